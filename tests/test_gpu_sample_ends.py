"""sample at temperatures next to the ends of f32, on the GPU, against the statement in 64 bits of tests/more_ops_f64.py."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_sample import same, uniform  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [300, 5001, 40000])
def test_sample_temperatures_next_to_the_ends_of_f32(vocab):
    """Logits whose differences pass f32's range and temperatures as large; logits and temperatures below 2^-126."""
    r = np.random.default_rng(vocab)
    for scale, temperatures in ((3.4e38, [1e38, 3e38, 2.4e37, 2e37, 1e37]), (1e-37, [1e-38, 3e-38, 2e-37]), (3e-44, [1.4e-45, 1e-44, 1e-40])):
        x = torch.from_numpy(((2 * r.random((len(temperatures), vocab)) - 1) * scale).astype(np.float32)).cuda()
        t = torch.tensor(temperatures, device="cuda")
        for i, s in enumerate([{}, dict(top_k=5), dict(top_k=200), dict(top_k=vocab - 3), dict(top_p=0.7), dict(min_p=0.3), dict(top_k=100, top_p=0.5, min_p=0.1)]):
            for seed in range(4):
                same(x, uniform(len(temperatures), seed=10 * i + seed), temperature=t, **s)
