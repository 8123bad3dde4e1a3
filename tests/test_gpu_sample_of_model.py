"""A loaded model's tokens drawn on the device: forward_batch_device and ops.sample on the library's stream, a step after
the other without the host, against host logits and the statement in 64 bits of tests/more_ops_f64.py."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from redukt_amd import ffi, ops, rbin, synth  # noqa: E402
from tests import more_ops_f64 as f64  # noqa: E402

pytestmark = pytest.mark.gpu

SETTINGS = [dict(temperature=0.8, top_k=50, top_p=0.95), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=0.0)]


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "-".join(s))
def test_generating_on_the_device(tmp_path, settings):
    n, steps = 4, 6
    path = str(tmp_path / "m.rbin")
    dims = rbin.MambaDims(vocab=1000, d_model=96, n_layer=3)
    synth.write_synthetic_mamba(path, dims, seed=5)
    u = torch.rand(steps, n, generator=torch.Generator().manual_seed(3))
    first = [3, 141, 59, 265]
    with ffi.PluginBackend(path, profile=2) as be:
        be.batch_init(2 * n)
        slots = torch.arange(n, 2 * n, dtype=torch.int32, device="cuda")
        tokens, d_u = torch.tensor(first, dtype=torch.int32, device="cuda"), u.cuda()
        drawn = torch.empty(steps, n, dtype=torch.int32, device="cuda")
        logits = torch.empty(n, be.vocab, device="cuda")
        torch.cuda.synchronize()            # (from here on everything is ordered by the library's stream)
        for t in range(steps):
            be.forward_batch_device(n, slots.data_ptr(), tokens.data_ptr() if t == 0 else drawn[t - 1].data_ptr(), logits.data_ptr())
            ops.sample(logits, d_u[t], out=drawn[t], stream=be.stream(), **settings)
        assert be.device_status() == ffi.BackendResult.OK        # (waits)
        now, host = first, np.empty((n, be.vocab), np.float32)
        for t in range(steps):
            be.forward_batch(list(range(n)), now, host)
            now = [f64.draw(host[i], u[t, i].item(), **settings) for i in range(n)]
            assert drawn[t].tolist() == now, t
