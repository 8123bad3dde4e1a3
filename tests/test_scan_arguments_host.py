"""ops.scan's checks of its arguments, without a GPU."""
import pytest

torch = pytest.importorskip("torch")

from redukt_amd import ops  # noqa: E402
from tests.test_more_ops_host import F32, layer, lib, recorded, refused  # noqa: E402,F401


@pytest.mark.parametrize("name", [*layer(), "state_in", "cu_seqlens"])
def test_what_is_no_tensor_or_of_another_type_is_refused(recorded, name):  # noqa: F811
    t = dict(layer(dtype=F32), state_in=torch.zeros(1, 64, 16), cu_seqlens=torch.tensor([0, 3], dtype=torch.int32))
    ops.scan(**t)
    assert len(recorded.calls) == 1
    for wrong in (5, "x", t[name].to(torch.float64), t[name][None], t[name].tolist()):
        refused(lambda: ops.scan(**dict(t, **{name: wrong})))
    if name in ("x", "dt", "a", "b", "c", "cu_seqlens"):
        refused(lambda: ops.scan(**dict(t, **{name: None})))
    assert len(recorded.calls) == 1
