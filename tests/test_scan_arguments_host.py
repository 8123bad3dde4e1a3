"""ops.scan's checks of its arguments and scan_chunk's workspace, without a GPU."""
import itertools
import random

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


@pytest.mark.parametrize("n,piece", [(8, 64), (16, 64), (32, 32), (64, 32)])
def test_the_workspace_grows_with_the_rows_and_not_with_sequences_that_need_none(n, piece):
    """Two places (a state and a sum of each channel) for each piece that the rows make, at most."""
    for rows, seqs in ((65536, 65536), (65536, 20), (20011, 37), (70000, 65536), (piece + 1, 2), (piece + 1, 65536)):
        size = ops.scan_chunk_workspace(rows, seqs, 1536, 1, n)
        assert 0 < size <= min(2 * rows // piece, rows // piece + seqs) * 1536 * (n + 1) * 4, (rows, seqs)
    assert ops.scan_chunk_workspace(piece, 65536, 1536, 1, n) == 0


def test_places_of_pieces_do_not_meet():
    """The two ways that pieces get places in the workspace, as the kernels have them: for sequences of more than one piece, those of each are
    apart from all others' and within the workspace; over all short lengths, and random ones."""
    r = random.Random(1)
    P = 4
    cases = [(start, c) for start in range(P) for c in itertools.product(range(11), repeat=3)]
    cases += [(r.randrange(9), [r.choice([0, 1, 2, P, P + 1, 2 * P, 2 * P + 1, r.randrange(40)]) for _ in range(r.randrange(1, 30))]) for _ in range(3000)]
    for start, lens in cases:
        rows = start + sum(lens)
        for spread in (False, True):
            at, end = start, 0
            for i, n in enumerate(lens):
                first, count = 2 * at // P if spread else at // P + i, -(-n // P)
                if count > 1:
                    assert first >= end, (start, lens, i, spread)
                    end = first + count
                at += n
            assert end <= (2 * rows // P if spread else rows // P + len(lens)), (start, lens, spread)
