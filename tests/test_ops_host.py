"""The operators on caller tensors without a GPU: the header and its Python mirror, and what is refused
before anything is launched."""
import ctypes
import os
import re
import subprocess

import pytest

torch = pytest.importorskip("torch")

from redukt_amd import ffi, ops  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "redukt_ops.h")
BAD, OK = int(ffi.BackendResult.INVALID_ARGUMENT), int(ffi.BackendResult.OK)
P = 1 << 20        # an aligned address that no call may reach


@pytest.fixture(scope="module")
def lib():
    return ops._load()


def test_every_declared_operator_is_exported(lib):
    names = set(re.findall(r"\b(redukt_op_\w+)\s*\(", open(HEADER).read()))
    assert len(names) >= 5 and all(hasattr(lib, n) for n in names)


def test_the_structs_are_the_headers(tmp_path):
    structs = {"redukt_delta_rows": ops.DeltaRows, "redukt_quantize_rows": ops.QuantizeRows, "redukt_int8_matmul": ops.Int8Matmul}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "redukt_ops.h"', "int main(void) {"]
    want = []
    for name, cls in structs.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, f))
            want.append(getattr(cls, f).offset)
    src = tmp_path / "s.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    assert [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()] == want


def rows(**over):
    v = dict(dtype=0, rows=4, hk=2, hv=4, dk=64, dv=64, flags=0, scale=1.0, q=P, k=P, v=P, out=P, q_stride=128, k_stride=128,
             v_stride=256, out_stride=256, g=P, beta=P, g_stride=4, beta_stride=4)
    v.update(over)
    return ops.DeltaRows(**v)


BAD_ROWS = [dict(dtype=3), dict(hk=0), dict(hv=0), dict(hk=3), dict(hv=4100, hk=1), dict(dk=32), dict(dk=96), dict(dk=0), dict(dv=0),
            dict(dv=16), dict(dv=288), dict(flags=2), dict(rows=1 << 31), dict(q=None), dict(k=None), dict(v=None), dict(out=None),
            dict(g=None), dict(beta=None), dict(q=P + 8), dict(k=P + 2), dict(v=P + 4), dict(out=P + 8), dict(g=P + 2),
            dict(beta=P + 1), dict(q_stride=132), dict(k_stride=127), dict(v_stride=128), dict(out_stride=0), dict(out_stride=128),
            dict(q_stride=-128), dict(g_stride=-1),
            dict(q_stride=0), dict(v_stride=0), dict(k_stride=(1 << 22) + 8), dict(out_stride=1 << 30)]


@pytest.mark.parametrize("over", BAD_ROWS, ids=str)
def test_delta_rows_refused(lib, over):
    a = rows(**over)
    assert lib.redukt_op_delta_step(ctypes.byref(a), P, 8, P, None) == BAD
    assert lib.redukt_op_delta_chunk(ctypes.byref(a), P, 2, P, P, 8, P, P, 1 << 40, None) == BAD


def test_delta_step_refused(lib):
    a = ctypes.byref(rows())
    assert lib.redukt_op_delta_step(None, P, 8, P, None) == BAD
    assert lib.redukt_op_delta_step(a, None, 8, P, None) == BAD
    assert lib.redukt_op_delta_step(a, P + 4, 8, P, None) == BAD          # states unaligned
    assert lib.redukt_op_delta_step(a, P, 8, P + 2, None) == BAD          # slots unaligned
    assert lib.redukt_op_delta_step(a, P, 3, None, None) == BAD           # four entries, three slots
    assert lib.redukt_op_delta_step(a, P, 1 << 31, P, None) == BAD
    assert lib.redukt_op_delta_step(ctypes.byref(rows(rows=65537)), P, 1 << 20, P, None) == BAD
    assert lib.redukt_op_delta_step(ctypes.byref(rows(rows=0, q=None)), None, 0, None, None) == OK
    # sizes are right, but no device owns the address
    assert lib.redukt_op_delta_step(a, P, 8, P, None) == BAD


def test_delta_chunk_refused(lib):
    a = ctypes.byref(rows())
    big = 1 << 40
    call = lib.redukt_op_delta_chunk
    assert call(None, P, 2, P, P, 8, P, P, big, None) == BAD
    assert call(a, None, 2, P, P, 8, P, P, big, None) == BAD
    assert call(a, P + 2, 2, P, P, 8, P, P, big, None) == BAD
    assert call(a, P, 65537, P, P, 1 << 20, P, P, big, None) == BAD
    assert call(a, P, 2, P + 4, P, 8, P, P, big, None) == BAD
    assert call(a, P, 2, P, P + 8, 8, P, P, big, None) == BAD
    assert call(a, P, 2, P, P + 1024, 8, P, P, big, None) == BAD         # pools that overlap in part
    assert call(a, P, 9, P, P, 8, None, P, big, None) == BAD             # nine sequences, eight slots
    assert call(a, P, 2, None, None, 0, P, P, big, None) == BAD          # slots of no pool
    assert call(a, P, 0, None, None, 0, None, None, 0, None) == OK
    need = lib.redukt_op_delta_chunk_workspace(a, 2)
    if need:
        assert call(a, P, 2, P, P, 8, P, None, big, None) == BAD
        assert call(a, P, 2, P, P, 8, P, P + 4, big, None) == BAD
        assert call(a, P, 2, P, P, 8, P, P, need - 1, None) == BAD
    assert call(a, P, 2, P, P, 8, P, P, big, None) == BAD                # no device owns the address


def test_workspace_of_sizes_that_are_not_taken(lib):
    for over in BAD_ROWS[:12]:
        assert lib.redukt_op_delta_chunk_workspace(ctypes.byref(rows(**over)), 2) == 0
    assert lib.redukt_op_delta_chunk_workspace(None, 2) == 0
    assert lib.redukt_op_delta_chunk_workspace(ctypes.byref(rows()), 65537) == 0


def quantize_args(**over):
    v = dict(dtype=0, rows=4, cols=100, x=P, x_stride=100, codes=P, codes_stride=100, scales=P)
    v.update(over)
    return ctypes.byref(ops.QuantizeRows(**v))


def test_quantize_rows_refused(lib):
    call = lib.redukt_op_quantize_rows
    assert call(None, None) == BAD
    for over in (dict(dtype=3), dict(rows=1 << 31), dict(cols=1 << 31), dict(x=None), dict(codes=None), dict(scales=None), dict(x=P + 1),
                 dict(scales=P + 2), dict(x_stride=99), dict(codes_stride=99), dict(codes_stride=0), dict(x_stride=-100), {}):
        assert call(quantize_args(**over), None) == BAD, over
    assert call(quantize_args(rows=0, x=None), None) == OK


def matmul_args(**over):
    v = dict(dtype=0, m=4, n=6, k=100, x=P, x_stride=100, x_scales=P, w=P, w_stride=100, w_scales=P, bias=P, out=P, out_stride=6)
    v.update(over)
    return ctypes.byref(ops.Int8Matmul(**v))


def test_int8_matmul_refused(lib):
    call = lib.redukt_op_int8_matmul
    assert call(None, None) == BAD
    for over in (dict(dtype=3), dict(m=1 << 31), dict(n=1 << 31), dict(k=131001), dict(x=None), dict(w=None), dict(x_scales=None),
                 dict(w_scales=None), dict(out=None), dict(x_scales=P + 2), dict(w_scales=P + 1), dict(bias=P + 2), dict(out=P + 1),
                 dict(out_stride=5), dict(x_stride=99), dict(w_stride=99), dict(x_stride=-100), {}):
        assert call(matmul_args(**over), None) == BAD, over
    assert call(matmul_args(m=0, out=None), None) == OK
    assert call(matmul_args(n=0, out=None), None) == OK


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(2, 2, 64)
    g = torch.zeros(2, 2)
    pool = torch.zeros(2, 2, 64, 64)
    codes, s = torch.zeros(2, 16, dtype=torch.int8), torch.ones(2)
    for call in (lambda: ops.delta_step(x, x, x, g, g, pool), lambda: ops.delta_chunk(x, x, x, g, g, torch.zeros(2, dtype=torch.int32)),
                 lambda: ops.quantize_rows(x[0]), lambda: ops.int8_matmul(codes, s, codes, s), lambda: ops.quantize_rows(None),
                 lambda: ops.delta_chunk_workspace(1, 1, 1, 1, 64, 64, torch.int32)):
        with pytest.raises(ffi.BackendError) as e:
            call()
        assert e.value.result == ffi.BackendResult.INVALID_ARGUMENT


# ---------------------------------------------------------------- the Python layer on its own

class Recorded:
    """Stands for the library: what is called, with which arguments."""
    def __init__(self, lib):
        self.calls = []
        self.redukt_op_delta_chunk_workspace = lib.redukt_op_delta_chunk_workspace
        for name in ("delta_step", "delta_chunk", "quantize_rows", "int8_matmul"):
            setattr(self, "redukt_op_" + name, lambda *a: self.calls.append(a) or OK)


@pytest.fixture
def recorded(lib, monkeypatch):
    """The operators on CPU tensors, with nothing behind the checks of arguments."""
    r = Recorded(lib)
    monkeypatch.setattr(ops, "_device", lambda op, t: t.get_device() if isinstance(t, torch.Tensor) else ops._refuse(op))
    monkeypatch.setattr(ops, "_stream", lambda *a: None)
    monkeypatch.setattr(ops, "_load", lambda: r)
    return r


def refused(call):
    with pytest.raises(ffi.BackendError) as e:
        call()
    assert e.value.result == ffi.BackendResult.INVALID_ARGUMENT


def rule_tensors(T=3, hk=2, hv=4, dk=64, dv=64, dtype=torch.bfloat16):
    return (torch.zeros(T, hk, dk, dtype=dtype), torch.zeros(T, hk, dk, dtype=dtype), torch.zeros(T, hv, dv, dtype=dtype),
            torch.zeros(T, hv), torch.zeros(T, hv))


def test_a_workspace_that_is_not_one_block_is_refused(recorded):
    x, cu = rule_tensors(), torch.tensor([0, 3], dtype=torch.int32)
    need = ops.delta_chunk_workspace(3, 1, 2, 4, 64, 64, torch.bfloat16)
    assert need > 0
    refused(lambda: ops.delta_chunk(*x, cu, workspace=torch.zeros(1, dtype=torch.uint8).expand(need)))
    refused(lambda: ops.delta_chunk(*x, cu, workspace=torch.zeros(2 * need, dtype=torch.uint8)[::2]))
    assert not recorded.calls
    ops.delta_chunk(*x, cu, workspace=torch.zeros(2 * need, dtype=torch.uint8)[need:])
    assert len(recorded.calls) == 1


def pools_and_calls():
    """Each operator on tensors of its own: (floating-point inputs and outputs by name, a call of them)."""
    f32, bf16 = torch.float32, torch.bfloat16
    rows = dict(zip(("q", "k", "v", "g", "beta"), rule_tensors()), out=torch.zeros(3, 4, 64, dtype=bf16))
    cu = torch.tensor([0, 3], dtype=torch.int32)
    step = dict(rows, states=torch.zeros(3, 4, 64, 64))
    chunk = dict(rows, state_in=torch.zeros(1, 4, 64, 64), state_out=torch.zeros(1, 4, 64, 64))
    codes = torch.zeros(3, 16, dtype=torch.int8)
    return {"delta_step": (step, lambda t: ops.delta_step(**t)),
            "delta_chunk": (chunk, lambda t: ops.delta_chunk(cu_seqlens=cu, **t)),
            "quantize_rows": (dict(x=torch.zeros(3, 16), scales=torch.zeros(3)), lambda t: ops.quantize_rows(codes=codes, **t)),
            "int8_matmul": (dict(x_scales=torch.ones(3), w_scales=torch.ones(3), bias=torch.zeros(3), out=torch.zeros(3, 3, dtype=f32)),
                            lambda t: ops.int8_matmul(x=codes, w=codes, **t))}


TENSORS = [(op, name) for op, (t, _) in pools_and_calls().items() for name in t]


@pytest.mark.parametrize("op,name", TENSORS)
def test_every_tensor_that_asks_for_a_gradient_is_refused(recorded, op, name):
    tensors, call = pools_and_calls()[op]
    call(tensors)
    tensors[name].requires_grad_()
    refused(lambda: call(tensors))
    assert len(recorded.calls) == 1
    with torch.no_grad():
        call(tensors)
    assert len(recorded.calls) == 2


@pytest.mark.parametrize("op,name", TENSORS)
def test_every_tensor_with_a_tangent_is_refused(recorded, op, name):
    from torch.autograd import forward_ad

    tensors, call = pools_and_calls()[op]
    with forward_ad.dual_level():
        call(tensors)                                                     # (a level alone is nothing to refuse)
        dual = dict(tensors, **{name: forward_ad.make_dual(tensors[name], torch.ones_like(tensors[name]))})
        refused(lambda: call(dual))
    refused(lambda: torch.func.jvp(lambda t: call(dict(tensors, **{name: t})), (tensors[name],), (torch.ones_like(tensors[name]),)))
    assert len(recorded.calls) == 1


@pytest.mark.parametrize("op,written", [("delta_step", ["states", "out"]), ("delta_chunk", ["state_out", "out"]),
                                        ("quantize_rows", ["scales"]), ("int8_matmul", ["out"])])
def test_what_a_call_writes_is_counted_as_written(recorded, op, written):
    """A tensor that autograd has saved and a call overwrites is noticed by backward."""
    tensors, call = pools_and_calls()[op]
    before = {n: t._version for n, t in tensors.items()}
    call(tensors)
    for n, t in tensors.items():
        assert (t._version > before[n]) == (n in written), n
    w = torch.ones((), requires_grad=True)
    loss = (w * tensors[written[0]]).sum()
    call(tensors)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_codes_and_workspaces_are_counted_as_written(recorded):
    codes = torch.zeros(3, 16, dtype=torch.int8)
    ops.quantize_rows(torch.zeros(3, 16), codes=codes)
    work = torch.zeros(ops.delta_chunk_workspace(3, 1, 2, 4, 64, 64, torch.bfloat16), dtype=torch.uint8)
    ops.delta_chunk(*rule_tensors(), torch.tensor([0, 3], dtype=torch.int32), workspace=work)
    assert codes._version == 1 and work._version == 1


def test_tensors_of_inference_mode(recorded):
    """They keep no count of writes, and none is missed."""
    with torch.inference_mode():
        tensors, call = pools_and_calls()["delta_step"]
    with torch.no_grad():
        call(tensors)
    assert len(recorded.calls) == 1


# ---------------------------------------------------------------- sizes that do not fit the library's fields

BIG = 2 ** 32 + 5


def test_sizes_past_32_bits_are_refused(recorded):
    """They would arrive as what is left of them modulo 2^32.  (Tensors of stride 0: no memory is behind them.)"""
    byte, one = torch.zeros(1, 1, dtype=torch.int8), torch.ones(1)
    codes, scales = byte.expand(BIG, 1), one.expand(BIG)
    for rows, cols in ((BIG, 1), (1, BIG), (2 ** 31, 1)):
        refused(lambda: ops.quantize_rows(torch.zeros(1, 1).expand(rows, cols), codes=byte.expand(rows, cols)))
    refused(lambda: ops.int8_matmul(codes, scales, byte, one, out=torch.zeros(1, 1).expand(BIG, 1)))
    refused(lambda: ops.int8_matmul(byte, one, codes, scales, out=torch.zeros(1, 1).expand(1, BIG)))
    refused(lambda: ops.int8_matmul(byte.expand(1, BIG), one, byte.expand(1, BIG), one))
    x = [t[:1].expand(BIG, *t.shape[1:]) for t in rule_tensors(1, 1, 1, 64, 32)]
    refused(lambda: ops.delta_step(*x, torch.zeros(1, 1, 64, 32), out=x[2]))
    refused(lambda: ops.delta_chunk(*x, torch.zeros(2, dtype=torch.int32), out=x[2]))
    assert not recorded.calls


def test_sizes_of_a_workspace_past_32_bits_are_refused(lib):
    sizes = (100, 2, 2, 4, 64, 64)
    assert ops.delta_chunk_workspace(*sizes, torch.bfloat16) > 0
    for i, size in enumerate(sizes):
        for wrong in (size + 2 ** 32, size - 2 ** 32, -1, 2 ** 31):
            refused(lambda: ops.delta_chunk_workspace(*sizes[:i], wrong, *sizes[i + 1:], torch.bfloat16))


@pytest.mark.parametrize("op,name", TENSORS)
def test_what_is_no_tensor_is_refused(recorded, op, name):
    tensors, call = pools_and_calls()[op]
    refused(lambda: call(dict(tensors, **{name: 5})))
    assert not recorded.calls
