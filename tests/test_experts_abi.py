"""CPU tests of libmi_experts.so (include/mi_experts.h): every declared symbol
is exported, and bad calls are rejected before any launch; and what the torch
side refuses without a GPU."""
import ctypes
import os
import re

import pytest
import torch

import flashinfer_amd as fa

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# made-up device addresses: only where no kernel could be launched on them
cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="passes fake device pointers; CPU-only session")
P = 1 << 20  # a 256-byte aligned address that is never read


def lib():
    L = ctypes.CDLL(os.path.join(ROOT, "flashinfer_amd", "libmi_experts.so"))
    L.mi_experts_last_error.restype = ctypes.c_char_p
    for n in ("mi_experts_sort_workspace_size", "mi_experts_int8_workspace_size"):
        getattr(L, n).restype = ctypes.c_size_t
    return L


def test_exports_every_declared_symbol():
    src = open(os.path.join(ROOT, "include", "mi_experts.h")).read()
    names = sorted(set(re.findall(r"\b(mi_experts_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", src, flags=re.S))))
    assert names == ["mi_experts_int8_matmul", "mi_experts_int8_workspace_size", "mi_experts_last_error",
                     "mi_experts_permute", "mi_experts_quantize_int8", "mi_experts_sort",
                     "mi_experts_sort_workspace_size", "mi_experts_unpermute", "mi_experts_unpermute_backward"]
    L = lib()
    for name in names:
        assert hasattr(L, name), name


i32, i64, ptr, size = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t


def call(name, types, args):
    L = lib()
    f = getattr(L, name)
    f.argtypes = types
    return f(*args), L.mi_experts_last_error().decode()


def refused(name, types, good, changes, code=1):
    for at, value, word in changes:
        args = list(good)
        args[at] = value
        rc, msg = call(name, types, args)
        assert rc == code and word in msg and msg.startswith(name), (at, value, rc, msg)


@cpu_only
def test_sort_refuses():
    types = [ptr, i64, i32, i32, i64, ptr, ptr, ptr, ptr, size, ptr]
    good = [P, 16, 8, 32, 0, P, P, P, None, 0, None]
    refused("mi_experts_sort", types, good, [
        (0, None, "NULL"), (5, None, "NULL"), (6, None, "NULL"), (7, None, "NULL"), (0, P + 2, "misaligned"),
        (1, -1, "num_tokens"), (1, (1 << 24) + 1, "num_tokens"), (2, 0, "top_k"), (2, 65, "top_k"),
        (3, 0, "num_experts"), (3, 1025, "num_experts")])
    large = list(good)
    large[1] = 1 << 20
    need = lib().mi_experts_sort_workspace_size(i64(8 << 20), i32(32))
    assert 0 < need <= 256 * 33 * 4
    refused("mi_experts_sort", types, large, [(8, None, "workspace")], code=2)
    large[8], large[9] = P, need - 1
    refused("mi_experts_sort", types, large, [(9, need - 1, "workspace")], code=2)


@cpu_only
def test_moves_refuse():
    types = [ptr, i64, i64, i32, i64, ptr, ptr, ptr, i64, i32, ptr]
    refused("mi_experts_permute", types, [P, 256, 16, 8, 256, P, P, P, 256, 1, None], [
        (0, None, "NULL"), (5, None, "NULL"), (6, None, "NULL"), (7, None, "NULL"), (5, P + 1, "misaligned"),
        (1, -4, "stride"), (8, 255, "stride"), (4, 0, "row length"), (4, (1 << 23) + 1, "row length"),
        (3, 65, "top_k"), (2, 1 << 40, "num_tokens")])
    types = [i32, ptr, i64, i64, i32, i64, ptr, ptr, ptr, ptr, i64, ptr]
    refused("mi_experts_unpermute", types, [0, P, 64, 16, 8, 64, P, P, P, P, 64, None], [
        (0, 3, "dtype"), (1, None, "NULL"), (1, P + 1, "misaligned"), (8, P + 2, "misaligned"), (9, None, "NULL"),
        (10, 63, "stride"), (2, -1, "stride"), (5, 0, "row length"), (5, 1 << 23, "row length"), (4, 0, "top_k")])
    types = [i32, ptr, i64, ptr, i64, i64, i32, i64, ptr, ptr, ptr, ptr, i64, i32, ptr, ptr]
    refused("mi_experts_unpermute_backward", types,
            [0, P, 64, P, 64, 16, 8, 64, P, P, P, P, 64, 1, P, None], [
                (0, -1, "dtype"), (1, None, "NULL"), (3, None, "NULL"), (8, None, "NULL"), (9, None, "NULL"),
                (12, 63, "stride"), (14, P + 2, "misaligned"), (7, 0, "row length"), (5, -1, "num_tokens")])


@cpu_only
def test_quantize_refuses():
    types = [i32, ptr, i64, i64, i64, i32, ptr, i32, ptr, i64, ptr, ptr]
    refused("mi_experts_quantize_int8", types, [1, P, 64, 16, 64, 0, None, 1, P, 64, P, None], [
        (0, 7, "dtype"), (1, None, "NULL"), (8, None, "NULL"), (10, None, "NULL"), (1, P + 2, "misaligned"),
        (9, 63, "stride"), (2, -1, "stride"), (4, 0, "row length"), (3, -1, "rows"), (3, 1 << 31, "rows")])


class Args(ctypes.Structure):
    _fields_ = ([(n, ptr) for n in ("a", "a_scale", "b", "b_scale", "bias", "out", "expert_offsets", "row_ids")]
                + [(n, i64) for n in ("a_rows", "rows", "N", "K", "a_stride", "b_stride", "b_expert_stride",
                                      "out_stride")]
                + [(n, i32) for n in ("num_experts", "out_dtype", "bias_dtype", "zero_rest")]
                + [("workspace", ptr), ("workspace_bytes", size)])


@cpu_only
def test_int8_matmul_refuses():
    good = dict(a=P, a_scale=P, b=P, b_scale=P, out=P, a_rows=4, rows=4, N=8, K=64, a_stride=64, b_stride=64,
                out_stride=8)
    grouped = dict(good, num_experts=2, expert_offsets=P, b_expert_stride=512)
    for base, change, word in [
            (good, dict(a=None), "NULL"), (good, dict(b=None), "NULL"), (good, dict(out=None), "NULL"),
            (good, dict(a_scale=None), "NULL"), (good, dict(b_scale=P + 1), "misaligned"), (good, dict(K=0), "K 0"),
            (good, dict(K=131072), "131072"), (good, dict(rows=5), "rows"), (good, dict(out_stride=7), "stride"),
            (good, dict(out_dtype=5), "dtype"), (good, dict(bias=P, bias_dtype=5), "dtype"),
            (good, dict(row_ids=P), "grouped"),
            (good, dict(expert_offsets=P), "grouped"), (good, dict(num_experts=-1), "num_experts"),
            (good, dict(N=1 << 29, rows=1 << 20, a_rows=1 << 20, out_stride=1 << 29), "too many"),
            (good, dict(a_rows=-1, rows=-1), "size"), (grouped, dict(expert_offsets=None), "NULL"),
            (grouped, dict(a_rows=0, row_ids=P), "no rows"), (grouped, dict(bias=P), "bias"), (grouped, dict(num_experts=1025), "num_experts")]:
        a = Args(**dict(base, **change))
        rc, msg = call("mi_experts_int8_matmul", [ctypes.POINTER(Args), ptr], [ctypes.byref(a), None])
        assert rc == 1 and word in msg, (change, rc, msg)
    # rows of no multiple of 16 bytes are copied from a size on
    copied = dict(good, a_rows=4096, rows=4096, N=4096, K=1025, a_stride=1025, b_stride=1025, out_stride=4096)
    need = lib().mi_experts_int8_workspace_size(i64(4096), i64(4096), i64(1025), i32(0))
    assert need == 8192 * 1040
    for workspace, nbytes, code, word in ((None, 0, 2, "workspace"), (P, need - 1, 2, "workspace"), (P + 16, need, 1, "misaligned")):
        a = Args(**dict(copied, workspace=workspace, workspace_bytes=nbytes))
        rc, msg = call("mi_experts_int8_matmul", [ctypes.POINTER(Args), ptr], [ctypes.byref(a), None])
        assert rc == code and word in msg, (workspace, rc, msg)
    assert lib().mi_experts_int8_workspace_size(i64(4096), i64(4096), i64(1024), i32(0)) == 0
    rc, msg = call("mi_experts_int8_matmul", [ctypes.POINTER(Args), ptr], [None, None])
    assert rc == 1 and "NULL" in msg


def test_no_cpu_path():
    ids = torch.zeros(2, 3, dtype=torch.int32)
    plan = fa.ExpertPlan(torch.zeros(5, dtype=torch.int32), torch.zeros(6, dtype=torch.int32), ids)
    x, q = torch.zeros(2, 16), torch.zeros(2, 16, dtype=torch.int8)
    s = torch.ones(2)
    for f in (lambda: fa.sort_experts(ids, 4), lambda: fa.permute(x, plan), lambda: fa.unpermute(x, plan),
              lambda: fa.quantize_int8(x), lambda: fa.swiglu_quantize_int8(x), lambda: fa.int8_matmul(q, s, q, s)):
        with pytest.raises(ValueError, match="no CPU path"):
            f()
    with pytest.raises(TypeError):
        fa.sort_experts(ids.float(), 4)
    with pytest.raises(TypeError):
        fa.int8_matmul(x, s, q, s)
    with pytest.raises(TypeError):
        fa.permute([1], plan)


def test_tangents_are_refused():
    """A dual tensor does not require a gradient, so its tangent would be lost
    without a word; one that autograd was told to leave alone may go on."""
    import torch.autograd.forward_ad as fwd
    ids = torch.zeros(2, 3, dtype=torch.int32)
    plan = fa.ExpertPlan(torch.zeros(5, dtype=torch.int32), torch.zeros(6, dtype=torch.int32), ids)
    x, rows, w = torch.zeros(2, 16), torch.zeros(6, 16), torch.zeros(2, 3)
    q, b, s = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(1, 2, 16, dtype=torch.int8), torch.ones(2)
    offs = torch.zeros(2, dtype=torch.int32)
    calls = [(x, lambda t: fa.permute(t, plan)), (rows, lambda t: fa.permute(x, plan, out=t)),
             (rows, lambda t: fa.unpermute(t, plan)), (w, lambda t: fa.unpermute(rows, plan, t)),
             (x, lambda t: fa.unpermute(rows, plan, out=t)), (x, fa.quantize_int8), (x, fa.swiglu_quantize_int8),
             (s, lambda t: fa.quantize_int8(x, scale=t)), (s, lambda t: fa.int8_matmul(q, t, q, s)),
             (s, lambda t: fa.int8_matmul(q, s, q, t)), (s, lambda t: fa.int8_matmul(q, s, q, s, bias=t)),
             (x, lambda t: fa.int8_matmul(q, s, q, s, out=t)),
             (s, lambda t: fa.int8_grouped_matmul(q, t, b, s[None], offs)),
             (s, lambda t: fa.int8_grouped_matmul(q, s, b, t[None], offs))]
    with fwd.dual_level():
        for n, (t, call) in enumerate(calls):
            dual = fwd.make_dual(t, torch.ones_like(t))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                    call(dual)
                    print("not refused:", n)
            with pytest.raises(ValueError, match="no CPU path"):
                call(dual.detach())
            with torch.inference_mode(), pytest.raises(ValueError, match="no CPU path"):
                call(dual)
