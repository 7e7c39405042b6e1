"""CPU tests of libmi_layer.so (include/mi_layer.h): every declared symbol is
exported, and bad calls are rejected before any launch; and what the torch side
refuses without a GPU."""
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
i32, i64, ptr, size = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t


def lib():
    L = ctypes.CDLL(os.path.join(ROOT, "flashinfer_amd", "libmi_layer.so"))
    L.mi_layer_last_error.restype = ctypes.c_char_p
    for n in ("mi_layer_balance_workspace_size", "mi_layer_int4_workspace_size"):
        getattr(L, n).restype = size
    return L


def test_exports_every_declared_symbol():
    src = open(os.path.join(ROOT, "include", "mi_layer.h")).read()
    names = sorted(set(re.findall(r"\b(mi_layer_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", src, flags=re.S))))
    assert names == ["mi_layer_balance", "mi_layer_balance_backward", "mi_layer_balance_workspace_size",
                     "mi_layer_int4_matmul", "mi_layer_int4_workspace_size", "mi_layer_last_error",
                     "mi_layer_pack_int4", "mi_layer_quantize_int4", "mi_layer_swiglu", "mi_layer_swiglu_backward"]
    L = lib()
    for name in names:
        assert hasattr(L, name), name


class Balance(ctypes.Structure):
    _fields_ = ([(n, ptr) for n in ("logits", "topk_ids", "seq_offsets", "mask", "loss", "counts", "weights")]
                + [(n, i64) for n in ("num_tokens", "num_seqs", "logits_stride")]
                + [(n, i32) for n in ("num_experts", "top_k", "dtype", "score")]
                + [("workspace", ptr), ("workspace_bytes", size)])


class Swiglu(ctypes.Structure):
    _fields_ = ([(n, ptr) for n in ("x", "grad", "out", "num_rows", "seed_ptr")] + [("seed", ctypes.c_uint64)]
                + [(n, i64) for n in ("max_rows", "I", "x_stride", "grad_stride", "out_stride")]
                + [(n, i32) for n in ("dtype", "threshold", "zero_rest", "reserved")])


class Int4(ctypes.Structure):
    _fields_ = ([(n, ptr) for n in ("x", "w", "scale", "bias", "out", "expert_offsets", "row_ids")]
                + [(n, i64) for n in ("x_rows", "rows", "N", "K", "x_stride", "out_stride")]
                + [(n, i32) for n in ("group_size", "num_experts", "x_dtype", "scale_dtype", "bias_dtype", "out_dtype",
                                      "zero_rest", "reserved")]
                + [("workspace", ptr), ("workspace_bytes", size)])


def refused(name, make, good, changes, *rest, code=1):
    L = lib()
    f = getattr(L, name)
    for change, word in changes:
        a = make(**dict(good, **change))
        rc = f(ctypes.byref(a), *rest)
        msg = L.mi_layer_last_error().decode()
        assert rc == code and word in msg and msg.startswith(name), (change, rc, msg)


@cpu_only
def test_balance_refuses():
    need = lib().mi_layer_balance_workspace_size(i64(100), i64(3), i32(16))
    assert need > 0
    good = dict(logits=P, topk_ids=P, seq_offsets=P, mask=P, loss=P, counts=P, weights=P, num_tokens=100, num_seqs=3,
                logits_stride=16, num_experts=16, top_k=2, dtype=1, score=0, workspace=P, workspace_bytes=need)
    both = [(dict(logits=None), "NULL"), (dict(weights=None), "NULL"), (dict(logits=P + 2), "misaligned"),
            (dict(seq_offsets=P + 1), "misaligned"), (dict(dtype=3), "dtype"), (dict(score=2), "score"),
            (dict(num_experts=0), "num_experts"), (dict(num_experts=1025), "num_experts"),
            (dict(num_tokens=-1), "num_tokens"), (dict(num_tokens=1 << 31), "num_tokens"), (dict(num_seqs=0), "num_seqs"),
            (dict(seq_offsets=None), "num_seqs"), (dict(logits_stride=-1), "stride")]
    refused("mi_layer_balance", Balance, good, both + [
        (dict(topk_ids=None), "NULL"), (dict(loss=None), "NULL"), (dict(counts=None), "NULL"),
        (dict(topk_ids=P + 2), "misaligned"), (dict(top_k=0), "top_k"), (dict(top_k=65), "top_k"), (dict(num_tokens=1 << 30), "num_tokens"),
        (dict(workspace=P + 16), "misaligned")], None)
    refused("mi_layer_balance", Balance, good, [(dict(workspace=None), "workspace"),
                                                (dict(workspace_bytes=need - 1), "workspace")], None, code=2)
    rest = ptr(P), ptr(P), i64(16), None
    refused("mi_layer_balance_backward", Balance, good, both, *rest)
    refused("mi_layer_balance_backward", Balance, good, [({}, "NULL")], None, ptr(P), i64(16), None)
    refused("mi_layer_balance_backward", Balance, good, [({}, "NULL")], ptr(P), None, i64(16), None)
    refused("mi_layer_balance_backward", Balance, good, [({}, "stride")], ptr(P), ptr(P), i64(15), None)
    refused("mi_layer_balance_backward", Balance, good, [({}, "misaligned")], ptr(P), ptr(P + 2), i64(16), None)


@cpu_only
def test_swiglu_refuses():
    good = dict(x=P, grad=P, out=P, max_rows=4, I=64, x_stride=128, grad_stride=64, out_stride=128, dtype=1)
    both = [(dict(x=None), "NULL"), (dict(out=None), "NULL"), (dict(x=P + 2), "misaligned"), (dict(out=P + 1), "misaligned"),
            (dict(num_rows=P + 2), "misaligned"), (dict(seed_ptr=P + 4), "misaligned"), (dict(dtype=5), "dtype"),
            (dict(max_rows=-1), "rows"), (dict(max_rows=1 << 31), "rows"), (dict(I=0), "row length"),
            (dict(I=1 << 28), "row length"), (dict(I=1 << 27, max_rows=1 << 15, out_stride=1 << 28), "row length"),
            (dict(threshold=-1), "threshold"), (dict(threshold=65536), "threshold"), (dict(x_stride=-1), "stride"),
            (dict(out_stride=63), "stride")]
    refused("mi_layer_swiglu", Swiglu, good, both, None)
    refused("mi_layer_swiglu_backward", Swiglu, good, both + [
        (dict(grad=None), "NULL"), (dict(grad=P + 2), "misaligned"), (dict(grad_stride=-1), "stride"),
        (dict(out_stride=127), "stride")], None)


@cpu_only
def test_int4_refuses():
    good = dict(x=P, w=P, scale=P, out=P, x_rows=4, rows=4, N=8, K=64, x_stride=64, out_stride=8, group_size=32)
    grouped = dict(good, num_experts=2, expert_offsets=P)
    refused("mi_layer_int4_matmul", Int4, good, [
        (dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(scale=None), "NULL"), (dict(out=None), "NULL"),
        (dict(x=P + 1), "misaligned"), (dict(w=P + 8), "misaligned"), (dict(scale=P + 4), "misaligned"),
        (dict(out=P + 1), "misaligned"), (dict(bias=P + 2, bias_dtype=1), "misaligned"), (dict(x_dtype=1), "dtype"),
        (dict(scale_dtype=2), "dtype"), (dict(out_dtype=3), "dtype"), (dict(bias=P, bias_dtype=3), "dtype"),
        (dict(K=0), "K 0"), (dict(K=(1 << 24) + 1), "K"), (dict(N=-1), "N"), (dict(group_size=16), "group_size"),
        (dict(group_size=96), "group_size"), (dict(num_experts=-1), "num_experts"), (dict(rows=5), "rows"),
        (dict(rows=-1, x_rows=-1), "size"), (dict(x_stride=-1), "stride"), (dict(out_stride=7), "stride"),
        (dict(row_ids=P), "grouped"), (dict(expert_offsets=P), "grouped"),
        (dict(N=1 << 24, rows=1 << 20, x_rows=1 << 20, out_stride=1 << 24), "too many")], None)
    refused("mi_layer_int4_matmul", Int4, grouped, [
        (dict(expert_offsets=None), "NULL"), (dict(bias=P), "bias"), (dict(num_experts=1025), "num_experts"),
        (dict(x_rows=0, row_ids=P), "no rows"), (dict(row_ids=P + 2), "misaligned")], None)
    need = lib().mi_layer_int4_workspace_size(i64(4), i64(63), i32(0))
    assert need == 4 * 64 * 2 and lib().mi_layer_int4_workspace_size(i64(4), i64(64), i32(1)) == 0
    for odd in (dict(K=63), dict(x=P + 2), dict(x_stride=66)):
        refused("mi_layer_int4_matmul", Int4, dict(good, **odd), [
            ({}, "workspace"), (dict(workspace=P, workspace_bytes=need - 1), "workspace")], None, code=2)
        refused("mi_layer_int4_matmul", Int4, dict(good, **odd), [
            (dict(workspace=P + 16, workspace_bytes=need), "misaligned")], None)


@cpu_only
def test_int4_weights_refuse():
    L = lib()
    for name, types, good, changes in (
            ("mi_layer_pack_int4", [ptr, i64, i64, ptr, i32, i64, i64, i64, i32, ptr, ptr, ptr],
             [P, 0, 64, P, 1, 0, 8, 64, 32, P, P, None],
             [(0, None, "NULL"), (3, None, "NULL"), (9, None, "NULL"), (10, None, "NULL"), (3, P + 2, "misaligned"),
              (9, P + 8, "misaligned"), (10, P + 4, "misaligned"), (1, -1, "stride"), (2, -1, "stride"), (4, 4, "dtype"),
              (5, 1025, "num_experts"), (6, 1 << 25, "N"), (7, 0, "K"), (8, 31, "group_size")]),
            ("mi_layer_quantize_int4", [i32, ptr, i64, i64, i64, i64, i64, i32, ptr, ptr, ptr],
             [1, P, 0, 64, 0, 8, 64, 32, P, P, None],
             [(0, 9, "dtype"), (1, None, "NULL"), (8, None, "NULL"), (9, None, "NULL"), (1, P + 2, "misaligned"),
              (2, -1, "stride"), (4, -1, "num_experts"), (6, 0, "K"), (7, 48, "group_size")])):
        f = getattr(L, name)
        f.argtypes = types
        for at, value, word in changes:
            args = list(good)
            args[at] = value
            rc, msg = f(*args), L.mi_layer_last_error().decode()
            assert rc == 1 and word in msg and msg.startswith(name), (at, value, rc, msg)


@cpu_only
def test_null_arguments():
    L = lib()
    for f in (L.mi_layer_balance, L.mi_layer_swiglu, L.mi_layer_swiglu_backward, L.mi_layer_int4_matmul):
        assert f(None, None) == 1 and b"NULL" in L.mi_layer_last_error()
    assert L.mi_layer_balance_backward(None, None, None, i64(1), None) == 1


def test_no_cpu_path():
    l, ids, x = torch.zeros(2, 4), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(16, 64, dtype=torch.int8), torch.ones(16, 2)
    w = fa.Int4Weights(torch.zeros(1, 1, 1024, dtype=torch.uint8), torch.ones(2, 16), 16, 64, 32)
    for f in (lambda: fa.balance_loss(l, ids), lambda: fa.swiglu(l), lambda: fa.pack_int4(q, s, 32),
              lambda: fa.quantize_int4(s), lambda: fa.int4_matmul(x, w)):
        with pytest.raises(ValueError, match="no CPU path"):
            f()
    for f in (lambda: fa.balance_loss(ids, ids), lambda: fa.balance_loss(l, l), lambda: fa.swiglu(ids),
              lambda: fa.pack_int4(s, s, 32), lambda: fa.quantize_int4(q), lambda: fa.int4_matmul(l, w)):
        with pytest.raises(TypeError):
            f()


def test_tangents_and_gradients_are_refused():
    import torch.autograd.forward_ad as fwd
    l, ids, x = torch.zeros(2, 4), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(16, 64, dtype=torch.int8), torch.ones(16, 2)
    w = fa.Int4Weights(torch.zeros(1, 1, 1024, dtype=torch.uint8), torch.ones(2, 16), 16, 64, 32)
    calls = [(l, lambda t: fa.balance_loss(t, ids)), (l, fa.swiglu), (torch.zeros(2, 2), lambda t: fa.swiglu(l, out=t)),
             (s, lambda t: fa.pack_int4(q, t, 32)), (s, fa.quantize_int4), (x, lambda t: fa.int4_matmul(t, w)),
             (w.scale, lambda t: fa.int4_matmul(x, w._replace(scale=t))),
             (torch.zeros(16), lambda t: fa.int4_matmul(x, w, bias=t)),
             (torch.zeros(2, 16), lambda t: fa.int4_matmul(x, w, out=t))]
    with fwd.dual_level():
        for n, (t, call) in enumerate(calls):
            dual = fwd.make_dual(t, torch.ones_like(t))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                    call(dual)
                    print("not refused:", n)
            with pytest.raises(ValueError, match="no CPU path"):
                call(dual.detach())
