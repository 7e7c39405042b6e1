"""sort_experts, permute and unpermute (flashinfer_amd.experts) against plain
64-bit formulas: tables and moved rows exactly, sums within the bounds that
fp32 sums and one rounding of the result give."""
import pytest
import torch

import flashinfer_amd as fa
from flashinfer_amd import kernel

pytestmark = pytest.mark.gpu
F64 = torch.float64
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24  # half a step of fp32, relative


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def ids_of(T, k, G, seed, repeats=False):
    g = torch.Generator().manual_seed(seed)
    if repeats:  # an expert may come twice; ids that no shard has, too
        return torch.randint(-2, G + 2, (T, k), generator=g, dtype=torch.int32)
    return torch.rand(T, G, generator=g).argsort(dim=1)[:, :k].to(torch.int32)


def plan_of(ids, E, offset):
    """The tables by Python's stable sort, on the CPU."""
    T, k = ids.shape
    flat = [int(i) - offset for i in ids.reshape(-1)]
    key = [b if 0 <= b < E else E for b in flat]
    order = sorted(range(T * k), key=lambda s: key[s])
    row = [0] * (T * k)
    for p, s in enumerate(order):
        row[s] = p
    counts = [0] * (E + 1)
    for b in key:
        counts[b] += 1
    offs = [0]
    for c in counts[:E]:
        offs.append(offs[-1] + c)
    i32 = torch.int32
    return (torch.tensor(offs, dtype=i32), torch.tensor([s // k for s in order], dtype=i32),
            torch.tensor(row, dtype=i32).view(T, k))


SORTS = [  # T, k, G, E, offset
    (0, 8, 8, 8, 0), (1, 1, 1, 1, 0), (1, 8, 256, 256, 0), (1, 8, 256, 32, 224), (7, 3, 16, 16, 0),
    (64, 8, 256, 32, 64), (65, 1, 5, 5, 0), (333, 6, 128, 16, 16), (1000, 8, 256, 256, 0),
    (1024, 8, 64, 8, 8), (512, 8, 1024, 1024, 0), (513, 8, 1024, 1024, 0), (1025, 8, 1024, 1024, 0), (5000, 7, 256, 255, 1), (3001, 64, 1024, 1000, 3),
    (70000, 8, 256, 32, 32), (1500, 2, 64, 64, 0), (3001, 1, 64, 8, 8), (1281, 8, 256, 256, 0), (4097, 8, 1024, 1024, 0)]


@pytest.mark.parametrize("case", SORTS, ids=str)
@pytest.mark.parametrize("repeats", [False, True])
def test_sort_tables(case, repeats):
    T, k, G, E, offset = case
    ids = ids_of(T, k, G, T + k, repeats)
    plan = fa.sort_experts(ids.cuda(), E, offset)
    for got, want, name in zip(plan, plan_of(ids, E, offset), plan._fields):
        assert torch.equal(got.cpu(), want), name
    again = fa.sort_experts(ids.cuda(), E, offset)
    assert all(torch.equal(a, b) for a, b in zip(plan, again))


def test_sort_of_one_expert_and_of_none():
    ids = torch.full((2000, 8), 3, dtype=torch.int32, device="cuda")
    for E, offset, S in ((8, 0, 16000), (2, 4, 0), (1, 3, 16000), (4, -(1 << 62), 0)):
        plan = fa.sort_experts(ids, E, offset)
        assert int(plan.expert_offsets[-1]) == S
        # one bucket holds everything: slots keep their order
        assert torch.equal(plan.row_of_slot.view(-1).cpu(), torch.arange(16000, dtype=torch.int32))


def test_sort_takes_routes_and_strided_ids():
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn(300, 256, generator=g, device="cuda")
    ids, w = kernel.route(logits, torch.zeros(256, device="cuda"), 2.5)
    plan = fa.sort_experts(ids, 32, 64)
    offs, tok, sw, _ = kernel.sort(ids, w, 64)
    S = int(offs[-1])
    assert torch.equal(plan.expert_offsets, offs) and torch.equal(plan.token_of_row[:S], tok)
    assert torch.equal(w.view(-1)[torch.argsort(plan.row_of_slot.view(-1))][:S], sw)
    wide = torch.stack([ids, ids + 1], dim=2).flatten(1)[:, ::2]  # every other column
    assert not wide.is_contiguous()
    assert all(torch.equal(a, b) for a, b in zip(plan, fa.sort_experts(wide, 32, 64)))


# T, k, G, E, offset, H
MOVES = [(1, 8, 256, 256, 0, 7168), (1, 1, 4, 4, 0, 1), (3, 2, 8, 4, 4, 7), (17, 8, 64, 64, 0, 130),
         (64, 6, 128, 16, 32, 4096), (129, 8, 256, 32, 0, 1000), (40, 20, 64, 16, 8, 264),
         (5, 3, 8, 8, 0, 9001), (300, 8, 256, 256, 0, 2048), (2, 64, 256, 256, 0, 64), (31, 4, 8, 2, 100, 96)]


def _rand(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _rounded(ref, other, dtype):
    """Bound of |got - ref|: `other`, the error before the last rounding, and that rounding."""
    eps = torch.finfo(dtype).eps / 2
    return other * (1 + eps) + ref.abs() * eps + torch.finfo(dtype).smallest_normal * eps * 2


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", MOVES, ids=str)
def test_permute_and_gradient(case, dtype):
    T, k, G, E, offset, H = case
    ids = ids_of(T, k, G, 5).cuda()
    plan = fa.sort_experts(ids, E, offset)
    S, row = int(plan.expert_offsets[-1]), plan.row_of_slot.long()
    x = _rand((T, H), dtype, 1).requires_grad_()
    rows = fa.permute(x, plan)
    want = torch.zeros(T * k, H, dtype=dtype, device="cuda")
    want[:S] = x.detach()[plan.token_of_row[:S].long()]
    assert torch.equal(rows, want)
    # a buffer: the rows behind the local ones stay
    buf = torch.full_like(want, 7.0)
    with torch.no_grad():
        assert fa.permute(x, plan, out=buf).data_ptr() == buf.data_ptr()
    assert torch.equal(buf[:S], want[:S]) and bool((buf[S:] == 7.0).all())
    grad = _rand((T * k, H), dtype, 2)
    grad[S:] = float("nan")  # rows of other shards are not read
    (dx,) = torch.autograd.grad(rows, x, grad)
    mine = torch.where((row < S)[:, :, None], grad.to(F64)[row], 0.0)
    ref = mine.sum(dim=1)
    assert dx.dtype == dtype
    assert bool(((dx.to(F64) - ref).abs() <= _rounded(ref, (k - 1) * U * mine.abs().sum(dim=1), dtype)).all())


@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", MOVES, ids=str)
def test_unpermute_and_gradients(case, dtype, weighted):
    T, k, G, E, offset, H = case
    ids = ids_of(T, k, G, 6).cuda()
    plan = fa.sort_experts(ids, E, offset)
    S, row = int(plan.expert_offsets[-1]), plan.row_of_slot.long()
    rows = _rand((T * k, H), dtype, 3)
    rows[S:] = float("nan")  # not read
    rows.requires_grad_()
    w = _rand((T, k), torch.float32, 4).requires_grad_() if weighted else None
    local = row < S
    w64 = torch.where(local, w.detach().to(F64) if weighted else torch.ones(T, k, dtype=F64, device="cuda"), 0.0)
    mine = torch.where(local[:, :, None], rows.detach().to(F64)[row], 0.0)
    terms = mine * w64[:, :, None]
    ref = terms.sum(dim=1)
    y = fa.unpermute(rows, plan, w)
    assert y.dtype == dtype
    bound = _rounded(ref, k * U * terms.abs().sum(dim=1), dtype)
    assert bool(((y.to(F64) - ref).abs() <= bound).all())
    buf = torch.full_like(y, 3.0)
    with torch.no_grad():
        fa.unpermute(rows, plan, w, out=buf)
    assert torch.equal(buf, y)
    grad = _rand((T, H), dtype, 5)
    got = torch.autograd.grad(y, (rows, w) if weighted else (rows,), grad)
    ref = torch.zeros(T * k, H, dtype=F64, device="cuda")
    ref[row.view(-1)] = (w64[:, :, None] * grad.to(F64)[:, None, :]).view(T * k, H)
    assert bool(((got[0].to(F64) - ref).abs() <= _rounded(ref, ref.abs() * U, dtype)).all())
    assert bool((got[0][S:] == 0).all())
    if weighted:
        terms = mine * grad.to(F64)[:, None, :]
        # H products summed in fp32 in some order
        assert bool(((got[1].to(F64) - terms.sum(dim=2)).abs() <= (H + 1) * U * terms.abs().sum(dim=2)).all())
        (only,) = torch.autograd.grad(fa.unpermute(rows.detach(), plan, w), w, grad)
        assert torch.equal(only, got[1])
        (only,) = torch.autograd.grad(fa.unpermute(rows, plan, w.detach()), rows, grad)
        assert torch.equal(only, got[0])


def test_gradients_by_differences():
    """Directional derivatives of a loss through permute, a product and unpermute."""
    T, k, E, H = 13, 3, 6, 24
    plan = fa.sort_experts(ids_of(T, k, E + 2, 9).cuda(), E, 1)
    x, w = _rand((T, H), torch.float32, 1), torch.softmax(_rand((T, k), torch.float32, 2), 1)
    m = _rand((H, H), torch.float32, 3) / H ** 0.5
    c = _rand((T, H), torch.float32, 4)

    def loss(x, w):
        return (fa.unpermute(torch.tanh(fa.permute(x, plan) @ m), plan, w) * c).to(F64).sum()

    x.requires_grad_(), w.requires_grad_()
    gx, gw = torch.autograd.grad(loss(x, w), (x, w))
    for seed in (5, 6):
        dx, dw = _rand((T, H), torch.float32, seed), _rand((T, k), torch.float32, seed + 10)
        h = 2.0 ** -7
        with torch.no_grad():
            by_diff = float((loss(x + h * dx, w + h * dw) - loss(x - h * dx, w - h * dw)) / (2 * h))
        got = float((gx.to(F64) * dx).sum() + (gw.to(F64) * dw).sum())
        # third derivatives times h^2 / 6, and fp32 differences over 2h, of sums of ~300 terms
        assert abs(got - by_diff) <= 1e-2 * max(1.0, abs(by_diff)), (got, by_diff)


def test_rows_that_are_not_dense():
    plan = fa.sort_experts(ids_of(50, 4, 8, 1).cuda(), 8)
    base = _rand((50, 300), torch.bfloat16, 1)
    dense = fa.permute(base[:, 8:136].contiguous(), plan)
    for x in (base[:, 8:136], base[:, 9:137], base.t().contiguous().t()[:, 8:136], base[:, 8:264:2]):
        assert torch.equal(fa.permute(x, plan), fa.permute(x.contiguous(), plan))
    assert torch.equal(fa.permute(base[:, 8:136], plan), dense)
    one = base[:1, :128].expand(50, 128)  # one row for all tokens
    assert torch.equal(fa.permute(one, plan), one.contiguous()[plan.token_of_row.long()])
    out = torch.zeros(200, 256, dtype=torch.bfloat16, device="cuda")
    fa.permute(base[:, 8:136], plan, out=out[:, 64:192])
    assert torch.equal(out[:, 64:192], dense) and not out[:, :64].any() and not out[:, 192:].any()
    y = fa.unpermute(dense, plan)
    wide = torch.zeros(200, 131, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:] = dense
    assert torch.equal(fa.unpermute(wide[:, 3:], plan), y)
    # broadcast gradients (stride 0), as sum().backward() makes them
    x = base[:, :128].contiguous().requires_grad_()
    (g,) = torch.autograd.grad(fa.permute(x, plan).sum(), x)
    assert bool((g == 4).all())
    rows = dense.clone().requires_grad_()
    w = torch.rand(50, 4, device="cuda").t().contiguous().t().requires_grad_()
    gr, gw = torch.autograd.grad(fa.unpermute(rows, plan, w).sum(), (rows, w))
    ref = dense.to(F64).sum(1)[plan.row_of_slot.long()]
    assert bool(((gw.to(F64) - ref).abs() <= 129 * U * dense.to(F64).abs().sum(1)[plan.row_of_slot.long()]).all())
    assert torch.equal(gr[:, 0], w.detach().reshape(-1)[torch.argsort(plan.row_of_slot.view(-1))].bfloat16())


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn, torch.int32, torch.float64, torch.bool])
def test_permute_other_types(dtype):
    plan = fa.sort_experts(ids_of(20, 4, 8, 2).cuda(), 4, 2)
    x = (torch.rand(20, 33, device="cuda") * 8 - 4).to(dtype)
    S = int(plan.expert_offsets[-1])
    rows = fa.permute(x, plan)
    as_bytes = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    assert torch.equal(as_bytes(rows[:S]), as_bytes(x)[plan.token_of_row[:S].long()].view(S, -1))
    assert not as_bytes(rows[S:]).any()


def test_nonfinite_rows_reach_their_tokens_only():
    plan = fa.sort_experts(torch.tensor([[0, 1], [2, 1], [2, 3]], dtype=torch.int32, device="cuda"), 3)
    rows = torch.ones(6, 16, device="cuda")
    rows[int(plan.row_of_slot[0, 0])] = float("inf")
    rows[int(plan.row_of_slot[2, 1])] = float("nan")  # expert 3 is not local
    y = fa.unpermute(rows, plan, torch.full((3, 2), 0.5, device="cuda"))
    assert bool(torch.isinf(y[0]).all()) and bool((y[1] == 1).all()) and bool((y[2] == 0.5).all())


def test_offsets_past_32_bits():
    """More than 2^31 elements of rows: the last rows are where they belong."""
    T, k, H = 40000, 8, 7168
    ids = (torch.arange(T * k, device="cuda", dtype=torch.int32) % 16).view(T, k)
    plan = fa.sort_experts(ids, 16)
    x = torch.randint(-8, 8, (T, H), device="cuda", dtype=torch.int8).to(torch.bfloat16)
    rows = fa.permute(x, plan)
    at = torch.randint(T * k - 5000, T * k, (500,), device="cuda")
    assert torch.equal(rows[at], x[plan.token_of_row[at].long()])
    y = fa.unpermute(rows, plan)  # sums of small whole numbers: exact
    assert torch.equal(y, x * k)


def test_graph_replays_and_streams():
    """sort, permute and unpermute captured together: every replay equals the
    eager result of its inputs; two graphs replayed in turn keep apart."""
    T, k, E, H = 1500, 8, 32, 512  # sorted with a workspace
    made = []
    for seed in (1, 2):
        ids, x = ids_of(T, k, 64, seed).cuda(), _rand((T, H), torch.bfloat16, seed)
        w = torch.rand(T, k, device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fa.unpermute(fa.permute(x, fa.sort_experts(ids, E, 16)), fa.sort_experts(ids, E, 16), w)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan = fa.sort_experts(ids, E, 16)
            rows = fa.permute(x, plan)
            y = fa.unpermute(rows, plan, w)
        made.append((graph, ids, x, w, plan, rows, y))
    for rep in range(3):
        for n, (graph, ids, x, w, plan, rows, y) in enumerate(made):
            ids.copy_(ids_of(T, k, 64, 10 * rep + n))
            x.copy_(_rand((T, H), torch.bfloat16, 10 * rep + n + 5))
        for graph, *_ in made:
            graph.replay()
        torch.cuda.synchronize()
        for graph, ids, x, w, plan, rows, y in made:
            p = fa.sort_experts(ids, E, 16)
            assert all(torch.equal(a, b) for a, b in zip(p, plan))
            r = fa.permute(x, p)
            assert torch.equal(r, rows) and torch.equal(fa.unpermute(r, p, w), y)


def test_captured_backward_on_leaves_of_its_own():
    T, k, E, H = 33, 4, 8, 256
    plan = fa.sort_experts(ids_of(T, k, E, 1).cuda(), E)
    x = _rand((T, H), torch.float32, 1).requires_grad_()
    w = torch.rand(T, k, device="cuda").requires_grad_()
    g = _rand((T, H), torch.float32, 2)

    def step():
        return torch.autograd.grad(fa.unpermute(fa.permute(x, plan), plan, w), (x, w), g)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for rep in range(3):
        with torch.no_grad():
            x.copy_(_rand((T, H), torch.float32, 7 + rep))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_refusals():
    plan = fa.sort_experts(ids_of(6, 2, 4, 1).cuda(), 4)
    x = torch.zeros(6, 16, device="cuda", dtype=torch.bfloat16)
    rows = torch.zeros(12, 16, device="cuda", dtype=torch.bfloat16)
    leaf = x.clone().requires_grad_()
    bad = [
        (ValueError, lambda: fa.permute(x[:5], plan)),
        (ValueError, lambda: fa.permute(x[0], plan)),
        (ValueError, lambda: fa.permute(x.cpu(), plan)),
        (ValueError, lambda: fa.permute(x[:, :0], plan)),
        (ValueError, lambda: fa.permute(x, fa.ExpertPlan(*(t.cpu() for t in plan)))),
        (TypeError, lambda: fa.permute(x, plan._replace(row_of_slot=plan.row_of_slot.long()))),
        (ValueError, lambda: fa.permute(x, plan, out=rows[:11])),
        (TypeError, lambda: fa.permute(x, plan, out=rows.float())),
        (ValueError, lambda: fa.permute(x, plan, out=rows[:1].expand(12, 16))),
        (ValueError, lambda: fa.permute(rows[:6], plan, out=rows)),
        (ValueError, lambda: fa.unpermute(rows, plan, out=rows[6:])),
        (ValueError, lambda: fa.permute(leaf, plan, out=rows)),
        (TypeError, lambda: fa.permute(x.double().requires_grad_(), plan)),
        (TypeError, lambda: fa.unpermute(rows.double(), plan)),
        (ValueError, lambda: fa.unpermute(rows[:11], plan)),
        (TypeError, lambda: fa.unpermute(rows, plan, torch.zeros(6, 2, device="cuda", dtype=torch.bfloat16))),
        (ValueError, lambda: fa.unpermute(rows, plan, torch.zeros(2, 6, device="cuda"))),
        (ValueError, lambda: fa.unpermute(rows.requires_grad_(), plan, out=x)),
        (TypeError, lambda: fa.sort_experts(torch.zeros(2, 2, device="cuda"), 4)),
        (ValueError, lambda: fa.sort_experts(torch.zeros(4, device="cuda", dtype=torch.int32), 4)),
        (ValueError, lambda: fa.sort_experts(torch.zeros(4, 65, device="cuda", dtype=torch.int32), 4)),
        (ValueError, lambda: fa.sort_experts(torch.zeros(4, 2, device="cuda", dtype=torch.int32), 0)),
        (ValueError, lambda: fa.sort_experts(torch.zeros(4, 2, device="cuda", dtype=torch.int32), 1025)),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    y = fa.permute(leaf, plan)
    g = torch.ones_like(y).requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, leaf, g, create_graph=True)


def test_long_rows():
    """Rows of 8 MB in single bytes: more column chunks than a launch takes with many tokens."""
    T, H = 600, 1 << 23
    x = torch.zeros(1, H, dtype=torch.uint8, device="cuda").random_(0, 256)
    plan = fa.sort_experts(torch.zeros(T, 1, dtype=torch.int32, device="cuda"), 1)
    out = torch.zeros(T, H + 1, dtype=torch.uint8, device="cuda")
    fa.permute(x.expand(T, H), plan, out=out[:, 1:])
    assert torch.equal(out[0, 1:], x[0]) and torch.equal(out[T // 2, 1:], x[0]) and torch.equal(out[-1, 1:], x[0])
    assert not out[:, 0].any()


def test_no_tokens():
    plan = fa.sort_experts(torch.zeros(0, 4, dtype=torch.int32, device="cuda"), 8)
    assert plan.expert_offsets.tolist() == [0] * 9 and plan.token_of_row.shape == (0,)
    x = torch.zeros(0, 64, device="cuda").requires_grad_()
    rows = fa.permute(x, plan)
    assert rows.shape == (0, 64)
    w = torch.zeros(0, 4, device="cuda").requires_grad_()
    y = fa.unpermute(rows, plan, w)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert gx.shape == (0, 64) and gw.shape == (0, 4)


def test_gradients_with_tangents_are_refused():
    """Forward over backward: a gradient's tangent would be lost on its way to the leaves."""
    import torch.autograd.forward_ad as fwd
    plan = fa.sort_experts(ids_of(6, 2, 4, 1).cuda(), 4)
    x, rows = torch.ones(6, 16, device="cuda", requires_grad=True), torch.ones(12, 16, device="cuda", requires_grad=True)
    w = torch.ones(6, 2, device="cuda", requires_grad=True)
    for y, leaves in ((fa.permute(x, plan), (x,)), (fa.unpermute(rows, plan, w), (rows, w))):
        g = torch.ones_like(y)
        with fwd.dual_level():
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(y, leaves, fwd.make_dual(g, g), retain_graph=True)
            with pytest.raises(ValueError, match="forward-mode"):
                fa.permute(fwd.make_dual(x, torch.ones_like(x)), plan)
        assert all(bool((t == 2 if t is x else t >= 1).all()) for t in torch.autograd.grad(y, leaves, g))


def test_negated_views():
    """The imaginary part of a conjugate is a view whose sign is changed only when it is read; so may a gradient be."""
    plan = fa.sort_experts(ids_of(5, 2, 4, 1).cuda(), 4)
    row = plan.token_of_row.long()
    for H in (1, 24):
        z = torch.complex(_rand((5, H), torch.float32, 1), _rand((5, H), torch.float32, 2)).conj()
        x = z.imag
        assert x.is_neg() and torch.equal(fa.permute(x, plan), x.resolve_neg()[row])
        rows, w = fa.permute(x.resolve_neg(), plan), torch.complex(torch.ones(5, 2), torch.full((5, 2), 0.5)).cuda().conj().imag
        y = fa.unpermute(rows, plan, w)
        assert torch.equal(y, -fa.unpermute(rows, plan, -w.resolve_neg())) and torch.equal(y, -x.resolve_neg())
        out = torch.zeros(10, H, dtype=torch.complex64, device="cuda").conj().imag
        with pytest.raises(ValueError, match="negated"):
            fa.permute(x, plan, out=out)
        leaf = x.resolve_neg().clone().requires_grad_()
        g = torch.ones(10, H, dtype=torch.complex64, device="cuda").mul_(1j).conj().imag  # -1
        assert g.is_neg() and bool((torch.autograd.grad(fa.permute(leaf, plan), leaf, g)[0] == -2).all())
    one = torch.ones(1, dtype=torch.complex64, device="cuda").mul_(2j).conj().imag  # -2, contiguous
    assert one.is_neg() and one.is_contiguous()
    plan = fa.sort_experts(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), 1)
    rows = torch.ones(1, 8, device="cuda", requires_grad=True)
    y = fa.unpermute(rows, plan, one.view(1, 1))
    assert bool((y == -2).all()) and bool((torch.autograd.grad(y.sum(), rows)[0] == -2).all())


def test_columns_of_one_buffer():
    """What a call reads and writes may lie side by side in one buffer, single rows and vectors too."""
    H = 32
    for T, k in ((1, 4), (3, 4), (4, 1), (1, 1)):
        plan = fa.sort_experts(ids_of(T, k, 4, T).cuda(), 4)
        n = T * k
        x, rows, w = _rand((T, H), torch.float32, 1), _rand((n, H), torch.float32, 2), _rand((T, k), torch.float32, 3)
        buf = torch.zeros(max(n, T * k), 2 * H + k, device="cuda")
        buf[:T, H:2 * H] = x
        assert torch.equal(fa.permute(buf[:T, H:2 * H], plan, out=buf[:n, :H]), fa.permute(x, plan))
        buf[:n, H:2 * H], buf[:T, 2 * H:] = rows, w
        y = fa.unpermute(buf[:n, H:2 * H], plan, buf[:T, 2 * H:], out=buf[:T, :H])
        assert torch.equal(y, fa.unpermute(rows, plan, w))
        if n > 1:
            for lo in (0, 1, H - 1):
                with pytest.raises(ValueError, match="shares memory"):
                    fa.permute(buf[:T, lo:lo + H], plan, out=buf[:n, :H])
                with pytest.raises(ValueError, match="shares memory"):
                    fa.unpermute(buf[:n, :H], plan, out=buf[:T, lo:lo + H])
            with pytest.raises(ValueError, match="shares memory"):  # into the next row
                fa.permute(buf.view(-1)[2 * H + k - 1:][:H].view(1, H).expand(T, H), plan, out=buf[:n, :H])
    # a column of scales beside the rows
    q = torch.ones(6, 16, dtype=torch.int8, device="cuda")
    buf = torch.full((6, 17), 0.5, device="cuda")
    out = fa.int8_matmul(q, buf[:, 16], q[:1].expand(16, 16), torch.ones(16, device="cuda"), out=buf[:, :16])
    assert bool((out == 8).all())
    with pytest.raises(ValueError, match="shares memory"):
        fa.int8_matmul(q, buf[:, 15], q[:1].expand(16, 16), torch.ones(16, device="cuda"), out=buf[:, :16])
