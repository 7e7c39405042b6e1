"""The balance loss and swiglu (flashinfer_amd.layer) against 64-bit formulas,
within the roundings of their fp32 steps and of the result; and a layer made of
these and the other expert operators."""
import pytest
import torch

import flashinfer_amd as fa

pytestmark = pytest.mark.gpu
F64 = torch.float64
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, seed, scale=1.0):
    return (scale * torch.randn(shape, generator=_gen(seed), device="cuda")).to(dtype)


def _within(got, ref, before):
    """A result rounded once, whose value before that is off by at most `before`."""
    eps = torch.finfo(got.dtype).eps / 2
    bound = before * (1 + eps) + ref.abs() * eps + torch.finfo(got.dtype).smallest_normal * eps * 2
    bad = ~((got.to(F64) - ref).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:3], ref[bad][:3])


# ------------------------------------------------------------- balance loss


def _balance64(logits, ids, cuts, mask, score):
    """loss, counts, P, slope dP/dl's factor, w = dloss/dP, from the definition."""
    l = logits.to(F64)
    if score == "softmax":
        p, slope = torch.softmax(l, dim=1), torch.ones_like(l)
    else:
        s = torch.sigmoid(l)
        p, slope = s / s.sum(dim=1, keepdim=True), torch.sigmoid(-l)
    T, E = l.shape
    k = ids.shape[1]
    keep = torch.ones(T, dtype=torch.bool, device="cuda") if mask is None else mask
    counts, w, losses = [], torch.zeros_like(l), []
    for a, b in zip(cuts[:-1], cuts[1:]):
        rows = torch.arange(a, b, device="cuda")[keep[a:b]]
        named = ids[rows].long().flatten()
        named = named[(named >= 0) & (named < E)]
        c = torch.zeros(E, dtype=F64, device="cuda").scatter_add_(0, named, torch.ones_like(named, dtype=F64))
        counts.append(c)
        n = len(rows)
        if n:
            losses.append((c * p[rows].sum(dim=0)).sum() * (E / (k * n * n)))
            w[rows] = c * (E / (k * n * n))
    share = 1 / max(1, len(losses))
    return sum(losses, torch.zeros((), dtype=F64, device="cuda")) * share, torch.stack(counts).int(), p, slope, w * share


def _check_balance(logits, ids, cuts, mask, score, given_cuts=True):
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda") if given_cuts else None
    leaf = logits.detach().requires_grad_()
    loss, counts = fa.balance_loss(leaf, ids, seq_offsets=offsets, mask=mask, score=score)
    ref, want, p, slope, w = _balance64(logits, ids, cuts, mask, score)
    assert torch.equal(counts, want if given_cuts else want[0])
    assert loss.shape == () and loss.dtype == torch.float32
    # P: the difference to the row's maximum (U of it, which the exponential makes
    # relative), exponential, sums over at most 32 values and lanes, quotient
    live = (w.sum(dim=1) > 0) if mask is None else mask
    l = logits.to(F64)[live]
    spread = 0.0
    if l.numel():
        far = torch.where(l.isinf(), 0.0, l.amax(dim=1, keepdim=True) - l)  # -inf is 0 exactly
        spread = float(far.amax()) if score == "softmax" else 0.0
        if score == "sigmoid" and float(l.amax(dim=1).min()) < -60:
            spread = float(torch.where(l.isinf(), 0.0, l).abs().amax())
    rel = (spread + 48) * U
    # sums of P over a chunk and the chunks, all of one sign: at most 400 in a row
    assert abs(loss.item() - float(ref)) <= float(ref) * (rel + 420 * U) + 1e-37, (loss.item(), float(ref))
    g = torch.full((), 0.37, device="cuda")
    (grad,) = torch.autograd.grad(loss, leaf, g)
    out = w.sum(dim=1) == 0  # tokens that do not count (or whose sequence's slots name none)
    p = torch.where(out[:, None], 0.0, p)
    slope = torch.where(out[:, None], 0.0, slope)
    dot = (p * w).sum(dim=1, keepdim=True)
    exact = float(g) * p * slope * (w - dot)
    _within(grad, exact, float(g) * p * slope * (w + dot) * (2 * rel + 60 * U))
    same = fa.balance_loss(logits.detach(), ids, seq_offsets=offsets, mask=mask, score=score)
    assert torch.equal(same[0], loss.detach()) and torch.equal(same[1], counts)


def _top(logits, k):
    return logits.float().topk(k, dim=1).indices.to(torch.int32)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_balance_sizes(dtype, score):
    for T, E, k in ((1, 1, 1), (1, 256, 8), (15, 7, 3), (16, 64, 6), (17, 65, 1), (64, 256, 8), (100, 33, 4),
                    (257, 128, 8), (300, 1024, 64), (1000, 8, 2), (129, 511, 5), (70, 640, 2), (9000, 256, 8),
                    (40000, 12, 2)):
        logits = _randn((T, E), dtype, T, 1.5)
        _check_balance(logits, _top(logits, min(k, E)), [0, T], None, score, given_cuts=False)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_balance_sequences_and_masks(score):
    for T, E, k, cuts in ((40, 16, 2, [0, 1, 1, 17, 40]), (300, 128, 6, [0, 0, 0, 299, 300]),
                          (500, 256, 8, [3, 50, 50, 420]), (64, 8, 2, [0] * 70 + [5, 64]),
                          (2000, 64, 4, list(range(0, 2001, 10))), (9000, 40, 2, [0, 8999, 9000]), (33, 5, 1, [7, 7])):
        logits = _randn((T, E), torch.bfloat16, T, 1.5)
        ids = _top(logits, k)
        ids[::7, 0] = -1  # count nowhere
        ids[::11, 0] = E
        ids[::5, -1] = ids[::5, 0]  # an expert named twice counts twice
        _check_balance(logits, ids, cuts, None, score)
        mask = torch.rand(T, generator=_gen(2), device="cuda") > 0.3
        mask[cuts[0]:cuts[1] + 1] = False  # a sequence without a token
        held = logits.clone()
        held[~mask] = float("nan")  # what a token that is left out holds
        for l in (logits, held):
            _check_balance(torch.where(mask[:, None], l, l), ids, cuts, mask, score)
    none = torch.zeros(33, dtype=torch.bool, device="cuda")
    _check_balance(logits, ids, [0, 10, 33], none, score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_balance_more_slots_than_lanes(score):
    """More slots for a token than lanes hold it, and than there are experts."""
    for T, E, k in ((50, 8, 33), (5000, 30, 64), (3, 2, 9)):
        ids = torch.randint(-2, E + 2, (T, k), generator=_gen(T), device="cuda", dtype=torch.int32)
        for dtype in (torch.float32, torch.bfloat16):
            _check_balance(_randn((T, E), dtype, T), ids, [0, T], None, score, given_cuts=False)


def test_balance_far_scores():
    """Rows of -inf, rows whose sigmoids leave fp32, a masked expert, large scores."""
    E = 20
    logits = _randn((6, E), torch.float32, 1)
    ids = torch.arange(12, dtype=torch.int32, device="cuda").view(6, 2)
    logits[1] -= 300.0
    logits[2, :5] = float("-inf")
    logits[3, 4] = 150.0
    logits[4] = -95.0
    for score in ("softmax", "sigmoid"):
        _check_balance(logits, ids, [0, 6], None, score)
        row = logits.clone()
        row[5] = float("-inf")
        leaf = row.requires_grad_()
        loss, _ = fa.balance_loss(leaf, ids, score=score)
        (grad,) = torch.autograd.grad(loss, leaf)
        _, _, p, _, w = _balance64(logits, ids, [0, 6], None, score)
        p[5] = 0  # such a row has no probabilities
        assert abs(loss.item() - float((p * w).sum())) < 1e-5 and not grad[5].any() and bool(grad.isfinite().all())


def test_balance_gradient_against_differences():
    logits = _randn((20, 12), torch.float32, 3)
    ids = _top(logits, 3)
    cuts = torch.tensor([0, 7, 20], dtype=torch.int32, device="cuda")
    leaf = logits.clone().requires_grad_()
    (grad,) = torch.autograd.grad(fa.balance_loss(leaf, ids, cuts, score="sigmoid")[0], leaf)
    for t, e in ((0, 0), (6, 11), (7, 3), (19, 5)):
        h = torch.zeros_like(logits, dtype=F64)
        h[t, e] = 1e-4
        up, down = (_balance64(logits.to(F64) + s * h, ids, cuts.tolist(), None, "sigmoid")[0] for s in (1, -1))
        # the difference is off by h^2 f''' / 6, far below the gradient's roundings
        assert abs(float((up - down) / 2e-4) - float(grad[t, e])) < 1e-7


def test_balance_strides():
    T, E, k = 90, 24, 3
    wide = _randn((T, 2 * E + 3), torch.float32, 1)
    ids = _top(wide[:, :E], k)
    for l in (wide[:, 1:1 + E], wide[:, :2 * E:2], wide[:1, :E].expand(T, E), wide[:, 4:4 + E]):
        i = torch.stack([ids, ids], dim=2)[:, :, 0]
        _check_balance(l, i, [0, T], None, "softmax", given_cuts=False)
    loss, counts = fa.balance_loss(torch.zeros(0, 8, device="cuda"), ids[:0])
    assert float(loss) == 0 and counts.tolist() == [0] * 8
    leaf = torch.zeros(0, 8, device="cuda", requires_grad=True)
    assert torch.autograd.grad(fa.balance_loss(leaf, ids[:0])[0], leaf)[0].shape == (0, 8)
    # counts alone: no gradient, and none asked of the loss
    leaf = wide[:, :E].clone().requires_grad_()
    loss, counts = fa.balance_loss(leaf, ids)
    assert loss.requires_grad and not counts.requires_grad


# ------------------------------------------------------------------- swiglu


def _keep(seed, threshold, rows, cols):
    """Philox4x32-10 from its definition, in whole numbers of Python."""
    key, out = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF], []
    for m in range(rows):
        row = []
        for b in range(-(-cols // 8)):
            c, k = [b, m, 0, 0], list(key)
            for _ in range(10):
                x, y = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
                c = [(y >> 32) ^ c[1] ^ k[0], y & 0xFFFFFFFF, (x >> 32) ^ c[3] ^ k[1], x & 0xFFFFFFFF]
                k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
            for w in c:
                row += [w & 0xFFFF, w >> 16]
        out.append([v >= threshold for v in row[:cols]])
    return torch.tensor(out, dtype=torch.bool).view(rows, cols).cuda()


def _check_swiglu(x, grad, rows, keep=None, scale=1.0, **args):
    """The sigmoid is off by at most 6 U of it (exponent, exponential, sum,
    quotient with one step), a product of up to four factors by 4 U more; in
    1 + u (1 - s) the terms are each off by 8 U of 1 + |u|."""
    M, I = x.shape[0], x.shape[1] // 2
    leaf = x.detach().requires_grad_()
    y = fa.swiglu(leaf, **args)
    (dx,) = torch.autograd.grad(y, leaf, grad)
    v, u, g = x[:, :I].to(F64), x[:, I:].to(F64), grad.to(F64)
    s = torch.sigmoid(u)
    f = torch.full((M, I), scale, dtype=F64, device="cuda")
    if keep is not None:
        f = f * keep
    f[rows:] = 0
    ref = v * u * s * f
    _within(y.detach(), ref, 12 * U * ref.abs() + 1e-38)
    dv, du = g * u * s * f, g * v * s * (1 + u * (1 - s)) * f
    _within(dx[:, :I], dv, 12 * U * dv.abs() + 1e-38)
    _within(dx[:, I:], du, 20 * U * (g * v * s * f).abs() * (1 + u.abs()) + 1e-38)
    assert not y[rows:].any() and not dx[rows:].any()
    return y.detach()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_swiglu(dtype):
    for M, I in ((1, 1), (1, 8), (2, 7), (16, 2048), (33, 1536), (5, 100), (130, 264), (3, 2056), (2, 20000), (700, 32)):
        x, g = _randn((M, 2 * I), dtype, M, 3.0), _randn((M, I), dtype, I)
        y = _check_swiglu(x, g, M)
        assert torch.equal(fa.swiglu(x), y)
        for rows in {0, 1, M // 3, M}:
            n = torch.tensor([rows], dtype=torch.int32, device="cuda")
            assert torch.equal(_check_swiglu(x, g, rows, num_rows=n)[:rows], y[:rows])
            out = torch.full((M, I), 9.0, dtype=dtype, device="cuda")
            assert fa.swiglu(x, num_rows=n, out=out) is out
            assert torch.equal(out[:rows], y[:rows]) and bool((out[rows:] == 9).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_swiglu_dropout(dtype):
    for M, I, p, seed in ((1, 1, 0.5, 0), (3, 20, 0.1, 12345678901234567), (40, 64, 0.9, -1), (9, 33, 0.25, 2**64 - 1)):
        x, g = _randn((M, 2 * I), dtype, M), _randn((M, I), dtype, I)
        threshold = round(p * 65536)
        keep, scale = _keep(seed % 2**64, threshold, M, I), 65536 / (65536 - threshold)
        y = _check_swiglu(x, g, M, keep, scale, dropout=p, seed=seed)
        on_device = torch.tensor([seed if seed < 2**63 else seed - 2**64], device="cuda")
        assert torch.equal(fa.swiglu(x, dropout=p, seed=on_device), y)
        # what is dropped is zero, whatever it was
        bad = x.clone()
        bad[:, :I][~keep] = float("nan")
        assert torch.equal(fa.swiglu(bad, dropout=p, seed=seed), y)
        n = torch.tensor([M // 2], dtype=torch.int32, device="cuda")
        _check_swiglu(x, g, M // 2, keep, scale, dropout=p, seed=seed, num_rows=n)
    x = torch.ones(512, 1024, device="cuda", dtype=dtype)
    for p in (0.01, 0.5):  # how many, to 6 standard deviations; and other seeds drop others
        a, b = (fa.swiglu(x, dropout=p, seed=s) == 0 for s in (1, 2))
        n = a.numel()
        assert abs(int(a.sum()) - n * p) < 6 * (n * p * (1 - p)) ** 0.5
        assert abs(int((a & b).sum()) - n * p * p) < 6 * (n * p * p) ** 0.5


def test_swiglu_far_values():
    """Gates over the whole range of the types; infinities and NaN where the formula has them."""
    for dtype in DTYPES:
        big = float(torch.finfo(dtype).max)
        u = torch.tensor([0.0, -0.0, 1e-30, 20.0, -20.0, 86.9, -86.9, 87.1, -87.1, 88.7, -88.7, 100.0, -100.0, -104.0,
                          1000.0, -1000.0, big, -big], device="cuda").to(dtype)
        I = len(u)
        x = torch.cat([torch.ones(I, device="cuda", dtype=dtype), u])[None]
        y = _check_swiglu(x, torch.ones(1, I, device="cuda", dtype=dtype), 1)
        assert bool(y.isfinite().all())
    x = torch.tensor([[1.0, 2.0, 1.0, float("nan"), float("inf"), float("nan"), 1.0, 1.0]], device="cuda")
    y = fa.swiglu(x)
    assert float(y[0, 0]) == float("inf") and bool(y[0, 1].isnan()) and bool(y[0, 3].isnan())


def test_swiglu_strides():
    for dtype in (torch.bfloat16, torch.float32):
        wide = _randn((40, 150), dtype, 1)
        for x in (wide[:, 3:3 + 128], wide[:, :128], wide[::2, 8:136], wide[:1, :128].expand(40, 128), wide[:, :128].t()[:, :40]):
            M, I = x.shape[0], x.shape[1] // 2
            assert torch.equal(fa.swiglu(x), fa.swiglu(x.contiguous()))
            a, b = x.detach().requires_grad_(), x.contiguous().requires_grad_()
            g = _randn((I, M), dtype, 2).t()
            assert torch.equal(torch.autograd.grad(fa.swiglu(a, 0.3, 5), a, g)[0],
                               torch.autograd.grad(fa.swiglu(b, 0.3, 5), b, g.contiguous())[0])
            one = torch.ones((), dtype=dtype, device="cuda").expand(M, I)
            assert torch.equal(torch.autograd.grad(fa.swiglu(a), a, one)[0],
                               torch.autograd.grad(fa.swiglu(b), b, one.contiguous())[0])
            buf = torch.full((M, I + 5), 9.0, dtype=dtype, device="cuda")
            fa.swiglu(x, out=buf[:, 2:2 + I])
            assert torch.equal(buf[:, 2:2 + I], fa.swiglu(x)) and bool((buf[:, :2] == 9).all()) and bool((buf[:, 2 + I:] == 9).all())
    leaf = torch.zeros(0, 16, device="cuda", requires_grad=True)
    y = fa.swiglu(leaf)
    assert y.shape == (0, 8) and torch.autograd.grad(y, leaf, y)[0].shape == (0, 16)


def test_swiglu_gradient_against_differences():
    x = _randn((4, 20), torch.float32, 1)
    leaf = x.clone().requires_grad_()
    g = _randn((4, 10), torch.float32, 2)
    (dx,) = torch.autograd.grad(fa.swiglu(leaf, 0.2, 9), leaf, g)
    keep = _keep(9, round(0.2 * 65536), 4, 10) * (65536 / (65536 - round(0.2 * 65536)))

    def f(z):
        return (g.to(F64) * keep * z[:, :10] * z[:, 10:] * torch.sigmoid(z[:, 10:])).sum()
    for i in range(0, 80, 7):
        h = torch.zeros(80, dtype=F64, device="cuda")
        h[i] = 1e-4
        h = h.view(4, 20)
        assert abs(float((f(x.to(F64) + h) - f(x.to(F64) - h)) / 2e-4) - float(dx.view(-1)[i])) < 1e-5


# ------------------------------------------------------------ both together


def test_refusals():
    l = torch.zeros(6, 4, device="cuda")
    ids = torch.zeros(6, 2, dtype=torch.int32, device="cuda")
    x, leaf = torch.zeros(6, 16, device="cuda"), torch.zeros(6, 16, device="cuda", requires_grad=True)
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.zeros(6, 8, device="cuda")
    bad = [
        (ValueError, lambda: fa.balance_loss(l, ids[:5])), (ValueError, lambda: fa.balance_loss(l[0], ids)),
        (TypeError, lambda: fa.balance_loss(l.double(), ids)), (TypeError, lambda: fa.balance_loss(l, ids.long())),
        (ValueError, lambda: fa.balance_loss(l, ids.cpu())), (ValueError, lambda: fa.balance_loss(l.cpu(), ids)),
        (ValueError, lambda: fa.balance_loss(l[:, :0], ids)), (ValueError, lambda: fa.balance_loss(l, ids[:, :0])),
        (ValueError, lambda: fa.balance_loss(torch.zeros(6, 1025, device="cuda"), ids)),
        (ValueError, lambda: fa.balance_loss(l, torch.zeros(6, 65, dtype=torch.int32, device="cuda"))),
        (ValueError, lambda: fa.balance_loss(l, ids, score="tanh")), (ValueError, lambda: fa.balance_loss(l, ids, n)),
        (TypeError, lambda: fa.balance_loss(l, ids, n.long().expand(3))),
        (TypeError, lambda: fa.balance_loss(l, ids, mask=torch.ones(6, device="cuda"))),
        (ValueError, lambda: fa.balance_loss(l, ids, mask=torch.ones(5, device="cuda", dtype=torch.bool))),
        (ValueError, lambda: fa.swiglu(x[:, :15])), (ValueError, lambda: fa.swiglu(x[0])),
        (TypeError, lambda: fa.swiglu(x.double())), (ValueError, lambda: fa.swiglu(x.cpu())),
        (ValueError, lambda: fa.swiglu(x, dropout=1.0, seed=1)), (ValueError, lambda: fa.swiglu(x, dropout=-0.1, seed=1)),
        (ValueError, lambda: fa.swiglu(x, dropout=float("nan"), seed=1)), (ValueError, lambda: fa.swiglu(x, dropout=0.1)),
        (ValueError, lambda: fa.swiglu(x, dropout=0.1, seed=2**64)), (TypeError, lambda: fa.swiglu(x, dropout=0.1, seed=1.5)),
        (TypeError, lambda: fa.swiglu(x, 0.1, n)),
        (ValueError, lambda: fa.swiglu(x, 0.1, torch.zeros(2, dtype=torch.int64, device="cuda"))),
        (ValueError, lambda: fa.swiglu(x, 0.1, torch.zeros(1, dtype=torch.int64))),
        (TypeError, lambda: fa.swiglu(x, num_rows=n.long())), (ValueError, lambda: fa.swiglu(x, num_rows=n.expand(2))),
        (ValueError, lambda: fa.swiglu(leaf, out=out)), (TypeError, lambda: fa.swiglu(x, out=out.half())),
        (ValueError, lambda: fa.swiglu(x, out=x[:, :8])), (ValueError, lambda: fa.swiglu(x, out=out[:5])),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            print("not refused:", i)
    for make, leaf in ((lambda t: fa.balance_loss(t, ids)[0], l.clone().requires_grad_()), (fa.swiglu, leaf)):
        y = make(leaf)
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y, leaf, torch.ones_like(y), create_graph=True)
        y = make(leaf)
        with torch.no_grad():
            leaf.add_(1.0)
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(y, leaf, torch.ones_like(y))


def _layer(tokens, router, w1, w2, plan_of, seed, experts):
    """A layer of one's own, trained: products in torch, all else operators."""
    logits = tokens @ router.t()
    ids, weights = plan_of(logits)
    aux, _ = fa.balance_loss(logits, ids, score="sigmoid")
    plan = fa.sort_experts(ids, experts)
    rows = fa.permute(tokens, plan)
    cuts = plan.expert_offsets.tolist()
    parts = list(zip(range(experts), cuts[:-1], cuts[1:]))
    h = torch.cat([rows[a:b] @ w1[e].t() for e, a, b in parts])
    h = fa.swiglu(h, dropout=0.1, seed=seed, num_rows=plan.expert_offsets[-1:])
    y = torch.cat([h[a:b] @ w2[e].t() for e, a, b in parts])
    return fa.unpermute(y, plan, weights), aux


def test_layer_trained_and_served():
    """route -> balance loss -> permute -> product -> swiglu -> product ->
    unpermute and back in fp32 against 64 bits, then served with 4-bit weights."""
    T, H, I, E, k = 70, 64, 96, 8, 2
    shapes = ((T, H), (E, H), (E, 2 * I, H), (E, H, I))
    leaves = [_randn(s, torch.float32, n, 0.3).requires_grad_() for n, s in enumerate(shapes)]
    keep = _keep(77, round(0.1 * 65536), T * k, I) * (65536 / (65536 - round(0.1 * 65536)))

    def plan_of(logits):
        s = torch.sigmoid(logits)
        ids = s.topk(k, dim=1).indices
        w = s.gather(1, ids)
        return ids.to(torch.int32), w / w.sum(dim=1, keepdim=True)

    out, aux = _layer(*leaves, plan_of, 77, E)
    g = _randn((T, H), torch.float32, 9)
    got = torch.autograd.grad((out * g).sum() + 0.5 * aux, leaves)

    x, router, w1, w2 = (t.detach().to(F64).requires_grad_() for t in leaves)
    logits = x @ router.t()
    ids, w = plan_of(logits)
    plan = fa.sort_experts(ids, E)
    row = plan.row_of_slot.long()
    v, u = torch.einsum("th,tkjh->tkj", x, w1[ids.long()]).chunk(2, dim=2)
    h = v * u * torch.sigmoid(u) * keep[row]
    ref = (torch.einsum("tki,tkhi->tkh", h, w2[ids.long()]) * w[:, :, None]).sum(dim=1)
    p = torch.sigmoid(logits)
    p = p / p.sum(dim=1, keepdim=True)
    c = torch.bincount(ids.flatten().long(), minlength=E).to(F64)
    loss = (c * p.sum(dim=0)).sum() * E / (k * T * T)
    want = torch.autograd.grad((ref * g.to(F64)).sum() + 0.5 * loss, (x, router, w1, w2))
    # fp32 sums of at most T * k terms of 2 H products and a few factors each: far below 1e-4 of the largest
    for a, b in zip((out, aux, *got), (ref, loss, *want)):
        assert (a.to(F64) - b).abs().max().item() <= 1e-4 * b.abs().max().item()

    with torch.no_grad():
        q1, q2 = fa.quantize_int4(leaves[2], 32), fa.quantize_int4(leaves[3], 32)
        tokens = leaves[0].to(torch.bfloat16)
        plan = fa.sort_experts(ids, E)
        h = fa.int4_grouped_matmul(tokens, q1, plan.expert_offsets, row_ids=plan.token_of_row)
        h = fa.swiglu(h, num_rows=plan.expert_offsets[-1:])
        y = fa.int4_grouped_matmul(h, q2, plan.expert_offsets)
        y = fa.unpermute(y, plan, w.float())

        def dequant(q, rows, cols):  # one-hot rows read the weights back
            eye = torch.eye(cols, device="cuda", dtype=torch.bfloat16)
            return torch.stack([fa.int4_matmul(eye, fa.Int4Weights(q.packed[e], q.scale[e], *q[2:]),
                                               out_dtype=torch.float32).t() for e in range(E)]).to(F64)
        d1, d2 = dequant(q1, 2 * I, H), dequant(q2, H, I)
        # half a step is the most that a weight moves
        for d, t, q in ((d1, leaves[2], q1), (d2, leaves[3], q2)):
            top = t.abs().view(*t.shape[:2], -1, 32).amax(-1, keepdim=True).expand(*t.shape[:2], -1, 32).reshape(t.shape)
            assert bool(((d - t).abs() <= top / 14 * 1.001).all())
        v, u = torch.einsum("th,tkjh->tkj", tokens.to(F64), d1[ids.long()]).chunk(2, dim=2)
        h = v * u * torch.sigmoid(u)
        parts = torch.einsum("tki,tkhi->tkh", h, d2[ids.long()])
        ref = (parts * w[:, :, None]).sum(dim=1)
        # bf16 roundings of v and u (each with a slope of at most 1.1 of the other), of h, of y and of the result
        most = torch.einsum("tki,tkhi->tkh", v.abs() * u.abs().clamp_min(1.0), d2[ids.long()].abs()) * w[:, :, None]
        assert bool(((y.to(F64) - ref).abs() <= 2.0 ** -8 * (3.5 * most.sum(dim=1) + 2 * ref.abs().amax())).all())


def test_captured_training_step():
    """Forward and backward in a graph whose leaves no eager graph holds, with a
    seed that is read anew; every replay equals the eager step."""
    T, E, k, I = 50, 16, 2, 40
    logits, x = _randn((T, E), torch.float32, 1).requires_grad_(), _randn((T, 2 * I), torch.float32, 2).requires_grad_()
    ids, g = _top(logits.detach(), k), _randn((T, I), torch.float32, 3)
    mask = torch.rand(T, generator=_gen(4), device="cuda") > 0.2
    cuts = torch.tensor([0, 20, 45], dtype=torch.int32, device="cuda")
    seed = torch.tensor([5], device="cuda")
    n = torch.tensor([T], dtype=torch.int32, device="cuda")

    def step():
        loss, counts = fa.balance_loss(logits, ids, cuts, mask)
        y = fa.swiglu(x, 0.2, seed, n)
        return [loss.detach(), counts, y.detach(), *torch.autograd.grad((loss, y), (logits, x), (torch.ones_like(loss), g))]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    made = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made.append((graph, step()))
    for rep in range(3):
        with torch.no_grad():
            logits.copy_(_randn((T, E), torch.float32, 7 + rep))
            x.copy_(_randn((T, 2 * I), torch.float32, 17 + rep))
            seed.fill_(rep * 1000)
            n.fill_(T - rep)
            mask.copy_(torch.rand(T, generator=_gen(rep), device="cuda") > 0.2)
        for graph, _ in made:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, got in made:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
