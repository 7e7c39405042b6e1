"""The int8 quantisers and products (flashinfer_amd.int8) against 64-bit
formulas: the plain quantiser bit for bit, products within the roundings of
their fp32 epilogue and of the result."""
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


def _ints(shape, seed, lo=-128):
    return torch.empty(shape, dtype=torch.int8, device="cuda").random_(lo, 128, generator=_gen(seed))


def _scales(shape, seed):
    return torch.empty(shape, device="cuda").uniform_(0.0005, 0.002, generator=_gen(seed))


def _check(got, acc, sa, sb, bias=None):
    """|got - exact| within: int32 to fp32, two products, the bias's sum, the last rounding."""
    y = acc * sa.to(F64)[:, None] * sb.to(F64)
    ref = y if bias is None else y + bias.to(F64)
    eps = torch.finfo(got.dtype).eps / 2
    before = 3.001 * U * y.abs() + (U * ref.abs() * 1.001 if bias is not None else 0)
    bound = before * (1 + eps) + ref.abs() * eps + torch.finfo(got.dtype).smallest_normal * eps * 2
    bad = (got.to(F64) - ref).abs() > bound
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


def _exact(a, b):
    return torch.matmul(a.to(F64), b.to(F64).t())  # whole numbers below 2^53: exact


SHAPES = [  # M, N, K
    (1, 1, 1), (1, 16, 64), (1, 4096, 7168), (2, 100, 4096), (3, 17, 33), (5, 64, 128), (16, 4096, 2048),
    (17, 130, 1024), (31, 48, 272), (33, 1000, 528), (64, 256, 7168), (65, 64, 16), (100, 7168, 2048),
    (128, 128, 128), (130, 515, 1040), (200, 4096, 512), (256, 256, 256), (257, 300, 130), (300, 264, 784),
    (511, 513, 96), (600, 1024, 2048), (1024, 2048, 1024), (1111, 999, 400), (2050, 1536, 4096), (4097, 31, 160),
    (2049, 2050, 4101), (8200, 4100, 1025)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matmul(shape, dtype):
    M, N, K = shape
    a, b, sa, sb = _ints((M, K), 1), _ints((N, K), 2), _scales(M, 3), _scales(N, 4)
    acc = _exact(a, b)
    y = fa.int8_matmul(a, sa, b, sb, out_dtype=dtype)
    assert y.dtype == dtype and y.shape == (M, N)
    _check(y, acc, sa, sb)
    bias = torch.randn(N, generator=_gen(5), device="cuda").to(DTYPES[M % 3])
    z = fa.int8_matmul(a, sa, b, sb, bias=bias, out_dtype=dtype)
    _check(z, acc, sa, sb, bias)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_matmul_at_the_largest_sums(M):
    """K at its limit and every product 2^14: the int32 sums do not wrap."""
    K = 131071
    a = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    b = torch.full((33, K), -128, dtype=torch.int8, device="cuda")
    b[1::2] = 127
    one = torch.ones(M, device="cuda"), torch.ones(33, device="cuda")
    y = fa.int8_matmul(a, one[0], b, one[1], out_dtype=torch.float32)
    want = torch.full((M, 33), float(K * 16384), device="cuda")
    want[:, 1::2] = float(-K * 128 * 127)
    assert torch.equal(y, want)
    with pytest.raises(ValueError, match="131071"):
        fa.int8_matmul(torch.zeros(1, K + 1, dtype=torch.int8, device="cuda"), one[0][:1],
                       torch.zeros(1, K + 1, dtype=torch.int8, device="cuda"), one[1][:1])


@pytest.mark.parametrize("M", [1, 20, 150, 700])
def test_matmul_strides_and_alignment(M):
    N, K = 200, 512
    big_a, big_b = _ints((M, 700), 1), _ints((N, 800), 2)
    sa, sb = _scales(2 * M, 3), _scales(2 * N, 4)
    for oa, ob in ((0, 0), (16, 32), (1, 0), (0, 3), (8, 8)):
        a, b = big_a[:, oa:oa + K], big_b[:, ob:ob + K]
        y = fa.int8_matmul(a, sa[::2], b, sb[1::2])
        assert torch.equal(y, fa.int8_matmul(a.contiguous(), sa[::2].contiguous(), b.contiguous(),
                                             sb[1::2].contiguous()))
        _check(y, _exact(a, b), sa[::2], sb[1::2])
    assert torch.equal(fa.int8_matmul(a.t().contiguous().t(), sa[::2], b, sb[1::2]), y)
    one = big_a[:1, :K].expand(M, K)
    _check(fa.int8_matmul(one, sa[:M], b, sb[:N]), _exact(one, b), sa[:M], sb[:N])
    for pad in (8, 3):  # a destination inside a wider one
        buf = torch.full((M, N + 2 * pad), 5.0, dtype=torch.bfloat16, device="cuda")
        out = fa.int8_matmul(a, sa[::2], b, sb[1::2], out=buf[:, pad:pad + N])
        assert torch.equal(out, y) and torch.equal(buf[:, pad:pad + N], y)
        assert bool((buf[:, :pad] == 5).all()) and bool((buf[:, pad + N:] == 5).all())


# rows of each expert, tokens (0: rows of a directly), N, K, spare rows behind the last
GROUPS = [([1], 0, 64, 128, 0), ([0, 0, 3], 0, 16, 64, 2), ([5, 0, 1, 0, 64, 65], 0, 130, 272, 7),
          ([1] * 40, 13, 256, 1024, 8), ([2, 0, 5, 1] * 8, 64, 4096, 2048, 100), ([0] * 5, 4, 64, 64, 9),
          ([300, 0, 17, 129, 256, 1], 500, 512, 640, 30), ([257], 100, 300, 1040, 1), ([1000, 3, 500], 0, 768, 2048, 0),
          ([0, 2500, 0, 40], 1024, 1024, 512, 64), ([3] * 1024, 0, 33, 48, 1), ([70] * 32, 300, 512, 1536, 5)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", GROUPS, ids=lambda c: f"{len(c[0])}x{sum(c[0])}-{c[1]}-{c[2]}-{c[3]}")
def test_grouped(case, dtype):
    counts, tokens, N, K, spare = case
    E, R = len(counts), sum(counts) + spare
    offs = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()
    M = tokens or R
    a, b, sa, sb = _ints((M, K), 1), _ints((E, N, K), 2), _scales(M, 3), _scales((E, N), 4)
    ids = torch.randint(0, M, (R,), generator=_gen(5), device="cuda", dtype=torch.int32) if tokens else None
    if tokens:
        ids[sum(counts):] = -1  # not read
    y = fa.int8_grouped_matmul(a, sa, b, sb, offs, row_ids=ids, out_dtype=dtype)
    assert y.shape == (R, N) and not y[sum(counts):].any()
    lo = 0
    for e, c in enumerate(counts):
        if c:
            src = ids[lo:lo + c].long() if tokens else slice(lo, lo + c)
            _check(y[lo:lo + c], _exact(a[src], b[e]), sa[src], sb[e])
        lo += c
    buf = torch.full((R, N), 9.0, dtype=dtype, device="cuda")
    fa.int8_grouped_matmul(a, sa, b, sb, offs, row_ids=ids, out=buf)
    assert torch.equal(buf[:lo], y[:lo]) and bool((buf[lo:] == 9).all())


def _leave_behind(like):
    """A freed block of the result's size that holds no zeros, for the next result to get."""
    torch.full_like(like, 9)


@pytest.mark.parametrize("tile", range(9))
@pytest.mark.parametrize("shape", [(264, 400), (130, 515)], ids=str)
def test_rows_without_an_expert_are_zeros(tile, shape, monkeypatch):
    """Those behind the last expert's, and those before the first one's."""
    monkeypatch.setenv("MI_INT8_TILE", str(tile))
    N, K = shape
    for offs, R in (([3, 3, 10, 300], 340), ([0, 0, 0, 0], 70), ([70, 70, 70, 70], 70), ([0, 1, 1, 1], 1)):
        offs = torch.tensor(offs, dtype=torch.int32, device="cuda")
        a, b, sa, sb = _ints((R, K), 1), _ints((3, N, K), 2), _scales(R, 3), _scales((3, N), 4)
        buf = torch.full((R, N), 9.0, dtype=torch.bfloat16, device="cuda")
        fa.int8_grouped_matmul(a, sa, b, sb, offs, out=buf)
        _leave_behind(buf)
        y = fa.int8_grouped_matmul(a, sa, b, sb, offs)
        first, end = int(offs[0]), int(offs[-1])
        assert torch.equal(y[first:end], buf[first:end])
        assert not y[:first].any() and not y[end:].any()
        assert bool((buf[:first] == 9).all()) and bool((buf[end:] == 9).all())


@pytest.mark.parametrize("K", [33, 96, 2048, 5000])
@pytest.mark.parametrize("swiglu", [False, True])
def test_quantize_clears_rows_past_those_in_use(K, swiglu):
    f = fa.swiglu_quantize_int8 if swiglu else fa.quantize_int8
    M = 700
    x = torch.randn(M, K * (1 + swiglu), generator=_gen(1), device="cuda").bfloat16()
    q0, s0 = f(x)
    for n in (-5, 0, 1, 699, 700, 5000):
        count = torch.tensor([n], dtype=torch.int32, device="cuda")
        _leave_behind(q0), _leave_behind(s0)
        q, s = f(x, num_rows=count)
        n = min(max(n, 0), M)
        assert torch.equal(q[:n], q0[:n]) and torch.equal(s[:n], s0[:n])
        assert not q[n:].any() and not s[n:].any()
        s2 = torch.full_like(s0, 9)  # one buffer passed in, one new
        q2, _ = f(x, num_rows=count, scale=s2)
        assert torch.equal(q2, q) and torch.equal(s2[:n], s0[:n]) and bool((s2[n:] == 9).all())


# the tiles of csrc/int8_common.hpp, each at sizes that end inside it
@pytest.mark.parametrize("tile", range(9))
@pytest.mark.parametrize("shape", [(1, 8, 144), (70, 90, 272), (130, 264, 2048), (259, 515, 1040), (300, 40, 7),
                                   (520, 700, 1111), (1030, 1000, 128)], ids=str)
def test_every_tile(tile, shape, monkeypatch):
    monkeypatch.setenv("MI_INT8_TILE", str(tile))
    M, N, K = shape
    a, b, sa, sb = _ints((M, K), 1), _ints((4, N, K), 2), _scales(M, 3), _scales((4, N), 4)
    bias = torch.randn(N, generator=_gen(5), device="cuda")
    for dtype in (torch.bfloat16, torch.float32):
        _check(fa.int8_matmul(a, sa, b[1], sb[1], bias=bias, out_dtype=dtype), _exact(a, b[1]), sa, sb[1], bias)
    # experts whose rows end inside, at and behind a tile's end, one without rows
    ends = [0, M // 7, M // 7, M // 7 + min(128, M // 2), M]
    offs = torch.tensor(ends, dtype=torch.int32, device="cuda")
    ids = torch.randperm(M, generator=_gen(6), device="cuda").to(torch.int32)
    for rows in (None, ids):
        y = fa.int8_grouped_matmul(a, sa, b, sb, offs, row_ids=rows)
        for e in range(4):
            at = torch.arange(ends[e], ends[e + 1], device="cuda")
            src = at if rows is None else ids[at].long()
            if len(at):
                _check(y[at], _exact(a[src], b[e]), sa[src], sb[e])


# few, some and many rows after each other, in all orders: at most 128, 129 to 192, up to 256, several tiles
MIXED = [100, 300, 1, 0, 190, 256, 64, 64, 520, 128, 129, 700, 33, 256, 256, 140, 90, 150, 600, 300, 5, 130] * 2


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("K", [144, 256, 400, 640, 1040])  # 2, 2, 4, 5 and 9 steps; the last of 16 or 128 bytes
def test_large_tiles_of_experts_in_turn(K, gather, monkeypatch):
    """Workgroups with several 256 x 256 tiles, whose experts and row counts change from one to the next."""
    monkeypatch.setenv("MI_INT8_TILE", "8")
    E, R, N, dtype = len(MIXED), sum(MIXED), 4088, torch.float32 if K == 640 else torch.bfloat16
    tiles = sum((c + 255) // 256 for c in MIXED) * 16
    assert tiles > 3 * 256
    offs = torch.tensor([0] + MIXED).cumsum(0).to(torch.int32).cuda()
    M = 1500 if gather else R
    a, b, sa, sb = _ints((M, K), 1), _ints((E, N, K), 2), _scales(M, 3), _scales((E, N), 4)
    ids = torch.randint(0, M, (R,), generator=_gen(5), device="cuda", dtype=torch.int32) if gather else None
    y = fa.int8_grouped_matmul(a, sa, b, sb, offs, row_ids=ids, out_dtype=dtype)
    lo = 0
    for e, c in enumerate(MIXED):
        src = ids[lo:lo + c].long() if gather else slice(lo, lo + c)
        _check(y[lo:lo + c], _exact(a[src], b[e]), sa[src], sb[e])
        lo += c


@pytest.mark.parametrize("K", [512, 515])
@pytest.mark.parametrize("rows", [30, 400])
def test_grouped_strided_weights_and_bad_ids(rows, K):
    E, N, M = 3, 96, 50
    w = _ints((E, N + 8, K + 16), 1)[:, 4:4 + N, :K]
    a, sa, sb = _ints((M, K), 2), _scales(M, 3), _scales((E, N), 4)
    offs = torch.tensor([0, rows // 3, rows // 2, rows], dtype=torch.int32, device="cuda")
    ids = torch.randint(0, M, (rows,), generator=_gen(5), device="cuda", dtype=torch.int32)
    good = fa.int8_grouped_matmul(a, sa, w.contiguous(), sb, offs, row_ids=ids)
    assert torch.equal(fa.int8_grouped_matmul(a, sa, w, sb, offs, row_ids=ids), good)
    ids[::7] = M
    ids[3] = -5
    y = fa.int8_grouped_matmul(a, sa, w, sb, offs, row_ids=ids)
    out = (ids < 0) | (ids >= M)
    assert bool(torch.isnan(y[out]).all()) and torch.equal(y[~out], good[~out])
    # offsets past the rows are cut to them
    far = torch.tensor([0, rows // 3, rows // 2, 1 << 30], dtype=torch.int32, device="cuda")
    assert torch.equal(fa.int8_grouped_matmul(a, sa, w, sb, far, row_ids=ids)[~out], good[~out])


QUANT = [(1, 1), (1, 7168), (3, 7), (5, 1024), (64, 1025), (33, 2048), (7, 4100), (100, 8192), (2, 40000), (4096, 64)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", QUANT, ids=str)
def test_quantize_is_the_formula(shape, dtype):
    M, K = shape
    x = (torch.randn(M, K, generator=_gen(1), device="cuda") * torch.logspace(-3, 3, M, device="cuda")[:, None]).to(dtype)
    x[M // 2] = 0
    q, s = fa.quantize_int8(x)
    xc = x.cpu().float()
    want_s = xc.abs().amax(dim=1).clamp_min(1e-10) / 127.0
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu(), torch.round(xc / want_s[:, None]).to(torch.int8))
    # rows at a distance, and odd ones
    wide = torch.zeros(M, K + 5, dtype=dtype, device="cuda")
    wide[:, 5:] = x
    q2, s2 = fa.quantize_int8(wide[:, 5:])
    assert torch.equal(q2, q) and torch.equal(s2, s)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", QUANT, ids=str)
def test_swiglu_quantize(shape, dtype):
    M, K = shape
    x = torch.randn(M, 2 * K, generator=_gen(2), device="cuda").mul_(3).to(dtype)
    q, s = fa.swiglu_quantize_int8(x)
    v = x.to(F64)
    v = v[:, K:] * torch.sigmoid(v[:, K:]) * v[:, :K]
    want = v.abs().amax(dim=1).clamp_min(1e-10) / 127.0
    # exp within 2 steps (4 U), then sum, quotient and product (3 U), the scale's quotient (1 U)
    assert bool(((s.to(F64) - want).abs() <= 8 * U * want * 1.001).all())
    # q is rint of a quotient that is within 7 + 8 + 1 U of the exact one
    assert bool(((q.to(F64) - v / want[:, None]).abs() <= 0.5 + 127 * 16.1 * U).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("K", [5, 64])
def test_swiglu_of_extreme_gates(K, dtype):
    """Gates up to the type's largest value; those below -90 give (next to) nothing."""
    most = torch.finfo(dtype).max
    gates = torch.tensor([most, most / 2, 3e4, 90.0, 87.0, 86.5, -86.5, -87.0, -90.0, -most], dtype=F64)
    x = torch.empty(len(gates), 2 * K, dtype=F64).uniform_(-0.5, 0.5, generator=torch.Generator().manual_seed(1))
    x[:, K] = gates
    x = x.to(dtype).cuda()
    q, s = fa.swiglu_quantize_int8(x)
    v = x.to(F64)
    v = v[:, K:] * torch.sigmoid(v[:, K:]) * v[:, :K]
    want = v.abs().amax(dim=1) / 127.0
    assert bool(((s.to(F64) - want).abs() <= 8 * U * want * 1.001).all())
    assert bool(((q.to(F64) - v / want[:, None]).abs() <= 0.5 + 127 * 16.1 * U).all())


def test_quantize_rows_in_use_and_poisoned_rows():
    x = torch.randn(10, 96, generator=_gen(1), device="cuda")
    n = torch.tensor([6], dtype=torch.int32, device="cuda")
    q0, s0 = fa.quantize_int8(x)
    q, s = fa.quantize_int8(x, num_rows=n)
    assert torch.equal(q[:6], q0[:6]) and torch.equal(s[:6], s0[:6]) and not q[6:].any() and not s[6:].any()
    qb, sb = torch.full_like(q, 5), torch.full_like(s, 5.0)
    fa.quantize_int8(x, num_rows=n, q=qb, scale=sb)
    assert torch.equal(qb[:6], q0[:6]) and bool((qb[6:] == 5).all()) and bool((sb[6:] == 5).all())
    x[2, 50], x[4, 0] = float("nan"), float("-inf")
    q, s = fa.quantize_int8(x)
    y = fa.int8_matmul(q, s, _ints((16, 96), 3), torch.ones(16, device="cuda"))
    bad = torch.tensor([2, 4], device="cuda")
    assert bool(torch.isnan(y[bad]).all())
    keep = [i for i in range(10) if i not in (2, 4)]
    assert bool(torch.isfinite(y[keep]).all()) and torch.equal(q[keep], q0[keep])


def test_offsets_past_32_bits():
    """More than 2^31 outputs, and weights of more than 2^31 bytes."""
    M, N, K = 70000, 32768, 32
    a, b, sa, sb = _ints((M, K), 1), _ints((N, K), 2), _scales(M, 3), _scales(N, 4)
    y = fa.int8_matmul(a, sa, b, sb)
    _check(y[-300:], _exact(a[-300:], b), sa[-300:], sb)
    del y
    E, N, K = 3, 16384, 65536
    w = torch.zeros(E, N, K, dtype=torch.int8, device="cuda")
    w[2] = _ints((N, K), 5)
    offs = torch.tensor([0, 1, 2, 40], dtype=torch.int32, device="cuda")
    a, sa, sb = _ints((40, K), 6), _scales(40, 7), _scales((E, N), 8)
    y = fa.int8_grouped_matmul(a, sa, w, sb, offs)
    _check(y[2:, -200:], _exact(a[2:], w[2, -200:]), sa[2:], sb[2, -200:])
    assert not y[:2].any()


def test_gathered_rows_past_32_bits():
    """Tokens whose rows lie more than 2^32 bytes into a."""
    M, K, N = 140000, 32768, 64
    a = torch.zeros(M, K, dtype=torch.int8, device="cuda")
    a[-50:] = _ints((50, K), 1)
    b, sa, sb = _ints((2, N, K), 2), _scales(M, 3), _scales((2, N), 4)
    ids = torch.arange(M - 50, M, device="cuda", dtype=torch.int32).flip(0)
    offs = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    y = fa.int8_grouped_matmul(a, sa, b, sb, offs, row_ids=ids)
    for e, rows in enumerate((slice(0, 20), slice(20, 50))):
        _check(y[rows], _exact(a[ids[rows].long()], b[e]), sa[ids[rows].long()], sb[e])


def test_gathered_overlapping_rows_at_32_bits():
    """Rows that overlap (16 bytes apart, 128 long): the last ones' ends lie past 2^32 bytes, their starts before."""
    M, K, N = 2 ** 28 - 1, 128, 64
    line = torch.zeros((M - 1) * 16 + K, dtype=torch.int8, device="cuda")
    line[:4096], line[-4096:] = _ints(4096, 1), _ints(4096, 2)
    a = line.as_strided((M, K), (16, 1))
    b, sb = _ints((2, N, K), 3), _scales((2, N), 4)
    sa = torch.ones(M, device="cuda")
    ids = torch.cat([torch.arange(M - 40, M), torch.arange(10)]).to(torch.int32).cuda()
    offs = torch.tensor([0, 30, 50], dtype=torch.int32, device="cuda")
    y = fa.int8_grouped_matmul(a, sa, b, sb, offs, row_ids=ids)
    for e, rows in enumerate((slice(0, 30), slice(30, 50))):
        _check(y[rows], _exact(a[ids[rows].long()], b[e]), sa[ids[rows].long()], sb[e])


def test_copied_product_in_graphs():
    """Large products of rows at any address copy them to a workspace: two
    captured graphs, replayed in turn, keep theirs apart."""
    M, N, K = 2048, 2112, 4111
    made = []
    for seed in (1, 2):
        a, b, sa, sb = _ints((M, K), seed), _ints((N, K), seed + 2), _scales(M, 3), _scales(N, 4)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            fa.int8_matmul(a, sa, b, sb)
        torch.cuda.current_stream().wait_stream(st)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fa.int8_matmul(a, sa, b, sb)
        made.append((graph, a, b, sa, sb, y))
    for rep in range(3):
        for n, (_, a, *_) in enumerate(made):
            a.copy_(_ints((M, K), 10 * rep + n))
        for graph, *_ in made:
            graph.replay()
        torch.cuda.synchronize()
        for _, a, b, sa, sb, y in made:
            assert torch.equal(y, fa.int8_matmul(a, sa, b, sb))
    _check(y, _exact(a, b), sa, sb)


def test_buffers_are_apart_and_counted_as_written():
    a, b, sa, sb = _ints((64, 64), 1), _ints((64, 64), 2), _scales(64, 3), _scales(64, 4)
    big = torch.zeros(64, 128, dtype=torch.float32, device="cuda")
    as_int8 = big.view(torch.int8)  # [64, 512]
    with pytest.raises(ValueError, match="shares memory"):
        fa.int8_matmul(as_int8[:, :64], sa, b, sb, out=big[:, :64])
    fa.int8_matmul(as_int8[:, 256:320], sa, b, sb, out=big[:, :64])  # other columns of one buffer
    x = torch.randn(4, 64, device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        fa.quantize_int8(x, q=x.view(torch.int8)[:, :64])
    buf = torch.ones(64, 64, dtype=torch.bfloat16, device="cuda")
    p = torch.randn(64, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = (p * buf).sum()  # keeps buf for its gradient
    with torch.no_grad():
        fa.int8_matmul(a, sa, b, sb, out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


@pytest.mark.parametrize("T", [1, 3, 40, 700])
def test_expert_layer_in_int8(T):
    """route, sort, gathered product, SwiGLU and quantiser, second product,
    and back: against the same layer in 64 bits, quantised at the same places."""
    from flashinfer_amd import kernel
    H, I, E, off = 1024, 512, 32, 64
    g = _gen(T)
    logits = torch.randn(T, 256, generator=g, device="cuda")
    logits[:, off:off + E] += 1.5
    ids, w = kernel.route(logits, torch.zeros(256, device="cuda"), 2.5)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    w1, w2 = _ints((E, 2 * I, H), 1), _ints((E, H, I), 2)
    s1, s2 = _scales((E, 2 * I), 3), _scales((E, H), 4)

    def layer():
        plan = fa.sort_experts(ids, E, off)
        q, s = fa.quantize_int8(x)
        h = fa.int8_grouped_matmul(q, s, w1, s1, plan.expert_offsets, row_ids=plan.token_of_row)
        q, s = fa.swiglu_quantize_int8(h, num_rows=plan.expert_offsets[-1:])
        return plan, h, q, s, fa.unpermute(fa.int8_grouped_matmul(q, s, w2, s2, plan.expert_offsets), plan, w)

    plan, h, q, s, y = layer()
    S = int(plan.expert_offsets[-1])
    ref = torch.zeros(T, H, dtype=F64, device="cuda")
    qx, sx = fa.quantize_int8(x)
    for t in range(T) if T <= 40 else (0, 1, T // 2, T - 1):
        for j in range(8):
            e = int(ids[t, j]) - off
            if 0 <= e < E:
                p = int(plan.row_of_slot[t, j])
                assert p < S
                _check(h[p:p + 1], _exact(qx[t:t + 1], w1[e]), sx[t:t + 1], s1[e])
                row = (_exact(q[p:p + 1], w2[e]) * s[p].to(F64) * s2[e].to(F64))[0]
                ref[t] += float(w[t, j]) * row
    # bf16 rows (2^-8 of each term), summed in fp32, rounded once more
    rows = [t for t in (range(T) if T <= 40 else (0, 1, T // 2, T - 1))]
    size = torch.zeros_like(ref)
    for t in rows:
        for j in range(8):
            e = int(ids[t, j]) - off
            if 0 <= e < E:
                p = int(plan.row_of_slot[t, j])
                size[t] += abs(float(w[t, j])) * (_exact(q[p:p + 1], w2[e]) * s[p].to(F64) * s2[e].to(F64))[0].abs()
    bound = size * (2.0 ** -8 + 16 * U) * 1.01 + ref.abs() * 2.0 ** -8
    assert bool(((y[rows].to(F64) - ref[rows]).abs() <= bound[rows]).all())
    # captured and replayed
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        layer()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        *_, z = layer()
    for rep in range(3):
        x.copy_(torch.randn(T, H, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, layer()[-1])


@pytest.mark.parametrize("tile", [0, 1, 2])
def test_forced_tiles_of_a_large_product(tile, monkeypatch):
    """2^32 outputs: 32 x 32 tiles of 1024 threads would be 2^32 threads, the rule's tile is taken."""
    n, K = 65536, 16
    a, b, sa, sb = _ints((n, K), 1), _ints((n, K), 2), _scales(n, 3), _scales(n, 4)
    monkeypatch.setenv("MI_INT8_TILE", str(tile))
    y = fa.int8_matmul(a, sa, b, sb)
    for rows in (slice(0, 40), slice(n // 2, n // 2 + 40), slice(n - 40, n)):
        _check(y[rows], _exact(a[rows], b), sa[rows], sb)


@pytest.mark.parametrize("T", [1, 700])
def test_expert_layer_into_buffers(T):
    """On a shard whose experts have a part of the rows: buffers passed in, whose other rows hold anything, give what
    new results give, and those rows stay."""
    H, I, E, off, k = 256, 128, 8, 16, 4
    ids = torch.rand(T, 64, generator=_gen(T), device="cuda").argsort(1)[:, :k].to(torch.int32)
    ids[0, 0] = off
    x, w = torch.randn(T, H, generator=_gen(1), device="cuda").bfloat16(), torch.rand(T, k, generator=_gen(2), device="cuda")
    w1, w2 = _ints((E, 2 * I, H), 3), _ints((E, H, I), 4)
    s1, s2 = _scales((E, 2 * I), 5), _scales((E, H), 6)
    nan = float("nan")
    h = torch.full((T * k, 2 * I), nan, dtype=torch.bfloat16, device="cuda")
    qb, sb = torch.full((T * k, I), 77, dtype=torch.int8, device="cuda"), torch.full((T * k,), nan, device="cuda")
    y = torch.full((T * k, H), nan, dtype=torch.bfloat16, device="cuda")

    def layer(h, qb, sb, y):
        plan = fa.sort_experts(ids, E, off)
        q, s = fa.quantize_int8(x)
        g = fa.int8_grouped_matmul(q, s, w1, s1, plan.expert_offsets, row_ids=plan.token_of_row, out=h)
        q, s = fa.swiglu_quantize_int8(g, num_rows=plan.expert_offsets[-1:], q=qb, scale=sb)
        return plan, fa.unpermute(fa.int8_grouped_matmul(q, s, w2, s2, plan.expert_offsets, out=y), plan, w)

    want = layer(None, None, None, None)[1]
    plan, got = layer(h, qb, sb, y)
    S = int(plan.expert_offsets[-1])
    assert torch.equal(got, want) and bool(torch.isfinite(got).all()) and 0 < S < T * k
    assert bool((qb[S:] == 77).all()) and all(bool(torch.isnan(t[S:]).all()) for t in (h, sb, y))


def test_two_streams_and_threads():
    import threading
    a, b, sa, sb = _ints((200, 2048), 1), _ints((1024, 2048), 2), _scales(200, 3), _scales(1024, 4)
    want = fa.int8_matmul(a, sa, b, sb)
    torch.cuda.synchronize()
    bad = []

    def work():
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                got = [fa.int8_matmul(a[:m], sa[:m], b, sb) for m in (1, 16, 64, 200)]
            st.synchronize()
        bad.extend(0 for y in got if not torch.equal(y, want[:len(y)]))

    threads = [threading.Thread(target=work) for _ in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_streams_and_threads_with_workspaces():
    """Calls that take a workspace, and those that clear what they do not use, on three streams at once:
    every result is that of its own inputs."""
    import threading
    M, N, K, E, k = 2048, 2112, 4111, 8, 4
    b, sb, w, sw = _ints((N, K), 1), _scales(N, 2), _ints((E, 512, 256), 3), _scales((E, 512), 4)
    sa = _scales(M, 5)

    def step(ids, a, x):
        plan = fa.sort_experts(ids, E, 2)
        q, s = fa.quantize_int8(x, num_rows=plan.expert_offsets[-1:])
        return (*plan, q, s, fa.int8_grouped_matmul(q, s, w, sw, plan.expert_offsets), fa.int8_matmul(a, sa, b, sb))

    inputs, want = [], []
    for n in range(3):
        ids = torch.randint(0, E + 4, (1500, k), generator=_gen(n), device="cuda", dtype=torch.int32)
        inputs.append((ids, _ints((M, K), 10 + n), torch.randn(1500 * k, 256, generator=_gen(20 + n), device="cuda").half()))
        want.append(step(*inputs[-1]))
    _check(want[0][-1], _exact(inputs[0][1], b), sa, sb)
    torch.cuda.synchronize()
    bad = []

    def work(n):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            got = [step(*inputs[n]) for _ in range(10)]
            st.synchronize()
        bad.extend((n, i, j) for i, out in enumerate(got) for j in range(len(out)) if not torch.equal(out[j], want[n][j]))

    threads = [threading.Thread(target=work, args=(n,)) for n in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_refusals():
    a, b = _ints((4, 32), 1), _ints((8, 32), 2)
    sa, sb = _scales(4, 3), _scales(8, 4)
    w, sw = _ints((2, 8, 32), 2), _scales((2, 8), 4)
    offs = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    out = torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(4, 32, device="cuda")
    bad = [
        (TypeError, lambda: fa.int8_matmul(a.float(), sa, b, sb)),
        (TypeError, lambda: fa.int8_matmul(a, sa, b.view(torch.uint8), sb)),
        (TypeError, lambda: fa.int8_matmul(a, sa.half(), b, sb)),
        (TypeError, lambda: fa.int8_matmul(a, sa, b, sb, out_dtype=torch.float64)),
        (TypeError, lambda: fa.int8_matmul(a, sa, b, sb, bias=torch.zeros(8, device="cuda", dtype=torch.float64))),
        (ValueError, lambda: fa.int8_matmul(a[:, :16], sa, b, sb)),
        (ValueError, lambda: fa.int8_matmul(a, sa[:3], b, sb)),
        (ValueError, lambda: fa.int8_matmul(a, sa[:, None], b, sb)),
        (ValueError, lambda: fa.int8_matmul(a, sa, b, sb, bias=torch.zeros(1, device="cuda"))),
        (ValueError, lambda: fa.int8_matmul(a, sa, b.cpu(), sb)),
        (ValueError, lambda: fa.int8_matmul(a.cpu(), sa, b, sb)),
        (ValueError, lambda: fa.int8_matmul(a, sa, b, sb, out=out[:3])),
        (ValueError, lambda: fa.int8_matmul(a, sa, b, sb, out=out[:1].expand(4, 8))),
        (ValueError, lambda: fa.int8_matmul(a, sa, b, sb.clone().requires_grad_())),
        (ValueError, lambda: fa.int8_matmul(a[:, :0], sa, b[:, :0], sb)),
        (ValueError, lambda: fa.int8_grouped_matmul(a, sa, b, sb, offs)),
        (ValueError, lambda: fa.int8_grouped_matmul(a, sa, w, sw, offs[:2])),
        (TypeError, lambda: fa.int8_grouped_matmul(a, sa, w, sw, offs.long())),
        (TypeError, lambda: fa.int8_grouped_matmul(a, sa, w, sw, offs, row_ids=offs.long())),
        (ValueError, lambda: fa.int8_grouped_matmul(a, sa, w, sw[0], offs)),
        (ValueError, lambda: fa.int8_grouped_matmul(a[:0], sa[:0], w, sw, offs, row_ids=offs)),
        (TypeError, lambda: fa.quantize_int8(x.double())),
        (ValueError, lambda: fa.quantize_int8(x[0])),
        (ValueError, lambda: fa.quantize_int8(x.clone().requires_grad_())),
        (ValueError, lambda: fa.swiglu_quantize_int8(x[:, :31])),
        (TypeError, lambda: fa.quantize_int8(x, num_rows=torch.zeros(1, device="cuda"))),
        (ValueError, lambda: fa.quantize_int8(x, num_rows=offs)),
        (TypeError, lambda: fa.quantize_int8(x, q=x)),
        (ValueError, lambda: fa.quantize_int8(x, scale=sa[:2])),
        (ValueError, lambda: fa.quantize_int8(x, scale=sa.clone().requires_grad_())),
    ]
    for n, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            print("not refused:", n)
    assert fa.int8_matmul(a[:0], sa[:0], b, sb).shape == (0, 8)
    assert fa.int8_matmul(a, sa, b[:0], sb[:0]).shape == (4, 0)
    assert fa.int8_grouped_matmul(a[:0], sa[:0], w, sw, offs * 0).shape == (0, 8)
    q, s = fa.quantize_int8(x[:0])
    assert q.shape == (0, 32) and s.shape == (0,)


def test_negated_views():
    """The imaginary part of a conjugate is a view whose sign is changed only when it is read."""
    def neg(v, shape):
        t = torch.full(shape, v * 1j, dtype=torch.complex64, device="cuda").conj().imag  # -v
        assert t.is_neg()
        return t

    q, s = fa.quantize_int8(neg(3.0, (4, 1)))
    assert bool((q == -127).all())
    a, b = torch.ones(1, 16, dtype=torch.int8, device="cuda"), torch.ones(1, 16, dtype=torch.int8, device="cuda")
    two, one = neg(2.0, (1,)), torch.ones(1, device="cuda")
    assert two.is_contiguous()
    f32 = torch.float32
    assert float(fa.int8_matmul(a, two, b, one, out_dtype=f32)) == -32
    assert float(fa.int8_matmul(a, one, b, two, out_dtype=f32)) == -32
    assert float(fa.int8_matmul(a, one, b, one, bias=two, out_dtype=f32)) == 14
    offs = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    assert float(fa.int8_grouped_matmul(a, two, b[None], two[None], offs, out_dtype=f32)) == 64
    with pytest.raises(ValueError, match="negated"):
        fa.int8_matmul(a, one, b, one, out=neg(0.0, (1, 1)))
