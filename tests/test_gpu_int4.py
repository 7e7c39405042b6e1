"""Products with 4-bit weights (flashinfer_amd.int4) against 64-bit formulas:
bit for bit on whole numbers whose sums are exact, and on others within the
roundings of fp32 sums and of the result."""
import pytest
import torch

import flashinfer_amd as fa

pytestmark = pytest.mark.gpu
F64 = torch.float64
TYPES = [torch.bfloat16, torch.float16]
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _q(shape, seed):
    return torch.empty(shape, dtype=torch.int8, device="cuda").random_(-8, 8, generator=_gen(seed))


def _whole(shape, dtype, seed):
    """Whole numbers of -4 .. 4."""
    return torch.empty(shape, device="cuda").random_(-4, 5, generator=_gen(seed)).to(dtype)


def _powers(shape, dtype, seed):
    """1 or 2: with |x| <= 4, |q| <= 8 and K <= 2^17 sums are whole numbers up to 2^23, exact in fp32."""
    return torch.empty(shape, device="cuda").random_(0, 2, generator=_gen(seed)).exp2().to(dtype)


def _dequant(q, scale, group):
    K = q.shape[-1]
    return q.to(F64) * scale.to(F64)[..., torch.arange(K, device="cuda") // group]


def _check(got, x, w, bias=None):
    """Each fp32 sum of K products (exact ones) and of their groups is off by at
    most (K + K / 32 + 2) U of the sum of magnitudes, twice that where the
    matrix cores cut instead of rounding; the scale's product by U; then the
    bias's sum and the last rounding."""
    x = x.to(F64)
    ref, most = torch.matmul(x, w.t()), torch.matmul(x.abs(), w.abs().t())
    if bias is not None:
        ref, most = ref + bias.to(F64), most + bias.to(F64).abs()
    eps = torch.finfo(got.dtype).eps / 2
    before = 2 * U * (1.04 * x.shape[1] + 8) * most
    bound = before * (1 + eps) + ref.abs() * eps + torch.finfo(got.dtype).smallest_normal * eps * 2
    bad = (got.to(F64) - ref).abs() > bound
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


SHAPES = [  # M, N, K
    (1, 1, 1), (1, 16, 128), (1, 4096, 7168), (2, 100, 4096), (3, 17, 33), (5, 64, 128), (8, 2048, 1000),
    (16, 4096, 2048), (17, 130, 1024), (31, 48, 272), (33, 1000, 528), (48, 640, 1536), (64, 256, 7168), (65, 64, 16),
    (100, 7168, 2048), (128, 128, 129), (130, 515, 1040), (200, 4096, 512), (256, 256, 256), (257, 300, 130),
    (300, 264, 784), (511, 513, 96), (600, 1024, 2048), (1024, 2048, 1024), (1111, 999, 408), (2050, 1536, 4096),
    (4097, 31, 160), (2049, 2050, 1101)]


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_exact_sums(shape, group):
    """Whole numbers: every element counts once, whatever the order of the sums."""
    M, N, K = shape
    dtype = TYPES[(M + group // 32) % 2]
    scale_type = torch.float32 if N % 2 else dtype
    q, x = _q((N, K), 1), _whole((M, K), dtype, 2)
    scale = _powers((N, -(-K // group)), scale_type, 3)
    w = fa.pack_int4(q, scale, group)
    assert (w.N, w.K, w.group_size) == (N, K, group) and w.scale.dtype == scale_type
    ref = torch.matmul(x.to(F64), _dequant(q, scale, group).t())
    y = fa.int4_matmul(x, w, out_dtype=torch.float32)
    assert torch.equal(y.to(F64), ref)
    bias = torch.arange(N, device="cuda", dtype=torch.float32) - 7
    assert torch.equal(fa.int4_matmul(x, w, bias=bias, out_dtype=torch.float32).to(F64), ref + bias)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matmul(shape, dtype):
    M, N, K = shape
    group = (32, 64, 128)[(M + K) % 3]
    q = _q((N, K), 1)
    scale = torch.empty(N, -(-K // group), device="cuda").uniform_(0.001, 0.02, generator=_gen(2)).to(dtype)
    x = torch.randn(M, K, generator=_gen(3), device="cuda").to(dtype)
    w, full = fa.pack_int4(q, scale, group), _dequant(q, scale, group)
    y = fa.int4_matmul(x, w)
    assert y.dtype == dtype and y.shape == (M, N)
    _check(y, x, full)
    bias = torch.randn(N, generator=_gen(5), device="cuda").to([torch.bfloat16, torch.float16, torch.float32][M % 3])
    _check(fa.int4_matmul(x, w, bias=bias, out_dtype=torch.float32), x, full, bias)


TILES = range(11)


@pytest.mark.parametrize("tile", TILES)
def test_every_tile(tile, monkeypatch):
    """Each kernel at sizes that are its own and at those that are not."""
    monkeypatch.setenv("MI_INT4_TILE", str(tile))
    for n, (M, N, K) in enumerate(((1, 1, 8), (16, 64, 128), (33, 200, 136), (70, 131, 1000), (300, 400, 776),
                                   (513, 260, 2048), (256, 192, 4104))):
        for group in (32, 64, 128, 512):
            dtype = TYPES[n % 2]
            for scale_type in (dtype, torch.float32):
                q, x = _q((N, K), n), _whole((M, K), dtype, n + 1)
                scale = _powers((N, -(-K // group)), scale_type, n + 2)
                y = fa.int4_matmul(x, fa.pack_int4(q, scale, group), out_dtype=torch.float32)
                assert torch.equal(y.to(F64), torch.matmul(x.to(F64), _dequant(q, scale, group).t())), (M, N, K, group)
                # results of 16 bits are these, rounded; in rows of a multiple of 16 bytes, too
                w = fa.pack_int4(q, scale, group)
                assert torch.equal(fa.int4_matmul(x, w), y.to(dtype))
                bias = torch.arange(N, device="cuda", dtype=torch.float32) - 7
                assert torch.equal(fa.int4_matmul(x, w, bias=bias, out_dtype=torch.bfloat16), (y + bias).bfloat16())
                buf = torch.full((M, -(-N // 8) * 8 + 8), 9.0, dtype=dtype, device="cuda")
                fa.int4_matmul(x, fa.pack_int4(q, scale, group), out=buf[:, :N])
                assert torch.equal(buf[:, :N], y.to(dtype)) and bool((buf[:, N:] == 9).all())


@pytest.mark.parametrize("tile", TILES)
def test_every_tile_grouped(tile, monkeypatch):
    """Tiles of experts that follow each other, gathered and not, some without rows; rows that no expert has."""
    monkeypatch.setenv("MI_INT4_TILE", str(tile))
    counts, N, K, spare = [300, 0, 17, 129, 256, 1], 200, 520, 30
    R, used = sum(counts) + spare, sum(counts)
    offs = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda() + 5
    q, scale = _q((6, N, K), 1), _powers((6, N, 9), torch.float16, 2)
    w = fa.pack_int4(q, scale, 64)
    x = _whole((R + 100, K), torch.float16, 3)
    ids = torch.randint(0, R + 100, (R,), generator=_gen(4), device="cuda", dtype=torch.int32)
    ids[:5], ids[40], ids[-25:] = -1, R + 100, -1
    for rows, table in ((x[:R], None), (x, ids)):
        torch.full((R, N), 9.0, device="cuda")  # a freed block that holds no zeros, for the result to get
        y = fa.int4_grouped_matmul(rows, w, offs, row_ids=table, out_dtype=torch.float32)
        ref = torch.zeros(R, N, dtype=F64, device="cuda")
        src = rows if table is None else rows[table.clamp(0, R + 99).long()]
        lo = 5
        for e, c in enumerate(counts):
            ref[lo:lo + c] = torch.matmul(src[lo:lo + c].to(F64), _dequant(q[e], scale[e], 64).t())
            lo += c
        if table is not None:
            assert bool(y[40].isnan().all())
            y[40] = ref[40] = 0
        assert torch.equal(y.to(F64), ref) and lo == used + 5
        half = torch.full((R, N), 9.0, dtype=torch.float16, device="cuda")
        fa.int4_grouped_matmul(rows, w, offs, row_ids=table, out=half)
        if table is not None:
            assert bool(half[40].isnan().all())
            half[40] = 0
        assert torch.equal(half[5:lo], ref[5:lo].to(torch.float16)) and bool((half[:5] == 9).all() & (half[lo:] == 9).all())


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("shape", [(8200, 4100, 136), (5000, 5555, 264), (33000, 777, 128)], ids=str)
def test_many_large_tiles(shape, group):
    """Several rounds of the largest tiles."""
    M, N, K = shape
    q, x = _q((N, K), 1), _whole((M, K), torch.bfloat16, 2)
    scale = _powers((N, -(-K // group)), torch.bfloat16, 3)
    y = fa.int4_matmul(x, fa.pack_int4(q, scale, group), out_dtype=torch.float32)
    assert torch.equal(y.to(F64), torch.matmul(x.to(F64), _dequant(q, scale, group).t()))


@pytest.mark.parametrize("used", [0, 1, 300, 767, 768, 1500, 3000])
def test_experts_that_have_a_part_of_the_rows(used):
    """The rows that the experts have, which the device alone knows, choose the tile: on both sides of the border."""
    E, N, K, R = 16, 130, 264, 3000
    cuts = torch.linspace(0, used, E + 1).round().to(torch.int32).cuda()
    q, scale, x = _q((E, N, K), 1), _powers((E, N, 3), torch.bfloat16, 2), _whole((R, K), torch.bfloat16, 3)
    torch.full((R, N), 9.0, device="cuda")  # a freed block that holds no zeros, for the result to get
    y = fa.int4_grouped_matmul(x, fa.pack_int4(q, scale), cuts, out_dtype=torch.float32)
    ref = torch.zeros(R, N, dtype=F64, device="cuda")
    for e, (lo, hi) in enumerate(zip(cuts.tolist()[:-1], cuts.tolist()[1:])):
        ref[lo:hi] = torch.matmul(x[lo:hi].to(F64), _dequant(q[e], scale[e], 128).t())
    assert torch.equal(y.to(F64), ref)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_weight_at_every_place(dtype):
    """One-hot rows read the weights back: all 16 values, each place of a tile, clamped ones too."""
    for N, K in ((16, 128), (40, 300)):
        q = (torch.arange(N * K, device="cuda") * 7 % 24 - 12).view(N, K).to(torch.int8)
        w = fa.pack_int4(q, torch.ones(N, -(-K // 32), device="cuda"), 32)
        y = fa.int4_matmul(torch.eye(K, device="cuda", dtype=dtype), w, out_dtype=torch.float32)
        assert torch.equal(y, q.clamp(-8, 7).t().float())


@pytest.mark.parametrize("M", [1, 20, 150, 700])
def test_strides_and_alignment(M):
    N, K = 200, 512
    big = _whole((M, 700), torch.bfloat16, 1)
    q, scale = _q((2 * N, 2 * K), 2), _powers((N, 8), torch.float32, 3)
    for o, ow in ((0, 0), (8, 32), (1, 1), (3, 5)):
        x, part = big[:, o:o + K], q[1::2, ow:ow + K]
        w = fa.pack_int4(part, scale, 64)
        assert all(torch.equal(a, b) for a, b in zip(w[:2], fa.pack_int4(part.contiguous(), scale, 64)[:2]))
        ref = torch.matmul(x.to(F64), _dequant(part, scale, 64).t())
        y = fa.int4_matmul(x, w, out_dtype=torch.float32)
        assert torch.equal(y.to(F64), ref)
    assert torch.equal(fa.int4_matmul(x.t().contiguous().t(), w, out_dtype=torch.float32), y)
    assert torch.equal(fa.int4_matmul(x[:1].expand(M, K), w, out_dtype=torch.float32), y[:1].expand(M, N))
    for pad in (8, 3):  # a destination inside a wider one
        buf = torch.full((M, N + 2 * pad), 5.0, device="cuda")
        out = fa.int4_matmul(x, w, out=buf[:, pad:pad + N])
        assert torch.equal(out, y) and torch.equal(buf[:, pad:pad + N], y)
        assert bool((buf[:, :pad] == 5).all()) and bool((buf[:, pad + N:] == 5).all())


# rows of each expert, tokens (0: rows of x directly), N, K, spare rows behind the last
GROUPS = [([1], 0, 64, 128, 0), ([0, 0, 3], 0, 16, 64, 2), ([5, 0, 1, 0, 64, 65], 0, 130, 272, 7),
          ([1] * 40, 13, 256, 1024, 8), ([2, 0, 5, 1] * 8, 64, 4096, 2048, 100), ([0] * 5, 4, 64, 64, 9),
          ([300, 0, 17, 129, 256, 1], 500, 512, 640, 30), ([257], 100, 300, 1041, 1), ([1000, 3, 500], 0, 768, 2048, 0),
          ([0, 2500, 0, 40], 1024, 1024, 512, 64), ([2] * 1024, 0, 33, 48, 1), ([70] * 32, 300, 512, 1536, 5)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", GROUPS, ids=lambda c: f"{len(c[0])}x{sum(c[0])}-{c[1]}-{c[2]}-{c[3]}")
def test_grouped(case, dtype):
    counts, tokens, N, K, spare = case
    E, R, used = len(counts), sum(counts) + spare, sum(counts)
    offs = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()
    M = tokens or R
    group = (32, 64, 128)[E % 3]
    q, x = _q((E, N, K), 1), _whole((M, K), dtype, 2)
    scale = _powers((E, N, -(-K // group)), dtype, 3)
    w = fa.pack_int4(q, scale, group)
    ids = torch.randint(0, M, (R,), generator=_gen(5), device="cuda", dtype=torch.int32) if tokens else None
    if tokens:
        ids[used:] = -1  # not read
    y = fa.int4_grouped_matmul(x, w, offs, row_ids=ids, out_dtype=torch.float32)
    assert y.shape == (R, N) and not y[used:].any()
    lo = 0
    for e, c in enumerate(counts):
        src = ids[lo:lo + c].long() if tokens else slice(lo, lo + c)
        ref = torch.matmul(x[src].to(F64), _dequant(q[e], scale[e], group).t())
        assert torch.equal(y[lo:lo + c].to(F64), ref), e
        lo += c
    one = fa.Int4Weights(w.packed[-1], w.scale[-1], *w[2:])  # an expert's slice is a dense layer's
    assert torch.equal(fa.int4_matmul(x[:1], one, out_dtype=torch.float32).to(F64),
                       torch.matmul(x[:1].to(F64), _dequant(q[-1], scale[-1], group).t()))
    buf = torch.full((R, N), 9.0, dtype=dtype, device="cuda")
    fa.int4_grouped_matmul(x, w, offs, row_ids=ids, out=buf)
    assert torch.equal(buf[:used], y[:used].to(dtype)) and bool((buf[used:] == 9).all())


@pytest.mark.parametrize("R", [12, 700])
def test_tables_that_leave_rows_out(R):
    """Rows before the first expert, entries past the end and below 0, ids that are no rows."""
    N, K = 80, 256
    q, x, scale = _q((3, N, K), 1), _whole((R, K), torch.float16, 2), _powers((3, N, 2), torch.float32, 3)
    w = fa.pack_int4(q, scale)
    a, b = R // 4, R // 2
    offs = torch.tensor([a, a, b, R + 100], dtype=torch.int32, device="cuda")
    torch.full((R, N), 9.0, device="cuda")  # a freed block that holds no zeros, for the result to get
    y = fa.int4_grouped_matmul(x, w, offs, out_dtype=torch.float32)
    ref = torch.zeros(R, N, dtype=F64, device="cuda")
    for e, (lo, hi) in ((1, (a, b)), (2, (b, R))):
        ref[lo:hi] = torch.matmul(x[lo:hi].to(F64), _dequant(q[e], scale[e], 128).t())
    assert torch.equal(y.to(F64), ref)
    offs = torch.tensor([-5, a, b, b], dtype=torch.int32, device="cuda")
    ids = torch.arange(R, dtype=torch.int32, device="cuda")
    ids[1], ids[2] = R, -1
    y = fa.int4_grouped_matmul(x, w, offs, row_ids=ids, out_dtype=torch.float32)
    assert bool(y[1:3].isnan().all()) and not y[b:].any()
    assert torch.equal(y[0].to(F64), torch.matmul(x[0].to(F64), _dequant(q[0], scale[0], 128).t()))


@pytest.mark.parametrize("M", [4, 40, 300])
def test_values_that_are_not_finite(M):
    """Those of a row stay in it, those of a scale in its channel, and infinities times whole numbers keep their signs."""
    N, K = 72, 640
    x = _whole((M, K), torch.bfloat16, 1)
    q = _q((N, K), 2)
    q[q == 0] = 1
    scale = torch.ones(N, 5, device="cuda")
    scale[7, 2] = float("nan")
    x[0, 5], x[1, 639] = float("inf"), float("nan")
    y = fa.int4_matmul(x, fa.pack_int4(q, scale), out_dtype=torch.float32)
    keep = torch.arange(N, device="cuda") != 7
    assert torch.equal(y[0, keep], float("inf") * q[keep, 5].float()) and bool(y[1].isnan().all())
    assert bool(y[:, 7].isnan().all()) and bool(y[2:, keep].isfinite().all())
    # past K in a copied row: nothing of its neighbour
    x = _whole((M, 131), torch.bfloat16, 1)
    x[1:] = float("inf")
    y = fa.int4_matmul(x[:, :129], fa.pack_int4(q[:, :129], scale[:, :2]), out_dtype=torch.float32)
    assert torch.equal(y[0].to(F64), torch.matmul(x[:1, :129].to(F64), q[:, :129].to(F64).t())[0])


@pytest.mark.parametrize("M", [3, 16, 70, 600])
def test_small_values(M):
    """float16 below its normal range (its steps of 2^-24), bfloat16 far below 1: multiplied as they are."""
    N, K = 200, 256
    q, one = _q((N, K), 1), torch.ones(N, 2, device="cuda")
    w = fa.pack_int4(q, one)
    for dtype, unit in ((torch.float16, 2.0 ** -24), (torch.bfloat16, 2.0 ** -100)):
        x = (_whole((M, K), torch.float32, 2) * unit).to(dtype)
        assert x.any()
        y = fa.int4_matmul(x, w, out_dtype=torch.float32)
        assert torch.equal(y.to(F64), torch.matmul(x.to(F64), q.to(F64).t()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_quantize(dtype):
    for shape, group in (((40, 200), 32), ((3, 17, 1000), 128), ((5, 64), 4096), ((1, 1), 32)):
        w = torch.randn(shape, generator=_gen(1), device="cuda").to(dtype)
        w.view(-1)[0] = 0.0
        got = fa.quantize_int4(w, group)
        K = shape[-1]
        parts = [w[..., i:i + group].float() for i in range(0, K, group)]
        # in 64 bits and rounded: torch multiplies fp32 by the reciprocal of a number
        scale = torch.stack([(p.abs().amax(-1).clamp_min(1e-10).to(F64) / 7).float() for p in parts], dim=-1)
        q = torch.cat([torch.round(p / scale[..., i:i + 1]) for i, p in enumerate(parts)], dim=-1).to(torch.int8)
        same = fa.pack_int4(q, scale, group)
        equal = torch.equal(got.packed, same.packed), torch.equal(got.scale, same.scale), got[2:] == same[2:]
        assert all(equal), equal
    w[:] = 0
    assert not fa.quantize_int4(w).packed.any()
    w = torch.randn(4, 256, generator=_gen(1), device="cuda").to(dtype)
    w[1, 3], w[2, 200] = float("nan"), float("-inf")
    scale = fa.quantize_int4(w).scale
    assert scale.shape == (2, 16) and not scale[:, 4:].any()
    bad = ~scale[:, :4].isfinite()
    assert bad.tolist() == [[False, True, False, False], [False, False, True, False]]
    wide = torch.randn(9, 300, generator=_gen(2), device="cuda").to(dtype)  # strides
    a, b = fa.quantize_int4(wide[1::2, 3:].t(), 64), fa.quantize_int4(wide[1::2, 3:].t().contiguous(), 64)
    assert torch.equal(a.packed, b.packed) and torch.equal(a.scale, b.scale)


def test_rows_past_32_bits():
    """Gathered rows that start 4 GiB and more into x, and results past 2^31 elements."""
    wide = torch.zeros(70000, 32768, dtype=torch.bfloat16, device="cuda")
    x, ids = wide[:, :264], torch.tensor([0, 65535, 65536, 69999, 5], dtype=torch.int32, device="cuda")
    x[ids.long()] = _whole((5, 264), torch.bfloat16, 1)
    q, scale = _q((2, 40, 264), 2), _powers((2, 40, 3), torch.float32, 3)
    w, offs = fa.pack_int4(q, scale), torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    for tiles in (1, 60):  # few rows, and many
        table = ids.repeat_interleave(tiles)
        y = fa.int4_grouped_matmul(x, w, offs * tiles, row_ids=table, out_dtype=torch.float32)
        for e, (lo, hi) in enumerate(((0, 2 * tiles), (2 * tiles, 5 * tiles))):
            ref = torch.matmul(x[table[lo:hi].long()].to(F64), _dequant(q[e], scale[e], 128).t())
            assert torch.equal(y[lo:hi].to(F64), ref)
    del wide, x
    M, N = 70000, 32768
    x = _whole((M, 8), torch.float16, 1)
    q = _q((N, 8), 2)
    y = fa.int4_matmul(x, fa.pack_int4(q, torch.ones(N, 1, device="cuda"), 32))
    for rows in (slice(0, 100), slice(65500, 65600), slice(M - 100, M)):
        assert torch.equal(y[rows].to(F64), torch.matmul(x[rows].to(F64), q.to(F64).t()))


def test_graph_replays_and_streams():
    """Captured with a copy of unaligned rows: every replay equals the eager result, two graphs keep apart."""
    R, N, K = 50, 96, 330
    q, scale = _q((4, N, K), 1), _powers((4, N, 11), torch.float32, 2)
    w = fa.pack_int4(q, scale, 32)
    made = []
    for seed in (3, 4):
        x = _whole((R, K + 1), torch.bfloat16, seed)
        offs = torch.tensor([0, 10, 10, 30, 45], dtype=torch.int32, device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fa.int4_grouped_matmul(x[:, 1:], w, offs)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fa.int4_grouped_matmul(x[:, 1:], w, offs)
        made.append((graph, x, offs, y))
    for rep in range(3):
        for n, (graph, x, offs, y) in enumerate(made):
            x.copy_(_whole(x.shape, x.dtype, 10 * rep + n))
            offs[1] = 5 + rep
        for graph, *_ in made:
            graph.replay()
        torch.cuda.synchronize()
        for graph, x, offs, y in made:
            assert torch.equal(y, fa.int4_grouped_matmul(x[:, 1:], w, offs))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        z = fa.int4_grouped_matmul(x[:, 1:], w, offs)
    s.synchronize()
    assert torch.equal(z, y)


def test_refusals():
    x = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)
    q, scale = _q((8, 64), 1), torch.ones(8, 2, device="cuda")
    w = fa.pack_int4(q, scale, 32)
    we = fa.pack_int4(q[None], scale[None], 32)
    offs = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    leaf = x.clone().requires_grad_()
    out = torch.zeros(4, 8, device="cuda", dtype=torch.bfloat16)
    buf = torch.zeros(4, 64 + 8, device="cuda", dtype=torch.bfloat16)
    bad = [
        (TypeError, lambda: fa.int4_matmul(x.float(), w)), (ValueError, lambda: fa.int4_matmul(x[:, :63], w)),
        (ValueError, lambda: fa.int4_matmul(x[0], w)), (ValueError, lambda: fa.int4_matmul(x.cpu(), w)),
        (ValueError, lambda: fa.int4_matmul(x, we)), (ValueError, lambda: fa.int4_grouped_matmul(x, w, offs)),
        (ValueError, lambda: fa.int4_matmul(x, w._replace(N=24))), (ValueError, lambda: fa.int4_matmul(x, w._replace(K=200))),
        (ValueError, lambda: fa.int4_matmul(x, w._replace(group_size=48))),
        (ValueError, lambda: fa.int4_matmul(x, w._replace(group_size=64))),
        (TypeError, lambda: fa.int4_matmul(x, w._replace(scale=w.scale.half()))),
        (ValueError, lambda: fa.int4_matmul(x, w._replace(packed=w.packed.cpu()))),
        (ValueError, lambda: fa.int4_matmul(x, w, bias=torch.zeros(7, device="cuda"))),
        (TypeError, lambda: fa.int4_matmul(x, w, bias=torch.zeros(8, device="cuda", dtype=torch.int32))),
        (TypeError, lambda: fa.int4_matmul(x, w, out_dtype=torch.float64)),
        (ValueError, lambda: fa.int4_matmul(x, w, out=out[:3])), (ValueError, lambda: fa.int4_matmul(leaf, w)),
        (ValueError, lambda: fa.int4_matmul(x, w._replace(scale=w.scale.clone().requires_grad_()))),
        (ValueError, lambda: fa.int4_matmul(buf[:, :64], w, out=buf[:, 60:68])),
        (TypeError, lambda: fa.int4_grouped_matmul(x, we, offs.long())),
        (ValueError, lambda: fa.int4_grouped_matmul(x, we, offs[:1])),
        (TypeError, lambda: fa.int4_grouped_matmul(x, we, offs, row_ids=offs.long())),
        (ValueError, lambda: fa.int4_grouped_matmul(x[:0], we, offs, row_ids=offs)),
        (TypeError, lambda: fa.pack_int4(q.float(), scale, 32)), (ValueError, lambda: fa.pack_int4(q, scale, 64)),
        (ValueError, lambda: fa.pack_int4(q, scale, 48)), (ValueError, lambda: fa.pack_int4(q, scale, 16)),
        (ValueError, lambda: fa.pack_int4(q[:0], scale[:0], 32)), (ValueError, lambda: fa.pack_int4(q[0], scale[0], 32)),
        (TypeError, lambda: fa.quantize_int4(q)), (ValueError, lambda: fa.quantize_int4(leaf)),
    ]
    for n, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            print("not refused:", n)
    # columns of one buffer side by side are no overlap; nothing to do is no error
    assert not fa.int4_matmul(buf[:, :64], w, out=buf[:, 64:]).any()
    assert fa.int4_matmul(x[:0], w).shape == (0, 8)
    assert fa.int4_grouped_matmul(x, we, offs, row_ids=offs[:0]).shape == (0, 8)
    with torch.no_grad():
        assert not fa.int4_matmul(leaf, w).any()
