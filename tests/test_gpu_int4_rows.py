"""Products with 4-bit weights on both sides of the borders between tiles, and of
as many rows as a call can have: 32 bits hold their number, and not much more.
There every row is one row of x at distance 0, so that results alone take
memory."""
import pytest
import torch

import flashinfer_amd as fa

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _equal_everywhere(y, value):
    return all(bool((part == value).all()) for part in y.view(-1).split(1 << 28))


@pytest.mark.parametrize("rows", [2139127681, 2147483391, 2147483647])
def test_dense_rows_up_to_32_bits(rows):
    """From the first number of rows that passes 31 bits with their 8355968 tiles of 256 added."""
    K = 32
    x = torch.arange(-5, K - 5, device="cuda").to(torch.bfloat16)[None]
    q = torch.full((1, K), 3, dtype=torch.int8, device="cuda")
    w = fa.pack_int4(q, torch.full((1, 1), 0.5, device="cuda"), 32)
    out = torch.full((rows, 1), float("nan"), dtype=torch.bfloat16, device="cuda")
    fa.int4_matmul(x.expand(rows, K), w, out=out)
    assert _equal_everywhere(out, 504.0)  # 1.5 times the sum of -5 .. 26, exact in bfloat16


@pytest.mark.parametrize("rows", [2147483633, 2147483647])
def test_an_expert_with_rows_up_to_32_bits(rows):
    """From the first number of rows that passes 31 bits with 15 added."""
    K = 32
    x = torch.arange(-5, K - 5, device="cuda").to(torch.bfloat16)[None]
    q = torch.full((1, 1, K), 3, dtype=torch.int8, device="cuda")
    w = fa.pack_int4(q, torch.full((1, 1, 1), 0.5, device="cuda"), 32)
    out = torch.full((rows, 1), float("nan"), dtype=torch.bfloat16, device="cuda")
    fa.int4_grouped_matmul(x.expand(rows, K), w, torch.tensor([0, rows], dtype=torch.int32, device="cuda"), out=out)
    assert _equal_everywhere(out, 504.0)


# rows, channels: the last of a tile and the first of the next
BORDERS = [(64, 2048), (65, 2048), (128, 4096), (129, 4096), (256, 4096), (257, 4096), (160, 6144), (161, 6144),
           (144, 7168), (145, 7168), (204, 4700), (512, 2048), (513, 2048), (1024, 2048), (1025, 2048),
           (1536, 4096), (1537, 4096), (2048, 2048)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", BORDERS, ids=str)
def test_borders_between_tiles(shape, group):
    """Whole numbers: every element counts once, whatever the order of the sums."""
    (M, N), K = shape, 264
    dtype = torch.bfloat16 if M % 2 else torch.float16
    g = torch.Generator(device="cuda").manual_seed(M)
    q = torch.empty((N, K), dtype=torch.int8, device="cuda").random_(-8, 8, generator=g)
    x = torch.empty((M, K), device="cuda").random_(-4, 5, generator=g).to(dtype)
    scale = torch.empty((N, -(-K // group)), device="cuda").random_(0, 2, generator=g).exp2()
    y = fa.int4_matmul(x, fa.pack_int4(q, scale, group), out_dtype=torch.float32)
    w = q.double() * scale.double()[:, torch.arange(K, device="cuda") // group]
    assert torch.equal(y.double(), torch.matmul(x.double(), w.t()))


@pytest.mark.parametrize("used", [0, 800, 1279, 1280, 1281, 2999])
def test_experts_on_both_sides_of_the_large_tiles(used):
    """80 rows of an expert on average: the rows that the experts have, which the device alone knows, choose."""
    E, N, K, R = 16, 130, 264, 3000
    cuts = torch.linspace(0, used, E + 1).round().to(torch.int32).cuda()
    g = torch.Generator(device="cuda").manual_seed(used)
    q = torch.empty((E, N, K), dtype=torch.int8, device="cuda").random_(-8, 8, generator=g)
    x = torch.empty((R, K), device="cuda").random_(-4, 5, generator=g).to(torch.bfloat16)
    scale = torch.empty((E, N, 3), device="cuda").random_(0, 2, generator=g).exp2()
    torch.full((R, N), 9.0, device="cuda")  # a freed block that holds no zeros, for the result to get
    y = fa.int4_grouped_matmul(x, fa.pack_int4(q, scale), cuts, out_dtype=torch.float32)
    w = q.double() * scale.double()[..., torch.arange(K, device="cuda") // 128]
    ref = torch.zeros(R, N, dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(zip(cuts.tolist()[:-1], cuts.tolist()[1:])):
        ref[lo:hi] = torch.matmul(x[lo:hi].double(), w[e].t())
    assert torch.equal(y.double(), ref)
