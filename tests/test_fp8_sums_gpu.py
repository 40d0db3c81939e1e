"""How the 8-bit product adds up (w2c_matmul_fp8, w2c_matmul_fp8_fast), on numbers whose sums show every lost bit.

Exact by construction: products and all their partial sums, in any order, are whole multiples of one unit below 2^24 of it, so an f32 sum has no rounding and
the output is the sum rounded once to its type.  `fast` cuts products below 2^-13 of the largest of 8 neighbours: exact where all of a block of
128 have one magnitude.

On normal data: with -sum as the bias the output is the error itself.  A default sum makes at most one rounding of U = 2^-24 for each 16 products added, independent
ones: sqrt(K / 16) U of the running sum's norm, below 2^-20 for K up to 4096, and the bias's own rounding U.  Of `fast` the header says about
1.5e-5 of the norm; twice that, 2^-15, is the bound."""
import pytest
import torch

from multiagentperception_amd import ops, train_ops
from multiagentperception_amd._native import W2CError

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu

# up to 24 rows, blocks of 4 and of 16 waves; then the three tiles; rows of scales that are whole dwords and others; reductions in parts
SHAPES = [(1, 33, 512), (16, 100, 640), (17, 257, 128), (24, 40, 4100), (5, 50, 2048), (1, 4096, 8192), (9, 120, 7200), (24, 40, 8200), (25, 65, 1500), (130, 259, 512), (40, 100, 8192), (33, 65, 8200), (1000, 700, 4096),
          (1900, 1910, 384), (1900, 1910, 512), (3300, 3200, 384), (3300, 3200, 512)]


def _blocks(values, exponents, cols):
    """values f32 [R, cols] that e4m3 holds exactly, exponents [R or ceil(R / 128), ceil(cols / 128)]"""
    codes = torch.nn.functional.pad(values, (0, -cols % 128)).to(E4M3)
    return ops.Fp8Blocks(codes.cuda(), (exponents + 127).to(torch.uint8).view(E8M0).cuda(), cols)


def _signs(g, *shape):
    return torch.randint(0, 2, shape, generator=g).float() * 2 - 1


def _product(va, vb):
    """va [M, K], vb [N, K] small multiples of one unit: exact in f64 in any order"""
    return (va.double().cuda() @ vb.double().t().contiguous().cuda()).cpu()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_small_products_beside_large_ones_that_cancel(M, N, K, dtype):
    """pairs of +-64 that add to nothing among products of 2^-9: at most 400 of the former, so sums stay below 400 * 64 + K 2^-9 < 2^24 2^-9"""
    g = torch.Generator().manual_seed(M + N + K)
    k = torch.arange(K)
    pair = (k % 8 < 2) & (k < 1600) & (k - k % 2 + 1 < K)
    b = _signs(g, N, K)
    b[:, 1::2] = torch.where(pair[1::2], b[:, :K - K % 2:2], b[:, 1::2])          # both of a pair meet the same sign
    small = _signs(g, M, K) * (torch.rand(M, K, generator=g) < 0.7) * 2.0 ** -9
    large = _signs(g, M, 1) * torch.where(k % 2 == 0, 64.0, -64.0)
    a = torch.where(pair, large, small)
    rows, cols = torch.arange(M) % 5, torch.arange(-(-N // 128)) % 3
    blocks = -(-K // 128)
    qa = _blocks(a, rows[:, None].expand(M, blocks).contiguous(), K)
    qb = _blocks(b, cols[:, None].expand(len(cols), blocks).contiguous(), K)
    unit = 2.0 ** rows[:, None].double() * 2.0 ** cols.repeat_interleave(128)[:N].double()
    want = (_product(a, b) * unit).to(F32).to(dtype)
    assert want.any() and torch.equal(ops.matmul_fp8(qa, qb, out_dtype=dtype).cpu(), want)


@pytest.mark.parametrize("fast", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_every_product_is_in_the_sum_once(M, N, K, dtype, fast):
    """products of 0 and +-1 times a block's 1, 2 or 4: whole numbers below 2^15"""
    g = torch.Generator().manual_seed(M + N + K + 1)
    a, b = torch.randint(-1, 2, (M, K), generator=g).float(), _signs(g, N, K)
    blocks = -(-K // 128)
    ea, eb = torch.randint(0, 2, (M, blocks), generator=g), torch.randint(0, 2, (N, blocks), generator=g)
    bias = torch.randint(-8, 9, (N,), generator=g).float()
    va, vb = (v * (2.0 ** e).repeat_interleave(128, 1)[:, :K] for v, e in ((a, ea), (b, eb)))
    want = (_product(va, vb) + bias).to(F32).to(dtype)
    assert torch.equal(ops.matmul_fp8(_blocks(a, ea, K), _blocks(b, eb, K), bias.cuda(), dtype, fast=fast).cpu(), want)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,N,K", [(1, 4000, 1024), (20, 3000, 4096), (64, 3000, 2000), (200, 40000, 1024), (2500, 4500, 500)])
def test_error_against_the_norm(M, N, K, dtype):
    """all rows of a alike, the bias their exact result negated: what comes out is the error of each element"""
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randn(1, K, generator=g, device="cuda").expand(M, K).contiguous()
    a, b = ops.quantize_fp8(x).rows, ops.quantize_fp8(torch.randn(N, K, generator=g, device="cuda"), 128).rows
    value = lambda t, tile: t.codes.cpu().double() * t.scale.cpu().double().repeat_interleave(tile, 0)[:t.codes.shape[0]].repeat_interleave(128, 1)     # noqa: E731
    want = (value(b, 128).cuda() @ value(a, 1)[0].cuda()).float()
    norm = float(want.double().norm()) * M ** 0.5
    for fast, bound in ((False, 2.0 ** -20), (True, 2.0 ** -15)):
        y = ops.matmul_fp8(a, b, -want, dtype, fast=fast)
        off = float(y.double().norm()) / norm
        print(M, N, K, dtype, "fast" if fast else "default", off, flush=True)
        assert off <= bound


def test_f32_outputs_are_the_same_with_and_without_fast():
    g = torch.Generator(device="cuda").manual_seed(1)
    for M in (9, 300):
        a, b = ops.quantize_fp8(torch.randn(M, 700, generator=g, device="cuda")).rows, ops.quantize_fp8(torch.randn(90, 700, generator=g, device="cuda")).rows
        assert torch.equal(ops.matmul_fp8(a, b, out_dtype=F32), ops.matmul_fp8(a, b, out_dtype=F32, fast=True))


def test_linear_layer_hands_fast_to_its_three_products():
    g = torch.Generator(device="cuda").manual_seed(2)
    x, dy = torch.randn(70, 400, generator=g, device="cuda", dtype=BF16), torch.randn(70, 300, generator=g, device="cuda", dtype=BF16)
    for fast in (False, True):
        m = train_ops.LinearFp8(400, 300, fast=fast, device="cuda", dtype=BF16)
        with torch.no_grad():
            m.weight.copy_(torch.randn(300, 400, generator=torch.Generator().manual_seed(3)))
        t = x.clone().requires_grad_()
        y = m(t)
        dx, dw = torch.autograd.grad(y, (t, m.weight), dy)
        qx, qw, qy = ops.quantize_fp8(x, columns=True), ops.quantize_fp8(m.weight.detach(), 128, columns=True), ops.quantize_fp8(dy, columns=True)
        assert torch.equal(y, ops.matmul_fp8(qx.rows, qw.rows, m.bias.detach().float(), BF16, fast))
        assert torch.equal(dx, ops.matmul_fp8(qy.rows, qw.columns, None, BF16, fast)) and torch.equal(dw, ops.matmul_fp8(qy.columns, qx.columns, None, BF16, fast))
        with torch.no_grad():
            assert torch.equal(train_ops.linear_fp8(x, qw.rows, m.bias, fast), y)


def test_the_fast_entry_refuses_f32():
    from multiagentperception_amd import _native
    p = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    a = p.data_ptr()
    assert _native.lib().w2c_matmul_fp8_fast(a, a, 1, a, a, 1, 8, 8, 128, 0, a, 0, 0, 0, 0) == -1
