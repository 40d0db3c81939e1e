"""The 8-bit block-scaled product and its quantiser (w2c_matmul_fp8, w2c_quantize_fp8) against their definitions in 64 bits.

Tolerances: U = 2^-24.  Codes and scales are exact by definition, so they must be equal.  A product of two codes is exact in f32; the sum of K of them is off by at
most K roundings of the running sum, which is bounded by the sum of magnitudes S: K U S.  bf16 and f16 outputs come from the scaled 8-bit matrix instructions,
which cut products below 2^-13 of the largest of their group of 8: at most 7 of a group lose less than 2^-13 of its largest, and the groups' largest add up to
at most S, so 7 2^-13 S more.  The output adds half a step of its type."""
import pytest
import torch

from multiagentperception_amd import ops, train_ops
from multiagentperception_amd._native import W2CError

pytestmark = pytest.mark.gpu
U, CUT = 2.0 ** -24, 7 * 2.0 ** -13
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _value(t):
    """Fp8Blocks -> f64 on the CPU, exactly (both are finite sets of numbers with few bits)"""
    codes, scale = t.codes.cpu().double(), t.scale.cpu().double()
    tile = 1 if scale.shape[0] == codes.shape[0] else 128
    return codes * scale.repeat_interleave(tile, 0)[:codes.shape[0]].repeat_interleave(128, 1)


def _reference(x, tile):
    """x f64 CPU [R, C] -> (values, scales as biased exponents)"""
    R, C = x.shape
    pr, pc = -R % tile, -C % 128
    fin = torch.where(x.isfinite(), x, torch.zeros_like(x))
    t = torch.nn.functional.pad(fin, (0, pc, 0, pr)).view((R + pr) // tile, tile, (C + pc) // 128, 128)
    amax = t.abs().amax((1, 3))
    m, e = torch.frexp(amax / 448.0)                      # amax / 448 = m 2^e, m in [0.5, 1)
    e = torch.where(m == 0.5, e - 1, e)                   # an exact power of two is its own scale
    e = torch.where(amax == 448.0 * torch.ldexp(torch.ones_like(amax), e), e, e)
    e = torch.where(amax > 0, e.clamp(-127, 127), torch.zeros_like(e))
    unit = torch.ldexp(torch.ones_like(amax), e).repeat_interleave(tile, 0)[:R].repeat_interleave(128, 1)[:, :C]
    u = fin / unit
    step = torch.ldexp(torch.ones_like(u), (torch.frexp(u)[1] - 1).clamp(min=-6) - 3)
    q = torch.round(u / step) * step * unit
    return torch.where(x.isfinite(), q, torch.full_like(q, float("nan"))), (e + 127).to(torch.uint8)


def _same(a, b):
    return bool(torch.equal(a.isnan(), b.isnan())) and bool(torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0)))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tile", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1), (3, 130), (128, 128), (129, 127), (300, 500), (77, 1025), (1000, 64)])
def test_quantiser(shape, tile, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape[0], 1, generator=g))).to(dtype)
    x[0, 0] = 0.0
    if shape[0] > 4:
        x[2] = 0.0                                            # a block of zeros
        x[3, :] = 448.0                                       # exactly the largest code
    q = ops.quantize_fp8(x.cuda(), tile, rows=True, columns=True, sums=True)
    for t, ref in ((q.rows, x.double()), (q.columns, x.double().t().contiguous())):
        v, s = _reference(ref, tile)
        assert torch.equal(t.scale.cpu().view(torch.uint8), s)
        assert _same(_value(t)[:, :ref.shape[1]], v) and not _value(t)[:, ref.shape[1]:].any()
    S = x.double().abs().sum(0)
    assert ((q.sums.cpu().double() - x.double().sum(0)).abs() <= (shape[0] + 1) * U * S).all()
    only = ops.quantize_fp8(x.cuda(), tile)
    assert only.columns is None and only.sums is None and torch.equal(only.rows.codes.view(torch.uint8), q.rows.codes.view(torch.uint8))


def test_quantiser_extremes_and_what_is_not_finite():
    x = torch.zeros(6, 256)
    x[0, :4] = torch.tensor([1e-45, -3e-42, 1e-38, 0.0])      # subnormal f32: the scale stops at 2^-127
    x[1, :3] = torch.tensor([3.4028234663852886e38, 1.0, -1e30])
    x[2, :4] = torch.tensor([float("nan"), 2.0, float("inf"), -float("inf")])
    x[3, 128:] = float("nan")
    x[4, :3] = torch.tensor([449.0, 1.0, 0.9])
    for tile in (1, 128):
        q = ops.quantize_fp8(x.cuda(), tile, columns=True)
        for t, ref in ((q.rows, x.double()), (q.columns, x.double().t().contiguous())):
            v, s = _reference(ref, tile)
            assert torch.equal(t.scale.cpu().view(torch.uint8), s) and _same(_value(t)[:, :ref.shape[1]], v)


def test_quantiser_reads_rows_of_a_wider_tensor():
    x = torch.randn(50, 300, device="cuda", dtype=BF16)
    a, b = ops.quantize_fp8(x[:, 3:200], columns=True), ops.quantize_fp8(x[:, 3:200].contiguous(), columns=True)
    for p, q in zip(a[:2], b[:2]):
        assert torch.equal(p.codes.view(torch.uint8), q.codes.view(torch.uint8)) and torch.equal(p.scale.view(torch.uint8), q.scale.view(torch.uint8))


def _operands(M, N, K, b_tile, seed, a_tile=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
    w = torch.randn(N, K, generator=g) * torch.exp(torch.randn(N, 1, generator=g))
    return ops.quantize_fp8(x.cuda(), a_tile).rows, ops.quantize_fp8(w.cuda(), b_tile).rows, torch.randn(N, generator=g)


def _check(M, N, K, b_tile=1, dtype=F32, bias=False, a_tile=1):
    a, b, c = _operands(M, N, K, b_tile, M + N + K, a_tile)
    y = ops.matmul_fp8(a, b, c.cuda() if bias else None, dtype)
    va, vb = _value(a).cuda(), _value(b).t().contiguous().cuda()
    want, S = va @ vb, va.abs() @ vb.abs()
    if bias:
        want, S = want + c.double().cuda(), S + c.double().abs().cuda()
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    tol = half * want.abs() + (1 + half) * ((K + 1) * U + (CUT if dtype != F32 else 0)) * S + (2.0 ** -25 if dtype == F16 else 0)
    assert y.shape == (M, N) and y.dtype == dtype
    assert ((y.double() - want).abs() <= tol).all(), float(((y.double() - want).abs() - tol).max())
    return y


@pytest.mark.parametrize("K", [1, 128, 300, 640, 1900])
@pytest.mark.parametrize("M,N", [(1, 1), (1, 33), (16, 16), (17, 100), (31, 257), (33, 40), (64, 129), (65, 1), (128, 128), (130, 259), (257, 511)])
def test_product(M, N, K):
    _check(M, N, K)
    _check(M, N, K, b_tile=128, dtype=BF16, bias=True)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_product_on_large_tiles(dtype):
    _check(3300, 3200, 384, b_tile=128, dtype=dtype, bias=True)
    _check(3073, 3333, 700, b_tile=1, dtype=dtype)


def test_both_operands_with_tile_scales_and_a_long_reduction():
    _check(300, 200, 5000, b_tile=128, a_tile=128)
    _check(7, 200, 5000, b_tile=128, a_tile=128)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,N,K", [(40, 100, 8192), (33, 65, 8200), (1000, 700, 4100), (1000, 700, 2000)])
def test_a_long_reduction_in_parts(M, N, K, dtype):
    _check(M, N, K, b_tile=128, dtype=dtype, bias=True)


def test_a_nan_stays_in_its_row_or_column_and_a_scale_can_be_nan():
    a, b, _ = _operands(200, 300, 256, 1, 1)
    clean = ops.matmul_fp8(a, b, None, F32)
    a.codes.view(torch.uint8)[5, 17] = 0x7F
    b.scale.view(torch.uint8)[9, 1] = 255
    y = ops.matmul_fp8(a, b, None, F32)
    bad = torch.zeros(200, 300, dtype=torch.bool, device="cuda")
    bad[5], bad[:, 9] = True, True
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], clean[~bad])
    few = ops.matmul_fp8(ops.Fp8Blocks(a.codes[:8], a.scale[:8], 256), b, None, F32)
    assert torch.equal(few.isnan(), bad[:8])


def test_the_same_bits_every_time():
    for M in (9, 300):
        a, b, _ = _operands(M, 500, 2000, 128, M)
        assert torch.equal(ops.matmul_fp8(a, b), ops.matmul_fp8(a, b))


@pytest.mark.parametrize("dtype,wtype", [(BF16, F32), (F32, F32), (F16, F16)])
@pytest.mark.parametrize("shape,N", [((5, 100), 70), ((2, 90, 300), 257), ((1, 16), 1), ((300, 129), 128)])
def test_linear_layer_and_its_gradients(shape, N, dtype, wtype):
    g = torch.Generator().manual_seed(N)
    K = shape[-1]
    x = torch.randn(shape, generator=g).to(dtype).cuda().requires_grad_()
    w = torch.randn(N, K, generator=g).to(wtype).cuda().requires_grad_()
    b = torch.randn(N, generator=g).cuda().requires_grad_()
    dy = torch.randn(shape[:-1] + (N,), generator=g).to(dtype).cuda()
    y = train_ops.linear_fp8(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x2, dy2 = x.detach().double().reshape(-1, K).cpu(), dy.double().reshape(-1, N).cpu()
    q = lambda t, tile: _reference(t.contiguous(), tile)[0]                        # noqa: E731
    wq = q(w.detach().double().cpu(), 128)

    def near(got, left, right, extra=0.0):
        want, S = left @ right + extra, left.abs() @ right.abs() + abs(extra)
        half = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
        tol = half * want.abs() + (1 + half) * ((left.shape[1] + 1) * U + (CUT if got.dtype != F32 else 0)) * S + (2.0 ** -25 if got.dtype == F16 else 0)
        assert ((got.double().cpu().reshape(want.shape) - want).abs() <= tol).all()

    near(y.detach(), q(x2, 1), wq.t(), b.detach().double().cpu())
    near(dx, q(dy2, 1), wq)
    near(dw, q(dy2.t(), 1), q(x2.t(), 1).t())
    assert dx.dtype == dtype and dw.dtype == wtype and dx.shape == x.shape
    assert ((db.double().cpu() - dy2.sum(0)).abs() <= (dy2.shape[0] + 1) * U * dy2.abs().sum(0)).all()
    held = train_ops.linear_fp8(x.detach(), ops.quantize_fp8(w.detach(), 128).rows, b.detach())
    assert torch.equal(held, y.detach())


def test_module_frozen_parts_and_no_rows():
    m = train_ops.LinearFp8(40, 24).cuda()
    x = torch.randn(6, 40, device="cuda", requires_grad=True)
    (gx,) = torch.autograd.grad(m(x).sum(), x)
    assert gx.shape == x.shape
    m.weight.requires_grad_(False)
    m(x.detach()).sum().backward()
    assert m.weight.grad is None and torch.equal(m.bias.grad, torch.full((24,), 6.0, device="cuda"))
    m.weight.requires_grad_(True)
    e = torch.zeros(0, 40, device="cuda", requires_grad=True)
    y = m(e)
    gx, gw, gb = torch.autograd.grad(y, (e, m.weight, m.bias), torch.zeros_like(y))
    assert y.shape == (0, 24) and gx.shape == (0, 40) and not gw.any() and not gb.any()


def test_quantised_weights_take_a_half_bias_and_a_frozen_module():
    m = train_ops.LinearFp8(40, 24).cuda().bfloat16().requires_grad_(False)
    x = torch.randn(6, 40, device="cuda", dtype=BF16)
    held = ops.quantize_fp8(m.weight, 128).rows
    assert torch.equal(train_ops.linear_fp8(x, held, m.bias), m(x))                 # the same operands in the same product
    with pytest.raises(W2CError):
        train_ops.linear_fp8(x, held, m.bias.clone().requires_grad_())
    for w in (torch.zeros(0, 40, device="cuda"), torch.zeros(24, 0, device="cuda")):
        with pytest.raises(W2CError):
            train_ops.linear_fp8(x[:, :w.shape[1]], w)


def test_replays_of_a_captured_linear_step():
    m = train_ops.LinearFp8(300, 200).cuda()
    x, dy = torch.randn(100, 300, device="cuda", requires_grad=True), torch.randn(100, 200, device="cuda")
    with ops.capture(thread_local=False) as graph:
        got = torch.autograd.grad(m(x), (x, m.weight, m.bias), dy)
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(100, 300, generator=torch.Generator().manual_seed(k)).cuda())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, torch.autograd.grad(m(x), (x, m.weight, m.bias), dy)):
            assert torch.equal(a, b)


def test_refusals():
    x = torch.randn(10, 200, device="cuda")
    q = ops.quantize_fp8(x).rows
    B = ops.Fp8Blocks
    for bad in (lambda: ops.quantize_fp8(x.cpu()), lambda: ops.quantize_fp8(x.double()), lambda: ops.quantize_fp8(x[0]), lambda: ops.quantize_fp8(x.t()),
                lambda: ops.quantize_fp8(x, 64), lambda: ops.quantize_fp8(x, rows=False), lambda: ops.quantize_fp8(x[:, :0]),
                lambda: ops.matmul_fp8(q, B(q.codes[:, :128].contiguous(), q.scale[:, :1].contiguous(), 128)), lambda: ops.matmul_fp8(q, B(q.codes, q.scale, 199)),
                lambda: ops.matmul_fp8(q, B(q.codes, q.scale[:9], 200)), lambda: ops.matmul_fp8(q, B(q.codes.view(torch.uint8), q.scale, 200)),
                lambda: ops.matmul_fp8(q, q, out_dtype=torch.float64), lambda: ops.matmul_fp8(q, q, bias=x[0]), lambda: ops.matmul_fp8(q, B(q.codes.cpu(), q.scale, 200)),
                lambda: ops.matmul_fp8(B(q.codes.t(), q.scale, 200), q), lambda: train_ops.linear_fp8(x, x[:, :100]), lambda: train_ops.linear_fp8(x[:, :100], q),
                lambda: train_ops.linear_fp8(x.clone().requires_grad_(), q)):
        with pytest.raises(W2CError):
            bad()
