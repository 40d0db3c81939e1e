"""The head's operators on tensors of more than 2^31 elements: their last rows have the bits that the same call answers for a view of those rows alone."""
import pytest
import torch

from multiagentperception_amd import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
FAR = 1 << 31


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def _normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=BF16)


def test_layer_norm():
    rows, D, tail = 524300, 4097, 9
    assert rows * D > FAR
    x = _normal(1, rows, D)
    w, b = _normal(2, D), _normal(3, D)
    y, h, mean, rstd = ops.layer_norm_forward(x, w, b, residual=x)
    part = ops.layer_norm_forward(x[-tail:], w, b, residual=x[-tail:])
    for a, p in zip((y, h, mean, rstd), part):
        assert torch.equal(a[-tail:], p)
    del y, x
    dy = torch.zeros_like(h)
    dy[-1] = w
    dx, dw, db = ops.layer_norm_backward(dy, h, w, mean, rstd)
    p = ops.layer_norm_backward(dy[-tail:], h[-tail:], w, mean[-tail:], rstd[-tail:])
    assert torch.equal(dx[-tail:], p[0]) and torch.equal(dw, p[1]) and torch.equal(db, p[2])      # one row has a gradient: no order to its sum
    assert dx[-1].any() and not dx[-1 - (1 << 20) // D:-1].any()


@pytest.mark.parametrize("shape,dim,tail", [((42800, 50177), 1, 4200), ((700, 40, 76800), 1, 1)])
def test_log_probs(shape, dim, tail):
    x = _normal(4, *shape)
    assert x.numel() > FAR
    rest = shape[:dim] + shape[dim + 1:]
    target = torch.randint(0, shape[dim], rest, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    r = ops.log_probs_forward(x, target, 2, dim)
    p = ops.log_probs_forward(x[-tail:], target[-tail:], 2, dim)
    for a, b in zip(r, p):
        assert torch.equal(a[-tail:], b)
    g = torch.ones(rest, device="cuda")
    d = ops.log_probs_backward(x, target, r, g, g, torch.ones(rest + (2,), device="cuda"), dim)
    e = ops.log_probs_backward(x[-tail:], target[-tail:], p, g[-tail:], g[-tail:], torch.ones(rest + (2,), device="cuda")[-tail:], dim)
    assert torch.equal(d[-tail:], e)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(bits):
    n, tail, blocks = FAR + 1000, 1512, 6                       # the tail is six blocks of 256, the last one of 232
    assert (n - tail) % ops.ADAMW_STATE_BLOCK == 0
    p, g = torch.zeros(n, dtype=BF16, device="cuda"), torch.zeros(n, dtype=BF16, device="cuda")
    p[-tail:], g[-tail:] = _normal(6, tail), _normal(7, tail)

    def state(n):
        if bits == 32:
            return torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        kinds = ((n, torch.float8_e4m3fn), (-(-n // ops.ADAMW_STATE_BLOCK), torch.float8_e8m0fnu)) * 2
        return tuple(torch.zeros(k, dtype=torch.uint8, device="cuda").view(t) for k, t in kinds)

    q, s, t = p[-tail:].clone(), state(n), state(tail)
    norm = ops.adamw_step([p], [g], [s], [torch.zeros((), device="cuda")], max_norm=1.0)
    part = ops.adamw_step([q], [g[-tail:].clone()], [t], [torch.zeros((), device="cuda")], max_norm=1.0)
    # the norms are sums in 64 bits in another order, rounded to f32: the gradients' factors differ by one such rounding, the moments and the update (at most
    # 0.001) by a few, and a bf16 parameter by the step that this may tip over
    assert abs(float(norm) - float(part)) <= 2.0 ** -23 * float(part)
    assert ((p[-tail:].double() - q.double()).abs() <= 2.0 ** -7 * q.double().abs() + 2.0 ** -28).all()
    if bits == 32:
        for a, b in zip(s, t):
            assert b.all() and ((a[-tail:].double() - b.double()).abs() <= 2.0 ** -20 * b.double().abs()).all() and not a[-tail - 4096:-tail].any()
    else:
        for k in (0, 2):
            assert (t[k].view(torch.uint8) & 0x7F).any() and not s[k].view(torch.uint8)[-tail - 4096:-tail].any()
            assert (s[k + 1].view(torch.uint8)[-blocks:].int() - t[k + 1].view(torch.uint8).int()).abs().max() <= 1


def test_quantiser_and_products():
    rows, cols, tail = 524300, 4097, 12                         # the last 12 rows are a block of 128 by themselves
    x = _normal(8, rows, cols)
    q, t = ops.quantize_fp8(x, columns=True, sums=True), ops.quantize_fp8(x[-tail:], columns=True)
    same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))       # noqa: E731
    assert q.rows.codes.numel() > FAR and q.columns.codes.numel() > FAR
    assert same(q.rows.codes[-tail:], t.rows.codes) and same(q.rows.scale[-tail:], t.rows.scale)
    assert same(q.columns.codes[:, -128:].contiguous(), t.columns.codes) and same(q.columns.scale[:, -1:].contiguous(), t.columns.scale)
    b = ops.quantize_fp8(_normal(9, 200, cols)).rows
    some = 65548                                                # both calls have enough rows for the largest tiles
    c = ops.matmul_fp8(q.rows, b)
    assert torch.equal(c[-some:], ops.matmul_fp8(ops.Fp8Blocks(q.rows.codes[-some:], q.rows.scale[-some:], cols), b))
    del c, q
    x[:-tail] = 0                                               # along the rows: nothing but the last block of the reduction counts
    dy = torch.zeros(rows, 300, dtype=BF16, device="cuda")
    dy[-tail:] = _normal(10, tail, 300)
    long = ops.matmul_fp8(ops.quantize_fp8(dy, rows=False, columns=True).columns, ops.quantize_fp8(x, rows=False, columns=True).columns, out_dtype=F32)
    short = ops.matmul_fp8(ops.quantize_fp8(dy[-tail:], rows=False, columns=True).columns, t.columns, out_dtype=F32)
    assert torch.equal(long, short)


def test_a_product_with_a_far_end():
    M = 46400
    assert M * M > FAR
    a, b = ops.quantize_fp8(_normal(11, M, 100)).rows, ops.quantize_fp8(_normal(12, M, 100)).rows
    c = ops.matmul_fp8(a, b)
    assert torch.equal(c[-512:], ops.matmul_fp8(ops.Fp8Blocks(a.codes[-512:], a.scale[-512:], 100), b))
