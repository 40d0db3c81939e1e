"""The head's operators on more rows or columns than one launch has work-items for (2^32): the parts of the work at the seams and at the end have the bits that
the same call answers for a view of them alone."""
import pytest
import torch

from multiagentperception_amd import ops, train_ops
from multiagentperception_amd._native import W2CError

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


# 16 rows to a block of the short rows' forward, 4 to one of their backward and of both up to 2 048 classes, 1 beyond
@pytest.mark.parametrize("rows,classes,seam", [((1 << 28) + 5, 65, 16 * (0xFFFFFFFF // 256)), ((1 << 26) + 9, 513, 4 * (0xFFFFFFFF // 256)), ((1 << 24) + 3, 2049, 0xFFFFFFFF // 256)])
def test_log_probs_of_many_rows(rows, classes, seam):
    n = 1100
    x = torch.zeros(rows, classes, dtype=BF16, device="cuda")
    target = torch.zeros(rows, dtype=torch.int64, device="cuda")
    assert rows - n < seam < rows                                 # (views of 1 024 rows and more: fewer rows of 2 049 classes are split into parts and joined)
    places = [slice(0, n), slice(rows - n, rows)] + ([slice((1 << 26) - n, (1 << 26) + 7)] if rows > 1 << 27 else [])
    g = torch.Generator(device="cuda").manual_seed(rows)
    for s in places:
        x[s] = torch.randn(x[s].shape, generator=g, device="cuda").to(BF16)
        target[s] = torch.randint(0, classes, target[s].shape, generator=g, device="cuda")
    ones = torch.ones(rows, device="cuda")
    r = ops.log_probs_forward(x, target, 2)
    d = ops.log_probs_backward(x, target, r, ones, ones)
    for s in places:
        p = ops.log_probs_forward(x[s], target[s], 2)
        for a, b in zip(r, p):
            assert torch.equal(a[s], b)
        assert torch.equal(d[s], ops.log_probs_backward(x[s], target[s], p, ones[s], ones[s]))
    some = slice(rows // 2, rows // 2 + 4)                        # zeros: every class alike
    assert torch.equal(r.top_index[some], torch.tensor([[0, 1]] * 4, device="cuda")) and not d[some][:, 1:].isnan().any()


def test_weight_gradients_of_a_norm_over_many_columns():
    D = (1 << 28) + 77
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(1, D, generator=g, device="cuda") for _ in range(2))
    w = torch.ones(D, device="cuda")
    y, h, mean, rstd = ops.layer_norm_forward(x, w)
    dw, db = ops.layer_norm_backward(dy, h, w, mean, rstd)[1:]
    assert torch.equal(db, dy[0])                                 # one row: no sum
    for s in (slice(0, 100), slice(64 * (0xFFFFFFFF // 1024) - 50, 64 * (0xFFFFFFFF // 1024) + 50), slice(D - 100, D)):
        want = dy[0, s].double() * (x[0, s].double() - mean.double()) * rstd.double()
        assert ((dw[s].double() - want).abs() <= 4 * 2.0 ** -24 * (dy[0, s].double() * rstd.double()).abs() * (x[0, s].double().abs() + mean.double().abs())).all()


def test_column_sums_of_many_columns():
    rows, cols = 129, (1 << 28) + 200                              # two tiles of rows: the sums are joined by a second launch
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    seam = 64 * (0xFFFFFFFF // 1024)
    g = torch.Generator(device="cuda").manual_seed(2)
    places = (slice(0, 300), slice(seam - 300, seam + 300), slice(cols - 300, cols))
    for s in places:
        x[:, s] = torch.randn(x[:, s].shape, generator=g, device="cuda").to(BF16)
    sums = ops.quantize_fp8(x, rows=False, sums=True).sums
    for s in places:
        v = x[:, s].double()
        assert ((sums[s].double() - v.sum(0)).abs() <= 130 * 2.0 ** -24 * v.abs().sum(0)).all()
    assert not sums[300:seam - 300].any()


@pytest.mark.parametrize("rows", [(1 << 22) + 1, ops.FP8_MOST])
def test_a_linear_step_over_as_many_rows_as_its_forward_takes(rows):
    """the gradient of the weights is a sum over all rows; 300 of them are not zero, so that many roundings at most"""
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy = torch.zeros(rows, 16, device="cuda"), torch.zeros(rows, 24, device="cuda")
    at = torch.randint(0, rows, (300,), generator=g, device="cuda")
    at[0] = rows - 1
    x[at], dy[at] = torch.randn(300, 16, generator=g, device="cuda"), torch.randn(300, 24, generator=g, device="cuda")
    x.requires_grad_()
    w = torch.randn(24, 16, generator=g, device="cuda", requires_grad=True)
    y = train_ops.linear_fp8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    held = lambda t: t.codes[:, :rows].float().double() * t.scale.float().double().repeat_interleave(128, 1)[:, :rows]       # noqa: E731
    a, b = (held(ops.quantize_fp8(t.detach(), rows=False, columns=True).columns)[:, at.unique()] for t in (dy, x))
    assert ((dw.double() - a @ b.t()).abs() <= 301 * 2.0 ** -24 * (a.abs() @ b.abs().t())).all() and dw.any()
    some = at.sort()[0][-20:]
    by_rows = lambda t, tile: (t.codes.float().double() * t.scale.float().double().repeat_interleave(tile, 0)[:t.codes.shape[0]])[:, :t.cols]       # noqa: E731
    qw = ops.quantize_fp8(w.detach(), 128, columns=True)
    for got, left, right in ((y, x, qw.rows), (dx, dy, qw.columns)):               # one block of 128 either way
        p, q = by_rows(ops.quantize_fp8(left.detach()[some]).rows, 1), by_rows(right, 128)
        assert ((got.detach()[some].double() - p @ q.t()).abs() <= 25 * 2.0 ** -24 * (p.abs() @ q.abs().t())).all()


def test_more_rows_are_refused_by_the_forward():
    x = torch.zeros(ops.FP8_MOST + 1, 16, device="cuda", requires_grad=True)
    with pytest.raises(W2CError, match="at most"):
        train_ops.linear_fp8(x, torch.zeros(24, 16, device="cuda"))
    c = torch.zeros(2, ops.FP8_MOST + 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    q = ops.Fp8Blocks(c, torch.zeros(2, c.shape[1] // 128, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu), c.shape[1])
    with pytest.raises(W2CError, match="at most"):
        ops.matmul_fp8(q, q)


def _codes(n, first, seed, t, x, positive):
    """the e4m3 values and scales of x f64 [n], elements first .. of a tensor, by the definition: rounded up or down by a hash of (seed, step, place)"""
    low = 0xFFFFFFFF
    place = torch.arange(n, dtype=torch.int64, device=x.device) + first
    h = ((place & low) * 0xA3D8F62B + (place >> 32) * 0xC2B2AE35 + ((seed * 0x9E3779B1 + t * 0x85EBCA6B) & low)) & low
    h = ((h ^ (h >> 15)) * 0xC58B3E95) & low
    h = ((h ^ (h >> 13)) * 0x9E3779B1) & low
    h = h ^ (h >> 16)
    noise = (((h >> 16) if positive else (h & 0xFFFF)).double() + 0.5) / 65536
    two_to = lambda e: ((e.long() + 1023) << 52).view(torch.float64)                # noqa: E731
    top = torch.nn.functional.pad(x.float().abs(), (0, -n % 256)).view(-1, 256).amax(1)
    m, e = torch.frexp(top / 448.0)
    e = torch.where(top > 0, torch.where(m == 0.5, e - 1, e), torch.zeros_like(e))
    unit = two_to(e).repeat_interleave(256)[:n]
    u = x / unit
    step = two_to(torch.clamp(torch.frexp(u)[1] - 1, min=-6) - 3)
    q = (torch.floor(u.abs() / step + noise) * step).clamp(max=448.0) * u.sign()
    if positive:
        q = torch.where(u > 0, q.clamp(min=2.0 ** -9), q)
    return q * unit, step * unit, (e + 127).to(torch.uint8)


@pytest.mark.parametrize("tail_first", [(1 << 32) - 256 * 3, 1 << 32])
def test_8_bit_moments_beyond_2_to_the_32(tail_first):
    """the last elements' codes are those of the definition, which counts places in 64 bits.  A moment a few roundings of f32 off may round the other way: one
    element in 2^20 / 2^7 of a step, so none or one of these"""
    n, seed, hp = (1 << 32) + 1000, 77, dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)
    p, g = torch.zeros(n, dtype=BF16, device="cuda"), torch.zeros(n, dtype=BF16, device="cuda")
    tail = slice(tail_first, n)
    gen = torch.Generator(device="cuda").manual_seed(5)
    p[tail], g[tail] = (torch.randn(n - tail_first, generator=gen, device="cuda").to(BF16) for _ in range(2))
    old = p[tail].double()
    kinds = ((n, torch.float8_e4m3fn), (-(-n // 256), torch.float8_e8m0fnu)) * 2
    state = tuple(torch.zeros(k, dtype=torch.uint8, device="cuda").view(t) for k, t in kinds)
    ops.adamw_step([p], [g], [state], [torch.zeros((), device="cuda")], seed=seed, **hp)
    gd = g[tail].double()
    off = 0
    for (code, scale), x, positive in ((state[:2], 0.1 * gd, False), (state[2:], 0.1 * gd.abs(), True)):
        want, step, e = _codes(n - tail_first, tail_first, seed, 1, x, positive)
        blocks = slice(tail_first // 256, None)
        assert torch.equal(scale[blocks].view(torch.uint8), e)
        got = code[tail].float().double() * scale[blocks].float().double().repeat_interleave(256)[:n - tail_first]
        assert ((got - want).abs() <= step * (1 + 1e-9)).all()
        off += int((got != want).sum())
        assert not code[tail_first - 512:tail_first].view(torch.uint8).any()
    assert off <= 1
    assert ((p[tail].double() - (old * (1 - 1e-3) - 1e-2 * gd.sign())).abs() <= 2.0 ** -8 * old.abs() + 2.0 ** -8 * 0.011 + 1e-6).all()
