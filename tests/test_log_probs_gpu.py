"""Log probabilities, entropy and alternatives (w2c_log_probs_forward / _backward) against the definition in 64 bits.

Tolerances: U = 2^-24 is half a step of f32.  The hardware exponential is within 2 U relative and its argument d * log2(e) within 2 U |d|, |d| <= R the row's
range of values that count; sums of positive terms add at most 64 roundings (a chain per thread in chunks, then a tree), n_chain more where one thread
walks the row.  So log s is off by at most E = (64 + n_chain + 4 R) U, a log probability by E + 4 U |log p|, and the entropy by E (1 + R) + 4 U R."""
import math

import pytest
import torch

from multiagentperception_amd import loss, ops
from multiagentperception_amd._native import W2CError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def _reference(x, target, top, ignore):
    """x f64 [rows, C]"""
    empty = (x == -INF).all(1, keepdim=True)
    lp = torch.log_softmax(x.masked_fill(empty, 0), 1).masked_fill(empty, -INF)
    p = lp.exp()
    H = -(p * lp.masked_fill(p == 0, 0)).sum(1)
    lt = lp.gather(1, target.clamp(0, x.shape[1] - 1).unsqueeze(1)).squeeze(1)
    lt = lt.masked_fill((target < 0) | (target >= x.shape[1]), float("nan")).masked_fill(target == ignore, 0)
    idx = x.sort(dim=1, descending=True, stable=True)[1][:, :top]
    return lp, p, H, lt, lp.gather(1, idx), idx, empty


def _check(outer, C, inner, dtype, top, seed, spread=3.0, masked=0.0, values=None, ignore=-100, pitch=0):
    g = torch.Generator().manual_seed(seed)
    shape = (outer, C) + ((inner,) if inner > 1 else ())
    x = torch.randn(shape, generator=g) * spread
    if values:
        x = torch.tensor(values)[torch.randint(0, len(values), shape, generator=g)]
    if masked:
        x[torch.rand(shape, generator=g) < masked] = -INF
    x = x.to(dtype).cuda()
    if pitch:
        wide = torch.randn(outer, C + pitch, generator=g).to(dtype).cuda()
        wide[:, :C] = x
        x = wide[:, :C]
    rest = shape[:1] + shape[2:]
    t = torch.randint(0, C, rest, generator=g)
    t[torch.rand(rest, generator=g) < 0.2] = ignore
    t = t.cuda()
    f32 = lambda s: torch.randn(s, generator=g).cuda()                            # noqa: E731
    g_logp, g_H, g_top = f32(rest), f32(rest), f32(rest + (top,)) if top else None
    r = ops.log_probs_forward(x, t, top, 1, ignore)
    d = ops.log_probs_backward(x, t, r, g_logp, g_H, g_top, 1, ignore)
    xd = x.double().movedim(1, -1).reshape(-1, C)
    lp, p, H, lt, tl, ti, empty = _reference(xd, t.reshape(-1), top, ignore)
    if top:
        same = bool(torch.equal(r.top_index.reshape(-1, top), ti))
        assert same
    fin = xd.masked_fill(xd == -INF, 0)
    top_x = xd.amax(1, keepdim=True).masked_fill(empty, 0)
    reach = (top_x - fin).masked_fill((xd == -INF) | (top_x - fin > 104), 0).amax(1)         # beyond e^-104 nothing counts
    chain = C if (inner > 1 or C <= 64) else 0
    E = (64 + chain + 4 * reach) * U

    def near(got, want, tol):
        got, want = got.double().reshape(want.shape), want
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got == -INF, want == -INF)
        ok = (got - want).abs() <= tol
        assert (ok | want.isnan() | (want == -INF)).all(), float(((got - want).abs() - tol)[want.isfinite()].max())

    near(r.logp, lt, E + 4 * U * lt.abs().nan_to_num(0, 0, 0))
    near(r.entropy, H, E * (1 + reach) + 4 * U * reach)
    if top:
        near(r.top_logp, tl, E[:, None] + 4 * U * tl.abs().nan_to_num(0, 0, 0))
    a = g_logp.double().reshape(-1, 1) * (t.reshape(-1, 1) != ignore)
    dr = torch.zeros_like(xd).scatter_(1, t.reshape(-1, 1).clamp_min(0), a)
    size = dr.abs()
    whole, wsize = a, a.abs()
    if top:
        gt = g_top.double().reshape(-1, top)
        dr.scatter_add_(1, ti, gt)
        size.scatter_add_(1, ti, gt.abs())
        whole, wsize = a + gt.sum(1, keepdim=True), a.abs() + gt.abs().sum(1, keepdim=True)
    c = g_H.double().reshape(-1, 1)
    lpf = lp.masked_fill(p == 0, 0)
    dr = (dr - p * whole - c * p * (lpf + H[:, None])).masked_fill(empty, 0)
    Ep = (E[:, None] + 8 * U + 4 * U * lpf.abs()) * p                                # of p
    e_l = E[:, None] + 4 * U * lpf.abs() + (E * (1 + reach) + 4 * U * reach)[:, None]
    inner_size = wsize + c.abs() * (lpf.abs() + H[:, None])
    tol = Ep * inner_size + p * (c.abs() * e_l + (top + 4) * U * inner_size) + 4 * U * (size + p * inner_size)
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    tol = half * dr.abs() + (1 + half) * tol + (2.0 ** -25 if dtype == F16 else 2.0 ** -126)      # the type's smallest step
    got = d.double().movedim(1, -1).reshape(-1, C)
    assert ((got - dr).abs() <= tol).all(), float(((got - dr).abs() - tol).max())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("outer,C,top", [(1, 1, 1), (3, 2, 2), (200, 11, 0), (70, 64, 5), (5, 65, 8), (9, 100, 20), (6, 1000, 0), (4, 2047, 32), (3, 2048, 1),
                                         (5, 2049, 8), (1, 50257, 5), (7, 33001, 32), (2, 128000, 1), (1030, 2500, 2)])
def test_rows(outer, C, top, dtype):
    _check(outer, C, 1, dtype, top, seed=outer + C, masked=0.0 if outer % 2 else 0.3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("outer,C,top", [(4099, 70, 3), (16389, 253, 8), (16386, 254, 20), (16387, 505, 0), (4097, 509, 32)])
def test_many_short_rows(outer, C, top, dtype):
    _check(outer, C, 1, dtype, top, seed=outer + C, masked=0.3)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("outer,C,inner,top", [(2, 11, 35, 2), (1, 2, 1000, 1), (3, 19, 3, 8), (2, 40, 130, 20), (1, 33, 70, 32), (2, 1100, 5, 3)])
def test_class_dimension_in_front(outer, C, inner, top, dtype):
    _check(outer, C, inner, dtype, top, seed=C + inner, masked=0.3 if C % 2 else 0.0)


@pytest.mark.parametrize("C", [33, 300, 5000])
def test_equal_values_go_to_the_lower_class(C):
    _check(8, C, 1, BF16, min(32, C), seed=C, values=[1.0, 1.0, 2.0])
    _check(8, C, 1, F32, min(32, C), seed=C + 1, values=[0.0, -0.0])
    _check(3, C, 1, F32, 8, seed=C + 2, values=[-INF, -INF, -INF, -2.0])
    _check(2, C, 1, F32, 8, seed=C + 3, values=[-INF])
    _check(2, C, 1, F32, 4, seed=C + 4, values=[-3.4028234663852886e38, 5.0])        # the type's lowest value as a mask
    _check(2, C, 1, F32, 4, seed=C + 5, values=[-3.4028234663852886e38])
    _check(2, 8, C, F32, 8, seed=C + 6, values=[-INF, 3.0, 3.0])


@pytest.mark.parametrize("C", [30, 700, 9000])
def test_ascending_and_descending_rows(C):
    x = torch.arange(C, dtype=torch.float32, device="cuda").repeat(3, 1) * 0.01
    for v in (x, x.flip(1).contiguous()):
        r = ops.log_probs_forward(v, None, 20)
        assert torch.equal(r.top_index, v.sort(dim=1, descending=True, stable=True)[1][:, :20]) and r.logp is None


@pytest.mark.parametrize("top", [1, 31, 32])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("C", [257, 1999, 9001, 40000])
def test_rows_with_many_equal_or_rising_values(C, dtype, top):
    """hundreds of values reach the bound that the alternatives are looked for from"""
    i = torch.arange(C, device="cuda")
    access, threads = i // (4 if dtype == F32 else 8), 64 if C <= 2048 else 256
    column = access % threads
    rows = torch.stack([torch.ones(C, device="cuda"), (i // 3).float(), (column < 31) * 10.0 + (column == 31) * 5.0, torch.where(i % 5 == 0, -INF, 1.0)]).to(dtype)
    wide = torch.zeros(4, C + 3, dtype=dtype, device="cuda")
    wide[:, :C] = rows
    for x in (rows, wide[:, :C]):
        assert torch.equal(ops.log_probs_forward(x, None, top).top_index, rows.float().sort(dim=1, descending=True, stable=True)[1][:, :top])


def test_large_logits_keep_their_digits():
    _check(4, 500, 1, F32, 3, seed=1, spread=2000.0)
    _check(3, 20000, 1, F32, 3, seed=2, spread=2000.0)


@pytest.mark.parametrize("C,pitch", [(11, 5), (129, 7), (5000, 3)])
def test_rows_of_a_wider_tensor(C, pitch):
    _check(6, C, 1, BF16, 4, seed=C, pitch=pitch)


@pytest.mark.parametrize("C", [20, 600, 6000])
def test_nan_and_infinity_answer_nan_in_their_row_alone(C):
    x = torch.randn(5, C, generator=torch.Generator().manual_seed(C)).cuda()
    t = torch.full((5,), 3, device="cuda")
    x[1, C - 1], x[2, 0], x[3, :] = float("nan"), INF, float("nan")
    r = ops.log_probs_forward(x, t, 4)
    d = ops.log_probs_backward(x, t, r, torch.ones(5, device="cuda"), torch.ones(5, device="cuda"), torch.ones(5, 4, device="cuda"))
    bad = torch.tensor([False, True, True, True, False], device="cuda")
    for v in (r.logp, r.entropy, r.top_logp[:, 0], r.top_logp[:, 3], d[:, 3]):
        assert torch.equal(v.isnan(), bad)
    assert ((r.top_index >= 0) & (r.top_index < C)).all()
    assert torch.equal(r.top_index[1], x[1].masked_fill(x[1].isnan(), -INF).sort(descending=True, stable=True)[1][:4]) and int(r.top_index[2, 0]) == 0


@pytest.mark.parametrize("C", [20, 600, 6000])
def test_targets_outside_answer_nan_and_ignored_ones_zero(C):
    x = torch.randn(6, C, generator=torch.Generator().manual_seed(C)).cuda()
    t = torch.tensor([0, C, -1, -100, 1 << 40, C - 1], device="cuda")
    r = ops.log_probs_forward(x, t)
    assert r.logp.isnan().tolist() == [False, True, True, False, True, False] and float(r.logp[3]) == 0.0
    d = ops.log_probs_backward(x, t, r, g_logp=torch.ones(6, device="cuda"))
    assert d.isnan().any(1).tolist() == [False, True, True, False, True, False] and not d[3].any()
    again = ops.log_probs_forward(x, torch.full((6,), 250, device="cuda"), ignore_index=250)
    assert not again.logp.any()


def test_no_rows_and_refusals():
    x = torch.randn(4, 16, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    r = ops.log_probs_forward(x[:0], t[:0], 2)
    assert r.logp.shape == (0,) and r.top_index.shape == (0, 2) and ops.log_probs_backward(x[:0], t[:0], r, r.logp).shape == (0, 16)
    good = ops.log_probs_forward(x, t, 2)
    for bad in (lambda: ops.log_probs_forward(x.cpu()), lambda: ops.log_probs_forward(x.double()), lambda: ops.log_probs_forward(x.t()),
                lambda: ops.log_probs_forward(x, t.int()), lambda: ops.log_probs_forward(x, t[:3]), lambda: ops.log_probs_forward(x, t.cpu()),
                lambda: ops.log_probs_forward(x, t, 17), lambda: ops.log_probs_forward(x, t, -1), lambda: ops.log_probs_forward(x, t, dim=2),
                lambda: ops.log_probs_forward(torch.randn(2, 64, device="cuda"), None, 33), lambda: ops.log_probs_forward(x[:, :0]),
                lambda: ops.log_probs_backward(x, None, good, g_logp=good.logp), lambda: ops.log_probs_backward(x, t, good, g_logp=good.logp.double()),
                lambda: ops.log_probs_backward(x, t, good, g_logp=good.logp[:2]), lambda: ops.log_probs_backward(x, t, good, g_top=good.logp),
                lambda: ops.log_probs_backward(x, t, ops.log_probs_forward(x, t), g_top=good.top_logp),
                lambda: ops.log_probs_backward(x[:2], t[:2], good, g_entropy=good.entropy[:2])):
        with pytest.raises(W2CError):
            bad()


def test_the_same_bits_every_time():
    x = torch.randn(3, 60000, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    a, b = ops.log_probs_forward(x, None, 8), ops.log_probs_forward(x, None, 8)
    for p, q in zip(a[1:], b[1:]):
        assert torch.equal(p, q)


@pytest.mark.parametrize("shape,dim", [((4, 7, 30), -1), ((2, 11, 5, 6), 1), ((3, 4000), 1)])
def test_loss_function_and_its_gradient_against_differences(shape, dim):
    g = torch.Generator().manual_seed(9)
    rest = list(shape)
    del rest[dim]
    x = torch.randn(shape, generator=g)
    t = torch.randint(0, shape[dim], rest, generator=g)
    a, c, b = torch.randn(rest, generator=g), torch.randn(rest, generator=g), torch.randn(rest + [3], generator=g)

    def value(r):
        f = lambda q: q.to(r.entropy)                                             # noqa: E731
        return (r.logp * f(a)).sum() + (r.entropy * f(c)).sum() + (r.top_logp * f(b)).sum()

    xg = x.cuda().requires_grad_()
    r = loss.log_probs(xg, t.cuda(), top=3, dim=dim)
    value(r).backward()
    xc = x.clone().requires_grad_()
    rc = loss.log_probs(xc, t, top=3, dim=dim)                                   # stock ops
    value(rc).backward()
    assert torch.equal(r.top_index.cpu(), rc.top_index) and not r.top_index.requires_grad
    scale = float(xc.grad.abs().max())
    assert float((xg.grad.cpu() - xc.grad).abs().max()) <= 400 * U * scale * 4      # both are f32: 200 roundings each of terms up to 4 times the largest
    xd, step = x.double(), 1e-5
    lse = lambda v: torch.log_softmax(v, dim).movedim(dim, -1)                    # noqa: E731

    def exact(v):
        lp = lse(v)
        p = lp.exp()
        return float((lp.gather(-1, t.unsqueeze(-1)).squeeze(-1) * a).sum() - ((p * lp).sum(-1) * c).sum() + (lp.gather(-1, rc.top_index) * b).sum())

    for k in (0, x.numel() // 2, x.numel() - 1):
        e = torch.zeros(x.numel(), dtype=torch.float64)
        e[k] = step
        diff = (exact(xd + e.view(shape)) - exact(xd - e.view(shape))) / (2 * step)
        assert abs(float(xg.grad.reshape(-1)[k]) - diff) <= 1e-5 * max(1.0, scale)


def test_replays_of_a_captured_loss():
    x = torch.randn(2, 40000, device="cuda", requires_grad=True)
    t = torch.randint(0, 40000, (2,), device="cuda")
    one = torch.ones(2, device="cuda")

    def step():
        r = loss.log_probs(x, t, top=4)
        g = torch.autograd.grad((r.logp, r.entropy, r.top_logp), x, (one, one, r.top_logp.detach()))
        return (*(v.detach() for v in r), *g)             # (no autograd graph of x outlives this)

    with ops.capture(thread_local=False) as graph:
        got = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(2, 40000, generator=torch.Generator().manual_seed(k)).cuda())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
