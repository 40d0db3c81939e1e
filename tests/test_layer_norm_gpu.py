"""Layer norm (w2c_layer_norm_forward / _backward) against the formulas in 64 bits.

Tolerances count roundings.  U = 2^-24 is half a step of f32, H half a step of the tensors' type relative to the value.  A sum over a row is a chain of at
most 32 values per thread and 10 tree levels, so K = 64 roundings bound every f32 quantity below, relative to the sum of magnitudes it is made of."""
import pytest
import torch

from multiagentperception_amd import ops, train_ops
from multiagentperception_amd._native import W2CError

pytestmark = pytest.mark.gpu
U, K = 2.0 ** -24, 64
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _make(shape, dtype, wtype, seed, residual=True, affine=True, shift=0.5):
    g = torch.Generator().manual_seed(seed)
    r = lambda s, k=1.0: (torch.randn(s, generator=g) * k)                       # noqa: E731
    x = (r(shape, 1.5) + shift).to(dtype).cuda()
    res = r(shape).to(dtype).cuda() if residual else None
    w = (r(shape[-1], 0.3) + 1).to(wtype).cuda() if affine else None
    b = r(shape[-1], 0.3).to(wtype).cuda() if affine else None
    return x, res, w, b, r(shape).to(dtype).cuda(), r(shape).to(dtype).cuda()


def _check(shape, dtype, wtype, seed, residual=True, affine=True, shift=0.5, eps=1e-5):
    x, res, w, b, dy, dh = _make(shape, dtype, wtype, seed, residual, affine, shift)
    if not residual:
        dh = None
    y, h, mean, rstd = ops.layer_norm_forward(x, w, b, eps, residual=res)
    dx, dw, db = ops.layer_norm_backward(dy, h, w, mean, rstd, dh=dh)
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    D = shape[-1]
    hd = h.double().reshape(-1, D)
    if residual:
        assert torch.equal(h, (x.float() + res.float()).to(dtype))
    else:
        assert h is x
    one = torch.ones(D, dtype=torch.float64, device="cuda")
    wd, bd = (one, one * 0) if w is None else (w.double(), b.double())
    mu = hd.mean(1, keepdim=True)
    rs = 1.0 / (((hd - mu) ** 2).mean(1, keepdim=True) + eps).sqrt()
    n = (hd - mu) * rs
    big = hd.abs().amax(1, keepdim=True)
    e_n = K * U * (n.abs() + rs * big) * (1 + n.abs())            # of n: the mean's error, and rstd's through the squared differences
    yr = n * wd + bd
    tol = half * yr.abs() + (1 + half) * (e_n * wd.abs() + 4 * U * (yr.abs() + bd.abs())) + (2.0 ** -24 if dtype == F16 else 0)
    assert ((y.double().reshape(-1, D) - yr).abs() <= tol).all()
    assert ((mean.double().reshape(-1, 1) - mu).abs() <= K * U * hd.abs().mean(1, keepdim=True) + 1e-30).all()
    gy = dy.double().reshape(-1, D)
    g = gy * wd
    avg = lambda t: t.mean(1, keepdim=True)                                       # noqa: E731
    dr = rs * (g - avg(g) - n * avg(g * n))
    e = rs * (K * U * (g.abs() + avg(g.abs()) + 2 * n.abs() * avg((g * n).abs())) + e_n * avg((g * n).abs()) + n.abs() * avg(g.abs() * e_n)
              + (1 + n.abs()) * K * U * rs * big * (g - avg(g) - n * avg(g * n)).abs())
    if residual:
        dr = dr + dh.double().reshape(-1, D)
    tol = half * dr.abs() + (1 + half) * (e + 4 * U * dr.abs()) + (2.0 ** -24 if dtype == F16 else 0)
    assert ((dx.double().reshape(-1, D) - dr).abs() <= tol).all()
    R = gy.shape[0]
    whalf = torch.finfo(wtype).eps / 2 if wtype != F32 else 0.0
    db_r = gy.sum(0)
    assert ((db.double() - db_r).abs() <= whalf * db_r.abs() + (1 + whalf) * (R + 2) * U * gy.abs().sum(0)).all()
    if affine:
        dw_r = (gy * n).sum(0)
        tol = whalf * dw_r.abs() + (1 + whalf) * ((R + 4) * U * (gy * n).abs().sum(0) + (gy.abs() * e_n).sum(0))
        assert ((dw.double() - dw_r).abs() <= tol).all() and dw.dtype == wtype
    else:
        assert dw is None


@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)])
@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (5, 7), (1, 64), (9, 255), (2, 3, 512), (6, 1001), (130, 2047), (3, 2049), (5, 4100), (3, 8191),
                                   (2, 16385), (3, 33000), (4099, 24)])
def test_forward_and_backward_match_the_formulas(shape, dtype, wtype):
    _check(shape, dtype, wtype, seed=sum(shape))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1), (7, 513), (3, 20000)])
def test_without_residual_and_without_weights(shape, dtype):
    _check(shape, dtype, F32 if dtype == F32 else dtype, seed=1, residual=False, affine=False)
    _check(shape, dtype, F32, seed=2, residual=False)


def test_a_large_mean_loses_no_digits_to_cancellation():
    _check((33, 768), F32, F32, seed=3, shift=3000.0)


def test_rows_that_start_at_odd_addresses():
    """a view one element into a buffer: contiguous, aligned to one element only"""
    for dtype in (F32, BF16, F16):
        flat = torch.randn(5 * 301 + 1, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
        x = flat[1:].view(5, 301)
        y = ops.layer_norm_forward(x)[0]
        z = ops.layer_norm_forward(x.clone())[0]
        assert x.data_ptr() % 16 and torch.equal(y, z)


def test_no_rows():
    x = torch.empty(0, 32, device="cuda")
    w = torch.ones(32, device="cuda")
    y, h, mean, rstd = ops.layer_norm_forward(x, w, w)
    dx, dw, db = ops.layer_norm_backward(x, h, w, mean, rstd)
    assert y.shape == x.shape and mean.shape == (0,) and dx.shape == x.shape and not dw.any() and not db.any()


def test_nan_and_infinity_stay_in_their_row():
    x = torch.randn(4, 300, device="cuda")
    clean = ops.layer_norm_forward(x)[0]
    x2 = x.clone()
    x2[1, 5], x2[2, 299] = float("nan"), float("inf")
    y = ops.layer_norm_forward(x2)[0]
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3]) and y[1].isnan().all() and y[2].isnan().any()


def test_the_same_bits_every_time_and_on_another_stream():
    x, res, w, b, dy, dh = _make((700, 1536), BF16, F32, 5)
    def both():
        y, h, mean, rstd = ops.layer_norm_forward(x, w, b, residual=res)
        return (y, h) + ops.layer_norm_backward(dy, h, w, mean, rstd, dh=dh)
    a = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = both()
    torch.cuda.current_stream().wait_stream(s)
    for p, q, r in zip(a, both(), c):
        assert torch.equal(p, q) and torch.equal(p, r)


def test_module_trains_like_the_formula_and_takes_strided_inputs():
    m = train_ops.LayerNormHip(96).cuda()
    g = torch.Generator().manual_seed(6)
    with torch.no_grad():
        m.weight.copy_(torch.randn(96, generator=g))
        m.bias.copy_(torch.randn(96, generator=g))
    x = torch.randn(96, 10, 4, generator=g).cuda().permute(2, 1, 0).requires_grad_()          # strides (1, 4, 40)
    r = torch.randn(4, 10, 96, generator=g).cuda().requires_grad_()
    up, uh = torch.randn(4, 10, 96, generator=g).cuda(), torch.randn(4, 10, 96, generator=g).cuda()
    y, h = m(x, r)
    ((y * up).sum() + (h * uh).sum()).backward()
    xd, rd, wd, bd = (t.detach().double().requires_grad_() for t in (x, r, m.weight, m.bias))
    hd = xd + rd
    yd = torch.nn.functional.layer_norm(hd, (96,), wd, bd, m.eps)
    ((yd * up.double()).sum() + (hd * uh.double()).sum()).backward()
    for a, b in ((x.grad, xd.grad), (r.grad, rd.grad), (m.weight.grad, wd.grad), (m.bias.grad, bd.grad)):
        assert float((a.double() - b).abs().max()) <= 256 * U * float(b.abs().max())
    y, h = m(x.detach(), r)
    assert torch.equal(torch.autograd.grad(h.sum(), r)[0], torch.ones_like(r))               # only h is used


def test_a_frozen_norm_hands_the_gradient_on():
    m = train_ops.LayerNormHip(300).cuda()
    x = torch.randn(40, 300, device="cuda", requires_grad=True)
    dy = torch.randn(40, 300, device="cuda")
    (want,) = torch.autograd.grad(m(x), x, dy)
    got = []
    for weight, bias in ((False, True), (True, False), (False, False)):
        m.weight.requires_grad_(weight)
        m.bias.requires_grad_(bias)
        (gx, *rest) = torch.autograd.grad(m(x), [x] + [p for p in m.parameters() if p.requires_grad], dy)
        assert torch.equal(gx, want)
        got.append(rest)
    m.requires_grad_(True)
    dw, db = torch.autograd.grad(m(x), (m.weight, m.bias), dy)
    assert torch.equal(got[0][0], db) and torch.equal(got[1][0], dw) and not got[2]


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(7)
    x, w, b, up = (torch.randn(s, generator=g).cuda() for s in ((3, 40), (40,), (40,), (3, 40)))
    x.requires_grad_()
    (gx,) = torch.autograd.grad((train_ops.layer_norm(x, w, b) * up).sum(), x)
    f = lambda t: (torch.nn.functional.layer_norm(t, (40,), w.double(), b.double()) * up.double()).sum()          # noqa: E731
    d = 1e-5
    for i, j in ((0, 0), (1, 17), (2, 39)):
        e = torch.zeros(3, 40, dtype=torch.float64, device="cuda")
        e[i, j] = d
        diff = float(f(x.detach().double() + e) - f(x.detach().double() - e)) / (2 * d)
        assert abs(float(gx[i, j]) - diff) <= 1e-5 * float(gx.abs().max())       # d^2 of the differences, K U of the kernel


def test_replays_of_a_captured_step():
    m = train_ops.LayerNormHip(512).cuda()
    x = torch.randn(64, 512, device="cuda", requires_grad=True)
    up = torch.randn(64, 512, device="cuda")
    with ops.capture(thread_local=False) as graph:            # (no autograd graph of these leaves outlives its statement)
        got = torch.autograd.grad(m(x), (x, m.weight, m.bias), up)
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(64, 512, generator=torch.Generator().manual_seed(k)).cuda())
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(m(x), (x, m.weight, m.bias), up)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_refusals():
    x = torch.randn(4, 16, device="cuda")
    for bad in (lambda: ops.layer_norm_forward(x.t()), lambda: ops.layer_norm_forward(x.double()), lambda: ops.layer_norm_forward(x[:, :0]),
                lambda: ops.layer_norm_forward(x, torch.ones(15, device="cuda")), lambda: ops.layer_norm_forward(x, torch.ones(16)),
                lambda: ops.layer_norm_forward(x, torch.ones(16, device="cuda"), torch.ones(16, device="cuda", dtype=BF16)),
                lambda: ops.layer_norm_forward(x, residual=x[:2]), lambda: ops.layer_norm_forward(x, residual=x.half()),
                lambda: ops.layer_norm_backward(x[:2], x, None, x[:, 0].contiguous(), x[:, 0].contiguous()),
                lambda: ops.layer_norm_backward(x, x, None, x[0].contiguous(), x[:, 0].contiguous()),
                lambda: train_ops.LayerNormHip((4, 4)), lambda: train_ops.LayerNormHip(8).cuda()(x)):
        with pytest.raises(W2CError):
            bad()
