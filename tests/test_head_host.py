"""CPU: the stock branches of the head's operators, and the C ABI's refusals (checked before anything is launched, so they need no GPU)."""
import ctypes
import math

import pytest
import torch

from multiagentperception_amd import loss, ops, optim, train_ops
from multiagentperception_amd._native import W2CError

INF = float("inf")


@pytest.fixture(scope="module")
def lib():
    from multiagentperception_amd import _build, _native
    _build.build()
    return _native.lib()


def test_log_probs_on_the_cpu():
    x = torch.tensor([[1.0, 2.0, 2.0, -INF], [-INF, -INF, -INF, -INF], [0.0, 0.0, 0.0, 0.0], [1.0, 0.0, 0.0, 0.0]])
    r = loss.log_probs(x, torch.tensor([0, 1, -100, 4]), top=3)
    p = [1 / (1 + 2 * math.e), math.e / (1 + 2 * math.e)]
    assert r.logp[0].item() == pytest.approx(math.log(p[0]), abs=1e-6) and r.logp[1].item() == -INF and r.logp[2].item() == 0.0 and r.logp[3].isnan()
    assert r.entropy[0].item() == pytest.approx(-p[0] * math.log(p[0]) - 2 * p[1] * math.log(p[1]), abs=1e-6)
    assert r.entropy[1].item() == 0.0 and r.entropy[2].item() == pytest.approx(math.log(4), abs=1e-6)
    assert r.top_index.tolist()[:3] == [[1, 2, 0], [0, 1, 2], [0, 1, 2]]
    y = x.clone().requires_grad_()
    loss.log_probs(y, top=1).entropy.sum().backward()
    assert not y.grad[1].any() and not y.grad.isnan().any()
    maps = torch.randn(2, 5, 3, 4)
    a, b = loss.log_probs(maps, torch.zeros(2, 3, 4), top=2, dim=1), loss.log_probs(maps.movedim(1, -1), torch.zeros(2, 3, 4), top=2)
    assert torch.equal(a.logp, b.logp) and torch.equal(a.top_index, b.top_index) and a.top_index.shape == (2, 3, 4, 2)


@pytest.mark.parametrize("classes,top", [(4, 5), (40, 33), (4, -1)])
def test_log_probs_on_the_cpu_refuses_what_the_kernels_refuse(classes, top):
    with pytest.raises(W2CError, match="top must lie in"):
        loss.log_probs(torch.randn(2, classes), top=top)


def test_layers_on_the_cpu_are_the_stock_ones():
    torch.manual_seed(0)
    n, stock = train_ops.LayerNormHip(12), torch.nn.LayerNorm(12)
    x, r = torch.randn(3, 12), torch.randn(3, 12)
    y, h = n(x, r)
    assert torch.equal(h, x + r) and torch.equal(y, stock(x + r)) and torch.equal(n(x), stock(x))
    l = train_ops.LinearFp8(12, 5)
    assert torch.equal(l(x), torch.nn.functional.linear(x, l.weight, l.bias)) and set(l.state_dict()) == {"weight", "bias"}


def test_tensor_level_operators_refuse_the_cpu():
    x = torch.randn(4, 8)
    q = ops.Fp8Blocks(torch.zeros(4, 128, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu), 8)
    for f in (lambda: ops.layer_norm_forward(x), lambda: ops.log_probs_forward(x), lambda: ops.quantize_fp8(x), lambda: ops.matmul_fp8(q, q),
              lambda: ops.grad_squares([x]), lambda: ops.adamw_step([x], [x.clone()], [(x.clone(), x.clone())], [torch.zeros(1)])):
        with pytest.raises(W2CError, match="no CPU fallback"):
            f()
    opt = optim.AdamW([torch.nn.Parameter(x)])
    opt.param_groups[0]["params"][0].grad = x.clone()
    with pytest.raises(W2CError):
        opt.step()


def test_quantised_weights_refuse_to_lose_a_gradient():
    q = ops.Fp8Blocks(torch.zeros(4, 128, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu), 8)
    for x, bias in ((torch.randn(3, 8), torch.zeros(4, requires_grad=True)), (torch.randn(3, 8, requires_grad=True), None)):
        with pytest.raises(W2CError, match="inference"):
            train_ops.linear_fp8(x, q, bias)


P = 1 << 20                       # an address that a refused call never touches


@pytest.mark.parametrize("change", [dict(x=0), dict(y=0), dict(mean=0), dict(rstd=0), dict(dtype=3), dict(wtype=2), dict(rows=0), dict(rows=1 << 31), dict(cols=0),
                                    dict(cols=(1 << 30) + 1), dict(res=P, h=0)])
def test_layer_norm_forward_refuses(lib, change):
    a = dict(x=P, res=0, dtype=1, rows=4, cols=8, w=P, b=P, wtype=0, eps=1e-5, y=P, h=0, mean=P, rstd=P)
    a.update(change)
    assert lib.w2c_layer_norm_forward(a["x"], a["res"], a["dtype"], a["rows"], a["cols"], a["w"], a["b"], a["wtype"], a["eps"], a["y"], a["h"], a["mean"], a["rstd"], 0) == -1


@pytest.mark.parametrize("change", [dict(dy=0), dict(h=0), dict(dx=0), dict(dtype=-1), dict(wtype=2), dict(rows=0), dict(cols=0), dict(ws=0), dict(nbytes=7)])
def test_layer_norm_backward_refuses(lib, change):
    a = dict(dy=P, h=P, dtype=1, rows=4, cols=8, wtype=0, dx=P, ws=P, nbytes=lib.w2c_layer_norm_workspace_bytes(4, 8, 1))
    assert a["nbytes"] > 0
    a.update(change)
    assert lib.w2c_layer_norm_backward(a["dy"], a["h"], 0, a["dtype"], a["rows"], a["cols"], P, a["wtype"], P, P, a["dx"], P, P, a["ws"], a["nbytes"], 0) == -1


@pytest.mark.parametrize("change", [dict(x=0), dict(entropy=0), dict(stats=0), dict(dtype=3), dict(outer=0), dict(outer=1 << 31), dict(C=0), dict(C=(1 << 28) + 1), dict(inner=0),
                                    dict(stride=9999), dict(target=0), dict(logp=0), dict(top=-1), dict(top=33), dict(C=4, stride=4, top=5), dict(tl=0), dict(ti=0),
                                    dict(ws=0), dict(nbytes=3), dict(ws=P + 4), dict(inner=2, stride=10000), dict(inner=2, C=8193, stride=16386)])
def test_log_probs_forward_refuses(lib, change):
    a = dict(x=P, dtype=1, outer=3, C=10000, inner=1, stride=10000, target=P, top=4, logp=P, entropy=P, tl=P, ti=P, stats=P, ws=P,
             nbytes=lib.w2c_log_probs_workspace_bytes(3, 10000, 1, 4))
    assert a["nbytes"] > 0
    a.update(change)
    assert lib.w2c_log_probs_forward(a["x"], a["dtype"], a["outer"], a["C"], a["inner"], a["stride"], a["target"], -100, a["top"], a["logp"], a["entropy"], a["tl"],
                                     a["ti"], a["stats"], a["ws"], a["nbytes"], 0) == -1


@pytest.mark.parametrize("change", [dict(x=0), dict(dx=0), dict(target=0), dict(top=0), dict(ti=0), dict(stride=9), dict(top=33)])
def test_log_probs_backward_refuses(lib, change):
    a = dict(x=P, dtype=1, outer=3, C=10, inner=1, stride=10, target=P, top=4, ti=P, gt=P, dx=P)
    a.update(change)
    assert lib.w2c_log_probs_backward(a["x"], a["dtype"], a["outer"], a["C"], a["inner"], a["stride"], a["target"], -100, P, P, a["top"], a["ti"], P, P, a["gt"], a["dx"], 0) == -1


def _rows(*rows):
    flat = [v for r in rows for v in r]
    return (ctypes.c_longlong * len(flat))(*flat)


GOOD = [P, P, P, P, P, P, P, 100, 0]


@pytest.mark.parametrize("change", [dict(n=0), dict(bits=16), dict(ws=0), dict(nbytes=31), dict(ws=P + 8), dict(squares=0, n_squares=3), dict(n_squares=-1), dict(row=(0, 0)),
                                    dict(row=(1, 0)), dict(row=(2, 0)), dict(row=(3, 0)), dict(row=(4, 0)), dict(row=(5, 0)), dict(row=(6, 0)), dict(row=(7, -1)), dict(row=(8, 3))])
def test_adamw_step_refuses(lib, change):
    a = dict(n=1, bits=8, squares=P, n_squares=1, ws=P, nbytes=lib.w2c_adamw_workspace_bytes(1), row=(8, 0))
    a.update(change)
    row = list(GOOD)
    row[a["row"][0]] = a["row"][1]
    assert lib.w2c_adamw_step(_rows(row), a["n"], a["bits"], 1e-3, 0, 0.9, 0.999, 1e-8, 0.0, a["squares"], a["n_squares"], 1.0, 0, 0, a["ws"], a["nbytes"], 0) == -1


def test_grad_squares_counts_blocks_and_refuses(lib):
    assert lib.w2c_grad_squares_count(_rows(GOOD), 1) == 1 and lib.w2c_grad_squares_count(_rows(GOOD[:7] + [0, 0]), 1) == 0
    many = _rows(*[GOOD[:7] + [1 << 20, k % 3] for k in range(600)])          # 64 chunks each; 200 tensors of a type in launches of at most 190: at most 1 024 blocks a launch
    assert lib.w2c_grad_squares_count(many, 600) == 3 * (1024 + 640)
    assert lib.w2c_grad_squares_count(0, 1) == -1 and lib.w2c_grad_squares(_rows(GOOD), 1, 0, 1, 0) == -1 and lib.w2c_grad_squares(_rows(GOOD), 1, P, 0, 0) == -1


@pytest.mark.parametrize("change", [dict(a=0), dict(sa=0), dict(b=0), dict(sb=0), dict(c=0), dict(M=0), dict(N=0), dict(K=0), dict(K=100), dict(K=1 << 23), dict(ta=2), dict(tb=64),
                                    dict(dtype=3), dict(a=P + 8), dict(b=P + 1), dict(ws=0), dict(nbytes=5), dict(ws=P + 4)])
def test_matmul_fp8_refuses(lib, change):
    a = dict(a=P, sa=P, ta=1, b=P, sb=P, tb=128, M=100, N=100, K=4096, c=P, dtype=1, ws=P, nbytes=lib.w2c_matmul_fp8_workspace_bytes(100, 100, 4096))
    assert a["nbytes"] > 0 and lib.w2c_matmul_fp8_workspace_bytes(1, 100, 4096) == 0 and lib.w2c_matmul_fp8_workspace_bytes(0, 1, 128) == -1
    a.update(change)
    assert lib.w2c_matmul_fp8(a["a"], a["sa"], a["ta"], a["b"], a["sb"], a["tb"], a["M"], a["N"], a["K"], 0, a["c"], a["dtype"], a["ws"], a["nbytes"], 0) == -1


@pytest.mark.parametrize("change", [dict(x=0), dict(dtype=3), dict(rows=0), dict(cols=0), dict(stride=9), dict(tile=2), dict(codes=0, codes_t=0, sums=0), dict(scale=0), dict(scale_t=0),
                                    dict(rows=65535 * 128 + 1), dict(codes_t=P + 8), dict(ws=0), dict(nbytes=1)])
def test_quantize_fp8_refuses(lib, change):
    assert lib.w2c_quantize_fp8_workspace_bytes(128, 10) == 0 and lib.w2c_quantize_fp8_workspace_bytes(0, 10) == -1
    a = dict(x=P, dtype=0, rows=200, cols=10, stride=10, tile=1, codes=P, scale=P, codes_t=P, scale_t=P, sums=P, ws=P, nbytes=lib.w2c_quantize_fp8_workspace_bytes(200, 10))
    a.update(change)
    assert lib.w2c_quantize_fp8(a["x"], a["dtype"], a["rows"], a["cols"], a["stride"], a["tile"], a["codes"], a["scale"], a["codes_t"], a["scale_t"], a["sums"], a["ws"],
                                a["nbytes"], 0) == -1
