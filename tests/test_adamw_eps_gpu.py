"""AdamW with eps = 0, where the root of the second moment alone is under the update."""
import pytest
import torch

from multiagentperception_amd import ops, optim

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _first_step(g, bits, **hp):
    p = torch.linspace(-1, 1, g.numel(), device="cuda").to(g.dtype)
    state = tuple(optim.AdamW._fresh(p, bits).values())[1:]
    before = p.double()
    ops.adamw_step([p], [g], [state], [torch.zeros((), device="cuda")], lr=0.25, beta1=0.5, beta2=0.75, eps=0.0, weight_decay=0.0, **hp)
    return before, p.double()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size", [1e-17, 1e-19, 3e-21])
def test_small_gradients(size, bits):
    """the first step moves by lr * sign(g), whatever g's size: m / (1 - b1) = g, v / (1 - b2) = g^2.  v = g^2 / 4 is a multiple of 2^-149 within two halves of it;
    the root halves that relative error.  The rest is f32's: 16 roundings of the update, 3 of the parameter (U = 2^-24)."""
    U = 2.0 ** -24
    g = torch.randn(3000, generator=torch.Generator().manual_seed(1)).mul(size).cuda()
    before, after = _first_step(g, bits)
    v = g.double() ** 2 / 4
    there = v >= 2.0 ** -147
    assert there.sum() > 1500
    tol = 0.25 * (16 * U + 2.0 ** -149 / v.clamp(min=2.0 ** -147)) + 3 * U * (before.abs() + 0.25)
    assert ((after - (before - 0.25 * g.double().sign())).abs() <= tol)[there].all()
    assert after.isfinite().all() and ((after - before).abs() <= 0.25 * 2.001).all()             # v of 2^-149, half of its last bit: at most a root of 4 off


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_no_gradient_leaves_an_element_as_it_is(bits, dtype):
    g = torch.zeros(700, dtype=dtype, device="cuda")
    g[::7] = 0.5
    before, after = _first_step(g, bits)
    still = g == 0
    assert torch.equal(after[still], before[still]) and (after != before)[~still].all() and after.isfinite().all()
    before, after = _first_step(g, bits, max_norm=1e-30)                  # clipped to where the square is below f32
    assert after.isfinite().all()


@pytest.mark.parametrize("bits", [32, 8])
def test_what_is_not_a_number_stays_one(bits):
    g = torch.zeros(300, device="cuda")
    g[5], g[6] = float("nan"), float("inf")
    before, after = _first_step(g, bits)
    assert after.isnan().nonzero().flatten().tolist() == [5, 6]
