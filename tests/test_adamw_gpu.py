"""AdamW over many tensors (w2c_adamw_step, optim.AdamW) against the formulas in 64 bits.

Tolerances: U = 2^-24.  A moment is two products and a sum, the clipped gradient one product more: 4 U of the magnitudes.  The update is a hardware root and
reciprocal (1 step of f32 = 2 U each), their operands' 6 U and four more roundings: 16 U of itself; the parameter adds 3 U and, where it has fewer bits, half a
step of its type.  An 8-bit moment is the e4m3 multiple below or above the value in units of its block's scale, chosen by the hash: within one step,
2^-3 of the value's power of two, never below 2^-9 of the scale; with the same hash and a value 8 U off, one element in 2^20 / 2^7 may round the other way."""
import copy
import math

import pytest
import torch

from multiagentperception_amd import ops, optim
from multiagentperception_amd._native import W2CError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
HP = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)


def _tensors(sizes, dtypes, bits, seed, t0=3.0, gscale=0.3):
    g = torch.Generator().manual_seed(seed)
    r = lambda n, k: torch.randn(n, generator=g) * k                              # noqa: E731
    p = [r(n, 1.0).to(d).cuda() for n, d in zip(sizes, dtypes)]
    gr = [r(n, gscale).to(d).cuda() for n, d in zip(sizes, dtypes)]
    m, v = [r(n, 0.1).cuda() for n in sizes], [(r(n, 0.1) ** 2 + 1e-8).cuda() for n in sizes]
    steps = [torch.tensor(t0 + i % 3, device="cuda") for i in range(len(sizes))]
    if bits == 32:
        return p, gr, list(zip(m, v)), steps
    held = [(*_encode(a.double(), torch.full_like(a.double(), 0.5), False), *_encode(b.double().sqrt(), torch.full_like(a.double(), 0.5), True))
            for a, b in zip(m, v)]
    return p, gr, [(mc.to(E4M3), ms.view(torch.uint8).view(E8M0), vc.to(E4M3), vs) for mc, ms, vc, vs in held], steps


def _two_to(e):
    """2^e in 64 bits by its exponent field: the GPU's pow is a step off now and then"""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(x, noise, positive):
    """-> (values of the codes, f64; scales) of x f64 [n] with the noise in [0, 1)"""
    n = x.numel()
    t = torch.cat([x, x.new_zeros(-n % 256)]).view(-1, 256)
    top = t.float().abs().amax(1).double()
    e = torch.where(top > 0, torch.ceil(torch.log2(top / 448.0)), torch.zeros_like(top))
    e = torch.where(top > 448.0 * _two_to(e), e + 1, torch.where((top > 0) & (top <= 224.0 * _two_to(e)), e - 1, e))
    u = (t / _two_to(e)[:, None]).view(-1)[:n]
    step = _two_to(torch.clamp(torch.frexp(u)[1] - 1, min=-6) - 3)
    q = (torch.floor(u.abs() / step + noise) * step).clamp(max=448.0)
    if positive:
        q = torch.where(u > 0, q.clamp(min=2.0 ** -9), q)
    return q * torch.sign(u), (e + 127).to(torch.uint8).view(E8M0)


def _hash(n, seed, t):
    low = 0xFFFFFFFF
    i = torch.arange(n, device="cuda", dtype=torch.int64)
    x = (i * 0xA3D8F62B + ((seed * 0x9E3779B1 + t * 0x85EBCA6B) & low)) & low
    x = ((x ^ (x >> 15)) * 0xC58B3E95) & low
    x = ((x ^ (x >> 13)) * 0x9E3779B1) & low
    return x ^ (x >> 16)


def _value(codes, scale):
    return codes.double() * scale.double().repeat_interleave(256)[:codes.numel()]


def _check(sizes, dtypes, bits, seed=1, max_norm=None, hp=HP, **kw):
    p, g, states, steps = _tensors(sizes, dtypes, bits, seed, **kw)
    before = [t.double() for t in p]
    held = [((s[0].double(), s[1].double()) if bits == 32 else (_value(s[0], s[1]), _value(s[2], s[3]) ** 2)) for s in states]
    t = [float(s) + 1 for s in steps]
    norm = ops.adamw_step(p, g, states, steps, max_norm=max_norm, seed=seed, **hp)
    factor = 1.0
    if max_norm is not None:
        want = math.sqrt(sum(float((x.double() ** 2).sum()) for x in g))
        assert abs(float(norm) - want) <= 2 * U * want
        factor = min(1.0, max_norm / (want + 1e-6))
    else:
        assert norm is None
    flips = total = 0
    for i, n in enumerate(sizes):
        assert float(steps[i]) == t[i]
        gd = g[i].double() * factor
        m0, v0 = held[i]
        m = hp["beta1"] * m0 + (1 - hp["beta1"]) * gd
        v = hp["beta2"] * v0 + (1 - hp["beta2"]) * gd * gd
        msize = hp["beta1"] * m0.abs() + (1 - hp["beta1"]) * gd.abs()
        den = (v / (1 - hp["beta2"] ** t[i])).sqrt() + hp["eps"]
        k = hp["lr"] / (1 - hp["beta1"] ** t[i])
        want = before[i] * (1 - hp["lr"] * hp["weight_decay"]) - k * m / den
        half = torch.finfo(dtypes[i]).eps / 2 if dtypes[i] != F32 else 0.0
        tol = half * want.abs() + (1 + half) * (16 * U * k * msize / den + 3 * U * (before[i].abs() + want.abs()))
        assert ((p[i].double() - want).abs() <= tol + (2.0 ** -24 if dtypes[i] == F16 else 0)).all()
        if bits == 32:
            assert ((states[i][0].double() - m).abs() <= 4 * U * msize + 1e-45).all()
            assert ((states[i][1].double() - v).abs() <= 6 * U * v + 1e-45).all()
        else:
            r = _hash(n, seed, int(t[i]))
            for x, code, scale, noise, positive in ((m, states[i][0], states[i][1], (r & 0xFFFF), False), (v.sqrt(), states[i][2], states[i][3], r >> 16, True)):
                q, s = _encode(x, (noise.double() + 0.5) / 65536, positive)
                assert torch.equal(scale.view(torch.uint8), s.view(torch.uint8))
                unit = s.double().repeat_interleave(256)[:n]
                step = unit * _two_to(torch.clamp(torch.frexp(x / unit)[1] - 1, min=-6) - 3)
                off = (_value(code, scale) - q * unit).abs()
                assert (off <= step * (1 + 1e-9)).all()
                flips += int((off > 0).sum())
                total += n
    assert flips <= 1 + total / 2 ** 13 * 4


MIX = [1, 3, 255, 256, 257, 4096, 4097, 70000, 2, 9000]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F16], [F32, BF16, F16]])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e9])
def test_a_step_over_a_mix_of_tensors(dtypes, bits, max_norm):
    _check(MIX, [dtypes[i % len(dtypes)] for i in range(len(MIX))], bits, max_norm=max_norm)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_launch_takes(bits):
    sizes = [(i * 37) % 600 + 1 for i in range(301)]
    _check(sizes, [F32] * 301, bits, seed=2, max_norm=1.0)
    _check([300000, 5], [BF16, BF16], bits, seed=3)


def test_first_step_large_and_small_gradients_and_no_decay():
    for scale in (1e-12, 1e12):
        _check([1000], [F32], 32, seed=4, t0=0.0, gscale=scale, hp=dict(HP, weight_decay=0.0))
        _check([1000], [F32], 8, seed=4, t0=0.0, gscale=scale, max_norm=3.0)


def test_zeros_stay_zeros_and_empty_tensors_only_count():
    p = [torch.zeros(300, device="cuda"), torch.zeros(0, device="cuda")]
    g = [torch.zeros_like(t) for t in p]
    steps = [torch.zeros(1, device="cuda") for _ in p]
    for bits in (8, 32):
        st = [tuple(optim.AdamW._fresh(t, bits).values())[1:] for t in p]
        ops.adamw_step(p, g, st, steps, max_norm=1.0)
        assert not p[0].any() and not st[0][0].float().any() and not st[0][2 if bits == 8 else 1].float().any()
    assert [float(t) for t in steps] == [2.0, 2.0]


def test_what_is_not_finite_stays_in_its_element():
    for bits in (32, 8):
        p, g, st, steps = _tensors([600], [F32], bits, 5)
        g[0][7], g[0][300] = float("nan"), float("inf")
        ops.adamw_step(p, g, st, steps, **HP)
        bad = torch.zeros(600, dtype=torch.bool, device="cuda")
        bad[7] = bad[300] = True
        assert torch.equal(p[0].isnan(), bad)
        for t in (st[0][0], st[0][1 if bits == 32 else 2]):
            assert torch.equal(~t.float().isfinite(), bad)
        ops.adamw_step(p, [torch.zeros_like(g[0])], st, steps, **HP)
        assert torch.equal(p[0].isnan(), bad)


def test_the_second_moment_decays_in_8_bits():
    """100 steps without gradients: sqrt(v) falls by 0.99^50 on the average, though a step moves it by half a per cent of itself"""
    n = 1 << 16
    p, g, st, steps = _tensors([n], [F32], 8, 6)
    start = _value(st[0][2], st[0][3]) ** 2
    zero = [torch.zeros_like(g[0])]
    for _ in range(100):
        ops.adamw_step(p, zero, st, steps, seed=9, **HP)
    end = _value(st[0][2], st[0][3]) ** 2
    # the mean of n independent roundings: its deviation is far below 3 % of the decay that is asked for
    assert abs(float(end.sum() / start.sum()) / 0.99 ** 100 - 1) <= 0.1


def test_the_same_bits_every_time_and_another_seed_others():
    def once(seed):
        p, g, st, steps = _tensors([50000, 77], [BF16, BF16], 8, 7)
        ops.adamw_step(p, g, st, steps, seed=seed, max_norm=1.0, **HP)
        return p + [t.view(torch.uint8) for s in st for t in s]
    a, b, c = once(1), once(1), once(2)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and not torch.equal(a[2], c[2])


class _Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.conv = torch.nn.Conv2d(8, 16, 3).to(memory_format=torch.channels_last)
        self.a, self.b = torch.nn.Linear(40, 30), torch.nn.Linear(30, 5)
        self.unused = torch.nn.Parameter(torch.zeros(3))


def _grads(net, seed):
    g = torch.Generator().manual_seed(seed)
    for p in net.parameters():
        if p is not net.unused:
            p.grad = torch.randn(p.shape, generator=g).to(p.dtype).cuda()          # contiguous: not the channels_last parameter's layout


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_against_torch_and_through_a_state_dict(bits):
    torch.manual_seed(1)
    net = _Net().cuda()
    twin = copy.deepcopy(net)
    groups = lambda m: [{"params": list(m.conv.parameters()), "lr": 3e-3}, {"params": [*m.a.parameters(), *m.b.parameters(), m.unused]}]   # noqa: E731
    opt = optim.AdamW(groups(net), lr=1e-3, weight_decay=0.05, state_bits=bits, max_norm=0.7)
    ref = torch.optim.AdamW(groups(twin), lr=1e-3, weight_decay=0.05)
    versions = [p._version for p in net.parameters()]
    for k in range(4):
        _grads(net, k)
        _grads(twin, k)
        want = torch.nn.utils.clip_grad_norm_(twin.parameters(), 0.7)
        opt.step()
        ref.step()
        assert abs(float(opt.last_norm) - float(want)) <= 1e-5 * float(want)
    assert not opt.state[net.unused] and all(p._version > v for p, v in zip(net.parameters(), versions) if p is not net.unused)
    # 32 bits: the same formula in f32, 40 roundings a step of terms up to lr and |p|; 8 bits: an update is at most a quarter off (a code's step is an eighth)
    for p, q in zip(net.parameters(), twin.parameters()):
        tol = 4 * 40 * U * (float(q.abs().max()) + 3e-3) if bits == 32 else 4 * 3e-3 * 1.25
        assert float((p - q).abs().max()) <= tol
    saved = copy.deepcopy(opt.state_dict())
    other = _Net().cuda()
    other.load_state_dict(net.state_dict())
    opt2 = optim.AdamW(groups(other), lr=1.0, state_bits=bits, max_norm=0.7)
    opt2.load_state_dict(saved)
    for o, m in ((opt, net), (opt2, other)):
        _grads(m, 10)
        o.step()
    for p, q in zip(net.parameters(), other.parameters()):
        assert torch.equal(p, q)
        for k, v in opt.state[p].items():
            assert v.dtype == opt2.state[q][k].dtype


def test_half_parameters_keep_their_moments_through_a_state_dict():
    p = torch.nn.Parameter(torch.randn(500, device="cuda", dtype=BF16))
    opt = optim.AdamW([p])
    p.grad = torch.randn_like(p)
    opt.step()
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert opt.state[p]["exp_avg"].dtype == F32 and opt.state[p]["step"].dtype == F32
    opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_of_a_captured_step_equal_eager_steps_and_follow_a_tensor_lr(bits):
    lr = torch.full((1,), 1e-2, device="cuda")
    p, q = (torch.nn.Parameter(torch.linspace(-1, 1, 5000, device="cuda")) for _ in range(2))
    opt, eager = (optim.AdamW([t], lr=lr, state_bits=bits, max_norm=1.0) for t in (p, q))
    p.grad, q.grad = torch.randn(5000, device="cuda"), torch.zeros(5000, device="cuda")
    q.grad.copy_(p.grad)
    opt.step()
    eager.step()
    with ops.capture(thread_local=False) as graph:
        opt.step()
    for k in range(4):
        lr.fill_(1e-2 / (k + 1))
        new = torch.randn(5000, generator=torch.Generator().manual_seed(k)).cuda()
        p.grad.copy_(new)
        q.grad.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        eager.step()
        assert torch.equal(p, q)


def test_refusals():
    p, g, st, steps = _tensors([300, 300], [F32, F32], 32, 8)
    p8, g8, st8, steps8 = _tensors([300, 300], [F32, F32], 8, 8)
    wide = torch.zeros(300, 2, device="cuda")
    for bad in (lambda: ops.adamw_step([], [], [], []), lambda: ops.adamw_step(p, g[:1], st, steps), lambda: ops.adamw_step(p, g, st[:1], steps),
                lambda: ops.adamw_step(p, g, st, steps[:1]), lambda: ops.adamw_step([p[0], p[0]], g, st, steps), lambda: ops.adamw_step(p, g, [st[0], st[0]], steps),
                lambda: ops.adamw_step(p, g, st, [steps[0], steps[0]]), lambda: ops.adamw_step(p, [g[0], g[1].half()], st, steps),
                lambda: ops.adamw_step(p, [g[0], g[1][:299]], st, steps), lambda: ops.adamw_step(p, [g[0], g[1].cpu()], st, steps),
                lambda: ops.adamw_step([t.cpu() for t in p], [t.cpu() for t in g], st, steps), lambda: ops.adamw_step([p[0], p[1].double()], [g[0], g[1].double()], st, steps),
                lambda: ops.adamw_step(p, g, [st[0], (st[1][0].half(), st[1][1])], steps), lambda: ops.adamw_step(p, g, st, [steps[0], steps[1].double()]),
                lambda: ops.adamw_step(p, g, [st[0], st8[1]], steps), lambda: ops.adamw_step(p8, g8, [st8[0], (st8[1][0], st8[1][1][:1], *st8[1][2:])], steps8),
                lambda: ops.adamw_step(p, g, st, steps, max_norm=0.0), lambda: ops.adamw_step(p, g, st, steps, lr=torch.zeros(1)),
                lambda: ops.adamw_step(p, g, st, steps, max_norm=1.0, squares=torch.ones(3, device="cuda")),
                lambda: ops.adamw_step([wide[:, 0], p[1]], [wide[:, 1], g[1]], st, steps)):
        with pytest.raises(W2CError):
            bad()
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(max_norm=0.0)):
        with pytest.raises(ValueError):
            optim.AdamW([torch.nn.Parameter(p[0])], **kw)
