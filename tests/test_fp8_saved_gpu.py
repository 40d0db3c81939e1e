"""What an 8-bit linear layer keeps for its backward: tensors that autograd knows of."""
import pytest
import torch
import torch.utils.checkpoint

from multiagentperception_amd import ops, train_ops

pytestmark = pytest.mark.gpu
F8 = (torch.float8_e4m3fn, torch.float8_e8m0fnu)


def _layer(rows=300, width=400, out=256):
    g = torch.Generator(device="cuda").manual_seed(rows)
    m = train_ops.LinearFp8(width, out, device="cuda")
    with torch.no_grad():
        m.weight.copy_(torch.randn(out, width, generator=g, device="cuda"))
    return m, torch.randn(rows, width, generator=g, device="cuda", requires_grad=True), torch.randn(rows, out, generator=g, device="cuda")


def test_a_second_backward_is_refused_and_a_retained_one_gives_the_same():
    m, x, dy = _layer()
    y = m(x)
    first = torch.autograd.grad(y, (x, m.weight), dy, retain_graph=True)
    second = torch.autograd.grad(y, (x, m.weight), dy)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, (x, m.weight), dy)


def test_a_backward_frees_what_the_layers_keep_while_the_loss_is_held():
    layers = [_layer(4096, 1024, 1024)[0] for _ in range(4)]
    x = torch.randn(4096, 1024, device="cuda")
    y = x
    for m in layers:
        y = m(y)
    loss = y.sum()
    del y
    held = torch.cuda.memory_allocated()
    loss.backward()
    for m in layers:
        m.zero_grad(set_to_none=True)
    # each layer kept its 4 MiB of transposed input codes; those after the first the transposed weights' too
    assert held - torch.cuda.memory_allocated() >= 4 * 4096 * 1024


def test_hooks_of_saved_tensors_see_the_operands():
    m, x, dy = _layer()
    want = torch.autograd.grad(m(x), (x, m.weight, m.bias), dy)
    seen = []

    def pack(t):
        seen.append(t.dtype)
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        y = m(x)
    assert [seen.count(d) for d in F8] == [2, 2]
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, m.weight, m.bias), dy), want))


@pytest.mark.parametrize("reentrant", [False, True])
def test_under_a_checkpoint_the_gradients_are_the_same(reentrant):
    m, x, dy = _layer()
    want = torch.autograd.grad(m(x), (x, m.weight, m.bias), dy)
    torch.utils.checkpoint.checkpoint(m, x, use_reentrant=reentrant).backward(dy)
    assert all(torch.equal(a, b) for a, b in zip((x.grad, m.weight.grad, m.bias.grad), want))


def test_frozen_parts_are_not_kept():
    m, x, dy = _layer()
    seen = []
    hooks = lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(t.dtype), t)[1], lambda t: t)        # noqa: E731
    with hooks():
        y = m(x.detach())
    assert len(seen) == 2 and torch.autograd.grad(y, m.weight, dy)[0].any()                # the transposed input alone
    m.weight.requires_grad_(False)
    seen.clear()
    with hooks():
        y = m(x)
    assert len(seen) == 2 and torch.autograd.grad(y, x, dy)[0].any()                       # the transposed weights alone


def test_without_gradients_nothing_is_transposed(monkeypatch):
    m, x, dy = _layer()
    asked, real = [], ops.quantize_fp8

    def spy(t, tile=1, rows=True, columns=False, sums=False):
        asked.append((rows, columns, sums))
        return real(t, tile, rows, columns, sums)

    monkeypatch.setattr(ops, "quantize_fp8", spy)
    y = m(x)
    assert asked == [(True, True, False)] * 2
    asked.clear()
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            assert torch.equal(m(x), y)
    assert asked == [(True, False, False)] * 4
