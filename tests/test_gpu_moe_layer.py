"""The top-k mixture-of-experts layer on the GPU: forward, gradients and
serving against the same layer in 64 bits on the values that the 8-bit
weights stand for."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from neuralscript_b200.moe_topk import MoETopk  # noqa: E402


def values(q, s):
    E, N, K = q.shape
    return q.double() * s.double().repeat_interleave(128, 1)[:, :N].repeat_interleave(128, 2)[:, :, :K]


def reference(layer, x, idx):
    """y, and the leaves x, gate, w1, w2, with the choice held."""
    x = x.double().requires_grad_(True)
    gate = layer.gate16.double().requires_grad_(True)
    w1, w2 = values(*layer.q1).requires_grad_(True), values(*layer.q2).requires_grad_(True)
    p = torch.sigmoid(x @ gate.t()).gather(1, idx.long())
    w = p / p.sum(1, keepdim=True)
    y = 0
    for j in range(idx.shape[1]):
        e = idx[:, j].long()
        h = torch.nn.functional.gelu(torch.einsum("thd,td->th", w1[e], x))
        y = y + w[:, j:j + 1] * torch.einsum("tdh,th->td", w2[e], h)
    return y, (x, gate, w1, w2)


def off(a, b):
    return float((a.double() - b.detach()).norm() / b.detach().norm())


# An e4m3 rounding is off by at most 2^-4, on average over a step's range about
# 2^-5.5 = 0.022 of a value; a product's error is that of its two operands (one
# exact here on the weights' side in forward and input gradient), and at most
# four roundings lie one after another.
ONE = 0.03


@pytest.mark.parametrize("M,E,k", [(1, 4, 2), (200, 8, 2), (333, 5, 3)])
def test_layer_against_64_bits(M, E, k):
    layer = MoETopk(128, 256, E, k, seed=M)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = torch.randn(M, 128, device="cuda", generator=g).to(torch.bfloat16)
    dy = torch.randn(M, 128, device="cuda", generator=g)
    y, kept = layer.forward(x, align=128)
    ref, leaves = reference(layer, x, kept["idx"])
    assert off(y, ref) < 2 * ONE
    (ref * dy.double()).sum().backward()
    for got, leaf in zip(layer.backward(dy, kept), leaves):
        assert off(got, leaf.grad) < 4 * ONE
    served, _ = layer.forward(x)  # without padding
    assert off(served, y.double()) < 1e-5


def test_layer_trains_and_serves_single_tokens():
    layer, teacher = MoETopk(128, 128, 8, 2, groups=4, topk_groups=2, seed=1), MoETopk(128, 128, 8, 2, seed=2)
    x = torch.randn(512, 128, device="cuda", dtype=torch.bfloat16)
    target, _ = teacher.forward(x)
    losses = [float(layer.train_step(x, target, 3e-3)) for _ in range(40)]
    assert losses[-1] < 0.5 * losses[0]
    y, _ = layer.forward(x)
    one, _ = layer.forward(x[17:18])
    assert off(one[0], y[17].double()) < 1e-5


@pytest.mark.parametrize("align", [1, 64])
def test_backward_refuses_unaligned_segments(align):
    """64 tokens, 2 experts each: 128 pairs, so that every buffer's shape fits and only the sums would be wrong."""
    layer = MoETopk(128, 128, 4, 2, seed=3)
    x = torch.randn(64, 128, device="cuda").to(torch.bfloat16)
    y, kept = layer.forward(x, align=align)
    with pytest.raises(ValueError, match="align"):
        layer.backward(torch.ones_like(y), kept)


def test_forward_refuses_other_inputs():
    layer = MoETopk(128, 128, 4, 2, seed=4)
    x = torch.randn(256, 256, device="cuda").to(torch.bfloat16)
    for bad in (x, x[:, :64], x[:, :128].float(), x[:128].t()[:, :128], x[0, :128], x[:, :128].cpu()):
        with pytest.raises(ValueError, match="wanted"):
            layer.forward(bad)
    assert torch.equal(layer.forward(x[:, 64:192])[0], layer.forward(x[:, 64:192].contiguous())[0])


def test_failed_products_stop_the_step(monkeypatch):
    layer = MoETopk(128, 128, 4, 2, seed=5)
    x = torch.randn(64, 128, device="cuda").to(torch.bfloat16)
    layer.err.fill_(102)  # (no product runs while it is set)
    with pytest.raises(RuntimeError, match="102"):
        layer.check()
    layer.check()  # read once
    before = [w.clone() for w in (layer.gate, layer.w1, layer.w2)]

    def failed():
        raise RuntimeError("device error 101")

    monkeypatch.setattr(layer, "check", failed)
    with pytest.raises(RuntimeError, match="101"):
        layer.train_step(x, x.float(), 1e-3)
    assert all(torch.equal(a, b) for a, b in zip(before, (layer.gate, layer.w1, layer.w2)))
    monkeypatch.undo()
    layer.train_step(x, x.float(), 1e-3)
    assert not torch.equal(before[1], layer.w1)
