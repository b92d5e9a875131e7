"""The attention layer put together from the operators: gradients against
autograd in 64 bits, and prompt and single tokens against the whole sequence."""
import pytest
import torch

from attention_ref import half_step, mask

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def layer_of(window, sinks, **kw):
    from neuralscript_b200.attention_layer import AttentionLayer
    return AttentionLayer(96, 6, 2, 40, window=window, sinks=sinks, **kw)


def whole(layer, x, wqkv, wo, lens):
    """The layer from its definition, in x's type, from rows x of sequences of these lengths."""
    out, at = [], 0
    Hq, Hkv, dh = layer.Hq, layer.Hkv, layer.dh
    for n in lens:
        h = (x[at:at + n] @ wqkv.t()).view(n, Hq + 2 * Hkv, dh)
        at += n
        a = (torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * layer.freq.double()[None])[:, None]
        x0, x1 = h[:, :Hq + Hkv, :dh // 2], h[:, :Hq + Hkv, dh // 2:]
        t = torch.cat([x0 * a.cos() - x1 * a.sin(), x1 * a.cos() + x0 * a.sin()], -1)
        q, k = t[:, :Hq].transpose(0, 1), t[:, Hq:].transpose(0, 1).repeat_interleave(Hq // Hkv, 0)
        v = h[:, Hq + Hkv:].transpose(0, 1).repeat_interleave(Hq // Hkv, 0)
        z = (q @ k.transpose(1, 2) / dh ** 0.5).masked_fill(~mask(n, n, layer.seen["window"], layer.seen["sinks"], "cuda"), -torch.inf)
        out.append((torch.softmax(z, -1) @ v).transpose(0, 1).reshape(n, Hq * dh) @ wo.t())
    return torch.cat(out)


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_gradients(window, sinks):
    lens = [130, 1, 77]
    layer = layer_of(window, sinks)
    T = sum(lens)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = torch.randn(T, 96, device="cuda", generator=g).to(BF)
    dy = torch.randn(T, 96, device="cuda", generator=g).to(BF)
    offsets = torch.tensor([0, 130, 131, 208], dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(n, dtype=torch.int32, device="cuda") for n in lens])
    y, kept = layer.forward(x, offsets, pos)
    grads = layer.backward(dy, kept)
    leaves = [t.double().requires_grad_() for t in (x, layer.wqkv16, layer.wo16)]
    want = whole(layer, *leaves, lens)
    # what each passes through in bf16, half a step at a time: heads, the rotation, weights, ctx; back dctx, P and dS,
    # the heads' gradients and their rotation. Their errors are independent; the sum of their bounds holds all the same
    steps = 8 * half_step(BF)
    assert off(y, want.detach()) <= steps
    want.backward(dy.double())
    for name, got, leaf in zip(("dx", "dwqkv", "dwo"), grads, leaves):
        assert off(got, leaf.grad) <= steps, name


@pytest.mark.parametrize("window,sinks", [(0, 0), (16, 2)])
def test_prompt_then_tokens(window, sinks):
    from neuralscript_b200.attention_layer import PagedCache
    layer = layer_of(window, sinks, seed=4)
    lens, steps = [50, 9], 12
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    rows = [torch.randn(n + steps, 96, device="cuda", generator=g).to(BF) for n in lens]
    want = [whole(layer, r.double(), layer.wqkv16.double(), layer.wo16.double(), [r.shape[0]]) for r in rows]
    cache = PagedCache(layer, 2, pages=12, page=8)
    y = layer.prompt(cache, torch.cat([r[:n] for r, n in zip(rows, lens)]), lens)
    bound = 4 * half_step(BF)  # heads, their rotation, the weights, ctx
    assert off(y, torch.cat([w[:n] for w, n in zip(want, lens)])) <= bound
    for i in range(steps):
        y = layer.token(cache, torch.stack([r[n + i] for r, n in zip(rows, lens)]))
        assert off(y, torch.stack([w[n + i] for w, n in zip(want, lens)])) <= bound
    with pytest.raises(ValueError, match="no room"):
        cache.grow([1000, 0])
    with pytest.raises(ValueError, match="empty"):
        layer.prompt(cache, rows[0], [62, 0])
    had = len(cache.free)
    cache.release(0)
    assert len(cache.free) == had + 8


def test_training_and_serving_run(capsys):
    from neuralscript_b200 import attention_layer
    attention_layer.main()
    assert "serving" in capsys.readouterr().out


def test_refusals():
    from neuralscript_b200.attention_layer import AttentionLayer
    for bad in ((64, 3, 2, 64), (64, 2, 2, 60), (64, 2, 2, 136), (60, 2, 2, 64)):
        with pytest.raises(ValueError):
            AttentionLayer(*bad)
    layer = layer_of(0, 0)
    for x in (torch.zeros(4, 96, device="cuda"), torch.zeros(4, 95, device="cuda", dtype=BF), torch.zeros(96, 4, device="cuda", dtype=BF).t()):
        with pytest.raises(ValueError):
            layer._heads(x)
