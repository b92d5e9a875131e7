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


def state(cache):
    return list(cache.lens), [list(h) for h in cache.host], sorted(cache.free), cache.table.clone()


def same(a, b):
    return a[:3] == b[:3] and torch.equal(a[3], b[3])


@pytest.mark.parametrize("window,sinks", [(0, 0), (16, 2)])
def test_sequences_come_and_go(window, sinks):
    """A released sequence is served again beside one that goes on, with prompts and tokens of some sequences alone."""
    from neuralscript_b200.attention_layer import PagedCache
    layer = layer_of(window, sinks, seed=4)
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    a, b, c = (torch.randn(n, 96, device="cuda", generator=g).to(BF) for n in (70, 30, 40))
    want = [whole(layer, r.double(), layer.wqkv16.double(), layer.wo16.double(), [r.shape[0]]) for r in (a, b, c)]
    bound = 4 * half_step(BF)  # heads, their rotation, the weights, ctx
    cache = PagedCache(layer, 3, pages=14, page=8)
    y = layer.prompt(cache, torch.cat([a[:50], b[:20]]), [50, 20], which=[2, 0])
    assert cache.lens == [20, 0, 50]
    assert off(y, torch.cat([want[0][:50], want[1][:20]])) <= bound
    for i in range(10):
        y = layer.token(cache, torch.stack([b[20 + i], a[50 + i]]), which=[0, 2])
        assert off(y, torch.stack([want[1][20 + i], want[0][50 + i]])) <= bound
    cache.release(0)
    y = layer.prompt(cache, c[:35], [35], which=[1])
    assert off(y, want[2][:35]) <= bound
    y = layer.token(cache, torch.stack([c[35], a[60], b[0]]), which=[1, 2, 0])  # (the third begins with its token)
    assert off(y, torch.stack([want[2][35], want[0][60], want[1][0]])) <= bound
    y = layer.token(cache, torch.stack([b[1], c[36], a[61]]))  # all of them, in order
    assert off(y, torch.stack([want[1][1], want[2][36], want[0][61]])) <= bound
    assert cache.lens == [2, 37, 62]


def test_refused_calls_leave_the_cache_as_it_was():
    from neuralscript_b200.attention_layer import PagedCache
    layer = layer_of(0, 0)
    x = torch.zeros(60, 96, device="cuda", dtype=BF)
    cache = PagedCache(layer, 3, pages=6, page=8, width=5)
    layer.prompt(cache, x[:9], [9], which=[1])
    was = state(cache)
    for call in (lambda: layer.prompt(cache, x[:9], [9], which=[1]), lambda: layer.prompt(cache, x[:9], [8], which=[0]),
                 lambda: layer.prompt(cache, x[:9], [9], which=[3]), lambda: layer.prompt(cache, x[:9], [4, 5], which=[0, 0]),
                 lambda: layer.prompt(cache, x[:9], [10, -1], which=[0, 2]), lambda: layer.prompt(cache, x[:9], [4, 5], which=[0]),
                 lambda: layer.prompt(cache, x[:9].float(), [9], which=[0]), lambda: layer.prompt(cache, x[:40], [20, 20], which=[0, 2]),
                 lambda: layer.prompt(cache, x[:41], [41], which=[0]), lambda: layer.prompt(cache, x[:9], [9]),
                 lambda: layer.token(cache, x[:2]), lambda: layer.token(cache, x[:2], which=[1]), lambda: layer.token(cache, x[:2], which=[1, 1]),
                 lambda: layer.token(cache, x[:1], which=[-1]), lambda: layer.token(cache, x[:1].float(), which=[1]),
                 lambda: cache.grow([20, 20, 20]), lambda: cache.grow([1, 1])):
        with pytest.raises(ValueError):
            call()
        assert same(state(cache), was)
    assert layer.token(cache, x[:0], which=[]).shape == layer.prompt(cache, x[:0], [0, 0], which=[0, 2]).shape == (0, 96)
    assert same(state(cache), was)
    layer.token(cache, x[:3])
    assert cache.lens == [1, 10, 1]
