"""An attention layer that answers token by token: rotary positions, a sliding
window with a few first tokens that stay visible, and a paged cache of keys and
values, the operators of ``ops`` put together as a program uses them.

    y = Wo attention(rope(Wq x), rope(Wk x), Wv x)

Training runs over packed sequences, forward and backward. Serving writes a
prompt's keys and values into the cache and then takes one token a sequence at a
time. ``python -m neuralscript_b200.attention_layer`` trains a small layer and
serves it.

torch holds the buffers; every product, rotation and attention is a kernel of
this package.
"""
from __future__ import annotations

import torch

from . import ops

BF16 = torch.bfloat16


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class PagedCache:
    """Keys and values of up to B sequences in pages of `page` places, given out as sequences grow."""

    def __init__(self, layer, B, pages, page=32, width=None):
        shape = (pages, page, layer.Hkv, layer.dh)
        self.k, self.v = (torch.empty(shape, dtype=BF16, device="cuda") for _ in "kv")
        self.page, self.free = page, list(range(pages))
        self.host = [[] for _ in range(B)]  # pages of every sequence
        self.lens = [0] * B
        self.width = pages if width is None else width  # fixed, so that a captured step finds its table again
        self.table = torch.zeros(B, self.width, dtype=torch.int32, device="cuda")

    def chosen(self, which):
        """The sequences' numbers: all, or those of `which`, each once."""
        B = len(self.lens)
        which = list(range(B) if which is None else which)
        if len(set(which)) != len(which) or not all(0 <= b < B for b in which):
            raise ValueError(f"sequences {which} where different ones of 0 to {B - 1} are wanted")
        return which

    def grow(self, new, which=None):
        """Room for new[i] tokens more of sequence which[i] (of every sequence): of all of them or, where it does not
        suffice, of none."""
        which, new = self.chosen(which), list(new)
        if len(new) != len(which) or min(new, default=0) < 0:
            raise ValueError(f"{new} tokens for {len(which)} sequences")
        places, left = [], len(self.free)
        for b, n in zip(which, new):
            had, need = len(self.host[b]), -(-(self.lens[b] + n) // self.page)
            left -= max(0, need - had)
            if need > self.width or left < 0:
                raise ValueError(f"sequence {b}: no room for {self.lens[b] + n} tokens")
            places += [(b, i) for i in range(had, need)]
        if places:
            for b, _ in places:
                self.host[b].append(self.free.pop())
            rows, cols = zip(*places)
            rows, cols, pages = _ints([rows, cols, [self.host[b][i] for b, i in places]])
            self.table[rows, cols] = pages

    def release(self, b):
        """Gives sequence b's pages back; a prompt or a token may begin it again."""
        self.free += self.host[b]
        self.host[b], self.lens[b] = [], 0


class AttentionLayer:
    """Wqkv [(Hq + 2 Hkv) dh, D] and Wo [D, Hq dh], in fp32; dh a multiple of 8, at most 128."""

    def __init__(self, D, Hq, Hkv, dh, window=0, sinks=0, theta=10000.0, seed=0):
        if Hq % Hkv or dh % 8 or dh > 128 or D % 8:
            raise ValueError("Hkv divides Hq, dh is a multiple of 8 of at most 128, D a multiple of 8")
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.D, self.Hq, self.Hkv, self.dh = D, Hq, Hkv, dh
        self.N = (Hq + 2 * Hkv) * dh
        self.seen = dict(window=window, sinks=sinks)
        self.freq = (theta ** (-torch.arange(dh // 2, dtype=torch.float64) / (dh // 2))).float().cuda()
        self.wqkv = torch.randn(self.N, D, device="cuda", generator=g) / D ** 0.5
        self.wo = torch.randn(D, Hq * dh, device="cuda", generator=g) / (Hq * dh) ** 0.5
        self.count = 0
        self._moments = [(torch.zeros_like(w), torch.zeros_like(w)) for w in (self.wqkv, self.wo)]
        self.refresh()

    def refresh(self):
        """Rounds the weights to the products' type (after they change)."""
        self.wqkv16, self.wo16 = self.wqkv.to(BF16), self.wo.to(BF16)

    def _check(self, x):
        if x.dtype != BF16 or x.dim() != 2 or x.shape[1] != self.D or not x.is_contiguous():
            raise ValueError(f"x: {x.dtype} {tuple(x.shape)} where rows of {self.D} bfloat16 are wanted")

    def _heads(self, x):
        """Queries, keys and values [T, Hq + 2 Hkv, dh] of x [T, D] (bf16, contiguous)."""
        self._check(x)
        T = x.shape[0]
        heads = torch.empty(T, self.N, dtype=BF16, device="cuda")
        ops.gemm(x, self.wqkv16, T, self.N, self.D, self.D, 0, self.D, 0, c16=heads)
        return heads.view(T, -1, self.dh)

    def _split(self, heads):
        Hq, Hkv = self.Hq, self.Hkv
        return heads[:, :Hq], heads[:, Hq:Hq + Hkv], heads[:, Hq + Hkv:]

    def _out(self, ctx):
        T, HD = ctx.shape[0], self.Hq * self.dh
        y = torch.empty(T, self.D, device="cuda")
        ops.gemm(ctx, self.wo16, T, self.D, HD, HD, 0, HD, 0, c32=y)
        return y

    def forward(self, x, offsets, pos):
        """y [T, D] (fp32) of packed sequences x [T, D] (bf16; offsets [B + 1], pos [T], int32), and what the backward
        pass needs."""
        T = x.shape[0]
        heads = self._heads(x)
        turned = heads[:, :self.Hq + self.Hkv]
        ops.rope(turned, pos, self.freq, turned)
        ctx, lse = torch.zeros(T, self.Hq, self.dh, dtype=BF16, device="cuda"), torch.empty(self.Hq, T, device="cuda")
        ops.attention_window(*self._split(heads), ctx, lse=lse, offsets=offsets, **self.seen)
        return self._out(ctx), dict(x=x, heads=heads, ctx=ctx, lse=lse, offsets=offsets, pos=pos)

    def backward(self, dy, kept):
        """Gradients (dx [T, D], dWqkv, dWo) of the loss whose gradient in y is dy [T, D]."""
        x, heads, ctx = kept["x"], kept["heads"], kept["ctx"]
        T, D, HD, N = x.shape[0], self.D, self.Hq * self.dh, self.N
        dy = dy.to(BF16).contiguous()
        dctx = torch.empty(T, HD, dtype=BF16, device="cuda")
        ops.gemm(dy, self.wo16, T, HD, D, D, 0, HD, 1, c16=dctx)
        dwo = torch.empty(D, HD, device="cuda")
        ops.gemm(dy, ctx, D, HD, T, D, 1, HD, 1, c32=dwo)
        dheads = torch.zeros_like(heads)
        ops.attention_window_bwd(*self._split(heads), ctx, kept["lse"], dctx.view(T, self.Hq, self.dh), *self._split(dheads),
                                 offsets=kept["offsets"], **self.seen)
        turned = dheads[:, :self.Hq + self.Hkv]
        ops.rope_bwd(turned, kept["pos"], self.freq, turned)
        dx, dwqkv = torch.empty(T, D, device="cuda"), torch.empty(N, D, device="cuda")
        ops.gemm(dheads, self.wqkv16, T, D, N, N, 0, D, 1, c32=dx)
        ops.gemm(dheads, x, N, D, T, N, 1, D, 1, c32=dwqkv)
        return dx, dwqkv, dwo

    def train_step(self, x, offsets, pos, target, lr):
        """Mean squared error before the step."""
        y, kept = self.forward(x, offsets, pos)
        diff = y - target
        loss = diff.square().mean()
        _, *grads = self.backward(diff * (2 / diff.numel()), kept)
        self.count += 1
        for w, g, (m, v) in zip((self.wqkv, self.wo), grads, self._moments):
            ops.adamw(w, g, m, v, self.count, lr)
        self.refresh()
        return loss

    def prompt(self, cache, x, new, which=None):
        """y [T, D] of prompts x [T, D], new[i] rows of sequence which[i] (of every sequence), which enter the cache; it
        holds nothing of these sequences yet."""
        self._check(x)
        which, new = cache.chosen(which), list(new)
        if any(cache.lens[b] for b in which):
            raise ValueError("a prompt begins a sequence: its cache is empty")
        if sum(new) != x.shape[0]:
            raise ValueError(f"{sum(new)} rows of prompts where x has {x.shape[0]}")
        if not x.shape[0]:
            return torch.empty(0, self.D, device="cuda")
        cache.grow(new, which)
        at = _ints([i for n in new for i in range(n)])
        seq = _ints([b for b, n in zip(which, new) for _ in range(n)])
        offsets = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        y, kept = self.forward(x, offsets, at)
        _, k, v = self._split(kept["heads"])
        ops.kv_append(k, v, seq, at, cache.table, cache.k, cache.v)  # (keys are rotated already)
        for b, n in zip(which, new):
            cache.lens[b] = n
        return y

    def token(self, cache, x, which=None):
        """y [n, D] of one more token, x [n, D], of the sequences `which` (of every sequence, where one that the cache
        holds nothing of begins with it)."""
        self._check(x)
        which = cache.chosen(which)
        n = len(which)
        if x.shape[0] != n:
            raise ValueError(f"{x.shape[0]} rows of tokens for {n} sequences")
        if not n:
            return torch.empty(0, self.D, device="cuda")
        cache.grow([1] * n, which)
        at, seq = _ints([cache.lens[b] for b in which]), _ints(which)
        q, k, v = self._split(self._heads(x))
        turned, ctx = (torch.empty(n, self.Hq, self.dh, dtype=BF16, device="cuda") for _ in "qc")
        ops.kv_append(k, v, seq, at, cache.table, cache.k, cache.v, pos=at, freq=self.freq, q=q, q_out=turned)
        for b in which:
            cache.lens[b] += 1
        table = cache.table if which == list(range(len(cache.lens))) else cache.table[seq]
        ops.attention_paged(turned, cache.k, cache.v, table, at + 1, ctx, **self.seen)
        return self._out(ctx)


def main():
    D, Hq, Hkv, dh, T = 256, 8, 2, 64, 1024
    how = dict(window=128, sinks=4)
    layer, teacher = AttentionLayer(D, Hq, Hkv, dh, **how, seed=2), AttentionLayer(D, Hq, Hkv, dh, **how, seed=3)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn(T, D, device="cuda", generator=g).to(BF16)
    lens = [400, 0, 623, 1]
    offsets = _ints([sum(lens[:b]) for b in range(len(lens) + 1)])
    pos = _ints([i for n in lens for i in range(n)])
    target, _ = teacher.forward(x, offsets, pos)
    losses = [float(layer.train_step(x, offsets, pos, target, 3e-3)) for _ in range(60)]
    print(f"training: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {len(losses)} steps of {T} tokens")
    whole, _ = layer.forward(x, offsets, pos)
    cache = PagedCache(layer, B=2, pages=64)
    layer.prompt(cache, torch.cat([x[:390], x[400:1000]]), [390, 600])
    for i in range(10):  # serving: one token a sequence at a time
        y = layer.token(cache, torch.stack([x[390 + i], x[1000 + i]]))
        want = torch.stack([whole[390 + i], whole[1000 + i]])
        if i % 3 == 0:
            print(f"serving token {i}: {float((y - want).norm() / want.norm()):.1e} off its rows in the batch")
    ops.check_errors()


if __name__ == "__main__":
    main()
