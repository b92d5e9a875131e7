"""A mixture-of-experts layer with k experts a token, its products in 8-bit
floating point: the operators of ``ops`` put together as a program uses them.

    y[t] = sum over the k experts e of token t of  w[t,e] W2[e] gelu(W1[e] x[t])

Training quantises every operand in both orientations: forward and input
gradient take the weights' 128 x 128 blocks (one quantisation serves both),
the weight gradients a scale for each 128 tokens. Serving orders the pairs
without padding and needs no second orientation. ``python -m
neuralscript_b200.moe_topk`` trains a small layer and serves it.

torch holds the buffers; every product, routing and quantisation is a kernel
of this package.
"""
from __future__ import annotations

import torch

from . import ops

F8 = torch.float8_e4m3fn
GELU = 6


def _codes(rows, cols):
    """Codes with rows on 16-byte boundaries."""
    return torch.empty(rows, ops.fp8_ld(cols), dtype=F8, device="cuda")[:, :cols]


def _floats(*shape):
    return torch.empty(*shape, device="cuda")


class MoETopk:
    """W1 [E, H, D] and W2 [E, D, H] of the experts and the gate [E, D], in fp32; D and H multiples of 128."""

    def __init__(self, D, H, E, k, score="sigmoid", groups=1, topk_groups=1, seed=0):
        if D % 128 or H % 128:
            raise ValueError("D and H are multiples of 128")
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.D, self.H, self.E, self.k = D, H, E, k
        self.how = dict(score=score, renorm=True, scale=1.0)
        self.choice = dict(bias=torch.zeros(E, device="cuda"), groups=groups, topk_groups=topk_groups)
        draw = lambda *s: torch.randn(*s, device="cuda", generator=g) / s[-1] ** 0.5  # noqa: E731
        self.gate, self.w1, self.w2 = draw(E, D), draw(E, H, D), draw(E, D, H)
        self.step = 0
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")  # of all its products
        self._moments = [(torch.zeros_like(w), torch.zeros_like(w)) for w in (self.gate, self.w1, self.w2)]
        self.refresh()

    def _blocks(self, w):
        """Codes and scales of the experts' matrices w [E, N, K] as products take them, and of their transposes: one
        pass over all experts, whose transposes then lie side by side in rows of E * N codes."""
        E, N, K = w.shape
        q, s = _codes(E * N, K), _floats(E * N // 128, K // 128)
        qt, st = _codes(K, E * N), _floats(K // 128, E * N // 128)
        ops.fp8_quantize_block(w.view(E * N, K), q, s, qt, st)
        return ((q.view(E, N, K), s.view(E, N // 128, K // 128)),
                (qt.view(K, E, N).transpose(0, 1), st.view(K // 128, E, N // 128).transpose(0, 1)))

    def refresh(self):
        """Quantises the weights (after they change)."""
        self.gate16 = self.gate.to(torch.bfloat16)
        self.q1, self.q1t = self._blocks(self.w1)
        self.q2, self.q2t = self._blocks(self.w2)

    def check(self):
        """Waits for the current stream and raises RuntimeError where a product gave up a bounded wait since the last
        check. train_step calls it; who serves calls it where the results are read."""
        code = int(self.err)
        if code:
            self.err.zero_()
            raise RuntimeError(f"device error {code} in a product of the layer")

    def _product(self, a, sa, order, b, N, rows=None):
        out = torch.zeros(order["rows"].numel(), N, device="cuda")
        ops.moe_gemm_fp8(a, sa, order["offsets"], order["counts"], *b, out, rows=rows, row_div=self.k,
                         err=self.err)
        return out

    def forward(self, x, align=1):
        """y [M, D] of x [M, D] (bf16, contiguous rows), and what the backward pass needs."""
        D, E, k = self.D, self.E, self.k
        if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] != D or x.stride(1) != 1 or x.device != self.gate.device:
            raise ValueError(f"x: {x.dtype} {tuple(x.shape)} with strides {x.stride()} on {x.device} where rows of {D} "
                             f"bfloat16 on {self.gate.device} are wanted")
        M = x.shape[0]
        i32 = dict(dtype=torch.int32, device="cuda")
        logits = _floats(M, E)
        ops.gemm(x, self.gate16, M, E, D, x.stride(0), 0, D, 0, c32=logits, err=self.err)
        idx, w = torch.empty(M, k, **i32), _floats(M, k)
        ops.moe_topk_route(logits, idx, w, **self.choice, **self.how)
        order = dict(offsets=torch.empty(E + 1, **i32), counts=torch.empty(E, **i32),
                     rows=torch.empty(ops.moe_dispatch_rows(M, k, E, align), **i32), pos=torch.empty(M, k, **i32))
        ops.moe_dispatch(idx, E, **order, align=align)
        R = order["rows"].numel()
        xq, xs = _codes(M, D), _floats(D // 128, M)
        ops.fp8_quantize(x, xq, xs)
        z = self._product(xq, xs, order, self.q1, self.H, rows=order["rows"])
        hq, hs = _codes(R, self.H), _floats(self.H // 128, R)
        ops.fp8_quantize(z, hq, hs, act=GELU)
        o = self._product(hq, hs, order, self.q2, D)
        y = _floats(M, D)
        ops.moe_combine(o, order["pos"], y, w=w)
        return y, dict(x=x, logits=logits, idx=idx, w=w, order=order, z=z, o=o, align=align)

    def backward(self, dy, kept):
        """Gradients (dx [M, D], dgate, dw1, dw2) of the loss whose gradient in y is dy [M, D] (fp32); the forward
        pass ran with align=128 (the weight gradients sum whole blocks of 128 rows: without padding a block holds
        rows of two experts)."""
        if kept["align"] % 128:
            raise ValueError(f"backward after a forward pass with align={kept['align']}, which is no multiple of 128")
        x, order, k, E, D, H = kept["x"], kept["order"], self.k, self.E, self.D, self.H
        rows, M = order["rows"], x.shape[0]
        R = rows.numel()

        def both(v, row_div, act=0, by_rows=True):
            """Codes of v in the order of the pairs: by rows, and transposed with zeros in the padding."""
            C = v.shape[1]
            q, s = (_codes(R, C), _floats(C // 128, R)) if by_rows else (None, None)
            qt, st = _codes(C, R), _floats(R // 128, C)
            ops.fp8_quantize(v, q, s, qt, st, act=act, rows=rows, row_div=row_div)
            return (q, s), (qt, st)

        do, dw = _floats(R, D), _floats(M, k)
        ops.moe_combine_bwd(dy, kept["o"], rows, order["pos"], kept["w"], do, dw)
        dlogits = _floats(M, E)
        ops.moe_topk_route_bwd(dw, kept["logits"], kept["idx"], dlogits, **self.how)
        (dq, ds), dt = both(do, 0)
        _, ht = both(kept["z"], 0, act=GELU, by_rows=False)
        dw2 = _floats(E, D, H)
        ops.moe_wgrad_fp8(*dt, *ht, order["offsets"], order["counts"], dw2, err=self.err)
        dz = _floats(R, H)
        ops.act_bwd(self._product(dq, ds, order, self.q2t, H), kept["z"], GELU, dz)
        (zq, zs), zt = both(dz, 0)
        _, xt = both(x, k, by_rows=False)
        dw1 = _floats(E, H, D)
        ops.moe_wgrad_fp8(*zt, *xt, order["offsets"], order["counts"], dw1, err=self.err)
        dx = _floats(M, D)
        ops.moe_combine(self._product(zq, zs, order, self.q1t, D), order["pos"], dx)
        x32 = x.float()
        dgate = _floats(E, D)
        ops.gemm(dlogits, x32, E, D, M, E, 1, D, 1, c32=dgate, err=self.err)
        total = _floats(M, D)
        ops.gemm(dlogits, self.gate, M, D, E, E, 0, D, 1, add=dx, c32=total, err=self.err)
        return total, dgate, dw1, dw2

    def update(self, grads, lr):
        """One AdamW step of the gate and the experts."""
        self.step += 1
        for w, g, (m, v) in zip((self.gate, self.w1, self.w2), grads, self._moments):
            ops.adamw(w, g, m, v, self.step, lr)
        self.refresh()

    def train_step(self, x, target, lr):
        """Mean squared error before the step. A step whose products failed changes no weight."""
        y, kept = self.forward(x, align=128)
        diff = y - target
        loss = diff.square().mean()
        _, *grads = self.backward(diff * (2 / diff.numel()), kept)
        self.check()
        self.update(grads, lr)
        return loss


def main():
    torch.manual_seed(1)
    D, H, E, k, M = 256, 512, 16, 4, 2048
    layer, teacher = MoETopk(D, H, E, k, groups=4, topk_groups=2, seed=2), MoETopk(D, H, E, k, seed=3)
    x = torch.randn(M, D, device="cuda", dtype=torch.bfloat16)
    target, _ = teacher.forward(x)
    losses = [float(layer.train_step(x, target, 3e-3)) for _ in range(60)]
    print(f"training: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {len(losses)} steps of {M} tokens")
    whole, _ = layer.forward(x, align=128)
    for t in (0, 7, M - 1):  # serving: one token at a time
        y, _ = layer.forward(x[t:t + 1])
        off = float((y - whole[t]).norm() / whole[t].norm())
        print(f"serving token {t}: {off:.1e} off its row in the batch")
    layer.check()


if __name__ == "__main__":
    main()
