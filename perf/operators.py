"""Cases for the operators of a mixture of experts with k experts a token and
8-bit (e4m3) products: routing, the order of (token, expert) pairs, block
quantisation, the block-scaled product, and the experts' products.

Each case is one call of one operator as a program makes it, on what that
program holds before the call. `run` computes it with the framework's kernels
where `own` is true, and with elementary torch operations in 32 bits where it
is not.
"""
import math

import torch

own = False

DEV = "cuda"
TOP = 448.0  # largest finite e4m3 value
FLOOR = 2.0 ** -100  # smallest scale of a block


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # routing of one decode step's tokens: sigmoid scores, balance bias, expert groups
        dict(name="route_decode", op="route", M=32, E=128, k=8, score="sigmoid", bias=True, dead=0, groups=8,
             topk_groups=4, renorm=True, scale=2.5, dtype="bf16", train=False),
        # routing and its gradient in a training step of 16384 tokens
        dict(name="route_train", op="route", M=16384, E=256, k=8, score="sigmoid", bias=True, dead=3, groups=8,
             topk_groups=4, renorm=True, scale=2.5, dtype="f32", train=True),
        # ordering the pairs of a decode step by expert and adding up the experts' outputs
        dict(name="order_decode", op="order", M=24, k=8, E=128, D=2048, align=1, dtype="bf16", train=False),
        # the same for a training step, with the gradients of the outputs and of the weights
        dict(name="order_train", op="order", M=8192, k=4, E=64, D=2048, align=128, dtype="bf16", train=True),
        # activations of a training step behind a GELU, in both orientations (forward and weight gradient)
        dict(name="quantize_rows", op="quantize", kind="rows", both=True, M=16384, K=2048, pad=0, act=6, dtype="bf16"),
        # a master weight after the optimizer's step, in both orientations; odd size, rows of a wider buffer
        dict(name="quantize_weight", op="quantize", kind="block", both=True, M=4000, K=1544, pad=8, act=0, dtype="f32"),
        # one token through a dense layer
        dict(name="product_decode", op="product", M=1, N=4096, K=4096, rows=False, out="bf16"),
        # a prompt batch, or a training step's forward, through a dense layer
        dict(name="product_prefill", op="product", M=8192, N=4096, K=4096, rows=False, out="bf16"),
        # a weight gradient (both operands scaled by row) of odd size
        dict(name="product_wgrad", op="product", M=2000, N=1544, K=8100, rows=True, out="f32"),
        # a decode step's tokens through the experts' first matrices
        dict(name="experts_decode", op="experts", kind="rows", M=24, k=4, E=64, N=2048, K=1024, align=1, gather=True,
             out="bf16"),
        # a prompt batch through the experts' first matrices, rows gathered by the product
        dict(name="experts_prefill", op="experts", kind="rows", M=8192, k=4, E=16, N=2048, K=2048, align=128,
             gather=True, out="bf16"),
        # the experts' weight gradients of a training step
        dict(name="experts_wgrad", op="experts", kind="wgrad", M=8192, k=2, E=8, N=1024, K=1024, align=128,
             gather=False, out="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "order", "quantize", "product", "product", "experts", "experts"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        E = groups * rng.randint(2, 256 // groups) if groups > 1 else rng.randint(4, 256)
        tg = rng.randint(max(1, groups // 2), groups)
        dead = rng.choice([0, 0, rng.randint(0, E // 4)])
        k = rng.randint(1, min(8, E))
        return dict(op=op, M=_log(rng, 1, 16384), E=E, k=k, score=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.5, dead=dead, groups=groups, topk_groups=tg, renorm=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["bf16", "f32"]), train=rng.random() < 0.5)
    if op == "order":
        E = rng.randint(2, 128)
        return dict(op=op, M=_log(rng, 1, 8192), k=rng.randint(1, min(4, E)), E=E, D=rng.randint(64, 2048),
                    align=rng.choice([1, 128]), dtype=rng.choice(["bf16", "bf16", "f32"]), train=rng.random() < 0.5)
    if op == "quantize":
        kind = rng.choice(["rows", "rows", "block", "grouped"])
        return dict(op=op, kind=kind, both=rng.random() < 0.5, M=_log(rng, 1, 8192), K=rng.randint(1, 2048),
                    pad=rng.choice([0, 8, 24]), act=rng.choice([0, 0, 5, 6]) if kind != "block" else 0,
                    dtype=rng.choice(["bf16", "f32"]))
    if op == "product":
        rows = rng.random() < 0.3
        return dict(op=op, M=_log(rng, 1, 8192), N=rng.randint(1, 512) * 8, K=rng.randint(1, 4096), rows=rows,
                    out=rng.choice(["bf16", "f32"]))
    kind = rng.choice(["rows", "rows", "wgrad"])
    E = rng.choice([4, 8, 16, 64])
    return dict(op=op, kind=kind, M=_log(rng, 1, 4096), k=rng.randint(1, 4), E=E, N=rng.randint(2, 128) * 8,
                K=rng.randint(2, 128) * 16, align=128 if kind == "wgrad" else rng.choice([1, 128]),
                gather=kind == "rows" and rng.random() < 0.6, out="f32" if kind == "wgrad" else "bf16")


def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _up(n, m):
    return -(-n // m) * m


def _capacity(M, k, E, align):
    """Rows that ordered pairs take at most: each expert that has any rounds up to `align`."""
    return _up(M * k + min(E, M * k) * (align - 1), align)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
class _Maker:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, device=DEV, generator=self.g)

    def uniform(self, *shape):
        return torch.rand(*shape, device=DEV, generator=self.g)

    def activations(self, *shape):
        """Values of a hidden state: normal, with channels of up to ten times the usual size."""
        return self.normal(*shape) * (1 + 9 * self.uniform(shape[-1]) ** 16)

    def choices(self, M, k, E):
        """k different experts a token, some experts more popular than others."""
        pull = self.normal(1, E) * 0.5
        noise = -torch.log(-torch.log(self.uniform(M, E).clamp(1e-7, 1 - 1e-7)))
        return (pull + noise).topk(min(k, E), dim=1).indices.to(torch.int32).contiguous()


def _codes_rows(x):
    """Codes and scales (one for each 128 along a row, block-major) of [R, K], the codes' rows on 16-byte boundaries."""
    R, K = x.shape
    KB = -(-K // 128)
    full = torch.zeros(R, KB * 128, device=DEV)
    full[:, :K] = x
    b = full.view(R, KB, 128)
    s = torch.clamp(b.abs().amax(2) / TOP, min=FLOOR)
    q = (b / s[:, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn).view(R, KB * 128)
    code = torch.zeros(R, _up(K, 16), device=DEV, dtype=torch.float8_e4m3fn)
    code[:, :K] = q[:, :K]
    scale = torch.ones(KB, _up(R, 4), device=DEV)
    scale[:, :R] = s.t()
    return code[:, :K], scale[:, :R]


def _codes_block(w):
    """Codes and scales (one for each 128 x 128) of [E, N, K]."""
    E, N, K = w.shape
    NB, KB = -(-N // 128), -(-K // 128)
    full = torch.zeros(E, NB * 128, KB * 128, device=DEV)
    full[:, :N, :K] = w
    b = full.view(E, NB, 128, KB, 128)
    s = torch.clamp(b.abs().amax((2, 4)) / TOP, min=FLOOR)
    q = (b / s[:, :, None, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn).view(E, NB * 128, KB * 128)
    code = torch.zeros(E, N, _up(K, 16), device=DEV, dtype=torch.float8_e4m3fn)
    code[:, :, :K] = q[:, :N, :K]
    return code[:, :, :K], s.contiguous()


def _order(idx, E, align):
    """Experts' segments of the pairs in idx [M, k]: offsets [E + 1], counts [E], rows [capacity], pos [M, k]."""
    M, k = idx.shape
    cap = _capacity(M, k, E, align)
    flat = idx.reshape(-1).long()
    key = torch.where(flat >= 0, flat, E)
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(E + 1, dtype=torch.long, device=DEV).index_add_(0, key, torch.ones_like(key))
    padded = (counts[:E] + align - 1) // align * align
    zero = torch.zeros(1, dtype=torch.long, device=DEV)
    offsets = torch.cat([zero, padded.cumsum(0)])
    first = torch.cat([zero, counts.cumsum(0)])[:E + 1]
    ek = key[order]
    at = torch.where(ek < E, offsets[ek] + torch.arange(M * k, device=DEV) - first[ek], cap)
    rows = torch.full((cap + 1,), -1, dtype=torch.int32, device=DEV)
    rows[at] = order.to(torch.int32)
    pos = torch.empty(M * k, dtype=torch.long, device=DEV)
    pos[order] = torch.where(ek < E, at, -1)
    return offsets.to(torch.int32), counts[:E].to(torch.int32), rows[:cap], pos.view(M, k).to(torch.int32)


def prepare(case, seed):
    m = _Maker(seed)
    c = dict(case)
    s = {"case": c}
    op = c["op"]
    if op == "route":
        M, E = c["M"], c["E"]
        s["logits"] = (m.normal(M, E) + 0.5 * m.normal(1, E)).to(_type(c["dtype"]))
        s["bias"] = 0.05 * m.normal(E) if c["bias"] else None
        s["active"] = None
        if c["dead"]:
            active = torch.ones(E, dtype=torch.uint8, device=DEV)
            active[torch.randperm(E, device=DEV, generator=m.g)[:c["dead"]]] = 0
            s["active"] = active
        s["idx"] = torch.empty(M, c["k"], dtype=torch.int32, device=DEV)
        s["w"] = torch.empty(M, c["k"], device=DEV)
        if c["train"]:
            s["dw"] = m.normal(M, c["k"])
            s["dlogits"] = torch.empty_like(s["logits"])
    elif op == "order":
        M, k, E, D = c["M"], c["k"], c["E"], c["D"]
        cap = _capacity(M, k, E, c["align"])
        t = _type(c["dtype"])
        s["idx"] = m.choices(M, k, E)
        s["w"] = torch.softmax(m.normal(M, k), 1)
        s["o"] = m.normal(cap, D).to(t)
        s["offsets"] = torch.empty(E + 1, dtype=torch.int32, device=DEV)
        s["counts"] = torch.empty(E, dtype=torch.int32, device=DEV)
        s["rows"] = torch.empty(cap, dtype=torch.int32, device=DEV)
        s["pos"] = torch.empty(M, k, dtype=torch.int32, device=DEV)
        s["y"] = torch.empty(M, D, dtype=t, device=DEV)
        if c["train"]:
            s["dy"] = m.normal(M, D).to(t)
            s["do"] = torch.empty(cap, D, dtype=t, device=DEV)
            s["dw"] = torch.empty(M, k, device=DEV)
    elif op == "quantize":
        M, K = c["M"], c["K"]
        wide = m.activations(M, K + c["pad"]) if c["kind"] != "block" else 0.02 * m.normal(M, K + c["pad"])
        s["x"] = wide.to(_type(c["dtype"]))[:, :K]
        R = M
        if c["kind"] == "grouped":  # two experts a token of eight, each expert's rows from a multiple of 128 on
            _, _, s["rows"], _ = _order(m.choices(M, 2, 8), 8, 128)
            R = s["rows"].numel()
        KB, RB = -(-K // 128), -(-R // 128)
        f8 = torch.float8_e4m3fn
        if c["kind"] != "grouped":
            s["q"] = torch.empty(M, _up(K, 16), dtype=f8, device=DEV)[:, :K]
            s["s"] = torch.empty(RB, KB, device=DEV) if c["kind"] == "block" else torch.empty(KB, _up(M, 4), device=DEV)[:, :M]
        if c["both"] or c["kind"] == "grouped":
            s["qt"] = torch.empty(K, _up(R, 16), dtype=f8, device=DEV)[:, :R]
            s["st"] = torch.empty(KB, RB, device=DEV) if c["kind"] == "block" else torch.empty(RB, _up(K, 4), device=DEV)[:, :K]
    elif op == "product":
        M, N, K = c["M"], c["N"], c["K"]
        s["a"], s["sa"] = _codes_rows(m.activations(M, K))
        if c["rows"]:
            s["b"], s["sb"] = _codes_rows(m.activations(N, K))
        else:
            b, sb = _codes_block(0.02 * m.normal(1, N, K))
            s["b"], s["sb"] = b[0], sb[0]
        s["c"] = torch.empty(M, N, dtype=_type(c["out"]), device=DEV)
    else:
        M, k, E, N, K = c["M"], c["k"], c["E"], c["N"], c["K"]
        s["offsets"], s["counts"], s["rows"], _ = _order(m.choices(M, k, E), E, c["align"])
        cap = s["rows"].numel()
        s["most"] = int(s["counts"].max())  # rows of the busiest expert: the plain form's padded batches have this many
        if c["kind"] == "rows":
            s["a"], s["sa"] = _codes_rows(m.activations(M if c["gather"] else cap, K))
            s["b"], s["sb"] = _codes_block(0.02 * m.normal(E, N, K))
            s["c"] = torch.zeros(cap, N, dtype=_type(c["out"]), device=DEV)
        else:
            real = (s["rows"] >= 0).float()
            s["a"], s["sa"] = _codes_rows(m.normal(N, cap) * 0.01 * real)
            s["b"], s["sb"] = _codes_rows(m.activations(cap, K).t() * real)
            s["c"] = torch.empty(E, N, K, dtype=_type(c["out"]), device=DEV)
    return s


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------
def _plain_scores(c, logits, active):
    x = logits.float()
    if c["score"] == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    if active is not None:
        x = x.masked_fill(active[None] == 0, -math.inf)
    e = torch.exp(x - x.amax(1, keepdim=True))
    return e / e.double().sum(1, keepdim=True).float()


def _plain_route(s):
    c = s["case"]
    M, E, k, G = c["M"], c["E"], c["k"], c["groups"]
    p = _plain_scores(c, s["logits"], s["active"])
    key = p if s["bias"] is None else p + s["bias"]
    if s["active"] is not None:
        key = key.masked_fill(s["active"][None] == 0, -math.inf)
    if G > 1:
        best = key.view(M, G, E // G).topk(min(2, E // G), dim=2).values
        if best.shape[2] == 2:
            group = best[:, :, 0] + torch.where(best[:, :, 1] > -math.inf, best[:, :, 1], 0)
        else:
            group = best[:, :, 0]
        kept = torch.sort(group, dim=1, descending=True, stable=True).indices[:, :c["topk_groups"]]
        keep = torch.zeros(M, G, dtype=torch.bool, device=DEV).scatter_(1, kept, True)
        key = key.masked_fill(~keep.repeat_interleave(E // G, dim=1), -math.inf)
    top = torch.sort(key, dim=1, descending=True, stable=True)
    there = top.values[:, :k] > -math.inf
    idx = top.indices[:, :k]
    chosen = torch.where(there, p.gather(1, idx), 0)
    total = chosen.sum(1, keepdim=True) + 1e-20 if c["renorm"] else 1.0
    out = {"idx": torch.where(there, idx, -1).to(torch.int32), "w": c["scale"] * chosen / total}
    if c["train"]:
        dw = torch.where(there, s["dw"], 0)
        if c["renorm"]:
            ds = c["scale"] * (dw - (dw * chosen).sum(1, keepdim=True) / total) / total
        else:
            ds = c["scale"] * dw
        ds = torch.zeros(M, E, device=DEV).scatter_add_(1, idx, torch.where(there, ds, 0))
        if c["score"] == "sigmoid":
            d = ds * p * (1 - p)
        else:
            d = p * (ds - (ds * p).sum(1, keepdim=True))
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _plain_order(s):
    c = s["case"]
    offsets, counts, rows, pos = _order(s["idx"], c["E"], c["align"])
    at = pos.long()
    there = (at >= 0)[:, :, None]
    o = s["o"][at.clamp(min=0)].float()
    y = torch.where(there, o * s["w"][:, :, None], 0).sum(1).to(s["o"].dtype)
    out = {"offsets": offsets, "counts": counts, "rows": rows, "pos": pos, "y": y}
    if c["train"]:
        dy = s["dy"].float()
        out["dw"] = torch.where(there, o * dy[:, None], 0).sum(2)
        pair = rows.long().clamp(min=0)
        do = dy[pair // c["k"]] * s["w"].reshape(-1)[pair][:, None]
        out["do"] = torch.where((rows >= 0)[:, None], do, 0).to(s["o"].dtype)
    return out


def _plain_act(x, act):
    if act == 5:
        return x / (1 + torch.exp(-x))
    if act == 6:
        return 0.5 * x * (1 + torch.erf(x / 1.41421356))
    return x


def _plain_scale(amax):
    return torch.clamp(amax / TOP, min=FLOOR)


def _plain_quantize_rows(x):
    """Codes [R, K] and block-major scales [KB, R] of x, a scale for each 128 along a row."""
    R, K = x.shape
    KB = -(-K // 128)
    b = torch.nn.functional.pad(x, (0, KB * 128 - K)).view(R, KB, 128)
    scale = _plain_scale(b.abs().amax(2))
    q = (b * (1 / scale)[:, :, None]).to(torch.float8_e4m3fn)
    return q.view(R, KB * 128)[:, :K], scale.t()


def _plain_quantize(s):
    c = s["case"]
    M, K = c["M"], c["K"]
    x = _plain_act(s["x"].float(), c["act"])
    out = {}
    if c["kind"] == "block":
        MB, KB = -(-M // 128), -(-K // 128)
        b = torch.nn.functional.pad(x, (0, KB * 128 - K, 0, MB * 128 - M)).view(MB, 128, KB, 128)
        scale = _plain_scale(b.abs().amax((1, 3)))
        q = (b * (1 / scale)[:, None, :, None]).to(torch.float8_e4m3fn).view(MB * 128, KB * 128)[:M, :K]
        out = {"q": q, "s": scale}
        if c["both"]:
            out |= {"qt": q.t(), "st": scale.t()}
        return out
    if c["kind"] == "rows":
        out["q"], out["s"] = _plain_quantize_rows(x)
    else:
        x = torch.where((s["rows"] >= 0)[:, None], x[s["rows"].long().clamp(min=0) // 2], 0)
    if c["both"] or c["kind"] == "grouped":
        out["qt"], out["st"] = _plain_quantize_rows(x.t())
    return out


def _plain_values_rows(q, scale):
    K = q.shape[-1]
    return q.float() * scale.t().repeat_interleave(128, dim=1)[:, :K]


def _plain_values_block(q, scale):
    N, K = q.shape[-2:]
    wide = scale.repeat_interleave(128, dim=-2)[..., :N, :].repeat_interleave(128, dim=-1)[..., :K]
    return q.float() * wide


def _plain_product(s):
    a = _plain_values_rows(s["a"], s["sa"])
    b = _plain_values_rows(s["b"], s["sb"]) if s["case"]["rows"] else _plain_values_block(s["b"], s["sb"])
    return (a @ b.t()).to(s["c"].dtype)


def _plain_experts(s):
    c = s["case"]
    E, N, K, most = c["E"], c["N"], c["K"], s["most"]
    cap = s["rows"].numel()
    step = torch.arange(most, device=DEV)
    inside = step[None] < s["counts"][:, None]  # [E, most]: the rows that each expert has
    at = torch.where(inside, s["offsets"][:E, None] + step[None], cap).long()
    if c["kind"] == "rows":
        a = _plain_values_rows(s["a"], s["sa"])
        src = at.clamp(max=cap - 1)
        if c["gather"]:
            src = s["rows"].long().clamp(min=0)[src] // c["k"]
        out = torch.bmm(a[src], _plain_values_block(s["b"], s["sb"]).transpose(1, 2))
        full = torch.zeros(cap + 1, N, dtype=s["c"].dtype, device=DEV)
        full[at.view(-1)] = out.view(E * most, N).to(full.dtype)
        return full[:cap]
    zero = torch.zeros(1, cap + 1, device=DEV)
    a = torch.cat([_plain_values_rows(s["a"], s["sa"]), zero[:, :1].expand(N, 1)], 1)[:, at].permute(1, 0, 2)
    b = torch.cat([_plain_values_rows(s["b"], s["sb"]), zero[:, :1].expand(K, 1)], 1)[:, at].permute(1, 2, 0)
    return torch.bmm(a, b).to(s["c"].dtype)


def _plain(s):
    op = s["case"]["op"]
    if op == "route":
        return _plain_route(s)
    if op == "order":
        return _plain_order(s)
    if op == "quantize":
        return _plain_quantize(s)
    return _plain_product(s) if op == "product" else _plain_experts(s)


# --------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------
def _framework(s):
    from neuralscript_b200 import ops

    c = s["case"]
    op = c["op"]
    if op == "route":
        how = dict(score=c["score"], active=s["active"], renorm=c["renorm"], scale=c["scale"])
        ops.moe_topk_route(s["logits"], s["idx"], s["w"], bias=s["bias"], groups=c["groups"],
                           topk_groups=c["topk_groups"], **how)
        out = {"idx": s["idx"], "w": s["w"]}
        if c["train"]:
            ops.moe_topk_route_bwd(s["dw"], s["logits"], s["idx"], s["dlogits"], **how)
            out["dlogits"] = s["dlogits"]
        return out
    if op == "order":
        ops.moe_dispatch(s["idx"], c["E"], s["offsets"], s["counts"], s["rows"], s["pos"], align=c["align"])
        ops.moe_combine(s["o"], s["pos"], s["y"], w=s["w"])
        out = {n: s[n] for n in ("offsets", "counts", "rows", "pos", "y")}
        if c["train"]:
            ops.moe_combine_bwd(s["dy"], s["o"], s["rows"], s["pos"], s["w"], s["do"], s["dw"])
            out |= {"do": s["do"], "dw": s["dw"]}
        return out
    if op == "quantize":
        if c["kind"] == "block":
            ops.fp8_quantize_block(s["x"], s["q"], s["s"], s.get("qt"), s.get("st"))
        elif c["kind"] == "rows":
            ops.fp8_quantize(s["x"], s["q"], s["s"], s.get("qt"), s.get("st"), act=c["act"])
        else:
            ops.fp8_quantize(s["x"], None, None, s["qt"], s["st"], act=c["act"], rows=s["rows"], row_div=2)
        return {n: s[n] for n in ("q", "s", "qt", "st") if n in s}
    if op == "product":
        ops.gemm_fp8(s["a"], s["sa"], s["b"], s["sb"], s["c"])
        return s["c"]
    if c["kind"] == "rows":
        ops.moe_gemm_fp8(s["a"], s["sa"], s["offsets"], s["counts"], s["b"], s["sb"], s["c"],
                         rows=s["rows"] if c["gather"] else None, row_div=c["k"])
    else:
        ops.moe_wgrad_fp8(s["a"], s["sa"], s["b"], s["sb"], s["offsets"], s["counts"], s["c"])
    return s["c"]


def run(state):
    return _framework(state) if own else _plain(state)


# --------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# --------------------------------------------------------------------------
def _e4m3(v):
    """The nearest e4m3 value, ties to the even one, of v in 64 bits (|v| up to the largest)."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 4, min=-9))  # three bits behind the leading one
    return torch.clamp(torch.round(v / step) * step, -TOP, TOP)


def _exact_quantize(blocks, dims):
    scale = (blocks.abs().amax(dims, keepdim=True) / TOP).clamp(min=FLOOR)
    return _e4m3(blocks / scale), scale


def _blocked(x, rows, cols):
    """x [R, C] in zero-filled blocks: [RB, rows, CB, cols]."""
    R, C = x.shape
    RB, CB = -(-R // rows), -(-C // cols)
    out = torch.zeros(RB * rows, CB * cols, dtype=torch.float64, device=DEV)
    out[:R, :C] = x
    return out.view(RB, rows, CB, cols)


def _exact_route(s):
    c = s["case"]
    M, E, k, G = c["M"], c["E"], c["k"], c["groups"]
    z = s["logits"].double()
    live = torch.ones(E, dtype=torch.bool, device=DEV) if s["active"] is None else s["active"] != 0
    if c["score"] == "softmax":
        p = torch.softmax(torch.where(live, z, -math.inf), 1)
    else:
        p = torch.sigmoid(z)
    key = torch.where(live, p + (s["bias"].double() if c["bias"] else 0), -math.inf)
    if G > 1:
        each = key.view(M, G, -1).sort(2, descending=True).values[:, :, :2]
        score = torch.where(each > -math.inf, each, 0).sum(2) + torch.where(each[:, :, 0] > -math.inf, 0, -math.inf)
        rank = score.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
        key = torch.where((rank < c["topk_groups"])[:, torch.arange(E, device=DEV) // (E // G)], key, -math.inf)
    rank = key.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
    on = (rank < k) & (key > -math.inf)
    total = (p * on).sum(1, keepdim=True) + 1e-20 if c["renorm"] else torch.ones(M, 1, dtype=torch.float64, device=DEV)
    at = rank.argsort(dim=1)[:, :k]
    out = {"idx": None, "w": (c["scale"] * p * on / total).gather(1, at)}
    if c["train"]:
        dw = torch.zeros(M, E, dtype=torch.float64, device=DEV).scatter_(1, at, s["dw"].double()) * on
        dp = c["scale"] * dw / total
        if c["renorm"]:
            dp = dp - on * c["scale"] * (dw * p).sum(1, keepdim=True) / total ** 2
        out["dlogits"] = dp * p * (1 - p) if c["score"] == "sigmoid" else p * dp - p * (p * dp).sum(1, keepdim=True)
    return out


def _exact_order(s):
    c = s["case"]
    _, _, rows, pos = _order(s["idx"], c["E"], c["align"])
    M, k, D = c["M"], c["k"], c["D"]
    y = torch.zeros(M, D, dtype=torch.float64, device=DEV)
    dw = torch.zeros(M, k, dtype=torch.float64, device=DEV)
    for j in range(k):
        on = (pos[:, j] >= 0).double()[:, None]
        o = s["o"][pos[:, j].long().clamp(min=0)].double() * on
        y += s["w"][:, j:j + 1].double() * o
        if c["train"]:
            dw[:, j] = (o * s["dy"].double()).sum(1)
    out = {"offsets": None, "counts": None, "rows": None, "pos": None, "y": y}
    if c["train"]:
        t, j = rows.long() // k, rows.long() % k
        do = s["dy"].double()[t] * s["w"].double()[t, j][:, None]
        out |= {"do": torch.where(rows[:, None] < 0, 0, do), "dw": dw}
    return out


def _exact_activation(x, act):
    x = x.double()
    return torch.nn.functional.gelu(x) if act == 6 else torch.nn.functional.silu(x) if act == 5 else x


def _exact_quantized(s):
    c = s["case"]
    x = _exact_activation(s["x"], c["act"])
    M, K = x.shape
    if c["kind"] == "block":
        q, scale = _exact_quantize(_blocked(x, 128, 128), (1, 3))
        q, scale = q.reshape(q.shape[0] * 128, -1)[:M, :K], scale[:, 0, :, 0]
        return {"q": q, "s": scale, **({"qt": q.t(), "st": scale.t()} if c["both"] else {})}
    out = {}
    if c["kind"] == "rows":
        q, scale = _exact_quantize(_blocked(x, 1, 128), (3,))
        out = {"q": q.reshape(M, -1)[:, :K], "s": scale[:, 0, :, 0].t()}
    else:
        r = s["rows"].long()
        x = torch.where((r < 0)[:, None], 0, x[r.clamp(min=0) // 2])
    if c["both"] or c["kind"] == "grouped":
        q, scale = _exact_quantize(_blocked(x, 128, 1), (1,))
        out |= {"qt": q.reshape(-1, K)[:x.shape[0]].t(), "st": scale[:, 0, :, 0]}
    return out


def _exact_values(q, scale, block):
    R, K = q.shape
    r, k = torch.arange(R, device=DEV), torch.arange(K, device=DEV)
    at = scale[(r // 128)[:, None], (k // 128)[None]] if block else scale[(k // 128)[None], r[:, None]]
    return q.double() * at.double()


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "route":
        return _exact_route(s)
    if c["op"] == "order":
        return _exact_order(s)
    if c["op"] == "quantize":
        return _exact_quantized(s)
    if c["op"] == "product":
        return _exact_values(s["a"], s["sa"], False) @ _exact_values(s["b"], s["sb"], not c["rows"]).t()
    E, k = c["E"], c["k"]
    offsets, counts = s["offsets"].tolist(), s["counts"].tolist()
    a = _exact_values(s["a"], s["sa"], False)
    if c["kind"] == "wgrad":
        b = _exact_values(s["b"], s["sb"], False)
        return torch.stack([a[:, o:o + n] @ b[:, o:o + n].t() for o, n in zip(offsets, counts)])
    out = torch.zeros(s["rows"].numel(), c["N"], dtype=torch.float64, device=DEV)
    for e in range(E):
        o, n = offsets[e], counts[e]
        rows = s["rows"][o:o + n].long() // k if c["gather"] else torch.arange(o, o + n, device=DEV)
        out[o:o + n] = a[rows] @ _exact_values(s["b"][e], s["sb"][e], True).t()
    return out


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    c = case
    op = c["op"]
    if op == "route":
        M, E, k = c["M"], c["E"], c["k"]
        item = 2 if c["dtype"] == "bf16" else 4
        moved = M * E * item + M * k * 8 + (4 * E if c["bias"] else 0) + (E if c["dead"] else 0)
        flops = 6 * M * E
        if c["train"]:  # dw and the chosen experts in, the logits once more (their scores are not kept), the gradient out
            moved += M * k * 8 + 2 * M * E * item
            flops += 6 * M * E
        return {"bytes": moved, "flops": flops}
    if op == "order":
        M, k, E, D = c["M"], c["k"], c["E"], c["D"]
        item = 2 if c["dtype"] == "bf16" else 4
        cap = _capacity(M, k, E, c["align"])
        moved = M * k * 4 + (2 * E + 1) * 4 + cap * 4 + M * k * 4  # choices in, segments, rows and places out
        moved += M * k * D * item + M * k * 4 + M * D * item
        flops = 2 * M * k * D
        if c["train"]:
            moved += M * D * item + M * k * D * item + cap * D * item + M * k * 4
            flops += 3 * M * k * D
        return {"bytes": moved, "flops": flops}
    if op == "quantize":
        M, K = c["M"], c["K"]
        item = 2 if c["dtype"] == "bf16" else 4
        R = _capacity(M, 2, 8, 128) if c["kind"] == "grouped" else M
        per = 4 / (128 * 128) if c["kind"] == "block" else 4 / 128
        out = (R * K if c["kind"] == "grouped" else M * K * (2 if c["both"] else 1)) * (1 + per)
        return {"bytes": M * K * item + out + (4 * R if c["kind"] == "grouped" else 0), "flops": 4 * M * K}
    if op == "product":
        M, N, K = c["M"], c["N"], c["K"]
        KB = -(-K // 128)
        item = 2 if c["out"] == "bf16" else 4
        scales = 4 * KB * (M + (N if c["rows"] else -(-N // 128)))
        return {"bytes": M * K + N * K + scales + M * N * item, "flops": 2 * M * N * K}
    M, k, E, N, K = c["M"], c["k"], c["E"], c["N"], c["K"]
    item = 2 if c["out"] == "bf16" else 4
    if c["kind"] == "wgrad":
        return {"bytes": M * k * (N + K) * (1 + 4 / 128) + E * N * K * item, "flops": 2 * M * k * N * K}
    used = E * (1 - (1 - k / E) ** M)  # experts that some token chooses, on average
    rows = M if c["gather"] else M * k
    return {"bytes": used * N * K + rows * K * (1 + 4 / 128) + M * k * N * item, "flops": 2 * M * k * N * K}
