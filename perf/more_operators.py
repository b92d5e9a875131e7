"""Cases for the operators of attention that answers token by token: rotary
positions, appending to a paged cache of keys and values, attention of one new
token over that cache, and attention with a sliding window and a few first
tokens that stay visible, for prompts and training.

Each case is one call of one operator (a training step's: forward and
backward) as a program makes it, on what that program holds before the call.
`run` computes it with the framework's kernels where `own` is true, and with
elementary torch operations in 32 bits where it is not.
"""
import math
import random

import torch

own = False

DEV = "cuda"


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
# mix: seed of the sequences' lengths. Heads are (Hq query heads, Hkv key heads of dh columns).
def listed():
    return [
        # queries and keys of a training step, heads beside the values' in one buffer; rotation and its gradient
        dict(name="rope_train", op="rope", T=16384, H=20, beside=4, dh=128, pairs=64, axes=1, interleaved=False,
             reach=8192, dtype="bf16", train=True),
        # patches of a video (time, height, width), odd head size, in fp32
        dict(name="rope_video", op="rope", T=9001, H=12, beside=0, dh=80, pairs=40, axes=3, interleaved=True, reach=600,
             dtype="f32", train=True),
        # one decode step's tokens: keys and values to the cache, queries rotated beside them
        dict(name="append_decode", op="append", B=32, new=1, longest=2000, Hq=16, Hkv=2, dh=128, page=32, pairs=64, axes=1,
             interleaved=False, heads_first=False, queries=True, pad=0, dtype="bf16", mix=1),
        # prompts of five sequences behind what the cache holds of them, padded to a fixed number of rows
        dict(name="append_prompt", op="append", B=5, new=1600, longest=30000, Hq=8, Hkv=8, dh=64, page=16, pairs=32, axes=1,
             interleaved=False, heads_first=True, queries=False, pad=77, dtype="bf16", mix=2),
        # one short dialogue, the heads of this repository's transformer
        dict(name="paged_single", op="paged", B=1, longest=900, Hq=8, Hkv=8, dh=64, page=16, heads_first=False, window=0,
             sinks=0, empty=False, dtype="bf16", mix=3),
        # a batch of sequences of very different lengths, one of them without a token
        dict(name="paged_batch", op="paged", B=64, longest=4096, Hq=24, Hkv=4, dh=128, page=32, heads_first=False, window=0,
             sinks=0, empty=True, dtype="bf16", mix=4),
        # two long documents
        dict(name="paged_long", op="paged", B=2, longest=120000, Hq=16, Hkv=2, dh=128, page=48, heads_first=True, window=0,
             sinks=0, empty=False, dtype="bf16", mix=5),
        # a large batch behind a window, in fp32
        dict(name="paged_window", op="paged", B=96, longest=9000, Hq=8, Hkv=8, dh=64, page=64, heads_first=False, window=1024,
             sinks=4, empty=False, dtype="f32", mix=6),
        # a training step over packed documents, rows behind the last one unused
        dict(name="window_train", op="window", T=8192, B=3, spare=100, Hq=16, Hkv=4, dh=128, window=1024, sinks=4, dtype="bf16",
             train=True, mix=7),
        # a small training step in fp32, some of its sequences very short
        dict(name="window_small", op="window", T=700, B=6, spare=0, Hq=8, Hkv=8, dh=64, window=100, sinks=2, dtype="f32",
             train=True, mix=8),
        # a long prompt, every token before it visible
        dict(name="window_prompt", op="window", T=8192, B=1, spare=0, Hq=16, Hkv=2, dh=128, window=0, sinks=0, dtype="bf16",
             train=False, mix=9),
        # a training step over one long document of few heads
        dict(name="window_long", op="window", T=20000, B=1, spare=0, Hq=4, Hkv=1, dh=64, window=4000, sinks=16, dtype="bf16",
             train=True, mix=10),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most=16):
    Hkv = rng.choice([1, 2, 4, 8])
    return Hkv * rng.randint(1, max(1, min(8, most // Hkv))), Hkv


def draw(rng):
    op = rng.choice(["rope", "append", "paged", "paged", "window", "window"])
    dh = rng.choice([32, 64, 64, 80, 96, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    mix = rng.randrange(1 << 30)
    turn = dict(pairs=rng.choice([dh // 2, dh // 2, dh // 4]), axes=rng.choice([1, 1, 2, 3]), interleaved=rng.random() < 0.4)
    if op == "rope":
        return dict(op=op, T=_log(rng, 1, 6000), H=rng.randint(1, 24), beside=rng.choice([0, 0, 4]), dh=dh, **turn,
                    reach=_log(rng, 100, 1000000), dtype=dtype, train=rng.random() < 0.5)
    Hq, Hkv = _heads(rng, 32 if op == "paged" else 16)
    cache = dict(Hq=Hq, Hkv=Hkv, dh=dh, page=rng.choice([1, 16, 24, 32, 64, 128]), heads_first=rng.random() < 0.5)
    if op == "append":
        B = _log(rng, 1, 64)
        return dict(op=op, B=B, new=rng.choice([1, 1, _log(rng, 2, 6000 // B)]), longest=_log(rng, 100, 20000), **cache, **turn,
                    queries=rng.random() < 0.5, pad=rng.choice([0, 0, rng.randint(1, 50)]), dtype=dtype, mix=mix)
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 1, 4096), rng.choice([0, 1, 4, 64]))])
    if op == "paged":
        B = _log(rng, 1, 96)
        value = 2 if dtype == "bf16" else 4
        longest = _log(rng, 1, min(60000, int(160e6 / (value * dh * Hkv * max(1.0, 0.6 * B)))))
        return dict(op=op, B=B, longest=longest, **cache, window=window, sinks=sinks, empty=rng.random() < 0.3, dtype=dtype, mix=mix)
    train = rng.random() < 0.6
    most = math.isqrt(int(4e11 / ((14 if train else 4) * Hq * dh)))
    T = _log(rng, 1, 2000 if dtype == "f32" else min(most, 12000))
    return dict(op=op, T=T, B=rng.randint(1, min(6, T)), spare=rng.choice([0, 0, rng.randint(1, 200)]), Hq=Hq, Hkv=Hkv, dh=dh,
                window=window, sinks=sinks, dtype=dtype, train=train, mix=mix)


def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _lengths(c):
    """The sequences' lengths, from the case alone: keys in the cache (append: before the new ones), or packed rows."""
    r = random.Random(c["mix"])
    if c["op"] == "window":
        cuts = sorted(r.randint(0, c["T"]) for _ in range(c["B"] - 1))
        return [b - a for a, b in zip([0] + cuts, cuts + [c["T"]])]
    some = [max(1, int(c["longest"] * r.random() ** 1.5)) for _ in range(c["B"])]
    some[r.randrange(c["B"])] = c["longest"]
    if c.get("empty"):
        some[r.randrange(c["B"])] = 0
    return some


def _sections(c):
    """Pairs of each axis: the first axes get what does not divide."""
    n, A = c["pairs"], c["axes"]
    return tuple(n // A + (a < n % A) for a in range(A))


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
class _Maker:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, device=DEV, generator=self.g).to(dtype)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, device=DEV, generator=self.g, dtype=torch.int32)

    def order(self, n):
        return torch.randperm(n, device=DEV, generator=self.g)


def _freq(n):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float().to(DEV)


def _cache(m, c, lens, s):
    """Pages in any order, a table of them, and what they hold; `most`: keys that the table has room for."""
    page, Hkv, dh = c["page"], c["Hkv"], c["dh"]
    wide = max(1, -(-max(lens) // page))
    pages = sum(-(-n // page) for n in lens) + 3
    order = m.order(pages).to(torch.int32)
    table = torch.zeros(len(lens), wide, dtype=torch.int32)
    order, at = order.cpu(), 0
    for b, n in enumerate(lens):
        k = -(-n // page)
        table[b, :k] = order[at:at + k]
        at += k
    s["table"] = table.to(DEV)
    for name in ("k_cache", "v_cache"):
        if c["heads_first"]:
            s[name] = m.normal(pages, Hkv, page, dh, dtype=_type(c["dtype"])).transpose(1, 2)
        else:
            s[name] = m.normal(pages, page, Hkv, dh, dtype=_type(c["dtype"]))


def prepare(case, seed):
    m = _Maker(seed)
    c = dict(case)
    s = {"case": c}
    t = _type(c["dtype"])
    if c["op"] == "rope":
        T, H, dh = c["T"], c["H"], c["dh"]
        s["x"] = m.normal(T, H + c["beside"], dh, dtype=t)[:, :H]
        s["pos"] = m.ints(0, c["reach"], c["axes"], T)
        s["freq"] = _freq(c["pairs"])
        s["y"] = torch.empty(T, H, dh, dtype=t, device=DEV)
        if c["train"]:
            s["dy"] = m.normal(T, H, dh, dtype=t)
            s["dx"] = torch.empty(T, H, dh, dtype=t, device=DEV)
    elif c["op"] == "append":
        B, new, Hq, Hkv, dh = c["B"], c["new"], c["Hq"], c["Hkv"], c["dh"]
        lens = _lengths(c)
        _cache(m, c, [n + new for n in lens], s)
        T = B * new + c["pad"]
        heads = m.normal(T, Hq + 2 * Hkv, dh, dtype=t)  # one product gives all three
        s["q"], s["k"], s["v"] = heads[:, :Hq], heads[:, Hq:Hq + Hkv], heads[:, Hq + Hkv:]
        seq = torch.full((T,), -1, dtype=torch.int32, device=DEV)
        at = torch.zeros(T, dtype=torch.int32, device=DEV)
        seq[:B * new] = torch.arange(B, device=DEV, dtype=torch.int32).repeat_interleave(new)
        at[:B * new] = (torch.tensor(lens, device=DEV, dtype=torch.int32)[:, None]
                        + torch.arange(new, device=DEV, dtype=torch.int32)[None]).reshape(-1)
        s["seq"], s["at"] = seq, at
        s["pos"] = at[None] if c["axes"] == 1 else torch.cat([at[None], m.ints(0, 500, c["axes"] - 1, T)])
        s["freq"] = _freq(c["pairs"])
        s["q_out"] = torch.zeros(T, Hq, dh, dtype=t, device=DEV) if c["queries"] else None
    elif c["op"] == "paged":
        lens = _lengths(c)
        _cache(m, c, lens, s)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["q"] = 1.5 * m.normal(c["B"], c["Hq"], c["dh"], dtype=t)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(c["B"], c["Hq"], device=DEV)
    else:
        T, Hq, Hkv, dh = c["T"], c["Hq"], c["Hkv"], c["dh"]
        lens = _lengths(c)
        s["most"] = max(lens)
        s["offsets"] = torch.tensor([sum(lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
        rows = T + c["spare"]
        heads = m.normal(rows, Hq + 2 * Hkv, dh, dtype=t)
        s["q"], s["k"], s["v"] = heads[:, :Hq], heads[:, Hq:Hq + Hkv], heads[:, Hq + Hkv:]
        s["out"] = torch.zeros(rows, Hq, dh, dtype=t, device=DEV)
        s["lse"] = torch.zeros(Hq, rows, device=DEV)
        if c["train"]:
            s["dout"] = m.normal(rows, Hq, dh, dtype=t)
            grads = torch.zeros_like(heads)
            s["dq"], s["dk"], s["dv"] = grads[:, :Hq], grads[:, Hq:Hq + Hkv], grads[:, Hq + Hkv:]
    return s


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------
def _plain_angles(s):
    """cos and sin [T, 1, pairs] of every token's angles, computed in 64 bits."""
    c = s["case"]
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=DEV), torch.tensor(_sections(c), device=DEV),
                                   output_size=c["pairs"])
    a = s["pos"][axis].double() * s["freq"].double()[:, None]
    return torch.cos(a).float().t()[:, None], torch.sin(a).float().t()[:, None]


def _plain_turn(x, cos, sin, interleaved):
    n = cos.shape[-1]
    x = x.float()
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_rope(s):
    c = s["case"]
    cos, sin = _plain_angles(s)
    out = {"y": _plain_turn(s["x"], cos, sin, c["interleaved"]).to(s["x"].dtype)}
    if c["train"]:
        out["dx"] = _plain_turn(s["dy"], cos, -sin, c["interleaved"]).to(s["x"].dtype)
    return out


def _plain_append(s):
    c = s["case"]
    n = c["B"] * c["new"]  # the rows behind are padding
    cos, sin = _plain_angles(s)
    t = s["k"].dtype
    at = s["at"][:n].long()
    page = s["table"][s["seq"][:n].long(), at // c["page"]].long()
    s["k_cache"][page, at % c["page"]] = _plain_turn(s["k"][:n], cos[:n], sin[:n], c["interleaved"]).to(t)
    s["v_cache"][page, at % c["page"]] = s["v"][:n]
    out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if c["queries"]:
        s["q_out"][:n] = _plain_turn(s["q"][:n], cos[:n], sin[:n], c["interleaved"]).to(t)
        out["q_out"] = s["q_out"]
    return out


def _plain_visible(c, i, j):
    """Whether the query at i sees the key at j."""
    near = j <= i
    if c["window"]:
        near = near & ((i - j < c["window"]) | (j < c["sinks"]))
    return near


def _plain_softmax(scores, seen):
    """Weights and log-sum-exp of the scores that are seen; a row without any: zeros and -inf."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top > -math.inf, top, 0))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1), (top + torch.log(total)).squeeze(-1)


def _plain_paged(s):
    c = s["case"]
    B, Hq, Hkv, dh = c["B"], c["Hq"], c["Hkv"], c["dh"]
    table = s["table"].long()
    k = s["k_cache"][table].reshape(B, -1, Hkv, dh).float()
    v = s["v_cache"][table].reshape(B, -1, Hkv, dh).float()
    j = torch.arange(k.shape[1], device=DEV)[None]
    seen = _plain_visible(c, s["lens"][:, None] - 1, j)[:, None, None]
    v = torch.where((j < s["lens"][:, None])[:, :, None, None], v, 0)
    q = s["q"].view(B, Hkv, Hq // Hkv, dh).float()
    w, lse = _plain_softmax(torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(dh), seen)
    out = torch.matmul(w, v.transpose(1, 2))
    return {"out": out.view(B, Hq, dh).to(s["q"].dtype), "lse": lse.view(B, Hq)}


def _plain_window(s):
    c = s["case"]
    B, L, Hq, Hkv, dh = c["B"], s["most"], c["Hq"], c["Hkv"], c["dh"]
    G = Hq // Hkv
    first, end = s["offsets"][:-1, None].long(), s["offsets"][1:, None].long()
    l = torch.arange(L, device=DEV)
    row = first + l[None]
    real = row < end
    row = torch.where(real, row, 0)
    there = real[:, :, None, None]

    def spread(x, H):  # [rows, H, dh] -> [B, Hkv, H / Hkv, L, dh], zeros behind a sequence's end
        return torch.where(there, x[row].float(), 0).view(B, L, Hkv, H // Hkv, dh).permute(0, 2, 3, 1, 4)

    q, k, v = spread(s["q"], Hq), spread(s["k"], Hkv), spread(s["v"], Hkv)
    scale = 1 / math.sqrt(dh)
    seen = _plain_visible(c, l[:, None], l[None])
    w, lse = _plain_softmax(torch.matmul(q, k.transpose(-1, -2)) * scale, seen)
    o = torch.matmul(w, v)

    def pack(x, into):  # [B, Hkv, G, L, dh] -> rows of the packed buffer
        into[row[real]] = x.permute(0, 3, 1, 2, 4).reshape(B, L, -1, dh)[real].to(into.dtype)
        return into

    out = {"out": pack(o, s["out"])}
    s["lse"].t()[row[real]] = lse.permute(0, 3, 1, 2).reshape(B, L, Hq)[real]
    out["lse"] = s["lse"]
    if c["train"]:
        do = spread(s["dout"], Hq)
        dv = torch.matmul(w.transpose(-1, -2), do).sum(2, keepdim=True)
        dw = torch.matmul(do, v.transpose(-1, -2))
        ds = w * (dw - (do * o).sum(-1, keepdim=True))
        dq = torch.matmul(ds, k) * scale
        dk = torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True) * scale
        out |= {"dq": pack(dq, s["dq"]), "dk": pack(dk, s["dk"]), "dv": pack(dv, s["dv"])}
    return out


def _plain(s):
    op = s["case"]["op"]
    if op == "rope":
        return _plain_rope(s)
    if op == "append":
        return _plain_append(s)
    return _plain_paged(s) if op == "paged" else _plain_window(s)


# --------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------
def _framework(s):
    from neuralscript_b200 import ops

    c = s["case"]
    if c["op"] in ("rope", "append"):
        turn = dict(sections=_sections(c), interleaved=c["interleaved"])
    if c["op"] == "rope":
        ops.rope(s["x"], s["pos"], s["freq"], s["y"], **turn)
        out = {"y": s["y"]}
        if c["train"]:
            ops.rope_bwd(s["dy"], s["pos"], s["freq"], s["dx"], **turn)
            out["dx"] = s["dx"]
        return out
    if c["op"] == "append":
        ops.kv_append(s["k"], s["v"], s["seq"], s["at"], s["table"], s["k_cache"], s["v_cache"], pos=s["pos"], freq=s["freq"],
                      q=s["q"] if c["queries"] else None, q_out=s["q_out"], **turn)
        out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return out | {"q_out": s["q_out"]} if c["queries"] else out
    seen = dict(window=c["window"], sinks=c["sinks"])
    if c["op"] == "paged":
        ops.attention_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["out"], lse=s["lse"], **seen)
        return {"out": s["out"], "lse": s["lse"]}
    ops.attention_window(s["q"], s["k"], s["v"], s["out"], lse=s["lse"], offsets=s["offsets"], **seen)
    out = {"out": s["out"], "lse": s["lse"]}
    if c["train"]:
        ops.attention_window_bwd(s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], s["dq"], s["dk"], s["dv"],
                                 offsets=s["offsets"], **seen)
        out |= {"dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}
    return out


def run(state):
    return _framework(state) if own else _plain(state)


# --------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# --------------------------------------------------------------------------
def _exact_turn(s, x, sign=1):
    """The rotation as a product with complex numbers of modulus 1."""
    c = s["case"]
    n = c["pairs"]
    axis = [a for a, k in enumerate(_sections(c)) for _ in range(k)]
    angle = s["pos"].double()[axis].t() * s["freq"].double()
    unit = torch.polar(torch.ones_like(angle), sign * angle)[:, None]
    x = x.double().clone()
    if c["interleaved"]:
        z = torch.view_as_complex(x[..., :2 * n].unflatten(-1, (n, 2)).contiguous()) * unit
        x[..., :2 * n] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()) * unit
        x[..., :n], x[..., n:2 * n] = z.real, z.imag
    return x


def _exact_append(s):
    c = s["case"]
    turned = _exact_turn(s, s["k"])
    k, v = s["k_cache"].double(), s["v_cache"].double()
    table = s["table"].tolist()
    lens = _lengths(c)
    for b in range(c["B"]):
        at = torch.arange(lens[b], lens[b] + c["new"], device=DEV)
        page = torch.tensor(table[b], device=DEV)[torch.div(at, c["page"], rounding_mode="floor")]
        k[page, at % c["page"]] = turned[b * c["new"]:(b + 1) * c["new"]]
        v[page, at % c["page"]] = s["v"][b * c["new"]:(b + 1) * c["new"]].double()
    out = {"k_cache": k, "v_cache": v}
    if c["queries"]:
        q = _exact_turn(s, s["q"])
        q[c["B"] * c["new"]:] = 0
        out["q_out"] = q
    return out


def _exact_mask(c, queries, keys):
    """[queries, keys]: 0 where the key is visible, -inf where not; both at their positions in the sequence."""
    back = queries[:, None] - keys[None, :]
    hidden = back < 0
    if c["window"] > 0:
        hidden |= (back >= c["window"]) & (keys[None, :] >= c["sinks"])
    return torch.zeros(back.shape, dtype=torch.float64, device=DEV).masked_fill_(hidden, -math.inf)


def _exact_paged(s):
    c = s["case"]
    out = torch.zeros(c["B"], c["Hq"], c["dh"], dtype=torch.float64, device=DEV)
    lse = torch.full((c["B"], c["Hq"]), -math.inf, dtype=torch.float64, device=DEV)
    G = c["Hq"] // c["Hkv"]
    for b, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        j = torch.arange(n, device=DEV)
        page = s["table"][b].long()[j // c["page"]]
        k = s["k_cache"][page, j % c["page"]].double().repeat_interleave(G, 1)
        v = s["v_cache"][page, j % c["page"]].double().repeat_interleave(G, 1)
        z = torch.einsum("hd,jhd->hj", s["q"][b].double(), k) / c["dh"] ** 0.5 + _exact_mask(c, j[-1:], j)
        lse[b] = torch.logsumexp(z, 1)
        out[b] = torch.einsum("hj,jhd->hd", torch.softmax(z, 1), v)
    return {"out": out, "lse": lse}


def _exact_window(s):
    c = s["case"]
    rows, G = c["T"] + c["spare"], c["Hq"] // c["Hkv"]
    zeros = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device=DEV)  # noqa: E731
    out, lse = zeros(rows, c["Hq"], c["dh"]), zeros(c["Hq"], rows)
    dq, dk, dv = zeros(rows, c["Hq"], c["dh"]), zeros(rows, c["Hkv"], c["dh"]), zeros(rows, c["Hkv"], c["dh"])
    at = 0
    for n in _lengths(c):
        mine = slice(at, at + n)
        at += n
        place = torch.arange(n, device=DEV)
        for h in range(c["Hq"] if n else 0):
            q, k, v = s["q"][mine, h].double(), s["k"][mine, h // G].double(), s["v"][mine, h // G].double()
            for lo in range(0, n, 4096):  # queries, some at a time
                part = slice(at - n + lo, min(at, at - n + lo + 4096))
                z = q[lo:lo + 4096] @ k.t()
                z /= c["dh"] ** 0.5
                z += _exact_mask(c, place[lo:lo + 4096], place)
                lse[h, part] = torch.logsumexp(z, 1)
                w = torch.softmax(z, 1)
                out[part, h] = w @ v
                if c["train"]:
                    do = s["dout"][part, h].double()
                    dv[mine, h // G] += w.t() @ do
                    dz = do @ v.t()
                    dz -= (dz * w).sum(1, keepdim=True)
                    dz *= w
                    dz /= c["dh"] ** 0.5
                    dq[part, h] = dz @ k
                    dk[mine, h // G] += dz.t() @ q[lo:lo + 4096]
    found = {"out": out, "lse": lse}
    return found | {"dq": dq, "dk": dk, "dv": dv} if c["train"] else found


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "rope":
        out = {"y": _exact_turn(s, s["x"])}
        return out | {"dx": _exact_turn(s, s["dy"], -1)} if c["train"] else out
    if c["op"] == "append":
        return _exact_append(s)
    return _exact_paged(s) if c["op"] == "paged" else _exact_window(s)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def _pairs_seen(c, n):
    """Pairs of a query and a key that it sees in a sequence of n."""
    if not c["window"]:
        return n * (n + 1) // 2
    w, k = c["window"], c["sinks"]
    return sum(min(i + 1, w + min(k, max(0, i + 1 - w))) for i in range(n))


def work(case):
    c = case
    e = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "rope":
        passes = 2 if c["train"] else 1
        values = c["T"] * c["H"] * c["dh"]
        return {"bytes": passes * 2 * values * e + 4 * c["axes"] * c["T"] + 4 * c["pairs"],
                "flops": passes * 6 * c["T"] * c["H"] * c["pairs"]}
    if c["op"] == "append":
        T = c["B"] * c["new"]
        heads = 2 * c["Hkv"] + (c["Hq"] if c["queries"] else 0)
        return {"bytes": 2 * T * heads * c["dh"] * e + T * (8 + 4 * c["axes"]) + 4 * T + 4 * c["pairs"],
                "flops": 6 * T * (heads - c["Hkv"]) * c["pairs"]}
    if c["op"] == "paged":
        seen = [n if not c["window"] else min(n, c["window"] + min(c["sinks"], max(0, n - c["window"]))) for n in _lengths(c)]
        pages = sum(-(-n // c["page"]) for n in seen)
        return {"bytes": 2 * sum(seen) * c["Hkv"] * c["dh"] * e + 4 * pages + 4 * c["B"] + c["B"] * c["Hq"] * (2 * c["dh"] * e + 4),
                "flops": 4 * sum(seen) * c["Hq"] * c["dh"]}
    pairs = sum(_pairs_seen(c, n) for n in _lengths(c))
    q, kv = c["T"] * c["Hq"] * c["dh"] * e, c["T"] * c["Hkv"] * c["dh"] * e
    size = 2 * q + 2 * kv + 4 * c["T"] * c["Hq"]
    if c["train"]:
        size += 4 * q + 4 * kv + 4 * c["T"] * c["Hq"]
    return {"bytes": size, "flops": (14 if c["train"] else 4) * pairs * c["Hq"] * c["dh"]}
