"""What attention keeps of its weights where tensors are bf16: against the
definitions in 64 bits (attention_ref), with tolerances that leave no room for
weights rounded to bf16."""
import math

import pytest
import torch

from attention_ref import close, half_step, packed, turn, turn_tolerance
from neuralscript_b200 import ops
from test_gpu_attention_cache import run_window

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def normal(*shape, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g)


@pytest.mark.parametrize("Hq,Hkv,dh", [(8, 8, 64), (8, 2, 128), (32, 2, 64), (24, 1, 128)])
def test_weights_over_the_cache(Hq, Hkv, dh):
    """A weight takes part to 2^-16 of itself (eight digits, and the next rounded to eight: 2^-7 2^-9), the result is
    rounded once."""
    lens, page = [3, 17, 40, 1, 300], 16
    need = [-(-n // page) for n in lens]
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(n) + sum(need[:b])
    kc, vc = (normal(sum(need), page, Hkv, dh, seed=s).to(BF) for s in (1, 2))
    q = (0.25 * normal(len(lens), Hq, dh, seed=3)).to(BF)  # flat: weights that are no power of two
    out, scale = torch.empty_like(q), dh ** -0.5
    ops.attention_paged(q, kc, vc, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), out)
    for b, n in enumerate(lens):
        pages = table[b, :need[b]].cuda().long()
        k, v = (c[pages].reshape(-1, Hkv, dh)[:n].double().repeat_interleave(Hq // Hkv, 1) for c in (kc, vc))
        z = scale * torch.einsum("hd,jhd->hj", q[b].double(), k)
        size = scale * torch.einsum("hd,jhd->hj", q[b].double().abs(), k.abs()).amax(1)[:, None]
        p = torch.softmax(z, 1)
        want = torch.einsum("hj,jhd->hd", p, v)
        # scores and sums in fp32, twice (weights and their sum), as attention_ref counts them
        off = 4 * ((dh + 4) * size + n) * 2.0 ** -24 + 2.0 ** -19 + 2.0 ** -16
        tol = half_step(BF) * want.abs() + off * torch.einsum("hj,jhd->hd", p, v.abs())
        close(out[b], want, tol, f"out {b}")


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("lens", [[9], [9, 700], [2000]])  # finished by one warp, by a block, joined
def test_infinite_values_over_the_cache(lens, dtype):
    """An infinite value makes its column infinite, with its sign, also where its weight is a power of two; both: NaN."""
    page, dh = 16, 64
    pages = [-(-n // page) for n in lens]
    table = torch.zeros(len(lens), max(pages), dtype=torch.int32)
    for b, n in enumerate(pages):
        table[b, :n] = torch.arange(n) + sum(pages[:b])
    kc, vc = (normal(sum(pages), page, 1, dh, seed=s).to(dtype) for s in (1, 2))
    kc *= 0.1
    for q_of in (0.0, 1.0):  # equal weights, and any
        q = (q_of * normal(len(lens), 2, dh, seed=3)).to(dtype)
        for b, n in enumerate(lens):
            for j, col, to in ((0, 5, math.inf), (n - 1, 6, -math.inf), (n // 2, 7, math.inf), (n - 2, 7, -math.inf)):
                vc[int(table[b, j // page]), j % page, 0, col] = to
        out = torch.empty_like(q)
        ops.attention_paged(q, kc, vc, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), out)
        assert (out[..., 5] == math.inf).all() and (out[..., 6] == -math.inf).all() and out[..., 7].isnan().all()
        assert out[..., [c for c in range(dh) if c not in (5, 6, 7)]].isfinite().all()


@pytest.mark.parametrize("dh", [64, 128, 20, 100])  # (the last two: not on the tensor cores)
@pytest.mark.parametrize("lens,window,sinks", [([700], 2, 1), ([700, 300], 9, 4), ([700], 50, 3), ([600], 1, 63), ([2, 3, 5, 9, 40, 256], 0, 0)])
def test_gradients_of_rows_with_few_keys_and_first_tokens(lens, window, sinks, dh):
    """D = sum P dP, not the rounded output's, wherever rows see few keys: first tokens beside the window, any alignment."""
    run_window(lens, 4, 2, dh, window, sinks, BF, True, summed=True)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("window,sinks", [(0, 0), (11, 2)])
def test_prompt_then_tokens_by_the_rotated_heads(window, sinks, dtype):
    """Prompts, then single tokens, through rotation, cache and both attentions, against the definition on the queries
    that the calls gave and the keys and values that the cache holds: attention's tolerance alone. The same definition
    on mistaken places, sequences or windows is far outside it."""
    Hq, Hkv, dh, page, prompts, steps = 4, 2, 64, 8, [30, 5], 12
    total = [p + steps for p in prompts]
    whole = [normal(t, Hq + 2 * Hkv, dh, seed=b + 1).to(dtype) for b, t in enumerate(total)]
    freq = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().cuda()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    empty = lambda *s: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
    order = torch.randperm(sum(-(-t // page) for t in total), generator=torch.Generator().manual_seed(1)).tolist()
    table = [[order.pop() for _ in range(-(-t // page))] for t in total]
    pages, wide = sum(map(len, table)), max(map(len, table))
    kc, vc = (torch.full((pages, page, Hkv, dh), math.nan, dtype=dtype, device="cuda") for _ in "kv")
    on_device = ints([row + [-1] * (wide - len(row)) for row in table])
    seen = dict(window=window, sinks=sinks)

    def append(heads, seq, at):
        q = empty(heads.shape[0], Hq, dh)
        ops.kv_append(heads[:, Hq:Hq + Hkv], heads[:, Hq + Hkv:], seq, at, on_device, kc, vc, pos=at, freq=freq, q=heads[:, :Hq], q_out=q)
        return q

    heads = torch.cat([w[:p] for w, p in zip(whole, prompts)])
    T, at = sum(prompts), ints([i for p in prompts for i in range(p)])
    q = append(heads, ints([b for b, p in enumerate(prompts) for _ in range(p)]), at)
    k, out = empty(T, Hkv, dh), empty(T, Hq, dh)
    ops.rope(heads[:, Hq:Hq + Hkv], at, freq, k)
    ops.attention_window(q, k, heads[:, Hq + Hkv:], out, offsets=ints([0, prompts[0], T]), **seen)
    queries, found = ([[x[:prompts[0]]], [x[prompts[0]:]]] for x in (q, out))
    for s in range(steps):
        at = ints([p + s for p in prompts])
        q = append(torch.stack([w[p + s] for w, p in zip(whole, prompts)]), ints([0, 1]), at)
        out = empty(2, Hq, dh)
        ops.attention_paged(q, kc, vc, on_device, at + 1, out, **seen)
        for b in range(2):
            queries[b].append(q[b:b + 1])
            found[b].append(out[b:b + 1])
    ops.check_errors()
    queries, found = [torch.cat(x) for x in queries], [torch.cat(x) for x in found]
    held = [[c[ints(table[b]).long()].flatten(0, 1)[:total[b]] for b in range(2)] for c in (kc, vc)]
    for b, t in enumerate(total):
        k, v = held[0][b], held[1][b]
        assert torch.equal(v, whole[b][:, Hq + Hkv:])
        x = whole[b]
        turned = turn(x, torch.arange(t, device="cuda")[None], freq, torch.zeros(32, dtype=torch.long, device="cuda"), False, 1.0)
        tol = turn_tolerance(x, 32, False, 1.0, dtype, turned)
        close(queries[b], turned[:, :Hq], tol[:, :Hq], "queries")
        close(k, turned[:, Hq:Hq + Hkv], tol[:, Hq:Hq + Hkv], "keys")
        want, tol = packed(queries[b], k, v, [0, t], window, sinks, 0.125, dtype)["out"]
        assert tol.max() < 0.05  # of values with a spread of 1
        close(found[b], want, tol, "out")
        wrong = [(k, v.roll(1, 0), window, sinks), (k.roll(1, 0), v, window, sinks), (k, v, 7, sinks), (k, v.flip(1), window, sinks)]
        for other in wrong:
            want, tol = packed(queries[b], *other[:2], [0, t], *other[2:], 0.125, dtype)["out"]
            off = (found[b].double() - want).abs() > tol
            # (row 9 is the first that a window of 7 and 2 first tokens changes: row 8 sees 2 to 8, and 0 and 1)
            assert off[9:].any(-1).float().mean() > 0.9, other[2:]
