"""Rotary positions, the paged cache, attention over it and attention with a
window against their definitions in 64 bits (attention_ref), at the sizes and
masks where they can go wrong."""
import math

import pytest
import torch

from attention_ref import attend, close, half_step, mask, packed, turn, turn_tolerance
from neuralscript_b200 import ops

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


def normal(*shape, dtype=F, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def freqs(n):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float().cuda()


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,dh,sections", [(1, 1, 64, (32,)), (3, 5, 128, (64,)), (37, 3, 80, (8, 16, 16)), (2, 2, 6, (1, 0, 1)),
                                             (5, 4, 64, (5, 6)), (1301, 2, 48, (8,)), (2, 1, 1024, (500, 12)), (9, 7, 32, (4, 4, 4, 4))])
def test_rope_and_its_gradient(T, H, dh, sections, interleaved, dtype):
    n, A = sum(sections), len(sections)
    axis = torch.repeat_interleave(torch.arange(A), torch.tensor(sections)).cuda()
    freq = freqs(n)
    pos = torch.randint(-5, 100000, (A, T), device="cuda", dtype=torch.int32)
    x = normal(T, H, dh, dtype=dtype)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    kw = dict(sections=sections, interleaved=interleaved, scale=1.25)
    ops.rope(x, pos, freq, y, **kw)
    want = turn(x, pos, freq, axis, interleaved, 1.25)
    close(y, want, turn_tolerance(x, n, interleaved, 1.25, dtype, want), "y")
    assert torch.equal(y[..., 2 * n:], x[..., 2 * n:])
    ops.rope_bwd(x, pos, freq, dx, **kw)
    want = turn(x, pos, freq, axis, interleaved, 1.25, back=True)
    close(dx, want, turn_tolerance(x, n, interleaved, 1.25, dtype, want), "dx")
    ops.rope(x, pos, freq, x, **kw)  # in place
    assert torch.equal(x, y)


def test_rope_gradient_against_differences():
    """<rope(x), g> is linear in x: its change along e is <e, rope_bwd(g)>."""
    x, g, e = (normal(11, 3, 64, seed=s) for s in (1, 2, 3))
    pos, freq = ints(list(range(11))), freqs(20)
    a, b, dx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    ops.rope(x + e, pos, freq, a)
    ops.rope(x - e, pos, freq, b)
    ops.rope_bwd(g, pos, freq, dx)
    got, want = ((a - b).double() * g.double()).sum() / 2, (e.double() * dx.double()).sum()
    # every term carries a few roundings of fp32
    assert abs(got - want) <= 2.0 ** -20 * (g.double().abs() * (x.abs() + e.abs()).double()).sum()


@pytest.mark.parametrize("dtype", [BF, F])
def test_rope_strides_and_far_positions(dtype):
    """Heads of a wider buffer, rows that start between 16-byte boundaries, positions up to 2^31 - 1."""
    wide = normal(50, 9, 65, dtype=dtype)
    pos = torch.randint(0, 2 ** 31 - 1, (50,), device="cuda", dtype=torch.int32)
    freq = freqs(32)
    axis = torch.zeros(32, dtype=torch.long, device="cuda")
    for x in (wide[:, 2:5, :64], wide[:, 1:8:2, 1:], wide.transpose(0, 1).contiguous().transpose(0, 1)[:, 3:, :64]):
        T = x.shape[0]
        out = torch.full((T, x.shape[1] + 1, 66), 7.0, dtype=dtype, device="cuda")
        y = out[:, :-1, 1:65]
        ops.rope(x, pos[:T], freq, y)
        want = turn(x, pos[None, :T], freq, axis, False, 1.0)
        # the angle's own error in 64 bits: 2^31 * 2^-52
        close(y, want, turn_tolerance(x, 32, False, 1.0, dtype, want), "y")
        assert (out[:, -1] == 7).all() and (out[..., 0] == 7).all() and (out[..., 65] == 7).all()


def test_rope_of_no_tokens():
    x = torch.empty(0, 2, 64, device="cuda")
    ops.rope(x, torch.empty(0, dtype=torch.int32, device="cuda"), freqs(8), x)


# ---------------------------------------------------------------------------
# the paged cache
# ---------------------------------------------------------------------------
def empty_cache(pages, page, H, dh, dtype, heads_first, fill=math.nan):
    if heads_first:
        return torch.full((pages, H, page, dh), fill, dtype=dtype, device="cuda").transpose(1, 2)
    return torch.full((pages, page, H, dh), fill, dtype=dtype, device="cuda")


def make_table(lens, page, seed=0, spare=2):
    """Pages in any order; entries behind a sequence's last page name no page."""
    g = torch.Generator()
    g.manual_seed(seed)
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    table = torch.full((len(lens), max(need + [1])), -9, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
    return table.cuda(), sum(need) + spare


def fill_cache(cache, table, lens, rows):
    """rows: one tensor [len, H, dh] a sequence."""
    page = cache.shape[1]
    for b, n in enumerate(lens):
        for j in range(0, n, page):
            k = min(page, n - j)
            cache[int(table[b, j // page]), :k] = rows[b][j:j + k]


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("page,heads_first", [(1, False), (5, True), (16, False), (64, True)])
@pytest.mark.parametrize("Hq,Hkv,dh,n,interleaved", [(4, 2, 64, 32, False), (3, 1, 80, 20, True), (0, 3, 20, 0, False), (8, 8, 128, 64, True),
                                                     (2, 2, 6, 2, False)])
def test_append(page, heads_first, Hq, Hkv, dh, n, interleaved, dtype):
    had, new, pad = [0, 13, 64, 7], [5, 1, 17, 0], 3
    after = [a + b for a, b in zip(had, new)]
    table, pages = make_table(after, page)
    kc, vc = (empty_cache(pages, page, Hkv, dh, dtype, heads_first, fill) for fill in (5.0, 6.0))
    T = sum(new) + pad
    seq = [b for b, k in enumerate(new) for _ in range(k)] + [-1, -7, -1]
    at = [had[b] + i for b, k in enumerate(new) for i in range(k)] + [-3, 0, 2 ** 31 - 1]
    order = torch.randperm(T).tolist()  # tokens in any order
    seq, at = [seq[i] for i in order], [at[i] for i in order]
    heads = normal(T, Hq + 2 * Hkv, dh, dtype=dtype)
    q, k, v = heads[:, :Hq], heads[:, Hq:Hq + Hkv], heads[:, Hq + Hkv:]
    q_out = torch.full((T, Hq, dh), 3.0, dtype=dtype, device="cuda")
    pos = torch.randint(0, 5000, (2, T), device="cuda", dtype=torch.int32)
    kw, axis = {}, None
    if n:
        sections = (n - n // 4, n // 4)
        axis = torch.repeat_interleave(torch.arange(2), torch.tensor(sections)).cuda()
        kw = dict(pos=pos, freq=freqs(n), sections=sections, interleaved=interleaved, scale=0.75)
    if Hq:
        kw |= dict(q=q, q_out=q_out)
    ops.kv_append(k, v, ints(seq), ints(at), table, kc, vc, **kw)
    ops.check_errors()
    spin = lambda x: turn(x, pos, freqs(n), axis, interleaved, 0.75) if n else x.double()  # noqa: E731
    tol = lambda x, y: turn_tolerance(x, n, interleaved, 0.75, dtype, y) if n else torch.zeros_like(y)  # noqa: E731
    want_k, want_v = torch.full_like(kc, 5.0).double(), torch.full_like(vc, 6.0)
    tol_k = torch.zeros_like(want_k)
    real = [t for t in range(T) if seq[t] >= 0]
    where = (torch.tensor([int(table[seq[t], at[t] // page]) for t in real]), torch.tensor([at[t] % page for t in real]))
    want_k[where], tol_k[where] = spin(k)[real], tol(k, spin(k))[real]
    want_v[where] = v[real]
    close(kc, want_k, tol_k, "k_cache")
    assert torch.equal(vc, want_v)
    if Hq:
        close(q_out[real], spin(q)[real], tol(q, spin(q))[real], "q_out")
        assert (q_out[[t for t in range(T) if seq[t] < 0]] == 3).all()  # padding is left as it was


def test_append_leaves_out_and_reports_what_has_no_place():
    table = ints([[0, 7], [1, -1]])  # pages 7 and -1 are none
    seq, at = ints([0, 0, 1, 1, 2, 0, 0]), ints([0, 4, 3, 4, 0, 8, -1])
    k = normal(7, 1, 16)
    kc, vc = (empty_cache(3, 4, 1, 16, F, False, 0.0) for _ in "kv")
    ops.check_errors()
    ops.kv_append(k, k, seq, at, table, kc, vc)
    with pytest.raises(RuntimeError, match="index past"):
        ops.check_errors()
    ops.check_errors()
    want = torch.zeros_like(kc)
    want[0, 0], want[1, 3] = k[0], k[2]
    assert torch.equal(kc, want) and torch.equal(vc, want)


# ---------------------------------------------------------------------------
# one new token over the cache
# ---------------------------------------------------------------------------
def paged_case(lens, Hq, Hkv, dh, page, dtype, heads_first=False, window=0, sinks=0, scale=None, seed=0):
    table, pages = make_table(lens, page, seed)
    kc, vc = (empty_cache(pages, page, Hkv, dh, dtype, heads_first) for _ in "kv")  # NaN behind the sequences
    k, v = ([normal(n, Hkv, dh, dtype=dtype, seed=seed + 10 * b + i) for b, n in enumerate(lens)] for i in (1, 2))
    fill_cache(kc, table, lens, k)
    fill_cache(vc, table, lens, v)
    q = 2 * normal(len(lens), Hq, dh, dtype=dtype, seed=seed + 3)
    out, lse = torch.empty_like(q), torch.empty(len(lens), Hq, device="cuda")
    return dict(q=q, kc=kc, vc=vc, table=table, lens=ints(lens), out=out, lse=lse, k=k, v=v)


def check_paged(c, lens, Hq, Hkv, dh, dtype, window, sinks, scale):
    for b, n in enumerate(lens):
        for h in range(Hq):
            hk = h // (Hq // Hkv)
            if n == 0:
                assert (c["out"][b, h] == 0).all() and c["lse"][b, h] == -math.inf
                continue
            got = attend(c["q"][b, h][None].double(), c["k"][b][:, hk].double(), c["v"][b][:, hk].double(),
                         mask(1, n, window, sinks, "cuda"), scale, dtype)
            close(c["out"][b, h][None], *got["out"], f"out {b} {h}")
            close(c["lse"][b, h][None], *got["lse"], f"lse {b} {h}")


def run_paged(c, window, sinks, scale=None, **kw):
    ops.attention_paged(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["out"], lse=c["lse"], window=window, sinks=sinks,
                        scale=scale, **kw)


HEADS = [(1, 1, 64), (8, 2, 128), (6, 2, 64), (24, 4, 80), (16, 1, 96), (40, 2, 128), (3, 3, 20), (5, 1, 7), (4, 4, 128)]


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Hq,Hkv,dh", HEADS)
@pytest.mark.parametrize("page,heads_first", [(16, False), (24, True)])
def test_paged(Hq, Hkv, dh, page, heads_first, dtype):
    lens = [1, 0, 63, 64, 65, 700, 15, 16, 17, 129]
    c = paged_case(lens, Hq, Hkv, dh, page, dtype, heads_first)
    run_paged(c, 0, 0)
    check_paged(c, lens, Hq, Hkv, dh, dtype, 0, 0, dh ** -0.5)
    ops.check_errors()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 2), (64, 0), (100, 70), (64, 64), (128, 1000), (5000, 3), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_paged_window(window, sinks, dtype):
    lens = [1, 2, 5, 6, 66, 171, 1000, 333]
    c = paged_case(lens, 8, 2, 64, 8, dtype)
    run_paged(c, window, sinks, 0.3)
    check_paged(c, lens, 8, 2, 64, dtype, window, sinks, 0.3)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("lens,Hq,Hkv,page", [([20000], 4, 1, 32), ([20000, 3], 16, 2, 1), ([1] * 300, 2, 2, 16),
                                              ([9000, 1, 0, 0, 12000, 2], 12, 1, 48)])
def test_paged_long_and_many(lens, Hq, Hkv, page, dtype):
    """One sequence over all blocks, and more sequences than blocks; the same bits every time."""
    c = paged_case(lens, Hq, Hkv, 128, page, dtype)
    run_paged(c, 0, 0)
    check_paged(c, lens, Hq, Hkv, 128, dtype, 0, 0, 128 ** -0.5)
    first = c["out"].clone(), c["lse"].clone()
    for _ in range(3):
        run_paged(c, 0, 0)
        assert torch.equal(first[0], c["out"]) and torch.equal(first[1], c["lse"])


@pytest.mark.parametrize("dtype", [BF, F])
def test_paged_strides(dtype):
    """Heads of wider rows between 16-byte boundaries, caches side by side in one buffer, a wider table, a workspace of
    the caller's."""
    lens = [40, 129]
    c = paged_case(lens, 4, 2, 64, 16, dtype)
    both = torch.full((c["kc"].shape[0], 16, 3, 2, 70), math.nan, dtype=dtype, device="cuda")
    kc, vc = both[:, :, 1:, 0, 3:67], both[:, :, :2, 1, 5:69]
    kc.copy_(c["kc"]), vc.copy_(c["vc"])
    q = torch.empty(2, 5, 67, dtype=dtype, device="cuda")[:, 1:, 2:66]
    q.copy_(c["q"])
    out = torch.full((2, 4, 90), 4.0, dtype=dtype, device="cuda")
    table = torch.full((2, 20), 99, dtype=torch.int32, device="cuda")
    table[:, :c["table"].shape[1]] = c["table"]
    space = torch.empty(ops.attention_paged_workspace(2, 4, 2, 64), dtype=torch.uint8, device="cuda")
    ops.attention_paged(q, kc, vc, table[:, :c["table"].shape[1]], c["lens"], out[:, :, 7:71], lse=c["lse"], workspace=space)
    c["out"] = out[:, :, 7:71]
    check_paged(c, lens, 4, 2, 64, dtype, 0, 0, 0.125)
    assert (out[:, :, :7] == 4).all() and (out[:, :, 71:] == 4).all()


@pytest.mark.parametrize("dtype", [BF, F])
def test_paged_far_pages(dtype):
    """Pages more than 2^31 elements behind the cache's start."""
    lens, page, H, dh = [100, 50], 32, 2, 64
    pages = (2 ** 31) // (page * H * dh) + 9
    kc = torch.empty(pages, page, H, dh, dtype=dtype, device="cuda")
    vc = torch.empty(pages, page, H, dh, dtype=dtype, device="cuda")
    table = ints([[pages - 1, 0, pages - 3, pages - 4], [pages - 2, 5, 0, 0]])
    T = sum(lens)
    k, v = normal(T, H, dh, dtype=dtype), normal(T, H, dh, dtype=dtype, seed=2)
    seq, at = ints([0] * 100 + [1] * 50), ints(list(range(100)) + list(range(50)))
    ops.kv_append(k, v, seq, at, table, kc, vc)
    c = dict(q=normal(2, 4, dh, dtype=dtype, seed=3), kc=kc, vc=vc, table=table, lens=ints(lens), k=[k[:100], k[100:]], v=[v[:100], v[100:]],
             out=torch.empty(2, 4, dh, dtype=dtype, device="cuda"), lse=torch.empty(2, 4, device="cuda"))
    run_paged(c, 0, 0)
    check_paged(c, lens, 4, H, dh, dtype, 0, 0, 0.125)
    ops.check_errors()


@pytest.mark.parametrize("dtype", [BF, F])
def test_paged_bad_pages_and_lengths(dtype):
    """Pages that are none are left out, lengths past the table cut, both reported."""
    lens = [100, 64]
    c = paged_case(lens, 2, 1, 64, 16, dtype)
    c["table"][0, 2], c["table"][1, 3] = -1, 10 ** 6
    c["lens"] = ints([100, 64])
    run_paged(c, 0, 0)
    with pytest.raises(RuntimeError, match="index past"):
        ops.check_errors()
    c["k"] = [torch.cat([c["k"][0][:32], c["k"][0][48:]]), c["k"][1][:48]]
    c["v"] = [torch.cat([c["v"][0][:32], c["v"][0][48:]]), c["v"][1][:48]]
    check_paged(c, [84, 48], 2, 1, 64, dtype, 0, 0, 0.125)
    c = paged_case([96, 64], 2, 1, 64, 16, dtype)
    c["table"][1] = c["table"][0]  # two sequences may share pages
    c["k"][1], c["v"][1] = c["k"][0], c["v"][0]
    c["lens"] = ints([97, 2 ** 31 - 1])
    run_paged(c, 0, 0)
    with pytest.raises(RuntimeError, match="index past"):
        ops.check_errors()
    check_paged(c, [96, 96], 2, 1, 64, dtype, 0, 0, 0.125)
    c["lens"] = ints([-5, 96])
    run_paged(c, 0, 0)
    check_paged(c, [0, 96], 2, 1, 64, dtype, 0, 0, 0.125)
    ops.check_errors()


@pytest.mark.parametrize("dtype", [BF, F])
def test_paged_infinite_scores(dtype):
    """A key that gives -inf weighs nothing; where every key does, nothing is seen. +inf and NaN give NaN, in their head alone."""
    c = paged_case([20, 3], 4, 2, 64, 8, dtype)
    c["q"].abs_()
    for j, to in ((4, -math.inf), (7, -math.inf)):
        c["kc"][int(c["table"][0, j // 8]), j % 8, 0] = to
        c["k"][0][j, 0] = to
    run_paged(c, 0, 0)
    keep = [j for j in range(20) if j not in (4, 7)]
    for h in (0, 1):
        got = attend(c["q"][0, h][None].double(), c["k"][0][keep, 0].double(), c["v"][0][keep, 0].double(),
                     mask(1, 18, 0, 0, "cuda"), 0.125, dtype)
        close(c["out"][0, h][None], *got["out"])
    for j in range(3):
        c["kc"][int(c["table"][1, 0]), j, 0] = -math.inf
    c["kc"][int(c["table"][0, 1]), 1, 1] = math.nan
    run_paged(c, 0, 0)
    assert (c["out"][1, :2] == 0).all() and (c["lse"][1, :2] == -math.inf).all()
    assert c["out"][0, 2:].isnan().all() and c["lse"][0, 2:].isnan().all()
    assert c["out"][0, :2].isfinite().all() and c["out"][1, 2:].isfinite().all()


def test_paged_of_no_sequences():
    c = paged_case([3], 2, 1, 64, 8, BF)
    ops.attention_paged(c["q"][:0], c["kc"], c["vc"], c["table"][:0], c["lens"][:0], c["out"][:0])


# ---------------------------------------------------------------------------
# packed sequences with a window
# ---------------------------------------------------------------------------
def run_window(lens, Hq, Hkv, dh, window, sinks, dtype, train, spare=0, scale=None, amp=1.5, seed=1, lead=0, summed=False):
    """Fills rows of no sequence with NaN, and checks that they stay."""
    offsets = [lead]
    for n in lens:
        offsets.append(offsets[-1] + n)
    T = offsets[-1] + spare
    heads = normal(T, Hq + 2 * Hkv, dh, dtype=dtype, seed=seed)
    heads[:, :Hq] *= amp
    dout = normal(T, Hq, dh, dtype=dtype, seed=seed + 1)
    for x in (heads, dout):
        x[:lead] = math.nan
        x[offsets[-1]:] = math.nan
    q, k, v = heads[:, :Hq], heads[:, Hq:Hq + Hkv], heads[:, Hq + Hkv:]
    out = torch.full((T, Hq, dh), 9.0, dtype=dtype, device="cuda")
    lse = torch.full((Hq, T + 3), 9.0, device="cuda")[:, :T]
    kw = dict(offsets=ints(offsets), window=window, sinks=sinks, scale=scale)
    if scale is None:
        scale = dh ** -0.5
    ops.attention_window(q, k, v, out, lse=lse, **kw)
    want = packed(q, k, v, offsets, window, sinks, scale, dtype, dout if train else None, summed)
    mine = slice(offsets[0], offsets[-1])
    close(out[mine], *(x[mine] for x in want["out"]), "out")
    close(lse[:, mine], *(x[:, mine] for x in want["lse"]), "lse")
    outside = [i for i in range(T) if i < lead or i >= offsets[-1]]
    assert (out[outside] == 9).all() and (lse[:, outside] == 9).all()
    if train:
        grads = torch.full_like(heads, 9.0)
        dq, dk, dv = grads[:, :Hq], grads[:, Hq:Hq + Hkv], grads[:, Hq + Hkv:]
        ops.attention_window_bwd(q, k, v, out, lse, dout, dq, dk, dv, **kw)
        for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):
            close(x[mine], *(y[mine] for y in want[name]), name)
        assert (grads[outside] == 9).all()
        again = torch.empty_like(grads)
        ops.attention_window_bwd(q, k, v, out, lse, dout, again[:, :Hq], again[:, Hq:Hq + Hkv], again[:, Hq + Hkv:], **kw)
        assert torch.equal(again[mine], grads[mine])
    ops.check_errors()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Hq,Hkv,dh", [(1, 1, 64), (4, 2, 128), (3, 1, 64), (6, 3, 80), (2, 2, 32), (2, 1, 20), (1, 1, 7), (8, 1, 96)])
def test_window_heads(Hq, Hkv, dh, dtype):
    run_window([1, 0, 63, 65, 200], Hq, Hkv, dh, 50, 3, dtype, True, spare=5)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (64, 0), (65, 1), (127, 130), (128, 4), (129, 64), (300, 2), (2 ** 31 - 1, 2 ** 31 - 1),
                                          (40, 300)])
def test_window_masks(window, sinks, dh, dtype):
    run_window([129, 2, 520], 2, 1, dh, window, sinks, dtype, True, spare=1)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("n", [1, 2, 64, 127, 128, 129, 255, 256, 257, 383, 385, 1000])
def test_window_lengths(n, dtype):
    run_window([n], 2, 2, 64, 0, 0, dtype, True)
    run_window([n], 4, 1, 128, 100, 5, dtype, True, spare=130, lead=3)


@pytest.mark.parametrize("dtype", [BF, F])
def test_window_many_sequences(dtype):
    """More than a warp counts at once, empty ones among them."""
    lens = [(7 * i) % 31 for i in range(75)] + [0, 0, 140, 0]
    run_window(lens, 2, 1, 64, 9, 1, dtype, True, spare=3)


@pytest.mark.parametrize("dtype,amp", [(BF, 12.0), (F, 12.0), (BF, 0.01), (F, 0.01)])
def test_window_sharp_and_flat(dtype, amp):
    """Scores of some hundreds, so that maxima rise by much from tile to tile, and scores next to 0."""
    run_window([700], 2, 1, 64, 0, 0, dtype, True, scale=1.0, amp=amp)
    run_window([700], 2, 1, 128, 300, 7, dtype, True, scale=0.5, amp=amp)


@pytest.mark.parametrize("dtype", [BF, F])
def test_window_rising_scores(dtype):
    """Every key scores higher than all before it."""
    n, dh = 600, 64
    k = torch.zeros(n, 1, dh, device="cuda", dtype=dtype)
    k[:, 0, 0] = torch.arange(n, device="cuda", dtype=F).div(4).round().to(dtype)
    q = torch.zeros(n, 1, dh, device="cuda", dtype=dtype)
    q[:, 0, 0] = 1
    v, dout = normal(n, 1, dh, dtype=dtype), normal(n, 1, dh, dtype=dtype, seed=2)
    out, lse = torch.empty_like(q), torch.empty(1, n, device="cuda")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
    ops.attention_window(q, k, v, out, lse=lse, scale=1.0)
    ops.attention_window_bwd(q, k, v, out, lse, dout, dq, dk, dv, scale=1.0)
    want = packed(q, k, v, [0, n], 0, 0, 1.0, dtype, dout)
    for name, x in dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv).items():
        close(x, *want[name], name)


@pytest.mark.parametrize("dtype", [BF, F])
def test_window_unaligned(dtype):
    """Heads that start between 16-byte boundaries, in rows of odd length; heads outermost."""
    T, dh = 150, 64
    wide = normal(T, 3, 67, dtype=dtype)
    for q, k, v in ((wide[:, :2, 1:65], wide[:, 2:, 3:], wide[:, 1:2, 2:66]),
                    tuple(normal(H, T, dh, dtype=dtype, seed=s).transpose(0, 1) for H, s in ((2, 1), (1, 2), (1, 3)))):
        dout = normal(T, 2, dh, dtype=dtype, seed=5)
        out, lse = torch.empty(T, 2, 71, dtype=dtype, device="cuda")[..., 5:69], torch.empty(2, T, device="cuda")
        dq, dk, dv = (torch.empty(T, H, 65, dtype=dtype, device="cuda")[..., 1:] for H in (2, 1, 1))
        ops.attention_window(q, k, v, out, lse=lse, window=77, sinks=1)
        ops.attention_window_bwd(q, k, v, out, lse, dout, dq, dk, dv, window=77, sinks=1)
        want = packed(q, k, v, [0, T], 77, 1, 0.125, dtype, dout)
        for name, x in dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv).items():
            close(x, *want[name], name)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("lens,window", [([2, 3, 5, 9, 40, 256], 0), ([700, 1, 130], 2), ([300, 129], 100)])
def test_window_gradient_of_rows_with_few_keys(lens, window, dh):
    run_window(lens, 4, 2, dh, window, 0, BF, True, summed=True)


def test_window_gradient_against_differences():
    """The change of <out, g> along directions of q, k and v, in fp32 with a step of 2^-6 (its cube's share is below the
    tolerance of 2 %), against the gradients."""
    T, H, dh = 40, 2, 32
    x = {n: normal(T, 2 if n == "q" else 1, dh, seed=s) for n, s in (("q", 1), ("k", 2), ("v", 3))}
    g, lse, step = normal(T, H, dh, seed=4), torch.empty(H, T, device="cuda"), 2.0 ** -6

    def value(**kw):
        out = torch.empty(T, H, dh, device="cuda")
        ops.attention_window(*({**x, **kw}[n] for n in "qkv"), out, lse=lse, window=9, sinks=2)
        return out

    out = value()
    grads = [torch.empty_like(x[n]) for n in "qkv"]
    ops.attention_window_bwd(*(x[n] for n in "qkv"), out, lse, g, *grads, window=9, sinks=2)
    for n, d in zip("qkv", grads):
        e = d / d.norm()  # along the gradient itself, where the change is largest
        up, down = value(**{n: x[n] + step * e}), value(**{n: x[n] - step * e})
        got = ((up - down).double() * g.double()).sum() / (2 * step)
        want = (d.double() * e.double()).sum()
        assert abs(got - want) <= 0.02 * abs(want), (n, got, want)


@pytest.mark.parametrize("dtype", [BF, F])
def test_window_bad_offsets(dtype):
    """Falling offsets and ones past the rows are cut and reported."""
    T = 100
    q = normal(T, 1, 64, dtype=dtype)
    for bad in ([0, 50, 40, 100], [0, 101], [-1, 100]):
        out = torch.zeros_like(q)
        ops.attention_window(q, q, q, out, offsets=ints(bad))
        with pytest.raises(RuntimeError, match="index past"):
            ops.check_errors()
    ops.attention_window(q, q, q, out, offsets=ints([7]))  # no sequence


@pytest.mark.parametrize("dtype", [BF, F])
def test_window_row_without_a_finite_score(dtype):
    """A query whose every score is -inf sees nothing: out 0, lse -inf, no gradient of it."""
    T, dh = 70, 64
    q, k, v, g = (normal(T, 1, dh, dtype=dtype, seed=s) for s in (1, 2, 3, 4))
    q[0] = -3e38  # times 1e38 summed: -inf
    k[0] = 1e38
    q[1:] = q[1:] * 1e-30
    out, lse = torch.empty_like(q), torch.empty(1, T, device="cuda")
    ops.attention_window(q, k, v, out, lse=lse, window=1)
    assert (out[0] == 0).all() and lse[0, 0] == -math.inf and out[1:].isfinite().all()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
    ops.attention_window_bwd(q, k, v, out, lse, g, dq, dk, dv, window=1)
    assert (dq[0] == 0).all() and (dk[0] == 0).all() and (dv[0] == 0).all()
    assert torch.equal(dv[1:], g[1:])


# ---------------------------------------------------------------------------
# together: a prompt, then token by token
# ---------------------------------------------------------------------------
def decode_all(dtype, window, sinks, stream=None):
    """Two sequences through prompt and single tokens; every token's output as the whole sequence gives it."""
    Hq, Hkv, dh, page, prompts, steps = 4, 2, 64, 8, [30, 5], 12
    B, n = 2, 32
    total = [p + steps for p in prompts]
    freq = freqs(n)
    whole = [normal(t, Hq + 2 * Hkv, dh, dtype=dtype, seed=b + 1) for b, t in enumerate(total)]
    table, pages = make_table(total, page)
    kc, vc = (empty_cache(pages, page, Hkv, dh, dtype, False) for _ in "kv")
    # prompts, packed
    heads = torch.cat([w[:p] for w, p in zip(whole, prompts)])
    T = sum(prompts)
    seq = ints([b for b, p in enumerate(prompts) for _ in range(p)])
    at = ints([i for p in prompts for i in range(p)])
    q_out, k_out = torch.empty(T, Hq, dh, dtype=dtype, device="cuda"), torch.empty(T, Hkv, dh, dtype=dtype, device="cuda")
    q, k, v = heads[:, :Hq], heads[:, Hq:Hq + Hkv], heads[:, Hq + Hkv:]
    ops.kv_append(k, v, seq, at, table, kc, vc, pos=at, freq=freq, q=q, q_out=q_out)
    ops.rope(k, at, freq, k_out)
    out = torch.empty(T, Hq, dh, dtype=dtype, device="cuda")
    ops.attention_window(q_out, k_out, v, out, offsets=ints([0, prompts[0], T]), window=window, sinks=sinks)
    found = [[out[:prompts[0]]], [out[prompts[0]:]]]
    for s in range(steps):
        now = torch.stack([w[p + s] for w, p in zip(whole, prompts)])
        at = ints([p + s for p in prompts])
        q_out = torch.empty(B, Hq, dh, dtype=dtype, device="cuda")
        ops.kv_append(now[:, Hq:Hq + Hkv], now[:, Hq + Hkv:], ints([0, 1]), at, table, kc, vc, pos=at, freq=freq, q=now[:, :Hq],
                      q_out=q_out)
        out = torch.empty(B, Hq, dh, dtype=dtype, device="cuda")
        ops.attention_paged(q_out, kc, vc, table, at + 1, out, window=window, sinks=sinks)
        for b in range(B):
            found[b].append(out[b:b + 1])
    return [torch.cat(f) for f in found], whole, total, freq


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("window,sinks", [(0, 0), (11, 2)])
def test_prompt_then_tokens(window, sinks, dtype):
    found, whole, total, freq = decode_all(dtype, window, sinks)
    axis = torch.zeros(32, dtype=torch.long, device="cuda")
    for got, w, t in zip(found, whole, total):
        pos = torch.arange(t, device="cuda", dtype=torch.int32)[None]
        q, k = (turn(x, pos, freq, axis, False, 1.0).to(dtype) for x in (w[:, :4], w[:, 4:6]))
        want, tol = packed(q, k, w[:, 6:], [0, t], window, sinks, 0.125, dtype)["out"]
        # a rotated value next to the middle of two steps may round to the other one: a step more of q and k in the scores
        size = 2 * half_step(dtype) * 0.125 * (q.double().abs().amax() * k.double().abs().amax() * 64)
        close(got, want, tol + 4 * size * w[:, 6:].double().abs().amax(), "out")
    ops.check_errors()


def test_other_stream_and_graph():
    """A decode step captured and replayed: lengths, places and tokens are read from the device each time."""
    Hq, Hkv, dh, page = 4, 2, 128, 16
    table = ints([[0, 1, 2], [3, 4, 5]])
    kc, vc = (empty_cache(6, page, Hkv, dh, BF, False, 0.0) for _ in "kv")
    at, seq = ints([0, 20]), ints([0, 1])
    lens = at + 1
    heads = normal(2, Hq + 2 * Hkv, dh, dtype=BF)
    q_out, out = torch.empty(2, Hq, dh, dtype=BF, device="cuda"), torch.empty(2, Hq, dh, dtype=BF, device="cuda")
    freq = freqs(64)

    def step():
        ops.kv_append(heads[:, Hq:Hq + Hkv], heads[:, Hq + Hkv:], seq, at, table, kc, vc, pos=at, freq=freq, q=heads[:, :Hq], q_out=q_out)
        ops.attention_paged(q_out, kc, vc, table, lens, out)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    for g in (one, two):
        with torch.cuda.graph(g):
            step()
    for i in range(14):
        at.copy_(ints([i, 20 + i]))
        lens.copy_(at + 1)
        heads.copy_(normal(2, Hq + 2 * Hkv, dh, dtype=BF, seed=50 + i))
        (one if i % 3 else two).replay()
        got = out.clone()
        kc2, vc2 = kc.clone(), vc.clone()
        step()
        assert torch.equal(got, out) and torch.equal(kc, kc2) and torch.equal(vc, vc2)
    ops.check_errors()


def test_training_step_in_a_graph():
    T, Hq, Hkv, dh = 300, 4, 2, 64
    heads, dout = normal(T, Hq + 2 * Hkv, dh, dtype=BF), normal(T, Hq, dh, dtype=BF, seed=2)
    q, k, v = heads[:, :Hq], heads[:, Hq:Hq + Hkv], heads[:, Hq + Hkv:]
    out, lse, grads = torch.empty(T, Hq, dh, dtype=BF, device="cuda"), torch.empty(Hq, T, device="cuda"), torch.empty_like(heads)
    offsets = ints([0, 100, 300])

    def step():
        ops.attention_window(q, k, v, out, lse=lse, offsets=offsets, window=64, sinks=2)
        ops.attention_window_bwd(q, k, v, out, lse, dout, grads[:, :Hq], grads[:, Hq:Hq + Hkv], grads[:, Hq + Hkv:], offsets=offsets,
                                 window=64, sinks=2)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    heads.copy_(normal(T, Hq + 2 * Hkv, dh, dtype=BF, seed=9))
    offsets.copy_(ints([0, 170, 290]))
    grads.zero_()
    graph.replay()
    got = out.clone(), lse.clone(), grads.clone()
    step()
    for a, b in zip(got, (out, lse, grads)):
        assert torch.equal(a[..., :290, :] if a.dim() == 3 else a[:, :290], b[..., :290, :] if b.dim() == 3 else b[:, :290])


def test_two_streams_at_once():
    """Calls that overlap work in workspaces of their own."""
    cases = [paged_case([3000 + 50 * i, 10], 8, 2, 128, 16, BF, seed=100 * i) for i in range(4)]
    for c in cases:
        run_paged(c, 0, 0)
    want = [c["out"].clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                run_paged(c, 0, 0)
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c["out"], w)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(window=2 ** 31), dict(window=2 ** 32 + 5), dict(sinks=2 ** 32), dict(sinks=-2 ** 32), dict(window=-1)])
def test_window_past_32_bits(kw):
    c = paged_case([20], 4, 2, 64, 8, BF)
    with pytest.raises(ValueError):
        ops.attention_paged(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["out"], **kw)
    q, k, o, l = normal(4, 4, 64, dtype=BF), normal(4, 2, 64, dtype=BF), normal(4, 4, 64, dtype=BF), torch.empty(4, 4, device="cuda")
    with pytest.raises(ValueError):
        ops.attention_window(q, k, k, o, **kw)
    with pytest.raises(ValueError):
        ops.attention_window_bwd(q, k, k, o, l, o, q, k, k, **kw)


def test_python_refusals():
    c = paged_case([20], 4, 2, 64, 8, BF)
    q, kc, vc, t, n, out = c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["out"]
    for bad in (dict(q=q.half()), dict(q=q.float()), dict(kc=kc.float()), dict(vc=vc[:, :4]), dict(t=t.long()), dict(n=n.cpu()),
                dict(out=out[:, :2]), dict(n=n[None]), dict(q=q.transpose(1, 2)), dict(kc=kc[:, :, :1]), dict(t=t.cpu())):
        a = dict(q=q, kc=kc, vc=vc, t=t, n=n, out=out) | bad
        with pytest.raises((ValueError, RuntimeError)):
            ops.attention_paged(a["q"], a["kc"], a["vc"], a["t"], a["n"], a["out"])
    for kw in (dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
               dict(workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.attention_paged(q, kc, vc, t, n, out, **kw)
    x, pos, f = normal(4, 2, 64), ints([0, 1, 2, 3]), freqs(16)
    for a in ((x.half(), pos, f, x), (x, pos.long(), f, x), (x, pos[:3], f, x), (x, pos, f.double(), x), (x, pos, freqs(33), x),
              (x, pos, f, x[:, :1]), (x[..., :63], pos, f, x[..., :63]), (x, torch.stack([pos, pos]), f, x), (x, pos, f[:0], x)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.rope(*a)
    for s in ((8, 7), (16, 0, 0), (17, -1)):
        with pytest.raises(ValueError):
            ops.rope(x, torch.stack([pos, pos]), f, x, sections=s)
    k = normal(4, 2, 64, dtype=BF)
    for kw in (dict(pos=pos), dict(freq=f), dict(q=k), dict(q_out=k)):
        with pytest.raises(ValueError):
            ops.kv_append(k, k, pos, pos, t, kc, vc, **kw)
    q, o, l = normal(4, 4, 64, dtype=BF), normal(4, 4, 64, dtype=BF), torch.empty(4, 4, device="cuda")
    for a, kw in (((q, k, k[:, :1], o), {}), ((q[:, :3], k, k, o[:, :3]), {}), ((q, k, k, o.float()), {}), ((q, k, k, o), dict(window=-2)),
                  ((q, k, k, o), dict(lse=l[:, :2])), ((q, k, k, o), dict(offsets=pos.long())), ((q, k, k, o), dict(scale=0.0))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.attention_window(*a, **kw)
    with pytest.raises(ValueError):
        ops.attention_window_bwd(q, k, k, o, l, o, q, k, k[:2])


@pytest.mark.parametrize("dtype,dh", [(BF, 8), (BF, 7), (F, 8)])
def test_paged_of_the_longest_lengths(dtype, dh):
    """2^31 - 1 keys, of pages that are all one: cut to 2^31 - 16 (units of 16 are counted in 32 bits) and reported."""
    page, H = 1 << 20, 1
    kc, vc = normal(1, page, H, dh, dtype=dtype), torch.ones(1, page, H, dh, dtype=dtype, device="cuda")
    table = torch.zeros(1, (1 << 31) // page, dtype=torch.int32, device="cuda")
    q, out, lse = torch.zeros(1, H, dh, dtype=dtype, device="cuda"), torch.empty(1, H, dh, dtype=dtype, device="cuda"), torch.empty(1, H, device="cuda")
    for n, cut in ((2 ** 31 - 17, False), (2 ** 31 - 16, False), (2 ** 31 - 15, True), (2 ** 31 - 1, True)):
        out.zero_()
        ops.attention_paged(q, kc, vc, table, ints([n]), out, lse=lse)
        if cut:
            with pytest.raises(RuntimeError, match="index past"):
                ops.check_errors()
        ops.check_errors()
        # equal scores: the mean of ones, and the logarithm of how many; sums of up to 2^13 parts in fp32
        assert (out.double() - 1).abs().max() <= half_step(dtype) + 2.0 ** -11
        assert abs(float(lse) - math.log(min(n, 2 ** 31 - 16))) <= 2.0 ** -10


def test_sizes_past_32_bits():
    """ValueError from every entry that can meet them (the tensors have one row, seen 2^31 times)."""
    n = 2 ** 31
    x, many = torch.zeros(1, 1, 64, dtype=BF, device="cuda"), torch.zeros(1, 1, 64, dtype=BF, device="cuda").expand(n, 1, 64)
    cache, i = torch.zeros(1, 1, 1, 64, dtype=BF, device="cuda").expand(n, 1, 1, 64), ints([0])
    for call in (lambda: ops.rope(x.expand(1, n, 64), i, freqs(8), x.expand(1, n, 64)),
                 lambda: ops.kv_append(x, x, i, i, i[None], cache, cache),
                 lambda: ops.attention_paged(x, cache, cache, i[None], i, x),
                 lambda: ops.attention_window(many, many, many, many)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("n", [5, 16, 90, 3000])  # finished by a warp, by a block, joined
def test_paged_infinite_values_of_scores_of_minus_infinity(n, dtype):
    """Where every score is -inf nothing is seen, whatever the values are."""
    c = paged_case([n, n], 4, 2, 64, 8, dtype)
    c["q"].abs_()
    for j in range(n):
        c["kc"][int(c["table"][0, j // 8]), j % 8, 0] = -math.inf
    c["vc"][int(c["table"][0, 0]), 0, 0, 3::4] = math.inf
    c["vc"][int(c["table"][0, 0]), 1, 0, 2::4] = math.nan
    run_paged(c, 0, 0)
    assert (c["out"][0, :2] == 0).all() and (c["lse"][0, :2] == -math.inf).all()
    assert c["out"][0, 2:].isfinite().all() and c["out"][1].isfinite().all()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("B,Hq,Hkv,dh", [(900, 6, 2, 128), (2500, 4, 1, 64), (8192, 2, 1, 128)])
def test_paged_of_large_batches(B, Hq, Hkv, dh, dtype):
    """Up to the most sequences of a call, whose sums take shared memory from the rings."""
    lens = [(37 * b) % 61 for b in range(B)]
    lens[B // 2], lens[-1] = 900, 5
    c = paged_case(lens, Hq, Hkv, dh, 16, dtype)
    run_paged(c, 40, 3)
    some = sorted({0, 1, B // 2, B - 1} | set(range(7, B, B // 40)))
    part = {k: [c[k][b] for b in some] for k in ("k", "v")} | {k: c[k][some] for k in ("q", "out", "lse")}
    check_paged(part, [lens[b] for b in some], Hq, Hkv, dh, dtype, 40, 3, dh ** -0.5)
    assert c["out"].isfinite().all()
    ops.check_errors()
