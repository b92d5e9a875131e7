"""Mixture of experts with k experts a token on the GPU: routing, order of
the pairs, weighted sum and their gradients, against plain forms in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from neuralscript_b200 import ops  # noqa: E402

DEV = "cuda"
EPS = 2.0 ** -24  # half an ulp of fp32


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def apart(M, E, seed, step=0.02):
    """[M, E] values of which no two in a row are nearer than step, so that fp32 and fp64 order them alike."""
    g = gen(seed)
    order = torch.rand(M, E, device=DEV, generator=g).argsort(1)
    return ((order - E / 2) * step + torch.rand(M, 1, device=DEV, generator=g)).float()


def scores(x, active, score):
    x = x.double()
    if score == "sigmoid":
        return torch.sigmoid(x)
    if active is not None:
        x = torch.where(active[None] != 0, x, -math.inf)
    return torch.softmax(x, 1)


def route_ref(x, k, score, bias=None, active=None, groups=1, topk_groups=1, renorm=True, scale=1.0):
    """idx, w by a loop over rows on the host, in 64 bits."""
    p = scores(x, active, score).cpu()
    M, E = p.shape
    live = [True] * E if active is None else [bool(v) for v in active.cpu()]
    b = [0.0] * E if bias is None else [float(v) for v in bias.double().cpu()]
    idx = torch.full((M, k), -1, dtype=torch.int32)
    w = torch.zeros(M, k, dtype=torch.float64)
    for r in range(M):
        key = {e: float(p[r, e]) + b[e] for e in range(E) if live[e]}
        key = {e: v for e, v in key.items() if v > -math.inf}
        per = E // groups
        if groups > 1:
            best = {}
            for g in range(groups):
                two = sorted((key[e] for e in range(g * per, (g + 1) * per) if e in key), reverse=True)[:2]
                if two:
                    best[g] = sum(two)
            kept = sorted(best, key=lambda g: (-best[g], g))[:topk_groups]
            key = {e: v for e, v in key.items() if e // per in kept}
        top = sorted(key, key=lambda e: (-key[e], e))[:k]
        total = sum(float(p[r, e]) for e in top) + 1e-20 if renorm else 1.0
        for j, e in enumerate(top):
            idx[r, j] = e
            w[r, j] = scale * float(p[r, e]) / total
    return idx, w


def route(x, k, **how):
    M = x.shape[0]
    idx = torch.full((M, k), -7, dtype=torch.int32, device=DEV)
    w = torch.full((M, k), math.nan, device=DEV)
    ops.moe_topk_route(x, idx, w, **how)
    return idx, w


@pytest.mark.parametrize("M,E,k,groups,tg", [(1, 4, 1, 1, 1), (3, 8, 2, 1, 1), (5, 33, 8, 1, 1), (37, 60, 6, 4, 2),
                                             (64, 128, 8, 8, 4), (9, 256, 8, 8, 1), (4, 160, 32, 5, 5),
                                             (2, 1024, 32, 512, 20), (6, 7, 7, 1, 1), (130, 300, 5, 3, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_against_rows(M, E, k, groups, tg, score, renorm):
    x = apart(M, E, E + k, 4.0 / E)
    bias = torch.randn(E, device=DEV, generator=gen(k)) * 0.1 if renorm else None
    active = None
    if E % 2 == 0:
        active = (torch.rand(E, device=DEV, generator=gen(3)) > 0.2).to(torch.uint8)
        active[0] = 1
    how = dict(score=score, bias=bias, active=active, groups=groups, topk_groups=tg, renorm=renorm, scale=1.5)
    idx, w = route(x, k, **how)
    ref_i, ref_w = route_ref(x, k, **how)
    assert torch.equal(idx.cpu(), ref_i)
    # exp and division of a few ulps each, a sum of at most 32 terms
    assert torch.all((w.cpu().double() - ref_w).abs() <= 64 * EPS * ref_w.abs() + 1e-30)


def test_route_bf16_rows_of_a_wider_buffer_and_ties():
    wide = torch.randn(50, 80, device=DEV, generator=gen(1)).to(torch.bfloat16)
    wide[:, 70] = wide[:, 12]  # ties: bf16 logits also have their own
    x = wide[:, 3:75]
    idx, w = route(x, 6)
    key = x.float()
    ref = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :6]
    assert torch.equal(idx.long(), ref)
    p = torch.softmax(x.double(), 1).gather(1, ref)
    assert torch.all((w.double() - p / p.sum(1, keepdim=True)).abs() <= 64 * EPS)
    zeros = torch.zeros(5, 40, device=DEV)
    idx, w = route(zeros, 3, score="sigmoid", groups=4, topk_groups=2)
    assert torch.equal(idx.cpu(), torch.tensor([[0, 1, 2]] * 5, dtype=torch.int32))
    assert torch.all((w - 1 / 3).abs() <= 4 * EPS)


def test_route_rows_that_masks_leave_short_or_empty():
    x = torch.randn(4, 12, device=DEV, generator=gen(2))
    active = torch.zeros(12, dtype=torch.uint8, device=DEV)
    idx, w = route(x, 3, active=active)
    assert (idx == -1).all() and (w == 0).all()
    active[5] = 1
    for dead in (math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min, torch.finfo(torch.float32).max):
        x[:, :5] = dead
        x[:, 6:] = dead
        for score in ("softmax", "sigmoid"):
            idx, w = route(x, 3, score=score, active=active, groups=3, topk_groups=2)
            assert torch.equal(idx.cpu(), torch.tensor([[5, -1, -1]] * 4, dtype=torch.int32)), (dead, score)
            assert torch.all((w[:, 0] - 1).abs() <= 4 * EPS) and (w[:, 1:] == 0).all()
    # the lowest finite logit scores zero, but its expert lives
    x = torch.full((2, 6), torch.finfo(torch.float32).min, device=DEV)
    x[:, 4] = 1.0
    idx, w = route(x, 2)
    assert torch.equal(idx.cpu(), torch.tensor([[4, 0]] * 2, dtype=torch.int32)) and (w[:, 1] == 0).all()
    # no score: -inf everywhere, NaN, +inf
    for bad in (-math.inf, math.nan, math.inf):
        x = torch.full((1, 6), bad, device=DEV)
        idx, w = route(x, 2)
        assert (idx == -1).all() and (w == 0).all(), bad
    bias = torch.zeros(6, device=DEV)
    bias[1] = -math.inf
    idx, _ = route(torch.zeros(1, 6, device=DEV), 6, bias=bias)
    assert idx.cpu().tolist() == [[0, 2, 3, 4, 5, -1]]


def weights_of(x, idx, active, score, renorm, scale):
    """w as a function of the logits with the choice held, in 64 bits."""
    p = scores(x, active, score)
    on = idx >= 0
    c = torch.where(on, p.gather(1, idx.long().clamp(min=0)), 0)
    return scale * c / (c.sum(1, keepdim=True) + 1e-20) if renorm else scale * c


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("M,E,k", [(1, 2, 1), (7, 20, 3), (33, 130, 8), (3, 515, 32)])
def test_route_gradient_against_formula_and_differences(M, E, k, score, renorm):
    x = apart(M, E, 5 * E, 4.0 / E)
    active = torch.ones(E, dtype=torch.uint8, device=DEV)
    if E > 2:
        active[1] = 0
        x[0, 1] = math.nan
    how = dict(score=score, active=active, renorm=renorm, scale=2.5)
    idx, _ = route(x, k, **how)
    if M > 2:
        idx[1] = -1  # a row without any expert
        idx[2, 0] = -1
    dw = torch.randn(M, k, device=DEV, generator=gen(9))
    dw[idx < 0] = math.nan  # not looked at
    got = torch.full((M, E), math.nan, device=DEV)
    ops.moe_topk_route_bwd(dw, x, idx, got, **how)
    z = torch.where(active[None] != 0, x, 0).double().requires_grad_(True)
    f = lambda v: (weights_of(v, idx, active, score, renorm, 2.5) * torch.where(idx >= 0, dw, 0).double()).sum()  # noqa: E731
    f(z).backward()
    ref = z.grad * (active != 0)
    size = 2.5 * torch.where(idx >= 0, dw, 0).abs().sum(1, keepdim=True).double()
    assert torch.all((got.double() - ref).abs() <= 128 * EPS * size + 1e-30)
    if M > 2:
        assert (got[1] == 0).all()
    h = 1e-4
    for e in range(min(E, 4)):
        d = torch.zeros(M, E, dtype=torch.float64, device=DEV)
        d[:, e] = h * float(active[e])
        with torch.no_grad():
            for r in range(min(M, 3)):
                one = torch.zeros_like(d)
                one[r] = d[r]
                diff = (f(z + one) - f(z - one)) / (2 * h)
                # third derivatives of a (renormalised) score are below 8
                assert abs(float(got[r, e]) - float(diff)) <= 8 * h * h * float(size[r]) + 128 * EPS * float(size[r]) + 1e-9


def test_route_gradient_bf16():
    x = apart(40, 64, 4, 0.05).to(torch.bfloat16)
    idx, _ = route(x, 4)
    dw = torch.randn(40, 4, device=DEV, generator=gen(8))
    buf = torch.zeros(40, 72, device=DEV, dtype=torch.bfloat16)
    ops.moe_topk_route_bwd(dw, x, idx, buf[:, 1:65])
    z = x.double().requires_grad_(True)
    (weights_of(z, idx, None, "softmax", True, 1.0) * dw.double()).sum().backward()
    # one rounding to bf16
    assert torch.all((buf[:, 1:65].double() - z.grad).abs() <= 2.0 ** -8 * z.grad.abs() + 1e-6)
    assert (buf[:, 0] == 0).all() and (buf[:, 65:] == 0).all()


def dispatch(idx, E, align):
    M, k = idx.shape
    i32 = dict(dtype=torch.int32, device=DEV)
    out = [torch.full((E + 1,), -9, **i32), torch.full((E,), -9, **i32),
           torch.full((ops.moe_dispatch_rows(M, k, E, align),), -9, **i32), torch.full((M, k), -9, **i32)]
    ops.moe_dispatch(idx, E, *out, align=align)
    return out


@pytest.mark.parametrize("M,k,E,align", [(1, 1, 1, 1), (1, 8, 64, 128), (5, 3, 4, 1), (24, 8, 128, 1), (33, 2, 1024, 16),
                                         (1000, 4, 7, 128), (4099, 8, 60, 128), (40000, 2, 16, 1), (0, 2, 5, 128)])
def test_dispatch_against_a_stable_sort(M, k, E, align):
    idx = torch.randint(-1, E, (M, k), device=DEV, generator=gen(M + E), dtype=torch.int32)
    if M > 100:
        idx[:, 0] = E // 2  # one busy expert
        idx[3, 1] = E + 5   # outside: as none
    offsets, counts, rows, pos = (t.cpu() for t in dispatch(idx, E, align))
    flat = idx.reshape(-1).cpu().long()
    at = 0
    want_rows, want_pos = torch.full_like(rows, -1), torch.full((M * k,), -1, dtype=torch.int32)
    for e in range(E):
        pairs = (flat == e).nonzero()[:, 0].to(torch.int32)
        assert offsets[e] == at and counts[e] == len(pairs)
        want_rows[at:at + len(pairs)] = pairs
        want_pos[pairs.long()] = torch.arange(at, at + len(pairs), dtype=torch.int32)
        at += -(-len(pairs) // align) * align
    assert offsets[E] == at <= len(rows)
    assert torch.equal(rows, want_rows) and torch.equal(pos.reshape(-1), want_pos)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,k,E,D,align,pad", [(1, 1, 2, 1, 1, 0), (3, 2, 4, 8, 1, 0), (17, 8, 16, 136, 128, 8),
                                               (50, 3, 5, 77, 1, 3), (9, 4, 8, 2048, 128, 0), (260, 2, 8, 520, 128, 8),
                                               (5, 32, 40, 1030, 1, 2)])
def test_combine_and_gradient(dtype, M, k, E, D, align, pad):
    g = gen(D + M)
    idx = torch.rand(M, E, device=DEV, generator=g).argsort(1)[:, :k].to(torch.int32).contiguous()
    idx[0, 0] = -1
    if M > 2:
        idx[2] = -1
    _, _, rows, pos = dispatch(idx, E, align)
    R = rows.numel()
    wide = lambda n: torch.randn(n, D + pad, device=DEV, generator=g).to(dtype)[:, pad // 2:pad // 2 + D]  # noqa: E731
    o, dy, y, do = wide(R), wide(M), wide(M), wide(R)
    o[rows < 0] = math.nan  # padding is not read
    w = torch.randn(M, k, device=DEV, generator=g)
    w[pos < 0] = math.nan
    dw = torch.full((M, k), math.nan, device=DEV)
    ops.moe_combine(o, pos, y, w=w)
    ops.moe_combine_bwd(dy, o, rows, pos, w, do, dw)
    there = (pos >= 0)[:, :, None]
    os = torch.where(there, o[pos.long().clamp(min=0)].double(), 0)
    ws = torch.where(there[:, :, 0], w.double(), 0)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else EPS  # the one rounding of an output
    ref = (os * ws[:, :, None]).sum(1)
    size = (os * ws[:, :, None]).abs().sum(1)
    assert torch.all((y.double() - ref).abs() <= half * ref.abs() + 2 * k * EPS * size)
    ref_dw = (os * dy.double()[:, None]).sum(2)
    size = (os * dy.double()[:, None]).abs().sum(2)
    assert torch.all((dw.double() - ref_dw).abs() <= 2 * D * EPS * size)
    assert (dw[pos < 0] == 0).all()
    pair = rows.long().clamp(min=0)
    ref_do = torch.where((rows >= 0)[:, None], dy.double()[pair // k] * w.double().reshape(-1)[pair][:, None], 0)
    assert torch.all((do.double() - ref_do).abs() <= half * ref_do.abs())
    # differences: <y(o + h e) - y(o - h e)> / 2h along a random direction is <do, e>, for y is linear in o
    e = torch.randn(R, D, device=DEV, generator=g, dtype=torch.float64) * (rows >= 0)[:, None]
    es = torch.where(there, e[pos.long().clamp(min=0)], 0)
    diff = ((es * ws[:, :, None]).sum(1) * dy.double()).sum()
    assert abs(float((do.double() * e).sum() - diff)) <= 2 * half * float((ref_do * e).abs().sum()) + 1e-12
    # without weights: the gradient of a gather
    ops.moe_combine(o, pos, y)
    ref = os.sum(1)
    assert torch.all((y.double() - ref).abs() <= half * ref.abs() + 2 * k * EPS * os.abs().sum(1))
    again = do.clone()
    ops.moe_combine_bwd(dy, None, rows, pos, w, do)
    assert torch.equal(again, do)


def test_route_to_combine_on_a_side_stream():
    s = torch.cuda.Stream()
    x = torch.randn(300, 16, device=DEV, generator=gen(4))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        x2 = x * 2
        idx, w = route(x2, 2)
        _, _, rows, pos = dispatch(idx, 16, 1)
        y = torch.empty(300, 4, device=DEV)
        ops.moe_combine(torch.ones(600, 4, device=DEV), pos, y, w=w)
    s.synchronize()
    ref_i, _ = route(x * 2, 2)
    assert torch.equal(idx, ref_i)
    assert torch.all((y - 1).abs() <= 8 * EPS)  # renormalised weights of ones


def test_offsets_beyond_32_bits():
    """Rows so far apart that an element's number passes 2^31."""
    far = 2 ** 30
    wide = torch.empty(3 * far + 64, dtype=torch.bfloat16, device=DEV)
    x = wide.as_strided((4, 64), (far, 1))
    x.copy_(torch.randn(4, 64, device=DEV, generator=gen(1)))
    idx, w = route(x, 3)
    ref, ref_w = route(x.contiguous(), 3)
    assert torch.equal(idx, ref) and torch.equal(w, ref_w)
    pos = torch.tensor([[3, 0], [2, -1]], dtype=torch.int32, device=DEV)
    w = torch.randn(2, 2, device=DEV, generator=gen(2))
    y, near = torch.empty(2, 64, dtype=torch.bfloat16, device=DEV), torch.empty(2, 64, dtype=torch.bfloat16, device=DEV)
    ops.moe_combine(x, pos, y, w=w)
    ops.moe_combine(x.contiguous(), pos, near, w=w)
    assert torch.equal(y, near)
    rows = torch.tensor([1, -1, 2, 0], dtype=torch.int32, device=DEV)
    dw, dw_near = torch.empty(2, 2, device=DEV), torch.empty(2, 2, device=DEV)
    do = torch.empty(4, 64, dtype=torch.bfloat16, device=DEV)
    ops.moe_combine_bwd(y, x.contiguous(), rows, pos, w, do, dw_near)
    far_do = torch.empty(3 * far + 64, dtype=torch.bfloat16, device=DEV).as_strided((4, 64), (far, 1))
    ops.moe_combine_bwd(y, x, rows, pos, w, far_do, dw)
    assert torch.equal(far_do, do) and torch.equal(dw, dw_near)


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    idx = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    w = torch.zeros(4, 2, device=DEV)
    with pytest.raises(ValueError):
        ops.moe_topk_route(x.double(), idx, w)
    with pytest.raises(ValueError):
        ops.moe_topk_route(x, idx.long(), w)
    with pytest.raises(ValueError):
        ops.moe_topk_route(x.t(), idx[:, :1].contiguous(), w)
    with pytest.raises(ValueError):
        ops.moe_topk_route(x.cpu(), idx, w)
    with pytest.raises(RuntimeError):
        ops.moe_topk_route(x, idx, w, groups=3)
    with pytest.raises(RuntimeError):
        ops.moe_topk_route(x, idx, w, groups=8)  # one expert a group
    with pytest.raises(RuntimeError):
        ops.moe_topk_route(x, idx, w, groups=2, topk_groups=3)
    with pytest.raises(RuntimeError):
        ops.moe_topk_route(x, torch.zeros(4, 9, dtype=torch.int32, device=DEV), torch.zeros(4, 9, device=DEV))
    with pytest.raises(ValueError):
        ops.moe_dispatch(idx, 8, *(torch.zeros(n, dtype=torch.int32, device=DEV) for n in (9, 8, 9, 8)))
    with pytest.raises(ValueError):
        ops.moe_combine(torch.zeros(8, 4, device=DEV), idx, torch.zeros(4, 4, device=DEV, dtype=torch.bfloat16), w=w)
    with pytest.raises(ValueError):
        ops.moe_combine_bwd(torch.zeros(4, 4, device=DEV), None, idx.view(-1), idx, w, torch.zeros(8, 4, device=DEV), w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_tokens(dtype):
    """Every operator of the path takes a batch of no tokens."""
    f8, i32 = torch.float8_e4m3fn, dict(dtype=torch.int32, device=DEV)
    x, logits = torch.empty(0, 64, dtype=dtype, device=DEV), torch.empty(0, 16, dtype=dtype, device=DEV)
    idx, w, dw = torch.empty(0, 2, **i32), torch.empty(0, 2, device=DEV), torch.empty(0, 2, device=DEV)
    ops.moe_topk_route(logits, idx, w)
    ops.moe_topk_route_bwd(dw, logits, idx, torch.empty_like(logits))
    offsets, counts = torch.full((17,), -7, **i32), torch.full((16,), -7, **i32)
    rows, pos = torch.empty(0, **i32), torch.empty(0, 2, **i32)
    ops.moe_dispatch(idx, 16, offsets, counts, rows, pos, align=128)
    assert (offsets == 0).all() and (counts == 0).all()
    q, s = torch.empty(0, 64, dtype=f8, device=DEV), torch.empty(1, 0, device=DEV)
    qt, st = torch.empty(64, 0, dtype=f8, device=DEV), torch.empty(0, 64, device=DEV)
    ops.fp8_quantize(x, q, s, qt, st)
    ops.fp8_quantize(x, qt=qt, st=st, rows=rows, row_div=2)
    ops.fp8_quantize_block(x, q, torch.empty(0, 1, device=DEV), qt, torch.empty(1, 0, device=DEV))
    c = torch.empty(0, 32, dtype=dtype, device=DEV)
    ops.gemm_fp8(q, s, torch.zeros(32, 64, device=DEV).to(f8), torch.ones(1, 1, device=DEV), c)
    y = torch.empty(0, 32, dtype=dtype, device=DEV)
    ops.moe_combine(c, pos, y, w)
    ops.moe_combine_bwd(y, c, rows, pos, w, torch.empty_like(c), dw)
    torch.cuda.synchronize()


def test_indices_past_the_rows_are_left_out_and_reported():
    """Guarded by the kernels' own comparison with the number of rows."""
    f8, i32 = torch.float8_e4m3fn, dict(dtype=torch.int32, device=DEV)
    ops.check_errors()
    o = torch.randn(6, 40, device=DEV, generator=gen(1))
    pos = torch.tensor([[0, 6], [5, 2 ** 31 - 1], [1000000, -1]], **i32)
    y = torch.empty(3, 40, device=DEV)
    ops.moe_combine(o, pos, y)
    assert torch.equal(y[0], o[0]) and torch.equal(y[1], o[5]) and (y[2] == 0).all()
    with pytest.raises(RuntimeError, match="111"):
        ops.check_errors()
    ops.check_errors()  # read once
    dy, do, dw = torch.randn(3, 40, device=DEV, generator=gen(2)), torch.empty(4, 40, device=DEV), torch.empty(3, 2, device=DEV)
    rows, pos = torch.tensor([0, 6, 2 ** 31 - 1, 5], **i32), torch.tensor([[0, -1], [-1, -1], [-1, 3]], **i32)
    ops.moe_combine_bwd(dy, o[:4], rows, pos, None, do, dw)
    assert torch.equal(do[0], dy[0]) and torch.equal(do[3], dy[2]) and (do[1:3] == 0).all()
    assert (dw.flatten()[1:5] == 0).all() and dw[0, 0] != 0 and dw[2, 1] != 0
    with pytest.raises(RuntimeError, match="111"):
        ops.check_errors()
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(5, 48, device=DEV, generator=gen(3)).to(dtype)
        rows = torch.tensor([9, 10, 2 ** 31 - 1, 0, -1], **i32)
        q, s, qt, st = (torch.empty(5, 48, device=DEV).to(f8), torch.empty(1, 5, device=DEV),
                        torch.empty(48, 16, device=DEV).to(f8)[:, :5], torch.empty(1, 48, device=DEV))
        ops.fp8_quantize(x, q, s, qt, st, rows=rows, row_div=2)
        with pytest.raises(RuntimeError, match="111"):
            ops.check_errors()
        want, ws = torch.empty(2, 48, device=DEV).to(f8), torch.empty(1, 2, device=DEV)
        ops.fp8_quantize(x[[4, 0]], want, ws)
        assert torch.equal(q[[0, 3]].float(), want.float()) and torch.equal(s[:, [0, 3]], ws)
        assert (q[[1, 2, 4]].float() == 0).all() and (qt[:, [1, 2, 4]].float() == 0).all()
        assert (s[0, [1, 2, 4]] == 2.0 ** -100).all()
    ops.check_errors()


def test_dispatch_from_two_threads():
    """Orders of few and of many experts, whose launches take different amounts of shared memory, at the same time."""
    import threading
    errors = []

    def work(E, calls=3000):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                idx = torch.randint(0, E, (40, 2), device=DEV, dtype=torch.int32)
                i32 = dict(dtype=torch.int32, device=DEV)
                out = [torch.empty(E + 1, **i32), torch.empty(E, **i32), torch.empty(80, **i32), torch.empty(40, 2, **i32)]
                for _ in range(calls):
                    ops.moe_dispatch(idx, E, *out)
                assert int(out[1].sum()) == 80
        except Exception as e:
            errors.append((E, e))

    threads = [threading.Thread(target=work, args=(E,)) for E in (1024, 400, 1000, 512)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors


def test_dispatch_of_more_pairs_than_a_block_holds():
    """From 16 blocks x 32 warps x 256 pairs on a warp loads its pairs a second time to place them."""
    M, k, E = 40000, 4, 96
    assert M * k > 16 * 32 * 256
    idx = torch.randint(-1, E, (M, k), device=DEV, generator=gen(1), dtype=torch.int32)
    offsets, counts, rows, pos = dispatch(idx, E, 16)
    flat = idx.reshape(-1).long()
    key = torch.where(flat >= 0, flat, E)
    perm = torch.argsort(key, stable=True)
    n = torch.bincount(key, minlength=E + 1)[:E]
    start = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), ((n + 15) // 16 * 16).cumsum(0)])
    assert torch.equal(offsets.long(), start) and torch.equal(counts.long(), n)
    first = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), n.cumsum(0)])
    e = key[perm]
    there = e < E
    at = start[e[there]] + torch.arange(M * k, device=DEV)[there] - first[e[there]]
    want_rows, want_pos = torch.full_like(rows, -1), torch.full((M * k,), -1, dtype=torch.int32, device=DEV)
    want_rows[at] = perm[there].to(torch.int32)
    want_pos[perm[there]] = at.to(torch.int32)
    assert torch.equal(rows, want_rows) and torch.equal(pos.reshape(-1), want_pos)


def test_dispatch_in_a_graph():
    """One block, 8 and 16 of them, of few and of many experts, replayed on other choices."""
    for M, E in ((100, 8), (1000, 1024), (9000, 1024)):
        idx = torch.randint(0, E, (M, 2), device=DEV, generator=gen(M), dtype=torch.int32)
        out = dispatch(idx, E, 1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.moe_dispatch(idx, E, *out)
        idx.copy_(torch.randint(0, E, (M, 2), device=DEV, generator=gen(M + 1), dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, dispatch(idx, E, 1)))
