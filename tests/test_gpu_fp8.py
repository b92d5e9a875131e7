"""8-bit (e4m3) quantisation with a scale for each block of 128 and its
products on the GPU, against plain forms in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from neuralscript_b200 import ops  # noqa: E402

DEV = "cuda"
F8 = torch.float8_e4m3fn
EPS = 2.0 ** -24


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def up(n, m):
    return -(-n // m) * m


def codes(R, K, extra=0):
    """[R, K] codes with rows on 16-byte boundaries, filled with a value that shows where nothing was written."""
    return torch.full((R, up(K, 16) + extra), 0x55, dtype=torch.uint8, device=DEV).view(F8)[:, :K]


def scales(R, C, pad=0):
    return torch.full((R, C + pad), math.nan, device=DEV)[:, :C]


def ref_rows(x):
    """Codes [R, K] and scales [KB, R] in fp32, as defined: every operation is a single IEEE one."""
    R, K = x.shape
    KB = up(K, 128) // 128
    b = torch.nn.functional.pad(x.float(), (0, KB * 128 - K)).view(R, KB, 128)
    amax = torch.where(b.isnan(), 0, b.abs()).amax(2)
    s = torch.clamp(amax / 448, min=2.0 ** -100)
    q = (b * (1 / s)[:, :, None]).to(F8).view(R, KB * 128)[:, :K]
    return q, s.t()


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,off,pad", [(1, 1, 0, 0), (1, 128, 0, 0), (3, 300, 0, 4), (128, 128, 0, 0), (129, 1000, 1, 7),
                                         (257, 136, 8, 8), (40, 2050, 3, 2), (1000, 16, 0, 8)])
def test_quantize_rows_and_columns(dtype, M, K, off, pad):
    x = (torch.randn(M, off + K + pad, device=DEV, generator=gen(M + K)) * 3).to(dtype)[:, off:off + K]
    if M > 2:
        x[1] = 0
        x[2, : K // 2] *= 1e-30
    q, qt = codes(M, K), codes(K, M, 16)
    s, st = scales(up(K, 128) // 128, M, 3), scales(up(M, 128) // 128, K)
    ops.fp8_quantize(x, q, s, qt, st)
    rq, rs = ref_rows(x)
    assert torch.equal(s, rs) and same(q, rq)
    rq, rs = ref_rows(x.t())
    assert torch.equal(st, rs) and same(qt, rq)
    # each alone
    q2, s2, qt2, st2 = codes(M, K), scales(*s.shape), codes(K, M), scales(*st.shape)
    ops.fp8_quantize(x, q2, s2)
    ops.fp8_quantize(x, qt=qt2, st=st2)
    assert same(q, q2) and same(qt, qt2) and torch.equal(s, s2) and torch.equal(st, st2)


def test_quantize_writes_nothing_beside_its_rows():
    x = torch.randn(5, 37, device=DEV, generator=gen(1))
    buf = torch.full((7, 64), 0x55, dtype=torch.uint8, device=DEV)
    s = scales(1, 5)
    ops.fp8_quantize(x, buf.view(F8)[1:6, :37], s)
    assert (buf[0] == 0x55).all() and (buf[6] == 0x55).all() and (buf[1:6, 37:] == 0x55).all()


def test_quantize_infinities_nan_and_extremes():
    x = torch.randn(8, 256, device=DEV, generator=gen(2))
    x[0, 5] = math.nan
    x[1, 7] = math.inf
    x[2, 9] = -math.inf
    x[3] = torch.finfo(torch.float32).max
    x[4] = torch.finfo(torch.float32).tiny / 8
    x[5] = -0.0
    q, s = codes(8, 256), scales(2, 8)
    ops.fp8_quantize(x, q, s)
    v = q.float() * s.t().repeat_interleave(128, 1)
    assert v[0, 5].isnan() and v[0].isnan().sum() == 1
    for r in (1, 2):  # an infinity turns its own block to NaN, and no other
        assert v[r, :128].isnan().all() and not v[r, 128:].isnan().any()
    assert torch.all((v[3] / torch.finfo(torch.float32).max - 1).abs() < 1e-6)
    assert (v[4].abs() <= x[4].abs() * 2).all() and (v[5] == 0).all()


@pytest.mark.parametrize("act", [1, 5, 6])
def test_quantize_behind_an_activation(act):
    x = torch.randn(70, 200, device=DEV, generator=gen(act)).to(torch.bfloat16)
    q, s, qt, st = codes(70, 200), scales(2, 70), codes(200, 70), scales(1, 200)
    ops.fp8_quantize(x, q, s, qt, st, act=act)
    z = x.double()
    z = {1: torch.relu, 5: torch.nn.functional.silu, 6: torch.nn.functional.gelu}[act](z)
    for v, sc, ref in ((q, s, z), (qt, st, z.t())):
        wide = sc.t().double().repeat_interleave(128, 1)[:, :ref.shape[1]]
        # half a step of e4m3, and the activation's own few ulps
        step = torch.maximum(ref.abs() * 2.0 ** -4, wide * 2.0 ** -10)
        assert torch.all((v.double() * wide - ref).abs() <= step * (1 + 1e-5) + 1e-6 * ref.abs())


def activated(x, act):
    """The activations in 64 bits, as the fp32 ones treat infinities and NaN."""
    x = x.double()
    if act == 1:
        return torch.where(x > 0, x, 0)
    if act == 2:
        return torch.where(x > 0, x, 0.01 * x)
    if act == 3:
        return 1 / (1 + torch.exp(-x))
    if act == 4:
        return torch.tanh(x)
    if act == 5:
        return x / (1 + torch.exp(-x))
    return 0.5 * x * (1 + torch.erf(x / math.sqrt(2))) if act else x


def read_back_ok(q, s, z):
    """Codes and scales (of 128 along a row) of z: an infinity turns its block to NaN, a NaN only itself, all else is
    within half a step of e4m3 and 1e-5 (above what the fp32 activations are off by) of its value."""
    R, K = z.shape
    wide = s.t().double().repeat_interleave(128, 1)[:, :K]
    v = q.double() * wide
    blocks = torch.nn.functional.pad(z, (0, up(K, 128) - K)).view(R, -1, 128)
    lost = blocks.isinf().any(2).repeat_interleave(128, 1)[:, :K] | z.isnan()
    ok = torch.where(lost, v.isnan(), (v - z).abs() <= torch.maximum(z.abs() * 2.0 ** -4, wide * 2.0 ** -10) + 1e-5 * z.abs())
    return ok.all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", range(8))
def test_quantize_infinities_and_nan_behind_activations(act, dtype):
    M, K = 300, 270
    x = torch.randn(M, K, device=DEV, generator=gen(act)).to(dtype)
    for i, bad in enumerate((math.inf, -math.inf, math.nan)):
        x[3 + i, 5 + i] = x[140 + i, 100 + 40 * i] = x[299 - i, 269 - i] = bad
    x[200, 200], x[210, 210] = torch.finfo(dtype).max, -torch.finfo(dtype).max
    for a in (x, torch.cat([x, x], 1)[:, 1:K + 1]):  # on 16-byte boundaries and off them
        z = activated(a, act)
        q, s, qt, st = codes(M, K), scales(up(K, 128) // 128, M), codes(K, M), scales(up(M, 128) // 128, K)
        ops.fp8_quantize(a, q, s, qt, st, act=act)
        assert read_back_ok(q, s, z) and read_back_ok(qt, st, z.t())


def test_quantize_behind_gelu_far_out():
    """Blocks of one value, so that the scale tells GELU's own error. Roundings of x^2 / 2 log2(e) (constants and
    operations: seven halves of an ulp) are multiplied by x^2 / 2; the rest is below 3e-6."""
    x = torch.cat([torch.linspace(-13, -1e-3, 4000), torch.linspace(1e-3, 30, 1000)]).to(DEV)[:, None]
    q, s = codes(5000, 1), scales(1, 5000)
    ops.fp8_quantize(x, q, s, act=6)
    z = 0.5 * x.double() * torch.special.erfc(-x.double() / math.sqrt(2))
    want = torch.clamp(z.abs() / 448, min=2.0 ** -100)[:, 0]
    assert ((s[0].double() - want).abs() <= want * (x[:, 0].double() ** 2 / 2 * 7 * EPS + 3e-6)).all()
    far = torch.tensor([[-13.3], [-20.0], [-1e10], [-torch.finfo(torch.float32).max]], device=DEV)
    q, s = codes(4, 1), scales(1, 4)
    ops.fp8_quantize(far, q, s, act=6)
    assert (q.float() == 0).all() and (s == 2.0 ** -100).all()


def test_quantize_block_infinities_and_nan():
    x = torch.randn(300, 400, device=DEV, generator=gen(1))
    x[130, 7], x[5, 300], x[299, 399], x[0, 0] = math.inf, -math.inf, math.nan, math.nan
    q, s, qt, st = codes(300, 400), scales(3, 4), codes(400, 300), scales(4, 3)
    ops.fp8_quantize_block(x, q, s, qt, st)
    wide = s.double().repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :400]
    v = q.double() * wide
    lost = x.isnan()
    lost[128:256, :128] = True
    lost[:128, 256:384] = True
    near = (v - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, wide * 2.0 ** -10) * (1 + 1e-6)
    assert torch.where(lost, v.isnan(), near).all()
    assert same(qt, q.t()) and torch.equal(st, s.t())


def test_quantize_gathered_rows():
    x = torch.randn(50, 90, device=DEV, generator=gen(3)).to(torch.bfloat16)
    rows = torch.randint(-1, 150, (300,), device=DEV, generator=gen(4), dtype=torch.int32)
    full = torch.where((rows >= 0)[:, None], x[rows.long().clamp(min=0) // 3], 0)
    qt, st, q, s = codes(90, 300), scales(3, 90), codes(300, 90), scales(1, 300)
    ops.fp8_quantize(x, q, s, qt, st, rows=rows, row_div=3)
    rq, rs = ref_rows(full.t())
    assert same(qt, rq) and torch.equal(st, rs)
    rq, rs = ref_rows(full)
    assert same(q, rq) and torch.equal(s, rs)
    y = torch.randn(300, 90, device=DEV, generator=gen(5))
    y[rows < 0] = math.nan
    ops.fp8_quantize(y, qt=qt, st=st, rows=rows, row_div=0)
    rq, rs = ref_rows(torch.where((rows >= 0)[:, None], y, 0).t())
    assert same(qt, rq) and torch.equal(st, rs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K", [(1, 1), (128, 128), (130, 260), (77, 1000), (512, 24)])
def test_quantize_block(dtype, M, K):
    x = torch.randn(M, K + 1, device=DEV, generator=gen(M * K)).to(dtype)[:, 1:]
    MB, KB = up(M, 128) // 128, up(K, 128) // 128
    q, s, qt, st = codes(M, K), scales(MB, KB, 1), codes(K, M), scales(KB, MB)
    ops.fp8_quantize_block(x, q, s, qt, st)
    b = torch.nn.functional.pad(x.float(), (0, KB * 128 - K, 0, MB * 128 - M)).view(MB, 128, KB, 128)
    rs = torch.clamp(b.abs().amax((1, 3)) / 448, min=2.0 ** -100)
    rq = (b * (1 / rs)[:, None, :, None]).to(F8).view(MB * 128, KB * 128)[:M, :K]
    assert torch.equal(s, rs) and same(q, rq) and torch.equal(st, rs.t()) and same(qt, rq.t())


# --------------------------------------------------------------------------
# products
# --------------------------------------------------------------------------
def values_rows(q, s):
    return q.double() * s.t().double().repeat_interleave(128, 1)[:, :q.shape[1]]


def values_block(q, s):
    N, K = q.shape
    return q.double() * s.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]


def rows_of(x, pad=0):
    R, K = x.shape
    q, s = codes(R, K), scales(up(K, 128) // 128, R, pad)
    ops.fp8_quantize(x, q, s)
    return q, s


def block_of(x):
    N, K = x.shape
    q, s = codes(N, K), scales(up(N, 128) // 128, up(K, 128) // 128)
    ops.fp8_quantize_block(x, q, s)
    return q, s


def near(c, a, b, K):
    """c against a b^T: sums of 128 in fp32 (a lost bit an addition at most), those summed, one rounding."""
    ref, size = a @ b.t(), a.abs() @ b.abs().t()
    half = 2.0 ** -8 if c.dtype == torch.bfloat16 else EPS
    return torch.all((c.double() - ref).abs() <= half * ref.abs() + (128 + up(K, 128) // 128) * 2 * EPS * size)


def wild(R, K, seed):
    """Values whose 128-blocks differ in size by many powers of two."""
    g = gen(seed)
    x = torch.randn(R, K, device=DEV, generator=g)
    return x * torch.exp2(torch.randint(-8, 9, (R, 1), device=DEV, generator=g).float()) * \
        torch.exp2(torch.randint(-6, 7, (1, up(K, 128) // 128), device=DEV, generator=g).float()).repeat_interleave(128, 1)[:, :K]


SIZES = [(1, 1, 1), (1, 8, 128), (1, 4096, 512), (2, 130, 129), (5, 24, 1000), (16, 512, 384), (17, 256, 127), (33, 1000, 640),
         (64, 128, 16), (100, 520, 1032), (128, 256, 256), (129, 257, 513), (300, 72, 2048), (700, 1000, 300),
         (2000, 384, 136), (1024, 1024, 1024)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("by_rows", [False, True])
def test_product(M, N, K, out, by_rows):
    a, sa = rows_of(wild(M, K, M + 1), 1)
    b, sb = rows_of(wild(N, K, N + 2)) if by_rows else block_of(wild(N, K, N + 2))
    c = torch.full((M + 2, N), math.nan, dtype=out, device=DEV)
    ops.gemm_fp8(a, sa, b, sb, c[1:M + 1])
    assert near(c[1:M + 1], values_rows(a, sa), values_rows(b, sb) if by_rows else values_block(b, sb), K)
    assert c[0].isnan().all() and c[M + 1].isnan().all()


@pytest.mark.parametrize("M,N,K", [(3900, 2500, 300), (4096, 2304, 128), (2900, 3400, 1000)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product_of_many_tiles(M, N, K, out):
    """Sizes from which pairs of CTAs share tiles, some of whose second halves are empty."""
    a, sa = rows_of(wild(M, K, 1), 3)
    b, sb = block_of(wild(N, K, 2))
    c = torch.full((M + 1, N), math.nan, dtype=out, device=DEV)
    ops.gemm_fp8(a, sa, b, sb, c[:M])
    assert near(c[:M], values_rows(a, sa), values_block(b, sb), K)
    assert c[M].isnan().all()


@pytest.mark.parametrize("M", [3, 200])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product_into_rows_of_a_wider_buffer(M, out):
    N, K = 300, 400
    a, sa = rows_of(wild(M, K, 1))
    b, sb = block_of(wild(N, K, 2))
    for off, ld in ((0, 304), (8, 320), (1, 303), (3, 305)):
        c = torch.full((M, ld), 7.0, dtype=out, device=DEV)
        ops.gemm_fp8(a, sa, b, sb, c[:, off:off + N])
        assert near(c[:, off:off + N], values_rows(a, sa), values_block(b, sb), K)
        assert (c[:, :off] == 7).all() and (c[:, off + N:] == 7).all()


def test_product_propagates_nan():
    x = torch.randn(130, 256, device=DEV, generator=gen(1))
    x[3, 200] = math.nan
    x[129, 0] = math.inf
    for M in (130, 4):
        a, sa = rows_of(x[:M])
        b, sb = block_of(torch.randn(70, 256, device=DEV, generator=gen(2)))
        c = torch.empty(M, 70, device=DEV)
        ops.gemm_fp8(a, sa, b, sb, c)
        bad = c.isnan().all(1).nonzero()[:, 0].tolist()
        assert bad == ([3, 129] if M == 130 else [3]) and c.isnan().any(1).sum() == len(bad)


@pytest.mark.parametrize("M,N,K", [(200, 256, 384), (1000, 136, 272)])
def test_gradients_of_a_linear_layer(M, N, K):
    """y = x w^T: the input gradient takes the weight's transposed codes, the weight gradient two transposed
    quantisations; against the formula on the quantised values, and against differences of the double loss."""
    x, w, dy = wild(M, K, 1), wild(N, K, 2), torch.randn(M, N, device=DEV, generator=gen(3))
    kb, nb, mb = up(K, 128) // 128, up(N, 128) // 128, up(M, 128) // 128
    wq, ws, wqt, wst = codes(N, K), scales(nb, kb), codes(K, N), scales(kb, nb)
    ops.fp8_quantize_block(w, wq, ws, wqt, wst)
    g, sg, gt, sgt = codes(M, N), scales(nb, M), codes(N, M), scales(mb, N)
    ops.fp8_quantize(dy, g, sg, gt, sgt)
    xt, sxt = codes(K, M), scales(mb, K)
    ops.fp8_quantize(x, qt=xt, st=sxt)
    dx, dw = torch.empty(M, K, dtype=torch.bfloat16, device=DEV), torch.empty(N, K, device=DEV)
    ops.gemm_fp8(g, sg, wqt, wst, dx)
    ops.gemm_fp8(gt, sgt, xt, sxt, dw)
    gv, wv = values_rows(g, sg), values_block(wq, ws)
    gtv, xv = values_rows(gt, sgt), values_rows(xt, sxt).t()
    assert near(dx, gv, wv.t(), N)
    assert near(dw, gtv, xv.t(), M)
    # loss L = <dy, x w^T>: a difference along a direction is the gradient's product with it
    e = torch.randn(N, K, device=DEV, generator=gen(4), dtype=torch.float64)
    h = 1e-3
    loss = lambda v: (gtv.t() * (xv @ v.t())).sum()  # noqa: E731
    diff = (loss(wv + h * e) - loss(wv - h * e)) / (2 * h)
    size = ((gtv.abs() @ xv.abs()) * e.abs()).sum()
    assert abs(float((dw.double() * e).sum() - diff)) <= 300 * EPS * float(size)


def order(idx, E, align):
    M, k = idx.shape
    i32 = dict(dtype=torch.int32, device=DEV)
    out = [torch.empty(E + 1, **i32), torch.empty(E, **i32), torch.empty(ops.moe_dispatch_rows(M, k, E, align), **i32),
           torch.empty(M, k, **i32)]
    ops.moe_dispatch(idx, E, *out, align=align)
    return out


def choose(M, k, E, seed):
    idx = torch.rand(M, E, device=DEV, generator=gen(seed)).argsort(1)[:, :k].to(torch.int32).contiguous()
    if E > 3:
        idx[idx == 2] = 3 if k == 1 else -1  # an expert without rows
    return idx


@pytest.mark.parametrize("M,k,E,N,K,align", [(1, 1, 2, 128, 128, 1), (1, 4, 8, 24, 48, 1), (24, 4, 64, 256, 128, 1),
                                             (24, 2, 8, 136, 400, 128), (300, 2, 4, 520, 272, 1), (300, 4, 8, 256, 512, 128),
                                             (2000, 2, 8, 72, 144, 128), (1500, 3, 5, 384, 1040, 1), (7, 1, 1, 8, 16, 1)])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_experts_product(M, k, E, N, K, align, gather, out):
    offsets, counts, rows, pos = order(choose(M, k, E, M + E), E, align)
    R = rows.numel()
    a, sa = rows_of(wild(M if gather else R, K, 1), 2)
    ws = [block_of(wild(N, K, 10 + e)) for e in range(E)]
    b, sb = torch.stack([q.view(torch.uint8) for q, _ in ws]), torch.stack([s for _, s in ws])
    wide = torch.zeros(E, N + 1, up(K, 16), dtype=torch.uint8, device=DEV)  # experts a row further apart
    wide[:, :N, :K] = b
    b = wide.view(F8)[:, :N, :K]
    c = torch.full((R, N), 7.0, dtype=out, device=DEV)
    ops.moe_gemm_fp8(a, sa, offsets, counts, b, sb, c, rows=rows if gather else None, row_div=k)
    av = values_rows(a, sa)
    written = torch.zeros(R, dtype=torch.bool, device=DEV)
    for e in range(E):
        o, n = int(offsets[e]), int(counts[e])
        src = rows[o:o + n].long() // k if gather else torch.arange(o, o + n, device=DEV)
        assert near(c[o:o + n], av[src], values_block(*ws[e]), K), e
        written[o:o + n] = True
    assert (c[~written] == 7).all()


@pytest.mark.parametrize("M,k,E,N,K", [(1, 1, 2, 8, 16), (40, 2, 4, 136, 72), (700, 2, 8, 256, 384), (3000, 4, 16, 130, 520)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_experts_weight_gradient(M, k, E, N, K, out):
    offsets, counts, rows, pos = order(choose(M, k, E, M), E, 128)
    R = rows.numel()
    x, dz = wild(M, K, 1), torch.randn(R, N, device=DEV, generator=gen(2))
    dz[rows < 0] = math.nan
    xt, sx, gt, sg = codes(K, R), scales(R // 128, K), codes(N, R), scales(R // 128, N)
    ops.fp8_quantize(x, qt=xt, st=sx, rows=rows, row_div=k)
    ops.fp8_quantize(dz, qt=gt, st=sg, rows=rows, row_div=0)
    c = torch.full((E, N, K), math.nan, dtype=out, device=DEV)
    ops.moe_wgrad_fp8(gt, sg, xt, sx, offsets, counts, c)
    gv, xv = values_rows(gt, sg), values_rows(xt, sx)
    for e in range(E):
        o, n = int(offsets[e]), int(counts[e])
        assert near(c[e], gv[:, o:o + n], xv[:, o:o + n], n), e
        if n == 0:
            assert (c[e] == 0).all()


def test_experts_without_tokens():
    i32 = dict(dtype=torch.int32, device=DEV)
    offsets, counts = torch.zeros(4, **i32), torch.zeros(3, **i32)
    c = torch.full((3, 16, 32), math.nan, device=DEV)
    e8 = lambda r, k: torch.empty(r, k, dtype=torch.uint8, device=DEV).view(F8)  # noqa: E731
    ops.moe_wgrad_fp8(e8(16, 0), scales(0, 16), e8(32, 0), scales(0, 32), offsets, counts, c)
    assert (c == 0).all()
    ops.moe_gemm_fp8(e8(0, 32), scales(1, 0), offsets, counts, e8(48, 32).view(3, 16, 32), scales(3, 1).view(3, 1, 1),
                     torch.empty(0, 16, device=DEV))


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_sums_of_nothing(out):
    """K = 0: zeros, in the experts' own rows alone."""
    i32 = dict(dtype=torch.int32, device=DEV)
    c = torch.full((9, 40), 7.0, dtype=out, device=DEV)
    ops.gemm_fp8(codes(5, 0), scales(0, 5), codes(24, 0), scales(1, 0), c[2:7, 8:32])
    want = torch.full_like(c, 7)
    want[2:7, 8:32] = 0
    assert torch.equal(c, want)
    offsets, counts = torch.tensor([0, 128, 256, 384], **i32), torch.tensor([5, 0, 100], **i32)
    c = torch.full((384, 24), 7.0, dtype=out, device=DEV)
    ops.moe_gemm_fp8(codes(384, 0), scales(0, 384), offsets, counts, codes(72, 0).view(3, 24, 0),
                     torch.empty(3, 1, 0, device=DEV), c)
    want = torch.full_like(c, 7)
    want[:5] = want[256:356] = 0
    assert torch.equal(c, want)


def test_product_on_a_side_stream_and_in_a_graph():
    a, sa = rows_of(wild(20, 512, 1))
    b, sb = block_of(wild(256, 512, 2))
    c = torch.empty(20, 256, device=DEV)
    ops.gemm_fp8(a, sa, b, sb, c)
    want = c.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.gemm_fp8(a, sa, b, sb, c)
    c.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, want)


def test_offsets_beyond_32_bits():
    """Rows so far apart that an element's number passes 2^31 (and a byte's 2^32)."""
    far = 2 ** 30
    x = torch.empty(3 * far + 256, dtype=torch.bfloat16, device=DEV).as_strided((4, 256), (far, 1))
    x.copy_(wild(4, 256, 1))
    q = torch.empty(3 * far + 256, dtype=torch.uint8, device=DEV).view(F8).as_strided((4, 256), (far, 1))
    s = scales(2, 4)
    ops.fp8_quantize(x, q, s)
    rq, rs = ref_rows(x)
    assert torch.equal(s, rs) and same(q, rq)
    b, sb = block_of(wild(72, 256, 2))
    c = x[:, :72]  # the same storage
    ops.gemm_fp8(q, s, b, sb, c)
    assert near(c, values_rows(q, s), values_block(b, sb), 256)
    del x, c
    b = torch.empty(2 * far + 300 * 256, dtype=torch.uint8, device=DEV).view(F8).as_strided((3, 72, 256), (far, 256, 1))
    sb = torch.empty(3, 1, 2, device=DEV)
    for e in range(3):
        qe, se = block_of(wild(72, 256, 3 + e))
        b[e].view(torch.uint8).copy_(qe.view(torch.uint8))
        sb[e] = se
    offsets, counts, rows, _ = order(torch.arange(6, device=DEV, dtype=torch.int32).view(6, 1) % 3, 3, 1)
    c = torch.empty(6, 72, device=DEV)
    a, sa = rows_of(wild(6, 256, 9))
    ops.moe_gemm_fp8(a, sa, offsets, counts, b, sb, c, rows=rows)
    for e in range(3):
        assert near(c[2 * e:2 * e + 2], values_rows(a, sa)[rows[2 * e:2 * e + 2].long()], values_block(b[e], sb[e]), 256)


def test_refusals():
    f = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    with pytest.raises(ValueError):
        ops.fp8_quantize(f(4, 64), f(4, 64), f(1, 4))  # codes of another type
    with pytest.raises(ValueError):
        ops.fp8_quantize(f(4, 64), codes(4, 64), f(4, 1))  # scales the other way round
    with pytest.raises(ValueError):
        ops.fp8_quantize(f(64, 4).t(), codes(4, 64), f(1, 4))
    with pytest.raises(RuntimeError):
        ops.fp8_quantize(f(4, 64))  # nothing asked for
    off = torch.zeros(4, 88, dtype=torch.uint8, device=DEV).view(F8)
    with pytest.raises(RuntimeError):
        ops.fp8_quantize(f(4, 64), off[:, :64], f(1, 4))  # rows off a 16-byte boundary
    with pytest.raises(RuntimeError):
        ops.gemm_fp8(off[:, 8:72], f(1, 4), codes(8, 64), f(1, 1), f(4, 8))
    with pytest.raises(ValueError):
        ops.gemm_fp8(codes(4, 64), f(1, 4), codes(8, 65), f(1, 1), f(4, 8))
    with pytest.raises(ValueError):
        ops.gemm_fp8(codes(4, 64), f(1, 4), codes(8, 64), f(1, 1), f(4, 8).half())
    with pytest.raises(ValueError):
        ops.moe_gemm_fp8(codes(4, 64), f(1, 4), f(3).int(), f(2).int(), codes(8, 64).view(1, 8, 64), f(1, 1, 1), f(4, 8))


def test_error_words():
    a, sa = rows_of(wild(20, 512, 1))
    b, sb = block_of(wild(256, 512, 2))
    c = torch.empty(20, 256, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.gemm_fp8(a, sa, b, sb, c, err=err)
    assert int(err) == 0
    ops.gemm_fp8(a, sa, b, sb, c)
    ops.check_errors()
    for bad in (err.long(), torch.zeros(2, dtype=torch.int32, device=DEV), err.cpu(), err.view(())):
        with pytest.raises(ValueError):
            ops.gemm_fp8(a, sa, b, sb, c, err=bad)


def test_first_call_of_a_process_may_be_captured():
    """Loading, attributes and the error word's address are no allocation of the stream's."""
    code = """
import torch
from neuralscript_b200 import ops
f8 = torch.float8_e4m3fn
a, b = torch.ones(20, 512, device="cuda").to(f8), torch.ones(256, 512, device="cuda").to(f8)
sa, sb, c = torch.ones(4, 20, device="cuda"), torch.ones(2, 4, device="cuda"), torch.zeros(20, 256, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ops.gemm_fp8(a, sa, b, sb, c)
g.replay()
ops.check_errors()
assert (c == 512).all()
"""
    import pathlib
    import subprocess
    import sys
    root = pathlib.Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# --------------------------------------------------------------------------
# Blocks that take several tiles in turn: what a tile leaves behind (rings,
# parts of TMEM, staging, shared memory) is the next one's start. Each case
# says how many tiles there are, by the rules of the launches.
# --------------------------------------------------------------------------
SMS = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148


def tiles_of(m_tiles, N, by_rows=False):
    """Width and number of the large products' tiles: the least rounds x (width + 64)."""
    cost = lambda bn: -(-m_tiles * -(-N // bn) // SMS) * (bn + 64)  # noqa: E731
    if by_rows and cost(192) < cost(256) and cost(192) <= cost(128):
        bn = 192
    else:
        bn = 128 if cost(128) < cost(256) else 256
    return bn, m_tiles * -(-N // bn)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K", [(2500, 2184), (5001, 2184), (3000, 2179)])
@pytest.mark.parametrize("gathered", [False, True])
def test_quantize_many_tiles(dtype, M, K, gathered):
    assert up(M, 128) // 128 * (up(K, 128) // 128) > 2 * SMS  # two blocks an SM
    x = wild(M, K, M).to(dtype)
    full, how = x, {}
    if gathered:
        rows = torch.randint(-1, 2 * M, (M,), device=DEV, generator=gen(4), dtype=torch.int32)
        full, how = torch.where((rows >= 0)[:, None], x[rows.long().clamp(min=0) // 2], 0), dict(rows=rows, row_div=2)
    rq, rs = ref_rows(full)
    rqt, rst = ref_rows(full.t())
    for both in ("q", "qt", "both"):
        q, s, qt, st = codes(M, K), scales(up(K, 128) // 128, M), codes(K, M), scales(up(M, 128) // 128, K)
        out = (dict(q=q, s=s) if both != "qt" else {}) | (dict(qt=qt, st=st) if both != "q" else {})
        ops.fp8_quantize(x, **out, **how)
        if both != "qt":
            assert same(q, rq) and torch.equal(s, rs), both
        if both != "q":
            assert same(qt, rqt) and torch.equal(st, rst), both


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K", [(2500, 2184), (5001, 2179)])
@pytest.mark.parametrize("transposed", [False, True])
def test_quantize_block_many_tiles(dtype, M, K, transposed):
    x = wild(M, K, M).to(dtype)
    MB, KB = up(M, 128) // 128, up(K, 128) // 128
    assert MB * KB > 2 * SMS
    q, s, qt, st = codes(M, K), scales(MB, KB), codes(K, M), scales(KB, MB)
    ops.fp8_quantize_block(x, q, s, *((qt, st) if transposed else ()))
    b = torch.nn.functional.pad(x.float(), (0, KB * 128 - K, 0, MB * 128 - M)).view(MB, 128, KB, 128)
    rs = torch.clamp(b.abs().amax((1, 3)) / 448, min=2.0 ** -100)
    rq = (b * (1 / rs)[:, None, :, None]).to(F8).view(MB * 128, KB * 128)[:M, :K]
    assert torch.equal(s, rs) and same(q, rq)
    if transposed:
        assert torch.equal(st, rs.t()) and same(qt, rq.t())


@pytest.mark.parametrize("M,N,K,bn", [(3500, 2800, 300, 192), (5000, 2000, 136, 192), (3000, 3500, 260, 256),
                                      (4000, 4100, 130, 256), (20000, 120, 300, 128)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product_scaled_by_rows_of_many_tiles(M, N, K, bn, out):
    width, tiles = tiles_of(up(M, 128) // 128, N, True)
    assert width == bn and tiles > SMS
    a, sa = rows_of(wild(M, K, 1), 3)
    b, sb = rows_of(wild(N, K, 2), 1)
    c = torch.full((M + 1, N), math.nan, dtype=out, device=DEV)
    ops.gemm_fp8(a, sa, b, sb, c[:M])
    assert near(c[:M], values_rows(a, sa), values_rows(b, sb), K)
    assert c[M].isnan().all()


@pytest.mark.parametrize("M,N,K", [(4096, 2560, 128), (4000, 2570, 100), (4100, 2560, 272)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product_on_pairs(M, N, K, out):
    """From one 256 x 256 tile an SM on: one k-block, a ragged one, and a last pair whose second half is empty."""
    assert up(M, 256) // 256 * (up(N, 256) // 256) >= SMS
    a, sa = rows_of(wild(M, K, 1), 3)
    b, sb = block_of(wild(N, K, 2))
    c = torch.full((M + 1, N), math.nan, dtype=out, device=DEV)
    ops.gemm_fp8(a, sa, b, sb, c[:M])
    assert near(c[:M], values_rows(a, sa), values_block(b, sb), K)
    assert c[M].isnan().all()


@pytest.mark.parametrize("M,N", [(5, 1000), (30, 300), (100, 1000), (40, 72)])
@pytest.mark.parametrize("by_rows", [False, True])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product_split_with_empty_shares(M, N, by_rows, out):
    """17 k-blocks over 8 CTAs in shares of 3: the last two have none."""
    K = 17 * 128 - 5
    rows, slots = (16 if M <= 16 else 32, 2 * SMS) if M <= 32 else (128, SMS)
    assert up(M, rows) // rows * (up(N, 128) // 128) * 8 <= slots
    a, sa = rows_of(wild(M, K, 1))
    b, sb = rows_of(wild(N, K, 2)) if by_rows else block_of(wild(N, K, 2))
    c = torch.full((M + 1, N), math.nan, dtype=out, device=DEV)
    ops.gemm_fp8(a, sa, b, sb, c[:M])
    assert near(c[:M], values_rows(a, sa), values_rows(b, sb) if by_rows else values_block(b, sb), K)
    assert c[M].isnan().all()


@pytest.mark.parametrize("M", [3, 30])
@pytest.mark.parametrize("by_rows", [False, True])
def test_small_product_of_many_tiles(M, by_rows):
    N, K = 40000, 5 * 128 + 16
    assert up(N, 128) // 128 > 2 * SMS
    a, sa = rows_of(wild(M, K, 1))
    b, sb = rows_of(wild(N, K, 2)) if by_rows else block_of(wild(N, K, 2))
    c = torch.full((M + 1, N), math.nan, device=DEV)
    ops.gemm_fp8(a, sa, b, sb, c[:M])
    assert near(c[:M], values_rows(a, sa), values_rows(b, sb) if by_rows else values_block(b, sb), K)
    assert c[M].isnan().all()


def uneven(pairs, E, seed):
    """One choice a token: expert 1 has none, expert 0 one, and the others shares that differ by powers of two."""
    g = gen(seed)
    share = torch.exp2(-torch.arange(E, device=DEV).float() / 2)
    share[:2] = 0
    idx = torch.multinomial(share, pairs, replacement=True, generator=g).to(torch.int32)
    idx[pairs // 2] = 0
    return idx[:, None].contiguous()


@pytest.mark.parametrize("pairs,E,N,K,align,bn", [(8000, 6, 2056, 272, 1, 256), (7000, 6, 2050, 136, 128, 256),
                                                  (19000, 7, 120, 400, 128, 128), (2000, 40, 2100, 200, 1, 0),
                                                  (500, 40, 2104, 272, 1, 0)])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_experts_product_of_many_tiles(pairs, E, N, K, align, bn, gather, out):
    """bn 0: the small kernel, for up to 128 rows an expert."""
    offsets, counts, rows, pos = order(uneven(pairs, E, N), E, align)
    R = rows.numel()
    n = counts.tolist()
    if bn:
        assert R > 128 * E and tiles_of(up(R, 128) // 128, N)[0] == bn
        assert sum(-(-v // 128) for v in n) * -(-N // bn) > SMS
    else:
        wide = 16 if -(-R // E) <= 16 else 32
        assert -(-R // E) <= 128 and sum(-(-v // wide) for v in n) * -(-N // 128) > 2 * SMS
    a, sa = rows_of(wild(pairs if gather else R, K, 1), 2)
    ws = [block_of(wild(N, K, 10 + e)) for e in range(E)]
    b = torch.zeros(E, N, up(K, 16), dtype=torch.uint8, device=DEV)
    b[:, :, :K] = torch.stack([q.view(torch.uint8) for q, _ in ws])
    b, sb = b.view(F8)[:, :, :K], torch.stack([s for _, s in ws])
    c = torch.full((R, N), 7.0, dtype=out, device=DEV)
    ops.moe_gemm_fp8(a, sa, offsets, counts, b, sb, c, rows=rows if gather else None)
    av = values_rows(a, sa)
    written = torch.zeros(R, dtype=torch.bool, device=DEV)
    for e in range(E):
        o = int(offsets[e])
        src = rows[o:o + n[e]].long() if gather else torch.arange(o, o + n[e], device=DEV)
        assert near(c[o:o + n[e]], av[src], values_block(*ws[e]), K), e
        written[o:o + n[e]] = True
    assert (c[~written] == 7).all()


@pytest.mark.parametrize("M,N,E,bn", [(520, 1000, 16, 256), (260, 600, 33, 192), (260, 120, 100, 128), (258, 602, 33, 192)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_experts_weight_gradient_of_many_tiles(M, N, E, bn, out):
    width, tiles = tiles_of(up(M, 128) // 128 * E, N, True)
    assert width == bn and tiles > 2 * SMS
    offsets, counts, rows, pos = order(uneven(6000, E, M), E, 128)
    R = rows.numel()
    x, dz = wild(6000, N, 1), torch.randn(R, M, device=DEV, generator=gen(2))
    xt, sx, gt, sg = codes(N, R), scales(R // 128, N), codes(M, R), scales(R // 128, M)
    ops.fp8_quantize(x, qt=xt, st=sx, rows=rows)
    ops.fp8_quantize(dz, qt=gt, st=sg, rows=rows, row_div=0)
    c = torch.full((E, M, N), math.nan, dtype=out, device=DEV)
    ops.moe_wgrad_fp8(gt, sg, xt, sx, offsets, counts, c)
    gv, xv = values_rows(gt, sg), values_rows(xt, sx)
    for e in range(E):
        o, n = int(offsets[e]), int(counts[e])
        assert near(c[e], gv[:, o:o + n], xv[:, o:o + n], n), e
    assert (c[1] == 0).all()  # no rows


def test_products_on_another_stream_than_the_current_one_before():
    """Inputs made late on a side stream: a launch on any other stream would read what was there before."""
    s = torch.cuda.Stream()
    for M, N, K in ((20, 256, 512), (300, 512, 640)):
        x, w = wild(M, K, 1), wild(N, K, 2)
        a, sa = rows_of(torch.zeros_like(x))
        b, sb = block_of(torch.zeros_like(w))
        c = torch.full((M, N), math.nan, device=DEV)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(20_000_000)
            ops.fp8_quantize(x, a, sa)
            ops.fp8_quantize_block(w, b, sb)
            ops.gemm_fp8(a, sa, b, sb, c)
        s.synchronize()
        assert near(c, values_rows(a, sa), values_block(b, sb), K) and (c != 0).any()
