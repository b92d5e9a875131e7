"""Argument checks of the top-k mixture-of-experts and 8-bit operators at the
C entries: every refusal comes before anything is launched, so none needs a
GPU."""

import pytest

from neuralscript_b200 import ops

X = 0x10000  # an address that is never read


def rc(name, *args):
    return getattr(ops.L(), name)(*args, None)


def route(**kw):
    a = dict(logits=X, dtype=0, ld=16, M=4, E=16, k=2, score=0, bias=None, active=None, groups=1, topk_groups=1, renorm=1,
             scale=1.0, idx=X, w=X) | kw
    return rc("nsb_op_moe_topk_route", *a.values())


@pytest.mark.parametrize("bad", [dict(k=0), dict(k=17), dict(E=0, ld=0), dict(E=1025, ld=1025), dict(k=33, E=64, ld=64),
                                 dict(M=-1), dict(ld=15), dict(dtype=2), dict(score=2), dict(groups=3), dict(groups=0),
                                 dict(groups=16), dict(groups=4, topk_groups=5), dict(topk_groups=0), dict(logits=None),
                                 dict(idx=None), dict(w=None)])
def test_route_refuses(bad):
    assert route(**bad) == -1


def test_route_of_no_tokens():
    assert route(M=0) == 0


def test_route_gradient_refuses():
    ok = [X, X, 0, 16, 4, 16, 2, 0, None, 1, 1.0, X, X, 16]
    for at, v in ((0, None), (1, None), (2, 5), (3, 8), (6, 0), (7, 9), (11, None), (12, None), (13, 15)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_moe_topk_route_bwd", *a) == -1, at


def test_dispatch_refuses():
    ok = [X, 4, 2, 8, 128, X, X, X, X]
    for at, v in ((0, None), (1, -1), (2, 0), (2, 33), (3, 0), (3, 1025), (4, 0), (5, None), (6, None), (7, None), (8, None)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_moe_dispatch", *a) == -1, at
    assert rc("nsb_op_moe_dispatch", X, 2 ** 30, 2, 8, 128, X, X, X, X) == -2


@pytest.mark.parametrize("M,k,E,align,rows", [(3, 2, 8, 1, 6), (3, 2, 8, 128, 768), (100, 2, 8, 128, 1280),
                                              (0, 2, 8, 128, 0), (1, 1, 8, 16, 16)])
def test_dispatch_rows(M, k, E, align, rows):
    got = ops.moe_dispatch_rows(M, k, E, align)
    assert got % align == 0 and got >= M * k
    assert got == rows


def test_combine_refuses():
    ok = [X, 0, 64, X, X, 4, 2, 64, X, 64]
    for at, v in ((0, None), (1, 3), (2, 63), (3, None), (5, -1), (6, 0), (6, 33), (7, 0), (8, None), (9, 63)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_moe_combine", *a) == -1, at
    ok = [X, X, 0, 64, 64, X, X, X, 4, 2, 8, 64, X, 64, X]
    for at, v in ((0, None), (1, None), (2, 3), (3, 63), (4, 63), (5, None), (6, None), (8, -1), (9, 0), (10, -1), (11, 0),
                  (12, None), (13, 63)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_moe_combine_bwd", *a) == -1, at


def test_quantize_refuses():
    ok = [X, 0, 64, 4, 64, 0, None, 1, X, 64, X, 4, X, 16, X, 64]
    for at, v in ((0, None), (1, 2), (2, 63), (3, -1), (4, 0), (5, 8), (5, -1), (8, X + 8), (9, 48), (9, 72), (10, None),
                  (11, 3), (12, X + 1), (13, 8), (14, None), (15, 63)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_fp8_quantize", *a) == -1, at
    a = list(ok)
    a[6], a[7] = X, -1
    assert rc("nsb_op_fp8_quantize", *a) == -1
    a = list(ok)
    a[8] = a[12] = None
    assert rc("nsb_op_fp8_quantize", *a) == -1
    ok = [X, 0, 300, 200, 300, X, 304, X, 3, X, 208, X, 2]
    for at, v in ((0, None), (1, 7), (2, 299), (4, 0), (6, 288), (7, None), (8, 2), (10, 192), (11, None), (12, 1)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_fp8_quantize_block", *a) == -1, at


def test_products_refuse():
    ok = [4, 200, 300, X, 304, X, 4, X, 304, X, 3, 0, X, 0, 200, None]
    for at, v in ((0, -1), (1, -1), (2, -1), (3, None), (3, X + 4), (4, 288), (4, 308), (5, None), (6, 3), (7, None),
                  (7, X + 8), (8, 300), (9, None), (10, 2), (12, None), (13, 2), (14, 199)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_gemm_fp8", *a) == -1, at
    a = list(ok)
    a[11], a[10] = 1, 199  # row scales
    assert rc("nsb_op_gemm_fp8", *a) == -1
    ok = [8, 4, 200, 300, X, 304, 8, X, 8, None, 1, X, X, X, 304, 304 * 200, X, 3, 6, X, 0, 200, None]
    for at, v in ((1, 0), (4, None), (5, 300), (6, 7), (8, 7), (11, None), (12, None), (13, None), (15, 8), (17, 2), (19, None),
                  (21, 199)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_moe_gemm_fp8", *a) == -1, at
    a = list(ok)
    a[1] = 1025
    assert rc("nsb_op_moe_gemm_fp8", *a) == -2
    a = list(ok)
    a[9], a[10] = X, 0
    assert rc("nsb_op_moe_gemm_fp8", *a) == -1
    ok = [64, 48, 256, 4, X, 256, X, 64, X, 256, X, 48, X, X, X, 0, 48, 64 * 48, None]
    for at, v in ((3, 0), (4, None), (5, 240), (7, 63), (8, None), (11, 47), (12, None), (13, None), (14, None), (16, 47)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_moe_wgrad_fp8", *a) == -1, at


def test_products_of_nothing():
    assert rc("nsb_op_gemm_fp8", 0, 200, 300, X, 304, X, 4, X, 304, X, 3, 0, X, 0, 200, None) == 0
    assert rc("nsb_op_gemm_fp8", 4, 0, 300, X, 304, X, 4, X, 304, X, 3, 0, X, 0, 200, None) == 0


def test_nothing_has_no_address():
    """A tensor without elements has the address 0: no refusal."""
    assert route(M=0, logits=None, idx=None, w=None) == 0
    assert rc("nsb_op_moe_topk_route_bwd", None, None, 0, 16, 0, 16, 2, 0, None, 1, 1.0, None, None, 16) == 0
    assert rc("nsb_op_moe_combine", None, 0, 64, None, None, 0, 2, 64, None, 64) == 0
    assert rc("nsb_op_moe_combine_bwd", None, None, 0, 64, 64, None, None, None, 0, 2, 0, 64, None, 64, None) == 0
    assert rc("nsb_op_fp8_quantize", None, 0, 64, 0, 64, 0, None, 1, None, 64, None, 0, None, 0, None, 64) == 0
    assert rc("nsb_op_fp8_quantize_block", None, 0, 64, 0, 64, None, 64, None, 1, None, 0, None, 0) == 0


def test_device_error_refuses():
    assert ops.L().nsb_op_device_error(None, None) == -1


def test_check_errors_raises(monkeypatch):
    """A code in the device's word is raised, and a failure to read it."""
    class Lib:
        code, rc = 0, 0

        def nsb_op_device_error(self, code, stream):
            code._obj.value = self.code
            return self.rc

    lib = Lib()
    monkeypatch.setattr(ops, "_bound", lib)
    monkeypatch.setattr(ops, "_f32", object())
    monkeypatch.setattr(ops, "_device", lambda: 0)
    monkeypatch.setattr(ops, "_stream_of", lambda d: 0)
    ops.check_errors()
    lib.code = 102
    with pytest.raises(RuntimeError, match="102"):
        ops.check_errors()
    lib.code, lib.rc = 0, -5
    with pytest.raises(RuntimeError, match="-5"):
        ops.check_errors()


def test_bounded_entries_refuse():
    ok = [X, 0, 64, 8, X, X, 4, 2, 64, X, 64]
    for at, v in ((0, None), (1, 3), (2, 63), (3, -1), (4, None), (6, -1), (7, 0), (7, 33), (8, 0), (9, None), (10, 63)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_moe_combine_rows", *a) == -1, at
    ok = [X, 0, 64, 4, 4, 64, 0, X, 0, X, 64, X, 4, X, 16, X, 64]
    for at, v in ((0, None), (3, 3), (3, -1), (8, -1), (9, X + 8), (10, 48), (11, None)):
        a = list(ok)
        a[at] = v
        assert rc("nsb_op_fp8_quantize_rows", *a) == -1, at
    a = list(ok)
    a[3], a[7], a[8] = 3, None, 1  # no list: the rows themselves
    assert rc("nsb_op_fp8_quantize_rows", *a) == -1


def test_missing_library_is_reported_by_every_call(monkeypatch):
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(ops, "_bound", None)
    monkeypatch.setattr(ops, "_f32", None)

    def missing():
        raise RuntimeError("libns_b200.so missing")

    monkeypatch.setattr(ops, "_core_lib", missing)
    idx, w = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="missing"):
            ops.moe_topk_route(torch.zeros(4, 8), idx, w)
        with pytest.raises(RuntimeError, match="missing"):
            ops.check_errors()


def test_names_are_published_behind_the_library(monkeypatch):
    """A thread that comes while another one loads the library sees all names or none."""
    monkeypatch.setattr(ops, "_f32", None)
    monkeypatch.setattr(ops, "_f8", None)
    seen = []
    load = ops.L
    monkeypatch.setattr(ops, "L", lambda: (seen.append(ops._f32), load())[1])
    assert ops._torch() is load() and seen == [None] and ops._f8 is not None


class Far:
    """What the entries ask of a tensor, of one that no process here could hold."""

    def __init__(self, shape, dtype, device=0):
        self.shape, self.dtype, self.device = tuple(shape), dtype, f"cuda:{device}"
        self.at = device

    def get_device(self):
        return self.at

    is_cuda = True

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return X

    def stride(self):
        out = [1]
        for n in reversed(self.shape[1:]):
            out.insert(0, out[0] * n)
        return tuple(out)


def calls():
    """Every entry with shapes and types of all its tensors: (entry, arguments, named arguments)."""
    torch = pytest.importorskip("torch")
    f, i, q, u, h = torch.float32, torch.int32, torch.float8_e4m3fn, torch.uint8, torch.bfloat16
    o = ops
    yield o.moe_topk_route, [((4, 16), f), ((4, 2), i), ((4, 2), f)], dict(bias=((16,), f), active=((16,), u))
    yield o.moe_topk_route_bwd, [((4, 2), f), ((4, 16), h), ((4, 2), i), ((4, 16), h)], dict(active=((16,), u))
    yield o.moe_dispatch, [((4, 2), i), 8, ((9,), i), ((8,), i), ((8,), i), ((4, 2), i)], {}
    yield o.moe_combine, [((8, 64), f), ((4, 2), i), ((4, 64), f)], dict(w=((4, 2), f))
    yield o.moe_combine_bwd, [((4, 64), h), ((8, 64), h), ((8,), i), ((4, 2), i), ((4, 2), f), ((8, 64), h)], dict(dw=((4, 2), f))
    yield o.fp8_quantize, [((8, 64), f)], dict(q=((4, 64), q), s=((1, 4), f), qt=((64, 4), q), st=((1, 64), f), rows=((4,), i))
    yield o.fp8_quantize_block, [((4, 64), f)], dict(q=((4, 64), q), s=((1, 1), f), qt=((64, 4), q), st=((1, 1), f))
    yield o.gemm_fp8, [((4, 64), q), ((1, 4), f), ((8, 64), q), ((1, 8), f), ((4, 8), h)], dict(err=((1,), i))
    yield (o.moe_gemm_fp8, [((4, 64), q), ((1, 4), f), ((3,), i), ((2,), i), ((2, 8, 64), q), ((2, 1, 1), f), ((6, 8), f)],
           dict(rows=((6,), i), err=((1,), i)))
    yield (o.moe_wgrad_fp8, [((8, 256), q), ((2, 8), f), ((16, 256), q), ((2, 16), f), ((3,), i), ((2,), i), ((2, 8, 16), f)],
           dict(err=((1,), i)))


def test_every_tensor_is_on_the_current_device(monkeypatch):
    class Lib:
        def nsb_op_moe_dispatch_rows(self, M, k, E, align):
            return M * k

        def __getattr__(self, name):
            return lambda *a: 0

    ops._torch()
    monkeypatch.setattr(ops, "_bound", Lib())
    monkeypatch.setattr(ops, "_device", lambda: 0)
    monkeypatch.setattr(ops, "_stream_of", lambda d: 0)
    for f, args, named in calls():
        every = list(enumerate(args)) + list(named.items())

        def call(elsewhere):
            make = lambda at, a: Far(*a, 1 if at == elsewhere else 0) if isinstance(a, tuple) else a  # noqa: E731
            f(*(make(n, a) for n, a in enumerate(args)), **{n: make(n, a) for n, a in named.items()})

        call(None)
        for at, a in every:
            if isinstance(a, tuple):
                with pytest.raises(ValueError, match="cuda:1"):
                    call(at)
