"""ctypes bindings of the kernel-level C-ABI (include/ns_b200_ops.h) taking
torch CUDA tensors; device memory comes from torch (plumbing only)."""
from __future__ import annotations

import ctypes as C

from . import lib as _core_lib

F32, BF16 = 0, 1
AUTO, SIMT, TENSOR = 0, 1, 2

_sigs = {
    "nsb_op_gemm": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_void_p,
                              C.c_int, C.c_longlong, C.c_int, C.c_float, C.c_void_p, C.c_longlong, C.c_int,
                              C.c_void_p, C.c_longlong, C.c_void_p, C.c_longlong, C.c_int, C.c_void_p, C.c_size_t,
                              C.c_void_p, C.c_void_p]),
    "nsb_op_gemm_workspace_floats": (C.c_size_t, [C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_int, C.c_longlong,
                                                  C.c_int, C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_int]),
    "nsb_op_gemm_uses_tensor_cores": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_int, C.c_longlong,
                                                C.c_int, C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_int]),
    "nsb_op_embedding_fwd": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p,
                                       C.c_void_p]),
    "nsb_op_embedding_bwd_scratch_bytes": (C.c_size_t, [C.c_int, C.c_int]),
    "nsb_op_embedding_bwd": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p,
                                       C.c_void_p]),
    "nsb_op_layernorm_fwd": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]),
    "nsb_op_layernorm_bwd": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p,
                                       C.c_void_p]),
    "nsb_op_attention_fwd": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_longlong,
                                       C.c_void_p, C.c_longlong, C.c_void_p, C.c_void_p]),
    "nsb_op_attention_bwd": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_longlong,
                                       C.c_void_p, C.c_longlong, C.c_void_p, C.c_void_p, C.c_longlong, C.c_void_p,
                                       C.c_longlong, C.c_void_p, C.c_void_p]),
    "nsb_op_cross_entropy": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_float, C.c_void_p,
                                       C.c_void_p, C.c_void_p, C.c_void_p]),
    "nsb_op_reduce_sum": (C.c_int, [C.c_void_p, C.c_int, C.c_float, C.c_void_p, C.c_void_p]),
    "nsb_op_adamw": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_longlong, C.c_longlong,
                               C.c_float, C.c_float, C.c_float, C.c_float, C.c_float, C.c_float, C.c_float,
                               C.c_void_p]),
    "nsb_op_mgs": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_void_p]),
    "nsb_op_moe_route": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p,
                                   C.c_void_p, C.c_void_p, C.c_void_p]),
    "nsb_op_act_fwd": (C.c_int, [C.c_void_p, C.c_size_t, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]),
    "nsb_op_act_bwd": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_size_t, C.c_void_p, C.c_void_p]),
    "nsb_op_moe_topk_route": (C.c_int, [C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_int,
                                        C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_float, C.c_void_p,
                                        C.c_void_p, C.c_void_p]),
    "nsb_op_moe_topk_route_bwd": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_int,
                                            C.c_int, C.c_void_p, C.c_int, C.c_float, C.c_void_p, C.c_void_p,
                                            C.c_longlong, C.c_void_p]),
    "nsb_op_moe_dispatch_rows": (C.c_size_t, [C.c_int, C.c_int, C.c_int, C.c_int]),
    "nsb_op_moe_dispatch": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p,
                                      C.c_void_p, C.c_void_p, C.c_void_p]),
    "nsb_op_moe_combine": (C.c_int, [C.c_void_p, C.c_int, C.c_longlong, C.c_void_p, C.c_void_p, C.c_int, C.c_int,
                                     C.c_int, C.c_void_p, C.c_longlong, C.c_void_p]),
    "nsb_op_moe_combine_rows": (C.c_int, [C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_void_p, C.c_void_p, C.c_int,
                                          C.c_int, C.c_int, C.c_void_p, C.c_longlong, C.c_void_p]),
    "nsb_op_moe_combine_bwd": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_longlong, C.c_longlong, C.c_void_p,
                                         C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p,
                                         C.c_longlong, C.c_void_p, C.c_void_p]),
    "nsb_op_fp8_quantize": (C.c_int, [C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_void_p,
                                      C.c_int] + [C.c_void_p, C.c_longlong] * 4 + [C.c_void_p]),
    "nsb_op_fp8_quantize_rows": (C.c_int, [C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_int,
                                           C.c_void_p, C.c_int] + [C.c_void_p, C.c_longlong] * 4 + [C.c_void_p]),
    "nsb_op_fp8_quantize_block": (C.c_int, [C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_int]
                                  + [C.c_void_p, C.c_longlong] * 4 + [C.c_void_p]),
    "nsb_op_device_error": (C.c_int, [C.POINTER(C.c_int), C.c_void_p]),
    "nsb_op_gemm_fp8": (C.c_int, [C.c_int, C.c_int, C.c_int] + [C.c_void_p, C.c_longlong] * 4
                        + [C.c_int, C.c_void_p, C.c_int, C.c_longlong, C.c_void_p, C.c_void_p]),
    "nsb_op_moe_gemm_fp8": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_longlong, C.c_int,
                                      C.c_void_p, C.c_longlong, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p,
                                      C.c_void_p, C.c_longlong, C.c_longlong, C.c_void_p, C.c_longlong, C.c_longlong,
                                      C.c_void_p, C.c_int, C.c_longlong, C.c_void_p, C.c_void_p]),
    "nsb_op_moe_wgrad_fp8": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int] + [C.c_void_p, C.c_longlong] * 4
                             + [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_longlong, C.c_longlong, C.c_void_p,
                                C.c_void_p]),
}
_bound = None


def L():
    global _bound
    if _bound is None:
        lib = _core_lib()
        for n, (res, args) in _sigs.items():
            f = getattr(lib, n)
            f.restype = res
            f.argtypes = args
        _bound = lib
    return _bound


def p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _check(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} returned {rc}")


def _dt(t):
    import torch
    return BF16 if t.dtype == torch.bfloat16 else F32


def gemm(A, B, M, N, K, lda, a_mn, ldb, b_mn, alpha=1.0, add=None, act=0, c32=None, c16=None, engine=AUTO,
         err=None):
    """C = act(alpha * A.B^T + add); see include/ns_b200_ops.h for layouts."""
    import torch
    ws_n = L().nsb_op_gemm_workspace_floats(M, N, K, p(A), _dt(A), lda, a_mn, p(B), _dt(B), ldb, b_mn, engine)
    ws = torch.empty(max(ws_n, 1), dtype=torch.float32, device=A.device) if ws_n else None
    ld32 = c32.stride(0) if c32 is not None else 0
    ld16 = c16.stride(0) if c16 is not None else 0
    ldadd = add.stride(0) if add is not None else 0
    rc = L().nsb_op_gemm(M, N, K, p(A), _dt(A), lda, a_mn, p(B), _dt(B), ldb, b_mn, alpha, p(add), ldadd, act,
                         p(c32), ld32, p(c16), ld16, engine, p(ws), ws_n, p(err), _stream())
    _check(rc, "nsb_op_gemm")


def uses_tensor_cores(A, B, M, N, K, lda, a_mn, ldb, b_mn, engine=AUTO) -> bool:
    return bool(L().nsb_op_gemm_uses_tensor_cores(M, N, K, p(A), _dt(A), lda, a_mn, p(B), _dt(B), ldb, b_mn, engine))


def embedding_fwd(W, ids, out32=None, out16=None):
    V, D = W.shape
    _check(L().nsb_op_embedding_fwd(p(W), p(ids), ids.numel(), V, D, p(out32), p(out16), _stream()), "embedding_fwd")


def embedding_bwd(dout, ids, V, dW):
    import torch
    M, D = dout.shape
    n = L().nsb_op_embedding_bwd_scratch_bytes(M, V)
    scratch = torch.empty(n, dtype=torch.uint8, device=dout.device)
    _check(L().nsb_op_embedding_bwd(p(dout), p(ids), M, V, D, p(dW), p(scratch), _stream()), "embedding_bwd")


def layernorm_fwd(x, out32=None, out16=None):
    M, D = x.shape
    _check(L().nsb_op_layernorm_fwd(p(x), M, D, p(out32), p(out16), _stream()), "layernorm_fwd")


def layernorm_bwd(dy, x, add=None, dx32=None, dx16=None):
    M, D = x.shape
    _check(L().nsb_op_layernorm_bwd(p(dy), p(x), p(add), M, D, p(dx32), p(dx16), _stream()), "layernorm_bwd")


def attention_fwd(B, S, H, D, qkv, ctx, lse):
    _check(L().nsb_op_attention_fwd(B, S, H, D, _dt(qkv), p(qkv), qkv.stride(0), p(ctx), ctx.stride(0), p(lse),
                                    _stream()), "attention_fwd")


def attention_bwd(B, S, H, D, qkv, ctx, lse, dctx, dqkv, dvec):
    _check(L().nsb_op_attention_bwd(B, S, H, D, _dt(qkv), p(qkv), qkv.stride(0), p(ctx), ctx.stride(0), p(lse),
                                    p(dctx), dctx.stride(0), p(dqkv), dqkv.stride(0), p(dvec), _stream()),
           "attention_bwd")


def cross_entropy(logits, labels=None, targets=None, denom=None, row_loss=None, d32=None, d16=None):
    M, Cc = logits.shape
    _check(L().nsb_op_cross_entropy(p(logits), p(labels), p(targets), M, Cc, float(M if denom is None else denom),
                                    p(row_loss), p(d32), p(d16), _stream()), "cross_entropy")


def reduce_sum(x, scale, out):
    _check(L().nsb_op_reduce_sum(p(x), x.numel(), scale, p(out), _stream()), "reduce_sum")


def adamw(w, g, m, v, t, lr, beta1=0.9, beta2=0.999, omb1=0.1, omb2=0.001, eps=1e-8, decay=0.01):
    _check(L().nsb_op_adamw(p(w), p(g), p(m), p(v), w.numel(), t, lr, beta1, beta2, omb1, omb2, eps, decay,
                            _stream()), "adamw")


def mgs(G):
    r, c = G.shape
    _check(L().nsb_op_mgs(p(G), r, c, _stream()), "mgs")


def act_fwd(x, act, out32):
    _check(L().nsb_op_act_fwd(p(x), x.numel(), act, p(out32), None, _stream()), "act_fwd")


def act_bwd(dy, z, act, out32):
    _check(L().nsb_op_act_bwd(p(dy), p(z), act, dy.numel(), p(out32), _stream()), "act_bwd")


def moe_route(x, Wg, active, best, pb, probs=None):
    M, D = x.shape
    E = Wg.shape[1]
    _check(L().nsb_op_moe_route(p(x), p(Wg), p(active), M, D, E, p(best), p(pb), p(probs), _stream()), "moe_route")


# ---------------------------------------------------------------------------
# Mixture of experts with k experts a token, and 8-bit (e4m3) products with a
# scale for each block of 128. Tensors that do not fit raise ValueError before
# anything is launched; see include/ns_b200_ops.h for the definitions.
# ---------------------------------------------------------------------------
_SCORE = {"softmax": 0, "sigmoid": 1}
_f32 = _bf16 = _i32 = _u8 = _f8 = _stream_of = _device = None


def _torch():
    """torch's names that every call below needs, looked up once (a decode step's kernels take a few microseconds)."""
    global _f32, _bf16, _i32, _u8, _f8, _stream_of, _device
    import torch
    lib = L()  # raises where the library is missing, in this call and in the next
    _stream_of, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
    _bf16, _i32, _u8, _f8 = torch.bfloat16, torch.int32, torch.uint8, torch.float8_e4m3fn
    _f32 = torch.float32  # last: where it is set, other threads find all the rest
    return lib


def _refuse(t, what, dtype, shape):
    if dtype is not None and t.dtype is not dtype:
        raise ValueError(f"{what}: {t.dtype} where {dtype} is wanted")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: shape {tuple(t.shape)} where {tuple(shape)} is wanted")
    if t.get_device() != _device():
        raise ValueError(f"{what}: on {t.device}, but the kernels run on the current CUDA device, {_device()}")
    raise ValueError(f"{what}: strides {t.stride()} are not those of contiguous rows (or of a dense tensor where one is "
                     "wanted)")


def _dense(d, t, what, dtype, shape):
    """Address of a tensor of this dtype and shape without gaps, on device d."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != d or not t.is_contiguous():
        _refuse(t, what, dtype, shape)
    return t.data_ptr()


def _rows(d, t, what, dtype, rows, cols):
    """Address and leading dimension of a matrix of this dtype and shape, on device d, whose rows are
    contiguous. (torch does not look at the stride of a single row; the kernels do.)"""
    if t.dtype is not dtype or t.shape != (rows, cols) or t.get_device() != d:
        _refuse(t, what, dtype, (rows, cols))
    ld, one = t.stride()
    if one != 1 and cols > 1:
        _refuse(t, what, dtype, (rows, cols))
    return t.data_ptr(), ld if rows > 1 else max(ld, cols)


def _float(d, t, what, rows, cols):
    """As _rows, fp32 or bf16: address, type code and leading dimension."""
    dt = t.dtype
    if dt is not _f32 and dt is not _bf16:
        raise ValueError(f"{what}: {dt} where float32 or bfloat16 is wanted")
    at, ld = _rows(d, t, what, dt, rows, cols)
    return at, F32 if dt is _f32 else BF16, ld


def _codes(d, t, what, rows, cols):
    """As _rows for codes, whose rows start on 16-byte boundaries."""
    at, ld = _rows(d, t, what, _f8, rows, cols)
    return at, ld if rows > 1 else -(-cols // 16) * 16


def _stack(d, t, what, dtype, n, rows, cols):
    """As _rows for n matrices: address, leading dimension and the stride from one to the next."""
    if t.dtype is not dtype or t.shape != (n, rows, cols) or t.get_device() != d:
        _refuse(t, what, dtype, (n, rows, cols))
    apart, ld, one = t.stride()
    if one != 1 and cols > 1:
        _refuse(t, what, dtype, (n, rows, cols))
    return t.data_ptr(), ld if rows > 1 else max(ld, -(-cols // 16) * 16 if dtype is _f8 else cols), apart


def moe_topk_route(logits, idx, w, score="softmax", bias=None, active=None, groups=1, topk_groups=1, renorm=True,
                   scale=1.0):
    """idx, w [M, k] (int32, float32) <- the k experts of each row of logits [M, E] and their weights."""
    lib = _bound if _f32 else _torch()
    d = _device()
    M, E = logits.shape
    k = idx.shape[1]
    rc = lib.nsb_op_moe_topk_route(
        *_float(d, logits, "logits", M, E), M, E, k, _SCORE[score],
        None if bias is None else _dense(d, bias, "bias", _f32, (E,)),
        None if active is None else _dense(d, active, "active", _u8, (E,)), groups, topk_groups, renorm, scale,
        _dense(d, idx, "idx", _i32, (M, k)), _dense(d, w, "w", _f32, (M, k)), _stream_of(d))
    if rc:
        _check(rc, "nsb_op_moe_topk_route")


def moe_topk_route_bwd(dw, logits, idx, dlogits, score="softmax", active=None, renorm=True, scale=1.0):
    """dlogits [M, E] (the logits' type) <- the gradient of moe_topk_route's w."""
    lib = _bound if _f32 else _torch()
    d = _device()
    M, E = logits.shape
    k = idx.shape[1]
    rc = lib.nsb_op_moe_topk_route_bwd(
        _dense(d, dw, "dw", _f32, (M, k)), *_float(d, logits, "logits", M, E), M, E, k, _SCORE[score],
        None if active is None else _dense(d, active, "active", _u8, (E,)), renorm, scale,
        _dense(d, idx, "idx", _i32, (M, k)), *_rows(d, dlogits, "dlogits", logits.dtype, M, E), _stream_of(d))
    if rc:
        _check(rc, "nsb_op_moe_topk_route_bwd")


def moe_dispatch_rows(M, k, E, align=1) -> int:
    """Rows that moe_dispatch orders M * k pairs into at most."""
    return L().nsb_op_moe_dispatch_rows(M, k, E, align)


def moe_dispatch(idx, E, offsets, counts, rows, pos, align=1):
    """offsets [E + 1], counts [E], rows [moe_dispatch_rows(...)], pos [M, k] (int32) <- the pairs of idx by expert."""
    lib = _bound if _f32 else _torch()
    d = _device()
    M, k = idx.shape
    rc = lib.nsb_op_moe_dispatch(
        _dense(d, idx, "idx", _i32, (M, k)), M, k, E, align, _dense(d, offsets, "offsets", _i32, (E + 1,)),
        _dense(d, counts, "counts", _i32, (E,)),
        _dense(d, rows, "rows", _i32, (lib.nsb_op_moe_dispatch_rows(M, k, E, align),)),
        _dense(d, pos, "pos", _i32, (M, k)), _stream_of(d))
    if rc:
        _check(rc, "nsb_op_moe_dispatch")


def moe_combine(o, pos, y, w=None):
    """y [M, D] <- sum over j of w[:, j] * o[pos[:, j]] (w None: 1). Negative entries of pos are left out, and so are
    those past o's rows, which check_errors raises."""
    lib = _bound if _f32 else _torch()
    d = _device()
    M, k = pos.shape
    R, D = o.shape
    rc = lib.nsb_op_moe_combine_rows(
        *_float(d, o, "o", R, D), R, _dense(d, pos, "pos", _i32, (M, k)),
        None if w is None else _dense(d, w, "w", _f32, (M, k)), M, k, D, *_rows(d, y, "y", o.dtype, M, D),
        _stream_of(d))
    if rc:
        _check(rc, "nsb_op_moe_combine_rows")


def moe_combine_bwd(dy, o, rows, pos, w, do, dw=None):
    """do [R, D], dw [M, k] <- the gradients of moe_combine's o and w (dw None: do alone; o may be None then)."""
    lib = _bound if _f32 else _torch()
    d = _device()
    M, k = pos.shape
    D = dy.shape[1]
    R = rows.shape[0]
    if dw is not None and o is None:
        raise ValueError("dw needs o")
    at, dt, ld = _float(d, dy, "dy", M, D)
    o_at, o_ld = (None, 0) if o is None else _rows(d, o, "o", dy.dtype, R, D)
    rc = lib.nsb_op_moe_combine_bwd(
        at, o_at, dt, ld, o_ld, _dense(d, rows, "rows", _i32, (R,)), _dense(d, pos, "pos", _i32, (M, k)),
        None if w is None else _dense(d, w, "w", _f32, (M, k)), M, k, R, D, *_rows(d, do, "do", dy.dtype, R, D),
        None if dw is None else _dense(d, dw, "dw", _f32, (M, k)), _stream_of(d))
    if rc:
        _check(rc, "nsb_op_moe_combine_bwd")


def fp8_ld(n) -> int:
    """Leading dimension of n codes a row: rows start on 16-byte boundaries."""
    return -(-n // 16) * 16


_NOTHING = (None, 0, None, 0)


def fp8_quantize(x, q=None, s=None, qt=None, st=None, act=0, rows=None, row_div=1):
    """q [M, K] with s [ceil(K / 128), M], and / or qt [K, M] with st [ceil(M / 128), K] <- codes and scales of act(x).

    q, qt: float8_e4m3fn with rows on 16-byte boundaries. rows [M] (int32) gathers rows[r] / row_div of x first
    (row_div 0: only puts zeros where rows is negative); an entry past x's rows gives zeros, and check_errors raises
    it."""
    lib = _bound if _f32 else _torch()
    d = _device()
    n, K = x.shape
    M = n if rows is None else rows.shape[0]
    if rows is not None and row_div == 0 and n < M:
        raise ValueError(f"x: {n} rows where {M} are wanted")
    rc = lib.nsb_op_fp8_quantize_rows(
        *_float(d, x, "x", n, K), n, M, K, act, None if rows is None else _dense(d, rows, "rows", _i32, (M,)), row_div,
        *(_NOTHING if q is None else _codes(d, q, "q", M, K) + _rows(d, s, "s", _f32, -(-K // 128), M)),
        *(_NOTHING if qt is None else _codes(d, qt, "qt", K, M) + _rows(d, st, "st", _f32, -(-M // 128), K)),
        _stream_of(d))
    if rc:
        _check(rc, "nsb_op_fp8_quantize_rows")


def fp8_quantize_block(x, q=None, s=None, qt=None, st=None):
    """q [M, K] with s [ceil(M / 128), ceil(K / 128)], and / or their transposes qt, st <- codes and scales of x."""
    lib = _bound if _f32 else _torch()
    d = _device()
    M, K = x.shape
    mb, kb = -(-M // 128), -(-K // 128)
    rc = lib.nsb_op_fp8_quantize_block(
        *_float(d, x, "x", M, K), M, K,
        *(_NOTHING if q is None else _codes(d, q, "q", M, K) + _rows(d, s, "s", _f32, mb, kb)),
        *(_NOTHING if qt is None else _codes(d, qt, "qt", K, M) + _rows(d, st, "st", _f32, kb, mb)), _stream_of(d))
    if rc:
        _check(rc, "nsb_op_fp8_quantize_block")


def _word(d, err):
    """Address of a caller's error word; None for the device's own."""
    return None if err is None else _dense(d, err, "err", _i32, (1,))


def check_errors():
    """Waits for the current stream and raises RuntimeError where since the last call a product without an `err` of
    its own gave up a bounded wait (its result is not to be used), or an index was past its tensor's rows."""
    lib = _bound if _f32 else _torch()
    d = _device()
    code = C.c_int(0)
    _check(lib.nsb_op_device_error(C.byref(code), _stream_of(d)), "nsb_op_device_error")
    if code.value:
        why = "an index past its tensor's rows" if code.value == 111 else "a product's wait ran out"
        raise RuntimeError(f"device error {code.value} since the last check: {why}")


def gemm_fp8(a, sa, b, sb, c, err=None):
    """c [M, N] (fp32 or bf16) <- A B^T of codes a [M, K] with row scales sa, b [N, K] with scales sb: of rows
    [ceil(K / 128), N], or of blocks [ceil(N / 128), ceil(K / 128)] (both have that shape only where they are the same:
    N = 1 and K at most 128). err (one int32): receives the code of a wait that ran out, in place of the word that
    check_errors reads."""
    lib = _bound if _f32 else _torch()
    d = _device()
    M, K = a.shape
    N = b.shape[0]
    kb = -(-K // 128)
    by_rows = sb.shape == (kb, N)
    at, dt, ld = _float(d, c, "c", M, N)
    rc = lib.nsb_op_gemm_fp8(
        M, N, K, *_codes(d, a, "a", M, K), *_rows(d, sa, "sa", _f32, kb, M), *_codes(d, b, "b", N, K),
        *(_rows(d, sb, "sb", _f32, kb, N) if by_rows else _rows(d, sb, "sb", _f32, -(-N // 128), kb)), by_rows,
        at, dt, ld, _word(d, err), _stream_of(d))
    if rc:
        _check(rc, "nsb_op_gemm_fp8")


def moe_gemm_fp8(a, sa, offsets, counts, b, sb, c, rows=None, row_div=1, err=None):
    """Rows of c [R, N] of each expert e <- those of A times B[e]^T: a [R, K] (with rows [R]: [any, K], of which
    row r takes rows[r] / row_div) with row scales sa, b [E, N, K] with block scales sb."""
    lib = _bound if _f32 else _torch()
    d = _device()
    n, K = a.shape
    E, N, _ = b.shape
    R = c.shape[0]
    kb = -(-K // 128)
    at, dt, ld = _float(d, c, "c", R, N)
    rc = lib.nsb_op_moe_gemm_fp8(
        R, E, N, K, *_codes(d, a, "a", n if rows is not None else R, K), n, *_rows(d, sa, "sa", _f32, kb, n),
        None if rows is None else _dense(d, rows, "rows", _i32, (R,)), row_div,
        _dense(d, offsets, "offsets", _i32, (E + 1,)), _dense(d, counts, "counts", _i32, (E,)),
        *_stack(d, b, "b", _f8, E, N, K), *_stack(d, sb, "sb", _f32, E, -(-N // 128), kb), at, dt, ld,
        _word(d, err), _stream_of(d))
    if rc:
        _check(rc, "nsb_op_moe_gemm_fp8")


def moe_wgrad_fp8(a, sa, b, sb, offsets, counts, c, err=None):
    """c [E, M, N] <- for each expert the sum over its columns of a [M, R] and b [N, R] (row scales sa, sb)."""
    lib = _bound if _f32 else _torch()
    d = _device()
    M, R = a.shape
    N = b.shape[0]
    E = c.shape[0]
    rb = -(-R // 128)
    if c.dtype is not _f32 and c.dtype is not _bf16:
        raise ValueError(f"c: {c.dtype} where float32 or bfloat16 is wanted")
    at, ld, apart = _stack(d, c, "c", c.dtype, E, M, N)
    rc = lib.nsb_op_moe_wgrad_fp8(
        M, N, R, E, *_codes(d, a, "a", M, R), *_rows(d, sa, "sa", _f32, rb, M), *_codes(d, b, "b", N, R),
        *_rows(d, sb, "sb", _f32, rb, N), _dense(d, offsets, "offsets", _i32, (E + 1,)),
        _dense(d, counts, "counts", _i32, (E,)), at, F32 if c.dtype is _f32 else BF16, ld, apart,
        _word(d, err), _stream_of(d))
    if rc:
        _check(rc, "nsb_op_moe_wgrad_fp8")
