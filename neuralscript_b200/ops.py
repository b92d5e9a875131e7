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
    "nsb_op_moe_combine_bwd": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_longlong, C.c_longlong, C.c_void_p,
                                         C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p,
                                         C.c_longlong, C.c_void_p, C.c_void_p]),
    "nsb_op_fp8_quantize": (C.c_int, [C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_void_p,
                                      C.c_int] + [C.c_void_p, C.c_longlong] * 4 + [C.c_void_p]),
    "nsb_op_fp8_quantize_block": (C.c_int, [C.c_void_p, C.c_int, C.c_longlong, C.c_int, C.c_int]
                                  + [C.c_void_p, C.c_longlong] * 4 + [C.c_void_p]),
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


def _is(t, what, dtype, *shape):
    """t is a CUDA tensor of the dtype and shape (None: any size) whose last dimension is contiguous."""
    if t.dtype is not dtype:
        raise ValueError(f"{what}: {t.dtype} where {dtype} is wanted")
    if t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise ValueError(f"{what}: shape {tuple(t.shape)} where {shape} is wanted")
    if not t.is_cuda:
        raise ValueError(f"{what}: not on a CUDA device")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: its last dimension has stride {t.stride(-1)}")
    return t.data_ptr()


def _dense(t, what, dtype, *shape):
    """As _is, without gaps between rows."""
    at = _is(t, what, dtype, *shape)
    if not t.is_contiguous():
        raise ValueError(f"{what}: not contiguous")
    return at


def _float(t, what, *shape):
    """As _is, fp32 or bf16; its address, type code and leading dimension."""
    import torch
    if t.dtype is not torch.float32 and t.dtype is not torch.bfloat16:
        raise ValueError(f"{what}: {t.dtype} where float32 or bfloat16 is wanted")
    return _is(t, what, t.dtype, *shape), F32 if t.dtype is torch.float32 else BF16, _ld(t)


def _ld(t, dim=0):
    """Stride of a dimension (that of a single row is not looked at by torch, but is by the kernels)."""
    return max(t.stride(dim), t.shape[-1] if t.shape[dim] < 2 else 0)


def _ld16(t, dim=0):
    """As _ld for codes: a single row has no stride of its own."""
    return t.stride(dim) if t.shape[dim] > 1 else -(-t.shape[-1] // 16) * 16


def _run(name, *args):
    import torch
    rc = getattr(L(), name)(*args, torch.cuda.current_stream().cuda_stream)
    if rc != 0:
        raise RuntimeError(f"{name} returned {rc}")


def moe_topk_route(logits, idx, w, score="softmax", bias=None, active=None, groups=1, topk_groups=1, renorm=True,
                   scale=1.0):
    """idx, w [M, k] (int32, float32) <- the k experts of each row of logits [M, E] and their weights."""
    import torch
    M, E = logits.shape
    k = idx.shape[1]
    at, dt, ld = _float(logits, "logits", M, E)
    _run("nsb_op_moe_topk_route", at, dt, ld, M, E, k, _SCORE[score],
         _dense(bias, "bias", torch.float32, E) if bias is not None else None,
         _dense(active, "active", torch.uint8, E) if active is not None else None, groups, topk_groups, int(renorm),
         scale, _dense(idx, "idx", torch.int32, M, k), _dense(w, "w", torch.float32, M, k))


def moe_topk_route_bwd(dw, logits, idx, dlogits, score="softmax", active=None, renorm=True, scale=1.0):
    """dlogits [M, E] (the logits' type) <- the gradient of moe_topk_route's w."""
    import torch
    M, E = logits.shape
    k = idx.shape[1]
    at, dt, ld = _float(logits, "logits", M, E)
    _run("nsb_op_moe_topk_route_bwd", _dense(dw, "dw", torch.float32, M, k), at, dt, ld, M, E, k, _SCORE[score],
         _dense(active, "active", torch.uint8, E) if active is not None else None, int(renorm), scale,
         _dense(idx, "idx", torch.int32, M, k), _is(dlogits, "dlogits", logits.dtype, M, E), _ld(dlogits))


def moe_dispatch_rows(M, k, E, align=1) -> int:
    """Rows that moe_dispatch orders M * k pairs into at most."""
    return L().nsb_op_moe_dispatch_rows(M, k, E, align)


def moe_dispatch(idx, E, offsets, counts, rows, pos, align=1):
    """offsets [E + 1], counts [E], rows [moe_dispatch_rows(...)], pos [M, k] (int32) <- the pairs of idx by expert."""
    import torch
    M, k = idx.shape
    i32 = torch.int32
    if rows.shape[0] != moe_dispatch_rows(M, k, E, align):
        raise ValueError(f"rows: {rows.shape[0]} where {moe_dispatch_rows(M, k, E, align)} are wanted")
    _run("nsb_op_moe_dispatch", _dense(idx, "idx", i32, M, k), M, k, E, align, _dense(offsets, "offsets", i32, E + 1),
         _dense(counts, "counts", i32, E), _dense(rows, "rows", i32, None), _dense(pos, "pos", i32, M, k))


def moe_combine(o, pos, y, w=None):
    """y [M, D] <- sum over j of w[:, j] * o[pos[:, j]] (w None: 1)."""
    import torch
    M, k = pos.shape
    D = y.shape[1]
    at, dt, ld = _float(o, "o", None, D)
    _run("nsb_op_moe_combine", at, dt, ld, _dense(pos, "pos", torch.int32, M, k),
         _dense(w, "w", torch.float32, M, k) if w is not None else None, M, k, D, _is(y, "y", o.dtype, M, D), _ld(y))


def moe_combine_bwd(dy, o, rows, pos, w, do, dw=None):
    """do [R, D], dw [M, k] <- the gradients of moe_combine's o and w (dw None: do alone; o may be None then)."""
    import torch
    M, k = pos.shape
    D = dy.shape[1]
    R = rows.shape[0]
    at, dt, ld = _float(dy, "dy", M, D)
    if dw is not None and o is None:
        raise ValueError("dw needs o")
    _run("nsb_op_moe_combine_bwd", at, _is(o, "o", dy.dtype, R, D) if o is not None else None, dt, ld,
         _ld(o) if o is not None else 0, _dense(rows, "rows", torch.int32, R), _dense(pos, "pos", torch.int32, M, k),
         _dense(w, "w", torch.float32, M, k) if w is not None else None, M, k, R, D, _is(do, "do", dy.dtype, R, D),
         _ld(do), _dense(dw, "dw", torch.float32, M, k) if dw is not None else None)


def fp8_ld(n) -> int:
    """Leading dimension of n codes a row: rows start on 16-byte boundaries."""
    return -(-n // 16) * 16


def _quantized(q, s, what, rows, cols, srows, scols):
    import torch
    if q is None:
        return None, 0, None, 0
    return (_is(q, what, torch.float8_e4m3fn, rows, cols), _ld16(q),
            _is(s, what + "'s scales", torch.float32, srows, scols), _ld(s))


def fp8_quantize(x, q=None, s=None, qt=None, st=None, act=0, rows=None, row_div=1):
    """q [M, K] with s [ceil(K / 128), M], and / or qt [K, M] with st [ceil(M / 128), K] <- codes and scales of act(x).

    q, qt: float8_e4m3fn with rows on 16-byte boundaries. rows [M] (int32) gathers rows[r] / row_div of x first
    (row_div 0: only puts zeros where rows is negative)."""
    import torch
    n, K = x.shape
    M = n if rows is None else rows.shape[0]
    if rows is not None and row_div == 0 and n < M:
        raise ValueError(f"x: {n} rows where {M} are wanted")
    at, dt, ld = _float(x, "x", n, K)
    _run("nsb_op_fp8_quantize", at, dt, ld, M, K, act,
         _dense(rows, "rows", torch.int32, M) if rows is not None else None, row_div,
         *_quantized(q, s, "q", M, K, -(-K // 128), M), *_quantized(qt, st, "qt", K, M, -(-M // 128), K))


def fp8_quantize_block(x, q=None, s=None, qt=None, st=None):
    """q [M, K] with s [ceil(M / 128), ceil(K / 128)], and / or their transposes qt, st <- codes and scales of x."""
    M, K = x.shape
    mb, kb = -(-M // 128), -(-K // 128)
    at, dt, ld = _float(x, "x", M, K)
    _run("nsb_op_fp8_quantize_block", at, dt, ld, M, K, *_quantized(q, s, "q", M, K, mb, kb),
         *_quantized(qt, st, "qt", K, M, kb, mb))


def gemm_fp8(a, sa, b, sb, c, err=None):
    """c [M, N] (fp32 or bf16) <- A B^T of codes a [M, K] with row scales sa, b [N, K] with scales sb: of rows
    [ceil(K / 128), N], or of blocks [ceil(N / 128), ceil(K / 128)]. Where both have that shape (K > 128 and N both
    in one block: N = ceil(N / 128) = ceil(K / 128) = 1) they are the same."""
    import torch
    f8, f32 = torch.float8_e4m3fn, torch.float32
    M, K = a.shape
    N = b.shape[0]
    kb = -(-K // 128)
    by_rows = tuple(sb.shape) == (kb, N)
    c_at, c_dt, ldc = _float(c, "c", M, N)
    _run("nsb_op_gemm_fp8", M, N, K, _is(a, "a", f8, M, K), _ld16(a), _is(sa, "sa", f32, kb, M), _ld(sa),
         _is(b, "b", f8, N, K), _ld16(b),
         _is(sb, "sb", f32, kb, N) if by_rows else _is(sb, "sb", f32, -(-N // 128), kb), _ld(sb), int(by_rows),
         c_at, c_dt, ldc, p(err))


def moe_gemm_fp8(a, sa, offsets, counts, b, sb, c, rows=None, row_div=1, err=None):
    """Rows of c [R, N] of each expert e <- those of A times B[e]^T: a [R, K] (with rows [R]: [any, K], of which
    row r takes rows[r] / row_div) with row scales sa, b [E, N, K] with block scales sb."""
    import torch
    f8, f32, i32 = torch.float8_e4m3fn, torch.float32, torch.int32
    n, K = a.shape
    E, N, _ = b.shape
    R = c.shape[0]
    kb = -(-K // 128)
    c_at, c_dt, ldc = _float(c, "c", R, N)
    _run("nsb_op_moe_gemm_fp8", R, E, N, K, _is(a, "a", f8, n if rows is not None else R, K), _ld16(a), n,
         _is(sa, "sa", f32, kb, n), _ld(sa), _dense(rows, "rows", i32, R) if rows is not None else None, row_div,
         _dense(offsets, "offsets", i32, E + 1), _dense(counts, "counts", i32, E), _is(b, "b", f8, E, N, K),
         _ld16(b, 1), b.stride(0), _is(sb, "sb", f32, E, -(-N // 128), kb), _ld(sb, 1), sb.stride(0), c_at, c_dt, ldc,
         p(err))


def moe_wgrad_fp8(a, sa, b, sb, offsets, counts, c, err=None):
    """c [E, M, N] <- for each expert the sum over its columns of a [M, R] and b [N, R] (row scales sa, sb)."""
    import torch
    f8, f32, i32 = torch.float8_e4m3fn, torch.float32, torch.int32
    M, R = a.shape
    N = b.shape[0]
    E = c.shape[0]
    rb = -(-R // 128)
    c_at, c_dt, _ = _float(c, "c", E, M, N)
    _run("nsb_op_moe_wgrad_fp8", M, N, R, E, _is(a, "a", f8, M, R), _ld16(a), _is(sa, "sa", f32, rb, M), _ld(sa),
         _is(b, "b", f8, N, R), _ld16(b), _is(sb, "sb", f32, rb, N), _ld(sb), _dense(offsets, "offsets", i32, E + 1),
         _dense(counts, "counts", i32, E), c_at, c_dt, _ld(c, 1), c.stride(0), p(err))
