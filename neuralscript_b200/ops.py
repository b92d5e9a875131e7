"""ctypes bindings of the kernel-level C-ABI (include/ns_b200_ops.h) taking
torch CUDA tensors; device memory comes from torch (plumbing only)."""
from __future__ import annotations

import ctypes as C
import functools
import struct

from . import lib as _core_lib

F32, BF16 = 0, 1
AUTO, SIMT, TENSOR = 0, 1, 2

# arguments that several entries have: a tensor of heads, a cache, a rotation, packed attention
_heads_args = [C.c_void_p, C.c_longlong, C.c_longlong]
_cache_args = [C.c_void_p] + [C.c_longlong] * 3
_turn_args = [C.c_void_p, C.c_longlong, C.c_int, C.POINTER(C.c_int), C.c_void_p, C.c_int, C.c_int, C.c_float]
_window_args = _heads_args * 3 + [C.c_int] * 5 + [C.c_void_p] + [C.c_int] * 3 + [C.c_float]

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
    "nsb_op_rope": (C.c_int, [C.c_void_p, C.c_int, C.c_longlong, C.c_longlong, C.c_int, C.c_int, C.c_int] + _turn_args
                    + _heads_args + [C.c_void_p]),
    "nsb_op_rope_bwd": (C.c_int, [C.c_void_p, C.c_int, C.c_longlong, C.c_longlong, C.c_int, C.c_int, C.c_int] + _turn_args
                        + _heads_args + [C.c_void_p]),
    "nsb_op_kv_append": (C.c_int, _heads_args * 2 + [C.c_int] * 4 + [C.c_void_p] * 3 + [C.c_longlong] + [C.c_int] * 4
                         + _cache_args * 2 + _turn_args + _heads_args + [C.c_int] + _heads_args + [C.c_void_p]),
    "nsb_op_attention_paged_workspace_bytes": (C.c_size_t, [C.c_int] * 4),
    "nsb_op_attention_paged": (C.c_int, _heads_args + [C.c_int] * 5 + _cache_args * 2
                               + [C.c_int, C.c_int, C.c_void_p, C.c_longlong, C.c_int, C.c_void_p, C.c_int, C.c_int,
                                  C.c_float] + _heads_args + [C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]),
    "nsb_op_attention_window": (C.c_int, _window_args + _heads_args + [C.c_void_p, C.c_longlong, C.c_void_p]),
    "nsb_op_attention_window_bwd": (C.c_int, _window_args + _heads_args + [C.c_void_p, C.c_longlong] + _heads_args * 4
                                    + [C.c_void_p, C.c_size_t, C.c_void_p]),
    "nsb_op_attention_window_bwd_workspace_bytes": (C.c_size_t, [C.c_int] * 5),
    "nsb_op_from_block": (C.c_int, [C.c_int, C.c_char_p, C.c_size_t]),
}
_letters = {C.c_void_p: "P", C.POINTER(C.c_int): "P", C.c_int: "i", C.c_longlong: "q", C.c_float: "f", C.c_size_t: "N"}
# entries that _call takes, in the order of the header's numbers, and what packs their arguments
_BLOCKS = ("nsb_op_rope", "nsb_op_rope_bwd", "nsb_op_kv_append", "nsb_op_attention_paged", "nsb_op_attention_window",
           "nsb_op_attention_window_bwd")
_ROPE, _ROPE_BWD, _APPEND, _PAGED, _WINDOW, _WINDOW_BWD = range(6)
_packs = [struct.Struct("".join(_letters[t] for t in _sigs[n][1])).pack for n in _BLOCKS]
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


def _call(lib, which, *args):
    """An entry with its arguments in one block: ctypes takes 0.1 us for each of up to 60. Addresses are ints, 0: none."""
    try:
        block = _packs[which](*args)
    except struct.error as e:  # sizes past 32 bits, numbers that are none
        raise ValueError(f"{_BLOCKS[which]}: {e}") from None
    rc = lib.nsb_op_from_block(which, block, len(block))
    if rc:
        _check(rc, _BLOCKS[which])


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
_f32 = _bf16 = _i32 = _u8 = _f8 = _stream_of = _device = _empty = None


def _torch():
    """torch's names that every call below needs, looked up once (a decode step's kernels take a few microseconds)."""
    global _f32, _bf16, _i32, _u8, _f8, _stream_of, _device, _empty
    import torch
    lib = L()  # raises where the library is missing, in this call and in the next
    _stream_of, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
    _empty = torch.empty
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


# ---------------------------------------------------------------------------
# Attention that answers token by token: rotary positions, a paged cache of
# keys and values, one new token over it, and packed sequences with a window.
# Tensors of heads are [rows, heads, dh], fp32 or bf16, with any strides but a
# head's columns side by side. Tensors that do not fit raise ValueError before
# anything is launched; see include/ns_b200_ops.h for the definitions.
# ---------------------------------------------------------------------------
def _heads(d, t, what, dtype, rows, heads, dh):
    """Address and strides (row, head) of a tensor of heads of this dtype and shape, on device d."""
    if t.dtype is not dtype or t.shape != (rows, heads, dh) or t.get_device() != d:
        _refuse(t, what, dtype, (rows, heads, dh))
    row, head, one = t.stride()
    if one != 1 and dh > 1:
        _refuse(t, what, dtype, (rows, heads, dh))
    return t.data_ptr(), row, head


def _kind(t, what):
    dt = t.dtype
    if dt is not _f32 and dt is not _bf16:
        raise ValueError(f"{what}: {dt} where float32 or bfloat16 is wanted")
    return F32 if dt is _f32 else BF16


def _workspace(need, d):
    """Scratch of this call: the allocator hands it on to calls of the same stream alone, and a graph's keeps to itself."""
    return _empty(need, dtype=_u8, device=_cuda[d])


class _Devices(dict):
    def __missing__(self, d):
        import torch
        self[d] = torch.device("cuda", d)
        return self[d]


_cuda = _Devices()
_NO_TURN = (0, 0, 0, 0, 0, 0, 0, 1.0)


@functools.lru_cache(maxsize=None)  # (kept: entries are given the address)
def _sections(sections, axes, pairs):
    """Pairs of each axis as the entries take them."""
    if len(sections) != axes or sum(sections) != pairs or min(sections) < 0:
        raise ValueError(f"sections {sections} where {axes} of sum {pairs} are wanted")
    return (C.c_int * axes)(*sections)


def _turn(d, pos, freq, T, sections, interleaved, scale):
    """The arguments of a rotation: pos [T] or [axes, T], freq [pairs], sections: pairs of each axis."""
    if pos.dim() == 1:
        pos = pos[None]
    axes = pos.shape[0]
    pairs = freq.shape[0]
    at, ld = _rows(d, pos, "pos", _i32, axes, T)
    if sections is not None:
        sections = C.addressof(_sections(tuple(sections), axes, pairs))
    elif axes != 1:
        raise ValueError(f"pos has {axes} axes: sections say how many pairs belong to each")
    else:
        sections = 0
    return at, ld, axes, sections, _dense(d, freq, "freq", _f32, (pairs,)), pairs, interleaved, scale


def _rope(which, x, pos, freq, y, sections, interleaved, scale):
    lib = _bound if _f32 else _torch()
    d = _device()
    dt = x.dtype
    T, H, dh = x.shape
    at, row, head = _heads(d, x, "x", dt, T, H, dh)
    _call(lib, which, at, _kind(x, "x"), row, head, T, H, dh, *_turn(d, pos, freq, T, sections, interleaved, scale),
          *_heads(d, y, "y", dt, T, H, dh), _stream_of(d))


def rope(x, pos, freq, y, sections=None, interleaved=False, scale=1.0):
    """y [T, H, dh] <- x with the pairs of its heads turned by pos * freq: pos [T] or [axes, T] (int32), freq [pairs]
    (float32), a pair (i, i + pairs), or (2 i, 2 i + 1) where interleaved; sections: pairs of each axis. y may be x."""
    _rope(_ROPE, x, pos, freq, y, sections, interleaved, scale)


def rope_bwd(dy, pos, freq, dx, sections=None, interleaved=False, scale=1.0):
    """dx [T, H, dh] <- the gradient of rope's x. dx may be dy."""
    _rope(_ROPE_BWD, dy, pos, freq, dx, sections, interleaved, scale)


def _pages(d, t, what, dtype, pages, page, heads, dh):
    """Address and strides (page, place, head) of a cache."""
    if t.dtype is not dtype or t.shape != (pages, page, heads, dh) or t.get_device() != d:
        _refuse(t, what, dtype, (pages, page, heads, dh))
    a, b, c, one = t.stride()
    if one != 1 and dh > 1:
        _refuse(t, what, dtype, (pages, page, heads, dh))
    return t.data_ptr(), a, b, c


def kv_append(k, v, seq, at, table, k_cache, v_cache, pos=None, freq=None, sections=None, interleaved=False, scale=1.0,
              q=None, q_out=None):
    """k, v [T, Hkv, dh] into k_cache, v_cache [pages, page, Hkv, dh] at key at[t] of sequence seq[t], by table [B, width]
    (all int32); with freq the keys are turned as by rope, and q_out [T, Hq, dh] <- q turned. Tokens with a negative seq
    are left out, and so are those without a place, which check_errors raises."""
    lib = _bound if _f32 else _torch()
    d = _device()
    kind = _kind(k, "k")
    dt = k.dtype
    T, Hkv, dh = k.shape
    B, width = table.shape
    pages, page = k_cache.shape[:2]
    if (q is None) != (q_out is None) or (pos is None) != (freq is None):
        raise ValueError("q goes with q_out, and pos with freq")
    Hq = 0 if q is None else q.shape[1]
    _call(
        lib, _APPEND, *_heads(d, k, "k", dt, T, Hkv, dh), *_heads(d, v, "v", dt, T, Hkv, dh), kind, T, Hkv, dh,
        _dense(d, seq, "seq", _i32, (T,)), _dense(d, at, "at", _i32, (T,)), *_rows(d, table, "table", _i32, B, width), B, width,
        pages, page, *_pages(d, k_cache, "k_cache", dt, pages, page, Hkv, dh),
        *_pages(d, v_cache, "v_cache", dt, pages, page, Hkv, dh),
        *(_NO_TURN if freq is None else _turn(d, pos, freq, T, sections, interleaved, scale)),
        *((0, 0, 0) if q is None else _heads(d, q, "q", dt, T, Hq, dh)), Hq,
        *((0, 0, 0) if q is None else _heads(d, q_out, "q_out", dt, T, Hq, dh)), _stream_of(d))


def attention_paged_workspace(B, Hq, Hkv, dh) -> int:
    """Bytes that attention_paged works in."""
    return L().nsb_op_attention_paged_workspace_bytes(B, Hq, Hkv, dh)


@functools.lru_cache(maxsize=256)
def _paged_bytes(d, B, Hq, Hkv, dh):
    """The same on device d (d: its multiprocessors count), without a call into the library a token."""
    return attention_paged_workspace(B, Hq, Hkv, dh)


def attention_paged(q, k_cache, v_cache, table, lens, out, lse=None, window=0, sinks=0, scale=None, workspace=None):
    """out [B, Hq, dh] (and lse [B, Hq]) <- attention of one token a sequence, q [B, Hq, dh], over the first lens[b] keys
    of caches [pages, page, Hkv, dh] by table [B, width]: with window the last `window` of them and the first `sinks`.
    scale: 1 / sqrt(dh). workspace (uint8): attention_paged_workspace(...) bytes, allocated where it is not given."""
    lib = _bound if _f32 else _torch()
    d = _device()
    kind = _kind(q, "q")
    dt = q.dtype
    B, Hq, dh = q.shape
    pages, page, Hkv, _ = k_cache.shape
    width = table.shape[1]
    if workspace is None:
        have = _paged_bytes(d, B, Hq, Hkv, dh)
        workspace = _workspace(have, d)
        room = workspace.data_ptr()
    else:
        have = workspace.numel()
        room = _dense(d, workspace, "workspace", _u8, (have,))
    _call(
        lib, _PAGED, *_heads(d, q, "q", dt, B, Hq, dh), kind, B, Hq, Hkv, dh, *_pages(d, k_cache, "k_cache", dt, pages, page, Hkv, dh),
        *_pages(d, v_cache, "v_cache", dt, pages, page, Hkv, dh), pages, page, *_rows(d, table, "table", _i32, B, width), width,
        _dense(d, lens, "lens", _i32, (B,)), *_reach(window, sinks), dh ** -0.5 if scale is None else scale,
        *_heads(d, out, "out", dt, B, Hq, dh), 0 if lse is None else _dense(d, lse, "lse", _f32, (B, Hq)),
        room, have, _stream_of(d))


def _reach(window, sinks):
    """Both as the entries take them: an int of 32 bits would drop the digits above."""
    if not 0 <= window < 2147483648 or not 0 <= sinks < 2147483648:
        raise ValueError(f"window {window}, sinks {sinks} where 0 to 2^31 - 1 is wanted")
    return window, sinks


def _packed(d, q, k, v, offsets, window, sinks, scale):
    kind = _kind(q, "q")
    dt = q.dtype
    T, Hq, dh = q.shape
    Hkv = k.shape[1]
    B = 1 if offsets is None else offsets.shape[0] - 1
    return (*_heads(d, q, "q", dt, T, Hq, dh), *_heads(d, k, "k", dt, T, Hkv, dh), *_heads(d, v, "v", dt, T, Hkv, dh), kind,
            T, Hq, Hkv, dh, 0 if offsets is None else _dense(d, offsets, "offsets", _i32, (B + 1,)), B,
            *_reach(window, sinks), dh ** -0.5 if scale is None else scale)


def attention_window(q, k, v, out, lse=None, offsets=None, window=0, sinks=0, scale=None):
    """out [T, Hq, dh] (and lse [Hq, T]) <- causal attention of packed sequences, q [T, Hq, dh] and k, v [T, Hkv, dh]:
    rows offsets[b] to offsets[b + 1] (int32, [B + 1]; None: one sequence) are sequence b. With window a query sees the
    last `window` keys up to its own, and the first `sinks`. Rows behind the last sequence are left as they are."""
    lib = _bound if _f32 else _torch()
    d = _device()
    T, Hq, dh = q.shape
    _call(lib, _WINDOW, *_packed(d, q, k, v, offsets, window, sinks, scale), *_heads(d, out, "out", q.dtype, T, Hq, dh),
          *((0, 0) if lse is None else _rows(d, lse, "lse", _f32, Hq, T)), _stream_of(d))


def attention_window_bwd_workspace(T, Hq, Hkv, dh, dtype) -> int:
    """Bytes that attention_window_bwd works in; dtype: the tensors'."""
    lib = _bound if _f32 else _torch()
    return lib.nsb_op_attention_window_bwd_workspace_bytes(T, Hq, Hkv, dh, F32 if dtype is _f32 else BF16)


def attention_window_bwd(q, k, v, out, lse, dout, dq, dk, dv, offsets=None, window=0, sinks=0, scale=None,
                         workspace=None):
    """dq [T, Hq, dh], dk, dv [T, Hkv, dh] <- the gradients of attention_window's q, k, v for out's gradient dout, from
    its out and lse. workspace (uint8): attention_window_bwd_workspace(...) bytes, allocated where it is not given."""
    lib = _bound if _f32 else _torch()
    d = _device()
    dt = q.dtype
    T, Hq, dh = q.shape
    Hkv = k.shape[1]
    args = _packed(d, q, k, v, offsets, window, sinks, scale)
    if workspace is None:
        need = lib.nsb_op_attention_window_bwd_workspace_bytes(T, Hq, Hkv, dh, F32 if dt is _f32 else BF16)
        workspace = _workspace(need, d)
    have = workspace.numel()
    _call(
        lib, _WINDOW_BWD, *args, *_heads(d, out, "out", dt, T, Hq, dh), *_rows(d, lse, "lse", _f32, Hq, T),
        *_heads(d, dout, "dout", dt, T, Hq, dh), *_heads(d, dq, "dq", dt, T, Hq, dh), *_heads(d, dk, "dk", dt, T, Hkv, dh),
        *_heads(d, dv, "dv", dt, T, Hkv, dh), _dense(d, workspace, "workspace", _u8, (have,)), have, _stream_of(d))
