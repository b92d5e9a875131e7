"""Argument checks of rotary positions, the paged cache and attention with a
window at the C entries: every refusal comes before anything is launched, so
none needs a GPU."""
import ctypes as C

import pytest

from neuralscript_b200 import ops

X = 0x10000  # an address that is never read


def call(name, ok, bad):
    return getattr(ops.L(), name)(*(ok | bad).values(), None)


def ints(*v):
    return (C.c_int * len(v))(*v)


ROPE = dict(x=X, dtype=0, row=64, head=64, T=4, H=1, dh=64, pos=X, ld_pos=4, axes=1, sections=None, freq=X, pairs=32, interleaved=0,
            scale=1.0, y=X, y_row=64, y_head=64)


@pytest.mark.parametrize("name", ["nsb_op_rope", "nsb_op_rope_bwd"])
@pytest.mark.parametrize("bad", [dict(x=None), dict(dtype=2), dict(T=-1), dict(H=0), dict(dh=63), dict(dh=0), dict(dh=1026), dict(pos=None),
                                 dict(axes=0), dict(axes=5), dict(axes=2, ld_pos=4), dict(axes=2, ld_pos=3, sections=ints(16, 16)),
                                 dict(axes=2, sections=ints(16, 15)), dict(axes=2, sections=ints(33, -1)),
                                 dict(axes=2, sections=ints(33, 0)), dict(freq=None), dict(pairs=33), dict(pairs=0), dict(pairs=-1),
                                 dict(scale=float("nan")), dict(y=None)])
def test_rope_refuses(name, bad):
    assert call(name, ROPE, bad) == -1


def test_rope_limits():
    assert call("nsb_op_rope", ROPE, dict(H=(1 << 20) + 1)) == -2
    assert call("nsb_op_rope", ROPE, dict(T=0)) == 0


APPEND = dict(k=X, k_row=64, k_head=64, v=X, v_row=64, v_head=64, dtype=1, T=4, Hkv=1, dh=64, seq=X, at=X, table=X, ld_table=3, B=2, width=3,
              pages=9, page=16, kc=X, kc_page=1024, kc_slot=64, kc_head=64, vc=X, vc_page=1024, vc_slot=64, vc_head=64, pos=X, ld_pos=4,
              axes=1, sections=None, freq=X, pairs=32, interleaved=0, scale=1.0, q=X, q_row=64, q_head=64, Hq=1, q_out=X, qo_row=64, qo_head=64)


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(dtype=3), dict(T=-1), dict(Hkv=0), dict(dh=65), dict(seq=None), dict(at=None),
                                 dict(table=None), dict(ld_table=2), dict(B=-1), dict(width=-1), dict(pages=-1), dict(page=0), dict(kc=None),
                                 dict(vc=None), dict(pos=None), dict(freq=None), dict(pairs=33), dict(q=None), dict(q_out=None), dict(Hq=0)])
def test_append_refuses(bad):
    assert call("nsb_op_kv_append", APPEND, bad) == -1


def test_append_of_no_tokens():
    assert call("nsb_op_kv_append", APPEND, dict(T=0)) == 0


@pytest.mark.parametrize("big", [dict(Hkv=1 << 30), dict(Hkv=(1 << 26) + 1), dict(Hq=(1 << 31) - 1), dict(Hq=1 << 20)])
def test_append_limits(big):
    assert call("nsb_op_kv_append", APPEND, big) == -2


PAGED = dict(q=X, q_row=64, q_head=64, dtype=1, B=2, Hq=4, Hkv=2, dh=64, kc=X, kc_page=1024, kc_slot=64, kc_head=64, vc=X, vc_page=1024, vc_slot=64,
             vc_head=64, pages=9, page=16, table=X, ld_table=3, width=3, lens=X, window=0, sinks=0, scale=0.125, out=X, o_row=64, o_head=64,
             lse=X, workspace=X, bytes=1 << 30)


@pytest.mark.parametrize("bad", [dict(q=None), dict(dtype=2), dict(B=-1), dict(Hq=3), dict(Hq=1), dict(Hkv=0), dict(dh=0), dict(dh=129), dict(kc=None),
                                 dict(vc=None), dict(pages=-1), dict(page=0), dict(table=None), dict(ld_table=2), dict(width=-1), dict(lens=None),
                                 dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
                                 dict(scale=float("nan")), dict(out=None), dict(workspace=None), dict(workspace=X + 8), dict(bytes=100)])
def test_paged_refuses(bad):
    assert call("nsb_op_attention_paged", PAGED, bad) == -1


def test_paged_limits():
    assert call("nsb_op_attention_paged", PAGED, dict(B=8193)) == -2
    assert call("nsb_op_attention_paged", PAGED, dict(B=8192, width=2 ** 30, ld_table=2 ** 30)) == -2
    assert call("nsb_op_attention_paged", PAGED, dict(B=8192, Hq=1 << 20, Hkv=1 << 20, width=1)) == -2
    assert call("nsb_op_attention_paged", PAGED, dict(B=0)) == 0
    size = ops.L().nsb_op_attention_paged_workspace_bytes
    assert size(0, 4, 2, 64) == size(2, 3, 2, 64) == size(2, 4, 2, 129) == size(2, 4, 0, 64) == 0
    assert size(2, 4, 2, 64) > 0 and size(2, 4, 2, 64) % 8 == 0


def test_block_of_arguments():
    """The same refusals through the call that takes its arguments in one block, and those of the block."""
    for which, (ok, cases) in enumerate([
            (ROPE, [(dict(dh=63), -1), (dict(H=(1 << 20) + 1), -2), (dict(T=0), 0)]), (ROPE, [(dict(axes=5), -1), (dict(T=0), 0)]),
            (APPEND, [(dict(page=0), -1), (dict(Hkv=1 << 30), -2), (dict(T=0), 0)]), (PAGED, [(dict(scale=0.0), -1), (dict(B=8193), -2), (dict(B=0), 0)]),
            (WINDOW, [(dict(ld_lse=3), -1), (dict(Hq=131072, Hkv=65536), -2), (dict(T=0), 0)]),
            (GRADS, [(dict(bytes=63), -1), (dict(Hq=131072, Hkv=65536), -2), (dict(B=0), 0)])]):
        for bad, want in cases:
            block = ops._packs[which](*(0 if v is None else v for v in (ok | bad).values()), 0)
            call_block = ops.L().nsb_op_from_block
            assert call_block(which, block, len(block)) == want, (which, bad)
            assert call_block(which, block[:-1], len(block) - 1) == call_block(which, block + b"\0", len(block) + 1) == -1
            assert call_block(which, None, len(block)) == call_block(6, block, len(block)) == call_block(-1, block, len(block)) == -1


WINDOW = dict(q=X, q_row=64, q_head=64, k=X, k_row=64, k_head=64, v=X, v_row=64, v_head=64, dtype=1, T=4, Hq=4, Hkv=2, dh=64, offsets=X, B=2,
              window=0, sinks=0, scale=0.125, out=X, o_row=64, o_head=64, lse=X, ld_lse=4)
GRADS = WINDOW | dict(dout=X, do_row=64, do_head=64, dq=X, dq_row=64, dq_head=64, dk=X, dk_row=64, dk_head=64, dv=X, dv_row=64, dv_head=64, workspace=X,
                      bytes=1 << 30)
BAD = [dict(q=None), dict(k=None), dict(v=None), dict(dtype=2), dict(T=-1), dict(Hq=3), dict(Hkv=0), dict(dh=0), dict(dh=129),
       dict(offsets=None), dict(B=-1), dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(out=None),
       dict(ld_lse=3)]


@pytest.mark.parametrize("bad", BAD)
def test_window_refuses(bad):
    assert call("nsb_op_attention_window", WINDOW, bad) == -1


@pytest.mark.parametrize("bad", BAD + [dict(lse=None), dict(dout=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(workspace=None),
                                       dict(workspace=X + 8), dict(bytes=63)])
def test_window_gradient_refuses(bad):
    assert call("nsb_op_attention_window_bwd", GRADS, bad) == -1


def test_window_limits():
    for name, ok in (("nsb_op_attention_window", WINDOW), ("nsb_op_attention_window_bwd", GRADS)):
        assert call(name, ok, dict(T=0)) == 0
        assert call(name, ok, dict(B=0)) == 0
        assert call(name, ok, dict(Hq=131072, Hkv=65536)) == -2
        assert call(name, ok, dict(T=(1 << 30) + 1, ld_lse=1 << 31)) == -2
        assert call(name, ok, dict(T=1 << 30, Hq=65535, Hkv=1, ld_lse=1 << 31)) == -2


@pytest.mark.parametrize("which,ok,bad", [(0, ROPE, dict(T=1 << 31)), (1, ROPE, dict(H=1 << 32)), (2, APPEND, dict(pages=1 << 31)), (3, PAGED, dict(B=1 << 31)),
                                          (4, WINDOW, dict(T=1 << 31)), (4, WINDOW, dict(scale="0.1")),
                                          (5, GRADS, dict(T=-(1 << 31) - 1)), (5, GRADS, dict(B=2.5))])
def test_numbers_past_their_types_raise_value_errors(which, ok, bad):
    """Before anything reaches the library."""
    with pytest.raises(ValueError, match=ops._BLOCKS[which]):
        ops._call(None, which, *(0 if v is None else v for v in (ok | bad).values()), 0)
