"""The batched step's launches without a GPU: what they say of themselves (grid, block and shared memory as they are launched), and what
the C binds refuse that the Python classes never ask for."""

import pytest
import torch

from sgl_muse_mega_b200.common import host
from sgl_muse_mega_b200.muse_spark.b200 import batch as BT

I32, I64, BF, F32 = torch.int32, torch.int64, torch.bfloat16, torch.float32


def z(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=dtype)


def shape(op):
    i = op.launch.info()
    return i.kernels, i.grid, i.block, i.smem, i.cluster


def tables(batch, pool, width, rows):
    return BT.BlockTables(host.library(), None, seq_lens=z(batch, dtype=I64), new_lens=z(batch, dtype=I64), req_pool_indices=z(batch, dtype=I64),
                          req_to_page=z(pool, width), pages_owned=z(pool), free_pages=z(8), free_words=z(2, dtype=I64), page_size=16,
                          rows=rows)  # fmt: skip


def test_block_tables():
    # a block a 1024 entries of a request or 256 rows, at most two an SM; 24 bytes a request and two bits a pool row
    assert shape(tables(3, 33, 2000, 10)) == (1, 6, 256, (3 * 6 + 1) * 4 + 2 * 8, 1)
    assert shape(tables(3, 32, 8, 1500)) == (1, 6, 256, (3 * 6 + 1) * 4 + 8, 1)
    assert shape(tables(400, 400, 8, 8)) == (1, 296, 256, (400 * 6 + 1) * 4 + 13 * 8, 1)


def test_rope_table():
    def op(rows, rot):
        return BT.RopeTable(host.library(), None, rows=rows, rot=rot, theta=1e4, device="cpu")

    assert shape(op(37, 64)) == (1, (10 * 8 + 127) // 128, 128, 0, 1)  # 4 positions and 4 frequencies a thread
    assert shape(op(131072, 128)) == (1, 8192 * 16 // 128, 128, 0, 1)  # 16 positions


def test_rotary():
    def op(rows, qh, kvh, dim, rot, inter):
        return BT.Rotary(host.library(), None, q=z(rows, qh, dim, dtype=BF), k=z(rows, kvh, dim, dtype=BF), k_out=z(rows, kvh, dim, dtype=BF),
                         positions=z(rows, dtype=I64), cos_sin_cache=z(4, rot, dtype=F32), interleaved=inter)  # fmt: skip

    assert shape(op(7, 2, 1, 64, 64, False)) == (1, 7, 32, 0, 1)  # 3 heads of 4 pieces
    assert shape(op(7, 5, 5, 80, 24, False)) == (1, 7, 192, 0, 1)  # 10 heads of 3 + 14 pieces of 8 bytes
    assert shape(op(9, 64, 8, 128, 64, True)) == (1, 9, 256, 0, 1)


def test_prefix_attention():
    def op(rows, qh, dim):
        return BT.PrefixAttention(host.library(), None, q=z(rows, qh, dim, dtype=BF), k_cache=z(64, 2, dim, dtype=BF), v_cache=z(64, 2, dim, dtype=BF),
                                  block_table=z(2, 4), kv_lens=z(2), cu_rows=z(3), prefix_len=z(1), page_size=16, max_new=2, scale=0.125)  # fmt: skip

    # 148 CTAs of twelve warps, 12 tiles of 16 KB or 7 of 32 KB; the merge takes a block per 8 rows, at most 12 an SM
    assert shape(op(4, 4, 64)) == (2, 148, 384, 12 * 16384 + 1024, 1)
    assert shape(op(4, 4, 128)) == (2, 148, 384, 7 * 32768 + 1024, 1)
    assert shape(op(500, 16, 64)) == (2, 1000, 384, 12 * 16384 + 1024, 1)
    assert shape(op(5000, 16, 64)) == (2, 12 * 148, 384, 12 * 16384 + 1024, 1)


@pytest.mark.parametrize("over,msg", [
    (dict(k_row=64), "k_cache: row stride"), (dict(v_row=64, v_head=64 * 64), "v_cache: row stride"), (dict(k_head=0), "k_cache: head stride"),
    (dict(q_head=32), "q: head stride"), (dict(q_row=64, q_head=4 * 64), "q: row stride"), (dict(q_row=0), "q: row stride"), (dict(k_row=0), "k_cache: row stride"),
    (dict(q_head=0), "head stride"), (dict(k_row=136), None), (dict(q_row=512, q_head=128), None),
])  # fmt: skip
def test_prefix_attention_strides(over, msg):
    """Heads-outermost pools and rows inside one another have no tensor map."""
    lib = host.library()
    op = BT.PrefixAttention(lib, None, q=z(4, 4, 64, dtype=BF), k_cache=z(64, 2, 64, dtype=BF), v_cache=z(64, 2, 64, dtype=BF), block_table=z(2, 4),
                            kv_lens=z(2), cu_rows=z(3), prefix_len=z(1), page_size=16, max_new=2, scale=0.125)  # fmt: skip
    for name, value in over.items():
        setattr(op.bind, name, value)
    if msg is None:
        lib.bind("mk_prefix_attn_bind", None, op.bind)
        return
    with pytest.raises(RuntimeError, match=msg):
        lib.bind("mk_prefix_attn_bind", None, op.bind)


def test_heads_outermost_is_refused():
    with pytest.raises(ValueError, match="heads outermost"):
        BT.PrefixAttention(host.library(), None, q=z(4, 4, 64, dtype=BF), k_cache=z(2, 64, 64, dtype=BF).transpose(0, 1), v_cache=z(64, 2, 64, dtype=BF),
                           block_table=z(2, 4), kv_lens=z(2), cu_rows=z(3), prefix_len=z(1), page_size=16, max_new=2, scale=0.125)  # fmt: skip


@pytest.mark.parametrize("scaling", [
    dict(kind="linear", factor=1e-310), dict(kind="ntk", factor=1e300), dict(kind="ntk", factor=1e-320),
    dict(kind="llama3", factor=1e-310, low_freq_factor=1.0, high_freq_factor=4.0, original_len=1),  # a sixth of a turn: all scaled
    dict(kind="yarn", factor=1e-310, beta_fast=32.0, beta_slow=1.0, original_len=8192),
])  # fmt: skip
def test_rope_table_whose_frequencies_are_not_numbers(scaling):
    """A table of NaN, or of cos 0 throughout, is no table."""
    with pytest.raises(RuntimeError, match="factor"):
        BT.RopeTable(host.library(), None, rows=5, rot=8, theta=1e4, device="cpu", scaling=scaling)
