"""The batched step's operators without a GPU: what their binds refuse (pack-only records) and the definitions that the GPU tests
compare with."""

import math

import pytest
import torch

import batch_ref as R
from sgl_muse_mega_b200.common import host
from sgl_muse_mega_b200.muse_spark.b200 import batch as BT

I32, I64, BF, F32 = torch.int32, torch.int64, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def lib():
    return host.library()


def z(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=dtype)


def tables_args(**over):
    kw = dict(seq_lens=z(4, dtype=I64), new_lens=z(4, dtype=I64), req_pool_indices=z(4, dtype=I64), req_to_page=z(6, 10),
              pages_owned=z(6), free_pages=z(60), free_words=z(2, dtype=I64), page_size=16, rows=8)  # fmt: skip
    return dict(kw, **over)


def rotary_args(rows=4, qh=4, kvh=2, dim=64, rot=64, **over):
    kw = dict(q=z(rows, qh, dim, dtype=BF), k=z(rows, kvh, dim, dtype=BF), v=z(rows, kvh, dim, dtype=BF), positions=z(rows, dtype=I64),
              cos_sin_cache=z(32, rot, dtype=F32), slots=z(rows, dtype=I64), k_cache=z(16, kvh, dim, dtype=BF),
              v_cache=z(16, kvh, dim, dtype=BF))  # fmt: skip
    return dict(kw, **over)


def attn_args(rows=4, qh=4, kvh=2, dim=64, batch=2, **over):
    kw = dict(q=z(rows, qh, dim, dtype=BF), k_cache=z(64, kvh, dim, dtype=BF), v_cache=z(64, kvh, dim, dtype=BF), block_table=z(batch, 4),
              kv_lens=z(batch), cu_rows=z(batch + 1), prefix_len=z(1), page_size=16, max_new=2, scale=0.125)  # fmt: skip
    return dict(kw, **over)


def test_binds_without_a_module(lib):
    for op in (BT.BlockTables(lib, None, **tables_args()), BT.Rotary(lib, None, **rotary_args()), BT.PrefixAttention(lib, None, **attn_args()),
               BT.RopeTable(lib, None, rows=5, rot=64, theta=1e4, device="cpu")):  # fmt: skip
        with pytest.raises(RuntimeError, match="pack-only"):
            op.launch(0)
    a = BT.PrefixAttention(lib, None, **attn_args())
    assert a.consts.kernels == 2 and a.consts.ws_bytes == a.ws.numel() and a.launch.info().kernels == 2


@pytest.mark.parametrize("over,error,msg", [
    (dict(seq_lens=z(4)), ValueError, "seq_lens"), (dict(new_lens=z(3, dtype=I64)), ValueError, "new_lens"),
    (dict(req_to_page=z(6, 20)[:, ::2]), ValueError, "contiguous"), (dict(pages_owned=z(5)), ValueError, "pages_owned"),
    (dict(free_words=z(2)), ValueError, "free_words"), (dict(page_size=0), RuntimeError, "page_size"),
    (dict(rows=0), ValueError, "rows"), (dict(page_size=1 << 19, req_to_page=z(6, 3000)), RuntimeError, "2\\^30"),
])  # fmt: skip
def test_block_tables_refusals(lib, over, error, msg):
    with pytest.raises(error, match=msg):
        BT.BlockTables(lib, None, **tables_args(**over))


def test_block_tables_batch_limit(lib):
    with pytest.raises(RuntimeError, match="batch"):
        n = 4097
        BT.BlockTables(lib, None, **tables_args(seq_lens=z(n, dtype=I64), new_lens=z(n, dtype=I64), req_pool_indices=z(n, dtype=I64)))


@pytest.mark.parametrize("over,error,msg", [
    (dict(rot=12), ValueError, "rot"), (dict(rot=264), RuntimeError, "rot"), (dict(rows=0), ValueError, "row"), (dict(theta=1.0), RuntimeError, "theta"),
    (dict(theta=math.nan), RuntimeError, "theta"), (dict(first=-1), RuntimeError, "first"), (dict(scaling=dict(kind="cubic")), ValueError, "kind"),
    (dict(scaling=dict(kind="linear")), ValueError, "factor"), (dict(scaling=dict(kind="linear", factor=0.0)), RuntimeError, "factor"),
    (dict(scaling=dict(kind="ntk", factor=2.0, beta_fast=1.0)), ValueError, "takes"),
    (dict(scaling=dict(kind="llama3", factor=8.0, low_freq_factor=4.0, high_freq_factor=1.0, original_len=8192)), RuntimeError, "freq_factor"),
    (dict(scaling=dict(kind="yarn", factor=8.0, beta_fast=1.0, beta_slow=32.0, original_len=8192)), RuntimeError, "beta"),
    (dict(scaling=dict(kind="yarn", factor=8.0, beta_fast=32.0, beta_slow=1.0, original_len=0)), RuntimeError, "original_len"),
])  # fmt: skip
def test_rope_table_refusals(lib, over, error, msg):
    with pytest.raises(error, match=msg):
        BT.RopeTable(lib, None, **dict(dict(rows=5, rot=64, theta=1e4, device="cpu"), **over))


@pytest.mark.parametrize("over,error,msg", [
    (dict(q=z(4, 4, 64, dtype=F32)), ValueError, "dtype"), (dict(k=z(4, 2, 64, dtype=torch.float16)), ValueError, "dtype"),
    (dict(v=z(4, 1, 64, dtype=BF)), ValueError, "shape"), (dict(positions=z(4)), ValueError, "positions"),
    (dict(cos_sin_cache=z(32, 72, dtype=F32)), RuntimeError, "rot"), (dict(cos_sin_cache=z(32, 12, dtype=F32)), RuntimeError, "rot"),
    (dict(slots=None), RuntimeError, "slots"), (dict(v=None), RuntimeError, "go together"), (dict(k=None, v=None), ValueError, "k_cache"),
    (dict(q=z(4, 4, 128, dtype=BF)[..., ::2]), ValueError, "strided"), (dict(q=z(4, 4, 66, dtype=BF)[..., :64]), RuntimeError, "16 bytes"),
    (dict(q=z(1, 4, 64, dtype=BF).expand(4, 4, 64)), ValueError, "overlap"),
    (dict(k_cache=None, v_cache=None, v=None, slots=None), RuntimeError, "place"),
])  # fmt: skip
def test_rotary_refusals(lib, over, error, msg):
    with pytest.raises(error, match=msg):
        BT.Rotary(lib, None, **rotary_args(**over))


def test_rotary_head_dim_refusal(lib):
    with pytest.raises(RuntimeError, match="head_dim"):
        BT.Rotary(lib, None, **rotary_args(dim=264))


@pytest.mark.parametrize("over,error,msg", [
    (dict(q=z(4, 4, 96, dtype=BF), k_cache=z(64, 2, 96, dtype=BF), v_cache=z(64, 2, 96, dtype=BF)), RuntimeError, "head_dim"),
    (dict(q=z(4, 5, 64, dtype=BF)), RuntimeError, "heads"), (dict(k_cache=z(64, 2, 64, dtype=F32)), ValueError, "dtype"),
    (dict(v_cache=z(32, 2, 64, dtype=BF)), ValueError, "shape"), (dict(block_table=z(3, 4)), ValueError, "block_table"),
    (dict(block_table=z(2, 8)[:, ::2]), ValueError, "strided"), (dict(kv_lens=z(2, dtype=I64)), ValueError, "kv_lens"),
    (dict(cu_rows=z(2)), ValueError, "cu_rows"), (dict(prefix_len=z(2)), ValueError, "prefix_len"), (dict(max_new=0), RuntimeError, "max_new"),
    (dict(max_new=5), RuntimeError, "max_new"), (dict(scale=0.0), RuntimeError, "scale"), (dict(scale=math.inf), RuntimeError, "scale"),
    (dict(window=-1), RuntimeError, "window"), (dict(page_size=0), RuntimeError, "page_size"), (dict(out=z(4, 4, 64, dtype=F32)), ValueError, "out"),
])  # fmt: skip
def test_prefix_attention_refusals(lib, over, error, msg):
    with pytest.raises(error, match=msg):
        BT.PrefixAttention(lib, None, **attn_args(**over))


def test_prefix_attention_scratch_is_checked(lib):
    a = BT.PrefixAttention(lib, None, **attn_args())
    bind = a.bind
    bind.ws_bytes = a.consts.ws_bytes - 1
    with pytest.raises(RuntimeError, match="ws_bytes"):
        lib.bind("mk_prefix_attn_bind", None, bind)


def test_reference_tables_by_hand():
    got = R.tables([5, 0, 16], [4, 0, 1], [2, -7, 0], [[10, 11, -1], [-1] * 3, [3, -1, -1]], [2, 0, 1], [7, 8, 9], [4, 6], 8, 6)
    # request 0: tokens 5..8, page 1 comes from ring entry 4 % 3; request 2 owns two pages and needs a third
    assert got["block_table"] == [[3, 8, -1], [-1] * 3, [10, 11, 9]]
    assert got["slots"] == [29, 30, 31, 64, 72] and got["positions"] == [5, 6, 7, 8, 16]
    assert got["cu_rows"] == [0, 4, 4, 5] and got["kv_lens"] == [9, 0, 17] and got["free_words"] == [6, 6] and got["pages_owned"] == [3, 0, 2]


def test_reference_rotation_is_its_own_gradient():
    """The rotation's gradient is the rotation back: against central differences of a weighted sum."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(3, 2, 24, generator=g, dtype=torch.float64), torch.randn(3, 2, 24, generator=g, dtype=torch.float64)
    tab = R.rope_table(3, 16, 1e4, None, 5)
    for inter in (False, True):
        grad = R.rotate(w, tab, inter, True)
        for i in (0, 7, 9, 15, 20):
            d = torch.zeros_like(x)
            d[..., i] = 1e-4
            diff = ((R.rotate(x + d, tab, inter, False) - R.rotate(x - d, tab, inter, False)) * w).sum(-1) / 2e-4
            assert torch.allclose(diff, grad[..., i], atol=1e-9)
