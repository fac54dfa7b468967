"""The batched step's operators against what the framework's one-request launches do on the same rows, pool and tables: the
target's head and attention, the draft's rotation, the window feeds."""

import pytest
import torch

from oracle import dflash_draft as D
from oracle import muse_layer as O
from sgl_muse_mega_b200.common import host
from sgl_muse_mega_b200.muse_spark.b200 import batch as BT
from sgl_muse_mega_b200.muse_spark.b200 import headtail as HT
from sgl_muse_mega_b200.muse_spark.b200 import layer as L
from sgl_muse_mega_b200.muse_spark.b200 import synthetic
from sgl_muse_mega_b200.muse_spark.b200.dflash.weights import rope_cos_sin
from sgl_muse_mega_b200.muse_spark.b200.head import QkvHead
from sgl_muse_mega_b200.muse_spark.config import Config

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
I32, I64, F32, BF = torch.int32, torch.int64, torch.float32, torch.bfloat16


def stream():
    return torch.cuda.current_stream().cuda_stream


def ctx():
    lib = host.library()
    return lib, lib.load()


def steps_apart(a, b):
    """How many steps of bf16 two tensors lie apart (values of one sign, or both next to 0)."""
    x, y = (t.contiguous().view(torch.int16).int() for t in (a, b))
    x, y = (torch.where(t < 0, -(t & 0x7FFF), t) for t in (x, y))
    return (x - y).abs()


def test_rotation_and_append_of_the_target():
    """The target's head norms q and k, scales q and turns neighbouring pairs over the 64-wide head. Its rows without the rotation, then
    `Rotary(interleaved=True)`, are its rows with it, and the pool is the same; the half layout is another rotation."""
    lib, module = ctx()
    rows, hidden, qh, kvh = 16, 1024, 16, 2
    g = torch.Generator().manual_seed(3)
    w = (torch.randn(2 * (qh + kvh) * 64, hidden, generator=g) / hidden**0.5).to(BF).to(DEV)
    x = torch.randn(rows, hidden, generator=g).to(BF).to(DEV)
    table = BT.RopeTable(lib, module, rows=8448, rot=64, theta=500000.0, device=DEV)
    table.launch(stream())
    pos = torch.randint(0, 8448, (rows,), generator=g).to(DEV)
    loc = torch.randperm(64, generator=g)[:rows].to(DEV)
    pools = [torch.zeros(64, kvh * 64, dtype=BF, device=DEV) for _ in range(6)]
    kw = dict(w=w, x=x, q_heads=qh, kv_heads=kvh, q_scale=43.7840518911 / 8, eps=1e-5, cache_loc=loc.int())
    turned = QkvHead(lib, module, cos_sin=table.cos_sin[pos], k_cache=pools[0], v_cache=pools[1], **kw)
    plain = QkvHead(lib, module, cos_sin=None, k_cache=pools[2], v_cache=pools[3], **kw)
    turned.launch(stream())
    plain.launch(stream())

    def heads(t):
        q, k, v, _ = t.split((qh * 64, kvh * 64, kvh * 64, qh * 64), 1)
        return q.unflatten(1, (qh, 64)), k.unflatten(1, (kvh, 64)), v.unflatten(1, (kvh, 64))

    q, k, v = heads(plain.out)
    kc, vc = (t.unflatten(1, (kvh, 64)) for t in pools[4:])
    bind = dict(q=q, k=k, v=v, positions=pos, cos_sin_cache=table.cos_sin, slots=loc, k_cache=kc, v_cache=vc)
    op = BT.Rotary(lib, module, interleaved=True, **bind)
    op.launch(stream())
    torch.cuda.synchronize()
    want_q, want_k, _ = heads(turned.out)
    # the same f32 products in sums that may be fused differently: next to a border they round to neighbours; where the pair's products cancel a
    # rounding of 2^-24 of them may be several steps of the result
    for got, want, src in ((op.q_out, want_q, q), (kc[loc], want_k, k)):
        pair = src.float().unflatten(2, (32, 2)).norm(dim=-1).repeat_interleave(2, -1)
        near = (got.float() - want.float()).abs() <= pair * 2.0**-22
        assert ((steps_apart(got, want) <= 1) | near).all()
        assert (got == want).float().mean() > 0.99
    assert torch.equal(pools[5], pools[1]) and op.status[0].item() == 0
    empty = torch.ones(64, dtype=torch.bool, device=DEV)
    empty[loc] = False
    assert not pools[4][empty].any()
    half = BT.Rotary(lib, module, **bind)
    half.launch(stream())
    assert (half.q_out.float() - want_q.float()).norm() > 0.5 * want_q.float().norm()

    # layers without a rotation: row 0 of the table turns by nothing, and the append is the head's
    kc.zero_()
    vc.zero_()
    op = BT.Rotary(lib, module, interleaved=True, **dict(bind, positions=torch.zeros_like(pos)))
    op.launch(stream())
    torch.cuda.synchronize()
    assert torch.equal(op.q_out, q) and torch.equal(pools[4], pools[2]) and torch.equal(pools[5], pools[3])


def test_rotation_of_the_draft():
    """The draft turns halves of its 128-wide heads: products and sums rounded one by one, then to bf16."""
    lib, module = ctx()
    g = torch.Generator().manual_seed(4)
    rows, qh, kvh = 16, 8, 2
    x = torch.randn(rows, qh + kvh, 128, generator=g).to(BF)
    pos = torch.arange(500, 500 + rows)
    cos, sin = rope_cos_sin(pos, 128, 1e6)
    ones = torch.ones(128, dtype=BF)
    want = D.head_norm_rope(x, ones, 1e-6, cos, sin, True)
    normed = D.head_norm_rope(x, ones, 1e-6, torch.ones_like(cos), torch.zeros_like(sin), True)
    dev = normed.to(DEV)
    op = BT.Rotary(lib, module, q=dev[:, :qh], k=dev[:, qh:], k_out=torch.zeros(rows, kvh, 128, dtype=BF, device=DEV), positions=torch.arange(rows).to(DEV),
                   cos_sin_cache=torch.cat((cos, sin), 1).float().to(DEV))  # fmt: skip
    op.launch(stream())
    got = torch.cat((op.q_out, op.k_out), 1).cpu()
    pair = normed.float().unflatten(2, (2, 64)).norm(dim=2).repeat(1, 1, 2)
    near = (got.float() - want.float()).abs() <= pair * 2.0**-22
    assert ((steps_apart(got, want) <= 1) | near).all() and (got == want).float().mean() > 0.99


@pytest.mark.parametrize("global_attn", [False, True])
def test_attention_of_a_layer(global_attn):
    """The target's attention of one request's window and `PrefixAttention` on the same rows and pool, token by token (page size 1): the
    request alone, and beside a copy of itself, which shares its context. Then the layer's norm and gate, and its own bound."""
    cfg = Config(hidden=1024, q_heads=16, kv_heads=2, experts=16, topk=8, moe_hidden=1024, moe_inter=1024, swa_window=100,
                 bf16_moe_layers=(), tp=1, node_ranks=1)  # fmt: skip
    rows, n = 16, 600
    case = synthetic.layer_case(cfg, rows=rows, ctx=n, global_attn=global_attn, seed=5)
    rank = L.LayerWorld(case, DEV).ranks[0]
    rank.launch_record.step(stream(), 0, 2)  # attention split + merge
    torch.cuda.synchronize()
    assert rank.launch_record.status(stream()).code == 0
    q, _, _, gate = O.split_heads(rank.w["qkv_in"], 16, 2)
    want = rank.o["x_attn"].cpu()
    lib, module = ctx()
    kc, vc = (t.unflatten(1, (2, 64)) for t in (rank.k_cache, rank.v_cache))
    table = (rank.page_table // (2 * 64 * 2)).int()
    for batch in (1, 2):
        op = BT.PrefixAttention(lib, module, q=q.repeat(batch, 1, 1), k_cache=kc, v_cache=vc, block_table=table.repeat(batch, 1),
                                kv_lens=torch.full((batch,), n + rows, dtype=I32, device=DEV), page_size=1, max_new=rows, scale=O.SOFTMAX_SCALE,
                                cu_rows=torch.arange(0, (batch + 1) * rows, rows, dtype=I32, device=DEV),
                                prefix_len=torch.tensor([n], dtype=I32, device=DEV), window=0 if global_attn else cfg.swa_window)  # fmt: skip
        op.launch(stream())
        torch.cuda.synchronize()
        assert op.status[0].item() == 0
        for out in op.out.float().cpu().split(rows):
            y = out * torch.rsqrt(out.square().mean(-1, keepdim=True) + O.ONORM_EPS) * torch.sigmoid(gate.float().cpu())
            # each within the layer's bound of the exact value, and the rows' rounding before the norm here
            _, rel, ok = O.compare(y.to(BF).reshape(rows, -1), want, "x_attn", tol=2 * O.TOLERANCES["x_attn"] + 2.0**-9)
            assert ok, (batch, rel)


def test_tables_of_a_window():
    """Page size 1: the slots and positions of one request's 16 new tokens, fed to the window feeds, and its row of the request table
    that both read."""
    lib, module = ctx()
    width, n, rows, row_bytes = 700, 601, 16, 256
    g = torch.Generator().manual_seed(6)
    ids = torch.randperm(4000, generator=g).int()
    r2t = torch.full((3, width), -1, dtype=I32)
    r2t[1, :n] = ids[:n]
    seq, req = torch.tensor([n], device=DEV), torch.tensor([1], device=DEV)
    r2t = r2t.to(DEV)
    tab = BT.BlockTables(lib, module, seq_lens=seq, new_lens=torch.tensor([rows], device=DEV), req_pool_indices=req, req_to_page=r2t,
                         pages_owned=torch.tensor([0, n, 0], dtype=I32, device=DEV), free_pages=ids[n:].to(DEV),
                         free_words=torch.tensor([5, 3000], device=DEV), page_size=1, rows=rows)  # fmt: skip
    table = torch.randn(2000, 64, generator=g).to(DEV)
    tab.launch(stream())
    feeds = HT.WindowFeeds(lib, module, positions=tab.positions, cos_sin_cache=table, out_cache_loc=tab.slots, swa_out_cache_loc=None, seq_lens=seq,
                           req_pool_indices=req, req_to_token=r2t, full_to_swa=None, kv_row_bytes=row_bytes)  # fmt: skip
    feeds.launch(stream())
    torch.cuda.synchronize()
    assert torch.equal(feeds.loc_full.long(), tab.slots) and torch.equal(feeds.kv_len, tab.kv_lens) and tab.kv_lens.item() == n + rows
    assert torch.equal(feeds.pt_full[: n + rows], tab.block_table[0, : n + rows].long() * row_bytes)
    assert torch.equal(feeds.pt_full[n : n + rows], tab.slots * row_bytes)
    assert torch.equal(feeds.cos_sin, table[n : n + rows]) and feeds.launch.status(stream()).code == 0
