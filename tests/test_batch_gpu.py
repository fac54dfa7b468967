"""The batched step's operators on the GPU against their plain 64-bit forms (``batch_ref.py``)."""

import math
import random

import pytest
import torch

import batch_ref as R
from sgl_muse_mega_b200.common import host
from sgl_muse_mega_b200.muse_spark.b200 import batch as BT

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
I32, I64, F32, BF, HF = torch.int32, torch.int64, torch.float32, torch.bfloat16, torch.float16


def stream():
    return torch.cuda.current_stream().cuda_stream


def ctx():
    lib = host.library()
    return lib, lib.load()


def dev(x, dtype):
    return torch.tensor(x, dtype=dtype, device=DEV)


# ---- block tables ---------------------------------------------------------------------------------------------------
def tables_case(seed, batch, page, ctx_hi, new_hi, spare_pages=3, ring_extra=0):
    g = random.Random(seed)
    seq = [g.choice([0, 1, page - 1, page, g.randint(0, ctx_hi)]) for _ in range(batch)]
    new = [g.choice([0, 1, g.randint(0, new_hi)]) for _ in range(batch)]
    pool = batch + 2
    width = max(-(-(s + n) // page) for s, n in zip(seq, new)) + 2
    req = g.sample(range(pool), batch)
    ids = list(range(pool * width + spare_pages))
    g.shuffle(ids)
    r2p, owned = [[-1] * width for _ in range(pool)], [0] * pool
    for s, r in zip(seq, req):
        owned[r] = min(width, -(-s // page) + g.choice([0, 0, 1]))
        for p in range(owned[r]):
            r2p[r][p] = ids.pop()
    n = len(ids) + ring_extra
    head = g.randint(0, 3 * n)
    ring = [-1] * n
    for i, x in enumerate(ids):
        ring[(head + i) % n] = x
    return dict(seq=seq, new=new, req=req, req_to_page=r2p, owned=owned, ring=ring, words=[head, head + len(ids)], page=page)


def bind_tables(c, rows):
    lib, module = ctx()
    return BT.BlockTables(
        lib, module, seq_lens=dev(c["seq"], I64), new_lens=dev(c["new"], I64), req_pool_indices=dev(c["req"], I64),
        req_to_page=dev(c["req_to_page"], I32), pages_owned=dev(c["owned"], I32), free_pages=dev(c["ring"], I32),
        free_words=dev(c["words"], I64), page_size=c["page"], rows=rows,
    )  # fmt: skip


def check_tables(op, c, rows, filler=0):
    want = R.tables(c["seq"], c["new"], c["req"], c["req_to_page"], c["owned"], c["ring"], c["words"], c["page"], rows)
    keep = op.keep
    n = len(want["slots"])
    assert op.block_table.tolist() == want["block_table"]
    assert op.slots.tolist() == want["slots"] + [filler] * (rows - n)
    assert op.positions.tolist() == want["positions"] + [filler] * (rows - n)
    assert op.cu_rows.tolist() == want["cu_rows"] and op.kv_lens.tolist() == want["kv_lens"]
    assert keep[3].tolist() == want["req_to_page"] and keep[4].tolist() == want["pages_owned"] and keep[6].tolist() == want["free_words"]
    assert op.ticket.item() == 0
    return want


@pytest.mark.parametrize("batch,page,ctx_hi,new_hi", [(1, 1, 40, 16), (1, 64, 3000, 700), (5, 16, 200, 1), (33, 7, 90, 40), (260, 16, 64, 3),
                                                       (64, 128, 9000, 500), (1, 1, 5000, 1), (4096, 16, 20, 2)])  # fmt: skip
def test_tables(batch, page, ctx_hi, new_hi):
    c = tables_case(batch + page, batch, page, ctx_hi, new_hi)
    rows = sum(c["new"]) + 5
    op = bind_tables(c, rows)
    op.slots.fill_(-9)
    op.positions.fill_(-9)
    op.launch(stream())
    torch.cuda.synchronize()
    want = check_tables(op, c, rows, -9)
    assert op.status[0].item() == 0
    # the same lengths again: nothing is left to take
    op.launch(stream())
    torch.cuda.synchronize()
    assert op.block_table.tolist() == want["block_table"] and op.keep[6].tolist() == want["free_words"] and op.ticket.item() == 0


def test_tables_all_padding():
    c = dict(seq=[0, 0], new=[0, 0], req=[-5, 99], req_to_page=[[-1, -1]], owned=[0], ring=[4], words=[0, 1], page=16)
    op = bind_tables(c, 3)
    op.launch(stream())
    torch.cuda.synchronize()
    check_tables(op, c, 3)
    assert op.status[0].item() == 0


@pytest.mark.parametrize("change,code", [
    (dict(seq=[-1, 5, 9]), 4), (dict(new=[1, -3, 2]), 4), (dict(req=[0, 7, 2]), 4), (dict(req=[0, -1, 2]), 4), (dict(req=[1, 0, 1]), 4),
    (dict(seq=[3, 5, 1 << 40]), 4), (dict(seq=[3, 500, 9]), 4), (dict(owned=[1, 0, 1, 0]), 4), (dict(owned=[1, 900, 1, 0]), 4),
    (dict(words=[5, 4]), 4), (dict(words=[0, 99]), 4), (dict(words=[7, 7]), 5), (dict(rows=4), 5),
    (dict(new=[30, 40, 2]), 4),  # 5 + 40 tokens exceed a row's 4 x 10 (recorded first), and 30 + 2 rows the buffers' 8
])  # fmt: skip
def test_tables_that_do_not_fit(change, code):
    """What contradicts the extents counts as padding, a step without room is not granted at all; both are recorded."""
    c = dict(seq=[3, 5, 9], new=[1, 3, 2], req=[0, 1, 2], req_to_page=[[20, -1, -1, -1], [21, -1, -1, -1], [22, -1, -1, -1], [-1] * 4],
             owned=[1, 1, 1, 0], ring=[30, 31, 32], words=[4, 6], page=10)  # fmt: skip
    rows = change.pop("rows", 8) if "rows" in change else 8
    c.update(change)
    op = bind_tables(c, rows)
    op.launch(stream())
    torch.cuda.synchronize()
    check_tables(op, c, rows)
    assert op.status[0].item() == code


# ---- rope table -----------------------------------------------------------------------------------------------------
SCALINGS = [None, dict(kind="linear", factor=4.0), dict(kind="ntk", factor=3.0),
            dict(kind="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_len=8192),
            dict(kind="yarn", factor=16.0, beta_fast=32.0, beta_slow=1.0, original_len=4096)]  # fmt: skip


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("rows,rot,theta,first", [(1, 8, 1e4, 0), (37, 64, 5e5, 100000), (5000, 128, 1e4, 1 << 20), (40001, 64, 5e5, 3)])
def test_rope_table(scaling, rows, rot, theta, first):
    lib, module = ctx()
    op = BT.RopeTable(lib, module, rows=rows, rot=rot, theta=theta, device=DEV, scaling=scaling, first=first)
    op.launch(stream())
    want = R.rope_table(rows, rot, theta, scaling, first)
    # half a step of f32, and the angle: 2^-52 of up to 2^20 radians on both sides and 16 turns by a step of 2^-52 each
    tol = want.abs() * 2.0**-24 + (2.0**-31 + 2.0**-46) * (1 + first / 2**20)
    assert ((op.cos_sin.double().cpu() - want).abs() <= tol).all()


# ---- rotary ---------------------------------------------------------------------------------------------------------
def rotary_tol(x, cos_sin, want, dt, interleaved, inverse):
    """Half a step of the type, and the f32 products and sum: three roundings of 2^-24 of |x c| + |y s| each."""
    mass = R.rotate(x.double().abs(), cos_sin.double().abs(), interleaved, True)
    mass = torch.maximum(mass.abs(), R.rotate(x.double().abs(), cos_sin.double().abs(), interleaved, False).abs()) + want.abs()
    tiny = 2.0**-25 if dt == HF else 0.0
    return want.abs() * torch.finfo(dt).eps / 2 * (1 + 2.0**-10) + 4 * mass * 2.0**-24 + tiny


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("rows,qh,kvh,dim,rot,inter,inverse", [
    (16, 16, 2, 64, 64, False, False), (1, 1, 1, 64, 64, True, False), (7, 5, 5, 80, 24, False, False), (33, 64, 8, 128, 64, True, True),
    (3, 3, 1, 256, 128, False, True), (9, 8, 1, 72, 8, False, False), (130, 2, 2, 40, 40, True, False), (5, 40, 8, 128, 128, False, False),
])  # fmt: skip
def test_rotary(dt, rows, qh, kvh, dim, rot, inter, inverse):
    lib, module = ctx()
    g = torch.Generator(device=DEV).manual_seed(rows * dim + rot)
    row = torch.randn(rows, (qh + 2 * kvh) * dim, generator=g, device=DEV).to(dt)  # one fused row: strided q, k, v
    q, k, v = (t.unflatten(1, (-1, dim)) for t in row.split([qh * dim, kvh * dim, kvh * dim], 1))
    n_slots = rows + 9
    slots = torch.randperm(n_slots, generator=g, device=DEV)[:rows]
    if rows > 2:
        slots[rows // 2] = -1  # rotated, not appended
    pos = torch.randint(0, 500, (rows,), generator=g, device=DEV)
    table = R.rope_table(500, rot, 1e4, None, 0).float().to(DEV)
    pool = torch.randn(n_slots, 2, kvh, dim, generator=g, device=DEV).to(dt)  # K and V interleaved in one pool: strided rows
    kc, vc = pool[:, 0], pool[:, 1]
    before = pool.clone()
    live = rows - 1 if rows > 4 else rows
    q_out = torch.full((rows, qh, dim), 7.0, dtype=dt, device=DEV)
    k_out = torch.full((rows, kvh, dim), 7.0, dtype=dt, device=DEV)
    op = BT.Rotary(lib, module, q=q, k=k, v=v, positions=pos, cos_sin_cache=table, slots=slots, k_cache=kc, v_cache=vc, q_out=q_out, k_out=k_out,
                   n_rows=dev([live], I32), interleaved=inter, inverse=inverse)  # fmt: skip
    op.launch(stream())
    torch.cuda.synchronize()
    tab = table[pos]
    for x, got in ((q, q_out), (k, k_out)):
        want = R.rotate(x, tab, inter, inverse)
        tol = rotary_tol(x.cpu(), tab.cpu(), want, dt, inter, inverse)
        assert ((got.double().cpu() - want).abs() <= tol)[:live].all()
        assert (got[live:] == 7.0).all()
    want = before.clone()
    for r in range(live):
        if slots[r] >= 0:
            want[slots[r], 0], want[slots[r], 1] = k_out[r], v[r]
    assert torch.equal(pool, want) and op.status[0].item() == 0


def test_rotary_in_place_and_back():
    """In place, then the inverse in place: the input up to two roundings of each pair's length."""
    lib, module = ctx()
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(11, 6, 64, generator=g, device=DEV).half()
    k = torch.randn(11, 2, 64, generator=g, device=DEV).half()
    was = q.double(), k.double()
    pos = torch.arange(11, device=DEV) * 40
    table = R.rope_table(500, 64, 1e4, None, 0).float().to(DEV)
    kw = dict(q=q, k=k, positions=pos, cos_sin_cache=table, q_out=q, k_out=k)
    BT.Rotary(lib, module, **kw).launch(stream())
    assert (q.double() - was[0]).abs().max() > 0.1
    BT.Rotary(lib, module, inverse=True, **kw).launch(stream())
    for x, w in zip((q, k), was):
        pair = (w[..., :32] ** 2 + w[..., 32:] ** 2).sqrt().repeat(1, 1, 2)
        # the first rounding moves each of the pair's two values by 2^-11 of at most the pair's length, the second the result
        assert ((x.double() - w).abs() <= pair * (2 * 2.0**-11 + 2.0**-11 + 2.0**-20) + 2.0**-23).all()


def test_rotary_records_bad_positions_and_slots():
    lib, module = ctx()
    table = R.rope_table(8, 64, 1e4, None, 0).float().to(DEV)
    q = torch.ones(3, 1, 64, dtype=BF, device=DEV)
    kc = torch.zeros(4, 1, 64, dtype=BF, device=DEV)
    kw = dict(q=q, k=q.clone(), v=q.clone(), cos_sin_cache=table, k_cache=kc, v_cache=kc.clone())
    op = BT.Rotary(lib, module, positions=dev([0, 8, -1], I64), slots=dev([0, 1, 2], I64), **kw)
    op.launch(stream())
    torch.cuda.synchronize()
    assert op.status[0].item() == 4 and (op.q_out == 1).all()  # row 0 of the table: no rotation
    op = BT.Rotary(lib, module, positions=dev([0, 0, 0], I64), slots=dev([4, 1 << 40, 3], I64), **kw)
    kc.zero_()
    op.launch(stream())
    torch.cuda.synchronize()
    assert op.status[0].item() == 4 and (kc[:3] == 0).all() and (kc[3] == 1).all()


# ---- attention ------------------------------------------------------------------------------------------------------
class AttnCase:
    """A batch with `kv[b]` keys and `new[b]` rows a request over pages in random order; slots that no request names hold NaN."""

    def __init__(self, seed, kv, new, prefix, qh, kvh, dim, page, dt, window=0, rows=None, max_new=None, layout="plain", q_mult=None):
        g = torch.Generator().manual_seed(seed)
        self.kv, self.new, self.prefix, self.page, self.dt, self.window = kv, new, prefix, page, dt, window
        self.qh, self.kvh, self.dim = qh, kvh, dim
        B = len(kv)
        shared = prefix // page
        pages = [max(-(-L // page), 0) for L in kv]
        width = max(max(pages), shared, 1)
        total = shared + sum(max(p - shared, 0) for p in pages) + 3
        ids = torch.randperm(total, generator=g).tolist()
        common = [ids.pop() for _ in range(shared)]
        table = [(common[: min(p, shared)] + [ids.pop() for _ in range(max(p - shared, 0))] + [-1] * width)[:width] for p in pages]
        self.table = torch.tensor(table, dtype=I32)
        slots = total * page
        k, v = torch.full((slots, kvh, dim), math.nan), torch.full((slots, kvh, dim), math.nan)
        body = torch.randn(2, max(prefix, 1), kvh, dim, generator=g)
        for b in range(B):
            p = torch.arange(kv[b])
            s = self.table[b, p // page].long() * page + p % page
            k[s], v[s] = torch.randn(kv[b], kvh, dim, generator=g), torch.randn(kv[b], kvh, dim, generator=g)
        for b in range(B):  # the shared tokens' values, also where the prefix ends inside a page of each request's own
            n = min(prefix, kv[b])
            p = torch.arange(n)
            s = self.table[b, p // page].long() * page + p % page
            k[s], v[s] = body[0, :n], body[1, :n]
        self.cu = [0]
        for n in new:
            self.cu.append(self.cu[-1] + n)
        self.rows = rows or max(self.cu[-1], 1)
        mult = q_mult if q_mult is not None else 3.0 / math.sqrt(dim) * 8
        q = torch.randn(self.rows, qh, dim, generator=g) * mult
        if layout == "fused":  # q inside a projection row, K and V interleaved in one pool
            row = torch.zeros(self.rows, qh * dim + 64, dtype=dt, device=DEV)
            self.q = row[:, : qh * dim].unflatten(1, (qh, dim))
            pool = torch.zeros(slots, 2, kvh, dim, dtype=dt, device=DEV)
            self.k, self.v = pool[:, 0], pool[:, 1]
        else:
            self.q = torch.zeros(self.rows, qh, dim, dtype=dt, device=DEV)
            self.k, self.v = (torch.zeros(slots, kvh, dim, dtype=dt, device=DEV) for _ in range(2))
        self.q.copy_(q)
        self.k.copy_(k)
        self.v.copy_(v)
        self.max_new = max_new or max(max(new), 1)
        self.scale = 0.125

    def bind(self, **over):
        lib, module = ctx()
        self.lens = dict(block_table=self.table.to(DEV), kv_lens=dev(self.kv, I32), cu_rows=dev(self.cu, I32), prefix_len=dev([self.prefix], I32))
        kw = dict(q=self.q, k_cache=self.k, v_cache=self.v, page_size=self.page, max_new=self.max_new, scale=self.scale, window=self.window, lse=True)
        op = BT.PrefixAttention(lib, module, **dict(kw, **self.lens, **over))
        op.out.fill_(5.0)
        op.lse.fill_(5.0)
        return op

    def check(self, op, kv=None, cu=None):
        kv, cu = kv or self.kv, cu or self.cu
        out, lse, mass = R.attention(self.q, self.k, self.v, self.table, kv, cu, self.page, self.scale, self.window)
        n = cu[-1]
        eps = torch.finfo(self.dt).eps / 2
        # P is rounded to the type once (eps of the weighted mean of |v|), the result once; scores: f32 sums of products, whose
        # absolute terms come to less than 64 in the exponent, 2^-20 of that, and an exponential good to 4e-6 (1e-4 of mass)
        tol = out.abs() * eps + mass * (eps + 1e-4) + 1e-6
        if self.dt == HF:  # probabilities below 2^-14 of the largest have a fixed step of 2^-24
            tol = tol + max(max(kv), 1) * 2.0**-25 * 5
        got, got_lse = op.out.double().cpu(), op.lse.double().cpu()
        assert torch.isfinite(got[:n]).all()
        bad = ((got - out).abs() > tol)[:n]
        assert not bad.any(), (int(bad.sum()), float((got - out).abs()[:n].max()))
        empty = lse[:n] == -math.inf
        assert (got_lse[:n][empty] == -math.inf).all() and (got[:n][empty] == 0).all()
        assert ((got_lse - lse).abs()[:n][~empty] <= 1e-4 + lse[:n][~empty].abs() * 2.0**-22).all()
        assert (op.out[n:] == 5.0).all() and (op.lse[n:] == 5.0).all()  # rows behind the batch stay


ATTN = {
    "one token alone": dict(kv=[1], new=[1], prefix=0, qh=1, kvh=1, dim=64, page=16),
    "window of 16 rows, page 1": dict(kv=[300], new=[16], prefix=0, qh=16, kvh=2, dim=64, page=1, window=127),
    "ragged decode behind a prefix": dict(kv=[200, 201, 330, 456, 700], new=[1] * 5, prefix=200, qh=16, kvh=2, dim=64, page=16),
    "prefix ends inside a page": dict(kv=[139, 150, 400], new=[2, 1, 3], prefix=137, qh=8, kvh=1, dim=128, page=64),
    "requests without rows, without keys": dict(kv=[300, 0, 257, 0, 260], new=[1, 0, 2, 1, 0], prefix=256, qh=14, kvh=2, dim=64, page=32),
    "fewer keys than rows": dict(kv=[2, 5, 130], new=[4, 5, 4], prefix=0, qh=8, kvh=2, dim=64, page=16),
    "a request shorter than the prefix": dict(kv=[500, 90, 400], new=[2, 2, 1], prefix=384, qh=8, kvh=1, dim=64, page=128),
    "every request shorter than the prefix": dict(kv=[50, 90], new=[2, 2], prefix=384, qh=8, kvh=1, dim=128, page=16),
    "one live request": dict(kv=[0, 400, 0], new=[0, 3, 0], prefix=256, qh=8, kvh=1, dim=64, page=16),
    "more than 256 rows a request": dict(kv=[700, 64, 300], new=[40, 33, 1], prefix=0, qh=16, kvh=2, dim=64, page=24),
    "17 heads a group, odd page": dict(kv=[260, 400], new=[5, 9], prefix=129, qh=34, kvh=2, dim=128, page=7),
    "window inside the prefix": dict(kv=[1000, 1010, 1300], new=[3, 1, 8], prefix=990, qh=8, kvh=1, dim=64, page=16, window=100),
    "window behind the prefix": dict(kv=[1000, 1500], new=[3, 1], prefix=300, qh=8, kvh=4, dim=128, page=8, window=250),
    "window of one key": dict(kv=[77, 300], new=[3, 1], prefix=0, qh=4, kvh=4, dim=64, page=16, window=1),
    "33 requests": dict(kv=[128 + 5 * i for i in range(33)], new=[1 + i % 3 for i in range(33)], prefix=128, qh=4, kvh=1, dim=64, page=16),
    "130 requests": dict(kv=[130 + i for i in range(130)], new=[1] * 130, prefix=128, qh=8, kvh=1, dim=64, page=128),
    "700 requests": dict(kv=[(37 * i) % 190 for i in range(700)], new=[min(i % 4, (37 * i) % 190) for i in range(700)], prefix=0, qh=8, kvh=2, dim=64,
                         page=16),
    "halves of a tile": dict(kv=[63, 64, 65, 127, 128, 129, 191, 192, 193], new=[4, 4, 4, 4, 4, 4, 4, 4, 4], prefix=0, qh=8, kvh=1, dim=64, page=16),
    "windows of half a tile": dict(kv=[200, 257, 320, 130], new=[16, 3, 1, 16], prefix=0, qh=8, kvh=1, dim=64, page=1, window=63),
    "windows of half a tile, wide": dict(kv=[200, 257, 320, 130], new=[16, 3, 1, 16], prefix=64, qh=8, kvh=2, dim=128, page=8, window=64),
    "nothing behind the prefix": dict(kv=[256, 256, 256], new=[1, 4, 2], prefix=256, qh=8, kvh=1, dim=64, page=16),
    "128 heads a group": dict(kv=[200, 300], new=[2, 1], prefix=160, qh=128, kvh=1, dim=128, page=16),
    "256 heads a group": dict(kv=[200, 300], new=[2, 1], prefix=0, qh=256, kvh=1, dim=64, page=16),
    "a million keys": dict(kv=[1000003], new=[2], prefix=0, qh=2, kvh=1, dim=64, page=128),
    "many splits of one item": dict(kv=[30000, 29000], new=[1, 1], prefix=28672, qh=8, kvh=1, dim=64, page=64),
    "tall prefix": dict(kv=[2100] * 9, new=[16] * 9, prefix=2048, qh=16, kvh=1, dim=128, page=128),
}  # fmt: skip


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("name", list(ATTN))
def test_attention(name, dt):
    c = AttnCase(len(name), dt=dt, rows=sum(ATTN[name]["new"]) + 3, layout="fused" if len(name) % 2 else "plain", **ATTN[name])
    op = c.bind()
    op.launch(stream())
    torch.cuda.synchronize()
    c.check(op)
    assert op.status[0].item() == 0
    first = op.out.clone(), op.lse.clone()
    op.launch(stream())
    torch.cuda.synchronize()
    assert torch.equal(op.out, first[0]) and torch.equal(op.lse, first[1])  # sums in a fixed order


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_scores_that_grow_along_the_keys(dim):
    """The running maximum moves in nearly every tile, by more and by less than the step that rescales O, down to -inf-like
    scores in front: keys along one direction with rising length."""
    c = AttnCase(4, kv=[900, 900], new=[2, 1], prefix=640, qh=8, kvh=1, dim=dim, page=16, dt=BF, q_mult=0.0)
    c.q[..., 0] = torch.linspace(0.2, 4.0, 8, device=DEV).to(BF)
    for b in range(2):
        p = torch.arange(900)
        s = (c.table[b, p // 16].long() * 16 + p % 16).to(DEV)
        c.k[s, 0, 0] = torch.linspace(-200, 200, 900, device=DEV).to(BF)
    op = c.bind()
    op.launch(stream())
    torch.cuda.synchronize()
    c.check(op)


def test_attention_non_finite_scores():
    """A NaN or +inf score makes its own row NaN and no other; -inf scores are keys of weight 0; the type's lowest value too."""
    c = AttnCase(5, kv=[300, 300], new=[4, 1], prefix=256, qh=2, kvh=1, dim=64, page=16, dt=BF)
    p = torch.arange(300)
    s = (c.table[0, p // 16].long() * 16 + p % 16).to(DEV)
    c.q[:, :, 0] = 1.0
    c.q[1, 0, 0], c.q[2, 1, 0] = math.nan, math.inf
    c.k[s[100], 0] = 0.0
    c.k[s[100], 0, 0] = torch.finfo(BF).min  # -2^125 or so times the scale: no weight
    op = c.bind()
    op.launch(stream())
    torch.cuda.synchronize()
    nan = torch.zeros(5, 2, dtype=torch.bool)
    nan[1, 0] = nan[2, 1] = True
    assert torch.equal(op.out.isnan().all(-1).cpu(), nan) and torch.equal(op.out.isnan().any(-1).cpu(), nan)
    assert torch.equal(op.lse.isnan().cpu(), nan)
    out, _, mass = R.attention(c.q, c.k, c.v, c.table, c.kv, c.cu, 16, 0.125, 0)
    ok = ~nan
    assert ((op.out.double().cpu() - out).abs() <= out.abs() * 2.0**-9 + mass * (2.0**-8 + 1e-4) + 1e-6)[ok].all()


def test_attention_bad_pages_and_lengths_are_recorded():
    base = dict(kv=[100, 120, 90], new=[1, 2, 1], prefix=64, qh=8, kvh=1, dim=64, page=16, dt=BF)
    c = AttnCase(6, **base)
    op = c.bind()
    c.lens["block_table"][1, 5] = 1 << 30  # an own page of request 1 outside the pool: its keys read as zero rows
    op.launch(stream())
    torch.cuda.synchronize()
    assert op.status[0].item() == 4 and torch.isfinite(op.out[:4]).all()
    out, _, _ = R.attention(c.q, c.k, c.v, c.table, c.kv, c.cu, 16, 0.125, 0)
    for r in (0, 3):  # the other requests are what they are
        assert (op.out[r].double().cpu() - out[r]).abs().max() < 0.05
    for bad in (dict(kv_lens=[100, 1 << 20, 90]), dict(cu_rows=[0, 1, 4, 5]), dict(prefix_len=[-3]), dict(cu_rows=[0, 1, 0, 1]),
                dict(cu_rows=[2**31 - 1, -(2**31), 3, 4]), dict(cu_rows=[0, 2**31 - 1, -(2**31), 4]), dict(cu_rows=[-5, -4, -2, 4])):
        c = AttnCase(6, **base)
        op = c.bind()
        for k, v in bad.items():
            c.lens[k].copy_(dev(v, I32))
        op.launch(stream())
        torch.cuda.synchronize()
        assert op.status[0].item() == 4, bad
        assert torch.isfinite(op.out).all()


def test_attention_captured_replays_follow_the_lengths():
    """One capture, replayed with other lengths, prefixes and row counts (padded requests); two captures of two binds interleave."""
    lib, module = ctx()
    kv = [[400, 300, 350, 290], [257, 0, 500, 288], [300, 310, 0, 0]]
    new = [[1, 3, 2, 1], [2, 0, 1, 1], [3, 1, 0, 0]]
    c = AttnCase(7, kv=[512] * 4, new=[3] * 4, prefix=256, qh=8, kvh=2, dim=64, page=16, dt=BF)
    a, b = c.bind(), c.bind()
    lens_b = c.lens
    a = BT.PrefixAttention(lib, module, q=c.q, k_cache=c.k, v_cache=c.v, page_size=16, max_new=3, scale=0.125, lse=True, **lens_b)
    graphs = []
    for op in (a, b):
        op.launch(stream())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            op.launch(stream())
        graphs.append(g)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for L, n, prefix in zip(kv, new, (256, 250, 0)):
        cu = [0]
        for x in n:
            cu.append(cu[-1] + x)
        lens_b["kv_lens"].copy_(dev(L, I32))
        lens_b["cu_rows"].copy_(dev(cu, I32))
        lens_b["prefix_len"].fill_(prefix)
        for op in (a, b):
            op.out.fill_(5.0)
            op.lse.fill_(5.0)
        torch.cuda.synchronize()
        for st, g in zip(s, graphs):  # both at once on two streams: each bind has its own scratch and outputs
            with torch.cuda.stream(st):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for op in (a, b):
            c.check(op, L, cu)
    for g in graphs:
        g.reset()


def test_attention_in_a_pool_beyond_32_bit_offsets():
    """Rows whose element offset passes 2^31 and whose byte offset passes 2^32."""
    kvh, dim, page = 8, 128, 16
    n_pages = 140000  # x 16 rows x 1024 elements = 2.29e9 elements, 4.6 GB a pool
    lib, module = ctx()
    g = torch.Generator().manual_seed(8)
    k, v = (torch.empty(n_pages * page, kvh, dim, dtype=BF, device=DEV) for _ in range(2))
    kv, new = [60, 70], [1, 2]
    table = torch.tensor([[n_pages - 1 - i for i in range(5)], [n_pages - 1, 3, n_pages - 9, 0, n_pages // 2]], dtype=I32)
    for b in range(2):
        p = torch.arange(kv[b])
        s = (table[b, p // page].long() * page + p % page).to(DEV)
        k[s], v[s] = torch.randn(2, kv[b], kvh, dim, generator=g).to(BF).to(DEV)
    q = torch.randn(3, 16, dim, generator=g).to(BF).to(DEV)
    op = BT.PrefixAttention(lib, module, q=q, k_cache=k, v_cache=v, block_table=table.to(DEV), kv_lens=dev(kv, I32), cu_rows=dev([0, 1, 3], I32),
                            prefix_len=dev([0], I32), page_size=page, max_new=2, scale=0.125)  # fmt: skip
    op.launch(stream())
    torch.cuda.synchronize()
    out, _, mass = R.attention(q, k, v, table, kv, [0, 1, 3], page, 0.125, 0)
    assert ((op.out.double().cpu() - out).abs() <= out.abs() * 2.0**-9 + mass * (2.0**-8 + 1e-4) + 1e-6).all()


# ---- the run of them --------------------------------------------------------------------------------------------------
def test_steps_of_a_batch():
    """Requests behind one prefix take steps of several tokens: tables, rotation with append and attention on the tables' own
    outputs, eager and as one captured step; each step's rows against the whole history in 64 bits. Some drafts are rejected
    between steps (a length goes back), one request ends and another joins in its place."""
    lib, module = ctx()
    g = torch.Generator(device=DEV).manual_seed(11)
    B, page, width, qh, kvh, D, prefix, rows = 4, 16, 12, 8, 2, 64, 48, 16
    pool = 6
    r2p = torch.full((pool, width), -1, dtype=I32, device=DEV)
    owned = torch.zeros(pool, dtype=I32, device=DEV)
    n_pages = 64
    ring = torch.randperm(n_pages, generator=g, device=DEV).int()
    words = dev([0, n_pages], I64)
    shared = ring[:3].clone()  # the prefix's pages are taken by hand
    words[0] += 3
    r2p[:, :3], owned[:] = shared, 3
    kc, vc = (torch.full((n_pages * page, kvh, D), math.nan, dtype=BF, device=DEV) for _ in range(2))
    hist = [[torch.randn(prefix, kvh, D, generator=g, device=DEV).to(BF) for _ in range(2)]] * pool  # rotated keys, values of each pool row
    at = (shared[:, None].long() * page + torch.arange(page, device=DEV)).flatten()
    kc[at], vc[at] = hist[0]
    seq, new, req = (torch.zeros(B, dtype=I64, device=DEV) for _ in range(3))
    tab = BT.BlockTables(lib, module, seq_lens=seq, new_lens=new, req_pool_indices=req, req_to_page=r2p, pages_owned=owned, free_pages=ring,
                         free_words=words, page_size=page, rows=rows)  # fmt: skip
    rope = BT.RopeTable(lib, module, rows=width * page, rot=D, theta=1e4, device=DEV)
    rope.launch(stream())
    qkv = torch.zeros(rows, (qh + 2 * kvh) * D, dtype=BF, device=DEV)
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([qh * D, kvh * D, kvh * D], 1))
    rot = BT.Rotary(lib, module, q=q, k=k, v=v, positions=tab.positions, cos_sin_cache=rope.cos_sin, slots=tab.slots, k_cache=kc, v_cache=vc,
                    n_rows=tab.cu_rows[B:])  # fmt: skip
    att = BT.PrefixAttention(lib, module, q=rot.q_out, k_cache=kc, v_cache=vc, block_table=tab.block_table, kv_lens=tab.kv_lens,
                             cu_rows=tab.cu_rows, prefix_len=dev([prefix], I32), page_size=page, max_new=8, scale=0.125)  # fmt: skip
    ops = (tab, rot, att)

    def step(pdl):
        for op in ops:
            op.launch(stream(), pdl)

    lens, reqs = [prefix] * B, [0, 1, 2, 3]
    graph = None
    for turn, take in enumerate([[1, 5, 8, 2], [3, 0, 1, 8], [8, 1, 2, 1], [1, 1, 1, 1], [2, 7, 0, 4]]):
        if turn == 3:  # request 1 ends: its own pages go back behind the ring's tail; pool row 4 joins
            give = r2p[1, 3 : int(owned[1])].clone()
            tail = int(words[1])
            ring[(tail + torch.arange(give.numel(), device=DEV)) % n_pages] = give
            words[1] += give.numel()
            owned[1] = 3
            reqs[1], lens[1] = 4, prefix
        seq.copy_(dev(lens, I64))
        new.copy_(dev(take, I64))
        req.copy_(dev(reqs, I64))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=DEV))
        att.out.fill_(3.0)
        if turn < 2:
            step(pdl=turn == 1)
        else:
            if graph is None:
                s = torch.cuda.Stream()
                graph = torch.cuda.CUDAGraph()
                torch.cuda.synchronize()
                with torch.cuda.graph(graph, stream=s):
                    step(pdl=True)
            graph.replay()
        torch.cuda.synchronize()
        assert all(op.status[0].item() == 0 for op in ops)
        r = 0
        cos_sin = rope.cos_sin.cpu()
        for b in range(B):
            pos = torch.arange(lens[b], lens[b] + take[b])
            rk = R.rotate(k[r : r + take[b]], cos_sin[pos], False, False).to(BF).to(DEV)
            hk, hv = hist[reqs[b]]
            hk, hv = torch.cat((hk[: lens[b]], rk)), torch.cat((hv[: lens[b]], v[r : r + take[b]]))
            hist = hist[: reqs[b]] + [[hk, hv]] + hist[reqs[b] + 1 :]
            rq = R.rotate(q[r : r + take[b]], cos_sin[pos], False, False).to(BF).to(DEV)
            n = hk.shape[0]
            ref, _, mass = R.attention(rq, hk, hv, torch.arange(n)[None], [n], [0, take[b]], 1, 0.125, 0)
            got = att.out[r : r + take[b]].double().cpu()
            # the reference's rounding of q and k may differ from the kernel's by one step where f32 falls on the other side: two
            # steps of 2^-8 on a score's terms, which come to less than 8
            assert ((got - ref).abs() <= ref.abs() * 2.0**-9 + mass * (2.0**-8 + 2 * 8 * 2.0**-8) + 1e-6).all()
            r += take[b]
        assert (att.out[r:] == 3.0).all()
        # two of the new tokens of each request are rejected where it brought more than two
        lens = [n + t - (2 if t > 2 else 0) for n, t in zip(lens, take)]
    graph.reset()
    used = torch.cat([r2p[x, 3 : int(owned[x])] for x in range(pool) if x != 1]).tolist()
    free = [int(ring[i % n_pages]) for i in range(int(words[0]), int(words[1]))]
    assert sorted(used + free + shared.tolist()) == list(range(n_pages))  # no page lost, none twice


def test_binds_refuse_host_memory():
    lib, module = ctx()
    with pytest.raises(RuntimeError, match="device"):
        BT.RopeTable(lib, module, rows=5, rot=64, theta=1e4, device="cpu")
