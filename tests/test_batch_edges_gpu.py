"""The batched step's attention at the edges of what its rows see: keys in front of every window, infinite scores, scores far from
zero, many keys of little weight, lengths that contradict the extents. Plain 64-bit forms: ``batch_ref.py``."""

import math

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


def dev(x, dtype):
    return torch.tensor(x, dtype=dtype, device=DEV)


class Batch:
    """`kv[b]` keys and `new[b]` rows a request; the whole pages of the first `prefix` keys are shared, the others lie in random
    order, and the shared keys' values are the same in each request. The pool is finite everywhere."""

    def __init__(self, seed, kv, new, prefix, qh, kvh, dim, page, dt, window=0, q_std=1.0):
        g = torch.Generator().manual_seed(seed)
        self.kv, self.new, self.prefix, self.page, self.window, self.dt = kv, new, prefix, page, window, dt
        shared, pages = prefix // page, [-(-n // page) for n in kv]
        total = shared + sum(max(p - shared, 0) for p in pages)
        ids = torch.randperm(total, generator=g).tolist()
        common, width = [ids.pop() for _ in range(shared)], max(pages)
        rows = [common[: min(p, shared)] + [ids.pop() for _ in range(max(p - shared, 0))] for p in pages]
        self.table = torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=I32)
        self.k, self.v = (torch.randn(total * page, kvh, dim, generator=g).to(dt).to(DEV) for _ in range(2))
        if prefix % page:
            body = torch.randn(2, prefix % page, kvh, dim, generator=g).to(dt).to(DEV)
            for b in range(len(kv)):
                n = min(prefix, kv[b]) - shared * page
                if n > 0:
                    s = self.slots(b, range(shared * page, shared * page + n))
                    self.k[s], self.v[s] = body[0, :n], body[1, :n]
        self.cu = [0]
        for n in new:
            self.cu.append(self.cu[-1] + n)
        self.q = (torch.randn(self.cu[-1], qh, dim, generator=g) * q_std).to(dt).to(DEV)

    def slots(self, b, keys):
        p = torch.tensor(list(keys))
        return (self.table[b, p // self.page].long() * self.page + p % self.page).to(DEV)

    def launch(self, **over):
        lib = host.library()
        self.lens = dict(block_table=self.table.to(DEV), kv_lens=dev(self.kv, I32), cu_rows=dev(self.cu, I32), prefix_len=dev([self.prefix], I32))
        self.lens.update(over)
        op = BT.PrefixAttention(lib, lib.load(), q=self.q, k_cache=self.k, v_cache=self.v, page_size=self.page, max_new=max(self.new),
                                scale=0.125, window=self.window, lse=True, **self.lens)  # fmt: skip
        op.out.fill_(5.0)
        op.lse.fill_(5.0)
        op.launch(stream())
        torch.cuda.synchronize()
        return op

    def want(self):
        return R.attention(self.q, self.k, self.v, self.table, self.kv, self.cu, self.page, 0.125, self.window)

    def check(self, op, rows=slice(None)):
        """The probabilities are rounded to the type once and the result once; f32 sums and the exponential are good to 1e-4 of the
        weighted mean of |v| (scores of a few dozen: 2^-19 in the exponent, an exponential good to 4e-6). In f16 a probability has
        a fixed step of 2^-24 below 2^-14; a row's largest is at least 2^7, so half such steps of all keys come to less than
        keys x 2^-32 x 5."""
        out, lse, mass = self.want()
        eps = torch.finfo(self.dt).eps / 2
        tol = out.abs() * eps + mass * (eps + 1e-4) + 1e-6 + (max(self.kv) * 2.0**-32 * 5 if self.dt == HF else 0.0)
        err = (op.out.double().cpu() - out).abs()
        assert (err <= tol)[rows].all(), float((err - tol)[rows].max())
        assert ((op.lse.double().cpu() - lse).abs() <= 1e-4 + lse.abs() * 2.0**-22)[rows].all()


# ---- many keys of little weight ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [BF, HF])
def test_many_keys_of_little_weight(dt):
    """Two keys of weight 1 beside 32,766 of 2^-25.2 each, 4e-4 of the row together, by one CTA: they stay in the result."""
    n, B, page = 32768, 160, 128
    k, v = torch.zeros(n, 1, 64, dtype=dt, device=DEV), torch.ones(n, 1, 64, dtype=dt, device=DEV)
    k[..., 0] = -140.0  # a score of -17.5
    for one in (3, 200):  # a tile of each parity
        k[one], v[one] = 0.0, 0.0
    q = torch.zeros(B, 1, 64, dtype=dt, device=DEV)
    q[..., 0] = 1.0
    table = torch.arange(n // page, dtype=I32, device=DEV).repeat(B, 1)
    lib = host.library()
    op = BT.PrefixAttention(lib, lib.load(), q=q, k_cache=k, v_cache=v, block_table=table, kv_lens=dev([n] * B, I32),
                            cu_rows=dev(list(range(B + 1)), I32), prefix_len=dev([0], I32), page_size=page, max_new=1, scale=0.125, lse=True)  # fmt: skip
    op.launch(stream())
    torch.cuda.synchronize()
    low = (n - 2) * math.exp(-17.5)
    out = low / (2 + low)
    # a probability's rounding (f16: half a step of 2^-24 of the 2^7 that the largest is held at, over a sum of 2), the result's (f16 has a
    # step of 2^-24 here too); the exponential 4e-6, f32 sums of 32 K values 2^-17
    step = n * 2.0**-33 + 2.0**-25 if dt == HF else out * 2.0**-9
    assert ((op.out.double() - out).abs() <= out * (torch.finfo(dt).eps / 2 + 2.0**-16) + step).all()
    assert ((op.lse.double() - math.log(2 + low)).abs() <= 2.0**-16).all()


# ---- keys in front of every window ------------------------------------------------------------------------------------
FRONT = {
    "inside the prefix": dict(kv=[700, 705, 760], new=[2, 1, 3], prefix=640, window=100),  # first key that a row sees: 598
    "inside the prefix, more rows than a block": dict(kv=[700, 705, 760], new=[40, 1, 3], prefix=640, window=90),
    "behind the prefix": dict(kv=[700, 900], new=[2, 1], prefix=300, window=77),
    "alone": dict(kv=[700], new=[16], prefix=0, window=127),
    "no prefix": dict(kv=[700, 431, 90], new=[3, 1, 2], prefix=0, window=50),
}


@pytest.mark.parametrize("dt,dim", [(BF, 64), (HF, 64), (BF, 128)])
@pytest.mark.parametrize("page", [1, 7, 8, 16, 24, 128])
@pytest.mark.parametrize("name", list(FRONT))
def test_keys_in_front_of_every_window(name, page, dt, dim):
    """Rows that no window reaches are not read: NaN and infinities there change nothing, neither do page ids outside the pool for
    pages that have slid out of every window."""
    c = Batch(page, qh=8, kvh=1, dim=dim, page=page, dt=dt, **FRONT[name])
    firsts = [max(0, n - m - c.window) for n, m in zip(c.kv, c.new)]
    low = min(firsts)
    for b, n in enumerate(c.kv):
        gone = [k for k in range(n) if k < low or c.prefix <= k < firsts[b]]
        if gone:
            s = c.slots(b, gone)
            c.k[s], c.v[s] = math.nan, math.nan
            c.v[s[::2]] = math.inf
    clean = c.table.clone()
    for b in range(len(c.kv)):
        for p in range(clean.shape[1]):
            last = (p + 1) * page - 1  # the page's last key
            if last < low or (p * page >= c.prefix and last < firsts[b]):
                c.table[b, p] = -1 if p % 2 else 1 << 30
    op = c.launch()
    assert op.status[0].item() == 0
    c.table = clean
    c.check(op)


# ---- scores of -inf ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 1), (128, 64)])
def test_scores_of_minus_infinity(dt, dim, page):
    """A key whose score is -inf has weight 0, whatever its V row holds; a row that has only such keys is 0 with lse -inf."""
    c = Batch(3, kv=[700, 640, 650], new=[2, 1, 2], prefix=384, qh=8, kvh=1, dim=dim, page=page, dt=dt)
    c.q[:, :, 0] = 1.0
    big = torch.finfo(dt).max
    for b, keys in ((0, [5, 200, 383, 384, 500]), (2, range(384, 600))):  # shared and own ones; whole tiles of request 2
        s = c.slots(b, keys)
        c.k[s, :, 0], c.v[s] = -math.inf, big
    op = c.launch()
    c.check(op)
    for b in range(3):  # and now all of them, in tiles that nothing masks
        c.k[c.slots(b, range(c.kv[b])), :, 0] = -math.inf
    c.k[c.slots(1, [639]), :, 0] = 0.0  # the one key that request 1's row keeps
    op = c.launch()
    out, lse = op.out.double().cpu(), op.lse.double().cpu()
    for r in (0, 1, 3, 4):
        assert (out[r] == 0).all() and (lse[r] == -math.inf).all(), r
    assert torch.equal(op.out[2], c.v[c.slots(1, [639])][0].expand(8, dim)) and op.status[0].item() == 0


# ---- scores far from zero ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt,length,step", [(BF, 2.0**8, 8.0), (HF, 2.0**8, 8.0), (BF, 2.0**11, 64.0), (HF, 2.0**11, 64.0), (BF, 2.0**15, 512.0),
                                            (HF, 2.0**15, 512.0), (BF, 2.0**30, 2.0**40)])  # fmt: skip
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_far_from_zero(dt, length, step, sign, dim):
    """Only the scores' differences count: up to 3 length^2 / 8 with steps of `step` / 8 between the keys, all of them exact in f32.
    Some references are large enough that a rounded one would be off by more than f16's or f32's exponents."""
    c = Batch(7, kv=[900, 800, 555], new=[2, 1, 3], prefix=512, qh=8, kvh=1, dim=dim, page=16, dt=dt)
    g = torch.Generator().manual_seed(int(math.log2(length)))
    c.q.zero_()
    c.k.zero_()
    c.q[..., :3] = (length * (1 - torch.arange(8) / 32.0))[None, :, None].to(dt).to(DEV)  # a length of its own for each head
    c.q[..., 3] = math.sqrt(step) if step > 2.0**16 else 1.0
    c.k[..., :3] = sign * length
    level = torch.randint(-8, 9, c.k.shape[:2], generator=g).to(DEV)
    c.k[..., 3] = (level * (step / c.q[0, 0, 3].double())).to(dt)
    op = c.launch()
    assert torch.isfinite(op.out).all() and op.status[0].item() == 0
    c.check(op)


# ---- lengths that contradict the extents ------------------------------------------------------------------------------
@pytest.mark.parametrize("change,out", [
    (dict(kv_lens=[700, 1 << 20, 650]), [1]), (dict(kv_lens=[-1, 640, 650]), [0]), (dict(cu_rows=[0, 2, 6, 7]), [1]),
    (dict(prefix_len=[-3]), []), (dict(prefix_len=[1 << 20]), []), (dict(cu_rows=[0, 2, 3, 9]), [0, 1, 2]),
    (dict(cu_rows=[-2, 0, 3, 6]), [0]),
])  # fmt: skip
@pytest.mark.parametrize("dim", [64, 128])
def test_lengths_that_contradict_the_extents(change, out, dim):
    """A request left out keeps its rows as they were, the others are what they are."""
    c = Batch(9, kv=[700, 640, 650], new=[2, 1, 3], prefix=384, qh=8, kvh=2, dim=dim, page=16, dt=BF)
    cu = change.get("cu_rows", c.cu)
    c.q = torch.cat((c.q, c.q[:1]))  # 7 rows
    op = c.launch(**{k: dev(v, I32) for k, v in change.items()})
    assert op.status[0].item() == 4
    c.cu = [0, 2, 3, 6] if cu[3] > 7 else [max(x, 0) for x in cu]
    rows = torch.zeros(7, dtype=torch.bool)
    for b in range(3):
        if b not in out:
            rows[c.cu[b] : c.cu[b + 1]] = True
    for b in out:  # the plain form takes no request that is left out
        c.kv = [n if i != b else 0 for i, n in enumerate(c.kv)]
    assert (op.out[~rows] == 5.0).all() and (op.lse[~rows.to(DEV)] == 5.0).all()
    if rows.any():
        c.check(op, rows)


def test_requests_that_name_more_rows_than_there_are():
    """Requests over and over on the same rows: nothing is done, and it is recorded. (Steps are counted in 32 bits, which the bind
    provides for as far as requests share the rows out.)"""
    B, rows, width = 4095, 256, 8192
    lib = host.library()
    q = torch.ones(rows, 8, 64, dtype=BF, device=DEV)
    kv = torch.ones(128, 8, 64, dtype=BF, device=DEV)
    cu = torch.zeros(B + 1, dtype=I32, device=DEV)
    cu[1::2] = rows
    op = BT.PrefixAttention(lib, lib.load(), q=q, k_cache=kv, v_cache=kv.clone(), block_table=torch.zeros(B, width, dtype=I32, device=DEV),
                            kv_lens=torch.full((B,), width * 128, dtype=I32, device=DEV), cu_rows=cu, prefix_len=dev([0], I32), page_size=128,
                            max_new=rows, scale=0.125)  # fmt: skip
    op.out.fill_(5.0)
    op.launch(stream())
    torch.cuda.synchronize()
    assert (op.out == 5.0).all() and op.status[:2].tolist() == [4, 520]  # the first to be recorded: every second request's rows


# ---- a step's own tensors ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt,dim,page", [(BF, 64, 16), (HF, 128, 1), (HF, 64, 24)])
def test_steps_on_the_pool_as_it_stands(dt, dim, page):
    """Three captured steps of tables, rotation with append and attention: the attention against the rotated rows, pool and tables that
    the launches in front of it left, so no rounding of theirs has to be allowed for."""
    lib = host.library()
    module = lib.load()
    g = torch.Generator(device=DEV).manual_seed(12)
    B, qh, kvh, prefix, rows = 5, 8, 2, 96, 24
    width, pool = -(-200 // page), 7
    n_pages = pool * width
    ring = torch.randperm(n_pages, generator=g, device=DEV).int()
    shared = prefix // page
    r2p = torch.full((pool, width), -1, dtype=I32, device=DEV)
    r2p[:, :shared] = ring[:shared]
    owned = torch.full((pool,), shared, dtype=I32, device=DEV)
    words = dev([shared, n_pages], I64)
    kc, vc = (torch.full((n_pages * page, kvh, dim), math.nan, dtype=dt, device=DEV) for _ in range(2))
    at = (ring[:shared, None].long() * page + torch.arange(page, device=DEV)).flatten()
    kc[at], vc[at] = (torch.randn(len(at), kvh, dim, generator=g, device=DEV).to(dt) for _ in range(2))
    lens = [shared * page] * B
    seq, new, req = dev(lens, I64), dev([0] * B, I64), dev([3, 0, 6, 1, 4], I64)
    tab = BT.BlockTables(lib, module, seq_lens=seq, new_lens=new, req_pool_indices=req, req_to_page=r2p, pages_owned=owned, free_pages=ring,
                         free_words=words, page_size=page, rows=rows)  # fmt: skip
    rope = BT.RopeTable(lib, module, rows=width * page, rot=dim, theta=5e5, device=DEV)
    rope.launch(stream())
    qkv = torch.zeros(rows, (qh + 2 * kvh) * dim, dtype=dt, device=DEV)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([qh * dim, kvh * dim, kvh * dim], 1))
    rot = BT.Rotary(lib, module, q=q, k=k, v=v, positions=tab.positions, cos_sin_cache=rope.cos_sin, slots=tab.slots, k_cache=kc, v_cache=vc,
                    n_rows=tab.cu_rows[B:], interleaved=True)  # fmt: skip
    att = BT.PrefixAttention(lib, module, q=rot.q_out, k_cache=kc, v_cache=vc, block_table=tab.block_table, kv_lens=tab.kv_lens,
                             cu_rows=tab.cu_rows, prefix_len=dev([shared * page], I32), page_size=page, max_new=8, scale=0.125, lse=True)  # fmt: skip
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        for op in (tab, rot, att):
            op.launch(stream(), True)
    c = Batch.__new__(Batch)
    c.k, c.v, c.page, c.window, c.dt = kc, vc, page, 0, dt
    for take in ([8, 1, 3, 5, 7], [1, 0, 8, 2, 1], [4, 4, 1, 8, 6]):
        new.copy_(dev(take, I64))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=DEV))
        att.out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(op.status[0].item() == 0 for op in (tab, rot, att))
        c.q, c.table, c.kv, c.cu = rot.q_out, tab.block_table.cpu(), tab.kv_lens.tolist(), tab.cu_rows.tolist()
        n = sum(take)
        assert c.cu[-1] == n and c.kv == [a + b for a, b in zip(lens, take)] and (att.out[n:] == 5.0).all()
        c.check(att, slice(0, n))
        lens = c.kv
        seq.copy_(dev(lens, I64))
    graph.reset()


# ---- long rows, rows that see a NaN -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [BF, HF])
def test_a_million_keys(dt):
    """Against outputs of a few hundredths, with the bound of every other case."""
    c = Batch(10, kv=[1000003], new=[2], prefix=0, qh=2, kvh=1, dim=64, page=128, dt=dt, q_std=3.0)
    c.check(c.launch())


@pytest.mark.parametrize("dim,window", [(64, 0), (64, 200), (128, 0)])
def test_a_nan_in_a_key_reaches_the_rows_that_see_it(dim, window):
    """The second of a request's four new keys, and a shared key that some windows have left behind."""
    c = Batch(11, kv=[700, 640, 650], new=[4, 1, 2], prefix=512, qh=8, kvh=2, dim=dim, page=16, dt=BF, window=window)
    shared = 490  # in front of what the first request's rows see through a window of 200 (496 and on), not of what the others' see
    at = [(0, 697)] + [(b, shared) for b in range(3)]
    for b, key in at:
        c.k[c.slots(b, [key])] = math.nan
    op = c.launch()
    hit = torch.zeros(7, dtype=torch.bool)
    hit[1:4] = True
    if window == 0:
        hit[:] = True
    else:
        hit[4:] = True
    assert torch.equal(op.out.isnan().flatten(1).all(1).cpu(), hit) and torch.equal(op.out.isnan().flatten(1).any(1).cpu(), hit)
    for b, key in at:  # the plain form multiplies by zero too
        c.k[c.slots(b, [key])] = 0.0
    if window:
        c.check(op, ~hit)
