"""What the kernels of the batched decode step are measured on: cases, inputs, plain forms and 64-bit definitions.

Four operators (``sgl_muse_mega_b200/muse_spark/b200/batch.py``), in the order a batched step runs them:

* ``tables``     pages, slots and positions of a step's new tokens from the requests' lengths (``BlockTables``)
* ``rope_table`` cos | sin rows of a position range, with the usual scalings for long contexts (``RopeTable``)
* ``rotary``     rotation of q and k, store of q, append of k and v at their slots (``Rotary``)
* ``attention``  the batch's new rows over the paged cache, whose first ``prefix`` tokens all requests share
                 (``PrefixAttention``)

``run`` computes a case in its plain form (elementary torch operations) or, with ``own`` set, through the framework's
launches, which ``prepare`` has bound to the inputs as a serving process binds them once.
"""

import math

import torch

own = False

# heads of one rank of the target (128 / 16 heads of 64 over 8 or 1 ranks) and of its draft (64 / 8 heads of 128)
THETA = 500000.0


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one request's 16-row verify window on the framework's token-granular request table (page size 1)
        dict(name="tables_window_b1", op="tables", batch=1, lo=8192, hi=8192, new_lo=16, new_hi=16, page=1, spare=0),
        # a decode step of a large batch with contexts up to 32 K tokens, pages of 16
        dict(name="tables_decode_b256", op="tables", batch=256, lo=1, hi=32768, new_lo=1, new_hi=1, page=16, spare=0),
        # prompts of odd lengths enter a batch (chunked prefill), pages of 64, row buffers that are larger than the step
        dict(name="tables_prefill_b61", op="tables", batch=61, lo=0, hi=5000, new_lo=0, new_hi=2047, page=64, spare=777),
        # the target's rope cache for an 8 K context
        dict(name="rope_table_8k", op="rope_table", rows=8448, rot=64, theta=THETA, kind="none", factor=1.0),
        # a 128 K context reached by yarn scaling (x 16 of an 8 K model), heads of 128
        dict(name="rope_table_131k_yarn", op="rope_table", rows=131072, rot=128, theta=10000.0, kind="yarn", factor=16.0),
        # the 16 rows of a verify window, one rank's heads
        dict(name="rotary_window16", op="rotary", rows=16, live=16, qh=16, kvh=2, dim=64, rot=64, inter=False, inverse=False,
             fp16=False, max_pos=8448),
        # a padded decode batch, the interleaved layout over half of a 128-wide head
        dict(name="rotary_decode_inter", op="rotary", rows=256, live=237, qh=64, kvh=8, dim=128, rot=64, inter=True,
             inverse=False, fp16=True, max_pos=32768),
        # a prefill chunk of the whole model's heads
        dict(name="rotary_prefill", op="rotary", rows=8192, live=8192, qh=128, kvh=16, dim=64, rot=64, inter=False,
             inverse=False, fp16=False, max_pos=131072),
        # one request's verify window on a sliding-window layer: the smallest call, bound by latency
        dict(name="attn_window_b1", op="attention", batch=1, prefix=0, lo=8192, hi=8192, new=16, qh=16, kvh=2, dim=64, page=1,
             window=2047, fp16=False, lse=False),
        # a decode batch behind one 8 K system prompt, answers of up to 1000 tokens so far
        dict(name="attn_decode_b64", op="attention", batch=64, prefix=8192, lo=1, hi=1000, new=1, qh=16, kvh=2, dim=64, page=16,
             window=0, fp16=False, lse=True),
        # 32 verify windows over one 32 K document (one rank's heads): bound by arithmetic
        dict(name="attn_verify_b32", op="attention", batch=32, prefix=32768, lo=16, hi=700, new=16, qh=16, kvh=2, dim=64, page=64,
             window=0, fp16=False, lse=False),
        # long answers of their own behind a short shared prefix, the draft's heads: bound by the cache's bytes
        dict(name="attn_suffix_b96", op="attention", batch=96, prefix=1021, lo=33, hi=4096, new=1, qh=64, kvh=8, dim=128, page=32,
             window=0, fp16=True, lse=False),
    ]  # fmt: skip


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tables", "rope_table", "rotary", "attention", "attention", "attention"])
    if op == "tables":
        lo = rng.choice([0, 1, 100])
        return dict(op=op, batch=_log(rng, 1, 256), lo=lo, hi=lo + _log(rng, 1, 16000), new_lo=rng.choice([0, 1]),
                    new_hi=_log(rng, 1, 512), page=rng.choice([1, 7, 16, 64, 128]), spare=rng.choice([0, 5, 100]))  # fmt: skip
    if op == "rope_table":
        return dict(op=op, rows=_log(rng, 1, 131072), rot=rng.choice([16, 32, 64, 80, 128]), theta=rng.choice([10000.0, THETA]),
                    kind=rng.choice(["none", "linear", "ntk", "llama3", "yarn"]), factor=rng.choice([1.5, 4.0, 16.0]))  # fmt: skip
    if op == "rotary":
        rows = _log(rng, 1, 4096)
        qh, kvh = rng.choice([(16, 2), (8, 1), (64, 8), (5, 5), (12, 4)])
        dim = rng.choice([64, 80, 128, 256])
        rot = rng.choice([r for r in (16, 24, 32, 64, 80, 128) if r <= dim])
        return dict(op=op, rows=rows, live=max(1, rows - rng.choice([0, 0, 1, 37])), qh=qh, kvh=kvh, dim=dim, rot=rot,
                    inter=rng.random() < 0.5, inverse=rng.random() < 0.3, fp16=rng.random() < 0.5,
                    max_pos=_log(rng, 64, 131072))  # fmt: skip
    dim, new = rng.choice([64, 128]), rng.choice([1, 1, 2, 5, 8, 16])
    qh, kvh = rng.choice([(16, 2), (8, 1), (16, 16), (14, 2), (32, 4)])
    batch, hi = _log(rng, 1, 64), _log(rng, 32, 2000)
    return dict(op="attention", batch=batch, prefix=rng.choice([0, _log(rng, 1, 32768 // max(1, new * batch * qh // 2048))]),
                lo=min(hi, new + rng.choice([0, 0, 20])), hi=max(hi, new), new=new, qh=qh, kvh=kvh, dim=dim,
                page=rng.choice([1, 16, 24, 64, 128]), window=rng.choice([0, 0, 127, 2047]), fp16=rng.random() < 0.4,
                lse=rng.random() < 0.5)  # fmt: skip


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def _lens(lo, hi, n, g):
    """n lengths in lo .. hi; the longest is there, so that every seed costs the same buffers."""
    x = torch.randint(lo, hi + 1, (n,), generator=g)
    x[n // 2] = hi
    return x


def _tables_state(c, seed):
    g = _gen(seed, "cpu")
    B, ps = c["batch"], c["page"]
    seq, new = _lens(c["lo"], c["hi"], B, g), _lens(c["new_lo"], c["new_hi"], B, g)
    width = -(-(c["hi"] + c["new_hi"]) // ps)
    pool = B + 3
    owned_b = -(-seq // ps)
    # some requests still hold the pages of rejected draft tokens
    owned_b = torch.minimum(owned_b + (torch.rand(B, generator=g) < 0.25).long(), torch.full((B,), width))
    n_pages = pool * width
    ids = torch.randperm(n_pages, generator=g).int()
    idx = torch.randperm(pool, generator=g)[:B]
    req_to_page = torch.full((pool, width), -1, dtype=torch.int32)
    owned = torch.zeros(pool, dtype=torch.int32)
    owned[idx] = owned_b.int()
    req_to_page[torch.arange(width)[None] < owned[:, None]] = ids[: int(owned_b.sum())]
    ring = torch.full((n_pages,), -1, dtype=torch.int32)
    left = ids[int(owned_b.sum()) :]
    head = int(torch.randint(0, n_pages, (1,), generator=g))  # the ring's free part may wrap around
    ring[(head + torch.arange(left.numel())) % n_pages] = left
    rows = B * c["new_hi"] + c["spare"]  # the buffers hold the largest step, most steps leave their end as it was
    s = dict(seq_lens=seq, new_lens=new, req_pool_indices=idx, req_to_page=req_to_page, pages_owned=owned, free_pages=ring,
             free_words=torch.tensor([head, head + left.numel()]))  # fmt: skip
    s = {k: v.cuda() for k, v in s.items()}
    return dict(s, rows=rows, page=ps)


def _rotary_state(c, seed):
    g = _gen(seed)
    dt = torch.float16 if c["fp16"] else torch.bfloat16
    R, qh, kvh, D = c["rows"], c["qh"], c["kvh"], c["dim"]
    # one fused projection row [q | k | v] per token, as the qkv GEMM leaves it
    row = torch.randn(R, (qh + 2 * kvh) * D, generator=g, device="cuda").to(dt)
    slots = torch.randperm(R + 64, generator=g, device="cuda")[:R]
    pos = torch.randint(0, c["max_pos"], (R,), generator=g, device="cuda")
    ang = torch.arange(c["max_pos"], device="cuda", dtype=torch.float64)[:, None] * (
        THETA ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"]))
    table = torch.cat((ang.cos(), ang.sin()), 1).float()
    q, k, v = (t.unflatten(1, (-1, D)) for t in row.split([qh * D, kvh * D, kvh * D], 1))
    cache = [torch.randn(R + 64, kvh, D, generator=g, device="cuda").to(dt) for _ in range(2)]
    n = torch.tensor([c["live"]], dtype=torch.int32, device="cuda")
    return dict(q=q, k=k, v=v, positions=pos, cos_sin_cache=table, slots=slots, k_cache=cache[0], v_cache=cache[1], n_rows=n)


def _attn_state(c, seed):
    g, gc = _gen(seed), _gen(seed, "cpu")
    dt = torch.float16 if c["fp16"] else torch.bfloat16
    B, n, ps, P, D, kvh = c["batch"], c["new"], c["page"], c["prefix"], c["dim"], c["kvh"]
    own_len = _lens(c["lo"], c["hi"], B, gc)
    kv = P + own_len
    width = -(-int(P + c["hi"]) // ps)
    shared = P // ps  # whole pages are shared; the prefix's last tokens may sit in a page of each request's own ...
    pages = -(-kv // ps)
    total = shared + int((pages - shared).sum())
    ids = torch.randperm(total, generator=gc).int()
    table = torch.full((B, width), -1, dtype=torch.int32)
    table[:, :shared] = ids[:shared]
    mask = (torch.arange(width)[None] >= shared) & (torch.arange(width)[None] < pages[:, None])
    table[mask] = ids[shared:]
    slots = total * ps
    # queries and keys as the qk norm leaves them: rows of unit mean square, queries scaled by 43.78 / sqrt(dim)
    q = torch.randn(B * n, c["qh"], D, generator=g, device="cuda")
    q = (q * torch.rsqrt(q.square().mean(-1, keepdim=True)) * (43.7840518911 / math.sqrt(D))).to(dt)
    k = torch.empty(slots, kvh, D, dtype=dt, device="cuda")
    v = torch.empty_like(k)
    for t in (k, v):
        for a in range(0, slots, 1 << 16):
            m = min(1 << 16, slots - a)
            t[a : a + m] = torch.randn(m, kvh, D, generator=g, device="cuda").to(dt)
    table = table.cuda()
    if P % ps:  # ... with the same contents in each
        p = torch.arange(shared * ps, P, device="cuda")
        src = table[0, p // ps].long() * ps + p % ps
        dst = table[:, shared].long()[:, None] * ps + (p % ps)[None]
        k[dst], v[dst] = k[src][None], v[src][None]
    return dict(q=q, k_cache=k, v_cache=v, block_table=table, kv_lens=kv.int().cuda(),
                cu_rows=(torch.arange(B + 1) * n).int().cuda(), prefix_len=torch.tensor([P], dtype=torch.int32).cuda(),
                lens=[int(x) for x in kv])  # fmt: skip


def _scaling(c):
    kind, f = c["kind"], c["factor"]
    return {"none": None, "linear": dict(kind="linear", factor=f), "ntk": dict(kind="ntk", factor=f),
            "llama3": dict(kind="llama3", factor=f, low_freq_factor=1.0, high_freq_factor=4.0, original_len=8192),
            "yarn": dict(kind="yarn", factor=f, beta_fast=32.0, beta_slow=1.0, original_len=8192)}[kind]  # fmt: skip


def prepare(case, seed):
    c = case
    if c["op"] == "tables":
        s = _tables_state(c, seed)
        if not own:
            z = torch.zeros(s["rows"], dtype=torch.int64, device="cuda")
            s.update(slots=z, positions=z.clone())
    elif c["op"] == "rope_table":
        s = dict(first=(seed % 977) * 16)  # tables may start anywhere: a rank of a sequence-parallel world, a shifted window
    elif c["op"] == "rotary":
        s = _rotary_state(c, seed)
        if not own:
            s.update(q_out=torch.zeros(c["rows"], c["qh"], c["dim"], dtype=s["q"].dtype, device="cuda"))
    else:
        s = _attn_state(c, seed)
    s["case"] = c
    if own:
        from sgl_muse_mega_b200.common import host
        from sgl_muse_mega_b200.muse_spark.b200 import batch as BT

        lib = host.library()
        module = lib.load()
        if c["op"] == "tables":
            keys = ("seq_lens", "new_lens", "req_pool_indices", "req_to_page", "pages_owned", "free_pages", "free_words")
            s["launch"] = BT.BlockTables(lib, module, **{k: s[k] for k in keys}, page_size=c["page"], rows=s["rows"])
        elif c["op"] == "rope_table":
            s["launch"] = BT.RopeTable(lib, module, rows=c["rows"], rot=c["rot"], theta=c["theta"], scaling=_scaling(c),
                                       first=s["first"], device=torch.device("cuda"))  # fmt: skip
        elif c["op"] == "rotary":
            keys = ("q", "k", "v", "positions", "cos_sin_cache", "slots", "k_cache", "v_cache", "n_rows")
            s["launch"] = BT.Rotary(lib, module, **{k: s[k] for k in keys}, interleaved=c["inter"], inverse=c["inverse"])
        else:
            keys = ("q", "k_cache", "v_cache", "block_table", "kv_lens", "cu_rows", "prefix_len")
            s["launch"] = BT.PrefixAttention(lib, module, **{k: s[k] for k in keys}, page_size=c["page"], max_new=c["new"],
                                             scale=0.125, window=c["window"], lse=c["lse"])  # fmt: skip
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if own:
        op = s["launch"]
        op.launch(torch.cuda.current_stream().cuda_stream)
        if c["op"] == "tables":
            return dict(block_table=op.block_table, slots=op.slots, positions=op.positions, cu_rows=op.cu_rows, kv_lens=op.kv_lens,
                        req_to_page=s["req_to_page"], pages_owned=s["pages_owned"], free_words=s["free_words"])  # fmt: skip
        if c["op"] == "rope_table":
            return op.cos_sin
        if c["op"] == "rotary":
            return dict(q=op.q_out, k_cache=s["k_cache"], v_cache=s["v_cache"])
        return dict(out=op.out, lse=op.lse) if c["lse"] else op.out
    return {"tables": _plain_tables, "rope_table": _plain_rope_table, "rotary": _plain_rotary, "attention": _plain_attention}[c["op"]](s, c)


def _plain_tables(s, c):
    ps, idx, seq, new = s["page"], s["req_pool_indices"], s["seq_lens"], s["new_lens"]
    owned, old = s["pages_owned"][idx].long(), s["req_to_page"][idx]
    need = (seq + new + ps - 1) // ps
    take = (need - owned).clamp(min=0)
    p = torch.arange(old.shape[1], device=idx.device)[None]
    j = p - owned[:, None]
    fresh = (j >= 0) & (j < take[:, None])
    ring = s["free_pages"]
    got = ring[(s["free_words"][0] + (take.cumsum(0) - take)[:, None] + j) % ring.numel()]
    page = torch.where(fresh, got, old)
    s["req_to_page"][idx] = page
    s["pages_owned"][idx] = torch.maximum(owned, need).int()
    s["free_words"][0] += take.sum()
    table = torch.where(p < need[:, None], page, torch.full_like(page, -1))
    cu = torch.cat((new.new_zeros(1), new.cumsum(0)))
    r = torch.arange(s["rows"], device=idx.device)
    b = torch.searchsorted(cu, r, right=True).clamp(max=idx.numel()) - 1
    live = r < cu[-1]
    pos = torch.where(live, seq[b] + r - cu[b], 0)
    slot = table[b, pos // ps].long() * ps + pos % ps
    s["slots"].copy_(torch.where(live, slot, s["slots"]))
    s["positions"].copy_(torch.where(live, pos, s["positions"]))
    return dict(block_table=table, slots=s["slots"], positions=s["positions"], cu_rows=cu.int(), kv_lens=(seq + new).int(),
                req_to_page=s["req_to_page"], pages_owned=s["pages_owned"], free_words=s["free_words"])  # fmt: skip


def _plain_rope_table(s, c):
    # angles in 64 bits: a far position times a frequency has lost the angle's fraction in 32
    rot, theta, f = c["rot"], c["theta"], c["factor"]
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    mult = 1.0
    if c["kind"] == "ntk":
        theta = theta * f ** (rot / (rot - 2))
    inv = theta ** (-i / rot)
    if c["kind"] == "linear":
        inv = inv / f
    elif c["kind"] == "llama3":
        wave = 2 * math.pi / inv
        smooth = (8192 / wave - 1.0) / (4.0 - 1.0)
        mixed = (1 - smooth) * inv / f + smooth * inv
        inv = torch.where(wave < 8192 / 4.0, inv, torch.where(wave > 8192 / 1.0, inv / f, mixed))
    elif c["kind"] == "yarn":
        dim = [rot * math.log(8192 / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(dim[0]), 0), min(math.ceil(dim[1]), rot - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        inv = inv / f * ramp + inv * (1 - ramp)
        mult = 0.1 * math.log(f) + 1.0
    ang = torch.arange(s["first"], s["first"] + c["rows"], dtype=torch.float64, device="cuda")[:, None] * inv[None]
    return (torch.cat((ang.cos(), ang.sin()), 1) * mult).float()


def _rotate(x, cos, sin, rot, inter):
    if inter:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., rot:]), -1)
    a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rot:]), -1)


def _rotary_in(s, c, dtype):
    row = s["cos_sin_cache"][s["positions"]].to(dtype)[:, None]
    cos, sin = row[..., : c["rot"] // 2], row[..., c["rot"] // 2 :]
    if c["inverse"]:
        sin = -sin
    return [_rotate(s[n].to(dtype), cos, sin, c["rot"], c["inter"]) for n in ("q", "k")]


def _plain_rotary(s, c):
    q, k = _rotary_in(s, c, torch.float32)
    live = (torch.arange(c["rows"], device="cuda") < s["n_rows"])[:, None, None]
    s["q_out"].copy_(torch.where(live, q.to(s["q"].dtype), s["q_out"]))
    for cache, new in ((s["k_cache"], k.to(s["k"].dtype)), (s["v_cache"], s["v"])):
        cache[s["slots"]] = torch.where(live, new, cache[s["slots"]])
    return dict(q=s["q_out"], k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_attention(s, c):
    B, n, ps, P, D, kvh = c["batch"], c["new"], c["page"], c["prefix"], c["dim"], c["kvh"]
    G, dev = c["qh"] // kvh, s["q"].device
    kv = s["kv_lens"].long()
    pos_q = (kv[:, None] - n + torch.arange(n, device=dev)).repeat_interleave(G, 1)  # [B, n G]
    q = s["q"].float().view(B, n, kvh, G, D).permute(2, 0, 1, 3, 4).reshape(kvh, B, n * G, D) * 0.125

    def see(p):  # p [.., keys] against pos_q [B, n G]
        ok = (p <= pos_q[..., None]) & (p < kv[:, None, None])
        return ok if c["window"] == 0 else ok & (p + c["window"] >= pos_q[..., None])

    parts = []
    if P > 0:  # the shared keys, once for all requests
        p = torch.arange(P, device=dev)
        slot = s["block_table"][0, p // ps].long() * ps + p % ps
        k, v = (s[x][slot].float().transpose(0, 1) for x in ("k_cache", "v_cache"))  # [kvh, P, D]
        sc = (q.reshape(kvh, B * n * G, D) @ k.transpose(1, 2)).view(kvh, B, n * G, P).masked_fill_(~see(p), -math.inf)
        parts.append((sc, v[:, None]))
    p = P + torch.arange(c["hi"], device=dev)
    page = s["block_table"][:, (p // ps).clamp(max=s["block_table"].shape[1] - 1)].long().clamp(min=0)
    slot = page * ps + p % ps
    k, v = (s[x][slot].float().permute(2, 0, 1, 3) for x in ("k_cache", "v_cache"))  # [kvh, B, keys, D]
    parts.append(((q @ k.transpose(2, 3)).masked_fill_(~see(p), -math.inf), v))
    m = parts[0][0].amax(-1)
    if len(parts) > 1:
        m = torch.maximum(m, parts[1][0].amax(-1))
    m0 = torch.where(m == -math.inf, 0.0, m)
    o, l = 0.0, 0.0
    for sc, v in parts:
        e = sc.sub_(m0[..., None]).exp_()
        l = l + e.sum(-1)
        o = o + (e @ v if v.shape[1] > 1 or B == 1 else (e.view(kvh, B * n * G, -1) @ v[:, 0]).view(kvh, B, n * G, D))
    out = torch.where(l[..., None] > 0, o / l[..., None], 0.0)
    out = out.view(kvh, B, n, G, D).permute(1, 2, 0, 3, 4).reshape(B * n, c["qh"], D).to(s["q"].dtype)
    if not c["lse"]:
        return out
    lse = m + l.log()
    return dict(out=out, lse=lse.view(kvh, B, n, G).permute(1, 2, 0, 3).reshape(B * n, c["qh"]))


# ---- 64-bit definitions ----------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    c, was = case, own
    own = False  # inputs only: no launches are bound here
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["op"] == "tables":
        return None  # whole numbers
    if c["op"] == "rope_table":
        return _exact_rope_table(c, s["first"])
    if c["op"] == "rotary":
        q, k = _rotary_in(s, c, torch.float64)
        n = c["live"]
        out = torch.zeros_like(q)
        out[:n] = q[:n]
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        kc[s["slots"][:n]], vc[s["slots"][:n]] = k[:n], s["v"][:n].double()
        return dict(q=out, k_cache=kc, v_cache=vc)
    return _exact_attention(s, c)


def _exact_rope_table(c, first):
    rot, f = c["rot"], c["factor"]
    inv, mult = [], 1.0
    for i in range(rot // 2):
        base = c["theta"] * (f ** (rot / (rot - 2)) if c["kind"] == "ntk" else 1.0)
        w = base ** (-2.0 * i / rot)
        if c["kind"] == "linear":
            w /= f
        elif c["kind"] == "llama3":
            turns = 8192 * w / (2 * math.pi)  # turns within the original context
            if turns < 1.0:
                w /= f
            elif turns <= 4.0:
                t = (turns - 1.0) / 3.0
                w = (1 - t) * w / f + t * w
        elif c["kind"] == "yarn":
            def at(turns):
                return rot * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(c["theta"]))

            lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
            r = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = w / f * r + w * (1 - r)
            mult = 0.1 * math.log(f) + 1.0
        inv.append(w)
    ang = torch.arange(first, first + c["rows"], dtype=torch.float64, device="cuda")[:, None] * torch.tensor(
        inv, dtype=torch.float64, device="cuda")
    return torch.cat((ang.cos(), ang.sin()), 1) * mult


def _exact_attention(s, c):
    n, ps, G = c["new"], c["page"], c["qh"] // c["kvh"]
    dev = s["q"].device
    out, lse = [], []
    for b, L in enumerate(s["lens"]):
        first = max(0, L - n - c["window"]) if c["window"] else 0
        p = torch.arange(first, L, device=dev)
        slot = s["block_table"][b, p // ps].long() * ps + p % ps
        k, v = (s[x][slot].double().transpose(0, 1) for x in ("k_cache", "v_cache"))  # [kvh, L, D]
        q = s["q"][b * n : (b + 1) * n].double().transpose(0, 1).reshape(c["kvh"], G, n, -1)
        sc = torch.einsum("hgnd,hkd->hgnk", q, k) * 0.125
        at = L - n + torch.arange(n, device=dev)
        hide = p[None] > at[:, None]
        if c["window"]:
            hide |= p[None] < at[:, None] - c["window"]
        sc = sc.masked_fill(hide, -math.inf)
        lse.append(sc.logsumexp(-1).reshape(c["qh"], n).transpose(0, 1))
        o = torch.einsum("hgnk,hkd->hgnd", torch.softmax(sc, -1), v)
        out.append(o.reshape(c["qh"], n, -1).transpose(0, 1))
    out = torch.cat(out)
    return dict(out=out, lse=torch.cat(lse)) if c["lse"] else out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "tables":
        B, width = c["batch"], -(-(c["hi"] + c["new_hi"]) // c["page"])
        rows = B * (c["new_lo"] + c["new_hi"]) / 2
        ids = B * (c["lo"] + c["hi"]) / 2 / c["page"] * 4  # page ids of the context
        return dict(bytes=ids + B * width * 4 + rows * 16 + B * 40, flops=0)
    if c["op"] == "rope_table":
        return dict(bytes=c["rows"] * c["rot"] * 4, flops=c["rows"] * c["rot"])
    if c["op"] == "rotary":
        heads = c["qh"] + 2 * c["kvh"]
        return dict(bytes=c["live"] * (heads * c["dim"] * 4 + c["rot"] * 4 + 16),
                    flops=c["live"] * (c["qh"] + c["kvh"]) * c["rot"] * 3)  # fmt: skip
    B, n, D = c["batch"], c["new"], c["dim"]
    suffix = (c["lo"] + c["hi"]) / 2
    if c["window"]:
        shared, own_keys = min(c["prefix"], c["window"] + n), min(suffix, c["window"] + n)
        seen = min(c["prefix"] + suffix, c["window"] + 1)
    else:
        shared, own_keys, seen = c["prefix"], suffix, c["prefix"] + suffix
    keys = shared + B * own_keys
    return dict(bytes=keys * c["kvh"] * D * 4 + B * n * c["qh"] * D * 4, flops=4.0 * B * n * c["qh"] * D * seen)
