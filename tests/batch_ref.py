"""Plain 64-bit forms of the batched step's operators, written request by request from their definitions."""

import math

import torch


def tables(seq, new, req, req_to_page, owned, ring, words, page, rows):
    """Python integers in, Python lists out: what one launch leaves (the state is not touched). Requests that contradict the
    extents count as padding; a step that finds no room grants nothing."""
    pool, width = len(owned), len(req_to_page[0])
    r2p, own, head, tail = [list(x) for x in req_to_page], list(owned), words[0], words[1]
    names = [r for s, n, r in zip(seq, new, req) if (s or n) and 0 <= r < pool and 0 <= s and 0 <= n and s + n <= width * page]
    live = []
    for s, n, r in zip(seq, new, req):
        ok = (s or n) and 0 <= r < pool and 0 <= s and 0 <= n and s + n <= width * page
        ok = ok and names.count(r) == 1 and -(-s // page) <= own[r] <= width
        live.append(bool(ok))
    need = [-(-(s + n) // page) if ok else 0 for s, n, ok in zip(seq, new, live)]
    take = [max(0, k - own[r]) if ok else 0 for k, r, ok in zip(need, req, live)]
    total = sum(n for n, ok in zip(new, live) if ok)
    ring_ok = 0 <= head <= tail and tail - head <= len(ring)
    grant = total <= rows and (sum(take) == 0 or (ring_ok and sum(take) <= tail - head))
    new = [n if ok and grant else 0 for n, ok in zip(new, live)]
    table, slots, positions, cu, kv = [], [], [], [0], []
    for b, ok in enumerate(live):
        s = seq[b] if ok else 0
        k = -(-(s + new[b]) // page)
        if ok:
            for p in range(own[req[b]], k):
                r2p[req[b]][p] = ring[head % len(ring)]
                head += 1
            own[req[b]] = max(own[req[b]], k)
        table.append((r2p[req[b]][:k] if ok else []) + [-1] * (width - k))
        for x in range(s, s + new[b]):
            slots.append(table[b][x // page] * page + x % page)
            positions.append(x)
        cu.append(cu[-1] + new[b])
        kv.append(s + new[b])
    return dict(block_table=table, slots=slots, positions=positions, cu_rows=cu, kv_lens=kv, req_to_page=r2p, pages_owned=own,
                free_words=[head, tail])  # fmt: skip


def frequencies(rot, theta, scaling):
    sc = dict(scaling or {})
    kind, f = sc.get("kind", "none"), sc.get("factor", 1.0)
    if kind == "ntk":
        theta = theta * f ** (rot / (rot - 2))
    out, mult = [], 1.0
    for i in range(rot // 2):
        w = theta ** (-2 * i / rot)
        if kind == "linear":
            w /= f
        if kind == "llama3":
            turns = sc["original_len"] * w / (2 * math.pi)
            lo, hi = sc["low_freq_factor"], sc["high_freq_factor"]
            t = min(max((turns - lo) / (hi - lo), 0.0), 1.0)
            w = (1 - t) * w / f + t * w
        if kind == "yarn":

            def dim(turns):
                return rot * math.log(sc["original_len"] / (turns * 2 * math.pi)) / (2 * math.log(theta))

            lo, hi = max(math.floor(dim(sc["beta_fast"])), 0), min(math.ceil(dim(sc["beta_slow"])), rot - 1)
            t = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = w / f * t + w * (1 - t)
            mult = 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
        out.append(w)
    return out, mult


def rope_table(rows, rot, theta, scaling, first):
    w, mult = frequencies(rot, theta, scaling)
    ang = torch.arange(first, first + rows, dtype=torch.float64)[:, None] * torch.tensor(w, dtype=torch.float64)
    return torch.cat((ang.cos(), ang.sin()), 1) * mult


def rotate(x, cos_sin, interleaved, inverse):
    """x [rows, heads, dim] and its table rows [rows, rot] -> the rotated rows in 64 bits."""
    rot = cos_sin.shape[1]
    x, cos_sin = x.double().cpu(), cos_sin.double().cpu()[:, None]
    c, s = cos_sin[..., : rot // 2], cos_sin[..., rot // 2 :] * (-1 if inverse else 1)
    out = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def attention(q, k_cache, v_cache, table, kv_lens, cu_rows, page, scale, window):
    """-> (out, lse, mass): mass is the softmax-weighted mean of |v|, what a relative error of the probabilities can move."""
    rows, qh, dim = q.shape
    kvh = k_cache.shape[1]
    out = torch.zeros(rows, qh, dim, dtype=torch.float64)
    lse = torch.full((rows, qh), -math.inf, dtype=torch.float64)
    mass = torch.zeros(rows, qh, dim, dtype=torch.float64)
    for b, L in enumerate(kv_lens):
        n = cu_rows[b + 1] - cu_rows[b]
        if n == 0 or L <= 0:
            continue
        p = torch.arange(L)
        slot = table[b, p // page].long() * page + p % page
        k, v = (t[slot.to(t.device)].double().cpu().transpose(0, 1).repeat_interleave(qh // kvh, 0) for t in (k_cache, v_cache))
        for j in range(n):
            at = L - n + j
            see = p <= at
            if window:
                see &= p >= at - window
            if not see.any():
                continue
            r = cu_rows[b] + j
            s = torch.einsum("hd,hkd->hk", q[r].double().cpu(), k[:, see]) * scale
            w = torch.softmax(s, -1)
            out[r] = torch.einsum("hk,hkd->hd", w, v[:, see])
            mass[r] = torch.einsum("hk,hkd->hd", w, v[:, see].abs())
            lse[r] = s.logsumexp(-1)
    return out, lse, mass
