// Attention of a batch's new rows over a paged K/V cache whose first tokens all requests share.
//
//   out[t, h] = sum_k p_k V[k] / sum_k p_k,  p_k = exp(scale q[t, h] . K[k]),  k over the keys that row t sees:
//   the row at position x of request b sees the keys max(0, x - window) .. x (window 0: 0 .. x), x = kv_len - new + its index
//
// The keys below prefix_len are the same cache rows for every request, so they are visited once for all of them: the
// query rows of the whole batch (tokens x the G query heads of a kv head) stand in one tall operand, and a K / V tile that
// was brought in serves 256 of them. The keys behind the prefix are visited per request. Softmax pieces (m, l, O) over
// disjoint key sets merge exactly, so any split of the work gives the same result up to f32 rounding.
//
// Work. An item is (kv head, block of up to 256 rows, its key tiles of 128): first the prefix items, then each request's
// own. A step is one 128-row x 128-key tile product: an item of more than 128 rows takes two steps a key tile (its two
// row halves), one of at most 128 rows takes one. All items' steps form one sequence that is cut evenly over the CTAs
// (one an SM), whatever the lengths; they are read on the device, so a captured launch follows the batch. The piece of
// item i that CTA c computes goes to slot i + c of the scratch: walking the sequence, every new piece moves to the next
// item or the next CTA, so the slots are distinct. prefix_merge_kernel adds the pieces of each row, in slot order.
//
// A CTA's twelve warps: two softmax warpgroups (a thread holds one query row, its scores are one TMEM lane), a warp that issues
// the products S = Q K^T, one that issues O += P V, one that brings in queries and K rows, one V rows (TMA boxes of a page's
// rows, or gathers of four rows where pages are small or odd). Steps alternate between the two warpgroups, each with its
// own S, P and O in tensor memory: while one takes the exponentials of its step the tensor core works for the other.
//
// Measured (both kernels, a pass inside a CUDA graph; passes on a stream take 1.5 - 2.5 us more): 32 requests x 16 rows over 32 K shared
// tokens, 16 heads of 64 on 2 kv heads: 121 us = 572 TFLOP/s, bound by the softmax's phases that depend on one another (two steps a CTA
// take about 3300 cycles; a warp's two halves of exponentials 740 + 950 of them, the unit they go through 2000 for both, the products 920);
// 96 requests over 2 K tokens of their own, 64 heads of 128 on 8: 153 us = 5.4 TB/s, DRAM, in a long run 163 - 176 at the board's power
// limit; 64 requests behind 8 K shared tokens 26 us, one request of 16 rows over a window of 2047 keys 17 us: latency.
#include "batch.h"
#include "umma.cuh"
#include "util.cuh"

namespace mk {

using namespace umma;

constexpr int kTile = 128;  // rows of a step and keys of a tile
constexpr int kAttnThreads = 384;
constexpr float kLn2 = 0.69314718055994530942f;

// ---- the plan: the same numbers in every warp of both kernels ---------------------------------------------------------
struct PlanHead {  // in front of the scratch, for the merge kernel
    unsigned total, tiles, per_head, prefix, tokens, pad[3];
};

struct Req {
    int first, n, len;  // its first row, its rows, its keys
};
// the lengths of request b as far as they are usable: what contradicts the launch's extents is left out (and recorded)
__device__ __forceinline__ Req usable(const PrefixAttnArgs& a, int b, int c0, int c1, int len, int* status) {
    Req r{c0, c1 - c0, len};
    if (r.n < 0 || r.n > a.max_new || r.first < 0 || r.first > a.rows - r.n) {
        if (status != nullptr) batch_status(status, 4, 520, b, r.n);
        r.n = 0;
    }
    if (r.len < 0 || r.len > a.width * a.page) {
        if (status != nullptr) batch_status(status, 4, 521, b, r.len);
        r.n = 0;
    }
    return r;
}
__device__ __forceinline__ Req request(const PrefixAttnArgs& a, int b) {
    return usable(a, b, __ldg(a.cu_rows + b), __ldg(a.cu_rows + b + 1), __ldg(a.kv_lens + b), nullptr);
}
// steps of one key tile over all row blocks of `rows` rows: two for every 256 rows, one for a rest of up to 128
__device__ __forceinline__ unsigned steps_of_rows(int rows) { return (unsigned)((rows + kTile - 1) / kTile); }
__device__ __forceinline__ int own_first(const PrefixAttnArgs& a, const Req& r, int prefix) {  // first key of its own tiles
    const int lo = a.window > 0 ? max(0, r.len - r.n - a.window) : 0;
    return max(prefix, lo);
}
// where its tile 0 starts: the runs of cache rows that one copy brings in begin at multiples of their length
__device__ __forceinline__ int own_start(const PrefixAttnArgs& a, const Req& r, int prefix) { return own_first(a, r, prefix) & ~(a.run - 1); }
__device__ __forceinline__ unsigned own_tiles(const PrefixAttnArgs& a, const Req& r, int prefix) {
    if (r.n <= 0 || r.len <= own_first(a, r, prefix)) return 0u;
    return (unsigned)(r.len - own_start(a, r, prefix) + kTile - 1) / kTile;
}
__device__ __forceinline__ int row_blocks(int rows) { return (rows + 2 * kTile - 1) / (2 * kTile); }
// what an item costs besides its tiles (its queries in, its O out, the tensor core's start), counted in steps
__device__ __forceinline__ unsigned lead(const PrefixAttnArgs& a, bool pair) { return a.item_steps + (pair ? a.pair_steps : 0); }
// steps of all row blocks of `rows` rows over `tiles` key tiles, for one kv head
__device__ __forceinline__ unsigned head_steps(const PrefixAttnArgs& a, unsigned tiles, int rows) {
    const unsigned pairs = (rows + kTile - 1) / (2 * kTile);  // blocks of more than kTile rows
    return tiles > 0 ? tiles * steps_of_rows(rows) + row_blocks(rows) * a.item_steps + pairs * a.pair_steps : 0u;
}
__device__ __forceinline__ unsigned own_steps(const PrefixAttnArgs& a, const Req& r, int prefix) {
    return head_steps(a, own_tiles(a, r, prefix), r.n * a.G) * a.kvh;
}
__device__ __forceinline__ int own_items(const PrefixAttnArgs& a, const Req& r) { return row_blocks(r.n * a.G) * a.kvh; }
// the key tiles of an item that the steps [lo, hi) of it stand for; a range that ends inside a pair of steps leaves the pair
// to the range that starts it
__device__ __forceinline__ void tiles_of(unsigned lo, unsigned hi, unsigned lead, int sh, unsigned& t0, unsigned& t1) {
    t0 = ((lo > lead ? lo - lead : 0u) + sh) >> sh;
    t1 = ((hi > lead ? hi - lead : 0u) + sh) >> sh;
}

struct Plan {
    int prefix;         // shared keys (0: none shared)
    int first;          // first shared key that any row sees
    int p_lo;           // where tile 0 of the prefix items starts: a multiple of kTile
    int ref;            // the request whose table row names the shared pages
    int tokens;         // rows of the batch
    unsigned tiles;     // key tiles of a prefix item
    unsigned per_head;  // steps of a kv head's prefix items
    unsigned prefix_steps, total;
};

// inclusive sums over the lanes
__device__ __forceinline__ void scan(unsigned& x, int& y, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned u = __shfl_up_sync(0xffffffffu, x, o);
        const int v = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) x += u, y += v;
    }
}

// The batch's lengths as a warp holds them: request b in lane b % 32. The first 128 stay in registers, requested all at once
// when the kernel starts; later ones are read again from L1.
struct Lens {
    static constexpr int kHeld = 4;
    Req r[kHeld];
    int want, tokens;
    __device__ __forceinline__ void load(const PrefixAttnArgs& a, int lane) {
        want = __ldg(a.prefix_len);
        tokens = __ldg(a.cu_rows + a.batch);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int b = min(32 * i + lane, a.batch - 1);
            r[i].first = __ldg(a.cu_rows + b);
            r[i].n = __ldg(a.cu_rows + b + 1);
            r[i].len = __ldg(a.kv_lens + b);
        }
    }
    // what the loads brought, as far as it is usable
    __device__ __forceinline__ void check(const PrefixAttnArgs& a, int lane, int* status) {
        const int cap = a.width * a.page;  // up to 2^30
        if (want < 0 || want > cap) {
            if (status != nullptr) batch_status(status, 4, 522, want, cap);
            want = 0;
        }
        if (tokens < 0 || tokens > a.rows) {
            if (status != nullptr) batch_status(status, 4, 523, tokens, a.rows);
            tokens = 0;
        }
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int b = 32 * i + lane;
            r[i] = b < a.batch ? usable(a, b, r[i].first, r[i].n, r[i].len, status) : Req{0, 0, 0};
        }
    }
    // fn(request, b) for blocks of 32 requests in order, b = the lane's request (an empty one past the batch); fn returns false
    // to stop. Whole warps.
    template <typename Fn>
    __device__ __forceinline__ void each(const PrefixAttnArgs& a, int lane, Fn&& fn) const {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            if (32 * i >= a.batch) return;
            if (!fn(r[i], 32 * i + lane)) return;
        }
        for (int b0 = 32 * kHeld; b0 < a.batch; b0 += 32) {
            const int b = b0 + lane;
            Req x{0, 0, 0};
            if (b < a.batch) x = request(a, b);
            if (!fn(x, b)) return;
        }
    }
};

// One warp; every lane gets the result. `cum`: first step and first item of each request, for the merge.
__device__ __forceinline__ Plan make_plan(const PrefixAttnArgs& a, const Lens& lens, int lane, int* status, unsigned* cum) {
    Plan p;
    const int want = lens.want;
    p.tokens = lens.tokens;
    int live = 0, ref = 0x7fffffff, lo = 0x7fffffff, hi = 0, all = 0;
    lens.each(a, lane, [&](const Req& r, int b) {
        if (status != nullptr && b >= 32 * Lens::kHeld && b < a.batch)
            usable(a, b, __ldg(a.cu_rows + b), __ldg(a.cu_rows + b + 1), __ldg(a.kv_lens + b), status);  // to be recorded
        all = min(all + r.n, 1 << 21);  // as far as it matters: a launch has up to 2^20 rows
        if (r.n > 0 && r.len > 0) {
            ++live;
            if (r.len >= want) ref = min(ref, b);
            lo = min(lo, a.window > 0 ? max(0, r.len - r.n - a.window) : 0);
            hi = max(hi, min(want, r.len));
        }
        return true;
    });
    // requests that name more rows than there are (where max_new lets them): their steps together could pass 32 bits, so nothing is done
    if ((long long)a.batch * a.max_new > a.rows && (all = __reduce_add_sync(0xffffffffu, all)) > a.rows) {
        if (status != nullptr && lane == 0) batch_status(status, 4, 525, all, a.rows);
        return Plan{0, 0, 0, 0, 0, 0u, 0u, 0u, 0u};
    }
    live = __reduce_add_sync(0xffffffffu, live);
    ref = __reduce_min_sync(0xffffffffu, ref);
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    // one request shares with nobody, and a prefix that no request holds whole cannot be read through one table row
    p.prefix = live > 1 && ref != 0x7fffffff ? want : 0;
    p.ref = p.prefix > 0 ? ref : 0;
    p.first = p.prefix > 0 ? lo : 0;
    p.p_lo = p.first / kTile * kTile;
    p.tiles = p.prefix > 0 && hi > p.p_lo ? (unsigned)(hi - p.p_lo + kTile - 1) / kTile : 0u;
    p.per_head = head_steps(a, p.tiles, p.tokens * a.G);
    p.prefix_steps = p.per_head * a.kvh;
    unsigned sum = 0;
    if (cum == nullptr) {
        lens.each(a, lane, [&](const Req& r, int) {
            sum += own_steps(a, r, p.prefix);
            return true;
        });
        p.total = p.prefix_steps + __reduce_add_sync(0xffffffffu, sum);
        return p;
    }
    sum = p.prefix_steps;
    int items = 0;
    lens.each(a, lane, [&](const Req& r, int b) {
        const unsigned x = own_steps(a, r, p.prefix);
        const int it = own_items(a, r);
        unsigned inc = x;
        int ci = it;
        scan(inc, ci, lane);
        if (b < a.batch) {
            cum[b] = sum + inc - x;
            cum[a.batch + b] = (unsigned)(items + ci - it);
        }
        sum += __shfl_sync(0xffffffffu, inc, 31);
        items += __shfl_sync(0xffffffffu, ci, 31);
        return true;
    });
    p.total = sum;
    return p;
}

// The work is cut for this many CTAs (one an SM), a constant so that no division by a variable stands in front of the work.
// No CTA waits for another, so a part with fewer SMs would only run them in turn.
constexpr unsigned kCtas = kAttnCtas;
__device__ __forceinline__ unsigned range_lo(unsigned total, unsigned c) {  // first step of CTA c's range: floor(total c / kCtas)
    const unsigned q = total / kCtas;
    if (q == 0) return min(c, total);  // fewer steps than CTAs: one each
    return q * c + (total - q * kCtas) * c / kCtas;
}
__device__ __forceinline__ int cta_of(unsigned step, unsigned total) {  // whose range holds the step
    if (total < kCtas) return (int)step;
    if (total < (1u << 24)) return (int)(((step + 1) * kCtas - 1) / total);  // kCtas < 2^8
    return (int)((((unsigned long long)step + 1) * kCtas - 1) / total);
}

// An item's piece in one CTA's range
struct Piece {
    int b;            // request, -1: the prefix
    int h, rb;        // kv head, row block
    int index;        // number of the item within its kind (slot = index + CTA)
    int rows;         // rows of the block (1 .. 256)
    int n;            // request rows (own items)
    int first, len;   // the request's first row and keys
    int key0;         // first key of the item's tile 0
    int seen;         // first key that any of its rows sees: those in front are not read
    unsigned t0, t1;  // key tiles [t0, t1)
    __device__ __forceinline__ bool pair() const { return rows > kTile; }
    __device__ __forceinline__ unsigned steps() const { return (t1 - t0) << (rows > kTile ? 1 : 0); }
};

// Walks a CTA's range of steps item by item. Every role of the CTA has its own walker with the same sequence.
struct Walker {
    const PrefixAttnArgs& a;
    const Plan& p;
    unsigned left;  // steps left
    int b;          // -1 while in the prefix
    int items;      // own items before request b
    int h, rb;      // the next item
    unsigned off;   // steps of it that lie before the range
    Req r;
    unsigned tiles;
    int row_total, blocks, key0, seen;

    __device__ __forceinline__ Walker(const PrefixAttnArgs& a_, const Plan& p_, const Lens& lens, int cta, int lane) : a(a_), p(p_) {
        unsigned pos = range_lo(p.total, cta);
        left = range_lo(p.total, cta + 1) - pos;
        b = -1;
        items = 0;
        h = rb = 0;
        off = 0;
        blocks = 0;
        if (left == 0) return;
        if (pos >= p.prefix_steps) {  // starts in a request's items: find it, the whole warp together
            unsigned sum = p.prefix_steps;
            lens.each(a, lane, [&](const Req& q, int bb) {
                const unsigned x = own_steps(a, q, p.prefix);
                const int it = own_items(a, q);
                unsigned inc = x;
                int ci = it;
                scan(inc, ci, lane);
                const unsigned hit = __ballot_sync(0xffffffffu, pos < sum + inc);
                const int l = hit != 0u ? __ffs(hit) - 1 : 31;
                if (hit != 0u) {
                    b = bb - lane + l;
                    pos -= sum + __shfl_sync(0xffffffffu, inc - x, l);
                    items += __shfl_sync(0xffffffffu, ci - it, l);
                    return false;
                }
                sum += __shfl_sync(0xffffffffu, inc, 31);
                items += __shfl_sync(0xffffffffu, ci, 31);
                return true;
            });
        }
        load();
        const unsigned per_head = head_steps(a, tiles, row_total), block = 2 * tiles + lead(a, true);
        h = (int)(pos / per_head);
        pos -= h * per_head;
        rb = (int)(pos / block);
        off = pos - rb * block;
    }
    __device__ __forceinline__ void load() {
        if (b < 0) {
            tiles = p.tiles;
            r = Req{0, p.tokens, p.prefix};
            key0 = p.p_lo;
            seen = p.first;
        } else {
            r = request(a, b);
            tiles = own_tiles(a, r, p.prefix);
            key0 = own_start(a, r, p.prefix);
            seen = own_first(a, r, p.prefix);
        }
        row_total = r.n * a.G;
        blocks = row_blocks(row_total);
    }
    // the next piece, false at the end of the range
    __device__ bool next(Piece& x) {
        while (left > 0) {
            while (tiles == 0 || h == a.kvh) {  // on to the next request that has steps
                if (b >= 0) items += blocks * a.kvh;
                if (++b >= a.batch) {  // only where the lengths changed under the kernel
                    left = 0;
                    return false;
                }
                h = 0;
                load();
            }
            x.b = b;
            x.h = h;
            x.rb = rb;
            x.rows = min(2 * kTile, row_total - rb * 2 * kTile);
            x.first = r.first;
            x.n = r.n;
            x.len = r.len;
            x.key0 = key0;
            x.seen = seen;
            x.index = (b < 0 ? 0 : items) + h * blocks + rb;
            const int sh = x.rows > kTile ? 1 : 0;
            const unsigned front = lead(a, sh != 0), len = (tiles << sh) + front, stop = min(off + left, len);
            tiles_of(off, stop, front, sh, x.t0, x.t1);
            left -= stop - off;
            off = 0;
            if (++rb == blocks) rb = 0, ++h;
            if (x.t1 > x.t0) return true;
        }
        return false;
    }
};

// ---- scratch ----------------------------------------------------------------------------------------------------------
// A slot holds two parts (the row halves of a pair, or the even and odd tiles of a single); a part of R rows: O as
// [D / 4][R] float4, then m [R] and l [R].
__host__ __device__ constexpr long long part_bytes(int rows, int dim) { return (long long)rows * (dim + 2) * 4; }

// ---- the kernel --------------------------------------------------------------------------------------------------------
template <int D>
struct Cfg {
    static constexpr int kAtoms = D / 64;                 // 64-wide column blocks of a K / V tile
    static constexpr int kTileBytes = kTile * D * 2;      // K, V or Q tile
    static constexpr int kRingK = D == 64 ? 4 : 2, kRingV = D == 64 ? 4 : 2;  // K stages, V stages
    static constexpr int kQ = D == 64 ? 4 : 3;            // query tiles
    static constexpr int kSmem = (kRingK + kRingV + kQ) * kTileBytes + 1024;
    static constexpr bool kAlias = D == 128;              // P over S: tensor memory holds 2 x (128 + 128) columns then
    // tensor-memory columns (512): S of each warpgroup, P, O
    static constexpr uint32_t kS = 0, kP = D == 64 ? 256 : 0, kPStep = D == 64 ? 64 : 128, kO = D == 64 ? 384 : 256, kOStep = D;
};

struct Bars {
    uint64_t k_full[6], k_empty[6], v_full[6], v_empty[6], q_full[6], q_empty[6];
    uint64_t s_full[2], s_free[2], p_ready[2], o_full[2], pv_done[2];
    uint64_t drain[2];
    uint32_t tmem;
    int abort;
};

__device__ __forceinline__ void gather4(void* dst, const CUtensorMap* map, int x, int y0, int y1, int y2, int y3, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y0), "r"(y1), "r"(y2), "r"(y3), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void load_box2(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void load_box3(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// D[128 x N] (+)= A B^T, both operands in shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        :
        : "r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
        : "memory");
}
// the same with A in tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t at, uint64_t bd, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        :
        : "r"(d), "r"(at), "l"(bd), "r"(idesc), "r"(acc)
        : "memory");
}
// f32 accumulator, A and B f16 (0) or bf16 (1), A K-major, B K-major or (bit 16) N-major
__host__ __device__ constexpr uint32_t idesc_f16(bool half, bool b_n_major, int m, int n) {
    return (1u << 4) | ((half ? 0u : 1u) << 7) | ((half ? 0u : 1u) << 10) | ((b_n_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}
// An item of at most 16 rows takes products of 64 rows instead of 128: rows 0 .. 15 lie in the same lanes in both shapes, and the
// tensor core does half the padding's work. (96 decodes over their own 2 K keys, which run at the board's power limit: 187 -> 175 us
// in a long run, 161 -> 157 us in a short one.)
constexpr int kFew = 16;
// V as the N-major operand: 64 columns (128 bytes, swizzled) x 8 keys form an atom of 1024 bytes; the next 8 keys follow
// it (stride offset), the next 64 columns lie a whole tile of 128-byte rows further (leading offset)
__device__ __forceinline__ uint64_t desc_v(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)((kTile * 128) >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}

__device__ __forceinline__ void tmem_ld32(uint32_t t, float* r) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
        "%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]),
          "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]),
          "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]),
          "=r"(u[31])
        : "r"(t));
}
// waits for this thread's loads; the registers pass through it, so that nothing that uses them moves in front
__device__ __forceinline__ void tmem_arrived32(float* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]),
                   "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]), "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]),
                   "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]),
                   "+f"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two f32 operations an instruction
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y), "f"(z.x), "f"(z.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
    return r;
}
__device__ __forceinline__ float max_nan(float x, float y) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float max_nan(float x, float y, float z) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
// 2^x for two x on the FMA pipe: x = k + f with k the nearest whole number, 2^f on [-1/2, 1/2] by the polynomial of degree 4 with
// p(0) = 1 and the least relative error (2.9e-6; a linear program), k added to the exponent. x is kept at or above -127, whose result is
// exactly 0 (p = 1 with its exponent's 127 taken off), so a score of -inf weighs nothing; between -127 and -126 it is some number below 2^-126.
// The special-function unit yields 16 results a clock and SM; kPolyOf8 of 8 results come from here instead, except in the few tiles with
// masked keys. (0 of 8: 128.5 us for the 32 x 16 rows over 32 K tokens, 1: 125, 2: 125.5, 3: 129.)
__device__ __forceinline__ float2 exp2_poly(float2 x) {
    const float2 magic = make_float2(12582912.f, 12582912.f), back = make_float2(-12582912.f, -12582912.f);
    x.x = fmaxf(x.x, -127.f);
    x.y = fmaxf(x.y, -127.f);
    const float2 r = add2(x, magic);  // k in the low bits
    const float2 f = fma2(add2(r, back), make_float2(-1.f, -1.f), x);
    float2 p = fma2(f, make_float2(0x1.3a007ap-7f, 0x1.3a007ap-7f), make_float2(0x1.c9fd1ep-5f, 0x1.c9fd1ep-5f));
    p = fma2(p, f, make_float2(0x1.ec0382p-3f, 0x1.ec0382p-3f));
    p = fma2(p, f, make_float2(0x1.62e12ap-1f, 0x1.62e12ap-1f));
    p = fma2(p, f, make_float2(1.f, 1.f));
    return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23)), __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23)));
}
template <int N>
struct Int {
    static constexpr int value = N;
};
constexpr int kPolyOf8 = 1;

// The probabilities p = 2^(score - m) are held as p 2^kLift, and l and O with them. f16 has no exponents below 2^-24: at 2^0 all keys of
// less than 2^-25 of the largest one's weight left O and stayed in l (32 K keys of 2^-25.2 beside two of weight 1, in one CTA: 0 instead of
// 4e-4, the two's V being 0).
// At 2^7 the largest p is 2^(7 + 8) (m lags by up to 8), below f16's 65504; bf16 has f32's exponents.
template <bool kHalf>
constexpr float kLift = kHalf ? 7.f : 0.f;
// From here on (in the exponent) the differences of scores are taken before they are scaled; below, the reference is rounded by at most
// 2^-15, which is what the pieces of a row may differ by. The test for it costs a vote a step (verify 121.8 -> 123.8 us, 64 decodes
// 27.7 -> 28.3); a vote only where the reference moves, a loop of its own for such scores, or one vote for this and the rescaling cost more.
constexpr float kFar = 1024.f;

template <bool kHalf>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (kHalf) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Called by whole warps; one expired wait ends every role of the CTA.
__device__ __forceinline__ bool attn_wait(uint64_t* bar, uint32_t parity, Bars* s, int* status, int where) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const bool ok = mbar_wait(bar, parity, &s->abort);
    if (__all_sync(0xffffffffu, ok)) return true;  // the whole warp goes the same way
    if (!ok && atomicExch(&s->abort, 1) == 0) batch_status(status, 3, where, 0, 0);
    return false;
}

// the request and index of token t of the batch (bisection over cu_rows, which is in L1)
__device__ __forceinline__ int request_of(const PrefixAttnArgs& a, int t) {
    int lo = 0, hi = a.batch;  // the last b with cu[b] <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(a.cu_rows + mid) <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}
// the same by a whole warp for one token: 32 probes a round
__device__ __forceinline__ int request_of_warp(const PrefixAttnArgs& a, int t, int lane) {
    int lo = 0, n = a.batch;  // the last b in [lo, lo + n) with cu[b] <= t
    while (n > 1) {
        const int step = (n + 31) / 32, b = lo + lane * step;
        const bool le = lane * step < n && (lane == 0 || __ldg(a.cu_rows + b) <= t);
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, le));
        lo += last * step;
        n = min(step, n - last * step);
    }
    return lo;
}
// the keys [lo, hi) that row `rr` of a piece sees, within the piece's keys
__device__ __forceinline__ void row_keys(const PrefixAttnArgs& a, const Plan& p, const Piece& x, int rr, int& lo, int& hi) {
    lo = hi = 0;
    if (rr >= x.rows) return;
    const int j = (x.rb * 2 * kTile + rr) / a.G;  // token of the item
    int n = x.n, len = x.len, idx = j;
    if (x.b < 0) {
        const int b = request_of(a, j);
        const Req r = request(a, b);
        n = r.n;
        len = r.len;
        idx = j - r.first;
        if (idx >= n) return;  // a request that was left out
    }
    const int at = len - n + idx;  // its position
    lo = max(x.b < 0 ? 0 : p.prefix, a.window > 0 ? at - a.window : 0);
    hi = min(at + 1, x.b < 0 ? p.prefix : len);
    if (hi < lo) hi = lo;
}

template <int D, bool kHalf>
__global__ void __launch_bounds__(kAttnThreads, 1)
    prefix_attn_kernel(const __grid_constant__ PrefixAttnArgs a, const __grid_constant__ PrefixAttnMaps maps) {
    typedef Cfg<D> C;
    extern __shared__ unsigned char raw[];
    __shared__ Bars S;
    unsigned char* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    unsigned char* Ks = smem;
    unsigned char* Vs = Ks + C::kRingK * C::kTileBytes;
    unsigned char* Qs = Vs + C::kRingV * C::kTileBytes;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();
    Lens lens;
    lens.load(a, lane);  // under the set-up below
    if (warp == 9 && lane < 5) {
        const CUtensorMap* m = lane == 0 ? &maps.k_run : lane == 1 ? &maps.v_run : lane == 2 ? &maps.k_row : lane == 3 ? &maps.v_row : &maps.q;
        if (lane < 4 || a.q_box) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < 6; ++i) {
            mbar_init(&S.k_full[i], 1);
            mbar_init(&S.k_empty[i], 1);
            mbar_init(&S.v_full[i], 1);
            mbar_init(&S.v_empty[i], 1);
            mbar_init(&S.q_full[i], a.q_box ? 1 : 32);
            mbar_init(&S.q_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&S.s_full[i], 1);
            mbar_init(&S.s_free[i], 4);
            mbar_init(&S.p_ready[i], 4);
            mbar_init(&S.o_full[i], 1);
            mbar_init(&S.pv_done[i], 1);
        }
        mbar_init(&S.drain[0], 1);
        mbar_init(&S.drain[1], 1);
        S.abort = 0;
        mbar_fence_init();
    }
    if (warp == 8) tmem_alloc(&S.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t*)&S.tmem;

    unsigned* cum = (unsigned*)(a.ws + 256);
    const bool writer = blockIdx.x == 0 && warp == 0;
    lens.check(a, lane, writer ? a.status : nullptr);
    const Plan p = make_plan(a, lens, lane, writer ? a.status : nullptr, writer ? cum : nullptr);
    if (writer && lane == 0) *(PlanHead*)a.ws = PlanHead{p.total, p.tiles, p.per_head, (unsigned)p.prefix, (unsigned)p.tokens, 0u, 0u, 0u};
    Walker walk(a, p, lens, blockIdx.x, lane);
    Piece x;
    const int cap = a.width * a.page;
    unsigned issued = 0, q_count = 0;  // tiles that this warp has asked for

    if (warp < 8) {
        // ---- softmax ----
        const int wg = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // 32 (warp % 4) lanes in bits 16 ..
        const uint32_t tS = tmem + lanes + C::kS + wg * 128, tP = tmem + lanes + C::kP + wg * C::kPStep, tO = tmem + lanes + C::kO + wg * C::kOStep;
        unsigned g = 0;  // steps of earlier pieces
        uint32_t s_par = 0, o_par = 0, pv_par = 1;  // pv: the wait for the step before the first returns at once
        const float2 scale2 = make_float2(a.scale_log2, a.scale_log2);
        bool ok = true;
        int lo = 0, hi = 0, rr = 0;
        unsigned ns = 0, sub = 0;
        auto advance = [&]() -> bool {  // the next piece in which this warpgroup has steps
            while (walk.next(x)) {
                ns = x.steps();
                sub = (wg - g) & 1;
                g += ns;
                if (sub >= ns) continue;
                rr = row + (x.pair() ? (int)sub * kTile : 0);
                row_keys(a, p, x, rr, lo, hi);
                return true;
            }
            return false;
        };
        bool more = advance();
        while (more) {
            const bool pair = x.pair();
            const bool busy = (rr & ~31) < x.rows;  // this warp has rows
            float m = -INFINITY, l = 0.f;
            for (unsigned st = sub; st < ns; st += 2) {
                const int kb = x.key0 + (int)(x.t0 + (pair ? st >> 1 : st)) * kTile;
                if (!(ok = attn_wait(&S.s_full[wg], s_par, &S, a.status, 530))) break;
                s_par ^= 1;
                tc_fence_after();
                if (busy) {
                    // Two passes over the scores, 32 columns at a time from tensor memory (the next 32 on their way): the
                    // maximum, then the probabilities. Loops of few instructions: a step's code unrolled over 128 columns
                    // ran at the pace of instruction fetch where it ran once or twice (a launch of few steps: 4 us a step).
                    const bool whole = __all_sync(0xffffffffu, (lo <= kb && hi >= kb + kTile) || rr >= x.rows);
                    // Otherwise each half of the columns is looked at: one that no row of the warp sees is passed over, one that
                    // all see whole needs no mask; in the others a bit a column says what the row sees.
                    unsigned part = 0, none = 0;  // halves in 64 columns: seen in part, not seen
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int c0 = lo - kb - 64 * i, c1 = hi - kb - 64 * i;
                            const bool idle = rr >= x.rows;
                            if (__all_sync(0xffffffffu, c1 <= 0 || c0 >= 64 || c0 >= c1 || idle)) none |= 1u << i;
                            else if (!__all_sync(0xffffffffu, (c0 <= 0 && c1 >= 64) || idle)) part |= 1u << i;
                        }
                    }
                    float s0[32], s1[32];
                    auto hide = [&](float* s, int col) {
                        const int c0 = max(lo - kb - col, 0), c1 = min(hi - kb - col, 32);
                        const unsigned see = c0 < c1 ? (0xffffffffu >> (32 - (c1 - c0))) << c0 : 0u;
#pragma unroll
                        for (int i = 0; i < 32; ++i) s[i] = see & (1u << i) ? s[i] : -INFINITY;
                    };
                    float mx[2] = {-INFINITY, -INFINITY};
                    auto highest = [&](float* s) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            mx[0] = max_nan(mx[0], s[i], s[i + 1]);
                            mx[1] = max_nan(mx[1], s[i + 2], s[i + 3]);
                        }
                    };
                    tmem_ld32(tS, s0);
                    tmem_ld32(tS + 32, s1);
                    auto first_pass = [&](auto masks) {
#pragma unroll 1
                        for (int i = 0; i < 128; i += 64) {
                            tmem_arrived32(s0);
                            tmem_arrived32(s1);
                            if (decltype(masks)::value && ((part | none) & (i == 0 ? 1u : 2u))) {
                                hide(s0, i);
                                hide(s1, i + 32);
                            }
                            highest(s0);
                            highest(s1);
                            tmem_ld32(tS + ((i + 64) & 127), s0);  // at the end: the first columns again, for the second pass
                            tmem_ld32(tS + ((i + 64) & 127) + 32, s1);
                        }
                    };
                    // (a test of the mask inside the loop of whole tiles: 32 x 16 rows over 32 K tokens 123 us instead of 121)
                    if (whole) first_pass(Int<0>());
                    else first_pass(Int<1>());
                    const float top = max_nan(mx[0], mx[1]);
                    if (!(top < INFINITY)) l = NAN;  // a score that is NaN or +inf: so is the row's softmax
                    // The reference score m (not scaled) follows the maximum only when that has grown by more than 2^8 (a factor that
                    // P's type and the f32 sums carry without loss), so O is seldom rescaled. (m = the maximum
                    // where it moves: a key that carries the row has a power of two as its p, which P's type holds exactly.)
                    const bool grow = (top - m) * a.scale_log2 > 8.f && rr < x.rows;
                    const bool any = __any_sync(0xffffffffu, grow);
                    const float f = grow ? ex2((m - top) * a.scale_log2) : 1.f;  // m = -inf: the factor is 0
                    if (grow) m = top;
                    l *= f;
                    // the P V product of this warpgroup's last step has read P and updated O
                    if (!C::kAlias && !(ok = attn_wait(&S.pv_done[wg], pv_par, &S, a.status, 540))) break;
                    if (any && st != sub) {
                        tc_fence_after();
#pragma unroll 1
                        for (int i = 0; i < D; i += 16) {
                            uint32_t o[16];
                            tmem_ld16(tO + i, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            tmem_st16(tO + i, o);
                        }
                    }
                    // Exponents are scale s - scale m in one FMA, whose second term is rounded. All weights of a row have the same
                    // factor from that, so it is of no account until its half step passes the exponents that P's type can carry
                    // (2^27 and up with f16: NaN). Where it counts the differences s - m are taken first.
                    const float ref = m == -INFINITY ? 0.f : m;
                    const bool far = __any_sync(0xffffffffu, fabsf(ref * a.scale_log2) >= kFar);
                    const float shift = far ? kLift<kHalf> : kLift<kHalf> - ref * a.scale_log2;
                    const float2 neg = make_float2(shift, shift);
                    const unsigned slow = part | none | (far ? 3u : 0u);  // halves that are masked, or whose scores are far from zero
                    float2 sum[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] = make_float2(0.f, 0.f);
                    auto probabilities = [&](float* s, uint32_t* u, auto poly) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            float2 e = fma2(make_float2(s[2 * j], s[2 * j + 1]), scale2, neg);
                            if (j % 8 < decltype(poly)::value) e = exp2_poly(e);
                            else e = make_float2(ex2(e.x), ex2(e.y));
                            sum[j & 3] = add2(sum[j & 3], e);
                            u[j] = pack2<kHalf>(e.x, e.y);
                        }
                    };
#pragma unroll 1
                    for (int i = 0; i < 128; i += 64) {
                        tmem_arrived32(s0);
                        tmem_arrived32(s1);
                        if (i != 0 && !C::kAlias) {  // all scores are in registers: the tensor core may write the next ones
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&S.s_free[wg]);
                        }
                        uint32_t u0[16], u1[16];
                        const unsigned bit = i == 0 ? 1u : 2u;
                        if (!(slow & bit)) {
                            probabilities(s0, u0, Int<kPolyOf8>());
                            probabilities(s1, u1, Int<kPolyOf8>());
                        } else if (none & bit) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) u0[j] = u1[j] = 0u;
                        } else {
                            if (far) {
#pragma unroll
                                for (int j = 0; j < 32; ++j) s0[j] -= ref, s1[j] -= ref;
                            }
                            hide(s0, i);
                            hide(s1, i + 32);
                            probabilities(s0, u0, Int<0>());
                            probabilities(s1, u1, Int<0>());
                        }
                        if (i == 0) {
                            tmem_ld32(tS + 64, s0);
                            tmem_ld32(tS + 96, s1);
                        }
                        tmem_st16(tP + i / 2, u0);  // where P lies over S: columns that have been read
                        tmem_st16(tP + i / 2 + 16, u1);
                    }
                    l += ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y)) + ((sum[2].x + sum[2].y) + (sum[3].x + sum[3].y));
                    tmem_st_wait();
                    tc_fence_before();
                } else if (!C::kAlias) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S.s_free[wg]);
                    if (!(ok = attn_wait(&S.pv_done[wg], pv_par, &S, a.status, 540))) break;
                }
                pv_par ^= 1;
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.p_ready[wg]);
            }
            if (!ok) break;
            // while the last product runs: where this piece goes, and the next one
            const int R = x.b < 0 ? kTile : a.suffix_rows;
            unsigned char* dst =
                a.ws + (x.b < 0 ? a.ws_prefix : a.ws_suffix) + ((long long)(x.index + (int)blockIdx.x) * 2 + sub) * part_bytes(R, D);
            const bool mine = rr < x.rows;
            more = advance();
            if (!(ok = attn_wait(&S.o_full[wg], o_par, &S, a.status, 531))) break;
            o_par ^= 1;
            if (busy) {
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    float o[32];
                    tmem_ld32(tO + 32 * i, o);
                    tmem_ld_wait();
                    if (mine) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            ((float4*)dst)[(8 * i + j) * R + row] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                    }
                }
                if (mine) {
                    float* ml = (float*)dst + (long long)R * D;
                    ml[row] = m;
                    ml[R + row] = l;
                }
                tc_fence_before();
            }
        }
    } else if (warp == 8) {
        // ---- S = Q K^T ----
        // What the issuing thread hands to the tensor core is made uniform over the warp first (shuffles from lane 0): the
        // compiler then keeps descriptors in uniform registers.
        const uint64_t q_desc = desc_sw128(smem_u32(Qs)), k_desc = desc_sw128(smem_u32(Ks));
        unsigned n = 0, ki = 0, kpar = 0, qi = 0, qpar = 0;  // step; ring places and their phases
        bool ok = true;
        while (ok && walk.next(x)) {
            const bool pair = x.pair();
            const uint32_t id_s = __shfl_sync(0xffffffffu, x.rows <= kFew ? idesc_f16(kHalf, false, 64, kTile) : idesc_f16(kHalf, false, kTile, kTile), 0);
            const unsigned ns = x.steps(), tiles_q = pair ? 2 : 1;
            for (unsigned st = 0; st < ns; ++st, ++n) {
                const int w = __shfl_sync(0xffffffffu, (int)(n & 1), 0);
                unsigned qq = qi + (pair ? st & 1 : 0), qp = qpar;
                if (qq >= C::kQ) qq -= C::kQ, qp ^= 1;
                const int qs = __shfl_sync(0xffffffffu, (int)qq, 0), ks = __shfl_sync(0xffffffffu, (int)ki, 0);
                const bool last_k = !pair || (st & 1);
                if (st < tiles_q && !(ok = attn_wait(&S.q_full[qs], qp, &S, a.status, 532))) break;
                if ((!pair || !(st & 1)) && !(ok = attn_wait(&S.k_full[ks], kpar, &S, a.status, 533))) break;
                // the scores of step n - 2 have left S (where P lies over S: its P V product has ended)
                if (!(ok = attn_wait(C::kAlias ? &S.pv_done[w] : &S.s_free[w], ((n >> 1) & 1) ^ 1, &S, a.status, 536))) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t qd = q_desc + (uint64_t)(qs * (C::kTileBytes >> 4)), kd = k_desc + (uint64_t)(ks * (C::kTileBytes >> 4));
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint64_t o = ((k >> 2) * (kTile * 128) + (k & 3) * 32) >> 4;
                        mma_ss(tmem + C::kS + w * 128, qd + o, kd + o, id_s, k > 0);
                    }
                    tc_commit(&S.s_full[w]);
                    if (last_k) tc_commit(&S.k_empty[ks]);
                    if (st + tiles_q >= ns) tc_commit(&S.q_empty[qs]);
                }
                __syncwarp();
                if (last_k && ++ki == C::kRingK) ki = 0, kpar ^= 1;
            }
            qi += tiles_q;
            if (qi >= C::kQ) qi -= C::kQ, qpar ^= 1;
        }
        // the tensor core has to be done before its memory is given back
        if (elect_one()) tc_commit(&S.drain[0]);
        __syncwarp();
        for (uint32_t i = 0; i < kWaitPolls && !mbar_try_wait(&S.drain[0], 0); ++i) {
        }
    } else if (warp == 11) {
        // ---- O += P V: a warp of its own, because one thread that issued both products and kept both sides' barriers spent
        // more time on those than the products take ----
        const uint64_t v_desc = desc_v(smem_u32(Vs));
        unsigned n = 0, vi = 0, vpar = 0;
        bool ok = true;
        while (ok && walk.next(x)) {
            const bool pair = x.pair();
            const uint32_t id_o = __shfl_sync(0xffffffffu, x.rows <= kFew ? idesc_f16(kHalf, true, 64, D) : idesc_f16(kHalf, true, kTile, D), 0);
            const unsigned ns = x.steps();
            for (unsigned st = 0; st < ns; ++st, ++n) {
                const int w = __shfl_sync(0xffffffffu, (int)(n & 1), 0), vs = __shfl_sync(0xffffffffu, (int)vi, 0);
                const unsigned more = __shfl_sync(0xffffffffu, st >= 2 ? 1u : 0u, 0);  // adds to O
                const bool last_v = !pair || (st & 1);
                if ((!pair || !(st & 1)) && !(ok = attn_wait(&S.v_full[vs], vpar, &S, a.status, 534))) break;
                if (!(ok = attn_wait(&S.p_ready[w], (n >> 1) & 1, &S, a.status, 535))) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t vd = v_desc + (uint64_t)(vs * (C::kTileBytes >> 4));
#pragma unroll
                    for (int k = 0; k < kTile / 16; ++k)
                        mma_ts(tmem + C::kO + w * C::kOStep, tmem + C::kP + w * C::kPStep + 8 * k, vd + (uint64_t)(k * 2048 >> 4), id_o, k > 0 ? 1u : more);
                    tc_commit(&S.pv_done[w]);
                    if (last_v) tc_commit(&S.v_empty[vs]);
                    if (st + 2 >= ns) tc_commit(&S.o_full[w]);
                }
                __syncwarp();
                if (last_v && ++vi == C::kRingV) vi = 0, vpar ^= 1;
            }
        }
        if (elect_one()) tc_commit(&S.drain[1]);
        __syncwarp();
        for (uint32_t i = 0; i < kWaitPolls && !mbar_try_wait(&S.drain[1], 0); ++i) {
        }
    } else {
        // ---- queries and K rows (warp 9), V rows (warp 10) ----
        // Where pages hold runs of 8 or more aligned rows, a lane copies a run as one box; else a lane gathers four rows. Rows
        // in front of the first key that any of the piece's rows sees and past its last one are asked for behind the pool's end,
        // which reads zeros: a probability of zero times whatever a stale row holds would not be zero. So the runs that the first
        // and the last key lie in are gathered row by row (V), and page ids outside [first, last] are not looked at.
        const bool is_v = warp == 10;
        const CUtensorMap *run_map = is_v ? &maps.v_run : &maps.k_run, *row_map = is_v ? &maps.v_row : &maps.k_row;
        unsigned char* ring = is_v ? Vs : Ks;
        uint64_t *full = is_v ? S.v_full : S.k_full, *empty = is_v ? S.v_empty : S.k_empty;
        const unsigned stages = is_v ? C::kRingV : C::kRingK;
        unsigned place = 0, phase = 0;  // of the ring
        const int head = is_v ? a.v_head : a.k_head;
        const bool runs = a.run >= 8;
        const int per = runs ? a.run : 4, mine = lane * per;  // this lane's keys of a tile
        bool ok = true;
        while (ok && walk.next(x)) {
            const int* trow = a.table + (long long)(x.b < 0 ? p.ref : x.b) * a.table_row;
            const int stop = min(x.len, cap), col = x.h * head;
            auto slot_of = [&](int k, int n) -> int {  // pool row of key k, of n rows that lie in one page
                if (k >= stop || k + n <= x.seen) return a.kv_rows;
                const int pg = a.page_shift >= 0 ? k >> a.page_shift : k / a.page;
                const long long slot = (long long)__ldg(trow + pg) * a.page + (k - pg * a.page);
                if (slot >= 0 && slot + n <= a.kv_rows) return (int)slot;
                batch_status(a.status, 4, 524, x.b, k);
                return a.kv_rows;
            };
            auto slots_of = [&](unsigned t, int (&y)[4]) {
                const int k = x.key0 + (int)t * kTile + mine;
                if (runs) {
                    if (mine < kTile) y[0] = slot_of(k, min(per, stop - k));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = slot_of(k + i, 1);
                }
            };
            int y[4] = {0, 0, 0, 0};
            slots_of(x.t0, y);
            for (int half = 0; !is_v && half < (x.pair() ? 2 : 1); ++half, ++q_count) {
                const unsigned i = q_count % C::kQ;
                if (!(ok = attn_wait(&S.q_empty[i], ((q_count / C::kQ) & 1) ^ 1, &S, a.status, 539))) break;
                unsigned char* dst = Qs + i * C::kTileBytes;
                const int ir = x.rb * 2 * kTile + half * kTile;  // the tile's first row in the item
                if (a.q_box) {                                   // 128 / G whole tokens: one box a 64-wide column block
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&S.q_full[i], C::kTileBytes);
#pragma unroll
                        for (int c = 0; c < C::kAtoms; ++c)
                            load_box3(dst + c * (kTile * 128), &maps.q, 64 * c, x.h * a.G, x.first + ir / a.G, &S.q_full[i]);
                    }
                    __syncwarp();
                } else {
#pragma unroll 1
                    for (int r = lane; r < kTile; r += 32) {
                        const bool valid = half * kTile + r < x.rows;
                        const int tok = (ir + r) / a.G, head = x.h * a.G + ir + r - tok * a.G;
                        const unsigned char* src =
                            (const unsigned char*)a.q + (valid ? ((long long)(x.first + tok) * a.q_row + head * a.q_head) * 2 : 0);
#pragma unroll
                        for (int c = 0; c < D / 8; ++c)
                            cp_async16(dst + (c >> 3) * (kTile * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), src + c * 16, valid);
                    }
                    cp_async_commit();
                    cp_async_wait<0>();
                    fence_proxy_async_smem();
                    mbar_arrive(&S.q_full[i]);
                }
            }
            if (!ok) break;
            for (unsigned t = x.t0; t < x.t1; ++t) {
                const unsigned i = place;
                if (!(ok = attn_wait(&empty[i], phase ^ 1, &S, a.status, 537))) break;
                if (lane == 0) mbar_arrive_expect_tx(&full[i], C::kTileBytes);
                __syncwarp();
                unsigned char* dst = ring + i * C::kTileBytes + mine * 128;
                if (mine < kTile) {
                    const int k = x.key0 + (int)t * kTile + mine;
                    if (!runs) {
#pragma unroll
                        for (int c = 0; c < C::kAtoms; ++c)
                            gather4(dst + c * (kTile * 128), row_map, col + 64 * c, y[0], y[1], y[2], y[3], &full[i]);
                    } else if (is_v && ((k < stop && k + per > stop) || (k < x.seen && k + per > x.seen))) {
                        for (int j = 0; j < per; j += 4) {
                            int z[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int key = k + j + e;
                                z[e] = y[0] < a.kv_rows && key >= x.seen && key < stop ? y[0] + j + e : a.kv_rows;
                            }
#pragma unroll
                            for (int c = 0; c < C::kAtoms; ++c)
                                gather4(dst + c * (kTile * 128) + j * 128, row_map, col + 64 * c, z[0], z[1], z[2], z[3], &full[i]);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < C::kAtoms; ++c) load_box2(dst + c * (kTile * 128), run_map, col + 64 * c, y[0], &full[i]);
                    }
                }
                ++issued;
                if (++place == stages) place = 0, phase ^= 1;
                if (t + 1 < x.t1) slots_of(t + 1, y);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if ((warp == 9 || warp == 10) && *(volatile int*)&S.abort) {
        // a role gave up: copies may still be on their way into this CTA's shared memory, so the last of each stage lands first
        auto landed = [&](uint64_t* full, unsigned stages, unsigned count) {
            for (unsigned i = 0; i < stages; ++i) {
                const unsigned n = count > i ? (count - i + stages - 1) / stages : 0;  // copies into stage i
                for (uint32_t j = 0; n > 0 && j < kWaitPolls && !mbar_try_wait(full + i, (n - 1) & 1); ++j) {
                }
            }
        };
        landed(warp == 10 ? S.v_full : S.k_full, warp == 10 ? C::kRingV : C::kRingK, issued);
        if (warp == 9) landed(S.q_full, C::kQ, q_count);
    }
}

// ---- merge --------------------------------------------------------------------------------------------------------------
// out = sum O_i w_i / L over the pieces of the row's prefix item and own item, w_i = 2^(scale (m_i - M)), M = max m_i, L = sum l_i w_i. A
// warp takes one row. Its lanes look up a candidate piece each (a CTA of the item's range, a part of its slot): which slot, m
// and l, all requested at once; then D / 4 lanes read a piece's O (a float4 each), kAhead loads in flight, in the order of the
// candidates. What rests on the lengths alone is done before the wait for the first kernel. The time is the chain of
// three round trips to L2 (plan, m and l, O) behind that kernel's end.
template <int D, bool kHalf, int kAhead>
__global__ void __launch_bounds__(256, kAhead > 4 ? 2 : 3) prefix_merge_kernel(const __grid_constant__ PrefixAttnArgs a) {
    constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes;  // lanes of a piece, pieces read side by side
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)a.rows * a.qh;
    bool waited = false;
    for (long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); id < rows; id += (long long)gridDim.x * 8) {
        const int tok = (int)(id / a.qh), head = (int)(id - (long long)tok * a.qh);
        const int b = request_of_warp(a, tok, lane);
        const Req r = request(a, b);
        const int j = tok - r.first, kv = head / a.G, hg = head - kv * a.G;
        if (!waited) griddep_wait();
        waited = true;
        const unsigned* cum = (const unsigned*)(a.ws + 256);
        const PlanHead h = *(const PlanHead*)a.ws;
        const unsigned cum_step = cum[b], cum_item = cum[a.batch + b];
        if (tok >= (int)h.tokens) return;  // so are all later ones
        if (j < 0 || j >= r.n) continue;

        // the prefix item and the own item: first step, steps, first CTA and number of candidates, slot of CTA 0, place of the row
        struct Item {
            unsigned first, len, front;
            int sh, c0, n, index, R, row, half;
        };
        const bool alone = h.total < kCtas;  // one step a CTA: no second parts
        auto item = [&](unsigned tiles, int rows, int gr, unsigned first, int index, int R) {
            Item e;
            const int block = gr / (2 * kTile), rr = gr - block * 2 * kTile, left = min(2 * kTile, rows - block * 2 * kTile);
            e.sh = left > kTile ? 1 : 0;
            e.front = lead(a, e.sh != 0);
            e.first = first + kv * head_steps(a, tiles, rows) + block * (2 * tiles + lead(a, true));
            e.len = (tiles << e.sh) + e.front;
            e.index = index + kv * row_blocks(rows) + block;
            e.R = R;
            e.row = rr & (kTile - 1);
            e.half = rr >> 7;
            e.c0 = tiles > 0 ? cta_of(e.first + e.front, h.total) : 0;
            e.n = tiles > 0 ? (cta_of(e.first + e.len - 1, h.total) - e.c0 + 1) << (e.sh || alone ? 0 : 1) : 0;
            return e;
        };
        const Item pre = item(h.tiles, (int)h.tokens * a.G, tok * a.G + hg, 0u, 0, kTile);
        const Item ind = item(own_tiles(a, r, (int)h.prefix), r.n * a.G, j * a.G + hg, cum_step, (int)cum_item, a.suffix_rows);
        float M = -INFINITY, Ls = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < pre.n + ind.n; k0 += 32) {
            const int k = k0 + lane;
            const bool own = k >= pre.n;
            const int q = own ? k - pre.n : k, n = own ? ind.n : pre.n, sh = own ? ind.sh : pre.sh, R = own ? ind.R : pre.R, row = own ? ind.row : pre.row;
            const bool one = sh != 0 || alone;
            const int c = (own ? ind.c0 : pre.c0) + (one ? q : q >> 1), s = sh != 0 ? (own ? ind.half : pre.half) : one ? 0 : q & 1;
            const unsigned first = own ? ind.first : pre.first, len = own ? ind.len : pre.len;
            bool on = false;
            if (q < n) {
                const unsigned lo = max(range_lo(h.total, c), first), hi = min(range_lo(h.total, c + 1), first + len);
                unsigned t0 = 0, t1 = 0;
                if (hi > lo) tiles_of(lo - first, hi - first, own ? ind.front : pre.front, sh, t0, t1);
                on = t1 > t0 + (sh != 0 ? 0 : s);
            }
            const float4* src =
                (const float4*)(a.ws + (own ? a.ws_suffix : a.ws_prefix) + ((long long)((own ? ind.index : pre.index) + c) * 2 + s) * part_bytes(R, D)) + row;
            float m = -INFINITY, l = 0.f;
            if (on) {
                const float* ml = (const float*)(src - row + R * (D / 4)) + row;
                m = ml[0];
                l = ml[R];
            }
            unsigned there = __ballot_sync(0xffffffffu, on);
            const unsigned owned = __ballot_sync(0xffffffffu, own);
            bool weighed = false;
            float g = 0.f;
            while (there != 0u) {  // O is asked for before m and l are looked at
                float4 v[kAhead];
                int from[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    from[i] = 32;
#pragma unroll
                    for (int y = 0; y < kAtOnce; ++y) {
                        const int f = there != 0u ? __ffs(there) - 1 : 32;
                        there &= there - 1;
                        if (lane / kLanes == y) from[i] = f;
                    }
                    const float4* p = (const float4*)__shfl_sync(0xffffffffu, (unsigned long long)src, from[i] & 31);
                    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (from[i] < 32) v[i] = p[(lane % kLanes) * ((owned >> from[i]) & 1u ? a.suffix_rows : kTile)];
                }
                if (!weighed) {
                    weighed = true;
                    const float mn = fmaxf(M, warp_max(m));
                    const float f = M == mn ? 1.f : ex2((M - mn) * a.scale_log2);           // of what is there
                    g = l == 0.f ? 0.f : m == mn ? 1.f : ex2((m - mn) * a.scale_log2);  // of this lane's piece (l is NaN where a score was)
                    M = mn;
                    Ls = Ls * f + warp_sum(l * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] *= f;
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const float w = __shfl_sync(0xffffffffu, g, from[i] & 31);
                    if (from[i] < 32 && w != 0.f) {
                        o[0] += v[i].x * w;
                        o[1] += v[i].y * w;
                        o[2] += v[i].z * w;
                        o[3] += v[i].w * w;
                    }
                }
            }
        }
        if (kAtOnce == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += __shfl_xor_sync(0xffffffffu, o[i], 16);
        }
        const float inv = Ls == 0.f ? 0.f : 1.f / Ls;  // a row that saw no key is zero
        if (lane < kLanes)
            *(uint2*)((unsigned char*)a.out + ((long long)tok * a.o_row + head * a.o_head + lane * 4) * 2) =
                make_uint2(pack2<kHalf>(o[0] * inv, o[1] * inv), pack2<kHalf>(o[2] * inv, o[3] * inv));
        if (a.lse != nullptr && lane == 0) a.lse[(long long)tok * a.qh + head] = Ls == 0.f ? -INFINITY : (M * a.scale_log2 + (log2f(Ls) - kLift<kHalf>)) * kLn2;
    }
}

// Loads in flight of a merging thread where rows are so few that every block has its place at once: the rows' chains are what it
// takes (64 decodes: 27.9 us with 4, 26.8 with 6, 8 or 10). Where blocks come in rounds, registers for a third block an SM do
// more (32 x 16 rows: two blocks 125 us, three 121).
constexpr int kWide = 8;
BatchDims prefix_attn_dims(int dim) { return {kCtas, kAttnThreads, (size_t)(dim == 64 ? Cfg<64>::kSmem : Cfg<128>::kSmem)}; }
BatchDims prefix_merge_dims(const PrefixAttnArgs& a) {
    // at most four rounds of three blocks an SM: rows beyond the batch's must not cost a block each
    const long long blocks = ((long long)a.rows * a.qh + 7) / 8, most = 12ll * kCtas;
    return {(unsigned)(blocks < most ? blocks : most), 256, 0};
}
template <int D, bool kHalf>
static cudaError_t prefix_attn_run(const PrefixAttnArgs& a, const PrefixAttnMaps& maps, cudaStream_t s, bool pdl) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    const BatchDims d = prefix_attn_dims(D), merge = prefix_merge_dims(a);
    cfg.gridDim = dim3(d.grid);
    cfg.blockDim = dim3(d.block);
    cfg.dynamicSmemBytes = d.smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, prefix_attn_kernel<D, kHalf>, a, maps);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(merge.grid);
    cfg.blockDim = dim3(merge.block);
    cfg.dynamicSmemBytes = merge.smem;
    cfg.numAttrs = 1;  // its wait is its first statement, so it may always start under the first kernel's tail
    if (merge.grid <= 2 * kCtas) return cudaLaunchKernelEx(&cfg, prefix_merge_kernel<D, kHalf, kWide>, a);
    return cudaLaunchKernelEx(&cfg, prefix_merge_kernel<D, kHalf, 4>, a);
}

cudaError_t prefix_attn_launch(const PrefixAttnArgs& a, const PrefixAttnMaps& maps, int dim, bool fp16, cudaStream_t s, bool pdl) {
    if (dim == 64) return fp16 ? prefix_attn_run<64, true>(a, maps, s, pdl) : prefix_attn_run<64, false>(a, maps, s, pdl);
    return fp16 ? prefix_attn_run<128, true>(a, maps, s, pdl) : prefix_attn_run<128, false>(a, maps, s, pdl);
}

cudaError_t prefix_attn_prepare() {
    cudaError_t e = cudaFuncSetAttribute(prefix_attn_kernel<64, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<64>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(prefix_attn_kernel<64, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<64>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(prefix_attn_kernel<128, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<128>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(prefix_attn_kernel<128, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<128>::kSmem);
    return e;
}

}  // namespace mk
