// The cache path of a batched decode step, up to its attention:
//
//   block_tables   pages, slots and positions of the step's new tokens from the requests' lengths
//   rope_table     cos | sin rows of a range of positions
//   rotary         rotation of q and k, store of q, append of k and v at their slots
//
// None has more than a few operations a byte: they are bound by memory, and at a decode step's sizes by the latency of
// their few dependent loads, so each is one launch whose CTAs repeat the small common work instead of meeting.
#include "batch.h"
#include "util.cuh"

namespace mk {

// ---- block tables ---------------------------------------------------------------------------------------------------
// need_b = ceil((seq_b + new_b) / page), take_b = max(0, need_b - owned_b); the first row of request b is the sum of the
// earlier requests' new_b, its first page from the ring the sum of their take_b. Every CTA computes both prefix sums over
// the whole batch into shared memory (24 bytes a request; two dependent round trips to L2), then fills its share of the
// table entries and rows. Table entries below owned_b come from the request's own row, the others straight from the ring,
// so no CTA reads what another writes. The two words that every CTA reads and the launch advances (pages owned, ring
// head) are written by the CTA that arrives last, after all have read them. One request: 5.2 us inside a graph, 256 requests x 2064
// pages (3.2 MB): 6.8 us, bound by those dependent loads; 7.8 and 8.5 a call on a stream.
struct TablesShared {
    int *seq, *cu, *off, *own, *need, *row;
    unsigned *seen, *twice;
};
__device__ __forceinline__ TablesShared tables_carve(unsigned char* p, int batch, int words) {
    TablesShared s;
    s.seq = (int*)p;
    s.cu = s.seq + batch;
    s.off = s.cu + batch + 1;
    s.own = s.off + batch;
    s.need = s.own + batch;
    s.row = s.need + batch;
    s.seen = (unsigned*)(s.row + batch);
    s.twice = s.seen + words;
    return s;
}
static size_t block_tables_smem(int batch, int pool_rows) { return ((size_t)batch * 6 + 1) * 4 + (size_t)((pool_rows + 31) / 32) * 8; }

constexpr int kTablesThreads = 256;

__global__ void __launch_bounds__(kTablesThreads) block_tables_kernel(const BlockTablesArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ long long w_rows[kTablesThreads / 32], w_take[kTablesThreads / 32];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int words = (a.pool_rows + 31) / 32;
    const TablesShared s = tables_carve(smem, a.batch, words);
    for (int i = tid; i < 2 * words; i += kTablesThreads) s.seen[i] = 0u;
    __syncthreads();
    griddep_wait();

    const long long cap = (long long)a.width * a.page;  // tokens a request's row can hold
    const long long head = a.words[0], tail = a.words[1];
    // pass 1: lengths and request rows; a request row named twice is found through one bit a row
    for (int b = tid; b < a.batch; b += kTablesThreads) {
        const long long seq = a.seq_lens[b], nw = a.new_lens[b], rq = a.req[b];
        int row = -1, sq = 0, n = 0, own = 0;
        if (seq != 0 || nw != 0) {
            if (seq < 0 || nw < 0 || seq > cap || nw > cap || seq + nw > cap || rq < 0 || rq >= a.pool_rows) {
                batch_status(a.status, 4, 500, b, 0);
            } else {
                row = (int)rq;
                sq = (int)seq;
                n = (int)nw;
                own = a.owned[row];
                if (atomicOr(&s.seen[row >> 5], 1u << (row & 31)) & (1u << (row & 31))) atomicOr(&s.twice[row >> 5], 1u << (row & 31));
            }
        }
        s.seq[b] = sq;
        s.cu[b] = n;
        s.own[b] = own;
        s.row[b] = row;
    }
    __syncthreads();
    // pass 2: what each request needs, and the two prefix sums
    long long rows_sum = 0, take_sum = 0;  // of the requests before this round
    for (int b0 = 0; b0 < a.batch; b0 += kTablesThreads) {
        const int b = b0 + tid;
        int n = 0, take = 0, need = 0;
        if (b < a.batch && s.row[b] >= 0) {
            const int row = s.row[b], own = s.own[b];
            const int held = (int)(((long long)s.seq[b] + a.page - 1) / a.page);
            if ((s.twice[row >> 5] >> (row & 31)) & 1u) {
                batch_status(a.status, 4, 501, b, row);
                s.row[b] = -1;
                s.seq[b] = 0;
            } else if (own < held || own > a.width) {
                batch_status(a.status, 4, 502, b, own);
                s.row[b] = -1;
                s.seq[b] = 0;
            } else {
                n = s.cu[b];
                need = (int)(((long long)s.seq[b] + n + a.page - 1) / a.page);
                take = need > own ? need - own : 0;
            }
        }
        long long xr = n, xt = take;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long yr = __shfl_up_sync(0xffffffffu, xr, o), yt = __shfl_up_sync(0xffffffffu, xt, o);
            if (lane >= o) xr += yr, xt += yt;
        }
        if (lane == 31) w_rows[warp] = xr, w_take[warp] = xt;
        __syncthreads();
        long long br = rows_sum, bt = take_sum, tr = 0, tt = 0;
#pragma unroll
        for (int w = 0; w < kTablesThreads / 32; ++w) {
            if (w < warp) br += w_rows[w], bt += w_take[w];
            tr += w_rows[w];
            tt += w_take[w];
        }
        if (b < a.batch) {
            // sums beyond 32 bits only occur in steps that are refused below
            s.cu[b] = (int)(br + xr - n);
            s.off[b] = (int)(bt + xt - take);
            s.need[b] = need;
        }
        rows_sum += tr;
        take_sum += tt;
        __syncthreads();
    }
    const bool ring_ok = head >= 0 && tail >= head && tail - head <= a.ring_len;
    const bool grant = rows_sum <= a.rows && (take_sum == 0 || (ring_ok && take_sum <= tail - head));
    if (!grant) {  // all or nothing: the step gets no rows and no pages
        if (tid == 0 && blockIdx.x == 0) {
            if (rows_sum > a.rows) batch_status(a.status, 5, 503, (int)min(rows_sum, 0x7fffffffll), a.rows);
            else if (!ring_ok) batch_status(a.status, 4, 505, (int)head, (int)tail);
            else batch_status(a.status, 5, 504, (int)min(take_sum, 0x7fffffffll), (int)min(tail - head, 0x7fffffffll));
        }
        for (int b = tid; b < a.batch; b += kTablesThreads) {
            s.cu[b] = 0;
            s.need[b] = (int)(((long long)s.seq[b] + a.page - 1) / a.page);
        }
        rows_sum = take_sum = 0;
    }
    if (tid == 0) s.cu[a.batch] = (int)rows_sum;
    __syncthreads();
    // this CTA has read the words that the last to get here advances
    if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
        __threadfence();
    }
    __syncthreads();
    if (s_last) {
        for (int b = tid; b < a.batch; b += kTablesThreads)
            if (s.row[b] >= 0 && s.need[b] > s.own[b]) a.owned[s.row[b]] = s.need[b];
        if (tid == 0) {
            a.words[0] = head + take_sum;
            *a.ticket = 0u;
        }
    }
    if (blockIdx.x == 0) {
        for (int b = tid; b <= a.batch; b += kTablesThreads) {
            a.cu_rows[b] = s.cu[b];
            if (b < a.batch) a.kv_lens[b] = s.seq[b] + (s.cu[b + 1] - s.cu[b]);
        }
    }
    const long long head_at = ring_ok ? head % a.ring_len : 0;
    auto page_of = [&](int b, int p) -> int {  // page p < need_b of request b
        if (p < s.own[b]) return a.req_to_page[(long long)s.row[b] * a.width + p];
        long long at = head_at + s.off[b] + (p - s.own[b]);
        if (at >= a.ring_len) at -= a.ring_len;
        return a.ring[at];
    };
    // the table, 1024 entries of one request at a time
    const int per = (a.width + 1023) / 1024;
    for (long long c = blockIdx.x; c < (long long)a.batch * per; c += gridDim.x) {
        const int b = (int)(c / per), p0 = (int)(c - (long long)b * per) * 1024;
        const int need = s.need[b];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = p0 + i * kTablesThreads + tid;
            if (p >= a.width) break;
            int page = -1;
            if (p < need) {
                page = page_of(b, p);
                if (p >= s.own[b]) a.req_to_page[(long long)s.row[b] * a.width + p] = page;
            }
            a.table[(long long)b * a.width + p] = page;
        }
    }
    // the new tokens' rows: the request by bisection of cu_rows in shared memory
    for (long long r = (long long)blockIdx.x * kTablesThreads + tid; r < rows_sum; r += (long long)gridDim.x * kTablesThreads) {
        int lo = 0, hi = a.batch;  // the last b with cu[b] <= r
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s.cu[mid] <= r) lo = mid;
            else hi = mid;
        }
        const int pos = s.seq[lo] + ((int)r - s.cu[lo]), p = pos / a.page;
        a.slots[r] = (long long)page_of(lo, p) * a.page + (pos - p * a.page);
        a.positions[r] = pos;
    }
}

// ---- rope table -----------------------------------------------------------------------------------------------------
// out[r] = {cos(pos f_i) | sin(pos f_i)} mult, pos = first + r. Angles are held in turns in 64 bits (pos f_i / 2 pi less its
// whole part, exact to 2^-52 of the angle), because a far position times a frequency keeps too few bits of its fraction
// in 32. A 64-bit sine pair costs about a hundred double operations, so a thread evaluates it once for kRows positions of a
// frequency and turns on from one position to the next by the addition theorem with the pair of a single step (from the
// host): four double operations a pair, error at most kRows 2^-52 against the 2^-24 of the result's own rounding. 131,072 x 128
// (67 MB): 15.1 us a table of three in turn, 4.4 TB/s of stores; 8,448 x 64: 2.5 us, one thread's chain.
template <int kRows>
__global__ void __launch_bounds__(128) rope_table_kernel(const RopeTableArgs a) {
    const int F = a.rot / 2, groups = F / 4;  // a thread: four neighbouring frequencies of kRows positions
    const long long id = (long long)blockIdx.x * 128 + threadIdx.x;
    const int f = (int)(id % groups) * 4;
    const long long r0 = id / groups * kRows;
    double c[4], s[4], cs[4], sn[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        cs[j] = a.step[f + j].x;
        sn[j] = a.step[f + j].y;
        const double t = (double)(a.first + r0) * a.turns[f + j];
        sincospi(2.0 * (t - rint(t)), &s[j], &c[j]);
        c[j] *= a.mult;
        s[j] *= a.mult;
    }
    griddep_wait();
    float* out = a.out + r0 * a.rot + f;
#pragma unroll 4
    for (int l = 0; l < kRows; ++l) {
        if (r0 + l >= a.rows) return;
        *(float4*)out = make_float4((float)c[0], (float)c[1], (float)c[2], (float)c[3]);
        *(float4*)(out + F) = make_float4((float)s[0], (float)s[1], (float)s[2], (float)s[3]);
        out += a.rot;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double x = c[j];
            c[j] = x * cs[j] - s[j] * sn[j];
            s[j] = s[j] * cs[j] + x * sn[j];
        }
    }
}

// ---- rotary ---------------------------------------------------------------------------------------------------------
// A pair (x, y) of the first `rot` dims becomes (x c - y s, y c + x s), in f32 with one rounding at the end; half layout:
// y = x's index + rot / 2, interleaved: neighbours. A CTA takes one token. A thread keeps the cos / sin of its dims in
// registers and walks the heads with it, so the table row is read once a token and not once a head; every value is read
// and written once, in 16-byte pieces (8-byte ones where half of rot is no multiple of 8). Bound by DRAM: 8192 rows x 160 heads of
// 64 (338 MB) take 63 us, 5.4 TB/s; 16 rows 2.5 us, two dependent loads.
template <typename T>
struct Pair;
template <>
struct Pair<__half> {
    typedef __half2 type;
    static __device__ __forceinline__ float2 up(__half2 v) { return __half22float2(v); }
    static __device__ __forceinline__ __half2 down(float x, float y) { return __floats2half2_rn(x, y); }
};
template <>
struct Pair<__nv_bfloat16> {
    typedef __nv_bfloat162 type;
    static __device__ __forceinline__ float2 up(__nv_bfloat162 v) { return __bfloat1622float2(v); }
    static __device__ __forceinline__ __nv_bfloat162 down(float x, float y) { return __floats2bfloat162_rn(x, y); }
};
template <int N>
struct Words;
template <>
struct Words<8> {
    typedef uint4 type;
};
template <>
struct Words<4> {
    typedef uint2 type;
};

template <typename T, int N, bool kInter>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
    typedef typename Words<N>::type W;
    typedef Pair<T> P2;
    typedef typename P2::type T2;
    griddep_wait();
    // Rows that are not live cost one word. Nothing else waits for what it does not need: the row's words and the first heads
    // are asked for together, the table row follows the position, the checks come behind all loads.
    const int r = blockIdx.x;
    if (a.n_rows != nullptr && r >= *a.n_rows) return;
    long long pos = a.positions[r];
    long long slot = a.k_cache != nullptr ? a.slots[r] : -1;
    const T* qr = (const T*)a.q + r * a.q_row;
    const T* kr = (const T*)a.k + r * a.k_row;
    T* qo = (T*)a.q_out + r * a.qo_row;
    T* ko = a.k_out != nullptr ? (T*)a.k_out + r * a.ko_row : nullptr;
    const int half = a.rot / 2;
    // pieces of a head: the rotated ones (a piece holds N pairs in the half layout, N / 2 in the interleaved one), then the rest
    const int turn = kInter ? a.rot / N : half / N, pieces = turn + (a.dim - a.rot) / N;
    const int step = blockDim.x / pieces, c = threadIdx.x % pieces;
    constexpr int kHeads = 3;  // heads in flight a thread
    const bool mine = (int)threadIdx.x < step * pieces, turned = c < turn;
    const int at = turned ? c * N : a.rot + (c - turn) * N;
    int h0 = mine ? (int)threadIdx.x / pieces : a.qh + a.kvh;
    W w0[kHeads], w1[kHeads];
    auto load_heads = [&]() {
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int hh = h0 + i * step;
            if (hh < a.qh + a.kvh) {
                const T* src = hh < a.qh ? qr + hh * a.q_head : kr + (hh - a.qh) * a.k_head;
                w0[i] = *(const W*)(src + at);
                if (!kInter && turned) w1[i] = *(const W*)(src + half + at);
            }
        }
    };
    load_heads();
    // v: from the block's last thread backwards, as the first threads have the heads' remainder
    const T* vr = (const T*)a.v + r * a.v_row;
    const int vp = a.dim / 8, v0 = blockDim.x - 1 - threadIdx.x;
    uint4 vw = make_uint4(0, 0, 0, 0);
    if (a.v != nullptr && v0 < a.kvh * vp) vw = *(const uint4*)(vr + v0 / vp * a.v_head + v0 % vp * 8);
    if (pos < 0 || pos >= a.cos_rows) {
        if (threadIdx.x == 0) batch_status(a.status, 4, 510, (int)pos, (int)min(a.cos_rows, 0x7fffffffll));
        pos = 0;
    }
    if (slot >= a.kv_rows && a.k_cache != nullptr) {
        if (threadIdx.x == 0) batch_status(a.status, 4, 511, (int)min(slot, 0x7fffffffll), (int)min(a.kv_rows, 0x7fffffffll));
        slot = -1;
    }
    T* kc = slot >= 0 ? (T*)a.k_cache + slot * a.kc_row : nullptr;
    const float* tab = a.cos_sin + pos * a.rot;
    if (mine) {
        float cs[N], sn[N];
        if (turned) {
            constexpr int n = kInter ? N / 2 : N;
#pragma unroll
            for (int j = 0; j < n; j += 2) {
                const float2 x = *(const float2*)(tab + c * n + j), y = *(const float2*)(tab + half + c * n + j);
                cs[j] = x.x, cs[j + 1] = x.y;
                sn[j] = a.inverse ? -y.x : y.x, sn[j + 1] = a.inverse ? -y.y : y.y;
            }
        }
        while (true) {
#pragma unroll
            for (int i = 0; i < kHeads; ++i) {
                const int hh = h0 + i * step;
                if (hh >= a.qh + a.kvh) break;
                const bool isq = hh < a.qh;
                const int h = isq ? hh : hh - a.qh;
                auto put = [&](int d, const W& w) {
                    if (isq) *(W*)(qo + h * a.qo_head + d) = w;
                    else {
                        if (ko != nullptr) *(W*)(ko + h * a.ko_head + d) = w;
                        if (kc != nullptr) *(W*)(kc + h * a.kc_head + d) = w;
                    }
                };
                T2* x0 = (T2*)&w0[i];
                T2* x1 = (T2*)&w1[i];
                if (turned) {
                    if (kInter) {
#pragma unroll
                        for (int j = 0; j < N / 2; ++j) {
                            const float2 v = P2::up(x0[j]);
                            x0[j] = P2::down(v.x * cs[j] - v.y * sn[j], v.y * cs[j] + v.x * sn[j]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < N / 2; ++j) {
                            const float2 x = P2::up(x0[j]), y = P2::up(x1[j]);
                            x0[j] = P2::down(x.x * cs[2 * j] - y.x * sn[2 * j], x.y * cs[2 * j + 1] - y.y * sn[2 * j + 1]);
                            x1[j] = P2::down(y.x * cs[2 * j] + x.x * sn[2 * j], y.y * cs[2 * j + 1] + x.y * sn[2 * j + 1]);
                        }
                        put(half + at, w1[i]);
                    }
                }
                put(at, w0[i]);
            }
            h0 += kHeads * step;
            if (h0 >= a.qh + a.kvh) break;
            load_heads();
        }
    }
    if (a.v != nullptr && slot >= 0) {
        T* vc = (T*)a.v_cache + slot * a.vc_row;
        for (int i = v0; i < a.kvh * vp; i += blockDim.x) {
            const int h = i / vp, d = (i - h * vp) * 8;
            *(uint4*)(vc + h * a.vc_head + d) = i == v0 ? vw : *(const uint4*)(vr + h * a.v_head + d);
        }
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------
template <typename K, typename A>
static cudaError_t launch_batch(K kern, const BatchDims& d, cudaStream_t s, bool pdl, const A& a) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(d.grid);
    cfg.blockDim = dim3(d.block);
    cfg.dynamicSmemBytes = d.smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

BatchDims block_tables_dims(const BlockTablesArgs& a, int sms) {
    const long long chunks = (long long)a.batch * ((a.width + 1023) / 1024), rows = ((long long)a.rows + kTablesThreads - 1) / kTablesThreads;
    long long grid = chunks > rows ? chunks : rows;
    if (grid > 2 * sms) grid = 2 * sms;
    return {(unsigned)grid, kTablesThreads, block_tables_smem(a.batch, a.pool_rows)};
}
cudaError_t block_tables_launch(const BlockTablesArgs& a, int sms, cudaStream_t s, bool pdl) {
    return launch_batch(block_tables_kernel, block_tables_dims(a, sms), s, pdl, a);
}

// 16 positions a thread once that fills the SMs; 4 for short tables, whose time is one thread's chain
static int rope_rows(const RopeTableArgs& a, int sms) { return (a.rows + 15) / 16 * (a.rot / 8) >= 256ll * sms ? 16 : 4; }
BatchDims rope_table_dims(const RopeTableArgs& a, int sms) {
    const long long rows = rope_rows(a, sms), groups = a.rot / 8;
    return {(unsigned)(((a.rows + rows - 1) / rows * groups + 127) / 128), 128, 0};
}
cudaError_t rope_table_launch(const RopeTableArgs& a, int sms, cudaStream_t s, bool pdl) {
    if (rope_rows(a, sms) == 16) return launch_batch(rope_table_kernel<16>, rope_table_dims(a, sms), s, pdl, a);
    return launch_batch(rope_table_kernel<4>, rope_table_dims(a, sms), s, pdl, a);
}

static bool rotary_wide(const RotaryArgs& a, bool inter) { return inter || (a.rot / 2) % 8 == 0; }
BatchDims rotary_dims(const RotaryArgs& a, bool inter) {
    const int n = rotary_wide(a, inter) ? 8 : 4, pieces = (inter ? a.rot / n : a.rot / 2 / n) + (a.dim - a.rot) / n;
    int threads = ((a.qh + a.kvh) * pieces + 31) / 32 * 32;
    if (threads > 256) threads = 256;
    return {(unsigned)a.rows, (unsigned)threads, 0};
}
template <typename T>
static cudaError_t rotary_typed(const RotaryArgs& a, bool inter, cudaStream_t s, bool pdl) {
    const BatchDims d = rotary_dims(a, inter);
    if (inter) return launch_batch(rotary_kernel<T, 8, true>, d, s, pdl, a);
    if (rotary_wide(a, inter)) return launch_batch(rotary_kernel<T, 8, false>, d, s, pdl, a);
    return launch_batch(rotary_kernel<T, 4, false>, d, s, pdl, a);
}
cudaError_t rotary_launch(const RotaryArgs& a, bool fp16, bool interleaved, cudaStream_t s, bool pdl) {
    return fp16 ? rotary_typed<__half>(a, interleaved, s, pdl) : rotary_typed<__nv_bfloat16>(a, interleaved, s, pdl);
}

cudaError_t batch_prepare() {
    cudaError_t e = cudaFuncSetAttribute(block_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)block_tables_smem(kMaxBatch, kMaxPoolRows));
    return e;
}

}  // namespace mk
