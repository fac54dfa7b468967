// Argument records and launchers of the batched decode step's cache path: block tables and slot maps, rope tables, the
// rotation with its K/V append, attention over a paged cache whose first tokens the batch shares.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mk {

// status words shared by the four (params: a caller-owned i32 [16] block): the first recorder wins
__device__ __forceinline__ void batch_status(int* status, int code, int where, int observed, int expected) {
    if (status != nullptr && atomicCAS(status, 0, code) == 0) {
        status[1] = where;
        status[2] = (int)blockIdx.x;
        status[3] = observed;
        status[4] = expected;
    }
}

constexpr int kMaxBatch = 4096;        // requests of a block-table or attention launch
constexpr int kAttnCtas = 148;         // CTAs of an attention launch: one an SM
constexpr int kMaxPoolRows = 1 << 18;  // rows of the request table (two bits each in shared memory)

struct BlockTablesArgs {
    const long long* seq_lens;
    const long long* new_lens;
    const long long* req;
    int* req_to_page;
    int pool_rows, width;
    int* owned;
    const int* ring;
    long long ring_len;
    long long* words;
    int page;
    int batch, rows;
    int* table;
    long long* slots;
    long long* positions;
    int* cu_rows;
    int* kv_lens;
    unsigned* ticket;
    int* status;
};

constexpr int kMaxRot = 256;
struct RopeTableArgs {
    float* out;
    long long rows, first;
    int rot;
    double mult;
    double turns[kMaxRot / 2];  // turns per position of each frequency: inv_freq / 2 pi
    double2 step[kMaxRot / 2];  // cos and sin of one position's angle
};

struct RotaryArgs {
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    void* k_out;
    long long q_row, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head, ko_row, ko_head;  // strides in elements
    const long long* positions;
    const float* cos_sin;
    long long cos_rows;
    const long long* slots;
    void* k_cache;
    void* v_cache;
    long long kc_row, kc_head, vc_row, vc_head, kv_rows;
    const int* n_rows;
    int rows, qh, kvh, dim, rot, inverse;
    int* status;
};

struct PrefixAttnArgs {
    const void* q;
    long long q_row, q_head;
    void* out;
    long long o_row, o_head;
    float* lse;
    const int* table;
    long long table_row;
    int width;
    const int* kv_lens;
    const int* cu_rows;
    const int* prefix_len;
    int batch, rows, max_new, qh, kvh, G, page, page_shift, kv_rows, window, suffix_rows;
    int k_head, v_head;  // elements between the heads of a cache row
    int item_steps;      // what an item costs besides its steps, counted in steps
    int pair_steps;      // the same of one of more than 128 rows, beyond that
    int run;             // rows of a copy: the largest power of two up to 128 that divides the page
    int q_box;           // the queries of a tile are 128 / G whole tokens: copied as a box
    float scale_log2;
    unsigned char* ws;
    long long ws_prefix, ws_suffix;  // byte offsets of the partials in ws
    int* status;
};

// tensor maps of 64-element wide columns: boxes of `run` cache rows, single cache rows (for gathers), G heads x 128 / G tokens
struct PrefixAttnMaps {
    CUtensorMap k_run, v_run, k_row, v_row, q;
};

// a kernel's launch shape
struct BatchDims {
    unsigned grid, block;
    size_t smem;
};
BatchDims block_tables_dims(const BlockTablesArgs& a, int sms);
BatchDims rope_table_dims(const RopeTableArgs& a, int sms);
BatchDims rotary_dims(const RotaryArgs& a, bool interleaved);
BatchDims prefix_attn_dims(int dim);                        // its first kernel
BatchDims prefix_merge_dims(const PrefixAttnArgs& a);       // its second
cudaError_t block_tables_launch(const BlockTablesArgs& a, int sms, cudaStream_t s, bool pdl);
cudaError_t rope_table_launch(const RopeTableArgs& a, int sms, cudaStream_t s, bool pdl);
cudaError_t rotary_launch(const RotaryArgs& a, bool fp16, bool interleaved, cudaStream_t s, bool pdl);
cudaError_t prefix_attn_launch(const PrefixAttnArgs& a, const PrefixAttnMaps& maps, int dim, bool fp16, cudaStream_t s, bool pdl);
cudaError_t batch_prepare();
cudaError_t prefix_attn_prepare();

}  // namespace mk
