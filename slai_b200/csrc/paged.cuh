// Shared by the kernels over a paged key / value cache (paged.cu: handle and entry points; paged_append.cu; paged_attention.cu).
#pragma once
#include "common.cuh"
#include "paged_plan.h"

namespace paged {

// One launch's view of the cache and of the step.
struct Cache {
    const int* plan;      // the step's device copy (paged_plan.h)
    int count_at, rows_at;  // offsets of the number of its rows, and of these
    char *keys, *values;
    long long page_stride, head_stride, pos_stride;  // elements
    Div page_size, group;
    int n_kv, hs;
};

struct AttnArgs {
    Cache c;
    int starts_at, joins_at, count_at;  // offsets of the blocks' starts, of the joins, of the joins' number
    const float* q;
    float* out;
    long long q_ld, out_ld;  // floats between tokens
    float scale;
    int n_pages;
    int tile_rows, unit;     // of the lane
    int recorded;            // the launch has room for any step: blocks and joins that this one does not have
    int vec;                 // rows of the cache can be read in 16-byte pieces
    int qvec;                // ... and rows of q and out
    float* part;             // [block][2][tile_rows][hs]: sums of (tile, head) pairs that lie on several blocks
    float* part_ml;          // [block][2][tile_rows][2]: their largest scores (times log2 e) and sums of weights
    unsigned int* err_flag;
    unsigned int wait_limit;
};

#ifdef __CUDACC__
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ Start load_start(const int* plan, int starts_at, int block) {
    Start s;
    const int4* g = reinterpret_cast<const int4*>(plan + starts_at) + 4 * (size_t)block;
    int4* d = reinterpret_cast<int4*>(&s);
#pragma unroll
    for (int i = 0; i < 4; i++) d[i] = __ldcg(g + i);
    return s;
}
__device__ __forceinline__ Tile load_tile(const int* plan, int tiles_at, int tile) {
    Tile t;
    const int4* g = reinterpret_cast<const int4*>(plan + tiles_at) + 2 * (size_t)tile;
    int4* d = reinterpret_cast<int4*>(&t);
    d[0] = __ldcg(g);
    d[1] = __ldcg(g + 1);
    return t;
}
// Place of position `p` of a sequence in the cache, in elements, for one cache head.
__device__ __forceinline__ long long place_of(const Cache& c, int table, int p, int head) {
    const int i = p / c.page_size;
    return __ldcg(c.plan + table + i) * c.page_stride + head * c.head_stride + (p - i * c.page_size) * c.pos_stride;
}
#endif

}  // namespace paged

bool paged_attention_few(int kv_dtype, int hs);
paged::Lane paged_attention_lane(int kv_dtype, int hs, int group, int sms);
// One lane's kernel with `blocks` blocks, and the joins of at most `joins` pairs of at most `longest` results.
int paged_attention_launch(slai_ctx* ctx, paged::AttnArgs& A, int kv_dtype, int lane, int blocks, int joins, int longest, bool pdl);

// paged_prompt.cu, paged_prompt32.cu
paged::Lane paged_prompt_lane(int sms);
int paged_prompt_launch(slai_ctx* ctx, const paged::AttnArgs& A, int blocks, bool pdl);
paged::Lane paged_prompt32_lane(int sms);
int paged_prompt32_launch(slai_ctx* ctx, const paged::AttnArgs& A, int blocks, bool pdl);

// paged_append.cu
struct QkArgs {
    int rows, counted;            // counted: there are as many rows as the step has when the kernel runs, `rows` at most
    int hs, n_q, n_kv, variant;
    float eps;
    const float *q_norm, *k_norm;
    const float *q, *k, *v;       // v null: no cache (k goes to k_out)
    float *q_out, *k_out;
    long long q_ld, k_ld, v_ld, q_out_ld, k_out_ld;
    const int* pos;               // [rows], without a cache
    const double* turns;          // turns per position of each pair (null: no rotation)
    paged::Cache cache;           // with a cache
    int kv_f16;
};
int qk_launch(slai_ctx* ctx, QkArgs& A, bool pdl);
