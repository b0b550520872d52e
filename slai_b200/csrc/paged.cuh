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
    int page_size, n_kv, group, hs;
};

struct AttnArgs {
    Cache c;
    int lane, starts_at;  // kind of kernel, offset of its blocks' starts
    const float* q;
    float* out;
    long long q_ld, out_ld;  // floats between tokens
    float scale;
    int tile_rows, unit;     // of the lane
    int vec;                 // rows of the cache can be read in 16-byte pieces
    int qvec;                // ... and rows of q and out
    float* part;             // [block][2][tile_rows][hs]: sums of (tile, head) pairs that lie on several blocks
    float* part_ml;          // [block][2][tile_rows][2]: their largest scores (times log2 e) and sums of weights
    unsigned int* tickets;   // [block], zero between launches
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
// The block that has unit `x` of the line, and which blocks share a (tile, head) pair.
__device__ __forceinline__ int block_of(const Start& s, long long x) { return (int)(((x + 1) * s.blocks - 1) / s.units); }

// Joins the results of a pair that lies on several blocks.  All threads of the block call it after their stores to the block's slot of `part`; true in the
// block that comes last, which then reads the slots of blocks first .. last (of the first: slot 1, of the others: slot 0).  `flag`: shared memory.
__device__ __forceinline__ bool last_to_come(unsigned int* ticket, int n, int* flag) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned int before = atomicAdd(ticket, 1u);
        const bool last = before == (unsigned int)(n - 1);
        if (last) *ticket = 0;  // for the next launch
        *flag = last;
    }
    __syncthreads();
    __threadfence();
    return *flag != 0;
}

// Rows of a tile: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the blocks' results in order of their positions.  A block that saw nothing of a
// row has m = -inf, l = 0, o = 0.
template <int THREADS>
__device__ __forceinline__ void join(const AttnArgs& A, const Tile& t, int head, int first, int last) {
    const int hs = A.c.hs, lanes = hs % 4 == 0 ? hs / 4 : hs, w = hs % 4 == 0 ? 4 : 1;
    const size_t rows = (size_t)A.tile_rows;
    for (int i = threadIdx.x; i < t.rows * lanes; i += THREADS) {
        const int r = i / lanes, d = (i - r * lanes) * w;
        float M = -INFINITY;
        for (int b = first; b <= last; b++) M = fmaxf(M, __ldcg(A.part_ml + (((size_t)b * 2 + (b == first)) * rows + r) * 2));
        float num[4] = {}, den = 0.f;
        for (int b = first; b <= last; b++) {
            const size_t slot = ((size_t)b * 2 + (b == first)) * rows + r;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(A.part_ml) + slot);
            const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
            den = fmaf(f, ml.y, den);
            if (w == 4) {
                const float4 o = __ldcg(reinterpret_cast<const float4*>(A.part + slot * hs + d));
                num[0] = fmaf(f, o.x, num[0]); num[1] = fmaf(f, o.y, num[1]); num[2] = fmaf(f, o.z, num[2]); num[3] = fmaf(f, o.w, num[3]);
            } else {
                num[0] = fmaf(f, __ldcg(A.part + slot * hs + d), num[0]);
            }
        }
        const int pr = t.first + r, tok = pr / A.c.group, qh = head * A.c.group + pr % A.c.group;
        float* o = A.out + (t.row0 + tok) * A.out_ld + (long long)qh * hs + d;
        for (int e = 0; e < w; e++) o[e] = num[e] / den;
    }
}
#endif

}  // namespace paged

bool paged_attention_few(int kv_dtype, int hs);
int paged_attention_launch(slai_ctx* ctx, paged::AttnArgs& A, int kv_dtype, int lane, int blocks, bool pdl);

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
