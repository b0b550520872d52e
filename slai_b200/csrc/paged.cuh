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
// row has m = -inf, l = 0, o = 0.  All (m, l) of some rows come to shared memory at once (`room` pairs), the o's eight at a time: one pair at a time, a
// sequence over 37 blocks took a trip to L2 for each.
template <int THREADS>
__device__ __forceinline__ void join(const AttnArgs& A, const Tile& t, int head, int first, int last, float2* ml, int room) {
    const int hs = A.c.hs, w = hs % 4 == 0 ? 4 : 1, lanes = hs / w, nb = last - first + 1;
    const size_t rows = (size_t)A.tile_rows;
    auto slot = [&](int i, int r) { return ((size_t)(first + i) * 2 + (i == 0)) * rows + r; };
    const int at_once = max(1, min(t.rows, room / nb));
    for (int r0 = 0; r0 < t.rows; r0 += at_once) {
        const int nr = min(at_once, t.rows - r0);
        __syncthreads();
        for (int i = threadIdx.x; i < nr * nb && i < room; i += THREADS) ml[i] = __ldcg(reinterpret_cast<const float2*>(A.part_ml) + slot(i % nb, r0 + i / nb));
        __syncthreads();
        for (int i = threadIdx.x; i < nr * lanes; i += THREADS) {
            const int r = i / lanes, d = (i - r * lanes) * w;
            const float2* x = ml + r * nb;
            float M = -INFINITY;
            for (int b = 0; b < nb; b++) M = fmaxf(M, b < room ? x[b].x : __ldcg(A.part_ml + 2 * slot(b, r0 + r)));
            float num[4] = {}, den = 0.f;
            for (int b0 = 0; b0 < nb; b0 += 8) {
                float4 o[8];
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (b0 + u < nb) {
                        const float* p = A.part + slot(b0 + u, r0 + r) * hs + d;
                        if (w == 4) o[u] = __ldcg(reinterpret_cast<const float4*>(p));
                        else o[u].x = __ldcg(p);
                    }
                }
#pragma unroll
                for (int u = 0; u < 8; u++)
                    if (b0 + u < nb) {
                        const float2 y = b0 + u < room ? x[b0 + u] : __ldcg(reinterpret_cast<const float2*>(A.part_ml) + slot(b0 + u, r0 + r));
                        const float f = y.x == -INFINITY ? 0.f : exp2f(y.x - M);
                        den = fmaf(f, y.y, den);
                        num[0] = fmaf(f, o[u].x, num[0]); num[1] = fmaf(f, o[u].y, num[1]); num[2] = fmaf(f, o[u].z, num[2]); num[3] = fmaf(f, o[u].w, num[3]);
                    }
            }
            const int pr = t.first + r0 + r, tok = pr / A.c.group, qh = head * A.c.group + pr % A.c.group;
            float* o = A.out + (t.row0 + tok) * A.out_ld + (long long)qh * hs + d;
            for (int e = 0; e < w; e++) o[e] = num[e] / den;
        }
    }
    __syncthreads();
}
#endif

}  // namespace paged

bool paged_attention_few(int kv_dtype, int hs);
paged::Lane paged_attention_lane(int kv_dtype, int hs, int sms);
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
