// Causal attention of a step's new tokens to the keys and values that their sequences hold in pages: out = softmax(q K^T scale) V, each token over the
// positions up to its own, a cache head shared by `group` query heads.  (The reference's operator has one token and one dense cache:
// crates/slai/src/ops/batched_multiquery_attention.rs:32-156.)  Who computes what: paged_plan.h.
#include "paged_rows.cuh"

using namespace paged;

namespace {

// ---- any head size, either cache type, any alignment ---------------------------------------------------------------------
// 16 rows at a time, positions in tiles of 32 brought into shared memory as f32; warp w has rows 4w .. 4w + 3; scores: lane = position, sums of values:
// lane = dimensions.  Plain f32 arithmetic, one pass with the running maximum and sum of each row.
constexpr int GT = 128, GR = 16, GP = 32;

template <typename T>
__device__ __forceinline__ void load_rows(const T* base, const long long* place, int rows, int hs, int hsp, bool vec, float* s, int stride, int tid) {
    constexpr int VEC = 16 / (int)sizeof(T);
    if (vec) {
        const int ppr = hs / VEC;
        for (int i = tid; i < GP * ppr; i += GT) {
            const int r = i / ppr, c = i - r * ppr;
            float v[VEC];
            if (r < rows) {
                const uint4 raw = __ldcg(reinterpret_cast<const uint4*>(base + place[r]) + c);
                const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
                for (int j = 0; j < VEC; j++) v[j] = to_float<T>(e[j]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j++) v[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < VEC; j += 4) *reinterpret_cast<float4*>(s + r * stride + c * VEC + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
    } else {
        for (int i = tid; i < GP * hsp; i += GT) {
            const int r = i / hsp, d = i - r * hsp;
            s[r * stride + d] = r < rows && d < hs ? to_float<T>(base[place[r] + d]) : 0.f;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(GT) paged_attn_any_kernel(const __grid_constant__ AttnArgs A) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Cache& c = A.c;
    const Start s = load_start(c.plan, A.starts_at, blockIdx.x);
    const int hs = c.hs, hsp = (hs + 3) & ~3, ks = hsp + 4;
    extern __shared__ __align__(16) float sm[];
    float* q_s = sm;                // [16][hsp], times the scale
    float* k_s = q_s + GR * hsp;    // [32][hsp + 4]
    float* v_s = k_s + GP * ks;     // [32][hsp]
    float* p_s = v_s + GP * hsp;    // [16][32]
    __shared__ long long place[GP];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    Tile t = s.t;
    int head = s.head, unit = s.unit, tile = s.tile;
    for (int left = s.count; left > 0;) {
        const int n = min(left, t.units - unit);
        const bool whole = n == t.units;
        const size_t slot = ((size_t)s.me * 2 + (unit == 0)) * A.tile_rows;
        for (int g0 = 0; g0 < t.rows; g0 += GR) {
            const int nr = min(GR, t.rows - g0);
            int vis[4];  // last position that this warp's rows see
#pragma unroll
            for (int i = 0; i < 4; i++) vis[i] = 4 * warp + i < nr ? t.pos0 + (t.first + g0 + 4 * warp + i) / c.group : -1;
            const int last = min(t.pos0 + (t.first + g0 + nr - 1) / c.group, (unit + n) * A.unit - 1);
            const int warp_last = max(max(vis[0], vis[1]), max(vis[2], vis[3]));
            __syncthreads();
            for (int i = tid; i < GR * hsp; i += GT) {
                const int r = i / hsp, d = i - r * hsp, pr = t.first + g0 + r, tok = pr / c.group;
                q_s[i] = r < nr && d < hs ? __ldcg(A.q + (t.row0 + tok) * A.q_ld + (long long)(head * c.group + pr % c.group) * hs + d) * A.scale : 0.f;
            }
            float m[4], l[4], acc[4][2][4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                m[i] = -INFINITY;
                l[i] = 0.f;
#pragma unroll
                for (int k = 0; k < 2; k++) acc[i][k][0] = acc[i][k][1] = acc[i][k][2] = acc[i][k][3] = 0.f;
            }
            for (int p0 = unit * A.unit; p0 <= last; p0 += GP) {
                const int cnt = min(GP, last + 1 - p0);
                __syncthreads();  // the tile before has been read
                if (tid < cnt) place[tid] = place_of(c, t.table, p0 + tid, head);
                __syncthreads();
                load_rows<T>(reinterpret_cast<const T*>(c.keys), place, cnt, hs, hsp, A.vec, k_s, ks, tid);
                load_rows<T>(reinterpret_cast<const T*>(c.values), place, cnt, hs, hsp, A.vec, v_s, hsp, tid);
                __syncthreads();
                if (p0 > warp_last) continue;
                float sc[4] = {};
                const float* kr = k_s + lane * ks;
                const float* qr = q_s + 4 * warp * hsp;
                for (int d = 0; d < hsp; d += 4) {
                    const float4 kv = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float4 qv = *reinterpret_cast<const float4*>(qr + i * hsp + d);
                        sc[i] = fmaf(kv.x, qv.x, fmaf(kv.y, qv.y, fmaf(kv.z, qv.z, fmaf(kv.w, qv.w, sc[i]))));
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool seen = lane < cnt && p0 + lane <= vis[i];
                    float mt = seen ? sc[i] : -INFINITY;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
                    const float m_new = fmaxf(m[i], mt);
                    const float p = !seen || sc[i] == -INFINITY ? 0.f : expf(sc[i] - m_new);
                    float ps = p;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
                    const float resc = m[i] == -INFINITY ? 1.f : expf(m[i] - m_new);  // (nothing but zeros so far, or a NaN, which stays)
                    l[i] = l[i] * resc + ps;
                    m[i] = m_new;
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        acc[i][k][0] *= resc; acc[i][k][1] *= resc; acc[i][k][2] *= resc; acc[i][k][3] *= resc;
                    }
                    p_s[(4 * warp + i) * GP + lane] = p;
                }
                __syncwarp();
                for (int j = 0; j < cnt; j++) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const int d = 128 * k + 4 * lane;
                        if (d < hsp) {
                            const float4 vv = *reinterpret_cast<const float4*>(v_s + j * hsp + d);
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if (p0 + j <= vis[i]) {  // what a row does not see is not multiplied: it may be infinite
                                    const float p = p_s[(4 * warp + i) * GP + j];
                                    acc[i][k][0] = fmaf(p, vv.x, acc[i][k][0]);
                                    acc[i][k][1] = fmaf(p, vv.y, acc[i][k][1]);
                                    acc[i][k][2] = fmaf(p, vv.z, acc[i][k][2]);
                                    acc[i][k][3] = fmaf(p, vv.w, acc[i][k][3]);
                                }
                        }
                    }
                }
                __syncwarp();
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = 4 * warp + i;
                if (r >= nr) continue;
                const int pr = t.first + g0 + r, tok = pr / c.group;
                float* o = whole ? A.out + (t.row0 + tok) * A.out_ld + (long long)(head * c.group + pr % c.group) * hs : A.part + (slot + g0 + r) * hs;
                const float f = whole ? 1.f / l[i] : 1.f;
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int d = 128 * k + 4 * lane + e;
                        if (d < hs) o[d] = acc[i][k][e] * f;
                    }
                if (!whole && lane == 0) *reinterpret_cast<float2*>(A.part_ml + (slot + g0 + r) * 2) = make_float2(m[i] * LOG2E, l[i]);
            }
        }
        left -= n + PAIR_COST;
        unit = 0;
        if (left > 0 && ++head == c.n_kv) {
            head = 0;
            t = load_tile(c.plan, s.tiles, ++tile);
        }
    }
}

template <typename T>
int launch_any(slai_ctx* ctx, const AttnArgs& A, int blocks, bool pdl) {
    auto kern = paged_attn_any_kernel<T>;
    const int hsp = (A.c.hs + 3) & ~3;
    const size_t smem = sizeof(float) * (size_t)(GR * hsp + GP * (hsp + 4) + GP * hsp + GR * GP);
    static PerDeviceOnce attr;
    if (attr.need(ctx->device)) {
        SLAI_CHECK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024));
        attr.set(ctx->device);
    }
    return launch_dependent(ctx, kern, dim3((unsigned)blocks), GT, smem, pdl, A);
}

// ---- pairs that lie on several blocks ------------------------------------------------------------------------------------------
// Rows of a tile: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the blocks' results in the order of their positions (a block that saw nothing of a row
// has m = -inf, l = 0, o = 0).  A launch of its own behind the other's end, whose blocks read all results at once: done by the block that comes last, a
// token over 32750 positions (37 blocks a pair) took 12 us from its loop's end to the result, and over 515 positions 5.
__device__ __forceinline__ float join_weight(float m, float M) { return m == -INFINITY ? 0.f : exp2f(m - M); }
struct JoinOf {  // one pair
    int row0, first, rows, head, begin, nb;
};
__device__ __forceinline__ JoinOf load_join(const AttnArgs& A, int i) {
    const int4* g = reinterpret_cast<const int4*>(A.c.plan + A.joins_at) + 2 * i;
    const int4 a = __ldcg(g), b = __ldcg(g + 1);
    return {a.x, a.y, a.z, a.w, b.x, b.y - b.x + 1};
}
__device__ __forceinline__ size_t part_slot(const AttnArgs& A, const JoinOf& j, int i, int r) { return ((size_t)(j.begin + i) * 2 + (i == 0)) * A.tile_rows + r; }
__device__ __forceinline__ float* join_out(const AttnArgs& A, const JoinOf& j, int r) {
    const int pr = j.first + r, tok = pr / A.c.group;
    return A.out + (j.row0 + tok) * A.out_ld + (long long)(j.head * A.c.group + pr % A.c.group) * A.c.hs;
}
// elements d .. d + 3 of a result where heads are whole quads, else d
__device__ __forceinline__ float4 join_load(const AttnArgs& A, size_t slot, int d, bool quads) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d >= A.c.hs) return o;
    if (quads) return __ldcg(reinterpret_cast<const float4*>(A.part + slot * A.c.hs + d));
    o.x = __ldcg(A.part + slot * A.c.hs + d);
    return o;
}
__device__ __forceinline__ void join_add(float4& a, float f, float4 o) {
    a.x = fmaf(f, o.x, a.x); a.y = fmaf(f, o.y, a.y); a.z = fmaf(f, o.z, a.z); a.w = fmaf(f, o.w, a.w);
}

// A few results to a pair: a warp takes four rows; eight lanes of it have a row's weights.
constexpr int JT = 64, JR = 4, JROWS = JT / 32 * JR;
// Rows r0 .. r0 + JR - 1 of a pair, by one warp.
__device__ __forceinline__ void join_rows(const AttnArgs& A, const JoinOf& j, int r0, int lane) {
    const int n = min(JR, j.rows - r0), hs = A.c.hs;
    if (n <= 0) return;
    const float2* ml = reinterpret_cast<const float2*>(A.part_ml);
    const int mine = min(lane >> 3, n - 1), b8 = lane & 7;
    const bool quads = hs % 4 == 0;
    for (int d0 = 0; d0 < hs; d0 += quads ? 128 : 32) {
        const int d = d0 + (quads ? 4 * lane : lane);
        float4 num[JR];
#pragma unroll
        for (int r = 0; r < JR; r++) num[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f, M = -INFINITY;
        for (int c0 = 0; c0 < j.nb; c0 += 8) {  // eight results at a time, with a running maximum; loads first, all at once
            const float2 y = c0 + b8 < j.nb ? __ldcg(ml + part_slot(A, j, c0 + b8, r0 + mine)) : make_float2(-INFINITY, 0.f);
            const int m = min(8, j.nb - c0);
            float4 o[2][JR];
            auto load = [&](int u) {
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int r = 0; r < JR; r++) o[k][r] = join_load(A, part_slot(A, j, c0 + min(u + k, m - 1), r0 + min(r, n - 1)), d, quads);
            };
            load(0);
            float Mn = y.x;
#pragma unroll
            for (int i = 4; i > 0; i >>= 1) Mn = fmaxf(Mn, __shfl_xor_sync(0xffffffffu, Mn, i));
            Mn = fmaxf(M, Mn);
            const float f = join_weight(y.x, Mn), resc = join_weight(M, Mn);
            M = Mn;
            den = fmaf(den, resc, f * y.y);
            if (c0 > 0) {
#pragma unroll
                for (int r = 0; r < JR; r++) {
                    const float by = __shfl_sync(0xffffffffu, resc, 8 * r);
                    num[r].x *= by; num[r].y *= by; num[r].z *= by; num[r].w *= by;
                }
            }
            for (int u = 0; u < m; u += 2) {
                if (u > 0) load(u);
#pragma unroll
                for (int k = 0; k < 2; k++)
                    if (u + k < m) {
#pragma unroll
                        for (int r = 0; r < JR; r++) join_add(num[r], __shfl_sync(0xffffffffu, f, 8 * r + u + k), o[k][r]);
                    }
            }
        }
#pragma unroll
        for (int i = 4; i > 0; i >>= 1) den += __shfl_xor_sync(0xffffffffu, den, i);
#pragma unroll
        for (int r = 0; r < JR; r++) {
            const float by = 1.f / __shfl_sync(0xffffffffu, den, 8 * r);
            if (r < n && d < hs) {
                float* o = join_out(A, j, r0 + r) + d;
                if (quads && A.qvec) {
                    *reinterpret_cast<float4*>(o) = make_float4(num[r].x * by, num[r].y * by, num[r].z * by, num[r].w * by);
                } else {
                    const float v[4] = {num[r].x, num[r].y, num[r].z, num[r].w};
                    for (int e = 0; e < (quads ? 4 : 1); e++) o[e] = v[e] * by;
                }
            }
        }
    }
}
// MORE: there may be more pairs than blocks for them.
template <bool MORE>
__global__ void __launch_bounds__(JT) paged_join_kernel(const __grid_constant__ AttnArgs A) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int joins = __ldcg(A.c.plan + A.count_at);
    JoinOf j = load_join(A, blockIdx.x);  // (there is room for it, whether it is one or not)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int r0 = (int)blockIdx.y * JROWS + warp * JR;
    if ((int)blockIdx.x < joins) join_rows(A, j, r0, lane);
    if (MORE)
        for (int i = blockIdx.x + gridDim.x; i < joins; i += gridDim.x) join_rows(A, load_join(A, i), r0, lane);
}

// Many results to a pair (one long sequence over many blocks): a block takes a row, its warps every LW-th result.
constexpr int LT = 128, LW = LT / 32, JOIN_MANY = 8;
// Row r of a pair, by the block.
__device__ __forceinline__ void join_row(const AttnArgs& A, const JoinOf& j, int r, float (&num_s)[LW][256], float (&den_s)[LW]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hs = A.c.hs;
    const float2* ml = reinterpret_cast<const float2*>(A.part_ml);
    float M = -INFINITY;
    for (int b = lane; b < j.nb; b += 32) M = fmaxf(M, __ldcg(ml + part_slot(A, j, b, r)).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const bool quads = hs % 4 == 0;
    for (int d0 = 0; d0 < hs; d0 += quads ? 128 : 32) {
        const int d = d0 + (quads ? 4 * lane : lane);
        float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
        for (int b0 = warp; b0 < j.nb; b0 += 8 * LW) {
            float4 o[8];
            float2 y[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int b = b0 + u * LW;
                y[u] = b < j.nb ? __ldcg(ml + part_slot(A, j, b, r)) : make_float2(-INFINITY, 0.f);
                o[u] = join_load(A, part_slot(A, j, min(b, j.nb - 1), r), b < j.nb ? d : hs, quads);
            }
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const float f = join_weight(y[u].x, M);
                den = fmaf(f, y[u].y, den);
                join_add(num, f, o[u]);
            }
        }
        const float v[4] = {num.x, num.y, num.z, num.w};
        for (int e = 0; e < (quads ? 4 : 1) && d < hs; e++) num_s[warp][d + e] = v[e];
        if (lane == 0) den_s[warp] = den;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < hs; d += LT) {
        float n = 0.f, den = 0.f;
#pragma unroll
        for (int w = 0; w < LW; w++) {
            n += num_s[w][d];
            den += den_s[w];
        }
        join_out(A, j, r)[d] = n / den;
    }
}
// MORE: there may be more pairs than blocks for them.
template <bool MORE>
__global__ void __launch_bounds__(LT) paged_join_many_kernel(const __grid_constant__ AttnArgs A) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int r = (int)blockIdx.y;
    const int joins = __ldcg(A.c.plan + A.count_at);
    JoinOf j = load_join(A, blockIdx.x);  // (there is room for it, whether it is one or not)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float num_s[LW][256];
    __shared__ float den_s[LW];
    if ((int)blockIdx.x < joins && r < j.rows) join_row(A, j, r, num_s, den_s);
    if (MORE)
        for (int i = blockIdx.x + gridDim.x; i < joins; i += gridDim.x) {
            j = load_join(A, i);
            __syncthreads();  // the sums before have been read
            if (r < j.rows) join_row(A, j, r, num_s, den_s);
        }
}

// `longest`: most results of a pair.  us of the call, a warp for four rows / a block for each: 272 pairs of 2 or 3 results of 8 rows 98.8 / 102; 8 pairs of 37 results
// 38.8 / 32.5; 141 pairs of 2 or 3 of 256 rows 475 / 494.
template <bool MORE>
int launch_join(slai_ctx* ctx, const AttnArgs& A, int joins, int longest, bool pdl) {
    if (joins <= 0) return SLAI_OK;
    if (longest > JOIN_MANY && A.tile_rows <= 16) return launch_dependent(ctx, paged_join_many_kernel<MORE>, dim3((unsigned)joins, (unsigned)A.tile_rows), LT, 0, pdl, A);
    return launch_dependent(ctx, paged_join_kernel<MORE>, dim3((unsigned)joins, (unsigned)((A.tile_rows + JROWS - 1) / JROWS)), JT, 0, pdl, A);
}

// ---- PTX wrappers --------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// ---- few rows: the end of a block's part of a pair ------------------------------------------------------------------------------
// Each of the block's FW warps has a maximum, a sum and an output of every row for its own positions: `so` [warp][rows][HS] (WF floats apart), ml_s; outputs and sums are
// `carried` times their size apart.  They become the result, or the block's slot of `part`.
constexpr int FW = 4, FT = 32 * FW, FS = 3, FB = 2, FR = 8;  // warps, threads, stages of a warp, blocks an SM, rows
template <int HS, typename T>
__device__ __forceinline__ void few_end(const AttnArgs& A, const Start& s, const Tile& t, int head, int unit, bool whole, int lo, int hi, const float* so, int WF,
                                        const float2 (*ml_s)[FR], unsigned int& bad, float carried) {
    const Cache& c = A.c;
    const int tid = threadIdx.x, warp = tid >> 5, hs = c.hs;
    if (tid == 0) bad = 0;
    __syncthreads();
    const size_t slot = ((size_t)s.me * 2 + (unit == 0)) * A.tile_rows;
    for (int i = tid; i < t.rows * (hs / 4); i += FT) {
        const int r = i / (hs / 4), d = 4 * (i - r * (hs / 4));
        float M = -INFINITY, den = 0.f, num[4] = {};
#pragma unroll
        for (int w = 0; w < FW; w++) M = fmaxf(M, ml_s[w][r].x);
#pragma unroll
        for (int w = 0; w < FW; w++) {
            const float2 x = ml_s[w][r];
            const float f = x.x == -INFINITY ? 0.f : ex2(x.x - M);
            const float4 o = *reinterpret_cast<const float4*>(so + w * WF + r * HS + d);
            den = fmaf(f, x.y, den);
            num[0] = fmaf(f, o.x, num[0]); num[1] = fmaf(f, o.y, num[1]); num[2] = fmaf(f, o.z, num[2]); num[3] = fmaf(f, o.w, num[3]);
        }
        if (!(fabsf(num[0] + num[1] + num[2] + num[3] + den) < INFINITY)) atomicOr(&bad, 1u << r);
        const float f = whole ? carried / den : carried;
        const int pr = t.first + r, tok = pr / c.group;
        float* o = whole ? A.out + (t.row0 + tok) * A.out_ld + (long long)(head * c.group + pr % c.group) * hs + d : A.part + (slot + r) * hs + d;
        if (!whole || A.qvec) {
            *reinterpret_cast<float4*>(o) = make_float4(num[0] * f, num[1] * f, num[2] * f, num[3] * f);
        } else {
            for (int e = 0; e < 4; e++) o[e] = num[e] * f;
        }
        if (!whole && d == 0) *reinterpret_cast<float2*>(A.part_ml + (slot + r) * 2) = make_float2(M, den);
    }
    __syncthreads();
    if (bad) {
        for (int r = warp; r < t.rows; r += FW)
            if (bad >> r & 1) {
                const int pr = t.first + r, tok = pr / c.group;
                float* o = whole ? A.out + (t.row0 + tok) * A.out_ld + (long long)(head * c.group + pr % c.group) * hs : A.part + (slot + r) * hs;
                row_again<T>(A, t, head, r, lo, hi, o, whole ? nullptr : A.part_ml + (slot + r) * 2);
            }
        __syncthreads();
    }
}

// ---- f16 caches, few rows: tokens of sequences that answer ---------------------------------------------------------------------
// Up to 8 rows (a token's or a few tokens' query heads of one cache head).  Queries and weights are pairs of halves (22 bits); the 16 rows of the matrix
// instruction are the 8 high parts and, below them, the 8 low ones, so one product does both and a lane holds both results of its row.  Sums end every 16
// positions (the matrix unit truncates when it adds) and go on in registers.
// What such a call costs is reading the cache: each of the block's warps has a ring of its own of stages of 16 positions, brought in by asynchronous
// copies that go around the registers, and takes every FW-th 16 positions of the block's share with a running maximum and sum of its own; they are joined in shared
// memory at the end.  A token of each of 64 sequences of 100 to 3900 positions, 64 heads on 8: 529 MB in 96 to 100 us, 82 to 85 % of the copy rate; a token at 32750: 134 MB in
// 33 us, 27 of them this kernel's (24 us of loop, of which the first positions' way takes 6), the rest the join's.  us of the two by warps, stages, blocks an
// SM: 4, 3, 2 102, 33; 4, 2, 3 97, 42; 6, 2, 2 103, 46; 8, 3, 1 119, 31.  (16 rows to an instruction, high and low parts one after the other: 161, 53.)
constexpr int FP = 16;
template <int HS>
constexpr int FEW_SMEM = FW * FS * 2 * FP * HS * 2;

// ALIGNED: pages hold a multiple of 16 positions, so 16 of them have one page.
template <int HS, bool ALIGNED>
__global__ void __launch_bounds__(FT, FB) paged_attn_few_kernel(const __grid_constant__ AttnArgs A) {
    constexpr int ROW = HS * 2, CH = HS / 8, TILE = FP * ROW, STAGE = 2 * TILE, KS = HS / 16, NT8 = HS / 8;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(128) unsigned char few_sm[];
    __shared__ float2 ml_s[FW][FR];
    __shared__ unsigned int bad;
    const Cache& c = A.c;
    const Start s = load_start(c.plan, A.starts_at, blockIdx.x);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3, hs = c.hs, chunks = hs / 8;
    const uint32_t sm = (uint32_t)__cvta_generic_to_shared(few_sm), ring = sm + warp * FS * STAGE;
    const char *keys = c.keys, *values = c.values;

    bool behind = false;
    if (s.count <= 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    Tile t = s.t;
    int head = s.head, unit = s.unit, tile = s.tile;
    for (int left = s.count; left > 0;) {
        const int n = min(left, t.units - unit);
        const bool whole = n == t.units;
        const int lo = unit * A.unit, hi = min((unit + n) * A.unit, t.pos0 + (t.first + t.rows - 1) / c.group + 1);  // positions [lo, hi)
        const int subs = (hi - lo + FP - 1) / FP, mine = subs > warp ? (subs - warp + FW - 1) / FW : 0;
        // Where this warp's i-th 16 positions are, in bytes: of the first of them (ALIGNED), or of position (lane & 15).
        auto place = [&](int i) -> long long {
            const int p = lo + (warp + i * FW) * FP + (ALIGNED ? 0 : lane & 15);
            return i < mine && p < hi ? 2 * place_of(c, t.table, p, head) : 0;
        };
        auto request = [&](int i, long long at) {
            if (i < mine) {
                const uint32_t dst = ring + (i % FS) * STAGE;
                const int valid = hi - (lo + (warp + i * FW) * FP), ch = lane % CH, r0 = lane / CH;
                constexpr int STEP = 32 / CH;  // rows a pass of the warp covers
                const char *k0 = keys + at + 16 * ch, *v0 = values + at + 16 * ch;
#pragma unroll
                for (int k = 0; k < FP / STEP; k++) {
                    const int r = r0 + STEP * k;
                    const uint32_t off = r * ROW + ((ch ^ (r & 7)) << 4), bytes = r < valid && ch < chunks ? 16u : 0u;  // (none: zeros, nothing is read)
                    long long a = r * 2 * c.pos_stride;
                    if (!ALIGNED) a = __shfl_sync(0xffffffffu, at, r) - at;
                    if (bytes == 0) a = -at - 16 * ch;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + off), "l"(__cvta_generic_to_global(k0 + a)), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + TILE + off), "l"(__cvta_generic_to_global(v0 + a)), "r"(bytes) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        {
            long long at[FS - 1];
#pragma unroll
            for (int i = 0; i < FS - 1; i++) at[i] = place(i);
            // The plan is there before any kernel of its step starts (it comes by a copy, which no launch overtakes); all else is the kernel before's.
            if (!behind) asm volatile("griddepcontrol.wait;" ::: "memory");
            behind = true;
#pragma unroll
            for (int i = 0; i < FS - 1; i++) request(i, at[i]);
        }
        long long next = place(FS - 1);

        // queries of row g: high parts in the instruction's row g, low ones in row g + 8
        uint32_t qf[KS][4];
        float cexp;  // the row's scores to powers of two
        const int pr_g = t.first + g, tok_g = pr_g / c.group, vis = g < t.rows ? t.pos0 + tok_g : -1;  // last position the row sees
        {
            float2 v[KS][2];
            float mx = 0.f;
            const float* qr = A.q + (g < t.rows ? (t.row0 + tok_g) * A.q_ld + (long long)(head * c.group + pr_g % c.group) * hs : 0);
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int d = 16 * k + 2 * t4 + 8 * i;
                    v[k][i] = make_float2(0.f, 0.f);
                    if (vis >= 0 && d < hs) {
                        if (A.qvec) v[k][i] = __ldcg(reinterpret_cast<const float2*>(qr + d));
                        else v[k][i] = make_float2(__ldcg(qr + d), __ldcg(qr + d + 1));
                    }
                    v[k][i].x *= A.scale;
                    v[k][i].y *= A.scale;
                    mx = fmaxf(mx, fmaxf(fabsf(v[k][i].x), fabsf(v[k][i].y)));
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float up = power_up(mx, cexp);
            cexp *= LOG2E;
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int i = 0; i < 2; i++) split2(v[k][i].x * up, v[k][i].y * up, qf[k][2 * i], qf[k][2 * i + 1]);
        }
        float acc[NT8][2];
#pragma unroll
        for (int i = 0; i < NT8; i++) acc[i][0] = acc[i][1] = 0.f;
        float m = -INFINITY, l = 0.f;  // m: largest score so far, as a power of two's exponent

        for (int i = 0; i < mine; i++) {
            request(i + FS - 1, next);
            next = place(i + FS);
            asm volatile("cp.async.wait_group %0;" ::"n"(FS - 1) : "memory");
            __syncwarp();
            const uint32_t ks = ring + (i % FS) * STAGE, vs = ks + TILE;
            const int p0 = lo + (warp + i * FW) * FP;
            float sc[4];
#pragma unroll
            for (int nn = 0; nn < 2; nn++) {
                float c0[4] = {}, c1[4] = {};
                uint32_t b[KS / 2][4];
                const int r = 8 * nn + (lane & 7);
#pragma unroll
                for (int k2 = 0; k2 < KS / 2; k2++) ldsm4(ks + r * ROW + (((4 * k2 + (lane >> 3)) ^ (r & 7)) << 4), b[k2]);
#pragma unroll
                for (int k = 0; k < KS; k++) mma_f16((k & 1) ? c1 : c0, qf[k], b[k >> 1][2 * (k & 1)], b[k >> 1][2 * (k & 1) + 1]);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float x = ((c0[e] + c1[e]) + (c0[e + 2] + c1[e + 2])) * cexp;
                    sc[2 * nn + e] = p0 + 8 * nn + 2 * t4 + e > vis ? -INFINITY : x;
                }
            }
            float mt = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
            const float m_new = fmaxf(m, mt), base = m_new == -INFINITY ? 0.f : m_new, resc = ex2(m - base);
            m = m_new;
            float ps = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float p = ex2(sc[e] - base);
                ps += p;
                sc[e] = p * 4096.f;
            }
            l = l * resc + ps;  // (this lane's positions only)
            uint32_t pf[4];
            split2(sc[0], sc[1], pf[0], pf[1]);
            split2(sc[2], sc[3], pf[2], pf[3]);
#pragma unroll
            for (int n2 = 0; n2 < NT8 / 2; n2++) {
                float d0[4] = {}, d1[4] = {};
                uint32_t b[4];
                const int r = lane & 15;
                ldsm4t(vs + r * ROW + (((2 * n2 + (lane >> 4)) ^ (r & 7)) << 4), b);
                mma_f16(d0, pf, b[0], b[1]);
                mma_f16(d1, pf, b[2], b[3]);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    acc[2 * n2][e] = fmaf(acc[2 * n2][e], resc, d0[e] + d0[e + 2]);
                    acc[2 * n2 + 1][e] = fmaf(acc[2 * n2 + 1][e], resc, d1[e] + d1[e + 2]);
                }
            }
            __syncwarp();  // the stage is requested again next round
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t4 == 0) ml_s[warp][g] = make_float2(m, l);
        // the warps' sums meet where the stages were (each in its own ring)
        float* so = reinterpret_cast<float*>(few_sm);
        constexpr int WF = FS * STAGE / 4;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NT8; i++) *reinterpret_cast<float2*>(so + warp * WF + g * HS + 8 * i + 2 * t4) = make_float2(acc[i][0], acc[i][1]);
        few_end<HS, __half>(A, s, t, head, unit, whole, lo, hi, so, WF, ml_s, bad, 1.f / 4096.f);
        left -= n + PAIR_COST;
        unit = 0;
        if (left > 0 && ++head == c.n_kv) {
            head = 0;
            t = load_tile(c.plan, s.tiles, ++tile);
        }
    }
}

template <int HS, bool ALIGNED>
int launch_few(slai_ctx* ctx, const AttnArgs& A, int blocks, bool pdl) {
    auto kern = paged_attn_few_kernel<HS, ALIGNED>;
    static PerDeviceOnce attr;
    if (attr.need(ctx->device)) {
        SLAI_CHECK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM<HS>));
        attr.set(ctx->device);
    }
    return launch_dependent(ctx, kern, dim3((unsigned)blocks), FT, FEW_SMEM<HS>, pdl, A);
}

// ---- f32 caches, few rows ----------------------------------------------------------------------------------------------------------
// The same with f32 arithmetic: stages of 8 positions; four lanes take a position's score (a quarter of the dimensions each, the queries from shared memory), a lane
// four dimensions of the output.  R: rows that there is room for (1, 4 or 8; 1 where a cache head has one query head: 69 -> 55 us for the following).  Reading the
// cache bounds it: a token of each of 8 sequences of 515 to 1546 positions, 32 heads, pages of 20: 271 MB in 55 us, 76 % of the copy rate.
constexpr int EP = 8;
template <int HS, int R>
constexpr int FEW32_SMEM = FW * FS * 2 * EP * HS * 4 + R * HS * 4 + FW * EP * R * 4;

template <int HS, int R, bool ALIGNED>
__global__ void __launch_bounds__(FT, FB) paged_attn_few32_kernel(const __grid_constant__ AttnArgs A) {
    constexpr int ROW = HS * 4, CH = HS / 4, TILE = EP * ROW, STAGE = 2 * TILE, STEP = 32 / CH;  // STEP: rows a pass of the warp covers
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(128) unsigned char few_sm[];
    float* q_s = reinterpret_cast<float*>(few_sm + FW * FS * STAGE);  // [R][HS]
    __shared__ float2 ml_s[FW][FR];
    __shared__ unsigned int bad;
    const Cache& c = A.c;
    const Start s = load_start(c.plan, A.starts_at, blockIdx.x);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, p8 = lane >> 2, c4 = lane & 3, hs = c.hs, chunks = hs / 4, ch = lane % CH, rl = lane / CH;
    float* p_s = q_s + R * HS + warp * EP * R;                         // [8][R], this warp's
    unsigned char* ring = few_sm + warp * FS * STAGE;
    const uint32_t ring_a = (uint32_t)__cvta_generic_to_shared(ring);
    const char *keys = c.keys, *values = c.values;
    // a piece's place in its row: rows of odd positions lie the other way round, so that two rows' pieces share no bank
    auto piece = [](int r, int i) { return 4 * (i ^ ((r & 1) << 2)); };

    asm volatile("griddepcontrol.wait;" ::: "memory");
    Tile t = s.t;
    int head = s.head, unit = s.unit, tile = s.tile;
    for (int left = s.count; left > 0;) {
        const int n = min(left, t.units - unit);
        const bool whole = n == t.units;
        const int lo = unit * A.unit, hi = min((unit + n) * A.unit, t.pos0 + (t.first + t.rows - 1) / c.group + 1);  // positions [lo, hi)
        const int subs = (hi - lo + EP - 1) / EP, mine = subs > warp ? (subs - warp + FW - 1) / FW : 0;
        auto place = [&](int i) -> long long {
            const int p = lo + (warp + i * FW) * EP + (ALIGNED ? 0 : lane & 7);
            return i < mine && p < hi ? 4 * place_of(c, t.table, p, head) : 0;
        };
        auto request = [&](int i, long long at) {
            if (i < mine) {
                const uint32_t dst = ring_a + (i % FS) * STAGE;
                const int valid = hi - (lo + (warp + i * FW) * EP);
#pragma unroll
                for (int k = 0; k < EP / STEP; k++) {
                    const int r = rl + STEP * k;
                    const uint32_t off = r * ROW + 4 * piece(r, ch), bytes = r < valid && ch < chunks ? 16u : 0u;  // (none: zeros, nothing is read)
                    const long long a = ALIGNED ? at + r * 4 * c.pos_stride : __shfl_sync(0xffffffffu, at, r);
                    const long long src = bytes ? a + 16 * ch : 0;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + off), "l"(__cvta_generic_to_global(keys + src)), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + TILE + off), "l"(__cvta_generic_to_global(values + src)), "r"(bytes) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        {
            long long at[FS - 1];
#pragma unroll
            for (int i = 0; i < FS - 1; i++) at[i] = place(i);
#pragma unroll
            for (int i = 0; i < FS - 1; i++) request(i, at[i]);
        }
        long long next = place(FS - 1);
        const float by = A.scale * LOG2E;  // scores as powers of two's exponents
#pragma unroll
        for (int k = 0; k < (R * HS + FT - 1) / FT; k++) {
            const int i = tid + k * FT;
            if (i >= R * HS) break;
            const int r = i / HS, d = i % HS, pr = t.first + r, tok = pr / c.group;
            q_s[i] = r < t.rows && d < hs ? __ldcg(A.q + (t.row0 + tok) * A.q_ld + (long long)(head * c.group + pr % c.group) * hs + d) * by : 0.f;
        }
        int vis[R];  // last position a row sees
#pragma unroll
        for (int r = 0; r < R; r++) vis[r] = r < t.rows ? t.pos0 + (t.first + r) / c.group : -1;
        __syncthreads();
        f32x2 acc[R][2];
        float m[R], l[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            acc[r][0] = acc[r][1] = 0;
            m[r] = -INFINITY;
            l[r] = 0.f;
        }
        for (int i = 0; i < mine; i++) {
            request(i + FS - 1, next);
            next = place(i + FS);
            asm volatile("cp.async.wait_group %0;" ::"n"(FS - 1) : "memory");
            __syncwarp();
            const float* ks = reinterpret_cast<const float*>(ring + (i % FS) * STAGE);
            const float* vs = ks + TILE / 4;
            const int p = lo + (warp + i * FW) * EP + p8;
            f32x2 sc[R][2];
#pragma unroll
            for (int r = 0; r < R; r++) sc[r][0] = sc[r][1] = 0;
#pragma unroll
            for (int j = 0; j < HS / 16; j++) {
                const ulonglong2 k2 = *reinterpret_cast<const ulonglong2*>(ks + p8 * HS + piece(p8, 4 * j + c4));
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const ulonglong2 q2 = *reinterpret_cast<const ulonglong2*>(q_s + r * HS + 4 * (4 * j + c4));
                    sc[r][0] = fma2(k2.x, q2.x, sc[r][0]);
                    sc[r][1] = fma2(k2.y, q2.y, sc[r][1]);
                }
            }
            float w[R];
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float2 a = unpack2(sc[r][0]), b = unpack2(sc[r][1]);
                float x = (a.x + a.y) + (b.x + b.y);
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                w[r] = p > vis[r] ? -INFINITY : x;
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                float mt = w[r];
                mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 4));
                mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 8));
                mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 16));
                const float m_new = fmaxf(m[r], mt), base = m_new == -INFINITY ? 0.f : m_new, resc = ex2(m[r] - base);
                m[r] = m_new;
                w[r] = ex2(w[r] - base);
                l[r] = l[r] * resc + w[r];  // (this lane's positions only)
                const f32x2 f = pack2(resc, resc);
                acc[r][0] = mul2(acc[r][0], f);
                acc[r][1] = mul2(acc[r][1], f);
            }
#pragma unroll
            for (int r0 = 0; r0 < R; r0 += 4) {  // of the four lanes of a position, each writes one row of four
                const float x = R == 1 || c4 == 0 ? w[r0] : c4 == 1 ? w[(r0 + 1) % R] : c4 == 2 ? w[(r0 + 2) % R] : w[(r0 + 3) % R];
                if (r0 + c4 < R) p_s[p8 * R + r0 + c4] = x;
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < EP; k += STEP) {
                const int pos = k + rl;
                const ulonglong2 v2 = *reinterpret_cast<const ulonglong2*>(vs + pos * HS + piece(pos, ch));
#pragma unroll
                for (int r0 = 0; r0 < R; r0 += 4) {
                    float xs[4];
                    if (R == 1) xs[0] = p_s[pos];
                    else *reinterpret_cast<float4*>(xs) = *reinterpret_cast<const float4*>(p_s + pos * R + r0);
#pragma unroll
                    for (int r = 0; r < (R < 4 ? R : 4); r++) {
                        const f32x2 f = pack2(xs[r], xs[r]);
                        acc[r0 + r][0] = fma2(f, v2.x, acc[r0 + r][0]);
                        acc[r0 + r][1] = fma2(f, v2.y, acc[r0 + r][1]);
                    }
                }
            }
            __syncwarp();  // the stage is requested, the weights written again next round
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        float* so = reinterpret_cast<float*>(few_sm);
        constexpr int WF = FS * STAGE / 4;
#pragma unroll
        for (int r = 0; r < R; r++) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
            const float2 a = unpack2(acc[r][0]), b = unpack2(acc[r][1]);
            float4 v = make_float4(a.x, a.y, b.x, b.y);
            if (STEP == 2) {
                v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
                v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
                v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
                v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
            }
            if (rl == 0) *reinterpret_cast<float4*>(so + warp * WF + r * HS + 4 * ch) = v;
            if (lane == 0) ml_s[warp][r] = make_float2(m[r], l[r]);
        }
        few_end<HS, float>(A, s, t, head, unit, whole, lo, hi, so, WF, ml_s, bad, 1.f);
        left -= n + PAIR_COST;
        unit = 0;
        if (left > 0 && ++head == c.n_kv) {
            head = 0;
            t = load_tile(c.plan, s.tiles, ++tile);
        }
    }
}

template <int HS, int R, bool ALIGNED>
int launch_few32(slai_ctx* ctx, const AttnArgs& A, int blocks, bool pdl) {
    auto kern = paged_attn_few32_kernel<HS, R, ALIGNED>;
    static PerDeviceOnce attr;
    if (attr.need(ctx->device)) {
        SLAI_CHECK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW32_SMEM<HS, R>));
        attr.set(ctx->device);
    }
    return launch_dependent(ctx, kern, dim3((unsigned)blocks), FT, FEW32_SMEM<HS, R>, pdl, A);
}
template <int HS>
int launch_few32_of(slai_ctx* ctx, const AttnArgs& A, int blocks, bool pdl) {
    if (A.tile_rows == 1) return A.c.page_size % EP == 0 ? launch_few32<HS, 1, true>(ctx, A, blocks, pdl) : launch_few32<HS, 1, false>(ctx, A, blocks, pdl);
    if (A.c.page_size % EP == 0) return A.tile_rows <= 4 ? launch_few32<HS, 4, true>(ctx, A, blocks, pdl) : launch_few32<HS, 8, true>(ctx, A, blocks, pdl);
    return A.tile_rows <= 4 ? launch_few32<HS, 4, false>(ctx, A, blocks, pdl) : launch_few32<HS, 8, false>(ctx, A, blocks, pdl);
}

}  // namespace

// Whether a handle's few-row launches can take the kernels above (with rows that can be read in 16-byte pieces).
bool paged_attention_few(int kv_dtype, int hs) { return hs % (kv_dtype == SLAI_KV_F16 ? 8 : 4) == 0 && hs <= 128; }
Lane paged_attention_lane(int kv_dtype, int hs, int group, int sms) {
    Lane l;
    l.unit = 64;
    l.least = 2;
    if (paged_attention_few(kv_dtype, hs)) {
        l.rows = kv_dtype == SLAI_KV_F16 || group > 4 ? FR : group == 1 ? 1 : 4;
        l.blocks = FB * sms;
        // us a call, cut / not cut where it can be: one token, 32 heads, at position 300 8.4 / 7.0, 515 8.8 / 10.2; a token of each of 8 sequences, 32 heads, at
        // 100 10.4 / 5.3, 515 20.6 / 16.9, 1000 31.4 / 27.6; 64 heads on 8 at 300 9.9 / 8.6, 515 11.2 / 12.5.
        l.join = kv_dtype == SLAI_KV_F32 && l.rows == FR ? 1 : 5;  // (a unit of eight rows in f32 takes as long as the join: a token of 64 heads on 8 at 300 18.8 / 13.6 us if cut only at 5 / from 1)
        l.fixed = 5;
        l.each = kv_dtype == SLAI_KV_F16 ? 0.0054 : l.rows == 1 ? 0.004 : l.rows == FR ? 0.018 : 0.0126;
    } else {
        l.rows = GR;
        l.blocks = 4 * sms;
    }
    return l;
}
static int launch_lane(slai_ctx* ctx, const AttnArgs& A, int kv_dtype, int lane, int blocks, bool pdl) {
    if (lane == 1 && A.vec) {
        if (kv_dtype == SLAI_KV_F16) return paged_prompt_launch(ctx, A, blocks, pdl);
        return paged_prompt32_launch(ctx, A, blocks, pdl);
    }
    if (lane == 0 && A.vec && paged_attention_few(kv_dtype, A.c.hs)) {
        if (kv_dtype == SLAI_KV_F32) return A.c.hs <= 64 ? launch_few32_of<64>(ctx, A, blocks, pdl) : launch_few32_of<128>(ctx, A, blocks, pdl);
        if (A.c.page_size % FP == 0) return A.c.hs <= 64 ? launch_few<64, true>(ctx, A, blocks, pdl) : launch_few<128, true>(ctx, A, blocks, pdl);
        return A.c.hs <= 64 ? launch_few<64, false>(ctx, A, blocks, pdl) : launch_few<128, false>(ctx, A, blocks, pdl);
    }
    return kv_dtype == SLAI_KV_F16 ? launch_any<__half>(ctx, A, blocks, pdl) : launch_any<float>(ctx, A, blocks, pdl);
}
int paged_attention_launch(slai_ctx* ctx, AttnArgs& A, int kv_dtype, int lane, int blocks, int joins, int longest, bool pdl) {
    if (blocks <= 0) return SLAI_OK;
    const int rc = launch_lane(ctx, A, kv_dtype, lane, blocks, pdl);
    if (rc) return rc;
    // (recorded: a launch for the most pairs that there can be took 2 to 3 us when there were none)
    return A.recorded ? launch_join<true>(ctx, A, (joins + 3) / 4, longest, pdl) : launch_join<false>(ctx, A, joins, longest, pdl);
}
