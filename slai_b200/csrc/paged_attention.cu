// Causal attention of a step's new tokens to the keys and values that their sequences hold in pages: out = softmax(q K^T scale) V, each token over the
// positions up to its own, a cache head shared by `group` query heads.  (The reference's operator has one token and one dense cache:
// crates/slai/src/ops/batched_multiquery_attention.rs:32-156.)  Who computes what: paged_plan.h.
#include "paged.cuh"

using namespace paged;

namespace {

// ---- any head size, either cache type, any alignment ---------------------------------------------------------------------
// 16 rows at a time, positions in tiles of 32 brought into shared memory as f32; warp w has rows 4w .. 4w + 3; scores: lane = position, sums of values:
// lane = dimensions.  Plain f32 arithmetic, one pass with the running maximum and sum of each row.
constexpr int GT = 128, GR = 16, GP = 32;

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }

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
__global__ void __launch_bounds__(GT) paged_attn_any_kernel(const AttnArgs A) {
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
    __shared__ int flag;
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
                if (!whole && lane == 0) *reinterpret_cast<float2*>(A.part_ml + (slot + g0 + r) * 2) = make_float2(m[i], l[i]);
            }
        }
        if (!whole) {
            const long long at = (long long)t.line + (long long)head * t.units;
            const int first = block_of(s, at), end = block_of(s, at + t.units - 1);
            if (last_to_come(A.tickets + first, end - first + 1, &flag)) join<GT>(A, t, head, first, end);
        }
        left -= n;
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

}  // namespace

int paged_attention_launch(slai_ctx* ctx, AttnArgs& A, int kv_dtype, int lane, int blocks, bool pdl) {
    (void)lane;
    if (blocks <= 0) return SLAI_OK;
    return kv_dtype == SLAI_KV_F16 ? launch_any<__half>(ctx, A, blocks, pdl) : launch_any<float>(ctx, A, blocks, pdl);
}
