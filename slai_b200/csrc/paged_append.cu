// What happens to a step's q, k and v between their product and the attention, in one pass: RmsNorm of every head of q and k
// (y = x * rsqrt(mean x^2 + eps) * w), rotation of its pairs by the token's position, keys and values into the pages of their sequences.  (The reference does
// the parts as operators of their own: crates/slai/src/ops/rms_norm.rs:35-77, ops/rope.rs:45-85, key_cache.column(pos) at
// models/llama2/transformer.rs:329-334.)
//
// The angle of pair i at position p is p * base^(-2i / hs): far into a long context its f32 value has lost the digits that matter (at position 120000 it is off
// by up to 0.008), so the turns p * base^(-2i / hs) / 2 pi are formed in 64 bits, the whole ones dropped, and the rest goes to sincospi in f32.
#include "paged.cuh"

namespace {

constexpr int QT = 256, QU = 4;  // threads; heads a warp takes one after the other where there are many

// cos and sin of pair i at position p
__device__ __forceinline__ float2 turn(const double* turns, int i, int p) {
    const double t = (double)p * turns[i];
    float s, c;
    sincospif((float)(2.0 * (t - rint(t))), &s, &c);
    return make_float2(c, s);
}

// A head of one token: where it comes from and goes to.
struct Head {
    const float* in;
    float* out;         // f32 result, or
    char* cache;        // place in the cache (bytes)
    const float* norm;
    bool turn;
};
__device__ __forceinline__ Head head_of(const QkArgs& A, int row, int slot, int h) {
    Head H = {nullptr, nullptr, nullptr, nullptr, A.turns != nullptr};
    if (h < A.n_q) {
        H.in = A.q + row * A.q_ld + (long long)h * A.hs;
        H.out = A.q_out + row * A.q_out_ld + (long long)h * A.hs;
        H.norm = A.q_norm;
        return H;
    }
    const int kv = (h - A.n_q) % A.n_kv;
    const bool value = h >= A.n_q + A.n_kv;
    H.in = value ? A.v + row * A.v_ld + (long long)kv * A.hs : A.k + row * A.k_ld + (long long)kv * A.hs;
    H.norm = value ? nullptr : A.k_norm;
    if (value) H.turn = false;
    if (A.v) {
        const paged::Cache& c = A.cache;
        const int page = slot / c.page_size;
        H.cache = (value ? c.values : c.keys) + (A.kv_f16 ? 2 : 4) * (page * c.page_stride + kv * c.head_stride + (slot - page * c.page_size) * c.pos_stride);
    } else {
        H.out = A.k_out + row * A.k_out_ld + (long long)kv * A.hs;
    }
    return H;
}

// Any head size and alignment: a warp takes one head of one token.
__global__ void __launch_bounds__(QT) qk_any_kernel(const QkArgs A) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int heads = A.n_q + (A.v ? 2 : 1) * A.n_kv, lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * (QT / 32) + (threadIdx.x >> 5);
    if (w >= (long long)A.rows * heads) return;
    const int row = (int)(w / heads), h = (int)(w - (long long)row * heads);
    if (A.counted && row >= __ldcg(A.cache.plan + A.cache.count_at)) return;
    const int2 ps = A.v ? __ldcg(reinterpret_cast<const int2*>(A.cache.plan + A.cache.rows_at) + row) : make_int2(__ldcg(A.pos + row), 0);
    if (ps.x < 0) return;
    const Head H = head_of(A, row, ps.y, h);
    // pairs (lane + 32 j) of the head (variant 0: elements 2i, 2i + 1; else i, i + hs / 2), then the last element of an odd head
    const int half = A.hs / 2;
    float x[4][2], last = 0.f, ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = lane + 32 * j;
        x[j][0] = x[j][1] = 0.f;
        if (i < half) {
            x[j][0] = __ldcg(H.in + (A.variant == 0 ? 2 * i : i));
            x[j][1] = __ldcg(H.in + (A.variant == 0 ? 2 * i + 1 : i + half));
        }
        ss = fmaf(x[j][0], x[j][0], fmaf(x[j][1], x[j][1], ss));
    }
    const bool odd = (A.hs & 1) && lane == 0;
    if (odd) {
        last = __ldcg(H.in + A.hs - 1);
        ss = fmaf(last, last, ss);
    }
    if (H.norm) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = rsqrtf(ss / (float)A.hs + A.eps);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int i = lane + 32 * j;
            if (i < half) {
                x[j][0] = x[j][0] * r * H.norm[A.variant == 0 ? 2 * i : i];
                x[j][1] = x[j][1] * r * H.norm[A.variant == 0 ? 2 * i + 1 : i + half];
            }
        }
        if (odd) last = last * r * H.norm[A.hs - 1];
    }
    __syncwarp();
    auto put = [&](int e, float y) {
        if (H.out) H.out[e] = y;
        else if (A.kv_f16) reinterpret_cast<__half*>(H.cache)[e] = __float2half_rn(y);
        else reinterpret_cast<float*>(H.cache)[e] = y;
    };
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = lane + 32 * j;
        if (i >= half) continue;
        float2 cs = make_float2(1.f, 0.f);
        if (H.turn) cs = turn(A.turns, i, ps.x);
        const float a = H.turn ? x[j][0] * cs.x - x[j][1] * cs.y : x[j][0], b = H.turn ? x[j][0] * cs.y + x[j][1] * cs.x : x[j][1];
        put(A.variant == 0 ? 2 * i : i, a);
        put(A.variant == 0 ? 2 * i + 1 : i + half, b);
    }
    if (odd) put(A.hs - 1, last);
}

// Heads of a multiple of 8 elements on 16-byte boundaries: LPH lanes take a head, 8 elements a lane (two 16-byte pieces that hold four whole pairs in either
// variant), a warp 32 / LPH * U heads of one token, whose angles it needs once.  Memory bounds it: 4095 tokens of 64 + 8 heads of 128, 302 MB, 53 to 58 us (81 to 89 % of
// the copy rate); 1919 tokens of 64 + 8 + 8 appended, 149 MB, 29 to 31.5 us (73 to 79 %).  us of the two by U and blocks an SM: 1 x 6 70.2, 36.5; 2 x 4 60.2, 32.1; 2 x 6 63.9, 34.0;
// 4 x 3 57.5, 31.7; 8 x 2 64.7, 40.0; 4 x 3 with loads that leave L2 first 52.7, 29.2 (the best runs).
template <int LPH, int U, bool NEOX>
__global__ void __launch_bounds__(QT, 3) qk_vec_kernel(const QkArgs A) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int HPW = 32 / LPH;
    const int heads = A.n_q + (A.v ? 2 : 1) * A.n_kv, chunks = (heads + HPW * U - 1) / (HPW * U), lane = threadIdx.x & 31, l = lane % LPH;
    const long long w = (long long)blockIdx.x * (QT / 32) + (threadIdx.x >> 5);
    const int row = (int)(w / chunks), h0 = (int)(w - (long long)row * chunks) * HPW * U;
    if (row >= A.rows || (A.counted && row >= __ldcg(A.cache.plan + A.cache.count_at))) return;
    const int2 ps = A.v ? __ldcg(reinterpret_cast<const int2*>(A.cache.plan + A.cache.rows_at) + row) : make_int2(__ldcg(A.pos + row), 0);
    if (ps.x < 0) return;
    const bool mine = 8 * l < A.hs;
    const int e0 = NEOX ? 4 * l : 8 * l, e1 = NEOX ? A.hs / 2 + 4 * l : 8 * l + 4;
    float4 x[U][2];
#pragma unroll
    for (int u = 0; u < U; u++) {  // all loads on their way first (where they go is worked out again below: kept meanwhile, it took half of the registers)
        const int h = h0 + u * HPW + lane / LPH;
        x[u][0] = x[u][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (h < heads && mine) {
            const float* in = head_of(A, row, ps.y, h).in;
            x[u][0] = __ldcs(reinterpret_cast<const float4*>(in + e0));  // (read once: out of L2 before what the attention reads next)
            x[u][1] = __ldcs(reinterpret_cast<const float4*>(in + e1));
        }
    }
    float2 cs[4];
    if (A.turns && h0 < A.n_q + A.n_kv) {
#pragma unroll
        for (int i = 0; i < 4; i++) cs[i] = mine ? turn(A.turns, 4 * l + i, ps.x) : make_float2(1.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int h = h0 + u * HPW + lane / LPH;
        const Head H = head_of(A, row, ps.y, min(h, heads - 1));
        float v[8] = {x[u][0].x, x[u][0].y, x[u][0].z, x[u][0].w, x[u][1].x, x[u][1].y, x[u][1].z, x[u][1].w};
        if (A.q_norm || A.k_norm) {  // (the same for all lanes; the sum of a head that is not normalised goes unused)
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fmaf(v[i], v[i], ss);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (h < heads && mine && H.norm) {
                const float r = rsqrtf(ss / (float)A.hs + A.eps);
                const float4 w0 = *reinterpret_cast<const float4*>(H.norm + e0), w1 = *reinterpret_cast<const float4*>(H.norm + e1);
                const float wn[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = v[i] * r * wn[i];
            }
        }
        if (h >= heads || !mine) continue;
        if (H.turn) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float& a = v[NEOX ? i : 2 * i];
                float& b = v[NEOX ? i + 4 : 2 * i + 1];
                const float y = a * cs[i].x - b * cs[i].y;
                b = a * cs[i].y + b * cs[i].x;
                a = y;
            }
        }
        if (H.cache && A.kv_f16) {
            __half2 p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            __half* d = reinterpret_cast<__half*>(H.cache);
            *reinterpret_cast<uint2*>(d + e0) = *reinterpret_cast<uint2*>(p);
            *reinterpret_cast<uint2*>(d + e1) = *reinterpret_cast<uint2*>(p + 2);
        } else {
            float* d = H.out ? H.out : reinterpret_cast<float*>(H.cache);
            *reinterpret_cast<float4*>(d + e0) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(d + e1) = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
}

template <int LPH, bool NEOX>
int launch_vec(slai_ctx* ctx, QkArgs& A, long long heads, bool pdl) {
    constexpr int HPW = 32 / LPH;
    auto blocks = [&](int u) { return ((long long)A.rows * ((heads + HPW * u - 1) / (HPW * u)) + QT / 32 - 1) / (QT / 32); };
    // Several heads a warp where that leaves enough warps to keep the memory busy.
    const bool many = blocks(QU) >= 8 * (ctx->sm_count > 0 ? ctx->sm_count : 148);
    SLAI_REQUIRE(ctx, blocks(1) <= 0x7fffffffll, SLAI_ERR_SHAPE, "rows: too many (%d tokens of %lld heads)", A.rows, heads);
    return many ? launch_dependent(ctx, qk_vec_kernel<LPH, QU, NEOX>, dim3((unsigned)blocks(QU)), QT, 0, pdl, A)
                : launch_dependent(ctx, qk_vec_kernel<LPH, 1, NEOX>, dim3((unsigned)blocks(1)), QT, 0, pdl, A);
}

bool in_vectors(const QkArgs& A) {
    const int esz = A.kv_f16 ? 2 : 4;
    uintptr_t b = (uintptr_t)A.q | (uintptr_t)A.k | (uintptr_t)A.v | (uintptr_t)A.q_out | (uintptr_t)A.k_out | (uintptr_t)A.q_norm | (uintptr_t)A.k_norm;
    b |= (uintptr_t)(4 * (A.q_ld | A.k_ld | A.v_ld | A.q_out_ld | A.k_out_ld));
    if (A.v) b |= (uintptr_t)A.cache.keys | (uintptr_t)A.cache.values | (uintptr_t)(esz * (A.cache.page_stride | A.cache.head_stride | A.cache.pos_stride));
    return A.hs % 8 == 0 && (b & 15) == 0;
}

}  // namespace

int qk_launch(slai_ctx* ctx, QkArgs& A, bool pdl) {
    const long long heads = A.n_q + (A.v ? 2 : 1) * A.n_kv, warps = (long long)A.rows * heads;
    if (warps == 0) return SLAI_OK;
    if (in_vectors(A)) {
        if (A.variant == 0) return A.hs <= 64 ? launch_vec<8, false>(ctx, A, heads, pdl) : A.hs <= 128 ? launch_vec<16, false>(ctx, A, heads, pdl) : launch_vec<32, false>(ctx, A, heads, pdl);
        return A.hs <= 64 ? launch_vec<8, true>(ctx, A, heads, pdl) : A.hs <= 128 ? launch_vec<16, true>(ctx, A, heads, pdl) : launch_vec<32, true>(ctx, A, heads, pdl);
    }
    const long long blocks = (warps + QT / 32 - 1) / (QT / 32);
    SLAI_REQUIRE(ctx, blocks <= 0x7fffffffll, SLAI_ERR_SHAPE, "rows: too many (%d tokens of %lld heads)", A.rows, heads);
    return launch_dependent(ctx, qk_any_kernel, dim3((unsigned)blocks), QT, 0, pdl, A);
}
