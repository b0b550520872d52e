// What the paged attention kernels share on the device.
#pragma once
#include "paged.cuh"

namespace paged {

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }

// Two f32 at a time
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ f32x2 pack2(uint32_t a, uint32_t b) { return pack2(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ float2 unpack2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// v = hi + lo, 22 bits
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const __half2 l = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
// 2^x, of the sizes weights have
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The power of two that puts a row's largest query below 2^15, and its inverse: whatever their size they fit a pair of halves.
__device__ __forceinline__ float power_up(float largest, float& unit) {
    const int e = max((int)(__float_as_uint(largest) >> 23), 15);  // biased by 127
    unit = __uint_as_float((uint32_t)(e - 14) << 23);
    return __uint_as_float((uint32_t)(127 + 14 + 127 - e) << 23);
}

// ---- what the matrix units cannot carry ----------------------------------------------------------------------------------
// The kernels below multiply whole tiles: a weight of zero times an infinite value that its row does not see would be NaN.  A row whose sums are not finite (this,
// or the formula's own infinities and NaN) is computed again by one warp, position by position: [lo, hi) of the positions, as the formula says.
template <typename T>
__device__ __noinline__ void row_again(const AttnArgs& A, const Tile& t, int head, int r, int lo, int hi, float* out, float* ml) {
    const Cache& c = A.c;
    const int lane = threadIdx.x & 31, pr = t.first + r, tok = pr / c.group;
    const float* q = A.q + (t.row0 + tok) * A.q_ld + (long long)(head * c.group + pr % c.group) * c.hs;
    hi = min(hi, t.pos0 + tok + 1);
    float m = -INFINITY, l = 0.f, acc[8] = {};
    for (int p0 = lo; p0 < hi; p0 += 32) {
        const bool seen = p0 + lane < hi;
        const long long at = seen ? place_of(c, t.table, p0 + lane, head) : 0;
        float s = 0.f;
        if (seen)
            for (int d = 0; d < c.hs; d++) s = fmaf(__ldcg(q + d) * A.scale, to_float<T>(reinterpret_cast<const T*>(c.keys)[at + d]), s);
        float mt = seen ? s : -INFINITY;
        for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
        const float m_new = fmaxf(m, mt), resc = m == -INFINITY ? 1.f : expf(m - m_new);
        const float w = !seen || s == -INFINITY ? 0.f : expf(s - m_new);
        float ws = w;
        for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
        l = l * resc + ws;
        m = m_new;
        for (int j = 0; j < 8; j++) acc[j] *= resc;
        for (int i = 0; i < min(32, hi - p0); i++) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            const long long ai = __shfl_sync(0xffffffffu, at, i);
            for (int j = 0; j < 8; j++)
                if (lane + 32 * j < c.hs) acc[j] = fmaf(wi, to_float<T>(reinterpret_cast<const T*>(c.values)[ai + lane + 32 * j]), acc[j]);
        }
    }
    for (int j = 0; j < 8; j++)
        if (lane + 32 * j < c.hs) out[lane + 32 * j] = ml ? acc[j] : acc[j] / l;
    if (ml && lane == 0) *reinterpret_cast<float2*>(ml) = make_float2(m * LOG2E, l);
}

}  // namespace paged
