// Paged attention for many rows and f32 caches: chunks of prompts, on the 5th-generation tensor cores.
//
// A tile is 128 rows (token, query head of the group) against 32 positions at a time.  Queries, keys, weights and values are each two tf32 numbers, the value rounded to
// 11 bits and the rest cut to 11 bits (together 21, over f32's whole range of exponents), and a product is three of the tensor core's: high x high, high x low,
// low x high; low x low is below 2^-22 of it.  The tensor core truncates when it adds: the small terms of scores have columns of their own, those of the sum of values
// come first, and that sum ends with its 32 positions and goes on in its row's threads, f32, times the factor by which the running maximum moved.
//
//   warp 0       issues the products: QK(j + 1), then PV(j).  Queries are in tensor memory (2 x HS columns), scores, whose place the weights take, too (two stages of 64
//                columns), and one output.
//   warps 4-11   softmax, two threads a row, half of the positions and half of the dimensions each: queries into tensor memory, scores out of it, weights into it,
//                outputs out of it, results.
//   warps 12-27  keys and values, two sets of eight in turn: out of the pages two steps ahead into registers, in two parts each into shared memory, rows of 128 bytes in the tensor core's swizzle.
//                Values lie there with a row a dimension: a thread reads four positions of one dimension, a warp's threads next to each other.
//
// Barriers: a stage of scores, weights, keys and values has a unit's number's parity; a unit's QK and PV being complete is what frees them.  (The issuer waits for the PV of
// unit u - 1 before the QK of unit u + 1 takes its stage: paged_order.h.  It costs 1 % where power sets the clock, 211 for 208 us a call in a loop, and 8 % of
// one launch under the profiler, 229 for 212.)
// 1023 tokens of 32 heads behind 2000 positions 211 us, 199 TFLOP/s, 597 executed, where the card's power sets the clock (1.6 GHz); 37 tokens behind 300 15.2 us.  (f32 arithmetic
// of 64 rows and 32 positions in shared memory: 31 TFLOP/s, 25 us.)
// What bounds it: 32 positions took 2500 cycles (511 tokens) before that wait, of which the 44 products take 1960 (1540 at the full rate) and what their issuer waits for
// between them 540.
// Descriptors in uniform registers: 225 -> 208 us.  A thread a row: 209, but 19 for 17 us with few tokens.
// Tried and taken back: eight more warps for the outputs (251 us: one more hop in the chain); one set of loading warps (257).
// Every wait is bounded (common.cuh, bounded_wait).
#include <type_traits>

#include "paged_order.h"
#include "paged_tc.cuh"

using namespace paged;

namespace {

constexpr int XT = 896, XR = 128, XP = 32, XU = 64;  // threads, rows of a tile, positions at a time, positions of a unit of the plan
constexpr int LOADERS = 8;                           // warps of either set

// kind::tf32: f32 results (bits 4-5 = 1), tf32 operands (bits 7-9 and 10-12 = 2), N / 8 in bits 17-22, M / 16 in bits 24-28
__device__ __forceinline__ uint32_t idesc(int n) { return (1u << 4) | (2u << 7) | (2u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(XR >> 4) << 24); }
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate)
                 : "memory");
}
// v = hi + lo: the value rounded to tf32's 11 bits, and the rest, of which the tensor core takes 11 bits.  An infinite value leaves NaN in lo, a NaN one of hi's.
// (By cvt.rna.tf32, two a value: 244 us instead of 212 for 1023 tokens of 32 heads behind 2000.)
__device__ __forceinline__ void split(float v, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(v) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(v - __uint_as_float(hi));
}

// Shared memory, of two units: keys [32 dimensions][high, low][32 positions][128 bytes], values [high, low][HS dimensions][128 bytes]; the tile's rows in f32 (queries on
// their way in, results out).
template <int HS>
struct Smem {
    static constexpr int PART = HS * 128, SLOT = 2 * PART, KS = HS + 4, ROWS = 4 * SLOT;
    struct Rest {
        unsigned long long bars[12];
        float max_s[2][2][XR];      // of every second unit: what the two threads of a row tell one another
        float sum_s[2][XR];         // of a part
        unsigned int bad_s[2][2][4];
        uint32_t tmem_slot;
    };
    static constexpr int REST = ROWS + 4 * XR * KS, TOTAL = REST + (int)sizeof(Rest);
    static_assert(TOTAL <= 227 * 1024, "a block's shared memory");
};
struct Part {  // a block's part of one (tile, head) pair: positions [lo, hi), n times XP
    int unit, units, lo, hi, n;
    bool whole;
};
template <class F>
__device__ __forceinline__ void for_parts(const Start& s, const Cache& c, F f) {
    Tile t = s.t;
    int head = s.head, unit = s.unit, tile = s.tile;
    for (int left = s.count; left > 0;) {
        Part p;
        p.unit = unit;
        p.units = min(left, t.units - unit);
        p.whole = p.units == t.units;
        p.lo = unit * XU;
        p.hi = min((unit + p.units) * XU, t.pos0 + (t.first + t.rows - 1) / c.group + 1);
        p.n = (p.hi - p.lo + XP - 1) / XP;
        f(t, head, p);
        left -= p.units + PAIR_COST;
        unit = 0;
        if (left > 0 && ++head == c.n_kv) {
            head = 0;
            t = load_tile(c.plan, s.tiles, ++tile);
        }
    }
}

template <int HS>
__global__ void __launch_bounds__(XT, 1) paged_attn_prompt32_kernel(const __grid_constant__ AttnArgs A) {
    using L = Smem<HS>;
    extern __shared__ __align__(1024) unsigned char smem[];  // (the kernel has no other shared memory: the operands begin on the swizzle's boundary)
    typename L::Rest& rest = *reinterpret_cast<typename L::Rest*>(smem + L::REST);
    if (smem_u32(smem) & 1023) {
        if (threadIdx.x == 0) atomicExch(A.err_flag, (unsigned int)ERR_PAGED);
        return;
    }
    if (A.recorded && __ldcg(A.c.plan + A.starts_at + (int)(sizeof(Start) / 4) * blockIdx.x + 3) <= 0) {  // (count) there is room for more blocks than the step has
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const uint32_t sb = smem_u32(smem);
    const uint32_t k_full = smem_u32(rest.bars), v_full = k_full + 16, qk_done = v_full + 16, p_full = qk_done + 16, pv_done = p_full + 16, q_full = pv_done + 16, all_done = q_full + 8;
    const Cache& c = A.c;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, hs = c.hs;
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(k_full + 8 * i, LOADERS);
            mbar_init(v_full + 8 * i, LOADERS);
            mbar_init(qk_done + 8 * i, 1);
            mbar_init(p_full + 8 * i, 8);
            mbar_init(pv_done + 8 * i, 1);
        }
        mbar_init(q_full, 8);
        mbar_init(all_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&rest.tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = uniform(rest.tmem_slot), out_cols = tmem + 2 * HS, stages = tmem + 384;
    const Start s = load_start(c.plan, A.starts_at, blockIdx.x);  // (there before any kernel of its step starts)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    unsigned int limit = A.wait_limit;
    auto wait = [&](uint32_t bar, uint32_t parity) { return bounded_wait<false, true, ERR_PAGED>(bar, parity & 1, limit, A.err_flag); };
    constexpr int KB = 2 * XP * 128;            // 32 dimensions of the keys: the positions' high parts, their low parts
    constexpr int CH = HS / 4, STEP = 32 / CH;  // 16-byte pieces of a row, rows a pass of a warp covers
    const int ch = lane % CH, rl = lane / CH, chunks = hs / 4;

    // Registers: 4 x 32 x 40 + 8 x 32 x 128 + 16 x 32 x 48 = 62464 of the launch's 896 x 72.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0) {
            // ---- products ----
            const uint32_t id_qk = idesc(XP), id_qk2 = idesc(2 * XP), id_pv = idesc(HS);
            uint32_t u = 0, n_part = 0;  // the part's first unit
            for_parts(s, c, [&](const Tile&, int, const Part& p) {
                wait(q_full, n_part++);
                auto do_qk = [&](uint32_t i) {
                    const uint32_t g = uniform(i & 1), d = stages + 64 * g;
                    const uint64_t keys = desc_k(sb + 2 * g * L::SLOT);
                    wait(k_full + 8 * g, i >> 1);
                    tc_after();
                    __syncwarp();
                    if (elect_one() && limit) {
#pragma unroll
                        for (int k = 0; k < HS / 8; k++)  // high queries, high and low keys
                            umma_ts(d, tmem + 8 * k, keys + ((k / 4) * KB + 32 * (k % 4)) / 16, id_qk2, k > 0);
#pragma unroll
                        for (int k = 0; k < HS / 8; k++)  // low queries, high keys, to the low keys' columns
                            umma_ts(d + XP, tmem + HS + 8 * k, keys + ((k / 4) * KB + 32 * (k % 4)) / 16, id_qk, 1);
                        umma_commit(qk_done + 8 * g);
                    }
                    __syncwarp();
                };
                auto do_pv = [&](uint32_t i) {
                    const uint32_t g = uniform(i & 1), a = stages + 64 * g;
                    const uint64_t values = desc_k(sb + (2 * g + 1) * L::SLOT);
                    wait(v_full + 8 * g, i >> 1);
                    wait(p_full + 8 * g, i >> 1);
                    tc_after();
                    __syncwarp();
                    if (elect_one() && limit) {
#pragma unroll
                        for (int w = 0; w < 3; w++)
#pragma unroll
                            for (int k = 0; k < XP / 8; k++) umma_ts(out_cols, a + (w == 0 ? XP : 0) + 8 * k, values + ((w == 1 ? L::PART : 0) + 32 * k) / 16, id_pv, w > 0 || k > 0);
                        umma_commit(pv_done + 8 * g);
                    }
                    __syncwarp();
                };
                chunk_products(u, p.n, [&](uint32_t i) { wait(pv_done + 8 * (i & 1), i >> 1); }, do_qk, do_pv);
                u += p.n;
            });
            if (elect_one()) umma_commit(all_done);  // no product is under way when the block ends
            limit = LAST_POLLS;
            wait(all_done, 0);
            __syncwarp();
        }
    } else if (warp >= 12) {
        // ---- keys and values of every second unit: this warp's positions are 4 w .. + 3 of 32 ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        const int w = (warp - 12) & 7;
        const uint32_t g = (warp - 12) >> 3;
        unsigned char* slot = smem + 2 * g * L::SLOT;
        uint32_t u = 0;  // the part's first unit
        for_parts(s, c, [&](const Tile& t, int head, const Part& p) {
            auto place = [&](int j) {  // lane i: of position i % 4, -1 behind the last
                const int at = p.lo + XP * j + 4 * w + (lane & 3);
                return at < p.hi ? 4 * place_of(c, t.table, at, head) : -1;
            };
            float4 kr[4 / STEP];
            float vr[HS / 32][4];
            auto load_k = [&](long long at) {
#pragma unroll
                for (int i = 0; i < 4 / STEP; i++) {
                    const long long a = __shfl_sync(0xffffffffu, at, STEP * i + rl);
                    kr[i] = a >= 0 && ch < chunks ? __ldcg(reinterpret_cast<const float4*>(c.keys + a) + ch) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            };
            auto load_v = [&](long long at) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const long long a = __shfl_sync(0xffffffffu, at, i);
#pragma unroll
                    for (int d = 0; d < HS / 32; d++) vr[d][i] = a >= 0 && 32 * d + lane < hs ? __ldcg(reinterpret_cast<const float*>(c.values + a) + 32 * d + lane) : 0.f;
                }
            };
            auto put = [&](unsigned char* to, int low, float x, float y, float z, float e) {
                uint4 hi, lo;
                split(x, hi.x, lo.x);
                split(y, hi.y, lo.y);
                split(z, hi.z, lo.z);
                split(e, hi.w, lo.w);
                *reinterpret_cast<uint4*>(to) = hi;
                *reinterpret_cast<uint4*>(to + low) = lo;
            };
            int j = (u ^ g) & 1;
            if (j < p.n) {
                const long long at = place(j);
                load_k(at);
                load_v(at);
            }
            for (; j < p.n; j += 2) {
                const uint32_t round = (u + j) >> 1;
                const long long at = j + 2 < p.n ? place(j + 2) : -1;
                if (round > 0) wait(qk_done + 8 * g, round - 1);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4 / STEP; i++) {
                    const int row = 4 * w + STEP * i + rl;
                    put(slot + (ch >> 3) * KB + row * 128 + (((ch & 7) ^ (row & 7)) << 4), XP * 128, kr[i].x, kr[i].y, kr[i].z, kr[i].w);
                }
                fence_async();
                __syncwarp();
                if (lane == 0 && limit) mbar_arrive(k_full + 8 * g);
                if (round > 0) wait(pv_done + 8 * g, round - 1);
                __syncwarp();
#pragma unroll
                for (int d = 0; d < HS / 32; d++) put(slot + L::SLOT + (32 * d + lane) * 128 + ((w ^ (lane & 7)) << 4), L::PART, vr[d][0], vr[d][1], vr[d][2], vr[d][3]);
                fence_async();
                __syncwarp();
                if (lane == 0 && limit) mbar_arrive(v_full + 8 * g);
                if (j + 2 < p.n) {  // (not before: the fence waits for loads)
                    load_k(at);
                    load_v(at);
                }
            }
            u += p.n;
        });
    } else {
        // ---- softmax: two threads a row, half of the positions and then of the dimensions each ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
        constexpr int DH = HS / 2;
        const int q4 = warp & 3, g = (warp >> 3) & 1, r = 32 * q4 + lane;
        const uint32_t lanes = (uint32_t)(32 * q4) << 16;
        float* rows_s = reinterpret_cast<float*>(smem + L::ROWS) + 32 * q4 * L::KS;  // the two warps'
        float* own = rows_s + lane * L::KS + DH * g;
        auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + q4) : "memory"); };
        uint32_t u = 0, n_part = 0;
        for_parts(s, c, [&](const Tile& t, int head, const Part& p) {
            const int pr = t.first + min(r, t.rows - 1), tok = pr / c.group, vis = r < t.rows ? t.pos0 + tok : 0x7fffffff;  // last position the row sees (rows behind the last: all, so that they need no mask)
            const long long col = (long long)(head * c.group + pr % c.group) * hs, q_at = (t.row0 + tok) * A.q_ld + col;
            // queries: 16 rows a warp in whole pieces to shared memory, from there each thread's to tensor memory
#pragma unroll 8
            for (int i = 16 * g; i < 16 * g + 16; i += STEP) {
                const float* q = A.q + __shfl_sync(0xffffffffu, q_at, i + rl) + 4 * ch;
                float* to = rows_s + (i + rl) * L::KS + 4 * ch;
                const bool there = 32 * q4 + i + rl < t.rows && ch < chunks;
                if (A.qvec) {
                    const uint32_t bytes = there ? 16u : 0u;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(__cvta_generic_to_global(there ? q : A.q)), "r"(bytes) : "memory");
                } else {
                    *reinterpret_cast<float4*>(to) = there ? make_float4(__ldcg(q), __ldcg(q + 1), __ldcg(q + 2), __ldcg(q + 3)) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            meet();
#pragma unroll
            for (int k = 0; k < DH; k += 16) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(own + k + i);
                    split(v.x * A.scale, hi[i], lo[i]);
                    split(v.y * A.scale, hi[i + 1], lo[i + 1]);
                    split(v.z * A.scale, hi[i + 2], lo[i + 2]);
                    split(v.w * A.scale, hi[i + 3], lo[i + 3]);
                }
                tmem_st16(tmem + lanes + DH * g + k, hi);
                tmem_st16(tmem + lanes + HS + DH * g + k, lo);
            }
            tmem_wait_st();
            tc_before();
            __syncwarp();
            if (lane == 0 && limit) mbar_arrive(q_full);
            f32x2 acc[DH / 2];
#pragma unroll
            for (int d = 0; d < DH / 2; d++) acc[d] = 0;
            float m = -INFINITY, l = 0.f, resc = 0.f;
            auto add_outputs = [&](uint32_t i) {  // unit i's
                wait(pv_done + 8 * (i & 1), i >> 1);
                __syncwarp();
                tc_after();
                const f32x2 by = pack2(resc, resc);
#pragma unroll
                for (int k = 0; k < DH / 32; k++) {
                    uint32_t o[2][16];
                    tmem_ld16(out_cols + lanes + DH * g + 32 * k, o[0]);
                    tmem_ld16(out_cols + lanes + DH * g + 32 * k + 16, o[1]);
                    tmem_wait_ld();
#pragma unroll
                    for (int d = 0; d < 16; d++) acc[16 * k + d] = fma2(acc[16 * k + d], by, pack2(o[d >> 3][2 * d & 15], o[d >> 3][(2 * d & 15) + 1]));
                }
            };
            for (int j = 0; j < p.n; j++, u++) {
                const uint32_t reg = stages + 64 * (u & 1) + lanes + 16 * g;
                const int p0 = p.lo + XP * j + 16 * g;
                wait(qk_done + 8 * (u & 1), u >> 1);
                __syncwarp();
                tc_after();
                float moved;
                auto weights = [&](auto all_seen) {
                    constexpr bool ALL = decltype(all_seen)::value;
                    const int seen = vis - p0;  // positions 0 .. seen of this thread's 16
                    uint32_t x[16], y[16];      // scores, their small terms
                    tmem_ld16(reg, x);
                    tmem_ld16(reg + XP, y);
                    tmem_wait_ld();
                    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float2 v = unpack2(add2(pack2(x[i], x[i + 1]), pack2(y[i], y[i + 1])));
                        x[i] = __float_as_uint(v.x);
                        x[i + 1] = __float_as_uint(v.y);
                        mx[(i >> 1) & 1] = max3(mx[(i >> 1) & 1], ALL || i <= seen ? v.x : -INFINITY, ALL || i + 1 <= seen ? v.y : -INFINITY);
                    }
                    float* told = &rest.max_s[u & 1][g][r];
                    *told = fmaxf(mx[0], mx[1]);
                    meet();
                    const float m_new = fmaxf(m, fmaxf(*told, rest.max_s[u & 1][g ^ 1][r]) * LOG2E), base = m_new == -INFINITY ? 0.f : m_new;
                    moved = ex2(m - base);
                    m = m_new;
                    const f32x2 shift = pack2(-base, -base), slope = pack2(LOG2E, LOG2E);
                    f32x2 ps[2] = {0, 0};
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float2 e = unpack2(fma2(pack2(x[i], x[i + 1]), slope, shift));
                        const float a = ALL || i <= seen ? ex2(e.x) : 0.f, b = ALL || i + 1 <= seen ? ex2(e.y) : 0.f;
                        ps[(i >> 1) & 1] = add2(ps[(i >> 1) & 1], pack2(a, b));
                        split(a, hi[i], lo[i]);
                        split(b, hi[i + 1], lo[i + 1]);
                    }
                    tmem_st16(reg, hi);
                    tmem_st16(reg + XP, lo);
                    const float2 sum = unpack2(add2(ps[0], ps[1]));
                    l = l * moved + (sum.x + sum.y);  // (this thread's positions)
                };
                if (__all_sync(0xffffffffu, vis >= p0 + 15)) weights(std::true_type());
                else weights(std::false_type());
                if (j > 0) add_outputs(u - 1);
                resc = moved;
                tmem_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0 && limit) mbar_arrive(p_full + 8 * (u & 1));
            }
            add_outputs(u - 1);
            // ---- results: through shared memory, so that a row leaves in one piece ----
            rest.sum_s[g][r] = l;
            meet();
            l += rest.sum_s[g ^ 1][r];
            float sum = l;
#pragma unroll
            for (int d = 0; d < DH / 2; d++) {
                const float2 v = unpack2(acc[d]);
                sum += v.x + v.y;
            }
            const unsigned int bad = __ballot_sync(0xffffffffu, r < t.rows && !(fabsf(sum) < INFINITY));
            if (lane == 0) rest.bad_s[n_part & 1][g][q4] = bad;
            const float f = p.whole ? 1.f / l : 1.f;
#pragma unroll
            for (int d = 0; d < DH / 4; d++) {
                const float2 v = unpack2(acc[2 * d]), e = unpack2(acc[2 * d + 1]);
                *reinterpret_cast<float4*>(own + 4 * d) = make_float4(v.x * f, v.y * f, e.x * f, e.y * f);
            }
            meet();
            const size_t slot = ((size_t)s.me * 2 + (p.unit == 0)) * A.tile_rows;
            if (!p.whole && g == 0 && r < t.rows) *reinterpret_cast<float2*>(A.part_ml + (slot + r) * 2) = make_float2(m, l);
            float* o_at = p.whole ? A.out + (t.row0 + tok) * A.out_ld + col : A.part + (slot + min(r, t.rows - 1)) * hs;
            const bool vec = !p.whole || A.qvec;
#pragma unroll 8
            for (int i = 16 * g; i < 16 * g + 16; i += STEP) {
                float* o = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o_at), i + rl)) + 4 * ch;
                if (32 * q4 + i + rl < t.rows && ch < chunks) {
                    const float4 v = *reinterpret_cast<const float4*>(rows_s + (i + rl) * L::KS + 4 * ch);
                    if (vec) {
                        *reinterpret_cast<float4*>(o) = v;
                    } else {
                        o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
                    }
                }
            }
            const unsigned int again = rest.bad_s[n_part & 1][0][q4] | rest.bad_s[n_part & 1][1][q4];
            n_part++;
            if (again) {
                if (!p.whole) meet();  // (the first warp has written the maxima and sums)
                __syncwarp();
                for (int i = 16 * g; i < 16 * g + 16; i++)
                    if (again >> i & 1) {
                        float* o = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o_at), i));
                        row_again<float>(A, t, head, 32 * q4 + i, p.lo, p.hi, o, p.whole ? nullptr : A.part_ml + (slot + 32 * q4 + i) * 2);
                    }
            }
            meet();  // the next queries lie where the results were
        });
    }
    __syncwarp();
    tc_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <int HS>
int launch(slai_ctx* ctx, const AttnArgs& A, int blocks, bool pdl) {
    auto kern = paged_attn_prompt32_kernel<HS>;
    constexpr int bytes = Smem<HS>::TOTAL;
    static PerDeviceOnce attr;
    if (attr.need(ctx->device)) {
        SLAI_CHECK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        attr.set(ctx->device);
    }
    return launch_dependent(ctx, kern, dim3((unsigned)blocks), XT, bytes, pdl, A);
}

}  // namespace

Lane paged_prompt32_lane(int sms) {
    Lane l;
    l.rows = XR;
    l.unit = XU;
    l.blocks = sms;
    // us a call, units of 64, two at least / of 32, one / of 32, two: 16 heads on 2 behind 2000, 37 tokens 19.4 / 27.6 / 27.6; 32 heads behind 300, 128 tokens
    // 17.7 / 20.2 / 20.2, 37 tokens 15.3 / 16.6 / 16.5 (three of 64: 17.2).
    l.least = 2;
    l.fixed = 15;
    l.each = 0.007;
    l.join = 2;  // 32 heads behind 300, 16 tokens, five units: whole 20.6 us, cut 17.2 (when this was chosen; cut now 14.9)
    return l;
}

int paged_prompt32_launch(slai_ctx* ctx, const AttnArgs& A, int blocks, bool pdl) {
    return A.c.hs <= 64 ? launch<64>(ctx, A, blocks, pdl) : launch<128>(ctx, A, blocks, pdl);
}
