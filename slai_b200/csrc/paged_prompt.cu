// Paged attention for many rows and f16 caches: chunks of prompts, on the 5th-generation tensor cores.
//
// A tile is 256 rows (token, query head of the group), two halves A and B of 128 that share the keys and values: scores S = Q K^T of 128 x 128 positions and
// sums P V of them are products of tcgen05.mma with their f32 results in tensor memory, where a thread has a row.  Queries and weights are pairs of halves
// (22 bits), two products each: one rounding of either to f16 would put 1e-4 into the result, the pairs leave 3e-7.  The tensor core truncates when it adds:
// both sums end with their 128 positions, and a half's output goes on in its threads' registers, times the factor by which the running maximum moved.
//
//   warps 0-1    keys, warps 2-3 values into a ring of three tiles of shared memory (asynchronous 16-byte copies that write the swizzle themselves: pages of any
//                size, strides and order; positions behind the last are zeros)
//   warps 4-7    half A: softmax, a row a thread: S out of tensor memory once for its maximum and once more for the weights, which take its columns' place as the
//   warps 8-11   half B  next product's operand; then the product's result
//   warp 12      issues the products: QK_A(j), PV_B(j-1), QK_B(j), PV_A(j): while one half's threads are at its softmax the tensor cores are at the other's
//                products.  Three regions of 128 columns of tensor memory hold scores and weights in turn, one the outputs.
// A region is written again by the third QK after its own; by then the PV that read it is complete: before each PV its issuer waits until the output of the PV
// before has been read (one region for all of them), so that only the last PV issued can be under way.
//
// Every wait is bounded (common.cuh, bounded_wait).
#include "paged_rows.cuh"

using namespace paged;

namespace {

constexpr int PT = 512, PR = 128, PU = 128, PSLOTS = 3;  // threads, rows of a half, positions of a unit, tiles of keys or values in shared memory
constexpr int ERR_PAGED = 7;
constexpr float WEIGHT = 16.f;  // weights are carried 16 times their size: their low parts keep their bits, and the exponent's rounding stays below 2^-23

// ---- PTX wrappers ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t a, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(a), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t a) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(a) : "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Operand descriptors, rows of 128 bytes swizzled, 8-row groups 1024 bytes apart.  Rows along the product's inner dimension (values: row = position) are
// `blocks` bytes apart in the other direction: 64 dimensions to a row.
__device__ __forceinline__ uint64_t desc_k(uint32_t a) { return (uint64_t)((a >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t a, uint32_t blocks) {
    return (uint64_t)((a >> 4) & 0x3FFFu) | ((uint64_t)(blocks >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16: f32 results (bits 4-5 = 1), f16 operands, B's rows along the inner dimension (bit 16), N / 8 in bits 17-22, M / 16 in bits 24-28
__device__ __forceinline__ uint32_t idesc(int n, bool b_mn) { return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(PR >> 4) << 24); }
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
#define R32(r) "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), \
                "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),      \
                "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
#define W32(r) "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),   \
               "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),     \
               "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
                 "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : R32(r)
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
                 "%24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(a),
                 W32(r)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- shared memory -------------------------------------------------------------------------------------------------------
// Queries [half][high, low][64 dimensions][128 rows][128 bytes], then the ring [slot][64 dimensions][128 positions][128 bytes].
template <int HS>
struct Smem {
    static constexpr int BLOCK = 128 * 128, BLOCKS = HS / 64, Q = BLOCKS * BLOCK, TILE = BLOCKS * BLOCK;
    static constexpr int RING = 4 * Q, TOTAL = RING + PSLOTS * TILE;
};

// A block's part of one (tile, head) pair.
struct Part {
    int unit, n;      // units [unit, unit + n)
    int na, nb;       // of these, the ones that the halves' rows see
    int ra, rb;       // rows of the halves
    bool whole;
};
__device__ __forceinline__ Part part_of(const Tile& t, int unit, int left, int group) {
    Part p;
    p.unit = unit;
    p.n = min(left, t.units - unit);
    p.whole = p.n == t.units;
    p.ra = min(t.rows, PR);
    p.rb = t.rows - p.ra;
    auto seen = [&](int last_row) { return max(0, min(p.n, (t.pos0 + (t.first + last_row) / group) / PU + 1 - unit)); };
    p.na = seen(p.ra - 1);
    p.nb = p.rb > 0 ? seen(t.rows - 1) : 0;
    return p;
}
// The block's parts in order: f(tile, head, part).
template <class F>
__device__ __forceinline__ void for_parts(const Start& s, const Cache& c, F f) {
    Tile t = s.t;
    int head = s.head, unit = s.unit, tile = s.tile;
    for (int left = s.count; left > 0;) {
        const Part p = part_of(t, unit, left, c.group);
        f(t, head, p);
        left -= p.n + PAIR_COST;
        unit = 0;
        if (left > 0 && ++head == c.n_kv) {
            head = 0;
            t = load_tile(c.plan, s.tiles, ++tile);
        }
    }
}

template <int HS>
__global__ void __launch_bounds__(PT, 1) paged_attn_prompt_kernel(const __grid_constant__ AttnArgs A) {
    using L = Smem<HS>;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long bars[2 * PSLOTS + 10];
    __shared__ uint32_t tmem_slot;
    const uint32_t sb = smem_u32(smem), ring = sb + L::RING;
    const uint32_t kv_full = smem_u32(bars), kv_empty = kv_full + 8 * PSLOTS, q_full = kv_empty + 8 * PSLOTS, s_full = q_full + 16, p_full = s_full + 16, o_full = p_full + 16,
                   o_free = o_full + 16, all_done = o_free + 8;
    const Cache& c = A.c;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, hs = c.hs;
    if (tid == 0) {
        for (int i = 0; i < PSLOTS; i++) {
            mbar_init(kv_full + 8 * i, 2);   // the two warps that fill a tile
            mbar_init(kv_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(q_full + 8 * i, 4);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4);
            mbar_init(o_full + 8 * i, 1);
        }
        mbar_init(o_free, 4);
        mbar_init(all_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = tmem_slot, out_cols = tmem + 3 * 128;
    const Start s = load_start(c.plan, A.starts_at, blockIdx.x);  // (there before any kernel of its step starts)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    unsigned int limit = A.wait_limit;
    auto wait = [&](uint32_t bar, uint32_t parity) { return bounded_wait<false, true, ERR_PAGED>(bar, parity & 1, limit, A.err_flag); };

    if (warp < 4) {
        // ---- keys (warps 0, 1) and values (2, 3): tiles 0, 2, .. and 1, 3, .. of the ring's sequence ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        const bool value = warp >= 2;
        const char* base = value ? c.values : c.keys;
        const int r0 = 64 * (warp & 1);
        constexpr int CH = HS / 8, STEP = 32 / CH;  // 16-byte pieces of a row, rows a pass of the warp covers
        const int ch = lane % CH, rl = lane / CH, chunks = hs / 8;
        int tile = value;  // of the sequence keys 0, values 0, keys 1, ..
        for_parts(s, c, [&](const Tile& t, int head, const Part& p) {
            const int hi = t.pos0 + (t.first + t.rows - 1) / c.group + 1;
            auto place = [&](int j, int i) -> long long {  // of position 32 i + lane of this warp's 64, -1 behind the last
                const int at = (p.unit + j) * PU + r0 + 32 * i + lane;
                return at < hi ? 2 * place_of(c, t.table, at, head) : -1;
            };
            long long a0 = place(0, 0), a1 = place(0, 1);
            for (int j = 0; j < p.n; j++, tile += 2) {
                const int slot = tile % PSLOTS, round = tile / PSLOTS;
                if (round > 0) wait(kv_empty + 8 * slot, round - 1);
                if (!__any_sync(0xffffffffu, limit == 0)) {
                    const uint32_t dst = ring + slot * L::TILE;
#pragma unroll 8
                    for (int k = 0; k < 64 / STEP; k++) {
                        const int r = STEP * k + rl;  // of the warp's 64
                        const long long a = __shfl_sync(0xffffffffu, k < 32 / STEP ? a0 : a1, r & 31);
                        const int row = r0 + r;
                        const uint32_t off = (ch >> 3) * L::BLOCK + row * 128 + (((ch & 7) ^ (row & 7)) << 4), bytes = a >= 0 && ch < chunks ? 16u : 0u;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + off), "l"(__cvta_generic_to_global(base + (bytes ? a + 16 * ch : 0))), "r"(bytes) : "memory");
                    }
                    if (j + 1 < p.n) {
                        a0 = place(j + 1, 0);
                        a1 = place(j + 1, 1);
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    fence_async();  // before the tensor core's reads
                    __syncwarp();
                    if (lane == 0) mbar_arrive(kv_full + 8 * slot);
                }
            }
        });
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 12) {
            // ---- products ----
            const uint32_t id_qk = idesc(128, false), id_pv = idesc(HS, true);
            uint32_t n_q[2] = {0, 0}, n_s[2] = {0, 0}, n_pv = 0, qk = 0;  // phases: queries, scores of each half; outputs; scores of both
            uint32_t tile = 0;  // of the ring's sequence, at the part's first
            for_parts(s, c, [&](const Tile&, int, const Part& p) {
                const int n[2] = {p.na, p.nb};
                uint32_t first_s[2] = {n_s[0], n_s[1]};
                auto kv_wait = [&](uint32_t i) { wait(kv_full + 8 * (i % PSLOTS), i / PSLOTS); };
                auto region = [&](uint32_t k) { return tmem + 128 * (k % 3); };
                const uint32_t qk0 = qk;
                auto place_of_s = [&](int h, int j) { return qk0 + j + (h == 0 ? min(j, p.nb) : min(j + 1, p.na)); };  // number of half h's j-th QK
                auto do_qk = [&](int h, int j) {
                    if (j == 0) {
                        wait(q_full + 8 * h, n_q[h]);
                        n_q[h]++;
                    }
                    const uint32_t kt = tile + 2 * j;
                    kv_wait(kt);
                    tc_after();
                    __syncwarp();
                    if (elect_one() && limit) {
                        const uint32_t d = region(place_of_s(h, j)), q = sb + h * 2 * L::Q, b = ring + (kt % PSLOTS) * L::TILE;
#pragma unroll
                        for (int w = 1; w >= 0; w--)  // the low parts first
#pragma unroll
                            for (int k = 0; k < HS / 16; k++)
                                umma_ss(d, desc_k(q + w * L::Q + (k / 4) * L::BLOCK + 32 * (k % 4)), desc_k(b + (k / 4) * L::BLOCK + 32 * (k % 4)), id_qk, w == 0 || k > 0);
                        umma_commit(s_full + 8 * h);
                        if (h == 1 || j >= p.nb) umma_commit(kv_empty + 8 * (kt % PSLOTS));
                    }
                    __syncwarp();
                    qk++;
                };
                auto do_pv = [&](int h, int j) {
                    const uint32_t vt = tile + 2 * j + 1;
                    wait(p_full + 8 * h, first_s[h] + j);
                    kv_wait(vt);
                    if (n_pv > 0) wait(o_free, n_pv - 1);
                    tc_after();
                    __syncwarp();
                    if (elect_one() && limit) {
                        const uint32_t a = region(place_of_s(h, j)), b = ring + (vt % PSLOTS) * L::TILE;
#pragma unroll
                        for (int w = 1; w >= 0; w--)
#pragma unroll
                            for (int k = 0; k < PU / 16; k++)
                                umma_ts(out_cols, a + 32 * (k / 2) + 16 * w + 8 * (k % 2), desc_mn(b + 2048 * k, L::BLOCK), id_pv, w == 0 || k > 0);
                        umma_commit(o_full + 8 * h);
                        if (h == 1 || j >= p.nb) umma_commit(kv_empty + 8 * (vt % PSLOTS));
                    }
                    __syncwarp();
                    n_s[h]++;
                    n_pv++;
                };
                for (int j = 0; j <= p.n; j++) {
                    if (j < n[0]) do_qk(0, j);
                    if (j > 0 && j - 1 < n[1]) do_pv(1, j - 1);
                    if (j < n[1]) do_qk(1, j);
                    if (j < n[0]) do_pv(0, j);
                }
                tile += 2 * p.n;
            });
            if (elect_one()) umma_commit(all_done);  // no product is under way when the block ends
            limit = LAST_POLLS;
            wait(all_done, 0);
            __syncwarp();
        }
    } else {
        // ---- softmax: a row a thread ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int h = warp >= 8, q4 = warp & 3, r = 32 * q4 + lane;
        const uint32_t lanes = (uint32_t)(32 * q4) << 16, mine = sb + h * 2 * L::Q;
        unsigned char* mine_p = smem + h * 2 * L::Q;
        uint32_t n_s = 0, qk = 0;
        for_parts(s, c, [&](const Tile& t, int head, const Part& p) {
            const int n = h ? p.nb : p.na, rows = h ? p.rb : p.ra, row_first = t.first + PR * h;
            float acc[HS];
#pragma unroll
            for (int d = 0; d < HS; d++) acc[d] = 0.f;
            float m = -INFINITY, l = 0.f, cexp = 0.f;
            const int vis = r < rows ? t.pos0 + (row_first + r) / c.group : -1;
            if (n > 0) {
                // queries: a warp brings one row after the other, 4 elements a lane
#pragma unroll 4
                for (int i = 0; i < 32; i++) {
                    const int rr = 32 * q4 + i, pr = row_first + rr, tok = pr / c.group;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (rr < rows && 4 * lane < hs) {
                        const float* q = A.q + (t.row0 + tok) * A.q_ld + (long long)(head * c.group + pr % c.group) * hs + 4 * lane;
                        if (A.qvec) v = __ldcg(reinterpret_cast<const float4*>(q));
                        else v = make_float4(__ldcg(q), __ldcg(q + 1), __ldcg(q + 2), __ldcg(q + 3));
                    }
                    v.x *= A.scale; v.y *= A.scale; v.z *= A.scale; v.w *= A.scale;
                    float mx = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    float unit;
                    const float up = power_up(mx, unit);
                    if (lane == i) cexp = unit * LOG2E;
                    uint2 hi, lo;
                    split2(v.x * up, v.y * up, hi.x, lo.x);
                    split2(v.z * up, v.w * up, hi.y, lo.y);
                    if (4 * lane < HS) {
                        const int ch = (lane % 16) / 2, off = (lane / 16) * L::BLOCK + rr * 128 + ((ch ^ (rr & 7)) << 4) + 8 * (lane & 1);
                        *reinterpret_cast<uint2*>(mine_p + off) = hi;
                        *reinterpret_cast<uint2*>(mine_p + L::Q + off) = lo;
                    }
                }
                fence_async();
                __syncwarp();
                if (lane == 0 && limit) mbar_arrive(q_full + 8 * h);
            }
            for (int j = 0; j < n; j++) {
                const uint32_t reg = tmem + 128 * ((qk + j + (h == 0 ? min(j, p.nb) : min(j + 1, p.na))) % 3) + lanes;
                const int p0 = (p.unit + j) * PU;
                wait(s_full + 8 * h, n_s);
                __syncwarp();
                tc_after();
                const bool all_seen = __all_sync(0xffffffffu, vis >= p0 + PU - 1);
                float mx = -INFINITY;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t x[32];
                    tmem_ld32(reg + 32 * k, x);
                    tmem_wait_ld();
                    if (all_seen) {
#pragma unroll
                        for (int i = 0; i < 32; i++) mx = fmaxf(mx, __uint_as_float(x[i]));
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i++) mx = fmaxf(mx, p0 + 32 * k + i <= vis ? __uint_as_float(x[i]) : -INFINITY);
                    }
                }
                const float m_new = fmaxf(m, mx * cexp), base = m_new == -INFINITY ? 0.f : m_new, resc = ex2(m - base);
                m = m_new;
                const float shift = 4.f - base;  // log2(WEIGHT)
                float ps[4] = {};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t x[32], y[32];
                    tmem_ld32(reg + 32 * k, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float e0 = ex2(fmaf(__uint_as_float(x[i]), cexp, shift)), e1 = ex2(fmaf(__uint_as_float(x[i + 1]), cexp, shift));
                        if (!all_seen) {
                            e0 = p0 + 32 * k + i <= vis ? e0 : 0.f;
                            e1 = p0 + 32 * k + i + 1 <= vis ? e1 : 0.f;
                        }
                        ps[(i >> 1) & 3] += e0 + e1;
                        const int at = (i >> 4) * 8 + ((i & 15) >> 1);  // 16 positions: 8 columns of high parts; 16 further on the low ones
                        split2(e0, e1, y[at], y[16 + at]);
                    }
                    tmem_st32(reg + 32 * k, y);
                }
                l = l * resc + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
                tmem_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0 && limit) mbar_arrive(p_full + 8 * h);
                wait(o_full + 8 * h, n_s);
                __syncwarp();
                tc_after();
#pragma unroll
                for (int k = 0; k < HS / 32; k++) {
                    uint32_t x[32];
                    tmem_ld32(out_cols + lanes + 32 * k, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i++) acc[32 * k + i] = fmaf(acc[32 * k + i], resc, __uint_as_float(x[i]));
                }
                tc_before();
                __syncwarp();
                if (lane == 0 && limit) mbar_arrive(o_free);
                n_s++;
            }
            qk += p.na + p.nb;
            // ---- results: through shared memory (the queries' place), so that a row leaves in one piece ----
            const float f = p.whole ? 1.f / l : 1.f / WEIGHT;
            float sum = l;
#pragma unroll
            for (int d = 0; d < HS; d++) sum += acc[d];
            const unsigned int bad = __ballot_sync(0xffffffffu, r < rows && !(fabsf(sum) < INFINITY));
            float4* so = reinterpret_cast<float4*>(mine_p) + r * (HS / 4);
            __syncwarp();
#pragma unroll
            for (int d = 0; d < HS / 4; d++) so[d ^ (lane & (HS / 4 - 1))] = make_float4(acc[4 * d] * f, acc[4 * d + 1] * f, acc[4 * d + 2] * f, acc[4 * d + 3] * f);
            __syncwarp();
            const size_t slot = ((size_t)s.me * 2 + (p.unit == 0)) * A.tile_rows + PR * h;
            if (!p.whole && r < rows) *reinterpret_cast<float2*>(A.part_ml + (slot + r) * 2) = make_float2(m, l / WEIGHT);
            for (int i = 0; i < 32 && 32 * q4 + i < rows; i++) {
                const int rr = 32 * q4 + i, pr = row_first + rr, tok = pr / c.group;
                float* o = p.whole ? A.out + (t.row0 + tok) * A.out_ld + (long long)(head * c.group + pr % c.group) * hs : A.part + (slot + rr) * hs;
                if (bad >> i & 1) {
                    row_again<__half>(A, t, head, PR * h + rr, p.unit * PU, (p.unit + p.n) * PU, o, p.whole ? nullptr : A.part_ml + (slot + rr) * 2);
                } else if (4 * lane < hs) {
                    const float4 v = reinterpret_cast<const float4*>(mine_p)[rr * (HS / 4) + (lane ^ (i & (HS / 4 - 1)))];
                    if (!p.whole || A.qvec) {
                        *reinterpret_cast<float4*>(o + 4 * lane) = v;
                    } else {
                        o[4 * lane] = v.x; o[4 * lane + 1] = v.y; o[4 * lane + 2] = v.z; o[4 * lane + 3] = v.w;
                    }
                }
            }
            if (h) asm volatile("bar.sync 2, 128;" ::: "memory");  // the next queries lie across the four warps' results
            else asm volatile("bar.sync 1, 128;" ::: "memory");
        });
    }
    __syncwarp();
    tc_before();
    __syncthreads();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <int HS>
int launch(slai_ctx* ctx, const AttnArgs& A, int blocks, bool pdl) {
    auto kern = paged_attn_prompt_kernel<HS>;
    constexpr int bytes = Smem<HS>::TOTAL + 1024;
    static PerDeviceOnce attr;
    if (attr.need(ctx->device)) {
        SLAI_CHECK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        attr.set(ctx->device);
    }
    return launch_dependent(ctx, kern, dim3((unsigned)blocks), PT, bytes, pdl, A);
}

}  // namespace

Lane paged_prompt_lane(int sms) {
    Lane l;
    l.rows = 2 * PR;
    l.unit = PU;
    l.blocks = sms;
    l.least = 1;
    return l;
}

int paged_prompt_launch(slai_ctx* ctx, const AttnArgs& A, int blocks, bool pdl) {
    return A.c.hs <= 64 ? launch<64>(ctx, A, blocks, pdl) : launch<128>(ctx, A, blocks, pdl);
}
