// Paged attention for many rows and f16 caches: chunks of prompts, on the 5th-generation tensor cores.
//
// A tile is 256 rows (token, query head of the group), two halves A and B of 128 that share the keys and values: scores S = Q K^T of 128 x 128 positions and
// sums P V of them are products of tcgen05.mma with their f32 results in tensor memory, where a lane has a row.  Queries and weights are pairs of halves
// (22 bits), two products each: one rounding of either to f16 would put 1e-4 into the result, the pairs leave 5e-7 (1e-6 behind 7000 positions; f32 arithmetic 2e-6).
// A row of queries is carried times a power of two that puts its largest element below 2^15: elements down to 2^-17 of that keep their 22 bits, smaller ones are
// off by up to 2^-40 of the largest.  The tensor core truncates when it adds: both sums end with their 128 positions, and a half's output goes on in its
// threads' registers, times the factor by which the running maximum moved.
//
//   warp 0       issues the products: QK_A(j), PV_B(j-1), QK_B(j), PV_A(j): while one half's threads are at its softmax the tensor cores are at the other's
//                products.  Three regions of 128 columns of tensor memory hold scores and weights in turn, one the outputs.
//   warps 1-3    keys and values of 128 positions, in turn, into a tile of shared memory each: by TMA, a box per page, where pages divide 128 positions or are
//                divided by them, else (and where a sequence ends inside the tile: positions behind the last are zeros, whatever the page holds there) by
//                asynchronous 16-byte copies that write the swizzle themselves.  (All by the latter: 522 us instead of 494.)
//   warps 4-11   half A, warps 12-19 half B: softmax, two threads a row, 64 positions and then 64 dimensions each: S out of tensor memory once for its maximum and once
//                more for the weights, which take its columns' place as the next product's operand; then the product's result.
// Steps that are sooner done in tiles of 128 rows have half A alone (Lane::low): QK_A(j + 1) goes before PV_A(j), and a unit takes 2.6 us instead of 3.4.
// A region is written again by the third QK after its own; by then the PV that read it is complete: before each PV its issuer waits until the output of the PV
// before has been read (one region for all of them), so that only the last PV issued can be under way.
//
// What bounds it: 1023 tokens of 64 heads on 8 behind 7001 positions, 440 us, 572 TFLOP/s, 1140 executed; the kernel itself 388 us, 1300 executed, where the card's
// power allows 1400 (the clock falls to 1.55 GHz).  A unit of 128 positions takes 5400 cycles for products of 4096: a half's softmax (maximum 500, weights
// 2000: 16 exponentials a cycle and SM, the wait for tensor memory), its product, the read of that and the next scores are one chain, longer than the other half's
// products.  Few tokens: 511 of 32 heads 21 us in tiles of 128 rows, of which the queries' way to shared memory takes 5, the results' 3 (in tiles of 256: 24.1).  Registers are
// short: 180 bytes of spills stored, 404 loaded (heads up to 64: 116 and 180).
// Descriptors in uniform registers: 464 -> 445 us.  Tried and taken back: a row a thread with twice the registers (chunk 453 us, but 139 for 96 us with 2047 tokens of 32 heads); half of the exponentials by a
// polynomial (547 for 497); queries by eight lanes a row, in a function of their own or not (the softmax's registers came out worse: 480 to 580).
//
// Every wait is bounded (common.cuh, bounded_wait).
#include <type_traits>

#include <cuda.h>

#include "paged_order.h"
#include "paged_tc.cuh"

using namespace paged;

namespace {

constexpr int PT = 640, PR = 128, PU = 128, PSLOTS = 3;  // threads, rows of a half, positions of a unit, tiles of keys or values in shared memory
constexpr float WEIGHT = 16.f;  // weights are carried 16 times their size: their low parts keep their bits, and the exponent's rounding stays below 2^-23

// ---- PTX wrappers ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mbar_expect_tx(uint32_t a, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(a), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t mbar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(mbar), "r"(x),
                 "r"(y), "r"(z), "r"(w)
                 : "memory");
}
// Values: rows along the product's inner dimension (row = position), `blocks` bytes apart in the other direction: 64 dimensions to a row.
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
// ---- shared memory -------------------------------------------------------------------------------------------------------
// Queries [half][high, low][64 dimensions][128 rows][128 bytes], then the ring [slot][64 dimensions][128 positions][128 bytes].
template <int HS>
struct Smem {
    static constexpr int BLOCK = 128 * 128, BLOCKS = HS / 64, Q = BLOCKS * BLOCK, TILE = BLOCKS * BLOCK;
    struct Rest {
        unsigned long long bars[2 * PSLOTS + 12];
        float max_s[4 * PR];  // what the two threads of a row tell one another
        unsigned int bad_s[2][2][4];
        uint32_t tmem_slot;
    };
    static constexpr int RING = 4 * Q, REST = RING + PSLOTS * TILE, TOTAL = REST + (int)sizeof(Rest);
    static_assert(TOTAL <= 227 * 1024, "a block's shared memory");
};

// A block's part of one (tile, head) pair.
struct Part {
    int unit, n;      // units [unit, unit + n)
    int na, nb;       // of these, the ones that the halves' rows see
    int ra, rb;       // rows of the halves
    bool whole;
};
__device__ __forceinline__ Part part_of(const Tile& t, int unit, int left, const Div& group) {
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
__global__ void __launch_bounds__(PT, 1) paged_attn_prompt_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ CUtensorMap map_k,
                                                                  const __grid_constant__ CUtensorMap map_v, const int box) {
    using L = Smem<HS>;
    extern __shared__ __align__(1024) unsigned char smem_dyn[];  // (the kernel has no other shared memory: the operands begin on the swizzle's boundary)
    unsigned char* smem = smem_dyn;
    typename L::Rest& rest = *reinterpret_cast<typename L::Rest*>(smem + L::REST);
    unsigned long long* bars = rest.bars;
    uint32_t& tmem_slot = rest.tmem_slot;
    float* max_s = rest.max_s;
    auto& bad_s = rest.bad_s;
    if (smem_u32(smem) & 1023) {
        if (threadIdx.x == 0) atomicExch(A.err_flag, (unsigned int)ERR_PAGED);
        return;
    }
    if (A.recorded && __ldcg(A.c.plan + A.starts_at + (int)(sizeof(Start) / 4) * blockIdx.x + 3) <= 0) {  // (count) there is room for more blocks than the step has
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const uint32_t sb = smem_u32(smem), ring = sb + L::RING;
    const uint32_t kv_full = smem_u32(bars), kv_empty = kv_full + 8 * PSLOTS, q_full = kv_empty + 8 * PSLOTS, s_full = q_full + 16, p_full = s_full + 32, o_full = p_full + 16,
                   o_free = o_full + 16, all_done = o_free + 8;
    const Cache& c = A.c;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, hs = c.hs;
    if (tid == 0) {
        for (int i = 0; i < PSLOTS; i++) {
            mbar_init(kv_full + 8 * i, 1);
            mbar_init(kv_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(q_full + 8 * i, 8);
            mbar_init(s_full + 16 * i, 1);
            mbar_init(s_full + 16 * i + 8, 1);
            mbar_init(p_full + 8 * i, 8);
            mbar_init(o_full + 8 * i, 1);
        }
        mbar_init(o_free, 8);
        mbar_init(all_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = uniform(tmem_slot), out_cols = tmem + 3 * 128;
    const Start s = load_start(c.plan, A.starts_at, blockIdx.x);  // (there before any kernel of its step starts)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    unsigned int limit = A.wait_limit;
    auto wait = [&](uint32_t bar, uint32_t parity) { return bounded_wait<false, true, ERR_PAGED>(bar, parity & 1, limit, A.err_flag); };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp > 0) {
            // ---- keys and values: tile i of the sequence keys 0, values 0, keys 1, .. is warp i % 3 + 1's, in its slot ----
            const int slot = warp - 1;
            constexpr int CH = HS / 8, STEP = 32 / CH;  // 16-byte pieces of a row, rows a pass of the warp covers
            const int ch = lane % CH, rl = lane / CH, chunks = hs / 8;
            const uint32_t dst0 = ring + slot * L::TILE + (ch >> 3) * L::BLOCK;
            int next = slot, base = 0;  // number of this warp's next tile, of the part's first
            SlotFills fills;
            auto give_up = [&]() { return !fills.may_fill([&](uint32_t i) { return wait(kv_empty + 8 * slot, i), !__any_sync(0xffffffffu, limit == 0); }); };
            for_parts(s, c, [&](const Tile& t, int head, const Part& p) {
                const int hi = t.pos0 + (t.first + t.rows - 1) / c.group + 1;
                for (; next < base + 2 * p.n; next += PSLOTS) {
                    const int j = (next - base) >> 1, p0 = (p.unit + j) * PU;
                    const char* from = (next - base) & 1 ? c.values : c.keys;
                    if (box > 0 && p0 + PU <= hi) {
                        // a page is a box of `box` rows and 64 dimensions; lane i has the number of the tile's i-th
                        const int i_page = p0 / c.page_size, boxes = PU / box;
                        const int id = lane < boxes ? __ldcg(c.plan + t.table + i_page + (lane * box) / c.page_size) : 0;
                        if (give_up()) continue;
                        fills.filled();
                        if (elect_one()) mbar_expect_tx(kv_full + 8 * slot, L::TILE);
                        __syncwarp();
                        for (int i = 0; i < boxes; i++) {
                            const int page = __shfl_sync(0xffffffffu, id, i);
                            if (elect_one()) {
#pragma unroll
                                for (int d = 0; d < L::BLOCKS; d++)
                                    tma_load_4d(ring + slot * L::TILE + d * L::BLOCK + i * box * 128, (next - base) & 1 ? &map_v : &map_k, 64 * d, (p0 + i * box) % c.page_size, head, page,
                                                kv_full + 8 * slot);
                            }
                            __syncwarp();
                        }
                        continue;
                    }
                    long long at[4];  // places of positions 32 i + lane, -1 behind the last
#pragma unroll
                    for (int i = 0; i < 4; i++) at[i] = p0 + 32 * i + lane < hi ? 2 * place_of(c, t.table, p0 + 32 * i + lane, head) : -1;
                    if (give_up()) continue;
                    fills.filled();
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll 4
                        for (int k = 0; k < 32 / STEP; k++) {
                            const int r = STEP * k + rl, row = 32 * i + r;
                            const long long a = __shfl_sync(0xffffffffu, at[i], r);
                            const uint32_t off = row * 128 + (((ch & 7) ^ (row & 7)) << 4), bytes = a >= 0 && ch < chunks ? 16u : 0u;
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst0 + off), "l"(__cvta_generic_to_global(from + (bytes ? a + 16 * ch : 0))), "r"(bytes) : "memory");
                        }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    fence_async();  // before the tensor core's reads
                    __syncwarp();
                    if (lane == 0) mbar_arrive(kv_full + 8 * slot);
                }
                base += 2 * p.n;
            });
            asm volatile("cp.async.wait_all;" ::: "memory");
            limit = LAST_POLLS;
            fills.settle([&](uint32_t i) { wait(kv_full + 8 * slot, i); });  // the last copy lands before the block ends
        } else {
            // ---- products ----
            const uint32_t id_qk = idesc(128, false), id_pv = idesc(HS, true);
            uint32_t n_q[2] = {0, 0}, n_qk[2] = {0, 0}, n_s[2] = {0, 0}, n_pv = 0, qk = 0;  // phases: queries, scores, weights of each half; outputs; scores of both
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
                    const uint32_t slot = uniform(kt % PSLOTS), d = uniform(region(place_of_s(h, j)));
                    tc_after();
                    __syncwarp();
                    if (elect_one() && limit) {
                        const uint64_t queries = desc_k(sb + h * 2 * L::Q), keys = desc_k(ring + slot * L::TILE);
#pragma unroll
                        for (int w = 1; w >= 0; w--)  // the low parts first
#pragma unroll
                            for (int k = 0; k < HS / 16; k++)
                                umma_ss(d, queries + (w * L::Q + (k / 4) * L::BLOCK + 32 * (k % 4)) / 16, keys + ((k / 4) * L::BLOCK + 32 * (k % 4)) / 16, id_qk, w == 0 || k > 0);
                        umma_commit(s_full + 16 * h + 8 * (n_qk[h] & 1));
                        if (h == 1 || j >= p.nb) umma_commit(kv_empty + 8 * (kt % PSLOTS));
                    }
                    __syncwarp();
                    n_qk[h]++;
                    qk++;
                };
                auto do_pv = [&](int h, int j) {
                    const uint32_t vt = tile + 2 * j + 1;
                    wait(p_full + 8 * h, first_s[h] + j);
                    kv_wait(vt);
                    if (n_pv > 0) wait(o_free, n_pv - 1);
                    const uint32_t slot = uniform(vt % PSLOTS), a = uniform(region(place_of_s(h, j)));
                    tc_after();
                    __syncwarp();
                    if (elect_one() && limit) {
                        const uint64_t values = desc_mn(ring + slot * L::TILE, L::BLOCK);
#pragma unroll
                        for (int w = 1; w >= 0; w--)
#pragma unroll
                            for (int k = 0; k < PU / 16; k++)
                                umma_ts(out_cols, a + 16 * k + 8 * w, values + 2048 * k / 16, id_pv, w == 0 || k > 0);
                        umma_commit(o_full + 8 * h);
                        if (h == 1 || j >= p.nb) umma_commit(kv_empty + 8 * (vt % PSLOTS));
                    }
                    __syncwarp();
                    n_s[h]++;
                    n_pv++;
                };
                if (n[1] == 0) {  // half A alone: the next scores come before the product that waits for this one's weights
                    do_qk(0, 0);
                    for (int j = 0; j < n[0]; j++) {
                        if (j + 1 < n[0]) do_qk(0, j + 1);
                        do_pv(0, j);
                    }
                }
                for (int j = 0; j <= p.n && n[1] > 0; j++) {
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
        // ---- softmax: two threads a row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const int h = warp >= 12, q4 = warp & 3, g = (warp - 4) >> 2 & 1, r = 32 * q4 + lane, pair = 1 + 4 * h + q4;  // pair: the barrier of a quarter's two warps
        constexpr int DH = HS / 2;  // dimensions a thread
        const uint32_t lanes = (uint32_t)(32 * q4) << 16;
        unsigned char* mine = smem + h * 2 * L::Q;
        float* other = max_s + (2 * h + (g ^ 1)) * PR + r;
        float* own = max_s + (2 * h + g) * PR + r;
        auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory"); };
        uint32_t n_s = 0, qk = 0;
        for_parts(s, c, [&](const Tile& t, int head, const Part& p) {
            const int n = h ? p.nb : p.na, rows = h ? p.rb : p.ra, row_first = t.first + PR * h;
            const int pr = row_first + min(r, rows - 1), tok = pr / c.group, vis = r < rows ? t.pos0 + tok : 0x7fffffff;  // last position the row sees (rows behind the last: all, so that they need no mask)
            const long long col = (long long)(head * c.group + pr % c.group) * hs;
            float cexp = 0.f;
            if (n > 0) {
                // queries: a warp brings 16 rows, 4 elements a lane, all on their way at once
                const long long q_at = (t.row0 + tok) * A.q_ld + col;
                float4 v[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int rl = 16 * g + i;
                    const float* q = A.q + __shfl_sync(0xffffffffu, q_at, rl) + 4 * lane;
                    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (32 * q4 + rl < rows && 4 * lane < hs) {
                        if (A.qvec) v[i] = __ldcg(reinterpret_cast<const float4*>(q));
                        else v[i] = make_float4(__ldcg(q), __ldcg(q + 1), __ldcg(q + 2), __ldcg(q + 3));
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int rl = 16 * g + i, rr = 32 * q4 + rl;
                    v[i].x *= A.scale; v[i].y *= A.scale; v[i].z *= A.scale; v[i].w *= A.scale;
                    float mx = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    float unit;
                    const float up = power_up(mx, unit);
                    if (lane == rl) cexp = unit * LOG2E;
                    uint2 hi, lo;
                    split2(v[i].x * up, v[i].y * up, hi.x, lo.x);
                    split2(v[i].z * up, v[i].w * up, hi.y, lo.y);
                    if (4 * lane < HS) {
                        const int ch = (lane % 16) / 2, off = (lane / 16) * L::BLOCK + rr * 128 + ((ch ^ (rr & 7)) << 4) + 8 * (lane & 1);
                        *reinterpret_cast<uint2*>(mine + off) = hi;
                        *reinterpret_cast<uint2*>(mine + L::Q + off) = lo;
                    }
                }
                fence_async();
                if (lane >> 4 == g) {  // the rows' units to both of their threads
                    *own = cexp;
                    *other = cexp;
                }
                meet();
                cexp = *own;
                if (lane == 0 && limit) mbar_arrive(q_full + 8 * h);
            }
            f32x2 acc[DH / 2];
#pragma unroll
            for (int d = 0; d < DH / 2; d++) acc[d] = 0;
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < n; j++) {
                const uint32_t reg = tmem + 128 * ((qk + j + (h == 0 ? min(j, p.nb) : min(j + 1, p.na))) % 3) + lanes + 64 * g;
                const int p0 = (p.unit + j) * PU + 64 * g;
                wait(s_full + 16 * h + 8 * (n_s & 1), n_s >> 1);
                __syncwarp();
                tc_after();
                float resc;
                auto weights = [&](auto all_seen) {
                    constexpr bool ALL = decltype(all_seen)::value;
                    const int seen = vis - p0;  // positions 0 .. seen of this thread's 64
                    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        uint32_t x[2][16];
                        tmem_ld16(reg + 32 * k, x[0]);
                        tmem_ld16(reg + 32 * k + 16, x[1]);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float a = __uint_as_float(x[i >> 4][i & 15]), b = __uint_as_float(x[i >> 4][(i & 15) + 1]);
                            mx[(i >> 1) & 1] = max3(mx[(i >> 1) & 1], ALL || 32 * k + i <= seen ? a : -INFINITY, ALL || 32 * k + i + 1 <= seen ? b : -INFINITY);
                        }
                    }
                    *own = fmaxf(mx[0], mx[1]);
                    meet();
                    const float m_new = fmaxf(m, fmaxf(*own, *other) * cexp), base = m_new == -INFINITY ? 0.f : m_new;
                    resc = ex2(m - base);
                    m = m_new;
                    const f32x2 shift = pack2(4.f - base, 4.f - base), slope = pack2(cexp, cexp);  // log2(WEIGHT)
                    f32x2 ps[2] = {0, 0};
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        uint32_t x[16];
                        tmem_ld16(reg + 16 * k, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            uint32_t hi[4], lo[4];  // of 16 positions: 8 columns of high parts, 8 of low ones
#pragma unroll
                            for (int i = 0; i < 8; i += 2) {
                                const float2 e = unpack2(fma2(pack2(x[8 * u + i], x[8 * u + i + 1]), slope, shift));
                                const int at = 16 * k + 8 * u + i;
                                const float a = ALL || at <= seen ? ex2(e.x) : 0.f, b = ALL || at + 1 <= seen ? ex2(e.y) : 0.f;
                                ps[(i >> 1) & 1] = add2(ps[(i >> 1) & 1], pack2(a, b));
                                // the high part: the upper 11 bits, exactly an f16; the low part: the rest, rounded to one
                                const float ah = __uint_as_float(__float_as_uint(a) & 0xFFFFE000u), bh = __uint_as_float(__float_as_uint(b) & 0xFFFFE000u);
                                const __half2 hh = __floats2half2_rn(ah, bh), ll = __floats2half2_rn(a - ah, b - bh);
                                hi[i >> 1] = *reinterpret_cast<const uint32_t*>(&hh);
                                lo[i >> 1] = *reinterpret_cast<const uint32_t*>(&ll);
                            }
                            tmem_st4(reg + 16 * k + 4 * u, hi);
                            tmem_st4(reg + 16 * k + 8 + 4 * u, lo);
                        }
                    }
                    const float2 sum = unpack2(add2(ps[0], ps[1]));
                    l = l * resc + (sum.x + sum.y);  // (this thread's positions)
                };
                if (__all_sync(0xffffffffu, vis >= p0 + 63)) weights(std::true_type());
                else weights(std::false_type());
                tmem_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0 && limit) mbar_arrive(p_full + 8 * h);
                wait(o_full + 8 * h, n_s);
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
                    for (int i = 0; i < 16; i++) acc[16 * k + i] = fma2(acc[16 * k + i], by, pack2(o[i >> 3][2 * i & 15], o[i >> 3][(2 * i & 15) + 1]));
                }
                tc_before();
                __syncwarp();
                if (lane == 0 && limit) mbar_arrive(o_free);
                n_s++;
            }
            qk += p.na + p.nb;
            // ---- results: through shared memory (the queries' place), so that a row leaves in one piece ----
            meet();  // (both have read the last maxima)
            *own = l;
            meet();
            l += *other;
            float sum = l;
#pragma unroll
            for (int d = 0; d < DH / 2; d++) {
                const float2 v = unpack2(acc[d]);
                sum += v.x + v.y;
            }
            const unsigned int bad = __ballot_sync(0xffffffffu, r < rows && !(fabsf(sum) < INFINITY));
            const float f = p.whole ? 1.f / l : 1.f / WEIGHT;
            float4* so = reinterpret_cast<float4*>(mine) + r * (HS / 4);
#pragma unroll
            for (int d = 0; d < DH / 4; d++) {
                const float2 v = unpack2(acc[2 * d]), w = unpack2(acc[2 * d + 1]);
                so[(DH / 4 * g + d) ^ (lane & (HS / 4 - 1))] = make_float4(v.x * f, v.y * f, w.x * f, w.y * f);
            }
            if (lane == 0) bad_s[h][g][q4] = bad;
            const size_t slot = ((size_t)s.me * 2 + (p.unit == 0)) * A.tile_rows + PR * h;
            if (!p.whole && g == 0 && r < rows) *reinterpret_cast<float2*>(A.part_ml + (slot + r) * 2) = make_float2(m, l / WEIGHT);
            meet();
            float* o_at = p.whole ? A.out + (t.row0 + tok) * A.out_ld + col : A.part + (slot + min(r, rows - 1)) * hs;
            const bool vec = !p.whole || A.qvec;
#pragma unroll 8
            for (int i = 0; i < 16; i++) {
                const int rl = 16 * g + i, rr = 32 * q4 + rl;
                float* o = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o_at), rl)) + 4 * lane;
                if (rr < rows && 4 * lane < hs) {
                    const float4 v = reinterpret_cast<const float4*>(mine)[rr * (HS / 4) + (lane ^ (rl & (HS / 4 - 1)))];
                    if (vec) {
                        *reinterpret_cast<float4*>(o) = v;
                    } else {
                        o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
                    }
                }
            }
            const unsigned int again = bad_s[h][0][q4] | bad_s[h][1][q4];
            if (again) {
                __syncwarp();
                for (int i = 16 * g; i < 16 * g + 16; i++)
                    if (again >> i & 1) {
                        float* o = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o_at), i));
                        row_again<__half>(A, t, head, PR * h + 32 * q4 + i, p.unit * PU, (p.unit + p.n) * PU, o,
                                          p.whole ? nullptr : A.part_ml + (slot + 32 * q4 + i) * 2);
                    }
            }
            if (h) asm volatile("bar.sync 10, 256;" ::: "memory");  // the next queries lie across the eight warps' results
            else asm volatile("bar.sync 9, 256;" ::: "memory");
        });
    }
    __syncwarp();
    tc_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ---- host side -----------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}
// Pages as [page][head][position][dimension], whatever their order in memory, in boxes of 64 dimensions of `rows` positions.
bool make_map(CUtensorMap* map, const AttnArgs& A, const void* base, int rows) {
    const EncodeTiledFn enc = encode_tiled();
    const Cache& c = A.c;
    const cuuint64_t dims[4] = {(cuuint64_t)c.hs, (cuuint64_t)c.page_size, (cuuint64_t)c.n_kv, (cuuint64_t)A.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.pos_stride * 2, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t boxes[4] = {64, (cuuint32_t)rows, 1, 1}, elem[4] = {1, 1, 1, 1};
    return enc && enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HS>
int launch(slai_ctx* ctx, const AttnArgs& A, int blocks, bool pdl) {
    auto kern = paged_attn_prompt_kernel<HS>;
    constexpr int bytes = Smem<HS>::TOTAL;
    static PerDeviceOnce attr;
    if (attr.need(ctx->device)) {
        SLAI_CHECK_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        attr.set(ctx->device);
    }
    // (a stride that the copy engine does not take, 2^40 bytes and more: by 16-byte copies)
    const int ps = A.c.page_size;
    int box = ps % PU == 0 ? PU : ps >= 8 && PU % ps == 0 ? ps : 0;
    CUtensorMap k = {}, v = {};
    if (box > 0 && !(make_map(&k, A, A.c.keys, box) && make_map(&v, A, A.c.values, box))) box = 0;
    return launch_dependent(ctx, kern, dim3((unsigned)blocks), PT, bytes, pdl, A, k, v, box);
}

}  // namespace

Lane paged_prompt_lane(int sms) {
    Lane l;
    l.rows = 2 * PR;
    // us a call, tiles of 256 / of 128 rows: 32 heads, 256 tokens 17.5 / 14.4, 511 24.1 / 21.0, 1023 38 / 53; 64 heads on 8 behind 2000, 64 tokens
    // 27.5 / 28.4, 511 73 / 109; 8 heads, 1023 tokens 25.2 / 23.5, 2047 38 / 44; 16 heads on 2 behind 1000, 256 tokens 26.2 / 23.7, 1023 45 / 52.  (The better one of each
    // pair is taken but for 64 tokens of 64 heads.)
    l.low = PR;
    l.unit_us[0] = 3.4, l.whole_us[0] = 11, l.cut_us[0] = 25;  // (lines through these and longer ones, as they were before the last steps: all some us longer)
    l.unit_us[1] = 2.6, l.whole_us[1] = 12, l.cut_us[1] = 19;
    l.unit = PU;
    l.blocks = sms;
    l.fixed = 13;
    l.each = 0.0223;
    l.least = 1;
    l.join = 2;  // us a call, cut / not cut where it can be: 32 heads, 511 tokens 27.7 / 24.1, 1023 45 / 38; 64 heads on 8, 511 tokens behind 2000 81 / 73
    return l;
}

int paged_prompt_launch(slai_ctx* ctx, const AttnArgs& A, int blocks, bool pdl) {
    return A.c.hs <= 64 ? launch<64>(ctx, A, blocks, pdl) : launch<128>(ctx, A, blocks, pdl);
}
