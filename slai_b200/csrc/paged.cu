// Paged key / value cache: the handle with a step's plan, and the entry points of its operators (kernels: paged_append.cu, paged_attention.cu,
// paged_prompt.cu, paged_prompt32.cu).
#include <math.h>
#include <string.h>

#include <exception>

#include "paged.cuh"
#include "row_overlap.h"

using namespace paged;

namespace {
// Rows of a cache head that a sequence may bring and surely goes to the kernel for few rows, and may bring and perhaps does.  us of a call, kernel for few / for many:
// one sequence at 300, 32 heads: 64 rows 9.8 / 17.2; at 3000, 32 rows 34 / 34, 64 rows 56 / 35; 64 heads on 8 at 3000, 64 rows 20 / 27, 128 rows 30 / 28; 16
// sequences of 64 heads on 8 at 2000: 16 rows 44 / 54, 32 rows 88 / 55.  (The planner's costs are older than the chunk kernel's last steps: of these it takes the slower
// one for 64 rows of 64 heads on 8 at 3000.)
constexpr int FEW_ROWS = 16, PERHAPS_ROWS = 128;
constexpr int SLOTS = 2;  // pinned copies of a plan: the next step is planned while the last one's copy is on its way

bool capturing(slai_ctx* ctx) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    return cudaStreamIsCapturing(ctx->stream, &st) == cudaSuccess && st != cudaStreamCaptureStatusNone;
}

// base^(-2i / hs) / 2 pi for the pairs of a head, made once per head size and base (64 bits: paged_append.cu)
int turn_table(slai_ctx* ctx, int hs, float base, const double** out) {
    for (auto& t : ctx->turn_tables)
        if (t.head_size == hs && t.base == base) {
            *out = t.d_turns;
            return SLAI_OK;
        }
    SLAI_REQUIRE(ctx, !capturing(ctx), SLAI_ERR_INVALID_ARG,
                 "rotation: the first call with a head size and base makes their table and cannot be recorded; run it once eagerly");
    std::vector<double> h((size_t)std::max(1, hs / 2));
    for (int i = 0; i < hs / 2; i++) h[i] = pow((double)base, -2.0 * i / hs) / (2.0 * M_PI);
    TurnTable t = {hs, base, nullptr};
    SLAI_CHECK_CUDA(ctx, cudaMalloc(&t.d_turns, h.size() * sizeof(double)));
    cudaError_t e = cudaMemcpyAsync(t.d_turns, h.data(), h.size() * sizeof(double), cudaMemcpyHostToDevice, ctx->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) {
        cudaFree(t.d_turns);
        return slai_set_error(ctx, SLAI_ERR_CUDA, "rotation: %s", cudaGetErrorString(e));
    }
    ctx->turn_tables.push_back(t);
    *out = t.d_turns;
    return SLAI_OK;
}
}  // namespace

namespace {
// What the kernels of a handle read and write beside the caller's buffers.  Passes that were recorded with the handle have a share in it.
struct DeviceSide {
    int* plan = nullptr;
    float *part[2] = {}, *ml[2] = {};
    ~DeviceSide() {
        cudaFree(plan);
        for (int k = 0; k < 2; k++) {
            cudaFree(part[k]);
            cudaFree(ml[k]);
        }
    }
};
}  // namespace

struct slai_paged {
    slai_ctx* ctx = nullptr;
    Config cfg = {};
    Planner planner;
    Step step;
    std::shared_ptr<DeviceSide> dev = std::make_shared<DeviceSide>();
    int* h_plan[SLOTS] = {};
    cudaEvent_t copied[SLOTS] = {};
    int slot = 0;
    ~slai_paged() {
        for (int i = 0; i < SLOTS; i++) {
            if (h_plan[i]) cudaFreeHost(h_plan[i]);
            if (copied[i]) cudaEventDestroy(copied[i]);
        }
    }
};

namespace {

int make_handle(slai_ctx* ctx, slai_paged* p) {
    const Config& c = p->cfg;
    const int sms = ctx->sm_count > 0 ? ctx->sm_count : 148;
    const int group = c.n_q_heads / c.n_kv_heads;
    const bool f16 = c.kv_dtype == SLAI_KV_F16, fast = paged_attention_few(c.kv_dtype, c.head_size);
    const Lane few = paged_attention_lane(c.kv_dtype, c.head_size, group, sms);
    const int few_rows = f16 ? FEW_ROWS : std::max(few.rows, 4);
    Lane many;
    if (fast && (long long)c.max_tokens * group > few_rows) many = f16 ? paged_prompt_lane(sms) : paged_prompt32_lane(sms);
    p->planner.init(c, few, many, few_rows, PERHAPS_ROWS);
    const size_t bytes = (size_t)p->planner.lay().total * 4;
    SLAI_CHECK_CUDA(ctx, cudaMalloc(&p->dev->plan, bytes));
    for (int i = 0; i < SLOTS; i++) {
        SLAI_CHECK_CUDA(ctx, cudaMallocHost(&p->h_plan[i], bytes));
        SLAI_CHECK_CUDA(ctx, cudaEventCreateWithFlags(&p->copied[i], cudaEventDisableTiming));
    }
    for (int k = 0; k < 2; k++) {
        const Lane& l = p->planner.lane(k);
        if (l.blocks == 0) continue;
        SLAI_CHECK_CUDA(ctx, cudaMalloc(&p->dev->part[k], sizeof(float) * 2 * l.blocks * l.rows * c.head_size));
        SLAI_CHECK_CUDA(ctx, cudaMalloc(&p->dev->ml[k], sizeof(float) * 2 * l.blocks * l.rows * 2));
    }
    return SLAI_OK;
}

int fill_cache(slai_paged* p, const slai_paged_layer* layer, Cache* out) {
    slai_ctx* ctx = p->ctx;
    const Config& c = p->cfg;
    SLAI_REQUIRE(ctx, p->step.n_rows >= 0, SLAI_ERR_INVALID_ARG, "paged: slai_paged_step comes first");
    SLAI_REQUIRE(ctx, layer->d_keys && layer->d_values, SLAI_ERR_INVALID_ARG, "paged: the layer's pages are missing");
    SLAI_REQUIRE(ctx, layer->page_stride >= c.head_size && layer->head_stride >= c.head_size && layer->pos_stride >= c.head_size, SLAI_ERR_SHAPE,
                 "paged: strides (page %lld, head %lld, position %lld) must be at least head_size=%d", (long long)layer->page_stride,
                 (long long)layer->head_stride, (long long)layer->pos_stride, c.head_size);
    const uintptr_t esz = c.kv_dtype == SLAI_KV_F16 ? 2 : 4;
    SLAI_REQUIRE(ctx, ((uintptr_t)layer->d_keys | (uintptr_t)layer->d_values) % esz == 0, SLAI_ERR_INVALID_ARG, "paged: the pages are not aligned to their type");
    out->plan = p->dev->plan;
    out->count_at = p->planner.lay().count;
    out->rows_at = p->planner.lay().rows;
    out->keys = (char*)layer->d_keys;
    out->values = (char*)layer->d_values;
    out->page_stride = layer->page_stride;
    out->head_stride = layer->head_stride;
    out->pos_stride = layer->pos_stride;
    out->page_size = Div(c.page_size);
    out->n_kv = c.n_kv_heads;
    out->group = Div(c.n_q_heads / c.n_kv_heads);
    out->hs = c.head_size;
    return SLAI_OK;
}

// Checks and leading dimensions common to the two rotations; `packed`: leading dimension that 0 stands for.
int fill_qk(slai_ctx* ctx, const slai_qk_params* p, QkArgs& A) {
    SLAI_REQUIRE(ctx, p->head_size >= 1 && p->head_size <= 256, SLAI_ERR_SHAPE, "qk: head_size=%d must be 1 .. 256", p->head_size);
    SLAI_REQUIRE(ctx, p->n_q_heads >= 0 && p->n_kv_heads >= 0 && p->n_q_heads <= 65536 && p->n_kv_heads <= 65536, SLAI_ERR_SHAPE, "qk: head counts (%d, %d)",
                 p->n_q_heads, p->n_kv_heads);
    SLAI_REQUIRE(ctx, p->rope_variant >= -1 && p->rope_variant <= 1, SLAI_ERR_INVALID_ARG, "qk: unknown rotation %d", p->rope_variant);
    SLAI_REQUIRE(ctx, p->rope_variant < 0 || p->head_size % 2 == 0, SLAI_ERR_SHAPE, "qk: a rotation needs an even head_size (%d)", p->head_size);
    SLAI_REQUIRE(ctx, p->rope_variant < 0 || (p->rope_base_freq > 0.f && isfinite(p->rope_base_freq)), SLAI_ERR_INVALID_ARG, "qk: base frequency %g",
                 (double)p->rope_base_freq);
    const int64_t q = (int64_t)p->n_q_heads * p->head_size, k = (int64_t)p->n_kv_heads * p->head_size;
    A.hs = p->head_size; A.n_q = p->n_q_heads; A.n_kv = p->n_kv_heads;
    A.variant = p->rope_variant < 0 ? 0 : p->rope_variant;
    A.eps = p->norm_eps;
    A.q_norm = p->d_q_norm; A.k_norm = p->d_k_norm;
    A.q_ld = p->q_ld ? p->q_ld : q; A.k_ld = p->k_ld ? p->k_ld : k; A.v_ld = p->v_ld ? p->v_ld : k;
    A.q_out_ld = p->q_out_ld ? p->q_out_ld : q; A.k_out_ld = p->k_out_ld ? p->k_out_ld : k;
    SLAI_REQUIRE(ctx, A.q_ld >= q && A.q_out_ld >= q && A.k_ld >= k && A.k_out_ld >= k && A.v_ld >= k, SLAI_ERR_SHAPE, "qk: a row is shorter than its heads");
    A.turns = nullptr;
    return p->rope_variant < 0 ? (int)SLAI_OK : turn_table(ctx, p->head_size, p->rope_base_freq, &A.turns);
}

// Heads are written while others are still read: a result's rows are its own input's, or share no float with any.
struct Rows {
    const char* name;
    const float* at;
    int64_t ld, w;
};
int check_apart(slai_ctx* ctx, const char* call, const Rows& out, const Rows& in, bool in_place, int64_t n) {
    if (in_place && out.at == in.at && (out.ld == in.ld || n <= 1)) return SLAI_OK;
    SLAI_REQUIRE(ctx, !rows_overlap((uintptr_t)out.at, out.ld, out.w, (uintptr_t)in.at, in.ld, in.w, n), SLAI_ERR_INVALID_ARG,
                 "%s: %s (rows %lld apart) shares floats with %s (rows %lld apart)", call, out.name, (long long)out.ld, in.name, (long long)in.ld);
    return SLAI_OK;
}

}  // namespace

SLAI_API int slai_paged_create(slai_ctx* ctx, const slai_paged_config* cfg, slai_paged** out) {
    if (!ctx || !cfg || !out) return SLAI_ERR_INVALID_ARG;
    *out = nullptr;
    SLAI_ENTER(ctx);
    const Config c = {cfg->n_q_heads, cfg->n_kv_heads, cfg->head_size, cfg->page_size, cfg->n_pages, cfg->kv_dtype, cfg->max_seqs, cfg->max_tokens, cfg->max_table};
    const std::string why = check_config(c);
    SLAI_REQUIRE(ctx, why.empty(), SLAI_ERR_SHAPE, "paged: %s", why.c_str());
    SLAI_REQUIRE(ctx, !capturing(ctx), SLAI_ERR_INVALID_ARG, "paged: a handle cannot be made while a pass is recorded");
    slai_paged* p = nullptr;
    int rc;
    try {
        p = new slai_paged();
        p->ctx = ctx;
        p->cfg = c;
        rc = make_handle(ctx, p);
    } catch (const std::exception&) {  // (the table of pages: up to 8 GB for 2^31 pages of one position)
        rc = slai_set_error(ctx, SLAI_ERR_OOM, "paged: no host memory for %d pages and %d table entries", c.n_pages, c.max_table);
    }
    if (rc) {
        cudaGetLastError();
        delete p;
        return rc;
    }
    *out = p;
    return SLAI_OK;
}

SLAI_API int slai_paged_destroy(slai_paged* p) {
    if (!p) return SLAI_OK;
    SLAI_ENTER(p->ctx);
    SLAI_REQUIRE(p->ctx, !capturing(p->ctx), SLAI_ERR_INVALID_ARG, "paged: a handle cannot be destroyed while a pass is recorded");
    cudaStreamSynchronize(p->ctx->stream);
    delete p;
    return SLAI_OK;
}

SLAI_API int slai_paged_step(slai_paged* p, int n_seq, const int32_t* h_pos0, const int32_t* h_n_new, const int32_t* h_tables, int64_t table_ld) {
    if (!p) return SLAI_ERR_INVALID_ARG;
    slai_ctx* ctx = p->ctx;
    SLAI_ENTER(ctx);
    SLAI_REQUIRE(ctx, !capturing(ctx), SLAI_ERR_INVALID_ARG, "paged: a step cannot be recorded (a recorded pass reads the step that is current when it runs)");
    SLAI_CHECK_CUDA(ctx, cudaEventSynchronize(p->copied[p->slot]));  // the copy that last left this slot
    int* h = p->h_plan[p->slot];
    Step st;
    std::string why;
    try {
        why = p->planner.plan(n_seq, h_pos0, h_n_new, h_tables, table_ld, h, &st);
    } catch (const std::exception&) {
        return slai_set_error(ctx, SLAI_ERR_OOM, "paged step: no host memory");
    }
    SLAI_REQUIRE(ctx, why.empty(), SLAI_ERR_SHAPE, "paged step: %s", why.c_str());
    const Layout& L = p->planner.lay();
    const size_t head = (size_t)L.rows + 2 * (size_t)st.n_rows, gap = L.dynamic - head;
    if (gap <= 16384) {  // one copy of what lies between them too: 64 KB are less than a second request
        SLAI_CHECK_CUDA(ctx, cudaMemcpyAsync(p->dev->plan, h, 4 * ((size_t)L.dynamic + st.used), cudaMemcpyHostToDevice, ctx->stream));
    } else {
        SLAI_CHECK_CUDA(ctx, cudaMemcpyAsync(p->dev->plan, h, 4 * head, cudaMemcpyHostToDevice, ctx->stream));
        if (st.used) SLAI_CHECK_CUDA(ctx, cudaMemcpyAsync(p->dev->plan + L.dynamic, h + L.dynamic, 4 * (size_t)st.used, cudaMemcpyHostToDevice, ctx->stream));
    }
    SLAI_CHECK_CUDA(ctx, cudaEventRecord(p->copied[p->slot], ctx->stream));
    p->slot = (p->slot + 1) % SLOTS;
    p->step = st;
    return SLAI_OK;
}

SLAI_API int slai_qk_norm_rope(slai_ctx* ctx, const slai_qk_params* params, int n_tokens, const int32_t* d_pos, const float* d_q, const float* d_k,
                               float* d_q_out, float* d_k_out) {
    if (!ctx || !params || n_tokens < 0) return SLAI_ERR_INVALID_ARG;
    SLAI_ENTER(ctx);
    QkArgs A = {};
    const int rc = fill_qk(ctx, params, A);
    if (rc || n_tokens == 0) return rc;
    SLAI_REQUIRE(ctx, d_pos && (A.n_q == 0 || (d_q && d_q_out)) && (A.n_kv == 0 || (d_k && d_k_out)), SLAI_ERR_INVALID_ARG, "qk: rows or positions are missing");
    const int64_t qw = (int64_t)A.n_q * A.hs, kw = (int64_t)A.n_kv * A.hs;
    const Rows q = {"q", d_q, A.q_ld, qw}, k = {"k", d_k, A.k_ld, kw}, qo = {"q_out", d_q_out, A.q_out_ld, qw}, ko = {"k_out", d_k_out, A.k_out_ld, kw};
    int bad = check_apart(ctx, "qk", qo, q, true, n_tokens);
    if (!bad) bad = check_apart(ctx, "qk", ko, k, true, n_tokens);
    if (!bad) bad = check_apart(ctx, "qk", qo, k, false, n_tokens);
    if (!bad) bad = check_apart(ctx, "qk", ko, q, false, n_tokens);
    if (!bad) bad = check_apart(ctx, "qk", qo, ko, false, n_tokens);
    if (bad) return bad;
    A.rows = n_tokens;
    A.pos = d_pos;
    A.q = d_q; A.k = d_k; A.q_out = d_q_out; A.k_out = d_k_out;
    return qk_launch(ctx, A, ctx->use_pdl);
}

SLAI_API int slai_paged_append(slai_paged* p, const slai_paged_layer* layer, const slai_qk_params* params, const float* d_q, const float* d_k, const float* d_v,
                               float* d_q_out) {
    if (!p || !layer || !params || !d_k || !d_v) return SLAI_ERR_INVALID_ARG;
    slai_ctx* ctx = p->ctx;
    SLAI_ENTER(ctx);
    QkArgs A = {};
    int rc = fill_cache(p, layer, &A.cache);
    if (rc) return rc;
    SLAI_REQUIRE(ctx, rows_apart(p->cfg, layer->page_stride, layer->head_stride, layer->pos_stride), SLAI_ERR_SHAPE,
                 "paged append: by strides of %lld, %lld and %lld (page, head, position) rows of %d elements lie on one another", (long long)layer->page_stride,
                 (long long)layer->head_stride, (long long)layer->pos_stride, p->cfg.head_size);
    SLAI_REQUIRE(ctx, params->head_size == p->cfg.head_size && params->n_kv_heads == p->cfg.n_kv_heads && (params->n_q_heads == p->cfg.n_q_heads || params->n_q_heads == 0),
                 SLAI_ERR_SHAPE, "paged append: heads of %d, %d on %d, are not the cache's (%d, %d on %d)", params->head_size, params->n_q_heads, params->n_kv_heads,
                 p->cfg.head_size, p->cfg.n_q_heads, p->cfg.n_kv_heads);
    if ((rc = fill_qk(ctx, params, A))) return rc;
    SLAI_REQUIRE(ctx, A.n_q == 0 || (d_q && d_q_out), SLAI_ERR_INVALID_ARG, "paged append: queries are missing (n_q_heads 0: none)");
    A.rows = p->step.n_rows;
    A.q = d_q; A.k = d_k; A.v = d_v; A.q_out = d_q_out;
    A.kv_f16 = p->cfg.kv_dtype == SLAI_KV_F16;
    if (capturing(ctx)) {
        if ((rc = slai_keep_for_pass(ctx, p->dev))) return rc;
        A.rows = p->cfg.max_tokens;
        A.counted = 1;
    }
    const int64_t qw = (int64_t)A.n_q * A.hs, kw = (int64_t)A.n_kv * A.hs;
    const Rows qo = {"q_out", d_q_out, A.q_out_ld, qw};
    if ((rc = check_apart(ctx, "paged append", qo, {"q", d_q, A.q_ld, qw}, true, A.rows))) return rc;
    if ((rc = check_apart(ctx, "paged append", qo, {"k", d_k, A.k_ld, kw}, false, A.rows))) return rc;
    if ((rc = check_apart(ctx, "paged append", qo, {"v", d_v, A.v_ld, kw}, false, A.rows))) return rc;
    return qk_launch(ctx, A, ctx->use_pdl);
}

SLAI_API int slai_paged_attention(slai_paged* p, const slai_paged_layer* layer, const float* d_q, int64_t q_ld, float scale, float* d_out, int64_t out_ld) {
    if (!p || !layer || !d_q || !d_out) return SLAI_ERR_INVALID_ARG;
    slai_ctx* ctx = p->ctx;
    SLAI_ENTER(ctx);
    AttnArgs A = {};
    int rc = fill_cache(p, layer, &A.c);
    if (rc) return rc;
    const Config& c = p->cfg;
    const int64_t row = (int64_t)c.n_q_heads * c.head_size;
    A.q_ld = q_ld ? q_ld : row;
    A.out_ld = out_ld ? out_ld : row;
    SLAI_REQUIRE(ctx, A.q_ld >= row && A.out_ld >= row, SLAI_ERR_SHAPE, "paged attention: rows of %lld and %lld floats are shorter than %lld", (long long)A.q_ld,
                 (long long)A.out_ld, (long long)row);
    SLAI_REQUIRE(ctx, isfinite(scale), SLAI_ERR_INVALID_ARG, "paged attention: scale %g", (double)scale);
    SLAI_REQUIRE(ctx, d_q != d_out, SLAI_ERR_INVALID_ARG, "paged attention: queries are read while results are written, out cannot be q");
    const bool recording = capturing(ctx);
    if ((rc = check_apart(ctx, "paged attention", {"out", d_out, A.out_ld, row}, {"q", d_q, A.q_ld, row}, false, recording ? c.max_tokens : p->step.n_rows))) return rc;
    A.scale = scale == 0.f ? (float)(1.0 / sqrt((double)c.head_size)) : scale;
    A.q = d_q;
    A.out = d_out;
    A.n_pages = c.n_pages;
    const int esz = c.kv_dtype == SLAI_KV_F16 ? 2 : 4;
    const uintptr_t bits = (uintptr_t)layer->d_keys | (uintptr_t)layer->d_values | (uintptr_t)(layer->page_stride * esz) | (uintptr_t)(layer->head_stride * esz) |
                           (uintptr_t)(layer->pos_stride * esz) | (uintptr_t)(c.head_size * esz);
    A.vec = (bits & 15) == 0;
    A.qvec = (((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)(A.q_ld * 4) | (uintptr_t)(A.out_ld * 4) | (uintptr_t)(c.head_size * 4)) & 15) == 0;
    A.err_flag = ctx->d_counters + CNT_ERR_FLAG;
    A.wait_limit = ctx->wait_limit;
    if (recording && (rc = slai_keep_for_pass(ctx, p->dev))) return rc;
    A.recorded = recording;
    for (int k = 0; k < 2; k++) {
        const Lane& l = p->planner.lane(k);
        if (l.blocks == 0) continue;
        A.starts_at = p->planner.lay().starts[k];
        A.joins_at = p->planner.lay().joins[k];
        A.count_at = p->planner.lay().count + 1 + k;
        A.tile_rows = l.rows;
        A.unit = l.unit;
        A.part = p->dev->part[k];
        A.part_ml = p->dev->ml[k];
        if ((rc = paged_attention_launch(ctx, A, c.kv_dtype, k, recording ? l.blocks : p->step.blocks[k], recording ? l.blocks : p->step.joins[k],
                                         recording ? l.blocks : p->step.longest[k], ctx->use_pdl))) return rc;
    }
    return SLAI_OK;
}
