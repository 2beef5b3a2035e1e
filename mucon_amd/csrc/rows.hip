// C-ABI entry points of the row operators: a row's top logits (top_rows.hpp), the distillation loss and its gradient (distill.hpp), one token a row (sample.hpp).
// Declared in include/mucon_hip.h.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/mucon_hip.h"
#include "distill.hpp"
#include "sample.hpp"
#include "top_rows.hpp"

void mucon_internal_set_error(const char *msg);  // mucon_hip.hip: feeds mucon_last_error()

using namespace rows;

static int rfail(int code, const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    mucon_internal_set_error(buf);
    return code;
}
static int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MUCON_OK : rfail(MUCON_E_HIP, "%s: kernel launch failed: %s", what, hipGetErrorString(e));
}

static int rows_check(const char *what, int type, int64_t rows, int vocab, int64_t stride) {
    if (type < 0 || type > 2) return rfail(MUCON_E_ARG, "%s: element type %d (0 fp32, 1 bf16, 2 fp16)", what, type);
    if (vocab < 1 || vocab > MAX_VOCAB) return rfail(MUCON_E_ARG, "%s: rows of %d elements (1 .. %d)", what, vocab, MAX_VOCAB);
    // (a launch holds fewer than 2^32 threads: 1,024 a row, 64 a row of up to 64 elements)
    const int64_t most = vocab <= 64 ? MUCON_ROWS_MAX_SHORT : MUCON_ROWS_MAX;
    if (rows < 0 || rows > most) return rfail(MUCON_E_ARG, "%s: %lld rows (at most %lld)", what, (long long)rows, (long long)most);
    if (stride < vocab && rows > 1) return rfail(MUCON_E_ARG, "%s: row stride %lld below the row's %d elements", what, (long long)stride, vocab);
    return MUCON_OK;
}

// Of top logits and distillation.  Within these log2(e) / T and its products with the differences of a row's logits keep their bits in fp32 (beyond, 0 times infinity made
// rows NaN).
static bool temperature_ok(double t) { return t >= 1e-30 && t <= 1e30; }

#define BY_TYPE(type, F, ...)       \
    switch (type) {                 \
        case F32: F(F32, __VA_ARGS__); break; \
        case BF16: F(BF16, __VA_ARGS__); break; \
        default: F(F16, __VA_ARGS__); break;  \
    }

// Few long rows leave most of the chip idle as one workgroup each: up to 128 rows are cut, into slices of 8,192 elements or more so that there are no more than 256
// workgroups, but of no more than a workgroup of 1,024 holds in its registers; their first k together have to fit the list of the workgroup that joins them.
static Slices plan_slices(int type, int64_t rows, int vocab, int k) {
    const Slices whole{1, vocab, 0, nullptr, nullptr};
    if (vocab <= 8192 || rows < 1 || rows > 128) return whole;
    const int most = CUT * 1024 * (type == F32 ? 4 : 8);
    int count = (int)(256 / rows);
    if (count > vocab / 8192) count = vocab / 8192;
    if (count < (vocab + most - 1) / most) count = (vocab + most - 1) / most;
    if (count < 2) return whole;
    Slices sl = whole;
    sl.length = ((vocab + count - 1) / count + 255) / 256 * 256;
    sl.count = (vocab + sl.length - 1) / sl.length;
    sl.keep = LIST / sl.count;
    return sl.count < 2 || sl.length > most || sl.keep < k ? whole : sl;
}
static size_t slices_bytes(const Slices &sl, int64_t rows) {
    return sl.count < 2 ? 0 : (size_t)rows * sl.count * (sizeof(Slices::Part) + sizeof(u64) * (size_t)sl.keep);
}
static void place_slices(Slices &sl, int64_t rows, void *ws) {
    sl.kept = static_cast<u64 *>(ws);
    sl.part = reinterpret_cast<Slices::Part *>(sl.kept + (size_t)rows * sl.count * sl.keep);
}

extern "C" size_t mucon_top_logits_workspace_bytes(int32_t type, int64_t rows, int32_t vocab, int32_t k) {
    return type < 0 || type > 2 || vocab < 1 || vocab > MAX_VOCAB || k < 1 || k > MAX_K ? 0 : slices_bytes(plan_slices(type, rows, vocab, k), rows);
}

extern "C" int mucon_top_logits(int32_t type, int64_t rows, int32_t vocab, int64_t row_stride, int32_t k, double temperature, const void *logits, void *values,
                                int32_t *index, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = rows_check("top_logits", type, rows, vocab, row_stride);
    if (rc != MUCON_OK) return rc;
    if (k < 1 || k > MAX_K || k > vocab) return rfail(MUCON_E_ARG, "top_logits: k = %d of %d elements (1 .. min(vocab, %d))", k, vocab, MAX_K);
    if (!temperature_ok(temperature)) return rfail(MUCON_E_ARG, "top_logits: temperature %g (1e-30 .. 1e30)", temperature);
    if (rows == 0) return MUCON_OK;
    if (!logits || !values || !index || !lse) return rfail(MUCON_E_ARG, "top_logits: null pointer argument");
    TopArgs a{logits, row_stride, vocab, k, temperature, exponent_of(temperature), values, index, lse};
    hipStream_t s = static_cast<hipStream_t>(stream);
    Slices sl = plan_slices(type, rows, vocab, k);
    if (sl.count > 1) {
        if (!workspace || workspace_bytes < slices_bytes(sl, rows)) return rfail(MUCON_E_WORKSPACE, "top_logits workspace too small");
        place_slices(sl, rows, workspace);
#define TOP_CUT(TY, _)                                                                                                             \
    hipLaunchKernelGGL((top_cut_kernel<TY, 1024>), dim3((unsigned)(rows * sl.count)), dim3(1024), 0, s, a, sl);                      \
    hipLaunchKernelGGL((top_join_kernel<TY, 1024>), dim3((unsigned)rows), dim3(1024), 0, s, a, sl);
        BY_TYPE(type, TOP_CUT, 0)
        return launched("top_logits");
    }
    const int vectors = (vocab + (type == F32 ? 3 : 7)) / (type == F32 ? 4 : 8);
#define TOP_ROW(TY, NT, NV) hipLaunchKernelGGL((top_rows_kernel<TY, NT, NV>), dim3((unsigned)rows), dim3(NT), 0, s, a)
#define TOP_SMALL(TY, E) hipLaunchKernelGGL((top_small_kernel<TY, E>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, (long long)rows)
#define TOP(TY, _)                                                                                               \
    if (vocab <= 64)                                                                                             \
        TOP_SMALL(TY, 1);                                                                                        \
    else if (vocab <= 128)                                                                                       \
        TOP_SMALL(TY, 2);                                                                                        \
    else if (vocab <= 256)                                                                                       \
        TOP_SMALL(TY, 4);                                                                                        \
    else if (vectors <= 2048 && k <= 256)                                                                        \
        TOP_ROW(TY, 256, 8);                                                                                     \
    else if (vectors <= 4096 && k <= 512)                                                                        \
        TOP_ROW(TY, 512, 8);                                                                                     \
    else if (vectors <= 8192)                                                                                    \
        TOP_ROW(TY, 1024, 8);                                                                                    \
    else if (vectors <= 16384)                                                                                   \
        TOP_ROW(TY, 1024, 16);                                                                                   \
    else                                                                                                         \
        TOP_ROW(TY, 1024, 0);
    BY_TYPE(type, TOP, 0)
    return launched("top_logits");
}

// ---- distillation ----
static int distill_check(const mucon_distill_cfg *cfg) {
    if (!cfg) return rfail(MUCON_E_ARG, "distill: null cfg");
    int rc = rows_check("distill", cfg->type, cfg->rows, cfg->vocab, cfg->row_stride);
    if (rc != MUCON_OK) return rc;
    if (cfg->teacher_type < 0 || cfg->teacher_type > 2) return rfail(MUCON_E_ARG, "distill: teacher element type %d", cfg->teacher_type);
    if (cfg->k < 1 || cfg->k > MAX_K) return rfail(MUCON_E_ARG, "distill: %d listed entries a row (1 .. %d)", cfg->k, MAX_K);
    if (!temperature_ok(cfg->temperature)) return rfail(MUCON_E_ARG, "distill: temperature %g (1e-30 .. 1e30)", cfg->temperature);
    if (cfg->reduction < 0 || cfg->reduction > 2) return rfail(MUCON_E_ARG, "distill: reduction %d (0 none, 1 sum, 2 mean)", cfg->reduction);
    if (cfg->rows < 1) return rfail(MUCON_E_ARG, "distill: no rows");
    return MUCON_OK;
}

// workspace: [norm: 1 double, padded to 64 bytes][row records][row losses]
static size_t distill_stat_off() { return 64; }
static size_t distill_loss_off(int64_t rows) { return distill_stat_off() + sizeof(DistillRow) * (size_t)rows; }

extern "C" size_t mucon_distill_workspace_bytes(const mucon_distill_cfg *cfg) {
    if (distill_check(cfg) != MUCON_OK) return 0;
    return distill_loss_off(cfg->rows) + sizeof(float) * (size_t)cfg->rows;
}

static DistillArgs distill_args(const mucon_distill_cfg *cfg, const void *student, const void *tv, const int32_t *ti, const float *lse, const float *weight, void *ws) {
    DistillArgs a;
    a.s = student;
    a.stride = cfg->row_stride;
    a.t = tv;
    a.index = ti;
    a.lse = lse;
    a.weight = weight;
    a.vocab = cfg->vocab;
    a.k = cfg->k;
    a.tt = cfg->teacher_type;
    a.temperature = cfg->temperature;
    a.it = 1.0 / cfg->temperature;
    a.c = exponent_of(cfg->temperature);
    char *w = static_cast<char *>(ws);
    a.losses = reinterpret_cast<float *>(w + distill_loss_off(cfg->rows));
    a.stat = reinterpret_cast<DistillRow *>(w + distill_stat_off());
    a.grad = nullptr;
    a.upstream = nullptr;
    a.each = 0;
    a.norm = nullptr;
    a.scale = 1.0;
    return a;
}

static bool small_rows(const mucon_distill_cfg *cfg) { return cfg->vocab <= 64 && cfg->k <= 64; }

// MODE 0: losses and row records; 1: losses and gradient; 2: the gradient from the records
template <int TY, int MODE>
static int launch_distill(const mucon_distill_cfg *cfg, const DistillArgs &a, hipStream_t s) {
    if (small_rows(cfg)) {
        hipLaunchKernelGGL((distill_small_kernel<TY, MODE>), dim3((unsigned)((cfg->rows + 3) / 4)), dim3(256), 0, s, a, (long long)cfg->rows);
        return MUCON_OK;
    }
    const dim3 grid((unsigned)cfg->rows);
    const int vectors = (cfg->vocab + El<TY>::N - 1) / El<TY>::N;
    if constexpr (MODE == 2) {
        const int per = 256 * 4 * El<TY>::N, chunks = (cfg->vocab + per - 1) / per;
        if (cfg->rows * chunks > (1 << 24) - 1) return rfail(MUCON_E_ARG, "distill: %lld rows of %d are too many for one call", (long long)cfg->rows, cfg->vocab);
        hipLaunchKernelGGL((distill_bwd_kernel<TY, 256>), dim3((unsigned)(cfg->rows * chunks)), dim3(256), 0, s, a, chunks, (long long)cfg->rows);
        return MUCON_OK;
    } else {
        const size_t lds = sizeof(uint32_t) * (size_t)list_words(cfg->vocab, cfg->k);
#define ROW(NT, NV) hipLaunchKernelGGL((distill_row_kernel<TY, NT, NV, MODE == 1>), grid, dim3(NT), lds, s, a)
        if (vectors <= 64)
            ROW(64, 1);
        else if (vectors <= 256)
            ROW(64, 4);
        else if (vectors <= 1024)
            ROW(256, 4);
        else if (MODE == 1 && vectors <= 2048)
            ROW(256, 8);
        else if (MODE == 1)
            hipLaunchKernelGGL((distill_stream_kernel<TY, 512, true>), grid, dim3(512), lds, s, a);
        else
            hipLaunchKernelGGL((distill_stream_kernel<TY, 256, false>), grid, dim3(256), lds, s, a);
#undef ROW
        return MUCON_OK;
    }
}
template <int MODE>
static int launch_distill(const mucon_distill_cfg *cfg, const DistillArgs &a, hipStream_t s) {
    return cfg->type == F32 ? launch_distill<F32, MODE>(cfg, a, s) : cfg->type == BF16 ? launch_distill<BF16, MODE>(cfg, a, s) : launch_distill<F16, MODE>(cfg, a, s);
}

static int distill_pointers(const mucon_distill_cfg *cfg, const void *student, const void *tv, const int32_t *ti, const void *out, const void *ws, size_t bytes) {
    if (!student || !tv || !ti || !out || !ws) return rfail(MUCON_E_ARG, "distill: null pointer argument");
    if (bytes < mucon_distill_workspace_bytes(cfg)) return rfail(MUCON_E_WORKSPACE, "distill workspace too small");
    return MUCON_OK;
}

extern "C" int mucon_distill_fwd(const mucon_distill_cfg *cfg, const void *student, const void *teacher_values, const int32_t *teacher_index, const float *teacher_lse,
                                 const float *weight, float *losses, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = distill_check(cfg);
    if (rc != MUCON_OK) return rc;
    if ((rc = distill_pointers(cfg, student, teacher_values, teacher_index, losses, workspace, workspace_bytes)) != MUCON_OK) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    DistillArgs a = distill_args(cfg, student, teacher_values, teacher_index, teacher_lse, weight, workspace);
    if (cfg->reduction == 0) a.losses = losses;
    if ((rc = launch_distill<0>(cfg, a, s)) != MUCON_OK) return rc;
    if (cfg->reduction != 0)
        hipLaunchKernelGGL(distill_join_kernel, dim3(1), dim3(1024), 0, s, a.losses, weight, (long long)cfg->rows, cfg->reduction == 2 ? 1 : 0, losses,
                           static_cast<double *>(workspace));
    return launched("distill_fwd");
}

extern "C" int mucon_distill_bwd(const mucon_distill_cfg *cfg, const void *student, const void *teacher_values, const int32_t *teacher_index, const float *teacher_lse,
                                 const float *weight, const float *d_losses, void *d_student, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = distill_check(cfg);
    if (rc != MUCON_OK) return rc;
    if ((rc = distill_pointers(cfg, student, teacher_values, teacher_index, d_student, workspace, workspace_bytes)) != MUCON_OK) return rc;
    if (!d_losses) return rfail(MUCON_E_ARG, "distill: null pointer argument");
    DistillArgs a = distill_args(cfg, student, teacher_values, teacher_index, teacher_lse, weight, workspace);
    a.grad = d_student;
    a.upstream = d_losses;
    a.each = cfg->reduction == 0;
    a.norm = cfg->reduction == 2 ? static_cast<double *>(workspace) : nullptr;
    if ((rc = launch_distill<2>(cfg, a, static_cast<hipStream_t>(stream))) != MUCON_OK) return rc;
    return launched("distill_bwd");
}

extern "C" int mucon_distill_fwd_bwd(const mucon_distill_cfg *cfg, const void *student, const void *teacher_values, const int32_t *teacher_index, const float *teacher_lse,
                                     const float *weight, double grad_scale, float *losses, void *d_student, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = distill_check(cfg);
    if (rc != MUCON_OK) return rc;
    if ((rc = distill_pointers(cfg, student, teacher_values, teacher_index, losses, workspace, workspace_bytes)) != MUCON_OK) return rc;
    if (!d_student) return rfail(MUCON_E_ARG, "distill: null pointer argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    DistillArgs a = distill_args(cfg, student, teacher_values, teacher_index, teacher_lse, weight, workspace);
    if (cfg->reduction == 0) a.losses = losses;
    a.grad = d_student;
    a.scale = grad_scale;
    double *norm = static_cast<double *>(workspace);
    if (cfg->reduction == 2) {      // the sum of the weights comes first
        if (weight) {
            hipLaunchKernelGGL(distill_join_kernel, dim3(1), dim3(1024), 0, s, nullptr, weight, (long long)cfg->rows, 1, nullptr, norm);
            a.norm = norm;
        } else {
            a.scale /= (double)cfg->rows;
        }
    }
    if ((rc = launch_distill<1>(cfg, a, s)) != MUCON_OK) return rc;
    if (cfg->reduction != 0)
        hipLaunchKernelGGL(distill_join_kernel, dim3(1), dim3(1024), 0, s, a.losses, weight, (long long)cfg->rows, cfg->reduction == 2 ? 1 : 0, losses, nullptr);
    return launched("distill_fwd_bwd");
}

// ---- drawing ----
extern "C" int mucon_sample_logits(int32_t type, int64_t rows, int32_t vocab, int64_t row_stride, const void *logits, const float *uniform,
                                   const mucon_sample_params *params, int64_t *token, float *logp, void *stream) {
    int rc = rows_check("sample_logits", type, rows, vocab, row_stride);
    if (rc != MUCON_OK) return rc;
    if (!params) return rfail(MUCON_E_ARG, "sample_logits: null params");
    if (!params->temperatures && (!(params->temperature >= 0.f) || !isfinite(params->temperature)))
        return rfail(MUCON_E_ARG, "sample_logits: temperature %g", (double)params->temperature);
    if (!params->top_ps && !(params->top_p > 0.f)) return rfail(MUCON_E_ARG, "sample_logits: top_p %g (above 0; 1 keeps everything)", (double)params->top_p);
    if (!params->min_ps && !(params->min_p >= 0.f && params->min_p <= 1.f)) return rfail(MUCON_E_ARG, "sample_logits: min_p %g (0 .. 1)", (double)params->min_p);
    if (!params->top_ks && params->top_k < 0) return rfail(MUCON_E_ARG, "sample_logits: top_k %d (0: no limit)", params->top_k);
    if (rows == 0) return MUCON_OK;
    if (!logits || !uniform || !token || !logp) return rfail(MUCON_E_ARG, "sample_logits: null pointer argument");
    SampleArgs a;
    a.x = logits;
    a.stride = row_stride;
    a.vocab = vocab;
    a.uniform = uniform;
    a.temperature = params->temperature;
    a.top_p = params->top_p;
    a.min_p = params->min_p;
    a.top_k = params->top_k;
    a.temperatures = params->temperatures;
    a.top_ps = params->top_ps;
    a.min_ps = params->min_ps;
    a.top_ks = params->top_ks;
    a.token = reinterpret_cast<long long *>(token);
    a.logp = logp;
    hipStream_t s = static_cast<hipStream_t>(stream);
#define SAMPLE_SMALL(TY, E) hipLaunchKernelGGL((sample_small_kernel<TY, E>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, (long long)rows)
#define SAMPLE(TY, _)                                                                                              \
    if (vocab <= 64)                                                                                               \
        SAMPLE_SMALL(TY, 1);                                                                                       \
    else if (vocab <= 128)                                                                                         \
        SAMPLE_SMALL(TY, 2);                                                                                       \
    else if (vocab <= 256)                                                                                         \
        SAMPLE_SMALL(TY, 4);                                                                                       \
    else if (vocab <= 1024)                                                                                        \
        hipLaunchKernelGGL((sample_listed_kernel<TY, 256, 1, 1024>), dim3((unsigned)rows), dim3(256), 0, s, a);    \
    else if (vocab <= LIST)                                                                                        \
        hipLaunchKernelGGL((sample_listed_kernel<TY, 256, 4, LIST>), dim3((unsigned)rows), dim3(256), 0, s, a);    \
    else                                                                                                           \
        hipLaunchKernelGGL((sample_rows_kernel<TY, 1024>), dim3((unsigned)rows), dim3(1024), 0, s, a);
    BY_TYPE(type, SAMPLE, 0)
    return launched("sample_logits");
}
