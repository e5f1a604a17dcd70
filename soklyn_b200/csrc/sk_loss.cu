// Entry points of the losses over rows of logits: argument checks and launches.
#include <algorithm>
#include <cmath>

#include "sk_context.cuh"
#include "sk_loss.cuh"

namespace {
using namespace sk;

// Entry points may be called with another device current than the context's.
struct OnDevice {
    int before = -1;
    explicit OnDevice(const sk_ctx *c) {
        int now = 0;
        if (cudaGetDevice(&now) == cudaSuccess && now != c->device && cudaSetDevice(c->device) == cudaSuccess) before = now;
    }
    ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
};

inline bool overlaps(const sk_ctx *c) { return c->reserve_sms == 0; }   // blocks that wait for a predecessor would sit on reserved SMs
inline size_t size_of(uint32_t dtype) { return dtype == SK_F32 ? 4 : 2; }
inline bool on_elements(const void *p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

#define LOSS_DISPATCH(dtype, fn, ...)                       \
    ((dtype) == SK_F32 ? fn<float>(__VA_ARGS__)             \
     : (dtype) == SK_F16 ? fn<__half>(__VA_ARGS__) : fn<__nv_bfloat16>(__VA_ARGS__))

// The checks that every loss makes of its logits, and their kernel argument.
int make_rows(sk_ctx *c, const sk_logits *x, bool need_gradient, loss::Rows *out) {
    if (!c || !x) return SK_ERR_NULL_POINTER;
    c->fused_colsum_key = nullptr;   // column sums handed over by sk_hidden_error are for the very next call only
    if (x->dtype > SK_BF16) return fail(c, SK_ERR_INVALID_CONFIGURATION, "unknown dtype %u", x->dtype);
    const uint32_t classes = x->classes ? x->classes : x->cols;
    if (x->cols == 0) return fail(c, SK_ERR_INVALID_CONFIGURATION, "Input or output size cannot be 0.");
    if (classes > x->cols) return fail(c, SK_ERR_MISMATCHED_DIMENSIONS, "classes vs logit columns: expected at most %u, found %u", x->cols, classes);
    if (x->cols > (1u << 30) || x->rows > (1u << 30)) return fail(c, SK_ERR_ALLOCATION_LIMIT, "%u x %u logits: at most 2^30 rows and columns", x->rows, x->cols);
    if (!(x->temperature >= 1e-4f && x->temperature <= 1e4f))
        return fail(c, SK_ERR_INVALID_CONFIGURATION, "temperature %g must lie between 1e-4 and 1e4", (double)x->temperature);
    if (!std::isfinite(x->grad_scale)) return fail(c, SK_ERR_INVALID_CONFIGURATION, "gradient scale is not finite");
    if (x->rows && (!x->logits || (need_gradient && !x->d_logits))) return fail(c, SK_ERR_NULL_POINTER, "logits or their gradient pointer is NULL");
    if (!c->loss_err) return fail(c, SK_ERR_DRIVER, "the context has no error word");
    const size_t one = size_of(x->dtype), bytes = (size_t)x->rows * x->cols * one;
    if (!on_elements(x->logits, one) || !on_elements(x->d_logits, one))
        return fail(c, SK_ERR_INVALID_CONFIGURATION, "logits and gradient must be aligned to their elements");
    if (x->d_logits && x->d_logits != x->logits) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(x->logits), d = reinterpret_cast<uintptr_t>(x->d_logits);
        if (a < d + bytes && d < a + bytes) return fail(c, SK_ERR_INVALID_CONFIGURATION, "the gradient may be written over the logits, but not overlap them otherwise");
    }
    loss::Rows r{};
    r.x = x->logits; r.d = x->d_logits;
    r.rows = x->rows; r.cols = x->cols; r.classes = classes;
    const double base = 1.4426950408889634 / (double)x->temperature;
    r.c_hi = (float)base;
    if ((double)r.c_hi >= base) r.c_hi = std::nextafter(r.c_hi, 0.0f);
    r.c_lo = (float)(base - (double)r.c_hi);
    r.inv_t = 1.0 / (double)x->temperature;
    r.k = (float)((double)x->grad_scale / (double)x->temperature);
    r.err = c->loss_err;
    *out = r;
    return SK_OK;
}

// Threads of a block and blocks of a cluster for a row; the reasons stand beside Team. `twice`: the row is read again.
constexpr size_t kWarpRow = 32 * loss::kWarpUnits * 16, kPerThread = 256;
constexpr uint32_t kMostThreads = 256;
struct RowPlan { uint32_t threads, ranks; };
RowPlan plan_row(const sk_ctx *c, const loss::Rows &r, size_t one, bool twice) {
    const size_t bytes = (size_t)r.classes * one, rows = r.rows, sms = (size_t)c->num_sms;
    if (bytes <= kWarpRow) return RowPlan{32, 1};
    RowPlan plan{64, 1};
    while (plan.threads < kMostThreads && bytes > plan.threads * kPerThread) plan.threads *= 2;
    while (twice && plan.ranks < loss::kMaxCluster && bytes > plan.ranks * plan.threads * kPerThread) plan.ranks *= 2;
    // few rows: more threads for each, then more blocks, down to 32 bytes per thread
    while (plan.threads < kMostThreads && rows * plan.threads < sms * 1024 && bytes >= plan.threads * 64) plan.threads *= 2;
    while (plan.ranks < loss::kMaxCluster && rows * plan.ranks * 2 <= sms && bytes >= plan.ranks * plan.threads * 64) plan.ranks *= 2;
    return plan;
}
template <typename T, class Op, int SUMS, bool GRAD> cudaError_t launch_rows(sk_ctx *c, const loss::Rows &r, const Op &op) {
    constexpr int warp_sums = SUMS ? loss::kMasked : loss::kSums;
    const RowPlan plan = plan_row(c, r, sizeof(T), GRAD);
    c->launches++;
    c->loss_launches++;
    if (plan.threads == 32)
        return launch_step(c->stream, overlaps(c), dim3((r.rows + loss::kWarps - 1) / loss::kWarps), loss::kThreads, 0, dim3(1), loss::warp_kernel<T, Op, warp_sums, GRAD>, r, op);
    auto kernel = plan.threads == 64 ? loss::row_kernel<T, 64, Op, SUMS, GRAD> : plan.threads == 128 ? loss::row_kernel<T, 128, Op, SUMS, GRAD> : loss::row_kernel<T, kMostThreads, Op, SUMS, GRAD>;
    return launch_step(c->stream, overlaps(c), dim3(r.rows * plan.ranks), plan.threads, 0, dim3(plan.ranks), kernel, r, op);
}

template <typename T> cudaError_t label_impl(sk_ctx *c, const loss::Rows &r, const loss::LabelLogprob &op) {
    return op.entropy ? launch_rows<T, loss::LabelLogprob, loss::kEntropy, false>(c, r, op) : launch_rows<T, loss::LabelLogprob, loss::kSums, false>(c, r, op);
}
template <typename T> cudaError_t label_backward_impl(sk_ctx *c, const loss::Rows &r, const loss::LabelLogprobBackward &op) {
    return op.d_entropy ? launch_rows<T, loss::LabelLogprobBackward, loss::kEntropy, true>(c, r, op) : launch_rows<T, loss::LabelLogprobBackward, loss::kSums, true>(c, r, op);
}
template <typename T> cudaError_t policy_impl(sk_ctx *c, const loss::Rows &r, const loss::Policy &op) {
    if (op.entropy || op.eta != 0.0f) return r.d ? launch_rows<T, loss::Policy, loss::kEntropy, true>(c, r, op) : launch_rows<T, loss::Policy, loss::kEntropy, false>(c, r, op);
    return r.d ? launch_rows<T, loss::Policy, loss::kSums, true>(c, r, op) : launch_rows<T, loss::Policy, loss::kSums, false>(c, r, op);
}
template <typename T> cudaError_t sequence_impl(sk_ctx *c, const loss::Rows &r, const loss::SequenceLogprob &op) {
    return launch_rows<T, loss::SequenceLogprob, loss::kSums, false>(c, r, op);
}
template <typename T> cudaError_t sequence_gradient_impl(sk_ctx *c, const loss::Rows &r, const int32_t *labels, const loss::Kept *kept) {
    c->launches++;
    c->loss_launches++;
    const size_t bytes = (size_t)r.classes * sizeof(T);
    auto kernel = bytes <= 64 * kPerThread ? loss::sequence_gradient_kernel<T, 64> : bytes <= 128 * kPerThread ? loss::sequence_gradient_kernel<T, 128> : loss::sequence_gradient_kernel<T, 256>;
    const uint32_t threads = bytes <= 64 * kPerThread ? 64 : bytes <= 128 * kPerThread ? 128 : 256;
    return launch_step(c->stream, overlaps(c), dim3(r.rows), threads, 0, dim3(1), kernel, r, labels, kept);
}
template <typename T> cudaError_t distill_impl(sk_ctx *c, const loss::Rows &r, const loss::Distill &op) {
    RowPlan plan = plan_row(c, r, sizeof(T), r.d != nullptr);
    const uint32_t threads = std::max(plan.threads, 64u);
    // A block has 48 KB without asking for more, and a row's bits may take 128: more blocks share such a row (four at 2^20 classes).
    // One block with up to 128 KB leaves an SM one or two of them: 1000 bf16 rows of 2^20 classes took 1035 us against 421,
    // 80 rows 149 against 57, 1000 rows of 400000 210 against 172. A gradient's rows are shared by enough blocks for other reasons.
    constexpr size_t room = 48 * 1024 - sizeof(loss::DistillShared<kMostThreads>);
    while (plan.ranks < loss::kMaxCluster && loss::bit_bytes<T>(r.classes, plan.ranks) > room) plan.ranks *= 2;
    static_assert(loss::kMaxListClasses / loss::kMaxCluster / 8 + 64 <= room, "the bits of the widest row fit the blocks of a cluster");
    const size_t bytes = loss::bit_bytes<T>(r.classes, plan.ranks);
    auto kernel = threads == 64 ? loss::distill_kernel<T, 64> : threads == 128 ? loss::distill_kernel<T, 128> : loss::distill_kernel<T, kMostThreads>;
    c->launches++;
    c->loss_launches++;
    return launch_step(c->stream, overlaps(c), dim3(r.rows * plan.ranks), threads, bytes, dim3(plan.ranks), kernel, r, op);
}
} // namespace

extern "C" {

int sk_label_logprob(sk_ctx *c, const sk_logits *x, const int32_t *labels, float *logp, float *entropy) {
    loss::Rows r;
    int rc = make_rows(c, x, false, &r);
    if (rc || r.rows == 0) return rc;
    if (!labels || !logp) return fail(c, SK_ERR_NULL_POINTER, "label or log-probability pointer is NULL");
    r.d = nullptr;
    OnDevice guard(c);
    ProfScope ps(c, SK_PROF_OUTPUT_ERROR);
    const loss::LabelLogprob op{labels, logp, entropy};
    return check_cuda(c, LOSS_DISPATCH(x->dtype, label_impl, c, r, op), "label log-probability");
}

int sk_label_logprob_backward(sk_ctx *c, const sk_logits *x, const int32_t *labels, const float *d_logp, const float *d_entropy) {
    loss::Rows r;
    int rc = make_rows(c, x, true, &r);
    if (rc || r.rows == 0) return rc;
    if (!labels || !d_logp) return fail(c, SK_ERR_NULL_POINTER, "label or gradient pointer is NULL");
    OnDevice guard(c);
    ProfScope ps(c, SK_PROF_OUTPUT_ERROR);
    const loss::LabelLogprobBackward op{labels, d_logp, d_entropy};
    return check_cuda(c, LOSS_DISPATCH(x->dtype, label_backward_impl, c, r, op), "label log-probability backward");
}

int sk_distill_loss(sk_ctx *c, const sk_logits *x, const sk_distill *t) {
    loss::Rows r;
    int rc = make_rows(c, x, false, &r);
    if (rc) return rc;
    if (!t) return fail(c, SK_ERR_NULL_POINTER, "teacher pointer is NULL");
    if (t->values_dtype > SK_BF16) return fail(c, SK_ERR_INVALID_CONFIGURATION, "unknown dtype %u", t->values_dtype);
    if (t->k == 0 || t->k > loss::kMaxList) return fail(c, SK_ERR_INVALID_CONFIGURATION, "a teacher's list of %u entries (1 to %u)", t->k, loss::kMaxList);
    if (r.classes > loss::kMaxListClasses) return fail(c, SK_ERR_ALLOCATION_LIMIT, "distillation over %u classes (at most %u)", r.classes, loss::kMaxListClasses);
    if (r.rows == 0) return SK_OK;
    if (!t->indices || !t->values || !t->loss) return fail(c, SK_ERR_NULL_POINTER, "teacher or loss pointer is NULL");
    if (!on_elements(t->values, size_of(t->values_dtype))) return fail(c, SK_ERR_INVALID_CONFIGURATION, "teacher values must be aligned to their elements");
    OnDevice guard(c);
    ProfScope ps(c, SK_PROF_OUTPUT_ERROR);
    const loss::Distill op{t->indices, t->values, t->values_dtype, t->k, t->lse, t->weights, t->loss, (double)x->temperature * (double)x->temperature};
    return check_cuda(c, LOSS_DISPATCH(x->dtype, distill_impl, c, r, op), "distillation loss");
}

int sk_policy_loss(sk_ctx *c, const sk_logits *x, const sk_policy *p) {
    loss::Rows r;
    int rc = make_rows(c, x, false, &r);
    if (rc) return rc;
    if (!p) return fail(c, SK_ERR_NULL_POINTER, "policy pointer is NULL");
    if (!(p->clip_low >= 0.0f && p->clip_low <= 1.0f) || !(p->clip_high >= 0.0f)) return fail(c, SK_ERR_INVALID_CONFIGURATION, "clip range %g below and %g above 1", (double)p->clip_low, (double)p->clip_high);
    if (!std::isfinite(p->kl_coeff) || !std::isfinite(p->entropy_coeff)) return fail(c, SK_ERR_INVALID_CONFIGURATION, "policy coefficients must be finite");
    if (p->kl_coeff != 0.0f && !p->logp_ref && r.rows) return fail(c, SK_ERR_NULL_POINTER, "a KL term needs the reference's log-probabilities");
    if (r.rows == 0) return SK_OK;
    if (!p->actions || !p->logp_old || !p->advantages || !p->loss || !p->logp || !p->kl) return fail(c, SK_ERR_NULL_POINTER, "policy tensor pointer is NULL");
    OnDevice guard(c);
    ProfScope ps(c, SK_PROF_OUTPUT_ERROR);
    const loss::Policy op{p->actions, p->logp_old, p->advantages, p->logp_ref, p->weights, 1.0f - p->clip_low, 1.0f + p->clip_high,
                          p->kl_coeff, p->entropy_coeff, p->loss, p->logp, p->kl, p->entropy};
    return check_cuda(c, LOSS_DISPATCH(x->dtype, policy_impl, c, r, op), "policy loss");
}

int sk_preference_loss(sk_ctx *c, const sk_logits *x, const sk_preference *p) {
    loss::Rows r;
    int rc = make_rows(c, x, false, &r);
    if (rc) return rc;
    if (!p) return fail(c, SK_ERR_NULL_POINTER, "preference pointer is NULL");
    if (p->form > SK_PREFERENCE_SQUARED) return fail(c, SK_ERR_INVALID_CONFIGURATION, "preference form %u out of range", p->form);
    if (p->pairs > (1u << 29)) return fail(c, SK_ERR_ALLOCATION_LIMIT, "%u pairs: at most 2^29", p->pairs);
    if (!std::isfinite(p->beta) || !std::isfinite(p->target_margin)) return fail(c, SK_ERR_INVALID_CONFIGURATION, "beta and target margin must be finite");
    if (!(p->label_smoothing >= 0.0f && p->label_smoothing <= 1.0f)) return fail(c, SK_ERR_INVALID_CONFIGURATION, "label smoothing %g must lie between 0 and 1", (double)p->label_smoothing);
    if (p->label_smoothing != 0.0f && p->form != SK_PREFERENCE_SIGMOID) return fail(c, SK_ERR_INVALID_CONFIGURATION, "only the sigmoid form takes label smoothing");
    if (r.rows == 0 && p->pairs == 0) return SK_OK;
    if (!p->offsets || (r.rows && (!p->labels || !p->row_logp || !p->scratch)) || (p->pairs && (!p->loss || !p->margin || !p->logp)))
        return fail(c, SK_ERR_NULL_POINTER, "preference tensor pointer is NULL");
    OnDevice guard(c);
    ProfScope ps(c, SK_PROF_OUTPUT_ERROR);
    if (!on_elements(p->scratch, 16)) return fail(c, SK_ERR_INVALID_CONFIGURATION, "the scratch of a preference loss must be 16-byte aligned");
    loss::Kept *kept = reinterpret_cast<loss::Kept *>(p->scratch);
    if (r.rows) {
        const loss::SequenceLogprob op{p->labels, p->offsets, 2 * p->pairs, p->row_logp, kept};
        if ((rc = check_cuda(c, LOSS_DISPATCH(x->dtype, sequence_impl, c, r, op), "sequence log-probabilities"))) return rc;
    }
    if (p->pairs) {
        const loss::Pairs op{p->offsets, p->pairs, r.rows, p->form, p->average, p->logp_ref, p->weights, p->row_logp, kept, (double)p->beta,
                             (double)p->label_smoothing, (double)p->target_margin, p->loss, p->margin, p->logp, r.err};
        c->launches++;
        c->loss_launches++;
        if ((rc = check_cuda(c, launch_step(c->stream, overlaps(c), dim3(p->pairs), loss::kThreads, 0, dim3(1), loss::pair_kernel, op), "preference loss"))) return rc;
    }
    if (r.rows && r.d) return check_cuda(c, LOSS_DISPATCH(x->dtype, sequence_gradient_impl, c, r, p->labels, kept), "preference gradient");
    return SK_OK;
}

} // extern "C"
