// dlr_losses.cpp -- C entries of the softmax losses: every argument that the
// host can see is checked here, before anything is enqueued.
#include "dlr_losses.h"

#include <dlfcn.h>

#include <cmath>
#include <cstdio>
#include <initializer_list>

namespace {

thread_local char last_error[512] = "";

int refuse(int code, const char *call, const char *why) noexcept {
    (void)std::snprintf(last_error, sizeof last_error, "%s: %s", call, why);
    return code;
}

int fail_hip(const char *call, hipError_t e) noexcept { return refuse(DLR_E_HIP, call, hipGetErrorString(e)); }

// `device` current for the launch, the caller's device again afterwards.
class DeviceScope {
   public:
    explicit DeviceScope(int device) {
        err_ = hipGetDevice(&before_);
        if (err_ == hipSuccess && before_ != device) {
            err_ = hipSetDevice(device);
            set_ = err_ == hipSuccess;
        }
        if (err_ != hipSuccess) (void)hipGetLastError();  // reported here, not by the caller's next call
    }
    ~DeviceScope() {
        if (set_) (void)hipSetDevice(before_);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
    hipError_t error() const { return err_; }

   private:
    int before_ = 0;
    bool set_ = false;
    hipError_t err_;
};

int64_t element_bytes(int32_t dtype) { return dtype == DLR_DTYPE_F32 ? 4 : 2; }

bool aligned(const void *p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

// Rows x columns of `bytes`-byte elements whose addresses fit 63 bits.
bool spans(int64_t rows, int64_t cols, int64_t stride, int64_t bytes) {
    if (stride > (INT64_MAX / 16) / (rows > 1 ? rows : 1)) return false;
    return (rows - 1) * stride + cols <= INT64_MAX / 16 / bytes;
}

bool overlap(const void *a, int64_t a_bytes, const void *b, int64_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}

// Rows of `cols` bytes, `a_stride` and `b_stride` bytes apart.  Rows at the same
// distance may lie between each other's.
bool rows_overlap(const void *a, int64_t a_stride, const void *b, int64_t b_stride, int64_t rows, int64_t cols) {
    if (!overlap(a, (rows - 1) * a_stride + cols, b, (rows - 1) * b_stride + cols)) return false;
    if (rows == 1 || a_stride != b_stride || a_stride == 0) return true;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    const int64_t apart = (int64_t)((x < y ? y - x : x - y) % (uintptr_t)a_stride);
    return apart < cols || a_stride - apart < cols;
}

constexpr int64_t kMaxRows = INT64_C(0x7fffffff);
constexpr int64_t kMaxPairs = (INT64_C(1) << 22) - 1;  // one launch of at most 1,024 threads each
constexpr int64_t kMaxVocab = INT64_C(1) << 30;
constexpr int64_t kMaxDim = INT64_C(1) << 20;
constexpr int64_t kMaxClasses = INT64_C(1) << 28;  // a head call's
constexpr int64_t kMaxLogits = INT64_C(1) << 44;

const char *check_target(const void *target, int32_t bits, double temperature) {
    if (!target) return "target is NULL";
    if (bits != 32 && bits != 64) return "target_bits must be 32 or 64";
    if (!aligned(target, bits / 8)) return "target is not aligned to its type";
    if (!(temperature >= 1e-6 && temperature <= 1e6)) return "temperature must lie in [1e-6, 1e6]";
    return nullptr;
}

// nullptr: the logits can be used (rows may be 0).
const char *check_logits(const dlr_logits *x) {
    if (!x) return "the logits' descriptor is NULL";
    if (x->rows < 0 || x->rows > kMaxRows) return "rows must be 0 .. 2^31 - 1";
    if (x->vocab < 1 || x->vocab > kMaxVocab) return "vocab must be 1 .. 2^30";
    if (x->dtype != DLR_DTYPE_F32 && x->dtype != DLR_DTYPE_BF16 && x->dtype != DLR_DTYPE_F16)
        return "dtype must be DLR_DTYPE_F32, _BF16 or _F16";
    if (x->rows == 0) return nullptr;
    if (x->row_stride != 0 && x->row_stride < x->vocab && x->rows > 1)
        return "row_stride must be 0 or at least vocab";
    if (x->row_stride < 0 || !spans(x->rows, x->vocab, x->row_stride, 4)) return "row_stride is out of range";
    if (!x->data) return "the logits are NULL";
    if (!aligned(x->data, element_bytes(x->dtype))) return "the logits are not aligned to their type";
    return check_target(x->target, x->target_bits, x->temperature);
}

const char *check_grad(const dlr_logits *x, const void *grad, int64_t stride) {
    if (!aligned(grad, element_bytes(x->dtype))) return "grad_logits is not aligned to its type";
    if (x->rows > 1 && stride < x->vocab) return "grad_row_stride must be at least vocab";
    if (stride < 0 || !spans(x->rows, x->vocab, stride, 4)) return "grad_row_stride is out of range";
    const int64_t b = element_bytes(x->dtype);
    const bool same = grad == x->data && (stride == x->row_stride || x->rows == 1);
    if (!same && rows_overlap(x->data, x->row_stride * b, grad, stride * b, x->rows, x->vocab * b))
        return "grad_logits overlaps the logits and is not the logits themselves";
    if (same && x->rows > 1 && x->row_stride == 0) return "grad_logits cannot be logits whose rows share memory";
    return nullptr;
}

const char *check_workspace(const void *workspace, int64_t bytes, int64_t need) {
    if (need == 0) return nullptr;
    if (!workspace || bytes < need) return "the workspace is smaller than its size call says";
    if (!aligned(workspace, 256)) return "the workspace is not 256-byte aligned";
    return nullptr;
}

bool floats(std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (!aligned(p, 4)) return false;
    return true;
}

}  // namespace

extern "C" {

const char *dlr_losses_last_error(void) { return last_error; }

const char *dlr_losses_runtime(void) {
    Dl_info info;
    return dladdr(reinterpret_cast<const void *>(&hipGetDevice), &info) && info.dli_fname ? info.dli_fname : "";
}

int64_t dlr_logits_workspace(int64_t rows, int64_t vocab, int dtype) {
    if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > kMaxVocab || dtype < DLR_DTYPE_F32 || dtype > DLR_DTYPE_F16)
        return refuse(DLR_E_ARG, "dlr_logits_workspace", "rows, vocab or dtype is out of range");
    return dlr::logits_workspace(rows, vocab, dtype);
}

int dlr_token_logprob(int device, void *stream, const dlr_logits *x, void *workspace, int64_t workspace_bytes,
                      float *logprob, float *lse) {
    const char *call = "dlr_token_logprob";
    if (const char *why = check_logits(x)) return refuse(DLR_E_ARG, call, why);
    if (x->rows == 0) return DLR_OK;
    if (!logprob || !lse) return refuse(DLR_E_ARG, call, "logprob or lse is NULL");
    if (!floats({logprob, lse})) return refuse(DLR_E_ARG, call, "logprob or lse is not aligned");
    if (const char *why = check_workspace(workspace, workspace_bytes, dlr::logits_workspace(x->rows, x->vocab, x->dtype)))
        return refuse(DLR_E_ARG, call, why);
    DeviceScope d(device);
    if (d.error() != hipSuccess) return fail_hip(call, d.error());
    const hipError_t e = dlr::launch_token_logprob(static_cast<hipStream_t>(stream), *x, workspace, logprob, lse);
    return e == hipSuccess ? DLR_OK : fail_hip(call, e);
}

int dlr_token_logprob_grad(int device, void *stream, const dlr_logits *x, const float *lse, const float *grad,
                           void *grad_logits, int64_t grad_row_stride) {
    const char *call = "dlr_token_logprob_grad";
    if (const char *why = check_logits(x)) return refuse(DLR_E_ARG, call, why);
    if (x->rows == 0) return DLR_OK;
    if (!lse || !grad || !grad_logits) return refuse(DLR_E_ARG, call, "lse, grad or grad_logits is NULL");
    if (!floats({lse, grad})) return refuse(DLR_E_ARG, call, "lse or grad is not aligned");
    if (const char *why = check_grad(x, grad_logits, grad_row_stride)) return refuse(DLR_E_ARG, call, why);
    DeviceScope d(device);
    if (d.error() != hipSuccess) return fail_hip(call, d.error());
    const hipError_t e = dlr::launch_token_logprob_grad(static_cast<hipStream_t>(stream), *x, lse, grad, grad_logits,
                                                        grad_row_stride);
    return e == hipSuccess ? DLR_OK : fail_hip(call, e);
}

int dlr_policy_loss(int device, void *stream, const dlr_logits *x, const dlr_policy *p, void *workspace,
                    int64_t workspace_bytes, float *loss, float *logprob, float *kl, uint8_t *clipped,
                    void *grad_logits, int64_t grad_row_stride) {
    const char *call = "dlr_policy_loss";
    if (const char *why = check_logits(x)) return refuse(DLR_E_ARG, call, why);
    if (!p) return refuse(DLR_E_ARG, call, "the policy's descriptor is NULL");
    if (!(p->clip_low >= 0.0 && p->clip_low <= 1.0)) return refuse(DLR_E_ARG, call, "clip_low must lie in [0, 1]");
    if (!(p->clip_high >= 0.0) || !std::isfinite(p->clip_high))
        return refuse(DLR_E_ARG, call, "clip_high must be finite and not negative");
    if (!(p->kl_coef >= 0.0) || !std::isfinite(p->kl_coef))
        return refuse(DLR_E_ARG, call, "kl_coef must be finite and not negative");
    if (x->rows == 0) return DLR_OK;
    if (!p->ref_logprob && p->kl_coef != 0.0) return refuse(DLR_E_ARG, call, "kl_coef without ref_logprob");
    if (!p->old_logprob || !p->advantage) return refuse(DLR_E_ARG, call, "old_logprob or advantage is NULL");
    if (!loss || !logprob || !kl || !clipped) return refuse(DLR_E_ARG, call, "an output is NULL");
    if (!floats({p->old_logprob, p->ref_logprob, p->advantage, p->weight, loss, logprob, kl}))
        return refuse(DLR_E_ARG, call, "a float array is not aligned");
    if (grad_logits)
        if (const char *why = check_grad(x, grad_logits, grad_row_stride)) return refuse(DLR_E_ARG, call, why);
    if (const char *why = check_workspace(workspace, workspace_bytes, dlr::logits_workspace(x->rows, x->vocab, x->dtype)))
        return refuse(DLR_E_ARG, call, why);
    DeviceScope d(device);
    if (d.error() != hipSuccess) return fail_hip(call, d.error());
    const hipError_t e = dlr::launch_policy_loss(static_cast<hipStream_t>(stream), *x, *p, workspace, loss, logprob, kl,
                                                 clipped, grad_logits, grad_row_stride);
    return e == hipSuccess ? DLR_OK : fail_hip(call, e);
}

int dlr_preference_loss(int device, void *stream, const dlr_preference *p, float *loss, float *chosen_reward,
                        float *rejected_reward, float *grad) {
    const char *call = "dlr_preference_loss";
    if (!p) return refuse(DLR_E_ARG, call, "the descriptor is NULL");
    if (p->pairs < 0 || p->pairs > kMaxPairs) return refuse(DLR_E_ARG, call, "pairs must be 0 .. 2^22 - 1");
    if (p->tokens < 0 || p->tokens > (INT64_C(1) << 40)) return refuse(DLR_E_ARG, call, "tokens must be 0 .. 2^40");
    if (!(p->beta > 0.0) || !std::isfinite(p->beta)) return refuse(DLR_E_ARG, call, "beta must be positive and finite");
    if (!(p->label_smoothing >= 0.0 && p->label_smoothing <= 1.0))
        return refuse(DLR_E_ARG, call, "label_smoothing must lie in [0, 1]");
    if (!std::isfinite(p->margin)) return refuse(DLR_E_ARG, call, "margin must be finite");
    if (p->average != 0 && p->average != 1) return refuse(DLR_E_ARG, call, "average must be 0 or 1");
    if (p->pairs == 0 && (p->tokens == 0 || !grad)) return DLR_OK;
    if (p->pairs && (!p->offsets || !loss || !chosen_reward || !rejected_reward))
        return refuse(DLR_E_ARG, call, "offsets or an output is NULL");
    if (p->pairs && p->tokens && !p->logprob) return refuse(DLR_E_ARG, call, "logprob is NULL");
    if (!floats({p->logprob, p->ref_logprob, p->weight, loss, chosen_reward, rejected_reward, grad}))
        return refuse(DLR_E_ARG, call, "a float array is not aligned");
    if (!aligned(p->offsets, 8)) return refuse(DLR_E_ARG, call, "offsets is not aligned");
    if (grad && p->tokens) {
        const int64_t b = p->tokens * 4;
        if (overlap(grad, b, p->logprob, b) || (p->ref_logprob && overlap(grad, b, p->ref_logprob, b)))
            return refuse(DLR_E_ARG, call, "grad overlaps an input");
    }
    DeviceScope d(device);
    if (d.error() != hipSuccess) return fail_hip(call, d.error());
    const hipError_t e = dlr::launch_preference_loss(static_cast<hipStream_t>(stream), *p, loss, chosen_reward,
                                                     rejected_reward, grad);
    return e == hipSuccess ? DLR_OK : fail_hip(call, e);
}

int64_t dlr_head_logprob_workspace(int64_t rows, int64_t vocab, int64_t dim) {
    if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > kMaxClasses || dim < 1 || dim > kMaxDim ||
        rows * vocab > kMaxLogits)
        return refuse(DLR_E_ARG, "dlr_head_logprob_workspace", "rows, vocab or dim is out of range");
    return dlr::head_workspace(rows, vocab, dim);
}

int dlr_head_logprob(int device, void *stream, const dlr_head *h, void *workspace, int64_t workspace_bytes,
                     float *logprob, float *lse) {
    const char *call = "dlr_head_logprob";
    if (!h) return refuse(DLR_E_ARG, call, "the descriptor is NULL");
    if (h->rows < 0 || h->rows > kMaxRows) return refuse(DLR_E_ARG, call, "rows must be 0 .. 2^31 - 1");
    if (h->vocab < 1 || h->vocab > kMaxClasses) return refuse(DLR_E_ARG, call, "vocab must be 1 .. 2^28");
    if (h->dim < 1 || h->dim > kMaxDim) return refuse(DLR_E_ARG, call, "dim must be 1 .. 2^20");
    if (h->rows * h->vocab > kMaxLogits) return refuse(DLR_E_ARG, call, "rows * vocab must be at most 2^44");
    if (h->dtype != DLR_DTYPE_BF16 && h->dtype != DLR_DTYPE_F16)
        return refuse(DLR_E_ARG, call, "dtype must be DLR_DTYPE_BF16 or DLR_DTYPE_F16");
    if (h->rows == 0) return DLR_OK;
    if (!h->hidden || !h->head) return refuse(DLR_E_ARG, call, "hidden or head is NULL");
    if (!aligned(h->hidden, 2) || !aligned(h->head, 2)) return refuse(DLR_E_ARG, call, "hidden or head is not aligned");
    if (h->hidden_stride < 0 || (h->rows > 1 && h->hidden_stride != 0 && h->hidden_stride < h->dim) ||
        !spans(h->rows, h->dim, h->hidden_stride, 2))
        return refuse(DLR_E_ARG, call, "hidden_stride must be 0 or at least dim");
    if (h->head_stride < 0 || (h->vocab > 1 && h->head_stride < h->dim) ||
        !spans(h->vocab, h->dim, h->head_stride, 2))
        return refuse(DLR_E_ARG, call, "head_stride must be at least dim");
    if (const char *why = check_target(h->target, h->target_bits, h->temperature)) return refuse(DLR_E_ARG, call, why);
    if (!logprob || !lse) return refuse(DLR_E_ARG, call, "logprob or lse is NULL");
    if (!floats({logprob, lse})) return refuse(DLR_E_ARG, call, "logprob or lse is not aligned");
    if (const char *why = check_workspace(workspace, workspace_bytes, dlr::head_workspace(h->rows, h->vocab, h->dim)))
        return refuse(DLR_E_ARG, call, why);
    DeviceScope d(device);
    if (d.error() != hipSuccess) return fail_hip(call, d.error());
    const hipError_t e = dlr::launch_head_logprob(static_cast<hipStream_t>(stream), *h, workspace, logprob, lse);
    return e == hipSuccess ? DLR_OK : fail_hip(call, e);
}

}  // extern "C"
