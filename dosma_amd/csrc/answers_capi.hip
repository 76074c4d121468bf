// answers_capi.hip -- C entries of the operators on a network's answers (label_scores.hip, distill.hip): checks of the
// arguments, device and workspace handling, the host-array variants.
#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <numeric>

#include "answers.h"
#include "qmri_internal.h"

namespace {

int afail(int code, const char *fmt, ...) {
    char msg[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    qmri::set_last_error(msg);
    return code;
}

#define A_TRY(expr)                                                                            \
    do {                                                                                       \
        hipError_t e_ = (expr);                                                                \
        if (e_ != hipSuccess)                                                                  \
            return afail(e_ == hipErrorOutOfMemory ? QMRI_ERR_NOMEM : QMRI_ERR_HIP,            \
                         "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, __LINE__); \
    } while (0)
#define A_ARG(cond, ...)                                        \
    do {                                                        \
        if (!(cond)) return afail(QMRI_ERR_ARG, __VA_ARGS__);   \
    } while (0)

constexpr int kMaxDevices = 16;

// The caller's current device is put back on every way out: these entries are called from programs (torch) that keep one.
struct DeviceGuard {
    int before = -1;
    hipError_t set(int device) {
        int now = -1;
        hipError_t e = hipGetDevice(&now);
        if (e != hipSuccess || now == device) return e;
        e = hipSetDevice(device);
        if (e == hipSuccess) before = now;
        return e;
    }
    ~DeviceGuard() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

hipError_t compute_units(int device, int *out) {
    static std::atomic<int> known[kMaxDevices];
    int n = known[device].load(std::memory_order_relaxed);
    if (n == 0) {
        hipError_t e = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device);
        if (e != hipSuccess) return e;
        known[device].store(n, std::memory_order_relaxed);
    }
    *out = n;
    return hipSuccess;
}

struct Scratch {  // stream-ordered, given back to the pool on every way out
    void *p = nullptr;
    hipStream_t st = nullptr;
    ~Scratch() {
        if (p) (void)hipFreeAsync(p, st);
    }
};

// `given` if it is large enough, otherwise memory of the stream's pool; an allocation made while the stream is being captured
// would belong to the graph, so the caller has to bring the workspace then
int take_workspace(void *given, uint64_t given_bytes, size_t need, hipStream_t st, Scratch &s, void **out) {
    *out = nullptr;
    if (need == 0) return QMRI_OK;
    if (given) {
        A_ARG(given_bytes >= need, "workspace holds %llu bytes, %llu needed", (unsigned long long)given_bytes, (unsigned long long)need);
        A_ARG((reinterpret_cast<uintptr_t>(given) & 15) == 0, "workspace must be 16-byte aligned");
        *out = given;
        return QMRI_OK;
    }
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (st) A_TRY(hipStreamIsCapturing(st, &cs));
    A_ARG(cs == hipStreamCaptureStatusNone, "a captured call needs a workspace of %llu bytes", (unsigned long long)need);
    s.st = st;
    A_TRY(hipMallocAsync(&s.p, need, st));
    *out = s.p;
    return QMRI_OK;
}

int score_size(int dt) { return dt == QMRI_F32 ? 4 : (dt == QMRI_F16 || dt == QMRI_BF16) ? 2 : 0; }
int label_size(int kind) { return kind == QMRI_L_I32 ? 4 : kind == QMRI_L_U8 ? 1 : kind == QMRI_L_I16 ? 2 : kind == QMRI_L_I64 ? 8 : 0; }

int check_logits(const qmri_logits &l, int device, bool need_data) {
    A_ARG(score_size(l.dtype) != 0, "logits must be QMRI_F32, QMRI_F16 or QMRI_BF16, got dtype %d", l.dtype);
    A_ARG(l.rows >= 0, "rows < 0");
    A_ARG(l.classes >= 1 && l.classes <= (1 << 30), "classes must be 1 .. 2^30, got %d", l.classes);
    A_ARG(l.background == 0 || l.background == 1, "background must be 0 or 1");
    A_ARG(l.inner >= 1, "inner must be at least 1");
    A_ARG(l.stride_outer >= 0 && l.stride_inner >= 0 && l.stride_class >= 0, "negative stride");
    // (the kernels multiply by log2(e) / T in 32 bits)
    A_ARG(std::isfinite(l.temperature) && l.temperature >= 1e-30 && l.temperature <= 1e30, "temperature must be in [1e-30, 1e30]");
    A_ARG(device >= 0 && device < kMaxDevices, "bad device %d", device);
    A_ARG(!need_data || l.rows == 0 || l.data, "logits are NULL");
    return QMRI_OK;
}

// Two axes of n and m elements, s and t apart: do any i < n and j < m other than 0, 0 meet (i s = j t)?
bool axes_meet(int64_t n, int64_t s, int64_t m, int64_t t) {
    if (n <= 1 || m <= 1) return false;
    const int64_t g = std::gcd(s, t);
    return t / g < n && s / g < m;
}

int check_grad(const qmri_logits &l, const void *grad, int64_t so, int64_t si, int64_t sc) {
    A_ARG(l.rows == 0 || grad, "grad is NULL");
    const int64_t inner = l.inner < l.rows ? l.inner : l.rows, outer = l.rows == 0 ? 0 : (l.rows + inner - 1) / inner;
    A_ARG((l.classes == 1 || sc >= 1) && (inner <= 1 || si >= 1) && (outer <= 1 || so >= 1) && !axes_meet(l.classes, sc, inner, si) &&
              !axes_meet(l.classes, sc, outer, so) && !axes_meet(inner, si, outer, so),
          "grad must have a place of its own for every score (stride 0 or negative, or rows that meet)");
    return QMRI_OK;
}

qmri::LogitsK geometry(const qmri_logits &l) {
    qmri::LogitsK g;
    g.z = l.data;
    g.rows = l.rows;
    g.inner = l.inner;
    g.so = l.stride_outer;
    g.si = l.stride_inner;
    g.sc = l.stride_class;
    g.C = l.classes;
    g.bg = l.background;
    g.c2 = (float)(1.4426950408889634074 / l.temperature);
    g.invT = (float)(1.0 / l.temperature);
    qmri::set_division(g);
    return g;
}

int check_scores(const qmri_label_scores_args *a, bool grad, bool need_data) {
    A_ARG(a, "args is NULL");
    const int rc = check_logits(a->logits, a->device, need_data);
    if (rc != QMRI_OK) return rc;
    const qmri_logits &l = a->logits;
    A_ARG(!a->labels || label_size(a->l_kind), "unknown l_kind %d", a->l_kind);
    if (!grad) {
        A_ARG(a->top >= 0 && a->top <= QMRI_MAX_TOP, "top must be 0 .. %d, got %d", QMRI_MAX_TOP, a->top);
        A_ARG(a->top <= l.classes + l.background, "top = %d, but there are %d categories", a->top, l.classes + l.background);
        if (need_data && l.rows > 0) {
            A_ARG(a->top == 0 || (a->top_log_prob && a->top_label), "top_log_prob / top_label is NULL");
            A_ARG(!a->log_prob || a->labels, "log_prob needs labels");
        }
    } else if (l.rows > 0) {
        A_ARG(a->norm, "norm is NULL");
        A_ARG(!a->grad_log_prob || a->labels, "grad_log_prob needs labels");
        A_ARG(!a->grad_entropy || a->entropy, "grad_entropy needs entropy");
    }
    return grad ? check_grad(l, a->grad, a->grad_stride_outer, a->grad_stride_inner, a->grad_stride_class) : QMRI_OK;
}

qmri::ScoresK scores_args(const qmri_label_scores_args *a) {
    qmri::ScoresK k;
    std::memset(&k, 0, sizeof(k));
    k.g = geometry(a->logits);
    k.labels = a->labels;
    k.l_kind = a->l_kind;
    k.top = a->top;
    k.ignore = a->ignore_label;
    k.log_prob = a->log_prob;
    k.entropy = a->entropy;
    k.norm = a->norm;
    k.top_log_prob = a->top_log_prob;
    k.top_label = a->top_label;
    k.g_log_prob = a->grad_log_prob;
    k.g_entropy = a->grad_entropy;
    k.grad = a->grad;
    k.gso = a->grad_stride_outer;
    k.gsi = a->grad_stride_inner;
    k.gsc = a->grad_stride_class;
    return k;
}

int check_distill(const qmri_distill_args *a, bool grad, bool need_data) {
    A_ARG(a, "args is NULL");
    const int rc = check_logits(a->logits, a->device, need_data);
    if (rc != QMRI_OK) return rc;
    A_ARG(a->entries >= 1 && a->entries <= QMRI_MAX_TOP, "entries must be 1 .. %d, got %d", QMRI_MAX_TOP, a->entries);
    A_ARG(a->l_kind == QMRI_L_I32 || a->l_kind == QMRI_L_I64, "teacher labels must be int32 or int64");
    A_ARG(a->tail == 0 || a->tail == 1, "tail must be 0 or 1");
    A_ARG(a->tail ? a->v_dtype == QMRI_F32 : score_size(a->v_dtype) != 0,
          a->tail ? "with the tail the values are float32 log probabilities" : "values must be QMRI_F32, QMRI_F16 or QMRI_BF16");
    if (need_data && a->logits.rows > 0) {
        A_ARG(a->top_label && a->values, "top_label / values is NULL");
        if (grad) {
            A_ARG(a->norm && a->grad_loss, "norm / grad_loss is NULL");
            A_ARG(!a->tail || a->log_tail, "log_tail is NULL");
        }
    }
    return grad ? check_grad(a->logits, a->grad, a->grad_stride_outer, a->grad_stride_inner, a->grad_stride_class) : QMRI_OK;
}

qmri::DistillK distill_args(const qmri_distill_args *a) {
    qmri::DistillK k;
    std::memset(&k, 0, sizeof(k));
    k.g = geometry(a->logits);
    k.labels = a->top_label;
    k.values = a->values;
    k.l_kind = a->l_kind;
    k.v_dtype = a->v_dtype;
    k.K = a->entries;
    k.tail = a->tail;
    k.loss = a->loss;
    k.norm = a->norm;
    k.log_tail = a->log_tail;
    k.g_loss = a->grad_loss;
    k.grad = a->grad;
    k.gso = a->grad_stride_outer;
    k.gsi = a->grad_stride_inner;
    k.gsc = a->grad_stride_class;
    return k;
}

bool dense(const qmri_logits &l, int64_t si, int64_t sc) {
    return l.inner >= l.rows && (si == l.classes || l.rows <= 1) && (sc == 1 || l.classes == 1);
}

// A device copy of host memory (in), or device memory that is copied back (out).
struct Mirror {
    void *d = nullptr;
    ~Mirror() {
        if (d) (void)hipFree(d);
    }
    hipError_t in(const void *h, size_t bytes) {
        if (!h) return hipSuccess;
        hipError_t e = hipMalloc(&d, bytes);
        return e == hipSuccess ? hipMemcpy(d, h, bytes, hipMemcpyHostToDevice) : e;
    }
    hipError_t make(const void *h, size_t bytes) { return h ? hipMalloc(&d, bytes) : hipSuccess; }
    hipError_t out(void *h, size_t bytes) { return h ? hipMemcpy(h, d, bytes, hipMemcpyDeviceToHost) : hipSuccess; }
    template <typename T>
    T *as() const {
        return static_cast<T *>(d);
    }
};

}  // namespace

extern "C" {

int qmri_label_scores_workspace(const qmri_label_scores_args *a, uint64_t *bytes) {
    A_ARG(bytes, "bytes is NULL");
    *bytes = 0;
    const int rc = check_scores(a, false, false);
    if (rc != QMRI_OK) return rc;
    int cu = 0;
    A_TRY(compute_units(a->device, &cu));
    *bytes = qmri::label_scores_workspace_bytes(scores_args(a), a->logits.dtype, cu);
    return QMRI_OK;
}

int qmri_label_scores_device(const qmri_label_scores_args *a) {
    int rc = check_scores(a, false, true);
    if (rc != QMRI_OK || a->logits.rows == 0) return rc;
    DeviceGuard dev;
    A_TRY(dev.set(a->device));
    int cu = 0;
    A_TRY(compute_units(a->device, &cu));
    qmri::ScoresK k = scores_args(a);
    hipStream_t st = static_cast<hipStream_t>(a->stream);
    Scratch ws;
    rc = take_workspace(a->workspace, a->workspace_bytes, qmri::label_scores_workspace_bytes(k, a->logits.dtype, cu), st, ws, &k.ws);
    if (rc != QMRI_OK) return rc;
    A_TRY(qmri::label_scores_launch(k, a->logits.dtype, cu, st));
    return QMRI_OK;
}

int qmri_label_scores_grad_device(const qmri_label_scores_args *a) {
    const int rc = check_scores(a, true, true);
    if (rc != QMRI_OK || a->logits.rows == 0) return rc;
    DeviceGuard dev;
    A_TRY(dev.set(a->device));
    int cu = 0;
    A_TRY(compute_units(a->device, &cu));
    A_TRY(qmri::label_scores_grad_launch(scores_args(a), a->logits.dtype, cu, static_cast<hipStream_t>(a->stream)));
    return QMRI_OK;
}

int qmri_distill_workspace(const qmri_distill_args *a, uint64_t *bytes) {
    A_ARG(bytes, "bytes is NULL");
    *bytes = 0;
    const int rc = check_distill(a, false, false);
    if (rc != QMRI_OK) return rc;
    int cu = 0;
    A_TRY(compute_units(a->device, &cu));
    *bytes = qmri::distill_workspace_bytes(distill_args(a), a->logits.dtype, cu);
    return QMRI_OK;
}

int qmri_distill_device(const qmri_distill_args *a) {
    int rc = check_distill(a, false, true);
    if (rc != QMRI_OK || a->logits.rows == 0) return rc;
    DeviceGuard dev;
    A_TRY(dev.set(a->device));
    int cu = 0;
    A_TRY(compute_units(a->device, &cu));
    qmri::DistillK k = distill_args(a);
    hipStream_t st = static_cast<hipStream_t>(a->stream);
    Scratch ws;
    rc = take_workspace(a->workspace, a->workspace_bytes, qmri::distill_workspace_bytes(k, a->logits.dtype, cu), st, ws, &k.ws);
    if (rc != QMRI_OK) return rc;
    A_TRY(qmri::distill_launch(k, a->logits.dtype, cu, st));
    return QMRI_OK;
}

int qmri_distill_grad_device(const qmri_distill_args *a) {
    const int rc = check_distill(a, true, true);
    if (rc != QMRI_OK || a->logits.rows == 0) return rc;
    DeviceGuard dev;
    A_TRY(dev.set(a->device));
    int cu = 0;
    A_TRY(compute_units(a->device, &cu));
    A_TRY(qmri::distill_grad_launch(distill_args(a), a->logits.dtype, cu, static_cast<hipStream_t>(a->stream)));
    return QMRI_OK;
}

static int scores_host(const qmri_label_scores_args *a, bool grad) {
    int rc = check_scores(a, grad, true);
    if (rc != QMRI_OK || a->logits.rows == 0) return rc;
    const qmri_logits &l = a->logits;
    A_ARG(dense(l, l.stride_inner, l.stride_class) && (!grad || dense(l, a->grad_stride_inner, a->grad_stride_class)),
          "the host entry takes dense rows");
    DeviceGuard dev;
    A_TRY(dev.set(a->device));
    const size_t n = (size_t)l.rows, zb = n * l.classes * score_size(l.dtype);
    Mirror z, lab, lp, ent, norm, tv, ti, ga, gb, g;
    A_TRY(z.in(l.data, zb));
    if (a->labels) A_TRY(lab.in(a->labels, n * label_size(a->l_kind)));
    qmri_label_scores_args d = *a;
    d.logits.data = z.d;
    d.labels = lab.d;
    d.workspace = nullptr;
    d.stream = nullptr;
    if (grad) {
        A_TRY(norm.in(a->norm, n * 8));
        A_TRY(ent.in(a->entropy, n * 4));
        A_TRY(ga.in(a->grad_log_prob, n * 4));
        A_TRY(gb.in(a->grad_entropy, n * 4));
        A_TRY(g.make(a->grad, zb));
        d.grad_log_prob = ga.as<float>();
        d.grad_entropy = gb.as<float>();
        d.grad = g.d;
    } else {
        A_TRY(lp.make(a->log_prob, n * 4));
        A_TRY(ent.make(a->entropy, n * 4));
        A_TRY(norm.make(a->norm, n * 8));
        if (a->top) {
            A_TRY(tv.make(a->top_log_prob, n * a->top * 4));
            A_TRY(ti.make(a->top_label, n * a->top * 4));
        }
        d.log_prob = lp.as<float>();
        d.top_log_prob = tv.as<float>();
        d.top_label = ti.as<int32_t>();
    }
    d.entropy = ent.as<float>();
    d.norm = norm.as<float>();
    rc = grad ? qmri_label_scores_grad_device(&d) : qmri_label_scores_device(&d);
    if (rc != QMRI_OK) return rc;
    if (grad) {
        A_TRY(g.out(a->grad, zb));
    } else {
        A_TRY(lp.out(a->log_prob, n * 4));
        A_TRY(ent.out(a->entropy, n * 4));
        A_TRY(norm.out(a->norm, n * 8));
        if (a->top) {
            A_TRY(tv.out(a->top_log_prob, n * a->top * 4));
            A_TRY(ti.out(a->top_label, n * a->top * 4));
        }
    }
    A_TRY(hipStreamSynchronize(nullptr));
    return QMRI_OK;
}

int qmri_label_scores_host(const qmri_label_scores_args *a) { return scores_host(a, false); }
int qmri_label_scores_grad_host(const qmri_label_scores_args *a) { return scores_host(a, true); }

static int distill_host(const qmri_distill_args *a, bool grad) {
    int rc = check_distill(a, grad, true);
    if (rc != QMRI_OK || a->logits.rows == 0) return rc;
    const qmri_logits &l = a->logits;
    A_ARG(dense(l, l.stride_inner, l.stride_class) && (!grad || dense(l, a->grad_stride_inner, a->grad_stride_class)),
          "the host entry takes dense rows");
    DeviceGuard dev;
    A_TRY(dev.set(a->device));
    const size_t n = (size_t)l.rows, zb = n * l.classes * score_size(l.dtype), e = n * a->entries;
    Mirror z, lab, val, loss, norm, tail, gl, g;
    A_TRY(z.in(l.data, zb));
    A_TRY(lab.in(a->top_label, e * label_size(a->l_kind)));
    A_TRY(val.in(a->values, e * score_size(a->v_dtype)));
    qmri_distill_args d = *a;
    d.logits.data = z.d;
    d.top_label = lab.d;
    d.values = val.d;
    d.workspace = nullptr;
    d.stream = nullptr;
    if (grad) {
        A_TRY(norm.in(a->norm, n * 8));
        if (a->tail) A_TRY(tail.in(a->log_tail, n * 4));
        A_TRY(gl.in(a->grad_loss, n * 4));
        A_TRY(g.make(a->grad, zb));
        d.grad_loss = gl.as<float>();
        d.grad = g.d;
    } else {
        A_TRY(loss.make(a->loss, n * 4));
        A_TRY(norm.make(a->norm, n * 8));
        A_TRY(tail.make(a->log_tail, n * 4));
        d.loss = loss.as<float>();
    }
    d.norm = norm.as<float>();
    d.log_tail = tail.as<float>();
    rc = grad ? qmri_distill_grad_device(&d) : qmri_distill_device(&d);
    if (rc != QMRI_OK) return rc;
    if (grad) {
        A_TRY(g.out(a->grad, zb));
    } else {
        A_TRY(loss.out(a->loss, n * 4));
        A_TRY(norm.out(a->norm, n * 8));
        A_TRY(tail.out(a->log_tail, n * 4));
    }
    A_TRY(hipStreamSynchronize(nullptr));
    return QMRI_OK;
}

int qmri_distill_host(const qmri_distill_args *a) { return distill_host(a, false); }
int qmri_distill_grad_host(const qmri_distill_args *a) { return distill_host(a, true); }

}  // extern "C"
