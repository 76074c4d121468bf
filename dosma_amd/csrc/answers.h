// answers.h -- what the kernels on a network's answers share (label_scores.hip, distill.hip): the geometry of a batch of
// category scores, the running softmax statistics of a row and how two of them join.
#ifndef QMRI_ANSWERS_H
#define QMRI_ANSWERS_H

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "qmri.h"

namespace qmri {

// Row n of `rows` lies at z + (n / inner) * so + (n % inner) * si, its classes `sc` elements apart.  With `bg` an implicit
// category 0 of score 0 stands before the C classes: category = class + bg.
struct LogitsK {
    const void *z;
    long long rows, inner;
    long long so, si, sc;
    int C, bg;
    float c2;    // log2(e) / T: exp((z - M) / T) = exp2((z - M) * c2)
    float invT;  // 1 / T
};

struct ScoresK {
    LogitsK g;
    const void *labels;
    int l_kind;
    int top;
    long long ignore;
    float *log_prob, *entropy, *norm, *top_log_prob;
    int *top_label;
    // gradient: norm / entropy are inputs then
    const float *g_log_prob, *g_entropy;
    void *grad;
    long long gso, gsi, gsc;
    void *ws;  // workspace (the split rows of the forward pass)
};

struct DistillK {
    LogitsK g;
    const void *labels;  // [rows][K]
    const void *values;  // [rows][K]
    int l_kind, v_dtype;
    int K, tail;
    float *loss, *norm, *log_tail;
    const float *g_loss;
    void *grad;
    long long gso, gsi, gsc;
    void *ws;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_inff();

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    return static_cast<float>(v);
}
// 2-byte gradients are rounded once, to nearest even, from the 32-bit value
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    return static_cast<T>(v);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// kinds of QMRI_L_*: int32, uint8, int16, int64
__device__ __forceinline__ long long load_label(const void *p, int kind, long long i) {
    switch (kind) {
        case 0: return static_cast<const int *>(p)[i];
        case 1: return static_cast<const unsigned char *>(p)[i];
        case 2: return static_cast<const short *>(p)[i];
        default: return static_cast<const long long *>(p)[i];
    }
}

__device__ __forceinline__ long long row_base(const LogitsK &g, long long n, long long so, long long si) {
    if (g.inner >= g.rows) return n * si;
    // (a 64-bit division is some 100 instructions: rows that fit 32 bits take the short one)
    long long o;
    if (g.rows <= 0x7fffffffll) o = (unsigned)n / (unsigned)g.inner;
    else o = n / g.inner;
    return o * so + (n - o * g.inner) * si;
}

// Running statistics of a row or of a part of one: maximum m, s = sum exp2((z - m) c2), t = sum exp2((z - m) c2) (z - m) c2.
// Everything is held in 32 bits.  A part without any offered category is (-inf, 0, 0).
struct RowStat {
    float m, s, t;
};

// exponent of the change of reference from m to M >= m.  Clamped: -inf (nothing seen yet) times a zero sum must stay zero.
__device__ __forceinline__ float shift2(float m, float M, float c2) {
    return m == M ? 0.f : fmaxf((m - M) * c2, -1.0e4f);
}
__device__ __forceinline__ RowStat join(const RowStat &a, const RowStat &b, float c2) {
    RowStat r;
    r.m = fmaxf(a.m, b.m);
    const float da = shift2(a.m, r.m, c2), db = shift2(b.m, r.m, c2);
    const float fa = exp2_hw(da), fb = exp2_hw(db);
    r.s = a.s * fa + b.s * fb;
    r.t = fa * (a.t + da * a.s) + fb * (b.t + db * b.s);
    return r;
}

// what a wave's lanes have written to LDS is visible to its other lanes from here on
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// a better than b in the order of the alternatives: larger score, ties to the lower label
__device__ __forceinline__ bool better(float va, int ia, float vb, int ib) { return va > vb || (va == vb && ia < ib); }

hipError_t label_scores_launch(const ScoresK &k, int dtype, int num_cu, hipStream_t st);
size_t label_scores_workspace_bytes(const ScoresK &k, int dtype, int num_cu);
hipError_t label_scores_grad_launch(const ScoresK &k, int dtype, int num_cu, hipStream_t st);
hipError_t distill_launch(const DistillK &k, int dtype, int num_cu, hipStream_t st);
size_t distill_workspace_bytes(const DistillK &k, int dtype, int num_cu);
hipError_t distill_grad_launch(const DistillK &k, int dtype, int num_cu, hipStream_t st);

}  // namespace qmri
#endif
