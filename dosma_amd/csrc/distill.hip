// distill.hip -- the divergence of a student's answers from a teacher's stored best ones, and its gradient, for gfx950.
//
//   teacher entries (i_k, v_k), k < K <= 64;  student p = softmax(z / T) over all categories
//   tail = 0:  q = softmax(v / T) over the entries,            L = sum_k q_k (log q_k - log p_{i_k})
//   tail = 1:  q_k = e^{v_k}, q_t = 1 - sum q_k, p_t = sum_{j not in i} p_j,   L = (the same sum) + q_t (log q_t - log p_t)
//   g_j = w / T [ Q p_j - sum_{k: i_k = j} q_k - [j not in i] q_t p_j / p_t ],   Q = sum_k q_k + q_t
#include "answers.h"

namespace qmri {
namespace {

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

__device__ __forceinline__ float load_value(const DistillK &k, long long i) {
    if (k.v_dtype == QMRI_F32) return static_cast<const float *>(k.values)[i];
    if (k.v_dtype == QMRI_F16) return to_f32(static_cast<const f16_t *>(k.values)[i]);
    return to_f32(static_cast<const bf16_t *>(k.values)[i]);
}

// The teacher's side of a row, one entry a lane: label (-1: empty slot), q and log q; the mass outside the entries.
struct Teacher {
    int idx;
    float q, lq;
    float rest, total;  // q_t, Q: the same in every lane
    bool any;
};
__device__ __forceinline__ Teacher teacher_wave(const DistillK &k, long long n, int lane, int cats) {
    Teacher t = {-1, 0.f, kNegInf, 0.f, 0.f, false};
    float v = kNegInf;
    if (lane < k.K) {
        const long long l = load_label(k.labels, k.l_kind, n * k.K + lane);
        if (l >= 0 && l < cats) {
            t.idx = (int)l;
            v = load_value(k, n * k.K + lane);
        }
    }
    const bool ok = t.idx >= 0;
    t.any = __ballot(ok) != 0ull;
    const float m = wave_max(v);
    if (k.tail) {
        t.lq = v;
        t.q = ok ? expf(v) : 0.f;
        // q_t = (1 - e^{v_max}) - the other entries: exact for a teacher that is sure of itself
        const unsigned long long at = __ballot(ok && v == m);
        const int first = at ? __ffsll(at) - 1 : 0;
        const float others = wave_sum(lane == first ? 0.f : t.q);
        const float rest = -expm1f(m) - others;
        t.rest = (!t.any || rest <= (float)k.K * 5.9604645e-8f) ? 0.f : rest;
        t.total = wave_sum(t.q) + t.rest;
    } else {
        const float d = (v - m) * k.g.invT;
        const float e = (ok && m > kNegInf) ? expf(d) : (v != v ? v : 0.f);
        const float s = wave_sum(e);
        if (s == 0.f) t.any = false;
        t.q = (ok && s != 0.f) ? e / s : 0.f;
        t.lq = d - logf(s);
        t.total = t.any ? 1.f : 0.f;
    }
    return t;
}

// One wave a row, any strides.
template <typename T>
__global__ __launch_bounds__(256) void distill_wave_kernel(const DistillK k) {
    __shared__ int s_idx[4][64];
    const LogitsK &g = k.g;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, cats = g.C + g.bg;
    const long long nw = (long long)gridDim.x * 4;
    for (long long n = (long long)blockIdx.x * 4 + w; n < g.rows; n += nw) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        const Teacher t = teacher_wave(k, n, lane, cats);
        s_idx[w][lane] = t.idx;
        wave_sync();
        float M = kNegInf;
        for (int j = lane; j < cats; j += 64) M = fmaxf(M, (g.bg && j == 0) ? 0.f : to_f32(z[(long long)(j - g.bg) * g.sc]));
        M = wave_max(M);
        float s = 0.f, st = 0.f;
        for (int j = lane; j < cats; j += 64) {
            const float v = (g.bg && j == 0) ? 0.f : to_f32(z[(long long)(j - g.bg) * g.sc]);
            const float e = v == kNegInf ? 0.f : exp2_hw((v - M) * g.c2);
            s += e;
            if (k.tail) {
                bool in = false;
                for (int q = 0; q < k.K; ++q) in |= s_idx[w][q] == j;
                if (!in) st += e;
            }
        }
        s = wave_sum(s);
        st = wave_sum(st);
        const bool empty = M == kNegInf && s == 0.f;
        const float ls = logf(s), lt = logf(st) - ls;
        float part = 0.f;
        if (t.idx >= 0) {
            const float v = (g.bg && t.idx == 0) ? 0.f : to_f32(z[(long long)(t.idx - g.bg) * g.sc]);
            const float lp = (v - M) * g.invT - ls;
            part = t.q == 0.f ? 0.f : t.q * (t.lq - lp);
        }
        float loss = wave_sum(part);
        if (k.tail && t.rest != 0.f) loss += t.rest * (logf(t.rest) - lt);
        if (lane == 0) {
            if (k.loss) k.loss[n] = (empty || !t.any) ? 0.f : loss;
            if (k.norm) {
                k.norm[2 * n] = ls != ls ? ls : M;
                k.norm[2 * n + 1] = ls;
            }
            if (k.log_tail) k.log_tail[n] = empty ? kNegInf : lt;
        }
        wave_sync();
    }
}

template <typename T>
__global__ __launch_bounds__(256) void distill_grad_wave_kernel(const DistillK k) {
    __shared__ int s_idx[4][64];
    __shared__ float s_q[4][64];
    const LogitsK &g = k.g;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, cats = g.C + g.bg;
    const long long nw = (long long)gridDim.x * 4;
    for (long long n = (long long)blockIdx.x * 4 + w; n < g.rows; n += nw) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        T *out = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi);
        const Teacher t = teacher_wave(k, n, lane, cats);
        s_idx[w][lane] = t.idx;
        s_q[w][lane] = t.q;
        wave_sync();
        const float M = k.norm[2 * n], ls = k.norm[2 * n + 1];
        const float f = k.g_loss[n] * g.invT;
        const float lt = (k.tail && t.rest != 0.f) ? k.log_tail[n] : 0.f;
        const bool zero = (M == kNegInf && !(ls != ls)) || !t.any;
        for (int c = lane; c < g.C; c += 64) {
            const float v = to_f32(z[(long long)c * g.sc]);
            const float lp = (v - M) * g.invT - ls, p = exp2_hw(lp * kLog2e);
            float qs = 0.f;
            bool in = false;
            for (int q = 0; q < k.K; ++q)
                if (s_idx[w][q] == c + g.bg) {
                    in = true;
                    qs += s_q[w][q];
                }
            float r = t.total * p - qs;
            if (!in && t.rest != 0.f && p != 0.f) r -= t.rest * exp2_hw((lp - lt) * kLog2e);
            out[(long long)c * k.gsc] = from_f32<T>(zero ? 0.f : r * f);
        }
        wave_sync();
    }
}

unsigned wave_grid(long long rows, int num_cu) {
    long long b = (rows + 3) / 4;
    const long long cap = (long long)num_cu * 32;
    return (unsigned)(b < cap ? b : cap);
}

}  // namespace

size_t distill_workspace_bytes(const DistillK &, int, int) { return 0; }

hipError_t distill_launch(const DistillK &k, int dtype, int num_cu, hipStream_t st) {
    (void)hipGetLastError();
    const dim3 g(wave_grid(k.g.rows, num_cu)), b(256);
    if (dtype == QMRI_F32) hipLaunchKernelGGL(distill_wave_kernel<float>, g, b, 0, st, k);
    else if (dtype == QMRI_F16) hipLaunchKernelGGL(distill_wave_kernel<f16_t>, g, b, 0, st, k);
    else hipLaunchKernelGGL(distill_wave_kernel<bf16_t>, g, b, 0, st, k);
    return hipGetLastError();
}

hipError_t distill_grad_launch(const DistillK &k, int dtype, int num_cu, hipStream_t st) {
    (void)hipGetLastError();
    const dim3 g(wave_grid(k.g.rows, num_cu)), b(256);
    if (dtype == QMRI_F32) hipLaunchKernelGGL(distill_grad_wave_kernel<float>, g, b, 0, st, k);
    else if (dtype == QMRI_F16) hipLaunchKernelGGL(distill_grad_wave_kernel<f16_t>, g, b, 0, st, k);
    else hipLaunchKernelGGL(distill_grad_wave_kernel<bf16_t>, g, b, 0, st, k);
    return hipGetLastError();
}

}  // namespace qmri
