// label_scores.hip -- log probability of a given label, entropy and best alternatives of every row of category scores, and
// the gradient of the first two, for gfx950.
//
//   M = max z, s = sum exp((z - M) / T), log p_j = (z_j - M) / T - ln s, H = ln s - sum exp(d_j) d_j / s  (d_j = (z_j - M) / T)
//   g_j = [ a (delta_j,label - p_j) - b p_j (log p_j + H) ] / T
#include "answers.h"

namespace qmri {
namespace {

__device__ __forceinline__ RowStat wave_join(RowStat r, float c2) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const RowStat b = {__shfl_xor(r.m, o), __shfl_xor(r.s, o), __shfl_xor(r.t, o)};
        r = join(r, b, c2);
    }
    return r;
}

template <typename T>
__device__ __forceinline__ float category(const LogitsK &g, const T *z, int j) {
    return (g.bg && j == 0) ? 0.f : to_f32(z[(long long)(j - g.bg) * g.sc]);
}

// One wave a row, any strides: the row is read once for the statistics and once more for each alternative.
template <typename T>
__global__ __launch_bounds__(256) void scores_wave_kernel(const ScoresK k) {
    const LogitsK &g = k.g;
    const int lane = threadIdx.x & 63, cats = g.C + g.bg;
    const long long nw = (long long)gridDim.x * 4;
    for (long long n = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); n < g.rows; n += nw) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        RowStat r = {kNegInf, 0.f, 0.f};
        for (int j = lane; j < cats; j += 64) {
            const float v = category(g, z, j);
            const float M = fmaxf(r.m, v), sh = shift2(r.m, M, g.c2), f = exp2_hw(sh);
            const float d = v == M ? (v - v) : (v - M) * g.c2, e = v == kNegInf ? 0.f : exp2_hw(d);
            r.t = f * (r.t + sh * r.s) + e * fmaxf(d, -200.f);
            r.s = f * r.s + e;
            r.m = M;
        }
        r = wave_join(r, g.c2);
        const bool empty = r.m == kNegInf && r.s == 0.f;
        const float l2s = __log2f(r.s), ls = l2s * kLn2;
        if (lane == 0) {
            if (k.norm) {
                k.norm[2 * n] = ls != ls ? ls : r.m;
                k.norm[2 * n + 1] = ls;
            }
            if (k.entropy) k.entropy[n] = empty ? 0.f : (l2s - r.t / r.s) * kLn2;
            if (k.log_prob) {
                const long long l = load_label(k.labels, k.l_kind, n);
                float lp;
                if (l == k.ignore) lp = 0.f;
                else if (l < 0 || l >= cats) lp = __builtin_nanf("");
                else if (empty) lp = kNegInf;
                else lp = (category(g, z, (int)l) - r.m) * g.invT - ls;
                k.log_prob[n] = lp;
            }
        }
        float pv = __builtin_inff();
        int pi = -1;
        for (int q = 0; q < k.top; ++q) {
            float bv = kNegInf;
            int bi = -1;
            for (int j = lane; j < cats; j += 64) {
                const float v = category(g, z, j);
                if (v > kNegInf && better(pv, pi, v, j) && (bi < 0 || better(v, j, bv, bi))) {
                    bv = v;
                    bi = j;
                }
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const float ov = __shfl_xor(bv, o);
                const int oi = __shfl_xor(bi, o);
                if (oi >= 0 && (bi < 0 || better(ov, oi, bv, bi))) {
                    bv = ov;
                    bi = oi;
                }
            }
            if (lane == 0) {
                k.top_label[n * k.top + q] = bi;
                k.top_log_prob[n * k.top + q] = (bi < 0 && !(r.s != r.s)) ? kNegInf : (bv - r.m) * g.invT - ls;
            }
            if (bi < 0) {  // nothing left: the further slots stay empty too
                pv = kNegInf;
                pi = -1;
            } else {
                pv = bv;
                pi = bi;
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void scores_grad_wave_kernel(const ScoresK k) {
    const LogitsK &g = k.g;
    const int lane = threadIdx.x & 63, cats = g.C + g.bg;
    const long long nw = (long long)gridDim.x * 4;
    for (long long n = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); n < g.rows; n += nw) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        T *out = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi);
        const float M = k.norm[2 * n], ls = k.norm[2 * n + 1];
        float a = 0.f, b = 0.f, H = 0.f;
        long long l = -1;
        if (k.g_log_prob) {
            l = load_label(k.labels, k.l_kind, n);
            if (l == k.ignore) l = -1;
            else {
                a = k.g_log_prob[n];
                if (l < 0 || l >= cats) a = __builtin_nanf("");
            }
        }
        if (k.g_entropy) {
            b = k.g_entropy[n];
            H = k.entropy[n];
        }
        const bool empty = M == kNegInf && !(ls != ls);
        for (int c = lane; c < g.C; c += 64) {
            const float v = to_f32(z[(long long)c * g.sc]);
            const float lp = (v - M) * g.invT - ls, p = exp2_hw(lp * kLog2e);
            float r = -a * p - b * (p == 0.f ? 0.f : p * (lp + H));
            if (c + g.bg == l) r += a;
            out[(long long)c * k.gsc] = from_f32<T>(empty ? 0.f : r * g.invT);
        }
    }
}

unsigned wave_grid(long long rows, int num_cu) {
    long long b = (rows + 3) / 4;
    const long long cap = (long long)num_cu * 32;
    return (unsigned)(b < cap ? b : cap);
}

}  // namespace

size_t label_scores_workspace_bytes(const ScoresK &, int, int) { return 0; }

hipError_t label_scores_launch(const ScoresK &k, int dtype, int num_cu, hipStream_t st) {
    (void)hipGetLastError();
    const dim3 g(wave_grid(k.g.rows, num_cu)), b(256);
    if (dtype == QMRI_F32) hipLaunchKernelGGL(scores_wave_kernel<float>, g, b, 0, st, k);
    else if (dtype == QMRI_F16) hipLaunchKernelGGL(scores_wave_kernel<f16_t>, g, b, 0, st, k);
    else hipLaunchKernelGGL(scores_wave_kernel<bf16_t>, g, b, 0, st, k);
    return hipGetLastError();
}

hipError_t label_scores_grad_launch(const ScoresK &k, int dtype, int num_cu, hipStream_t st) {
    (void)hipGetLastError();
    const dim3 g(wave_grid(k.g.rows, num_cu)), b(256);
    if (dtype == QMRI_F32) hipLaunchKernelGGL(scores_grad_wave_kernel<float>, g, b, 0, st, k);
    else if (dtype == QMRI_F16) hipLaunchKernelGGL(scores_grad_wave_kernel<f16_t>, g, b, 0, st, k);
    else hipLaunchKernelGGL(scores_grad_wave_kernel<bf16_t>, g, b, 0, st, k);
    return hipGetLastError();
}

}  // namespace qmri
