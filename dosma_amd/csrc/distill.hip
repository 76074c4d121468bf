// distill.hip -- the divergence of a student's answers from a teacher's stored best ones, and its gradient, for gfx950.
//
//   teacher entries (i_k, v_k), k < K <= 64;  student p = softmax(z / T) over all categories
//   tail = 0:  q = softmax(v / T) over the entries,            L = sum_k q_k (log q_k - log p_{i_k})
//   tail = 1:  q_k = e^{v_k}, q_t = 1 - sum q_k, p_t = sum_{j not in i} p_j,   L = (the same sum) + q_t (log q_t - log p_t)
//   g_j = w / T [ Q p_j - sum_{k: i_k = j} q_k - [j not in i] q_t p_j / p_t ],   Q = sum_k q_k + q_t
//
// The student's scores are read once (and the gradient written once); p_t is summed over the categories outside the entries,
// never as a difference.  Who owns a row is as in label_scores.hip: a lane (up to 8 classes, or classes that do not lie
// together), 2 .. 64 lanes (up to 1024 contiguous classes), a wave, a block or several blocks (more).  The times at the kernels are
// those of whole calls on an MI355X, where a large copy moves 4.8 to 5.0 TB/s.
#include "answers.h"

namespace qmri {
namespace {

__device__ __forceinline__ float load_value(const DistillK &k, long long i) {
    if (k.v_dtype == QMRI_F32) return static_cast<const float *>(k.values)[i];
    if (k.v_dtype == QMRI_F16) return to_f32(static_cast<const f16_t *>(k.values)[i]);
    return to_f32(static_cast<const bf16_t *>(k.values)[i]);
}
// entry q of row n: its label (-1: empty slot) and value
__device__ __forceinline__ int load_entry(const DistillK &k, long long n, int q, int cats, float &v) {
    const long long l = load_label(k.labels, k.l_kind, n * k.K + q);
    v = load_value(k, n * k.K + q);
    return (l >= 0 && l < cats) ? (int)l : -1;
}

// ---- the teacher's side of a row ----------------------------------------------------------------------------------------------
// An entry's weight is q = exp2((v - m) * c2) * scale, its logarithm (v - m) * (1 / T) + lscale: with the tail m = 0, T = 1 and
// scale = 1, without it m is the largest value and scale = 1 / sum.
struct Teacher {
    float m, c2, invT, scale, lscale;
    float rest, total;  // q_t, Q
    bool some;          // any entry that counts
};
__device__ __forceinline__ float weight(const Teacher &t, float v) { return exp2_hw((v - t.m) * t.c2) * t.scale; }
__device__ __forceinline__ float log_weight(const Teacher &t, float v) { return (v - t.m) * t.invT + t.lscale; }
// 1 - e^x for x <= 0 (and a negative number beyond): near 0 the series, whose first term left out is below 2e-8 of the sum at -0.35
__device__ __forceinline__ float one_minus_exp(float x) {
    const float p = 1.f + x * 0.5f * (1.f + x * (1.f / 3.f) * (1.f + x * 0.25f * (1.f + x * 0.2f * (1.f + x * (1.f / 6.f) * (1.f + x * (1.f / 7.f))))));
    return fabsf(x) < 0.35f ? -x * p : 1.f - exp2_hw(x * kLog2e);
}
__device__ __forceinline__ float ln(float x) { return __builtin_amdgcn_logf(x) * kLn2; }
// From what the entries give together: their number, largest value m, sum of exp2((v - base) c2), base = m or (tail) 0, and in
// the tail the sum without one entry of the largest value.
__device__ __forceinline__ Teacher teacher_of(const DistillK &k, bool any, float m, float sum, float others) {
    Teacher t;
    if (k.tail) {
        t.m = 0.f;
        t.c2 = kLog2e;
        t.invT = 1.f;
        t.scale = 1.f;
        t.lscale = 0.f;
        // 1 - sum q as (1 - e^{v_max}) - the others: nothing cancels for a teacher that is sure of itself
        const float rest = one_minus_exp(m) - others;
        t.rest = (any && !(rest <= (float)k.K * 5.9604645e-8f)) ? rest : 0.f;
        t.total = sum + t.rest;
        t.some = any;
    } else {
        t.m = m;
        t.c2 = k.g.c2;
        t.invT = k.g.invT;
        t.scale = 1.f / sum;
        t.lscale = -ln(sum);
        t.rest = 0.f;
        t.some = any && sum != 0.f;
        t.total = t.some ? 1.f : 0.f;
    }
    return t;
}
__device__ __forceinline__ float teacher_term(const DistillK &k, float v, float m) {
    return k.tail ? exp2_hw(v * kLog2e) : (m == kNegInf ? (v != v ? v : 0.f) : exp2_hw((v - m) * k.g.c2));
}
// by a wave that holds an entry a lane (l < 0: none)
__device__ __forceinline__ Teacher teacher_wave(const DistillK &k, int l, float v) {
    const bool ok = l >= 0;
    const float m = group_max<64>(ok ? v : kNegInf);
    const float e = ok ? teacher_term(k, v, m) : 0.f;
    const unsigned long long at = __ballot(ok && v == m);
    const int first = at ? __ffsll(at) - 1 : -1;
    return teacher_of(k, __ballot(ok) != 0ull, m, group_sum<64>(e), group_sum<64>((int)(threadIdx.x & 63) == first ? 0.f : e));
}
// N entries of a row in registers: both loads are issued before either is looked at.
template <int N, typename L, typename V, int K>
__device__ __forceinline__ void load_pairs(const void *labels, const void *values, long long n, int cats, int (&l)[K], float (&v)[K]) {
    struct {
        L v[N];
    } rl;
    struct {
        V v[N];
    } rv;
    __builtin_memcpy(&rl, static_cast<const L *>(labels) + n * N, sizeof(rl));
    __builtin_memcpy(&rv, static_cast<const V *>(values) + n * N, sizeof(rv));
#pragma unroll
    for (int q = 0; q < N; ++q) {
        l[q] = rl.v[q] >= 0 && rl.v[q] < (L)cats ? (int)rl.v[q] : -1;
        v[q] = to_f32(rv.v[q]);
    }
}
template <int N, int K>
__device__ __forceinline__ void load_exactly(const DistillK &k, long long n, int cats, int (&l)[K], float (&v)[K]) {
    if (k.l_kind == QMRI_L_I32) {
        if (k.v_dtype == QMRI_F32) load_pairs<N, int, float>(k.labels, k.values, n, cats, l, v);
        else if (k.v_dtype == QMRI_F16) load_pairs<N, int, f16_t>(k.labels, k.values, n, cats, l, v);
        else load_pairs<N, int, bf16_t>(k.labels, k.values, n, cats, l, v);
    } else {
        if (k.v_dtype == QMRI_F32) load_pairs<N, long long, float>(k.labels, k.values, n, cats, l, v);
        else if (k.v_dtype == QMRI_F16) load_pairs<N, long long, f16_t>(k.labels, k.values, n, cats, l, v);
        else load_pairs<N, long long, bf16_t>(k.labels, k.values, n, cats, l, v);
    }
}
template <int K>
__device__ __forceinline__ void load_entries(const DistillK &k, long long n, int cats, int (&l)[K], float (&v)[K]) {
    // (the usual case by itself and first: of the ways below each gives its registers to a common set in the end, which waits)
    if (k.K == K && k.l_kind == QMRI_L_I32 && k.v_dtype == QMRI_F32) {
        __builtin_memcpy(&l, static_cast<const int *>(k.labels) + n * K, sizeof(l));
        __builtin_memcpy(&v, static_cast<const float *>(k.values) + n * K, sizeof(v));
#pragma unroll
        for (int q = 0; q < K; ++q) l[q] = (unsigned)l[q] < (unsigned)cats ? l[q] : -1;
        return;
    }
#pragma unroll
    for (int q = 0; q < K; ++q) {
        l[q] = -1;
        v[q] = 0.f;
    }
    if constexpr (K == 2) {
        if (k.K == 2) load_exactly<2>(k, n, cats, l, v);
        else load_exactly<1>(k, n, cats, l, v);
    } else if constexpr (K == 4) {
        if (k.K == 4) load_exactly<4>(k, n, cats, l, v);
        else load_exactly<3>(k, n, cats, l, v);
    } else {
        if (k.K == 8) load_exactly<8>(k, n, cats, l, v);
        else if (k.K == 7) load_exactly<7>(k, n, cats, l, v);
        else if (k.K == 6) load_exactly<6>(k, n, cats, l, v);
        else load_exactly<5>(k, n, cats, l, v);
    }
}
template <int K>
__device__ __forceinline__ Teacher teacher_lane(const DistillK &k, const int (&l)[K], const float (&v)[K]) {
    float m = kNegInf, sum = 0.f, others = 0.f;
    bool any = false, left_out = false;
#pragma unroll
    for (int q = 0; q < K; ++q)
        if (l[q] >= 0) {
            m = maxn(m, v[q]);
            any = true;
        }
#pragma unroll
    for (int q = 0; q < K; ++q) {
        const float e = l[q] >= 0 ? teacher_term(k, v[q], m) : 0.f;
        const bool first = l[q] >= 0 && v[q] == m && !left_out;
        sum += e;
        others += first ? 0.f : e;
        left_out |= first;
    }
    return teacher_of(k, any, m, sum, others);
}
// by one lane, the entries read from memory
__device__ __forceinline__ Teacher teacher_read(const DistillK &k, long long n, int cats) {
    float m = kNegInf;
    bool any = false;
    for (int q = 0; q < k.K; ++q) {
        float v;
        if (load_entry(k, n, q, cats, v) >= 0) {
            m = maxn(m, v);
            any = true;
        }
    }
    float sum = 0.f, others = 0.f;
    bool left_out = false;
    for (int q = 0; q < k.K; ++q) {
        float v;
        if (load_entry(k, n, q, cats, v) < 0) continue;
        const float e = teacher_term(k, v, m);
        sum += e;
        if (v == m && !left_out) left_out = true;
        else others += e;
    }
    return teacher_of(k, any, m, sum, others);
}

// v, or 0 where bit i of `marks` is set (two instructions: a sign extended from the bit, and a mask)
__device__ __forceinline__ float unless(float v, unsigned marks, int i) {
    return __int_as_float(__float_as_int(v) & __builtin_amdgcn_sbfe((int)~marks, i, 1));
}

// ---- results of a row -----------------------------------------------------------------------------------------------------------
// s: of all categories, so: of those outside the entries, both relative to reference(M)
struct Student {
    float ref, ls;
    bool empty;
};
__device__ __forceinline__ Student student_of(float M, float s) { return {reference(M), ln(s), s == 0.f}; }
__device__ __forceinline__ float entry_loss(const DistillK &k, const Teacher &t, const Student &p, float v, float z) {
    const float q = weight(t, v);
    const float lp = (z == kNegInf && p.ls == p.ls) ? kNegInf : (z - p.ref) * k.g.invT - p.ls;
    return q == 0.f ? 0.f : q * (log_weight(t, v) - lp);
}
template <typename T>
__device__ __forceinline__ float gather(const LogitsK &g, const T *z, int l) {
    return l < g.bg ? 0.f : to_f32(z[(long long)(l - g.bg) * g.sc]);
}
// ln of the sum outside the entries, relative to p.ref.  A student that leaves less than 2^-100 out there (its terms vanish next to
// the maximum's) has it summed again relative to the largest outside, where anyone asks: the G lanes read the row twice more.  Beyond 64
// categories each score is compared with the entries in memory, which a batch of such rows pays for (temperature 1, the best 120 above
// the others): 200000 x 500 in bf16 with 3 entries 0.58 ms instead of 0.08, 1024 x 100003 with 8 entries 5.6 ms and with 64 entries 33 ms
// instead of 0.04, planes of 117 classes with 5 entries 0.39 ms instead of 0.02 (147456 rows).
template <int G, typename T>
__device__ __forceinline__ float log_outside(const DistillK &k, long long n, const T *z, int gl, int cats, const Student &p, const Teacher &t, float so) {
    if (!k.tail) return 0.f;
    if (!(so < 7.888609e-31f) || (t.rest == 0.f && !k.log_tail) || p.empty) return ln(so);
    unsigned long long mask = 0ull;  // the entries of up to 64 categories
    if (cats <= 64) {
        float v;
        for (int q = 0; q < k.K; ++q) {
            const int l = load_entry(k, n, q, cats, v);
            mask |= l >= 0 ? 1ull << l : 0ull;
        }
        if (mask == ~0ull >> (64 - cats)) return kNegInf;
    }
    auto score = [&](int j) {
        const float z_j = gather(k.g, z, j);
        if (z_j == kNegInf) return kNegInf;
        if (cats <= 64) return mask >> j & 1ull ? kNegInf : z_j;
        float v;
        for (int q = 0; q < k.K; ++q)
            if (load_entry(k, n, q, cats, v) == j) return kNegInf;
        return z_j;
    };
    float m = kNegInf, s = 0.f;
    for (int j = gl; j < cats; j += G) m = maxn(m, score(j));
    m = group_max<G>(m);
    for (int j = gl; j < cats; j += G) s += exp2_hw((score(j) - reference(m)) * k.g.c2);
    s = group_sum<G>(s);
    return s == 0.f ? kNegInf : (m - p.ref) * k.g.invT + ln(s);
}
__device__ __forceinline__ void write_row(const DistillK &k, long long n, float M, float lso, const Student &p, const Teacher &t, float loss) {
    const float lt = p.empty ? kNegInf : lso - p.ls;
    if (k.tail && t.rest != 0.f) loss += t.rest * (ln(t.rest) - lt);
    if (k.loss) k.loss[n] = (p.empty || !t.some) ? 0.f : loss;
    if (k.norm) *reinterpret_cast<float2 *>(k.norm + 2 * n) = make_float2(p.ls != p.ls ? p.ls : M, p.ls);
    if (k.log_tail) k.log_tail[n] = lt;
}

// ---- small: one lane a row ----------------------------------------------------------------------------------------------------
// K: entries held in registers (as many or fewer of them in use); 0: any number, read again where they are needed.  Bound by memory:
// 384 x 384 x 160 rows of 4 fp32 classes and a background, two entries and the tail, 171 us (5.0 TB/s), the gradient 303 us (5.0 TB/s).
template <typename T, int N>
__device__ __forceinline__ void load_small(const LogitsK &g, const T *z, T (&v)[N]) {
    if (g.sc == 1) {
        __builtin_memcpy(&v, z, sizeof(v));
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = z[j * g.sc];
    }
}
template <typename T, int N, int K>
__global__ __launch_bounds__(256) void distill_small_kernel(const DistillK k) {
    const LogitsK &g = k.g;
    const int cats = N + g.bg;
    const long long stride = (long long)gridDim.x * 256;
    for (long long n = (long long)blockIdx.x * 256 + threadIdx.x; n < g.rows; n += stride) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        T raw[N];
        load_small<T, N>(g, z, raw);
        int el[K > 0 ? K : 1];
        float ev[K > 0 ? K : 1];
        if (K) load_entries(k, n, cats, el, ev);
        const Teacher t = K ? teacher_lane(k, el, ev) : teacher_read(k, n, cats);
        // x[0]: the implicit category, or one that is not offered; x[j + 1]: class j
        float x[N + 1], e[N + 1], s = 0.f, so = 0.f;
        x[0] = g.bg ? 0.f : kNegInf;
#pragma unroll
        for (int j = 0; j < N; ++j) x[j + 1] = to_f32(raw[j]);
        float M = x[0];
#pragma unroll
        for (int j = 1; j <= N; ++j) M = maxn(M, x[j]);
        const float ref = reference(M);
#pragma unroll
        for (int j = 0; j <= N; ++j) {
            e[j] = exp2_hw((x[j] - ref) * g.c2);
            s += e[j];
        }
        const Student p = student_of(M, s);
        unsigned in = 0u;
        float loss = 0.f;
        auto entry = [&](int l, float v) {
            if (l < 0) return;
            float zl = 0.f;
            const int at = l + 1 - g.bg;
            in |= 1u << at;
#pragma unroll
            for (int j = 0; j <= N; ++j) zl = at == j ? x[j] : zl;
            loss += entry_loss(k, t, p, v, zl);
        };
        if (K) {
#pragma unroll
            for (int q = 0; q < K; ++q) entry(el[q], ev[q]);
        } else {
            for (int q = 0; q < k.K; ++q) {
                float v;
                const int l = load_entry(k, n, q, cats, v);
                entry(l, v);
            }
        }
#pragma unroll
        for (int j = 0; j <= N; ++j) so += unless(e[j], in, j);
        write_row(k, n, M, log_outside<1>(k, n, z, 0, cats, p, t, so), p, t, loss);
    }
}

// What a row's gradient needs: g_j = f (total p_j - [outside] rest p_j / p_t) for the others, f (total p_j - sum q) for an entry's label
struct GradRow {
    float M, l2s, total, share, f;  // share = q_t / p_t
    bool zero;
};
__device__ __forceinline__ GradRow grad_row(const DistillK &k, long long n, const Teacher &t) {
    GradRow r;
    const float2 nm = *reinterpret_cast<const float2 *>(k.norm + 2 * n);
    r.M = nm.x;
    r.l2s = nm.y * kLog2e;
    r.total = t.total;
    // q_t / p_t reaches e^80 and more where the student leaves next to nothing outside: it is kept as a logarithm, in units of 2
    r.share = (k.tail && t.rest != 0.f) ? __builtin_amdgcn_logf(t.rest) - k.log_tail[n] * kLog2e : kNegInf;
    r.f = k.g_loss[n] * k.g.invT;
    r.zero = nm.x == kNegInf || !t.some;
    return r;
}
__device__ __forceinline__ float grad_outside(const GradRow &r, float c2, float v) {
    const float d = (v - r.M) * c2 - r.l2s, p = exp2_hw(d);
    const float o = v == kNegInf ? 0.f : exp2_hw(d + r.share);  // (the share of a row with nothing outside is infinite)
    return r.zero ? 0.f : r.f * fmaf(r.total, p, -o);
}
// q: the sum of the weights of the score's entries, negative where it has none
__device__ __forceinline__ float grad_either(const GradRow &r, float c2, float v, float q) {
    const float d = (v - r.M) * c2 - r.l2s, p = exp2_hw(d);
    const float o = v == kNegInf ? 0.f : exp2_hw(d + r.share);
    return r.zero ? 0.f : r.f * fmaf(r.total, p, -(q < 0.f ? o : q));
}
__device__ __forceinline__ float grad_inside(const GradRow &r, float c2, float v, float qs) {
    const float p = exp2_hw((v - r.M) * c2 - r.l2s);
    return r.zero ? 0.f : r.f * fmaf(r.total, p, -qs);
}

template <typename T, int N, int K>
__global__ __launch_bounds__(256) void distill_grad_small_kernel(const DistillK k) {
    const LogitsK &g = k.g;
    const int cats = N + g.bg;
    const long long stride = (long long)gridDim.x * 256;
    for (long long n = (long long)blockIdx.x * 256 + threadIdx.x; n < g.rows; n += stride) {
        T raw[N];
        load_small<T, N>(g, static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si), raw);
        T *out = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi);
        int el[K > 0 ? K : 1];
        float ev[K > 0 ? K : 1];
        if (K) load_entries(k, n, cats, el, ev);
        const Teacher t = K ? teacher_lane(k, el, ev) : teacher_read(k, n, cats);
        const GradRow r = grad_row(k, n, t);
        unsigned in = 0u;
        float qs[N];
#pragma unroll
        for (int j = 0; j < N; ++j) qs[j] = 0.f;
        auto entry = [&](int l, float v) {
            if (l < g.bg) return;
            const float w = weight(t, v);
            in |= 1u << (l - g.bg);
#pragma unroll
            for (int j = 0; j < N; ++j) qs[j] += l - g.bg == j ? w : 0.f;
        };
        if (K) {
#pragma unroll
            for (int q = 0; q < K; ++q) entry(el[q], ev[q]);
        } else {
            for (int q = 0; q < k.K; ++q) {
                float v;
                const int l = load_entry(k, n, q, cats, v);
                entry(l, v);
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float v = to_f32(raw[j]);
            raw[j] = from_f32<T>((in >> j) & 1u ? grad_inside(r, g.c2, v, qs[j]) : grad_outside(r, g.c2, v));
        }
        if (k.gsc == 1) {
            __builtin_memcpy(out, &raw, sizeof(raw));
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) out[j * k.gsc] = raw[j];
        }
    }
}

// ---- group: G lanes a row, 16 scores a lane ------------------------------------------------------------------------------------
// E > 0: a lane holds E entries in registers, every G-th of the row; the labels are marked in LDS, a 16-bit word for each lane's
// scores.  E 0: the same with any number of entries, in LDS.  E < 0: up to -E entries, all of them in every lane -- the exponents
// and logarithms of a few entries, worked out by all lanes alike, are less than the exchanges between them.
// More entries than registers are given to lie in LDS: those of a block's rows are one piece of memory, read side by side.  A row
// every K | 1 words (lanes that walk through rows of their own do not meet in a bank), rows behind the last are empty.
//
// 200000 x 500, three entries and the tail: fp32 91 us (4.5 TB/s), bf16 79 us (2.6 TB/s): a row's labels, its entries' scores and the
// exchanges for teacher, sums and loss follow each other, and eight waves a SIMD (64 registers) do not hide all of it.
struct StagedEntries {
    int *l;
    float *v;
    __device__ __forceinline__ void to_row(int row, int K) {
        l += row * (K | 1);
        v += row * (K | 1);
    }
    // the sum of the weights (v holds them then) of all entries with label x, in their order
    __device__ __forceinline__ float weights_of(int x, int K) const {
        float s = 0.f;
        int o = 0;
        for (; o + 8 <= K; o += 8) {
            int i[8];
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                i[e] = l[o + e];
                w[e] = v[o + e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) s += i[e] == x ? w[e] : 0.f;
        }
        for (; o < K; ++o) s += l[o] == x ? v[o] : 0.f;
        return s;
    }
};
constexpr size_t staged_bytes(int rows, int K) { return (size_t)rows * (K | 1) * 8; }
template <int THREADS, typename L, typename V>
__device__ __forceinline__ void stage_from(const StagedEntries &s, const L *labels, const V *values, int K, int all, long long left, int cats) {
    for (int i0 = threadIdx.x; i0 < all; i0 += 8 * THREADS) {  // (eight of each under way together)
        L l[8];
        V v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const long long i = i0 + e * THREADS, at = i < left ? i : left - 1;
            l[e] = labels[at];
            v[e] = values[at];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = i0 + e * THREADS, r = (unsigned)i / (unsigned)K, at = r * (K | 1) + i - r * K;
            if (i >= all) continue;
            s.l[at] = i < left && l[e] >= 0 && l[e] < (L)cats ? (int)l[e] : -1;
            s.v[at] = to_f32(v[e]);
        }
    }
}
template <int THREADS>
__device__ __forceinline__ StagedEntries stage_entries(const DistillK &k, void *lds, long long n0, int rows, int cats) {
    const StagedEntries s = {static_cast<int *>(lds), static_cast<float *>(lds) + rows * (k.K | 1)};
    const long long first = n0 * k.K, left = (k.g.rows - n0) * k.K;
    __syncthreads();  // (the block's last rows have been worked on)
    auto from = [&](const auto *labels, const auto *values) { stage_from<THREADS>(s, labels + first, values + first, k.K, rows * k.K, left, cats); };
    auto typed = [&](const auto *labels) {
        if (k.v_dtype == QMRI_F32) from(labels, static_cast<const float *>(k.values));
        else if (k.v_dtype == QMRI_F16) from(labels, static_cast<const f16_t *>(k.values));
        else from(labels, static_cast<const bf16_t *>(k.values));
    };
    if (k.l_kind == QMRI_L_I32) typed(static_cast<const int *>(k.labels));
    else typed(static_cast<const long long *>(k.labels));
    __syncthreads();
    return s;
}
template <int G, int V>
__device__ __forceinline__ void place_of(int c, int &owner, int &bit) {
    const int vec = c / V;
    owner = (int)(threadIdx.x / G) * G + vec % G;
    bit = (vec / G) * V + c % V;
}
template <int G, int E>
struct GroupEntries {
    int l[E > 0 ? E : 1];
    float v[E > 0 ? E : 1];
    const DistillK &k;
    StagedEntries at;  // E 0: the row's
    int gl;
    __device__ __forceinline__ GroupEntries(const DistillK &k_, long long n, int gl_, int cats, StagedEntries at_) : k(k_), at(at_), gl(gl_) {
        if constexpr (E > 0) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int q = gl + e * G;
                l[e] = -1;
                v[e] = 0.f;
                if (q < k.K) l[e] = load_entry(k, n, q, cats, v[e]);
            }
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        if constexpr (E > 0) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (l[e] >= 0) f(l[e], v[e]);
        } else {
            for (int q = gl; q < k.K; q += G)
                if (at.l[q] >= 0) f(at.l[q], at.v[q]);
        }
    }
    // which of the lane's scores are entries' (bits: LDS), and whether the implicit category is one
    template <int V>
    __device__ __forceinline__ unsigned marks(unsigned *bits, bool &back) const {
        float b = 0.f;
        if ((threadIdx.x & 1) == 0) bits[threadIdx.x >> 1] = 0u;
        wave_sync();
        each([&](int i, float) {
            if (i < k.g.bg) {
                b = 1.f;
            } else {
                int owner, bit;
                place_of<G, V>(i - k.g.bg, owner, bit);
                atomicOr(&bits[owner >> 1], 1u << ((owner & 1) * 16 + bit));
            }
        });
        wave_sync();
        const unsigned in = bits[threadIdx.x >> 1] >> ((threadIdx.x & 1) * 16) & 0xffffu;
        wave_sync();
        back = group_max<G>(b) > 0.f;
        return in;
    }
    // f(label, value, score): the scores of the entries in registers, or of 4, are under way together
    template <typename T, typename F>
    __device__ __forceinline__ void each_score(const T *z, F f) const {
        const int bg = k.g.bg;
        if constexpr (E > 0) {
            unsigned w[E];
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = load_bits(z + (l[e] > bg ? l[e] - bg : 0));
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (l[e] >= 0) f(l[e], v[e], l[e] < bg ? 0.f : widen<T>(w[e]));
        } else {
            for (int q0 = gl; q0 < k.K; q0 += 4 * G) {
                unsigned w[4];
                int i[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    i[e] = q0 + e * G < k.K ? at.l[q0 + e * G] : -1;
                    w[e] = load_bits(z + (i[e] > bg ? i[e] - bg : 0));
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i[e] >= 0) f(i[e], at.v[q0 + e * G], i[e] < bg ? 0.f : widen<T>(w[e]));
            }
        }
    }
    __device__ __forceinline__ Teacher teacher() const {
        float m = kNegInf, cnt = 0.f, sum = 0.f, others = 0.f;
        each([&](int, float x) {
            m = maxn(m, x);
            cnt = 1.f;
        });
        m = group_max<G>(m);
        const bool any = group_max<G>(cnt) > 0.f;
        bool left_out = false;
        each([&](int, float x) {
            const float e = teacher_term(k, x, m);
            sum += e;
            if (x == m && !left_out) left_out = true;
            else others += e;
        });
        // one entry of the largest value is left out, not one a lane
        const int one = group_min<G>(left_out ? gl : 0x7fffffff);
        if (left_out && one != gl) others += teacher_term(k, m, m);
        return teacher_of(k, any, m, group_sum<G>(sum), group_sum<G>(others));
    }
    __device__ __forceinline__ float total(float part) const { return group_sum<G>(part); }  // of what each gave
};
template <int G, int K>
struct AllEntries {
    int l[K];
    float v[K];
    const DistillK &k;
    __device__ __forceinline__ AllEntries(const DistillK &k_, long long n, int, int cats, StagedEntries) : k(k_) { load_entries(k, n, cats, l, v); }
    template <int V>
    __device__ __forceinline__ unsigned marks(unsigned *, bool &back) const {
        unsigned in = 0u;
        back = false;
#pragma unroll
        for (int q = 0; q < K; ++q) {
            int owner, bit;
            place_of<G, V>(l[q] - k.g.bg, owner, bit);
            const bool there = l[q] >= k.g.bg;
            back |= l[q] == 0 && !there;
            in |= there && owner == (int)threadIdx.x ? 1u << bit : 0u;
        }
        return in;
    }
    template <typename T, typename F>
    __device__ __forceinline__ void each_score(const T *z, F f) const {
        const int bg = k.g.bg;
        unsigned w[K];
#pragma unroll
        for (int q = 0; q < K; ++q) w[q] = load_bits(z + (l[q] > bg ? l[q] - bg : 0));
#pragma unroll
        for (int q = 0; q < K; ++q)
            if (l[q] >= 0) f(l[q], v[q], l[q] < bg ? 0.f : widen<T>(w[q]));
    }
    __device__ __forceinline__ Teacher teacher() const { return teacher_lane(k, l, v); }
    __device__ __forceinline__ float total(float part) const { return part; }
};
template <int G, int E>
using EntriesOf = std::conditional_t<(E < 0), AllEntries<G, E < 0 ? -E : 1>, GroupEntries<G, E < 0 ? 1 : E>>;
template <typename T, int G, int E>
__global__ __launch_bounds__(256, sizeof(T) == 4 || E == 0 ? 6 : 8) void distill_group_kernel(const DistillK k) {
    extern __shared__ float s_entries[];  // E 0
    __shared__ unsigned s_bits[128];
    const LogitsK &g = k.g;
    constexpr int V = kVec<T>, NV = 16 / V, ROWS = 256 / G;
    const int gl = threadIdx.x % G, cats = g.C + g.bg;
    for (long long n0 = (long long)blockIdx.x * ROWS; n0 < g.rows; n0 += (long long)gridDim.x * ROWS) {
        // (groups behind the last row work on it too and write nothing: the lane exchanges want whole waves)
        const long long nr = n0 + threadIdx.x / G;
        const bool live = nr < g.rows;
        const long long n = live ? nr : g.rows - 1;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        Vec<T> raw[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * G + gl) * V;
            raw[i] = load_vec(z + j - vec_back<T>(g.C - j));
        }
        StagedEntries staged = {nullptr, nullptr};
        if constexpr (E == 0) {
            staged = stage_entries<256>(k, s_entries, n0, ROWS, cats);
            staged.to_row(threadIdx.x / G, k.K);
        }
        const EntriesOf<G, E> entries(k, n, gl, cats, staged);
        unsigned in = 0u;
        bool back_in = false;  // the implicit category is an entry
        if (k.tail) in = entries.template marks<V>(s_bits, back_in);
        const Teacher t = entries.teacher();
        float x[16];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int back = vec_back<T>(g.C - (i * G + gl) * V);
            // (with more than 8 G scores in a row the first half of the vectors is whole)
            const Vec<T> v = G > 2 && 2 * i < NV ? raw[i] : drop_front(raw[i], back < V ? back : V);
#pragma unroll
            for (int e = 0; e < V; ++e) x[i * V + e] = get(v, e);
        }
        const float xb = (g.bg && gl == 0) ? 0.f : kNegInf;
        const float M = group_max<G>(maxn(max_of(x), xb)), ref = reference(M);
        float e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = exp2_hw((x[i] - ref) * g.c2);
        const float eb = exp2_hw((xb - ref) * g.c2);
        const float s = group_sum<G>(tree_sum(e) + eb);
        float so = 0.f;
        if (k.tail) {
#pragma unroll
            for (int i = 0; i < 16; ++i) e[i] = unless(e[i], in, i);
            so = group_sum<G>(tree_sum(e) + (back_in ? 0.f : eb));
        }
        const Student p = student_of(M, s);
        float loss = 0.f;
        entries.each_score(z, [&](int, float v, float zl) { loss += entry_loss(k, t, p, v, zl); });
        loss = entries.total(loss);
        const float lso = log_outside<G>(k, n, z, gl, cats, p, t, so);
        if (live && gl == 0) write_row(k, n, M, lso, p, t, loss);
    }
}

// The weights of the scores' entries lie in LDS, a column of 16 for a lane (-1: no entry); a row's last vector, moved to the front
// where it would end behind the row, finds its own in a column of the row's.  (The entries' scores written over after the others
// wait for the stores: 60 classes in fp32, six entries, 260 us and 218.)  200000 x 500, three entries and the tail: fp32 152 us (5.3 TB/s),
// bf16 107 us (3.8 TB/s).
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void distill_grad_group_kernel(const DistillK k) {
    constexpr int V = kVec<T>, NV = 16 / V, ROWS = 256 / G, COLS = 256 + ROWS;
    extern __shared__ float s_entries[];  // E 0
    __shared__ int s_l[E > 0 ? ROWS * ((G * E) | 1) : 1];  // entry q of a row at row * (G E | 1) + q
    __shared__ float s_q[E > 0 ? ROWS * ((G * E) | 1) : 1];
    __shared__ float s_w[16][COLS];
    const LogitsK &g = k.g;
    const int gl = threadIdx.x % G, cats = g.C + g.bg, row = threadIdx.x / G;
    for (long long n0 = (long long)blockIdx.x * ROWS; n0 < g.rows; n0 += (long long)gridDim.x * ROWS) {
        const long long nr = n0 + row;
        const bool live = nr < g.rows;
        const long long n = live ? nr : g.rows - 1;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        T *out = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi);
        Vec<T> x[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * G + gl) * V;
            x[i] = load_vec(z + j - vec_back<T>(g.C - j));
        }
        StagedEntries at = {nullptr, nullptr};
        if constexpr (E == 0) {
            at = stage_entries<256>(k, s_entries, n0, ROWS, cats);
            at.to_row(row, k.K);
        }
        const EntriesOf<G, E> entries(k, n, gl, cats, at);
        const Teacher t = entries.teacher();
        const GradRow r = grad_row(k, n, t);
#pragma unroll
        for (int i = 0; i < 16; ++i) s_w[i][threadIdx.x] = -1.f;
        for (int e = gl; e < V; e += G) s_w[e][256 + row] = -1.f;
        // the same label twice: the sum of all its entries, in their order
        const int last = g.C - V;  // the first class of the row's last vector
        if constexpr (E < 0) {
            wave_sync();
#pragma unroll
            for (int q = 0; q < -E; ++q) {
                const int c = entries.l[q] - g.bg;
                if (entries.l[q] < 0 || c < 0) continue;
                const float w = weight(t, entries.v[q]);
                int owner, bit;
                place_of<G, V>(c, owner, bit);
                if (owner == (int)threadIdx.x) s_w[bit][owner] = maxn(s_w[bit][owner], 0.f) + w;
                if (gl == 0 && c >= last) s_w[c - last][256 + row] = maxn(s_w[c - last][256 + row], 0.f) + w;
            }
        } else {
            // (the weights of a row's entries in one place)
            if constexpr (E > 0) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    s_l[row * ((G * E) | 1) + gl + e * G] = entries.l[e];
                    s_q[row * ((G * E) | 1) + gl + e * G] = entries.l[e] >= 0 ? weight(t, entries.v[e]) : 0.f;
                }
                at = {s_l + row * ((G * E) | 1), s_q + row * ((G * E) | 1)};
            } else {
                for (int q = gl; q < k.K; q += G) at.v[q] = at.l[q] >= 0 ? weight(t, at.v[q]) : 0.f;
            }
            wave_sync();
            if constexpr (G == 2) {  // (both lanes go through all entries)
                for (int q = 0; q < k.K; ++q) {
                    const int c = at.l[q] - g.bg;
                    if (at.l[q] < 0 || c < 0) continue;
                    const float w = at.v[q];
                    int owner, bit;
                    place_of<G, V>(c, owner, bit);
                    if (owner == (int)threadIdx.x) s_w[bit][owner] = maxn(s_w[bit][owner], 0.f) + w;
                    if (gl == 0 && c >= last) s_w[c - last][256 + row] = maxn(s_w[c - last][256 + row], 0.f) + w;
                }
            } else {
                entries.each([&](int l, float) {
                    const int c = l - g.bg;
                    if (c < 0) return;
                    const float qs = at.weights_of(l, k.K);
                    int owner, bit;
                    place_of<G, V>(c, owner, bit);
                    s_w[bit][owner] = qs;
                    if (c >= last) s_w[c - last][256 + row] = qs;
                });
            }
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * G + gl) * V, back = vec_back<T>(g.C - j);
            const float *w = back ? &s_w[0][256 + row] : &s_w[i * V][threadIdx.x];
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = grad_either(r, g.c2, get(x[i], e), w[e * COLS]);
            // (scores that another lane has too get the same value from both)
            if (live && j < g.C) store_vec(out + j - back, pack_vec<T>(y));
        }
        wave_sync();
    }
}

// ---- block: W waves a segment of a row -----------------------------------------------------------------------------------------
// The tail's sum leaves the entries' labels out: a bit a score in LDS, looked up a vector at a time.  Bound by memory with the row's
// beginning (its marks) and end (its loss) beside: 2048 x 65537 in bf16, 64 entries and the tail, 70 us (3.8 TB/s); 8192 x 16385 71 us.
constexpr int kLongest = 131072;  // scores of a segment then: 16 KB of marks

// wave 0, one entry a lane: the loss of a finished row
template <typename T>
__device__ __forceinline__ void finish_row(const DistillK &k, long long n, const T *z, float M, float s, float so) {
    const int lane = threadIdx.x & 63, cats = k.g.C + k.g.bg;
    float v = 0.f;
    const int l = lane < k.K ? load_entry(k, n, lane, cats, v) : -1;
    const float zl = l >= 0 ? gather(k.g, z, l) : 0.f;
    const Teacher t = teacher_wave(k, l, v);
    const Student p = student_of(M, s);
    float loss = l >= 0 ? entry_loss(k, t, p, v, zl) : 0.f;
    loss = group_sum<64>(loss);
    const float lso = log_outside<64>(k, n, z, lane, cats, p, t, so);
    if (lane == 0) write_row(k, n, M, lso, p, t, loss);
}

// x without the marked scores
template <int N>
__device__ __forceinline__ void add_outside(Running &r, const float (&x)[N], float c2, unsigned in) {
    raise<false>(r, max_of(x), c2);
    float e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = exp2_hw(fmaf(x[i], c2, -r.R));
    const float s = tree_sum(e);
    r.s += s;
    if (in) {
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = unless(e[i], in, i);
        r.t += tree_sum(e);
    } else {
        r.t += s;
    }
}
// 4-byte scores want 80 registers (4096 x 32000: 99 us, 121 with 64, which spill in the loop); 2-byte ones take 64 although 24 bytes a lane
// spill then, once a row outside the loop (10 MB for 2048 rows of 65537): with 72 or 80 they are slower.
template <typename T, bool TAIL, int W>
__global__ __launch_bounds__(64 * W, sizeof(T) == 4 ? 6 : 8) void distill_block_kernel(const DistillK k, const Cut cut) {
    __shared__ RowStat s_stat[W];
    extern __shared__ unsigned s_bits[];  // TAIL: cut.len bits
    __shared__ int s_back;
    const LogitsK &g = k.g;
    constexpr int V = kVec<T>, TILE = 1024;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), cats = g.C + g.bg;
    const long long work = g.rows * cut.segs;
    for (long long item = blockIdx.x; item < work; item += gridDim.x) {
        const long long n = cut.segs == 1 ? item : item / cut.segs;
        const int seg = cut.segs == 1 ? 0 : (int)(item - n * cut.segs);
        const int c0 = seg * cut.len, c1 = c0 + cut.len < g.C ? c0 + cut.len : g.C;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        int c = c0 + w * TILE;
        Tile<T> next;
        if (c < c1) next = load_tile(z + c, c1 - c);
        if (TAIL) {
            for (int i = threadIdx.x; i < (c1 - c0 + 31) / 32; i += 64 * W) s_bits[i] = 0u;
            if (threadIdx.x == 0) s_back = 0;
            __syncthreads();
            if ((int)threadIdx.x < k.K) {
                float v;
                const int l = load_entry(k, n, threadIdx.x, cats, v), j = l - g.bg - c0;
                if (l >= 0 && l < g.bg) s_back = 1;
                else if (l >= 0 && j >= 0 && j < c1 - c0) atomicOr(&s_bits[j >> 5], 1u << (j & 31));
            }
            __syncthreads();
        }
        // t holds the sum outside the entries here
        Running r = no_scores();
        const bool back = g.bg && seg == 0 && w == 0;
        if (back && lane == 0) r = {0.f, 0.f, 1.f, (TAIL && s_back) ? 0.f : 1.f};
        for (; c < c1; c += W * TILE) {
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = get(next.v[i / V], i % V);
            if (c + W * TILE < c1) next = load_tile(z + c + W * TILE, c1 - c - W * TILE);
            unsigned in = 0u;
            if (TAIL) {
#pragma unroll
                for (int u = 0; u < 16 / V; ++u) {
                    const int j = c + u * 64 * V + lane * V - c0;
                    in |= (j < c1 - c0 ? s_bits[j >> 5] >> (j & 31) & ((1u << V) - 1u) : 0u) << (u * V);
                }
            }
            add_outside(r, x, g.c2, in);
        }
        const float M = group_max<64>(r.m), ref = reference(M);
        RowStat st = {M, ref, 0.f, 0.f};
        if (far_scores(M, g.c2)) {  // (see answers.h)
            float s = 0.f, so = 0.f;
            for (int t0 = c0 + w * TILE; t0 < c1; t0 += W * TILE)
                for (int j = t0 + lane; j < t0 + TILE && j < c1; j += 64) {
                    const float e = exp2_hw((to_f32(z[j]) - ref) * g.c2);
                    s += e;
                    if (!TAIL || !(s_bits[(j - c0) >> 5] >> ((j - c0) & 31) & 1u)) so += e;
                }
            if (back && lane == 0) {
                const float e = exp2_hw((0.f - ref) * g.c2);
                s += e;
                if (!(TAIL && s_back)) so += e;
            }
            st.s = group_sum<64>(s);
            st.t = group_sum<64>(so);
        } else {
            float d;
            const float f = to_reference(r, M, g.c2, d);
            st.s = group_sum<64>(r.s * f);
            st.t = TAIL ? group_sum<64>(r.t * f) : 0.f;
        }
        if (lane == 0) s_stat[w] = st;
        __syncthreads();
        if (w == 0) {
            float MM = s_stat[0].m, s = 0.f, so = 0.f;
#pragma unroll
            for (int o = 1; o < W; ++o) MM = maxn(MM, s_stat[o].m);
            const float rr = reference(MM);
#pragma unroll
            for (int o = 0; o < W; ++o) {
                const float f = s_stat[o].ref == rr ? 1.f : exp2_hw(maxn((s_stat[o].ref - rr) * g.c2, -1.0e4f));
                s += s_stat[o].s * f;
                so += s_stat[o].t * f;
            }
            if (cut.segs > 1) {
                if (lane == 0) static_cast<float4 *>(k.ws)[item] = make_float4(MM, s, so, 0.f);
            } else {
                finish_row(k, n, z, MM, s, so);
            }
        }
        __syncthreads();
    }
}

// The segments' parts of a row together: one wave a row.
template <typename T>
__global__ __launch_bounds__(64) void distill_join_kernel(const DistillK k, const Cut cut) {
    const LogitsK &g = k.g;
    for (long long n = blockIdx.x; n < g.rows; n += gridDim.x) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        const float4 *p = static_cast<const float4 *>(k.ws) + n * cut.segs;
        float m = kNegInf;
        for (int q = threadIdx.x; q < cut.segs; q += 64) m = maxn(m, p[q].x);
        const float M = group_max<64>(m), ref = reference(M);
        float s = 0.f, so = 0.f;
        for (int q = threadIdx.x; q < cut.segs; q += 64) {
            const float4 a = p[q];
            const float r = reference(a.x), f = r == ref ? 1.f : exp2_hw(maxn((r - ref) * g.c2, -1.0e4f));
            s += a.y * f;
            so += a.z * f;
        }
        finish_row(k, n, z, M, group_sum<64>(s), group_sum<64>(so));
    }
}

// W waves take a segment of a row, 16 scores a lane at a time, as if none of them were an entry's label; those few are
// written over at the end, when the block's other stores have arrived.  2048 x 65537 in bf16 with 64 entries: 137 us (3.9 TB/s); 8192 x
// 8192 with five 53 us (5.0 TB/s).
template <typename T, int W>
__global__ __launch_bounds__(64 * W) void distill_grad_block_kernel(const DistillK k, const Cut cut) {
    constexpr int V = kVec<T>, NV = 16 / V, TILE = 1024 * W;
    __shared__ GradRow s_row;
    const LogitsK &g = k.g;
    for (long long item = blockIdx.x; item < g.rows * cut.segs; item += gridDim.x) {
        const long long n = cut.segs == 1 ? item : item / cut.segs;
        const int c0 = cut.segs == 1 ? 0 : (int)(item - n * cut.segs) * cut.len, c1 = c0 + cut.len < g.C ? c0 + cut.len : g.C;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        T *out = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi);
        Vec<T> nx[NV];
        auto fetch = [&](int c) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int j = c + (i * 64 * W + (int)threadIdx.x) * V;
                nx[i] = load_vec(z + j - vec_back<T>(g.C - j));  // (lanes behind the row: its last vector)
            }
        };
        fetch(c0);
        int mine = -1;  // wave 0: the class of a lane's entry if it lies in this segment, and its gradient
        T value = static_cast<T>(0.f);
        if (threadIdx.x < 64) {
            const int lane = threadIdx.x;
            float v = 0.f;
            const int l = lane < k.K ? load_entry(k, n, lane, g.C + g.bg, v) : -1, c = l - g.bg;
            const bool here = l >= 0 && c >= c0 && c < c1;
            const float zl = here ? to_f32(z[c]) : 0.f;
            const Teacher t = teacher_wave(k, l, v);
            const GradRow r = grad_row(k, n, t);
            if (lane == 0) s_row = r;
            const float q = l >= 0 ? weight(t, v) : 0.f;
            float qs = 0.f;  // (the same label twice: each of its lanes has the sum of all its entries, in their order)
            for (int o = 0; o < k.K; ++o) {
                const float oq = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(q), o));
                qs += __builtin_amdgcn_readlane(l, o) == l ? oq : 0.f;
            }
            if (here) {
                mine = c;
                value = from_f32<T>(grad_inside(r, g.c2, zl, qs));
            }
        }
        __syncthreads();
        const GradRow r = s_row;
        for (int c = c0; c < c1; c += TILE) {
            Vec<T> now[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) now[i] = nx[i];
            if (c + TILE < c1) fetch(c + TILE);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int j = c + (i * 64 * W + (int)threadIdx.x) * V, back = vec_back<T>(g.C - j);
                if (j >= c1) continue;
                float y[V];
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = grad_outside(r, g.c2, get(now[i], e));
                // (the row's last vector, moved to the front: what lies before j is another lane's)
                if (back == 0) store_vec(out + j, pack_vec<T>(y));
                else store_end(out + j - back, y, back);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (mine >= 0) out[mine] = value;
    }
}

// ---- planes: one lane a row, more than 8 classes that do not lie together ------------------------------------------------------
// K: entries in registers, as in small; 0: any number in LDS (blocks of one wave then).  8 x 384 x 384 rows of 60 classes in f16, five
// entries and the tail: 63 us (3.1 TB/s), bound by the entries' scores, each a line of its own, and the vector unit.
template <int K>
struct LaneEntries {
    int l[K > 0 ? K : 1];
    float v[K > 0 ? K : 1];
    const DistillK &k;
    StagedEntries at;  // K 0: the row's
    __device__ __forceinline__ LaneEntries(const DistillK &k_, long long n, int cats, StagedEntries at_) : k(k_), at(at_) {
        if constexpr (K > 0) load_entries(k, n, cats, l, v);
    }
    // f(label, value) for every entry that counts
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        if constexpr (K > 0) {
#pragma unroll
            for (int q = 0; q < K; ++q)
                if (l[q] >= 0) f(l[q], v[q]);
        } else {
            for (int q = 0; q < k.K; ++q)
                if (at.l[q] >= 0) f(at.l[q], at.v[q]);
        }
    }
    // f(label, value, score): the scores of up to 8 entries are under way together (an empty slot reads the first class's)
    template <typename T, typename F>
    __device__ __forceinline__ void each_score(const T *z, F f) const {
        const LogitsK &g = k.g;
        if constexpr (K > 0) {
            unsigned w[K];
#pragma unroll
            for (int q = 0; q < K; ++q) w[q] = load_bits(z + (l[q] > g.bg ? l[q] - g.bg : 0) * g.sc);
#pragma unroll
            for (int q = 0; q < K; ++q)
                if (l[q] >= 0) f(l[q], v[q], l[q] < g.bg ? 0.f : widen<T>(w[q]));
        } else {
            for (int q0 = 0; q0 < k.K; q0 += 8) {
                unsigned w[8];
                int i[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    i[q] = q0 + q < k.K ? at.l[q0 + q] : -1;
                    w[q] = load_bits(z + (i[q] > g.bg ? i[q] - g.bg : 0) * g.sc);
                }
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (i[q] >= 0) f(i[q], at.v[q0 + q], i[q] < g.bg ? 0.f : widen<T>(w[q]));
            }
        }
    }
    __device__ __forceinline__ Teacher teacher() const {
        if constexpr (K > 0) {
            return teacher_lane(k, l, v);
        } else {
            float m = kNegInf, sum = 0.f, others = 0.f;
            bool any = false, left_out = false;
            each([&](int, float x) {
                m = maxn(m, x);
                any = true;
            });
            each([&](int, float x) {
                const float e = teacher_term(k, x, m);
                sum += e;
                if (x == m && !left_out) left_out = true;
                else others += e;
            });
            return teacher_of(k, any, m, sum, others);
        }
    }
    // the values become weights
    __device__ __forceinline__ void to_weights(const Teacher &t) {
        if constexpr (K > 0) {
#pragma unroll
            for (int q = 0; q < K; ++q) v[q] = weight(t, v[q]);
        } else {
            for (int q = 0; q < k.K; ++q) at.v[q] = weight(t, at.v[q]);
        }
    }
    // which of the 32 categories from c are entries
    __device__ __forceinline__ unsigned marks(int c) const {
        unsigned in = 0u;
        each([&](int i, float) { in |= (unsigned)(i - c) < 32u ? 1u << (i - c) : 0u; });
        return in;
    }
};
template <int K>
constexpr int kPlaneThreads = K > 0 ? 256 : 64;
// CH: classes in flight (a divisor of 32).
template <typename T, int K, int CH>
__global__ __launch_bounds__(kPlaneThreads<K>) void distill_planes_kernel(const DistillK k) {
    extern __shared__ float s_entries[];  // K 0
    constexpr int B = kPlaneThreads<K>;
    const LogitsK &g = k.g;
    const int cats = g.C + g.bg;
    for (long long n0 = (long long)blockIdx.x * B; n0 < g.rows; n0 += (long long)gridDim.x * B) {
        const long long n = n0 + threadIdx.x;
        StagedEntries at = {nullptr, nullptr};
        if constexpr (K == 0) {
            at = stage_entries<B>(k, s_entries, n0, B, cats);
            at.to_row(threadIdx.x, k.K);
        }
        if (n >= g.rows) continue;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si), *p = z;
        unsigned next[CH];
        load_classes(p, g.sc, g.C, next);
        const LaneEntries<K> entries(k, n, cats, at);
        Running r = no_scores();  // (t: the sum outside the entries)
        if (g.bg) {
            const float x[1] = {0.f};
            add_outside(r, x, g.c2, k.tail ? entries.marks(0) & 1u : 0u);
        }
        unsigned in = 0u;
        for (int c = 0; c < g.C; c += CH) {
            if (k.tail && (c & 31) == 0) in = entries.marks(c + g.bg);
            float x[CH];
#pragma unroll
            for (int i = 0; i < CH; ++i) x[i] = widen<T>(next[i]);
            p += CH * g.sc;
            if (c + CH < g.C) load_classes(p, g.sc, g.C - c - CH, next);
            add_outside(r, x, g.c2, (in >> (c & 31)) & ((1u << CH) - 1u));
        }
        float sum = 0.f, so = 0.f;
        if (far_scores(r.m, g.c2)) {  // (see answers.h)
            for (int j = 0; j < cats; ++j) {
                if (k.tail && (j & 31) == 0) in = entries.marks(j);
                const float e = exp2_hw((gather(g, z, j) - reference(r.m)) * g.c2);
                sum += e;
                so += k.tail && (in >> (j & 31)) & 1u ? 0.f : e;
            }
        } else {
            float d;
            const float f = to_reference(r, r.m, g.c2, d);
            sum = r.s * f;
            so = r.t * f;
        }
        const Student st = student_of(r.m, sum);
        const Teacher t = entries.teacher();
        float loss = 0.f;
        entries.each_score(z, [&](int, float v, float zl) { loss += entry_loss(k, t, st, v, zl); });
        write_row(k, n, r.m, log_outside<1>(k, n, z, 0, cats, st, t, so), st, t, loss);
    }
}

// The same with too few rows for a lane each: a wave a row (8000 rows of 200 classes in f16: the kernel 9 us).
template <typename T>
__global__ __launch_bounds__(256) void distill_wave_kernel(const DistillK k) {
    __shared__ int s_l[4][64];
    const LogitsK &g = k.g;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, cats = g.C + g.bg;
    for (long long n = (long long)blockIdx.x * 4 + w; n < g.rows; n += (long long)gridDim.x * 4) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        float v;
        s_l[w][lane] = lane < k.K ? load_entry(k, n, lane, cats, v) : -1;
        wave_sync();
        Running r = no_scores();
        auto listed = [&](int j) {
            bool in = false;
            for (int q = 0; q < k.K; ++q) in |= s_l[w][q] == j;
            return in;
        };
        for (int j0 = 0; j0 < cats; j0 += 256) {
            float x[4];
            unsigned in = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = j0 + i * 64 + lane;
                x[i] = j < cats ? gather(g, z, j) : kNegInf;
            }
            if (k.tail) {
                for (int q = 0; q < k.K; ++q) {
                    const int at = s_l[w][q] - j0 - lane;
                    if ((at & 63) == 0 && at >= 0 && at < 256) in |= 1u << (at >> 6);
                }
            }
            add_outside(r, x, g.c2, in);
        }
        const float M = group_max<64>(r.m);
        float sum = 0.f, so = 0.f;
        if (far_scores(M, g.c2)) {  // (see answers.h)
            for (int j = lane; j < cats; j += 64) {
                const float e = exp2_hw((gather(g, z, j) - reference(M)) * g.c2);
                sum += e;
                so += k.tail && listed(j) ? 0.f : e;
            }
        } else {
            float d;
            const float f = to_reference(r, M, g.c2, d);
            sum = r.s * f;
            so = r.t * f;
        }
        finish_row(k, n, z, M, group_sum<64>(sum), group_sum<64>(so));
        wave_sync();
    }
}

// A block takes its rows and `len` classes of them.  The weights of 16 classes' entries lie in LDS while those are worked on, a column
// for a lane (-1: no entry); two entries are compared with each class in registers.  8 x 384 x 384 rows of 60 classes in f16, five entries
// and the tail: 86 us (4.1 TB/s); the entries' scores written over afterwards, each a line of its own: 128 us.
template <typename T, int K>
__global__ __launch_bounds__(kPlaneThreads<K>) void distill_grad_planes_kernel(const DistillK k, int parts, int len) {
    extern __shared__ float s_entries[];  // K 0
    constexpr int B = kPlaneThreads<K>, WIN = 16;
    __shared__ float s_w[K == 2 ? 1 : WIN][B];  // (a lane's own column)
    const LogitsK &g = k.g;
    const int cats = g.C + g.bg;
    const long long blocks = (g.rows + B - 1) / B;
    for (long long item = blockIdx.x; item < blocks * parts; item += gridDim.x) {
        const long long rb = parts == 1 ? item : item / parts;
        const int c0 = (int)(item - rb * parts) * len, c1 = c0 + len < g.C ? c0 + len : g.C;
        const long long n = rb * B + threadIdx.x;
        StagedEntries at = {nullptr, nullptr};
        if constexpr (K == 0) {
            at = stage_entries<B>(k, s_entries, rb * B, B, cats);
            at.to_row(threadIdx.x, k.K);
        }
        if (n >= g.rows) continue;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si), *p = z + c0 * g.sc;
        T *grad = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi), *out = grad + c0 * k.gsc;
        unsigned next[8];
        load_classes(p, g.sc, c1 - c0, next);
        LaneEntries<K> entries(k, n, cats, at);
        const Teacher t = entries.teacher();
        const GradRow r = grad_row(k, n, t);
        entries.to_weights(t);
        for (int c = c0; c < c1; c += 8) {
            const int w0 = (c - c0) & (WIN - 1);
            if (K != 2 && w0 == 0) {
#pragma unroll
                for (int i = 0; i < WIN; ++i) s_w[i][threadIdx.x] = -1.f;
                entries.each([&](int l, float w) {
                    const int j = l - g.bg - c;
                    if ((unsigned)j < (unsigned)WIN) s_w[j][threadIdx.x] = maxn(s_w[j][threadIdx.x], 0.f) + w;
                });
            }
            float y[8], q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[i] = widen<T>(next[i]);
                if constexpr (K == 2) {
                    q[i] = -1.f;
                    entries.each([&](int l, float w) { q[i] = l - g.bg == c + i ? maxn(q[i], 0.f) + w : q[i]; });
                } else {
                    q[i] = s_w[w0 + i][threadIdx.x];
                }
            }
            p += 8 * g.sc;
            if (c + 8 < c1) load_classes(p, g.sc, c1 - c - 8, next);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = grad_either(r, g.c2, y[i], q[i]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < c1) out[i * k.gsc] = from_f32<T>(y[i]);
            out += 8 * k.gsc;
        }
    }
}

// ---- dispatch ------------------------------------------------------------------------------------------------------------------
unsigned grid_of(long long blocks, int num_cu, int per_cu) {
    const long long cap = (long long)num_cu * per_cu;
    return (unsigned)(blocks < 1 ? 1 : blocks < cap ? blocks : cap);
}
bool contiguous(const LogitsK &g) { return g.sc == 1 || g.C == 1; }

template <typename T, int N>
void small(const DistillK &k, bool grad, int num_cu, hipStream_t st) {
    const dim3 grid(grid_of((k.g.rows + 255) / 256, num_cu, 64)), block(256);
    if (grad) {
        if (k.K <= 2) hipLaunchKernelGGL((distill_grad_small_kernel<T, N, 2>), grid, block, 0, st, k);
        else if (k.K <= 4) hipLaunchKernelGGL((distill_grad_small_kernel<T, N, 4>), grid, block, 0, st, k);
        else if (k.K <= 8) hipLaunchKernelGGL((distill_grad_small_kernel<T, N, 8>), grid, block, 0, st, k);
        else hipLaunchKernelGGL((distill_grad_small_kernel<T, N, 0>), grid, block, 0, st, k);
    } else {
        if (k.K <= 2) hipLaunchKernelGGL((distill_small_kernel<T, N, 2>), grid, block, 0, st, k);
        else if (k.K <= 4) hipLaunchKernelGGL((distill_small_kernel<T, N, 4>), grid, block, 0, st, k);
        else if (k.K <= 8) hipLaunchKernelGGL((distill_small_kernel<T, N, 8>), grid, block, 0, st, k);
        else hipLaunchKernelGGL((distill_small_kernel<T, N, 0>), grid, block, 0, st, k);
    }
}
template <typename T>
void small_of(const DistillK &k, bool grad, int num_cu, hipStream_t st) {
    switch (k.g.C) {
        case 1: return small<T, 1>(k, grad, num_cu, st);
        case 2: return small<T, 2>(k, grad, num_cu, st);
        case 3: return small<T, 3>(k, grad, num_cu, st);
        case 4: return small<T, 4>(k, grad, num_cu, st);
        case 5: return small<T, 5>(k, grad, num_cu, st);
        case 6: return small<T, 6>(k, grad, num_cu, st);
        case 7: return small<T, 7>(k, grad, num_cu, st);
        default: return small<T, 8>(k, grad, num_cu, st);
    }
}
// The kernel's limit of LDS raised to what any call of it asks for: the limit is the kernel's, not the call's, and another thread's
// call may come between this and the launch.
template <int ROWS, typename F>
hipError_t allow_staged(F *kernel) {
    return hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)staged_bytes(ROWS, QMRI_MAX_TOP));
}
template <typename T, int G>
hipError_t group(const DistillK &k, bool grad, int num_cu, hipStream_t st) {
    const dim3 grid(grid_of((k.g.rows + 256 / G - 1) / (256 / G), num_cu, 64)), block(256);
    // up to 16 entries a row in registers, or 64 where a row has that many lanes; 256 / G rows of more in LDS (G 2: at most 65 KB)
    constexpr int E = G >= 16 ? 64 / G : 16 / G > 4 ? 4 : 16 / G;
    // One or two entries: all of them in every lane (1000 classes: 74 us instead of 83); with more it pays only where two lanes share a
    // row (20 classes, three entries: 135 and 149 us; 500 classes: 85 and 81)
    if (k.K <= 2) {
        if (grad) hipLaunchKernelGGL((distill_grad_group_kernel<T, G, -2>), grid, block, 0, st, k);
        else hipLaunchKernelGGL((distill_group_kernel<T, G, -2>), grid, block, 0, st, k);
        return hipSuccess;
    }
    if constexpr (G == 2) {
        if (k.K <= 4) {
            if (grad) hipLaunchKernelGGL((distill_grad_group_kernel<T, G, -4>), grid, block, 0, st, k);
            else hipLaunchKernelGGL((distill_group_kernel<T, G, -4>), grid, block, 0, st, k);
            return hipSuccess;
        }
        if (k.K <= 8 && grad) {  // (20 classes, six entries: 183 us and 230)
            hipLaunchKernelGGL((distill_grad_group_kernel<T, G, -8>), grid, block, 0, st, k);
            return hipSuccess;
        }
    }
    if (k.K <= G * E) {
        if (!grad) hipLaunchKernelGGL((distill_group_kernel<T, G, E>), grid, block, 0, st, k);
        if constexpr (G > 2) {
            if (grad) hipLaunchKernelGGL((distill_grad_group_kernel<T, G, E>), grid, block, 0, st, k);
        }
    } else if constexpr (G < 16) {
        const size_t lds = staged_bytes(256 / G, k.K);
        // (the gradient has 25 KB of its own)
        if (lds > 16 * 1024) {
            const hipError_t e = grad ? allow_staged<256 / G>(distill_grad_group_kernel<T, G, 0>) : allow_staged<256 / G>(distill_group_kernel<T, G, 0>);
            if (e != hipSuccess) return e;
        }
        if (grad) hipLaunchKernelGGL((distill_grad_group_kernel<T, G, 0>), grid, block, lds, st, k);
        else hipLaunchKernelGGL((distill_group_kernel<T, G, 0>), grid, block, lds, st, k);
    }
    return hipSuccess;
}
template <typename T>
void planes(const DistillK &k, int num_cu, hipStream_t st) {
    const dim3 grid(grid_of((k.g.rows + 255) / 256, num_cu, 64)), block(256);
    if constexpr (sizeof(T) == 2) {  // (117 classes in f16, two entries: 79 us instead of 86; 20 classes 30 and 25)
        if (k.K <= 4 && k.g.C > 48) {
            if (k.K <= 2) hipLaunchKernelGGL((distill_planes_kernel<T, 2, 16>), grid, block, 0, st, k);
            else hipLaunchKernelGGL((distill_planes_kernel<T, 4, 16>), grid, block, 0, st, k);
            return;
        }
    }
    if (k.K <= 2) hipLaunchKernelGGL((distill_planes_kernel<T, 2, 8>), grid, block, 0, st, k);
    else if (k.K <= 4) hipLaunchKernelGGL((distill_planes_kernel<T, 4, 8>), grid, block, 0, st, k);
    else if (k.K <= 8) hipLaunchKernelGGL((distill_planes_kernel<T, 8, 8>), grid, block, 0, st, k);
    else hipLaunchKernelGGL((distill_planes_kernel<T, 0, 8>), dim3(grid_of((k.g.rows + 63) / 64, num_cu, 64)), dim3(64), staged_bytes(64, k.K), st, k);
}
template <typename T>
void planes_grad(const DistillK &k, int num_cu, hipStream_t st) {
    int parts;
    const int len = cut_classes(k.g, num_cu, parts);
    const dim3 grid(grid_of((k.g.rows + 255) / 256 * parts, num_cu, 64)), block(256);
    if (k.K <= 2) hipLaunchKernelGGL((distill_grad_planes_kernel<T, 2>), grid, block, 0, st, k, parts, len);
    else if (k.K <= 4) hipLaunchKernelGGL((distill_grad_planes_kernel<T, 4>), grid, block, 0, st, k, parts, len);
    else if (k.K <= 8) hipLaunchKernelGGL((distill_grad_planes_kernel<T, 8>), grid, block, 0, st, k, parts, len);
    else hipLaunchKernelGGL((distill_grad_planes_kernel<T, 0>), dim3(grid_of((k.g.rows + 63) / 64 * parts, num_cu, 64)), dim3(64),
                            staged_bytes(64, k.K), st, k, parts, len);
}

template <typename T>
hipError_t launch(const DistillK &k, int num_cu, hipStream_t st) {
    const LogitsK &g = k.g;
    const bool contig = contiguous(g);
    if (g.C <= 8) {
        small_of<T>(k, false, num_cu, st);
        return hipSuccess;
    }
    if (!contig) {
        if (lane_rows(g, num_cu))
            planes<T>(k, num_cu, st);
        else
            hipLaunchKernelGGL(distill_wave_kernel<T>, dim3(grid_of((g.rows + 3) / 4, num_cu, 32)), dim3(256), 0, st, k);
        return hipSuccess;
    }
    if (g.C <= 32) return group<T, 2>(k, false, num_cu, st);
    if (g.C <= 64) return group<T, 4>(k, false, num_cu, st);
    if (g.C <= 128) return group<T, 8>(k, false, num_cu, st);
    if (g.C <= 256) return group<T, 16>(k, false, num_cu, st);
    if (g.C <= 512) return group<T, 32>(k, false, num_cu, st);
    if (g.C <= 1024) return group<T, 64>(k, false, num_cu, st);
    const Cut cut = cut_rows(g, num_cu, k.tail ? kLongest : 1 << 30);
    const dim3 grid(grid_of(g.rows * cut.segs, num_cu, 64));
    const unsigned marks = (unsigned)(cut.len + 31) / 32 * 4;
    // One wave a row as soon as every SIMD has two rows: its teacher and its loss are then worked out while other waves read (4096 x
    // 32000 in bf16: 58 us, with four waves a row 68; 1024 x 100003: 74 and 55).  Longer rows are better shared, of 4-byte scores sooner
    // (bf16 2048 x 131000: 122 and 113; fp32 8192 x 16385: 114 and 106, 50000 x 1999: 88 and 162).
    if (g.rows >= 8ll * num_cu && g.C <= (sizeof(T) == 4 ? 8192 : 32768)) {
        if (k.tail) hipLaunchKernelGGL((distill_block_kernel<T, true, 1>), grid, dim3(64), marks, st, k, cut);
        else hipLaunchKernelGGL((distill_block_kernel<T, false, 1>), grid, dim3(64), 0, st, k, cut);
    } else {
        if (k.tail) hipLaunchKernelGGL((distill_block_kernel<T, true, 4>), grid, dim3(256), marks, st, k, cut);
        else hipLaunchKernelGGL((distill_block_kernel<T, false, 4>), grid, dim3(256), 0, st, k, cut);
    }
    if (cut.segs > 1) hipLaunchKernelGGL(distill_join_kernel<T>, dim3(grid_of(g.rows, num_cu, 64)), dim3(64), 0, st, k, cut);
    return hipSuccess;
}

template <typename T>
hipError_t launch_grad(const DistillK &k, int num_cu, hipStream_t st) {
    const LogitsK &g = k.g;
    const bool contig = contiguous(g) && (k.gsc == 1 || g.C == 1);
    if (g.C <= 8) {
        small_of<T>(k, true, num_cu, st);
        return hipSuccess;
    }
    if (!contig) {
        planes_grad<T>(k, num_cu, st);
        return hipSuccess;
    }
    if (g.C <= 32) return group<T, 2>(k, true, num_cu, st);
    if (g.C <= 64) return group<T, 4>(k, true, num_cu, st);
    if (g.C <= 128) return group<T, 8>(k, true, num_cu, st);
    if (g.C <= 256) return group<T, 16>(k, true, num_cu, st);
    if (g.C <= 512) return group<T, 32>(k, true, num_cu, st);
    if (g.C <= 1024) return group<T, 64>(k, true, num_cu, st);
    // a row's setup (its teacher) is worth several rounds of loads; eight blocks on every compute unit hide it
    const long long most = (g.C + 4095) / 4096;
    long long want = (8ll * num_cu + g.rows - 1) / g.rows;
    if (want > most) want = most;
    Cut cut;
    cut.len = (int)(((g.C + want - 1) / want + 4095) / 4096 * 4096);
    cut.segs = (g.C + cut.len - 1) / cut.len;
    const dim3 grid(grid_of(g.rows * cut.segs, num_cu, 64));
    if (wave_rows_grad<T>(g, num_cu)) hipLaunchKernelGGL((distill_grad_block_kernel<T, 1>), grid, dim3(64), 0, st, k, cut);
    else hipLaunchKernelGGL((distill_grad_block_kernel<T, 4>), grid, dim3(256), 0, st, k, cut);
    return hipSuccess;
}

}  // namespace

size_t distill_workspace_bytes(const DistillK &k, int, int num_cu) {
    if (k.g.C <= QMRI_SHORT_ROW || !contiguous(k.g)) return 0;
    const Cut cut = cut_rows(k.g, num_cu, k.tail ? kLongest : 1 << 30);
    return cut.segs > 1 ? (size_t)k.g.rows * cut.segs * 16 : 0;
}

hipError_t distill_launch(const DistillK &k, int dtype, int num_cu, hipStream_t st) {
    (void)hipGetLastError();
    const hipError_t e = dtype == QMRI_F32 ? launch<float>(k, num_cu, st) : dtype == QMRI_F16 ? launch<f16_t>(k, num_cu, st) : launch<bf16_t>(k, num_cu, st);
    const hipError_t last = hipGetLastError();  // (cleared in either case)
    return e != hipSuccess ? e : last;
}

hipError_t distill_grad_launch(const DistillK &k, int dtype, int num_cu, hipStream_t st) {
    (void)hipGetLastError();
    const hipError_t e = dtype == QMRI_F32 ? launch_grad<float>(k, num_cu, st) : dtype == QMRI_F16 ? launch_grad<f16_t>(k, num_cu, st) : launch_grad<bf16_t>(k, num_cu, st);
    const hipError_t last = hipGetLastError();  // (cleared in either case)
    return e != hipSuccess ? e : last;
}

}  // namespace qmri
