// answers.h -- what the kernels on a network's answers share (label_scores.hip, distill.hip): the geometry of a batch of
// category scores, the running softmax statistics of a row and how two of them join.
#ifndef QMRI_ANSWERS_H
#define QMRI_ANSWERS_H

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <type_traits>

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
    // n / inner for n < 2^31 as (n * magic) >> shift: shift = 31 + ceil(log2 inner), magic = ceil(2^shift / inner) < 2^32; the
    // error magic * inner - 2^shift is below 2^(shift - 31), so n times it stays below 2^shift.  magic 0: rows do not fit 31 bits
    unsigned magic;
    int shift;
};
inline void set_division(LogitsK &g) {
    g.magic = 0;
    g.shift = 0;
    if (g.rows > 0x7fffffffll || g.inner >= g.rows) return;
    int b = 0;
    while ((1ll << b) < g.inner) ++b;
    g.shift = 31 + b;
    g.magic = (unsigned)(((1ull << g.shift) + (unsigned long long)g.inner - 1) / (unsigned long long)g.inner);
}

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
    const long long o = g.magic ? (long long)(((unsigned long long)(unsigned)n * g.magic) >> g.shift) : n / g.inner;
    return o * so + (n - o * g.inner) * si;
}

// ---- scores of a row ------------------------------------------------------------------------------------------------------
// A vector is 16 bytes of scores, at the alignment of one score: rows of odd length begin anywhere, and the memory takes a
// 16-byte load at any address (aligned ones are not split off: the peeling costs more than the odd line).  It is kept as four
// words and widened from there: as 2-byte elements the compiler would take it apart and put it together again.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);
template <typename T>
struct Vec {
    unsigned w[4];
};
template <typename T>
__device__ __forceinline__ float get(const Vec<T> &r, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[i]);
    else if constexpr (std::is_same_v<T, bf16_t>) return __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
    else return static_cast<float>(__builtin_bit_cast(T, (unsigned short)(i & 1 ? r.w[i / 2] >> 16 : r.w[i / 2])));
}
template <typename T>
__device__ __forceinline__ unsigned bits_of(T v) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(unsigned, v);
    else return __builtin_bit_cast(unsigned short, v);
}
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T *p) {
    Vec<T> r;
    __builtin_memcpy(&r, p, 16);
    return r;
}
// the vector without its first n scores, -inf behind the others
template <typename T>
__device__ __forceinline__ Vec<T> drop_front(Vec<T> r, int n) {
    constexpr unsigned fill = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, bf16_t> ? 0xff80ff80u : 0xfc00fc00u;
    int words = n;
    if constexpr (sizeof(T) == 2) {
        words = n >> 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = n & 1 ? __builtin_amdgcn_alignbit(i < 3 ? r.w[i < 3 ? i + 1 : 3] : fill, r.w[i], 16) : r.w[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = words & 1 ? (i < 3 ? r.w[i < 3 ? i + 1 : 3] : fill) : r.w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = words & 2 ? (i < 2 ? r.w[i < 2 ? i + 2 : 3] : fill) : r.w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = words >= 4 ? fill : r.w[i];
    return r;
}
// The vector at p of a row with n scores (any number, also none) from there on, -inf behind: where it would end behind the row, the
// row's last vector without what lies before p.  (One load for all lanes: the scores one by one in a branch cost a third of the
// time of rows that end inside a vector.)  The row has at least kVec<T> scores.
template <typename T>
__device__ __forceinline__ int vec_back(int n) {  // by how many scores the load is moved to the front
    return n < kVec<T> ? kVec<T> - n : 0;
}
template <typename T>
__device__ __forceinline__ Vec<T> load_part(const T *p, int n) {
    const int back = vec_back<T>(n);
    return drop_front(load_vec(p - back), back < kVec<T> ? back : kVec<T>);
}
// values rounded to T
template <typename T>
__device__ __forceinline__ Vec<T> pack_vec(const float (&v)[kVec<T>]) {
    Vec<T> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) r.w[i] = __float_as_uint(v[i]);
        else r.w[i] = bits_of(from_f32<T>(v[2 * i])) | (bits_of(from_f32<T>(v[2 * i + 1])) << 16);
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void store_vec(T *p, const Vec<T> &r) {
    __builtin_memcpy(p, &r, 16);
}
// without the first n of them
template <typename T>
__device__ __forceinline__ void store_end(T *p, const float (&v)[kVec<T>], int n) {
#pragma unroll
    for (int i = 1; i < kVec<T>; ++i)
        if (i >= n) p[i] = from_f32<T>(v[i]);
}
// 16 scores a lane: the wave's 1024 from p on, in vectors side by side; score i of a lane is the wave's tile_at<T>(lane, i)-th
template <typename T>
struct Tile {
    Vec<T> v[16 / kVec<T>];
};
template <typename T>
__device__ __forceinline__ int tile_at(int lane, int i) {
    constexpr int V = kVec<T>;
    return (i / V) * 64 * V + lane * V + i % V;
}
// n: scores of the row from p on (wave-uniform); what lies behind is -inf
template <typename T>
__device__ __forceinline__ Tile<T> load_tile(const T *p, int n) {
    constexpr int V = kVec<T>;
    const int lane = threadIdx.x & 63;
    Tile<T> r;
    if (n >= 1024) {
#pragma unroll
        for (int u = 0; u < 16 / V; ++u) r.v[u] = load_vec(p + u * 64 * V + lane * V);
    } else {
#pragma unroll
        for (int u = 0; u < 16 / V; ++u) {
            const int j = u * 64 * V + lane * V;
            r.v[u] = load_part(p + j, n - j);
        }
    }
    return r;
}

// The bits of N scores, a class `sc` apart, `left` of them there and -inf behind.  (Bits in words of their own, and the whole N
// without a condition: what is packed, converted or branched upon would be waited for on the spot, and these are meant to be in
// flight while the N before them are worked on.)
template <typename T>
__device__ __forceinline__ unsigned load_bits(const T *p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const unsigned *>(p);
    else return *reinterpret_cast<const unsigned short *>(p);
}
template <typename T>
__device__ __forceinline__ float widen(unsigned w) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else if constexpr (std::is_same_v<T, bf16_t>) return __uint_as_float(w << 16);
    else return static_cast<float>(__builtin_bit_cast(T, (unsigned short)w));
}
template <typename T, int N>
__device__ __forceinline__ void load_classes(const T *p, long long sc, int left, unsigned (&v)[N]) {
    if (left >= N) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = load_bits(p + i * sc);
    } else {
        const unsigned none = bits_of(static_cast<T>(kNegInf));
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < left ? load_bits(p + i * sc) : none;
    }
}
// Classes that do not lie together, a lane a row: into how many parts (of whole eights) a row is cut so that every compute unit has
// 16 waves.  Returns the classes of a part.
inline int cut_classes(const LogitsK &g, int num_cu, int &parts) {
    const long long waves = (g.rows + 63) / 64;
    long long want = (16ll * num_cu + waves - 1) / waves;
    const int eights = (g.C + 7) / 8;
    if (want > eights) want = eights;
    const int len = (int)((eights + want - 1) / want) * 8;
    parts = (g.C + len - 1) / len;
    return len;
}

// NaN goes through a maximum here (v_maximum3_f32), so a row's NaN reaches its statistics without a test of its own
__device__ __forceinline__ float maxn(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// exponents are kept above -200: exp2 of that is 0 already, and 0 * -200 is 0 where 0 * -inf would not be
__device__ __forceinline__ float clamp2(float d) { return maxn(d, -200.f); }

// what a row's sums refer to: its maximum, or the lowest finite value where nothing is offered
__device__ __forceinline__ float reference(float M) { return maxn(M, -3.4028234663852886e38f); }

// ---- reductions over 2, 4, .. 64 neighbouring lanes, the result in each of them: DPP moves and lane swaps, no LDS -------------
template <int STEP>
__device__ __forceinline__ void partner(unsigned x, unsigned &a, unsigned &b) {
    if constexpr (STEP == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        a = r[0];
        b = r[1];
    } else if constexpr (STEP == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        a = r[0];
        b = r[1];
    } else {
        // quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror: within 8 and 16 lanes the halves hold one value each by then
        constexpr int ctrl = STEP == 1 ? 0xB1 : STEP == 2 ? 0x4E : STEP == 4 ? 0x141 : 0x140;
        a = x;
        b = (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, ctrl, 0xf, 0xf, false);
    }
}
template <int G, int STEP = 1>
__device__ __forceinline__ float group_max(float x) {
    if constexpr (STEP < G) {
        unsigned a, b;
        partner<STEP>(__float_as_uint(x), a, b);
        return group_max<G, STEP * 2>(maxn(__uint_as_float(a), __uint_as_float(b)));
    }
    return x;
}
template <int G, int STEP = 1>
__device__ __forceinline__ float group_sum(float x) {
    if constexpr (STEP < G) {
        unsigned a, b;
        partner<STEP>(__float_as_uint(x), a, b);
        return group_sum<G, STEP * 2>(__uint_as_float(a) + __uint_as_float(b));
    }
    return x;
}
template <int G, int STEP = 1>
__device__ __forceinline__ unsigned group_maxu(unsigned x) {
    if constexpr (STEP < G) {
        unsigned a, b;
        partner<STEP>(x, a, b);
        return group_maxu<G, STEP * 2>(a > b ? a : b);
    }
    return x;
}
template <int G, int STEP = 1>
__device__ __forceinline__ int group_min(int x) {
    if constexpr (STEP < G) {
        unsigned a, b;
        partner<STEP>((unsigned)x, a, b);
        return group_min<G, STEP * 2>((int)a < (int)b ? (int)a : (int)b);
    }
    return x;
}

// sum of 2^k values as a tree
template <int N>
__device__ __forceinline__ float tree_sum(const float (&v)[N]) {
    float a[N];
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = v[i];
#pragma unroll
    for (int h = N / 2; h > 0; h >>= 1)
#pragma unroll
        for (int i = 0; i < h; ++i) a[i] += a[i + h];
    return a[0];
}

// Running statistics of a part of a row: the maximum m of its scores (-inf: none offered), and relative to a finite reference
// ref  s = sum exp2((z - ref) c2),  t = sum exp2((z - ref) c2) (z - ref) c2.  Everything is held in 32 bits.
struct RowStat {
    float m, ref, s, t;
};
__device__ __forceinline__ RowStat no_stat() { return {kNegInf, -3.4028234663852886e38f, 0.f, 0.f}; }
// the sums of r relative to another reference
__device__ __forceinline__ void rebase(RowStat &r, float ref, float c2) {
    const float d = r.ref == ref ? 0.f : maxn((r.ref - ref) * c2, -1.0e4f);
    const float f = exp2_hw(d);
    r.t = f * (r.t + d * r.s);
    r.s *= f;
    r.ref = ref;
}
// all lanes of a wave together
__device__ __forceinline__ RowStat wave_join(RowStat r, float c2) {
    const float M = group_max<64>(r.m);
    rebase(r, reference(M), c2);
    r.m = M;
    r.s = group_sum<64>(r.s);
    r.t = group_sum<64>(r.t);
    return r;
}
__device__ __forceinline__ RowStat join(RowStat a, RowStat b, float c2) {
    const float M = maxn(a.m, b.m), ref = reference(M);
    rebase(a, ref, c2);
    rebase(b, ref, c2);
    return {M, ref, a.s + b.s, a.t + b.t};
}

// A lane's running sums over many scores.  The reference is kept in the units of the exponents, R = ref * c2 rounded: an exponent
// is then one fused z * c2 - R, and as all of a row's terms are brought to one reference in the end, the rounding of R cancels.
// It follows the lane's maximum only when that has grown by more than a factor of 16: nearly no step pays for a change.
constexpr float kSlack = 4.f;
// Scores whose product with c2 leaves the range of 32 bits cannot be summed like that; a row of such (the lowest value of the type
// everywhere, for one) is summed again by differences (far_scores).
constexpr float kFar = 1.0e37f;
struct Running {
    float m, R, s, t;
};
__device__ __forceinline__ Running no_scores() { return {kNegInf, -1.0e38f, 0.f, 0.f}; }
template <int N>
__device__ __forceinline__ float max_of(const float (&x)[N]) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = maxn(m, x[i]);
    return m;
}
// cm: the largest of the scores that come next
template <bool T2>
__device__ __forceinline__ void raise(Running &r, float cm, float c2) {
    r.m = maxn(r.m, cm);
    if (fmaf(cm, c2, -r.R) > kSlack) {
        const float R = cm * c2, d = fmaxf(r.R - R, -1.0e4f), f = exp2_hw(d);
        r.t = T2 ? f * fmaf(d, r.s, r.t) : f * r.t;
        r.s *= f;
        r.R = R;
    }
}
// t as the sum of exp2(d) d; returns the largest of the scores
template <int N>
__device__ __forceinline__ float add_scores(Running &r, const float (&x)[N], float c2) {
    const float cm = max_of(x);
    raise<true>(r, cm, c2);
    float s[4] = {0.f, 0.f, 0.f, 0.f}, t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = clamp2(fmaf(x[i], c2, -r.R)), e = exp2_hw(d);
        s[i & 3] += e;
        t[i & 3] = fmaf(e, d, t[i & 3]);
    }
    r.s += tree_sum(s);
    r.t += tree_sum(t);
    return cm;
}
__device__ __forceinline__ bool far_scores(float M, float c2) { return M > kNegInf && !(fabsf(M) * c2 < kFar); }
// factor that brings a lane's sums to reference(M), M the maximum over the lanes; d its exponent
__device__ __forceinline__ float to_reference(const Running &r, float M, float c2, float &d) {
    d = fminf(maxn(fmaf(-reference(M), c2, r.R), -1.0e4f), 64.f);  // (a lane that saw nothing has no sums: any factor will do)
    return exp2_hw(d);
}
// the wave's sums together; far: the row's own scores again, j = first, first + step, .. of n, by differences
template <typename F>
__device__ __forceinline__ RowStat wave_stat(const Running &r, float c2, F score, int first, int step, int n) {
    const float M = group_max<64>(r.m);
    RowStat o = {M, reference(M), 0.f, 0.f};
    if (far_scores(M, c2)) {
        float s = 0.f, t = 0.f;
        for (int j = first; j < n; j += step) {
            const float d = clamp2((score(j) - o.ref) * c2), e = exp2_hw(d);
            s += e;
            t = fmaf(e, d, t);
        }
        o.s = group_sum<64>(s);
        o.t = group_sum<64>(t);
    } else {
        float d;
        const float f = to_reference(r, M, c2, d);
        o.s = group_sum<64>(r.s * f);
        o.t = group_sum<64>(f * fmaf(d, r.s, r.t));
    }
    return o;
}

// what a wave's lanes have written to LDS is visible to its other lanes from here on
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// a better than b in the order of the alternatives: larger score, ties to the lower label
__device__ __forceinline__ bool better(float va, int ia, float vb, int ib) { return va > vb || (va == vb && ia < ib); }

// How the rows of a call are cut for the kernels that give a block a row (contiguous classes, more than 1024 of them): segments
// of whole 16-byte vectors, of at most `longest` scores
struct Cut {
    int segs, len;
};
Cut cut_rows(const LogitsK &g, int num_cu, int longest);
// Classes that do not lie together: a lane a row as soon as every compute unit has 32 rows (half a wave), below that a wave a row (kernel
// times in f16, wave and lane: 200 classes 1000 rows 3.6 and 10.1 us, 8000 rows 7.4 and 10.3, 16000 rows 15.8 and 10.3; with the three
// best 7.3 and 14.1, 18.7 and 14.4, 31.2 and 14.6; distillation 4.6 and 16.0, 9.4 and 16.2, 20.0 and 16.2).  The rule does not look at the best:
// with them a wave a row is behind already at 8000 rows.  Rows of up to 64 classes are read by a lane in a few rounds: always.
inline bool lane_rows(const LogitsK &g, int num_cu) { return g.C <= 64 || g.rows >= 32ll * num_cu; }
// Gradients by a wave a row, once every SIMD has four rows; longer ones are better left to four waves, 4-byte ones sooner (8192 x 8192: bf16 53
// us by one wave and 56 by four, fp32 115 and 101; 50000 x 1999 with a teacher: bf16 105 and 194, fp32 178 and 212)
template <typename T>
bool wave_rows_grad(const LogitsK &g, int num_cu) {
    return g.C <= (sizeof(T) == 4 ? 2048 : 8192) && g.rows >= 16ll * num_cu;
}

hipError_t label_scores_launch(const ScoresK &k, int dtype, int num_cu, hipStream_t st);
size_t label_scores_workspace_bytes(const ScoresK &k, int dtype, int num_cu);
hipError_t label_scores_grad_launch(const ScoresK &k, int dtype, int num_cu, hipStream_t st);
hipError_t distill_launch(const DistillK &k, int dtype, int num_cu, hipStream_t st);
size_t distill_workspace_bytes(const DistillK &k, int dtype, int num_cu);
hipError_t distill_grad_launch(const DistillK &k, int dtype, int num_cu, hipStream_t st);
// (S, P, K) rows of float32 or int32 labels -> (K, P, S) planes of float32 or uint8, and back (answers_planes.hip)
hipError_t rows_to_planes_launch(const void *x, int is_label, long long P, int S, int K, void *y, hipStream_t stream);
hipError_t planes_to_rows_launch(const void *x, int kind, long long P, int S, int K, void *y, hipStream_t stream);

}  // namespace qmri
#endif
