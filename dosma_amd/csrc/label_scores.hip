// label_scores.hip -- log probability of a given label, entropy and best alternatives of every row of category scores, and
// the gradient of the first two, for gfx950.
//
//   M = max z, s = sum exp((z - M) / T), log p_j = (z_j - M) / T - ln s, H = ln s - sum exp(d_j) d_j / s  (d_j = (z_j - M) / T)
//   g_j = [ a (delta_j,label - p_j) - b p_j (log p_j + H) ] / T
//
// The scores are read once (and the gradient written once).  Who owns a row depends on its length and layout:
//   small   1 .. 8 classes, any layout: one lane a row, everything in registers, unrolled for the number of classes
//   group   9 .. 1024 contiguous classes: 2 .. 64 lanes a row, 16 scores a lane in registers
//   block   more contiguous classes: a block (or, with few rows, several) a row, running statistics per lane
//   planes  more than 8 classes that do not lie together: one lane a row, neighbouring rows side by side
//   wave    the same with too few rows for that: a wave a row
// The times at the kernels are those of whole calls on an MI355X, where a large copy moves 4.8 to 5.0 TB/s.
#include "answers.h"

namespace qmri {

Cut cut_rows(const LogitsK &g, int num_cu, int longest) {
    // enough blocks for every compute unit twice over, but at least 4096 scores (a round of a block's loads) for each
    long long want = g.rows >= 2ll * num_cu ? 1 : (2ll * num_cu + g.rows - 1) / g.rows;
    const long long most = (g.C + 4095) / 4096, least = (g.C + longest - 1) / longest;
    if (want > most) want = most;
    if (want < least) want = least;
    Cut c;
    c.len = (int)(((g.C + want - 1) / want + 63) / 64 * 64);
    c.segs = (g.C + c.len - 1) / c.len;
    return c;
}
namespace {

// ---- results of a row -------------------------------------------------------------------------------------------------------
// s and t refer to reference(M).  zl: score of the given label (NaN-free only where the label is a category)
__device__ __forceinline__ void write_row(const ScoresK &k, long long n, float M, float s, float t, bool has_label, bool ignored, float zl) {
    const float l2s = __builtin_amdgcn_logf(s), ls = l2s * kLn2;
    if (k.norm) {
        float2 v = make_float2(ls != ls ? ls : M, ls);
        *reinterpret_cast<float2 *>(k.norm + 2 * n) = v;
    }
    // (both terms are >= 0: no cancellation)
    if (k.entropy) k.entropy[n] = s == 0.f ? 0.f : (l2s - t / s) * kLn2;
    if (k.log_prob) {
        float lp = (zl - reference(M)) * k.g.invT - ls;
        if (s == 0.f || zl == kNegInf) lp = ls != ls ? ls : kNegInf;
        if (!has_label) lp = __builtin_nanf("");
        k.log_prob[n] = ignored ? 0.f : lp;
    }
}
__device__ __forceinline__ float top_value(const ScoresK &k, float v, int i, float M, float ls) {
    return i < 0 ? (ls != ls ? ls : kNegInf) : (v - reference(M)) * k.g.invT - ls;
}
__device__ __forceinline__ void write_top(const ScoresK &k, long long n, int q, float v, int i, float M, float ls) {
    k.top_label[n * k.top + q] = i;
    k.top_log_prob[n * k.top + q] = top_value(k, v, i, M, ls);
}
__device__ __forceinline__ void given_label(const ScoresK &k, long long n, int cats, int &l, bool &has, bool &ignored) {
    l = -1;
    has = ignored = false;
    if (!k.log_prob) return;
    const long long v = load_label(k.labels, k.l_kind, n);
    ignored = v == k.ignore;
    has = v >= 0 && v < cats;
    if (has) l = (int)v;
}

// ---- scores as keys -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned ordered(float f) {  // the order of floats as that of unsigned integers; -0 ranks as +0
    const int u = __float_as_int(f + 0.f);
    return (unsigned)(u ^ ((u >> 31) | (int)0x80000000));
}
__device__ __forceinline__ float unordered(unsigned o) {
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
constexpr unsigned kKeyNegInf = 0x007fffffu;  // ordered(-inf)
// significant bits of a widened score's key: the lower ones are all alike
template <typename T>
constexpr int kKeyBits = 32;
template <>
constexpr int kKeyBits<f16_t> = 19;
template <>
constexpr int kKeyBits<bf16_t> = 16;

// ---- small: one lane a row ----------------------------------------------------------------------------------------------------
// Bound by memory and, right behind, by the vector unit: a row of 4 scores in 32 bits is 16 bytes in and up to 32 out.  512 x 512 x
// 160 such rows with a background and the two best: 336 us, 5.1 TB/s.
template <typename T, int N, bool BG, bool CONTIG>
__global__ __launch_bounds__(256) void scores_small_kernel(const ScoresK k) {
    const LogitsK &g = k.g;
    constexpr int CATS = N + BG;
    const long long stride = (long long)gridDim.x * 256;
    for (long long n = (long long)blockIdx.x * 256 + threadIdx.x; n < g.rows; n += stride) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        float x[CATS];
        if (BG) x[0] = 0.f;
        if (CONTIG) {
            struct {
                T v[N];
            } r;
            __builtin_memcpy(&r, z, sizeof(r));
#pragma unroll
            for (int j = 0; j < N; ++j) x[j + BG] = to_f32(r.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) x[j + BG] = to_f32(z[j * g.sc]);
        }
        int l;
        bool has, ignored;
        given_label(k, n, CATS, l, has, ignored);
        float M = x[0];
#pragma unroll
        for (int j = 1; j < CATS; ++j) M = maxn(M, x[j]);
        const float ref = reference(M);
        float s = 0.f, t = 0.f, zl = kNegInf;
#pragma unroll
        for (int j = 0; j < CATS; ++j) {
            const float d = clamp2((x[j] - ref) * g.c2), e = exp2_hw(d);
            s += e;
            t = fmaf(e, d, t);
            zl = l == j ? x[j] : zl;
        }
        write_row(k, n, M, s, t, has, ignored, zl);
        const float ls = __builtin_amdgcn_logf(s) * kLn2;
        for (int q = 0; q < k.top; ++q) {
            float bv = x[0];
            int bi = 0;
#pragma unroll
            for (int j = 1; j < CATS; ++j) {
                const bool c = x[j] > bv || bv != bv;
                bv = c ? x[j] : bv;
                bi = c ? j : bi;
            }
            write_top(k, n, q, bv, bv > kNegInf ? bi : -1, M, ls);
#pragma unroll
            for (int j = 0; j < CATS; ++j) x[j] = bi == j ? kNegInf : x[j];
        }
    }
}

// ---- group: G lanes a row, 16 scores a lane -----------------------------------------------------------------------------------
// The fewest lanes that hold a row, so that the exchanges between lanes are few and shared by many rows of a wave.  The best are
// found one after the other: a maximum over 17 keys a lane, one over the lanes.  200000 x 500 in fp32 80 us (5.0 TB/s, memory), in bf16
// 51 us (4.0 TB/s); with the three best 111 and 84 us, bound by the vector unit.
// Without the best: 64 registers, eight waves a SIMD (500 classes in bf16, 200000 rows: 51 us instead of 55 with the code of both).
// With them 78: held to 64 they spill (104 us instead of 86).  Keys made two scores at a time in packed 16-bit integers are no faster.
template <typename T, int G, bool TOP>
__global__ __launch_bounds__(256, TOP ? 4 : 8) void scores_group_kernel(const ScoresK k) {
    const LogitsK &g = k.g;
    constexpr int V = kVec<T>, NV = 16 / V, ROWS = 256 / G;
    const int gl = threadIdx.x % G, cats = g.C + g.bg;
    for (long long n0 = (long long)blockIdx.x * ROWS; n0 < g.rows; n0 += (long long)gridDim.x * ROWS) {
        // groups behind the last row work on it too and write nothing: the lane exchanges below want whole waves
        const long long nr = n0 + threadIdx.x / G;
        const bool live = nr < g.rows;
        const long long n = live ? nr : g.rows - 1;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        float x[17];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * G + gl) * V;
            // (with more than 8 G scores in a row the first half of the vectors is whole)
            const Vec<T> r = G > 2 && 2 * i < NV ? load_vec(z + j) : load_part(z + j, g.C - j);
#pragma unroll
            for (int e = 0; e < V; ++e) x[i * V + e] = get(r, e);
        }
        x[16] = (g.bg && gl == 0) ? 0.f : kNegInf;
        int l;
        bool has, ignored;
        given_label(k, n, cats, l, has, ignored);
        const float zl = (has && l >= g.bg) ? to_f32(z[l - g.bg]) : 0.f;
        float M = x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) M = maxn(M, x[i]);
        M = group_max<G>(M);
        const float ref = reference(M);
        float e[16], et[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float d = clamp2((x[i] - ref) * g.c2);
            e[i] = exp2_hw(d);
            et[i] = e[i] * d;
        }
        const float db = clamp2((x[16] - ref) * g.c2), eb = exp2_hw(db);
        const float s = group_sum<G>(tree_sum(e) + eb), t = group_sum<G>(tree_sum(et) + eb * db);
        if (live && gl == 0) write_row(k, n, M, s, t, has, ignored, zl);
        if (!TOP) continue;
        const float ls = __builtin_amdgcn_logf(s) * kLn2;
        auto label_of = [&](int i) { return ((i / V) * G + gl) * V + i % V + g.bg; };
        if constexpr (sizeof(T) == 2) {
            // the significant bits of a score over the complement of its label (11 bits: up to 1024 classes), below 2^31: of the
            // differences key - last those of the keys already taken are small, the others wrap around, in their order
            constexpr int DOWN = 32 - kKeyBits<T>;
            auto key_of = [&](float v, int label) { return ((ordered(v) >> DOWN) << 11) | (2047u - (unsigned)label); };
            unsigned key[17];
#pragma unroll
            for (int i = 0; i < 16; ++i) key[i] = key_of(x[i], label_of(i));
            key[16] = key_of(x[16], 0);
            unsigned last = 0x80000000u;
            for (int q = 0; q < k.top; ++q) {
                unsigned m = key[16] - last;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const unsigned d = key[i] - last;
                    m = d > m ? d : m;
                }
                last += group_maxu<G>(m);
                const unsigned o = (last >> 11) << DOWN;
                const float v = unordered(o & 0x80000000u ? o : o | ((1u << DOWN) - 1u));
                if (live && gl == 0) write_top(k, n, q, v, v > kNegInf ? (int)(2047u - (last & 2047u)) : -1, M, ls);
            }
        } else {
            for (int q = 0; q < k.top; ++q) {
                float bv = x[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) bv = fmaxf(bv, x[i]);
                const float best = group_max<G>(bv);
                int bi = x[16] == best ? 0 : 0x7fffffff;
#pragma unroll
                for (int i = 15; i >= 0; --i) {
                    const int l = label_of(i);
                    bi = x[i] == best && l < bi ? l : bi;
                }
                const int at = group_min<G>(bi);
                if (live && gl == 0) write_top(k, n, q, best, best > kNegInf ? at : -1, M, ls);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = label_of(i) == at ? kNegInf : x[i];
                if (at == 0 && g.bg) x[16] = kNegInf;
            }
        }
    }
}

// ---- the best of a long row -----------------------------------------------------------------------------------------------------
// A score can belong to the k best only if it is above a floor for which k others are known.  What passes the floor goes into a
// buffer of the wave's in LDS; a full buffer is cut down to its k best, whose last is the new floor.  The order is (score falling,
// label rising), so the result does not depend on who came first.
// No two pairs of a buffer have the same label, and none is an empty slot (label -1): equal scores are told apart by their labels, so
// a cut leaves at most k <= 64 pairs, which is what makes room for the next 64 and what final_best reads.
// Which of the wave's 64 N (key, label) pairs are its k best; key 0: none.  The k-th largest key is found bit by bit.
template <int N, int BITS>
__device__ __forceinline__ unsigned select_best(const unsigned (&key)[N], const int (&id)[N], int k, bool (&win)[N]) {
    auto count = [&](auto f) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(f(i)));
        return c;
    };
    unsigned t = 0u;
#pragma unroll 1
    for (int bit = 31; bit >= 32 - BITS; --bit) {
        const unsigned at = t | (1u << bit);
        if (count([&](int i) { return key[i] >= at; }) >= k) t = at;
    }
    // keys that agree with t in the significant bits are equal scores: of those the lowest labels
    const unsigned top = BITS == 32 ? 0xffffffffu : ~((1u << (32 - BITS)) - 1u);
    const int above = count([&](int i) { return (key[i] & top) > t; });
    int last = 0x7fffffff;
    if (t != 0u && above + count([&](int i) { return (key[i] & top) == t; }) > k) {
        last = 0;
#pragma unroll 1
        for (int bit = 30; bit >= 0; --bit) {  // the largest label of which fewer than k - above equals lie below
            const int at = last | (1 << bit);
            if (count([&](int i) { return (key[i] & top) == t && id[i] < at; }) < k - above) last = at;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) win[i] = key[i] != 0u && ((key[i] & top) > t || ((key[i] & top) == t && id[i] <= last));
    return t;
}

constexpr int kBuf = 192;
struct WaveBest {
    float *v;  // [kBuf] in LDS, this wave's
    int *i;
    int n;     // pairs in it
    // a pair that does not come before (floor, bound) cannot be among the best
    float floor;
    int bound;
    int k;
    // where the set lanes of a ballot find their places
    static __device__ __forceinline__ int place(unsigned long long m) {
        return __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0u));
    }
    __device__ __forceinline__ bool passes(float x, int label) const { return x > floor || (x == floor && label < bound); }
    template <int BITS>
    __device__ __forceinline__ void cut() {
        wave_sync();
        const int lane = threadIdx.x & 63;
        unsigned key[kBuf / 64];
        int id[kBuf / 64];
        float sv[kBuf / 64];
        bool win[kBuf / 64];
#pragma unroll
        for (int q = 0; q < kBuf / 64; ++q) {
            const int j = q * 64 + lane;
            sv[q] = j < n ? v[j] : 0.f;
            id[q] = j < n ? i[j] : 0;
            key[q] = j < n ? ordered(sv[q]) : 0u;
        }
        select_best<kBuf / 64, BITS>(key, id, k, win);
        wave_sync();
        const bool full = n >= k;
        n = 0;
        float worst = __builtin_inff();
#pragma unroll
        for (int q = 0; q < kBuf / 64; ++q) {
            const unsigned long long m = __ballot(win[q]);
            if (win[q]) {
                v[n + place(m)] = sv[q];
                i[n + place(m)] = id[q];
                worst = fminf(worst, sv[q]);
            }
            n += __popcll(m);
        }
        if (full) {  // the last of the best
            floor = -group_max<64>(-worst);
            int last = -1;
#pragma unroll
            for (int q = 0; q < kBuf / 64; ++q) last = win[q] && sv[q] == floor && id[q] > last ? id[q] : last;
            bound = -group_min<64>(-last);
        }
        wave_sync();
    }
    // one pair a lane
    template <int BITS>
    __device__ __forceinline__ void take(float x, int label, bool in) {
        if (__ballot(in && passes(x, label)) == 0ull) return;
        if (n + 64 > kBuf) cut<BITS>();
        const bool yes = in && passes(x, label);
        const unsigned long long m = __ballot(yes);
        if (yes) {
            v[n + place(m)] = x;
            i[n + place(m)] = label;
        }
        n += __popcll(m);
    }
};

// The floor that 64 N values (N a lane) give: k of them are at least as large as the k-th, so only what is above a lower value
// can be among the best.
template <int N, int BITS>
__device__ __forceinline__ float first_floor(const float *m, int k) {
    const int lane = threadIdx.x & 63;
    unsigned key[N];
#pragma unroll
    for (int q = 0; q < N; ++q) key[q] = ordered(m[q * 64 + lane]);
    unsigned t = 0u;
    constexpr int LOW = BITS < 20 ? 32 - BITS : 12;  // (the upper 20 bits will do: a floor that is a little low only lets more through)
#pragma unroll 1
    for (int bit = 31; bit >= LOW; --bit) {
        const unsigned at = t | (1u << bit);
        int c = 0;
#pragma unroll
        for (int q = 0; q < N; ++q) c += __popcll(__ballot(key[q] >= at));
        if (c >= k) t = at;
    }
    return t > kKeyNegInf + (1u << LOW) ? unordered(t - (1u << LOW)) : kNegInf;  // (the next lower of these keys)
}

// Up to 64 winners, one a lane (i < 0: none), into falling order: every lane counts the better ones.
__device__ __forceinline__ int rank_of(float v, int i, int k) {
    int r = 0;
#pragma unroll 1
    for (int o = 0; o < k; ++o) {
        const float ov = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), o));
        const int oi = __builtin_amdgcn_readlane(i, o);
        r += (oi >= 0 && (i < 0 || better(ov, oi, v, i))) ? 1 : 0;
    }
    return r;
}

// a segment's part of a row in the workspace: m, s (relative to reference(m)), t, then its best scores and their labels
__device__ __forceinline__ size_t part_words(int k) { return 4 + 2 * (size_t)k; }

// The W waves' lists, up to 64 pairs each at v, i + w * kBuf (i < 0: none), together: the k best to lanes 0 .. k - 1 of the wave
// that asks, in falling order.  The lists are overwritten.
template <int W, int BITS>
__device__ __forceinline__ void final_best(float *tv, int *ti, int k, float &bv, int &bi) {
    const int lane = threadIdx.x & 63;
    int id[W];
    float sv[W];
    bool win[W];
    int all = 0;
#pragma unroll
    for (int q = 0; q < W; ++q) {
        id[q] = ti[q * kBuf + lane];
        sv[q] = tv[q * kBuf + lane];
        win[q] = id[q] >= 0;
        all += __popcll(__ballot(win[q]));
    }
    wave_sync();
    if (all > 64) {  // (up to 64 are put in order as they are)
        unsigned key[W];
#pragma unroll
        for (int q = 0; q < W; ++q) key[q] = win[q] ? ordered(sv[q]) : 0u;
        select_best<W, BITS>(key, id, k, win);
    }
    int n = 0;
#pragma unroll
    for (int q = 0; q < W; ++q) {
        const unsigned long long m = __ballot(win[q]);
        if (win[q]) {
            tv[n + WaveBest::place(m)] = sv[q];
            ti[n + WaveBest::place(m)] = id[q];
        }
        n += __popcll(m);
    }
    wave_sync();
    bv = lane < n ? tv[lane] : kNegInf;
    bi = lane < n ? ti[lane] : -1;
    const int r = rank_of(bv, bi, n);
    wave_sync();
    if (lane < n) {
        tv[r] = bv;
        ti[r] = bi;
    }
    wave_sync();
    bv = lane < n ? tv[lane] : kNegInf;
    bi = lane < n ? ti[lane] : -1;
}

// ---- block: W waves a segment of a row ------------------------------------------------------------------------------------------
// Per score: widen, half a maximum, one fused multiply, clamp, exp2 (two slots), one and a half sums -- about 8 issue slots, of
// the 16 that a 2-byte score has at 4.8 TB/s: memory first, the vector unit close behind.  1024 x 100003 in bf16: 47 us (4.3 TB/s);
// with the 8 best 63 us: the floors, the reading of candidates and the last order, none of which reads the scores, take the rest.
// Four waves a segment (eight wait longer for the one that finishes: 8192 x 16385 80 us instead of 68), one wave a row where there
// are rows enough.  64 registers without the best, for eight waves a SIMD; 80 with them: at 64 they spill, five times slower.
template <typename T, bool TOP, int W>
__global__ __launch_bounds__(64 * W, TOP ? 6 : sizeof(T) == 4 ? 6 : 8) void scores_block_kernel(const ScoresK k, const Cut cut) {
    __shared__ RowStat s_stat[W];
    __shared__ float s_max[TOP ? 64 * W : 1];  // the lanes' largest
    __shared__ float s_v[TOP ? W * kBuf : 1];
    __shared__ int s_i[TOP ? W * kBuf : 1];
    const LogitsK &g = k.g;
    constexpr int TILE = 1024, BITS = kKeyBits<T>;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long work = g.rows * cut.segs;
    for (long long item = blockIdx.x; item < work; item += gridDim.x) {
        const long long n = cut.segs == 1 ? item : item / cut.segs;
        const int seg = cut.segs == 1 ? 0 : (int)(item - n * cut.segs);
        const int c0 = seg * cut.len, c1 = c0 + cut.len < g.C ? c0 + cut.len : g.C;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        const bool back = g.bg && seg == 0 && w == 0;
        // the given label's score, needed last, is on its way from the start
        int l = -1;
        bool has = false, ignored = false;
        float zl = 0.f;
        if (w == 0 && cut.segs == 1) {
            given_label(k, n, g.C + g.bg, l, has, ignored);
            if (has && l >= g.bg) zl = to_f32(z[l - g.bg]);
        }
        Running r = no_scores();
        if (back && lane == 0) r = {0.f, 0.f, 1.f, 0.f};  // the implicit category: lane 0 has seen a score of 0
        WaveBest b = {s_v + (TOP ? w * kBuf : 0), s_i + (TOP ? w * kBuf : 0), 0, kNegInf, 0, k.top};
        // the best k of the lanes' largest so far: nothing below the last of them can be among the best of the row.  (What the
        // other waves have written meanwhile does not matter: older maxima are scores of the row as well.)
        auto raise_floor = [&](float m) {
            wave_sync();
            s_max[threadIdx.x] = m;
            wave_sync();
            const float f = first_floor<W, BITS>(s_max, k.top);
            if (f > b.floor) {
                b.floor = f;
                b.bound = 0;
            }
        };
        const int rounds = (c1 - c0 + W * TILE - 1) / (W * TILE);
        int c = c0 + w * TILE;
        Tile<T> next;
        if (c < c1) next = load_tile(z + c, c1 - c);
        for (int it = 0; it < rounds; ++it, c += W * TILE) {
            const bool mine = c < c1;
            float x[16];
            if (mine) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = get(next.v[i / kVec<T>], i % kVec<T>);
                if (c + W * TILE < c1) next = load_tile(z + c + W * TILE, c1 - c - W * TILE);
            }
            if (TOP && it == 0) {
                float cm = back && lane == 0 ? 0.f : kNegInf;
                if (mine) cm = fmaxf(cm, max_of(x));
                s_max[threadIdx.x] = cm;
                __syncthreads();
                raise_floor(cm);
                if (back && b.passes(0.f, 0)) {
                    if (lane == 0) {
                        b.v[0] = 0.f;
                        b.i[0] = 0;
                    }
                    b.n = 1;
                }
            }
            if (mine) {
                const float cm = add_scores(r, x, g.c2);
                if (TOP) {
                    // the 16 scores of lanes that hold something for the list are read again, four lanes' at a time, one a lane
                    for (unsigned long long m = __ballot(cm >= b.floor); m != 0ull;) {
                        int from = 0, have = 0;
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (m != 0ull) {
                                const int l = __ffsll(m) - 1;
                                from = (lane >> 4) == q ? l : from;
                                m &= m - 1;
                                have = q + 1;
                            }
                        const int j = c + tile_at<T>(from, lane & 15);
                        const bool in = (lane >> 4) < have && j < c1;
                        b.take<BITS>(in ? to_f32(z[j]) : kNegInf, j + g.bg, in);
                    }
                }
            }
            // every time the scores seen have quadrupled
            if (TOP && (it == 3 || it == 15 || it == 63) && it + 1 < rounds) raise_floor(r.m);
        }
        RowStat st = wave_stat(r, g.c2, [&](int j) {
            // (w's scores in the order of its tiles; -1: the implicit category, seen by lane 0)
            if (j < 0) return lane == 0 ? 0.f : kNegInf;
            const int at = c0 + (j / TILE) * W * TILE + w * TILE + j % TILE;
            return at < c1 ? to_f32(z[at]) : kNegInf;
        }, back ? lane - 64 : lane, 64, rounds * TILE);
        if (lane == 0) s_stat[w] = st;
        if (TOP) {
            if (b.n > 64) b.cut<BITS>();
            for (int q = b.n + lane; q < 64; q += 64) b.i[q] = -1;
        }
        __syncthreads();
        if (w == 0) {
            float bv = kNegInf;
            int bi = -1;
            if (TOP) final_best<W, BITS>(s_v, s_i, k.top, bv, bi);
            st = s_stat[0];
#pragma unroll
            for (int o = 1; o < W; ++o) st = join(st, s_stat[o], g.c2);
            if (cut.segs > 1) {
                float *p = static_cast<float *>(k.ws) + (size_t)item * part_words(TOP ? k.top : 0);
                if (lane == 0) {
                    p[0] = st.m;
                    p[1] = st.s;
                    p[2] = st.t;
                }
                if (TOP && lane < k.top) {
                    p[4 + lane] = bv;
                    reinterpret_cast<int *>(p)[4 + k.top + lane] = bi;
                }
            } else {
                const float ls = __builtin_amdgcn_logf(st.s) * kLn2;
                if (TOP && lane < k.top) write_top(k, n, lane, bv, bi, st.m, ls);
                if (lane == 0) write_row(k, n, st.m, st.s, st.t, has, ignored, zl);
            }
        }
        __syncthreads();
    }
}

// The segments' parts of a row together: a block a row, its waves a quarter of the segments each.  One row of 131071 scores in bf16
// with the 20 best: 8 us for its 32 segments and 8 us here, both of them latency (here: the bitwise searches over 640 pairs that are in order
// already).
template <typename T>
__global__ __launch_bounds__(256) void scores_join_kernel(const ScoresK k, const Cut cut) {
    __shared__ RowStat s_stat[4];
    __shared__ float s_max[256];
    __shared__ float s_v[4 * kBuf];
    __shared__ int s_i[4 * kBuf];
    constexpr int BITS = kKeyBits<T>;
    const LogitsK &g = k.g;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (long long n = blockIdx.x; n < g.rows; n += gridDim.x) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        const size_t words = part_words(k.top);
        const float *p = static_cast<const float *>(k.ws) + (size_t)n * cut.segs * words;
        int l = -1;
        bool has = false, ignored = false;
        float zl = 0.f;
        if (w == 0) {
            given_label(k, n, g.C + g.bg, l, has, ignored);
            if (has && l >= g.bg) zl = to_f32(z[l - g.bg]);
        }
        RowStat r = no_stat();
        for (int q = threadIdx.x; q < cut.segs; q += 256) {
            const float *a = p + q * words;
            r = join(r, {a[0], reference(a[0]), a[1], a[2]}, g.c2);
        }
        r = wave_join(r, g.c2);
        if (lane == 0) s_stat[w] = r;
        WaveBest b = {s_v + w * kBuf, s_i + w * kBuf, 0, kNegInf, 0, k.top};
        if (k.top) {
            const int pairs = cut.segs * k.top;
            // (the segments' first: k of them are at least as large as the k-th)
            if (cut.segs >= k.top) {
                s_max[threadIdx.x] = (int)threadIdx.x < cut.segs ? p[threadIdx.x * words + 4] : kNegInf;
                __syncthreads();
                b.floor = first_floor<4, BITS>(s_max, k.top);
            }
            for (int q0 = w * 64; q0 < pairs; q0 += 256) {
                const int q = q0 + lane, sg = q / k.top, at = q - sg * k.top;
                const float *a = p + sg * words + 4;
                // (a segment that offers fewer than k has empty slots behind its last: they are no pairs)
                const int id = q < pairs ? reinterpret_cast<const int *>(a)[k.top + at] : -1;
                b.take<BITS>(q < pairs ? a[at] : kNegInf, id, id >= 0);
            }
            if (b.n > 64) b.cut<BITS>();
            for (int q = b.n + lane; q < 64; q += 64) b.i[q] = -1;
        }
        __syncthreads();
        if (w == 0) {
            r = join(join(s_stat[0], s_stat[1], g.c2), join(s_stat[2], s_stat[3], g.c2), g.c2);
            if (lane == 0) write_row(k, n, r.m, r.s, r.t, has, ignored, zl);
            if (k.top) {
                float bv;
                int bi;
                final_best<4, BITS>(s_v, s_i, k.top, bv, bi);
                const float ls = __builtin_amdgcn_logf(r.s) * kLn2;
                if (lane < k.top) write_top(k, n, lane, bv, bi, r.m, ls);
            }
        }
        __syncthreads();
    }
}

// ---- planes: one lane a row, more than 8 classes ---------------------------------------------------------------------------
// Neighbouring lanes read neighbouring rows.  The best are a sorted list in registers.  A widened 2-byte score leaves the lower
// bits of its 32 unused: with the label's complement there, score and label are one unsigned key, and a key enters the list with
// one v_med3 a level; 4-byte scores carry the label beside.  The classes of one round are in flight while those before are worked
// on.  8 x 384 x 384 rows of 117 classes in f16: 65 us (4.3 TB/s), with the three best 84 (vector unit); in fp32 115 us (4.9 TB/s).
template <typename T>
constexpr int kLabelBits = 32 - kKeyBits<T>;
__device__ __forceinline__ unsigned minu(unsigned a, unsigned b) { return a < b ? a : b; }
__device__ __forceinline__ unsigned maxu(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned med3u(unsigned a, unsigned b, unsigned c) { return maxu(minu(a, b), minu(maxu(a, b), c)); }
template <typename T, int K>
struct LaneBest {  // any type: score and label side by side
    float v[K > 0 ? K : 1];
    int i[K > 0 ? K : 1];
    __device__ void clear() {
#pragma unroll
        for (int q = 0; q < K; ++q) {
            v[q] = kNegInf;
            i[q] = -1;
        }
    }
    __device__ void take(float x, int label) {
        if (K > 4 && __ballot(x > v[K > 0 ? K - 1 : 0]) == 0ull) return;
#pragma unroll
        for (int q = K - 1; q >= 0; --q) {
            const bool above = q > 0 && x > v[q > 0 ? q - 1 : 0], here = x > v[q];
            i[q] = above ? i[q > 0 ? q - 1 : 0] : (here ? label : i[q]);
            v[q] = above ? v[q > 0 ? q - 1 : 0] : (here ? x : v[q]);
        }
    }
    __device__ float score(int q) const { return v[q]; }
    __device__ int label(int q) const { return i[q]; }
};
template <typename T, int K>
struct LaneBestKey {  // 2-byte scores, labels that fit the unused bits
    static constexpr unsigned MASK = kLabelBits<T> < 32 ? (1u << (kLabelBits<T> % 32)) - 1u : 0u;
    unsigned key[K > 0 ? K : 1];
    __device__ void clear() {
#pragma unroll
        for (int q = 0; q < K; ++q) key[q] = 0u;
    }
    __device__ void take(float x, int label) {
        const unsigned k = (ordered(x) & ~MASK) | (MASK - (unsigned)label);
        if (K > 4 && __ballot(k > key[K > 0 ? K - 1 : 0]) == 0ull) return;
#pragma unroll
        for (int q = K - 1; q > 0; --q) key[q] = med3u(key[q - 1], key[q], k);
        if (K > 0) key[0] = maxu(key[0], k);
    }
    __device__ float score(int q) const {
        // (below the significant bits a negative score's key has ones)
        const unsigned o = key[q] & 0x80000000u ? key[q] & ~MASK : key[q] | MASK;
        return (key[q] & ~MASK) <= (kKeyNegInf & ~MASK) ? kNegInf : unordered(o);
    }
    __device__ int label(int q) const { return (int)(MASK - (key[q] & MASK)); }
};

//
// Long lists go out through LDS: 64 lanes that write each its own row ask for 64 lines a store.  A wave's rows lie one behind the
// other, so from LDS (a row every top | 1 words) they are written as one piece.
template <int K>
constexpr int kPlaneThreads = K > 32 ? 64 : 256;
template <typename T, int K, bool KEY, int CH>
__global__ __launch_bounds__(kPlaneThreads<K>) void scores_planes_kernel(const ScoresK k) {
    constexpr int B = kPlaneThreads<K>;
    extern __shared__ int s_top[];  // K > 4
    const LogitsK &g = k.g;
    const long long stride = (long long)gridDim.x * B;
    // (whole waves walk on together: the lists ask all lanes whether a score is worth entering)
    for (long long n0 = (long long)blockIdx.x * B + (threadIdx.x & ~63); n0 < g.rows; n0 += stride) {
        const long long nr = n0 + (threadIdx.x & 63);
        const bool live = nr < g.rows;
        const long long n = live ? nr : g.rows - 1;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        std::conditional_t<KEY, LaneBestKey<T, K>, LaneBest<T, K>> best;
        best.clear();
        Running r = no_scores();
        if (g.bg) {
            r = {0.f, 0.f, 1.f, 0.f};
            if (K) best.take(0.f, 0);
        }
        unsigned next[CH];
        load_classes(z, g.sc, g.C, next);
        const T *p = z;
        for (int c = 0; c < g.C; c += CH) {
            float x[CH];
#pragma unroll
            for (int i = 0; i < CH; ++i) x[i] = widen<T>(next[i]);
            p += CH * g.sc;
            if (c + CH < g.C) load_classes(p, g.sc, g.C - c - CH, next);
            add_scores(r, x, g.c2);
            if (K) {
#pragma unroll
                for (int i = 0; i < CH; ++i) best.take(x[i], c + i + g.bg);
            }
        }
        RowStat st = {r.m, reference(r.m), 0.f, 0.f};
        if (far_scores(r.m, g.c2)) {
            for (int c = -g.bg; c < g.C; ++c) {
                const float d = clamp2(((c < 0 ? 0.f : to_f32(z[(long long)c * g.sc])) - st.ref) * g.c2), e = exp2_hw(d);
                st.s += e;
                st.t = fmaf(e, d, st.t);
            }
        } else {
            float d;
            const float f = to_reference(r, r.m, g.c2, d);
            st.s = r.s * f;
            st.t = f * fmaf(d, r.s, r.t);
        }
        int l;
        bool has, ignored;
        given_label(k, n, g.C + g.bg, l, has, ignored);
        const float zl = (has && l >= g.bg) ? to_f32(z[(long long)(l - g.bg) * g.sc]) : 0.f;
        if (live) write_row(k, n, st.m, st.s, st.t, has, ignored, zl);
        if (K) {
            const float ls = __builtin_amdgcn_logf(st.s) * kLn2;
            if (K <= 4) {
#pragma unroll
                for (int q = 0; q < K; ++q) {
                    const float v = best.score(q);
                    if (live) write_top(k, n, q, v, v > kNegInf ? best.label(q) : -1, st.m, ls);
                }
            } else {
                const int lane = threadIdx.x & 63, step = k.top | 1;
                int *s = s_top + (threadIdx.x & ~63) * step;
                const long long left = g.rows - n0;
                const int all = (left < 64 ? (int)left : 64) * k.top;
                const float per = 1.f / (float)k.top;
                auto write_all = [&](auto value, auto out) {
#pragma unroll
                    for (int q = 0; q < K; ++q)
                        if (q < k.top) s[lane * step + q] = value(q);
                    wave_sync();
                    for (int i = lane; i < all; i += 64) {
                        const int r = (int)((i + 0.5f) * per);  // (i < 4096: exact)
                        out(n0 * k.top + i, s[r * step + i - r * k.top]);
                    }
                    wave_sync();
                };
                auto label = [&](int q) { return best.score(q) > kNegInf ? best.label(q) : -1; };
                write_all(label, [&](long long at, int v) { k.top_label[at] = v; });
                write_all([&](int q) { return __float_as_int(top_value(k, best.score(q), label(q), st.m, ls)); },
                          [&](long long at, int v) { k.top_log_prob[at] = __int_as_float(v); });
            }
        }
    }
}

// ---- wave: a wave a row, any strides -------------------------------------------------------------------------------------------
// Every score is a line of its own, so this is for calls whose rows are too few to fill lanes: latency.  8000 rows of 200 classes in
// f16, in planes: the kernel 7 us, with the three best 19.
template <typename T>
__device__ __forceinline__ float category(const LogitsK &g, const T *z, int j) {
    return (g.bg && j == 0) ? 0.f : to_f32(z[(long long)(j - g.bg) * g.sc]);
}
template <typename T>
__global__ __launch_bounds__(256) void scores_wave_kernel(const ScoresK k) {
    __shared__ float s_v[4 * kBuf];
    __shared__ int s_i[4 * kBuf];
    constexpr int BITS = kKeyBits<T>;
    const LogitsK &g = k.g;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, cats = g.C + g.bg;
    const long long nw = (long long)gridDim.x * 4;
    for (long long n = (long long)blockIdx.x * 4 + w; n < g.rows; n += nw) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        Running u = no_scores();
        WaveBest b = {s_v + w * kBuf, s_i + w * kBuf, 0, kNegInf, 0, k.top};
        auto score = [&](int j) { return j < cats ? category(g, z, j) : kNegInf; };
        for (int j0 = 0; j0 < cats; j0 += 256) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = score(j0 + i * 64 + lane);
            add_scores(u, x, g.c2);
            if (k.top) {
#pragma unroll 1
                for (int i = 0; i < 4; ++i) {
                    const float v = i == 0 ? x[0] : i == 1 ? x[1] : i == 2 ? x[2] : x[3];
                    b.take<BITS>(v, j0 + i * 64 + lane, true);
                }
            }
        }
        const RowStat r = wave_stat(u, g.c2, score, lane, 64, cats);
        if (lane == 0) {
            int l;
            bool has, ignored;
            given_label(k, n, cats, l, has, ignored);
            write_row(k, n, r.m, r.s, r.t, has, ignored, has ? category(g, z, l) : 0.f);
        }
        if (k.top) {
            b.cut<BITS>();
            float bv = lane < b.n ? b.v[lane] : kNegInf;
            int bi = lane < b.n ? b.i[lane] : -1;
            const int at = rank_of(bv, bi, b.n);
            const float ls = __builtin_amdgcn_logf(r.s) * kLn2;
            // (lanes without a winner keep their own slot: they come behind the winners)
            if (lane < k.top) write_top(k, n, lane < b.n ? at : lane, bv, bi, r.m, ls);
            wave_sync();
        }
    }
}

// ---- gradient ---------------------------------------------------------------------------------------------------------------
// One exponent a score from the row's maximum and sum; no exchange between lanes.  Bound by memory: small 26 us for 16 x 384 x 384
// rows of 4 fp32 classes in planes (4.8 TB/s), rows in registers 79 us for 200000 x 500 in bf16 (5.1 TB/s), blocks 86 us for 1024 x 100003
// in bf16 (4.8 TB/s), planes 115 us for 8 x 384 x 384 x 117 in f16 (4.9 TB/s).
struct GradRow {
    float M, l2s, ls, a, b, H;
    int l;
    bool zero;
};
__device__ __forceinline__ GradRow grad_row(const ScoresK &k, long long n, int cats) {
    GradRow r;
    const float2 nm = *reinterpret_cast<const float2 *>(k.norm + 2 * n);
    r.M = nm.x;
    r.ls = nm.y;
    r.l2s = nm.y * kLog2e;
    r.zero = nm.x == kNegInf;
    r.a = r.b = r.H = 0.f;
    r.l = -1;
    if (k.g_log_prob) {
        const long long l = load_label(k.labels, k.l_kind, n);
        if (l != k.ignore) {
            r.a = k.g_log_prob[n];
            if (l >= 0 && l < cats) r.l = (int)l;
            else r.a = __builtin_nanf("");
        }
    }
    if (k.g_entropy) {
        r.b = k.g_entropy[n];
        r.H = k.entropy[n];
    }
    return r;
}
// gradient of category j with score v
__device__ __forceinline__ float grad_score(const GradRow &r, float c2, float invT, float v, int j) {
    const float d = clamp2((v - r.M) * c2), p = exp2_hw(d - r.l2s);
    // log p + H; p log p is 0 where p is (the clamp keeps the logarithm finite)
    const float lp = fmaf(d, kLn2, r.H - r.ls);
    float q = -p * fmaf(r.b, lp, r.a);
    if (j == r.l) q += r.a;
    return r.zero ? 0.f : q * invT;
}

template <typename T, int N, bool CONTIG>
__global__ __launch_bounds__(256) void scores_grad_small_kernel(const ScoresK k) {
    const LogitsK &g = k.g;
    const long long stride = (long long)gridDim.x * 256;
    for (long long n = (long long)blockIdx.x * 256 + threadIdx.x; n < g.rows; n += stride) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        T *out = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi);
        struct {
            T v[N];
        } x;
        if (CONTIG) __builtin_memcpy(&x, z, sizeof(x));
        else
#pragma unroll
            for (int j = 0; j < N; ++j) x.v[j] = z[j * g.sc];
        const GradRow r = grad_row(k, n, g.C + g.bg);
#pragma unroll
        for (int j = 0; j < N; ++j) x.v[j] = from_f32<T>(grad_score(r, g.c2, g.invT, to_f32(x.v[j]), j + g.bg));
        if (CONTIG) __builtin_memcpy(out, &x, sizeof(x));
        else
#pragma unroll
            for (int j = 0; j < N; ++j) out[j * k.gsc] = x.v[j];
    }
}

template <typename T, int G>
__global__ __launch_bounds__(256) void scores_grad_group_kernel(const ScoresK k) {
    const LogitsK &g = k.g;
    constexpr int V = kVec<T>, NV = 16 / V, ROWS = 256 / G;
    const int gl = threadIdx.x % G;
    for (long long n = (long long)blockIdx.x * ROWS + threadIdx.x / G; n < g.rows; n += (long long)gridDim.x * ROWS) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        T *out = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi);
        Vec<T> x[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * G + gl) * V;
            x[i] = load_vec(z + j - vec_back<T>(g.C - j));
        }
        const GradRow r = grad_row(k, n, g.C + g.bg);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            // (the vector moved to the front: scores that another lane has too get the same value from both)
            const int j = (i * G + gl) * V, at = j - vec_back<T>(g.C - j);
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = grad_score(r, g.c2, g.invT, get(x[i], e), at + e + g.bg);
            if (j < g.C) store_vec(out + at, pack_vec<T>(y));
        }
    }
}

// W waves a segment of a row, 16 scores a lane at a time and the next 16 in flight.
template <typename T, int W>
__global__ __launch_bounds__(64 * W) void scores_grad_block_kernel(const ScoresK k, const Cut cut) {
    const LogitsK &g = k.g;
    constexpr int V = kVec<T>, NV = 16 / V, TILE = 1024 * W;
    for (long long item = blockIdx.x; item < g.rows * cut.segs; item += gridDim.x) {
        const long long n = cut.segs == 1 ? item : item / cut.segs;
        const int c0 = (int)(item - n * cut.segs) * cut.len, c1 = c0 + cut.len < g.C ? c0 + cut.len : g.C;
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
        const GradRow r = grad_row(k, n, g.C + g.bg);
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
                for (int e = 0; e < V; ++e) y[e] = grad_score(r, g.c2, g.invT, get(now[i], e), j - back + e + g.bg);
                // (the row's last vector, moved to the front: what lies before j is another lane's)
                if (back == 0) store_vec(out + j, pack_vec<T>(y));
                else store_end(out + j - back, y, back);
            }
        }
    }
}

// Classes that do not lie together: neighbouring lanes take neighbouring rows, a block 256 rows and `len` classes of them.
template <typename T>
__global__ __launch_bounds__(256) void scores_grad_planes_kernel(const ScoresK k, int parts, int len) {
    const LogitsK &g = k.g;
    const long long blocks = (g.rows + 255) / 256;
    for (long long item = blockIdx.x; item < blocks * parts; item += gridDim.x) {
        const long long rb = parts == 1 ? item : item / parts;
        const int c0 = (int)(item - rb * parts) * len, c1 = c0 + len < g.C ? c0 + len : g.C;
        const long long n = rb * 256 + threadIdx.x;
        if (n >= g.rows) continue;
        const T *p = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si) + c0 * g.sc;
        T *out = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi) + c0 * k.gsc;
        unsigned next[8];
        load_classes(p, g.sc, c1 - c0, next);
        const GradRow r = grad_row(k, n, g.C + g.bg);
        for (int c = c0; c < c1; c += 8) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = widen<T>(next[i]);
            p += 8 * g.sc;
            if (c + 8 < c1) load_classes(p, g.sc, c1 - c - 8, next);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = grad_score(r, g.c2, g.invT, y[i], c + i + g.bg);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < c1) out[i * k.gsc] = from_f32<T>(y[i]);
            out += 8 * k.gsc;
        }
    }
}

// ---- dispatch ---------------------------------------------------------------------------------------------------------------
unsigned grid_of(long long blocks, int num_cu, int per_cu) {
    const long long cap = (long long)num_cu * per_cu;
    return (unsigned)(blocks < 1 ? 1 : blocks < cap ? blocks : cap);
}
bool contiguous(const LogitsK &g) { return g.sc == 1 || g.C == 1; }

template <typename T, int N>
void small(const ScoresK &k, bool contig, int num_cu, hipStream_t st) {
    const dim3 grid(grid_of((k.g.rows + 255) / 256, num_cu, 64)), block(256);
    if (contig) {
        if (k.g.bg) hipLaunchKernelGGL((scores_small_kernel<T, N, true, true>), grid, block, 0, st, k);
        else hipLaunchKernelGGL((scores_small_kernel<T, N, false, true>), grid, block, 0, st, k);
    } else {
        if (k.g.bg) hipLaunchKernelGGL((scores_small_kernel<T, N, true, false>), grid, block, 0, st, k);
        else hipLaunchKernelGGL((scores_small_kernel<T, N, false, false>), grid, block, 0, st, k);
    }
}
template <typename T, int N>
void small_grad(const ScoresK &k, bool contig, int num_cu, hipStream_t st) {
    const dim3 grid(grid_of((k.g.rows + 255) / 256, num_cu, 64)), block(256);
    if (contig) hipLaunchKernelGGL((scores_grad_small_kernel<T, N, true>), grid, block, 0, st, k);
    else hipLaunchKernelGGL((scores_grad_small_kernel<T, N, false>), grid, block, 0, st, k);
}
template <typename T, int G>
void group(const ScoresK &k, bool grad, int num_cu, hipStream_t st) {
    const dim3 grid(grid_of((k.g.rows + 256 / G - 1) / (256 / G), num_cu, 64)), block(256);
    if (grad) hipLaunchKernelGGL((scores_grad_group_kernel<T, G>), grid, block, 0, st, k);
    else if (k.top) hipLaunchKernelGGL((scores_group_kernel<T, G, true>), grid, block, 0, st, k);
    else hipLaunchKernelGGL((scores_group_kernel<T, G, false>), grid, block, 0, st, k);
}
template <typename T, int K>
void planes(const ScoresK &k, int num_cu, hipStream_t st) {
    constexpr int B = kPlaneThreads<K>;
    const dim3 grid(grid_of((k.g.rows + B - 1) / B, num_cu, 64 * (256 / B))), block(B);
    const size_t lds = K > 4 ? (size_t)B * (k.top | 1) * 4 : 0;
    if constexpr (sizeof(T) == 2) {
        // (the last CH classes may reach CH - 1 labels beyond the last)
        const bool key = k.g.C + k.g.bg + 15 <= (1 << kLabelBits<T>);
        if constexpr (K <= 4) {
            // 16 classes in flight where 2-byte rows are long enough (117 classes in f16: 64 us instead of 73, with the best 75 and 82; 20
            // classes 22 and 19; nothing between is measured; 4-byte scores are no faster with it)
            if (key && k.g.C > 48) {
                hipLaunchKernelGGL((scores_planes_kernel<T, K, true, 16>), grid, block, lds, st, k);
                return;
            }
        }
        if (key) {
            hipLaunchKernelGGL((scores_planes_kernel<T, K, true, 8>), grid, block, lds, st, k);
            return;
        }
    }
    hipLaunchKernelGGL((scores_planes_kernel<T, K, false, 8>), grid, block, lds, st, k);
}

template <typename T>
void launch(const ScoresK &k, int num_cu, hipStream_t st) {
    const LogitsK &g = k.g;
    const bool contig = contiguous(g);
    if (g.C <= 8) {
        switch (g.C) {
            case 1: return small<T, 1>(k, contig, num_cu, st);
            case 2: return small<T, 2>(k, contig, num_cu, st);
            case 3: return small<T, 3>(k, contig, num_cu, st);
            case 4: return small<T, 4>(k, contig, num_cu, st);
            case 5: return small<T, 5>(k, contig, num_cu, st);
            case 6: return small<T, 6>(k, contig, num_cu, st);
            case 7: return small<T, 7>(k, contig, num_cu, st);
            default: return small<T, 8>(k, contig, num_cu, st);
        }
    }
    if (!contig) {
        if (!lane_rows(g, num_cu)) {
            hipLaunchKernelGGL(scores_wave_kernel<T>, dim3(grid_of((g.rows + 3) / 4, num_cu, 32)), dim3(256), 0, st, k);
            return;
        }
        switch (k.top) {
            case 0: return planes<T, 0>(k, num_cu, st);
            case 1: return planes<T, 1>(k, num_cu, st);
            case 2: return planes<T, 2>(k, num_cu, st);
            case 3: return planes<T, 3>(k, num_cu, st);
            case 4: return planes<T, 4>(k, num_cu, st);
        }
        if (k.top <= 8) return planes<T, 8>(k, num_cu, st);
        if (k.top <= 16) return planes<T, 16>(k, num_cu, st);
        if (k.top <= 32) return planes<T, 32>(k, num_cu, st);
        return planes<T, 64>(k, num_cu, st);
    }
    if (g.C <= 32) return group<T, 2>(k, false, num_cu, st);
    if (g.C <= 64) return group<T, 4>(k, false, num_cu, st);
    if (g.C <= 128) return group<T, 8>(k, false, num_cu, st);
    if (g.C <= 256) return group<T, 16>(k, false, num_cu, st);
    if (g.C <= 512) return group<T, 32>(k, false, num_cu, st);
    if (g.C <= 1024) return group<T, 64>(k, false, num_cu, st);
    const Cut cut = cut_rows(g, num_cu, 1 << 30);
    const dim3 grid(grid_of(g.rows * cut.segs, num_cu, 64));
    // A wave a row, with no other to wait for, where every SIMD has four rows: 50000 x 1999 in bf16 65 us, with the 8 best 116 (four waves
    // a row: 107, 226).  From 16 KB a row on there is nothing in it (8192 x 8192: 34 and 35), in 4-byte scores it loses (61 and 54).
    if (g.C <= 16384 / (int)sizeof(T) && g.rows >= 16ll * num_cu) {
        if (k.top) hipLaunchKernelGGL((scores_block_kernel<T, true, 1>), grid, dim3(64), 0, st, k, cut);
        else hipLaunchKernelGGL((scores_block_kernel<T, false, 1>), grid, dim3(64), 0, st, k, cut);
    } else if (k.top) {
        hipLaunchKernelGGL((scores_block_kernel<T, true, 4>), grid, dim3(256), 0, st, k, cut);
    } else {
        hipLaunchKernelGGL((scores_block_kernel<T, false, 4>), grid, dim3(256), 0, st, k, cut);
    }
    if (cut.segs > 1) hipLaunchKernelGGL(scores_join_kernel<T>, dim3(grid_of(g.rows, num_cu, 64)), dim3(256), 0, st, k, cut);
}

template <typename T>
void launch_grad(const ScoresK &k, int num_cu, hipStream_t st) {
    const LogitsK &g = k.g;
    const bool contig = contiguous(g) && (k.gsc == 1 || g.C == 1);
    if (g.C <= 8) {
        switch (g.C) {
            case 1: return small_grad<T, 1>(k, contig, num_cu, st);
            case 2: return small_grad<T, 2>(k, contig, num_cu, st);
            case 3: return small_grad<T, 3>(k, contig, num_cu, st);
            case 4: return small_grad<T, 4>(k, contig, num_cu, st);
            case 5: return small_grad<T, 5>(k, contig, num_cu, st);
            case 6: return small_grad<T, 6>(k, contig, num_cu, st);
            case 7: return small_grad<T, 7>(k, contig, num_cu, st);
            default: return small_grad<T, 8>(k, contig, num_cu, st);
        }
    }
    if (!contig) {
        int parts;
        const int len = cut_classes(g, num_cu, parts);
        hipLaunchKernelGGL(scores_grad_planes_kernel<T>, dim3(grid_of((g.rows + 255) / 256 * parts, num_cu, 64)), dim3(256), 0, st, k, parts, len);
        return;
    }
    if (g.C <= 32) return group<T, 2>(k, true, num_cu, st);
    if (g.C <= 64) return group<T, 4>(k, true, num_cu, st);
    if (g.C <= 128) return group<T, 8>(k, true, num_cu, st);
    if (g.C <= 256) return group<T, 16>(k, true, num_cu, st);
    if (g.C <= 512) return group<T, 32>(k, true, num_cu, st);
    if (g.C <= 1024) return group<T, 64>(k, true, num_cu, st);
    // a block a piece of 4096 scores, one round of its loads (4-byte scores: 8192 x 16384 in 190 us, by blocks that go on to the next
    // pieces 228); a wave a row where that leaves lanes without scores (50000 x 1999 in bf16: 92 us, in pieces 146)
    const bool wave = wave_rows_grad<T>(g, num_cu);
    const Cut cut = {wave ? 1 : (g.C + 4095) / 4096, wave ? g.C : 4096};
    if (wave) hipLaunchKernelGGL((scores_grad_block_kernel<T, 1>), dim3(grid_of(g.rows, num_cu, 64)), dim3(64), 0, st, k, cut);
    else hipLaunchKernelGGL((scores_grad_block_kernel<T, 4>), dim3(grid_of(g.rows * cut.segs, num_cu, 256)), dim3(256), 0, st, k, cut);
}

}  // namespace

size_t label_scores_workspace_bytes(const ScoresK &k, int, int num_cu) {
    if (k.g.C <= QMRI_SHORT_ROW || !contiguous(k.g)) return 0;
    const Cut cut = cut_rows(k.g, num_cu, 1 << 30);
    return cut.segs > 1 ? (size_t)k.g.rows * cut.segs * (4 + 2 * (size_t)k.top) * 4 : 0;
}

hipError_t label_scores_launch(const ScoresK &k, int dtype, int num_cu, hipStream_t st) {
    (void)hipGetLastError();
    if (dtype == QMRI_F32) launch<float>(k, num_cu, st);
    else if (dtype == QMRI_F16) launch<f16_t>(k, num_cu, st);
    else launch<bf16_t>(k, num_cu, st);
    return hipGetLastError();
}

hipError_t label_scores_grad_launch(const ScoresK &k, int dtype, int num_cu, hipStream_t st) {
    (void)hipGetLastError();
    if (dtype == QMRI_F32) launch_grad<float>(k, num_cu, st);
    else if (dtype == QMRI_F16) launch_grad<f16_t>(k, num_cu, st);
    else launch_grad<bf16_t>(k, num_cu, st);
    return hipGetLastError();
}

}  // namespace qmri
