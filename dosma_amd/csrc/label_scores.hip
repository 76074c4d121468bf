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
#include "answers.h"

namespace qmri {

Cut cut_rows(const LogitsK &g, int num_cu) {
    // enough blocks for every compute unit twice over, but at least 2048 scores (two rounds of a block's loads) for each
    long long want = g.rows >= 2ll * num_cu ? 1 : (2ll * num_cu + g.rows - 1) / g.rows;
    const long long most = (g.C + 2047) / 2048;
    if (want > most) want = most;
    const long long least = (g.C + 65535) / 65536;
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
__device__ __forceinline__ void write_top(const ScoresK &k, long long n, int q, float v, int i, float M, float ls) {
    k.top_label[n * k.top + q] = i;
    k.top_log_prob[n * k.top + q] = i < 0 ? (ls != ls ? ls : kNegInf) : (v - reference(M)) * k.g.invT - ls;
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

// ---- small: one lane a row ----------------------------------------------------------------------------------------------------
// Bound by memory and, right behind, by the vector unit: a row of 4 scores in 32 bits is 16 bytes in and up to 32 out.
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
template <typename T, int G>
__global__ __launch_bounds__(256) void scores_group_kernel(const ScoresK k) {
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
            const Vec<T> r = j + V <= g.C ? load_vec(z + j) : load_part(z + j, g.C - j);
#pragma unroll
            for (int e = 0; e < V; ++e) x[i * V + e] = to_f32(r.v[e]);
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
        if (k.top == 0) continue;
        const float ls = __builtin_amdgcn_logf(s) * kLn2;
        for (int q = 0; q < k.top; ++q) {
            // the largest of this lane's 16 (the first of equals: its labels rise with i only within a vector and from vector to vector)
            float bv = x[16];
            int bi = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool c = x[i] > bv;
                bv = c ? x[i] : bv;
                bi = c ? ((i / V) * G + gl) * V + i % V + g.bg : bi;
            }
            const float best = group_max<G>(bv);
            const int at = group_min<G>(bv == best ? bi : 0x7fffffff);
            if (live && gl == 0) write_top(k, n, q, best, best > kNegInf ? at : -1, M, ls);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = ((i / V) * G + gl) * V + i % V + g.bg == at ? kNegInf : x[i];
            if (at == 0 && g.bg) x[16] = kNegInf;
        }
    }
}

// ---- the best of a long row: a sorted list over the 64 lanes of a wave ----------------------------------------------------------
struct Best {
    float v;  // lane i: the i-th best score seen by this wave
    int i;    // its label
    float floor;  // scores that are not above it cannot enter the list (the same in every lane)
};
// lane i takes lane i - 1's value
__device__ __forceinline__ int from_left(int x) { return __builtin_amdgcn_update_dpp(x, x, 0x138, 0xf, 0xf, false); }
// (wave-uniform v, i): into the list behind everything that is better
__device__ __forceinline__ void best_insert(Best &b, float v, int i, int k) {
    const int lane = threadIdx.x & 63;
    const int pos = __popcll(__ballot(better(b.v, b.i, v, i)));
    const float lv = __int_as_float(from_left(__float_as_int(b.v)));
    const int li = from_left(b.i);
    b.v = lane > pos ? lv : (lane == pos ? v : b.v);
    b.i = lane > pos ? li : (lane == pos ? i : b.i);
    b.floor = fmaxf(b.floor, __int_as_float(__builtin_amdgcn_readlane(__float_as_int(b.v), k - 1)));
}
// k-th largest of the lanes' values, less one step: k scores at least as large as it are known to exist, so nothing at or below
// that step can belong to the best k.  A bitonic sort over the wave.
__device__ __forceinline__ float kth_floor(float c, int k) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int w = 2; w <= 64; w <<= 1)
#pragma unroll
        for (int o = w >> 1; o > 0; o >>= 1) {
            const float p = __shfl_xor(c, o);
            const bool up = (lane & w) != 0;        // (w = 64: every lane falls)
            const bool low = (lane & o) == 0;
            c = (up != low) ? fmaxf(c, p) : fminf(c, p);
        }
    const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(c), k - 1));
    if (!(f > kNegInf)) return kNegInf;
    const int u = __float_as_int(f);
    return f == 0.f ? __int_as_float(0x80000001u) : __int_as_float(f > 0.f ? u - 1 : u + 1);
}
// V neighbouring scores a lane, labels rising with the lane: what can still enter the list does.  In the order of the labels, so
// that of equal scores the lower label comes first and a later equal one is not above the floor.
template <int V>
__device__ __forceinline__ void best_take(Best &b, const float (&x)[V], float cm, int first, int k) {
    unsigned long long m = __ballot(cm > b.floor);
    if (m == 0ull) return;
    // many at once (the start of a row, or one that rises): sort the lanes' largest first, which leaves about k of them
    if (__popcll(m) > 12) {
        b.floor = fmaxf(b.floor, kth_floor(cm, k));
        m = __ballot(cm > b.floor);
    }
    while (m) {
        const int l = __ffsll(m) - 1;
        m &= m - 1;
        const int at = __builtin_amdgcn_readlane(first, l);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x[e]), l));
            if (v > b.floor) best_insert(b, v, at + e, k);
        }
    }
}

// a segment's part of a row in the workspace: m, s (relative to reference(m)), t, then the list's scores and labels
__device__ __forceinline__ size_t part_words(int k) { return 4 + 2 * (size_t)k; }

// ---- block: four waves a segment of a row -----------------------------------------------------------------------------------
// Per score: widen, subtract, multiply, clamp, exp2, two sums -- about 10 issue slots, of the 14 that a 2-byte score has at 5.5
// TB/s: memory first, the vector unit close behind.  A lane's reference follows its maximum only when that has grown by more than
// a factor of 16, so nearly no step pays for a change of reference.
constexpr float kSlack = 4.f;

template <typename T, bool TOP>
__global__ __launch_bounds__(256) void scores_block_kernel(const ScoresK k, const Cut cut) {
    __shared__ RowStat s_stat[4];
    __shared__ float s_v[4][64];
    __shared__ int s_i[4][64];
    const LogitsK &g = k.g;
    constexpr int V = kVec<T>, U = 16 / V, TILE = 64 * 16;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long long work = g.rows * cut.segs;
    for (long long item = blockIdx.x; item < work; item += gridDim.x) {
        const long long n = cut.segs == 1 ? item : item / cut.segs;
        const int seg = cut.segs == 1 ? 0 : (int)(item - n * cut.segs);
        const int c0 = seg * cut.len, c1 = c0 + cut.len < g.C ? c0 + cut.len : g.C;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        RowStat r = no_stat();
        Best b = {kNegInf, -1, kNegInf};
        if (g.bg && seg == 0 && w == 0) {  // the implicit category: lane 0 has seen a score of 0
            if (lane == 0) r = {0.f, 0.f, 1.f, 0.f};
            if (TOP) best_insert(b, 0.f, 0, k.top);
        }
        Vec<T> nx[U];
        auto fetch = [&](int c) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = c + u * 64 * V + lane * V;
                nx[u] = j + V <= c1 ? load_vec(z + j) : load_part(z + j, c1 - j);
            }
        };
        int c = c0 + w * TILE;
        if (c < c1) fetch(c);
        for (; c < c1; c += 4 * TILE) {
            Vec<T> now[U];
#pragma unroll
            for (int u = 0; u < U; ++u) now[u] = nx[u];
            if (c + 4 * TILE < c1) fetch(c + 4 * TILE);
            float x[16], um[U], cm = kNegInf;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                um[u] = kNegInf;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x[u * V + e] = to_f32(now[u].v[e]);
                    um[u] = maxn(um[u], x[u * V + e]);
                }
                cm = maxn(cm, um[u]);
            }
            r.m = maxn(r.m, cm);
            if ((cm - r.ref) * g.c2 > kSlack) rebase(r, cm, g.c2);
            float e[16], et[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float d = clamp2((x[i] - r.ref) * g.c2);
                e[i] = exp2_hw(d);
                et[i] = e[i] * d;
            }
            r.s += tree_sum(e);
            r.t += tree_sum(et);
            if (TOP) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float xv[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) xv[i] = x[u * V + i];
                    best_take<V>(b, xv, um[u], c + u * 64 * V + lane * V + g.bg, k.top);
                }
            }
        }
        r = wave_join(r, g.c2);
        if (lane == 0) s_stat[w] = r;
        if (TOP) {
            s_v[w][lane] = b.v;
            s_i[w][lane] = b.i;
        }
        __syncthreads();
        if (w == 0) {
            r = join(join(s_stat[0], s_stat[1], g.c2), join(s_stat[2], s_stat[3], g.c2), g.c2);
            if (TOP) {
                for (int o = 1; o < 4; ++o)
                    for (int q = 0; q < k.top; ++q) {
                        const float v = s_v[o][q];
                        const int i = s_i[o][q];
                        const float kv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(b.v), k.top - 1));
                        const int ki = __builtin_amdgcn_readlane(b.i, k.top - 1);
                        if (i < 0 || (ki >= 0 && !better(v, i, kv, ki))) break;  // (the other lists fall too)
                        best_insert(b, v, i, k.top);
                    }
            }
            if (cut.segs > 1) {
                float *p = static_cast<float *>(k.ws) + (size_t)item * part_words(TOP ? k.top : 0);
                if (lane == 0) {
                    p[0] = r.m;
                    p[1] = r.s;
                    p[2] = r.t;
                }
                if (TOP && lane < k.top) {
                    p[4 + lane] = b.v;
                    reinterpret_cast<int *>(p)[4 + k.top + lane] = b.i;
                }
            } else {
                const float ls = __builtin_amdgcn_logf(r.s) * kLn2;
                if (TOP && lane < k.top) write_top(k, n, lane, b.v, b.i, r.m, ls);
                if (lane == 0) {
                    int l;
                    bool has, ignored;
                    given_label(k, n, g.C + g.bg, l, has, ignored);
                    const float zl = (has && l >= g.bg) ? to_f32(z[l - g.bg]) : 0.f;
                    write_row(k, n, r.m, r.s, r.t, has, ignored, zl);
                }
            }
        }
        __syncthreads();
    }
}

// The segments' parts of a row together: one wave a row.
template <typename T>
__global__ __launch_bounds__(64) void scores_join_kernel(const ScoresK k, const Cut cut) {
    const LogitsK &g = k.g;
    const int lane = threadIdx.x;
    for (long long n = blockIdx.x; n < g.rows; n += gridDim.x) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        const size_t words = part_words(k.top);
        const float *p = static_cast<const float *>(k.ws) + (size_t)n * cut.segs * words;
        int l;
        bool has, ignored;
        given_label(k, n, g.C + g.bg, l, has, ignored);
        const float zl = (has && l >= g.bg) ? to_f32(z[l - g.bg]) : 0.f;
        RowStat r = no_stat();
        for (int q = lane; q < cut.segs; q += 64) {
            const float *a = p + q * words;
            RowStat o = {a[0], reference(a[0]), a[1], a[2]};
            r = join(r, o, g.c2);
        }
        r = wave_join(r, g.c2);
        if (lane == 0) write_row(k, n, r.m, r.s, r.t, has, ignored, zl);
        if (k.top) {
            Best b = {kNegInf, -1, kNegInf};
            for (int q0 = 0; q0 < cut.segs; q0 += 64) {
                // the segments' best, a lane a segment; a segment whose list cannot add anything is passed over
                for (int q = q0; q < cut.segs && q < q0 + 64; ++q) {
                    const float *a = p + q * words;
                    const float sv = lane < k.top ? a[4 + lane] : kNegInf;
                    const int si = lane < k.top ? reinterpret_cast<const int *>(a)[4 + k.top + lane] : -1;
                    for (int i = 0; i < k.top; ++i) {
                        const float v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sv), i));
                        const int id = __builtin_amdgcn_readlane(si, i);
                        if (id < 0 || !(v > b.floor)) break;  // (segments come in the order of their labels: an equal score is too late)
                        best_insert(b, v, id, k.top);
                    }
                }
            }
            const float ls = __builtin_amdgcn_logf(r.s) * kLn2;
            if (lane < k.top) write_top(k, n, lane, b.v, b.i, r.m, ls);
        }
    }
}

// ---- planes: one lane a row, more than 8 classes ---------------------------------------------------------------------------
// Neighbouring lanes read neighbouring rows.  The best are a sorted list in registers.  Of 2-byte scores a key of 32 bits, the
// ordered score over the complement of the label, enters it with one v_med3 a level; 4-byte scores carry the label beside.
__device__ __forceinline__ unsigned score_key(unsigned short u, int label) {
    const unsigned hi = (u == 0x8000u) ? 0u : (unsigned)u << 16;  // -0 ranks as +0
    const unsigned ordered = hi ^ ((unsigned)((int)hi >> 31) | 0x80000000u);
    return (ordered & 0xffff0000u) | (0xffffu - (unsigned)label);
}
__device__ __forceinline__ unsigned med3u(unsigned a, unsigned b, unsigned c) {
    const unsigned lo = a < b ? a : b, hi = a < b ? b : a;
    return hi < c ? hi : (lo > c ? lo : c);
}
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
    __device__ void take(T, float x, int label) {
        if (K > 4 && __ballot(x > v[K - 1]) == 0ull) return;
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
struct LaneBestKey {  // 2-byte scores, labels below 65536 (those of the last, partly filled step of 8 included)
    unsigned key[K > 0 ? K : 1];
    __device__ void clear() {
#pragma unroll
        for (int q = 0; q < K; ++q) key[q] = 0u;
    }
    __device__ void take(T raw, float, int label) {
        unsigned short u;
        __builtin_memcpy(&u, &raw, 2);
        const unsigned x = score_key(u, label);
        if (K > 4 && __ballot(x > key[K - 1]) == 0ull) return;
#pragma unroll
        for (int q = K - 1; q > 0; --q) key[q] = med3u(key[q - 1], key[q], x);
        if (K > 0) key[0] = key[0] > x ? key[0] : x;
    }
    __device__ float score(int q) const {
        const unsigned o = key[q] & 0xffff0000u;
        unsigned hi = (o & 0x80000000u) ? o ^ 0x80000000u : ~o & 0xffff0000u;
        if (key[q] == 0u) return kNegInf;
        const unsigned short u = (unsigned short)(hi >> 16);
        T r;
        __builtin_memcpy(&r, &u, 2);
        return to_f32(r);
    }
    __device__ int label(int q) const { return score(q) > kNegInf ? (int)(0xffffu - (key[q] & 0xffffu)) : -1; }
};

template <typename T, int K, bool KEY>
__global__ __launch_bounds__(256) void scores_planes_kernel(const ScoresK k) {
    const LogitsK &g = k.g;
    const long long stride = (long long)gridDim.x * 256;
    // (whole waves walk on together: the lists ask all lanes whether a score is worth entering)
    for (long long n0 = (long long)blockIdx.x * 256 + (threadIdx.x & ~63); n0 < g.rows; n0 += stride) {
        const long long nr = n0 + (threadIdx.x & 63);
        const bool live = nr < g.rows;
        const long long n = live ? nr : g.rows - 1;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        std::conditional_t<KEY, LaneBestKey<T, K>, LaneBest<T, K>> best;
        best.clear();
        RowStat r = no_stat();
        if (g.bg) {
            r = {0.f, 0.f, 1.f, 0.f};
            if (K) best.take(static_cast<T>(0.f), 0.f, 0);
        }
        for (int c = 0; c < g.C; c += 8) {
            T raw[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i] = c + i < g.C ? z[(long long)(c + i) * g.sc] : static_cast<T>(kNegInf);
            float x[8], cm = kNegInf;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = to_f32(raw[i]);
                cm = maxn(cm, x[i]);
            }
            r.m = maxn(r.m, cm);
            if ((cm - r.ref) * g.c2 > kSlack) rebase(r, cm, g.c2);
            float e[8], et[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = clamp2((x[i] - r.ref) * g.c2);
                e[i] = exp2_hw(d);
                et[i] = e[i] * d;
            }
            r.s += tree_sum(e);
            r.t += tree_sum(et);
            if (K) {
#pragma unroll
                for (int i = 0; i < 8; ++i) best.take(raw[i], x[i], c + i + g.bg);
            }
        }
        rebase(r, reference(r.m), g.c2);
        if (!live) continue;
        int l;
        bool has, ignored;
        given_label(k, n, g.C + g.bg, l, has, ignored);
        const float zl = (has && l >= g.bg) ? to_f32(z[(long long)(l - g.bg) * g.sc]) : 0.f;
        write_row(k, n, r.m, r.s, r.t, has, ignored, zl);
        if (K) {
            const float ls = __builtin_amdgcn_logf(r.s) * kLn2;
#pragma unroll
            for (int q = 0; q < K; ++q)
                if (q < k.top) {
                    const float v = best.score(q);
                    write_top(k, n, q, v, v > kNegInf ? best.label(q) : -1, r.m, ls);
                }
        }
    }
}

// ---- wave: a wave a row, any strides -------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float category(const LogitsK &g, const T *z, int j) {
    return (g.bg && j == 0) ? 0.f : to_f32(z[(long long)(j - g.bg) * g.sc]);
}
template <typename T>
__global__ __launch_bounds__(256) void scores_wave_kernel(const ScoresK k) {
    const LogitsK &g = k.g;
    const int lane = threadIdx.x & 63, cats = g.C + g.bg;
    const long long nw = (long long)gridDim.x * 4;
    for (long long n = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); n < g.rows; n += nw) {
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        RowStat r = no_stat();
        Best b = {kNegInf, -1, kNegInf};
        for (int j0 = 0; j0 < cats; j0 += 256) {
            float x[4], cm = kNegInf;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = j0 + i * 64 + lane;
                x[i] = j < cats ? category(g, z, j) : kNegInf;
                cm = maxn(cm, x[i]);
            }
            r.m = maxn(r.m, cm);
            if ((cm - r.ref) * g.c2 > kSlack) rebase(r, cm, g.c2);
            float e[4], et[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float d = clamp2((x[i] - r.ref) * g.c2);
                e[i] = exp2_hw(d);
                et[i] = e[i] * d;
            }
            r.s += tree_sum(e);
            r.t += tree_sum(et);
            if (k.top) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float xv[1] = {x[i]};
                    best_take<1>(b, xv, x[i], j0 + i * 64 + lane, k.top);
                }
            }
        }
        r = wave_join(r, g.c2);
        if (lane == 0) {
            int l;
            bool has, ignored;
            given_label(k, n, cats, l, has, ignored);
            write_row(k, n, r.m, r.s, r.t, has, ignored, has ? category(g, z, l) : 0.f);
        }
        const float ls = __builtin_amdgcn_logf(r.s) * kLn2;
        if (lane < k.top) write_top(k, n, lane, b.v, b.i, r.m, ls);
    }
}

// ---- gradient ---------------------------------------------------------------------------------------------------------------
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
            x[i] = j + V <= g.C ? load_vec(z + j) : load_part(z + j, g.C - j);
        }
        const GradRow r = grad_row(k, n, g.C + g.bg);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = (i * G + gl) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) x[i].v[e] = from_f32<T>(grad_score(r, g.c2, g.invT, to_f32(x[i].v[e]), j + e + g.bg));
            if (j + V <= g.C) __builtin_memcpy(out + j, &x[i], 16);
            else store_part(out + j, x[i], g.C - j);
        }
    }
}

// A block takes 256 lanes x 16 scores of a row at a time.
template <typename T>
__global__ __launch_bounds__(256) void scores_grad_block_kernel(const ScoresK k, long long tiles) {
    const LogitsK &g = k.g;
    constexpr int V = kVec<T>, NV = 16 / V, TILE = 256 * 16;
    for (long long item = blockIdx.x; item < g.rows * tiles; item += gridDim.x) {
        const long long n = item / tiles;
        const int c0 = (int)(item - n * tiles) * TILE;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        T *out = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi);
        Vec<T> x[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = c0 + (i * 256 + threadIdx.x) * V;
            x[i] = j + V <= g.C ? load_vec(z + j) : load_part(z + j, g.C - j);
        }
        const GradRow r = grad_row(k, n, g.C + g.bg);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = c0 + (i * 256 + threadIdx.x) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) x[i].v[e] = from_f32<T>(grad_score(r, g.c2, g.invT, to_f32(x[i].v[e]), j + e + g.bg));
            if (j + V <= g.C) __builtin_memcpy(out + j, &x[i], 16);
            else store_part(out + j, x[i], g.C - j);
        }
    }
}

// Classes that do not lie together: neighbouring lanes take neighbouring rows (planes), a block 256 rows and 32 classes.
template <typename T>
__global__ __launch_bounds__(256) void scores_grad_planes_kernel(const ScoresK k, int parts) {
    const LogitsK &g = k.g;
    const long long blocks = (g.rows + 255) / 256;
    for (long long item = blockIdx.x; item < blocks * parts; item += gridDim.x) {
        const long long rb = item / parts;
        const int c0 = (int)(item - rb * parts) * 32, c1 = c0 + 32 < g.C ? c0 + 32 : g.C;
        const long long n = rb * 256 + threadIdx.x;
        if (n >= g.rows) continue;
        const T *z = static_cast<const T *>(g.z) + row_base(g, n, g.so, g.si);
        T *out = static_cast<T *>(k.grad) + row_base(g, n, k.gso, k.gsi);
        const GradRow r = grad_row(k, n, g.C + g.bg);
        for (int c = c0; c < c1; c += 8) {
            T raw[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < c1) raw[i] = z[(long long)(c + i) * g.sc];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < c1) out[(long long)(c + i) * k.gsc] = from_f32<T>(grad_score(r, g.c2, g.invT, to_f32(raw[i]), c + i + g.bg));
        }
    }
}

// ---- dispatch ---------------------------------------------------------------------------------------------------------------
unsigned grid_of(long long blocks, int num_cu, int per_cu) {
    const long long cap = (long long)num_cu * per_cu;
    return (unsigned)(blocks < 1 ? 1 : blocks < cap ? blocks : cap);
}
bool contiguous(const LogitsK &g) { return g.sc == 1 || g.C == 1; }
// One lane a row wants 64 lanes on every compute unit; below that a wave a row is faster as soon as rows are long
bool lane_rows(const LogitsK &g, int num_cu) { return g.C <= 64 || g.rows >= 64ll * num_cu; }

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
    else hipLaunchKernelGGL((scores_group_kernel<T, G>), grid, block, 0, st, k);
}
template <typename T, int K>
void planes(const ScoresK &k, int num_cu, hipStream_t st) {
    const dim3 grid(grid_of((k.g.rows + 255) / 256, num_cu, 64)), block(256);
    if (sizeof(T) == 2 && k.g.C <= 65528) hipLaunchKernelGGL((scores_planes_kernel<T, K, sizeof(T) == 2>), grid, block, 0, st, k);
    else hipLaunchKernelGGL((scores_planes_kernel<T, K, false>), grid, block, 0, st, k);
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
    const Cut cut = cut_rows(g, num_cu);
    const dim3 grid(grid_of(g.rows * cut.segs, num_cu, 64));
    if (k.top) hipLaunchKernelGGL((scores_block_kernel<T, true>), grid, dim3(256), 0, st, k, cut);
    else hipLaunchKernelGGL((scores_block_kernel<T, false>), grid, dim3(256), 0, st, k, cut);
    if (cut.segs > 1) hipLaunchKernelGGL(scores_join_kernel<T>, dim3(grid_of(g.rows, num_cu, 64)), dim3(64), 0, st, k, cut);
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
        const int parts = (g.C + 31) / 32;
        hipLaunchKernelGGL(scores_grad_planes_kernel<T>, dim3(grid_of((g.rows + 255) / 256 * parts, num_cu, 64)), dim3(256), 0, st, k, parts);
        return;
    }
    if (g.C <= 32) return group<T, 2>(k, true, num_cu, st);
    if (g.C <= 64) return group<T, 4>(k, true, num_cu, st);
    if (g.C <= 128) return group<T, 8>(k, true, num_cu, st);
    if (g.C <= 256) return group<T, 16>(k, true, num_cu, st);
    if (g.C <= 512) return group<T, 32>(k, true, num_cu, st);
    if (g.C <= 1024) return group<T, 64>(k, true, num_cu, st);
    const long long tiles = (g.C + 4095) / 4096;
    hipLaunchKernelGGL(scores_grad_block_kernel<T>, dim3(grid_of(g.rows * tiles, num_cu, 256)), dim3(256), 0, st, k, tiles);
}

}  // namespace

size_t label_scores_workspace_bytes(const ScoresK &k, int, int num_cu) {
    if (k.g.C <= 1024 || !contiguous(k.g)) return 0;
    const Cut cut = cut_rows(k.g, num_cu);
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
