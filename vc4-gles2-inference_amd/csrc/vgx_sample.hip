// A token of each row of logits, by temperature, top-k, top-p and min-p.
//
// The tokens that stay are the first in a ranking by value and index, so every
// cut is a place in it, and so is the draw in the order of the indices: the token
// at which a count or a sum of weights reaches a number.
//
// Launch 1 (a workgroup a row and chunk) reads every logit once: the chunk's
// maximum, the maxima of its groups of 64 logits and, where the row needs it, the
// sum of its weights, under top-p alone by bins of an eighth of the temperature.
// Launch 2 (a workgroup a row) finds a value that all that may stay reach: from
// the bins, from min-p, or from the groups' maxima (as many tokens reach it as
// maxima do).  It reads the groups that reach it again and goes on with these
// tokens alone, a few hundred of tens of thousands: up to 128 compare themselves
// with each other, up to 4096 are counted into bins first.  Where top-p keeps
// more, the bins give all sums but the cut's own bin.  What is left is searched
// whole.
//
// Sums that are split at a place the data decides are taken in integers, which
// have no order: a weight is rounded to a multiple of 2^-q of the largest, q as
// large as the vocabulary's sum allows (2^-46 for 64402 tokens).  The tokens that
// stay under top-p < 1 weigh 2^-24 / vocab of the sum or more.  Without a cut the
// sums are launch 1's, in 64-bit floats.
#include <algorithm>
#include <string>

#include "vgx_logits.h"

#pragma clang fp contract(off)

namespace {

typedef unsigned long long u64;

struct Part {
    float m;   // the chunk's maximum (-inf: nothing)
    int arg;   // its first index (greedy rows)
    int n;     // tokens that are not masked (rows without a cut), or the bin of m
    int pad;
    double z;  // sum of exp((x - m) / T) (rows that need it)
};
struct SampleArgs {
    int nrows, vocab;
    const uint8_t* x;
    int64_t xs;  // bytes between rows
    const float* u;
    const float* temp;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    int* token;
    int* kept;
    float* prob;
    int q;       // weights are multiples of 2^-q
    Part* part;  // nrows x nch
    float* gmax; // nrows x ng: the groups' maxima
    u64* hist;   // nrows x nch x kHist: sums of weights by bins (top-p alone)
    int nch, k;  // chunks of a row; pieces of 16 bytes a thread and chunk
    int ng;
};

constexpr int kThreads = 256;  // of launch 1
constexpr int kRow = 512;      // of launch 2
constexpr int kWaves = kRow / 64;
constexpr int kBinBits = 10, kBins = 1 << kBinBits;
static_assert(kBins == 2 * kRow, "two bins a thread");
constexpr int kFew = 128;      // tokens that compare themselves with each other
constexpr int kList = 4096;    // tokens gathered from a row; under top-p alone
constexpr int kAbove = 1024;   // the first of these are for those above its bin
constexpr int kGroup = 64;     // logits of a group
constexpr int kHist = kThreads; // bins of a chunk; the last holds all below
constexpr int kMaxChunks = 520;
constexpr int kSides = kRow / kHist;  // of a launch 2's threads, chunks by turns
constexpr int kMaxVocab = 1 << 21;

// What a row asks for.
struct Ask {
    bool greedy, k, p, m;  // which cuts there are
    int top_k;
    double inv, top_p, min_p;
    // the sum of all weights is needed
    __device__ bool sum() const { return !greedy && !k && (p || !m); }
    __device__ bool none() const { return !k && !p && !m; }
    __device__ bool bins() const { return !greedy && p && !k && !m; }
    // A value's bin from above, as a whole float; bins are as wide as weights of
    // e^(1/8).
    __device__ float step() const { return (float)(8.0 * inv); }
};
__device__ __forceinline__ float bin_at(float x, float step) { return floorf(x * step); }
constexpr float kFar = 4194304.0f;  // bins past it are not whole numbers
// Where a chunk of maximum's bin n keeps its d-th bin from there: by the bin
// itself, so that a row's bins can be asked for before its maximum is known.
__device__ __forceinline__ int slot_of(int n, int d) { return (n - d) & (kHist - 1); }
__device__ __forceinline__ Ask ask_of(const SampleArgs& P, int r) {
    const float t = P.temp ? P.temp[r] : 1.0f;
    const float tp = P.top_p ? P.top_p[r] : 1.0f, mp = P.min_p ? P.min_p[r] : 0.0f;
    Ask a;
    a.top_k = P.top_k ? P.top_k[r] : 0;
    a.greedy = !(t > 0.0f) || a.top_k == 1 || tp <= 0.0f;
    a.k = a.top_k > 0 && a.top_k < P.vocab;
    a.p = tp < 1.0f;
    a.m = mp > 0.0f;
    a.inv = a.greedy ? 1.0 : fmin(1.0 / (double)t, 1e30);
    a.top_p = tp;
    a.min_p = a.m ? fmin((double)mp, 1.0) : 0.0;
    return a;
}

// A weight (0 .. 1) as a multiple of 2^-q, rounded to nearest: the low bits of a
// sum with 2^52.
__device__ __forceinline__ u64 fixed(double w, double scale) {
    return __builtin_bit_cast(u64, fma(w, scale, 4503599627370496.0)) - 0x4330000000000000ull;
}
// Sums and running sums over the lanes, as wave_sum and wave_scan.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_shift(u64 x) {
    const uint32x2 u = __builtin_bit_cast(uint32x2, x);
    const uint32x2 v = {(unsigned)__builtin_amdgcn_update_dpp(0, (int)u.x, CTRL, ROWS, 0xF, false),
                        (unsigned)__builtin_amdgcn_update_dpp(0, (int)u.y, CTRL, ROWS, 0xF, false)};
    return __builtin_bit_cast(u64, v);
}
__device__ __forceinline__ u64 wave_run(u64 x) {
    x += dpp_shift<0x111, 0xF>(x);
    x += dpp_shift<0x112, 0xF>(x);
    x += dpp_shift<0x114, 0xF>(x);
    x += dpp_shift<0x118, 0xF>(x);
    x += dpp_shift<0x142, 0xA>(x);
    return x + dpp_shift<0x143, 0xC>(x);
}
__device__ __forceinline__ u64 lane_of(u64 x, int l) {
    const uint32x2 u = __builtin_bit_cast(uint32x2, x);
    const uint32x2 v = {(unsigned)__builtin_amdgcn_readlane((int)u.x, l), (unsigned)__builtin_amdgcn_readlane((int)u.y, l)};
    return __builtin_bit_cast(u64, v);
}
__device__ __forceinline__ u64 wave_add(u64 x) { return lane_of(wave_run(x), 63); }

// The largest of 16 lanes (rows of 32-bit logits: 16 pieces are a group) or 8.
template <int LANES>
__device__ __forceinline__ float lanes_max(float x) {
    x = fmaxf(x, dpp<0xB1>(x));
    x = fmaxf(x, dpp<0x4E>(x));
    x = fmaxf(x, dpp<0x141>(x));
    if (LANES == 16) x = fmaxf(x, dpp<0x140>(x));
    return x;
}

// Bound by memory where no row needs a sum (640 rows of 64402 q16 logits, top-k: 82
// MB in 18.6 us, 4.4 TB/s), else by its 45 vector instructions a logit and, under
// top-p, a 64-bit LDS addition a logit: 160 rows of 64402 bf16 19 us, 48 of 73448 f32
// with all cuts among them 10.
template <int KIND, int K>
__global__ void __launch_bounds__(kThreads) sample_stats_kernel(const SampleArgs P) {
    constexpr int N = kPer<KIND>, LG = kGroup / N;  // lanes a group
    __shared__ double tab[64];
    __shared__ float sm[4];
    __shared__ int sa[4], sn[4];
    __shared__ double sz[4];
    __shared__ u64 hist[kHist];
    const int chunk = blockIdx.x, r = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const Row q = row_at<KIND>(P.x, P.xs, r);
    auto first = [&](int k) { return ((chunk * K + k) * kThreads + t) * N - q.off; };
    auto full = [&](int i0) { return i0 >= 0 && i0 + N <= P.vocab; };
    uint4 raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        raw[k] = make_uint4(0, 0, 0, 0);
        if (full(first(k))) raw[k] = *reinterpret_cast<const uint4*>(q.p + (int64_t)first(k) * kBytes<KIND>);
    }
    const Ask A = ask_of(P, r);
    const bool sum = A.sum(), bins = A.bins();
    if (sum) fill_table(tab);
    if (bins) hist[t] = 0;
    // q16 logits are integers, and the maximum less one of them is one of 0 ..
    // 65535 (65536: nothing): its weight is a product of two table entries, of the
    // low byte and of what is above it (two LDS reads instead of 12 operations of
    // 64 bits: 640 rows of 64402 without a cut 61 -> 52 us, by top-p 64 -> 60).
    __shared__ double low[KIND == VGX_E_Q16 ? 256 : 1], high[KIND == VGX_E_Q16 ? 257 : 1];
    if (KIND == VGX_E_Q16 && sum) {
        const Scale S = scale_of(0.0f, A.inv);
        __syncthreads();
        low[t] = exp_of((float)-t * (1.0f / 256), S, tab);
        high[t] = exp_of((float)-t, S, tab);
        if (t == 0) high[256] = 0.0;
    }
    float x[K][N], gm[K];
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        unpack<KIND>(raw[k], x[k]);
        const int i0 = first(k);
        if (!full(i0)) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                x[k][e] = i0 + e >= 0 && i0 + e < P.vocab ? one<KIND>(q.p, i0 + e) : -INFINITY;
        }
        gm[k] = x[k][0];
#pragma unroll
        for (int e = 1; e < N; ++e) gm[k] = fmaxf(gm[k], x[k][e]);
        m = fmaxf(m, gm[k]);
    }
    int a = 0x7fffffff;
    if (A.greedy) {  // the first index of the maximum
#pragma unroll
        for (int k = K - 1; k >= 0; --k)
#pragma unroll
            for (int e = N - 1; e >= 0; --e)
                if (x[k][e] == m) a = first(k) + e;
        wave_best(m, a);
    } else {
        m = wave_max(m);
        if (!A.none()) {
            float y = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const float g = lanes_max<LG>(gm[k]);
                if ((lane & (LG - 1)) == k) y = g;
            }
            // lane k of a group stores its k-th piece's
            const int k = lane & (LG - 1);
            if (k < K) P.gmax[(int64_t)r * P.ng + (chunk * K + k) * (kThreads / LG) + t / LG] = y;
        }
    }
    if (lane == 0) { sm[wave] = m; sa[wave] = a; }
    __syncthreads();
    m = sm[0];
    a = sa[0];
#pragma unroll
    for (int w = 1; w < 4; ++w)
        if (sm[w] > m || (sm[w] == m && sa[w] < a)) { m = sm[w]; a = sa[w]; }
    double z[2] = {0.0, 0.0};
    int n = 0;
    const Scale S = scale_of(m, A.inv);
    const float m256 = m * 256.0f;
    // (a masked one's is e^-690, or 0)
    auto weigh = [&](float x) {
        if constexpr (KIND == VGX_E_Q16) {
            const int d = (int)fminf(fmaf(x, -256.0f, m256), 65536.0f);
            return low[d & 255] * high[d >> 8];
        } else {
            return add_pow(fmax(((double)x - S.m) * S.a, -63700.0), 0.0, tab);
        }
    };
    if (bins) {
        // weights as multiples of 2^-50 of the chunk's largest: sums that do not
        // depend on their order
        const float step = A.step(), top = bin_at(m, step);
        if (m != -INFINITY) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const u64 f = fixed(weigh(x[k][e]), 0x1p50);
                    const int b = (int)fminf(top - bin_at(x[k][e], step), (float)(kHist - 1));
                    if (f) atomicAdd(&hist[b], f);
                }
        }
        __syncthreads();
        const u64 f = hist[t];
        n = m == -INFINITY ? -0x7fffffff : fabsf(m * step) < kFar ? (int)top : 0x7fffffff;
        P.hist[((int64_t)r * P.nch + chunk) * kHist + slot_of(n, t)] = f;
        const u64 w = wave_add(f);
        if (lane == 0) sz[wave] = (double)w;
        __syncthreads();
        z[0] = (sz[0] + sz[1] + sz[2] + sz[3]) * 0x1p-50;
    } else if (sum) {
        if (m != -INFINITY) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    z[e & 1] += weigh(x[k][e]);
                    n += x[k][e] != -INFINITY;
                }
        }
        const double w = wave_sum(z[0] + z[1]);
        n = (int)wave_add((u64)n);
        if (lane == 0) { sz[wave] = w; sn[wave] = n; }
        __syncthreads();
        z[0] = sz[0] + sz[1] + sz[2] + sz[3];
        n = sn[0] + sn[1] + sn[2] + sn[3];
    }
    if (t == 0) P.part[(int64_t)r * P.nch + chunk] = Part{m, a, n, 0, z[0]};
}

// The order of floats as unsigned integers (-0 as 0; never 0).
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// A place in the ranking: the tokens up to it stay.
struct Cut {
    unsigned key;
    int idx;
};
__device__ __forceinline__ bool stays(const Cut& c, unsigned key, int i) {
    return key > c.key || (key == c.key && i <= c.idx);
}
constexpr int kGroups = 2048;  // groups that are read again, at most
constexpr int kHoldBins = 10;  // chunks whose bins a thread holds

struct RowShared {
    double tab[64];
    u64 wave[kWaves];
    float m[kWaves], low[kWaves];
    int a[kWaves];
    union {
        struct {
            unsigned cnt[kBins];
            u64 sum[kBins];
        } h;
        struct {
            u64 order[kRow], w[kRow], before[kRow];
            unsigned rank[kRow];
            u64 sum[kWaves];
            int count[kWaves];
        } few;
        int groups[kGroups];
        struct {
            double sum[kMaxChunks];
            u64 more[kMaxChunks];
        } chunk;
        struct {
            double f[kRow], part[kSides][kHist], wave[4];
            int down[kRow];
        } merge;
    };
    unsigned key[kList];
    int idx[kList];
    int bin, n, above_n, stay, found, last;
    unsigned lo, hi;
    u64 above, total;
    double left, sum;
    int down[kSides * kHoldBins];  // the first chunks' bins below the row's
    double weight[kSides * kHoldBins];  // of their maxima
    u64 first[kSides * kHoldBins]; // the sums of their bins above top-p's
    Part one;
    float x;
    Cut at;
};

// The running sum over the workgroup's threads; total: of all.
__device__ __forceinline__ u64 block_scan(u64 x, u64* sm, u64& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    x = wave_run(x);
    __syncthreads();  // the last scan's sums are read
    if (lane == 63) sm[wave] = x;
    __syncthreads();
    u64 before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += sm[w];
        total += sm[w];
    }
    return x + before;
}
// Places for the lanes' c things each in a list whose length is *n: the first of
// a lane's.
__device__ __forceinline__ int place_of(int c, int* n) {
    int run = c;
    run += __builtin_amdgcn_update_dpp(0, run, 0x111, 0xF, 0xF, false);
    run += __builtin_amdgcn_update_dpp(0, run, 0x112, 0xF, 0xF, false);
    run += __builtin_amdgcn_update_dpp(0, run, 0x114, 0xF, 0xF, false);
    run += __builtin_amdgcn_update_dpp(0, run, 0x118, 0xF, 0xF, false);
    run += __builtin_amdgcn_update_dpp(0, run, 0x142, 0xA, 0xF, false);
    run += __builtin_amdgcn_update_dpp(0, run, 0x143, 0xC, 0xF, false);
    const int all = __builtin_amdgcn_readlane(run, 63);
    if (all == 0) return 0;
    int at = 0;
    if ((threadIdx.x & 63) == 0) at = atomicAdd(n, all);
    return __builtin_amdgcn_readfirstlane(at) + run - c;
}
// Of n <= kFew tokens (few.order, few.w) each one's rank and the weights before
// it: all threads take part, several a token.
__device__ __forceinline__ void compare_all(RowShared& H, int n) {
    const int t = threadIdx.x;
    const int cols = n <= 64 ? 64 : kFew, parts = kRow / cols;
    H.few.before[t] = 0;
    H.few.rank[t] = 0;
    __syncthreads();
    const int i = t & (cols - 1), per = (n + parts - 1) / parts, j0 = t / cols * per, j1 = min(n, j0 + per);
    const u64 mine = H.few.order[i];
    u64 s = 0;
    unsigned c = 0;
#pragma unroll 4
    for (int j = j0; j < j1; ++j) {
        const u64 o = H.few.order[j], w = H.few.w[j];
        const bool less = o < mine;
        s += less ? w : 0;
        c += less;
    }
    if (c) {
        atomicAdd(&H.few.before[i], s);
        atomicAdd(&H.few.rank[i], c);
    }
    __syncthreads();
}

// A row's piece g as it lies in memory; values outside the row are 0.
template <int KIND>
__device__ __forceinline__ uint4 raw_piece(const Row& q, int vocab, int g) {
    constexpr int N = kPer<KIND>;
    const int i0 = g * N - q.off;
    if (i0 >= 0 && i0 + N <= vocab) return *reinterpret_cast<const uint4*>(q.p + (int64_t)i0 * kBytes<KIND>);
    unsigned u[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (i0 + e >= 0 && i0 + e < vocab) {
            if (KIND == VGX_E_F32) u[e] = reinterpret_cast<const unsigned*>(q.p)[i0 + e];
            else u[e / 2] |= (unsigned)reinterpret_cast<const unsigned short*>(q.p)[i0 + e] << 16 * (e & 1);
        }
    return make_uint4(u[0], u[1], u[2], u[3]);
}
// The e-th value of a piece.
template <int KIND>
__device__ __forceinline__ float value_in(const uint4& v, int e) {
    const int w = KIND == VGX_E_F32 ? e : e / 2;
    const unsigned a = w & 1 ? v.y : v.x, b = w & 1 ? v.w : v.z;
    unsigned u = w & 2 ? b : a;
    if (KIND == VGX_E_F32) return clean(__uint_as_float(u));
    u = u >> 16 * (e & 1) & 0xffff;
    if (KIND == VGX_E_Q16) return (float)(short)u * (1.0f / 256);
    if (KIND == VGX_E_BF16) return clean(__uint_as_float(u << 16));
    return clean((float)__builtin_bit_cast(_Float16, (unsigned short)u));
}
// Which of a piece's n values, the first of index i, are inside the row.
__device__ __forceinline__ unsigned ends_of(int i, int n, int vocab) {
    unsigned r = 0;
    for (int e = 0; e < n; ++e) r |= (unsigned)(i + e >= 0 && i + e < vocab) << e;
    return r;
}
// f(value, index) of a piece's values inside the row, one after the other: a loop
// that shifts them down, as many copies of a long f would not stay in the
// instruction cache.
template <int KIND, class F>
__device__ __forceinline__ void each_of(uint4 v, int i0, int vocab, F f) {
    constexpr int N = kPer<KIND>;
#pragma unroll 1
    for (int e = 0; e < N; ++e) {
        float x;
        if (KIND == VGX_E_F32) x = clean(__uint_as_float(v.x));
        else if (KIND == VGX_E_Q16) x = (float)(short)(v.x & 0xffff) * (1.0f / 256);
        else if (KIND == VGX_E_BF16) x = clean(__uint_as_float(v.x << 16));
        else x = clean((float)__builtin_bit_cast(_Float16, (unsigned short)(v.x & 0xffff)));
        if (i0 + e >= 0 && i0 + e < vocab) f(x, i0 + e);
        if (KIND == VGX_E_F32) {
            v.x = v.y; v.y = v.z; v.z = v.w;
        } else {
            v.x = v.y << 16 | v.x >> 16;
            v.y = v.z << 16 | v.y >> 16;
            v.z = v.w << 16 | v.z >> 16;
            v.w >>= 16;
        }
    }
}
// The tokens of a row (f(key, index) of each that is not masked) ...
template <int KIND>
struct WholeRow {
    static constexpr bool kWhole = true;
    const SampleArgs& P;
    Row q;
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        constexpr int N = kPer<KIND>;
        const int pieces = (P.vocab + q.off + N - 1) / N;
        constexpr int U = 4;  // pieces a thread in one round trip
#pragma unroll 1
        for (int g0 = threadIdx.x; g0 < pieces; g0 += kRow * U) {
            uint4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                v[u] = make_uint4(0, 0, 0, 0);
                if (g0 + u * kRow < pieces) v[u] = raw_piece<KIND>(q, P.vocab, g0 + u * kRow);
            }
#pragma unroll 1
            for (int u = 0; u < U; ++u) {
                each_of<KIND>(v[0], (g0 + u * kRow) * N - q.off, P.vocab, [&](float x, int i) {
                    if (x != -INFINITY) f(key_of(x), i);
                });
#pragma unroll
                for (int w = 0; w + 1 < U; ++w) v[w] = v[w + 1];
            }
        }
    }
};
// ... or those gathered from it: the list's places i0 .. i0 + n - 1, and the
// first n0 ones.
struct Gathered {
    static constexpr bool kWhole = false;
    const RowShared& H;
    int n0, i0, n;
    __device__ __forceinline__ int place(int i) const { return i < n0 ? i : i - n0 + i0; }
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        for (int i = threadIdx.x; i < n0 + n; i += kRow) {
            const int at = place(i);
            f(H.key[at], H.idx[at]);
        }
    }
};

// The tokens that stay inside a cut, with their weights.
struct Weigh {
    Scale S;
    double scale, least;
    const double* tab;
    __device__ __forceinline__ double real(unsigned key) const { return weight(value_of(key), S, tab); }
    __device__ __forceinline__ u64 operator()(unsigned key) const {
        const double w = real(key);
        return w < least ? 0 : fixed(w, scale);
    }
};

// The token at which the tokens inside `in`, in the ranking's order or (BY_INDEX)
// that of their indices, reach `want` (of their total, once that is known): of
// tokens, or of weights (WEIGHTED).  False: they do not.  Bins over the values
// first (floats' keys spread over them badly), then over the keys of the bin that
// holds the place, then over the indices of one key, until few are left.  Of a
// whole row a bin's tokens are gathered as soon as there is room for them (640 rows
// of 64402 by top-k 5000 262 -> 186 us).
template <bool WEIGHTED, bool BY_INDEX, class Source, class Want>
__device__ __forceinline__ bool locate(RowShared& H, const Source& src, const Weigh& W, const Cut& in, float m, float range, int vocab,
                       Want want_of) {
    const int t = threadIdx.x;
    const float step = (float)(kBins - 1) / range;
    enum { VALUE, KEY, INDEX };
    int mode = BY_INDEX ? INDEX : VALUE;
    unsigned lo = BY_INDEX ? ~(unsigned)(vocab - 1) : 0, hi = ~0u, eq = 0;  // (INDEX: of the indices' complements)
    u64 before = 0, want = 0;
#pragma unroll 1
    for (bool first = true;; first = false) {
        const int sh = mode == VALUE ? 0 : max(0, 32 - __clz((int)(hi - lo)) - kBinBits);
        auto bin_of = [&](unsigned key, int i) -> int {
            if (!stays(in, key, i)) return -1;
            if (mode == VALUE) return kBins - 1 - (int)fminf(fmaxf((m - value_of(key)) * step, 0.0f), (float)(kBins - 1));
            if (mode == INDEX && !BY_INDEX && key != eq) return -1;
            const unsigned o = mode == KEY ? key : ~(unsigned)i;
            return o < lo || o > hi ? -1 : (int)((o - lo) >> sh);
        };
        __syncthreads();
        for (int i = t; i < kBins; i += kRow) { H.h.cnt[i] = 0; H.h.sum[i] = 0; }
        if (t == 0) { H.bin = -1; H.n = 0; H.lo = ~0u; H.hi = 0; }
        __syncthreads();
        src.each([&](unsigned key, int i) {
            const int b = bin_of(key, i);
            if (b < 0) return;
            if (WEIGHTED) {
                const u64 w = W(key);
                if (w) atomicAdd(&H.h.sum[b], w);
            }
            atomicAdd(&H.h.cnt[b], 1u);
        });
        __syncthreads();
        const int b0 = kBins - 1 - 2 * t;
        const unsigned c0 = H.h.cnt[b0], c1 = H.h.cnt[b0 - 1];
        const u64 v0 = WEIGHTED ? H.h.sum[b0] : c0, v1 = WEIGHTED ? H.h.sum[b0 - 1] : c1;
        u64 total;
        const u64 run = block_scan(v0 + v1, H.wave, total), at = before + run - v0 - v1;
        if (first) want = want_of(total);
        if (at < want && want <= before + run) {
            const bool low = want > at + v0;
            H.bin = low ? b0 - 1 : b0;
            H.above = low ? at + v0 : at;
            H.total = low ? c1 : c0;
        }
        __syncthreads();
        const int bin = H.bin;
        if (bin < 0) return false;
        before = H.above;
        const int c = (int)H.total;
        if (c <= kFew) {
            __syncthreads();  // (the bins' memory is used again)
            src.each([&](unsigned key, int i) {
                if (bin_of(key, i) != bin) return;
                const int at = atomicAdd(&H.n, 1);
                if (at >= kFew) return;  // (never)
                H.few.order[at] = BY_INDEX ? (u64)(unsigned)i << 32 | key : (u64)~key << 32 | (unsigned)i;
                H.few.w[at] = WEIGHTED ? W(key) : 1;
            });
            __syncthreads();
            compare_all(H, c);
            const u64 mine = t < c ? H.few.order[t] : 0, w = t < c ? H.few.w[t] : 0, s = before + H.few.before[t];
            if (t < c && s < want && want <= s + w)
                H.at = BY_INDEX ? Cut{(unsigned)mine, (int)(mine >> 32)} : Cut{~(unsigned)(mine >> 32), (int)(unsigned)mine};
            __syncthreads();
            return true;
        }
        if constexpr (Source::kWhole) {
            if (mode == VALUE && c <= kList) {  // the bin's tokens alone from here on
                src.each([&](unsigned key, int i) {
                    if (bin_of(key, i) != bin) return;
                    const int at = atomicAdd(&H.n, 1);
                    if (at >= kList) return;  // (never)
                    H.key[at] = key;
                    H.idx[at] = i;
                });
                __syncthreads();
                const u64 left = want - before;
                return locate<WEIGHTED, BY_INDEX>(H, Gathered{H, 0, 0, c}, W, in, m - (float)(kBins - 1 - bin) / step, 1.0f / step,
                                                  vocab, [&](u64) { return left; });
            }
        }
        if (mode == VALUE) {  // the keys of the bin
            unsigned a = ~0u, b = 0;
            src.each([&](unsigned key, int i) {
                if (bin_of(key, i) != bin) return;
                a = min(a, key);
                b = max(b, key);
            });
            if (a <= b) { atomicMin(&H.lo, a); atomicMax(&H.hi, b); }
            __syncthreads();
            lo = H.lo;
            hi = H.hi;
            mode = KEY;
        } else {
            lo += (unsigned)bin << sh;
            hi = min(hi, lo + ((1u << sh) - 1));
        }
        if (mode == KEY && lo == hi) {  // equal values: by their indices
            eq = lo;
            mode = INDEX;
            lo = ~(unsigned)(vocab - 1);
            hi = ~0u;
        }
    }
}

// Weights below 2^-q, which are 0, are this far below the maximum.
__device__ __forceinline__ float range_of(const SampleArgs& P, const Ask& A) {
    return (float)fmin((double)(P.q + 1) * 0.7 / A.inv, 1e30);
}
// Top-k's and top-p's place in a source that holds all that may stay (but for
// min_p, W.least: 0).  z: the sum of all weights, negative where the source holds
// them all.
template <class Source>
__device__ __forceinline__ Cut find_cut(const SampleArgs& P, RowShared& H, const Source& src, const Ask& A, const Weigh& W,
                                        float m, double z) {
    Cut cut{0, 0x7fffffff};
    const float range = range_of(P, A);
    if (A.k && locate<false, false>(H, src, W, cut, m, range, P.vocab, [&](u64) { return (u64)A.top_k; })) cut = H.at;
    if (A.p) {
        const bool some = locate<true, false>(H, src, W, cut, m, range, P.vocab, [&](u64 total) {
            const double y = ceil(A.top_p * (A.k || z < 0.0 ? (double)total : z * W.scale));
            return y < 1.0 ? 1ull : (u64)y;
        });
        if (some) cut = H.at;
    }
    __syncthreads();
    return cut;
}

// The cuts and the draw over such a source.
template <class Source>
__device__ __forceinline__ void cut_and_draw(const SampleArgs& P, RowShared& H, const Source& src, int r, const Ask& A, Weigh W, float m,
                             double z) {
    const int t = threadIdx.x;
    const double least = W.least, u = P.u[r];
    W.least = 0.0;
    const Cut cut = find_cut(P, H, src, A, W, m, z);
    W.least = least;
    // how many stay
    unsigned n = 0;
    if (t == 0) H.stay = 0;
    __syncthreads();
    src.each([&](unsigned key, int i) { n += stays(cut, key, i) && (least == 0.0 || W.real(key) >= least); });
    n = (unsigned)wave_add(n);
    if ((t & 63) == 0 && n) atomicAdd(&H.stay, (int)n);
    u64 sum = 0;
    // (a draw of 1 or more, or no number, takes the last token)
    locate<true, true>(H, src, W, cut, m, range_of(P, A), P.vocab, [&](u64 total) {
        sum = total;
        return u >= 0.0 && u < 1.0 ? min((u64)(u * (double)total), total - 1) + 1 : u < 0.0 ? 1ull : total;
    });
    if (t == 0) {
        P.token[r] = H.at.idx;
        if (P.kept) P.kept[r] = H.stay;
        if (P.prob) P.prob[r] = (float)(W.real(H.at.key) / ((double)sum / W.scale));
    }
}

// The same for up to kFew gathered tokens, each with its thread: its rank and the
// weights before it by comparing with all others, then the weights of those that
// stay with a lower index.
__device__ __forceinline__ void cut_and_draw_few(const SampleArgs& P, RowShared& H, const Gathered& src, int r,
                                                 const Ask& A, const Weigh& W, double z) {
    const int t = threadIdx.x, n = src.n0 + src.n;
    const double u = P.u[r];  // (here it comes in beside the first comparisons)
    const bool in = t < n;
    const unsigned key = in ? H.key[src.place(t)] : 0;
    const int idx = in ? H.idx[src.place(t)] : 0;
    const u64 mine = (u64)~key << 32 | (unsigned)idx;
    const double real = in ? W.real(key) : 0.0;
    u64 w = in ? fixed(real, W.scale) : 0;
    H.few.order[t] = in ? mine : ~0ull;
    H.few.w[t] = w;
    compare_all(H, n);
    const u64 before = H.few.before[t];
    bool stay = in && (!A.k || (int)H.few.rank[t] < A.top_k);
    const int lane = t & 63, wave = t >> 6;  // (all tokens are the first two waves')
    if (A.p) {
        double all = z * W.scale;
        if (A.k) {
            const u64 s = wave_add(stay ? w : 0);
            if (lane == 0) H.wave[wave] = s;
            __syncthreads();
            all = (double)(H.wave[0] + H.wave[1]);
        }
        const double y = ceil(A.top_p * all);
        stay = stay && before < (y < 1.0 ? 1ull : (u64)y);
    }
    stay = stay && real >= W.least;
    if (!stay) w = 0;
    const u64 s = wave_add(w);
    const int some = __popcll(__ballot(stay));
    if (lane == 0) {
        H.few.sum[wave] = s;
        H.few.count[wave] = some;
    }
    H.few.order[t] = stay ? (u64)(unsigned)idx : ~0ull;
    H.few.w[t] = w;
    compare_all(H, n);
    const u64 c = H.few.before[t], sum = H.few.sum[0] + H.few.sum[1];
    const u64 want = u >= 0.0 && u < 1.0 ? min((u64)(u * (double)sum), sum - 1) : u < 0.0 ? 0 : sum - 1;
    if (stay && c <= want && want < c + w) {
        P.token[r] = idx;
        if (P.kept) P.kept[r] = H.few.count[0] + H.few.count[1];
        if (P.prob) P.prob[r] = (float)(real / ((double)sum / W.scale));
    }
}

// The draw from the chunks' sums (H.chunk.sum, in 64-bit floats): the chunk, then
// the token in it from its weights.  stay(x, index): which of them count.
template <int KIND, class Stay>
__device__ __forceinline__ void draw_in_chunks(const SampleArgs& P, RowShared& H, int r, const Row& q, const Scale& S,
                                               int kept, Stay stay) {
    constexpr int N = kPer<KIND>;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    __shared__ double sw[kWaves];
    if (wave == 0) {
        auto sum_of = [&](int c) { return c < P.nch ? H.chunk.sum[c] : 0.0; };
        double total = 0.0;
        for (int c = lane; c < P.nch; c += 64) total += sum_of(c);
        total = wave_sum(total);
        const double un = P.u[r];
        // (a draw of 1 or more, or no number, takes the last token)
        const double want = un >= 0.0 ? un * total : un < 0.0 ? 0.0 : total;
        double before = 0.0, at = 0.0, some_at = 0.0;
        int pick = -1, some = -1;
        for (int c = 0; c < P.nch && pick < 0; c += 64) {
            const double v = sum_of(c + lane), run = wave_scan(v);
            const u64 past = __ballot(before + run > want && v > 0.0), any = __ballot(v > 0.0);
            if (past) {
                const int l = __ffsll(past) - 1;
                pick = c + l;
                at = before + lane_of(run, l) - lane_of(v, l);
            } else if (any) {
                const int l = 63 - __clzll((long long)any);
                some = c + l;
                some_at = before + lane_of(run, l) - lane_of(v, l);
            }
            before += lane_of(run, 63);
        }
        if (lane == 0) {
            H.bin = pick >= 0 ? pick : some;
            H.left = fmax(want - (pick >= 0 ? at : some_at), 0.0);
            H.sum = total;
            H.found = 0x7fffffff;
            H.last = -1;
        }
    }
    __syncthreads();
    const double left = H.left;
    // the chunk's pieces, consecutive ones of a thread
    const int pieces = P.k * kThreads, per = (pieces + kRow - 1) / kRow, g0 = H.bin * pieces;
    double s = 0.0;
    int mine = -1;
    float lastx = 0.0f;
    auto each = [&](auto f) {
        for (int k = 0; k < per; ++k) {
            const int j = t * per + k;
            if (j >= pieces) break;
            each_of<KIND>(raw_piece<KIND>(q, P.vocab, g0 + j), (g0 + j) * N - q.off, P.vocab, [&](float x, int i) {
                if (x != -INFINITY && stay(x, i)) f(x, i, weight(x, S, H.tab));
            });
        }
    };
    each([&](float x, int i, double w) {
        s += w;
        if (w > 0.0) { mine = i; lastx = x; }
    });
    const double run = wave_scan(s);
    if (lane == 63) sw[wave] = run;
    if (mine >= 0) atomicMax(&H.last, mine);
    __syncthreads();
    // (as the draft check takes it: only a thread with a weight, and of several
    // waves the first)
    double before = __shfl_up(run, 1, 64);
    if (lane == 0) before = 0.0;
    double base = 0.0;
    for (int v = 0; v < wave; ++v) base += sw[v];
    before += base;
    const u64 past = __ballot(mine >= 0 && base + run > left);
    int hit = -1;
    float hx = 0.0f;
    if (past) {
        // the first such thread's values, one a lane
        const int l = __ffsll(past) - 1;
        const double b = lane_of(before, l);
        const int fall = __builtin_amdgcn_readlane(mine, l);
        const float fallx = lane_of(lastx, l);
        const int i = (g0 + (wave * 64 + l) * per) * N - q.off + lane;
        const bool in = lane < per * N && i >= 0 && i < P.vocab;
        const float x = in ? one<KIND>(q.p, i) : -INFINITY;
        const double w = in && x != -INFINITY && stay(x, i) ? weight(x, S, H.tab) : 0.0;
        const double c = b + wave_scan(w);
        const u64 at = __ballot(w > 0.0 && c > left);
        const int k = __ffsll(at) - 1;
        hit = at ? __builtin_amdgcn_readlane(i, max(k, 0)) : fall;
        hx = at ? lane_of(x, max(k, 0)) : fallx;
        if (lane == 0) atomicMin(&H.found, hit);
    }
    __syncthreads();
    const bool none = H.found == 0x7fffffff;
    const int token = none ? H.last : H.found;
    if (!none && hit == token && lane == 0) H.x = hx;
    if (none && mine == token) H.x = lastx;
    __syncthreads();
    if (t == 0) {
        P.token[r] = token;
        if (P.kept) P.kept[r] = kept;
        if (P.prob) P.prob[r] = (float)(weight(H.x, S, H.tab) / H.sum);
    }
}
static_assert(4 * kThreads / kRow * 8 <= 64 && 8192 / kRow <= 64, "a thread's values of a chunk: a lane each");

// The cuts and the draw where what may stay was not gathered: the cut from passes
// over the whole row, then the chunks' sums of what stays.
template <int KIND>
__device__ __forceinline__ void cut_and_draw_whole(const SampleArgs& P, RowShared& H, int r, const Row& q, const Ask& A,
                                                   Weigh W, float m) {
    constexpr int N = kPer<KIND>;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const double least = W.least;
    W.least = 0.0;
    const Cut cut = find_cut(P, H, WholeRow<KIND>{P, q}, A, W, m, -1.0);
    auto stay = [&](float x, int i) { return stays(cut, key_of(x), i) && (least == 0.0 || weight(x, W.S, W.tab) >= least); };
    // (a row of one chunk: a part of it a wave)
    const int parts = P.nch == 1 ? kWaves : 1, units = P.nch * parts, per = P.k * kThreads / parts;
    if (t == 0) H.stay = 0;
    __syncthreads();
    int n = 0;
#pragma unroll 1
    for (int c = wave; c < units; c += kWaves) {
        double s = 0.0;
#pragma unroll 1
        for (int j0 = lane; j0 < per; j0 += 4 * 64) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                v[u] = make_uint4(0, 0, 0, 0);
                if (j0 + u * 64 < per) v[u] = raw_piece<KIND>(q, P.vocab, c * per + j0 + u * 64);
            }
#pragma unroll 1
            for (int u = 0; u < 4 && j0 + u * 64 < per; ++u) {
                const int i0 = (c * per + j0 + u * 64) * N - q.off;
                const unsigned inside = i0 >= 0 && i0 + N <= P.vocab ? (1u << N) - 1 : ends_of(i0, N, P.vocab);
                float x[N];
                unpack<KIND>(v[0], x);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const bool in = inside >> e & 1 && x[e] != -INFINITY && stays(cut, key_of(x[e]), i0 + e);
                    const double w = in ? weight(x[e], W.S, W.tab) : 0.0;
                    const bool some = in && w >= least;
                    s += some ? w : 0.0;
                    n += some;
                }
#pragma unroll
                for (int w = 0; w + 1 < 4; ++w) v[w] = v[w + 1];
            }
        }
        s = wave_sum(s);
        if (lane == 0) H.chunk.sum[c] = s;
    }
    n = (int)wave_add((u64)n);
    if (lane == 0) atomicAdd(&H.stay, n);
    __syncthreads();
    if (parts > 1 && t == 0)
        for (int w = 1; w < kWaves; ++w) H.chunk.sum[0] += H.chunk.sum[w];
    __syncthreads();
    draw_in_chunks<KIND>(P, H, r, q, W.S, H.stay, stay);
}

// The maximum of a row's chunks, and (greedy) its first index.
__device__ __forceinline__ float join_max(const SampleArgs& P, RowShared& H, const Part* part, bool first, int& a) {
    const int t = threadIdx.x;
    float m = -INFINITY;
    a = 0x7fffffff;
    for (int c = t; c < P.nch; c += kRow)
        if (part[c].m > m || (part[c].m == m && part[c].arg < a)) { m = part[c].m; a = part[c].arg; }
    if (first) wave_best(m, a);
    else m = wave_max(m);
    if ((t & 63) == 0) { H.m[t >> 6] = m; H.a[t >> 6] = a; }
    __syncthreads();
    m = H.m[0];
    a = H.a[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
        if (H.m[w] > m || (H.m[w] == m && H.a[w] < a)) { m = H.m[w]; a = H.a[w]; }
    return m;
}

// The least float of a bin; false where its search is long (products that
// underflow).
__device__ __forceinline__ bool first_in(float bin, float step, float& x) {
    auto next = [](float y, int d) {
        const unsigned k = key_of(y) + d;
        return value_of(k == 0x7fffffffu && d < 0 ? k - 1 : k);  // (-0 is 0)
    };
    x = bin / step;
    if (!(fabsf(x) < FLT_MAX)) return false;
    int n = 0;
    while (n < 64 && bin_at(x, step) < bin) { x = next(x, 1); ++n; }
    while (n < 64 && bin_at(next(x, -1), step) >= bin) { x = next(x, -1); ++n; }
    return n < 64;
}

// Top-p's bin from the chunks' bins: H.bin (-1: none of them, or they are not
// whole), the weights above it H.left, all weights H.sum.  held: the thread's slot
// of its first chunks (every kSides-th one).
__device__ __forceinline__ void find_bin(const SampleArgs& P, RowShared& H, const Part* part, const Part& own,
                                         const u64 (&held)[kHoldBins], int r, const Ask& A, const Scale& S, float top) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, slot = t & (kHist - 1), half = t / kHist;
    const u64* hist = P.hist + (int64_t)r * P.nch * kHist + slot;
    bool far = !(fabsf(top) < kFar);
    const int mine = ((far ? 0 : (int)top) - slot) & (kHist - 1);  // the row's bin that the slot is
    double v = 0.0, z = 0.0;
    for (int c0 = 0; c0 < P.nch; c0 += kRow) {
        __syncthreads();
        if (c0 + t < P.nch) {
            const Part x = c0 ? part[c0 + t] : own;
            const bool some = x.m != -INFINITY;
            const double f = some ? weight(x.m, S, H.tab) : 0.0;
            if (some && x.n == 0x7fffffff) far = true;
            H.merge.f[t] = f;
            H.merge.down[t] = some && !far ? (int)fminf(top - (float)x.n, (float)kHist) : kHist;
            if (c0 == 0 && t < kSides * kHoldBins) {
                H.down[t] = H.merge.down[t];
                H.weight[t] = f;
            }
            z += x.z * f;
        }
        __syncthreads();
        const int n = min(P.nch - c0, kRow);
        auto add = [&](int c, u64 w) {
            const int at = mine - H.merge.down[c];
            v += at >= 0 && at < kHist - 1 ? (double)w * H.merge.f[c] : 0.0;
        };
        if (c0 == 0) {
#pragma unroll
            for (int k = 0; k < kHoldBins; ++k)
                if (half + kSides * k < n) add(half + kSides * k, held[k]);
        }
#pragma unroll 4
        for (int c = half + (c0 ? 0 : kSides * kHoldBins); c < n; c += kSides) add(c, hist[(int64_t)(c0 + c) * kHist]);
    }
    // (z: threads in order; a row of up to 512 chunks has one each)
    z = wave_sum(z);
    far = __any(far);
    if (lane == 0) { H.wave[wave] = __builtin_bit_cast(u64, z); H.a[wave] = far; }
    H.merge.part[half][mine] = v;
    if (t == 0) { H.bin = -1; H.n = kHist; }
    __syncthreads();
    z = 0.0;
    far = false;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        z += __builtin_bit_cast(double, H.wave[w]);
        far = far || H.a[w];
    }
    v = half ? 0.0 : (H.merge.part[0][slot] + (kSides > 1 ? H.merge.part[kSides - 1][slot] : 0.0)) * 0x1p-50;
    double run = wave_scan(v);
    if (!half && lane == 63) H.merge.wave[wave] = run;
    __syncthreads();
    for (int w = 0; w < wave && !half; ++w) run += H.merge.wave[w];
    // (the least bin whose running sum reaches it: the scan's sums may be a
    // rounding apart from lane to lane)
    const u64 past = __ballot(!half && slot < kHist - 1 && run >= A.top_p * z && v > 0.0);
    if (past && lane == 0) atomicMin(&H.n, wave * 64 + __ffsll(past) - 1);
    __syncthreads();
    if (!half && slot == H.n && !far) {
        H.bin = slot;
        H.left = run - v;
    }
    if (t == 0) H.sum = z;
    __syncthreads();
}

// What launch 1 does, for a row that this launch holds whole: its groups' maxima
// (a group is a piece: u * kRow + t of thread t), the one chunk's statistics (H.one) and
// the thread's slot of its bins.
template <int KIND, int U>
__device__ __forceinline__ void read_row(const SampleArgs& P, RowShared& H, int r, const Row& q, float (&gm)[U], Part& own,
                                         u64& slot) {
    constexpr int N = kPer<KIND>;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i0 = (u * kRow + t) * N - q.off;
        raw[u] = make_uint4(0, 0, 0, 0);
        if (i0 >= 0 && i0 + N <= P.vocab) raw[u] = *reinterpret_cast<const uint4*>(q.p + (int64_t)i0 * kBytes<KIND>);
    }
    const Ask A = ask_of(P, r);
    fill_table(H.tab);
    if (t < kHist) H.h.sum[t] = 0;
    float x[U][N], m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i0 = (u * kRow + t) * N - q.off;
        unpack<KIND>(raw[u], x[u]);
        if (!(i0 >= 0 && i0 + N <= P.vocab)) {
#pragma unroll
            for (int e = 0; e < N; ++e) x[u][e] = i0 + e >= 0 && i0 + e < P.vocab ? one<KIND>(q.p, i0 + e) : -INFINITY;
        }
        gm[u] = x[u][0];
#pragma unroll
        for (int e = 1; e < N; ++e) gm[u] = fmaxf(gm[u], x[u][e]);
        m = fmaxf(m, gm[u]);
    }
    m = wave_max(m);
    if (lane == 0) H.m[wave] = m;
    if (t == 0) { H.found = 0x7fffffff; H.n = 0; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, H.m[w]);
    own = Part{m, 0x7fffffff, 0, 0, 0.0};
    slot = 0;
    if (A.greedy) {
        int a = 0x7fffffff;
#pragma unroll
        for (int u = U - 1; u >= 0; --u)
#pragma unroll
            for (int e = N - 1; e >= 0; --e)
                if (x[u][e] == m) a = (u * kRow + t) * N - q.off + e;
        if (a != 0x7fffffff) atomicMin(&H.found, a);
    }
    if (A.sum() && m != -INFINITY) {
        const Scale S = scale_of(m, A.inv);
        const float step = A.step(), top = bin_at(m, step);
        const bool bins = A.bins();
        double z = 0.0;
        int n = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const double w = add_pow(fmax(((double)x[u][e] - S.m) * S.a, -63700.0), 0.0, H.tab);
                if (bins) {
                    const u64 f = fixed(w, 0x1p50);
                    if (f) atomicAdd(&H.h.sum[(int)fminf(top - bin_at(x[u][e], step), (float)(kHist - 1))], f);
                } else {
                    z += w;
                    n += x[u][e] != -INFINITY;
                }
            }
        __syncthreads();
        if (bins) {
            own.n = fabsf(m * step) < kFar ? (int)top : 0x7fffffff;
            if (t < kHist) slot = H.h.sum[(own.n - t) & (kHist - 1)];
            const u64 f = wave_add(t < kHist ? slot : 0);
            z = (double)f * 0x1p-50;
        } else {
            z = wave_sum(z);
            n = (int)wave_add((u64)n);
        }
        if (lane == 0) {
            H.wave[wave] = __builtin_bit_cast(u64, z);
            if (!bins) atomicAdd(&H.n, n);
        }
    }
    __syncthreads();
    if (A.sum() && m != -INFINITY) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) own.z += __builtin_bit_cast(double, H.wave[w]);
        if (!A.bins()) own.n = H.n;
    }
    own.arg = H.found;
    if (t == 0) H.one = own;
    __syncthreads();
}

// A workgroup a row: a chain of LDS passes and barriers, with few bytes behind them.
// One row of 6400 (WHOLE) 9.5 us, 640 rows by top-k 24 (7 to 15 a row), 160 by top-p
// 36, where thousands stay: the bin's tokens gathered 15 to 18, its search 4, the
// chunks' sums 4, the draw 6.  512 threads: with 256
// 640 rows by top-k 400 took 45 us instead of 50 a call, 48 flat rows 86 instead of 51.
// WHOLE: a row of up to kSmall pieces, which one launch reads and decides: 6400
// logits 15.6 -> 11 us a call, as the second launch's 4 go.
template <int KIND>
constexpr int kSmall = 8192 / kPer<KIND>;
// BINS: a row may ask for top-p.  Calls without need neither the bins nor what
// follows from them, and in 80 registers three rows fit a CU instead of two (f32's
// would not without memory): 640 rows of 64402 by top-k 50 36 -> 32 us a call, 400 51
// -> 43, without a cut 51 -> 47.
template <int KIND, bool WHOLE, bool BINS>
__global__ void __launch_bounds__(kRow, BINS || KIND == VGX_E_F32 ? 1 : 6) sample_pick_kernel(const SampleArgs P) {
    constexpr int N = kPer<KIND>, LG = WHOLE ? 1 : kGroup / N, kHold = WHOLE ? kSmall<KIND> / kRow : 3;
    __shared__ RowShared H;
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const Row q = row_at<KIND>(P.x, P.xs, r);
    const Part* part = WHOLE ? &H.one : P.part + (int64_t)r * P.nch;
    const float* gmax = P.gmax + (int64_t)r * P.ng;
    // the thread's chunk, and the groups' maxima, the first ones held (not used where
    // the row has none)
    Part own;
    float held[kHold];
    u64 bins_of[kHoldBins];
    if constexpr (WHOLE) {
        read_row<KIND, kHold>(P, H, r, q, held, own, bins_of[0]);
    } else {
        own = part[min(t, P.nch - 1)];
#pragma unroll
        for (int i = 0; i < kHold; ++i) held[i] = gmax[min(t + i * kRow, P.ng - 1)];
    }
    auto each_group = [&](auto f) {
        if constexpr (WHOLE) {
#pragma unroll
            for (int i = 0; i < kHold; ++i) f(i * kRow + t, held[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kHold; ++i) {
                const bool in = t + i * kRow < P.ng;
                f(t + i * kRow, in ? held[i] : -INFINITY);
            }
            for (int g = t + kHold * kRow; g - t < P.ng; g += kRow) f(g, g < P.ng ? gmax[g] : -INFINITY);
        }
    };
    const Ask A = ask_of(P, r);
    const bool by_bins = BINS && A.bins();
    if constexpr (!WHOLE) {
        if (by_bins) {
            const u64* hist = P.hist + (int64_t)r * P.nch * kHist + (t & (kHist - 1));
#pragma unroll
            for (int k = 0; k < kHoldBins; ++k) bins_of[k] = hist[(int64_t)min(t / kHist + kSides * k, P.nch - 1) * kHist];
        }
        fill_table(H.tab);
    }
    int a;
    if (A.greedy || A.none()) {
        const float m = join_max(P, H, part, A.greedy, a);
        const bool nothing = m == -INFINITY;
        if (nothing || A.greedy) {
            if (t == 0) {
                P.token[r] = nothing ? -1 : a;
                if (P.kept) P.kept[r] = !nothing;
                if (P.prob) P.prob[r] = nothing ? 0.0f : 1.0f;
            }
            return;
        }
        const Scale S = scale_of(m, A.inv);
        int n = 0;
        for (int c = t; c < P.nch; c += kRow) {
            H.chunk.sum[c] = part[c].z * weight(part[c].m, S, H.tab);
            n += part[c].n;
        }
        u64 kept;
        block_scan((u64)n, H.wave, kept);
        return draw_in_chunks<KIND>(P, H, r, q, S, (int)kept, [](float, int) { return true; });
    }
    float m = -INFINITY, low = INFINITY;
    each_group([&](int, float x) {
        m = fmaxf(m, x);
        if (x != -INFINITY) low = fminf(low, x);
    });
    m = wave_max(m);
    low = -wave_max(-low);
    if (lane == 0) { H.m[wave] = m; H.low[wave] = low; }
    for (int i = t; i < kBins; i += kRow) H.h.cnt[i] = 0;
    if (t == 0) { H.n = 0; H.stay = 0; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        m = fmaxf(m, H.m[w]);
        low = fminf(low, H.low[w]);
    }
    if (m == -INFINITY) {
        if (t == 0) {
            P.token[r] = -1;
            if (P.kept) P.kept[r] = 0;
            if (P.prob) P.prob[r] = 0.0f;
        }
        return;
    }
    const Scale S = scale_of(m, A.inv);
    const Weigh W{S, __longlong_as_double((long long)(1023 + P.q) << 52), A.min_p, H.tab};
    const float hstep = A.step(), top = bin_at(m, hstep);
    double z = -1.0;
    // All that may stay: x >= floor_m, and in bins of the distance from m up to
    // last (not: every bin).
    float floor_m = -INFINITY, step = 0.0f;
    int last = kBins - 1;
    bool open = true;  // nothing is known of the row
    int must = 0;      // tokens that have to reach it
    if (by_bins) {
        find_bin(P, H, part, own, bins_of, r, A, S, top);
        z = H.sum;
        if (H.bin >= 0) {
            open = false;
            last = H.bin;
        }
    } else if (A.m && !A.k) {
        if (A.p) {  // (one wave's order for every thread)
            z = 0.0;
            for (int c = lane; c < P.nch; c += 64) z += part[c].z * weight(part[c].m, S, H.tab);
            z = wave_sum(z);
        }
        // a rounding below min-p's border
        if (A.inv > 0.0) {
            floor_m = (float)((double)m + log(A.min_p) / A.inv) - 1e-5f * (fabsf(m) + (float)(1.0 / A.inv));
            open = false;
        }
    } else {  // as many tokens as top-k keeps reach what as many groups' maxima do
        step = (float)(kBins - 1) / fmaxf(m - low, 1e-30f);
        each_group([&](int, float x) {
            if (x != -INFINITY) atomicAdd(&H.h.cnt[(int)fminf((m - x) * step, (float)(kBins - 1))], 1u);
        });
        __syncthreads();
        u64 groups;
        const unsigned c0 = H.h.cnt[2 * t], c1 = H.h.cnt[2 * t + 1];
        const u64 run = block_scan(c0 + c1, H.wave, groups);
        // Where k nears the number of groups that would be nearly all logits.  Of
        // logits that lie in no order a share f is found in 1 - (1 - f)^(a group's
        // size) of the groups; asked for is a quarter more than k, and whether k
        // reach it is counted.  (Up to a third of the groups that is above k.)
        u64 want = (u64)A.top_k;
        if (want * 3 > groups) {
            constexpr int size = WHOLE ? N : kGroup;
            const float f = 1.25f * (float)A.top_k / ((float)groups * size);
            const float likely = f < 1.0f ? (float)groups * (1.0f - expf(size * log1pf(-f))) : (float)groups;
            want = min(want, (u64)likely + 1);
        }
        if (run >= want && run - c0 - c1 < want) H.bin = run - c1 >= want ? 2 * t : 2 * t + 1;
        __syncthreads();
        if (want <= groups && A.top_k <= kList) {
            open = false;
            last = H.bin;
            if (want < (u64)A.top_k) must = A.top_k;
        }
    }
    bool bins = by_bins && last < kHist - 1;  // top-p's bin is known
    // What may stay is lo or more, what does (bins) hi or more.
    float lo = -FLT_MAX, hi = INFINITY;
    const float edge = top - (float)last;
    if (bins) {
        bins = first_in(edge, hstep, lo) && first_in(edge + 1.0f, hstep, hi);
        open = !bins;
        if (open) hi = INFINITY;
    } else if (floor_m > -INFINITY) {
        lo = fmaxf(floor_m, -FLT_MAX);
    } else if (last < kBins - 1) {  // (a rounding below the bin's border)
        lo = fmaxf(m - (float)(last + 1) / step * 1.000001f - fabsf(m) * 1e-6f, -FLT_MAX);
    }
    if (open && P.vocab <= kList) {  // all of it is gathered
        open = false;
        lo = -FLT_MAX;
    }
    if (!open) {
        __syncthreads();
        if (t == 0) { H.n = 0; H.above_n = 0; H.stay = 0; H.found = 0; }
        __syncthreads();
        each_group([&](int g, float x) {
            const bool some = x >= lo;
            const int at = place_of(some, &H.found);
            if (some && at < kGroups) H.groups[at] = g;
            const int sure = __popcll(__ballot(x >= hi));
            if (sure && lane == 0) atomicAdd(&H.stay, sure);
        });
        __syncthreads();
        // (groups with a token above top-p's bin: past half the list's room those
        // tokens are only counted)
        const bool listed = H.found <= kGroups;  // else all are read
        const int ngr = listed ? H.found : P.ng, i0 = bins ? kAbove : 0;
        auto group_of = [&](int j) { return listed ? H.groups[j / LG] * LG + j % LG : j; };
        const bool many = H.stay > kAbove / 2;
        __syncthreads();
        if (t == 0) H.stay = 0;
        // Pieces in one round trip, and one copy of what is done with them
        // (several would be fetched from memory for a run or two).
        constexpr int U = 4;
        const int pieces = ngr * LG;
        int sure = 0;
#pragma unroll 1
        for (int j0 = 0; j0 < pieces; j0 += kRow * U) {
            uint4 v[U];
            int at0[U];  // the index of a piece's first value
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + u * kRow + t;
                v[u] = make_uint4(0, 0, 0, 0);
                at0[u] = j < pieces ? group_of(j) * N - q.off : P.vocab;
                if (at0[u] >= 0 && at0[u] + N <= P.vocab)
                    v[u] = *reinterpret_cast<const uint4*>(q.p + (int64_t)at0[u] * kBytes<KIND>);
            }
#pragma unroll 1
            for (int u = 0; u < U && j0 + u * kRow < pieces; u += 2) {  // two a time
                // (as they lie in memory: NaN reaches nothing, infinity all)
                float x[2][N];
                const bool ends = at0[0] < 0 || at0[0] + N > P.vocab || at0[1] < 0 || at0[1] + N > P.vocab;
#pragma unroll
                for (int w = 0; w < 2; ++w) unpack<KIND, false>(v[w], x[w]);
                if (__any(ends)) {  // (a row's)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const unsigned inside = ends_of(at0[w], N, P.vocab);
                        if (inside) v[w] = raw_piece<KIND>(q, P.vocab, (at0[w] + q.off) / N);
                        unpack<KIND, false>(v[w], x[w]);
#pragma unroll
                        for (int e = 0; e < N; ++e) x[w][e] = inside >> e & 1 ? x[w][e] : -INFINITY;
                    }
                }
                // a bit a value: an addition with its carry each
                auto reach = [&](float y) {
                    unsigned r = 0, past;
#pragma unroll
                    for (int e = 2 * N - 1; e >= 0; --e) r = __builtin_addc(r, r, (unsigned)(x[e / N][e % N] >= y), &past);
                    return r;
                };
                const unsigned does = bins ? reach(hi) : 0, may = reach(lo) & ~does;
                auto put = [&](unsigned bits, int* n, int at, int most) {
                    at += place_of(__popc(bits), n);
                    for (; bits && at < most; bits &= bits - 1, ++at) {
                        const int k = __ffs(bits) - 1, e = k & (N - 1);
                        const bool second = k >= N;
                        const uint4 y = make_uint4(second ? v[1].x : v[0].x, second ? v[1].y : v[0].y,
                                                   second ? v[1].z : v[0].z, second ? v[1].w : v[0].w);
                        H.key[at] = key_of(value_in<KIND>(y, e));
                        H.idx[at] = (second ? at0[1] : at0[0]) + e;
                    }
                };
                put(may, &H.n, i0, kList);
                if (bins) {
                    if (many) sure += __popc(does);
                    else put(does, &H.above_n, 0, kAbove);
                }
#pragma unroll
                for (int w = 0; w + 2 < U; ++w) {
                    v[w] = v[w + 2];
                    at0[w] = at0[w + 2];
                }
            }
        }
        if (many) {
            sure = (int)wave_add((u64)sure);
            if (lane == 0) atomicAdd(&H.above_n, sure);
        }
        __syncthreads();
        const int n = H.n, above = bins ? H.above_n : 0;
        if (n <= kList - i0 && above <= kAbove && !many && n >= must) {
            const Gathered src{H, above, i0, n};
            if (above + n <= kFew) cut_and_draw_few(P, H, src, r, A, W, z);
            else cut_and_draw(P, H, src, r, A, W, m, z);
            return;
        }
        if (bins && n <= kList - kAbove) {
            // Thousands stay: all above top-p's bin, and of its own tokens, which
            // are gathered, those to be found.
            const int kept = above;
            const double left = H.left;
            Cut cut{0, 0x7fffffff};
            const double y = ceil((A.top_p * z - left) * W.scale);
            if (locate<true, false>(H, Gathered{H, 0, kAbove, n}, W, cut, (edge + 1.0f) / hstep, 1.0f / hstep, P.vocab,
                                    [&](u64) { return y < 1.0 ? 1ull : (u64)y; }))
                cut = H.at;
            __syncthreads();
            // the chunks' sums: their bins above the cut's (the first chunks' are
            // held), then those of the bin's tokens that stay
            const int per = P.k * kThreads * N;
            for (int c = t; c < P.nch; c += kRow) H.chunk.more[c] = 0;
            if (t < kSides * kHoldBins) H.first[t] = 0;
            __syncthreads();
            int more = 0;
            Gathered{H, 0, kAbove, n}.each([&](unsigned key, int i) {
                if (!stays(cut, key, i)) return;
                ++more;
                atomicAdd(&H.chunk.more[(i + q.off) / per], W(key));
            });
            more = (int)wave_add((u64)more);
            if (lane == 0) atomicAdd(&H.stay, more);
            const int mine = ((int)top - t) & (kHist - 1);
#pragma unroll
            for (int k = 0; k < kHoldBins; ++k) {
                const int c = t / kHist + kSides * k;
                if (c >= P.nch) continue;
                const int at = mine - H.down[c];
                const u64 f = wave_add(at >= 0 && at < kHist - 1 && mine < last ? bins_of[k] : 0);
                if (lane == 0 && f) atomicAdd(&H.first[c], f);
            }
            __syncthreads();
            if (t < min(P.nch, kSides * kHoldBins))
                H.chunk.sum[t] = (double)H.first[t] * 0x1p-50 * H.weight[t] + (double)H.chunk.more[t] / W.scale;
            for (int c = kSides * kHoldBins + wave; c < P.nch; c += kWaves) {
                const float cm = part[c].m;
                const int n = part[c].n, bins_in = cm == -INFINITY ? 0 : last - (int)fminf(top - (float)n, (float)kHist);
                u64 f = 0;
                for (int b = lane; b < bins_in; b += 64)
                    f += P.hist[((int64_t)r * P.nch + c) * kHist + slot_of(n, b)];
                f = wave_add(f);
                if (lane == 0)
                    H.chunk.sum[c] = (double)f * 0x1p-50 * weight(cm, S, H.tab) + (double)H.chunk.more[c] / W.scale;
            }
            __syncthreads();
            return draw_in_chunks<KIND>(P, H, r, q, S, kept + H.stay, [&](float x, int i) {
                return x >= hi || (x >= lo && stays(cut, key_of(x), i));
            });
        }
        __syncthreads();
    }
    cut_and_draw_whole<KIND>(P, H, r, q, A, W, m);
}

// Pieces a thread and chunk (K) and chunks of a row; chunks of 256 pieces while
// they are 1024 or fewer, 128 a row.
struct Chunks {
    int k, nch, ng;
};
Chunks chunks_of(int nrows, int vocab, int kind) {
    const int per = kind == VGX_E_F32 ? 4 : 8;
    Chunks c;
    if (vocab + per - 1 <= 8192) {  // one launch
        c.k = 8192 / per / kThreads;
        c.nch = c.ng = 0;
        return c;
    }
    c.k = 1;
    c.nch = (vocab + per - 1 + per * kThreads - 1) / (per * kThreads);
    if ((int64_t)nrows * c.nch > 1024 || c.nch > 128) {
        c.k = 4;
        c.nch = (vocab + per - 1 + per * kThreads * 4 - 1) / (per * kThreads * 4);
    }
    c.ng = c.nch * c.k * kThreads * per / kGroup;
    return c;
}

template <int KIND>
void launch(const SampleArgs& P, hipStream_t st) {
    if (P.ng == 0) {
        hipLaunchKernelGGL((sample_pick_kernel<KIND, true, true>), dim3(P.nrows), dim3(kRow), 0, st, P);
        return;
    }
    hipLaunchKernelGGL((P.k == 1 ? sample_stats_kernel<KIND, 1> : sample_stats_kernel<KIND, 4>), dim3(P.nch, P.nrows),
                       dim3(kThreads), 0, st, P);
    hipLaunchKernelGGL((P.top_p ? sample_pick_kernel<KIND, false, true> : sample_pick_kernel<KIND, false, false>), dim3(P.nrows),
                       dim3(kRow), 0, st, P);
}

bool kind_ok(int k) { return k == VGX_E_F32 || k == VGX_E_BF16 || k == VGX_E_F16 || k == VGX_E_Q16; }

}  // namespace

extern "C" {

size_t vgx_sample_ws(int nrows, int vocab, int kind) {
    if (nrows < 0 || vocab <= 0 || vocab > kMaxVocab || !kind_ok(kind)) return 0;
    const Chunks c = chunks_of(nrows, vocab, kind);
    return (size_t)nrows * (c.nch * (sizeof(Part) + kHist * sizeof(u64)) + c.ng * sizeof(float));
}

int vgx_sample(vgx_ctx* ctx, const vgx_sampling* a) {
    auto fail = [](int status, const char* what) { return vgx_fail(status, std::string("vgx_sample: ") + what); };
    if (!a) return fail(VGX_EINVAL, "NULL arguments");
    if (a->nrows < 0 || a->nrows > 65535) return fail(VGX_EINVAL, "nrows outside 0..65535");
    if (a->vocab <= 0 || a->vocab > kMaxVocab) return fail(VGX_EINVAL, "vocab outside 1..2^21");
    if (!kind_ok(a->kind)) return fail(VGX_EINVAL, "logits are f32, bf16, f16 or q16");
    if (a->nrows && (!a->logits || !a->u || !a->token)) return fail(VGX_EINVAL, "NULL logits, u or token");
    const int eb = a->kind == VGX_E_F32 ? 4 : 2;
    if (a->stride < a->vocab || a->stride > ((int64_t)1 << 40)) return fail(VGX_EINVAL, "a row stride below vocab or above 2^40");
    if ((uintptr_t)a->logits & (eb - 1)) return fail(VGX_EINVAL, "logits not aligned to their type");
    const size_t need = vgx_sample_ws(a->nrows, a->vocab, a->kind);
    if (need && (!a->ws || a->ws_bytes < need || ((uintptr_t)a->ws & 15)))
        return fail(VGX_EINVAL, "the workspace is missing, too small or not 16-byte aligned");
    const Chunks c = chunks_of(a->nrows, a->vocab, a->kind);
    if ((int64_t)c.nch * a->nrows >= (1 << 24)) return fail(VGX_ERANGE, "too many logits for one call");  // 2^32 threads
    if (!ctx) return fail(VGX_EINVAL, "no context");
    if (a->nrows == 0) return VGX_OK;
    SampleArgs P{};
    P.nrows = a->nrows; P.vocab = a->vocab;
    P.x = static_cast<const uint8_t*>(a->logits);
    P.xs = a->stride * eb;
    P.u = a->u;
    P.temp = a->temp; P.top_k = a->top_k; P.top_p = a->top_p; P.min_p = a->min_p;
    P.token = a->token; P.kept = a->kept; P.prob = a->prob;
    int lg = 0;
    while ((1 << lg) < a->vocab) ++lg;
    P.q = std::min(50, 62 - lg);
    P.nch = std::max(c.nch, 1); P.k = c.k; P.ng = c.ng;
    P.hist = static_cast<u64*>(a->ws);
    P.part = reinterpret_cast<Part*>(P.hist + (size_t)a->nrows * c.nch * kHist);
    P.gmax = reinterpret_cast<float*>(P.part + (size_t)a->nrows * c.nch);
    VGX_HIP(hipSetDevice(ctx->device));
    switch (a->kind) {
        case VGX_E_F32: launch<VGX_E_F32>(P, ctx->stream); break;
        case VGX_E_BF16: launch<VGX_E_BF16>(P, ctx->stream); break;
        case VGX_E_F16: launch<VGX_E_F16>(P, ctx->stream); break;
        default: launch<VGX_E_Q16>(P, ctx->stream); break;
    }
    VGX_LAUNCH_CHECK("sample launch");
    return VGX_OK;
}

}  // extern "C"
