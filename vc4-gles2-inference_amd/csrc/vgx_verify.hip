// Checking drafted tokens against the target's logits.
//
// p_r = softmax(l_r / T) of the target's row r, q_r of the draft's (1 at the
// drafted token where its logits are not given).  The row's draft t is taken
// when u q_r(t) < p_r(t); the first row that does not (or the sequence's last
// row, which has no draft) gives the next token: the least j whose running
// sum of w passes u' times the sum of all, w = max(p - q, 0) of a refused row
// and p of the last.  Integers come out, so the exponentials and sums run in
// 64 bits: a draw next to a border of the running sum has thousands of
// borders to be wrong at.
//
// Launch 1 reads every logit once (a workgroup a row and chunk): the chunk's
// maximum, its first index and its sum of exponentials.  With draft logits
// launch 2 sums the chunks of w for the refused rows.  The last launch (a
// workgroup a sequence) joins the rows' chunks, takes or refuses, finds the
// chunk the draw falls into from the chunks' sums and the token in it from a
// scan of that chunk alone.
//
// The exponentials (vgx_logits.h) are 12 of the 29 vector instructions a logit of
// launch 1; q16's go by two tables (stats16_kernel).
#include <string>
#include <type_traits>

#include "vgx_logits.h"

#pragma clang fp contract(off)

namespace {

struct VerifyArgs {
    int nseq, ntok, vocab;
    const int* qstart;
    const int* tokens;
    const uint8_t* x;
    const uint8_t* d;     // the draft's logits, or nullptr
    int64_t xs, ds;       // bytes between rows
    const float* temp;
    const float* ua;
    const float* un;
    int* accepted;
    int* next;
    float* prob;
    struct Part* px;      // ntok x nch
    struct Part* pd;
    double* w;            // nseq x nch: sums of w of the refused rows
    int nch, chunk;       // chunks of a row, pieces of a chunk
};

struct Part {
    float m;   // the chunk's maximum (-inf: nothing)
    int arg;   // its first index
    double z;  // sum of exp((x - m) / T)
};

constexpr int kThreads = 256;
// A chunk is K pieces of 16 bytes a thread of launch 1: 4, or 1 where the
// launch would leave CUs idle.
constexpr int kPick = 512;  // threads of the last launch: its waves take a row each

struct Temp {
    double inv;
    bool greedy;
};
__device__ __forceinline__ Temp temp_of(const VerifyArgs& P, int s) {
    const float t = P.temp ? P.temp[s] : 1.0f;
    Temp r;
    r.greedy = !(t > 0.0f);
    r.inv = r.greedy ? 1.0 : fmin(1.0 / (double)t, 1e30);
    return r;
}
// The sequence of row t (every lane active); nseq behind the last.
__device__ __forceinline__ int seq_of(const VerifyArgs& P, int t) {
    int s = 0;
    for (int b = 0; b < P.nseq; b += 64) {
        const int j = b + (int)(threadIdx.x & 63);
        s += __popcll(__ballot((j < P.nseq ? P.qstart[j + 1] : 0x7fffffff) <= t));
    }
    return s;
}

// What every launch-1 kernel ends with: the waves' statistics joined.
struct Joined {
    float m[4];
    int a[4];
    double z[4];
};
__device__ __forceinline__ void stats_best(Joined& J, bool greedy, float& m, int& a) {
    if (greedy) wave_best(m, a);
    else m = wave_max(m);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { J.m[wave] = m; J.a[wave] = a; }
    __syncthreads();
    m = J.m[0];
    a = J.a[0];
#pragma unroll
    for (int w = 1; w < 4; ++w)
        if (J.m[w] > m || (J.m[w] == m && J.a[w] < a)) { m = J.m[w]; a = J.a[w]; }
}
__device__ __forceinline__ void stats_put(Joined& J, Part* to, float m, int a, double z) {
    z = wave_sum(z);
    if ((threadIdx.x & 63) == 0) J.z[threadIdx.x >> 6] = z;
    __syncthreads();
    if (threadIdx.x == 0) *to = Part{m, a, J.z[0] + J.z[1] + J.z[2] + J.z[3]};
}

// 126 rows of 73448 f32 logits and the draft's, 20 us (3.7 TB/s): 14 us of vector
// instructions (29 a logit, at 2.4 GHz) and 12 of bytes, which overlap in part
// only: a workgroup loads its chunk, then computes.
template <int KIND, int K>
__global__ void __launch_bounds__(kThreads) stats_kernel(const VerifyArgs P) {
    constexpr int N = kPer<KIND>;
    __shared__ double tab[64];
    __shared__ Joined J;
    const int chunk = blockIdx.x, t = blockIdx.y;
    const bool draft = blockIdx.z;
    const Row q = row_at<KIND>(draft ? P.d : P.x, draft ? P.ds : P.xs, t);
    auto first = [&](int k) { return ((chunk * K + k) * kThreads + (int)threadIdx.x) * N - q.off; };
    // (a row's first and last piece may be short: read value by value)
    auto full = [&](int i0) { return i0 >= 0 && i0 + N <= P.vocab; };
    uint4 raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        raw[k] = make_uint4(0, 0, 0, 0);
        if (full(first(k))) raw[k] = *reinterpret_cast<const uint4*>(q.p + (int64_t)first(k) * kBytes<KIND>);
    }
    const int s = seq_of(P, t);
    fill_table(tab);
    if (s >= P.nseq) return;  // (uniform)
    const Temp T = temp_of(P, s);
    float x[K][N];
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
#pragma unroll
        for (int e = 0; e < N; ++e) m = fmaxf(m, x[k][e]);
    }
    int a = 0x7fffffff;
    if (T.greedy) {  // the first index of the maximum
#pragma unroll
        for (int k = K - 1; k >= 0; --k)
#pragma unroll
            for (int e = N - 1; e >= 0; --e)
                if (x[k][e] == m) a = first(k) + e;
    }
    stats_best(J, T.greedy, m, a);
    double z[2] = {0.0, 0.0};
    if (!T.greedy && m != -INFINITY) {
        const Scale S = scale_of(m, T.inv);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < N; ++e)
                z[e & 1] = add_pow(fmax(((double)x[k][e] - S.m) * S.a, -63700.0), z[e & 1], tab);
    }
    stats_put(J, (draft ? P.pd : P.px) + (int64_t)t * P.nch + chunk, m, a, z[0] + z[1]);
}

// q16 logits are integers, and the maximum less one of them, d, is one of
// 0 .. 65535: e^(-d / 256 T) is a product of two table entries, of d's low byte
// and of its high one.  exp16 is that product computed alone.
__device__ __forceinline__ double exp_low(int i, double a256, const double* tab) {
    return add_pow(fmax((double)-i * a256, -63700.0), 0.0, tab);
}
__device__ __forceinline__ double exp16(int d, const Scale& S, const double* tab) {
    const double a256 = S.a * (1.0 / 256);
    return exp_low(d & 255, a256, tab) * exp_low(d & 0xff00, a256, tab);
}
typedef short short2v __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));

// Launch 1 for q16: two LDS reads and one operation of 64 bits a logit instead of
// 12.  654 rows of 64402, 22 us (3.8 TB/s; 31 us by stats_kernel's way): 13 us of
// vector instructions (12 a logit) and 13 of bytes; the tables cost a thread 2
// exponentials beside its 8 or 32 logits.
template <int K>
__global__ void __launch_bounds__(kThreads) stats16_kernel(const VerifyArgs P) {
    constexpr int KIND = VGX_E_Q16, N = 8;
    __shared__ double tab[64], low[256], high[256];
    __shared__ Joined J;
    const int chunk = blockIdx.x, t = blockIdx.y, tid = threadIdx.x;
    const bool draft = blockIdx.z;
    const Row q = row_at<KIND>(draft ? P.d : P.x, draft ? P.ds : P.xs, t);
    auto first = [&](int k) { return ((chunk * K + k) * kThreads + tid) * N - q.off; };
    auto full = [&](int i0) { return i0 >= 0 && i0 + N <= P.vocab; };
    auto in = [&](int i) { return i >= 0 && i < P.vocab; };
    union Piece {
        uint4 v;
        unsigned u[4];
        short x[8];
    } raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        raw[k].v = make_uint4(0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u);  // (nothing: the least value)
        if (full(first(k))) raw[k].v = *reinterpret_cast<const uint4*>(q.p + (int64_t)first(k) * 2);
    }
    const int s = seq_of(P, t);
    fill_table(tab);
    if (s >= P.nseq) return;  // (uniform)
    const Temp T = temp_of(P, s);
    const Scale S = scale_of(0.0f, T.inv);
    __syncthreads();
    if (!T.greedy) {
        low[tid] = exp_low(tid, S.a * (1.0 / 256), tab);
        high[tid] = exp_low(tid << 8, S.a * (1.0 / 256), tab);
    }
    short2v best = {-32768, -32768};
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int i0 = first(k);
        if (!full(i0)) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (in(i0 + e)) raw[k].x[e] = reinterpret_cast<const short*>(q.p)[i0 + e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            best = __builtin_elementwise_max(best, __builtin_bit_cast(short2v, raw[k].u[e]));
    }
    const short top = best.x > best.y ? best.x : best.y;
    int a = 0x7fffffff;
    if (T.greedy) {
#pragma unroll
        for (int k = K - 1; k >= 0; --k)
#pragma unroll
            for (int e = N - 1; e >= 0; --e)
                if (raw[k].x[e] == top && in(first(k) + e)) a = first(k) + e;
    }
    // (a thread may have no value at all)
    bool some = false;
#pragma unroll
    for (int k = 0; k < K; ++k) some = some || (first(k) + N > 0 && first(k) < P.vocab);
    float m = some ? (float)top * (1.0f / 256) : -INFINITY;
    stats_best(J, T.greedy, m, a);
    double z[2] = {0.0, 0.0};
    if (!T.greedy && m != -INFINITY) {
        const unsigned short mi = (unsigned short)(short)(int)(m * 256.0f);
        const ushort2v m2 = {mi, mi};
        auto at = [](const double* p, unsigned byte8) {
            return *reinterpret_cast<const double*>(reinterpret_cast<const char*>(p) + byte8);
        };
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i0 = first(k);
            if (full(i0)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned d = __builtin_bit_cast(unsigned, m2 - __builtin_bit_cast(ushort2v, raw[k].u[e]));
                    const double y0 = at(low, (d & 255) << 3), y1 = at(high, (d >> 8 & 255) << 3);
                    const double y2 = at(low, (d >> 16 & 255) << 3), y3 = at(high, (d >> 24) << 3);
                    z[0] = fma(y0, y1, z[0]);
                    z[1] = fma(y2, y3, z[1]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (in(i0 + e)) {
                        const unsigned short d = mi - (unsigned short)raw[k].x[e];
                        z[0] = fma(low[d & 255], high[d >> 8], z[0]);
                    }
            }
            __builtin_amdgcn_sched_barrier(0);  // (all pieces' reads at once would spill)
        }
    }
    stats_put(J, (draft ? P.pd : P.px) + (int64_t)t * P.nch + chunk, m, a, z[0] + z[1]);
}

__device__ __forceinline__ Part part_of(const VerifyArgs& P, const Part* p, int c) {
    return c < P.nch ? p[c] : Part{-INFINITY, 0x7fffffff, 0.0};
}
// A row's chunks (p; x: the first 64, a lane each) joined by one wave: its
// maximum, with best its first index, and its sum.
__device__ __forceinline__ Part join(const VerifyArgs& P, const Part* p, Part x, double inv, bool best,
                                     const double* tab) {
    const int lane = threadIdx.x & 63;
    Part r = x;
#pragma unroll 1
    for (int c = lane + 64; c < P.nch; c += 64)
        if (p[c].m > r.m || (p[c].m == r.m && p[c].arg < r.arg)) { r.m = p[c].m; r.arg = p[c].arg; }
    if (best) wave_best(r.m, r.arg);
    else r.m = wave_max(r.m);
    const Scale S = scale_of(r.m, inv);
    r.z = 0.0;
#pragma unroll 1
    for (int c = 0;;) {
        r.z += x.z * weight(x.m, S, tab);
        c += 64;
        if (c >= P.nch) break;
        x = part_of(P, p, c + lane);
    }
    r.z = wave_sum(r.z);
    return r;
}

// What a sequence's rows decide: the first row that refuses its draft (the
// last row where none does), and that row joined, by every thread of the
// workgroup.  A wave takes a row's logits or its draft's, kGroup rows at a time.
constexpr int kGroup = 32;
struct Shared {
    double tab[64];
    Part x[2][kGroup];    // the target's rows, the draft's
    double p[2][kGroup];  // what they give the drafted token
    int tok[kGroup];      // the drafted token, and its logit
    float lx[kGroup];
};
struct Decision {
    int q0, n, acc;
    bool refused;
    Part x, d;
    int tok;  // of a refused row: its draft, and that one's logit
    float lx;
};
template <int KIND>
__device__ __forceinline__ Decision decide(const VerifyArgs& P, int s, const Temp& T, Shared& H, bool write) {
    Decision r{};
    r.q0 = min(max(P.qstart[s], 0), P.ntok);
    r.n = max(min(P.qstart[s + 1], P.ntok) - r.q0, 0);
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    const int sides = P.d && !T.greedy ? 2 : 1;
    // (the first row's loads are on their way while the table is made)
    int side, i, tok;
    const Part* p;
    Part x;
    auto load = [&](int g, int m, int w) {
        side = w >= m;
        i = side ? w - m : w;
        const int t = r.q0 + g + i;
        p = (side ? P.pd : P.px) + (int64_t)t * P.nch;
        x = part_of(P, p, lane);
        tok = g + i + 1 < r.n ? P.tokens[t + 1] : -1;
    };
    if (wave < min(r.n, kGroup) * sides) load(0, min(r.n, kGroup), wave);
    fill_table(H.tab);
    __syncthreads();
#pragma unroll 1
    for (int g = 0; g < r.n; g += kGroup) {
        const int m = min(r.n - g, kGroup);
        const bool drafted = lane < m && g + lane + 1 < r.n;
        const float ua = drafted ? P.ua[r.q0 + g + lane] : 0.0f;
        if (g) __syncthreads();  // the last group's values are read
#pragma unroll 1
        for (int w = wave; w < m * sides; w += waves) {
            if (g || w != wave) load(g, m, w);
            const int t = r.q0 + g + i;
            const bool in = tok >= 0 && tok < P.vocab;
            const float l = one<KIND>(side ? P.d + (int64_t)t * P.ds : P.x + (int64_t)t * P.xs, in ? tok : 0);
            const Part y = join(P, p, x, T.inv, T.greedy, H.tab);
            double v;
            if (T.greedy) v = y.m != -INFINITY && tok == y.arg ? 1.0 : 0.0;
            else v = in && y.z > 0.0 ? weight(l, y.m, T.inv, H.tab) / y.z : 0.0;
            if (lane == 0) {
                H.x[side][i] = y;
                H.p[side][i] = v;
                if (!side) { H.tok[i] = tok; H.lx[i] = l; }
            }
        }
        __syncthreads();
        const double pr = drafted ? H.p[0][lane & (kGroup - 1)] : 0.0;
        const double qr = drafted && sides == 2 ? H.p[1][lane & (kGroup - 1)] : 1.0;
        const bool ok = T.greedy ? pr > 0.0 : (double)ua * qr < pr;
        if (write && P.prob && wave == 0 && lane < m) P.prob[r.q0 + g + lane] = (float)pr;
        const unsigned long long no = __ballot(drafted && !ok);
        if (!r.refused && (no || g + m == r.n)) {
            r.refused = no != 0;
            const int k = no ? __ffsll(no) - 1 : m - 1;
            r.acc = g + k;
            r.x = H.x[0][k];
            if (sides == 2) r.d = H.x[1][k];
            r.tok = H.tok[k];
            r.lx = H.lx[k];
        }
        if (r.refused && !write) break;
    }
    return r;
}

// w of one value of the refused row t.
struct Residual {
    Scale sx, sd;
    double zx, zd;  // 1 / the sums
    int tok;        // without draft logits: the refused token
};
__device__ __forceinline__ Residual residual_of(const Decision& D, double inv, int tok) {
    return {scale_of(D.x.m, inv), scale_of(D.d.m, inv), D.x.z > 0.0 ? 1.0 / D.x.z : 0.0,
            D.d.z > 0.0 ? 1.0 / D.d.z : 0.0, tok};
}
// A draw from p alone needs no 1 / the sum: the weights of equal maxima are then
// 1, their sums exact, and a draw at a border of theirs is decided as defined.
__device__ __forceinline__ void unscaled(Residual& R) {
    R.zx = 1.0;
}
__device__ __forceinline__ double residual(const Residual& R, bool draft, float x, float d, int j, const double* tab) {
    const double p = weight(x, R.sx, tab) * R.zx;
    if (!draft) return j == R.tok ? 0.0 : p;
    // (sums of rows that lie differently are added in different orders, and the
    // exponentials are good to 2^-44: less than 2^-40 of p is no difference)
    const double r = p - weight(d, R.sd, tab) * R.zd;
    return r > p * 0x1p-40 ? r : 0.0;
}

// With draft logits: the sums of w over the chunks of the refused rows.  Every
// workgroup decides for itself, which a launch between would cost more than: 32
// sequences of 73448, 8.8 us, most of it that chain.
template <int KIND>
__global__ void __launch_bounds__(kPick) residual_kernel(const VerifyArgs P) {
    constexpr int N = kPer<KIND>;
    __shared__ Shared H;
    __shared__ double sz[kPick / 64];
    const int chunk = blockIdx.x, s = blockIdx.y;
    const Temp T = temp_of(P, s);
    const Decision D = decide<KIND>(P, s, T, H, false);
    if (!D.refused || T.greedy) return;
    const int t = D.q0 + D.acc;
    const Residual R = residual_of(D, T.inv, -1);
    const Row qx = row_at<KIND>(P.x, P.xs, t), qd = row_at<KIND>(P.d, P.ds, t);
    double w = 0.0;
    for (int g = chunk * P.chunk + threadIdx.x; g < (chunk + 1) * P.chunk; g += kPick) {
        float a[N], b[N];
        piece<KIND>(qx, P.vocab, g, a);
        if (qx.off == qd.off) {
            piece<KIND>(qd, P.vocab, g, b);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int j = g * N - qx.off + e;
                b[e] = j >= 0 && j < P.vocab ? one<KIND>(qd.p, j) : -INFINITY;
            }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) w += residual(R, true, a[e], b[e], 0, H.tab);
    }
    w = wave_sum(w);
    if ((threadIdx.x & 63) == 0) sz[threadIdx.x >> 6] = w;
    __syncthreads();
    if (threadIdx.x == 0) {
        w = 0.0;
        for (int i = 0; i < kPick / 64; ++i) w += sz[i];
        P.w[(int64_t)s * P.nch + chunk] = w;
    }
}

// 9 us for one sequence of 6400 logits, 12 for 128 of 64402: a chain of about ten
// dependent steps (chunks' statistics, decision, their walk, one chunk's logits).
template <int KIND, int K>
__global__ void __launch_bounds__(kPick) pick_kernel(const VerifyArgs P) {
    constexpr int N = kPer<KIND>, PP = K > 1 ? K * kThreads / kPick : 1;  // pieces a thread
    __shared__ Shared H;
    __shared__ double sw[kPick / 64], left;
    __shared__ int chosen, found, last, plain;
    const int s = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Temp T = temp_of(P, s);
    const double un = P.un[s];  // (asked for before the chain below)
    const Decision D = decide<KIND>(P, s, T, H, true);
    if (D.n <= 0) {
        if (threadIdx.x == 0) { P.accepted[s] = 0; P.next[s] = -1; }
        return;
    }
    const int t = D.q0 + D.acc;
    const Part& x = D.x;
    const double* tab = H.tab;
    if (threadIdx.x == 0) P.accepted[s] = D.acc;
    if (T.greedy || x.m == -INFINITY) {
        if (threadIdx.x == 0) P.next[s] = x.m == -INFINITY ? -1 : x.arg;
        return;
    }
    bool draft = P.d && D.refused;
    Residual R = residual_of(D, T.inv, D.refused && !P.d ? D.tok : -1);
    if (!draft) unscaled(R);
    const Row qx = row_at<KIND>(P.x, P.xs, t);
    // the chunks' sums, walked by one wave; without draft logits they are
    // launch 1's, less the refused token
    const int tchunk = R.tok >= 0 && R.tok < P.vocab ? (R.tok + qx.off) / N / P.chunk : -1;
    if (wave == 0) {
        // (what launch 1 has added for the refused token, but for the rounding of
        // its fused additions)
        auto taken = [&](float m) {
            const Scale S = scale_of(m, T.inv);
            return KIND == VGX_E_Q16 ? exp16((int)((m - D.lx) * 256.0f), S, tab) : weight(D.lx, S, tab);
        };
        auto sum_of = [&](int c) {
            if (c >= P.nch) return 0.0;
            if (draft) return P.w[(int64_t)s * P.nch + c];
            const Part p = P.px[(int64_t)t * P.nch + c];
            const double w = weight(p.m, R.sx, tab);
            double z = p.z;
            // A chunk whose sum passes 0 has to hold a token that can be drawn: one
            // whose maximum is all but cut beside the row's counts as nothing
            // without the refused token, as its other weights may be cut.  (Otherwise
            // what is left is 0 or above 2^-53, so some weight is above 2^-66 of
            // the maximum's.)
            if (c == tchunk) z = w < 0x1p-900 ? 0.0 : fmax(z - taken(p.m), 0.0);
            return z * w * R.zx;
        };
        double total, v0;
        if (lane == 0) plain = 0;
#pragma unroll 1
        for (;;) {
            total = 0.0;
#pragma unroll 1
            for (int c = 0; c < P.nch; c += 64) {
                const double v = sum_of(c + lane);
                if (c == 0) v0 = v;
                total += v;
            }
            total = wave_sum(total);
            if (!draft || total > 0.0) break;
            draft = false;  // p = q: the draw is from p
            unscaled(R);
            if (lane == 0) plain = 1;
        }
        const double want = un * total;
        double before = 0.0;
        int pick = -1, some = -1;
        double at = 0.0, some_at = 0.0;
#pragma unroll 1
        for (int c = 0; c < P.nch && pick < 0; c += 64) {
            const double v = c ? sum_of(c + lane) : v0;
            const double run = wave_scan(v);
            const unsigned long long past = __ballot(before + run > want && v > 0.0);
            const unsigned long long any = __ballot(v > 0.0);
            if (past) {
                const int l = __ffsll((unsigned long long)past) - 1;
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
            chosen = pick >= 0 ? pick : some;
            left = fmax(want - (pick >= 0 ? at : some_at), 0.0);
            found = 0x7fffffff;
            last = -1;
        }
    }
    __syncthreads();
    if (plain) {
        draft = false;
        unscaled(R);
    }
    if (chosen < 0) {  // nothing but the refused token has a weight
        if (threadIdx.x == 0) P.next[s] = -1;
        return;
    }
    // the chosen chunk, PP consecutive pieces a thread
    const Row qd = draft ? row_at<KIND>(P.d, P.ds, t) : qx;
    const int g0 = chosen * P.chunk + threadIdx.x * PP;
    const bool mine_in = (int)threadIdx.x * PP < P.chunk;
    double w[PP * N];
    double sum = 0.0;
    int mine = -1;  // the thread's last value with a weight
#pragma unroll
    for (int k = 0; k < PP; ++k) {
        float a[N], b[N];
#pragma unroll
        for (int e = 0; e < N; ++e) a[e] = b[e] = -INFINITY;
        if (mine_in) {
            piece<KIND>(qx, P.vocab, g0 + k, a);
            if (draft && qx.off == qd.off) {
                piece<KIND>(qd, P.vocab, g0 + k, b);
            } else if (draft) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int j = (g0 + k) * N - qx.off + e;
                    b[e] = j >= 0 && j < P.vocab ? one<KIND>(qd.p, j) : -INFINITY;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int j = (g0 + k) * N - qx.off + e;
            w[k * N + e] = residual(R, draft, a[e], b[e], j, tab);
            sum += w[k * N + e];
            if (w[k * N + e] > 0.0) mine = j;
        }
    }
    const double run = wave_scan(sum);
    if (lane == 63) sw[wave] = run;
    if (mine >= 0) atomicMax(&last, mine);
    __syncthreads();
    // The first thread with a weight whose running sum has passed the draw.  (The
    // lanes' sums are added in different orders, so a thread without a weight
    // may have one a rounding above its neighbour's: it takes no part.)  Several
    // waves may find one: the least index is the first's.
    double before = __shfl_up(run, 1, 64);
    if (lane == 0) before = 0.0;
    double base = 0.0;
    for (int v = 0; v < wave; ++v) base += sw[v];
    before += base;
    const unsigned long long past = __ballot(mine >= 0 && base + run > left);
    if (past && lane == __ffsll(past) - 1) {
        int hit = -1;
        double u = before;
#pragma unroll
        for (int i = 0; i < PP * N; ++i) {
            u += w[i];
            if (hit < 0 && u > left && w[i] > 0.0) hit = (g0 + i / N) * N - qx.off + i % N;
        }
        atomicMin(&found, hit >= 0 ? hit : mine);
    }
    __syncthreads();
    if (threadIdx.x == 0) P.next[s] = found != 0x7fffffff ? found : last;
}

// Pieces a thread and chunk (K) and chunks of a row.  A row may begin inside a
// piece.  Chunks of 256 pieces (2048 16-bit logits) while they are fewer than
// 1024; one row of 6400: 3.8 us against 8.5 with chunks of 1024.
struct Cut {
    int k, nch;
};
Cut cut_of(int ntok, int vocab, int kind, bool draft) {
    const int per = kind == VGX_E_F32 ? 4 : 8;
    Cut c;
    c.k = 1;
    c.nch = (vocab + per - 1 + per * kThreads - 1) / (per * kThreads);
    if ((int64_t)ntok * c.nch * (draft ? 2 : 1) > 1024 || c.nch > 64) {
        c.k = 4;
        c.nch = (vocab + per - 1 + per * kThreads * 4 - 1) / (per * kThreads * 4);
    }
    return c;
}

template <int KIND>
void launch(const VerifyArgs& P, int k, hipStream_t st) {
    if (P.ntok) {
        void (*stats)(const VerifyArgs);
        if constexpr (KIND == VGX_E_Q16) stats = k == 1 ? stats16_kernel<1> : stats16_kernel<4>;
        else stats = k == 1 ? stats_kernel<KIND, 1> : stats_kernel<KIND, 4>;
        hipLaunchKernelGGL(stats, dim3(P.nch, P.ntok, P.d ? 2 : 1), dim3(kThreads), 0, st, P);
        if (P.d) hipLaunchKernelGGL(residual_kernel<KIND>, dim3(P.nch, P.nseq), dim3(kPick), 0, st, P);
    }
    hipLaunchKernelGGL((k == 1 ? pick_kernel<KIND, 1> : pick_kernel<KIND, 4>), dim3(P.nseq), dim3(kPick), 0, st, P);
}

bool kind_ok(int k) { return k == VGX_E_F32 || k == VGX_E_BF16 || k == VGX_E_F16 || k == VGX_E_Q16; }

}  // namespace

extern "C" {

size_t vgx_draft_verify_ws(int nseq, int ntok, int vocab, int kind, int with_draft) {
    if (nseq < 0 || ntok < 0 || vocab <= 0 || vocab > (1 << 26) || !kind_ok(kind)) return 0;
    const size_t nch = cut_of(ntok, vocab, kind, with_draft).nch;
    return nch * ((size_t)ntok * (with_draft ? 2 : 1) * sizeof(Part) + (size_t)(with_draft ? nseq : 0) * sizeof(double));
}

int vgx_draft_verify(vgx_ctx* ctx, const vgx_draft* a) {
    if (!a) return vgx_fail(VGX_EINVAL, "vgx_draft_verify: NULL arguments");
    if (a->nseq < 0 || a->ntok < 0 || a->nseq > 65535 || a->ntok > 65535)
        return vgx_fail(VGX_EINVAL, "vgx_draft_verify: nseq or ntok outside 0..65535");
    if (a->vocab <= 0 || a->vocab > (1 << 26)) return vgx_fail(VGX_EINVAL, "vgx_draft_verify: vocab outside 1..2^26");
    if (!kind_ok(a->kind)) return vgx_fail(VGX_EINVAL, "vgx_draft_verify: logits are f32, bf16, f16 or q16");
    if (a->nseq && (!a->qstart || !a->accepted || !a->next || !a->u_next))
        return vgx_fail(VGX_EINVAL, "vgx_draft_verify: NULL qstart, u_next or output");
    if (a->nseq && a->ntok && (!a->logits || !a->tokens || !a->u_accept))
        return vgx_fail(VGX_EINVAL, "vgx_draft_verify: NULL logits, tokens or u_accept");
    const int eb = a->kind == VGX_E_F32 ? 4 : 2;
    if (a->stride < a->vocab || (a->draft && a->draft_stride < a->vocab))
        return vgx_fail(VGX_EINVAL, "vgx_draft_verify: a row stride below vocab");
    if (((uintptr_t)a->logits | (uintptr_t)a->draft) & (eb - 1))
        return vgx_fail(VGX_EINVAL, "vgx_draft_verify: logits not aligned to their type");
    const size_t need = vgx_draft_verify_ws(a->nseq, a->ntok, a->vocab, a->kind, a->draft != nullptr);
    if (a->nseq && need && (!a->ws || a->ws_bytes < need || ((uintptr_t)a->ws & 15)))
        return vgx_fail(VGX_EINVAL, "vgx_draft_verify: the workspace is missing, too small or not 16-byte aligned");
    const Cut cut = cut_of(a->ntok, a->vocab, a->kind, a->draft != nullptr);
    if ((int64_t)cut.nch * a->ntok * (a->draft ? 2 : 1) >= (1 << 24) || (int64_t)cut.nch * a->nseq >= (1 << 23))
        return vgx_fail(VGX_ERANGE, "vgx_draft_verify: too many logits for one call");  // 2^32 threads
    if (!ctx) return vgx_fail(VGX_EINVAL, "vgx_draft_verify: no context");
    if (a->nseq == 0) return VGX_OK;
    VerifyArgs P{};
    P.nseq = a->nseq; P.ntok = a->ntok; P.vocab = a->vocab;
    P.qstart = a->qstart; P.tokens = a->tokens;
    P.x = static_cast<const uint8_t*>(a->logits);
    P.d = static_cast<const uint8_t*>(a->draft);
    P.xs = a->stride * eb; P.ds = a->draft_stride * eb;
    P.temp = a->temp; P.ua = a->u_accept; P.un = a->u_next;
    P.accepted = a->accepted; P.next = a->next; P.prob = a->prob;
    P.nch = cut.nch;
    P.chunk = cut.k * kThreads;
    P.px = static_cast<Part*>(a->ws);
    P.pd = P.px + (size_t)a->ntok * P.nch;
    P.w = reinterpret_cast<double*>(P.pd + (a->draft ? (size_t)a->ntok * P.nch : 0));
    VGX_HIP(hipSetDevice(ctx->device));
    switch (a->kind) {
        case VGX_E_F32: launch<VGX_E_F32>(P, cut.k, ctx->stream); break;
        case VGX_E_BF16: launch<VGX_E_BF16>(P, cut.k, ctx->stream); break;
        case VGX_E_F16: launch<VGX_E_F16>(P, cut.k, ctx->stream); break;
        default: launch<VGX_E_Q16>(P, cut.k, ctx->stream); break;
    }
    VGX_LAUNCH_CHECK("draft verify launch");
    return VGX_OK;
}

}  // extern "C"
