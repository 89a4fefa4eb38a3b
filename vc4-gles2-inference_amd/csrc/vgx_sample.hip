// A token of each row of logits, by temperature, top-k, top-p and min-p.
//
// The tokens that stay are the first in a ranking by value and index, so a cut
// is a place in it: (key, index), the key being the float's bits in an order of
// integers.  top-k's is found by counting, top-p's by summing weights, in three
// levels of a radix search; the draw then sums the weights of the tokens that
// stay in index order.
//
// Sums that are split at a place the data decides are taken in integers, which
// have no order: a weight is rounded to a multiple of 2^-q of the largest, q as
// large as the vocabulary's sum allows (2^-46 for 64402 tokens).  The tokens that
// stay under top-p < 1 weigh 2^-24 / vocab of the sum or more.
#include <algorithm>
#include <string>

#include "vgx_logits.h"

#pragma clang fp contract(off)

namespace {

typedef unsigned long long u64;

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
};

constexpr int kRow = 1024;    // threads of a row
constexpr int kBins = 2048;
constexpr int kMaxVocab = 1 << 21;

// The order of floats as unsigned integers (-0 as 0; never 0).
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// The tokens before a place in the ranking, and the one there.
struct Cut {
    unsigned key;
    int idx;
};
__device__ __forceinline__ bool stays(const Cut& c, unsigned key, int i) {
    return key > c.key || (key == c.key && i <= c.idx);
}
// A weight (0 .. 1) as a multiple of 2^-q, rounded to nearest: the low bits of a
// sum with 2^52.
__device__ __forceinline__ u64 fixed(double w, double scale) {
    return __builtin_bit_cast(u64, fma(w, scale, 4503599627370496.0)) - 0x4330000000000000ull;
}

struct RowShared {
    double tab[64];
    float m[kRow / 64];
    int a[kRow / 64];
    unsigned cnt[kBins];
    u64 sum[kBins];
    u64 wave[kRow / 64];
    int bin;
    u64 above, value;
    int idx;
};

// The running sum over the workgroup's threads; total: of all.
__device__ __forceinline__ u64 block_scan(u64 x, u64* sm, u64& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the last scan's sums are read
    if (lane == 63) sm[wave] = x;
    __syncthreads();
    u64 before = 0;
    total = 0;
    for (int w = 0; w < kRow / 64; ++w) {
        if (w < wave) before += sm[w];
        total += sm[w];
    }
    return x + before;
}

template <int KIND>
struct RowOf {
    static constexpr int N = kPer<KIND>;
    const SampleArgs& P;
    RowShared& H;
    Row q;
    int slabs;     // of kRow pieces
    Scale S;
    double scale;  // 2^q
    __device__ __forceinline__ RowOf(const SampleArgs& P_, RowShared& H_, int r)
        : P(P_), H(H_), q(row_at<KIND>(P_.x, P_.xs, r)), S{}, scale(__longlong_as_double((long long)(1023 + P_.q) << 52)) {
        slabs = (P.vocab + q.off + kRow * N - 1) / (kRow * N);
    }
    // f(x, index) of every token of a slab that is not masked
    template <class F>
    __device__ __forceinline__ void slab(int k, F f) const {
        const int g = k * kRow + (int)threadIdx.x;
        float x[N];
        piece<KIND>(q, P.vocab, g, x);
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (x[e] != -INFINITY) f(x[e], g * N - q.off + e);
    }
    __device__ __forceinline__ u64 weigh(float x) const { return fixed(weight(x, S, H.tab), scale); }

    // The index of the n-th token (1 ..) of a value, inside a cut.
    __device__ int nth(unsigned key, const Cut& in, u64 n) const {
        u64 before = 0;
        for (int k = 0; k < slabs; ++k) {
            u64 c = 0;
            slab(k, [&](float x, int i) {
                const unsigned y = key_of(x);
                c += y == key && stays(in, y, i);
            });
            u64 total;
            const u64 run = before + block_scan(c, H.wave, total);
            if (run >= n && run - c < n) {
                u64 left = n - (run - c);
                slab(k, [&](float x, int i) {
                    const unsigned y = key_of(x);
                    if (y == key && stays(in, y, i) && --left == 0) H.idx = i;
                });
            }
            before += total;
            if (before >= n) break;
        }
        __syncthreads();
        const int r = H.idx;
        __syncthreads();
        return r;
    }

    // The cut after `want` tokens of those inside `in`, or (WEIGHTED) after the
    // token at which the sum of weights reaches top_p of theirs.
    template <bool WEIGHTED>
    __device__ Cut select(const Cut& in, u64 want, double top_p) const {
        u64 before = 0, value = 0;
        unsigned prefix = 0;
        const int t = threadIdx.x;
#pragma unroll 1
        for (int level = 0; level < 3; ++level) {
            const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
            for (int i = t; i < kBins; i += kRow) { H.cnt[i] = 0; H.sum[i] = 0; }
            if (t == 0) H.bin = -1;
            __syncthreads();
            for (int k = 0; k < slabs; ++k)
                slab(k, [&](float x, int i) {
                    const unsigned y = key_of(x);
                    if (!stays(in, y, i) || (level && y >> (shift + bits) != prefix)) return;
                    const int b = y >> shift & ((1 << bits) - 1);
                    atomicAdd(&H.cnt[b], 1u);
                    if (WEIGHTED) {
                        const u64 w = weigh(x);
                        if (w) atomicAdd(&H.sum[b], w);
                    }
                });
            __syncthreads();
            // bins from the largest down, two a thread
            const int b0 = kBins - 1 - 2 * t;
            const u64 v0 = WEIGHTED ? H.sum[b0] : H.cnt[b0], v1 = WEIGHTED ? H.sum[b0 - 1] : H.cnt[b0 - 1];
            u64 total;
            const u64 run = block_scan(v0 + v1, H.wave, total), at = before + run - v0 - v1;
            if (WEIGHTED && level == 0) {
                const double y = ceil(top_p * (double)total);
                want = y < 1.0 ? 1 : (u64)y;
            }
            if (at < want && want <= before + run) {
                const bool low = want > at + v0;
                H.bin = low ? b0 - 1 : b0;
                H.above = low ? at + v0 : at;
                H.value = low ? v1 : v0;
            }
            __syncthreads();
            const int bin = H.bin;
            if (bin < 0) return in;  // fewer tokens than that
            before = H.above;
            value = H.value;
            prefix = prefix << bits | (unsigned)bin;
            if (level < 2) __syncthreads();
        }
        const u64 ties = H.cnt[prefix & 1023];
        __syncthreads();
        u64 n = want - before;
        if (WEIGHTED) {
            const u64 w = value / ties;  // (equal ones)
            n = (n + w - 1) / w;
        }
        if (n >= ties) return Cut{prefix, prefix == in.key ? in.idx : 0x7fffffff};
        return Cut{prefix, nth(prefix, in, n)};
    }
};

template <int KIND>
__global__ void __launch_bounds__(kRow) sample_kernel(const SampleArgs P) {
    __shared__ RowShared H;
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    RowOf<KIND> R(P, H, r);
    fill_table(H.tab);
    float m = -INFINITY;
    int a = 0x7fffffff;
    for (int k = 0; k < R.slabs; ++k)
        R.slab(k, [&](float x, int i) {
            if (x > m) { m = x; a = i; }
        });
    wave_best(m, a);
    if (lane == 0) { H.m[wave] = m; H.a[wave] = a; }
    __syncthreads();
    m = H.m[0];
    a = H.a[0];
    for (int w = 1; w < kRow / 64; ++w)
        if (H.m[w] > m || (H.m[w] == m && H.a[w] < a)) { m = H.m[w]; a = H.a[w]; }
    const float T = P.temp ? P.temp[r] : 1.0f;
    const int top_k = P.top_k ? P.top_k[r] : 0;
    const float top_p = P.top_p ? P.top_p[r] : 1.0f;
    const float min_p = P.min_p ? P.min_p[r] : 0.0f;
    const bool none = m == -INFINITY;
    if (none || !(T > 0.0f) || top_k == 1 || top_p <= 0.0f) {
        if (t == 0) {
            P.token[r] = none ? -1 : a;
            if (P.kept) P.kept[r] = !none;
            if (P.prob) P.prob[r] = none ? 0.0f : 1.0f;
        }
        return;
    }
    R.S = scale_of(m, fmin(1.0 / (double)T, 1e30));
    Cut cut{0, 0x7fffffff};
    if (top_k > 0 && top_k < P.vocab) cut = R.template select<false>(cut, (u64)top_k, 0.0);
    if (top_p < 1.0f) cut = R.template select<true>(cut, 0, (double)top_p);
    const double least = min_p > 0.0f ? fmin((double)min_p, 1.0) : 0.0;
    // the slabs' sums, and how many tokens stay
    __shared__ u64 part[kMaxVocab / (kRow * 4) + 2];
    __shared__ unsigned kept;
    __shared__ int pick, last, found;
    __shared__ u64 left;
    __shared__ float lx;
    for (int k = t; k < R.slabs; k += kRow) part[k] = 0;
    if (t == 0) { kept = 0; found = 0x7fffffff; last = -1; }
    __syncthreads();
    unsigned n = 0;
    for (int k = 0; k < R.slabs; ++k) {
        u64 s = 0;
        R.slab(k, [&](float x, int i) {
            if (!stays(cut, key_of(x), i)) return;
            const double w = weight(x, R.S, H.tab);
            if (w < least) return;
            ++n;
            s += fixed(w, R.scale);
        });
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
        if (lane == 0 && s) atomicAdd(&part[k], s);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o, 64);
    if (lane == 0 && n) atomicAdd(&kept, n);
    __syncthreads();
    u64 sum = 0;
    for (int k = 0; k < R.slabs; ++k) sum += part[k];
    // (a draw of 1 or more, or no number, takes the last token)
    const double u = P.u[r];
    const u64 want = u >= 0.0 && u < 1.0 ? min((u64)(u * (double)sum), sum - 1) : u < 0.0 ? 0 : sum - 1;
    u64 before = 0;
    int k = 0;
    while (before + part[k] <= want) before += part[k++];
    u64 s = 0;
    auto each = [&](auto f) {
        R.slab(k, [&](float x, int i) {
            if (!stays(cut, key_of(x), i)) return;
            const double w = weight(x, R.S, H.tab);
            if (w >= least) f(x, i, fixed(w, R.scale));
        });
    };
    each([&](float, int, u64 w) { s += w; });
    u64 total;
    u64 run = before + block_scan(s, H.wave, total) - s;
    if (run <= want && want < run + s)
        each([&](float x, int i, u64 w) {
            if (run <= want && want < run + w) { found = i; lx = x; }
            run += w;
        });
    __syncthreads();
    if (t == 0) {
        P.token[r] = found;
        if (P.kept) P.kept[r] = (int)kept;
        if (P.prob) P.prob[r] = (float)(weight(lx, R.S, H.tab) / ((double)sum / R.scale));
    }
}

bool kind_ok(int k) { return k == VGX_E_F32 || k == VGX_E_BF16 || k == VGX_E_F16 || k == VGX_E_Q16; }

}  // namespace

extern "C" {

size_t vgx_sample_ws(int nrows, int vocab, int kind) { return 0; }

int vgx_sample(vgx_ctx* ctx, const vgx_sampling* a) {
    auto fail = [](int status, const char* what) { return vgx_fail(status, std::string("vgx_sample: ") + what); };
    if (!a) return fail(VGX_EINVAL, "NULL arguments");
    if (a->nrows < 0 || a->nrows > (1 << 20)) return fail(VGX_EINVAL, "nrows outside 0..2^20");
    if (a->vocab <= 0 || a->vocab > kMaxVocab) return fail(VGX_EINVAL, "vocab outside 1..2^21");
    if (!kind_ok(a->kind)) return fail(VGX_EINVAL, "logits are f32, bf16, f16 or q16");
    if (a->nrows && (!a->logits || !a->u || !a->token)) return fail(VGX_EINVAL, "NULL logits, u or token");
    const int eb = a->kind == VGX_E_F32 ? 4 : 2;
    if (a->stride < a->vocab || a->stride > ((int64_t)1 << 40)) return fail(VGX_EINVAL, "a row stride below vocab or above 2^40");
    if ((uintptr_t)a->logits & (eb - 1)) return fail(VGX_EINVAL, "logits not aligned to their type");
    const size_t need = vgx_sample_ws(a->nrows, a->vocab, a->kind);
    if (need && (!a->ws || a->ws_bytes < need || ((uintptr_t)a->ws & 15)))
        return fail(VGX_EINVAL, "the workspace is missing, too small or not 16-byte aligned");
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
    VGX_HIP(hipSetDevice(ctx->device));
    void (*fn)(const SampleArgs) = a->kind == VGX_E_F32    ? sample_kernel<VGX_E_F32>
                                   : a->kind == VGX_E_BF16 ? sample_kernel<VGX_E_BF16>
                                   : a->kind == VGX_E_F16  ? sample_kernel<VGX_E_F16>
                                                           : sample_kernel<VGX_E_Q16>;
    hipLaunchKernelGGL(fn, dim3(a->nrows), dim3(kRow), 0, ctx->stream, P);
    VGX_LAUNCH_CHECK("sample launch");
    return VGX_OK;
}

}  // extern "C"
