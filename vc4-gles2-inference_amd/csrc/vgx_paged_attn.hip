// Attention of a ragged batch's new tokens over a paged cache.
//
// Formulas.  For one sequence and KV head the queries are the columns of Q^T
// (row r of the sequence's new tokens, head u of the group: column r * grp +
// u).  Per tile of keys
//   S^T = K Q^T        32x32x16 MFMA, A = K rows, B = Q columns
//   m' = max(m, max_keys S), P = exp2(c S - c m'), l = l 2^(c(m - m')) + sum P
//   O^T = O^T 2^(c(m - m')) + V^T P    A = V^T, B = P
// with c = scale * log2(e); out = O / l.  Products in the compute type with
// 32-bit sums; P is rounded to it (relative error at most half a step a
// weight, as the inputs' own); m, l and O stay in 32 bits.
//
// Why transposed: a 32x32 product leaves column q's scores in lanes q and
// q + 32 (keys 8a + 4h + b in register 4a + b of half h), which is a B operand
// of the next product when its key order is taken as (4h + b, 8 + 4h + b): P
// never leaves the registers, a row's statistics are one lane's and its
// partner's, and the running scale is one multiply a register.  V^T in that
// order is two 64-bit transposing LDS reads a fragment.
#include <algorithm>
#include <cmath>
#include <string>

#include "vgx_paged.h"

#pragma clang fp contract(off)

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
    PagedDev A;
    const uint8_t* q;
    int64_t qstride;
    float c;       // scale * log2(e), the K step included: exponents of 2
    float scale;   // scale with the K step: scores
    int window;
    int split_len, nsplit;
    int out_q16;
    uint8_t* out;
    int64_t ostride;
    float* lse;
    float* po;     // nsplit x ntok x heads x hd partial sums
    float* pml;    // nsplit x ntok x heads x (m, l)
    int tm;        // columns of a tile (what combine needs to find a row's span)
};

template <int CK>
__device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
    if constexpr (CK == VGX_E_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}
template <int CK>
__device__ __forceinline__ short to_ct(float x) {
    if constexpr (CK == VGX_E_BF16) return __builtin_bit_cast(short, (bf16_t)x);
    else return __builtin_bit_cast(short, (f16_t)x);
}
template <int CK>
__device__ __forceinline__ float from_ct(short x) {
    if constexpr (CK == VGX_E_BF16) return __uint_as_float((unsigned)(unsigned short)x << 16);
    else return (float)__builtin_bit_cast(f16_t, x);
}
// Four cache bytes as two pairs of half floats, exact: 0x6400 | (b ^ 0x80) is
// 1024 + 128 + b.
__device__ __forceinline__ uint2 q8_to_f16(unsigned w) {
    const unsigned u = w ^ 0x80808080u;
    const unsigned a = __builtin_amdgcn_perm(0x64646464u, u, 0x05010500u);
    const unsigned b = __builtin_amdgcn_perm(0x64646464u, u, 0x05030502u);
    const f16x2 off = {(f16_t)-1152.0f, (f16_t)-1152.0f};
    uint2 r;
    r.x = __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, a) + off);
    r.y = __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, b) + off);
    return r;
}
// Whether a word of two 16-bit floats holds an infinity or NaN.
template <int CK>
__device__ __forceinline__ bool odd16(unsigned w) {
    constexpr unsigned e = CK == VGX_E_BF16 ? 0x7f80u : 0x7c00u;
    return (w & e) == e || (w & (e << 16)) == (e << 16);
}
// LDS written by the wave's lanes, then read by others of the same wave.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// max / sum of a lane and its partner in the other half of the wave.
__device__ __forceinline__ float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// A tile of keys in LDS.  K rows of HD values with 16 bytes between them (a
// lane's 16-byte pieces of 8 rows then lie in 8 different bank groups); V rows
// a pitch of 64 mod 128 bytes, so the 4 rows x 64 bytes that half a
// transposing read takes cover the 64 banks once.
template <int HD>
struct Geo {
    static constexpr int pk = HD * 2 + 16;
    static constexpr int pv = (HD * 2 + 63) / 128 * 128 + 64;
};
static_assert(Geo<64>::pv == 192 && Geo<96>::pv == 192 && Geo<128>::pv == 320 && Geo<256>::pv == 576, "");

// Staging of ROWS keys by THREADS threads: NL 16-byte pieces a thread of K and
// as many of V.  Lane r of a wave holds the page of row r % ROWS.
template <int KIND, int HD, bool EX, int ROWS, int THREADS>
struct Stage {
    static constexpr int CK = KIND == VGX_E_BF16 ? VGX_E_BF16 : VGX_E_F16;
    static constexpr int EB = KIND == VGX_E_Q8 ? 1 : 2;
    static constexpr int CPR = HD * EB / 16;  // pieces of a row
    static constexpr int NL = (ROWS * CPR + THREADS - 1) / THREADS;
    uint4 k[NL], v[NL];

    // The page of row j0 + lane % ROWS (the last row before `end` stands in
    // for those behind); a page outside the pool counts as page 0, with the
    // fault recorded.
    static __device__ __forceinline__ int page(const PagedDev& A, const int* tab, int j0, int end) {
        const int j = min(j0 + (int)(threadIdx.x & (ROWS - 1)), end - 1);
        int pg = tab[page_of(A, j)];
        if (pg < 0 || pg >= A.npages) {
            set_fault(A, VGX_FAULT_PAGE);
            pg = 0;
        }
        return pg;
    }
    // One of K and V (VALUE): a V row behind the end is zeros, whatever the
    // page holds there; a K row there is the last one again (its scores are
    // masked).
    template <bool VALUE>
    static __device__ __forceinline__ void load1(const PagedDev& A, const uint8_t* base, int pg, int j0, int end,
                                                 int tid, uint4 (&w)[NL]) {
        const int64_t ps = VALUE ? A.vpg : A.kpg, rs = VALUE ? A.vrow : A.krow;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int sl = i * THREADS + tid;
            const int row = sl / CPR, ch = sl - row * CPR;
            const int p = __shfl(pg, row & (ROWS - 1), 64);
            const bool use = (NL * THREADS == ROWS * CPR || row < ROWS) && (EX || ch * 16 < A.hd * EB);
            const int j = min(j0 + row, end - 1);
            const int slot = j - page_of(A, j) * A.psize;
            w[i] = make_uint4(0, 0, 0, 0);
            if (use && (!VALUE || j0 + row < end))
                w[i] = *reinterpret_cast<const uint4*>(base + (int64_t)p * ps + (int64_t)slot * rs + ch * 16);
        }
    }
    __device__ __forceinline__ void load(const PagedDev& A, const uint8_t* kh, const uint8_t* vh, int pg, int j0,
                                         int end, int tid) {
        load1<false>(A, kh, pg, j0, end, tid, k);
        load1<true>(A, vh, pg, j0, end, tid, v);
    }
    static __device__ __forceinline__ bool odd1(const uint4 (&w)[NL]) {
        bool r = false;
        if (KIND != VGX_E_Q8)
#pragma unroll
            for (int i = 0; i < NL; ++i)
                r = r || odd16<CK>(w[i].x) || odd16<CK>(w[i].y) || odd16<CK>(w[i].z) || odd16<CK>(w[i].w);
        return r;
    }
    __device__ __forceinline__ bool odd() const { return odd1(v); }
    static __device__ __forceinline__ void put(uint8_t* p, const uint4& w) {
        if (KIND == VGX_E_Q8) {
            const uint2 a = q8_to_f16(w.x), b = q8_to_f16(w.y), c = q8_to_f16(w.z), d = q8_to_f16(w.w);
            reinterpret_cast<uint4*>(p)[0] = make_uint4(a.x, a.y, b.x, b.y);
            reinterpret_cast<uint4*>(p)[1] = make_uint4(c.x, c.y, d.x, d.y);
        } else {
            *reinterpret_cast<uint4*>(p) = w;
        }
    }
    static __device__ __forceinline__ void store1(uint8_t* l, int pitch, int tid, const uint4 (&w)[NL]) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int sl = i * THREADS + tid;
            const int row = sl / CPR, ch = sl - row * CPR;
            if (NL * THREADS == ROWS * CPR || row < ROWS) put(l + row * pitch + ch * (32 / EB), w[i]);
        }
    }
    __device__ __forceinline__ void store(uint8_t* lk, uint8_t* lv, int tid) const {
        store1(lk, Geo<HD>::pk, tid, k);
        store1(lv, Geo<HD>::pv, tid, v);
    }
    // Load and store in one go, K then V through the same registers (heads of
    // more than 128 values leave none for a tile ahead); V's odd() comes back.
    static __device__ __forceinline__ bool fetch(const PagedDev& A, const uint8_t* kh, const uint8_t* vh, int pg,
                                                 int j0, int end, int tid, uint8_t* lk, uint8_t* lv) {
        uint4 w[NL];
        load1<false>(A, kh, pg, j0, end, tid, w);
        store1(lk, Geo<HD>::pk, tid, w);
        load1<true>(A, vh, pg, j0, end, tid, w);
        store1(lv, Geo<HD>::pv, tid, w);
        return odd1(w);
    }
};

// The running state of a wave's 32 columns.
template <int HD>
struct Acc {
    static constexpr int NB = HD / 32;
    f32x16 o[NB];
    float m, l;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
        m = -INFINITY;
        l = 0.0f;
    }
};

// The query columns as B operands: k-step t of column lane % 32 holds values
// 16 t + 8 (lane / 32) .. + 7.
template <int HD, bool EX>
__device__ __forceinline__ void load_q(const PagedDev& A, const uint8_t* qp, bool valid, s16x8 (&q)[HD / 16]) {
    const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (valid && (EX || 16 * t < A.hd)) w = *reinterpret_cast<const uint4*>(qp + (16 * t + 8 * h) * 2);
        q[t] = __builtin_bit_cast(s16x8, w);
    }
}

// One step over 32 * KB keys in LDS (lk, lv: the first row), the first of them
// key j0.  mask: some column does not see some key; vlo <= key < vhi are the
// lane's column's.  odd: an infinity or NaN among V (checked where mask is
// set): 0 * inf would reach the rows that do not see it, so the weighted sum
// then runs key by key over the visible ones (lp: a free LDS area of 4 KB
// a wave).
template <int CK, int HD, bool EX, int KB>
__device__ __forceinline__ void step(const PagedDev& A, const s16x8 (&q)[HD / 16], Acc<HD>& a, const uint8_t* lk,
                                     const uint8_t* lv, int j0, float c, bool mask, int vlo, int vhi, bool odd,
                                     float* lp) {
    const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
    f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) {
            if (!EX && 16 * t >= A.hd) continue;
            const s16x8 kf = *reinterpret_cast<const s16x8*>(lk + (kb * 32 + col) * Geo<HD>::pk + (2 * t + h) * 16);
            s[kb] = mfma<CK>(kf, q[t], s[kb]);
        }
    }
    if (mask) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = j0 + kb * 32 + 8 * (i / 4) + 4 * h + (i & 3);
                s[kb][i] = j >= vlo && j < vhi ? s[kb][i] : -INFINITY;
            }
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = fmaxf(half_max(mx), a.m);
    // (no key yet: subtract 0, so the exponents stay -inf and the weights 0)
    const float mc = (mx == -INFINITY ? 0.0f : mx) * c;
    const float alpha = exp2_(fmaf(a.m, c, -mc));
    a.m = mx;
    float sum = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[kb][i] = exp2_(fmaf(s[kb][i], c, -mc));
            sum += s[kb][i];
        }
    a.l = fmaf(a.l, alpha, sum);
#pragma unroll
    for (int b = 0; b < HD / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) a.o[b][i] *= alpha;
    if (odd) {
#pragma unroll 1
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float p = s[0][i];
#pragma unroll
                for (int u = 1; u < KB; ++u) p = kb == u ? s[u][i] : p;
                lp[(8 * (i / 4) + 4 * h + (i & 3)) * 32 + col] = p;
            }
            wave_sync();
            for (int r = 0; r < 32; ++r) {
                const int j = j0 + kb * 32 + r;
                const float p = lp[r * 32 + col];
                if (j >= vlo && j < vhi) {
#pragma unroll
                    for (int b = 0; b < HD / 32; ++b)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const s16x4 w = *reinterpret_cast<const s16x4*>(lv + (kb * 32 + r) * Geo<HD>::pv +
                                                                            (32 * b + 8 * g + 4 * h) * 2);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                a.o[b][4 * g + e] = fmaf(p, from_ct<CK>(w[e]), a.o[b][4 * g + e]);
                        }
                }
            }
            wave_sync();
        }
        return;
    }
    // lane 16 g + i's address: key row i / 4 of the half, dims 16 (g & 1) + 4 (i & 3)
    const int i16 = lane & 15;
    const uint8_t* vb = lv + (4 * h + (i16 >> 2)) * Geo<HD>::pv + (16 * ((lane >> 4) & 1) + 4 * (i16 & 3)) * 2;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s16x8 pf;
#pragma unroll
            for (int i = 0; i < 8; ++i) pf[i] = to_ct<CK>(s[kb][8 * t + i]);
#pragma unroll
            for (int b = 0; b < HD / 32; ++b) {
                if (!EX && 32 * b >= A.hd) continue;
                const uint8_t* p = vb + (kb * 32 + 16 * t) * Geo<HD>::pv + 64 * b;
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
                const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * Geo<HD>::pv));
                const s16x8 vf = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                a.o[b] = mfma<CK>(vf, pf, a.o[b]);
            }
        }
}

// Four values of one output row: dims d .. d+3.
template <int CK>
__device__ __forceinline__ void put_out(const AttnArgs& P, int64_t row, int head, int d, float4 v) {
    uint8_t* p = P.out + ((int64_t)row * P.ostride + (int64_t)head * P.A.hd + d) * 2;
    unsigned w[2];
    if (P.out_q16) {
        const float x[4] = {v.x, v.y, v.z, v.w};
        int z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float f = floorf(fmaf(x[e], 256.0f, 0.5f));
            f = fminf(fmaxf(f, -32768.0f), 32767.0f);
            z[e] = x[e] == x[e] ? (int)f : 0;
        }
        w[0] = (unsigned)(z[0] & 0xffff) | (unsigned)z[1] << 16;
        w[1] = (unsigned)(z[2] & 0xffff) | (unsigned)z[3] << 16;
    } else {
        w[0] = (unsigned)(unsigned short)to_ct<CK>(v.x) | (unsigned)(unsigned short)to_ct<CK>(v.y) << 16;
        w[1] = (unsigned)(unsigned short)to_ct<CK>(v.z) | (unsigned)(unsigned short)to_ct<CK>(v.w) << 16;
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}
__device__ __forceinline__ float lse_of(const AttnArgs& P, float m, float l) {
    return l > 0.0f || l != l ? fmaf(m, P.scale, logf(l)) : -INFINITY;
}
__device__ __forceinline__ float inv_l(const AttnArgs& P, float l) {
    return l == 0.0f ? 0.0f : P.A.vstep / l;
}

// A column's place: row of the batch, query head, position, what it sees.
struct Col {
    bool valid;
    int row, head, vlo, vhi;
};
__device__ __forceinline__ Col col_of(const AttnArgs& P, const SeqAt& q, int h, int m, int end) {
    Col r;
    r.valid = m < q.n * P.A.grp;
    const int i = m / P.A.grp;
    r.row = q.q0 + i;
    r.head = h * P.A.grp + (m - i * P.A.grp);
    const int pos = q.kv - q.n + i;
    r.vhi = r.valid ? min(pos + 1, end) : 0;
    r.vlo = P.window > 0 ? pos - P.window + 1 : 0;
    return r;
}

// Few rows a sequence (max_q * grp <= 32): a workgroup is one sequence, KV
// head and split; its 4 waves hold the same 32 columns and take tiles of 32
// keys in turn, each through LDS of its own without a barrier, and join at
// the end.
template <int KIND, int HD, bool EX>
__global__ void __launch_bounds__(256) paged_rows_kernel(const AttnArgs P) {
    using St = Stage<KIND, HD, EX, 32, 64>;
    constexpr int CK = St::CK;
    constexpr int kWave = 32 * (Geo<HD>::pk + Geo<HD>::pv);
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float sm[4][32], sl[4][32];
    const PagedDev& A = P.A;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31;
    const int s = blockIdx.x / A.kvh, h = blockIdx.x - s * A.kvh;
    const SeqAt q = seq_at(A, s);
    if (!q.ok && threadIdx.x == 0) set_fault(A, VGX_FAULT_LENGTH);
    if (q.n <= 0) return;
    const Span sp = span_of(q, 0, q.n - 1, P.window, P.split_len);
    const int split = blockIdx.y;
    if (split >= sp.nsp) return;
    const int start = sp.lo + split * P.split_len, end = min(sp.hi, start + P.split_len);
    const Col cl = col_of(P, q, h, col, end);
    s16x8 qf[HD / 16];
    load_q<HD, EX>(A, P.q + ((int64_t)cl.row * P.qstride + (int64_t)cl.head * A.hd) * 2, cl.valid, qf);
    uint8_t* lk = smem + wave * kWave;
    uint8_t* lv = lk + 32 * Geo<HD>::pk;
    const uint8_t* kh = A.k + (int64_t)h * A.khd;
    const uint8_t* vh = A.v + (int64_t)h * A.vhd;
    const int* tab = A.table + (int64_t)s * A.tstride;
    // keys every column sees: [all_lo, all_hi)
    const int all_hi = min(q.kv - q.n + 1, end);
    const int all_lo = P.window > 0 ? q.kv - P.window : 0;
    Acc<HD> a;
    a.clear();
    St st;
    int j0 = start + wave * 32;
    int pg = j0 < end ? St::page(A, tab, j0, end) : 0;
    if (HD <= 128 && j0 < end) st.load(A, kh, vh, pg, j0, end, lane);
    int pn = j0 + 128 < end ? St::page(A, tab, j0 + 128, end) : 0;
    while (j0 < end) {
        const bool mask = j0 + 32 > all_hi || j0 < all_lo;
        bool odd;
        wave_sync();
        if (HD <= 128) {
            odd = mask && __any(st.odd());
            st.store(lk, lv, lane);
        } else {
            odd = __any(St::fetch(A, kh, vh, pg, j0, end, lane, lk, lv)) && mask;
        }
        const int jn = j0 + 128;
        if (jn < end) {
            if (HD <= 128) st.load(A, kh, vh, pn, jn, end, lane);
            pg = pn;
            if (jn + 128 < end) pn = St::page(A, tab, jn + 128, end);
        }
        wave_sync();
        step<CK, HD, EX, 1>(A, qf, a, lk, lv, j0, P.c, mask, cl.vlo, cl.vhi, odd, reinterpret_cast<float*>(lk));
        j0 = jn;
    }
    // the waves' sums on a common maximum, joined in wave order
    const float l = half_sum(a.l);
    if (lane < 32) { sm[wave][col] = a.m; sl[wave][col] = l; }
    __syncthreads();
    float M = sm[0][col];
#pragma unroll
    for (int w = 1; w < 4; ++w) M = fmaxf(M, sm[w][col]);
    const float mc = (M == -INFINITY ? 0.0f : M) * P.c;
    float L = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) L = fmaf(sl[w][col], exp2_(fmaf(sm[w][col], P.c, -mc)), L);
    const float f = exp2_(fmaf(a.m, P.c, -mc));
    float* part = reinterpret_cast<float*>(smem + wave * kWave);
    const int hh = lane >> 5;
#pragma unroll
    for (int b = 0; b < HD / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(32 * b + 8 * (i / 4) + 4 * hh + (i & 3)) * 32 + col] = a.o[b][i] * f;
    __syncthreads();
    if (!cl.valid) return;
    // thread: column lane % 32, every eighth group of 4 dims
    const int64_t at = ((int64_t)split * A.ntok + cl.row) * A.heads + cl.head;
    const bool whole = sp.nsp == 1;
    const float r = whole ? inv_l(P, L) : 1.0f;
    for (int d = 4 * (threadIdx.x >> 5); d < A.hd; d += 32) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) x[e] += reinterpret_cast<const float*>(smem + w * kWave)[(d + e) * 32 + col];
            x[e] *= r;
        }
        const float4 v = make_float4(x[0], x[1], x[2], x[3]);
        if (whole) put_out<CK>(P, cl.row, cl.head, d, v);
        else *reinterpret_cast<float4*>(P.po + at * A.hd + d) = v;
    }
    if (threadIdx.x < 32) {
        if (!whole) {
            P.pml[2 * at] = M;
            P.pml[2 * at + 1] = L;
        } else if (P.lse) {
            P.lse[(int64_t)cl.row * A.heads + cl.head] = lse_of(P, M, L);
        }
    }
}

// The sequence and place of a tile of tm columns, tiles counted through the
// batch: false past the last.  Every lane of the wave is active.
__device__ __forceinline__ bool tile_at(const PagedDev& A, int tm, int tile, int& s, int& local) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b = 0; b < A.nseq; b += 64) {
        const int j = b + lane;
        const int n = j < A.nseq ? seq_at(A, j).n : 0;
        const int cnt = (int)(((int64_t)n * A.grp + tm - 1) / tm);
        int sum = cnt;  // the running sum over the lanes
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(sum, o, 64);
            if (lane >= o) sum += y;
        }
        const unsigned long long past = __ballot(base + sum > tile);
        if (past) {
            const int l = __ffsll(past) - 1;
            s = b + l;
            local = tile - (base + __shfl(sum, l, 64) - __shfl(cnt, l, 64));
            return true;
        }
        base += __shfl(sum, 63, 64);
    }
    return false;
}

// Many rows a sequence: a workgroup is a tile of 128 columns (4 waves x 32) of
// one KV head; the waves share tiles of 64 keys.
template <int KIND, int HD, bool EX>
__global__ void __launch_bounds__(256) paged_tile_kernel(const AttnArgs P) {
    constexpr int ROWS = 64;
    using St = Stage<KIND, HD, EX, ROWS, 256>;
    constexpr int CK = St::CK;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int any_odd;
    const PagedDev& A = P.A;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31;
    const int tile = blockIdx.x / A.kvh, h = blockIdx.x - tile * A.kvh;
    int s, local;
    if (!tile_at(A, 128, tile, s, local)) return;
    const SeqAt q = seq_at(A, s);
    if (!q.ok && threadIdx.x == 0) set_fault(A, VGX_FAULT_LENGTH);
    const int m0 = local * 128, m1 = min(m0 + 128, q.n * A.grp) - 1;
    const Span sp = span_of(q, m0 / A.grp, m1 / A.grp, P.window, P.split_len);
    const int split = blockIdx.y;
    if (split >= sp.nsp) return;
    const int start = sp.lo + split * P.split_len, end = min(sp.hi, start + P.split_len);
    const Col cl = col_of(P, q, h, m0 + wave * 32 + col, end);
    s16x8 qf[HD / 16];
    load_q<HD, EX>(A, P.q + ((int64_t)cl.row * P.qstride + (int64_t)cl.head * A.hd) * 2, cl.valid, qf);
    // the wave's rows: keys every column sees, and keys any column sees
    const int w0 = m0 + wave * 32, w1 = min(w0 + 31, m1);
    const bool any = w0 <= m1;
    const int base = q.kv - q.n;
    const int r0 = w0 / A.grp, r1 = w1 / A.grp;
    const int all_hi = min(base + r0 + 1, end), any_hi = any ? min(base + r1 + 1, end) : 0;
    const int all_lo = P.window > 0 ? base + r1 - P.window + 1 : 0;
    const int any_lo = P.window > 0 ? base + r0 - P.window + 1 : 0;
    uint8_t* lk = smem;
    uint8_t* lv = smem + ROWS * Geo<HD>::pk;
    float* lp = reinterpret_cast<float*>(smem + ROWS * (Geo<HD>::pk + Geo<HD>::pv)) + wave * 1024;
    const uint8_t* kh = A.k + (int64_t)h * A.khd;
    const uint8_t* vh = A.v + (int64_t)h * A.vhd;
    const int* tab = A.table + (int64_t)s * A.tstride;
    Acc<HD> a;
    a.clear();
    St st;
    if (threadIdx.x == 0) any_odd = 0;
    int pg = start < end ? St::page(A, tab, start, end) : 0;
    if (HD <= 128 && start < end) st.load(A, kh, vh, pg, start, end, threadIdx.x);
    int pn = start + ROWS < end ? St::page(A, tab, start + ROWS, end) : 0;
    // tiles of keys that some column of the workgroup does not wholly see
    const int tile_hi = min(base + m0 / A.grp + 1, end);
    const int tile_lo = P.window > 0 ? base + m1 / A.grp - P.window + 1 : 0;
    for (int j0 = start; j0 < end; j0 += ROWS) {
        const bool wide = j0 + ROWS > tile_hi || j0 < tile_lo;
        __syncthreads();  // the last tile's reads are done
        if (HD <= 128) {
            if (wide && st.odd()) any_odd = 1;
            st.store(lk, lv, threadIdx.x);
        } else if (St::fetch(A, kh, vh, pg, j0, end, threadIdx.x, lk, lv) && wide) {
            any_odd = 1;
        }
        __syncthreads();
        const bool odd = wide && any_odd;
        const int jn = j0 + ROWS;
        if (jn < end) {
            if (HD <= 128) st.load(A, kh, vh, pn, jn, end, threadIdx.x);
            pg = pn;
            if (jn + ROWS < end) pn = St::page(A, tab, jn + ROWS, end);
        }
        if (j0 < any_hi && j0 + ROWS > any_lo) {
            const bool mask = j0 + ROWS > all_hi || j0 < all_lo;
            step<CK, HD, EX, 2>(A, qf, a, lk, lv, j0, P.c, mask, cl.vlo, cl.vhi, odd && mask, lp);
        }
    }
    const float L = half_sum(a.l);
    if (!cl.valid) return;
    const int hh = lane >> 5;
    const int64_t at = ((int64_t)split * A.ntok + cl.row) * A.heads + cl.head;
    const bool whole = sp.nsp == 1;
    const float r = whole ? inv_l(P, L) : 1.0f;
#pragma unroll
    for (int b = 0; b < HD / 32; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * b + 8 * g + 4 * hh;
            if (!EX && d >= A.hd) continue;
            const float4 v = make_float4(a.o[b][4 * g] * r, a.o[b][4 * g + 1] * r, a.o[b][4 * g + 2] * r,
                                         a.o[b][4 * g + 3] * r);
            if (whole) put_out<CK>(P, cl.row, cl.head, d, v);
            else *reinterpret_cast<float4*>(P.po + at * A.hd + d) = v;
        }
    if (hh == 0) {
        if (!whole) {
            P.pml[2 * at] = a.m;
            P.pml[2 * at + 1] = L;
        } else if (P.lse) {
            P.lse[(int64_t)cl.row * A.heads + cl.head] = lse_of(P, a.m, L);
        }
    }
}

// Joins a row's splits, in split order: a wave a row and head.
template <int CK>
__global__ void __launch_bounds__(256) paged_join_kernel(const AttnArgs P) {
    const PagedDev& A = P.A;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = (int)(w / A.heads), head = (int)(w - (int64_t)t * A.heads);
    if (t >= A.ntok) return;
    const int lane = threadIdx.x & 63;
    const int s = seq_of_row(A, t);
    if (s >= A.nseq) return;
    const SeqAt q = seq_at(A, s);
    const int i = t - q.q0;
    if (i < 0 || i >= q.n) return;
    // the row's tile, as the kernels cut it
    const int m = i * A.grp + head % A.grp;
    const int m0 = m / P.tm * P.tm, m1 = min(m0 + P.tm, q.n * A.grp) - 1;
    const Span sp = span_of(q, m0 / A.grp, m1 / A.grp, P.window, P.split_len);
    if (sp.nsp == 1) return;
    const int64_t step = (int64_t)A.ntok * A.heads, at = (int64_t)t * A.heads + head;
    float M = -INFINITY;
    for (int k = 0; k < sp.nsp; ++k) M = fmaxf(M, P.pml[2 * (at + k * step)]);
    const float mc = (M == -INFINITY ? 0.0f : M) * P.c;
    float L = 0.0f;
    const int d = lane * 4;
    float4 o = make_float4(0, 0, 0, 0);
    for (int k = 0; k < sp.nsp; ++k) {
        const float f = exp2_(fmaf(P.pml[2 * (at + k * step)], P.c, -mc));
        L = fmaf(P.pml[2 * (at + k * step) + 1], f, L);
        if (d < A.hd) {
            const float4 x = *reinterpret_cast<const float4*>(P.po + (at + k * step) * A.hd + d);
            o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w);
        }
    }
    const float r = inv_l(P, L);
    if (d < A.hd) put_out<CK>(P, t, head, d, make_float4(o.x * r, o.y * r, o.z * r, o.w * r));
    if (lane == 0 && P.lse) P.lse[at] = lse_of(P, M, L);
}

typedef void (*AttnFn)(const AttnArgs);
struct Plan {
    AttnFn fn;
    int lds, tm;
    int64_t wgs;       // workgroups of one split
    int split_len, nsplit;
    size_t ws;
};

template <int KIND, int HD, bool EX>
void fn_of(bool rows, Plan& p) {
    const int row = Geo<HD>::pk + Geo<HD>::pv;
    p.fn = rows ? paged_rows_kernel<KIND, HD, EX> : paged_tile_kernel<KIND, HD, EX>;
    p.lds = rows ? 4 * 32 * row : 64 * row + 4 * 4096;
}
template <int KIND>
void fn_of(int hd, bool rows, Plan& p) {
    switch (hd) {
        case 64: return fn_of<KIND, 64, true>(rows, p);
        case 96: return fn_of<KIND, 96, true>(rows, p);
        case 128: return fn_of<KIND, 128, true>(rows, p);
        case 256: return fn_of<KIND, 256, true>(rows, p);
    }
    return hd < 128 ? fn_of<KIND, 128, false>(rows, p) : fn_of<KIND, 256, false>(rows, p);
}

Plan plan_of(const PagedDev& A, int kind, int window, int num_cu) {
    Plan p{};
    const bool rows = (int64_t)A.max_q * A.grp <= 32;
    if (kind == VGX_E_BF16) fn_of<VGX_E_BF16>(A.hd, rows, p);
    else if (kind == VGX_E_F16) fn_of<VGX_E_F16>(A.hd, rows, p);
    else fn_of<VGX_E_Q8>(A.hd, rows, p);
    p.tm = rows ? 32 : 128;
    // (a sequence with rows has at most rows * grp / tm + 1 tiles)
    const int64_t tiles = rows ? A.nseq : (int64_t)A.ntok * A.grp / p.tm + std::min(A.nseq, A.ntok);
    p.wgs = tiles * A.kvh;
    int64_t span = A.max_kv;
    if (window > 0) span = std::min<int64_t>(span, (int64_t)window + p.tm + 64);
    // enough workgroups for four a CU, splits of 256 keys or more
    const int64_t want = std::max<int64_t>(1, (int64_t)num_cu * 4 / p.wgs);
    int64_t len = (span + want - 1) / want;
    len = std::max<int64_t>((len + 255) / 256 * 256, 256);
    int64_t n = (span + len - 1) / len;
    p.split_len = (int)std::min<int64_t>(len, INT32_MAX / 2);
    p.nsplit = (int)std::max<int64_t>(n, 1);
    p.ws = p.nsplit > 1 ? (size_t)p.nsplit * A.ntok * A.heads * (A.hd + 2) * 4 : 0;
    return p;
}

}  // namespace

extern "C" {

size_t vgx_paged_attn_ws(vgx_ctx* ctx, const vgx_paged* cache, const vgx_ragged* batch, int window) {
    PagedDev A;
    if (vgx_paged_fill("vgx_paged_attn_ws", cache, batch, &A) != VGX_OK || !ctx || window < 0) return 0;
    if (A.ntok == 0 || A.nseq == 0) return 0;
    return plan_of(A, cache->kind, window, ctx->num_cu).ws;
}

int vgx_paged_attn(vgx_ctx* ctx, const vgx_paged* cache, const vgx_ragged* batch, const vgx_paged_query* r) {
    AttnArgs P{};
    const int st = vgx_paged_fill("vgx_paged_attn", cache, batch, &P.A);
    if (st != VGX_OK) return st;
    if (!r) return vgx_fail(VGX_EINVAL, "vgx_paged_attn: NULL query");
    const PagedDev& A = P.A;
    const int64_t width = (int64_t)A.heads * A.hd;
    if (r->q_stride < width || r->q_stride % 8 || r->out_stride < width || r->out_stride % 8)
        return vgx_fail(VGX_EINVAL, "vgx_paged_attn: a row stride below the width or not a multiple of 16 bytes");
    if (!(r->scale >= 0) || std::isinf(r->scale))
        return vgx_fail(VGX_EINVAL, "vgx_paged_attn: scale is negative or not a number");
    if (r->window < 0) return vgx_fail(VGX_EINVAL, "vgx_paged_attn: a negative window");
    if (r->out_kind != VGX_E_Q16 && r->out_kind != compute_kind(cache->kind))
        return vgx_fail(VGX_EINVAL, "vgx_paged_attn: out is the cache's compute type or q16");
    if (A.ntok && (!r->q || !r->out)) return vgx_fail(VGX_EINVAL, "vgx_paged_attn: NULL q or out");
    if (((uintptr_t)r->q | (uintptr_t)r->out | (uintptr_t)r->ws) & 15)
        return vgx_fail(VGX_EINVAL, "vgx_paged_attn: q, out or ws not 16-byte aligned");
    if (!ctx) return vgx_fail(VGX_EINVAL, "vgx_paged_attn: no context");
    if (A.ntok == 0 || A.nseq == 0) return VGX_OK;
    Plan p = plan_of(A, cache->kind, r->window, ctx->num_cu);
    if (p.nsplit > 1 && (!r->ws || r->ws_bytes < p.ws)) {
        p.nsplit = 1;
        p.split_len = INT32_MAX / 2;
    }
    if (p.wgs >= (1 << 24) || p.nsplit > 65535) return vgx_fail(VGX_ERANGE, "vgx_paged_attn: too many rows");
    P.q = static_cast<const uint8_t*>(r->q);
    P.qstride = r->q_stride;
    P.scale = (r->scale > 0 ? r->scale : 1.0f / std::sqrt((float)A.hd)) * A.kstep;
    P.c = P.scale * kLog2e;
    if (!(P.c > 1e-30f) || std::isinf(P.c))
        return vgx_fail(VGX_EINVAL, "vgx_paged_attn: scale times the K step outside 1e-30 .. 1e38");
    P.window = r->window;
    P.split_len = p.split_len;
    P.nsplit = p.nsplit;
    P.tm = p.tm;
    P.out_q16 = r->out_kind == VGX_E_Q16;
    P.out = static_cast<uint8_t*>(r->out);
    P.ostride = r->out_stride;
    P.lse = r->lse;
    P.po = static_cast<float*>(r->ws);
    P.pml = P.po ? P.po + (size_t)p.nsplit * A.ntok * A.heads * A.hd : nullptr;
    VGX_HIP(hipSetDevice(ctx->device));
    if (p.lds > 64 * 1024)
        VGX_HIP(hipFuncSetAttribute((const void*)p.fn, hipFuncAttributeMaxDynamicSharedMemorySize, p.lds));
    hipLaunchKernelGGL(p.fn, dim3((unsigned)p.wgs, (unsigned)p.nsplit), dim3(256), p.lds, ctx->stream, P);
    VGX_LAUNCH_CHECK("paged attention launch");
    if (p.nsplit > 1) {
        const int64_t jobs = (int64_t)A.ntok * A.heads;
        hipLaunchKernelGGL(compute_kind(cache->kind) == VGX_E_BF16 ? paged_join_kernel<VGX_E_BF16>
                                                                   : paged_join_kernel<VGX_E_F16>,
                           dim3((unsigned)((jobs + 3) / 4)), dim3(256), 0, ctx->stream, P);
        VGX_LAUNCH_CHECK("paged attention join launch");
    }
    return VGX_OK;
}

}  // extern "C"
