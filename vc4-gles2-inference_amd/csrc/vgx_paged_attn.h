// Attention of a ragged batch's new tokens over a paged cache.
//
// Formulas.  For one sequence and KV head the queries are the columns of Q^T
// (row r of the sequence's new tokens, head u of the group: column r * grp +
// u).  Per tile of keys
//   S^T = K Q^T        32x32x16 MFMA, A = K rows, B = Q columns
//   m' = max(m, max_keys S), P = exp2(c S - c m'), l = l 2^(c(m - m')) + sum P
//   O^T = O^T 2^(c(m - m')) + V^T P    A = V^T, B = P
// with c = scale * log2(e); out = O / l.  Products in the compute type with
// 32-bit sums; m, l and O stay in 32 bits.
//
// P is rounded to the compute type, which is what the second product multiplies;
// l sums it unrounded.  A weight is then off by at most half a step of its own
// (2^-8 of it in bf16, 2^-11 in f16), as K and V were when they were stored;
// carrying the rest of it in a second operand would double that product.  bf16
// has the exponents of 32 bits.  In f16 a weight below 2^-14 loses bits and one
// below 2^-25 all of them, which many such keys behind one that has nearly all
// the weight would notice: there the weights are 2^lift times as large, in P
// and in l (lift_of).
//
// Why transposed: a 32x32 product leaves column q's scores in lanes q and
// q + 32 (keys 8a + 4h + b in register 4a + b of half h), which is a B operand
// of the next product when its key order is taken as (4h + b, 8 + 4h + b): P
// never leaves the registers, a row's statistics are one lane's and its
// partner's, and the running scale is one multiply a register.  V^T in that
// order is two 64-bit transposing LDS reads a fragment.
//
// Over a tree (TREE) a row sees the positions before the new rows, and of those
// the ones that its mask names: where a tile of keys holds new rows, a column's
// visible keys are 32 or 64 bits of that mask, shifted to the tile; the tiles
// before those are untouched.  A call: one tree of 8 rows over 700 positions 8.6 us,
// a launch and its round trips; 24 of 5 to 61 rows over 300 to 8000 (16/8 heads of
// 64, f16) 57 with the join, 48 under a window of 4096 (16/2 of 64, q8) 42, both
// waiting for the next tile's loads 43% of the wave cycles (vector work 23 and 25%);
// 2 of 64 rows over 60001 (32/8 of 128, bf16) 189, of which the tiles are 171: 126
// GFLOP at 740 TFLOP/s, in one round of workgroups, two of which stage the same keys.
#pragma once

#include <algorithm>
#include <cmath>
#include <string>

#include "vgx_paged.h"

#pragma clang fp contract(off)

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
    PagedDev A;
    const uint8_t* q;
    int64_t qstride;
    float c;       // scale * log2(e), the K step included: exponents of 2
    float scale;   // scale with the K step: scores
    int window;
    int split_len, split_sh;
    int cmin, cmax;  // the sequences of this launch: cmin < columns a KV head <= cmax
    int out_q16;
    uint8_t* out;
    int64_t ostride;
    float* lse;
    // Partial results, numbered: hd sums and (m, l) each, without the lift.  Split
    // k of a row and head is number base + k * step; pn (ntok x heads) holds their
    // splits and base.  Numbers go by row and head, or by sequence, KV head and column (the
    // few rows of short sequences among many others').
    float* po;
    float2* pml;
    uint2* pn;
    unsigned pbase, pstep;
    int by_seq;
    // TREE: each row's depth (with a window), and its mask of words 64-bit words
    const int* depth;
    const uint64_t* see;
    int words;
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
__device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
    if constexpr (CK == VGX_E_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
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
// Four cache bytes as two pairs of half floats, exact.
__device__ __forceinline__ uint2 q8_to_f16(unsigned w) {
    const float a = (float)(signed char)w, b = (float)(signed char)(w >> 8), c = (float)(signed char)(w >> 16),
                d = (float)((int)w >> 24);
    uint2 r;
    r.x = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a, b));
    r.y = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(c, d));
    return r;
}
// Infinities and NaN among V.  Where a row does not see a key its weight is 0,
// but 0 * inf would reach it through the product, so tiles that some row does
// not wholly see go into LDS with these set to 0 (the main loop stays free of
// a second path, whose copies of the sums cost it up to 200 registers); if
// there were any, a pass after the loop adds them to the rows that do see
// them: a weight times an infinity or NaN is that value.
template <int CK>
__device__ __forceinline__ bool odd1(unsigned short x) {
    constexpr unsigned short e = CK == VGX_E_BF16 ? 0x7f80u : 0x7c00u;
    return (x & e) == e;
}
template <int CK>
__device__ __forceinline__ bool clear_odd(unsigned& w) {
    const bool lo = odd1<CK>((unsigned short)w), hi = odd1<CK>((unsigned short)(w >> 16));
    w = (lo ? 0 : w & 0xffffu) | (hi ? 0 : w & 0xffff0000u);
    return lo || hi;
}
template <int CK>
__device__ __forceinline__ bool clear_odd(uint4& w) {
    bool r = clear_odd<CK>(w.x);
    r = clear_odd<CK>(w.y) || r;
    r = clear_odd<CK>(w.z) || r;
    return clear_odd<CK>(w.w) || r;
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
// The exponent of the largest weight: f16 ends at 2^16, and the tile kernel lets
// weights pass its reference by 2^6.
template <int CK, bool TILE>
constexpr float lift_of = CK != VGX_E_F16 ? 0.0f : TILE ? 9.0f : 15.0f;
template <int CK, bool TILE>
constexpr float unlift_of = CK != VGX_E_F16 ? 1.0f : TILE ? 0x1p-9f : 0x1p-15f;
// What to subtract from the scores: 0 while there is no key, so that the
// exponents stay -inf and the weights 0.
__device__ __forceinline__ float ref_or_0(float m) { return m == -INFINITY ? 0.0f : m; }
// An exponent is c s - c m in one operation, whose c m is rounded alone.  From
// 2^12 on that rounding is more than 2^-12, and at 2^31 it passes what a float
// can hold the power of: there m is subtracted from the scores first.
__device__ __forceinline__ bool far(float mc) { return fabsf(mc) > 4096.0f; }

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

// The page of position j (of the last one where j is past it) as the table has
// it, and the page to read: 0 where the table's is outside the pool, with the
// fault noted if some row sees the position (tiles begin at multiples of 64, up
// to 63 positions before a window: pages behind it may be gone).  Apart, so that
// a load does not wait for the table's before it.
__device__ __forceinline__ int page_at(const PagedDev& A, const int* tab, int j, int end) {
    return tab[page_of(A, min(j, end - 1))];
}
__device__ __forceinline__ int page_ok(const PagedDev& A, int pg, bool& bad, bool used = true) {
    const bool in = (unsigned)pg < (unsigned)A.npages;
    bad = bad || (used && !in);
    return in ? pg : 0;
}

// EX: heads of exactly HD values in pages whose size is a multiple of 16: 16
// rows then lie one after the other and a wave's address is one scalar and an
// offset a lane that stays.  Otherwise (EX false) HD is the room for a head and
// every row is looked up.

// Staging of a tile of 64 keys by a workgroup of 4 waves: wave w takes rows
// 16 w .. 16 w + 15, NL 16-byte pieces a lane of K and as many of V (lane r
// holds the page of row r % 16).
template <int KIND, int HD, bool EX>
struct Stage {
    static constexpr int CK = KIND == VGX_E_BF16 ? VGX_E_BF16 : VGX_E_F16;
    static constexpr int EB = KIND == VGX_E_Q8 ? 1 : 2;
    static constexpr int CPR = HD * EB / 16;  // pieces of a row
    static constexpr int NL = (16 * CPR + 63) / 64;
    static constexpr bool kAll = NL * 64 == 16 * CPR;
    uint4 k[NL], v[NL];

    // the page of row j0 + 16 w + lane % 16
    static __device__ __forceinline__ int page(const PagedDev& A, const int* tab, int j0, int end) {
        return page_at(A, tab, j0 + 16 * (int)(threadIdx.x >> 6) + (int)(threadIdx.x & 15), end);
    }
    // One of K and V; rows behind the end are whatever is there.
    static __device__ __forceinline__ void load1(const PagedDev& A, const uint8_t* base, int64_t ps, int64_t rs, int pg,
                                                 int j0, int end, uint4 (&w)[NL]) {
        const int lane = threadIdx.x & 63, jw = j0 + 16 * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint8_t* sbase = base;
        if (EX) {
            const int j = min(jw, (end - 1) & ~15);
            const int slot = j - page_of(A, j) * A.psize;
            sbase += (int64_t)__builtin_amdgcn_readfirstlane(pg) * ps + (int64_t)slot * rs;
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int sl = i * 64 + lane, row = sl / CPR, ch = sl - row * CPR;
            const uint8_t* p;
            if (EX) {
                p = sbase + (unsigned)(row * (int)rs + ch * 16);
            } else {
                const int q = __shfl(pg, row & 15, 64);  // (every lane takes part)
                const int j = min(jw + row, end - 1);
                const int slot = j - page_of(A, j) * A.psize;
                p = base + (int64_t)q * ps + (int64_t)slot * rs + ch * 16;
            }
            w[i] = make_uint4(0, 0, 0, 0);
            if ((kAll || row < 16) && (EX || ch * 16 < A.hd * EB)) w[i] = *reinterpret_cast<const uint4*>(p);
        }
    }
    __device__ __forceinline__ void load(const PagedDev& A, const uint8_t* kh, const uint8_t* vh, int pg, int j0,
                                         int end) {
        load1(A, kh, A.kpg, A.krow, pg, j0, end, k);
        load1(A, vh, A.vpg, A.vrow, pg, j0, end, v);
    }
    static __device__ __forceinline__ void put(uint8_t* p, const uint4& w) {
        if (KIND == VGX_E_Q8) {
            const uint2 a = q8_to_f16(w.x), b = q8_to_f16(w.y), c = q8_to_f16(w.z), d = q8_to_f16(w.w);
            reinterpret_cast<uint4*>(p)[0] = make_uint4(a.x, a.y, b.x, b.y);
            reinterpret_cast<uint4*>(p)[1] = make_uint4(c.x, c.y, d.x, d.y);
        } else {
            *reinterpret_cast<uint4*>(p) = w;
        }
    }
    static __device__ __forceinline__ void store1(uint8_t* l, int pitch, const uint4 (&w)[NL]) {
        const int lane = threadIdx.x & 63;
        l += 16 * (threadIdx.x >> 6) * pitch;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int sl = i * 64 + lane, row = sl / CPR, ch = sl - row * CPR;
            if (kAll || row < 16) put(l + row * pitch + ch * (32 / EB), w[i]);
        }
    }
    // V rows at or behind the tile's `left`-th become zeros, whatever the page
    // holds there.
    static __device__ __forceinline__ void cut(uint4 (&w)[NL], int left) {
        const int lane = threadIdx.x & 63, r0 = 16 * (threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < NL; ++i)
            if (r0 + (i * 64 + lane) / CPR >= left) w[i] = make_uint4(0, 0, 0, 0);
    }
    static __device__ __forceinline__ bool clean(uint4 (&w)[NL]) {
        bool r = false;
        if (KIND != VGX_E_Q8)
#pragma unroll
            for (int i = 0; i < NL; ++i) r = clear_odd<CK>(w[i]) || r;
        return r;
    }
    // The loaded tile into LDS; wide: with V cut and cleaned.  Whether there
    // was something to clean.
    __device__ __forceinline__ bool store(uint8_t* lk, uint8_t* lv, int left, bool wide) {
        bool r = false;
        store1(lk, Geo<HD>::pk, k);
        if (wide) {
            cut(v, left);
            r = clean(v);
        }
        store1(lv, Geo<HD>::pv, v);
        return r;
    }
    // Load and store in one go, K then V through the same registers (heads of
    // more than 128 values leave none for a tile ahead).
    static __device__ __forceinline__ bool fetch(const PagedDev& A, const uint8_t* kh, const uint8_t* vh, int pg,
                                                 int j0, int end, uint8_t* lk, uint8_t* lv, bool wide) {
        uint4 w[NL];
        bool r = false;
        load1(A, kh, A.kpg, A.krow, pg, j0, end, w);
        store1(lk, Geo<HD>::pk, w);
        load1(A, vh, A.vpg, A.vrow, pg, j0, end, w);
        if (wide) {
            cut(w, end - j0);
            r = clean(w);
        }
        store1(lv, Geo<HD>::pv, w);
        return r;
    }
    static __device__ __forceinline__ void fetch_v(const PagedDev& A, const uint8_t* vh, int pg, int j0, int end,
                                                   uint8_t* lv) {
        uint4 w[NL];
        load1(A, vh, A.vpg, A.vrow, pg, j0, end, w);
        cut(w, end - j0);
        store1(lv, Geo<HD>::pv, w);
    }
};

// What the main loop left out of four sums of a column: the infinities and
// NaN of keys lo .. hi-1 of a tile in LDS (p: the first key's four values).
template <int CK>
__device__ __forceinline__ void add_odd(float (&x)[4], const uint8_t* p, int pitch, int lo, int hi) {
    for (int r = lo; r < hi; ++r) {
        const s16x4 w = *reinterpret_cast<const s16x4*>(p + r * pitch);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (odd1<CK>((unsigned short)w[e])) x[e] += from_ct<CK>(w[e]);
    }
}

// The same for the keys that vis names.
template <int CK>
__device__ __forceinline__ void add_odd_of(float (&x)[4], const uint8_t* p, int pitch, uint64_t vis) {
    for (; vis; vis &= vis - 1) {
        const s16x4 w = *reinterpret_cast<const s16x4*>(p + (__ffsll((unsigned long long)vis) - 1) * pitch);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (odd1<CK>((unsigned short)w[e])) x[e] += from_ct<CK>(w[e]);
    }
}

// The running state of a wave's 32 columns.
template <int HD>
struct Acc {
    static constexpr int NB = HD / 32;
    f32x16 o[NB];
    float m, l;
    bool big;  // some column's m is far from 0
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
        m = -INFINITY;
        l = 0.0f;
        big = false;
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
// lane's column's, or (TREE) those that vis_of names.
template <int CK, int HD, bool EX, int KB, bool TREE, class Vis>
__device__ __forceinline__ void step(const PagedDev& A, const s16x8 (&q)[HD / 16], Acc<HD>& a, const uint8_t* lk,
                                     const uint8_t* lv, int j0, float c, bool mask, int vlo, int vhi, Vis vis_of) {
    const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
    f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) {
        if (!EX && 16 * t >= A.hd) continue;
        // (reads far ahead of their products would spill)
        if (HD > 128 && t % 4 == 0) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const s16x8 kf = *reinterpret_cast<const s16x8*>(lk + (kb * 32 + col) * Geo<HD>::pk + (2 * t + h) * 16);
            s[kb] = mfma<CK>(kf, q[t], s[kb]);
        }
    }
    if constexpr (EX && HD <= 128) {  // four reads ahead of the products
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int t = 0; t < (KB * HD / 16 - 4) / 2; ++t) {
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    }
    if (mask) {
        const uint64_t vis = TREE ? vis_of(j0) : 0;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int k = kb * 32 + 8 * (i / 4) + 4 * h + (i & 3), j = j0 + k;
                s[kb][i] = (TREE ? (bool)(vis >> k & 1) : j >= vlo && j < vhi) ? s[kb][i] : -INFINITY;
            }
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = half_max(mx);
    // The reference value m is any that keeps the weights in range: it moves,
    // and the sums with it, only when some column's maximum has passed its m by
    // 2^6 (a weight then stays below 64 lifts, exact in no fewer bits).
    if (__any((mx - a.m) * c > 6.0f)) {
        const float m2 = fmaxf(mx, a.m);
        const float alpha = exp2_((a.m - ref_or_0(m2)) * c);
        a.m = m2;
        a.big = __any(far(ref_or_0(m2) * c));
        a.l *= alpha;
#pragma unroll
        for (int b = 0; b < HD / 32; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) a.o[b][i] *= alpha;
    }
    const float m0 = ref_or_0(a.m);
    constexpr float lift = lift_of<CK, true>;
    float mc = lift == 0.0f ? m0 * c : fmaf(m0, c, -lift);
    if (__builtin_expect(a.big, 0)) {
        mc = -lift;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] -= m0;
    }
    float sum = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[kb][i] = exp2_(fmaf(s[kb][i], c, -mc));
            sum += s[kb][i];
        }
    a.l += sum;
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

// Where a column's partial results begin.
__device__ __forceinline__ unsigned part_of(const AttnArgs& P, int s, int h, int m, int row, int head) {
    return P.pbase + (P.by_seq ? (unsigned)(s * P.A.kvh + h) * P.cmax + m : (unsigned)row * P.A.heads + head);
}
// A row's number of splits in the low half of pn.x, its numbering above.
constexpr unsigned kBySeq = 1u << 16;

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

// A column's place: row of the batch, query head, position, what it sees (of a
// tree: vlo .. vhi - 1 are the positions before the new rows).
struct Col {
    bool valid;
    int row, head, vlo, vhi;
};
template <bool TREE>
__device__ __forceinline__ Col col_of(const AttnArgs& P, const SeqAt& q, int h, int m, int end) {
    Col r;
    r.valid = m < q.n * P.A.grp;
    const int i = m / P.A.grp;
    r.row = q.q0 + i;
    r.head = h * P.A.grp + (m - i * P.A.grp);
    int pos = q.kv - q.n + i;
    r.vhi = r.valid ? min(TREE ? q.kv - q.n : pos + 1, end) : 0;
    if (TREE && P.window > 0 && r.valid) pos = q.kv - q.n + min(max(P.depth[r.row], 0), q.n - 1);
    r.vlo = P.window > 0 ? pos - P.window + 1 : 0;
    return r;
}
// The first word of a column's mask.
__device__ __forceinline__ uint64_t first_word(const AttnArgs& P, const Col& c) {
    return c.valid ? P.see[(int64_t)c.row * P.words] : 0;
}
// Which of the 64 keys from j0 on a column of a tree sees.  base: the first new
// row's position; w0: the mask's first word.
__device__ __forceinline__ uint64_t visible(const AttnArgs& P, const Col& c, uint64_t w0, int base, int j0, int end) {
    if (!c.valid) return 0;
    auto below = [](int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; };
    const uint64_t ctx = below(c.vhi - j0) & ~below(c.vlo - j0);
    const int off = j0 - base;  // the tile's first key among the new rows
    uint64_t rows = 0;
    if (off <= -64) {
    } else if (off < 0) {
        rows = w0 << -off;
    } else {
        const int w = off >> 6, sh = off & 63;
        const uint64_t* p = P.see + (int64_t)c.row * P.words;
        if (w < P.words) rows = (w ? p[w] : w0) >> sh;
        if (sh && w + 1 < P.words) rows |= p[w + 1] << (64 - sh);
    }
    return (ctx | rows) & below(end - j0);
}

// max / sum over the four lanes that hold a column (lane % 16).
__device__ __forceinline__ float quad_max(float x) {
    x = half_max(x);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
    x = half_sum(x);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A wave's tile of 32 keys on its way: K as the pieces its lanes multiply (key
// lane % 16 of each half, 16 bytes from byte 64 T + 16 (lane / 16) of the
// row), V as pieces of rows for LDS.
template <int KIND, int HD, bool EX>
struct Keys {
    static constexpr int CK = KIND == VGX_E_BF16 ? VGX_E_BF16 : VGX_E_F16;
    static constexpr int EB = KIND == VGX_E_Q8 ? 1 : 2;
    static constexpr int RB = HD * EB;             // bytes of a row
    static constexpr int KP = (RB + 63) / 64;      // K pieces a lane and half
    static constexpr int CPR = RB / 16;            // V pieces of a row
    static constexpr int NL = 32 * CPR / 64;       // V pieces a lane
    static_assert(32 * CPR % 64 == 0, "");
    uint4 k[2][KP], v[NL];

    // the page of row j0 + lane % 32
    static __device__ __forceinline__ int page(const PagedDev& A, const int* tab, int j0, int end) {
        return page_at(A, tab, j0 + (int)(threadIdx.x & 31), end);
    }
    // byte of a row that piece T of lane group g starts at; in the tail of a
    // q8 row of 32 mod 64 bytes, 8 bytes a lane
    static __device__ __forceinline__ int kbyte(int T, int g) {
        return RB - 64 * T >= 64 ? 64 * T + 16 * g : 64 * T + 8 * g;
    }
    template <class Addr>
    __device__ __forceinline__ void load_k(int rb, int g, int u, Addr addr) {
#pragma unroll
        for (int T = 0; T < KP; ++T) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (RB - 64 * T >= 64) {
                if (EX || 64 * T + 16 * g < rb) w = *reinterpret_cast<const uint4*>(addr + kbyte(T, g));
            } else if (EX || 64 * T + 8 * g < rb) {
                const uint2 x = *reinterpret_cast<const uint2*>(addr + kbyte(T, g));
                w.x = x.x;
                w.y = x.y;
            }
            k[u][T] = w;
        }
    }
    __device__ __forceinline__ void load_k(const PagedDev& A, const uint8_t* kh, int pg, int j0, int end) {
        const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, rb = A.hd * EB;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (EX) {
                const int p = __builtin_amdgcn_readlane(pg, 16 * u);
                const int j = min(j0 + 16 * u, (end - 1) & ~15);
                const int slot = j - page_of(A, j) * A.psize;
                load_k(rb, g, u, kh + (int64_t)p * A.kpg + (int64_t)slot * A.krow + (unsigned)(r * (int)A.krow));
            } else {
                const int p = __shfl(pg, 16 * u + r, 64);
                const int j = min(j0 + 16 * u + r, end - 1);
                const int slot = j - page_of(A, j) * A.psize;
                load_k(rb, g, u, kh + (int64_t)p * A.kpg + (int64_t)slot * A.krow);
            }
        }
    }
    __device__ __forceinline__ void load_v(const PagedDev& A, const uint8_t* vh, int pg, int j0, int end) {
        const int lane = threadIdx.x & 63, rb = A.hd * EB;
        const uint8_t* base[2];
        if (EX) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int p = __builtin_amdgcn_readlane(pg, 16 * u);
                const int j = min(j0 + 16 * u, (end - 1) & ~15);
                const int slot = j - page_of(A, j) * A.psize;
                base[u] = vh + (int64_t)p * A.vpg + (int64_t)slot * A.vrow;
            }
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int sl = i * 64 + lane, row = sl / CPR, ch = sl - row * CPR;
            const uint8_t* p;
            if (EX) {
                // (pieces 0 .. NL/2 - 1 are the first half's rows)
                p = base[i >= NL / 2] + (unsigned)((row & 15) * (int)A.vrow + ch * 16);
                if (NL & 1) p = (row < 16 ? base[0] : base[1]) + (unsigned)((row & 15) * (int)A.vrow + ch * 16);
            } else {
                const int q = __shfl(pg, row, 64);
                const int j = min(j0 + row, end - 1);
                const int slot = j - page_of(A, j) * A.psize;
                p = vh + (int64_t)q * A.vpg + (int64_t)slot * A.vrow + ch * 16;
            }
            v[i] = make_uint4(0, 0, 0, 0);
            if (EX || ch * 16 < rb) v[i] = *reinterpret_cast<const uint4*>(p);
        }
    }
    // V into LDS; wide: rows behind the end (the tile's `left`-th on) as zeros,
    // and cleaned.  Whether there was something to clean.
    __device__ __forceinline__ bool store_v(uint8_t* lv, int left, bool wide, bool keep_odd = false) {
        const int lane = threadIdx.x & 63;
        bool r = false;
        if (wide) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                if ((i * 64 + lane) / CPR >= left) v[i] = make_uint4(0, 0, 0, 0);
                if (KIND != VGX_E_Q8 && !keep_odd) r = clear_odd<CK>(v[i]) || r;
            }
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int sl = i * 64 + lane, row = sl / CPR, ch = sl - row * CPR;
            uint8_t* p = lv + row * Geo<HD>::pv + ch * (32 / EB);
            if (KIND == VGX_E_Q8) {
                const uint2 a = q8_to_f16(v[i].x), b = q8_to_f16(v[i].y), c = q8_to_f16(v[i].z), d = q8_to_f16(v[i].w);
                reinterpret_cast<uint4*>(p)[0] = make_uint4(a.x, a.y, b.x, b.y);
                reinterpret_cast<uint4*>(p)[1] = make_uint4(c.x, c.y, d.x, d.y);
            } else {
                *reinterpret_cast<uint4*>(p) = v[i];
            }
        }
        return r;
    }
    // K's A operand of k-step t (half u): values as Q's B operand has them.
    __device__ __forceinline__ s16x8 frag(int u, int t) const {
        if constexpr (KIND == VGX_E_Q8) {
            const uint4 w = k[u][t / 2];
            const uint2 a = q8_to_f16(t & 1 ? w.z : w.x), b = q8_to_f16(t & 1 ? w.w : w.y);
            return __builtin_bit_cast(s16x8, make_uint4(a.x, a.y, b.x, b.y));
        } else {
            return __builtin_bit_cast(s16x8, k[u][t]);
        }
    }
    // The first value of k-step t that lane group g holds.
    static __device__ __forceinline__ int qdim(int t, int g) {
        if (KIND != VGX_E_Q8) return 32 * t + 8 * g;
        return RB - 64 * (t / 2) >= 64 ? 64 * (t / 2) + 16 * g + 8 * (t & 1) : 64 * (t / 2) + 8 * g;
    }
};

// LDS of one wave: its V tile; at the end its columns' sums.
constexpr int rows_lds(int hd, int nb) {
    const int pv = (hd * 2 + 63) / 128 * 128 + 64;
    return 32 * pv > nb * (hd + 4) * 64 ? 32 * pv : nb * (hd + 4) * 64;
}

// Few rows a sequence (max_q * grp <= 16 NB): a workgroup is one sequence, KV
// head and split; its WV waves hold the same NB blocks of 16 columns and take
// tiles of 32 keys in turn, without a barrier, and join at the end.  The 16x16x32
// product leaves column lane % 16's scores of keys 4 g + i (g = lane / 16) in
// the lane; two of them are the next product's B operand.  Long caches are bound
// by their bytes: one token at 130001 positions, 32 / 8 heads of 128 in bf16,
// 92 us (5.8 TB/s); 64 at 200 .. 16000 in q8, 106 us (4.7 TB/s; in bf16, with the
// join, 200 us and 4.9: 2136 workgroups with keys are 4.2 rounds of those
// resident; the same with four workgroups a CU, and with pages of 16 to 256).
// Short ones by a chain of round trips (lengths and table, rows, the join): one
// token at 700, 8 / 4 heads of 96, 8.4 us.
template <int KIND, int HD, bool EX, int NB, int WV, bool TREE>
__device__ __forceinline__ void rows_body(const AttnArgs& P, int bx, int split) {
    using Ks = Keys<KIND, HD, EX>;
    constexpr int CK = Ks::CK, KS = HD / 32, DB = HD / 16;
    constexpr int kWave = rows_lds(HD, NB);
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float sm[WV][16 * NB], sl[WV][16 * NB];
    const PagedDev& A = P.A;
    // Every argument into scalar registers before the first use of one: the
    // loads then go out as one batch instead of a round trip at each first use.
    asm volatile("" ::"s"(A.k), "s"(A.v), "s"(A.kpg), "s"(A.khd), "s"(A.krow), "s"(A.vpg), "s"(A.vhd), "s"(A.vrow),
                 "s"(A.tstride), "s"(A.qstart), "s"(A.kvlen), "s"(A.table), "s"(P.q), "s"(P.qstride), "s"(P.out),
                 "s"(P.po), "s"(P.split_len), "s"(P.split_sh), "s"(P.window), "s"(P.c), "s"(A.kvh), "s"(A.grp), "s"(A.psize),
                 "s"(A.pmul), "s"(A.npages), "s"(A.max_kv), "s"(A.ntok), "s"(A.heads), "s"(A.max_q), "s"(A.tcols));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int s = bx / A.kvh, h = bx - s * A.kvh;
    const int* tab = A.table + (int64_t)s * A.tstride;
    // Without a window the keys begin at 0, so the table's entries are asked
    // for along with the lengths (an entry past the sequence's end is not used).
    int pg = 0;
    if (P.window <= 0) {
        const int64_t j = (int64_t)split * P.split_len + wave * 32 + (lane & 31);
        pg = tab[min(page_of(A, (int)min(j, (int64_t)A.max_kv)), A.tcols - 1)];
    }
    const SeqAt q = seq_at(A, s);
    if (!q.ok && threadIdx.x == 0) set_fault(A, VGX_FAULT_LENGTH);
    if (q.n <= 0 || q.n * A.grp > P.cmax) return;
    const Span sp = span_of(q, 0, q.n - 1, P.window, P.split_len, P.split_sh);
    if (split >= sp.nsp) return;
    const int start = sp.lo + split * sp.len, end = start + min(sp.hi - start, sp.len);
    const uint8_t* kh = A.k + (int64_t)h * A.khd;
    const uint8_t* vh = A.v + (int64_t)h * A.vhd;
    uint8_t* lv = smem + wave * kWave;
    Ks t;
    int j0 = start + wave * 32;
    int pn = 0;
    bool bad = false, odd = false;
    if (j0 < end) {
        if (P.window > 0 || sp.len != P.split_len) pg = Ks::page(A, tab, j0, end);
        pn = Ks::page(A, tab, j0 + 32 * WV, end);
    }
    Col cl[NB];
    uint64_t w0[NB];
    s16x8 qf[NB][KS];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        cl[b] = col_of<TREE>(P, q, h, b * 16 + col, end);
        if (TREE) w0[b] = first_word(P, cl[b]);
        const uint8_t* qp = P.q + ((int64_t)cl[b].row * P.qstride + (int64_t)cl[b].head * A.hd) * 2;
#pragma unroll
        for (int u = 0; u < KS; ++u) {
            uint4 w = make_uint4(0, 0, 0, 0);
            const int d = Ks::qdim(u, g);
            if (cl[b].valid && (EX || d < A.hd)) w = *reinterpret_cast<const uint4*>(qp + d * 2);
            qf[b][u] = __builtin_bit_cast(s16x8, w);
        }
    }
    const int seen = P.window > 0 ? q.kv - q.n - P.window + 1 : 0;  // the first key of any row
    if (j0 < end) {
        pg = page_ok(A, pg, bad, j0 + (lane & 31) < end && j0 + (lane & 31) >= seen);
        t.load_v(A, vh, pg, j0, end);
        t.load_k(A, kh, pg, j0, end);
    }
    // keys every column sees: [all_lo, all_hi)
    const int base = q.kv - q.n;
    const int all_hi = min(base + (TREE ? 0 : 1), end);
    const int all_lo = P.window > 0 ? q.kv - P.window : 0;
    f32x4 o[NB][DB];
    float m[NB], l[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        m[b] = -INFINITY;
        l[b] = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[b][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // a lane's address for the transposing read: key 4 g + i / 4, dims 4 (i & 3)
    const uint8_t* vb = lv + (4 * g + (col >> 2)) * Geo<HD>::pv + 8 * (col & 3);
    // (past the end the loads repeat the last rows: without a branch between
    // them each product waits for its own loads only)
    while (j0 < end) {
        const bool mask = j0 + 32 > all_hi || j0 < all_lo;
        const int jn = j0 + 32 * WV;
        wave_sync();
        odd = t.store_v(lv, end - j0, mask) || odd;
        pg = page_ok(A, pn, bad);
        pn = Ks::page(A, tab, jn + 32 * WV, end);
        t.load_v(A, vh, pg, jn, end);
        f32x4 sc[NB][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int b = 0; b < NB; ++b) sc[b][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const s16x8 kf = t.frag(u, k);
#pragma unroll
                for (int b = 0; b < NB; ++b) sc[b][u] = mfma16<CK>(kf, qf[b][k], sc[b][u]);
            }
        }
        t.load_k(A, kh, pg, jn, end);
        s16x8 pf[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (mask) {
                const unsigned vis = TREE ? (unsigned)visible(P, cl[b], w0[b], base, j0, end) >> 4 * g : 0;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = j0 + 16 * u + 4 * g + i;
                        sc[b][u][i] = (TREE ? (bool)(vis >> (16 * u + i) & 1) : j >= cl[b].vlo && j < cl[b].vhi)
                                          ? sc[b][u][i] : -INFINITY;
                    }
            }
            float mx = fmaxf(fmaxf(fmaxf(sc[b][0][0], sc[b][0][1]), fmaxf(sc[b][0][2], sc[b][0][3])),
                             fmaxf(fmaxf(sc[b][1][0], sc[b][1][1]), fmaxf(sc[b][1][2], sc[b][1][3])));
            mx = fmaxf(quad_max(mx), m[b]);
            const float m0 = ref_or_0(mx);
            constexpr float lift = lift_of<CK, false>;
            float mc = lift == 0.0f ? m0 * P.c : fmaf(m0, P.c, -lift);
            const float alpha = exp2_((m[b] - m0) * P.c);
            m[b] = mx;
            if (__builtin_expect(__any(far(mc)), 0)) {
                mc = -lift;
#pragma unroll
                for (int u = 0; u < 2; ++u) sc[b][u] -= m0;
            }
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[b][u][i] = exp2_(fmaf(sc[b][u][i], P.c, -mc));
                    sum += sc[b][u][i];
                    pf[b][4 * u + i] = to_ct<CK>(sc[b][u][i]);
                }
            l[b] = fmaf(l[b], alpha, sum);
#pragma unroll
            for (int d = 0; d < DB; ++d) o[b][d] *= alpha;
        }
        wave_sync();
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            if (!EX && 16 * d >= A.hd) continue;
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vb + 32 * d));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vb + 32 * d + 16 * Geo<HD>::pv));
            const s16x8 vf = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int b = 0; b < NB; ++b) o[b][d] = mfma16<CK>(vf, pf[b], o[b][d]);
        }
        j0 = jn;
    }
    if (KIND != VGX_E_Q8 && __builtin_expect(__any(odd), 0)) {
        for (j0 = start + wave * 32; j0 < end; j0 += 32 * WV) {
            if (j0 + 32 <= all_hi && j0 >= all_lo) continue;
            t.load_v(A, vh, page_ok(A, Ks::page(A, tab, j0, end), bad, j0 + (lane & 31) >= seen), j0, end);
            wave_sync();
            t.store_v(lv, end - j0, true, true);
            wave_sync();
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    float x[4] = {o[b][d][0], o[b][d][1], o[b][d][2], o[b][d][3]};
                    if (TREE)
                        add_odd_of<CK>(x, lv + (16 * d + 4 * g) * 2, Geo<HD>::pv,
                                       (unsigned)visible(P, cl[b], w0[b], base, j0, end));
                    else
                        add_odd<CK>(x, lv + (16 * d + 4 * g) * 2, Geo<HD>::pv, max(cl[b].vlo - j0, 0),
                                    min(cl[b].vhi - j0, 32));
                    o[b][d] = f32x4{x[0], x[1], x[2], x[3]};
                }
        }
    }
    if (__builtin_expect(bad, 0)) set_fault(A, VGX_FAULT_PAGE);
    // the waves' columns through LDS, each thread then joining its outputs in
    // wave order on their common maximum
    float* part = reinterpret_cast<float*>(smem + wave * kWave);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const float x = quad_sum(l[b]);
        if (lane < 16) { sm[wave][16 * b + col] = m[b]; sl[wave][16 * b + col] = x; }
#pragma unroll
        for (int d = 0; d < DB; ++d)
            *reinterpret_cast<f32x4*>(part + (16 * b + col) * (HD + 4) + 16 * d + 4 * g) = o[b][d];
    }
    __syncthreads();
    const bool whole = sp.nsp == 1;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        if (!cl[b].valid) continue;
        float f[WV], M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < WV; ++w) {
            f[w] = sm[w][16 * b + col];
            M = fmaxf(M, f[w]);
        }
        const float m0 = ref_or_0(M);
#pragma unroll
        for (int w = 0; w < WV; ++w) {
            f[w] = exp2_((f[w] - m0) * P.c) * unlift_of<CK, false>;
            L = fmaf(sl[w][16 * b + col], f[w], L);
        }
        const int64_t at = (int64_t)cl[b].row * A.heads + cl[b].head;
        const unsigned part0 = part_of(P, s, h, 16 * b + col, cl[b].row, cl[b].head);
        const int64_t to = part0 + (int64_t)split * P.pstep;
        const float r = whole ? inv_l(P, L) : 1.0f;
        // thread: column lane % 16, every (4 WV)-th group of 4 dims
        for (int d = 4 * (threadIdx.x >> 4); d < A.hd; d += 16 * WV) {
            f32x4 x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < WV; ++w) {
                const f32x4 y = *reinterpret_cast<const f32x4*>(smem + w * kWave + ((16 * b + col) * (HD + 4) + d) * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = fmaf(y[e], f[w], x[e]);
            }
            const float4 v = make_float4(x[0] * r, x[1] * r, x[2] * r, x[3] * r);
            if (whole) put_out<CK>(P, cl[b].row, cl[b].head, d, v);
            else *reinterpret_cast<float4*>(P.po + to * A.hd + d) = v;
        }
        if (threadIdx.x < 16) {
            if (!whole) {
                P.pml[to] = make_float2(M, L);
                if (split == 0) P.pn[at] = make_uint2(sp.nsp | (P.by_seq ? kBySeq : 0), part0);
            } else {
                if (P.pn) P.pn[at] = make_uint2(1, 0);
                if (P.lse) P.lse[at] = lse_of(P, M, L);
            }
        }
    }
}

template <int KIND, int HD, bool EX, int NB, int WV, bool TREE>
__global__ void __launch_bounds__(64 * WV, (NB == 1 ? HD <= 128 : NB * HD <= 256) ? 2 : 1)
    paged_rows_kernel(const AttnArgs P) {
    rows_body<KIND, HD, EX, NB, WV, TREE>(P, blockIdx.x, blockIdx.y);
}

// The sequence and place of a tile of tm columns, tiles counted through the
// batch: false past the last.  Every lane of the wave is active.
__device__ __forceinline__ bool tile_at(const PagedDev& A, int tm, int cmin, int tile, int& s, int& local) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b = 0; b < A.nseq; b += 64) {
        const int j = b + lane;
        const int n = j < A.nseq ? seq_at(A, j).n : 0;
        const int cnt = n * A.grp > cmin ? (n * A.grp + tm - 1) / tm : 0;  // (the host bounds n * grp)
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
// one KV head; the waves share tiles of 64 keys.  Bound by the products and, as
// two waves a SIMD do not wholly hide it, the softmax between them (6.7 vector
// instructions a product): 4000 rows at 8100 positions, 32 / 8 heads of 128 in
// bf16, 417 to 444 us by the card (900 to 959 TFLOP/s; a library product of
// 8192^3 reaches 1234).
template <int KIND, int HD, bool EX, bool TREE>
__device__ __forceinline__ void tile_body(const AttnArgs& P, int bx, int wgs, int split) {
    constexpr int ROWS = 64, kTile = 64 * (Geo<HD>::pk + Geo<HD>::pv);
    using St = Stage<KIND, HD, EX>;
    constexpr int CK = St::CK;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int any_odd;
    const PagedDev& A = P.A;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, col = lane & 31;
    // the last tiles, which see the most keys, first
    const int rev = bx / A.kvh, h = bx - rev * A.kvh;
    const int tile = wgs / A.kvh - 1 - rev;
    int s, local;
    if (!tile_at(A, 128, P.cmin, tile, s, local)) return;
    s = __builtin_amdgcn_readfirstlane(s);
    local = __builtin_amdgcn_readfirstlane(local);
    const SeqAt q = seq_at(A, s);
    if (!q.ok && threadIdx.x == 0) set_fault(A, VGX_FAULT_LENGTH);
    const int m0 = local * 128, m1 = min(m0 + 128, q.n * A.grp) - 1;
    // (of a tree any row may see the last one, or be of the least depth)
    const Span sp = span_of(q, TREE ? 0 : m0 / A.grp, TREE ? q.n - 1 : m1 / A.grp, P.window, P.split_len);
    if (split >= sp.nsp) return;
    const int start = sp.lo + split * sp.len, end = start + min(sp.hi - start, sp.len);
    Col cl = col_of<TREE>(P, q, h, m0 + wave * 32 + col, end);
    // A column's mask, in the few tiles that hold new rows: its place is found
    // anew there, as registers held for it through the loop would spill.
    auto col_anew = [&] {
        int c = threadIdx.x;
        asm volatile("" : "+v"(c));
        return col_of<TREE>(P, q, h, m0 + wave * 32 + (c & 31), end);
    };
    auto vis_of = [&](int j0) {
        const Col x = col_anew();
        return visible(P, x, first_word(P, x), q.kv - q.n, j0, end);
    };
    s16x8 qf[HD / 16];
    load_q<HD, EX>(A, P.q + ((int64_t)cl.row * P.qstride + (int64_t)cl.head * A.hd) * 2, cl.valid, qf);
    // the wave's rows: keys every column sees, and keys any column sees
    const int w0 = m0 + wave * 32, w1 = min(w0 + 31, m1);
    const bool any = w0 <= m1;
    const int base = q.kv - q.n;
    const int r0 = TREE ? 0 : w0 / A.grp, r1 = TREE ? q.n - 1 : w1 / A.grp;
    const int all_hi = min(base + (TREE ? 0 : r0 + 1), end), any_hi = any ? min(base + r1 + 1, end) : 0;
    const int all_lo = P.window > 0 ? base + r1 - P.window + 1 : 0;
    const int any_lo = P.window > 0 ? base + r0 - P.window + 1 : 0;
    uint8_t* lk = smem;
    uint8_t* lv = smem + ROWS * Geo<HD>::pk;
    const uint8_t* kh = A.k + (int64_t)h * A.khd;
    const uint8_t* vh = A.v + (int64_t)h * A.vhd;
    const int* tab = A.table + (int64_t)s * A.tstride;
    Acc<HD> a;
    a.clear();
    St st;
    if (threadIdx.x == 0) any_odd = 0;  // (read after the loop's barriers)
    // tiles of keys that some column of the workgroup does not wholly see
    const int tile_hi = min(base + (TREE ? 0 : m0 / A.grp + 1), end);
    const int tile_lo = P.window > 0 ? base + (TREE ? q.n - 1 : m1 / A.grp) - P.window + 1 : 0;
    auto wide = [&](int j) { return j + ROWS > tile_hi || j < tile_lo; };
    // the first key of any row, and the row of a tile that the lane looks up
    const int seen = P.window > 0 ? base + (TREE ? 0 : m0 / A.grp) - P.window + 1 : 0;
    const int row = 16 * wave + (lane & 15);
    // Two tiles in LDS (one for heads of more than 128 values): the next one is
    // loaded into registers before this one's products and stored after them,
    // so a tile costs one barrier.
    constexpr bool kTwo = HD <= 128;
    int pg = 0, pn = 0;
    bool odd = false, bad = false;
    if (start < end) {
        pg = St::page(A, tab, start, end);
        pn = St::page(A, tab, start + ROWS, end);
        pg = page_ok(A, pg, bad, start + row >= seen);
        if (kTwo) {
            st.load(A, kh, vh, pg, start, end);
            odd = st.store(lk, lv, end - start, wide(start));
        }
    }
    int buf = 0;
    for (int j0 = start; j0 < end; j0 += ROWS) {
        const int jn = j0 + ROWS;
        if (!kTwo) {
            __syncthreads();  // the last tile's reads are done
            odd = St::fetch(A, kh, vh, pg, j0, end, lk, lv, wide(j0)) || odd;
        }
        __syncthreads();
        const uint8_t* ck = lk + buf * kTile;
        const uint8_t* cv = lv + buf * kTile;
        // (past the end the loads repeat the last rows)
        pg = page_ok(A, pn, bad);
        if (kTwo) st.load(A, kh, vh, pg, jn, end);
        pn = St::page(A, tab, jn + ROWS, end);
        if (j0 < any_hi && j0 + ROWS > any_lo) {
            const bool mask = j0 + ROWS > all_hi || j0 < all_lo;
            if constexpr (HD <= 128) {
                step<CK, HD, EX, 2, TREE>(A, qf, a, ck, cv, j0, P.c, mask, cl.vlo, cl.vhi, vis_of);
            } else {  // (registers)
#pragma unroll 1
                for (int u = 0; u < 64; u += 32)
                    step<CK, HD, EX, 1, TREE>(A, qf, a, ck + u * Geo<HD>::pk, cv + u * Geo<HD>::pv, j0 + u, P.c, mask,
                                              cl.vlo, cl.vhi, vis_of);
            }
        }
        if (kTwo && jn < end) {
            buf ^= 1;
            odd = st.store(lk + buf * kTile, lv + buf * kTile, end - jn, wide(jn)) || odd;
        }
    }
    if (odd) any_odd = 1;
    __syncthreads();
    if (KIND != VGX_E_Q8 && any_odd) {
        for (int j0 = start; j0 < end; j0 += ROWS) {
            if (!wide(j0)) continue;
            __syncthreads();
            St::fetch_v(A, vh, page_ok(A, St::page(A, tab, j0, end), bad, j0 + row >= seen), j0, end, lv);
            __syncthreads();
            // (as the loop above skips and masks)
            if (j0 >= any_hi || j0 + ROWS <= any_lo) continue;
            const uint64_t vis = TREE ? vis_of(j0) : 0;
#pragma unroll
            for (int b = 0; b < HD / 32; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float x[4] = {a.o[b][4 * g], a.o[b][4 * g + 1], a.o[b][4 * g + 2], a.o[b][4 * g + 3]};
                    const uint8_t* p = lv + (32 * b + 8 * g + 4 * (lane >> 5)) * 2;
                    if (TREE) add_odd_of<CK>(x, p, Geo<HD>::pv, vis);
                    else add_odd<CK>(x, p, Geo<HD>::pv, max(cl.vlo - j0, 0), min(cl.vhi - j0, ROWS));
#pragma unroll
                    for (int e = 0; e < 4; ++e) a.o[b][4 * g + e] = x[e];
                }
        }
    }
    if (bad) set_fault(A, VGX_FAULT_PAGE);
    // (the lift leaves: powers of two, exact)
    constexpr float unlift = unlift_of<CK, true>;
    const float L = half_sum(a.l) * unlift;
    if (TREE) cl = col_anew();
    if (!cl.valid) return;
    const int hh = lane >> 5;
    const int64_t at = (int64_t)cl.row * A.heads + cl.head;
    const unsigned part0 = part_of(P, s, h, 0, cl.row, cl.head);
    const int64_t to = part0 + (int64_t)split * P.pstep;
    const bool whole = sp.nsp == 1;
    const float r = whole ? inv_l(P, L) * unlift : unlift;
#pragma unroll
    for (int b = 0; b < HD / 32; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * b + 8 * g + 4 * hh;
            if (!EX && d >= A.hd) continue;
            const float4 v = make_float4(a.o[b][4 * g] * r, a.o[b][4 * g + 1] * r, a.o[b][4 * g + 2] * r,
                                         a.o[b][4 * g + 3] * r);
            if (whole) put_out<CK>(P, cl.row, cl.head, d, v);
            else *reinterpret_cast<float4*>(P.po + to * A.hd + d) = v;
        }
    if (hh == 0) {
        if (!whole) {
            P.pml[to] = make_float2(a.m, L);
            if (split == 0) P.pn[at] = make_uint2(sp.nsp, part0);
        } else {
            if (P.pn) P.pn[at] = make_uint2(1, 0);
            if (P.lse) P.lse[at] = lse_of(P, a.m, L);
        }
    }
}

template <int KIND, int HD, bool EX, bool TREE>
__global__ void __launch_bounds__(256, HD <= 128 && EX ? 2 : 1) paged_tile_kernel(const AttnArgs P) {
    tile_body<KIND, HD, EX, TREE>(P, blockIdx.x, gridDim.x, blockIdx.y);
}

// Prompts and single tokens in one batch: the sequences of at most 16 columns a
// KV head (over trees 16 both_nb) as the rows kernel takes them, the others as
// tiles, in one launch (the
// tiles first), so that the ones' bytes come in while the others multiply: 512
// rows and 8 at 16000 positions, 117 us (178 as tiles only, 136 in two launches);
// 20 sequences of 1 .. 700 rows, window 1024, 16 / 8 heads of 64, 21 us, the
// longest tile's chain.
template <int HD, bool TREE>
constexpr int both_nb = !TREE ? 1 : HD == 64 ? 3 : 2;  // blocks of 16 columns of the rows' way
struct BothArgs {
    AttnArgs rows, tile;
    int rows_wgs, tile_wgs;   // workgroups of one split
    int tile_all;             // the tiles' workgroups of all splits
};
template <int KIND, int HD, bool EX, bool TREE>
__global__ void __launch_bounds__(256, EX ? 2 : 1) paged_both_kernel(const BothArgs B) {
    const int bx = blockIdx.x;
    if (bx < B.tile_all) {
        const int split = bx / B.tile_wgs;
        tile_body<KIND, HD, EX, TREE>(B.tile, bx - split * B.tile_wgs, B.tile_wgs, split);
    } else {
        const int r = bx - B.tile_all, split = r / B.rows_wgs;
        rows_body<KIND, HD, EX, both_nb<HD, TREE>, 4, TREE>(B.rows, r - split * B.rows_wgs, split);
    }
}

// Joins a row's splits.  Few splits (WIDE false): hd / 4 lanes (rounded up to a
// power of two, lg) a row and head, in split order.  Many: a workgroup a row and
// head, the splits dealt to groups of hd / 4 threads, each in split order, the
// groups in theirs.  Round trips again (entry, maxima, sums): 4 to 6 us.
struct JoinArgs {
    unsigned step_row, step_seq, total;  // between a row's splits, by its numbering; all partial results
};
template <int CK, bool WIDE>
__global__ void __launch_bounds__(256) paged_join_kernel(const AttnArgs P, int lg, const JoinArgs J) {
    const PagedDev& A = P.A;
    __shared__ float sw[4], sl[4];
    __shared__ float4 so[256];
    const int lane = threadIdx.x & 63;
    // (a wave's lanes are of one row: lg divides so, or is 6)
    const int64_t w0 = WIDE ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) << (6 - lg);
    const int t = (int)(w0 / A.heads);
    const int head = (int)(w0 - (int64_t)t * A.heads) + (WIDE ? 0 : lane >> lg);
    if (t >= A.ntok) return;
    // (the entry of a row before the first sequence or behind the last was
    // written by nobody, nor that of a row past the bounds)
    const uint2 e = t >= A.qstart[0] && t < A.qstart[A.nseq] ? P.pn[(int64_t)t * A.heads + head] : make_uint2(0, 0);
    const int nsp = e.x & 0xffff;
    const int64_t step = e.x & kBySeq ? J.step_seq : J.step_row, at = e.y;
    if (nsp <= 1 || at + (nsp - 1) * step >= J.total) return;
    const float2* ml = P.pml + at;
    const float4* po = reinterpret_cast<const float4*>(P.po);
    const int n4 = A.hd / 4;
    float4 o = make_float4(0, 0, 0, 0);
    float M = -INFINITY, L = 0.0f;
    if (!WIDE) {
        for (int k = 0; k < nsp; ++k) M = fmaxf(M, ml[k * step].x);
        const float m0 = ref_or_0(M);
#pragma unroll 4
        for (int k = 0; k < nsp; ++k) {
            const float2 x = ml[k * step];
            const float f = exp2_((x.x - m0) * P.c);
            L = fmaf(x.y, f, L);
            const float4 y = po[(at + k * step) * n4 + min(lane & ((1 << lg) - 1), n4 - 1)];
            o.x = fmaf(y.x, f, o.x); o.y = fmaf(y.y, f, o.y); o.z = fmaf(y.z, f, o.z); o.w = fmaf(y.w, f, o.w);
        }
    } else {
        for (int k = threadIdx.x; k < nsp; k += 256) M = fmaxf(M, ml[k * step].x);
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
        if (lane == 0) sw[threadIdx.x >> 6] = M;
        __syncthreads();
        M = fmaxf(fmaxf(sw[0], sw[1]), fmaxf(sw[2], sw[3]));
        const float m0 = ref_or_0(M);
        const int ng = 256 / n4, gr = threadIdx.x / n4, d = threadIdx.x - gr * n4;
        if (gr < ng) {
#pragma unroll 8
            for (int k = gr; k < nsp; k += ng) {
                const float2 x = ml[k * step];
                const float f = exp2_((x.x - m0) * P.c);
                const float4 y = po[(at + k * step) * n4 + d];
                o.x = fmaf(y.x, f, o.x); o.y = fmaf(y.y, f, o.y); o.z = fmaf(y.z, f, o.z); o.w = fmaf(y.w, f, o.w);
            }
        }
        for (int k = threadIdx.x; k < nsp; k += 256) {
            const float2 x = ml[k * step];
            L = fmaf(x.y, exp2_((x.x - m0) * P.c), L);
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) L += __shfl_xor(L, x, 64);
        if (lane == 0) sl[threadIdx.x >> 6] = L;
        so[threadIdx.x] = o;
        __syncthreads();
        L = (sl[0] + sl[1]) + (sl[2] + sl[3]);
        if ((int)threadIdx.x >= n4) return;
        for (int x = 1; x < ng; ++x) {
            const float4 y = so[x * n4 + threadIdx.x];
            o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
        }
    }
    const int d = WIDE ? threadIdx.x : lane & ((1 << lg) - 1);
    const float r = inv_l(P, L);
    if (d < n4) put_out<CK>(P, t, head, 4 * d, make_float4(o.x * r, o.y * r, o.z * r, o.w * r));
    if (d == 0 && P.lse) P.lse[(int64_t)t * A.heads + head] = lse_of(P, M, L);
}

typedef void (*AttnFn)(const AttnArgs);
typedef void (*BothFn)(const BothArgs);
typedef void (*JoinFn)(const AttnArgs, int, const JoinArgs);
// Positions up to which one workgroup takes a sequence whole.
constexpr int64_t kWhole = 1024;
// Rounds of resident workgroups that a tree's tiles are split into, at most.
constexpr int kTreeRounds = 16;

struct Launch {
    AttnFn fn;
    BothFn both;
    int lds, tm, threads;
    bool rows;
    int cmin, cmax;
    int64_t wgs;       // workgroups of one split
    int split_len, split_sh, nsplit;
};
struct Plan {
    Launch l[2];
    int n;
    int by_seq;        // the first one's partial results are numbered by sequence
    size_t parts;      // partial results
    size_t ws;
    unsigned step(const PagedDev& A, int i) const {
        return i == 0 && by_seq ? (unsigned)A.nseq * A.kvh * l[0].cmax : (unsigned)A.ntok * A.heads;
    }
};

// cols: the columns a sequence may have in a KV head.  Up to 48 the rows kernel
// (16 for heads of more than 128 values; more columns fill the registers).  few:
// under half a workgroup a CU, each of a whole sequence of up to 1024 positions:
// 8 waves then finish it sooner (8 sequences of 900, 8 / 4 heads of 96: 11.2 us
// against 12.1 with 4 waves, 11.9 with 4 splits; 128 workgroups: 20.0 against
// 18.7).
template <int KIND, int HD, bool EX, bool TREE>
void fn_of(int64_t cols, bool few, Launch& p) {
    p.threads = 256;
    p.both = nullptr;
    if constexpr (HD <= 128) p.both = paged_both_kernel<KIND, HD, EX, TREE>;
    if (cols <= (HD <= 128 ? 48 : 16)) {
        const int nb = (int)(cols + 15) / 16;
        p.fn = paged_rows_kernel<KIND, HD, EX, 1, 4, TREE>;
        if constexpr (HD <= 128) {
            if (nb == 1 && few) {
                p.fn = paged_rows_kernel<KIND, HD, EX, 1, 8, TREE>;
                p.threads = 512;
            }
            if (nb == 2) p.fn = paged_rows_kernel<KIND, HD, EX, 2, 4, TREE>;
            if (nb == 3) p.fn = paged_rows_kernel<KIND, HD, EX, 3, 4, TREE>;
        }
        p.lds = p.threads / 64 * rows_lds(HD, nb);
        p.tm = 16 * nb;
        p.rows = true;
    } else {
        p.fn = paged_tile_kernel<KIND, HD, EX, TREE>;
        p.lds = (HD <= 128 ? 2 : 1) * 64 * (Geo<HD>::pk + Geo<HD>::pv);
        p.tm = 128;
        p.rows = false;
    }
}
template <int KIND, bool TREE>
void fn_of(const PagedDev& A, int64_t cols, bool few, Launch& p) {
    const int hd = A.hd;
    const bool whole = A.psize % 16 == 0 && A.krow < (1 << 26) && A.vrow < (1 << 26);
    if (whole) switch (hd) {
        case 64: return fn_of<KIND, 64, true, TREE>(cols, few, p);
        case 96: return fn_of<KIND, 96, true, TREE>(cols, few, p);
        case 128: return fn_of<KIND, 128, true, TREE>(cols, few, p);
        case 256:
            if constexpr (KIND != VGX_E_Q8) return fn_of<KIND, 256, true, TREE>(cols, few, p);  // (q8: it would spill)
    }
    return hd <= 128 ? fn_of<KIND, 128, false, TREE>(cols, few, p) : fn_of<KIND, 256, false, TREE>(cols, few, p);
}

// The head size that fn_of's kernel has room for.
int fn_hd(const PagedDev& A) {
    const bool whole = A.psize % 16 == 0 && A.krow < (1 << 26) && A.vrow < (1 << 26);
    return whole && (A.hd == 64 || A.hd == 96) ? A.hd : A.hd <= 128 ? 128 : 256;
}

// The columns the rows kernel takes at most.
int64_t max_cols(const PagedDev& A) { return A.hd <= 128 ? 48 : 16; }

// A window of every position is none (and what is left keeps the kernels' sums
// of positions and windows inside 32 bits).
int window_of(const PagedDev& A, int window) { return window >= A.max_kv ? 0 : window; }

template <bool TREE>
Launch launch_of(const PagedDev& A, int kind, int window, int num_cu, int64_t cols, int cmin, bool alone) {
    Launch p{};
    int64_t span = A.max_kv;
    // a tile's rows (of a tree all), lo's rounding
    if (window > 0) span = std::min<int64_t>(span, (int64_t)window + (TREE ? A.max_q + 64 : 192));
    const bool few = alone && span <= kWhole && (int64_t)A.nseq * A.kvh < num_cu / 2;
    if (kind == VGX_E_BF16) fn_of<VGX_E_BF16, TREE>(A, cols, few, p);
    else if (kind == VGX_E_F16) fn_of<VGX_E_F16, TREE>(A, cols, few, p);
    else fn_of<VGX_E_Q8, TREE>(A, cols, few, p);
    p.cmin = cmin;
    p.cmax = p.rows ? p.tm : INT32_MAX;
    // (a sequence of more than cmin columns has at most columns / tm + 1 tiles)
    const int64_t all = (int64_t)A.ntok * A.grp;
    int64_t tiles = p.rows ? A.nseq : all / p.tm + std::min<int64_t>(A.nseq, std::max<int64_t>(all / (cmin + 1), 1));
    if (TREE && !p.rows) tiles = std::min<int64_t>(tiles, A.nseq * ((cols + p.tm - 1) / p.tm));
    p.wgs = tiles * A.kvh;
    // Splits.  A workgroup of the rows kernel costs about 8 us before and after
    // its keys (the tables' and first rows' round trips, the join of its waves),
    // so splits go no further than filling the chip once (two workgroups a CU
    // are resident, three of the tile kernel at heads of up to 64).  One
    // sequence: down to 256 keys.  Several, whose lengths the host does not
    // know: 512 keys or more (24 x 6 rows over 2800 positions, 16 / 2 heads of
    // 64: 26.6 us at 256, 19.2 at 512, 18.9 at 768, 27.8 at 2048), and no more
    // than 768 (1024 where the sequences alone fill the CUs), or the longest
    // one's workgroups run after all others (64 sequences of 200 to 16000
    // positions: 111 us at 1024, 124 at 512).
    const int fill = !p.rows && A.hd <= 64 ? 3 : 2;
    const int64_t want = std::max<int64_t>(1, (int64_t)num_cu * fill / p.wgs);
    int64_t len = std::max<int64_t>((span + want - 1) / want, 256);
    if (p.rows && A.nseq > 1)
        len = span <= kWhole ? span : std::min<int64_t>(std::max<int64_t>(len, 512), p.wgs >= num_cu ? 1024 : 768);
    // Trees: a tile launch is a tile or two a sequence and KV head, so its longest
    // sequence would run on after all others, and sequences are split to 1024 keys
    // or a sixteenth of the longest (whose parts the join has to read): 24 trees of 5
    // to 61 rows at 300 to 8000, 16 / 8 heads of 64, 59 us (75 by the rule above, 74
    // at 512 keys, 61 at 2048); 2 of 64 rows at 60001, 32 / 8 of 128, 207 (251; 290 at
    // 1024).  That ends at 16 rounds of resident workgroups by the bounds, as the
    // partial results of more cost memory and time: of 64 rows, 32 / 8 heads of 128,
    // 128 at 8192 1664 us with 0.55 GB (without the end 1878 and 1.09; at 8 rounds
    // 1565, at none 1474), 128 of 500 under a bound of 32768 164 (296; 160; 156), one
    // at 32768 among 127 of 500 427 (425 and 2.2 GB; 651; 980).  The rows kernel
    // beside it takes 1024 keys too (768: 3 us more).
    if (TREE && A.nseq > 1 && !alone && p.rows) len = std::max<int64_t>(len, 1024);
    if (TREE && A.nseq > 1 && !p.rows) {
        const int64_t most = std::max<int64_t>((int64_t)kTreeRounds * num_cu * fill / p.wgs, 1);
        len = std::min<int64_t>(std::max<int64_t>(len, 512),
                                std::max<int64_t>({1024, span / 16, (span + most - 1) / most}));
    }
    len = (len + 127) / 128 * 128;
    if (p.threads == 512) len = std::max<int64_t>(span, 128);
    p.split_len = (int)std::min<int64_t>(len, INT32_MAX);
    p.nsplit = (int)std::max<int64_t>((span + len - 1) / len, 1);
    p.split_sh = 31;
    // A bound far above the lengths costs an empty workgroup for each split
    // that no sequence has, so their number ends at 8192 in all (8 splits at
    // the least): longer sequences then take longer splits.  64 sequences of
    // 500, 32 / 8 heads of 128: 42 us under bounds of 16384 to 10^6 positions
    // (without this 81 at 65536, 889 at 10^6); one of 60000 positions among 24
    // of 500, 16 / 8 heads of 64: 59 us (4096 in all: 79).
    if (p.rows && A.nseq > 1) {
        int sh = 3;
        while (sh < 13 && (p.wgs << (sh + 1)) <= 8192) ++sh;
        if (p.nsplit > 1 << sh) {
            p.nsplit = 1 << sh;
            p.split_sh = sh;
        }
    }
    return p;
}

// One kind of sequences, or both where some may have many columns and others up
// to 16 both_nb: l[0] then takes these, whose long caches it splits, l[1] the others.
template <bool TREE>
Plan plan_of(const PagedDev& A, int kind, int window, int num_cu) {
    Plan p{};
    const int64_t cols = (int64_t)A.max_q * A.grp;
    const int64_t least = A.ntok - (int64_t)(A.nseq - 1) * A.max_q;  // rows of the shortest sequence, if all others are full
    // (the columns of the rows' way: what fn_of's kernels have for these heads)
    const int rows = 16 * (fn_hd(A) == 64 ? both_nb<64, TREE> : both_nb<128, TREE>);
    if (cols > max_cols(A) && A.hd <= 128 && A.grp <= rows && A.nseq > 1 && least * A.grp <= rows) {
        p.l[0] = launch_of<TREE>(A, kind, window, num_cu, rows, 0, false);
        p.l[1] = launch_of<TREE>(A, kind, window, num_cu, cols, rows, false);
        p.n = 2;
        p.by_seq = 1;
    } else {
        p.l[0] = launch_of<TREE>(A, kind, window, num_cu, cols, 0, true);
        p.n = 1;
    }
    for (int i = 0; i < p.n; ++i)
        if (p.l[i].nsplit > 1) p.parts += (size_t)p.l[i].nsplit * p.step(A, i);
    if (p.parts > INT32_MAX) p.parts = 0;  // (their numbers have 32 bits: such a batch fills the chip unsplit)
    p.ws = p.parts ? p.parts * (A.hd + 2) * 4 + (size_t)A.ntok * A.heads * 8 : 0;
    return p;
}

// LDS past 64 KB is granted per kernel, once a context (not on the launch path).
template <bool TREE>
hipError_t attn_init() {
    for (int hd : {64, 96, 128, 256, 80, 144})      // (the last two: the kernels without an exact head)
        for (int64_t cols : {16, 32, 48, 49})
            for (bool few : {false, true})
                for (int kind : {VGX_E_BF16, VGX_E_F16, VGX_E_Q8}) {
                    PagedDev A{};
                    A.hd = hd;
                    A.psize = 16;
                    Launch p{};
                    if (kind == VGX_E_BF16) fn_of<VGX_E_BF16, TREE>(A, cols, few, p);
                    else if (kind == VGX_E_F16) fn_of<VGX_E_F16, TREE>(A, cols, few, p);
                    else fn_of<VGX_E_Q8, TREE>(A, cols, few, p);
                    if (p.lds <= 64 * 1024) continue;
                    for (const void* fn : {(const void*)p.fn, (const void*)p.both}) {
                        if (!fn || (fn == (const void*)p.both && p.rows)) continue;  // (the tiles' LDS is the larger)
                        const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, p.lds);
                        if (e != hipSuccess) return e;
                    }
                }
    return hipSuccess;
}

template <bool TREE>
size_t attn_ws(const char* who, vgx_ctx* ctx, const vgx_paged* cache, const vgx_ragged* batch, int window) {
    PagedDev A;
    if (vgx_paged_fill(who, cache, batch, &A) != VGX_OK || !ctx || window < 0) return 0;
    if (A.ntok == 0 || A.nseq == 0) return 0;
    return plan_of<TREE>(A, cache->kind, window_of(A, window), ctx->num_cu).ws;
}

// vgx_paged_attn and, over a tree, vgx_paged_attn_tree.
template <bool TREE>
int attn_call(const char* who, vgx_ctx* ctx, const vgx_paged* cache, const vgx_ragged* batch, const vgx_paged_query* r,
              const vgx_tree* tree) {
    AttnArgs P{};
    const int st = vgx_paged_fill(who, cache, batch, &P.A);
    if (st != VGX_OK) return st;
    auto fail = [&](int status, const char* what) { return vgx_fail(status, std::string(who) + ": " + what); };
    if (!r) return fail(VGX_EINVAL, "NULL query");
    const PagedDev& A = P.A;
    const int64_t width = (int64_t)A.heads * A.hd;
    if (r->q_stride < width || r->q_stride % 8 || r->out_stride < width || r->out_stride % 8)
        return fail(VGX_EINVAL, "a row stride below the width or not a multiple of 16 bytes");
    if (!(r->scale >= 0) || std::isinf(r->scale))
        return fail(VGX_EINVAL, "scale is negative or not a number");
    if (r->window < 0) return fail(VGX_EINVAL, "a negative window");
    if (r->out_kind != VGX_E_Q16 && r->out_kind != compute_kind(cache->kind))
        return fail(VGX_EINVAL, "out is the cache's compute type or q16");
    if (A.ntok && (!r->q || !r->out)) return fail(VGX_EINVAL, "NULL q or out");
    if (((uintptr_t)r->q | (uintptr_t)r->out | (uintptr_t)r->ws) & 15)
        return fail(VGX_EINVAL, "q, out or ws not 16-byte aligned");
    if (TREE) {
        if (!tree) return fail(VGX_EINVAL, "NULL tree");
        if (tree->words <= 0 || tree->words > kTreeWords) return fail(VGX_EINVAL, "a tree's masks are 1 to 16 words a row");
        if (A.max_q > 64 * tree->words) return fail(VGX_ERANGE, "max_q past the rows that a tree's masks hold");
        if (A.ntok && !tree->see) return fail(VGX_EINVAL, "a tree without masks");
        if (A.ntok && r->window > 0 && !tree->depth) return fail(VGX_EINVAL, "a tree's window needs the rows' depths");
        P.depth = tree->depth;
        P.see = tree->see;
        P.words = tree->words;
    }
    if (!ctx) return fail(VGX_EINVAL, "no context");
    if (A.ntok == 0 || A.nseq == 0) return VGX_OK;
    P.window = window_of(A, r->window);
    Plan p = plan_of<TREE>(A, cache->kind, P.window, ctx->num_cu);
    const bool split = p.ws && r->ws && r->ws_bytes >= p.ws;
    for (int i = 0; i < p.n && !split; ++i) {
        p.l[i].nsplit = 1;
        p.l[i].split_len = INT32_MAX;
        p.l[i].split_sh = 31;
    }
    for (int i = 0; i < p.n; ++i)
        if (p.l[i].wgs >= (1 << 24) || p.l[i].nsplit > 65535)
            return fail(VGX_ERANGE, "too many rows");
    if ((int64_t)A.ntok * A.heads > INT32_MAX - 256)
        return fail(VGX_ERANGE, "too many rows");
    P.q = static_cast<const uint8_t*>(r->q);
    P.qstride = r->q_stride;
    P.scale = (r->scale > 0 ? r->scale : 1.0f / std::sqrt((float)A.hd)) * A.kstep;
    P.c = P.scale * kLog2e;
    if (!(P.c > 1e-30f) || std::isinf(P.c))
        return fail(VGX_EINVAL, "scale times the K step outside 1e-30 .. 1e38");
    P.out_q16 = r->out_kind == VGX_E_Q16;
    P.out = static_cast<uint8_t*>(r->out);
    P.ostride = r->out_stride;
    P.lse = r->lse;
    if (split) {
        P.po = static_cast<float*>(r->ws);
        P.pml = reinterpret_cast<float2*>(P.po + p.parts * A.hd);
        P.pn = reinterpret_cast<uint2*>(P.pml + p.parts);
    }
    VGX_HIP(hipSetDevice(ctx->device));
    JoinArgs J{(unsigned)A.ntok * A.heads, 0, (unsigned)p.parts};
    BothArgs B;
    int most = 1;
    for (int i = 0; i < p.n; ++i) {
        const Launch& l = p.l[i];
        P.split_len = l.split_len;
        P.split_sh = l.split_sh;
        P.cmin = l.cmin;
        P.cmax = l.cmax;
        P.by_seq = i == 0 && p.by_seq;
        P.pstep = p.step(A, i);
        if (P.by_seq) J.step_seq = P.pstep;
        (i == 0 ? B.rows : B.tile) = P;
        if (l.nsplit > 1) P.pbase += (unsigned)l.nsplit * P.pstep;
        most = std::max(most, l.nsplit);
    }
    if (p.n == 1) {
        const Launch& l = p.l[0];
        hipLaunchKernelGGL(l.fn, dim3((unsigned)l.wgs, (unsigned)l.nsplit), dim3(l.threads), l.lds, ctx->stream, B.rows);
    } else {
        B.rows_wgs = (int)p.l[0].wgs;
        B.tile_wgs = (int)p.l[1].wgs;
        const int64_t tiles = p.l[1].wgs * p.l[1].nsplit, grid = tiles + p.l[0].wgs * p.l[0].nsplit;
        if (grid >= (1 << 24)) return fail(VGX_ERANGE, "too many rows");
        B.tile_all = (int)tiles;
        hipLaunchKernelGGL(p.l[1].both, dim3((unsigned)grid), dim3(256), std::max(p.l[0].lds, p.l[1].lds), ctx->stream, B);
    }
    VGX_LAUNCH_CHECK("paged attention launch");
    if (most > 1) {
        const int64_t jobs = (int64_t)A.ntok * A.heads;
        // (a row's partials one after the other cost a round trip each four)
        const bool wide = most > 8 && p.n == 1 && jobs < (1 << 24);  // (both: few of the rows are split)
        const bool bf = compute_kind(cache->kind) == VGX_E_BF16;
        const JoinFn join = wide ? (bf ? paged_join_kernel<VGX_E_BF16, true> : paged_join_kernel<VGX_E_F16, true>)
                                 : (bf ? paged_join_kernel<VGX_E_BF16, false> : paged_join_kernel<VGX_E_F16, false>);
        int lg = A.hd <= 64 ? 4 : A.hd <= 128 ? 5 : 6;
        if (A.heads % (64 >> lg)) lg = 6;  // a wave's heads would be of two rows
        const int64_t grid = wide ? jobs : ((jobs >> (6 - lg)) + 3) / 4;
        if (grid >= (1 << 24)) return fail(VGX_ERANGE, "too many rows");
        hipLaunchKernelGGL(join, dim3((unsigned)grid), dim3(256), 0, ctx->stream, P, lg, J);
        VGX_LAUNCH_CHECK("paged attention join launch");
    }
    return VGX_OK;
}

}  // namespace
