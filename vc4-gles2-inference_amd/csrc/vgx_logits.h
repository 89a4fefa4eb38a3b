// Rows of logits and their weights e^((x - m) / T) in 64 bits, as the draft check
// and the sampler read and compute them.
//
// The exponential: e^y = 2^k 2^(i/64) e^(f ln 2 / 64) with 64 y / ln 2 = 64 k + i
// + f, |f| <= 1/2: a table of 64 powers in LDS and a polynomial of degree 4 in f
// (error (ln 2 / 128)^5 / 120 < 4e-14); a table lookup instead of a polynomial of degree 11 or more
// (P. T. P. Tang, ACM TOMS 15, 1989).  12 operations of 64 bits a logit.
#pragma once

#include <cfloat>
#include <cmath>

#include "vgx_internal.h"

#pragma clang fp contract(off)

namespace {

typedef unsigned uint32x2 __attribute__((ext_vector_type(2)));

template <int KIND>
constexpr int kBytes = KIND == VGX_E_F32 ? 4 : 2;
template <int KIND>
constexpr int kPer = 16 / kBytes<KIND>;  // values of a 16-byte piece

// NaN counts as masked (-inf), +inf as the largest float.
__device__ __forceinline__ float clean(float x) { return x == x ? fminf(x, FLT_MAX) : -INFINITY; }

template <int KIND>
__device__ __forceinline__ float one(const uint8_t* p, int i) {
    if (KIND == VGX_E_F32) return clean(reinterpret_cast<const float*>(p)[i]);
    const unsigned short u = reinterpret_cast<const unsigned short*>(p)[i];
    if (KIND == VGX_E_Q16) return (float)(short)u * (1.0f / 256);
    if (KIND == VGX_E_BF16) return clean(__uint_as_float((unsigned)u << 16));
    return clean((float)__builtin_bit_cast(_Float16, u));
}

// CLEAN: masks and infinities as they count.
template <int KIND, bool CLEAN = true>
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[kPer<KIND>]) {
    auto tidy = [](float y) { return CLEAN ? clean(y) : y; };
    const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (KIND == VGX_E_F32) {
            x[i] = tidy(__uint_as_float(u[i]));
        } else if constexpr (KIND == VGX_E_Q16) {
            x[2 * i] = (float)(short)(u[i] & 0xffff) * (1.0f / 256);
            x[2 * i + 1] = (float)((int)u[i] >> 16) * (1.0f / 256);
        } else if constexpr (KIND == VGX_E_BF16) {
            x[2 * i] = tidy(__uint_as_float(u[i] << 16));
            x[2 * i + 1] = tidy(__uint_as_float(u[i] & 0xffff0000u));
        } else {
            x[2 * i] = tidy((float)__builtin_bit_cast(_Float16, (unsigned short)(u[i] & 0xffff)));
            x[2 * i + 1] = tidy((float)__builtin_bit_cast(_Float16, (unsigned short)(u[i] >> 16)));
        }
    }
}

// A row as 16-byte pieces of the address space: piece g holds values
// g * per - off .. + per - 1; the ends' pieces are read value by value.
struct Row {
    const uint8_t* p;
    int off;
};
template <int KIND>
__device__ __forceinline__ Row row_at(const uint8_t* x, int64_t stride, int r) {
    Row q;
    q.p = x + (int64_t)r * stride;
    q.off = (int)(((uintptr_t)q.p & 15) / kBytes<KIND>);
    return q;
}
template <int KIND>
__device__ __forceinline__ void piece(const Row& q, int vocab, int g, float (&x)[kPer<KIND>]) {
    constexpr int N = kPer<KIND>;
    const int i0 = g * N - q.off;
    if (i0 >= 0 && i0 + N <= vocab) {
        unpack<KIND>(*reinterpret_cast<const uint4*>(q.p + (int64_t)i0 * kBytes<KIND>), x);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = i0 + e >= 0 && i0 + e < vocab ? one<KIND>(q.p, i0 + e) : -INFINITY;
    }
}

// 2^(i / 64), written into LDS by every workgroup, less i 2^14 in the high word:
// adding n 2^14 for n = 64 k + i then adds k to the exponent alone.
__device__ __forceinline__ void fill_table(double* t) {
    for (int i = threadIdx.x; i < 64; i += blockDim.x) {
        const unsigned long long u = __builtin_bit_cast(unsigned long long, exp2((double)i * (1.0 / 64)));
        t[i] = __builtin_bit_cast(double, u - ((unsigned long long)i << 46));
    }
}
// x, m -> e^((x - m) / T) for x <= m: a = 64 / (T ln 2).  Below e^-690 the
// weight stays there: nothing a sum of 1 or more would notice.
struct Scale {
    double a, m;
};
__device__ __forceinline__ Scale scale_of(float m, double inv) {
    return {inv * 92.33248261689366, m == -INFINITY ? 0.0 : (double)m};
}
// sum + 2^(z / 64), z in [-63700, 0].
__device__ __forceinline__ double add_pow(double z, double sum, const double* tab) {
    const double big = 6755399441055744.0;  // 1.5 * 2^52: the low bits hold the rounded value
    const double kb = z + big;
    const int n = (int)(unsigned)__builtin_bit_cast(unsigned long long, kb);
    const double f = z - (kb - big);
    // (ln 2 / 64)^i / i!
    double e = fma(f, 5.732851688640402e-10, 2.1173137155464776e-07);
    e = fma(e, f, 5.86490495505617e-05);
    e = fma(e, f, 0.010830424696249145);
    e = fma(e, f, 1.0);
    uint32x2 t = __builtin_bit_cast(uint32x2, tab[n & 63]);
    t.y += (unsigned)n << 14;
    return fma(e, __builtin_bit_cast(double, t), sum);
}
__device__ __forceinline__ double exp_of(float x, const Scale& S, const double* tab) {
    return add_pow(fmax(((double)x - S.m) * S.a, -63700.0), 0.0, tab);
}

// The same, with 0 for a masked x and below e^-690.
__device__ __forceinline__ double weight(float x, const Scale& S, const double* tab) {
    return x == -INFINITY || ((double)x - S.m) * S.a < -63700.0 ? 0.0 : exp_of(x, S, tab);
}
__device__ __forceinline__ double weight(float x, float m, double inv, const double* tab) {
    return weight(x, scale_of(m, inv), tab);
}

// Lane exchanges inside rows of 16 lanes (quad_perm [1,0,3,2], [2,3,0,1],
// row_half_mirror, row_mirror), the four rows then joined through readlane.
template <int CTRL>
__device__ __forceinline__ int dpp(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, false); }
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
    const uint32x2 u = __builtin_bit_cast(uint32x2, x);
    const uint32x2 v = {(unsigned)dpp<CTRL>((int)u.x), (unsigned)dpp<CTRL>((int)u.y)};
    return __builtin_bit_cast(double, v);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) { return __int_as_float(dpp<CTRL>(__float_as_int(x))); }
__device__ __forceinline__ double lane_of(double x, int l) {
    const uint32x2 u = __builtin_bit_cast(uint32x2, x);
    const uint32x2 v = {(unsigned)__builtin_amdgcn_readlane((int)u.x, l), (unsigned)__builtin_amdgcn_readlane((int)u.y, l)};
    return __builtin_bit_cast(double, v);
}
__device__ __forceinline__ float lane_of(float x, int l) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l));
}
__device__ __forceinline__ double wave_sum(double x) {
    x += dpp<0xB1>(x);
    x += dpp<0x4E>(x);
    x += dpp<0x141>(x);
    x += dpp<0x140>(x);
    return (lane_of(x, 0) + lane_of(x, 16)) + (lane_of(x, 32) + lane_of(x, 48));
}
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp<0xB1>(x));
    x = fmaxf(x, dpp<0x4E>(x));
    x = fmaxf(x, dpp<0x141>(x));
    x = fmaxf(x, dpp<0x140>(x));
    return fmaxf(fmaxf(lane_of(x, 0), lane_of(x, 16)), fmaxf(lane_of(x, 32), lane_of(x, 48)));
}
// The running sum over the lanes: inside rows of 16 (row_shr), then the rows
// before (row_bcast 15 and 31).
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double x) {
    const uint32x2 u = __builtin_bit_cast(uint32x2, x);
    const uint32x2 v = {(unsigned)__builtin_amdgcn_update_dpp(0, (int)u.x, CTRL, ROWS, 0xF, false),
                        (unsigned)__builtin_amdgcn_update_dpp(0, (int)u.y, CTRL, ROWS, 0xF, false)};
    return x + __builtin_bit_cast(double, v);
}
__device__ __forceinline__ double wave_scan(double x) {
    x = dpp_add<0x111, 0xF>(x);
    x = dpp_add<0x112, 0xF>(x);
    x = dpp_add<0x114, 0xF>(x);
    x = dpp_add<0x118, 0xF>(x);
    x = dpp_add<0x142, 0xA>(x);
    return dpp_add<0x143, 0xC>(x);
}
// (value, index): the larger value, the smaller index of equals.
__device__ __forceinline__ void wave_best(float& m, int& a) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const float m2 = __shfl_xor(m, o, 64);
        const int a2 = __shfl_xor(a, o, 64);
        if (m2 > m || (m2 == m && a2 < a)) { m = m2; a = a2; }
    }
}

}  // namespace
