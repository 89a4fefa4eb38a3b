// Appending a ragged batch's keys and values to a paged cache, with the
// per-head norm and the rotation on the way.
#include <algorithm>
#include <cmath>
#include <string>

#include "vgx_paged.h"

#pragma clang fp contract(off)

namespace {

// floor(log2 d) for d >= 1
int log2_floor(unsigned d) {
    int s = 0;
    while (d >>= 1) ++s;
    return s;
}

// Three strides over a buffer keep their positions apart: sorted by stride,
// each passes the extent of the ones below.  ext: values at one position.
bool apart(int64_t ext, int64_t n[3], int64_t st[3]) {
    int o[3] = {0, 1, 2};
    std::sort(o, o + 3, [&](int a, int b) { return st[a] < st[b]; });
    for (int i = 0; i < 3; ++i) {
        const int a = o[i];
        if (n[a] == 1) continue;  // its stride is never used
        if (st[a] < ext) return false;
        ext = (int64_t)std::min<__int128>(ext + (__int128)(n[a] - 1) * st[a], INT64_MAX);
    }
    return true;
}

}  // namespace

int vgx_paged_fill(const char* who, const vgx_paged* c, const vgx_ragged* b, PagedDev* d) {
    const std::string w = std::string(who) + ": ";
    if (!c || !b) return vgx_fail(VGX_EINVAL, w + "NULL cache or batch");
    if (c->kind != VGX_E_BF16 && c->kind != VGX_E_F16 && c->kind != VGX_E_Q8)
        return vgx_fail(VGX_EINVAL, w + "a cache is bf16, f16 or q8");
    if (c->heads <= 0 || c->kv_heads <= 0 || c->heads % c->kv_heads || c->heads > 1024)
        return vgx_fail(VGX_EINVAL, w + "heads must be a multiple of kv_heads, at most 1024");
    if (c->head_dim <= 0 || c->head_dim % 16 || c->head_dim > 256)
        return vgx_fail(VGX_EINVAL, w + "head_dim must be a multiple of 16, at most 256");
    if (c->page_size <= 0 || c->page_size > (1 << 20) || c->num_pages <= 0)
        return vgx_fail(VGX_EINVAL, w + "page_size outside 1..2^20 or no pages");
    if (!c->k || !c->v) return vgx_fail(VGX_EINVAL, w + "NULL pages");
    const int eb = elem_bytes(c->kind), per16 = 16 / eb;
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return vgx_fail(VGX_EINVAL, w + "pages not 16-byte aligned");
    for (int i = 0; i < 2; ++i) {
        int64_t st[3] = {i ? c->v_page : c->k_page, i ? c->v_head : c->k_head, i ? c->v_row : c->k_row};
        int64_t n[3] = {c->num_pages, c->kv_heads, c->page_size};
        for (int j = 0; j < 3; ++j)
            if (st[j] < 0 || st[j] > ((int64_t)1 << 40) || st[j] % per16)
                return vgx_fail(VGX_EINVAL, w + "a page, head or row stride is negative, above 2^40 or not a multiple of 16 bytes");
        if (!apart(c->head_dim, n, st)) return vgx_fail(VGX_EINVAL, w + "the page, head and row strides overlap");
    }
    for (float step : {c->k_step, c->v_step})  // (a NaN is refused; 1 / step and 128 step stay finite)
        if (step != 0 && !(step >= 0x1p-64f && step <= 0x1p64f))
            return vgx_fail(VGX_EINVAL, w + "a q8 step is neither 0 nor in 2^-64 .. 2^64");
    if (b->nseq < 0 || b->ntok < 0 || b->nseq > (1 << 20) || b->ntok > (1 << 24))
        return vgx_fail(VGX_EINVAL, w + "nseq outside 0..2^20 or ntok outside 0..2^24");
    if (b->max_q < 0 || b->max_kv < 0) return vgx_fail(VGX_EINVAL, w + "a negative bound");
    if (b->nseq && b->ntok) {
        if (!b->qstart || !b->kvlen || !b->table) return vgx_fail(VGX_EINVAL, w + "NULL qstart, kvlen or table");
        if (b->table_cols <= 0 || b->table_stride < b->table_cols)
            return vgx_fail(VGX_EINVAL, w + "a table without columns, or rows that overlap");
        // (positions, less a window and 2^24 rows, stay inside 32 bits)
        if ((int64_t)b->table_cols * c->page_size > INT32_MAX - (1 << 25))
            return vgx_fail(VGX_ERANGE, w + "a table's row holds 2^31 - 2^25 positions or more");
        if ((int64_t)b->max_kv > (int64_t)b->table_cols * c->page_size)
            return vgx_fail(VGX_ERANGE, w + "max_kv past what a table's row holds");
    }
    PagedDev& A = *d;
    A.k = static_cast<uint8_t*>(c->k);
    A.v = static_cast<uint8_t*>(c->v);
    A.kpg = c->k_page * eb; A.khd = c->k_head * eb; A.krow = c->k_row * eb;
    A.vpg = c->v_page * eb; A.vhd = c->v_head * eb; A.vrow = c->v_row * eb;
    A.heads = c->heads; A.kvh = c->kv_heads; A.grp = c->heads / c->kv_heads; A.hd = c->head_dim;
    A.psize = c->page_size; A.npages = c->num_pages;
    // a 31-bit j: floor(j / d) = mulhi(j, floor(2^(32+s) / d) + 1) >> s, s =
    // floor(log2 d), the product's excess being below 2^s; a power of two by
    // its shift
    const unsigned p = (unsigned)c->page_size;
    const int s = log2_floor(p);
    if (p == 1) { A.pmul = 0; A.psh = 0; }
    else if ((p & (p - 1)) == 0) { A.pmul = 0x80000000u; A.psh = s - 1; }
    else { A.pmul = (unsigned)((((unsigned __int128)1 << (32 + s)) / p) + 1); A.psh = s; }
    A.kstep = c->kind == VGX_E_Q8 ? (c->k_step > 0 ? c->k_step : 1.0f / 16) : 1.0f;
    A.vstep = c->kind == VGX_E_Q8 ? (c->v_step > 0 ? c->v_step : 1.0f / 16) : 1.0f;
    A.nseq = b->nseq; A.ntok = b->ntok; A.tcols = b->table_cols; A.tstride = b->table_stride;
    const int64_t held = (int64_t)b->table_cols * c->page_size;
    A.max_q = b->max_q > 0 ? std::min(b->max_q, b->ntok) : b->ntok;
    A.max_kv = b->max_kv > 0 ? b->max_kv : (int)std::min<int64_t>(held, INT32_MAX);
    A.qstart = b->qstart; A.kvlen = b->kvlen; A.table = b->table; A.fault = b->fault;
    return VGX_OK;
}

namespace {

struct AppendArgs {
    PagedDev A;
    const uint8_t* x;
    int64_t stride;  // elements
    const float* cs;
    const float* sn;
    int npos, rot, half;
    const float* qn;
    const float* kn;
    float eps;
    uint8_t* q;
    int64_t qstride;
    int vecs;        // heads + 2 * kvh
    int wpt;         // workgroups a row
};

template <int ACT>
__device__ __forceinline__ void load8(const uint8_t* p, float (&x)[8]) {
    if (ACT == VGX_E_F32) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (ACT == VGX_E_BF16) {
                x[2 * i] = __uint_as_float(u[i] << 16);
                x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            } else if (ACT == VGX_E_F16) {
                x[2 * i] = (float)__builtin_bit_cast(f16_t, (unsigned short)(u[i] & 0xffff));
                x[2 * i + 1] = (float)__builtin_bit_cast(f16_t, (unsigned short)(u[i] >> 16));
            } else {
                x[2 * i] = (float)(short)(u[i] & 0xffff) * (1.0f / 256);
                x[2 * i + 1] = (float)((int)u[i] >> 16) * (1.0f / 256);
            }
        }
    }
}

template <int KIND>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    if (KIND == VGX_E_BF16) {
        return (unsigned)__builtin_bit_cast(unsigned short, (bf16_t)a) |
               (unsigned)__builtin_bit_cast(unsigned short, (bf16_t)b) << 16;
    }
    return (unsigned)__builtin_bit_cast(unsigned short, (f16_t)a) |
           (unsigned)__builtin_bit_cast(unsigned short, (f16_t)b) << 16;
}
template <int KIND>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(pack2<KIND>(x[0], x[1]), pack2<KIND>(x[2], x[3]), pack2<KIND>(x[4], x[5]),
                      pack2<KIND>(x[6], x[7]));
}
// The 8-bit grid: floor(v / step + 1/2), clamped.  NaN gives 0.
__device__ __forceinline__ uint2 pack8_q8(const float (&x)[8], float inv) {
    unsigned w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float f = floorf(x[i] * inv + 0.5f);
        f = fminf(fmaxf(f, -128.0f), 127.0f);
        const int q = x[i] == x[i] ? (int)f : 0;
        w[i / 4] |= (unsigned)(q & 255) << (8 * (i & 3));
    }
    return make_uint2(w[0], w[1]);
}

// A head vector is LPV = 8, 16 or 32 lanes of 8 values (the least that holds
// head_dim), so a wave takes 64 / LPV head vectors at a time and a workgroup of 4
// waves 256 / LPV, PASS times (all loads first): the row's place, a chain of
// three round trips, is then looked up once for them.  The rotation's partner
// values are loaded a second time (the cache line is the wave's own) instead of
// exchanged: the partner of a piece of 8 is a piece of 8.  Bound by bytes where
// rows are many: 32 / 8 heads of 128, 4233
// bf16 rows, 24.3 us (4.3 TB/s; 26.5 us with one pass).
template <int KIND, int ACT, int LPV, int PASS>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs P) {
    const PagedDev& A = P.A;
    const int t = blockIdx.x / P.wpt, part = blockIdx.x - t * P.wpt;
    const int sub = threadIdx.x & (LPV - 1);
    const int d0 = sub * 8;
    constexpr int ab = ACT == VGX_E_F32 ? 4 : 2, VPP = 256 / LPV;  // head vectors a pass
    const uint8_t* row = P.x + (int64_t)t * P.stride * ab;
    const int half = P.rot / 2;
    const bool turn = d0 < P.rot, first = d0 < half;
    const int partner = P.half && turn ? (first ? d0 + half : d0 - half) : d0;
    const int ti = P.half ? (first ? d0 : d0 - half) : d0 / 2;  // the angle of the first value
    float x[PASS][8], y[PASS][8];
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
        const int vec = (part * PASS + p) * VPP + threadIdx.x / LPV;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[p][e] = y[p][e] = 0.0f;
        if (vec < P.vecs && d0 < A.hd) {
            load8<ACT>(row + ((int64_t)vec * A.hd + d0) * ab, x[p]);
            if (P.half && turn && vec < A.heads + A.kvh) load8<ACT>(row + ((int64_t)vec * A.hd + partner) * ab, y[p]);
        }
    }
    const int s = seq_of_row(A, t);
    if (s >= A.nseq) return;  // behind the last sequence
    const SeqAt sq = seq_at(A, s);
    const int i = t - sq.q0, pos = sq.kv - sq.n + i;
    const int cap = min(A.max_kv, P.rot ? P.npos : 0x7fffffff);
    if (!sq.ok || pos >= cap) {
        if (threadIdx.x == 0) set_fault(A, VGX_FAULT_LENGTH);
        return;
    }
    if (i < 0 || i >= sq.n || pos < 0) return;
    const int pi = page_of(A, pos), slot = pos - pi * A.psize;
    const int pg = A.table[(int64_t)s * A.tstride + pi];
    float c[8], n[8];
    if (turn && d0 < A.hd) {
        const float* cp = P.cs + (int64_t)pos * half + ti;
        const float* np = P.sn + (int64_t)pos * half + ti;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool use = P.half || e < 4;  // (neighbours: four angles)
            c[e] = use ? cp[e] : 1.0f;
            n[e] = use ? np[e] : 0.0f;
        }
    }
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
        const int vec = (part * PASS + p) * VPP + threadIdx.x / LPV;
        const bool in = vec < P.vecs && d0 < A.hd;
        const bool isv = vec >= A.heads + A.kvh, isq = vec < A.heads;
        // 32-bit sum of squares over the head's lanes
        if (P.qn) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(x[p][e], x[p][e], ss);
#pragma unroll
            for (int o = 1; o < LPV; o <<= 1) ss += __shfl_xor(ss, o, 64);
            if (in && !isv) {
                const float* nw = isq ? P.qn : P.kn;
                const float r = 1.0f / sqrtf(ss / (float)A.hd + P.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[p][e] = x[p][e] * r * nw[d0 + e];
                if (turn && P.half)
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[p][e] = y[p][e] * r * nw[partner + e];
            }
        }
        if (!in) continue;
        if (turn && !isv) {
            if (P.half) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[p][e] = fmaf(first ? -y[p][e] : y[p][e], n[e], x[p][e] * c[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = x[p][2 * e], b = x[p][2 * e + 1];
                    x[p][2 * e] = fmaf(-b, n[e], a * c[e]);
                    x[p][2 * e + 1] = fmaf(a, n[e], b * c[e]);
                }
            }
        }
        constexpr int CK = KIND == VGX_E_BF16 ? VGX_E_BF16 : VGX_E_F16;
        if (isq) {
            if (P.q) *reinterpret_cast<uint4*>(P.q + ((int64_t)t * P.qstride + vec * A.hd + d0) * 2) = pack8<CK>(x[p]);
            continue;
        }
        // (asked for here, behind the queries: before the norm it cost 4233 rows
        // 1.2 us)
        if (pg < 0 || pg >= A.npages) {
            if (sub == 0) set_fault(A, VGX_FAULT_PAGE);
            continue;
        }
        const int h = isv ? vec - A.heads - A.kvh : vec - A.heads;
        uint8_t* o = isv ? A.v + (int64_t)pg * A.vpg + (int64_t)h * A.vhd + (int64_t)slot * A.vrow
                         : A.k + (int64_t)pg * A.kpg + (int64_t)h * A.khd + (int64_t)slot * A.krow;
        if (KIND == VGX_E_Q8)
            *reinterpret_cast<uint2*>(o + d0) = pack8_q8(x[p], 1.0f / (isv ? A.vstep : A.kstep));
        else
            *reinterpret_cast<uint4*>(o + d0 * 2) = pack8<KIND>(x[p]);
    }
}

typedef void (*AppendFn)(const AppendArgs);
template <int KIND, int ACT, int PASS>
AppendFn append_lpv(int lpv) {
    return lpv == 8    ? append_kernel<KIND, ACT, 8, PASS>
           : lpv == 16 ? append_kernel<KIND, ACT, 16, PASS>
                       : append_kernel<KIND, ACT, 32, PASS>;
}
template <int KIND>
AppendFn append_act(int act, int lpv, bool three) {
    switch (act) {
        case VGX_E_F32: return three ? append_lpv<KIND, VGX_E_F32, 3>(lpv) : append_lpv<KIND, VGX_E_F32, 1>(lpv);
        case VGX_E_BF16: return three ? append_lpv<KIND, VGX_E_BF16, 3>(lpv) : append_lpv<KIND, VGX_E_BF16, 1>(lpv);
        case VGX_E_F16: return three ? append_lpv<KIND, VGX_E_F16, 3>(lpv) : append_lpv<KIND, VGX_E_F16, 1>(lpv);
    }
    return three ? append_lpv<KIND, VGX_E_Q16, 3>(lpv) : append_lpv<KIND, VGX_E_Q16, 1>(lpv);
}

}  // namespace

extern "C" int vgx_paged_append(vgx_ctx* ctx, const vgx_paged* cache, const vgx_ragged* batch,
                                const vgx_paged_rows* r) {
    AppendArgs P{};
    const int st = vgx_paged_fill("vgx_paged_append", cache, batch, &P.A);
    if (st != VGX_OK) return st;
    if (!r) return vgx_fail(VGX_EINVAL, "vgx_paged_append: NULL rows");
    if (r->kind != VGX_E_F32 && r->kind != VGX_E_BF16 && r->kind != VGX_E_F16 && r->kind != VGX_E_Q16)
        return vgx_fail(VGX_EINVAL, "vgx_paged_append: rows are f32, bf16, f16 or q16");
    const PagedDev& A = P.A;
    const int64_t width = (int64_t)(A.heads + 2 * A.kvh) * A.hd;
    const int per16 = 16 / elem_bytes(r->kind);
    if (r->stride < width || r->stride % per16)
        return vgx_fail(VGX_EINVAL, "vgx_paged_append: stride below a row's width or not a multiple of 16 bytes");
    if (r->rot < 0 || r->rot % 16 || r->rot > A.hd)
        return vgx_fail(VGX_EINVAL, "vgx_paged_append: rot must be a multiple of 16, at most head_dim");
    if (r->rot && (!r->cos || !r->sin || r->npos <= 0))
        return vgx_fail(VGX_EINVAL, "vgx_paged_append: a rotation without its table");
    if (!r->q_norm != !r->k_norm) return vgx_fail(VGX_EINVAL, "vgx_paged_append: one norm weight of two");
    if (r->q_norm && !(r->eps >= 0 && std::isfinite(r->eps)))
        return vgx_fail(VGX_EINVAL, "vgx_paged_append: eps is negative or not a number");
    if (r->q && (r->q_stride < (int64_t)A.heads * A.hd || r->q_stride % 8))
        return vgx_fail(VGX_EINVAL, "vgx_paged_append: q_stride below a row's width or not a multiple of 16 bytes");
    if (A.ntok && !r->qkv) return vgx_fail(VGX_EINVAL, "vgx_paged_append: NULL qkv");
    if (((uintptr_t)r->qkv | (uintptr_t)r->q) & 15)
        return vgx_fail(VGX_EINVAL, "vgx_paged_append: qkv or q not 16-byte aligned");
    if (!ctx) return vgx_fail(VGX_EINVAL, "vgx_paged_append: no context");
    if (A.ntok == 0 || A.nseq == 0) return VGX_OK;
    P.x = static_cast<const uint8_t*>(r->qkv);
    P.stride = r->stride;
    P.cs = r->cos; P.sn = r->sin; P.npos = r->npos; P.rot = r->rot; P.half = r->rope_half;
    P.qn = r->q_norm; P.kn = r->k_norm; P.eps = r->eps;
    P.q = static_cast<uint8_t*>(r->q);
    P.qstride = r->q_stride;
    P.vecs = A.heads + 2 * A.kvh;
    const int lpv = A.hd <= 64 ? 8 : A.hd <= 128 ? 16 : 32;
    // three passes a workgroup where the rows alone fill the chip (8 workgroups
    // a CU are resident)
    const int passes = (P.vecs * lpv + 255) / 256;
    const bool three = passes > 1 && A.ntok >= 8 * ctx->num_cu;
    P.wpt = three ? (passes + 2) / 3 : passes;
    const int64_t grid = (int64_t)A.ntok * P.wpt;
    if (grid >= (1 << 24)) return vgx_fail(VGX_ERANGE, "vgx_paged_append: too many rows");  // 2^32 threads
    const AppendFn fn = cache->kind == VGX_E_BF16  ? append_act<VGX_E_BF16>(r->kind, lpv, three)
                        : cache->kind == VGX_E_F16 ? append_act<VGX_E_F16>(r->kind, lpv, three)
                                                   : append_act<VGX_E_Q8>(r->kind, lpv, three);
    VGX_HIP(hipSetDevice(ctx->device));
    hipLaunchKernelGGL(fn, dim3((unsigned)grid), dim3(256), 0, ctx->stream, P);
    VGX_LAUNCH_CHECK("paged append launch");
    return VGX_OK;
}
