// Drafted trees: masks from parents, the walk to the accepted rows, and the
// rows and pages of a cache that are copied for them.
#include <algorithm>
#include <string>

#include "vgx_paged.h"

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
constexpr int kTreeRows = 64 * kTreeWords;

// The rows of a batch without its cache: of vgx_ragged nseq, ntok, max_q,
// qstart and fault.
int rows_fill(const char* who, const vgx_ragged* b, PagedDev* A) {
    auto fail = [&](int status, const char* what) { return vgx_fail(status, std::string(who) + ": " + what); };
    if (!b) return fail(VGX_EINVAL, "NULL batch");
    if (b->nseq < 0 || b->ntok < 0 || b->nseq > (1 << 20) || b->ntok > (1 << 24))
        return fail(VGX_EINVAL, "nseq outside 0..2^20 or ntok outside 0..2^24");
    if (b->max_q < 0) return fail(VGX_EINVAL, "a negative bound");
    if (b->nseq && !b->qstart) return fail(VGX_EINVAL, "NULL qstart");
    A->nseq = b->nseq;
    A->ntok = b->ntok;
    A->max_q = b->max_q > 0 ? std::min(b->max_q, b->ntok) : b->ntok;
    A->qstart = b->qstart;
    A->fault = b->fault;
    return VGX_OK;
}

// seq_at without a length.
__device__ __forceinline__ SeqAt rows_at(const PagedDev& A, int s) {
    SeqAt r;
    const int a = A.qstart[s], b = A.qstart[s + 1];
    r.q0 = min(max(a, 0), A.ntok);
    r.n = min(max(min(b, A.ntok) - r.q0, 0), A.max_q);
    r.kv = r.n;
    r.ok = a >= 0 && b >= a && b <= A.ntok && b - a <= A.max_q;
    return r;
}

// A wave takes 64 rows of a sequence: its parents go into LDS, and every lane
// walks up from its row.  A parent comes before its row, so a walk ends.  Bound by
// its chain (lengths, parents, the walk's LDS reads, one a level) and once a step
// for all layers: 4 us for 24 sequences of 5 to 61 rows.
__global__ void __launch_bounds__(64) tree_masks_kernel(const PagedDev A, const int* parent, int window, int words,
                                                        int* depth, uint64_t* see) {
    __shared__ int up[kTreeRows];
    __shared__ unsigned long long bits[64 * kTreeWords];
    const int s = blockIdx.x, lane = threadIdx.x, r0 = blockIdx.y * 64;
    const SeqAt q = rows_at(A, s);
    if (!q.ok && lane == 0 && r0 == 0) set_fault(A, VGX_FAULT_LENGTH);
    if (r0 >= q.n) return;
    const int n = min(r0 + 64, q.n);
    for (int i = lane; i < n; i += 64) {
        const int p = parent[q.q0 + i];
        up[i] = p >= 0 && p < i ? p : -1;
    }
    for (int i = lane; i < 64 * words; i += 64) bits[i] = 0;
    __syncthreads();
    const int i = r0 + lane;
    if (i >= n) return;
    int d = 0;
    for (int j = i; j >= 0; j = up[j], ++d)
        if (window <= 0 || d < window) bits[lane * words + (j >> 6)] |= 1ull << (j & 63);
    depth[q.q0 + i] = d - 1;
    uint64_t* to = see + (int64_t)(q.q0 + i) * words;
    for (int w = 0; w < words; ++w) to[w] = bits[lane * words + w];
}

// A wave walks one sequence's tree: the row's chosen token is compared with
// those of all its children at once.  A level is one LDS read after the other and
// a vote: 3.5 us for 12 sequences, 3.8 for 64.
__global__ void __launch_bounds__(64) tree_accept_kernel(const PagedDev A, const int* parent, const int* tokens,
                                                         const int* chosen, int* path, int* accepted, int* next) {
    __shared__ int up[kTreeRows], tok[kTreeRows], then[kTreeRows];
    const int s = blockIdx.x, lane = threadIdx.x;
    const SeqAt q = rows_at(A, s);
    if (!q.ok && lane == 0) set_fault(A, VGX_FAULT_LENGTH);
    if (q.n <= 0) {
        if (lane == 0) { accepted[s] = 0; next[s] = -1; }
        return;
    }
    for (int i = lane; i < q.n; i += 64) {
        up[i] = parent[q.q0 + i];
        tok[i] = tokens[q.q0 + i];
        then[i] = chosen[q.q0 + i];
    }
    __syncthreads();
    int cur = 0, k = 0;
    for (;;) {
        if (lane == 0) path[q.q0 + k] = cur;
        const int want = then[cur];
        int child = -1;
        for (int b = (cur + 1) & ~63; b < q.n && child < 0; b += 64) {
            const int i = b + lane;
            const unsigned long long fit =
                __ballot(i > cur && i < q.n && up[i] == cur && tok[i] == want && want >= 0);  // (-1: no token)
            if (fit) child = b + __ffsll(fit) - 1;
        }
        if (child < 0) break;
        cur = child;
        ++k;
    }
    for (int i = k + 1 + lane; i < q.n; i += 64) path[q.q0 + i] = -1;
    if (lane == 0) { accepted[s] = k; next[s] = then[cur]; }
}

// ---- rows and pages of several layers

constexpr int kLayers = 64;  // of one launch
struct Layers {
    uint8_t* p[2 * kLayers];  // K and V of each
};

// A thread owns 16 bytes of a KV head's vector, of K or V of one layer, for a
// whole path: it reads four rows, then writes them.  A row comes from its own
// place or from behind it, so nothing that is still to be read is written over.
// What bounds it is the chain of lengths, path, table and rows (four rows a time
// share one): 5.6 us for 12 sequences and 8 layers of 4 heads of 96, 8.5 for 64
// sequences and 14 layers of 8 heads of 64 (8 MB at most).
struct KeepArgs {
    PagedDev A;
    const int* path;
    const int* accepted;
    int pieces;  // of a position: kvh * hd * bytes / 16
    int ppr;     // of a head
    Layers L;
};
__global__ void __launch_bounds__(256) keep_kernel(const KeepArgs P) {
    const PagedDev& A = P.A;
    const int s = blockIdx.x, side = blockIdx.z & 1;
    const int piece = blockIdx.y * blockDim.x + threadIdx.x;
    const SeqAt q = seq_at(A, s);
    const int acc = P.accepted[s];
    const bool ok = q.ok && acc >= 0 && (acc < q.n || (acc == 0 && q.n == 0));
    if (!ok && threadIdx.x == 0) set_fault(A, VGX_FAULT_LENGTH);
    if (!ok || piece >= P.pieces) return;
    const int h = piece / P.ppr, ch = piece - h * P.ppr;
    const int64_t pg = side ? A.vpg : A.kpg, row = side ? A.vrow : A.krow;
    uint8_t* base = P.L.p[blockIdx.z] + (int64_t)h * (side ? A.vhd : A.khd) + ch * 16;
    const int* tab = A.table + (int64_t)s * A.tstride;
    const int b = q.kv - q.n;
    bool bad_row = false, bad_page = false;
    auto at = [&](int pos) -> uint8_t* {
        const int pi = page_of(A, pos), page = tab[pi];
        if ((unsigned)page >= (unsigned)A.npages) { bad_page = true; return nullptr; }
        return base + (int64_t)page * pg + (int64_t)(pos - pi * A.psize) * row;
    };
    for (int k = 1; k <= acc; k += 4) {
        u32x4 x[4];
        uint8_t* to[4];
        int from[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) from[e] = k + e <= acc ? P.path[q.q0 + k + e] : k + e;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = from[e];
            x[e] = u32x4{0, 0, 0, 0};
            to[e] = nullptr;
            if (i < k + e || (i >= q.n && k + e <= acc)) {
                bad_row = true;
            } else if (i > k + e && b + k + e >= 0) {
                const uint8_t* p = at(b + i);
                to[e] = at(b + k + e);
                if (!p) to[e] = nullptr;
                if (to[e]) x[e] = *reinterpret_cast<const u32x4*>(p);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (to[e]) *reinterpret_cast<u32x4*>(to[e]) = x[e];
    }
    if (bad_row) set_fault(A, VGX_FAULT_LENGTH);
    if (bad_page) set_fault(A, VGX_FAULT_PAGE);
}

// One side of a page as lines of consecutive 16-byte pieces: `heads` blocks
// `head` bytes apart, each of a line per position `row` bytes apart.  Heads
// that lie side by side are one longer line.
struct PageSide {
    int64_t page, head, row;
    int heads, ppr;
};
struct CopyArgs {
    PageSide s[2];
    int npages, psize;
    const int* src;
    const int* dst;
    const int* rows;
    int* fault;
    int chunks;  // workgroups a head block
    Layers L;
};
// HBM bounds it: 301 pages of 64 positions, 8 heads of 128, K and V of 8 layers are
// 1263 MB read and written in 242 us, 5.2 TB/s (a plain copy of 2 GiB: 4.94).
constexpr int kCopyPer = 8;  // pieces a thread, all loaded before the first is written
// DENSE: a block's lines lie one after the other, in K as in V.
template <bool DENSE>
__global__ void __launch_bounds__(256) copy_kernel(const CopyArgs P) {
    const bool v = blockIdx.z & 1;
    const PageSide S = {v ? P.s[1].page : P.s[0].page, v ? P.s[1].head : P.s[0].head, v ? P.s[1].row : P.s[0].row,
                        v ? P.s[1].heads : P.s[0].heads, v ? P.s[1].ppr : P.s[0].ppr};
    const int i = blockIdx.x, h = blockIdx.y / P.chunks, c = blockIdx.y - h * P.chunks;
    if (h >= S.heads) return;
    const int from = P.src[i], to = P.dst[i], rows = P.rows ? P.rows[i] : P.psize;
    int bad = 0;
    if ((unsigned)from >= (unsigned)P.npages || (unsigned)to >= (unsigned)P.npages) bad |= VGX_FAULT_PAGE;
    if (rows < 0 || rows > P.psize) bad |= VGX_FAULT_LENGTH;
    if (bad) {
        if (threadIdx.x == 0 && P.fault) atomicOr(P.fault, bad);
        return;
    }
    if (from == to) return;
    uint8_t* base = P.L.p[blockIdx.z] + (int64_t)h * S.head;
    const uint8_t* a = base + (int64_t)from * S.page;
    uint8_t* b = base + (int64_t)to * S.page;
    const int64_t n = (int64_t)rows * S.ppr, t0 = (int64_t)c * (256 * kCopyPer) + threadIdx.x;
    auto at = [&](int64_t t) {
        if (DENSE) return t * 16;
        const unsigned r = (unsigned)t / (unsigned)S.ppr;  // (fewer than 2^31 pieces: checked by the host)
        return (int64_t)r * S.row + (int64_t)((unsigned)t - r * (unsigned)S.ppr) * 16;
    };
    if (t0 - threadIdx.x + 256 * kCopyPer <= n) {
        u32x4 x[kCopyPer];
        int64_t o[kCopyPer];
#pragma unroll
        for (int e = 0; e < kCopyPer; ++e) o[e] = at(t0 + e * 256);
#pragma unroll
        for (int e = 0; e < kCopyPer; ++e) x[e] = *reinterpret_cast<const u32x4*>(a + o[e]);
#pragma unroll
        for (int e = 0; e < kCopyPer; ++e) *reinterpret_cast<u32x4*>(b + o[e]) = x[e];
        return;
    }
#pragma unroll 1
    for (int64_t t = t0; t < n; t += 256) {
        const int64_t o = at(t);
        *reinterpret_cast<u32x4*>(b + o) = *reinterpret_cast<const u32x4*>(a + o);
    }
}

// Checks the layers against the first.
int layers_check(const char* who, int ncache, const vgx_paged* c) {
    auto fail = [&](const char* what) { return vgx_fail(VGX_EINVAL, std::string(who) + ": " + what); };
    if (ncache < 1 || !c) return fail("no caches");
    for (int i = 1; i < ncache; ++i) {
        const vgx_paged& a = c[0];
        const vgx_paged& b = c[i];
        if (a.kv_heads != b.kv_heads || a.head_dim != b.head_dim || a.page_size != b.page_size ||
            a.num_pages != b.num_pages || a.kind != b.kind || a.k_page != b.k_page || a.k_head != b.k_head ||
            a.k_row != b.k_row || a.v_page != b.v_page || a.v_head != b.v_head || a.v_row != b.v_row)
            return fail("the caches differ in shape, type or strides");
        if (!b.k || !b.v || (((uintptr_t)b.k | (uintptr_t)b.v) & 15))
            return fail("NULL pages, or pages not 16-byte aligned");
    }
    return VGX_OK;
}

}  // namespace

extern "C" {

int vgx_tree_masks(vgx_ctx* ctx, const vgx_ragged* batch, const int* parent, int window, int words, int* depth,
                   uint64_t* see) {
    auto fail = [](int status, const char* what) { return vgx_fail(status, std::string("vgx_tree_masks: ") + what); };
    PagedDev A{};
    const int st = rows_fill("vgx_tree_masks", batch, &A);
    if (st != VGX_OK) return st;
    if (words <= 0 || words > kTreeWords) return fail(VGX_EINVAL, "a tree's masks are 1 to 16 words a row");
    if (A.max_q > 64 * words) return fail(VGX_ERANGE, "max_q past the rows that a tree's masks hold");
    if (window < 0) return fail(VGX_EINVAL, "a negative window");
    if (A.ntok && (!parent || !depth || !see)) return fail(VGX_EINVAL, "NULL parent, depth or see");
    if (!ctx) return fail(VGX_EINVAL, "no context");
    if (A.ntok == 0 || A.nseq == 0) return VGX_OK;
    VGX_HIP(hipSetDevice(ctx->device));
    hipLaunchKernelGGL(tree_masks_kernel, dim3(A.nseq, (A.max_q + 63) / 64), dim3(64), 0, ctx->stream, A, parent, window,
                       words, depth, see);
    VGX_LAUNCH_CHECK("tree masks launch");
    return VGX_OK;
}

int vgx_tree_accept(vgx_ctx* ctx, const vgx_ragged* batch, const int* parent, const int* tokens, const int* chosen,
                    int* path, int* accepted, int* next) {
    auto fail = [](int status, const char* what) { return vgx_fail(status, std::string("vgx_tree_accept: ") + what); };
    PagedDev A{};
    const int st = rows_fill("vgx_tree_accept", batch, &A);
    if (st != VGX_OK) return st;
    if (A.max_q > kTreeRows) return fail(VGX_ERANGE, "max_q past 1024 rows");
    if (A.nseq && (!accepted || !next)) return fail(VGX_EINVAL, "NULL accepted or next");
    if (A.nseq && A.ntok && (!parent || !tokens || !chosen || !path))
        return fail(VGX_EINVAL, "NULL parent, tokens, chosen or path");
    if (!ctx) return fail(VGX_EINVAL, "no context");
    if (A.nseq == 0) return VGX_OK;
    VGX_HIP(hipSetDevice(ctx->device));
    hipLaunchKernelGGL(tree_accept_kernel, dim3(A.nseq), dim3(64), 0, ctx->stream, A, parent, tokens, chosen, path,
                       accepted, next);
    VGX_LAUNCH_CHECK("tree accept launch");
    return VGX_OK;
}

int vgx_paged_keep(vgx_ctx* ctx, int ncache, const vgx_paged* caches, const vgx_ragged* batch, const int* path,
                   const int* accepted) {
    auto fail = [](int status, const char* what) { return vgx_fail(status, std::string("vgx_paged_keep: ") + what); };
    KeepArgs P{};
    int st = layers_check("vgx_paged_keep", ncache, caches);
    if (st == VGX_OK) st = vgx_paged_fill("vgx_paged_keep", caches, batch, &P.A);
    if (st != VGX_OK) return st;
    const PagedDev& A = P.A;
    if (A.nseq && A.ntok && (!path || !accepted)) return fail(VGX_EINVAL, "NULL path or accepted");
    P.path = path;
    P.accepted = accepted;
    P.ppr = A.hd * elem_bytes(caches->kind) / 16;
    P.pieces = A.kvh * P.ppr;
    const int threads = P.pieces <= 64 ? 64 : P.pieces <= 128 ? 128 : 256;
    const int64_t blocks = (P.pieces + threads - 1) / threads;
    if (blocks * A.nseq >= (1 << 24) / (2 * kLayers)) return fail(VGX_ERANGE, "too many sequences");  // 2^32 threads
    if (!ctx) return fail(VGX_EINVAL, "no context");
    if (A.nseq == 0 || A.ntok == 0) return VGX_OK;
    VGX_HIP(hipSetDevice(ctx->device));
    for (int l0 = 0; l0 < ncache; l0 += kLayers) {
        const int n = std::min(kLayers, ncache - l0);
        for (int l = 0; l < n; ++l) {
            P.L.p[2 * l] = static_cast<uint8_t*>(caches[l0 + l].k);
            P.L.p[2 * l + 1] = static_cast<uint8_t*>(caches[l0 + l].v);
        }
        hipLaunchKernelGGL(keep_kernel, dim3(A.nseq, (unsigned)blocks, 2 * n), dim3(threads), 0, ctx->stream, P);
        VGX_LAUNCH_CHECK("paged keep launch");
    }
    return VGX_OK;
}

int vgx_paged_copy(vgx_ctx* ctx, int ncache, const vgx_paged* caches, int n, const int* src, const int* dst,
                   const int* rows, int* fault) {
    auto fail = [](int status, const char* what) { return vgx_fail(status, std::string("vgx_paged_copy: ") + what); };
    PagedDev A{};
    int st = layers_check("vgx_paged_copy", ncache, caches);
    if (st == VGX_OK) st = vgx_cache_fill("vgx_paged_copy", caches, &A);
    if (st != VGX_OK) return st;
    if (n < 0 || n > (1 << 20)) return fail(VGX_EINVAL, "pages outside 0..2^20");
    if (n && (!src || !dst)) return fail(VGX_EINVAL, "NULL src or dst");
    CopyArgs P{};
    const int ppr = A.hd * elem_bytes(caches->kind) / 16;
    P.s[0] = PageSide{A.kpg, A.khd, A.krow, A.kvh, ppr};
    P.s[1] = PageSide{A.vpg, A.vhd, A.vrow, A.kvh, ppr};
    int blocks = 1;
    int64_t most = 0;
    for (PageSide& s : P.s) {
        if (s.head == (int64_t)s.ppr * 16 || s.heads == 1) { s.ppr *= s.heads; s.heads = 1; }
        blocks = std::max(blocks, s.heads);
        most = std::max(most, (int64_t)A.psize * s.ppr);
    }
    if (most > INT32_MAX) return fail(VGX_ERANGE, "pages too large");
    const bool dense = P.s[0].row == P.s[0].ppr * 16 && P.s[1].row == P.s[1].ppr * 16;
    P.npages = A.npages;
    P.psize = A.psize;
    P.fault = fault;
    const int64_t chunks = (most + 256 * kCopyPer - 1) / (256 * kCopyPer);
    if (chunks * blocks > 65535) return fail(VGX_ERANGE, "pages too large");
    if (!ctx) return fail(VGX_EINVAL, "no context");
    if (n == 0) return VGX_OK;
    P.chunks = (int)chunks;
    VGX_HIP(hipSetDevice(ctx->device));
    for (int l0 = 0; l0 < ncache; l0 += kLayers) {
        const int m = std::min(kLayers, ncache - l0);
        for (int l = 0; l < m; ++l) {
            P.L.p[2 * l] = static_cast<uint8_t*>(caches[l0 + l].k);
            P.L.p[2 * l + 1] = static_cast<uint8_t*>(caches[l0 + l].v);
        }
        // (a launch has fewer than 2^32 threads)
        const int per = (int)std::max<int64_t>(((1 << 24) - 1) / (chunks * blocks * 2 * m), 1);
        for (int i = 0; i < n; i += per) {
            P.src = src + i;
            P.dst = dst + i;
            P.rows = rows ? rows + i : nullptr;
            hipLaunchKernelGGL(dense ? copy_kernel<true> : copy_kernel<false>, dim3(std::min(per, n - i), (unsigned)(chunks * blocks), 2 * m), dim3(256), 0,
                               ctx->stream, P);
            VGX_LAUNCH_CHECK("paged copy launch");
        }
    }
    return VGX_OK;
}

}  // extern "C"
