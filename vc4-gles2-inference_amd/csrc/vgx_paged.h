// What the kernels over a paged KV cache share: the cache and batch as a
// launch carries them, and a row's or tile's place in the batch.
#pragma once

#include "vgx_internal.h"

struct PagedDev {
    uint8_t* k;
    uint8_t* v;
    int64_t kpg, khd, krow, vpg, vhd, vrow;  // bytes
    int heads, kvh, grp, hd;
    int psize, npages;
    unsigned pmul, psh;  // j / psize for 0 <= j < 2^31 (page_of)
    float kstep, vstep;
    // the batch
    int nseq, ntok, max_q, max_kv, tcols;
    int64_t tstride;
    const int* qstart;
    const int* kvlen;
    const int* table;
    int* fault;
};

// Checks the two descriptions (no device needed) and fills d.
int vgx_paged_fill(const char* who, const vgx_paged* c, const vgx_ragged* b, PagedDev* d);

inline int elem_bytes(int kind) { return kind == VGX_E_F32 ? 4 : kind == VGX_E_Q8 ? 1 : 2; }
inline int compute_kind(int cache_kind) { return cache_kind == VGX_E_BF16 ? VGX_E_BF16 : VGX_E_F16; }

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// j / psize by a multiplication (pmul 0: psize is 1).
__device__ __forceinline__ int page_of(const PagedDev& A, int j) {
    return A.pmul ? (int)(__umulhi((unsigned)j, A.pmul) >> A.psh) : j;
}

__device__ __forceinline__ void set_fault(const PagedDev& A, int bit) {
    if (A.fault) atomicOr(A.fault, bit);
}

// A sequence's rows and length, held inside what was promised: first row,
// number of rows, length (negative lengths count as 0).
struct SeqAt {
    int q0, n, kv;
    bool ok;  // false: a length outside the bounds
};
__device__ __forceinline__ SeqAt seq_at(const PagedDev& A, int s) {
    SeqAt r;
    const int a = A.qstart[s], b = A.qstart[s + 1], kv = A.kvlen[s];
    r.q0 = min(max(a, 0), A.ntok);
    r.n = min(max(min(b, A.ntok) - r.q0, 0), A.max_q);
    r.kv = min(max(kv, 0), A.max_kv);
    r.ok = a >= 0 && b >= a && b <= A.ntok && b - a <= A.max_q && kv >= 0 && kv <= A.max_kv;
    return r;
}

// The sequence that row t belongs to: the number of sequences that end at or
// before t (nseq: behind the last).  Every lane of the wave is active; the
// lanes count 64 sequences a load.
__device__ __forceinline__ int seq_of_row(const PagedDev& A, int t) {
    const int lane = threadIdx.x & 63;
    int s = 0;
    for (int b = 0; b < A.nseq; b += 64) {
        const int j = b + lane;
        const int e = j < A.nseq ? A.qstart[j + 1] : 0x7fffffff;
        s += __popcll(__ballot(e <= t));
    }
    return s;
}

// The positions a tile of a sequence's rows attends to, cut into splits:
// [lo, hi), a split's length and their number (at least 1).  first, last: the
// tile's rows.  lo is a multiple of 64, so a tile of keys never starts inside a
// page that its neighbour's tile also starts in.  Splits are split_len long, or
// where that would make more than 2^sh, a multiple of 128 that does not (sh 31:
// split_len is enough, and 128 or more).
struct Span {
    int lo, hi, len, nsp;
};
__device__ __forceinline__ Span span_of(const SeqAt& q, int first, int last, int window, int split_len, int sh = 31) {
    Span r;
    const int base = q.kv - q.n;
    r.hi = max(min(q.kv, base + last + 1), 0);
    r.lo = window > 0 ? max(base + first - window + 1, 0) & ~63 : 0;
    r.lo = min(r.lo, r.hi);
    const int n = max(r.hi - r.lo, 1);
    r.len = max(split_len, (((n - 1) >> sh >> 7) + 1) << 7);
    r.nsp = (int)(((unsigned)n + (unsigned)r.len - 1) / (unsigned)r.len);
    return r;
}
