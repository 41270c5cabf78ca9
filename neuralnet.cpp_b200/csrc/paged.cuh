// Paged key/value cache of batched decoding: what its kernels share.
// A pool of pages holds the rows of many sequences, so that sequences of unlike lengths share one allocation and several of
// them may read the same prompt.  Row t of a sequence is row t % page_size of page table[t / page_size] of its page table.
// A page is (kv_heads, page_size, head_dim): the rows of one head lie together, page_size * head_dim values in a run, which
// is what an attention block (one head) reads and what one bulk or vector copy moves.
// Page numbers and lengths are device data that no host check sees: the kernels take a page number outside the pool for a
// page whose rows do not exist.
#pragma once
#include "common.cuh"
#include "nnb200.h"

namespace nnb {

// the pages of one layer
template <typename T> struct PagedPool {
    T* k;
    T* v;
    int pages, page_shift, kv_heads, dk;
    // rows of one head from the start of the pool to row `row` of head `h` in page `page`: a pool has fewer than 2^31
    __device__ __forceinline__ int row_at(int page, int h, int row) const { return ((page * kv_heads + h) << page_shift) + row; }
    __device__ __forceinline__ long long at(int page, int h, int row) const { return static_cast<long long>(row_at(page, h, row)) * dk; }
    // the same for row t of a page table's sequence; -1 where the page is not there
    __device__ __forceinline__ int find(const int* table, int h, int t) const
    {
        const int page = __ldg(table + (t >> page_shift));
        return static_cast<unsigned>(page) < static_cast<unsigned>(pages) ? row_at(page, h, t & ((1 << page_shift) - 1)) : -1;
    }
};

// quotients of numbers below 2^31 by a divisor fixed on the host: n / d = (n * ceil(2^(32 + s) / d)) >> (32 + s) with 2^s >= d > 2^(s - 1)
// needs 33 bits of the factor; the missing one is added back (the round-up method for unsigned division by an invariant)
struct FastDiv {
    unsigned mul, shift, d;
    FastDiv() = default;
    explicit FastDiv(int divisor)
    {
        d = static_cast<unsigned>(divisor < 1 ? 1 : divisor);
        shift = 0;
        while ((1ull << shift) < d) ++shift;
        mul = static_cast<unsigned>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
#ifdef __CUDACC__
    __device__ __forceinline__ int div(int n) const { return static_cast<int>((__umulhi(static_cast<unsigned>(n), mul) + static_cast<unsigned>(n)) >> shift); }
    // quotient, and the remainder left in n
    __device__ __forceinline__ int split(int& n) const { const int q = div(n); n -= q * static_cast<int>(d); return q; }
#endif
};

inline int log2_of(int n) { int s = 0; while ((1 << s) < n) ++s; return s; }

// message, or null where the description is a usable one
inline const char* paged_kv_error(const nnb200_paged_kv* kv)
{
    if (!kv) return "null cache description";
    if (kv->dtype != 0 && kv->dtype != 1) return "dtype must be 0 (fp32) or 1 (bf16)";
    if (kv->page_size < 8 || kv->page_size > 256 || (kv->page_size & (kv->page_size - 1))) return "page_size must be a power of two from 8 to 256";
    if (kv->head_dim < 8 || kv->head_dim > 256 || kv->head_dim % 8) return "head_dim must be a multiple of 8 from 8 to 256";
    if (kv->kv_heads < 1 || kv->pages < 1 || kv->layers < 1) return "kv_heads, pages and layers must be positive";
    const long long page = static_cast<long long>(kv->kv_heads) * kv->page_size * kv->head_dim;
    if (kv->kv_heads > 65535 || page > INT_MAX) return "a page must have fewer than 2^31 elements and 65536 heads";
    if (static_cast<long long>(kv->pages) * kv->kv_heads * kv->page_size > INT_MAX) return "a layer's pages must hold fewer than 2^31 rows of a head";
    if (kv->layers > 1 && kv->layer_stride < page * kv->pages) return "layer_stride is shorter than a layer's pages";
    if (kv->layers > 1 && kv->layer_stride % 8) return "layer_stride must be a multiple of 8";
    if (!kv->k || !kv->v) return "null pages";
    if ((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v)) & 15) return "the pages must start on a 16-byte boundary";
    return nullptr;
}

template <typename T> inline PagedPool<T> paged_pool(const nnb200_paged_kv& kv, int layer)
{
    return {static_cast<T*>(kv.k) + layer * kv.layer_stride, static_cast<T*>(kv.v) + layer * kv.layer_stride, kv.pages, log2_of(kv.page_size), kv.kv_heads, kv.head_dim};
}

}  // namespace nnb

#define NNB_KV_CHECK(kv)                                                                      \
    do {                                                                                      \
        if (const char* msg__ = nnb::paged_kv_error(kv)) {                                    \
            fprintf(stderr, "nnb200: %s: %s\n", __func__, msg__);                             \
            return -1;                                                                        \
        }                                                                                     \
    } while (0)
