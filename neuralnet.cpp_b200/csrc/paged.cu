// Writing into the paged cache: new tokens' rows (nnb200_paged_append) and the states of chosen beams (nnb200_beam_reorder).
#include "paged.cuh"

namespace nnb {

// ---------------------------------------------------------------- append
// For each new token: k, q rotated to the token's position, k and v rounded once to the cache's type and stored at the
// token's row of its sequence's pages, q to q_out.  x[j] <- x[j] c - x[j+h/2] s, x[j+h/2] <- x[j+h/2] c + x[j] s, as rope_apply.
// A thread takes VEC columns of one head's first half and the same columns of the second half, 16 bytes of the narrower type at a
// time where alignment allows.  Bound by memory where there is work: 8192 tokens of 16 heads of 64, fp32 into bf16, 27.8 us, 5450
// GB/s; eight tokens of 12 heads take 2.0 us, a launch.
struct AppendArgs {
    const void *q, *k, *v;
    void* q_out;
    long long ldq, ldqo, ldkv;
    const int *seq_of, *row_of, *table, *rope_pos;
    const float* rope;
    int tokens, heads, seqs, table_stride, rope_len;
};

template <typename T, int N> __device__ __forceinline__ void load_vec(const T* p, float (&x)[N])
{
    constexpr int BYTES = N * sizeof(T) >= 16 ? 16 : N * static_cast<int>(sizeof(T));
    constexpr int PER = BYTES / sizeof(T);
#pragma unroll
    for (int i = 0; i < N; i += PER) {
        alignas(16) T t[PER];
        if constexpr (BYTES == 16) *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(p + i);
        else if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(t) = *reinterpret_cast<const uint2*>(p + i);
        else t[0] = p[i];
#pragma unroll
        for (int j = 0; j < PER; ++j) x[i + j] = to_f32(t[j]);
    }
}
template <typename T, int N> __device__ __forceinline__ void store_vec(T* p, const float (&x)[N])
{
    constexpr int BYTES = N * sizeof(T) >= 16 ? 16 : N * static_cast<int>(sizeof(T));
    constexpr int PER = BYTES / sizeof(T);
#pragma unroll
    for (int i = 0; i < N; i += PER) {
        alignas(16) T t[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) t[j] = from_f32<T>(x[i + j]);
        if constexpr (BYTES == 16) *reinterpret_cast<uint4*>(p + i) = *reinterpret_cast<const uint4*>(t);
        else if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(p + i) = *reinterpret_cast<const uint2*>(t);
        else p[i] = t[0];
    }
}

template <typename TS, typename T, int VEC>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedPool<T> pool, AppendArgs a)
{
    const int half = pool.dk / 2, vph = half / VEC, parts = a.heads + 2 * pool.kv_heads, per_token = parts * vph;
    const long long items = static_cast<long long>(a.tokens) * per_token;
    for (long long w = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; w < items; w += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int tok = static_cast<int>(w / per_token), r = static_cast<int>(w - static_cast<long long>(tok) * per_token);
        const int part = r / vph, j = (r - part * vph) * VEC;
        const bool is_q = part < a.heads, is_k = !is_q && part < a.heads + pool.kv_heads;
        if (is_q && !a.q) continue;
        const int h = is_q ? part : (is_k ? part - a.heads : part - a.heads - pool.kv_heads);
        const TS* src = is_q ? static_cast<const TS*>(a.q) + tok * a.ldq : static_cast<const TS*>(is_k ? a.k : a.v) + tok * a.ldkv;
        src += static_cast<long long>(h) * pool.dk + j;
        float lo[VEC], hi[VEC];                                 // on their way while the row's place is looked up
        load_vec<TS, VEC>(src, lo);
        load_vec<TS, VEC>(src + half, hi);
        const int seq = a.seq_of ? a.seq_of[tok] : tok, row = a.row_of[tok];
        if (seq < 0 || seq >= a.seqs || row < 0 || (row >> pool.page_shift) >= a.table_stride) continue;
        const int page = a.table[static_cast<long long>(seq) * a.table_stride + (row >> pool.page_shift)];
        const int pos = a.rope_pos ? a.rope_pos[tok] : row;
        if (page < 0 || page >= pool.pages || (a.rope && (pos < 0 || pos >= a.rope_len))) continue;
        if (a.rope && (is_q || is_k)) {
            const float* cs = a.rope + static_cast<long long>(pos) * half + j;
            const float* sn = cs + static_cast<long long>(a.rope_len) * half;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float x = lo[i], y = hi[i], c = cs[i], s = sn[i];
                lo[i] = x * c - y * s;
                hi[i] = y * c + x * s;
            }
        }
        T* dst = is_q ? static_cast<T*>(a.q_out) + tok * a.ldqo + static_cast<long long>(h) * pool.dk
                      : (is_k ? pool.k : pool.v) + pool.at(page, h, row & ((1 << pool.page_shift) - 1));
        store_vec<T, VEC>(dst + j, lo);
        store_vec<T, VEC>(dst + j + half, hi);
    }
}

template <typename TS, typename T>
static int append_t(const nnb200_paged_kv& kv, int layer, const AppendArgs& a, cudaStream_t s)
{
    const PagedPool<T> pool = paged_pool<T>(kv, layer);
    const int half = kv.head_dim / 2, parts = a.heads + 2 * kv.kv_heads;
    auto aligned = [](const void* p, long long ld, size_t es) { return !p || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * es % 16 == 0); };
    const bool vec = aligned(a.q, a.ldq, sizeof(TS)) && aligned(a.q_out, a.ldqo, sizeof(T)) && aligned(a.k, a.ldkv, sizeof(TS)) && aligned(a.v, a.ldkv, sizeof(TS));
    auto go = [&](auto* kernel, int v) {
        kernel<<<grid_for(static_cast<long long>(a.tokens) * parts * (half / v), 256), 256, 0, s>>>(pool, a);
        NNB_LAUNCH_CHECK();
        return 0;
    };
    if (!vec) return go(paged_append_kernel<TS, T, 1>, 1);
    if (sizeof(T) == 2 && half % 8 == 0) return go(paged_append_kernel<TS, T, 8>, 8);
    return go(paged_append_kernel<TS, T, 4>, 4);
}

// ---------------------------------------------------------------- reorder
// The state of slot b becomes that of its parent p: whole pages, which nobody writes any more, by copying table entries; the
// page that is partly filled, which both slots will go on writing, by copying its rows into the slot's spare page.  Everything
// is read from the old tables and written to new ones and to pages that no old table names, so no order matters.  A block each
// for a slot's and layer's keys and values.  Bound by memory: 192 slots of 16 layers of 8 bf16 heads of 128, 30 rows of a page of 32 each, 104 us, 755 MB read and written
// (parents that several slots share are read from L2); eight slots of 12 layers 4.1 us, a launch and a few trips to memory.  With keys
// and values in one block and a vector at a time they took 113 and 6.1 us.
struct ReorderArgs {
    const int *parent, *len, *table, *spare;
    int *len_out, *table_out, *spare_out;
    int beams, table_stride;
};

template <typename T>
__global__ void __launch_bounds__(256) beam_reorder_kernel(PagedPool<T> pool, long long layer_stride, ReorderArgs a)
{
    const int slot = blockIdx.x, layer = blockIdx.y, base = slot / a.beams * a.beams;
    int p = a.parent[slot];
    p = p < 0 || p >= a.beams ? slot : base + p;
    const int ps = 1 << pool.page_shift;
    const long long cap = static_cast<long long>(a.table_stride) << pool.page_shift;
    const int len = static_cast<int>(min(static_cast<long long>(max(a.len[p], 0)), cap)), full = len >> pool.page_shift, rest = len & (ps - 1);
    const int* from = a.table + static_cast<long long>(p) * a.table_stride;
    const int* mine = a.table + static_cast<long long>(slot) * a.table_stride;
    const int spare = a.spare[slot];
    if (layer == 0 && blockIdx.z == 0) {
        int* to = a.table_out + static_cast<long long>(slot) * a.table_stride;
        for (int j = threadIdx.x; j < a.table_stride; j += blockDim.x) to[j] = j < full ? from[j] : (j == full && rest ? spare : mine[j]);
        if (threadIdx.x == 0) {
            a.len_out[slot] = a.len[p];
            a.spare_out[slot] = rest ? mine[full] : spare;
        }
    }
    if (rest == 0) return;
    const int src = from[full];
    if (src < 0 || src >= pool.pages || spare < 0 || spare >= pool.pages || src == spare) return;
    constexpr int N = Vec16<T>::N;
    const int per_head = rest * pool.dk / N, all = per_head * pool.kv_heads;       // head_dim is a whole number of 16-byte vectors
    constexpr int U = 4;                                        // vectors of a thread on their way at a time
    T* const pages = (blockIdx.z == 0 ? pool.k : pool.v) + layer * layer_stride;
    for (int w0 = threadIdx.x; w0 < all; w0 += U * blockDim.x) {
        Vec16<T> v[U];
        T* to[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = w0 + u * blockDim.x, h = i / per_head, e = (i - h * per_head) * N;
            if (i >= all) { to[u] = nullptr; continue; }
            to[u] = pages + pool.at(spare, h, 0) + e;
            v[u] = ld16(pages + pool.at(src, h, 0) + e);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) if (to[u]) st16(to[u], v[u]);
    }
}

template <typename T>
static int reorder_t(const nnb200_paged_kv& kv, int slots, const ReorderArgs& a, cudaStream_t s)
{
    beam_reorder_kernel<T><<<dim3(static_cast<unsigned>(slots), static_cast<unsigned>(kv.layers), 2), 256, 0, s>>>(paged_pool<T>(kv, 0), kv.layer_stride, a);
    NNB_LAUNCH_CHECK();
    return 0;
}

}  // namespace nnb

using namespace nnb;

extern "C" {

int nnb200_paged_append(const nnb200_paged_kv* kv, int layer, const void* q, long long ldq, void* q_out, long long ldqo, const void* k, const void* v,
                        long long ldkv, int src_dtype, int tokens, int heads, const int32_t* seq_of, const int32_t* row_of, const int32_t* page_table,
                        int seqs, int table_stride, const float* rope, int rope_len, const int32_t* rope_pos, void* stream)
{
    NNB_KV_CHECK(kv);
    NNB_ARG_CHECK(layer >= 0 && layer < kv->layers, "layer out of range");
    NNB_ARG_CHECK(src_dtype == 0 || src_dtype == 1, "dtype must be 0 (fp32) or 1 (bf16)");
    NNB_ARG_CHECK(tokens >= 0 && seqs >= 0 && table_stride >= 0 && heads >= 0, "negative size");
    NNB_ARG_CHECK(heads <= 65535 && table_stride <= INT_MAX / 256, "too many heads, or a page table too wide");
    if (tokens == 0) return 0;
    NNB_ARG_CHECK(k && v && row_of && page_table, "null keys, values, rows or page table");
    NNB_ARG_CHECK(!q == !q_out, "queries need a place to go, and the other way round");
    NNB_ARG_CHECK(!q || heads > 0, "queries without heads");
    NNB_ARG_CHECK(seq_of || tokens <= seqs, "without seq_of token i belongs to sequence i: more tokens than sequences");
    const long long wide = static_cast<long long>(heads) * kv->head_dim, kv_wide = static_cast<long long>(kv->kv_heads) * kv->head_dim;
    NNB_ARG_CHECK(ldkv >= kv_wide && (!q || (ldq >= wide && ldqo >= wide)), "a row stride shorter than a row");
    NNB_ARG_CHECK(q != q_out || !q || (src_dtype == kv->dtype && ldq == ldqo), "queries rotated in place need the cache's type and one stride");
    NNB_ARG_CHECK(!rope || rope_len > 0, "an empty rotation table");
    AppendArgs a{q, k, v, q_out, ldq, ldqo, ldkv, seq_of, row_of, page_table, rope_pos, rope, tokens, q ? heads : 0, seqs, table_stride, rope_len};
    const cudaStream_t s = to_stream(stream);
    if (kv->dtype == 0) return src_dtype == 0 ? append_t<float, float>(*kv, layer, a, s) : append_t<bf16, float>(*kv, layer, a, s);
    return src_dtype == 0 ? append_t<float, bf16>(*kv, layer, a, s) : append_t<bf16, bf16>(*kv, layer, a, s);
}

int nnb200_beam_reorder(const nnb200_paged_kv* kv, int groups, int beams, const int32_t* parent, const int32_t* len, const int32_t* page_table,
                        const int32_t* spare, int32_t* len_out, int32_t* page_table_out, int32_t* spare_out, int table_stride, void* stream)
{
    NNB_KV_CHECK(kv);
    NNB_ARG_CHECK(groups >= 0 && beams >= 0 && table_stride >= 0, "negative size");
    NNB_ARG_CHECK(static_cast<long long>(groups) * beams <= INT_MAX && table_stride <= INT_MAX / 256 && kv->layers <= 65535, "too many beams or layers, or a page table too wide");
    if (groups == 0 || beams == 0) return 0;
    NNB_ARG_CHECK(parent && len && spare && len_out && spare_out && (table_stride == 0 || (page_table && page_table_out)), "null argument");
    NNB_ARG_CHECK(len != len_out && spare != spare_out && (table_stride == 0 || page_table != page_table_out), "the new tables must not be the old ones");
    ReorderArgs a{parent, len, page_table, spare, len_out, page_table_out, spare_out, beams, table_stride};
    const cudaStream_t s = to_stream(stream);
    if (kv->dtype == 0) return reorder_t<float>(*kv, groups * beams, a, s);
    return reorder_t<bf16>(*kv, groups * beams, a, s);
}

}  // extern "C"
