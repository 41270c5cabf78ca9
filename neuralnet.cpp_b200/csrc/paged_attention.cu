// Attention of batched decoding: one new query per sequence over the rows of a paged cache, first the prefix that the
// sequences of a group share, then the sequence's own rows (nnb200_paged_attention).
//   s_t = q . k_t / sqrt(dk) - slope_h (T - 1 - t),  out = sum_t softmax(s)_t v_t,  lse = log sum_t exp(s_t)
// with t over the T = prefix_len + seq_len rows the query sees; a query for which no row has weight (it sees none, or all
// its scores are -inf) gives 0 and -inf.
#include "paged.cuh"

namespace nnb {

struct PagedAttnArgs {
    const void* q;
    void* out;
    float* lse;
    long long ldq, ldo;
    const int *prefix_table, *prefix_len, *table, *len;
    int prefix_stride, table_stride, groups, size, heads, alibi;
};

// A block per (sequence, query head): warps take rows in turn, a lane every 32nd column, partial softmax states joined at the end.
template <typename T>
__global__ void __launch_bounds__(128) paged_attn_kernel(PagedPool<T> pool, PagedAttnArgs a, float scale)
{
    constexpr int C = 8, WARPS = 4;
    const int seq = blockIdx.x, h = blockIdx.y, hk = h / (a.heads / pool.kv_heads), g = seq / a.size;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dk = pool.dk, ps = 1 << pool.page_shift;
    const int own = a.table_stride ? a.len[seq] : min(a.len[seq], 0);
    const long long own_cap = static_cast<long long>(a.table_stride) << pool.page_shift, pre_cap = static_cast<long long>(a.prefix_stride) << pool.page_shift;
    const int n_own = static_cast<int>(min(static_cast<long long>(max(own, 0)), own_cap));
    const int n_pre = own < 0 || !a.prefix_stride ? 0 : static_cast<int>(min(static_cast<long long>(max(a.prefix_len[g], 0)), pre_cap));
    const T* qp = static_cast<const T*>(a.q) + seq * a.ldq + static_cast<long long>(h) * dk;
    float q[C], o[C], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) { const int c = lane + 32 * i; q[i] = c < dk ? to_f32(qp[c]) : 0.f; o[i] = 0.f; }
    const float slope = a.alibi ? exp2f(-8.0f * static_cast<float>(h) / static_cast<float>(a.heads)) : 0.f;
    const int total = n_pre + n_own;
    for (int t = warp; t < total; t += WARPS) {
        const int r = t < n_pre ? t : t - n_pre;
        const int* table = t < n_pre ? a.prefix_table + static_cast<long long>(g) * a.prefix_stride : a.table + static_cast<long long>(seq) * a.table_stride;
        const int page = table[r >> pool.page_shift];
        if (page < 0 || page >= pool.pages) continue;
        const long long at = pool.at(page, hk, r & (ps - 1));
        float s = 0.f, v[C];
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = lane + 32 * i;
            if (c < dk) s = fmaf(q[i], to_f32(pool.k[at + c]), s);
            v[i] = c < dk ? to_f32(pool.v[at + c]) : 0.f;
        }
        s = warp_sum(s) * scale - slope * static_cast<float>(total - 1 - t);
        const float nm = fmaxf(m, s), ref = nm == -INFINITY ? 0.f : nm, back = expf(m - ref), e = expf(s - ref);
        m = nm;
        l = l * back + e;
#pragma unroll
        for (int i = 0; i < C; ++i) o[i] = fmaf(e, v[i], o[i] * back);
    }
    __shared__ float sm[WARPS], sl[WARPS], so[WARPS][256];
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
    for (int i = 0; i < C; ++i) so[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float gm = -INFINITY, gl = 0.f;
    for (int w = 0; w < WARPS; ++w) gm = fmaxf(gm, sm[w]);
    const float ref = gm == -INFINITY ? 0.f : gm;
    for (int w = 0; w < WARPS; ++w) gl += sl[w] * expf(sm[w] - ref);
    for (int c = threadIdx.x; c < dk; c += blockDim.x) {
        float x = 0.f;
        for (int w = 0; w < WARPS; ++w) x = fmaf(so[w][c], expf(sm[w] - ref), x);
        static_cast<T*>(a.out)[seq * a.ldo + static_cast<long long>(h) * dk + c] = from_f32<T>(gl == 0.f ? 0.f : x / gl);
    }
    if (a.lse && threadIdx.x == 0) a.lse[static_cast<long long>(seq) * a.heads + h] = ref + logf(gl);
}

template <typename T>
static int attention_t(const nnb200_paged_kv& kv, int layer, const PagedAttnArgs& a, cudaStream_t s)
{
    const dim3 grid(static_cast<unsigned>(a.groups * a.size), static_cast<unsigned>(a.heads));
    paged_attn_kernel<T><<<grid, 128, 0, s>>>(paged_pool<T>(kv, layer), a, 1.0f / sqrtf(static_cast<float>(kv.head_dim)));
    NNB_LAUNCH_CHECK();
    return 0;
}

static const char* attention_shape_error(const nnb200_paged_kv* kv, int groups, int group_size, int heads, int prefix_stride, int table_stride)
{
    if (const char* e = paged_kv_error(kv)) return e;
    if (groups < 0 || group_size < 0 || prefix_stride < 0 || table_stride < 0) return "negative size";
    if (heads < 1 || heads > 65535 || heads % kv->kv_heads) return "heads must be a multiple of the cache's heads, up to 65535";
    if (static_cast<long long>(groups) * group_size * heads > INT_MAX / 512) return "too many queries for one call";
    if (prefix_stride > INT_MAX / 512 || table_stride > INT_MAX / 512) return "a page table too wide";
    return nullptr;
}

}  // namespace nnb

using namespace nnb;

extern "C" {

size_t nnb200_paged_attention_scratch_bytes(const nnb200_paged_kv* kv, int groups, int group_size, int heads, int prefix_stride, int table_stride)
{
    if (const char* e = attention_shape_error(kv, groups, group_size, heads, prefix_stride, table_stride)) {
        fprintf(stderr, "nnb200: %s: %s\n", __func__, e);
        return 0;
    }
    return 16;
}

int nnb200_paged_attention(const nnb200_paged_kv* kv, int layer, const void* q, long long ldq, void* out, long long ldo, float* lse,
                           const int32_t* prefix_table, int prefix_stride, const int32_t* prefix_len, const int32_t* page_table, int table_stride,
                           const int32_t* seq_len, int groups, int group_size, int heads, int alibi, void* scratch, size_t scratch_bytes, void* stream)
{
    const char* e = attention_shape_error(kv, groups, group_size, heads, prefix_stride, table_stride);
    NNB_ARG_CHECK(!e, e);
    NNB_ARG_CHECK(layer >= 0 && layer < kv->layers, "layer out of range");
    if (groups == 0 || group_size == 0) return 0;
    NNB_ARG_CHECK(q && out && seq_len, "null queries, output or lengths");
    NNB_ARG_CHECK(prefix_stride == 0 || (prefix_table && prefix_len), "a prefix needs its page table and lengths");
    NNB_ARG_CHECK(table_stride == 0 || page_table, "null page table");
    NNB_ARG_CHECK(ldq >= static_cast<long long>(heads) * kv->head_dim && ldo >= static_cast<long long>(heads) * kv->head_dim, "a row stride shorter than a row");
    NNB_ARG_CHECK(scratch && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "scratch must be there and start on a 16-byte boundary");
    NNB_ARG_CHECK(scratch_bytes >= nnb200_paged_attention_scratch_bytes(kv, groups, group_size, heads, prefix_stride, table_stride), "scratch too small");
    PagedAttnArgs a{q, out, lse, ldq, ldo, prefix_table, prefix_len, page_table, seq_len, prefix_stride, table_stride, groups, group_size, heads, alibi};
    if (kv->dtype == 0) return attention_t<float>(*kv, layer, a, to_stream(stream));
    return attention_t<bf16>(*kv, layer, a, to_stream(stream));
}

}  // extern "C"
