// Several continuations of one prompt a token at a time: the products of a step over all sequences' rows, their keys and values
// in a paged cache (nnb200_paged_append), attention over the prompt, once for all, and each sequence's own rows
// (nnb200_paged_attention).  fp32 activations and cache and fp32 or bf16 weights, as single decoding steps have them (decode.cu).
// What bounds a step of few sequences is the chain of about ten kernels a layer, not the weights they share: 1.0 ms a token with the
// selection and the reordering for 1 to 8 sequences of the 12-layer model of width 768 behind 501 tokens, 1.2 ms for 32.
#include <algorithm>
#include <vector>

#include "kernels.h"
#include "nnb200.h"
#include "paged.cuh"

namespace nnb {

constexpr int kBatchPage = 16;                                  // rows of a page: half of one is copied per reordered sequence on average

struct BatchWs {
    size_t k, v, fixed, state, fresh, x, xn, qkv, att, mid, h1, h2, stat, scratch, scratch_bytes, total;
    int prompt_pages, own_pages;                                // pages of the prompt, of a sequence
    // int32 arrays: prefix table | prefix length | position | row, each sequence's | 0 .. seq - 1 | seq zeros (fixed);
    // table | spare page | length (state, fresh)
    size_t fixed_ints, state_ints;
};
static nnb200_paged_kv batch_pool(const nnb200_gpt_config& c, const BatchWs& W, int seqs, uint8_t* ws)
{
    nnb200_paged_kv kv = {};
    kv.pages = W.prompt_pages + seqs * (W.own_pages + 1);
    kv.page_size = kBatchPage; kv.kv_heads = c.heads; kv.head_dim = c.d_model / c.heads; kv.dtype = 0; kv.layers = c.layers;
    kv.layer_stride = static_cast<int64_t>(kv.pages) * kBatchPage * c.d_model;
    kv.k = ws + W.k;
    kv.v = ws + W.v;
    return kv;
}
static BatchWs batch_ws(const nnb200_gpt_config& c, int seqs, int new_rows)
{
    BatchWs W;
    const size_t d = c.d_model, n = seqs, fc1 = c.act == 1 ? 2 * static_cast<size_t>(c.d_ff) : c.d_ff;
    W.prompt_pages = static_cast<int>(ceil_div(c.seq, kBatchPage));
    W.own_pages = static_cast<int>(ceil_div(new_rows, kBatchPage));
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off = (off + bytes + 255) / 256 * 256; return o; };
    const size_t pool = static_cast<size_t>(c.layers) * (W.prompt_pages + n * (W.own_pages + 1)) * kBatchPage * d * 4;
    W.k = take(pool); W.v = take(pool);
    W.fixed_ints = W.prompt_pages + 1 + 2 * n + 2 * static_cast<size_t>(c.seq);
    W.state_ints = n * (W.own_pages + 2);
    W.fixed = take(W.fixed_ints * 4); W.state = take(W.state_ints * 4); W.fresh = take(W.state_ints * 4);
    W.x = take(n * d * 4); W.xn = take(n * d * 4); W.qkv = take(n * 3 * d * 4); W.att = take(n * d * 4); W.mid = take(n * d * 4);
    W.h1 = take(n * fc1 * 4); W.h2 = take(n * c.d_ff * 4); W.stat = take(2 * n * 4);
    uint8_t* nowhere = reinterpret_cast<uint8_t*>(256);         // the size of the scratch does not depend on where things are
    const nnb200_paged_kv kv = batch_pool(c, W, seqs, nowhere);
    W.scratch_bytes = nnb200_paged_attention_scratch_bytes(&kv, 1, seqs, c.heads, W.prompt_pages, W.own_pages);
    W.scratch = take(W.scratch_bytes);
    W.total = off;
    return W;
}

// page tables, spare pages and lengths of sequences without rows; row and sequence numbers to append the prompt by
__global__ void batch_begin_kernel(int* fixed, int* state, int seqs, int prompt_pages, int own_pages, int prompt_len, int seq)
{
    const int i0 = blockIdx.x * blockDim.x + threadIdx.x, stride = gridDim.x * blockDim.x;
    for (int i = i0; i < prompt_pages; i += stride) fixed[i] = i;
    if (i0 == 0) fixed[prompt_pages] = prompt_len;
    int* rows = fixed + prompt_pages + 1 + 2 * seqs;
    for (int i = i0; i < seq; i += stride) { rows[i] = i; rows[seq + i] = 0; }
    for (int i = i0; i < seqs * own_pages; i += stride) state[i] = prompt_pages + i;
    for (int i = i0; i < seqs; i += stride) { state[seqs * own_pages + i] = prompt_pages + seqs * own_pages + i; state[seqs * (own_pages + 1) + i] = 0; }
}
// every sequence's next row is `row` of its own, at the position behind the prompt and the rows before it
__global__ void batch_row_kernel(const int* prompt_len, int* pos, int* row, int* len, int seqs, int at)
{
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < seqs) { pos[i] = prompt_len[0] + at; row[i] = at; len[i] = at + 1; }
}

template <typename WT>
static int batch_step_t(const nnb200_gpt_config& c, const float* P, const WT* Wt, const uint8_t* decode, uint8_t* ws, int seqs, int new_rows, int step, int prompt_len,
                        const int* tokens, float* logits, cudaStream_t s)
{
    const DecodeLayout L = decode_layout(c);
    const BatchWs W = batch_ws(c, seqs, new_rows);
    const int d = c.d_model, ff = c.d_ff, fc1 = c.act == 1 ? 2 * ff : ff;
    const bool ln = c.norm == 0;
    auto F = [&](size_t off) { return reinterpret_cast<float*>(ws + off); };
    auto PB = [&](long long off) { return off >= 0 ? P + off : nullptr; };
    const nnb200_paged_kv kv = batch_pool(c, W, seqs, ws);
    int *prefix_table = reinterpret_cast<int*>(ws + W.fixed), *prefix_len = prefix_table + W.prompt_pages, *pos = prefix_len + 1, *row = pos + seqs;
    int *table = reinterpret_cast<int*>(ws + W.state), *len = table + static_cast<size_t>(seqs) * (W.own_pages + 1);
    const float* tab = reinterpret_cast<const float*>(decode + decode_cache(c).table);
    float *x = F(W.x), *xn = F(W.xn), *qkv = F(W.qkv), *att = F(W.att), *mid = F(W.mid), *h1 = F(W.h1), *h2 = F(W.h2), *rinv = F(W.stat), *mean = rinv + seqs;
    batch_row_kernel<<<static_cast<unsigned>(ceil_div(seqs, 128)), 128, 0, s>>>(prefix_len, pos, row, len, seqs, step);
    NNB_LAUNCH_CHECK();
    const float* pos_table = c.pos == 0 ? P + L.pos_emb : (c.pos == 1 ? tab : nullptr);
    // all tokens stand at one position: its row of the table, for every token
    NNB_TRY(embed_fwd<float>(P + L.tok_emb, pos_table ? pos_table + static_cast<size_t>(prompt_len + step) * d : nullptr, tokens, x, seqs, 1, d, c.vocab, s));
    for (int l = 0; l < c.layers; ++l) {
        const DecodeLayer& lp = L.layers[l];
        NNB_TRY(norm_fwd<float>(x, P + lp.g1, PB(lp.be1), xn, rinv, mean, seqs, d, ln, s));
        NNB_TRY(prompt_linear(xn, Wt + lp.wqkv, P + lp.bqkv, nullptr, qkv, seqs, d, 3 * d, s));
        NNB_TRY(nnb200_paged_append(&kv, l, c.pos == 3 ? qkv : nullptr, 3 * d, c.pos == 3 ? qkv : nullptr, 3 * d, qkv + d, qkv + 2 * d, 3 * d, 0, seqs, c.heads, nullptr, row, table,
                                    seqs, W.own_pages, c.pos == 3 ? tab : nullptr, c.pos == 3 ? c.seq : 0, c.pos == 3 ? pos : nullptr, s));
        NNB_TRY(nnb200_paged_attention(&kv, l, qkv, 3 * d, att, d, nullptr, prefix_table, W.prompt_pages, prefix_len, table, W.own_pages, len, 1, seqs, c.heads,
                                       c.pos == 2 ? 1 : 0, ws + W.scratch, W.scratch_bytes, s));
        NNB_TRY(prompt_linear(att, Wt + lp.wo, P + lp.bo, x, mid, seqs, d, d, s));
        NNB_TRY(norm_fwd<float>(mid, P + lp.g2, PB(lp.be2), xn, rinv, mean, seqs, d, ln, s));
        NNB_TRY(prompt_linear(xn, Wt + lp.w1, P + lp.b1, nullptr, h1, seqs, d, fc1, s));
        NNB_TRY(act_fwd<float>(h1, h2, seqs, ff, c.act == 1, s));
        NNB_TRY(prompt_linear(h2, Wt + lp.w2, P + lp.b2, mid, x, seqs, ff, d, s));
    }
    NNB_TRY(norm_fwd<float>(x, P + L.lnf_g, PB(L.lnf_b), xn, rinv, mean, seqs, d, ln, s));
    return prompt_linear(xn, Wt + L.lm_w, P + L.lm_b, nullptr, logits, seqs, d, c.vocab, s);
}

static const char* batch_error(const nnb200_gpt_config* cfg, int seqs, int new_rows)
{
    if (nnb200_gpt_arena_elems(cfg) < 0) return "bad configuration";
    const int dk = cfg->d_model / cfg->heads;
    if (dk % 8 || dk > 256) return "the head size must be a multiple of 8, up to 256";
    if (seqs < 1 || seqs > 1024) return "1 to 1024 sequences";
    if (new_rows < 1 || new_rows > cfg->seq) return "new rows: from 1 to seq";
    // a layer's pages, counted in rows of a head, and the attention's queries and heads (its own limits)
    if (cfg->heads > 65535 || static_cast<long long>(seqs) * cfg->heads > INT_MAX / 512) return "too many heads for this many sequences";
    const long long pages = ceil_div(cfg->seq, kBatchPage) + static_cast<long long>(seqs) * (ceil_div(new_rows, kBatchPage) + 1);
    if (pages * cfg->heads * kBatchPage > INT_MAX || pages * (ceil_div(new_rows, kBatchPage) + 1) > INT_MAX) return "too many sequences for rows this long";
    return nullptr;
}

}  // namespace nnb

using namespace nnb;

extern "C" {

long long nnb200_gpt_batch_workspace_bytes(const nnb200_gpt_config* cfg, int seqs, int new_rows)
{
    if (const char* e = batch_error(cfg, seqs, new_rows)) { fprintf(stderr, "nnb200: %s: %s\n", __func__, e); return -1; }
    return static_cast<long long>(batch_ws(*cfg, seqs, new_rows).total);
}

int nnb200_gpt_batch_begin(const nnb200_gpt_config* cfg, const void* decode_workspace, void* workspace, int seqs, int new_rows, int prompt_len, void* stream)
{
    const char* e = batch_error(cfg, seqs, new_rows);
    NNB_ARG_CHECK(!e, e);
    NNB_ARG_CHECK(decode_workspace && workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "workspaces must be there, this one on a 256-byte boundary");
    NNB_ARG_CHECK(prompt_len >= 1 && prompt_len <= cfg->seq - new_rows, "the prompt and the new rows must fit into seq");
    const cudaStream_t s = to_stream(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const BatchWs W = batch_ws(*cfg, seqs, new_rows);
    const nnb200_paged_kv kv = batch_pool(*cfg, W, seqs, ws);
    int *fixed = reinterpret_cast<int*>(ws + W.fixed), *state = reinterpret_cast<int*>(ws + W.state), *rows = fixed + W.prompt_pages + 1 + 2 * seqs;
    batch_begin_kernel<<<static_cast<unsigned>(grid_for(std::max<long long>(W.fixed_ints, W.state_ints), 256)), 256, 0, s>>>(fixed, state, seqs, W.prompt_pages, W.own_pages, prompt_len, cfg->seq);
    NNB_LAUNCH_CHECK();
    // the prompt's rows as the decode cache has them, already rotated: the prompt is a sequence of its own, with the prefix table
    // for a page table
    const int d = cfg->d_model;
    const float* cache = reinterpret_cast<const float*>(static_cast<const uint8_t*>(decode_workspace) + decode_cache(*cfg).kv);
    for (int l = 0; l < cfg->layers; ++l) {
        const float* k = cache + static_cast<size_t>(l) * 2 * cfg->seq * d;
        NNB_TRY(nnb200_paged_append(&kv, l, nullptr, 0, nullptr, 0, k, k + static_cast<size_t>(cfg->seq) * d, d, 0, prompt_len, 0, rows + cfg->seq, rows, fixed, 1, W.prompt_pages,
                                    nullptr, 0, nullptr, s));
    }
    return 0;
}

int nnb200_gpt_batch_step(const nnb200_gpt_config* cfg, const float* params, const void* params_bf16, const void* decode_workspace, void* workspace, int seqs,
                          int new_rows, int prompt_len, int step, const int32_t* tokens, float* logits_out, void* stream)
{
    const char* e = batch_error(cfg, seqs, new_rows);
    NNB_ARG_CHECK(!e, e);
    NNB_ARG_CHECK(params && decode_workspace && workspace && tokens && logits_out, "null argument");
    NNB_ARG_CHECK(((reinterpret_cast<uintptr_t>(workspace) & 255) | (reinterpret_cast<uintptr_t>(params) & 15) | (reinterpret_cast<uintptr_t>(logits_out) & 15)) == 0,
                  "the workspace must start on a 256-byte boundary, parameters and logits on a 16-byte one");
    NNB_ARG_CHECK(prompt_len >= 1 && prompt_len <= cfg->seq - new_rows && step >= 0 && step < new_rows, "the prompt and the new rows must fit into seq, and the step into the new rows");
    const uint8_t* dec = static_cast<const uint8_t*>(decode_workspace);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (cfg->precision == 1) {
        NNB_ARG_CHECK(params_bf16 != nullptr, "bf16 mode needs the bf16 parameter shadow");
        return batch_step_t<bf16>(*cfg, params, static_cast<const bf16*>(params_bf16), dec, ws, seqs, new_rows, step, prompt_len, tokens, logits_out, to_stream(stream));
    }
    return batch_step_t<float>(*cfg, params, params, dec, ws, seqs, new_rows, step, prompt_len, tokens, logits_out, to_stream(stream));
}

int nnb200_gpt_batch_reorder(const nnb200_gpt_config* cfg, void* workspace, int seqs, int new_rows, const int32_t* parent, void* stream)
{
    const char* e = batch_error(cfg, seqs, new_rows);
    NNB_ARG_CHECK(!e, e);
    NNB_ARG_CHECK(workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && parent, "null parents, or a workspace that does not start on a 256-byte boundary");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const BatchWs W = batch_ws(*cfg, seqs, new_rows);
    const nnb200_paged_kv kv = batch_pool(*cfg, W, seqs, ws);
    int *old = reinterpret_cast<int*>(ws + W.state), *now = reinterpret_cast<int*>(ws + W.fresh);
    const size_t spare = static_cast<size_t>(seqs) * W.own_pages, len = spare + seqs;
    NNB_TRY(nnb200_beam_reorder(&kv, 1, seqs, parent, old + len, old, old + spare, now + len, now, now + spare, W.own_pages, stream));
    NNB_CUDA_CHECK(cudaMemcpyAsync(old, now, W.state_ints * 4, cudaMemcpyDeviceToDevice, to_stream(stream)));
    return 0;
}

}  // extern "C"
