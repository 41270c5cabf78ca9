// Beam search's selection (nnb200_beam_select): of the continuations (beam b, token v) of a group's beams, valued
//   score_b + logit_bv - log sum_u exp(logit_bu),
// the n best, best first; equal values go to the lower (b, v).
// Which of two continuations is better decides what a program answers, so values are compared in 64 bits: a score and a logit
// are exact, and the normaliser, the only rounded part, is the same for a whole beam.
#include "common.cuh"
#include "nnb200.h"

namespace nnb {

struct SelectArgs {
    const void* logits;
    long long ld;
    int groups, beams, vocab, n, eos;
    const float* scores;
    const int* ended;
    int *parent, *token, *ended_out;
    float* scores_out;
    double* norm;               // (groups * beams): score - log-sum-exp, NaN where the beam offers nothing by its logits
};

template <typename T>
__global__ void __launch_bounds__(256) select_norm_kernel(SelectArgs a)
{
    __shared__ float red[32];
    __shared__ double redd[8];
    const T* x = static_cast<const T*>(a.logits) + blockIdx.x * a.ld;
    float m = -INFINITY;
    bool bad = false;
    for (int i = threadIdx.x; i < a.vocab; i += 256) { const float v = to_f32(x[i]); bad |= !(v < INFINITY); m = fmaxf(m, v); }
    m = block_max(m, red);
    bad = __syncthreads_or(bad) || m == -INFINITY;
    double sum = 0.0;
    if (!bad) for (int i = threadIdx.x; i < a.vocab; i += 256) sum += exp(static_cast<double>(to_f32(x[i])) - m);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) redd[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) sum += redd[w];
        a.norm[blockIdx.x] = bad ? static_cast<double>(NAN) : static_cast<double>(m) + log(sum);
    }
}

struct Cand { double value; long long at; };
__device__ __forceinline__ bool better(const Cand& x, const Cand& y) { return x.value > y.value || (x.value == y.value && x.at < y.at); }

template <typename T>
__global__ void __launch_bounds__(256) select_pick_kernel(SelectArgs a)
{
    __shared__ Cand red[8];
    __shared__ Cand last;
    const int g = blockIdx.x;
    if (threadIdx.x == 0) last = {INFINITY, -1};
    __syncthreads();
    for (int k = 0; k < a.n; ++k) {
        Cand best{-INFINITY, LLONG_MAX};
        const Cand prev = last;
        for (int b = 0; b < a.beams; ++b) {
            const int row = g * a.beams + b;
            const double score = a.scores[row];
            if (a.ended && a.ended[row]) {
                const Cand c{score, static_cast<long long>(b) * a.vocab + a.eos};
                if (threadIdx.x == 0 && c.value > -INFINITY && better(prev, c) && better(c, best)) best = c;
                continue;
            }
            const double norm = a.norm[row];
            const T* x = static_cast<const T*>(a.logits) + row * a.ld;
            for (int v = threadIdx.x; v < a.vocab; v += 256) {
                const Cand c{score + (static_cast<double>(to_f32(x[v])) - norm), static_cast<long long>(b) * a.vocab + v};
                if (c.value > -INFINITY && better(prev, c) && better(c, best)) best = c;
            }
        }
        for (int o = 16; o > 0; o >>= 1) {
            const Cand c{__shfl_xor_sync(0xffffffffu, best.value, o), __shfl_xor_sync(0xffffffffu, best.at, o)};
            if (better(c, best)) best = c;
        }
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = best;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 8; ++w) if (better(red[w], best)) best = red[w];
            last = best;
            const bool none = best.value == -INFINITY;
            const int parent = none ? -1 : static_cast<int>(best.at / a.vocab), token = none ? -1 : static_cast<int>(best.at % a.vocab), to = g * a.n + k;
            a.parent[to] = parent;
            a.token[to] = token;
            a.scores_out[to] = static_cast<float>(best.value);
            if (a.ended_out) a.ended_out[to] = !none && ((a.ended && a.ended[g * a.beams + parent]) || token == a.eos) ? 1 : 0;
        }
        __syncthreads();
    }
}

template <typename T> static int select_t(const SelectArgs& a, cudaStream_t s)
{
    select_norm_kernel<T><<<static_cast<unsigned>(a.groups * a.beams), 256, 0, s>>>(a);
    NNB_LAUNCH_CHECK();
    select_pick_kernel<T><<<static_cast<unsigned>(a.groups), 256, 0, s>>>(a);
    NNB_LAUNCH_CHECK();
    return 0;
}

static const char* select_shape_error(int groups, int beams, int vocab, int n)
{
    if (groups < 0) return "negative size";
    if (beams < 1 || beams > 64) return "beams must be from 1 to 64";
    if (vocab < 1 || static_cast<long long>(beams) * vocab > INT_MAX) return "vocab must be positive, and beams * vocab below 2^31";
    if (n < 1 || n > 128 || n > static_cast<long long>(beams) * vocab) return "the number of continuations must be from 1 to 128, and at most beams * vocab";
    if (static_cast<long long>(groups) * beams > INT_MAX / 256) return "too many beams for one call";
    return nullptr;
}

}  // namespace nnb

using namespace nnb;

extern "C" {

size_t nnb200_beam_select_scratch_bytes(int groups, int beams, int vocab, int n)
{
    if (const char* e = select_shape_error(groups, beams, vocab, n)) {
        fprintf(stderr, "nnb200: %s: %s\n", __func__, e);
        return 0;
    }
    return static_cast<size_t>(groups) * beams * sizeof(double) + 16;
}

int nnb200_beam_select(const void* logits, long long ld, int dtype, int groups, int beams, int vocab, const float* scores, const int32_t* ended, int eos,
                       int n, int32_t* parent, int32_t* token, float* scores_out, int32_t* ended_out, void* scratch, size_t scratch_bytes, void* stream)
{
    const char* e = select_shape_error(groups, beams, vocab, n);
    NNB_ARG_CHECK(!e, e);
    NNB_ARG_CHECK(dtype == 0 || dtype == 1, "dtype must be 0 (fp32) or 1 (bf16)");
    if (groups == 0) return 0;
    NNB_ARG_CHECK(logits && scores && parent && token && scores_out, "null argument");
    NNB_ARG_CHECK(ld >= vocab, "a row stride shorter than a row");
    NNB_ARG_CHECK(!ended || (eos >= 0 && eos < vocab), "ended beams continue with the end token, which must be in the vocabulary");
    NNB_ARG_CHECK(scratch && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "scratch must be there and start on a 16-byte boundary");
    NNB_ARG_CHECK(scratch_bytes >= nnb200_beam_select_scratch_bytes(groups, beams, vocab, n), "scratch too small");
    SelectArgs a{logits, ld, groups, beams, vocab, n, eos, scores, ended, parent, token, ended_out, scores_out, static_cast<double*>(scratch)};
    if (dtype == 0) return select_t<float>(a, to_stream(stream));
    return select_t<bf16>(a, to_stream(stream));
}

}  // extern "C"
