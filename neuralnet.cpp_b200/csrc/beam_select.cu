// Beam search's selection (nnb200_beam_select): of the continuations (beam b, token v) of a group's beams, valued
//   score_b + logit_bv - log sum_u exp(logit_bu),
// the n best, best first; equal values go to the lower (b, v).
// Which of two continuations is better decides what a program answers.  A score and a logit are exact and values are compared
// in 64 bits; the normaliser, the only rounded part, is summed in 64 bits from exponentials in 32, off by less than 1.5e-6 of
// one (ex2 2^-22, its argument 2^-24 of about 10 twice, eight additions in 32 bits), most often by less than 1e-7.  Where
// continuations of two beams come closer than that, which happens to one group in some hundreds, their beams' normalisers
// are computed again in 64 bits, as sums of whole numbers: exact to 1e-12, and the same in whatever order a row holds its logits.
//
// Two kernels.  The first reads the logits once, bound by memory: a block per span of a row sums its exponentials and keeps its n
// best (value, token) pairs.  The order within a row does not depend on the normaliser, so that needs no second pass.  What
// makes it one pass is a threshold: n values are known to be at least as large, so that only larger ones, few after the first
// tile of a row, go to a list in shared memory.  The second, already resident when the first ends, joins the spans' sums
// and picks from the rows' lists.
#include <algorithm>

#include "common.cuh"
#include "nnb200.h"

namespace nnb {

constexpr int kSelThreads = 256, kSelWarps = kSelThreads / 32;
constexpr int kSelPer = 16, kSelTile = kSelThreads * kSelPer;   // logits of a thread, and of the block, at a time
constexpr int kSelMost = 128;                                   // continuations of a group
constexpr int kSelSlack = 256;                                  // a list this much longer than n is cut back to n
constexpr int kSelList = kSelTile + kSelMost + kSelSlack;       // a tile may go into the list whole

struct alignas(16) SpanSum { double sum; float ref; };          // of exponentials against the reference point

struct SelectArgs {
    const void* logits;
    long long ld;
    int groups, beams, vocab, n, eos, spans, span, vectors;
    const float* scores;
    const int* ended;
    int *parent, *token, *ended_out;
    float* scores_out;
    SpanSum* stat;              // (row, span)
    int2* list;                 // (row, span, n): value (its bits) and token, best first; token -1: no more
};

// order of floats as order of unsigned numbers; zeros of either sign are one number
__device__ __forceinline__ uint32_t order_of(float x)
{
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float exp_against(float x, float ref)
{
    // (x - ref) log2(e), the constant in two parts: its rounding alone would move sums by 1e-7
    const float d = x - ref;
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(d, 1.4426950216293335f, d * 1.925963033500e-8f)));
    return y;
}

// A bound that at least `want` of the threads' values reach, none of them counted twice: of each warp the k-th largest value for
// k = want / 8 and want / 4, of the warps the smallest of the one, and the fourth of the other.  0 where there are too few.
__device__ __forceinline__ uint32_t bound_for(uint32_t mine, int want, uint32_t (*sw)[2])
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k8 = (want + 7) / 8, k4 = (want + 3) / 4;
    uint32_t at8 = 0, top = 0;
    for (int k = 1; k <= k4; ++k) {
        top = __reduce_max_sync(0xffffffffu, mine);
        const uint32_t who = __ballot_sync(0xffffffffu, mine == top);
        if (lane == __ffs(who) - 1) mine = 0;
        if (k == k8) at8 = top;
    }
    if (lane == 0) { sw[warp][0] = at8; sw[warp][1] = top; }
    __syncthreads();
    uint32_t least = 0xffffffffu, fourth = 0;
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) {
        least = min(least, sw[w][0]);
        int above = 0;
#pragma unroll
        for (int v = 0; v < kSelWarps; ++v) above += sw[v][1] > sw[w][1] || (sw[v][1] == sw[w][1] && v < w) ? 1 : 0;
        if (above == 3) fourth = sw[w][1];
    }
    return max(least, fourth);
}

// a list entry: order of the value above, complement of the token below, so that the larger one is the better
using Entry = unsigned long long;
__device__ __forceinline__ Entry entry_of(float x, int token) { return static_cast<Entry>(order_of(x)) << 32 | static_cast<uint32_t>(~token); }

struct SelectShared {
    Entry list[kSelList];
    Entry best[kSelMost];
    uint32_t sw[kSelWarps][2];
    double sum[kSelWarps];
    float ref[kSelWarps];
    int count;
};

// Cuts the list back to its n best, sorted; sh.count entries before, returns how many after (all threads call it).
__device__ int cut_list(SelectShared& sh, int n)
{
    __syncthreads();
    int count = sh.count;
    // a long list is thinned first: a bound from one value per thread leaves little more than n
    for (int round = 0; round < 3 && count > n + 64; ++round) {
        constexpr int PER = (kSelList + kSelThreads - 1) / kSelThreads;
        Entry top = 0;
        for (int i = threadIdx.x; i < count; i += kSelThreads) top = max(top, sh.list[i]);
        Entry bound = static_cast<Entry>(bound_for(static_cast<uint32_t>(top >> 32), n, sh.sw)) << 32;
        // entries equal to the bound in value may be many: of those a bound of tokens
        uint32_t tie = 0;
        for (int i = threadIdx.x; i < count; i += kSelThreads) { const Entry e = sh.list[i]; if (e >> 32 == bound >> 32) tie = max(tie, static_cast<uint32_t>(e)); }
        __syncthreads();
        bound |= bound_for(tie, n, sh.sw);
        uint32_t keep = 0;
#pragma unroll 1
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x + j * kSelThreads;
            if (i < count && sh.list[i] >= bound) keep |= 1u << j;
        }
        if (__syncthreads_count(keep != 0) == 0) break;
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        // in place, a stretch of the list at a time: what is kept moves to the front, never past where it is read
#pragma unroll 1
        for (int j = 0; j * kSelThreads < count; ++j) {
            const int i = threadIdx.x + j * kSelThreads;
            const bool k = keep >> j & 1u;
            const Entry e = k ? sh.list[i] : 0;
            __syncthreads();
            if (k) sh.list[atomicAdd(&sh.count, 1)] = e;
            __syncthreads();
        }
        const int now = sh.count;
        __syncthreads();
        if (now == count) break;
        count = now;
    }
    // the rank of an entry is the number of better ones; no two are equal
    for (int i = threadIdx.x; i < count; i += kSelThreads) {
        const Entry e = sh.list[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += sh.list[j] > e;
        if (rank < n) sh.best[rank] = e;
    }
    __syncthreads();
    const int left = min(count, n);
    for (int i = threadIdx.x; i < left; i += kSelThreads) sh.list[i] = sh.best[i];
    if (threadIdx.x == 0) sh.count = left;
    __syncthreads();
    return left;
}

template <typename T>
__global__ void __launch_bounds__(kSelThreads) select_scan_kernel(const __grid_constant__ SelectArgs a)
{
    __shared__ SelectShared sh;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int row = static_cast<int>(blockIdx.x / a.spans), part = static_cast<int>(blockIdx.x) - row * a.spans;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (a.ended && a.ended[row]) return;                        // its only continuation is not in its logits
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    const int begin = part * a.span, end = min(begin + a.span, a.vocab);
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    constexpr int N = Vec16<T>::N, VECS = kSelPer / N;
    float ref = -INFINITY;                                      // this thread's exponentials are taken against ref, near its maximum
    double sum = 0.0;
    uint32_t floor_ = 0;                                        // order of a value that n others reach: equal ones come too late
    for (int t0 = begin; t0 < end; t0 += kSelTile) {
        float v[kSelPer];
        // logit j of this thread is token_of(j): vectors of neighbours lie side by side
        auto token_of = [&](int j) { return a.vectors ? t0 + (j / N * kSelThreads + static_cast<int>(threadIdx.x)) * N + j % N : t0 + j * kSelThreads + static_cast<int>(threadIdx.x); };
        if (a.vectors && t0 + kSelTile <= end) {
            Vec16<T> r[VECS];
#pragma unroll
            for (int i = 0; i < VECS; ++i) r[i] = ld16(x + token_of(i * N));
#pragma unroll
            for (int j = 0; j < kSelPer; ++j) v[j] = to_f32(r[j / N].v[j % N]);
        } else {
#pragma unroll
            for (int j = 0; j < kSelPer; ++j) { const int t = token_of(j); v[j] = t < end ? to_f32(x[t]) : -INFINITY; }
        }
        float top = v[0];
#pragma unroll
        for (int j = 1; j < kSelPer; ++j) top = fmaxf(top, v[j]);
        if (top > ref + 8.0f) { sum *= ref == -INFINITY ? 0.0 : exp(static_cast<double>(ref) - top); ref = top; }
        const float r = ref == -INFINITY ? 0.f : ref;
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < kSelPer; j += 2) { s0 += exp_against(v[j], r); s1 += exp_against(v[j + 1], r); }
        sum += static_cast<double>(s0 + s1);
        const bool first = t0 == begin;
        uint32_t least = floor_ + 1;
        if (first) least = max(bound_for(order_of(top), a.n, sh.sw), order_of(-INFINITY) + 1);
        if (order_of(top) >= least) {
#pragma unroll
            for (int j = 0; j < kSelPer; ++j)
                if (order_of(v[j]) >= least && v[j] == v[j]) sh.list[atomicAdd(&sh.count, 1)] = entry_of(v[j], token_of(j));
        }
        __syncthreads();
        const int count = sh.count;
        if (first || count > a.n + kSelSlack) {
            if (cut_list(sh, a.n) == a.n) floor_ = static_cast<uint32_t>(sh.list[a.n - 1] >> 32);
            else floor_ = order_of(-INFINITY);
        }
        __syncthreads();
    }
    // the block's sum, against the largest of the threads' points
    float m = ref;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) sh.ref[warp] = m;
    const int left = cut_list(sh, a.n);
    m = sh.ref[0];
#pragma unroll
    for (int w = 1; w < kSelWarps; ++w) m = fmaxf(m, sh.ref[w]);
    // a thread without a finite value adds what it has: 0, or NaN where there was one
    double s = ref == -INFINITY ? sum : sum * exp(static_cast<double>(ref) - m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sh.sum[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kSelWarps; ++w) s += sh.sum[w];
        a.stat[blockIdx.x] = {s, m};
    }
    int2* to = a.list + static_cast<long long>(blockIdx.x) * a.n;
    for (int i = threadIdx.x; i < a.n; i += kSelThreads) {
        int2 o = make_int2(0, -1);
        if (i < left) {
            const uint32_t k = static_cast<uint32_t>(sh.list[i] >> 32);
            o = make_int2(static_cast<int>(k & 0x80000000u ? k & 0x7fffffffu : ~k), static_cast<int>(~static_cast<uint32_t>(sh.list[i])));
        }
        to[i] = o;
    }
}

// ---------------------------------------------------------------- picking
struct Cand { double value; int at, beam; };                    // at: beam * vocab + token
__device__ __forceinline__ bool better(const Cand& x, const Cand& y) { return x.value > y.value || (x.value == y.value && x.at < y.at); }
constexpr int kPickList = 2048;
constexpr double kNear = 4e-6;                                  // values of two beams this close are compared again, exactly

struct PickShared {
    double norm[64];            // log-sum-exp of each beam; NaN: its logits offer nothing
    Cand list[kPickList];
    uint32_t sw[kSelWarps][2];
    Cand red[kSelWarps], last;
    unsigned long long part[kSelWarps], again;                  // again: beams whose normalisers have to be exact
    int count;
};

__device__ __forceinline__ void put(const SelectArgs& a, int g, int k, const Cand& c)
{
    const bool none = !(c.value > -INFINITY);
    const int to = g * a.n + k, token = none ? -1 : c.at - c.beam * a.vocab;
    a.parent[to] = none ? -1 : c.beam;
    a.token[to] = token;
    a.scores_out[to] = none ? -INFINITY : static_cast<float>(c.value);
    if (a.ended_out) a.ended_out[to] = !none && ((a.ended && a.ended[g * a.beams + c.beam]) || token == a.eos) ? 1 : 0;
}

// log-sum-exp of a row whose sum is finite, by the whole block: exponentials in 64 bits, added as multiples of 2^-shift, 62 bits in all
template <typename T>
__device__ double exact_norm(const SelectArgs& a, PickShared& sh, int row)
{
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, shift = 62 - (32 - __clz(a.vocab));
    float m = -INFINITY;                                        // the first entry of a span is its maximum
    for (int i = 0; i < a.spans; ++i) { const int2 e = a.list[(static_cast<long long>(row) * a.spans + i) * a.n]; if (e.y >= 0) m = fmaxf(m, __int_as_float(e.x)); }
    const double scale = static_cast<double>(1ull << shift);
    unsigned long long sum = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kSelThreads) sum += __double2ull_rn(exp(static_cast<double>(to_f32(x[i])) - m) * scale);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (lane == 0) sh.part[warp] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) sum += sh.part[w];
    return static_cast<double>(m) + log(static_cast<double>(sum) / scale);
}

template <typename T>
__global__ void __launch_bounds__(kSelThreads) select_pick_kernel(const __grid_constant__ SelectArgs a)
{
    __shared__ PickShared sh;
    const int g = static_cast<int>(blockIdx.x), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int b = warp; b < a.beams; b += kSelWarps) {           // a warp per beam
        const int row = g * a.beams + b;
        if (a.ended && a.ended[row]) { if (lane == 0) sh.norm[b] = NAN; continue; }
        const SpanSum* st = a.stat + static_cast<long long>(row) * a.spans;
        float m = -INFINITY;
        for (int i = lane; i < a.spans; i += 32) m = fmaxf(m, st[i].ref);
        m = warp_max(m);
        double s = 0.0;
        for (int i = lane; i < a.spans; i += 32) s += st[i].ref == -INFINITY ? st[i].sum : st[i].sum * exp(static_cast<double>(st[i].ref) - m);
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        // NaN from a NaN or +inf logit; a row of -inf has no maximum
        if (lane == 0) sh.norm[b] = m == -INFINITY ? static_cast<double>(NAN) : static_cast<double>(m) + log(s);
    }
    if (threadIdx.x == 0) { sh.count = 0; sh.again = 0; }
    __syncthreads();
    const int per = a.spans * a.n, lists = a.beams * per, all = lists + a.beams;
    const Cand nothing{-INFINITY, INT_MAX, -1};
    // candidate i: the entries of the beams' lists, then the ended beams' own
    auto cand = [&](int i) -> Cand {
        if (i < lists) {
            const int b = i / per;
            const double norm = sh.norm[b];
            if (norm != norm) return nothing;                   // also where the lists were not written
            const int2 e = a.list[static_cast<long long>(g) * lists + i];
            if (e.y < 0) return nothing;
            const double v = static_cast<double>(a.scores[g * a.beams + b]) + (static_cast<double>(__int_as_float(e.x)) - norm);
            return v > -INFINITY ? Cand{v, b * a.vocab + e.y, b} : nothing;
        }
        const int b = i - lists;
        if (!a.ended || !a.ended[g * a.beams + b]) return nothing;
        const double v = a.scores[g * a.beams + b];
        return v > -INFINITY ? Cand{v, b * a.vocab + a.eos, b} : nothing;
    };
    // a value that n candidates reach, in 32 bits (rounding keeps the order but for equality), and by kNear less once normalisers move
    uint32_t top = 0;
    for (int i = threadIdx.x; i < all; i += kSelThreads) {
        const Cand x = cand(i);
        if (x.value > -INFINITY) top = max(top, order_of(static_cast<float>(x.value)));
    }
    const uint32_t key = bound_for(top, a.n, sh.sw);
    double bound = -INFINITY;
    if (key) {
        const float b = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
        bound = static_cast<double>(b) - fabs(static_cast<double>(b)) * 0x1p-23 - 2.0 * kNear;
        if (!(bound > -INFINITY)) bound = b == INFINITY ? 3e38 : -INFINITY;
    }
    for (int pass = 0; pass < 2; ++pass) {
        for (int i = threadIdx.x; i < all; i += kSelThreads) {
            const Cand x = cand(i);
            if (x.value > -INFINITY && x.value >= bound) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kPickList) sh.list[at] = x;
            }
        }
        __syncthreads();
        const int count = sh.count;
        if (count > kPickList) {
            if (pass == 0 && threadIdx.x == 0) sh.again = ~0ull;
        } else {
            for (int i = threadIdx.x; i < count; i += kSelThreads) {
                const Cand x = sh.list[i];
                int rank = 0;
                unsigned long long near = 0;
                for (int j = 0; j < count; ++j) {
                    const Cand y = sh.list[j];
                    rank += better(y, x);
                    if (y.beam != x.beam && fabs(y.value - x.value) < kNear) near |= 1ull << y.beam | 1ull << x.beam;
                }
                if (rank < a.n) {
                    if (pass == 0 && near) atomicOr(&sh.again, near);
                    put(a, g, rank, x);
                }
            }
            for (int k = count + threadIdx.x; k < a.n; k += kSelThreads) put(a, g, k, nothing);
        }
        __syncthreads();
        const unsigned long long again = sh.again;
        if (pass == 1 || again == 0) {
            if (count <= kPickList) return;
            break;
        }
        if (threadIdx.x == 0) sh.count = 0;
        for (int b = 0; b < a.beams; ++b) {
            const double norm = sh.norm[b];
            if (!(again >> b & 1ull) || norm != norm) continue;  // the same for all threads; an ended beam has no normaliser
            const double exact = exact_norm<T>(a, sh, g * a.beams + b);
            __syncthreads();
            if (threadIdx.x == 0) sh.norm[b] = exact;
        }
        __syncthreads();
    }
    // more candidates near the bound than the list takes: one place at a time
    if (threadIdx.x == 0) sh.last = {INFINITY, -1, -1};
    __syncthreads();
    for (int k = 0; k < a.n; ++k) {
        const Cand prev = sh.last;
        Cand best = nothing;
        for (int i = threadIdx.x; i < all; i += kSelThreads) {
            const Cand x = cand(i);
            if (x.value > -INFINITY && better(prev, x) && better(x, best)) best = x;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Cand x{__shfl_xor_sync(0xffffffffu, best.value, o), __shfl_xor_sync(0xffffffffu, best.at, o), __shfl_xor_sync(0xffffffffu, best.beam, o)};
            if (better(x, best)) best = x;
        }
        if (lane == 0) sh.red[warp] = best;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kSelWarps; ++w) if (better(sh.red[w], best)) best = sh.red[w];
            sh.last = best;
            put(a, g, k, best);
        }
        __syncthreads();
    }
}

// Blocks for a row: as many as keep the machine busy where there are few rows, whole tiles each.
static int select_spans(int groups, int beams, int vocab)
{
    const long long rows = static_cast<long long>(groups) * beams, tiles = ceil_div(vocab, kSelTile);
    const long long want = std::max<long long>(1, 148 * 4 / rows), per = ceil_div(tiles, std::min(tiles, want));
    return static_cast<int>(ceil_div(tiles, per));
}

template <typename T> static int select_t(SelectArgs a, cudaStream_t s)
{
    a.vectors = ((reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.ld % Vec16<T>::N == 0) ? 1 : 0;
    select_scan_kernel<T><<<static_cast<unsigned>(a.groups * a.beams * a.spans), kSelThreads, 0, s>>>(a);
    NNB_LAUNCH_CHECK();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.groups));
    cfg.blockDim = dim3(kSelThreads);
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    NNB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, select_pick_kernel<T>, a));
    NNB_LAUNCH_CHECK();
    return 0;
}

static const char* select_shape_error(int groups, int beams, int vocab, int n)
{
    if (groups < 0) return "negative size";
    if (beams < 1 || beams > 64) return "beams must be from 1 to 64";
    if (vocab < 1 || static_cast<long long>(beams) * vocab > INT_MAX) return "vocab must be positive, and beams * vocab below 2^31";
    if (n < 1 || n > kSelMost || n > static_cast<long long>(beams) * vocab) return "the number of continuations must be from 1 to 128, and at most beams * vocab";
    if (static_cast<long long>(groups) * beams > INT_MAX / 256) return "too many beams for one call";
    if (static_cast<long long>(beams) * select_spans(groups, beams, vocab) * n > INT_MAX / 2) return "too many candidates for one call";
    return nullptr;
}
static size_t select_stat_bytes(int groups, int beams, int spans) { return static_cast<size_t>(groups) * beams * spans * sizeof(SpanSum); }

}  // namespace nnb

using namespace nnb;

extern "C" {

size_t nnb200_beam_select_scratch_bytes(int groups, int beams, int vocab, int n)
{
    if (const char* e = select_shape_error(groups, beams, vocab, n)) {
        fprintf(stderr, "nnb200: %s: %s\n", __func__, e);
        return 0;
    }
    const int spans = select_spans(groups, beams, vocab);
    return select_stat_bytes(groups, beams, spans) + static_cast<size_t>(groups) * beams * spans * n * sizeof(int2) + 16;
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
    SelectArgs a{logits, ld, groups, beams, vocab, n, eos};
    const int spans = select_spans(groups, beams, vocab);
    a.spans = spans;
    a.span = static_cast<int>(ceil_div(ceil_div(vocab, kSelTile), spans)) * kSelTile;
    a.scores = scores; a.ended = ended; a.parent = parent; a.token = token; a.scores_out = scores_out; a.ended_out = ended_out;
    a.stat = static_cast<SpanSum*>(scratch);
    a.list = reinterpret_cast<int2*>(static_cast<uint8_t*>(scratch) + select_stat_bytes(groups, beams, spans));
    if (dtype == 0) return select_t<float>(a, to_stream(stream));
    return select_t<bf16>(a, to_stream(stream));
}

}  // extern "C"
