// Beam search's selection (nnb200_beam_select): of the continuations (beam b, token v) of a group's beams, valued
//   score_b + logit_bv - log sum_u exp(logit_bu),
// the n best, best first; equal values go to the lower (b, v).
// Which of two continuations is better decides what a program answers.  A score and a logit are exact and values are compared
// in 64 bits; the normaliser, the only rounded part, is summed in 64 bits from exponentials in 32, off by less than 2.3e-6, most
// often by less than 1e-7.  An exponential of a distance d to the reference point is off by half a step of d and of
// d log2(e), 2^-22 for ex2 and six additions of 2^-24.  No d is above kSelAhead: 1.2e-6 for those from -8 up, 1.8e-6 for -16 to
// -8, 2.3e-6 for -22 to -16; all further below, 2.9e-6, is at most 2^31 e^-22 = 0.6 of the largest exponential.  Where
// continuations of two beams come closer than that, which happens to one group in some hundreds, their beams' normalisers
// are computed again in 64 bits, as sums of whole multiples of 2^-62: off by 2^-63 an exponential (5e-13 for 2^22 of them) and the
// roundings of exp and log, and the same in whatever order a row holds its logits.
//
// Two kernels.  The first reads the logits once, bound by memory and the exponentials: a block per span of a row sums its
// exponentials and keeps the maximum of each thread's share of each tile.  The order within a row does not depend on the
// normaliser, so its n best can be had from these: n threads' maxima bound them from below, and only the few shares that reach the
// bound are looked at again.  (Comparing each logit with a running threshold on the way took 2000 of a tile's 3800 clocks: with
// 1000 logits a warp and tile somebody always has one.)  The second kernel, already resident when the first ends, joins the spans'
// sums and picks from the rows' lists.
// 64 groups of 8 beams over 32768 bf16 logits, 16 continuations: 21.3 us.  Its 512 blocks are one wave: 11.7 us until the last has been
// through its eight tiles (the exponentials alone, at 16 an SM and clock and with four blocks an SM, take 4.3, the copy rate 5.2),
// 3.7 for what ends a span (the bound 1.3, the shares that reach it 1.3, sorting the list 0.7, the sum 0.4), 0.8 to the second kernel
// and 5 to 6 in it.  One group of 4 beams over 4096: 7.1 us, two launches of a few dependent steps.
#include <algorithm>

#include "common.cuh"
#include "nnb200.h"
#include "tc_ptx.cuh"

namespace nnb {

constexpr int kSelThreads = 128, kSelWarps = kSelThreads / 32;  // few warps: what a block does besides its logits is done by each
constexpr int kSelPer = 32, kSelTile = kSelThreads * kSelPer;   // logits of a thread, and of the block, at a time
constexpr int kSelMost = 128;                                   // continuations of a group
constexpr int kSelSlack = 256;                                  // a list this much longer than n is cut back to n
constexpr int kSelList = kSelTile + kSelMost + kSelSlack;       // a tile may go into the list whole
constexpr int kSelTiles = 16;                                   // tiles of a span at most
constexpr float kSelAhead = 8.0f;                               // what a logit may be above the reference point of its exponential
constexpr int kSelPieces = kSelList / kSelPer - 4;              // threads' shares of tiles that may go into the list together

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
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order); }
__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// exponentials of eight values against a reference point, added up: the argument is (x - ref) log2(e) with the constant in two
// parts, because its rounding alone would move sums by 1e-7
__device__ __forceinline__ float exps_against(const float* v, uint64_t minus_ref)
{
    const uint64_t hi = pack2(1.4426950216293335f, 1.4426950216293335f), lo = pack2(1.925963033500e-8f, 1.925963033500e-8f);
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const uint64_t d = add2(pack2(v[j], v[j + 1]), minus_ref);
        float x, y;
        unpack2(fma2(d, hi, mul2(d, lo)), x, y);
        const uint64_t e = pack2(exp2_approx(x), exp2_approx(y));
        sum = j ? add2(sum, e) : e;
    }
    float x, y;
    unpack2(sum, x, y);
    return x + y;
}

// A bound that at least `want` (up to 128) of the threads' values reach: of each of the W warps the k-th largest value, for
// k = want / W the smallest of the warps', for k = 2 want / W the (W / 2)-th largest.  0 where there are too few.
template <int W>
__device__ __forceinline__ uint32_t bound_for(uint32_t mine, int want, uint32_t (*sw)[2])
{
    static_assert(W >= 4 && W <= 32 && 128 / W <= 32, "a warp has that many values");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, all = (want + W - 1) / W, half = (2 * want + W - 1) / W, rounds = min(half, 32);
    uint32_t at = 0, top = 0;
    for (int k = 1; k <= rounds; ++k) {
        top = __reduce_max_sync(0xffffffffu, mine);
        const uint32_t who = __ballot_sync(0xffffffffu, mine == top);
        if (lane == __ffs(who) - 1) mine = 0;
        if (k == all) at = top;
    }
    if (lane == 0) { sw[warp][0] = at; sw[warp][1] = rounds == half ? top : 0; }
    __syncthreads();
    const uint32_t least = __reduce_min_sync(0xffffffffu, lane < W ? sw[lane][0] : 0xffffffffu), h = lane < W ? sw[lane][1] : 0;
    int above = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) { const uint32_t o = __shfl_sync(0xffffffffu, h, w); above += o > h || (o == h && w < lane) ? 1 : 0; }
    return max(least, __reduce_max_sync(0xffffffffu, lane < W && above == W / 2 - 1 ? h : 0));
}

// a list entry: order of the value above, complement of the token below, so that the larger one is the better
using Entry = unsigned long long;
__device__ __forceinline__ Entry entry_of(float x, int token) { return static_cast<Entry>(order_of(x)) << 32 | static_cast<uint32_t>(~token); }

struct SelectShared {
    Entry list[kSelList];
    Entry best[kSelMost];
    uint32_t sw[kSelWarps][2];
    double sum[kSelWarps];
    float ref[kSelWarps], top[kSelTiles][kSelThreads];          // top: maximum of each thread's share of each tile
    int count, pieces, piece[kSelPieces > kSelThreads ? kSelPieces : kSelThreads];
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
        Entry bound = static_cast<Entry>(bound_for<kSelWarps>(static_cast<uint32_t>(top >> 32), n, sh.sw)) << 32;
        // entries equal to the bound in value may be many: of those a bound of tokens
        uint32_t tie = 0;
        for (int i = threadIdx.x; i < count; i += kSelThreads) { const Entry e = sh.list[i]; if (e >> 32 == bound >> 32) tie = max(tie, static_cast<uint32_t>(e)); }
        __syncthreads();
        bound |= bound_for<kSelWarps>(tie, n, sh.sw);
        unsigned long long keep = 0;
        static_assert(PER <= 64, "a bit for each of a thread's entries");
#pragma unroll 1
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x + j * kSelThreads;
            if (i < count && sh.list[i] >= bound) keep |= 1ull << j;
        }
        if (__syncthreads_count(keep != 0) == 0) break;
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        // in place, a stretch of the list at a time: what is kept moves to the front, never past where it is read
#pragma unroll 1
        for (int j = 0; j * kSelThreads < count; ++j) {
            const int i = threadIdx.x + j * kSelThreads;
            const bool k = keep >> j & 1ull;
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
#pragma unroll 8
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
    if (threadIdx.x == 0) { sh.count = 0; sh.pieces = 0; }
    constexpr int N = Vec16<T>::N, VECS = kSelPer / N;
    // exponentials are taken against the first tile's maximum, or one of this thread's own where that is far behind
    float ref = -INFINITY, most = -INFINITY;
    double sum = 0.0;
    const int tiles = (end - begin + kSelTile - 1) / kSelTile;
    // whole tiles of aligned rows are read a tile ahead
    Vec16<T> raw[VECS];
    auto whole = [&](int t0) { return a.vectors && t0 + kSelTile <= end; };
    auto ahead = [&](int t0) {
        if (!whole(t0)) return;
#pragma unroll
        for (int i = 0; i < VECS; ++i) raw[i] = ld16(x + t0 + (i * kSelThreads + static_cast<int>(threadIdx.x)) * N);
    };
    // logit j of thread t in the tile at t0: vectors of neighbours lie side by side
    auto token_of = [&](int t0, int t, int j) { return a.vectors ? t0 + (j / N * kSelThreads + t) * N + j % N : t0 + j * kSelThreads + t; };
    ahead(begin);
    for (int i = 0; i < tiles; ++i) {
        const int t0 = begin + i * kSelTile;
        float v[kSelPer];
        if (whole(t0)) {
#pragma unroll
            for (int j = 0; j < kSelPer; ++j) v[j] = to_f32(raw[j / N].v[j % N]);
            ahead(t0 + kSelTile);
        } else {
#pragma unroll
            for (int j = 0; j < kSelPer; ++j) { const int t = token_of(t0, threadIdx.x, j); v[j] = t < end ? to_f32(x[t]) : -INFINITY; }
        }
        float top4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int j = 4; j < kSelPer; ++j) top4[j & 3] = fmaxf(top4[j & 3], v[j]);
        const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
        sh.top[i][threadIdx.x] = top;
        most = fmaxf(most, top);
        if (i == 0) {
            ref = warp_max(top);
            if (lane == 0) sh.ref[warp] = ref;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kSelWarps; ++w) ref = fmaxf(ref, sh.ref[w]);
        }
        if (top > ref + kSelAhead) { sum *= ref == -INFINITY ? 0.0 : exp(static_cast<double>(ref) - top); ref = top; }
        const float r = ref == -INFINITY ? 0.f : -ref;
        const uint64_t minus_ref = pack2(r, r);
        float part[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) part[h] = exps_against(v + 8 * h, minus_ref);
        sum += static_cast<double>((part[0] + part[1]) + (part[2] + part[3]));
    }
    // the shares that hold one of the n best, one warp each
    float least = value_of(max(bound_for<kSelWarps>(order_of(most), a.n, sh.sw), order_of(-INFINITY) + 1));
    auto look = [&](int pieces) {
        for (int p0 = warp; p0 < pieces; p0 += 4 * kSelWarps) {  // four of a warp's on their way at a time
            int t[4];
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int piece = sh.piece[min(p0 + u * kSelWarps, pieces - 1)];
                t[u] = token_of(begin + (piece >> 8) * kSelTile, piece & 255, lane);
                v[u] = p0 + u * kSelWarps < pieces && t[u] < end ? to_f32(x[t[u]]) : -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (v[u] >= least) sh.list[atomicAdd(&sh.count, 1)] = entry_of(v[u], t[u]);
        }
    };
    static_assert(kSelPer == 32 && kSelThreads <= 256, "a lane for each logit of a share");
    uint32_t reach = 0;
#pragma unroll
    for (int i = 0; i < kSelTiles; ++i) reach |= i < tiles && sh.top[i][threadIdx.x] >= least ? 1u << i : 0;
    static_assert(kSelTiles <= 32, "a bit for each tile");
    if (reach) {
        for (int at = atomicAdd(&sh.pieces, __popc(reach)); reach && at < kSelPieces; ++at, reach &= reach - 1)
            sh.piece[at] = (__ffs(reach) - 1) << 8 | static_cast<int>(threadIdx.x);
    }
    __syncthreads();
    if (sh.pieces <= kSelPieces) look(sh.pieces);
    else {
        // many equal values: tile by tile, in order, the list cut back on the way; what equals the n-th best comes too late from then on
        for (int i = 0; i < tiles; ++i) {
            __syncthreads();
            if (threadIdx.x == 0) sh.pieces = 0;
            __syncthreads();
            if (sh.top[i][threadIdx.x] >= least) sh.piece[atomicAdd(&sh.pieces, 1)] = i << 8 | static_cast<int>(threadIdx.x);
            __syncthreads();
            look(sh.pieces);
            __syncthreads();
            if (sh.count > a.n + kSelSlack && cut_list(sh, a.n) == a.n) least = fmaxf(least, value_of(static_cast<uint32_t>(sh.list[a.n - 1] >> 32) + 1));
        }
    }
    const int left = cut_list(sh, a.n);
    // the block's sum, against the largest of the threads' points
    float m = ref;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) sh.ref[warp] = m;
    __syncthreads();
    m = sh.ref[0];
#pragma unroll
    for (int w = 1; w < kSelWarps; ++w) m = fmaxf(m, sh.ref[w]);
    // a thread without a finite value adds what it has: 0, or NaN where there was one
    double s = ref == -INFINITY || ref == m ? sum : sum * exp(static_cast<double>(ref) - m);
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
// order of doubles as order of unsigned numbers; at: beam * vocab + token
struct Cand { unsigned long long key; int at, beam; };
__device__ __forceinline__ unsigned long long order_of(double x)
{
    const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(x + 0.0));
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double value_of(unsigned long long order) { return __longlong_as_double(static_cast<long long>(order >> 63 ? order & ~(1ull << 63) : ~order)); }
__device__ __forceinline__ bool better(const Cand& x, const Cand& y) { return x.key > y.key || (x.key == y.key && x.at < y.at); }
constexpr int kPickList = 2048;
constexpr double kNear = 5e-6;                                  // values of two beams this close are compared again, exactly: twice a normaliser's error

template <int W> struct PickShared {
    double norm[64];            // log-sum-exp of each beam; NaN: its logits offer nothing
    float score[64];
    Cand list[kPickList], best[kSelMost];
    uint32_t sw[W][2];
    Cand red[W], last;
    ulonglong2 part[W];
    unsigned long long again;                           // beams whose normalisers have to be exact
    int count, ended[64];
};

template <int W>
__device__ __forceinline__ void put(const SelectArgs& a, const PickShared<W>& sh, int g, int k, const Cand& c)
{
    const bool none = c.key == 0;
    const int to = g * a.n + k, token = none ? -1 : c.at - c.beam * a.vocab;
    a.parent[to] = none ? -1 : c.beam;
    a.token[to] = token;
    a.scores_out[to] = none ? -INFINITY : static_cast<float>(value_of(c.key));
    if (a.ended_out) a.ended_out[to] = !none && (sh.ended[c.beam] || token == a.eos) ? 1 : 0;
}

// log-sum-exp of a row whose sum is finite, by the whole block: exponentials in 64 bits, none above 1, added as multiples of 2^-62.  Their
// upper and lower 31 bits are added apart (x: below 2^32 each, y: below 2^31), so that 2^31 of them fit.
template <typename T, int W>
__device__ double exact_norm(const SelectArgs& a, PickShared<W>& sh, int row)
{
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = -INFINITY;                                        // the first entry of a span is its maximum
    for (int i = 0; i < a.spans; ++i) { const int2 e = a.list[(static_cast<long long>(row) * a.spans + i) * a.n]; if (e.y >= 0) m = fmaxf(m, __int_as_float(e.x)); }
    ulonglong2 sum = make_ulonglong2(0, 0);
    auto add = [&sum](unsigned long long hi, unsigned long long lo) { sum.x += hi; sum.y += lo; };
#pragma unroll 8
    for (int i = threadIdx.x; i < a.vocab; i += (W * 32)) {
        const unsigned long long e = __double2ull_rn(exp(static_cast<double>(to_f32(x[i])) - m) * 0x1p62);
        add(e >> 31, e & 0x7fffffffull);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) add(__shfl_xor_sync(0xffffffffu, sum.x, o), __shfl_xor_sync(0xffffffffu, sum.y, o));
    __syncthreads();
    if (lane == 0) sh.part[warp] = sum;
    __syncthreads();
    sum = make_ulonglong2(0, 0);
#pragma unroll
    for (int w = 0; w < W; ++w) add(sh.part[w].x, sh.part[w].y);
    // the same whole number whatever the order: first the carry, then to 64 bits of floating point
    sum.x += sum.y >> 31;
    return static_cast<double>(m) + log(static_cast<double>(sum.x) * 0x1p-31 + static_cast<double>(sum.y & 0x7fffffffull) * 0x1p-62);
}

template <typename T, int W>
__global__ void __launch_bounds__(W * 32) select_pick_kernel(const __grid_constant__ SelectArgs a)
{
    __shared__ PickShared<W> sh;
    const int g = static_cast<int>(blockIdx.x), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // written before the kernel in front of this one began
    if (static_cast<int>(threadIdx.x) < a.beams) {
        sh.score[threadIdx.x] = a.scores[g * a.beams + threadIdx.x];
        sh.ended[threadIdx.x] = a.ended ? a.ended[g * a.beams + threadIdx.x] : 0;
    }
    if (threadIdx.x == 0) { sh.count = 0; sh.again = 0; }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // candidate i: the rows' lists side by side, best entries first, then the ended beams' own.  A thread's candidates are then of
    // like places in different lists, and the best of each list with different threads: what the bound below lives on.
    const int rows = a.beams * a.spans, lists = rows * a.n, all = lists + a.beams;
    const Cand nothing{0, INT_MAX, -1};
    struct Raw { int2 e; int beam; };
    auto raw = [&](int i) -> Raw {
        if (i >= lists) return {make_int2(0, a.eos), i - lists};
        const int k = i / rows, r = i - k * rows, b = r / a.spans;
        if (sh.ended[b]) return {make_int2(0, -1), b};          // its lists were not written
        return {a.list[(static_cast<long long>(g) * rows + r) * a.n + k], b};
    };
    auto cand = [&](int i, const Raw& w) -> Cand {
        double v = sh.score[w.beam];
        if (i >= lists) { if (!sh.ended[w.beam]) return nothing; }
        else {
            if (w.e.y < 0) return nothing;
            v += static_cast<double>(__int_as_float(w.e.x)) - sh.norm[w.beam];
        }
        return v > -INFINITY ? Cand{order_of(v), w.beam * a.vocab + w.e.y, w.beam} : nothing;
    };
    const int first = threadIdx.x;
    Raw mine_raw{make_int2(0, -1), 0};
    if (first < all) mine_raw = raw(first);
    for (int b = warp; b < a.beams; b += W) {           // a warp per beam
        if (sh.ended[b]) { if (lane == 0) sh.norm[b] = NAN; continue; }
        const SpanSum* st = a.stat + static_cast<long long>(g * a.beams + b) * a.spans;
        const SpanSum own = lane < a.spans ? st[lane] : SpanSum{0.0, -INFINITY};
        float m = own.ref;
        for (int i = lane + 32; i < a.spans; i += 32) m = fmaxf(m, st[i].ref);
        m = warp_max(m);
        auto against = [&](const SpanSum& x) { return x.ref == -INFINITY || x.ref == m ? x.sum : x.sum * exp(static_cast<double>(x.ref) - m); };
        double s = against(own);
        for (int i = lane + 32; i < a.spans; i += 32) s += against(st[i]);
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        // NaN from a NaN or +inf logit; a row of -inf has no maximum
        if (lane == 0) sh.norm[b] = m == -INFINITY ? static_cast<double>(NAN) : static_cast<double>(m) + log(s);
    }
    __syncthreads();
    // a value that n candidates reach, in 32 bits (rounding keeps the order but for equality), and by kNear less once normalisers move
    Cand mine = first < all ? cand(first, mine_raw) : nothing;
    uint32_t top = mine.key ? order_of(static_cast<float>(value_of(mine.key))) : 0;
    for (int i = first + (W * 32); i < all; i += (W * 32)) {
        const Cand x = cand(i, raw(i));
        if (x.key) top = max(top, order_of(static_cast<float>(value_of(x.key))));
    }
    const uint32_t key = bound_for<W>(top, a.n, sh.sw);
    auto below = [](uint32_t k) -> unsigned long long {
        if (k == 0) return 1;
        const double b = value_of(k), less = b - fabs(b) * 0x1p-23 - 2.0 * kNear;
        return b == INFINITY ? order_of(3e38) : (less > -INFINITY ? order_of(less) : 1);
    };
    const unsigned long long bound = below(key);
    auto add = [&](const Cand& x) {
        if (x.key >= bound) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kPickList) sh.list[at] = x;
        }
    };
    for (int pass = 0; pass < 2; ++pass) {
        if (pass == 1 && first < all) mine = cand(first, mine_raw);
        add(mine);
        for (int i = first + (W * 32); i < all; i += (W * 32)) add(cand(i, raw(i)));
        __syncthreads();
        int count = sh.count;
        // a long list is thinned: with its entries spread over the threads a bound leaves little more than n
        for (int round = 0; round < 2 && count > a.n + 256 && count <= kPickList; ++round) {
            uint32_t most = 0;
            for (int i = threadIdx.x; i < count; i += (W * 32)) most = max(most, order_of(static_cast<float>(value_of(sh.list[i].key))));
            const unsigned long long tight = below(bound_for<W>(most, a.n, sh.sw));
            Cand kept[kPickList / (W * 32)];
#pragma unroll
            for (int j = 0; j < kPickList / (W * 32); ++j) {
                const int i = threadIdx.x + j * (W * 32);
                kept[j] = i < count && sh.list[i].key >= tight ? sh.list[i] : nothing;
            }
            __syncthreads();
            if (threadIdx.x == 0) sh.count = 0;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kPickList / (W * 32); ++j) if (kept[j].key) sh.list[atomicAdd(&sh.count, 1)] = kept[j];
            __syncthreads();
            count = sh.count;
            __syncthreads();
        }
        if (count > kPickList) {
            if (threadIdx.x == 0) sh.again = ~0ull;
        } else {
            // four threads an entry.  What is close to one of the n best may belong before it, and its beam's normaliser has
            // to be exact too
            for (int i = threadIdx.x >> 2; i < (count + 7) / 8 * 8; i += W * 8) {
                const Cand x = sh.list[min(i, count - 1)];
                const unsigned long long under = order_of(value_of(x.key) - kNear), over = order_of(value_of(x.key) + kNear);
                int rank = 0;
                unsigned long long near = 0;
                for (int j = threadIdx.x & 3; j < count; j += 4) {
                    const Cand y = sh.list[j];
                    rank += better(y, x);
                    if (y.key > under && y.key < over && y.beam != x.beam) near |= 1ull << y.beam | 1ull << x.beam;
                }
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) { rank += __shfl_xor_sync(0xffffffffu, rank, o); near |= __shfl_xor_sync(0xffffffffu, near, o); }
                if (i < count && (threadIdx.x & 3) == 0 && rank < a.n) {
                    sh.best[rank] = x;
                    if (pass == 0 && near) atomicOr(&sh.again, near);
                }
            }
            for (int k = count + threadIdx.x; k < a.n; k += (W * 32)) sh.best[k] = nothing;
        }
        __syncthreads();
        const unsigned long long again = sh.again;
        if (count <= kPickList && (pass == 1 || again == 0)) {
            for (int k = threadIdx.x; k < a.n; k += (W * 32)) put(a, sh, g, k, sh.best[k]);
            return;
        }
        if (pass == 1) break;
        if (threadIdx.x == 0) sh.count = 0;
        for (int b = 0; b < a.beams; ++b) {
            const double norm = sh.norm[b];
            if (!(again >> b & 1ull) || norm != norm) continue;  // the same for all threads; an ended beam has no normaliser
            const double exact = exact_norm<T, W>(a, sh, g * a.beams + b);
            __syncthreads();
            if (threadIdx.x == 0) sh.norm[b] = exact;
        }
        __syncthreads();
    }
    // more candidates near the bound than the list takes: one place at a time
    if (threadIdx.x == 0) sh.last = {~0ull, -1, -1};
    __syncthreads();
    for (int k = 0; k < a.n; ++k) {
        const Cand prev = sh.last;
        Cand best = nothing;
        for (int i = threadIdx.x; i < all; i += (W * 32)) {
            const Cand x = cand(i, raw(i));
            if (x.key && better(prev, x) && better(x, best)) best = x;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Cand x{__shfl_xor_sync(0xffffffffu, best.key, o), __shfl_xor_sync(0xffffffffu, best.at, o), __shfl_xor_sync(0xffffffffu, best.beam, o)};
            if (better(x, best)) best = x;
        }
        if (lane == 0) sh.red[warp] = best;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < W; ++w) if (better(sh.red[w], best)) best = sh.red[w];
            sh.last = best;
            put(a, sh, g, k, best);
        }
        __syncthreads();
    }
}

// Blocks for a row: as many as keep the machine busy where there are few rows, whole tiles each.
static int select_spans(int groups, int beams, int vocab)
{
    const long long rows = std::max(1LL, static_cast<long long>(groups) * beams), tiles = ceil_div(vocab, kSelTile);
    const long long want = std::max<long long>(1, 148 * 4 / rows), per = std::min<long long>(ceil_div(tiles, std::min(tiles, want)), kSelTiles);
    return static_cast<int>(ceil_div(tiles, per));
}

template <typename T> static int select_t(SelectArgs a, cudaStream_t s)
{
    a.vectors = ((reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.ld % Vec16<T>::N == 0) ? 1 : 0;
    select_scan_kernel<T><<<static_cast<unsigned>(a.groups * a.beams * a.spans), kSelThreads, 0, s>>>(a);
    NNB_LAUNCH_CHECK();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.groups));
    // candidates on most threads: the bound is the n-th of the threads' best
    const bool many = static_cast<long long>(a.beams) * a.spans * a.n > 1024;
    cfg.blockDim = dim3(many ? 512 : 128);
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    NNB_CUDA_CHECK(many ? cudaLaunchKernelEx(&cfg, select_pick_kernel<T, 16>, a) : cudaLaunchKernelEx(&cfg, select_pick_kernel<T, 4>, a));
    NNB_LAUNCH_CHECK();
    return 0;
}

static const char* select_shape_error(int groups, int beams, int vocab, int n)
{
    if (groups < 0) return "negative size";
    if (beams < 1 || beams > 64) return "beams must be from 1 to 64";
    if (vocab < 1 || static_cast<long long>(beams) * vocab > INT_MAX) return "vocab must be positive, and beams * vocab below 2^31";
    if (vocab > INT_MAX - kSelTiles * kSelTile) return "vocab must be below 2^31 - 2^16";        // tokens are counted to the end of a row's last span
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
