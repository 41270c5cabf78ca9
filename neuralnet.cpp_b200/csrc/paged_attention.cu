// Attention of batched decoding: one new query per sequence over the rows of a paged cache, first the prefix that the
// sequences of a group share, then the sequence's own rows (nnb200_paged_attention).
//   s_t = q . k_t / sqrt(dk) - slope_h (T - 1 - t),  out = sum_t softmax(s)_t v_t,  lse = log sum_t exp(s_t)
// with t over the T = prefix_len + seq_len rows the query sees; a query for which no row has weight (it sees none, or all
// its scores are -inf) gives 0 and -inf.
//
// A group's queries that read one head of the cache are the rows of one tile, so the prefix is read once for all of them; own
// rows are read by the query heads that share them.  Both are the same task, "rows of queries against a run of cached rows":
// the runs are split over blocks until the machine is full, each block leaves its unnormalised sums with their maximum and
// sum of exponentials in scratch, and a second kernel, already resident when the last block ends, joins them in fixed order.
#include "paged.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <type_traits>

namespace nnb {

struct PagedAttnArgs {
    const void* q;
    void* out;
    float* lse;
    long long ldq, ldo;
    const int *prefix_table, *prefix_len, *table, *len;
    int prefix_stride, table_stride, groups, size, heads, alibi;
    FastDiv m;                      // query heads per cached head
    FastDiv row_tiles, own_tiles;   // tiles of a group's rows, of a sequence's
    FastDiv pre_splits, own_splits; // blocks that share a prefix, a sequence's own rows (0: divisor 1, and no task)
    FastDiv by_size, by_kv_heads, by_vecs, by_heads;
    int slots, pre_slots, own_rows; // places of a query row's partial results, the prefix's among them; rows of an own tile
    int own_warps;                  // warps that share a task of own rows: 4, or 1 (four tasks in a block)
    int pre_blocks, tasks;          // tasks [0, pre_blocks) are prefixes, a block each; the others own rows
    int pairs;                      // queries may be read two columns at a time
    float c;                        // log2(e) / sqrt(head_dim): exponentials are powers of two
    float* part;                    // (query row, slot): head_dim sums
    float2* stat;                   // (query row, slot): maximum (in powers of two) and sum; sum 0: nothing there
};

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float alibi_slope2(int h, int heads) { return exp2f(-8.0f * static_cast<float>(h) / static_cast<float>(heads)) * 1.4426950408889634f; }

// What a block works on: `rows` query rows (row r is query head head0 + r % m of sequence seq0 + r / m) against rows
// [begin, end) of one page table.  Row t stands at position place + t of what sequence `seq` sees in all.
struct AttnTask {
    const int* table;
    int hk, first, rows, begin, end, place, slot, group;
};
// lengths are device data: clamped to [0, what the table holds]; negative own length: nothing is seen
__device__ __forceinline__ int held(int len, int stride, int shift)
{
    return static_cast<int>(min(static_cast<long long>(max(len, 0)), static_cast<long long>(stride) << shift));
}
// the share of split s: whole tiles of 64 rows, so that few rows go to few splits
__device__ __forceinline__ void share_of(int len, int splits, int s, int& begin, int& end)
{
    const int per = ((len + splits - 1) / splits + 63) & ~63;
    begin = static_cast<int>(min(static_cast<long long>(s) * per, static_cast<long long>(len)));
    end = min(len - begin, per) + begin;
}
template <int RT, typename T>
__device__ __forceinline__ AttnTask task_of(const PagedPool<T>& pool, const PagedAttnArgs& a, int b)
{
    AttnTask k;
    if (b < a.pre_blocks) {                                     // neighbours share their cached rows: row tiles, then splits
        int rest = a.row_tiles.split(b);                        // b: row tile
        int head = a.pre_splits.split(rest);                    // rest: split
        const int g = a.by_kv_heads.split(head);
        k.hk = head;
        k.group = g;
        k.first = b * RT;
        k.rows = min(a.size * static_cast<int>(a.m.d) - k.first, RT);
        k.table = a.prefix_table + static_cast<long long>(g) * a.prefix_stride;
        k.place = 0;
        k.slot = rest;
        share_of(held(a.prefix_len[g], a.prefix_stride, pool.page_shift), a.pre_slots, rest, k.begin, k.end);
        return k;
    }
    b -= a.pre_blocks;
    int rest = a.own_tiles.split(b), head = a.own_splits.split(rest);
    const int seq = a.by_kv_heads.split(head), m = static_cast<int>(a.m.d);
    k.hk = head;
    k.group = a.by_size.div(seq);
    k.first = (seq - k.group * a.size) * m + b * a.own_rows;
    k.rows = min(m - b * a.own_rows, a.own_rows);
    k.table = a.table + static_cast<long long>(seq) * a.table_stride;
    k.place = a.prefix_stride ? held(a.prefix_len[k.group], a.prefix_stride, pool.page_shift) : 0;
    k.slot = a.pre_slots + rest;
    share_of(held(a.len[seq], a.table_stride, pool.page_shift), static_cast<int>(a.own_splits.d), rest, k.begin, k.end);
    return k;
}
// query row r of a task
struct AttnRow { int seq, head; };
__device__ __forceinline__ AttnRow row_of(const PagedAttnArgs& a, const AttnTask& k, int r)
{
    int j = k.first + r;
    const int i = a.m.split(j);
    return {k.group * a.size + i, k.hk * static_cast<int>(a.m.d) + j};
}
// distance from row `place + t` to the last one the query sees is far_of - t
__device__ __forceinline__ int far_of(const PagedAttnArgs& a, int shift, const AttnTask& k, int seq)
{
    const int pre = a.prefix_stride ? held(a.prefix_len[k.group], a.prefix_stride, shift) : 0;
    return pre + (a.table_stride ? held(a.len[seq], a.table_stride, shift) : 0) - 1 - k.place;
}

// ---------------------------------------------------------------- bf16: mma.sync tiles
// 64 cached rows a step, a ring of STAGES steps filled by 16-byte asynchronous copies; WM warps take 16 query rows each, the
// 4 / WM warps of a set of rows take turns at the step's cached rows and are joined at the end.  Cached rows that do not
// exist are zero in shared memory (what lies there may be anything, and zero times it must be zero) and -inf as scores.
template <int DP> struct AttnTile {
    static constexpr int KT = 64, CPR = DP / 8;                // cached rows a step, 16-byte chunks a row
    static constexpr int STAGES = DP <= 64 ? 4 : (DP == 128 ? 3 : 2);
    static constexpr int BYTES = KT * DP * 2;
    static constexpr int SMEM = STAGES * 2 * BYTES + STAGES * (KT + 16) + 64;
    // chunk c of row r: eight rows of one chunk column fall into eight different 16-byte banks
    static __device__ __forceinline__ uint32_t at(int r, int c)
    {
        return static_cast<uint32_t>(r * (DP * 2) + ((CPR >= 8 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4));
    }
};

template <int DP> struct AttnLoader {
    using Tile = AttnTile<DP>;
    const PagedPool<bf16>& pool;
    const AttnTask& k;
    uint32_t base;                  // shared memory: K, V of each stage
    uint8_t* alive;                 // per stage: KT flags, then one per warp for "some row of the step is not there"
    __device__ __forceinline__ void load(int step, int stage) const
    {
        const int t0 = k.begin + step * Tile::KT, tid = threadIdx.x;
        bool gap = false;
#pragma unroll
        for (int i = 0; i < Tile::KT * Tile::CPR / 128; ++i) {
            const int idx = tid + i * 128, r = idx / Tile::CPR, c = idx % Tile::CPR, t = t0 + r;
            const int row = t < k.end ? pool.find(k.table, k.hk, t) : -1;
            const bool there = row >= 0;
            const long long off = there && c * 8 < pool.dk ? static_cast<long long>(row) * pool.dk + c * 8 : 0;
            const int bytes = there && c * 8 < pool.dk ? 16 : 0;
            const uint32_t dst = base + stage * 2 * Tile::BYTES + Tile::at(r, c);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(pool.k + off), "r"(bytes) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + Tile::BYTES), "l"(pool.v + off), "r"(bytes) : "memory");
            gap |= !there;
            if (c == 0) alive[stage * (Tile::KT + 16) + r] = there;
        }
        const bool any = __any_sync(0xffffffffu, gap);
        if ((tid & 31) == 0) alive[stage * (Tile::KT + 16) + Tile::KT + (tid >> 5)] = any;
    }
};

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t p)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t p)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Leaves a row's state: in scratch for the join, or finished where a row has one slot only.
__device__ __forceinline__ bool sees(const PagedAttnArgs& a, int seq) { return a.len[seq] >= 0; }
template <typename T>
__device__ __forceinline__ void leave(const PagedAttnArgs& a, const AttnTask& k, int dk, int r, int c, float4 o, float m, float l)
{
    const AttnRow w = row_of(a, k, r);
    const long long row = static_cast<long long>(w.seq) * a.heads + w.head;
    if (a.slots == 1) {
        const bool none = l == 0.f || !sees(a, w.seq);
        T* to = static_cast<T*>(a.out) + w.seq * a.ldo + static_cast<long long>(w.head) * dk + c;
        const float inv = none ? 0.f : 1.0f / l;
        to[0] = from_f32<T>(none ? 0.f : o.x * inv); to[1] = from_f32<T>(none ? 0.f : o.y * inv);
        to[2] = from_f32<T>(none ? 0.f : o.z * inv); to[3] = from_f32<T>(none ? 0.f : o.w * inv);
        if (c == 0 && a.lse) a.lse[row] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        return;
    }
    const long long at = row * a.slots + k.slot;
    *reinterpret_cast<float4*>(a.part + at * dk + c) = o;
    if (c == 0) a.stat[at] = make_float2(m, l);
}
template <typename T>
__device__ __forceinline__ void leave_nothing(const PagedAttnArgs& a, const AttnTask& k, int dk, int first, int stride)
{
    for (int r = first; r < k.rows; r += stride) {
        const AttnRow w = row_of(a, k, r);
        if (a.slots > 1) a.stat[(static_cast<long long>(w.seq) * a.heads + w.head) * a.slots + k.slot] = make_float2(-INFINITY, 0.f);
        else for (int c = 0; c < dk; c += 4) leave<T>(a, k, dk, r, c, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f);
    }
}

template <int DP, int WM>
__device__ __forceinline__ void attend_bf16(const PagedPool<bf16>& pool, const PagedAttnArgs& a, const AttnTask& k, uint8_t* smem)
{
    using Tile = AttnTile<DP>;
    constexpr int WK = 4 / WM, KW = Tile::KT / WK, NT = KW / 8, ND = DP / 8, KS = DP / 16, ST = Tile::STAGES;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wm = warp / WK, wk = warp % WK, dk = pool.dk;
    const int steps = (k.end - k.begin + Tile::KT - 1) / Tile::KT;
    uint8_t* alive = smem + ST * 2 * Tile::BYTES;
    const AttnLoader<DP> loader{pool, k, smem_u32(smem), alive};
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) { if (i < steps) loader.load(i, i); cp_commit(); }

    const int r0 = wm * 16 + (lane >> 2);                       // this thread's rows: r0 and r0 + 8
    uint32_t qf[KS][4];
    float slope[2] = {0.f, 0.f}, far[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = r0 + 8 * i;
        const bool live = r < k.rows;
        const bf16* q = static_cast<const bf16*>(a.q);
        if (live) {
            const AttnRow w = row_of(a, k, r);
            q += w.seq * a.ldq + static_cast<long long>(w.head) * dk;
            if (a.alibi) { slope[i] = alibi_slope2(w.head, a.heads); far[i] = static_cast<float>(far_of(a, pool.page_shift, k, w.seq)); }
        }
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = kk * 16 + j * 8 + (lane & 3) * 2;
                uint32_t v = 0;
                if (live && c < dk) {
                    if (a.pairs) v = *reinterpret_cast<const uint32_t*>(q + c);
                    else v = static_cast<uint32_t>(__bfloat16_as_ushort(q[c])) | static_cast<uint32_t>(__bfloat16_as_ushort(q[c + 1])) << 16;
                }
                qf[kk][j * 2 + i] = v;
            }
    }

    const float mul = a.alibi ? 1.f : a.c;                      // scores are scaled inside the exponent, or with the bias before it
    float o[ND][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][j] = 0.f;

    for (int step = 0; step < steps; ++step) {
        cp_wait<ST - 2>();
        __syncthreads();
        const int stage = step % ST;
        if (step + ST - 1 < steps) loader.load(step + ST - 1, (step + ST - 1) % ST);
        cp_commit();
        const uint32_t kb = smem_u32(smem) + stage * 2 * Tile::BYTES, vb = kb + Tile::BYTES;
        const int key0 = wk * KW;
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                uint32_t b[4];
                ldsm4(b, kb + Tile::at(key0 + n * 8 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
                mma_bf16(s[n], qf[kk], b[0], b[1]);
                mma_bf16(s[n + 1], qf[kk], b[2], b[3]);
            }
        const int t0 = k.begin + step * Tile::KT + key0 + (lane & 3) * 2;
        if (a.alibi) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[n][j] = s[n][j] * a.c - slope[j >> 1] * (far[j >> 1] - static_cast<float>(t0 + n * 8 + (j & 1)));
        }
        const uint8_t* al = alive + stage * (Tile::KT + 16);
        if (*reinterpret_cast<const uint32_t*>(al + Tile::KT)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (!al[key0 + n * 8 + (lane & 3) * 2 + j]) { s[n][j] = -INFINITY; s[n][j + 2] = -INFINITY; }
        }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[0] = fmaxf(top[0], fmaxf(s[n][0], s[n][1]));
            top[1] = fmaxf(top[1], fmaxf(s[n][2], s[n][3]));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
            top[i] = fmaxf(m[i], top[i] * mul);
        }
        float ref[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) ref[i] = top[i] == -INFINITY ? 0.f : top[i];
        if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float back = exp2_fast(m[i] - ref[i]);
                l[i] *= back;
#pragma unroll
                for (int n = 0; n < ND; ++n) { o[n][2 * i] *= back; o[n][2 * i + 1] *= back; }
                m[i] = top[i];
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) { s[n][j] = exp2_fast(fmaf(s[n][j], mul, -ref[j >> 1])); l[j >> 1] += s[n][j]; }
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            // the weights are rounded to bf16 for the tensor cores (their sum is not): 2^-9 of a weight, what rounding V costs too
            const uint32_t p[4] = {pack_bf16x2(s[n][0], s[n][1]), pack_bf16x2(s[n][2], s[n][3]), pack_bf16x2(s[n + 1][0], s[n + 1][1]), pack_bf16x2(s[n + 1][2], s[n + 1][3])};
#pragma unroll
            for (int d = 0; d < ND; d += 2) {
                uint32_t b[4];
                ldsm4_t(b, vb + Tile::at(key0 + n * 8 + (lane & 7) + (((lane >> 3) & 1) << 3), d + (lane >> 4)));
                mma_bf16(o[d], p, b[0], b[1]);
                mma_bf16(o[d + 1], p, b[2], b[3]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    // join the warps of a set of rows through shared memory, write rows with whole vectors
    cp_wait<0>();
    __syncthreads();
    constexpr int LD = DP + 8;
    float* so = reinterpret_cast<float*>(smem);                 // (warp, 16 rows, LD)
    float2* sml = reinterpret_cast<float2*>(so + 4 * 16 * LD);
    static_assert(4 * 16 * LD * 4 + 4 * 16 * 8 <= ST * 2 * Tile::BYTES, "the join fits the ring");
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *reinterpret_cast<float2*>(so + (warp * 16 + (lane >> 2) + 8 * i) * LD + n * 8 + (lane & 3) * 2) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
    if ((lane & 3) == 0) {
        sml[warp * 16 + (lane >> 2)] = make_float2(m[0], l[0]);
        sml[warp * 16 + (lane >> 2) + 8] = make_float2(m[1], l[1]);
    }
    __syncthreads();
    const int vecs = dk / 4;
    for (int idx = threadIdx.x; idx < k.rows * vecs; idx += 128) {
        const int r = a.by_vecs.div(idx), c = (idx - r * vecs) * 4, w0 = (r >> 4) * WK, rr = r & 15;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WK; ++w) top = fmaxf(top, sml[(w0 + w) * 16 + rr].x);
        const float ref = top == -INFINITY ? 0.f : top;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) {
            const float2 st = sml[(w0 + w) * 16 + rr];
            const float e = exp2_fast(st.x - ref);
            const float4 y = *reinterpret_cast<const float4*>(so + ((w0 + w) * 16 + rr) * LD + c);
            sum = fmaf(st.y, e, sum);
            x.x = fmaf(y.x, e, x.x); x.y = fmaf(y.y, e, x.y); x.z = fmaf(y.z, e, x.z); x.w = fmaf(y.w, e, x.w);
        }
        leave<bf16>(a, k, dk, r, c, x, top, sum);
    }
}

// Up to 16 query rows: nothing is shared between warps, so each warp streams cached rows through a ring of its own, KW rows a
// step, without a barrier, and the WT warps of a task (one, or the block's four) take its steps in turn and are joined at the
// end.  The products are transposed, S' = K Q' and O' = V' P', so that cached rows fill the 16 rows of a tensor core tile and
// queries its 8 columns (NQ = 1 or 2 of them): one query costs half of what it would as one of 16 rows.  P' comes out of the
// first product with cached rows down and queries across; the second wants it the other way round, an 8 x 8 transposition.
// A lane looks up one cached row of a step, a step before it is copied; the copies get it by shuffle.  Rows in shared memory
// are 16 bytes longer than they are: eight neighbours at one column meet no bank twice.  The reference point of the exponentials
// moves only when a score is more than 2^8 above it: scores then need no maximum across lanes.
template <int DP> struct AttnStream {
    static constexpr int KW = DP <= 32 ? 32 : 16, ST = DP <= 64 ? 3 : 2, PITCH = DP * 2 + 16, CPR = DP / 8;
    static constexpr int PLANE = KW * PITCH, STAGE = 2 * PLANE, RING = ST * STAGE;
    static constexpr int SMEM = 4 * (RING + 16);
};
// what a score may be above the reference point of its row's exponentials, in powers of two: sums stay far from overflow
constexpr float kAttnSlack = 8.0f;

__device__ __forceinline__ uint32_t transposed8x8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <int DP, int NQ>
__device__ __forceinline__ void stream_bf16(const PagedPool<bf16>& pool, const PagedAttnArgs& a, const AttnTask& k, uint8_t* smem, int wt)
{
    using Str = AttnStream<DP>;
    constexpr int KW = Str::KW, NK = KW / 16, ND = DP / 16, KS = DP / 16, ST = Str::ST, CPR = Str::CPR;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wk = wt == 1 ? 0 : warp, dk = pool.dk;
    const int all = (k.end - k.begin + KW - 1) / KW, steps = (all - wk + wt - 1) / wt;
    const uint32_t ring = smem_u32(smem) + warp * Str::RING;
    uint32_t* alive = reinterpret_cast<uint32_t*>(smem + 4 * Str::RING) + warp * 4;
    // the cached row this lane looks up for a step (lanes beyond KW: none)
    auto look = [&](int step) {
        const int t = k.begin + (step * wt + wk) * KW + lane;
        return step < steps && lane < KW && t < k.end ? pool.find(k.table, k.hk, t) : -1;
    };
    // lane l copies chunk l % CPR of rows l / CPR, l / CPR + RPI, ..
    constexpr int RPI = 32 / CPR;                               // rows the warp copies at once
    const int chunk = lane % CPR;
    const bool in = chunk * 8 < dk;
    const char* kbase = reinterpret_cast<const char*>(pool.k + (in ? chunk * 8 : 0));
    const char* vbase = reinterpret_cast<const char*>(pool.v + (in ? chunk * 8 : 0));
    const uint32_t dst0 = ring + (lane / CPR) * Str::PITCH + chunk * 16;
    auto fetch = [&](int row, int stage) {
        const uint32_t mask = __ballot_sync(0xffffffffu, row >= 0);
        if (lane == 0) alive[stage] = mask;
#pragma unroll
        for (int i = 0; i < KW / RPI; ++i) {
            const int r = __shfl_sync(0xffffffffu, row, i * RPI + lane / CPR);
            const long long off = static_cast<long long>(max(r, 0)) * (dk * 2);
            const int bytes = r >= 0 && in ? 16 : 0;
            const uint32_t dst = dst0 + stage * Str::STAGE + i * RPI * Str::PITCH;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(kbase + off), "r"(bytes) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + Str::PLANE), "l"(vbase + off), "r"(bytes) : "memory");
        }
    };
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) { const int row = look(i); if (i < steps) fetch(row, i); cp_commit(); }
    int next = look(ST - 1);

    const int g = lane >> 2, t2 = (lane & 3) * 2;               // queries as columns: g for loading them, t2 and t2 + 1 in the products
    uint32_t qf[NQ][KS][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = n * 8 + g;
        const bool live = r < k.rows;
        const AttnRow w = row_of(a, k, live ? r : 0);
        const bf16* q = static_cast<const bf16*>(a.q) + w.seq * a.ldq + static_cast<long long>(w.head) * dk + t2;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = kk * 16 + j * 8;
                uint32_t v = 0;
                if (live && c + t2 < dk) {
                    if (a.pairs) v = *reinterpret_cast<const uint32_t*>(q + c);
                    else v = static_cast<uint32_t>(__bfloat16_as_ushort(q[c])) | static_cast<uint32_t>(__bfloat16_as_ushort(q[c + 1])) << 16;
                }
                qf[n][kk][j] = v;
            }
    }
    float slope[NQ][2], far[NQ][2], m[NQ][2], l[NQ][2], o[ND][NQ][4];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            slope[n][i] = 0.f; far[n][i] = 0.f; m[n][i] = -INFINITY; l[n][i] = 0.f;
            if (a.alibi && n * 8 + t2 + i < k.rows) {
                const AttnRow w = row_of(a, k, n * 8 + t2 + i);
                slope[n][i] = alibi_slope2(w.head, a.heads);
                far[n][i] = static_cast<float>(far_of(a, pool.page_shift, k, w.seq));
            }
        }
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[d][n][j] = 0.f;
    const float mul = a.alibi ? 1.f : a.c;                      // scores are scaled inside the exponent, or with the bias before it

    int stage = 0;
    for (int step = 0; step < steps; ++step) {
        cp_wait<ST - 2>();
        __syncwarp();
        if (step + ST - 1 < steps) fetch(next, stage == 0 ? ST - 1 : stage - 1);
        cp_commit();
        next = look(step + ST);
        const uint32_t kb = ring + stage * Str::STAGE + ((lane & 7) + ((lane >> 3) & 1) * 8) * Str::PITCH + (lane >> 4) * 16;
        const uint32_t vb = ring + stage * Str::STAGE + Str::PLANE + ((lane & 7) + (lane >> 4) * 8) * Str::PITCH + ((lane >> 3) & 1) * 16;
        const uint32_t mask = alive[stage];
        stage = stage == ST - 1 ? 0 : stage + 1;
        float s[NK][NQ][4];                                     // cached row g (0, 1) or g + 8 (2, 3), query t2 (0, 2) or t2 + 1 (1, 3)
#pragma unroll
        for (int x = 0; x < NK; ++x) {
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[x][n][j] = 0.f;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                uint32_t f[4];
                ldsm4(f, kb + x * 16 * Str::PITCH + kk * 32);
#pragma unroll
                for (int n = 0; n < NQ; ++n) mma_bf16(s[x][n], f, qf[n][kk][0], qf[n][kk][1]);
            }
        }
        if (a.alibi) {
            const float t0 = static_cast<float>(k.begin + (step * wt + wk) * KW + g);
#pragma unroll
            for (int x = 0; x < NK; ++x)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[x][n][j] = s[x][n][j] * a.c - slope[n][j & 1] * (far[n][j & 1] - (t0 + static_cast<float>(x * 16 + (j >> 1) * 8)));
        }
        if (mask != (KW == 32 ? 0xffffffffu : (1u << (KW & 31)) - 1u)) {
#pragma unroll
            for (int x = 0; x < NK; ++x)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (!(mask >> (x * 16 + g + i * 8) & 1u)) {
#pragma unroll
                        for (int n = 0; n < NQ; ++n) { s[x][n][2 * i] = -INFINITY; s[x][n][2 * i + 1] = -INFINITY; }
                    }
        }
        bool ahead = false;
        float top[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                top[n][i] = fmaxf(s[0][n][i], s[0][n][i + 2]);
#pragma unroll
                for (int x = 1; x < NK; ++x) top[n][i] = fmaxf(top[n][i], fmaxf(s[x][n][i], s[x][n][i + 2]));
                top[n][i] *= mul;
                ahead |= top[n][i] > m[n][i] + kAttnSlack;
            }
        if (__any_sync(0xffffffffu, ahead)) {
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float x = top[n][i];
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
                    x = fmaxf(x, m[n][i]);
                    const float back = exp2_fast(m[n][i] - (x == -INFINITY ? 0.f : x));
                    m[n][i] = x;
                    l[n][i] *= back;
#pragma unroll
                    for (int d = 0; d < ND; ++d) { o[d][n][i] *= back; o[d][n][i + 2] *= back; }
                }
        }
        float ref[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) ref[n][i] = m[n][i] == -INFINITY ? 0.f : m[n][i];
#pragma unroll
        for (int x = 0; x < NK; ++x) {
            uint32_t p[NQ][2];
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                float e[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) { e[j] = exp2_fast(fmaf(s[x][n][j], mul, -ref[n][j & 1])); l[n][j & 1] += e[j]; }
                // the weights are rounded to bf16 for the tensor cores (their sum is not): half a step of 2^-8, what rounding V costs too
                p[n][0] = transposed8x8(pack_bf16x2(e[0], e[1]));
                p[n][1] = transposed8x8(pack_bf16x2(e[2], e[3]));
            }
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                uint32_t f[4];
                ldsm4_t(f, vb + x * 16 * Str::PITCH + d * 32);
#pragma unroll
                for (int n = 0; n < NQ; ++n) mma_bf16(o[d][n], f, p[n][0], p[n][1]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], w);
    cp_wait<0>();
    if (wt == 1) __syncwarp();
    else __syncthreads();
    // through shared memory, so that rows are written with whole vectors; the warps of a task are joined on the way
    constexpr int LD = DP + 4;
    static_assert(NQ * 8 * (LD * 4 + 8) <= Str::RING, "the join fits a warp's ring");
    float* so = reinterpret_cast<float*>(smem + warp * Str::RING);
    float2* sml = reinterpret_cast<float2*>(so + NQ * 8 * LD);
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = n * 8 + t2 + i;
            if (r < k.rows) {
#pragma unroll
                for (int d = 0; d < ND; ++d) { so[r * LD + d * 16 + g] = o[d][n][i]; so[r * LD + d * 16 + g + 8] = o[d][n][i + 2]; }
                if (g == 0) sml[r] = make_float2(m[n][i], l[n][i]);
            }
        }
    if (wt == 1) __syncwarp();
    else __syncthreads();
    const int vecs = dk / 4;
    for (int idx = wt == 1 ? lane : threadIdx.x; idx < k.rows * vecs; idx += 32 * wt) {
        const int r = a.by_vecs.div(idx), c = (idx - r * vecs) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, sum = 0.f;
        if (wt == 1) {
            x = *reinterpret_cast<const float4*>(so + r * LD + c);
            top = sml[r].x; sum = sml[r].y;
        } else {
            const float* s0 = reinterpret_cast<const float*>(smem);
            float2 st[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) { st[w] = *reinterpret_cast<const float2*>(s0 + w * (Str::RING / 4) + NQ * 8 * LD + 2 * r); top = fmaxf(top, st[w].x); }
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float e = exp2_fast(st[w].x - ref);
                const float4 y = *reinterpret_cast<const float4*>(s0 + w * (Str::RING / 4) + r * LD + c);
                sum = fmaf(st[w].y, e, sum);
                x.x = fmaf(y.x, e, x.x); x.y = fmaf(y.y, e, x.y); x.z = fmaf(y.z, e, x.z); x.w = fmaf(y.w, e, x.w);
            }
        }
        leave<bf16>(a, k, dk, r, c, x, top, sum);
    }
}

template <int DP, int WM, int NQ>
__global__ void __launch_bounds__(128) paged_attn_bf16_kernel(PagedPool<bf16> pool, const __grid_constant__ PagedAttnArgs a)
{
    extern __shared__ __align__(128) uint8_t smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int b = static_cast<int>(blockIdx.x);
    if (b < a.pre_blocks) {
        const AttnTask k = task_of<WM == 1 ? NQ * 8 : WM * 16>(pool, a, b);
        if (k.begin >= k.end) { leave_nothing<bf16>(a, k, pool.dk, threadIdx.x, 128); return; }
        if constexpr (WM == 1) stream_bf16<DP, NQ>(pool, a, k, smem, 4);
        else attend_bf16<DP, WM>(pool, a, k, smem);
        return;
    }
    // own rows: a task for the block, or one for each of its warps
    const int task = a.own_warps == 4 ? b : a.pre_blocks + (b - a.pre_blocks) * 4 + static_cast<int>(threadIdx.x >> 5);
    if (task >= a.tasks) return;
    const AttnTask k = task_of<WM == 1 ? NQ * 8 : WM * 16>(pool, a, task);
    if (k.begin >= k.end) { leave_nothing<bf16>(a, k, pool.dk, a.own_warps == 4 ? threadIdx.x : threadIdx.x & 31, 32 * a.own_warps); return; }
    stream_bf16<DP, NQ>(pool, a, k, smem, a.own_warps);
}

// ---------------------------------------------------------------- fp32: FMA tiles
// Up to 16 query rows against KT cached rows a step.  Scores: a thread takes one cached row and four to eight query rows; softmax:
// eight lanes a query row; values: a thread takes four columns and every KG-th cached row, for all query rows, and the KG
// parts are summed at the end.  Rows in shared memory are 16 bytes longer than they are, so that eight neighbours' 16-byte reads
// meet no bank twice.  fp32 products and sums throughout: infinities and NaN behave as in the formula, which splitting a
// number into parts for the tensor cores would not keep.
template <int DP> struct AttnTile32 {
    static constexpr int KT = DP <= 64 ? 64 : 4096 / DP, LD = DP + 4, CPR = DP / 4, STAGES = 2;
    static constexpr int G = 128 / KT, RPT = 16 / G;           // sets of query rows, rows of a thread
    static constexpr int KG = 512 / DP, PL = 20;               // sets of cached rows for the values, row of the weights
    static constexpr int FLOATS = KT * LD;                     // K, or V, of a stage
    static constexpr int RING = STAGES * 2 * FLOATS;
    static constexpr int SMEM = (RING + 16 * DP + KT * PL + 16 * 4) * 4 + STAGES * (KT + 16);
    static_assert(RING >= 128 * 64, "the join fits the ring");
    // query row i of set g: fours of rows in turn, so that few rows still spread over the sets
    static __device__ __forceinline__ int row(int g, int i) { return RPT >= 4 ? (i >> 2) * 4 * G + g * 4 + (i & 3) : g * RPT + i; }
};

template <int DP>
__device__ __forceinline__ void load_f32(const PagedPool<float>& pool, const AttnTask& k, uint32_t base, uint8_t* alive, int step, int stage)
{
    using Tile = AttnTile32<DP>;
    const int t0 = k.begin + step * Tile::KT, tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < Tile::KT * Tile::CPR / 128; ++i) {
        const int idx = tid + i * 128, r = idx / Tile::CPR, c = idx % Tile::CPR, t = t0 + r;
        const int row = t < k.end ? pool.find(k.table, k.hk, t) : -1;
        const bool there = row >= 0;
        const long long off = there && c * 4 < pool.dk ? static_cast<long long>(row) * pool.dk + c * 4 : 0;
        const int bytes = there && c * 4 < pool.dk ? 16 : 0;
        const uint32_t dst = base + (stage * 2 * Tile::FLOATS + r * Tile::LD + c * 4) * 4;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(pool.k + off), "r"(bytes) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + Tile::FLOATS * 4), "l"(pool.v + off), "r"(bytes) : "memory");
        if (c == 0) alive[stage * (Tile::KT + 16) + r] = there;
    }
}

template <int DP>
__global__ void __launch_bounds__(128) paged_attn_f32_kernel(PagedPool<float> pool, const __grid_constant__ PagedAttnArgs a)
{
    extern __shared__ __align__(128) uint8_t smem[];
    using Tile = AttnTile32<DP>;
    constexpr int KT = Tile::KT, ST = Tile::STAGES, PL = Tile::PL;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const AttnTask k = task_of<16>(pool, a, blockIdx.x);
    if (k.begin >= k.end) { leave_nothing<float>(a, k, pool.dk, threadIdx.x, 128); return; }
    const int tid = threadIdx.x, dk = pool.dk, steps = (k.end - k.begin + KT - 1) / KT;
    float* ring = reinterpret_cast<float*>(smem);
    float *sq = ring + Tile::RING, *sp = sq + 16 * DP, *sback = sp + KT * PL, *sslope = sback + 16, *sfar = sslope + 16;
    uint8_t* alive = reinterpret_cast<uint8_t*>(sfar + 32);
    const uint32_t base = smem_u32(ring);
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) { if (i < steps) load_f32<DP>(pool, k, base, alive, i, i); cp_commit(); }
    for (int i = tid; i < 16 * DP; i += 128) {
        const int r = i / DP, c = i - r * DP;
        const AttnRow w = row_of(a, k, r);
        sq[i] = r < k.rows && c < dk ? static_cast<const float*>(a.q)[w.seq * a.ldq + static_cast<long long>(w.head) * dk + c] : 0.f;
    }
    if (tid < 16) {
        const bool on = a.alibi && tid < k.rows;
        const AttnRow w = row_of(a, k, on ? tid : 0);
        sslope[tid] = on ? alibi_slope2(w.head, a.heads) : 0.f;
        sfar[tid] = on ? static_cast<float>(far_of(a, pool.page_shift, k, w.seq)) : 0.f;
    }
    const int key = tid % KT, set = tid / KT;                   // scores
    const int srow = tid >> 3, part = tid & 7;                  // softmax
    const int c4 = tid % (DP / 4), kg = tid / (DP / 4);         // values
    const int quads = (k.rows + 3) >> 2;
    float m = -INFINITY, l = 0.f, o[16][4];
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[r][j] = 0.f;

    for (int step = 0; step < steps; ++step) {
        cp_wait<ST - 2>();
        __syncthreads();
        const int stage = step % ST;
        if (step + ST - 1 < steps) load_f32<DP>(pool, k, base, alive, step + ST - 1, (step + ST - 1) % ST);
        cp_commit();
        const float *sk = ring + stage * 2 * Tile::FLOATS, *sv = sk + Tile::FLOATS;
        {
            float s[Tile::RPT];
#pragma unroll
            for (int i = 0; i < Tile::RPT; ++i) s[i] = 0.f;
#pragma unroll 4
            for (int d = 0; d < DP; d += 4) {
                const float4 kv = *reinterpret_cast<const float4*>(sk + key * Tile::LD + d);
#pragma unroll
                for (int i = 0; i < Tile::RPT; ++i) {
                    if (Tile::row(set, i) >= k.rows) continue;
                    const float4 q = *reinterpret_cast<const float4*>(sq + Tile::row(set, i) * DP + d);
                    s[i] = fmaf(q.x, kv.x, s[i]); s[i] = fmaf(q.y, kv.y, s[i]); s[i] = fmaf(q.z, kv.z, s[i]); s[i] = fmaf(q.w, kv.w, s[i]);
                }
            }
            const bool there = alive[stage * (KT + 16) + key];
            const float t = static_cast<float>(k.begin + step * KT + key);
#pragma unroll
            for (int i = 0; i < Tile::RPT; ++i) {
                const int r = Tile::row(set, i);
                s[i] = there ? s[i] * a.c - sslope[r] * (sfar[r] - t) : -INFINITY;
            }
            if constexpr (Tile::RPT >= 4) {
#pragma unroll
                for (int i = 0; i < Tile::RPT; i += 4) *reinterpret_cast<float4*>(sp + key * PL + Tile::row(set, i)) = make_float4(s[i], s[i + 1], s[i + 2], s[i + 3]);
            } else {
#pragma unroll
                for (int i = 0; i < Tile::RPT; ++i) sp[key * PL + Tile::row(set, i)] = s[i];
            }
        }
        __syncthreads();
        float s[KT / 8], top = m;
#pragma unroll
        for (int j = 0; j < KT / 8; ++j) { s[j] = sp[(part + 8 * j) * PL + srow]; top = fmaxf(top, s[j]); }
#pragma unroll
        for (int w = 1; w < 8; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float ref = top == -INFINITY ? 0.f : top, back = exp2f(m - ref);
        const bool moved = top != m;
        l *= back;
        m = top;
#pragma unroll
        for (int j = 0; j < KT / 8; ++j) {
            s[j] = exp2f(s[j] - ref);
            l += s[j];
            sp[(part + 8 * j) * PL + srow] = s[j];
        }
        if (part == 0) sback[srow] = back;
        if (__syncthreads_or(moved)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float b = sback[r];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[r][j] *= b;
            }
        }
#pragma unroll 2
        for (int t = kg; t < KT; t += Tile::KG) {
            const float4 v = *reinterpret_cast<const float4*>(sv + t * Tile::LD + c4 * 4);
#pragma unroll
            for (int rq = 0; rq < 4; ++rq) {
                if (rq >= quads) break;
                const float4 p = *reinterpret_cast<const float4*>(sp + t * PL + rq * 4);
                const float pr[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float* x = o[rq * 4 + i];
                    x[0] = fmaf(pr[i], v.x, x[0]); x[1] = fmaf(pr[i], v.y, x[1]); x[2] = fmaf(pr[i], v.z, x[2]); x[3] = fmaf(pr[i], v.w, x[3]);
                }
            }
        }
    }
#pragma unroll
    for (int w = 1; w < 8; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
    cp_wait<0>();
    __syncthreads();
    if (part == 0) { sslope[srow] = m; sfar[srow] = l; }
#pragma unroll
    for (int r = 0; r < 16; ++r)
        if (r < k.rows) *reinterpret_cast<float4*>(ring + (kg * 16 + r) * DP + c4 * 4) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
    __syncthreads();
    const int vecs = dk / 4;
    for (int idx = tid; idx < k.rows * vecs; idx += 128) {
        const int r = a.by_vecs.div(idx), c = (idx - r * vecs) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < Tile::KG; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(ring + (w * 16 + r) * DP + c);
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        leave<float>(a, k, dk, r, c, x, sslope[r], sfar[r]);
    }
}

// ---------------------------------------------------------------- the join
// A block per query row: groups of dk / 4 threads take the slots in turn.
template <typename T>
__global__ void __launch_bounds__(128) paged_attn_join_kernel(const __grid_constant__ PagedAttnArgs a, int dk)
{
    __shared__ float sx[128 * 4], sl[128], red[32];
    const long long row = blockIdx.x;
    int h = static_cast<int>(blockIdx.x);
    const int seq = a.by_heads.split(h), slots = a.slots;
    const bool live = sees(a, seq);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float2* st = a.stat + row * slots;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < slots; i += 128) m = fmaxf(m, st[i].x);
    m = block_max(m, red);
    const float ref = m == -INFINITY ? 0.f : m;
    const int vecs = dk / 4, sets = a.by_vecs.div(128), set = a.by_vecs.div(threadIdx.x), c = (threadIdx.x - set * vecs) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    if (set < sets)
        for (int i = set; i < slots; i += sets) {
            const float2 s = st[i];
            if (s.y == 0.f) continue;                           // nothing was left there, not even sums
            const float e = exp2f(s.x - ref);
            const float4 y = *reinterpret_cast<const float4*>(a.part + (row * slots + i) * dk + c);
            l = fmaf(s.y, e, l);
            x.x = fmaf(y.x, e, x.x); x.y = fmaf(y.y, e, x.y); x.z = fmaf(y.z, e, x.z); x.w = fmaf(y.w, e, x.w);
        }
    *reinterpret_cast<float4*>(sx + threadIdx.x * 4) = x;
    sl[threadIdx.x] = l;
    __syncthreads();
    if (set == 0) {
        for (int i = 1; i < sets; ++i) {
            const int o = (i * vecs + threadIdx.x);
            l += sl[o];
            x.x += sx[o * 4]; x.y += sx[o * 4 + 1]; x.z += sx[o * 4 + 2]; x.w += sx[o * 4 + 3];
        }
        const bool none = l == 0.f || !live;
        const float inv = none ? 0.f : 1.0f / l;
        T* to = static_cast<T*>(a.out) + seq * a.ldo + static_cast<long long>(h) * dk + c;
        to[0] = from_f32<T>(none ? 0.f : x.x * inv); to[1] = from_f32<T>(none ? 0.f : x.y * inv);
        to[2] = from_f32<T>(none ? 0.f : x.z * inv); to[3] = from_f32<T>(none ? 0.f : x.w * inv);
        if (a.lse && threadIdx.x == 0) a.lse[row] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
}

// ---------------------------------------------------------------- how the work is cut
struct AttnPlan { int rt, row_tiles, own_rows, own_tiles, pre_splits, own_splits, own_warps; };
static AttnPlan attn_plan(const nnb200_paged_kv& kv, int groups, int size, int heads, int prefix_stride, int table_stride)
{
    AttnPlan p;
    const int m = heads / kv.kv_heads;
    const long long rows = static_cast<long long>(size) * m;
    // fp32 tiles take 16 query rows; bf16 streams 8 or 16, the shared tiles 32 or 64
    p.rt = kv.dtype == 0 ? 16 : (rows <= 8 ? 8 : (rows <= 16 ? 16 : (rows <= 32 ? 32 : 64)));
    p.own_rows = kv.dtype == 1 && (rows <= 8 || (m <= 8 && rows > 16)) ? 8 : 16;
    p.row_tiles = static_cast<int>(ceil_div(rows, p.rt));
    p.own_tiles = static_cast<int>(ceil_div(m, p.own_rows));
    const long long pre = static_cast<long long>(prefix_stride) * kv.page_size, own = static_cast<long long>(table_stride) * kv.page_size;
    const long long pre_units = static_cast<long long>(groups) * kv.kv_heads * p.row_tiles, own_units = static_cast<long long>(groups) * size * kv.kv_heads * p.own_tiles;
    // cached rows for a block when the tables are full: enough blocks for the machine a few times over, at least two steps each
    const long long blocks = 148LL * 8;
    long long chunk = ceil_div(pre_units * pre + own_units * own, blocks);
    chunk = std::min<long long>(std::max<long long>(ceil_div(chunk, 64) * 64, 128), 1 << 20);
    p.pre_splits = static_cast<int>(ceil_div(pre, chunk));
    p.own_splits = static_cast<int>(ceil_div(own, chunk));
    p.own_warps = kv.dtype == 0 || ceil_div(own, std::max(1, p.own_splits)) > 512 ? 4 : 1;
    return p;
}

template <typename T>
static int attention_t(const nnb200_paged_kv& kv, int layer, PagedAttnArgs a, const AttnPlan& p, void* scratch, cudaStream_t s)
{
    const PagedPool<T> pool = paged_pool<T>(kv, layer);
    const long long rows = static_cast<long long>(a.groups) * a.size * a.heads;
    a.m = FastDiv(a.heads / kv.kv_heads);
    a.row_tiles = FastDiv(p.row_tiles); a.own_tiles = FastDiv(p.own_tiles); a.pre_splits = FastDiv(p.pre_splits); a.own_splits = FastDiv(p.own_splits);
    a.by_size = FastDiv(a.size); a.by_kv_heads = FastDiv(kv.kv_heads); a.by_vecs = FastDiv(kv.head_dim / 4); a.by_heads = FastDiv(a.heads);
    a.pre_slots = p.pre_splits; a.slots = p.pre_splits + p.own_splits; a.own_rows = p.own_rows; a.own_warps = p.own_warps;
    const long long pre_tasks = static_cast<long long>(a.groups) * kv.kv_heads * p.row_tiles * p.pre_splits;
    const long long own_tasks = static_cast<long long>(a.groups) * a.size * kv.kv_heads * p.own_tiles * p.own_splits;
    NNB_ARG_CHECK(pre_tasks + own_tasks <= INT_MAX, "too many queries for one call");
    a.pre_blocks = static_cast<int>(pre_tasks);
    a.tasks = static_cast<int>(pre_tasks + own_tasks);
    const long long blocks = pre_tasks + ceil_div(own_tasks, 4 / p.own_warps);
    a.c = 1.4426950408889634f / sqrtf(static_cast<float>(kv.head_dim));
    a.pairs = ((reinterpret_cast<uintptr_t>(a.q) & 3) == 0 && a.ldq % 2 == 0) ? 1 : 0;
    a.stat = static_cast<float2*>(scratch);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + (rows * a.slots * 8 + 15) / 16 * 16);
    if (blocks > 0) {
        auto go = [&](auto* kernel, int bytes, PerDeviceOnce& once) {
            NNB_TRY(once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); }));
            kernel<<<static_cast<unsigned>(blocks), 128, bytes, s>>>(pool, a);
            NNB_LAUNCH_CHECK();
            return 0;
        };
        auto width = [&](auto dp) {
            constexpr int DP = decltype(dp)::value;
            static PerDeviceOnce once[6];
            if constexpr (sizeof(T) == 4) return go(paged_attn_f32_kernel<DP>, AttnTile32<DP>::SMEM, once[0]);
            else {
                constexpr int both = std::max(AttnTile<DP>::SMEM, AttnStream<DP>::SMEM);
                const bool wide = p.own_rows == 16;
                if (p.rt <= 16) return wide ? go(paged_attn_bf16_kernel<DP, 1, 2>, AttnStream<DP>::SMEM, once[0]) : go(paged_attn_bf16_kernel<DP, 1, 1>, AttnStream<DP>::SMEM, once[1]);
                if (p.rt == 32) return wide ? go(paged_attn_bf16_kernel<DP, 2, 2>, both, once[2]) : go(paged_attn_bf16_kernel<DP, 2, 1>, both, once[3]);
                return wide ? go(paged_attn_bf16_kernel<DP, 4, 2>, both, once[4]) : go(paged_attn_bf16_kernel<DP, 4, 1>, both, once[5]);
            }
        };
        if (kv.head_dim <= 32) NNB_TRY(width(std::integral_constant<int, 32>()));
        else if (kv.head_dim <= 64) NNB_TRY(width(std::integral_constant<int, 64>()));
        else if (kv.head_dim <= 128) NNB_TRY(width(std::integral_constant<int, 128>()));
        else NNB_TRY(width(std::integral_constant<int, 256>()));
    }
    if (a.slots == 1) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows));
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = blocks > 0 ? 1 : 0;
    NNB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<T>, a, kv.head_dim));
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
    const AttnPlan p = attn_plan(*kv, groups, group_size, heads, prefix_stride, table_stride);
    const long long slots = static_cast<long long>(groups) * group_size * heads * (p.pre_splits + p.own_splits);
    return static_cast<size_t>((slots * 8 + 15) / 16 * 16 + slots * kv->head_dim * 4 + 16);
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
    const AttnPlan p = attn_plan(*kv, groups, group_size, heads, prefix_stride, table_stride);
    if (kv->dtype == 0) return attention_t<float>(*kv, layer, a, p, scratch, to_stream(stream));
    return attention_t<bf16>(*kv, layer, a, p, scratch, to_stream(stream));
}

}  // extern "C"
