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
    int own_warps;                  // warps that share a task of own rows: all of a block, or 1 (a task for each)
    int pre_blocks, tasks;          // tasks [0, pre_blocks) are prefixes, a block each; the others own rows
    int first_block;                // of this launch: the prefixes may be another's
    int direct;                     // a block takes a sequence's prefix and its own rows
    int pairs, vectors;             // queries may be read two columns, or 16 bytes, at a time
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
    const int *table, *table2;
    int hk, first, rows, begin, end, place, slot, group, end2;  // end2: rows of a second run, behind the first (short contexts, fp32)
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
    k.table2 = nullptr;
    k.end2 = 0;
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
    if (a.direct) {                                             // the prefix, then the sequence's own rows, by one block
        k.table2 = k.table;
        k.table = a.prefix_table + static_cast<long long>(k.group) * a.prefix_stride;
        k.begin = 0;
        k.end = a.len[seq] < 0 ? 0 : k.place;
        k.end2 = a.table_stride ? held(a.len[seq], a.table_stride, pool.page_shift) : 0;
        k.place = 0;
        k.slot = 0;
        return k;
    }
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
    return pre + (a.table_stride ? held(a.len[seq], a.table_stride, shift) : 0) - 1 - k.place;   // place is 0 where a task has both runs
}

// ---------------------------------------------------------------- bf16: mma.sync tiles
// 64 cached rows a step, a ring of STAGES steps filled by 16-byte asynchronous copies; WM warps take 16 query rows each, the
// 4 / WM warps of a set of rows take turns at the step's cached rows and are joined at the end.  Cached rows that do not
// exist are zero in shared memory (what lies there may be anything, and zero times it must be zero) and -inf as scores.
// Bound by the chain of a step: 64 rows of 16 heads of 64 behind 8192 cached rows (34 MB, 5 us of memory's) take 24.7 us with launch
// and join, one block an SM; more blocks with shorter runs leave more to join than they gain.  Three stages instead of four leave
// room for a fourth block of own rows: 20 queries with up to 512 rows each behind the same 21.4 us to 18.6.
template <int DP> struct AttnTile {
    static constexpr int KT = 64, CPR = DP / 8;                // cached rows a step, 16-byte chunks a row
    static constexpr int STAGES = DP <= 64 ? 3 : 2;
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
            // the weights are rounded to bf16 for the tensor cores (their sum is not): 2^-8 of a weight at most, what rounding V costs too
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
// step, without a barrier, and the warps of a task (one, or all NW of the block) take its steps in turn and are joined at the
// end.  The products are transposed, S' = K Q' and O' = V' P', so that cached rows fill the 16 rows of a tensor core tile and
// queries its 8 columns (NQ = 1 or 2 of them): one query costs half of what it would as one of 16 rows.  P' comes out of the
// first product with cached rows down and queries across; the second wants it the other way round, an 8 x 8 transposition.
// A lane looks up one cached row of a step, a step before it is copied; the copies get it by shuffle.  Rows in shared memory
// are 16 bytes longer than they are: eight neighbours at one column meet no bank twice.  The reference point of the exponentials
// moves only when a score is more than 2^8 above it: scores then need no maximum across lanes.
// Bound by memory, behind 7 us of launch, first rows and join: 16 prefixes of 2047 rows, 16 heads of 64, eight queries each, 134 MB,
// 27.5 us in all; 96 sequences' own rows, up to 1024, 8 heads of 128, 190 MB, 39 us.
template <int DP> struct AttnStream {
    static constexpr int KW = DP <= 32 ? 32 : 16, ST = DP <= 64 ? 3 : 2, PITCH = DP * 2 + 16, CPR = DP / 8;
    static constexpr int PLANE = KW * PITCH, STAGE = 2 * PLANE, RING = ST * STAGE;
    static constexpr int smem(int warps) { return warps * (RING + 16); }
};
// what a score may be above the reference point of its row's exponentials, in powers of two: sums stay far from overflow
constexpr float kAttnSlack = 8.0f;

__device__ __forceinline__ uint32_t transposed8x8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <int DP, int NQ, int NW>
__device__ __forceinline__ void stream_bf16(const PagedPool<bf16>& pool, const PagedAttnArgs& a, const AttnTask& k, uint8_t* smem, int wt)
{
    using Str = AttnStream<DP>;
    constexpr int KW = Str::KW, NK = KW / 16, ND = DP / 16, KS = DP / 16, ST = Str::ST, CPR = Str::CPR;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wk = wt == 1 ? 0 : warp, dk = pool.dk;
    const int run1 = (k.end - k.begin + KW - 1) / KW, all = run1 + (k.end2 + KW - 1) / KW, steps = (all - wk + wt - 1) / wt;
    const uint32_t ring = smem_u32(smem) + warp * Str::RING;
    uint32_t* alive = reinterpret_cast<uint32_t*>(smem + NW * Str::RING) + warp * 4;
    // the cached row this lane looks up for a step (lanes beyond KW: none)
    auto look = [&](int step) {
        const int at = step * wt + wk;
        const bool second = at >= run1;                         // short contexts: the sequence's own rows behind the prefix
        const int t = second ? (at - run1) * KW + lane : k.begin + at * KW + lane;
        return step < steps && lane < KW && t < (second ? k.end2 : k.end) ? pool.find(second ? k.table2 : k.table, k.hk, t) : -1;
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
#pragma unroll 2
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
            const int at = step * wt + wk;
            const float t0 = static_cast<float>((at >= run1 ? k.end + (at - run1) * KW : k.begin + at * KW) + g);
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
                // the weights are rounded to bf16 for the tensor cores (their sum is not): 2^-8 of a weight at most, what rounding V costs too
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
    else asm volatile("barrier.cta.sync 0, %0;" ::"n"(32 * NW) : "memory");
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
    else asm volatile("barrier.cta.sync 0, %0;" ::"n"(32 * NW) : "memory");
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
            float2 st[NW];
#pragma unroll
            for (int w = 0; w < NW; ++w) { st[w] = *reinterpret_cast<const float2*>(s0 + w * (Str::RING / 4) + NQ * 8 * LD + 2 * r); top = fmaxf(top, st[w].x); }
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float e = exp2_fast(st[w].x - ref);
                const float4 y = *reinterpret_cast<const float4*>(s0 + w * (Str::RING / 4) + r * LD + c);
                sum = fmaf(st[w].y, e, sum);
                x.x = fmaf(y.x, e, x.x); x.y = fmaf(y.y, e, x.y); x.z = fmaf(y.z, e, x.z); x.w = fmaf(y.w, e, x.w);
            }
        }
        leave<bf16>(a, k, dk, r, c, x, top, sum);
    }
}

// own rows, tasks counted from a.pre_blocks: block b of them takes one with all its warps, or one with each
template <int DP, int NQ, int NW, int RT>
__device__ __forceinline__ void own_bf16(const PagedPool<bf16>& pool, const PagedAttnArgs& a, int b, uint8_t* smem)
{
    const bool shared = a.own_warps != 1;
    const int task = a.pre_blocks + (shared ? b : b * NW + static_cast<int>(threadIdx.x >> 5));
    if (task >= a.tasks) return;
    const AttnTask k = task_of<RT>(pool, a, task);
    if (k.begin >= k.end && k.end2 == 0) { leave_nothing<bf16>(a, k, pool.dk, shared ? threadIdx.x : threadIdx.x & 31, shared ? 32 * NW : 32); return; }
    stream_bf16<DP, NQ, NW>(pool, a, k, smem, a.own_warps);
}

template <int DP, int WM, int NQ>
__global__ void __launch_bounds__(128) paged_attn_bf16_kernel(PagedPool<bf16> pool, const __grid_constant__ PagedAttnArgs a)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int RT = WM == 1 ? NQ * 8 : WM * 16;
    const int b = static_cast<int>(blockIdx.x) + a.first_block;
    if (b >= a.pre_blocks) { own_bf16<DP, NQ, 4, RT>(pool, a, b - a.pre_blocks, smem); return; }
    const AttnTask k = task_of<RT>(pool, a, b);
    if (k.begin >= k.end) { leave_nothing<bf16>(a, k, pool.dk, threadIdx.x, 128); return; }
    if constexpr (WM == 1) stream_bf16<DP, NQ, 4>(pool, a, k, smem, 4);
    else attend_bf16<DP, WM>(pool, a, k, smem);
}

// ---------------------------------------------------------------- bf16: tcgen05 tiles
// More than 64 query rows of heads up to 64 wide, more than 16 of heads up to 128, on the 5th-generation tensor cores: 128 rows (those
// that are not there are zero) against 128 cached rows a step.  S = Q K' (128 x 128) goes to TMEM, O (128 x DP) stays in TMEM across
// steps.
//   warp 0     looks up the step's pages and loads their rows by TMA, a box of a page (64 rows of a larger one) per lane; pages
//              that are not there are loaded from behind the pool's end, where TMA fills in zeros
//   warp 1     issues the products: S, and O += P V in two halves of 64 cached rows
//   warps 2-9  two threads per query row, half of the columns each: read their 64 scores, make P (bf16, over the scores, for 64
//              cached rows at a time) with the reference point of the exponentials moved, and O rescaled, only when a score is
//              more than 2^8 above it (the one thing the two must agree on); V's rows behind the end are zeroed by these warps
//              before P is handed over, because a page's unused rows may hold anything
// A step is a chain - S, maximum, exponentials, P, P V; two blocks an SM overlap two chains.  P stands in TMEM where its scores
// stood: with P in shared memory the products' operands, P and the arriving tiles asked for 3600 clocks of shared memory's
// bandwidth a step of both blocks, of 4200 that it took, although the next step's S could then start half a P V earlier.  64 cached rows a step instead (an S of 128 x 64 takes the tensor core as long as one of 128 x 128) had the issue
// of products as its bound: 2400 clocks for 64 rows and block, 12 products of 130 clocks.
// Every wait is bounded; one that gives up raises a status word, the others see it, and the block drains: loads and products that
// have been issued are waited for (again with a bound), the two threads of a row leave together, at the barrier where they
// compare notes, and the block's rows are NaN.
__device__ int g_paged_attn_error = 0;

template <int DP> struct AttnTc {
    static constexpr int NS = DP / 64, ST = DP == 64 ? 2 : 1, KT = 128;
    static constexpr int SUB = 128 * 128;                       // bytes of 128 rows by 64 columns
    static constexpr int TILE = NS * SUB;
    static constexpr int OFF_K = TILE, OFF_V = OFF_K + ST * TILE, OFF_X = OFF_V + ST * TILE, OFF_BAR = OFF_X + 2 * 128 * 4;
    static constexpr int TILES = OFF_BAR + 256;                 // two blocks fit an SM: 97.3 KB each with DP = 128, 81.3 KB with 64
    static constexpr uint32_t TMEM_COLS = 256;                  // scores [0, 128), O [128, 128 + DP)
};

// barrier of the two warps that share 32 query rows, and the OR of a flag over them
__device__ __forceinline__ bool pair_any(int quad, bool pred)
{
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 q, %2, 0;\n\t"
        "barrier.cta.red.or.pred p, %1, 64, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r) : "r"(quad + 1), "r"(static_cast<uint32_t>(pred)) : "memory");
    return r != 0;
}

template <int DP>
__device__ __forceinline__ void attend_tc(const PagedPool<bf16>& pool, const PagedAttnArgs& a, const AttnTask& k, const CUtensorMap* tk, const CUtensorMap* tv,
                                          uint8_t* smem)
{
    using Tc = AttnTc<DP>;
    constexpr int ST = Tc::ST, NS = Tc::NS, KT = Tc::KT;
    uint8_t *sQ = smem, *sK = smem + Tc::OFF_K, *sV = smem + Tc::OFF_V;
    float* sX = reinterpret_cast<float*>(smem + Tc::OFF_X);     // (half, row)
    float* sL = reinterpret_cast<float*>(sQ);                   // (half, row), once the query tile has been used
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Tc::OFF_BAR);
    const uint32_t bar0 = smem_u32(bars);
    const uint32_t k_full = bar0, k_empty = bar0 + 8 * ST, v_full = bar0 + 16 * ST, v_empty = bar0 + 24 * ST, s_full = bar0 + 32 * ST,
                   p_full = s_full + 8, pv_done = s_full + 24, q_full = s_full + 32, idle = s_full + 40;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 4 * ST + 6);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dk = pool.dk, ps = 1 << pool.page_shift;
    const int steps = (k.end - k.begin + KT - 1) / KT;
    const int high = min(ps, 64), boxes = KT / high;            // rows of a box, boxes of a step: a run begins at a multiple of 64

    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) { mbar_init(k_full + 8 * i, 1); mbar_init(k_empty + 8 * i, 1); mbar_init(v_full + 8 * i, 1); mbar_init(v_empty + 8 * i, 1); }
        mbar_init(s_full, 1); mbar_init(p_full, 8); mbar_init(p_full + 8, 8); mbar_init(pv_done, 1); mbar_init(q_full, 8); mbar_init(idle, 1);
        *abort_flag = (smem_u32(smem) & 1023u) ? 1 : 0;         // the swizzled tiles need a 1024-byte aligned base
        if (*abort_flag) atomicCAS(&g_paged_attn_error, 0, 9 << 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(Tc::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot, tmem_o = tmem + 128;
    constexpr uint32_t IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(KT >> 3) << 17) | (uint32_t(128 >> 4) << 24);
    constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (uint32_t(DP >> 3) << 17) | (uint32_t(128 >> 4) << 24);
    auto wait = [&](uint32_t bar, int parity, int code) -> bool { return mbar_wait(bar, parity & 1, abort_flag, code, &g_paged_attn_error); };
    auto wait_all = [&](uint32_t bar, int parity, int code) -> bool { return __all_sync(0xffffffffu, wait(bar, parity, code)); };
    // what this block has under way is waited for before it ends, whoever gave up
    auto drain = [&](uint32_t bar, int parity) {
        if (!mbar_drain(bar, parity & 1)) { *abort_flag = 1; atomicCAS(&g_paged_attn_error, 0, 3 << 16); }
    };
    // whether a page of the run is missing: looked over once, by every warp for itself
    bool gaps = false;
    for (int t = k.begin + lane * high; t < k.end; t += 32 * high) gaps |= pool.find(k.table, k.hk, t) < 0;
    gaps = __any_sync(0xffffffffu, gaps);
    // first row in the pool of the box this lane has of step i, -1: it is not there (the whole warp calls this)
    auto box_of = [&](int i) -> int {
        const int t = k.begin + i * KT + lane * high;
        return i < steps && lane < boxes && t < k.end ? pool.find(k.table, k.hk, t) : -1;
    };

    if (warp == 0) {
        const int nowhere = pool.pages * pool.kv_heads * ps;    // a row behind the pool
        bool ok = !*abort_flag;
        int row = box_of(0), k_loads = 0, v_loads = 0;          // steps whose loads have been issued
        for (int i = 0; ok && i < steps; ++i) {
            const int st = i % ST, use = i / ST, y = row < 0 ? nowhere : row;
            if (!(ok = wait_all(k_empty + 8 * st, use + 1, 1))) break;
            if (lane == 0) mbar_expect_tx(k_full + 8 * st, Tc::TILE);
            __syncwarp();
            if (lane < boxes) {
#pragma unroll
                for (int j = 0; j < NS; ++j) tma_load_2d(smem_u32(sK) + st * Tc::TILE + j * Tc::SUB + lane * high * 128, tk, k_full + 8 * st, j * 64, y);
            }
            k_loads = i + 1;
            row = box_of(i + 1);
            if (!(ok = wait_all(v_empty + 8 * st, use + 1, 2))) break;
            if (lane == 0) mbar_expect_tx(v_full + 8 * st, Tc::TILE);
            __syncwarp();
            if (lane < boxes) {
#pragma unroll
                for (int j = 0; j < NS; ++j) tma_load_2d(smem_u32(sV) + st * Tc::TILE + j * Tc::SUB + lane * high * 128, tv, v_full + 8 * st, j * 64, y);
            }
            v_loads = i + 1;
        }
        // a place's loads before its last ones have been used: only these can be under way
        if (lane == 0) {
            for (int i = max(0, k_loads - ST); i < k_loads; ++i) drain(k_full + 8 * (i % ST), i / ST);
            for (int i = max(0, v_loads - ST); i < v_loads; ++i) drain(v_full + 8 * (i % ST), i / ST);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            bool ok = !*abort_flag && wait(q_full, 0, 5);
            const uint64_t dq = smem_desc(smem_u32(sQ), 16, 1024), dkey = smem_desc(smem_u32(sK), 16, 1024),
                           dv = smem_desc(smem_u32(sV), Tc::SUB, 1024);          // addresses in units of 16 bytes: offsets are added below
            auto issue_s = [&](int i) -> bool {
                const int st = i % ST;
                if (!wait(k_full + 8 * st, i / ST, 6)) return false;
                tc_fence_after();
#pragma unroll
                for (int x = 0; x < DP / 16; ++x) {
                    const int o = ((x >> 2) * Tc::SUB + (x & 3) * 32) >> 4;
                    umma_bf16(tmem, dq + o, dkey + (st * Tc::TILE >> 4) + o, IDESC_S, x > 0 ? 1u : 0u);
                }
                umma_commit(s_full);
                umma_commit(k_empty + 8 * st);
                return true;
            };
            auto issue_pv = [&](int i, int part) -> bool {
                const int st = i % ST;
                if (!wait(p_full + 8 * part, i, 7)) return false;
                tc_fence_after();
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    umma_bf16_ta(tmem_o, tmem + part * 64 + (x >> 1) * 32 + (x & 1) * 8, dv + (st * Tc::TILE >> 4) + ((part * 4 + x) * 2048 >> 4), IDESC_PV, i > 0 || part > 0 || x > 0 ? 1u : 0u);
                return true;
            };
            if (ok) ok = issue_s(0);
            for (int i = 0; ok && i < steps; ++i) {
                const int st = i % ST;
                if (!(ok = wait(v_full + 8 * st, i / ST, 8))) break;
                if (!(ok = issue_pv(i, 0))) break;
                if (!(ok = issue_pv(i, 1))) break;
                umma_commit(pv_done);
                umma_commit(v_empty + 8 * st);
                if (i + 1 == steps) break;
                // the next scores take the columns of this step's, where P stands
                if (!(ok = wait(pv_done, i, 15))) break;
                if (!(ok = issue_s(i + 1))) break;
            }
            umma_commit(idle);                                  // every product that was issued
            drain(idle, 0);
        }
    } else {
        const int quad = warp & 3, half = (warp - 2) >> 2, row = quad * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const int sw = row & 7;
        const bool live = row < k.rows, work = quad * 32 < k.rows;   // of a warp without rows the scores serve as P: its rows of O are nobody's
        const AttnRow w = row_of(a, k, live ? row : 0);
        {   // half of the query row, zero where there is none
            const bf16* q = static_cast<const bf16*>(a.q) + w.seq * a.ldq + static_cast<long long>(w.head) * dk;
#pragma unroll 2
            for (int c = 0; c < DP / 16; ++c) {
                const int cc = half * (DP / 16) + c;
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (live && cc * 8 < dk) {
                    if (a.vectors) v = *reinterpret_cast<const uint4*>(q + cc * 8);
                    else {
                        alignas(16) bf16 x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = q[cc * 8 + e];
                        v = *reinterpret_cast<const uint4*>(x);
                    }
                }
                *reinterpret_cast<uint4*>(sQ + (cc >> 3) * Tc::SUB + row * 128 + (((cc & 7) ^ sw) << 4)) = v;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        const float mul = a.alibi ? 1.f : a.c;
        const float slope = a.alibi && live ? alibi_slope2(w.head, a.heads) : 0.f;
        const float far = a.alibi && live ? static_cast<float>(far_of(a, pool.page_shift, k, w.seq)) : 0.f;
        float m = -INFINITY, l = 0.f;
        bool bad = *abort_flag != 0;                            // a wait of this thread gave up
        for (int i = 0; i < steps; ++i) {
            const int st = i % ST;
            // bit r of there[p]: row p * 64 + half * 32 + r of the step is there; all of them but for the last step and missing pages
            const int t0 = k.begin + i * KT;
            const bool whole = !gaps && t0 + KT <= k.end;
            uint32_t there[2] = {0xffffffffu, 0xffffffffu};
            // before all else: it also says that the step before has used its V, whose place this step's takes
            bad |= !wait_all(s_full, i, 11);
            if (!whole) {
                // rows [from, from + count) of the step are this lane's, as bits of its 128
                const int from = lane * high, count = box_of(i) < 0 ? 0 : min(high, k.end - (t0 + from));
                uint32_t word[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int b0 = max(from - x * 32, 0), b1 = min(from + (lane < boxes ? count : 0) - x * 32, 32);
                    word[x] = __reduce_or_sync(0xffffffffu, b1 <= b0 ? 0u : (b1 - b0 == 32 ? 0xffffffffu : ((1u << (b1 - b0)) - 1u) << b0));
                }
                there[0] = half ? word[1] : word[0];
                there[1] = half ? word[3] : word[2];
                bad |= !wait_all(v_full + 8 * st, i / ST, 10);
                for (int idx = threadIdx.x - 64; idx < KT * NS * 8; idx += 256) {
                    const int r = (idx >> 3) % KT;
                    const uint32_t wd = r < 64 ? (r < 32 ? word[0] : word[1]) : (r < 96 ? word[2] : word[3]);
                    if (!(wd >> (r & 31) & 1u)) *reinterpret_cast<uint4*>(sV + st * Tc::TILE + (idx >> 3) / KT * Tc::SUB + r * 128 + (idx & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            // 32 scores of part p (cached rows [64 p, 64 p + 64) of the step), biased and masked
            auto scores = [&](int p, float (&x)[32]) {
                uint32_t r[32];
                tmem_ld32(tmem + lanes + p * 64 + half * 32, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(r[j]);
                if (a.alibi) {
                    const float f0 = far - static_cast<float>(t0 + p * 64 + half * 32);
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = x[j] * a.c - slope * (f0 - static_cast<float>(j));
                }
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) if (!(there[p] >> j & 1u)) x[j] = -INFINITY;
                }
            };
            float x[32];
            uint32_t pk[16];
            uint64_t sum0 = 0ull, sum1 = 0ull;
            auto most = [&](const float (&x)[32]) -> float {
                float top4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int j = 4; j < 32; ++j) top4[j & 3] = fmaxf(top4[j & 3], x[j]);
                return fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
            };
            auto exponentials = [&](const float (&x)[32]) {
                const float ref = m == -INFINITY ? 0.f : m;
                const uint64_t mul_2 = pack2(mul, mul), ref_2 = pack2(-ref, -ref);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    float e0, e1;
                    unpack2(fma2(pack2(x[2 * j], x[2 * j + 1]), mul_2, ref_2), e0, e1);
                    e0 = exp2_fast(e0);
                    e1 = exp2_fast(e1);
                    if (j & 1) sum1 = add2(sum1, pack2(e0, e1));
                    else sum0 = add2(sum0, pack2(e0, e1));
                    pk[j] = pack_bf16x2(e0, e1);                // rounded for the tensor cores, summed as they are
                }
            };
            auto hand_over = [&](int p) {
                if (work) {
                    tmem_st16(tmem + lanes + p * 64 + half * 32, pk);   // over scores that only this warp reads, and has read
                    tmem_st_wait();
                }
                tc_fence_before();
                if (!whole) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * p);     // a barrier for each part: a warp may be done with both before others with one
            };
            if (work) {
                tc_fence_after();
                // part 0 against the point so far, which is right but for the first steps
                scores(0, x);
                float top = most(x);
                exponentials(x);
                scores(1, x);
                top = fmaxf(top, most(x)) * mul;
                if (pair_any(quad, top > m + kAttnSlack || bad)) {
                    // both threads take the same point, the maximum itself: one that is rounded up lies above large scores by more
                    // than their exponentials can bear (a step of bf16 is 256 beyond 2^15)
                    sX[half * 128 + row] = top;
                    if (pair_any(quad, bad)) { bad = true; break; }              // both warps leave here
                    top = fmaxf(top, sX[(half ^ 1) * 128 + row]);
                    const bool move = top > m + kAttnSlack;
                    const float back = move ? exp2_fast(m - top) : 1.0f;          // 0 from -inf
                    if (move) m = top;
                    l *= back;
                    if (i > 0) {                                // the products of the step before are in: this one's scores came after them
#pragma unroll 1
                        for (int c = 0; c < DP / 2; c += 32) {
                            uint32_t r[32];
                            tmem_ld32(tmem_o + lanes + half * (DP / 2) + c, r);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * back);
                            tmem_st32(tmem_o + lanes + half * (DP / 2) + c, r);
                        }
                        tmem_st_wait();
                    }
                    sum0 = sum1 = 0ull;
                    scores(0, x);
                    exponentials(x);
                    scores(1, x);
                }
            }
            hand_over(0);
            if (work) exponentials(x);
            hand_over(1);
            float s0, s1;
            unpack2(add2(sum0, sum1), s0, s1);
            l += s0 + s1;
            if (!work && bad) break;
        }
        if (work) {
            bad |= !wait_all(pv_done, steps - 1, 14);
            sL[half * 128 + row] = l;
            if (!pair_any(quad, bad)) {
                l += sL[(half ^ 1) * 128 + row];
                tc_fence_after();
                // through shared memory (the last products have read K and V), so that a row is written by neighbouring threads
                constexpr int VECS = DP / 8, ROWS = 32 / VECS;  // 16 bytes at a time: a warp's half of a row, rows at a time
                static_assert(8 * 32 * VECS * 16 <= 2 * ST * Tc::TILE, "the sums fit the tiles");
                uint8_t* stage = sK + (warp - 2) * 32 * VECS * 16;
#pragma unroll 1
                for (int c = 0; c < DP / 2; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem_o + lanes + half * (DP / 2) + c, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *reinterpret_cast<uint4*>(stage + (lane * VECS + (((c + j) / 4) ^ sw)) * 16) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                }
                __syncwarp();
#pragma unroll 2
                for (int r0 = 0; r0 < 32; r0 += ROWS) {
                    const int r = r0 + lane / VECS, v = lane % VECS, c = half * (DP / 2) + v * 4;
                    const float4 o = *reinterpret_cast<const float4*>(stage + (r * VECS + (v ^ (r & 7))) * 16);
                    const float mr = __shfl_sync(0xffffffffu, m, r), lr = __shfl_sync(0xffffffffu, l, r);
                    if (quad * 32 + r < k.rows && c < dk) leave<bf16>(a, k, dk, quad * 32 + r, c, o, mr, lr);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    // a block that gave up has rows it did not write, or in part: NaN, which the join keeps, instead of an earlier call's
    if (*abort_flag)
        for (int idx = threadIdx.x; idx < k.rows * (dk / 4); idx += 320)
            leave<bf16>(a, k, dk, a.by_vecs.div(idx), (idx - a.by_vecs.div(idx) * (dk / 4)) * 4, make_float4(NAN, NAN, NAN, NAN), -INFINITY, NAN);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Tc::TMEM_COLS) : "memory");
    }
}

// Prefixes only.  The own rows' kernel goes first, 16 warps an SM as it needs them for memory's sake; this one's blocks move in as
// its last ones leave.
template <int DP>
__global__ void __launch_bounds__(320, 2) paged_attn_tc_kernel(PagedPool<bf16> pool, const __grid_constant__ PagedAttnArgs a, const __grid_constant__ CUtensorMap tk,
                                                               const __grid_constant__ CUtensorMap tv)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const AttnTask k = task_of<128>(pool, a, static_cast<int>(blockIdx.x));
    if (k.begin < k.end) attend_tc<DP>(pool, a, k, &tk, &tv, smem);
    else leave_nothing<bf16>(a, k, pool.dk, threadIdx.x, 320);
    // the join waits for this kernel; with this it has waited for the one in front too
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

int paged_attn_device_error(int* code)
{
    NNB_CUDA_CHECK(cudaMemcpyFromSymbol(code, g_paged_attn_error, sizeof(int)));
    if (*code) { const int z = 0; NNB_CUDA_CHECK(cudaMemcpyToSymbol(g_paged_attn_error, &z, sizeof(int))); }
    return 0;
}

// ---------------------------------------------------------------- fp32: FMA tiles
// RT (4, 8 or 16) query rows against KT cached rows a step, 256 threads.  Scores: a thread takes one cached row and RT KT / 256 query
// rows; softmax: up to a warp per query row; values: a thread takes four columns and every KG-th cached row, for all query rows,
// and the KG parts are summed at the end.  Rows in shared memory are 16 bytes longer than they are, so that eight neighbours'
// 16-byte reads meet no bank twice.  fp32 products and sums throughout: infinities and NaN behave as in the formula, which
// splitting a number into parts for the tensor cores would not keep.  With few rows a step is a chain of dependent
// instructions: eight warps and a fixed RT, instead of four that count rows, took 13.5 us to 10.9 for eight beams of 12 heads
// behind 901 rows (9.2 since the join and the runs were changed).
constexpr int kF32Threads = 256;
template <int DP, int RT> struct AttnTile32 {
    static constexpr int KT = DP <= 64 ? 64 : 4096 / DP, LD = DP + 4, CPR = DP / 4, STAGES = 2;
    static constexpr int SETS = kF32Threads / KT, RPT = RT > SETS ? RT / SETS : 1;      // sets of threads, query rows of each
    static constexpr int KG = kF32Threads * 4 / DP, PL = RT + 4;   // sets of cached rows for the values, row of the weights
    static constexpr int LPR = kF32Threads / RT < 32 ? kF32Threads / RT : 32, KPL = KT / LPR > 0 ? KT / LPR : 1;   // lanes of a softmax row, cached rows of each
    static constexpr int FLOATS = KT * LD;                     // K, or V, of a stage
    static constexpr int RING = STAGES * 2 * FLOATS > KG * RT * DP ? STAGES * 2 * FLOATS : KG * RT * DP;
    static constexpr int SMEM = (RING + RT * DP + KT * PL + 4 * RT) * 4 + STAGES * KT;
};

template <int DP, int RT>
__device__ __forceinline__ void attend_f32(const PagedPool<float>& pool, const PagedAttnArgs& a, const AttnTask& k, uint8_t* smem)
{
    using Tile = AttnTile32<DP, RT>;
    constexpr int KT = Tile::KT, ST = Tile::STAGES, PL = Tile::PL, NTH = kF32Threads;
    const int tid = threadIdx.x, dk = pool.dk, steps1 = max(0, (k.end - k.begin + KT - 1) / KT), steps = steps1 + (k.end2 + KT - 1) / KT;
    if (steps == 0) { leave_nothing<float>(a, k, dk, tid, NTH); return; }
    float* ring = reinterpret_cast<float*>(smem);
    float *sq = ring + Tile::RING, *sp = sq + RT * DP, *sback = sp + KT * PL, *sslope = sback + RT, *sfar = sslope + RT;
    uint8_t* alive = reinterpret_cast<uint8_t*>(sfar + 2 * RT);
    const uint32_t base = smem_u32(ring);
    auto load = [&](int step, int stage) {
        const bool second = step >= steps1;
        const int* table = second ? k.table2 : k.table;
        const int t0 = second ? (step - steps1) * KT : k.begin + step * KT, end = second ? k.end2 : k.end;
#pragma unroll
        for (int i = 0; i < KT * Tile::CPR / NTH; ++i) {
            const int idx = tid + i * NTH, r = idx / Tile::CPR, c = idx % Tile::CPR, t = t0 + r;
            const int row = t < end ? pool.find(table, k.hk, t) : -1;
            const bool there = row >= 0, in = there && c * 4 < dk;
            const long long off = in ? static_cast<long long>(row) * dk + c * 4 : 0;
            const uint32_t dst = base + (stage * 2 * Tile::FLOATS + r * Tile::LD + c * 4) * 4;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(pool.k + off), "r"(in ? 16 : 0) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + Tile::FLOATS * 4), "l"(pool.v + off), "r"(in ? 16 : 0) : "memory");
            if (c == 0) alive[stage * KT + r] = there;
        }
    };
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) { if (i < steps) load(i, i); cp_commit(); }
    for (int i = tid; i < RT * DP; i += NTH) {
        const int r = i / DP, c = i - r * DP;
        const AttnRow w = row_of(a, k, min(r, k.rows - 1));
        sq[i] = r < k.rows && c < dk ? static_cast<const float*>(a.q)[w.seq * a.ldq + static_cast<long long>(w.head) * dk + c] : 0.f;
    }
    if (tid < RT) {
        const bool on = a.alibi && tid < k.rows;
        const AttnRow w = row_of(a, k, on ? tid : 0);
        sslope[tid] = on ? alibi_slope2(w.head, a.heads) : 0.f;
        sfar[tid] = on ? static_cast<float>(far_of(a, pool.page_shift, k, w.seq)) : 0.f;
    }
    const int key = tid % KT, set = tid / KT;                   // scores: query rows set, set + SETS, ..
    const int srow = tid / Tile::LPR, part = tid % Tile::LPR;   // softmax
    const int c4 = tid % (DP / 4), kg = tid / (DP / 4);         // values
    float m = -INFINITY, l = 0.f, o[RT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[r][j] = 0.f;

    for (int step = 0; step < steps; ++step) {
        cp_wait<ST - 2>();
        __syncthreads();
        const int stage = step % ST;
        if (step + ST - 1 < steps) load(step + ST - 1, (step + ST - 1) % ST);
        cp_commit();
        const float *sk = ring + stage * 2 * Tile::FLOATS, *sv = sk + Tile::FLOATS;
        if (set < RT) {
            float s[Tile::RPT];
#pragma unroll
            for (int i = 0; i < Tile::RPT; ++i) s[i] = 0.f;
#pragma unroll 4
            for (int d = 0; d < DP; d += 4) {
                const float4 kv = *reinterpret_cast<const float4*>(sk + key * Tile::LD + d);
#pragma unroll
                for (int i = 0; i < Tile::RPT; ++i) {
                    const float4 q = *reinterpret_cast<const float4*>(sq + (set + Tile::SETS * i) * DP + d);
                    s[i] = fmaf(q.x, kv.x, s[i]); s[i] = fmaf(q.y, kv.y, s[i]); s[i] = fmaf(q.z, kv.z, s[i]); s[i] = fmaf(q.w, kv.w, s[i]);
                }
            }
            const bool there = alive[stage * KT + key];
            const float t = static_cast<float>((step >= steps1 ? k.end + (step - steps1) * KT : k.begin + step * KT) + key);
#pragma unroll
            for (int i = 0; i < Tile::RPT; ++i) {
                const int r = set + Tile::SETS * i;
                sp[key * PL + r] = there ? s[i] * a.c - sslope[r] * (sfar[r] - t) : -INFINITY;
            }
        }
        __syncthreads();
        bool moved = false;
        if (srow < RT) {
            float s[Tile::KPL], top = m;
#pragma unroll
            for (int j = 0; j < Tile::KPL; ++j) { s[j] = part + Tile::LPR * j < KT ? sp[(part + Tile::LPR * j) * PL + srow] : -INFINITY; top = fmaxf(top, s[j]); }
#pragma unroll
            for (int w = 1; w < Tile::LPR; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const float ref = top == -INFINITY ? 0.f : top, back = exp2f(m - ref);
            moved = top != m;
            l *= back;
            m = top;
#pragma unroll
            for (int j = 0; j < Tile::KPL; ++j) {
                s[j] = exp2f(s[j] - ref);
                l += s[j];
                if (part + Tile::LPR * j < KT) sp[(part + Tile::LPR * j) * PL + srow] = s[j];
            }
            if (part == 0) sback[srow] = back;
        }
        if (__syncthreads_or(moved)) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const float b = sback[r];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[r][j] *= b;
            }
        }
#pragma unroll 2
        for (int t = kg; t < KT; t += Tile::KG) {
            const float4 v = *reinterpret_cast<const float4*>(sv + t * Tile::LD + c4 * 4);
#pragma unroll
            for (int rq = 0; rq < RT / 4; ++rq) {
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
    for (int w = 1; w < Tile::LPR; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
    cp_wait<0>();
    __syncthreads();
    if (part == 0 && srow < RT) { sslope[srow] = m; sfar[srow] = l; }
#pragma unroll
    for (int r = 0; r < RT; ++r)
        if (r < k.rows) *reinterpret_cast<float4*>(ring + (kg * RT + r) * DP + c4 * 4) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
    __syncthreads();
    const int vecs = dk / 4;
    for (int idx = tid; idx < k.rows * vecs; idx += NTH) {
        const int r = a.by_vecs.div(idx), c = (idx - r * vecs) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < Tile::KG; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(ring + (w * RT + r) * DP + c);
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        leave<float>(a, k, dk, r, c, x, sslope[r], sfar[r]);
    }
}

// RT rows of a group against its prefix, RO of a sequence against its own rows
template <int DP, int RT, int RO>
__global__ void __launch_bounds__(kF32Threads) paged_attn_f32_kernel(PagedPool<float> pool, const __grid_constant__ PagedAttnArgs a)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int b = static_cast<int>(blockIdx.x);
    const AttnTask k = task_of<RT>(pool, a, b);
    if (RT == RO || b < a.pre_blocks) attend_f32<DP, RT>(pool, a, k, smem);
    else attend_f32<DP, RO>(pool, a, k, smem);
}

// ---------------------------------------------------------------- the join
// A block per query row: groups of dk / 4 threads take the slots in turn.  A few latencies of L2 and no work to speak of: about 2 us
// behind the last block of the kernel in front, 6 us for 96 queries of 32 heads of 128 and 13 places (20 MB) because not all blocks
// are resident at a time.  Loading the first places before their maximum is known took 0.8 us out.  Blocks of 64 threads where rows are
// many and narrow: 64 groups of eight behind 300 rows, 16 heads of 64, 75.9 us to 72.1 in all; of 128 columns no difference.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) paged_attn_join_kernel(const __grid_constant__ PagedAttnArgs a, int dk)
{
    __shared__ float sx[NT * 4], sl[NT], red[32];
    const long long row = blockIdx.x;
    int h = static_cast<int>(blockIdx.x);
    const int seq = a.by_heads.split(h), slots = a.slots;
    const bool live = sees(a, seq);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int vecs = dk / 4, sets = a.by_vecs.div(NT), set = a.by_vecs.div(threadIdx.x), c = (threadIdx.x - set * vecs) * 4;
    const float2* st = a.stat + row * slots;
    const float* part = a.part + row * slots * dk + c;
    // a thread's first places are under way before their maximum is known
    constexpr int AHEAD = 4;
    float2 s[AHEAD];
    float4 y[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        const int i = set + u * sets;
        const bool there = set < sets && i < slots;
        s[u] = there ? st[i] : make_float2(-INFINITY, 0.f);
        y[u] = there ? *reinterpret_cast<const float4*>(part + static_cast<long long>(i) * dk) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) m = fmaxf(m, s[u].x);
    for (int i = AHEAD * sets + threadIdx.x; i < slots; i += NT) m = fmaxf(m, st[i].x);
    m = block_max(m, red);
    const float ref = m == -INFINITY ? 0.f : m;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    auto add = [&](const float2& s, const float4& y) {
        if (s.y == 0.f) return;                                 // nothing was left there, not even sums
        const float e = exp2f(s.x - ref);
        l = fmaf(s.y, e, l);
        x.x = fmaf(y.x, e, x.x); x.y = fmaf(y.y, e, x.y); x.z = fmaf(y.z, e, x.z); x.w = fmaf(y.w, e, x.w);
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) add(s[u], y[u]);
    if (set < sets)
        for (int i = set + AHEAD * sets; i < slots; i += sets) add(st[i], *reinterpret_cast<const float4*>(part + static_cast<long long>(i) * dk));
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
struct AttnPlan { bool tc, direct; int rt, row_tiles, own_rows, own_tiles, pre_splits, own_splits, own_warps; };
static AttnPlan attn_plan(const nnb200_paged_kv& kv, int groups, int size, int heads, int prefix_stride, int table_stride)
{
    AttnPlan p;
    const int m = heads / kv.kv_heads;
    const long long rows = static_cast<long long>(size) * m;
    // bf16: warps stream up to 16 query rows; beyond that mma.sync tiles take up to 64 of heads up to 64 wide, and the tcgen05 tiles
    // all of wider ones and more than 64 (us, tcgen05 | mma.sync, heads of 64 behind 8192 rows and own ones: 20 rows 27.2 | 21.5,
    // 64 rows 36.5 | 31.0; heads of 128 behind 32768: 32 rows 44.5, 64 rows 46.7, where mma.sync tiles took 72 and 87, and 17 rows
    // of them 43.7 where the stream takes 47.0 for 16); heads over 128 have only mma.sync tiles
    p.tc = kv.dtype == 1 && rows > (kv.head_dim <= 64 ? 64 : 16) && kv.head_dim <= 128 && prefix_stride > 0;
    const int few = std::max<long long>(prefix_stride > 0 ? rows : 0, m) <= 4 ? 4 : (std::max<long long>(prefix_stride > 0 ? rows : 0, m) <= 8 ? 8 : 16);
    p.rt = kv.dtype == 0 ? few : (p.tc ? 128 : (rows <= 8 ? 8 : (rows <= 16 || prefix_stride == 0 ? 16 : (rows <= 32 && kv.head_dim <= 64 ? 32 : 64))));
    p.own_rows = kv.dtype == 0 ? (m <= 4 ? 4 : p.rt) : p.tc || (kv.dtype == 1 && (rows <= 8 || (m <= 8 && rows > 16))) ? 8 : 16;
    p.row_tiles = static_cast<int>(std::max(1LL, ceil_div(rows, p.rt)));
    p.own_tiles = static_cast<int>(ceil_div(m, p.own_rows));
    const long long pre = static_cast<long long>(prefix_stride) * kv.page_size, own = static_cast<long long>(table_stride) * kv.page_size;
    const long long pre_units = static_cast<long long>(groups) * kv.kv_heads * p.row_tiles, own_units = static_cast<long long>(groups) * size * kv.kv_heads * p.own_tiles;
    // Rows of a run that a block takes when the tables are full.  Fewer make more partial results to write and join, more leave
    // SMs idle behind the last ones (us, eight beams of 12 fp32 heads behind 901 rows: 64 rows 9.0, 128 10.5, 256 13.9, but behind
    // 2000, where 64 are more than two blocks an SM, 14.5, 11.3, 14.7; two sequences of 32 bf16 heads behind 4000: 128 rows
    // 15.2, 256 13.0; 64 queries of 16 heads behind 8192: 384 rows 41.5, 768 31.1, 2048 46).
    const bool f32 = kv.dtype == 0;
    const long long least = f32 ? (pre_units * ceil_div(pre, 64) <= 148 * 2 ? 64 : 128) : (p.rt <= 16 ? 256 : 128);
    const long long share = ceil_div(ceil_div(pre_units * pre + own_units * own, 148LL * (f32 ? 4 : 6)), 64) * 64;
    const long long chunk = std::min<long long>(std::max(share, least), 1 << 20);
    p.pre_splits = static_cast<int>(ceil_div(pre, chunk));
    if (p.tc) p.pre_splits = static_cast<int>(std::min<long long>(std::max<long long>(148 * 2 / std::max(pre_units, 1LL), 1), ceil_div(pre, 256)));
    // (tcgen05 tiles, one wave of blocks: 48 queries behind 901 rows, one head, 16.5 us with 256 rows a block at least, 22.9 with 512)
    // own rows in bf16: 128 a warp, and four warps a task where there are that many (64 sequences of 16 heads with up to 512: 34.6 us
    // with a warp for all of them, 31.5 with one for 128, 30.2 with a block; 128 sequences with up to 256: 41.0, 38.1, 39.4)
    p.own_warps = f32 || own >= 512 ? 4 : 1;
    p.own_splits = static_cast<int>(ceil_div(own, f32 ? chunk : 128 * p.own_warps));
    // a block for a short prefix and the own rows behind it, without the join (us against the three launches' work in two, four beams of
    // six heads: bf16 behind 41 rows 3.6 | 5.0, 200 rows 5.9 | 6.6; fp32, whose scores and values are plain products, behind 41 rows
    // 5.6 | 5.5 with a launch less, 90 rows 7.3 | 5.7)
    p.direct = !p.tc && pre > 0 && own > 0 && pre + own <= (f32 ? 64 : 256) && static_cast<long long>(groups) * size * kv.kv_heads <= 4 * 148;
    if (p.direct) {
        p.rt = p.own_rows = kv.dtype == 0 && m <= 4 ? 4 : (m <= 8 ? 8 : 16);
        p.own_tiles = static_cast<int>(ceil_div(m, p.own_rows));
        p.pre_splits = 0;
        p.own_splits = 1;
    }
    if (p.direct) p.own_warps = 4;
    return p;
}

// a launch that may begin while the kernel in front of it runs (`early`)
template <typename... P, typename... A>
static int launch_behind(void (*kernel)(P...), unsigned blocks, int threads, int bytes, bool early, cudaStream_t s, const A&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = early ? 1 : 0;
    NNB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
    NNB_LAUNCH_CHECK();
    return 0;
}

template <typename T>
static int attention_t(const nnb200_paged_kv& kv, int layer, PagedAttnArgs a, const AttnPlan& p, void* scratch, cudaStream_t s)
{
    const PagedPool<T> pool = paged_pool<T>(kv, layer);
    const long long rows = static_cast<long long>(a.groups) * a.size * a.heads;
    a.m = FastDiv(a.heads / kv.kv_heads);
    a.row_tiles = FastDiv(p.row_tiles); a.own_tiles = FastDiv(p.own_tiles); a.pre_splits = FastDiv(p.pre_splits); a.own_splits = FastDiv(p.own_splits);
    a.by_size = FastDiv(a.size); a.by_kv_heads = FastDiv(kv.kv_heads); a.by_vecs = FastDiv(kv.head_dim / 4); a.by_heads = FastDiv(a.heads);
    a.pre_slots = p.pre_splits; a.slots = p.pre_splits + p.own_splits; a.own_rows = p.own_rows; a.own_warps = p.own_warps; a.direct = p.direct ? 1 : 0;
    const long long pre_tasks = static_cast<long long>(a.groups) * kv.kv_heads * p.row_tiles * p.pre_splits;
    const long long own_tasks = static_cast<long long>(a.groups) * a.size * kv.kv_heads * p.own_tiles * p.own_splits;
    NNB_ARG_CHECK(pre_tasks + own_tasks <= INT_MAX, "too many queries for one call");
    a.pre_blocks = static_cast<int>(pre_tasks);
    a.tasks = static_cast<int>(pre_tasks + own_tasks);
    const long long blocks = pre_tasks + ceil_div(own_tasks, 4 / p.own_warps);
    a.c = 1.4426950408889634f / sqrtf(static_cast<float>(kv.head_dim));
    a.pairs = ((reinterpret_cast<uintptr_t>(a.q) & 3) == 0 && a.ldq % 2 == 0) ? 1 : 0;
    a.vectors = ((reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.ldq % 8 == 0) ? 1 : 0;
    a.stat = static_cast<float2*>(scratch);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + (rows * a.slots * 8 + 15) / 16 * 16);
    if (blocks > 0) {
        a.first_block = p.tc ? a.pre_blocks : 0;
        auto go = [&](auto* kernel, int bytes, PerDeviceOnce& once) {
            NNB_TRY(once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); }));
            if (blocks == a.first_block) return 0;
            kernel<<<static_cast<unsigned>(blocks - a.first_block), sizeof(T) == 4 ? kF32Threads : 128, bytes, s>>>(pool, a);
            NNB_LAUNCH_CHECK();
            return 0;
        };
        auto width = [&](auto dp) {
            constexpr int DP = decltype(dp)::value;
            static PerDeviceOnce once[6];
            if constexpr (sizeof(T) == 4) {
                const bool narrow = p.own_rows == 4;
                if (p.rt == 4) return go(paged_attn_f32_kernel<DP, 4, 4>, AttnTile32<DP, 4>::SMEM, once[0]);
                if (p.rt == 8) return narrow ? go(paged_attn_f32_kernel<DP, 8, 4>, AttnTile32<DP, 8>::SMEM, once[1]) : go(paged_attn_f32_kernel<DP, 8, 8>, AttnTile32<DP, 8>::SMEM, once[2]);
                return narrow ? go(paged_attn_f32_kernel<DP, 16, 4>, AttnTile32<DP, 16>::SMEM, once[3]) : go(paged_attn_f32_kernel<DP, 16, 16>, AttnTile32<DP, 16>::SMEM, once[4]);
            }
            else {
                const bool wide = p.own_rows == 16;
                constexpr int both = DP == 128 ? 0 : std::max(AttnTile<DP>::SMEM, AttnStream<DP>::smem(4));
                if constexpr (DP != 128) if (p.rt == 64) return wide ? go(paged_attn_bf16_kernel<DP, 4, 2>, both, once[2]) : go(paged_attn_bf16_kernel<DP, 4, 1>, both, once[3]);
                if constexpr (DP <= 64) if (p.rt == 32) return wide ? go(paged_attn_bf16_kernel<DP, 2, 2>, both, once[4]) : go(paged_attn_bf16_kernel<DP, 2, 1>, both, once[5]);
                return wide ? go(paged_attn_bf16_kernel<DP, 1, 2>, AttnStream<DP>::smem(4), once[0]) : go(paged_attn_bf16_kernel<DP, 1, 1>, AttnStream<DP>::smem(4), once[1]);
            }
        };
        if (kv.head_dim <= 32) NNB_TRY(width(std::integral_constant<int, 32>()));
        else if (kv.head_dim <= 64) NNB_TRY(width(std::integral_constant<int, 64>()));
        else if (kv.head_dim <= 128) NNB_TRY(width(std::integral_constant<int, 128>()));
        else NNB_TRY(width(std::integral_constant<int, 256>()));
        if constexpr (sizeof(T) == 2) if (p.tc) {
            const long long pool_rows = static_cast<long long>(kv.pages) * kv.kv_heads * kv.page_size;
            CUtensorMap tk, tv;
            NNB_TRY(tensor_map_2d(pool.k, kv.head_dim, pool_rows, kv.head_dim, 64, std::min(kv.page_size, 64), &tk, 2));
            NNB_TRY(tensor_map_2d(pool.v, kv.head_dim, pool_rows, kv.head_dim, 64, std::min(kv.page_size, 64), &tv, 2));
            auto tc = [&](auto* kernel, int bytes, PerDeviceOnce& once) {
                NNB_TRY(once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); }));
                return launch_behind(kernel, static_cast<unsigned>(a.pre_blocks), 320, bytes, own_tasks > 0, s, pool, a, tk, tv);
            };
            static PerDeviceOnce once[2];
            if (kv.head_dim <= 64) NNB_TRY(tc(paged_attn_tc_kernel<64>, AttnTc<64>::TILES, once[0]));
            else NNB_TRY(tc(paged_attn_tc_kernel<128>, AttnTc<128>::TILES, once[1]));
        }
    }
    if (a.slots == 1) return 0;
    if (rows > 148 * 16 && kv.head_dim <= 64) NNB_TRY(launch_behind(paged_attn_join_kernel<T, 64>, static_cast<unsigned>(rows), 64, 0, blocks > 0, s, a, kv.head_dim));
    else NNB_TRY(launch_behind(paged_attn_join_kernel<T, 128>, static_cast<unsigned>(rows), 128, 0, blocks > 0, s, a, kv.head_dim));
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
