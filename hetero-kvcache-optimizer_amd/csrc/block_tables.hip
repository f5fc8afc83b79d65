// Block tables of sequences that share INT4 records: extend, select, compact.
//
// State (HkvBlockTables): per row the ids of its ceil(len / 16) blocks, per block the number
// of rows that hold it, and a bitmap of the blocks that none holds.  The bitmap is what makes
// "the lowest free ids" cheap: 256K blocks are 32 KB, which one workgroup counts in one pass.
// Thread t counts the bits of its kept run of words, one scan over the threads gives the rank of
// every run's first free block, and each thread lists its own.
//
// Each operator decides in one workgroup (the plan kernel), as what it decides depends on
// every row and every bit, and does its bulk work, if any, in a second launch over the GPU.
// Both are bound by latency (launch, a chain of a few dependent loads, one scan for every sum)
// until the records that select and compact copy outweigh it.  Measured, plan + bulk kernel:
//   select   64 rows of 2043 tokens, beam step, 4 pools      4.5 + 5.0 us
//            one row of 28597 tokens to 16, 28 pools         4.0 + 4.4 us
//   extend   64 rows by a token 4.2 us; 16 rows by up to 8192 (5000 blocks) 7.6 us
//   compact  4 rows, 1 pool 4.5 + 3.6 us; 974 records of 8 pools, 275 MB 4.8 + 50 us (5.5 TB/s)
#include "hkv_internal.h"

namespace hkv {
namespace {

constexpr int kPlan = 1024;         // threads of a plan kernel, one per row
static_assert(kPlan == HKV_MAX_SEQUENCES, "one thread per row");
constexpr int kThreads = 256;       // of the compacting kernel
constexpr int kColumns = 16;        // table columns per workgroup of the bulk kernels (64-byte runs)
constexpr int64_t kMaxBlocks = 1 << 25;

// Words at the start of the workspace, written by the plan kernels.
enum : int { kOk = 0, kCount = 1, kMaxCols = 2, kLive = 3, kHeader = 16 };

struct Params {
    int32_t* table;
    int32_t* lens;
    int32_t* refs;
    uint32_t* bits;
    uint8_t* const* pools;
    int32_t* err;
    int32_t* ws;
    int S, stride, N, W, run;       // rows, table stride, blocks, bitmap words, words per plan thread
    int L, vecs;                    // pools, 16-byte pieces of a record
    int colwgs;                     // bulk kernels: workgroups of the table's columns
    const int32_t* rows;            // extend: tokens per row; select: source rows
    int32_t all;                    // extend: tokens of every row (rows null)
    int32_t* starts;                // extend
};

// Workspace of select: source rows' old lengths and change of count, each row's new last
// block (-1: the source's), the copies.
__host__ __device__ inline int ws_len(int) { return kHeader; }
__host__ __device__ inline int ws_delta(int S) { return kHeader + S; }
__host__ __device__ inline int ws_tail(int S) { return kHeader + 2 * S; }
__host__ __device__ inline int ws_from(int S) { return kHeader + 3 * S; }
__host__ __device__ inline int ws_to(int S) { return kHeader + 4 * S; }
// Workspace of compact: the held blocks before every run, the
// old bitmap, the blocks that move and where to, by rank.
constexpr int kWsBefore = kHeader, kWsBits = kHeader + kPlan;
__host__ __device__ inline int ws_moved(int W) { return kWsBits + (W + 3) / 4 * 4; }
__host__ __device__ inline int ws_hole(int W, int N) { return ws_moved(W) + (N + 1) / 2; }

__device__ __forceinline__ int blocks_of(int tokens) { return (tokens + kBlockTokens - 1) / kBlockTokens; }

// What the workgroup's kPlan threads tell each other, for one barrier: exclusive sums of two
// numbers with their totals, and the OR of error bits.  sm: kJoin words, for this call alone.
struct Joint {
    int a, b, total_a, total_b, err;
};
constexpr int kWaves = kPlan / 64, kJoin = 3 * kWaves;
__device__ __forceinline__ Joint join(int a, int b, int err, int* sm) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = a, y = b;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int xd = __shfl_up(x, d), yd = __shfl_up(y, d);
        if (lane >= d) {
            x += xd;
            y += yd;
        }
    }
    if (__any(err)) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) err |= __shfl_xor(err, d);
    }
    if (lane == 63) {
        sm[wave] = x;
        sm[kWaves + wave] = y;
        sm[2 * kWaves + wave] = err;
    }
    __syncthreads();
    Joint r = {x - a, y - b, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const int sa = sm[w], sb = sm[kWaves + w];
        r.a += w < wave ? sa : 0;
        r.b += w < wave ? sb : 0;
        r.total_a += sa;
        r.total_b += sb;
        r.err |= sm[2 * kWaves + w];
    }
    return r;
}

// Word w of the bitmap; what a caller may have left behind the last block is not free.
__device__ __forceinline__ uint32_t free_word(const Params& p, int w) {
    const int n = p.N - w * 32;
    return n >= 32 ? p.bits[w] : p.bits[w] & ((1u << n) - 1);
}

// Free blocks in this thread's run of words.
__device__ __forceinline__ int count_run(const Params& p) {
    const int w0 = threadIdx.x * p.run, w1 = min(w0 + p.run, p.W);
    int n = 0;
#pragma unroll 8   // as many loads on their way: 1M blocks 19.7 -> 9.2 us
    for (int w = w0; w < w1; ++w) n += __popc(free_word(p, w));
    return n;
}

// Lists this thread's free blocks (n of them, of ranks from `before`) of ranks [r0, r1): list[rank - r0].
__device__ __forceinline__ void list_free(const Params& p, int before, int n, int r0, int r1, int32_t* list) {
    if (before >= r1 || before + n <= r0) return;
    const int w1 = min((int)(threadIdx.x + 1) * p.run, p.W);
    for (int w = threadIdx.x * p.run; w < w1 && before < r1; ++w)
        for (uint32_t v = free_word(p, w); v != 0 && before < r1; v &= v - 1, ++before)
            if (before >= r0) list[before - r0] = w * 32 + __builtin_ctz(v);
}

// Clears the `taken` lowest free bits; this thread's run starts at rank `before`.
__device__ __forceinline__ void take_lowest(const Params& p, int before, int taken) {
    int left = taken - before;
    const int w1 = min((int)(threadIdx.x + 1) * p.run, p.W);
    for (int w = threadIdx.x * p.run; w < w1 && left > 0; ++w) {
        uint32_t v = free_word(p, w);
        const int n = __popc(v);
        if (left >= n) v = 0u;
        else
            for (int k = 0; k < left; ++k) v &= v - 1;
        p.bits[w] = v;
        left -= n;
    }
}

__device__ __forceinline__ void report(const Params& p, int err) {
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, err);
}

constexpr int kList = 8 * kPlan;   // 32 KB: blocks that extend hands out between two barriers
__global__ __launch_bounds__(kPlan) void blocks_extend_kernel(Params p) {
    touch_kernel_args(p);
    __shared__ int sm[kJoin], off[kPlan], have[kPlan], list[kList];
    const int i = threadIdx.x;
    const bool row = i < p.S;
    const int len = row ? p.lens[i] : 0;
    const int add = row ? (p.rows ? p.rows[i] : p.all) : 0;
    const int cap = p.stride * kBlockTokens;
    const bool bad = len < 0 || len > cap || add < 0, over = !bad && add > cap - len;
    const int need = bad || over ? 0 : blocks_of(len + add) - blocks_of(len);
    const int nfree = count_run(p);
    const Joint all = join(need, nfree, (bad ? HKV_ERR_BIT_SEQUENCE : 0) | (over ? HKV_ERR_BIT_SLOT : 0), sm);
    const int total = all.total_a, before = all.b, err = all.err | (total > all.total_b ? HKV_ERR_BIT_FULL : 0);
    if (row && p.starts) p.starts[i] = len;
    if (err) return report(p, err);
    off[i] = all.a;
    have[i] = blocks_of(len);
    if (row) p.lens[i] = len + add;
    for (int r0 = 0; r0 < total; r0 += kList) {
        const int r1 = min(r0 + kList, total);
        __syncthreads();   // (the list before this one has been read)
        list_free(p, before, nfree, r0, r1, list);
        __syncthreads();
#pragma unroll 2
        for (int r = r0 + i; r < r1; r += kPlan) {
            const int id = list[r - r0];
            int s = 0;   // the last row with off[s] <= r: rows without need end at the next one's
#pragma unroll
            for (int step = kPlan / 2; step > 0; step >>= 1)
                if (off[s + step] <= r) s += step;
            p.table[(int64_t)s * p.stride + have[s] + r - off[s]] = id;
            p.refs[id] = 1;
        }
    }
    take_lowest(p, before, total);
}

__global__ __launch_bounds__(kPlan) void blocks_select_plan_kernel(Params p) {
    touch_kernel_args(p);
    __shared__ int sm[kJoin], sm_cols, len[kPlan], takers[kPlan], first[kPlan], list[kPlan];
    const int i = threadIdx.x;
    const bool row = i < p.S;
    const int l = row ? p.lens[i] : 0, s = row ? p.rows[i] : -1;
    const bool bad = l < 0 || l > p.stride * kBlockTokens || s < -1 || s >= p.S;
    len[i] = bad ? 0 : l;
    takers[i] = 0;
    first[i] = kPlan;
    if (i == 0) sm_cols = 0;
    const int nfree = count_run(p);
    __syncthreads();
    if (!bad && s >= 0) {
        atomicAdd(&takers[s], 1);
        atomicMin(&first[s], i);
    }
    if (!bad && l > 0) atomicMax(&sm_cols, blocks_of(l));
    __syncthreads();
    const bool copies = !bad && s >= 0 && first[s] != i && len[s] % kBlockTokens != 0;
    const int from = copies ? p.table[(int64_t)s * p.stride + len[s] / kBlockTokens] : 0;
    const Joint all = join(copies ? 1 : 0, nfree,
                           (bad ? HKV_ERR_BIT_SEQUENCE : 0) | (from < 0 || from >= p.N ? HKV_ERR_BIT_BLOCK_ID : 0), sm);
    const int at = all.a, before = all.b, total = all.total_a;
    const int err = all.err | (total > all.total_b ? HKV_ERR_BIT_FULL : 0);
    if (i == 0) {
        p.ws[kOk] = err == 0;
        p.ws[kCount] = total;
        p.ws[kMaxCols] = sm_cols;
    }
    if (err) return report(p, err);
    if (total > 0) {
        list_free(p, before, nfree, 0, total, list);
        take_lowest(p, before, total);
        __syncthreads();
    }
    if (row) {
        int to = -1;
        if (copies) {
            to = list[at];
            p.refs[to] = 1;
            p.ws[ws_from(p.S) + at] = from;
            p.ws[ws_to(p.S) + at] = to;
        }
        p.ws[ws_len(p.S) + i] = l;
        p.ws[ws_delta(p.S) + i] = takers[i] - 1;
        p.ws[ws_tail(p.S) + i] = to;
        p.lens[i] = s >= 0 ? len[s] : 0;
    }
}

// One record, 16 bytes per thread and load, the whole of it (up to 32 KB with 256 threads) on its
// way before the first store: one round trip a record.  Past the caches (nontemporal), where
// nobody reads it again soon: a compaction of 275 MB takes 50 us so, 78 us through them.
template <int kT>
__device__ __forceinline__ void copy_record(const Params& p, uint8_t* pool, int from, int to) {
    typedef uint32_t Piece __attribute__((ext_vector_type(4)));
    const Piece* src = (const Piece*)pool + (int64_t)from * p.vecs;
    Piece* dst = (Piece*)pool + (int64_t)to * p.vecs;
    for (int o = threadIdx.x; o < p.vecs; o += 8 * kT) {
        Piece v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (o + k * kT < p.vecs) v[k] = __builtin_nontemporal_load(src + o + k * kT);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (o + k * kT < p.vecs) __builtin_nontemporal_store(v[k], dst + o + k * kT);
    }
}

// Sets bit `id` of the bitmap for the lanes that `give` it, all 16 of a row's columns taking part.
// Neighbours' ids are mostly neighbours: the first lane of those that share a word sets their
// bits at once, where 16 atomics would queue at the word.
__device__ __forceinline__ void free_blocks(const Params& p, int id, bool give) {
    const int word = id >> 5;
    uint32_t v = give ? 1u << (id & 31) : 0u;
#pragma unroll
    for (int d = 1; d < kColumns; d <<= 1) {
        const int other = __shfl_down(word, d, kColumns);
        const uint32_t theirs = __shfl_down(v, d, kColumns);
        if ((int)(threadIdx.x & (kColumns - 1)) + d < kColumns && other == word) v |= theirs;
    }
    const int before = __shfl_up(word, 1, kColumns);
    if (v != 0 && ((threadIdx.x & (kColumns - 1)) == 0 || before != word)) atomicOr(&p.bits[word], v);
}

// Workgroups [0, colwgs): kColumns columns of every row each, so that a column's old entries
// are all in LDS before the first new one is written, and the table changes in place.  The
// others copy records, one per workgroup and step.  64 rows are one pass of a workgroup: what a
// pass waits for (its loads, the counts' old values) is waited for once.
constexpr int kSelect = 1024;
__global__ __launch_bounds__(kSelect) void blocks_select_kernel(Params p) {
    touch_kernel_args(p);
    extern __shared__ int tile[];   // [S][kColumns], then [S] each: source, old length, change of count, new tail
    if ((int)blockIdx.x >= p.colwgs) {
        const int n = p.ws[kOk] ? p.ws[kCount] * p.L : 0;
        for (int u = (int)blockIdx.x - p.colwgs; u < n; u += (int)gridDim.x - p.colwgs) {
            const int k = u / p.L;
            copy_record<kSelect>(p, p.pools[u - k * p.L], p.ws[ws_from(p.S) + k], p.ws[ws_to(p.S) + k]);
        }
        return;
    }
    const int tc = threadIdx.x & (kColumns - 1), c0 = (int)blockIdx.x * kColumns, col = c0 + tc, r0 = threadIdx.x / kColumns;
    constexpr int kRows = kSelect / kColumns;
    int *source = tile + p.S * kColumns, *len = source + p.S, *delta = len + p.S, *tail = delta + p.S;
    const int ok = p.ws[kOk], cols = p.ws[kMaxCols];
    if ((int)threadIdx.x < p.S) {   // S <= kSelect
        source[threadIdx.x] = p.rows[threadIdx.x];
        len[threadIdx.x] = p.ws[ws_len(p.S) + threadIdx.x];
        delta[threadIdx.x] = p.ws[ws_delta(p.S) + threadIdx.x];
        tail[threadIdx.x] = p.ws[ws_tail(p.S) + threadIdx.x];
    }
    const bool in = col < p.stride;
    for (int i = r0; i < p.S; i += kRows) tile[i * kColumns + tc] = in ? p.table[(int64_t)i * p.stride + col] : -1;
    if (!ok || c0 >= cols) return;   // (the words behind ok are not set then, and nothing was stored)
    __syncthreads();
    bool bad = false;
    for (int i = r0; i < p.S; i += kRows) {
        // the block that row i held: as many holders more as rows take row i, less itself; of a
        // partial one no more than one
        const int mine = tile[i * kColumns + tc], l = len[i];
        const int d = col < l / kBlockTokens ? delta[i] : col < blocks_of(l) ? min(delta[i], 0) : 0;
        const bool in_pool = mine >= 0 && mine < p.N;
        int held = 0;
        if (d != 0 && in_pool) held = atomicAdd(&p.refs[mine], d) + d;
        const int s = source[i];
        int now = -1;
        if (s >= 0 && col < blocks_of(len[s])) now = tail[i] >= 0 && col == len[s] / kBlockTokens ? tail[i] : tile[s * kColumns + tc];
        if (now != mine) p.table[(int64_t)i * p.stride + col] = now;
        if (d != 0 && !in_pool) bad = true;
        free_blocks(p, mine, d != 0 && in_pool && held == 0);   // no order of the additions gives 0 before the last
    }
    if (bad && p.err) atomicOr(p.err, HKV_ERR_BIT_BLOCK_ID);
}

__global__ __launch_bounds__(kPlan) void blocks_compact_plan_kernel(Params p) {
    touch_kernel_args(p);
    __shared__ int sm[kJoin], sm_cols, sm_moves;
    const int i = threadIdx.x;
    const bool row = i < p.S;
    const int l = row ? p.lens[i] : 0;
    const bool bad = l < 0 || l > p.stride * kBlockTokens;
    if (i == 0) sm_cols = sm_moves = 0;   // (no word holds block `live` where no block is free)
    const int nfree = count_run(p);
    const Joint all = join(nfree, 0, bad ? HKV_ERR_BIT_SEQUENCE : 0, sm);
    const int before = all.a, live = p.N - all.total_a, err = all.err;
    if (!bad && l > 0) atomicMax(&sm_cols, blocks_of(l));
    // the free blocks below `live`: counted by the thread whose run holds its word
    const int lw = live >> 5;
    if (lw < p.W && lw / p.run == i) {
        int n = before;
        for (int w = i * p.run; w < lw; ++w) n += __popc(free_word(p, w));
        sm_moves = n + __popc(free_word(p, lw) & ((1u << (live & 31)) - 1));
    }
    __syncthreads();
    const int moves = sm_moves;
    if (i == 0) {
        p.ws[kOk] = err == 0;
        p.ws[kCount] = moves;
        p.ws[kMaxCols] = sm_cols;
        p.ws[kLive] = live;
    }
    if (err) return report(p, err);
    if (moves == 0) return;
    // The bitmap as it was, the held blocks before every run, and the blocks that move, by rank:
    // holes below `live`, held blocks at or above it.
    int hole = before, held = (i * p.run < p.W ? i * p.run * 32 : p.W * 32) - before, moved = held - (live - moves);
    p.ws[kWsBefore + i] = held;
    const int w1 = min((i + 1) * p.run, p.W);
    for (int w = i * p.run; w < w1; ++w) {
        const uint32_t v = free_word(p, w);
        p.ws[kWsBits + w] = (int)v;
        const int lo = live - w * 32, hi = p.N - w * 32;   // bits [lo, hi) of the word are free now
        const uint32_t below = lo <= 0 ? 0u : lo >= 32 ? ~0u : (1u << lo) - 1;
        const uint32_t valid = hi >= 32 ? ~0u : (1u << hi) - 1;
        p.bits[w] = valid & ~below;
        for (uint32_t f = v & below; f != 0; f &= f - 1) p.ws[ws_hole(p.W, p.N) + hole++] = w * 32 + __builtin_ctz(f);
        moved += __popc(~v & below);
        for (uint32_t m = ~v & valid & ~below; m != 0; m &= m - 1) p.ws[ws_moved(p.W) + moved++] = w * 32 + __builtin_ctz(m);
    }
}

// The free blocks of rank k below `live` take the held ones of rank k at or above it.  Nothing
// is both read and written: sources lie at or above `live`, destinations below.
__global__ __launch_bounds__(kThreads) void blocks_compact_kernel(Params p) {
    touch_kernel_args(p);
    const int4 head = *(const int4*)p.ws;   // kOk, kCount, kMaxCols, kLive
    const int moves = head.y, live = head.w;
    if (!head.x || moves == 0) return;
    const int32_t *from = p.ws + ws_moved(p.W), *to = p.ws + ws_hole(p.W, p.N);
    if ((int)blockIdx.x >= p.colwgs) {
        const int n = moves * p.L;
        for (int u = (int)blockIdx.x - p.colwgs; u < n; u += (int)gridDim.x - p.colwgs) {
            const int k = u / p.L, layer = u - k * p.L, a = from[k], b = to[k];
            if (layer == 0 && threadIdx.x == 0) {
                p.refs[b] = p.refs[a];
                p.refs[a] = 0;
            }
            copy_record<kThreads>(p, p.pools[layer], a, b);
        }
        return;
    }
    if ((int)blockIdx.x * kColumns >= head.z) return;
    const int col = blockIdx.x * kColumns + (threadIdx.x & (kColumns - 1));
    const uint32_t* bits = (const uint32_t*)p.ws + kWsBits;   // as they were
    bool bad = false;
    for (int i = threadIdx.x / kColumns; i < p.S; i += kThreads / kColumns) {
        if (col >= blocks_of(p.lens[i])) continue;
        const int id = p.table[(int64_t)i * p.stride + col];
        if (id < live && id >= 0) continue;
        if (id < 0 || id >= p.N || (bits[id >> 5] >> (id & 31) & 1u)) {   // outside, or a block that is not held
            bad = true;
            continue;
        }
        // the rank of id among the held blocks, less those that stay
        int w = (id >> 5) / p.run * p.run, k = p.ws[kWsBefore + (id >> 5) / p.run] - (live - moves);
        for (; w < id >> 5; ++w) k += __popc(~bits[w]);
        k += __popc(~bits[w] & ((1u << (id & 31)) - 1));
        p.table[(int64_t)i * p.stride + col] = to[k];
    }
    if (bad && p.err) atomicOr(p.err, HKV_ERR_BIT_BLOCK_ID);
}

int check(const HkvBlockTables* t, const char* name, Params& p) {
    HKV_REQUIRE(t != nullptr, HKV_ERR_ARG, "%s: null args", name);
    HKV_REQUIRE(t->head_dim == kHeadDim, HKV_ERR_UNSUPPORTED, "%s: head_dim %d != 128", name, t->head_dim);
    HKV_REQUIRE(t->num_sequences > 0 && t->num_sequences <= HKV_MAX_SEQUENCES, HKV_ERR_ARG,
                "%s: num_sequences %d outside [1, %d]", name, t->num_sequences, HKV_MAX_SEQUENCES);
    HKV_REQUIRE(t->num_blocks > 0 && t->num_blocks <= kMaxBlocks, HKV_ERR_ARG, "%s: num_blocks %lld outside [1, %lld]",
                name, (long long)t->num_blocks, (long long)kMaxBlocks);
    HKV_REQUIRE(t->table_stride > 0 && t->table_stride <= (1 << 26) && t->num_kv_heads > 0 && t->num_kv_heads <= 4096 &&
                    t->num_pools > 0 && t->num_pools <= 4096,
                HKV_ERR_ARG, "%s: bad table stride %d, kv heads %d or pools %d", name, t->table_stride, t->num_kv_heads,
                t->num_pools);
    HKV_REQUIRE((int64_t)t->num_sequences * t->table_stride <= INT32_MAX, HKV_ERR_ARG,
                "%s: a table of %d x %d entries (2^31 - 1 at most)", name, t->num_sequences, t->table_stride);
    HKV_REQUIRE(t->table && t->lens && t->refs && t->free_bits && t->pools && t->workspace, HKV_ERR_ARG, "%s: null pointer",
                name);
    HKV_REQUIRE((((uintptr_t)t->workspace) & 15) == 0, HKV_ERR_ARG, "%s: workspace must be 16-byte aligned", name);
    const size_t need = hkv_blocks_workspace_bytes(t->num_sequences, t->num_blocks);
    HKV_REQUIRE(t->workspace_bytes >= need, HKV_ERR_CAPACITY, "%s: workspace %zu bytes, need %zu", name, t->workspace_bytes,
                need);
    p = {};
    p.table = t->table;
    p.lens = t->lens;
    p.refs = t->refs;
    p.bits = t->free_bits;
    p.pools = t->pools;
    p.err = t->err_flag;
    p.ws = (int32_t*)t->workspace;
    p.S = t->num_sequences;
    p.stride = t->table_stride;
    p.N = (int)t->num_blocks;
    p.W = (p.N + 31) / 32;
    p.run = (p.W + kPlan - 1) / kPlan;
    p.L = t->num_pools;
    p.vecs = t->num_kv_heads * (kHeadPartBytes / 16);
    // a row holds num_blocks blocks at most, its further columns are never in use
    p.colwgs = ((p.stride < p.N ? p.stride : p.N) + kColumns - 1) / kColumns;
    return HKV_OK;
}

}  // namespace
}  // namespace hkv

using namespace hkv;

extern "C" size_t hkv_blocks_workspace_bytes(int32_t num_sequences, int64_t num_blocks) {
    if (num_sequences <= 0 || num_blocks <= 0 || num_blocks > kMaxBlocks) return 0;
    const size_t select = kHeader + 5 * (size_t)num_sequences, W = (size_t)(num_blocks + 31) / 32;
    const size_t compact = (size_t)ws_hole((int)W, (int)num_blocks) + (size_t)(num_blocks + 1) / 2;
    return ((select > compact ? select : compact) * sizeof(int32_t) + 255) / 256 * 256;
}

extern "C" int hkv_blocks_extend(const HkvBlockTables* t, const int32_t* tokens, int32_t tokens_all, int32_t* starts,
                                 void* stream) {
    clear_error();
    Params p;
    const int rc = check(t, "hkv_blocks_extend", p);
    if (rc != HKV_OK) return rc;
    HKV_REQUIRE(tokens || tokens_all >= 0, HKV_ERR_ARG, "hkv_blocks_extend: %d tokens", tokens_all);
    p.rows = tokens;
    p.all = tokens_all;
    p.starts = starts;
    hipLaunchKernelGGL(blocks_extend_kernel, dim3(1), dim3(kPlan), 0, (hipStream_t)stream, p);
    HKV_LAUNCH_CHECK("blocks_extend_kernel");
    return HKV_OK;
}

extern "C" int hkv_blocks_select(const HkvBlockTables* t, const int32_t* source, void* stream) {
    clear_error();
    Params p;
    const int rc = check(t, "hkv_blocks_select", p);
    if (rc != HKV_OK) return rc;
    HKV_REQUIRE(source != nullptr, HKV_ERR_ARG, "hkv_blocks_select: null source");
    p.rows = source;
    hipLaunchKernelGGL(blocks_select_plan_kernel, dim3(1), dim3(kPlan), 0, (hipStream_t)stream, p);
    HKV_LAUNCH_CHECK("blocks_select_plan_kernel");
    const int64_t copies = (int64_t)(p.S - 1) * p.L;   // at most
    const unsigned grid = (unsigned)(p.colwgs + (copies < 2048 ? copies : 2048));
    static std::atomic<uint64_t> raised;
    HKV_RAISE_LDS(blocks_select_kernel, kSelect * (kColumns + 4) * (int)sizeof(int), raised);
    hipLaunchKernelGGL(blocks_select_kernel, dim3(grid), dim3(kSelect), (size_t)p.S * (kColumns + 4) * sizeof(int),
                       (hipStream_t)stream, p);
    HKV_LAUNCH_CHECK("blocks_select_kernel");
    return HKV_OK;
}

extern "C" int hkv_blocks_compact(const HkvBlockTables* t, void* stream) {
    clear_error();
    Params p;
    const int rc = check(t, "hkv_blocks_compact", p);
    if (rc != HKV_OK) return rc;
    hipLaunchKernelGGL(blocks_compact_plan_kernel, dim3(1), dim3(kPlan), 0, (hipStream_t)stream, p);
    HKV_LAUNCH_CHECK("blocks_compact_plan_kernel");
    const int64_t copies = (int64_t)(p.N + 1) / 2 * p.L;   // at most
    const unsigned grid = (unsigned)(p.colwgs + (copies < 16384 ? copies : 16384));
    hipLaunchKernelGGL(blocks_compact_kernel, dim3(grid), dim3(kThreads), 0, (hipStream_t)stream, p);
    HKV_LAUNCH_CHECK("blocks_compact_kernel");
    return HKV_OK;
}
