// Decode attention for sequences that share a prefix, the prefix attended once per group.
//
// Math.  out = softmax(q K^T * sm_scale) V over the tokens of the shared prefix, of the
// sequence's own INT4 blocks and of its fp16 zones, as hkv_decode_attn's.  A softmax over a set
// of tokens merges from softmaxes over its parts, each with its maximum m, its sum l of
// 2^(s - m) and its o = sum of 2^(s - m) v:  M = max m_i, L = sum l_i 2^(m_i - M), O alike.  So
// the prefix is one problem of R = group x n_rep query rows per kv head that reads each record
// once, and the rest is a problem of n_rep rows per sequence.
//
// Bound.  A prefix token is 138 bytes and 512 R operations per kv head.  At the copy rate
// (5.13 TB/s) and the rate of a large matrix product (1216 TFLOP/s) these are equal at R = 64:
// few rows are bound by HBM, many by the matrix cores and, beside them, by the softmax's VALU
// work and the nibble decode, whose times mostly add to the products' (a third of the matrix
// cores' cycles lie beside VALU work).
//
// Work.  One launch: workgroups for ranges of the prefix and for the sequences' own tokens, every
// range leaving its state (o[128], m, l) in the workspace.  A sequence need not hold all of the prefix
// (its length or its group's count is short of it): its own blocks in there, "strays", are
// attended by the workgroups of the prefix, all of them, behind what they do for the group.  Few
// states are merged by whoever stores the last one of a (sequence, kv head) (kJoin), many by a
// second launch.  A wave streams its own run of block pairs, decodes a pair once into MFMA operands and multiplies it
// with NT tiles of 16 query rows, NT = 1 .. 4: the decode (~150 of ~400 VALU instructions at NT =
// 4) is paid once for them (a workgroup of more rows holds no more accumulators: 32 registers a
// tile); q lies in LDS.  With more than 64 rows several workgroups read a range, next to each
// other on one XCD, so that its L2 serves all but the first.
//
// Measured (both launches, us; floor: the larger of bytes and operations at the rates above):
//   samples x heads        shared tokens     us    floor
//         2 x 32/8                  1024   11.4      0.4   latency: ids, records, merges
//        16 x 32/8                 28608     29      9.2   7 to the first step, 4.4 for it and its loads, 2.6
//         8 x 28/4                126912     39       15     a further one (two waves a SIMD), 6 to merge
//                                                          eight waves, the last of them 2 behind; launch
//    6 x 10 x 24/8                  6000     32       16     + 4 to merge ranges
//       256 x 32/8                 16384    121       57   105 without own tokens (657 TFLOP/s), then
//                                                          those, 89 MB
// Tried and not kept: codes staged through LDS with wide loads; K operands of the next step decoded
// beside the products of this one (spills); 256 rows a workgroup, all waves sharing tiles that are
// decoded once into LDS: 8% fewer us in the prefix, all of which its four times as many states cost.
#include "hkv_internal.h"
#include "kv_tiles.h"

namespace hkv {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * 64;
constexpr int kMaxTiles = 4;                   // row tiles of 16 per workgroup
constexpr int kState = kHeadDim + 4;           // floats of a state: o[128], m, l, 2 pad (16-byte rows)
constexpr int kWindow = 64;                    // block ids a wave holds, one per lane
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kXcc = 8;                        // XCDs that workgroups go to round-robin
constexpr int kMaxRanges = 64;                 // of the prefix, and of a sequence's own tokens
constexpr int kFewStates = 12;                 // a row's states that one wave merges
constexpr int kJoinFew = 8;                    // a row's states that a thread merges without a second launch
constexpr int kDeviceScope = 16;               // cache policy of accesses that another XCD's see (sc1)

struct ZoneP {
    const uint16_t* k;
    const uint16_t* v;
    int cap;
    int max_len;
    const int32_t* lens;
};

struct Params {
    int B, Hkv, nrep, group;
    float scale_log2;
    int q_bf16, out_bf16;
    const uint16_t* q;
    int64_t q_sb, q_sh;
    int nz;
    ZoneP z[HKV_MAX_F16_ZONES];
    const uint8_t* pool;
    int64_t pool_blocks;
    const uint8_t* staging;
    int64_t staging_blocks;
    int fallback_id;
    const int32_t* bt;
    int bt_stride;
    const int32_t* int4_lens;
    int int4_max_len;
    uint16_t* out;
    int64_t o_sb, o_sh;
    int* err;
    float* states;              // [prefix ranges + own ranges + strays][B * Hq][kState]
    int* arrivals;              // [B][Hkv], with kJoin: states stored, zero again at the end
    const int32_t* counts;      // shared blocks of each group (null: shared_blocks)
    int shared_blocks;
    int row_tiles;              // workgroups of rows per prefix range
    int prefix_ranges, own_ranges;
    int strays;                 // states of a sequence's strays: as many as prefix ranges, or there can be none
    int own_waves;              // waves per own range: 1, or a workgroup's
    int prefix_wgs, own_wgs;
    int own_first;              // the order of these two kinds of workgroups: the longer ones first
};

__device__ __forceinline__ int row_len(const Params& p, int b) {
    return p.int4_lens ? min(max(load_uniform_i32(p.int4_lens, b), 0), p.int4_max_len) : p.int4_max_len;
}
// Shared blocks of a group.  A sequence shorter than these has no part in them.
__device__ __forceinline__ int shared_count(const Params& p, int group) {
    const int n = p.counts ? min(max(load_uniform_i32(p.counts, group), 0), p.shared_blocks) : p.shared_blocks;
    return min(n, p.int4_max_len / kBlockTokens);
}

// What a sequence of `len` tokens has of the first shared_blocks blocks beside its group's `count`
// shared ones: blocks [from, to).
struct Strays {
    int from, to;
    __device__ __forceinline__ Strays(const Params& p, int len, int count)
        : from(len >= count * kBlockTokens ? count : 0), to(min((len + kBlockTokens - 1) / kBlockTokens, p.shared_blocks)) {}
    __device__ __forceinline__ bool any() const { return from < to; }
};

// Row c's query values as an MFMA operand takes them: dims 32g + 8j .. +7 (at: dim 32g), zeros
// without a row.
__device__ __forceinline__ void load_query(const uint16_t* at, bool has, u4 (&w)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = has ? *(const u4*)(at + 8 * j) : u4{0u, 0u, 0u, 0u};
}
// bf16 values to fp16; a finite one that leaves its range is reported.
__device__ __forceinline__ void query_to_f16(const Params& p, u4 (&w)[4]) {
    if (!p.q_bf16) return;
    bool over = false;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float lo = __uint_as_float(w[j][e] << 16), hi = __uint_as_float(w[j][e] & 0xffff0000u);
            const uint32_t a = f2h_rn(lo), b = f2h_rn(hi);
            over |= (((a & 0x7fffu) == 0x7c00u) && fabsf(lo) < INFINITY) || (((b & 0x7fffu) == 0x7c00u) && fabsf(hi) < INFINITY);
            w[j][e] = a | (b << 16);
        }
    if (__ballot(over) && (threadIdx.x & 63) == 0 && p.err) atomicOr(p.err, HKV_ERR_BIT_RANGE);
}

// The largest value of the four lanes (c, 0 .. 3).
__device__ __forceinline__ float row_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Online softmax of NT row tiles.  m is a reference, and the scores relative to it, x = s - m, are at
// most `lim`.  What limits them is fp16: P = 2^x times a token's V scale goes into the products as
// fp16, so lim + log2 of the largest V scale (or a little more) is kTopP.  Thus P uses fp16's upper end
// whatever the size of V, and the likeliest token of V scales within a factor of 4 has 21 bits above the
// subnormals (with 2^x <= 1, V of some 2^-8 would have none).  When a score passes lim, m rises
// until it is kHeadroom below, and the scores a little larger that follow need no new reference and no
// pass over the accumulators.  `fresh`: a row may have had no score yet, or only -inf, and its m has to
// go by the first one whatever it is.  One branch for all tiles: with a branch for each, no product
// of one tile could run beside another's exponentials.
constexpr float kHeadroom = 4.0f;
constexpr int kTopP = 15;
struct Range {
    float lim = kTopP;
    float largest = 0.f;   // V scale that lim allows
};
template <int NT, int N>
__device__ __forceinline__ void raise_reference(bool& fresh, float lim, float (&x)[NT][N], f4 (&acc)[NT][8], float (&m)[NT],
                                                float (&l)[NT]) {
    float top[NT];
    bool any = fresh;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        top[nt] = x[nt][0];
#pragma unroll
        for (int i = 1; i < N; ++i) top[nt] = fmaxf(top[nt], x[nt][i]);
        any |= top[nt] > lim;
    }
    if (__ballot(any)) {
        bool waits = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float t = row_max(top[nt]);
            const bool first = fresh && row_max(l[nt]) == 0.f;
            waits |= first && t == -INFINITY;
            const float up = (first ? t > -INFINITY : t > lim) ? t - (lim - kHeadroom) : 0.f;
            if (__ballot(up != 0.f) == 0) continue;
            const float a = first ? 1.0f : fast_exp2(-up);
#pragma unroll
            for (int i = 0; i < N; ++i) x[nt][i] -= up;
#pragma unroll
            for (int n = 0; n < 8; ++n) acc[nt][n] *= a;
            l[nt] *= a;
            m[nt] += up;
        }
        fresh = fresh && __ballot(waits) != 0;
    }
}
// Another limit (uniform), and the references for it.
template <int NT>
__device__ __forceinline__ float set_limit(Range& range, float lim, f4 (&acc)[NT][8], float (&m)[NT], float (&l)[NT]) {
    const float up = range.lim - lim, a = fast_exp2(-up);
    range.lim = lim;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int n = 0; n < 8; ++n) acc[nt][n] *= a;
        l[nt] *= a;
        m[nt] += up;
    }
    return up;
}
// The limit for V scales up to `top` (a lane's), and up to twice as large ones, which seldom call for
// another.  Scales of 0 to 2^-47 are alike, and beyond 2^53 P may leave fp16.
template <int NT, int N>
__device__ __forceinline__ void fit_scales(Range& range, float top, float (&x)[NT][N], f4 (&acc)[NT][8], float (&m)[NT],
                                           float (&l)[NT]) {
    const int e = min(max((int)(__builtin_amdgcn_readfirstlane(__float_as_uint(row_max(top))) >> 23) - 127, -47), 53) + 2;
    range.largest = __uint_as_float((uint32_t)(e + 127) << 23);
    const float up = set_limit<NT>(range, (float)(kTopP - e), acc, m, l);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < N; ++i) x[nt][i] -= up;
}
// Probabilities relative to the reference, and their sum.
template <int N>
__device__ __forceinline__ void exponentiate(const float (&x)[N], float& l, float (&pr)[N]) {
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = pr[i] = fast_exp2(x[i]);
#pragma unroll
    for (int w = N / 2; w > 0; w >>= 1)
#pragma unroll
        for (int i = 0; i < w; ++i) sum[i] += sum[i + w];
    l += sum[0];
}

// The K and the V half of a block pair, loaded apart: K of the next pair is on its way while
// this one's softmax runs.
struct Half {
    u4 w;         // codes (Int4Blk::k or v)
    f4 s;         // scales of tokens 4g .. 4g + 3
    uint32_t z;   // zero points (Int4Blk::kz or vz)
};
struct Lane {
    int c, g, kzsh;
};
__device__ __forceinline__ void load_k(__amdgpu_buffer_rsrc_t r, const Lane& ln, Half& d) {
    d.w = ld16(r, kPartKc + ln.c * kCodeRowBytes + ln.g * 16);
    d.s = __builtin_bit_cast(f4, ld16(r, kPartKs + ln.g * 16));
    d.z = ld4(r, kPartKz + (ln.c & ~3));
}
__device__ __forceinline__ void load_v(__amdgpu_buffer_rsrc_t r, const Lane& ln, Half& d) {
    d.w = ld16(r, kPartVc + (ln.g * 16 + ln.c) * 16);
    d.s = __builtin_bit_cast(f4, ld16(r, kPartVs + ln.g * 16));
    d.z = ld4(r, kPartVz + ln.g * 4);
}

// Where a wave finds its blocks: this kv head's parts of up to kWindow of them, one address
// per lane (an address from an id in scalar registers costs eleven instructions, in a row, for
// every block: 2% of the time).
struct Blocks {
    uint32_t lo, hi;
    __device__ __forceinline__ void set(const Params& p, int h, int id) {
        const uint64_t at = (uint64_t)(id >= 0 ? p.pool : p.staging) + (uint32_t)RecordLayout::part(h) +
                            (uint64_t)(uint32_t)(id >= 0 ? id : ~id) * (uint32_t)(p.Hkv * kHeadPartBytes);
        lo = (uint32_t)at;
        hi = (uint32_t)(at >> 32);
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(int i) const {
        const uint64_t a = (uint32_t)__builtin_amdgcn_readlane(lo, i) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i) << 32;
        return rsrc((const void*)a, kHeadPartBytes);
    }
};

// Ids of blocks [b0, b0 + n), n <= kWindow, repeating the last; bad ones are replaced and reported.
__device__ __forceinline__ int request_ids(const int32_t* row, int b0, int n) {
    return row[b0 + min((int)(threadIdx.x & 63), n - 1)];
}
__device__ __forceinline__ int check_ids(const Params& p, int id) {
    const bool bad = id >= 0 ? (int64_t)id >= p.pool_blocks : (int64_t)(~id) >= p.staging_blocks;
    if (__ballot(bad)) {
        if ((threadIdx.x & 63) == 0 && p.err) atomicOr(p.err, HKV_ERR_BIT_BLOCK_ID);
        if (bad) id = p.fallback_id;
    }
    return id;
}

// INT4 blocks [b0, b1) of one sequence against NT row tiles; tokens at or past `len` are masked
// (score -inf, V scale 0), so what their slots hold does not matter.  ids: the first window's,
// requested.  stage() runs once the first loads are on their way, and by every wave: it makes
// the queries ready, q(nt, j) is dims 32g + 8j .. +7 of row c of tile nt.
template <int NT, class Stage, class Q>
__device__ __forceinline__ void attend_int4(const Params& p, const int32_t* row, int ids, int h, int b0, int b1, int len,
                                            const Lane& ln, const Stage& stage, const Q& q, bool& fresh, Range& range,
                                            f4 (&acc)[NT][8], float (&m)[NT], float (&l)[NT]) {
    Blocks bl;
    if (b0 >= b1) stage();
    for (int wb = b0; wb < b1; wb += kWindow) {
        const int n = min(kWindow, b1 - wb), np = (n + 1) >> 1;
        bl.set(p, h, check_ids(p, wb == b0 ? ids : request_ids(row, wb, n)));
        // (past the last block: it again, masked)
        Half kA, kB, vA, vB;
        load_k(bl.at(0), ln, kA);
        load_k(bl.at(min(1, n - 1)), ln, kB);
        load_v(bl.at(0), ln, vA);
        load_v(bl.at(min(1, n - 1)), ln, vB);
        if (wb == b0) {
            __builtin_amdgcn_sched_barrier(0);
            stage();
        }
        for (int i = 0; i < np; ++i) {
            const int lb = wb + 2 * i;
            const bool hasB = 2 * i + 1 < n;
            const int iA = min(2 * i + 2, n - 1), iB = min(2 * i + 3, n - 1);
            // tokens of the blocks; full: no slot to mask
            const int nA = len - lb * kBlockTokens, nB = hasB ? nA - kBlockTokens : 0;
            const bool full = nB >= kBlockTokens;
            // The two waves of a SIMD (w and w + 4) go first in turn, four steps each: the older one
            // would stay ahead, and the other end alone, without anything beside its waits (60
            // sequences of 10 x 3 rows over 6000 tokens 33.8 -> 31.8 us).
            if (NT > 1) {
                if ((i >> 2 ^ __builtin_amdgcn_readfirstlane(threadIdx.x) >> 8) & 1) __builtin_amdgcn_s_setprio(1);
                else __builtin_amdgcn_s_setprio(0);
            }
            // ---- scores: S^T[token][row], log2 domain.  One 32-dim step of all row tiles after
            // another, so that neighbouring products are of different sums, only one step's K
            // operands are decoded at a time, and the next step's queries are on their way.
            float x[NT][8];
            {
                const uint32_t za = __builtin_amdgcn_ubfe(kA.z, ln.kzsh, 8), zb = __builtin_amdgcn_ubfe(kB.z, ln.kzsh, 8);
                const h2 a1024 = zp1024(za, za), a64 = zp64(za, za), b1024 = zp1024(zb, zb), b64 = zp64(zb, zb);
                f4 SA[NT], SB[NT];
                h8 qf[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    SA[nt] = SB[nt] = f4{0.f, 0.f, 0.f, 0.f};
                    qf[nt] = q(nt, 0);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const h8 ka = k_operand(kA.w[j], a1024, a64), kb = k_operand(kB.w[j], b1024, b64);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        SA[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qf[nt], SA[nt], 0, 0, 0);
                        SB[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qf[nt], SB[nt], 0, 0, 0);
                        if (j < 3) qf[nt] = q(nt, j + 1);
                        if (NT > 1) __builtin_amdgcn_sched_barrier(0);
                    }
                }
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float sa = kA.s[v] * p.scale_log2, sb = kB.s[v] * p.scale_log2;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        x[nt][v] = __builtin_fmaf(SA[nt][v], sa, -m[nt]);
                        x[nt][4 + v] = __builtin_fmaf(SB[nt][v], sb, -m[nt]);
                    }
                }
                if (!full) {
                    asm volatile("");   // a branch, not 32 selects in every step
#pragma unroll
                    for (int v = 0; v < 4; ++v)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            x[nt][v] = 4 * ln.g + v < nA ? x[nt][v] : -INFINITY;
                            x[nt][4 + v] = 4 * ln.g + v < nB ? x[nt][4 + v] : -INFINITY;
                        }
                }
            }
            load_k(bl.at(iA), ln, kA);
            load_k(bl.at(iB), ln, kB);
            __builtin_amdgcn_sched_barrier(0);
            raise_reference<NT, 8>(fresh, range.lim, x, acc, m, l);
            // ---- V scales and operands
            float vs[8];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                vs[v] = vA.s[v];
                vs[4 + v] = vB.s[v];
            }
            if (!full) {
                asm volatile("");
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    vs[v] = 4 * ln.g + v < nA ? vs[v] : 0.f;
                    vs[4 + v] = 4 * ln.g + v < nB ? vs[4 + v] : 0.f;
                }
            }
            float scale = 0.f;
#pragma unroll
            for (int v = 0; v < 8; ++v) scale = fmaxf(scale, fabsf(vs[v]));
            if (__ballot(scale > range.largest)) fit_scales<NT, 8>(range, scale, x, acc, m, l);
            h8 V0[4], V1[4];
            {
                const h2 zA01 = zp1024(vA.z & 0xffu, (vA.z >> 8) & 0xffu), zA23 = zp64((vA.z >> 16) & 0xffu, vA.z >> 24);
                const h2 zB01 = zp1024(vB.z & 0xffu, (vB.z >> 8) & 0xffu), zB23 = zp64((vB.z >> 16) & 0xffu, vB.z >> 24);
#pragma unroll
                for (int mm = 0; mm < 4; ++mm) {
                    const NibPairs a = unpack_word(vA.w[mm], zA01, zA23), b = unpack_word(vB.w[mm], zB01, zB23);
                    V0[mm] = h8{a.p0[0], a.p0[1], a.p1[0], a.p1[1], b.p0[0], b.p0[1], b.p1[0], b.p1[1]};
                    V1[mm] = h8{a.p2[0], a.p2[1], a.p3[0], a.p3[1], b.p2[0], b.p2[1], b.p3[0], b.p3[1]};
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            // ---- probabilities, times the V scales, and O^T[dim][row] += V^T P^T, 32 tokens per
            // product: one tile's products beside the next one's exponentials
            h8 P;
#pragma unroll
            for (int nt = 0; nt <= NT; ++nt) {
                h8 Pn;
                if (nt < NT) {
                    float pr[8];
                    exponentiate<8>(x[nt], l[nt], pr);
                    asm volatile("" : "+v"(l[nt]));   // summed here, not behind the loads with 32 registers held for it
#pragma unroll
                    for (int v = 0; v < 8; ++v) Pn[v] = (_Float16)(pr[v] * vs[v]);
                }
                if (nt > 0) {
#pragma unroll
                    for (int mm = 0; mm < 4; ++mm) {
                        acc[nt - 1][2 * mm] = __builtin_amdgcn_mfma_f32_16x16x32_f16(V0[mm], P, acc[nt - 1][2 * mm], 0, 0, 0);
                        acc[nt - 1][2 * mm + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(V1[mm], P, acc[nt - 1][2 * mm + 1], 0, 0, 0);
                    }
                    if (nt < NT) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // an MFMA
                            __builtin_amdgcn_sched_group_barrier(0x402, 5, 0);   // and up to five VALU or exponentials
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                P = Pn;
            }
            load_v(bl.at(iA), ln, vA);
            load_v(bl.at(iB), ln, vB);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// fp16 tiles [t0, t1), counted over the zones, of sequence b.  There is no V scale in their P.
__device__ __forceinline__ void attend_f16(const Params& p, int b, int h, const int (&lens)[HKV_MAX_F16_ZONES], int t0, int t1,
                                           const Lane& ln, const h8 (&qf)[4], bool& fresh, Range& range, f4 (&acc)[1][8],
                                           float (&m)[1], float (&l)[1]) {
    if (range.lim != kTopP) set_limit<1>(range, kTopP, acc, m, l);
    const int64_t bh = (int64_t)b * p.Hkv + h;
    F16Tile buf[2];   // two tiles on their way
    int valid[2];
    const auto load = [&](int t, F16Tile& d, int& n) {
        int zi = 0, tile = t;
#pragma unroll
        for (int i = 0; i < HKV_MAX_F16_ZONES - 1; ++i) {
            const int k = (lens[i] + kBlockTokens - 1) / kBlockTokens;
            if (zi == i && tile >= k) {
                tile -= k;
                zi = i + 1;
            }
        }
        const ZoneP z = zi == 0 ? p.z[0] : zi == 1 ? p.z[1] : p.z[2];
        const int len = zi == 0 ? lens[0] : zi == 1 ? lens[1] : lens[2];
        const bool in = t < t1;
        n = in ? min(kBlockTokens, len - tile * kBlockTokens) : 0;
        const uint16_t* k = z.k + (bh * z.cap + (int64_t)tile * kBlockTokens) * kHeadDim;
        const uint16_t* v = z.v + (bh * (z.cap / kBlockTokens) + tile) * (kBlockTokens * kHeadDim);
        load_tile(rsrc(in ? k : z.k, in ? kTileBytes : 0), rsrc(in ? v : z.v, in ? kTileBytes : 0), ln.c, ln.g, d);
        __builtin_amdgcn_sched_barrier(0);
    };
    load(t0, buf[0], valid[0]);
    load(t0 + 1, buf[1], valid[1]);
    // rounds of two tiles; an empty second one has no valid token and adds nothing
    for (int t = t0; t < t1; t += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            F16Tile& d = buf[u];
            const int n = valid[u], g4 = 4 * ln.g;
            f4 S = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 4; ++j) S = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, d.k[j]), qf[j], S, 0, 0, 0);
            float x[1][4], pr[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) x[0][v] = g4 + v < n ? __builtin_fmaf(S[v], p.scale_log2, -m[0]) : -INFINITY;
            raise_reference<1, 4>(fresh, kTopP, x, acc, m, l);
            exponentiate<4>(x[0], l[0], pr);
            h4 P;
#pragma unroll
            for (int v = 0; v < 4; ++v) P[v] = (_Float16)pr[v];
            if (n < kBlockTokens) {
                // slots past the zone's length may hold anything: 0 times a NaN is not 0
                const uint32_t m01 = (g4 < n ? 0xFFFFu : 0u) | (g4 + 1 < n ? 0xFFFF0000u : 0u);
                const uint32_t m23 = (g4 + 2 < n ? 0xFFFFu : 0u) | (g4 + 3 < n ? 0xFFFF0000u : 0u);
#pragma unroll
                for (int j = 0; j < 4; ++j) d.v[j] &= u4{m01, m23, m01, m23};
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[0][2 * j] = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4, u2{d.v[j].x, d.v[j].y}), P, acc[0][2 * j], 0, 0, 0);
                acc[0][2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4, u2{d.v[j].z, d.v[j].w}), P, acc[0][2 * j + 1], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            load(t + 2 + u, d, valid[u]);
        }
    }
}

// The merge of the workgroup's eight states of one row tile through LDS: every wave puts its own,
// and behind a barrier every thread gets four dims of a row, and stores the rows that row(i),
// i < 16, maps to an output row (or -1).
constexpr int kMergeFloats = kWaves * 16 * kState;
__device__ __forceinline__ void merge_put(float* sm, int wave, const Lane& ln, const f4 (&acc)[8], float m, float l) {
    float* mine = sm + (wave * 16 + ln.c) * kState;
#pragma unroll
    for (int n = 0; n < 8; ++n) *(f4*)(mine + 16 * n + 4 * ln.g) = acc[n];
    l = row_sum(l);
    if (ln.g == 0) {
        mine[kHeadDim] = l == 0.f ? -INFINITY : m;   // no token: no reference
        mine[kHeadDim + 1] = l;
    }
}
// Stores a piece of a state that lies `at` floats behind `states` (uniform).  kJoin: past this
// XCD's L2, where another XCD's workgroup finds it.
template <bool kJoin, class V>
__device__ __forceinline__ void put_state(float* states, int64_t at, V v) {
    if constexpr (kJoin) {
        const auto r = rsrc(states, -1);
        if constexpr (sizeof(V) == 16) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), r, (int)((uint32_t)at * 4u), 0, kDeviceScope);
        else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, v), r, (int)((uint32_t)at * 4u), 0, kDeviceScope);
    } else {
        *(V*)(states + at) = v;
    }
}

template <bool kJoin, class Row>
__device__ __forceinline__ void merge_get(const float* sm, float* states, const Row& row) {
    const int i = threadIdx.x >> 5, d = (threadIdx.x & 31) * 4;   // 16 rows x 32 pieces of 4 dims
    static_assert(kThreads == 16 * 32, "one output piece per thread");
    const int to = row(i);
    if (to < 0) return;
    f2 ml[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) ml[w] = *(const f2*)(sm + (w * 16 + i) * kState + kHeadDim);
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, ml[w].x);
    f4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const float e = ml[w].x == -INFINITY ? 0.f : fast_exp2(ml[w].x - M);
        O += *(const f4*)(sm + (w * 16 + i) * kState + d) * e;
        L += ml[w].y * e;
    }
    put_state<kJoin>(states, (int64_t)to * kState + d, O);
    if (d == 0) put_state<kJoin>(states, (int64_t)to * kState + kHeadDim, f2{M, L});
}

// ---- the merge without a second launch
// The sums of shared_combine_kernel<1>, in its order, for pieces of rows: a thread merges dims d ..
// d + 3 of kRows rows (row[i] < 0: none; seq[i]: its sequence; states before first[i] have no part
// in it, those of its strays if stray[i]), whose states' loads are all on their way at once.
struct Sums {
    float m, l;
    f4 o;
};
__device__ __forceinline__ Sums add_sums(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m), wa = a.m == -INFINITY ? 0.f : fast_exp2(a.m - m), wb = b.m == -INFINITY ? 0.f : fast_exp2(b.m - m);
    Sums r = {m, __builtin_fmaf(b.l, wb, a.l * wa), {}};
#pragma unroll
    for (int v = 0; v < 4; ++v) r.o[v] = __builtin_fmaf(b.o[v], wb, a.o[v] * wa);
    return r;
}
template <int kRows>
__device__ __forceinline__ void join_states(const Params& p, int from, int n, const int (&row)[kRows], const int (&first)[kRows],
                                            int d, Sums (&sums)[kRows]) {
    const int Hq = p.Hkv * p.nrep;
    f4 o[kRows][kJoinFew];
    f2 ml[kRows][kJoinFew];
#pragma unroll
    for (int k = 0; k < kJoinFew; ++k)
        if (k < n) {
            const auto r = rsrc(p.states + (int64_t)(from + k) * p.B * Hq * kState, -1);
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const uint32_t at = (uint32_t)max(row[i], 0) * (kState * 4u);
                o[i][k] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(at + d * 4u), 0, kDeviceScope));
                ml[i][k] = __builtin_bit_cast(f2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)(at + kHeadDim * 4u), 0, kDeviceScope));
            }
        }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        float M = -INFINITY, e[8] = {};
        f4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kJoinFew; ++k)
            if (k < n && k >= first[i]) M = fmaxf(M, ml[i][k].x);
#pragma unroll
        for (int k = 0; k < kJoinFew; ++k)
            if (k < n && k >= first[i]) {
                const float w = ml[i][k].x == -INFINITY ? 0.f : fast_exp2(ml[i][k].x - M);
                e[k] = ml[i][k].y * w;
#pragma unroll
                for (int v = 0; v < 4; ++v) O[v] = __builtin_fmaf(o[i][k][v], w, O[v]);
            }
#pragma unroll
        for (int x = 1; x < 8; x <<= 1)
#pragma unroll
            for (int k = 0; k < 8; k += 2 * x) e[k] += e[k + x];
        sums[i] = {M, e[0], O};
    }
}
template <int kRows>
__device__ __forceinline__ void join_rows(const Params& p, const int (&row)[kRows], const int (&seq)[kRows],
                                          const int (&first)[kRows], const bool (&stray)[kRows], int d) {
    const int Hq = p.Hkv * p.nrep, T = p.prefix_ranges + p.own_ranges;
    Sums sums[kRows];
    join_states<kRows>(p, 0, T, row, first, d, sums);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (row[i] < 0) continue;
        if (__builtin_expect(stray[i], 0)) {
            const int one[1] = {row[i]}, all[1] = {0};
            Sums more[1];
            int from = T, n = p.strays;
            asm volatile("" : "+s"(from), "+s"(n));   // (its addresses are for this branch alone)
            join_states<1>(p, from, n, one, all, d, more);
            sums[i] = add_sums(sums[i], more[0]);
        }
        const float inv = sums[i].l > 0.f ? 1.0f / sums[i].l : sums[i].l;
        uint16_t* to = p.out + (int64_t)seq[i] * p.o_sb + (int64_t)(row[i] - seq[i] * Hq) * p.o_sh + d;
#pragma unroll
        for (int v = 0; v < 4; ++v) to[v] = p.out_bf16 ? f2bf_rn(sums[i].o[v] * inv) : f2h_rn(sums[i].o[v] * inv);
    }
}
// One more state of (b, h) is stored, by a range of the prefix (work or none) or of own tokens;
// true for the last one.
__device__ __forceinline__ bool arrive(const Params& p, int b, int h) {
    int* at = p.arrivals + (int64_t)b * p.Hkv + h;
    const bool last = __hip_atomic_fetch_add(at, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.prefix_ranges + p.own_ranges - 1;
    __atomic_signal_fence(__ATOMIC_SEQ_CST);   // the states are read behind this
    if (last) __hip_atomic_store(at, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return last;
}
// This wave's states have reached memory.
__device__ __forceinline__ void states_stored() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// The queries of a workgroup's row tiles in LDS: [tile][j][lane] operands of 16 bytes.
constexpr int query_bytes(int tiles) { return tiles * 4096; }

// Blocks [w0, w1) (a wave's) of a group's `count` shared ones, which table row `row` names, against rows
// r0 .. of the group.
template <int NT, bool kJoin>
__device__ __forceinline__ void prefix_rows(const Params& p, float* smem, int split, int b0, int h, int r0, const int32_t* row,
                                            int ids, int w0, int w1, int count, u4 (&qw)[4]) {
    f4 acc[NT][8];
    float m[NT], l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = 0.f;
        l[nt] = 0.f;
#pragma unroll
        for (int n = 0; n < 8; ++n) acc[nt][n] = f4{0.f, 0.f, 0.f, 0.f};
    }
    uint8_t* sm = (uint8_t*)smem;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), R = p.group * p.nrep;
    const Lane ln{lane & 15, lane >> 4, 8 * (lane & 3)};
    const auto stage = [&]() {
        if (wave < NT) {
            query_to_f16(p, qw);
#pragma unroll
            for (int j = 0; j < 4; ++j) *(u4*)(sm + ((wave * 4 + j) * 64 + lane) * 16) = qw[j];
        }
        __syncthreads();
    };
    const auto q = [&](int nt, int j) { return *(const h8*)(sm + ((nt * 4 + j) * 64 + lane) * 16); };
    bool fresh = true;
    Range range;
    attend_int4<NT>(p, row, ids, h, w0, w1, count * kBlockTokens, ln, stage, q, fresh, range, acc, m, l);
    float* states = p.states + (int64_t)split * p.B * p.Hkv * p.nrep * kState;
    float* buf = (float*)(sm + query_bytes(NT));
    // two tiles between barriers
#pragma unroll
    for (int n2 = 0; n2 < NT; n2 += 2) {
        if (n2 > 0) __syncthreads();
#pragma unroll
        for (int nt = n2; nt < NT && nt < n2 + 2; ++nt) merge_put(buf + (nt & 1) * kMergeFloats, wave, ln, acc[nt], m[nt], l[nt]);
        __syncthreads();
#pragma unroll
        for (int nt = n2; nt < NT && nt < n2 + 2; ++nt)
            merge_get<kJoin>(buf + (nt & 1) * kMergeFloats, states, [&](int i) {
                const int r = r0 + nt * 16 + i;
                return r < R ? (b0 + r / p.nrep) * (p.Hkv * p.nrep) + h * p.nrep + r % p.nrep : -1;
            });
    }
}

// A wave's blocks [w0, w1) of a sequence, which table row `row` names, against its rows.
__device__ __forceinline__ void own_rows(const Params& p, int h, const int32_t* row, int ids, int w0, int w1, int len,
                                         const Lane& ln, u4 (&qw)[4], bool& fresh, Range& range, f4 (&acc)[1][8], float (&m)[1],
                                         float (&l)[1]) {
#pragma unroll
    for (int n = 0; n < 8; ++n) acc[0][n] = f4{0.f, 0.f, 0.f, 0.f};
    attend_int4<1>(p, row, ids, h, w0, w1, len, ln, [&]() { query_to_f16(p, qw); },
                   [&](int, int j) { return __builtin_bit_cast(h8, qw[j]); }, fresh, range, acc, m, l);
}

// A range's part of the strays of the sequences whose first rows are r0 + i of a group, bit i of `rows`
// (buf: behind the last merge).
template <bool kJoin>
__device__ __forceinline__ void stray_ranges(const Params& p, float* buf, int split, int b0, int h, int r0, int count,
                                             uint64_t rows) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lane ln{lane & 15, lane >> 4, 8 * (lane & 3)};
    const int Hq = p.Hkv * p.nrep;
    for (; rows != 0; rows &= rows - 1) {
        const int b = b0 + (r0 + __builtin_ctzll(rows)) / p.nrep, len = row_len(p, b);
        const Strays st(p, len, count);
        const int nb = st.to - st.from, np = (nb + 1) >> 1, parts = p.prefix_ranges * kWaves, part = split * kWaves + wave;
        const int w0 = st.from + 2 * (np * part / parts), w1 = st.from + min(2 * (np * (part + 1) / parts), nb);
        const int32_t* row = p.bt + (int64_t)b * p.bt_stride;
        const int ids = w1 > w0 ? request_ids(row, w0, min(kWindow, w1 - w0)) : 0;
        u4 qw[4];
        const bool has = ln.c < p.nrep;
        load_query(p.q + (int64_t)b * p.q_sb + (int64_t)(h * p.nrep + (has ? ln.c : 0)) * p.q_sh + 32 * ln.g, has, qw);
        f4 acc[1][8];
        float m[1] = {0.f}, l[1] = {0.f};
        bool fresh = true;
        Range range;
        own_rows(p, h, row, ids, w0, w1, len, ln, qw, fresh, range, acc, m, l);
        __syncthreads();   // the merge before this one has been read
        merge_put(buf, wave, ln, acc[0], m[0], l[0]);
        __syncthreads();
        float* states = p.states + ((int64_t)(p.prefix_ranges + p.own_ranges + split) * p.B + b) * Hq * kState + (int64_t)h * p.nrep * kState;
        merge_get<kJoin>(buf, states, [&](int i) { return i < p.nrep ? i : -1; });
    }
}

template <int NT, bool kJoin>
__device__ __forceinline__ void prefix_range(const Params& p, float* smem, int id) {
    const int pairs = p.B / p.group * p.Hkv;
    // workgroups of the row tiles of one range follow one another on one XCD
    const int rest = id / kXcc, rt = rest % p.row_tiles;
    const int u = rest / p.row_tiles * kXcc + id % kXcc;
    if (u >= pairs * p.prefix_ranges) return;
    const int split = u / pairs, pair = u - split * pairs, group = pair / p.Hkv, h = pair - group * p.Hkv;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lane ln{lane & 15, lane >> 4, 8 * (lane & 3)};
    const int count = shared_count(p, group), b0 = group * p.group;
    // the range's block pairs, in runs of the waves
    const int np = (count + 1) >> 1, q0 = np * split / p.prefix_ranges, q1 = np * (split + 1) / p.prefix_ranges;
    const int w0 = 2 * (q0 + (q1 - q0) * wave / kWaves), w1 = min(2 * (q0 + (q1 - q0) * (wave + 1) / kWaves), count);
    // the first sequence that holds the shared blocks names them: nearly always the group's
    // first, whose ids are asked for before the lengths are known
    const int32_t* row = p.bt + (int64_t)b0 * p.bt_stride;
    const int n0 = min(kWindow, w1 - w0);
    int ids = n0 > 0 ? request_ids(row, w0, n0) : 0;
    const int R = p.group * p.nrep, r0 = rt * NT * 16;
    u4 qw[4];
    {   // wave nt of the first NT: row tile nt's queries
        const int r = r0 + wave * 16 + ln.c;
        const bool has = wave < NT && r < R;
        const int b = b0 + (has ? r / p.nrep : 0), hd = h * p.nrep + (has ? r % p.nrep : 0);
        load_query(p.q + (int64_t)b * p.q_sb + (int64_t)hd * p.q_sh + 32 * ln.g, has, qw);
    }
    // a sequence's strays are for the workgroup that has its first row: lane i looks at row r0 + i
    const int seq = (r0 + lane) / p.nrep;
    const bool first = p.strays > 0 && lane < NT * 16 && r0 + lane < R && seq * p.nrep == r0 + lane;
    int lead = count > 0 ? 0 : -1, len = p.int4_max_len;   // (lead -1: nobody holds the shared blocks)
    if (p.int4_lens) {
        len = min(p.int4_lens[b0 + min(seq, p.group - 1)], p.int4_max_len);
        lead = -1;
        for (int i = 0; i < p.group && lead < 0 && count > 0; i += 64) {
            const uint64_t has = __ballot(i + lane < p.group && p.int4_lens[b0 + min(i + lane, p.group - 1)] >= count * kBlockTokens);
            if (has) lead = i + __builtin_ctzll(has);
        }
        if (lead > 0) {
            row += (int64_t)lead * p.bt_stride;
            ids = n0 > 0 ? request_ids(row, w0, n0) : 0;
        }
    }
    const uint64_t strays = __ballot(first && Strays(p, len, count).any());
    if (lead >= 0) prefix_rows<NT, kJoin>(p, smem, split, b0, h, r0, row, ids, w0, w1, count, qw);
    if (__builtin_expect(strays != 0, 0)) stray_ranges<kJoin>(p, smem + query_bytes(NT) / sizeof(float), split, b0, h, r0, count, strays);
}
// Behind prefix_range of a group's only row tile: the merge of the sequences whose last state
// this workgroup stored.
__device__ __forceinline__ void prefix_join(const Params& p, float* smem, int id) {
    const int pairs = p.B / p.group * p.Hkv;
    if (id >= pairs * p.prefix_ranges) return;
    const int pair = id % pairs, group = pair / p.Hkv, h = pair - group * p.Hkv, b0 = group * p.group;
    const int i = threadIdx.x >> 5, d = (threadIdx.x & 31) * 4, s = i / p.nrep;   // 16 rows x 32 pieces of 4 dims
    const int b = b0 + min(s, p.group - 1), count = shared_count(p, group);
    const int len = p.int4_lens ? min(p.int4_lens[b], p.int4_max_len) : p.int4_max_len;
    const int first[1] = {count > 0 && len >= count * kBlockTokens ? 0 : p.prefix_ranges}, seq[1] = {b};
    const bool stray[1] = {p.strays > 0 && Strays(p, len, count).any()};
    states_stored();
    __syncthreads();
    int* last = (int*)smem;
    if (threadIdx.x < 64) {   // lane s: sequence s of the group, 16 at most
        const int lane = threadIdx.x;
        const uint64_t mask = __ballot(lane < p.group && arrive(p, b0 + min(lane, p.group - 1), h));
        if (lane == 0) *last = (int)mask;
    }
    __syncthreads();
    const int mask = *last;
    if (mask == 0) return;
    const int row[1] = {s < p.group && (mask >> s & 1) ? b * (p.Hkv * p.nrep) + h * p.nrep + i - s * p.nrep : -1};
    join_rows<1>(p, row, seq, first, stray, d);
}

template <bool kJoin>
__device__ __forceinline__ void own_range(const Params& p, float* smem, int wg) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lane ln{lane & 15, lane >> 4, 8 * (lane & 3)};
    const int pairs = p.B * p.Hkv, Hq = p.Hkv * p.nrep;
    const int u = p.own_waves == 1 ? wg * kWaves + wave : wg;
    if (u >= pairs * p.own_ranges) return;   // a wave of the last workgroup: own_waves is 1, no barrier follows
    const int split = u / pairs, pair = u - split * pairs, b = pair / p.Hkv, h = pair - b * p.Hkv;
    u4 qw[4];
    const bool has = ln.c < p.nrep;
    load_query(p.q + (int64_t)b * p.q_sb + (int64_t)(h * p.nrep + (has ? ln.c : 0)) * p.q_sh + 32 * ln.g, has, qw);
    const int len = row_len(p, b), all = (len + kBlockTokens - 1) / kBlockTokens, s0 = min(p.shared_blocks, all);
    int lens[HKV_MAX_F16_ZONES], tiles = 0;
#pragma unroll
    for (int i = 0; i < HKV_MAX_F16_ZONES; ++i) {
        lens[i] = 0;
        if (i < p.nz) lens[i] = p.z[i].lens ? min(max(load_uniform_i32(p.z[i].lens, b), 0), p.z[i].max_len) : p.z[i].max_len;
        tiles += (lens[i] + kBlockTokens - 1) / kBlockTokens;
    }
    // this wave's share of both kinds (at most 2^22 items in 512 parts: 32 bits)
    const uint32_t parts = p.own_ranges * p.own_waves, part = p.own_waves == 1 ? split : split * kWaves + wave;
    const int nb = all - s0, np = (nb + 1) >> 1;
    const int x0 = (uint32_t)np * part / parts, x1 = (uint32_t)np * (part + 1) / parts;
    const int f0 = (uint32_t)tiles * part / parts, f1 = (uint32_t)tiles * (part + 1) / parts;
    const int w0 = s0 + 2 * x0, w1 = s0 + min(2 * x1, nb);
    const int32_t* row = p.bt + (int64_t)b * p.bt_stride;
    const int ids = w1 > w0 ? request_ids(row, w0, min(kWindow, w1 - w0)) : 0;
    f4 acc[1][8];
    float m[1] = {0.f}, l[1] = {0.f};
    bool fresh = true;
    Range range;
    own_rows(p, h, row, ids, w0, w1, len, ln, qw, fresh, range, acc, m, l);
    if (f1 > f0) {
        h8 qf[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[j] = __builtin_bit_cast(h8, qw[j]);
        attend_f16(p, b, h, lens, f0, f1, ln, qf, fresh, range, acc, m, l);
    }
    float* states = p.states + ((int64_t)(p.prefix_ranges + split) * p.B + b) * Hq * kState + (int64_t)h * p.nrep * kState;
    int none = 0;        // prefix states that the sequence has no part in
    bool strays = false;
    if constexpr (kJoin) {
        const int count = p.prefix_ranges > 0 ? shared_count(p, b / p.group) : 0;
        none = count > 0 && len >= count * kBlockTokens ? 0 : p.prefix_ranges;
        strays = p.strays > 0 && Strays(p, len, count).any();
    }
    if (p.own_waves == 1) {
        const float sum = row_sum(l[0]);
        if (ln.c < p.nrep) {
#pragma unroll
            for (int n = 0; n < 8; ++n) put_state<kJoin>(states, ln.c * kState + 16 * n + 4 * ln.g, acc[0][n]);
            if (ln.g == 0) put_state<kJoin>(states, ln.c * kState + kHeadDim, f2{sum == 0.f ? -INFINITY : m[0], sum});
        }
        if constexpr (kJoin) {
            states_stored();
            int last = 0;
            if (lane == 0) last = arrive(p, b, h);
            if (!__builtin_amdgcn_readfirstlane(last)) return;
            for (int r = 0; r < p.nrep; r += 4) {   // two rows at a time and half wave
                int rows[2], seq[2], firsts[2];
                bool stray[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int i = r + 2 * k + (lane >> 5);
                    seq[k] = b;
                    firsts[k] = none;
                    stray[k] = strays;
                    rows[k] = i < p.nrep ? b * Hq + h * p.nrep + i : -1;
                }
                join_rows<2>(p, rows, seq, firsts, stray, (lane & 31) * 4);
            }
        }
    } else {
        merge_put(smem, wave, ln, acc[0], m[0], l[0]);
        __syncthreads();
        merge_get<kJoin>(smem, states, [&](int i) { return i < p.nrep ? i : -1; });
        if constexpr (kJoin) {
            states_stored();
            __syncthreads();
            int* last = (int*)smem;
            if (threadIdx.x == 0) *last = arrive(p, b, h);
            __syncthreads();
            if (!*last) return;
            const int i = threadIdx.x >> 5;
            const int row[1] = {i < p.nrep ? b * Hq + h * p.nrep + i : -1}, seq[1] = {b}, first[1] = {none};
            const bool stray[1] = {strays};
            join_rows<1>(p, row, seq, first, stray, (threadIdx.x & 31) * 4);
        }
    }
}

// 8 waves, two on a SIMD: up to 256 registers each.
template <int NT, bool kJoin>
__global__ __launch_bounds__(kThreads, 1) void shared_attn_kernel(Params p) {
    touch_kernel_args(p);
    extern __shared__ __align__(16) float smem[];
    const int id = (int)blockIdx.x;
    if (p.own_first ? id >= p.own_wgs : id < p.prefix_wgs) {
        prefix_range<NT, kJoin>(p, smem, p.own_first ? id - p.own_wgs : id);
        if constexpr (kJoin) prefix_join(p, smem, p.own_first ? id - p.own_wgs : id);
    } else {
        own_range<kJoin>(p, smem, p.own_first ? id : id - p.prefix_wgs);
    }
}

// Merges the states of an output row: kWavesRow waves take every kWavesRow-th state each, lane i
// of a wave holds the weight of its i-th, the lanes two dims each.  With few states a wave does a
// row, with many four waves do, whose loads are all on their way at once.
constexpr int kCombine = 4;   // waves of a workgroup
template <int kWavesRow>
__global__ __launch_bounds__(kCombine * 64) void shared_combine_kernel(Params p) {
    touch_kernel_args(p);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int Hq = p.Hkv * p.nrep, row = (int)blockIdx.x * (kCombine / kWavesRow) + (kWavesRow == 1 ? wave : 0);
    if (kWavesRow == 1 && row >= p.B * Hq) return;
    const int b = row / Hq, hd = row - b * Hq, part = kWavesRow == 1 ? 0 : wave;
    const int64_t stride = (int64_t)p.B * Hq * kState;   // between a row's states
    static_assert(2 * kMaxRanges <= kCombine * 64 && kFewStates <= 64, "a lane for every state");
    const float* st = p.states + (int64_t)row * kState + part * stride;
    // the sums of states [from, n) of every kWavesRow-th one at `at`; from(): asked for when the states
    // are on their way
    const auto sum_states = [&](const float* at, int n, const auto& from, float& M, float& L, float& o0, float& o1) {
        M = -INFINITY;
        L = o0 = o1 = 0.f;
        if (n <= 0) return;
        f2 ml = {-INFINITY, 0.f};
        if (lane < n) ml = *(const f2*)(at + lane * kWavesRow * stride + kHeadDim);
        f2 o[8];   // eight states on their way; past the last one it again, with weight 0
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = *(const f2*)(at + min(j, n - 1) * kWavesRow * stride + 2 * lane);
        const int first = from();
        if (lane < first) ml = f2{-INFINITY, 0.f};
        M = ml.x;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
        const float e = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
        L = ml.y * e;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) L += __shfl_xor(L, x);
        for (int i = 0; i < n; i += 8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e), min(i + j, 63)));   // past n: 0
                const bool in = i + j >= first && i + j < n;   // (past n: state n - 1 may have no part either)
                o0 = __builtin_fmaf(in ? o[j].x : 0.f, w, o0);
                o1 = __builtin_fmaf(in ? o[j].y : 0.f, w, o1);
                if (i + 8 < n) o[j] = *(const f2*)(at + min(i + 8 + j, n - 1) * kWavesRow * stride + 2 * lane);
            }
        }
    };
    const auto part_of = [&](int n) { return (n - part + kWavesRow - 1) / kWavesRow; };   // this wave's of n states
    const int T = p.prefix_ranges + p.own_ranges;
    float M, L, o0, o1;
    // A sequence that does not hold the shared blocks has no part in the prefix's states, which may
    // hold anything.
    bool stray = false;
    sum_states(st, part_of(T), [&]() {   // (asked in every wave: with several a row, T > kFewStates)
        if (p.prefix_ranges == 0) return 0;
        const int len = row_len(p, b), count = shared_count(p, b / p.group);
        stray = p.strays > 0 && Strays(p, len, count).any();
        return count > 0 && len >= count * kBlockTokens ? 0 : part_of(p.prefix_ranges);
    }, M, L, o0, o1);
    if (__builtin_expect(stray, 0)) {
        float M2, L2, p0, p1;
        sum_states(st + T * stride, part_of(p.strays), []() { return 0; }, M2, L2, p0, p1);
        const float top = fmaxf(M, M2), w = M == -INFINITY ? 0.f : fast_exp2(M - top), w2 = M2 == -INFINITY ? 0.f : fast_exp2(M2 - top);
        M = top;
        L = __builtin_fmaf(L2, w2, L * w);
        o0 = __builtin_fmaf(p0, w2, o0 * w);
        o1 = __builtin_fmaf(p1, w2, o1 * w);
    }
    if constexpr (kWavesRow > 1) {
        __shared__ float sm[kWavesRow][kHeadDim + 2];
        sm[wave][2 * lane] = o0;
        sm[wave][2 * lane + 1] = o1;
        if (lane == 0) {
            sm[wave][kHeadDim] = M;
            sm[wave][kHeadDim + 1] = L;
        }
        __syncthreads();
        if (wave != 0) return;
        M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWavesRow; ++w) M = fmaxf(M, sm[w][kHeadDim]);
        L = o0 = o1 = 0.f;
#pragma unroll
        for (int w = 0; w < kWavesRow; ++w) {
            const float mw = sm[w][kHeadDim], e = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
            L += sm[w][kHeadDim + 1] * e;
            o0 += sm[w][2 * lane] * e;
            o1 += sm[w][2 * lane + 1] * e;
        }
    }
    const float inv = L > 0.f ? 1.0f / L : L;   // without a token 0; NaN stays NaN
    o0 *= inv;
    o1 *= inv;
    uint16_t* to = p.out + (int64_t)b * p.o_sb + (int64_t)hd * p.o_sh + 2 * lane;
    to[0] = p.out_bf16 ? f2bf_rn(o0) : f2h_rn(o0);
    to[1] = p.out_bf16 ? f2bf_rn(o1) : f2h_rn(o1);
}

// ---- the work plan (host)
int num_cus() {
    static std::atomic<int> cached[64];   // per device (partition modes can differ)
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess) return 256;
    const int c = cached[dev & 63].load(std::memory_order_relaxed);
    if (c > 0) return c;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) return 256;
    cached[dev & 63].store(n, std::memory_order_relaxed);
    return n;
}

struct Plan {
    int tiles, row_tiles;          // row tiles per workgroup, workgroups of rows
    int prefix_ranges, own_ranges, own_waves, strays;
    int64_t prefix_wgs, own_wgs;
    bool own_first;
    double end;                    // of the workgroups, in us, as modelled
};

// What a workgroup takes, in us, where HBM keeps up: a prefix range kPrefixStart, for every row
// tile kPrefixMerge, and for every pair of blocks a wave takes kPrefixPair, and kPrefixTile for
// each row tile of it; a range of a sequence's own tokens kOwnStart, and kOwnItem for every pair
// of blocks or fp16 tile.
constexpr double kPrefixStart = 2.5, kPrefixMerge = 1.2, kPrefixPair = 0.7, kPrefixTile = 0.6, kOwnStart = 4.0, kOwnItem = 1.3;

// The ranges with the earliest end.  One workgroup is on a CU at a time, longer ones first; if not
// all find a CU at once, the end is the work over the CUs and half of a short workgroup, or
// the rounds of the long ones.
Plan make_plan(const HkvSharedArgs* s) {
    const HkvDecodeArgs* a = &s->decode;
    const int nrep = a->num_q_heads / a->num_kv_heads, rows = s->group * nrep;
    Plan p = {};
    p.row_tiles = (rows + kMaxTiles * 16 - 1) / (kMaxTiles * 16);
    p.tiles = (rows + p.row_tiles * 16 - 1) / (p.row_tiles * 16);
    const double cus = num_cus();
    const int64_t prefix_units = (int64_t)(a->batch / s->group) * a->num_kv_heads, own_units = (int64_t)a->batch * a->num_kv_heads;
    const int prefix_pairs = (s->shared_blocks + 1) / 2;
    int64_t items = 0;   // of a sequence's own tokens
    for (int i = 0; i < a->num_f16_zones; ++i) items += ((int64_t)a->f16[i].max_len + kBlockTokens - 1) / kBlockTokens;
    items += ((a->int4_max_len + kBlockTokens - 1) / kBlockTokens - s->shared_blocks + 1) / 2;
    const bool own = items > 0 || prefix_pairs == 0;
    double best = 0;
    for (int o = 1; o <= kMaxRanges; o *= 2) {
        // up to four ranges a wave each, beyond that (8, 16, ..) a workgroup of eight waves each
        const int waves = o <= 4 ? 1 : kWaves, own_ranges = o <= 4 ? o : o / kWaves;
        if (o > 1 && (!own || o > items)) break;
        const double own_one = kOwnStart + (double)((items + o - 1) / o) * kOwnItem;
        const int64_t own_wgs = own ? (waves == 1 ? (own_units * own_ranges + kWaves - 1) / kWaves : own_units * own_ranges) : 0;
        for (int n = 1; n <= kMaxRanges; ++n) {
            if (n > 1 && n * kWaves > prefix_pairs) break;
            const int steps = ((prefix_pairs + n - 1) / n + kWaves - 1) / kWaves;
            const double one = kPrefixStart + p.tiles * kPrefixMerge + steps * (kPrefixPair + p.tiles * kPrefixTile);
            const int64_t wgs = prefix_pairs > 0 ? (prefix_units * n + kXcc - 1) / kXcc * kXcc * p.row_tiles : 0;
            const double longer = wgs == 0 ? own_one : own_wgs == 0 || one > own_one ? one : own_one;
            double t = longer;
            if (wgs + own_wgs > cus) {
                const double even = (wgs * one + own_wgs * own_one) / cus;
                const double rounds = (int64_t)((wgs + cus - 1) / cus) * one;
                t = rounds > even ? rounds : even;
                if (own_wgs > 0) t += 0.5 * (one < own_one ? one : own_one);
                if (t < longer) t = longer;
            }
            if (best == 0 || t < best * 0.98) {
                p.end = best = t;
                p.prefix_ranges = prefix_pairs > 0 ? n : 0;
                p.prefix_wgs = wgs;
                p.own_ranges = own ? own_ranges : 0;
                p.own_waves = waves;
                p.own_wgs = own_wgs;
                p.own_first = own_wgs > 0 && own_one > one;
            }
            if (prefix_pairs == 0) break;
        }
    }
    // (how many there are is not known here: lengths and counts are the device's)
    p.strays = a->int4_lens || s->shared_counts ? p.prefix_ranges : 0;
    return p;
}

// A short call of few rows and states: no second launch.  That saves 2 us of the host's 14, which is
// what an eager short call takes (2 samples of 1024 tokens 13.9 -> 11.8 us, 4 of 512 14.2 -> 11.7), and nothing
// on the GPU: stores past the L2, a counter and the reads by one workgroup take what a launch does
// (11.5 and 11.4 us).  More row tiles lost (11 samples of 3 rows, 720 tokens: 15.2 and 17.0), more states too
// (12 of them: 0.7 us for the code alone, 24 KB that few waves run).
constexpr double kJoinEnd = 12.0;
bool joins(const HkvSharedArgs* s, const Plan& p) {
    return s->arrivals && p.end <= kJoinEnd && p.tiles == 1 && p.row_tiles == 1 && p.prefix_ranges + p.own_ranges <= kJoinFew;
}

size_t state_bytes(const HkvDecodeArgs* a, const Plan& p) {
    return (size_t)(p.prefix_ranges + p.own_ranges + p.strays) * a->batch * a->num_q_heads * kState * sizeof(float);
}

int check_shared(const HkvSharedArgs* s) {
    HKV_REQUIRE(s != nullptr, HKV_ERR_ARG, "hkv_shared_attn: null args");
    const HkvDecodeArgs* a = &s->decode;
    const int rc = check_decode_shape(a, "hkv_shared_attn");
    if (rc != HKV_OK) return rc;
    HKV_REQUIRE(s->group > 0 && a->batch % s->group == 0, HKV_ERR_ARG, "hkv_shared_attn: a batch of %d in groups of %d",
                a->batch, s->group);
    HKV_REQUIRE(a->int4_max_len >= 0 && a->int4_max_len <= kMaxZoneTokens && s->shared_blocks >= 0 &&
                    s->shared_blocks <= a->int4_max_len / kBlockTokens,
                HKV_ERR_ARG, "hkv_shared_attn: %d shared blocks in %d INT4 tokens", s->shared_blocks, a->int4_max_len);
    HKV_REQUIRE(!a->scores && !a->score_stats && a->splits_hint == 0, HKV_ERR_UNSUPPORTED,
                "hkv_shared_attn: no score output and no splits_hint");
    return HKV_OK;
}

}  // namespace
}  // namespace hkv

using namespace hkv;

extern "C" size_t hkv_shared_workspace_bytes(const HkvSharedArgs* s) {
    clear_error();
    if (check_shared(s) != HKV_OK) return 0;
    return state_bytes(&s->decode, make_plan(s));
}

extern "C" int hkv_shared_launches(const HkvSharedArgs* s) {
    clear_error();
    if (check_shared(s) != HKV_OK) return 0;
    return joins(s, make_plan(s)) ? 1 : 2;
}

extern "C" int hkv_shared_attn(const HkvSharedArgs* s, void* stream) {
    clear_error();
    int rc = check_shared(s);
    if (rc != HKV_OK) return rc;
    const HkvDecodeArgs* a = &s->decode;
    rc = check_decode_buffers(a, a->workspace, true, "hkv_shared_attn");
    if (rc != HKV_OK) return rc;
    const Plan plan = make_plan(s);
    const size_t need = state_bytes(a, plan);
    HKV_REQUIRE(a->workspace_bytes >= need, HKV_ERR_CAPACITY, "hkv_shared_attn: workspace %zu bytes, need %zu",
                a->workspace_bytes, need);
    HKV_REQUIRE((((uintptr_t)a->workspace) & 15) == 0, HKV_ERR_ARG, "hkv_shared_attn: workspace must be 16-byte aligned");
    HKV_REQUIRE((((uintptr_t)s->arrivals) & 3) == 0, HKV_ERR_ARG, "hkv_shared_attn: arrivals must be 4-byte aligned");
    Params p = {};
    p.B = a->batch;
    p.Hkv = a->num_kv_heads;
    p.nrep = a->num_q_heads / a->num_kv_heads;
    p.group = s->group;
    p.scale_log2 = a->sm_scale * kLog2e;
    p.q_bf16 = a->q_dtype == HKV_DTYPE_BF16;
    p.out_bf16 = a->out_dtype == HKV_DTYPE_BF16;
    p.q = a->q;
    p.q_sb = a->q_stride_b;
    p.q_sh = a->q_stride_h;
    p.nz = a->num_f16_zones;
    for (int i = 0; i < p.nz; ++i) p.z[i] = ZoneP{a->f16[i].k, a->f16[i].v, a->f16[i].capacity, a->f16[i].max_len, a->f16[i].lens};
    p.pool = a->pool;
    p.pool_blocks = a->pool ? a->pool_blocks : 0;
    p.staging = a->staging;
    p.staging_blocks = a->staging ? a->staging_blocks : 0;
    p.fallback_id = p.pool_blocks > 0 ? 0 : -1;
    p.bt = a->block_table;
    p.bt_stride = a->bt_stride;
    p.int4_lens = a->int4_lens;
    p.int4_max_len = a->int4_max_len;
    p.out = a->out;
    p.o_sb = a->out_stride_b;
    p.o_sh = a->out_stride_h;
    p.err = a->err_flag;
    p.states = (float*)a->workspace;
    p.counts = s->shared_counts;
    p.shared_blocks = s->shared_blocks;
    p.row_tiles = plan.row_tiles;
    p.prefix_ranges = plan.prefix_ranges;
    p.own_ranges = plan.own_ranges;
    p.strays = plan.strays;
    p.own_waves = plan.own_waves;
    p.prefix_wgs = (int)plan.prefix_wgs;
    p.own_wgs = (int)plan.own_wgs;
    p.own_first = plan.own_first;
    const bool join = joins(s, plan);
    p.arrivals = join ? s->arrivals : nullptr;
    static void (*const fns[kMaxTiles + 1])(Params) = {shared_attn_kernel<1, false>, shared_attn_kernel<2, false>,
                                                       shared_attn_kernel<3, false>, shared_attn_kernel<4, false>,
                                                       shared_attn_kernel<1, true>};
    static std::atomic<uint64_t> raised[kMaxTiles + 1];
    const int var = join ? kMaxTiles : plan.tiles - 1;
    const size_t lds = query_bytes(plan.tiles) + (plan.tiles > 1 ? 2 : 1) * kMergeFloats * sizeof(float);
    HKV_RAISE_LDS(fns[var], query_bytes(kMaxTiles) + 2 * kMergeFloats * (int)sizeof(float), raised[var]);
    hipLaunchKernelGGL(fns[var], dim3((unsigned)(plan.prefix_wgs + plan.own_wgs)), dim3(kThreads), lds, (hipStream_t)stream, p);
    HKV_LAUNCH_CHECK("shared_attn_kernel");
    if (join) return HKV_OK;
    const bool few = p.prefix_ranges + p.own_ranges <= kFewStates;
    const unsigned rows = (unsigned)(a->batch * a->num_q_heads);
    hipLaunchKernelGGL(few ? shared_combine_kernel<1> : shared_combine_kernel<kCombine>, dim3(few ? (rows + kCombine - 1) / kCombine : rows),
                       dim3(kCombine * 64), 0, (hipStream_t)stream, p);
    HKV_LAUNCH_CHECK("shared_combine_kernel");
    return HKV_OK;
}
