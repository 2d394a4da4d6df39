// flash_attn_bwd.cu - causal grouped-query flash attention backward for sm_100a, head_dim 128.
//
// Two launches, deterministic (no atomics):
//   1. attn_delta_kernel   delta[b,h,s] = sum_d dO * O                      (bandwidth bound)
//   2. attn_bwd_kernel, whose CTAs do one of two things:
//      dK / dV             one CTA per (kv tile, kv head, batch). It sweeps the query tiles at or
//                          below the diagonal of every query head of the group and accumulates
//                          dK and dV in tensor memory. Scores are computed transposed
//                          (S^T = K Q^T, dP^T = V dO^T) so that TMEM lanes are kv rows; the bf16
//                          P^T goes through shared memory and feeds dV += P^T dO from there, dS^T is
//                          written back over dP^T and feeds dK += dS^T Q as A operand straight from TMEM.
//      dQ                  one CTA per (q tile, head, batch): S = Q K^T, dP = dO V^T,
//                          dS -> TMEM, dQ += dS K.
// Q, K, V and dO tiles arrive by TMA from the packed activation; each shared-memory tile serves
// both as a K-major operand (for the score products) and as an MN-major operand (for the
// gradient products) through different UMMA descriptors, so nothing is transposed in memory.
//
// Roles per CTA: warp 0 issues TMA, warps 1 and 2 issue the MMAs, sixteen warps do the exponentials (four groups of
// four; a warp owns 32 TMEM lanes, a group 32 of the step's 128 score columns). What bounds a step is the latency chain
// of the compute warps, not the tensor pipe, so as little of that pipe's time as possible is left on the chain:
//   dK / dV: S^T(i+1) is computed as soon as the warps hold the scores of step i in registers. P^T leaves through shared
//            memory (in place of S^T it would hold up S^T(i+1) until dV(i) is done), before dP^T is looked at; dS^T goes
//            over dP^T in TMEM. Warp 1 issues S^T and dV, warp 2 dP^T and dK.
//   dQ:      warp 1 runs S ahead in two buffers, warp 2 alternates dP(j) and dQ(j).
// Two issuing warps because a wait costs the issuing thread 110-300 cycles even when it is already satisfied (its
// shared-memory access queues behind the operand reads of the MMAs): the other warp's MMAs run meanwhile. Each warp's MMAs
// execute in the order of issue, which is what protects dP / dS (one overwrites the other); the two warps share no
// operand that either writes. A thread keeps its 32 probabilities in fp32 registers until dP arrives. bf16 results in TMEM
// go over the first half of the 32 columns they came from, so the groups never touch each other's columns and need
// no barrier inside a step; a warp keeps the statistics of its queries in 32 words of its own. Every warp arrives once (not
// every thread) on a barrier. The softmax scale is applied once to the finished dK / dQ, and only diagonal tiles run the
// code path with the mask.
// Measured on a B200, before (one step at a time: scores, exponentials, gradients) and now, both back to back on one GPU:
// 8192 tokens, 32 / 8 heads: dK / dV 5390 -> 3700 cycles per 128 x 128 step and SM (1279 -> 1010 us: at 990 W the clock falls
// from 1900 to 1640 MHz), dQ 4240 -> 3030 cycles (986 -> 800 us). 4096 tokens, 16 / 8 heads: 203 -> 140 and 170 -> 111 us.
// P^T over S^T in TMEM, with S^T(i+1) behind dV(i): 8 % slower. Asking the barriers early without blocking, and fetching
// the next scores before dS^T is handed over: 2-10 % slower.
//
// The windowed form (kWindow; a window and sinks, sequences of any length) is the same two parts over lists of tiles: of dK / dV the query tiles that see a key tile, of dQ the key
// tiles that a query tile sees. It cuts dK / dV's sums into parts that a third kernel adds up in a fixed order (AttnWindowParts): over heads and query tiles in small
// grids, and the sinks' sums, which run over all later queries. Tensor maps with the sequences apart bring rows past a sequence's end as zeros and leave them out of the
// result. Warps that see nothing of a tile skip its exponentials. us: 4 x 4096 tokens, 16 / 8 heads, 4 sinks, window 1024 540 in a burst, 590 back to back at the power
// limit (985 W, 1657-1725 MHz; 560 TFLOP/s of the five products of what is seen; seven are computed), window 128 280; 16384 tokens, window 4096 1680; 333 tokens, 8 / 1 heads 14.8, 2 x 128,
// 2 / 1 heads 10.1. (Window 128 moves 62 us of bytes: a CTA has two to four steps there, and set-up, first loads, staging and writing, which take longer, overlap nothing: it has
// the SM's whole shared memory.) dQ from the same scores as dK / dV, added to in L2 in a fixed order, took 725 against 600: the additions go at some 30 bytes a cycle and SM.
//
// Replaces the reference's one-thread-per-query backward, which recomputes dp twice, scatters
// dK/dV with atomicAdd and never zeroes dq/dk/dv (src/cuda/cai_kernels.cu:110-143).
#include <math.h>

#include "attn_common.cuh"
#include "attn_window.cuh"
#include "cai_kernels.h"
#include "host_common.h"
#include "sm100.cuh"

namespace cai {

// How the dK / dV part of the windowed form is cut into CTAs. A key tile's sum runs over the query heads of its group and over the query tiles that see it: those of
// the window, and, where it holds sinks, all later ones. The heads are cut into `head_parts`, the window's query tiles into `near_parts` of `near_tiles`
// each, the later ones into `far_parts` of `far_tiles`. Tiles with more than one part leave sums in fp32 in the caller's scratch, 128 KB a part, which a
// second kernel adds up in a fixed order.
struct AttnWindowParts {
    int head_parts, near_parts, near_tiles, far_parts, far_tiles;
    int sink_tiles;          // key tiles that hold sinks and are seen by query tiles behind their window
    int near_ctas, far_ctas, near_slots;
};

// The part that CTA `lin` of the dK / dV part works on: those of the window first, key tiles slowest, heads and batch fastest.
struct WindowPart {
    int j, b, g, h_first, heads;    // key tile, batch, kv head, query heads
    int q_first, q_tiles;           // query tiles of each head (none or less: nothing to do, for the last parts of a late tile)
    int slot;                       // of the scratch; -1: the CTA has the whole sum
    __host__ __device__ WindowPart(const AttnWindow& w, const AttnWindowParts& c, int B, int S, int nh, int nkv, int lin) {
        const int rep = nh / nkv, nq = (S + kAttnTile - 1) / kAttnTile, stride = nkv * c.head_parts * B;
        const bool far = lin >= c.near_ctas;
        const int rest = (far ? lin - c.near_ctas : lin) / stride, at = lin % stride, y = at % (nkv * c.head_parts);   // near_ctas is a multiple of stride
        const int parts = far ? c.far_parts : c.near_parts, tiles = far ? c.far_tiles : c.near_tiles;
        j = rest / parts;
        b = at / (nkv * c.head_parts);
        g = y / c.head_parts;
        heads = rep / c.head_parts;
        h_first = g * rep + y % c.head_parts * heads;
        const int near_end = window_last_query_tile(w, j, nq) + 1, end = far ? nq : near_end;
        q_first = (far ? near_end : j) + (rest - j * parts) * tiles;
        q_tiles = (q_first + tiles < end ? q_first + tiles : end) - q_first;
        slot = c.head_parts * c.near_parts == 1 && (j >= c.sink_tiles || near_end >= nq) ? -1 : far ? c.near_slots + lin - c.near_ctas : lin;
    }
};

struct AttnBwdParams {
    int B, S, nh, nkv;
    float scale, scale_log2;
    const float* lse;
    const float* delta;
    __nv_bfloat16* dqkv;
    int* status;
    // dK / dV with one CTA per QUERY head (small grids): the heads of a kv group take turns adding their
    // contribution to the group's dK / dV rows; chain[b][g][kv tile] counts the heads that are done.
    int split_heads;
    unsigned int* chain;
    const float2* rope;          // (cos, sin) [S][64]: dQ and dK leave rotated back (null: as they are)
    AttnWindow win;              // of the windowed form
    AttnWindowParts cut;
    float* partial;
    long long ldq;               // row pitch of dqkv
};

// chain counters of the head-split dK / dV kernel: one per (batch, kv group, kv tile).
// ONE array serves every call on a device: each call clears the slots it uses (in stream order: the row sums' kernel, or a
// memset) before its kernel, so two attention backwards that overlap on one GPU (different streams) would reset each other's
// counters. Calls that take the head-split path must therefore be ordered against each other; the executor
// issues them from one stream. A CTA of turn t waits (bounded) for the CTA of turn t - 1 of the same kv tile,
// which has a lower linear block id: with no more of these CTAs than SMs, and nothing beside them that waits, every one of them gets
// an SM whatever the order of dispatch; the launcher only takes this path then.
constexpr size_t kAttnChainSlots = 65536;
__device__ unsigned int g_attn_chain[kAttnChainSlots];

// Sixteen lanes per (token, head), 16 bytes a lane from each tensor, kDeltaUnroll of them in flight per thread: what bounds this is
// bytes in flight (one pair of 8-byte loads per thread and a 64-bit division in front: 8192 tokens of
// 32 heads 47 -> 23 us, 6 x 640 tokens of 9 heads 8.5 -> 6.2 us). The tensors are walked as one array of
// 128-element rows. (dO starts on 16 bytes, or its tensor map is refused; O may start on 8.)
constexpr int kDeltaUnroll = 2;
__global__ void __launch_bounds__(256)
attn_delta_kernel(const __nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ dout, float* __restrict__ delta,
                  unsigned total, unsigned S, unsigned nh, bool out16, unsigned int* chain, unsigned chain_slots) {
    grid_dep_begin();
    if (blockIdx.x * 256u + threadIdx.x < chain_slots) chain[blockIdx.x * 256u + threadIdx.x] = 0;   // for the dK / dV kernel behind this one
    const unsigned w0 = blockIdx.x * (16u * kDeltaUnroll) + (threadIdx.x >> 4);
    const int sub = threadIdx.x & 15;
    uint4 a[kDeltaUnroll], d[kDeltaUnroll];
#pragma unroll
    for (int i = 0; i < kDeltaUnroll; ++i) {
        const unsigned w = w0 + 16u * i;
        a[i] = d[i] = make_uint4(0, 0, 0, 0);
        if (w < total) {
            const size_t off = static_cast<size_t>(w) * kAttnHD + sub * 8;
            if (out16) {
                a[i] = *reinterpret_cast<const uint4*>(out + off);
            } else {
                const uint2 lo = *reinterpret_cast<const uint2*>(out + off), hi = *reinterpret_cast<const uint2*>(out + off + 4);
                a[i] = make_uint4(lo.x, lo.y, hi.x, hi.y);
            }
            d[i] = *reinterpret_cast<const uint4*>(dout + off);
        }
    }
#pragma unroll
    for (int i = 0; i < kDeltaUnroll; ++i) {
        // two quads of elements per lane, added last: the tree of sums over quads 16, 8, 4, 2 and 1 apart
        float s0 = bf16_lo(a[i].x) * bf16_lo(d[i].x) + bf16_hi(a[i].x) * bf16_hi(d[i].x) + bf16_lo(a[i].y) * bf16_lo(d[i].y) +
                   bf16_hi(a[i].y) * bf16_hi(d[i].y);
        float s1 = bf16_lo(a[i].z) * bf16_lo(d[i].z) + bf16_hi(a[i].z) * bf16_hi(d[i].z) + bf16_lo(a[i].w) * bf16_lo(d[i].w) +
                   bf16_hi(a[i].w) * bf16_hi(d[i].w);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            s0 += __shfl_xor_sync(0xffffffffu, s0, o);
            s1 += __shfl_xor_sync(0xffffffffu, s1, o);
        }
        const float s = s0 + s1;
        const unsigned w = w0 + 16u * i;
        if (sub == 0 && w < total) {
            const unsigned row = w / nh, h = w - row * nh, b = row / S, at = row - b * S;
            delta[(static_cast<size_t>(b) * nh + h) * S + at] = s;
        }
    }
}

// Sixteen compute warps: every scheduler has four of them to hide the TMEM and shared-memory latencies.
constexpr int kAttnGroups = 4;
constexpr int kAttnComputeThreads = kAttnGroups * 128;
constexpr int kAttnBwdThreads = 128 + kAttnComputeThreads;  // warp 0 TMA, warps 1-2 MMA, warps 4-19 compute

__device__ __forceinline__ void bar_sync_compute() { asm volatile("bar.sync 1, 512;" ::: "memory"); }

// A finished 128 x 128 fp32 accumulator goes to its bf16 rows through shared memory (operands nobody reads any more), so that a warp writes, and where
// it adds to what is there reads, two whole rows at a time. From the registers a lane had a row of its own, 32 lines an access: a turn of the heads' chain
// took 9 us, now 3.4. us, both parts and the row sums, before / now: 4 x 128 tokens, 2 / 1 heads 18.6 / 13.5; 512 tokens, 8 / 1 heads 75.4 / 40.2;
// 2048, 8 / 2 72.2 / 51.5; 8192, 2 / 1 138 / 124. (The old rows read ahead of every store, still a row per lane: no change.)
// Staged: row r at r * 512, its 16-byte chunk c at c ^ (r & 7).
__device__ __forceinline__ void stage_acc_chunk(uint32_t tacc, uint32_t stage, int r, int c) {
    uint32_t v[32];
    tmem_ld_32x32(tacc + c * 32, v);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 8; ++k)
        st_shared_v4(stage + r * 512 + (((c * 8 + k) ^ (r & 7)) << 4), v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
}
// A thread of 512 takes kPieces times eight columns and the eight that are 64 further on: item `first` of eight a row, 128 rows a tile of 64 KB, then
// every 512th. Tile t leaves at dst[t], times mul[t]; where `rope` is given (the row of its table that belongs to row 0), tile 0 is rounded, as it
// would be in memory, and rotated back.
template <bool kAdd, int kPieces>
__device__ __forceinline__ void write_staged(uint32_t stage, __nv_bfloat16* const (&dst)[2], const float (&mul)[2], long long ld, int first, const float2* rope) {
    uint4 old[kPieces][2];
    if constexpr (kAdd) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int item = first + i * 512;
                old[i][h] = *reinterpret_cast<const uint4*>(dst[i >> 1] + ((item >> 3) & 127) * ld + h * 64 + (item & 7) * 8);
            }
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int item = first + i * 512, r = (item >> 3) & 127, c = (item & 7) * 2;
        const uint32_t row = stage + (i >> 1) * 65536 + r * 512;
        uint32_t o[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float4 f = ld_shared_f4(row + ((((h * 16) + c + k) ^ (r & 7)) << 4));
                v[4 * k] = f.x; v[4 * k + 1] = f.y; v[4 * k + 2] = f.z; v[4 * k + 3] = f.w;
            }
            const uint32_t ov[4] = {kAdd ? old[i][h].x : 0u, kAdd ? old[i][h].y : 0u, kAdd ? old[i][h].z : 0u, kAdd ? old[i][h].w : 0u};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float lo = v[2 * t] * mul[i >> 1], hi = v[2 * t + 1] * mul[i >> 1];
                if constexpr (kAdd) {
                    lo += bf16_lo(ov[t]);
                    hi += bf16_hi(ov[t]);
                }
                o[h][t] = pack_bf16(lo, hi);
            }
        }
        if (rope && (i >> 1) == 0) {
            const float4* cs = reinterpret_cast<const float4*>(rope + r * 64 + (item & 7) * 8);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float4 q = cs[t];      // of two columns
                float a0 = bf16_lo(o[0][t]), a1 = bf16_hi(o[0][t]), b0 = bf16_lo(o[1][t]), b1 = bf16_hi(o[1][t]);
                rope_rotate(a0, b0, q.x, -q.y);
                rope_rotate(a1, b1, q.z, -q.w);
                o[0][t] = pack_bf16(a0, a1);
                o[1][t] = pack_bf16(b0, b1);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<uint4*>(dst[i >> 1] + r * ld + h * 64 + (item & 7) * 8) = make_uint4(o[h][0], o[h][1], o[h][2], o[h][3]);
    }
}

// A part's sums in the scratch: four columns (of piece c of 32) of row r of dK or dV at this float, eight rows to a line of 128 bytes.
__device__ __forceinline__ int window_part_at(int which, int r, int c) { return which * 16384 + ((r >> 3) * 32 + c) * 32 + (r & 7) * 4; }

// The windowed form, which adds to nothing and turns nothing, leaves by TMA in bf16: 32 columns of a thread's row, times `mul`, to chunk `chunk` on of its row in a
// sub-tile of 64. (us, through write_staged / so: 2 x 128 tokens, 2 / 1 heads 10.1 / 9.6; 4 x 4096, 16 / 8 heads, window 128 290 / 283.)
__device__ __forceinline__ void window_stage(uint32_t tacc, uint32_t sub, int r, int chunk, float mul) {
    uint32_t v[32];
    tmem_ld_32x32(tacc, v);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint32_t o[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) o[t] = pack_bf16(__uint_as_float(v[8 * k + 2 * t]) * mul, __uint_as_float(v[8 * k + 2 * t + 1]) * mul);
        st_shared_v4(sub + r * 128 + (((chunk + k) ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
    }
}
// The groups that fill a sub-tile, `threads` of them, wait for each other; one stores it. Rows behind the sequence's end are not written.
__device__ __forceinline__ void window_store(const CUtensorMap& tm, const uint8_t* sub, int barrier, int threads, bool first, bool ok, int x, int row, int b) {
    fence_proxy_async_smem();
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
    if (first && ok) {
        tma_store_3d(&tm, sub, x, row, b);
        tma_store_commit();
        tma_store_wait0();
    }
}

// Probabilities of one thread's 32 score columns, in place: exp2(s * scale_log2 - lse2). In the transposed form (dK / dV)
// a column is a query with its own lse2; in the other (dQ) the thread's row is the query. One half (16 columns) per call.
template <bool kDiag, int kHalf>
__device__ __forceinline__ void prob_cols(uint32_t (&v)[32], const float4 (&ls)[4], float scale_log2, int r, int qb) {
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
        const float l[4] = {ls[e4].x, ls[e4].y, ls[e4].z, ls[e4].w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int e = kHalf * 16 + e4 * 4 + t;
            float pv = fast_exp2(__uint_as_float(v[e]) * scale_log2 - l[t]);
            if constexpr (kDiag) {
                if (r > qb + e) pv = 0.f;  // key (row r) may not lie after the query (column)
            }
            v[e] = __float_as_uint(pv);
        }
    }
}
template <bool kDiag>
__device__ __forceinline__ void prob_rows(uint32_t (&v)[32], float lse2, float scale_log2, int r, int kb) {
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        float pv = fast_exp2(__uint_as_float(v[e]) * scale_log2 - lse2);
        if constexpr (kDiag) {
            if (kb + e > r) pv = 0.f;
        }
        v[e] = __float_as_uint(pv);
    }
}
// The windowed form's, a bit of `seen` a column where `hides`, arithmetic on pairs: of half kHalf with the columns' own statistics (negated), or
// of all with the row's.
template <int kHalf>
__device__ __forceinline__ void window_prob_cols(uint32_t (&v)[32], const float4 (&neg_ls)[4], float scale_log2, bool hides, uint32_t seen) {
    const uint64_t scale2 = pair_of(scale_log2, scale_log2);
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
        const float l[4] = {neg_ls[e4].x, neg_ls[e4].y, neg_ls[e4].z, neg_ls[e4].w};
#pragma unroll
        for (int t = 0; t < 4; t += 2) {
            const int e = kHalf * 16 + e4 * 4 + t;
            const float2 x = floats_of(fma2(pair_of(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), scale2, pair_of(l[t], l[t + 1])));
            v[e] = __float_as_uint(fast_exp2(x.x));
            v[e + 1] = __float_as_uint(fast_exp2(x.y));
        }
    }
    if (hides) {
#pragma unroll
        for (int e = kHalf * 16; e < kHalf * 16 + 16; ++e)
            if (!(seen & (1u << e))) v[e] = 0;
    }
}
__device__ __forceinline__ void window_prob_rows(uint32_t (&v)[32], float neg_lse2, float scale_log2, bool hides, uint32_t seen) {
    const uint64_t scale2 = pair_of(scale_log2, scale_log2), l2 = pair_of(neg_lse2, neg_lse2);
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
        const float2 x = floats_of(fma2(pair_of(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), scale2, l2));
        v[e] = __float_as_uint(fast_exp2(x.x));
        v[e + 1] = __float_as_uint(fast_exp2(x.y));
    }
    if (hides) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
            if (!(seen & (1u << e))) v[e] = 0;
    }
}
// Two of dS = P (dP - delta), in bf16.
__device__ __forceinline__ uint32_t window_ds(const uint32_t p0, const uint32_t p1, const uint32_t dp0, const uint32_t dp1, float neg_d0, float neg_d1) {
    const float2 x = floats_of(mul2(pair_of(__uint_as_float(p0), __uint_as_float(p1)),
                                    add2(pair_of(__uint_as_float(dp0), __uint_as_float(dp1)), pair_of(neg_d0, neg_d1))));
    return pack_bf16(x.x, x.y);
}

// D[128,hd] (+)= A[128,128](TMEM, bf16 pairs) * B[128,hd] with B MN-major in two 16 KiB sub-tiles; the A operand sits in
// four pieces of 16 columns, 32 columns apart (each where one warp group read its 32 fp32 columns from).
// kCut: only the first `keys` (a multiple of 16) of the inner dimension.
template <bool kCut = false>
__device__ __forceinline__ void issue_pv_g16(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accumulate, int keys = kAttnTile) {
#pragma unroll
    for (int k = 0; k < kAttnTile / 16; ++k)
        if (!kCut || k * 16 < keys) umma_f16_ts(d_tmem, a_tmem + (k >> 1) * 32 + (k & 1) * 8, b_desc + k * (2048 >> 4), idesc, (accumulate || k > 0) ? 1u : 0u);
}
// D[128,hd] (+)= A[128,128] * B[128,hd], both in shared memory: A K-major, B MN-major.
__device__ __forceinline__ void issue_pd_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
#pragma unroll
    for (int k = 0; k < kAttnTile / 16; ++k)
        umma_f16_ss(d_tmem, a_desc + (((k >> 2) * kAttnSub + (k & 3) * 32) >> 4), b_desc + k * (2048 >> 4), idesc,
                    (accumulate || k > 0) ? 1u : 0u);
}

// A tile of the packed activation or of dO: the windowed form has the sequences apart (rows past a sequence's end come as zeros).
template <bool kWindow>
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* tm, uint64_t* bar, int x, int b, int S, int row) {
    if constexpr (kWindow) {
        tma_load_3d(dst, tm, bar, x, row, b);
        tma_load_3d(static_cast<uint8_t*>(dst) + kAttnSub, tm, bar, x + 64, row, b);
    } else {
        tma_load_2d(dst, tm, bar, x, b * S + row);
        tma_load_2d(static_cast<uint8_t*>(dst) + kAttnSub, tm, bar, x + 64, b * S + row);
    }
}

// ---------------------------------------------------------------------------- dK / dV
// One CTA's work: number `lin` of the (kv tile, batch, head) triples; kWindow: of the parts of AttnWindowParts, those of the window first.
template <bool kWindow>
__device__ __forceinline__ void attn_dkdv(const CUtensorMap& tm_qkv, const CUtensorMap& tm_do, const CUtensorMap& tm_dqkv, const AttnBwdParams& p, uint8_t* smem, int lin) {
    uint8_t* sK = smem;
    uint8_t* sV = smem + kAttnTileBytes;
    uint8_t* sQ = smem + 2 * kAttnTileBytes;   // 2 stages
    uint8_t* sdO = smem + 4 * kAttnTileBytes;  // 2 stages
    uint8_t* sP = smem + 6 * kAttnTileBytes;   // P^T, the A operand of dV
    float* sStat = reinterpret_cast<float*>(smem + 7 * kAttnTileBytes);  // [16 warps][32] lse * log2e, later delta, of its columns
    uint64_t* bars = reinterpret_cast<uint64_t*>(sStat + kAttnComputeThreads);
    uint64_t* kv_full = bars;
    uint64_t* q_full = bars + 1;      // [2]
    uint64_t* q_empty = bars + 3;     // [2] dK has read the tile (S^T long before)
    uint64_t* do_full = bars + 5;     // [2]
    uint64_t* do_empty = bars + 7;    // [2] dV and dP^T have read the tile
    uint64_t* s_full = bars + 9;
    uint64_t* s_empty = bars + 10;    // the compute warps have the scores in registers
    uint64_t* dp_full = bars + 11;
    uint64_t* p_ready = bars + 12;
    uint64_t* p_free = bars + 13;     // dV has read P^T
    uint64_t* ds_ready = bars + 14;
    uint64_t* final_bar = bars + 15;  // both issuing warps' last MMAs
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // kv tile slowest, heaviest first; heads and batch fastest. Heads are kv groups (a CTA sweeps the group's query heads) or,
    // with split_heads, query heads
    const WindowPart part(p.win, p.cut, p.B, p.S, p.nh, p.nkv, kWindow ? lin : 0);
    const int heads = p.split_heads ? p.nh : p.nkv, heads_all = heads * p.B;
    const int j = kWindow ? part.j : lin / heads_all;  // kv tile
    const int ysel = (lin % heads_all) % heads, b = kWindow ? part.b : (lin % heads_all) / heads;
    const int rep = p.nh / p.nkv;
    const int g = kWindow ? part.g : p.split_heads ? ysel / rep : ysel;
    const int h_first = kWindow ? part.h_first : p.split_heads ? ysel : g * rep;
    const int turn = !kWindow && p.split_heads ? ysel - g * rep : 0;   // my place in the group's accumulation chain
    const int nq = p.S / kAttnTile;
    const int q_first = kWindow ? part.q_first : j;
    const int per_head = kWindow ? part.q_tiles : nq - j;          // query tiles at or below the diagonal
    const int iters = (kWindow ? part.heads : p.split_heads ? 1 : rep) * per_head;
    if (kWindow && per_head <= 0) {
        grid_dep_wait();
        return;
    }
    const int row_base = b * p.S;
    const int col_k = (p.nh + g) * kAttnHD, col_v = (p.nh + p.nkv + g) * kAttnHD;

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_qkv);
        tma_prefetch_desc(&tm_do);
        mbar_init(kv_full, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], 1);
            mbar_init(&do_full[i], 1);
            mbar_init(&do_empty[i], 2);
        }
        mbar_init(s_full, 1);
        mbar_init(s_empty, kAttnComputeThreads / 32);
        mbar_init(dp_full, 1);
        mbar_init(p_ready, kAttnComputeThreads / 32);
        mbar_init(p_free, 1);
        mbar_init(ds_ready, kAttnComputeThreads / 32);
        mbar_init(final_bar, 2);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dep_wait();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tS = tmem_base, tdP = tmem_base + 128, tdV = tmem_base + 256, tdK = tmem_base + 384;

    if (warp == 0) {
        if (lane == 0) {
            mbar_expect_tx(kv_full, 2 * kAttnTileBytes);
            load_tile<kWindow>(sK, &tm_qkv, kv_full, col_k, b, p.S, j * kAttnTile);
            load_tile<kWindow>(sV, &tm_qkv, kv_full, col_v, b, p.S, j * kAttnTile);
            bool ok = true;
            for (int it = 0; it < iters && ok; ++it) {
                const int slot = it & 1;
                const uint32_t ph = (it >> 1) & 1;
                const int h = h_first + it / per_head;
                const int q_row = (q_first + it % per_head) * kAttnTile;
                if (!mbar_wait(&q_empty[slot], ph ^ 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                mbar_expect_tx(&q_full[slot], kAttnTileBytes);
                load_tile<kWindow>(sQ + slot * kAttnTileBytes, &tm_qkv, &q_full[slot], h * kAttnHD, b, p.S, q_row);
                if (!mbar_wait(&do_empty[slot], ph ^ 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                mbar_expect_tx(&do_full[slot], kAttnTileBytes);
                load_tile<kWindow>(sdO + slot * kAttnTileBytes, &tm_do, &do_full[slot], h * kAttnHD, b, p.S, q_row);
            }
            grid_dep_launch();
            if (!ok)
                for (int i = 0; i < 32; ++i) __nanosleep(50000);
        }
    } else if (warp == 1) {
        // ---------------- S^T = K Q^T, a step ahead of the compute warps; dV += P^T dO. The whole warp walks the loop
        // (descriptors in uniform registers).
        const uint32_t idesc_kk = umma_idesc_bf16(128, 128, 0, 0), idesc_mn = umma_idesc_bf16(128, 128, 0, 1);
        const uint64_t kd = umma_smem_desc_sw128(smem_u32(sK), 0, 1024), qd = umma_smem_desc_sw128(smem_u32(sQ), 0, 1024);
        const uint64_t pd = umma_smem_desc_sw128(smem_u32(sP), 0, 1024), dod = umma_smem_desc_sw128(smem_u32(sdO), kAttnSub, 1024);
        const bool leader = elect_one();
        bool ok = mbar_wait_warp(kv_full, 0, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
        for (int it = 0; it <= iters && ok; ++it) {
            if (it < iters) {
                const int slot = it & 1;
                if (!mbar_wait_warp(s_empty, (it & 1) ^ 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN) ||
                    !mbar_wait_warp(&q_full[slot], (it >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                tc_fence_after();
                if (leader) {
                    issue_kk(tS, kd, qd + slot * kTileDesc, idesc_kk);
                    umma_commit(s_full);
                }
            }
            if (it > 0) {
                const int slot = (it - 1) & 1;
                if (!mbar_wait_warp(&do_full[slot], ((it - 1) >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN) ||
                    !mbar_wait_warp(p_ready, (it - 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                tc_fence_after();
                if (leader) {
                    issue_pd_ss(tdV, pd, dod + slot * kTileDesc, idesc_mn, it > 1);
                    umma_commit(p_free);
                    umma_commit(&do_empty[slot]);
                    if (it == iters) umma_commit(final_bar);
                }
            }
        }
    } else if (warp == 2) {
        // ---------------- dP^T = V dO^T, dK += dS^T Q (unscaled). dK(i) comes after S^T(i), which the compute warps saw before
        // they gave dS^T(i): the commit that frees Q(i) covers both its readers.
        const uint32_t idesc_kk = umma_idesc_bf16(128, 128, 0, 0), idesc_mn = umma_idesc_bf16(128, 128, 0, 1);
        const uint64_t vd = umma_smem_desc_sw128(smem_u32(sV), 0, 1024), dod = umma_smem_desc_sw128(smem_u32(sdO), 0, 1024);
        const uint64_t qd = umma_smem_desc_sw128(smem_u32(sQ), kAttnSub, 1024);
        const bool leader = elect_one();
        bool ok = mbar_wait_warp(kv_full, 0, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
        for (int it = 0; it <= iters && ok; ++it) {
            if (it > 0) {
                const int slot = (it - 1) & 1;
                if (!mbar_wait_warp(&q_full[slot], ((it - 1) >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN) ||
                    !mbar_wait_warp(ds_ready, (it - 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                tc_fence_after();
                if (leader) {
                    issue_pv_g16(tdK, tdP, qd + slot * kTileDesc, idesc_mn, it > 1);
                    umma_commit(&q_empty[slot]);
                    if (it == iters) umma_commit(final_bar);
                }
            }
            if (it < iters) {
                const int slot = it & 1;
                if (!mbar_wait_warp(&do_full[slot], (it >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                tc_fence_after();
                if (leader) {
                    issue_kk(tdP, vd, dod + slot * kTileDesc, idesc_kk);
                    umma_commit(dp_full);
                    umma_commit(&do_empty[slot]);
                }
            }
        }
    } else if (warp >= 4) {
        const int r = (warp & 3) * 32 + lane;  // kv row inside the tile == TMEM lane
        const int grp = (warp - 4) >> 2;       // which 32 of the step's 128 query columns
        const uint32_t lane_bits = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const int qb = grp * 32;               // first of this warp's 32 query columns
        const uint32_t tSg = tS + lane_bits + qb, tdPg = tdP + lane_bits + qb;
        float* stat = sStat + (warp - 4) * 32;
        // P^T row r, its 16-byte chunk c (8 queries) at chunk c ^ (r & 7) of the 128-byte row, 64 queries per sub-tile
        const uint32_t prow = smem_u32(sP) + (grp >> 1) * kAttnSub + r * 128;
        const uint32_t pchunk = (grp & 1) * 4, psw = r & 7;
        bool ok = true;
        // statistics of this warp's queries (a lane holds one), fetched a step ahead; shared through the warp's own 32 words
        // (past the sequence's end there is none: a probability of exp2(-inf) = 0)
        auto stat_at = [&](const float* v, int it, float none) {
            const int h = h_first + it / per_head;
            const int i = q_first + it % per_head;
            if (kWindow && i * kAttnTile + qb + lane >= p.S) return none;
            return v[(static_cast<long long>(b) * p.nh + h) * p.S + i * kAttnTile + qb + lane];
        };
        float lse_next = stat_at(p.lse, 0, INFINITY), delta_next = stat_at(p.delta, 0, 0.f);
#pragma unroll 1
        for (int it = 0; it < iters; ++it) {
            const int i = q_first + it % per_head;
            const bool diag = kWindow ? window_masks(p.win, i, j) : it % per_head == 0;
            // kWindow: the 32 columns this thread's key is seen by, a bit each: from its own query on, to the window's end or, as a sink, without one
            uint32_t seen = ~0u;
            if (kWindow && diag) {
                const int from = (j - i) * kAttnTile + r - qb;
                seen = ~bits_below(from) & (j * kAttnTile + r < p.win.sinks ? ~0u : bits_below(from + p.win.window));
            }
            // Of a tile at either end of the window six of sixteen warps see nothing, of a sinks' tile behind it all but four for each 32 sinks begun: zeros, for no
            // exponentials.
            const bool none = kWindow && diag && !__any_sync(0xffffffffu, seen);
            const float delta = delta_next;
            if (!mbar_wait_warp(s_full, it & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
            tc_fence_after();
            uint32_t pr[32];
            if (none) {
#pragma unroll
                for (int e = 0; e < 32; ++e) pr[e] = 0;
            } else {
                tmem_ld_32x32(tSg, pr);
            }
            __syncwarp();
            stat[lane] = lse_next * (kWindow ? -1.4426950408889634f : 1.4426950408889634f);
            if (it + 1 < iters) {
                lse_next = stat_at(p.lse, it + 1, INFINITY);
                delta_next = stat_at(p.delta, it + 1, 0.f);
            }
            __syncwarp();
            float4 ls[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) ls[e] = reinterpret_cast<const float4*>(stat)[e];
            tmem_ld_wait();
            tc_fence_before();
            mbar_arrive_warp(s_empty);
            if constexpr (kWindow) { if (!none) window_prob_cols<0>(pr, ls, p.scale_log2, diag, seen); }
            else if (diag) prob_cols<true, 0>(pr, ls, p.scale_log2, r, qb);
            else prob_cols<false, 0>(pr, ls, p.scale_log2, r, qb);
#pragma unroll
            for (int e = 0; e < 4; ++e) ls[e] = reinterpret_cast<const float4*>(stat)[4 + e];
            if constexpr (kWindow) { if (!none) window_prob_cols<1>(pr, ls, p.scale_log2, diag, seen); }
            else if (diag) prob_cols<true, 1>(pr, ls, p.scale_log2, r, qb);
            else prob_cols<false, 1>(pr, ls, p.scale_log2, r, qb);
            __syncwarp();
            stat[lane] = kWindow ? -delta : delta;
            if (it > 0 && !mbar_wait_warp(p_free, (it - 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
            auto give_p = [&]() {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t o[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        o[t] = pack_bf16(__uint_as_float(pr[c * 8 + 2 * t]), __uint_as_float(pr[c * 8 + 2 * t + 1]));
                    st_shared_v4(prow + (((pchunk + c) ^ psw) << 4), o[0], o[1], o[2], o[3]);
                }
                fence_proxy_async_smem();
                mbar_arrive_warp(p_ready);
            };
            give_p();
            if (!mbar_wait_warp(dp_full, it & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
            tc_fence_after();
            uint32_t dp[32];
            uint32_t dk[16];
            if (none) {
#pragma unroll
                for (int e = 0; e < 16; ++e) dk[e] = 0;
            } else {
                tmem_ld_32x32(tdPg, dp);
                tmem_ld_wait();
#pragma unroll
                for (int e4 = 0; e4 < 8; ++e4) {
                    const float4 d = reinterpret_cast<const float4*>(stat)[e4];
                    const int e = e4 * 4;
                    if constexpr (kWindow) {
                        dk[e4 * 2] = window_ds(pr[e], pr[e + 1], dp[e], dp[e + 1], d.x, d.y);
                        dk[e4 * 2 + 1] = window_ds(pr[e + 2], pr[e + 3], dp[e + 2], dp[e + 3], d.z, d.w);
                        continue;
                    }
                    dk[e4 * 2] = pack_bf16(__uint_as_float(pr[e]) * (__uint_as_float(dp[e]) - d.x),
                                           __uint_as_float(pr[e + 1]) * (__uint_as_float(dp[e + 1]) - d.y));
                    dk[e4 * 2 + 1] = pack_bf16(__uint_as_float(pr[e + 2]) * (__uint_as_float(dp[e + 2]) - d.z),
                                               __uint_as_float(pr[e + 3]) * (__uint_as_float(dp[e + 3]) - d.w));
                }
            }
            tmem_st_32x16(tdPg, dk);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive_warp(ds_ready);
        }
        // every MMA of the tile is done, and with it every read of shared memory; groups 0, 1 stage dK, 2, 3 dV. A warp that gave up comes to the
        // barriers all the same.
        ok = ok && mbar_wait_warp(final_bar, 0, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
        const uint32_t stage = smem_u32(smem);
        if (ok) tc_fence_after();
        if (kWindow && part.slot < 0) {
            uint8_t* sub = smem + grp * kAttnSub;      // 64 columns of dK or dV
            const uint32_t acc = (grp < 2 ? tdK : tdV) + lane_bits + (grp & 1) * 64;
            if (ok) {
                window_stage(acc, smem_u32(sub), r, 0, grp < 2 ? p.scale : 1.f);
                window_stage(acc + 32, smem_u32(sub), r, 4, grp < 2 ? p.scale : 1.f);
            }
            window_store(tm_dqkv, sub, 1 + grp, 128, (threadIdx.x & 127) == 0, ok, (grp < 2 ? col_k : col_v) + (grp & 1) * 64, j * kAttnTile, b);
        } else if constexpr (kWindow) {
            // A part leaves its sums in fp32, of a sinks' tile behind the window the sinks' rows; the kernel behind this one adds the parts up.
            // (A whole warp reads tensor memory, whichever of its rows leave.)
            const int rows = lin < p.cut.near_ctas ? kAttnTile : p.win.sinks - j * kAttnTile;
            if (ok && (r & ~31) < rows) {
                float* to = p.partial + part.slot * 32768ll + window_part_at(grp >> 1, r, (grp & 1) * 16);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t v[32];
                    tmem_ld_32x32((grp < 2 ? tdK : tdV) + lane_bits + (grp & 1) * 64 + c * 32, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (r < rows) *reinterpret_cast<uint4*>(to + (c * 8 + k) * 32) = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                }
            }
        } else {
            if (ok) {
                const int c0 = (grp & 1) * 2;
                stage_acc_chunk((grp < 2 ? tdK : tdV) + lane_bits, stage + (grp >> 1) * 65536, r, c0);
                stage_acc_chunk((grp < 2 ? tdK : tdV) + lane_bits, stage + (grp >> 1) * 65536, r, c0 + 1);
            }
            bar_sync_compute();
        }
        if constexpr (!kWindow) {
            const long long ld = static_cast<long long>(p.nh + 2 * p.nkv) * kAttnHD;
            __nv_bfloat16* row0 = p.dqkv + (static_cast<long long>(row_base) + j * kAttnTile) * ld;
            __nv_bfloat16* const dst[2] = {row0 + col_k, row0 + col_v};
            const float mul[2] = {p.scale, 1.f};
            const int first = threadIdx.x - 128;
            unsigned int* cnt = p.split_heads ? p.chain + (static_cast<long long>(b) * p.nkv + g) * nq + j : nullptr;
            if (turn > 0 && ok) {
                // heads of the group add in turn: wait (bounded) until the heads before me are done
                ok = false;
                for (uint32_t spin = 0; spin < kSpinLimit && !ok; ++spin) {
                    unsigned int v;
                    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(cnt) : "memory");
                    ok = v >= static_cast<unsigned int>(turn);
                    if (!ok && spin > 16) __nanosleep(200);
                }
                if (!ok) atomicCAS(p.status, 0, CAI_DEV_TIMEOUT_ATTN);
            }
            if (ok) {
                // the last of the heads turns the finished sum
                const float2* rope = p.rope && (!p.split_heads || turn + 1 == rep) ? p.rope + static_cast<long long>(j) * kAttnTile * 64 : nullptr;
                if (turn == 0) write_staged<false, 4>(stage, dst, mul, ld, first, rope);
                else write_staged<true, 4>(stage, dst, mul, ld, first, rope);
            }
            if (p.split_heads) {
                __threadfence();
                bar_sync_compute();
                if (threadIdx.x == 128) {   // first compute thread: everyone's rows are written and fenced
                    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(cnt), "r"(static_cast<unsigned int>(turn + 1)) : "memory");
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// ---------------------------------------------------------------------------- dQ
template <bool kWindow>
__device__ __forceinline__ void attn_dq(const CUtensorMap& tm_qkv, const CUtensorMap& tm_do, const CUtensorMap& tm_dqkv, const AttnBwdParams& p, uint8_t* smem, int lin) {
    uint8_t* sQ = smem;
    uint8_t* sdO = smem + kAttnTileBytes;
    uint8_t* sK = smem + 2 * kAttnTileBytes;  // 3 stages: S runs a step ahead of the dQ that still needs the tile
    uint8_t* sV = smem + 5 * kAttnTileBytes;  // 2 stages
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 7 * kAttnTileBytes);
    uint64_t* q_full = bars;
    uint64_t* k_full = bars + 1;     // [3]
    uint64_t* k_empty = bars + 4;    // [3] dQ has read the tile
    uint64_t* v_full = bars + 7;     // [2]
    uint64_t* v_empty = bars + 9;    // [2]
    uint64_t* s_full = bars + 11;    // [2]
    uint64_t* s_empty = bars + 13;   // [2] the compute warps have read the scores
    uint64_t* dp_full = bars + 15;
    uint64_t* ds_ready = bars + 16;
    uint64_t* final_bar = bars + 17;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads_all = p.nh * p.B;
    const int i = (p.S + kAttnTile - 1) / kAttnTile - 1 - lin / heads_all;  // q tile, heaviest first across all heads
    const int h = (lin % heads_all) % p.nh, b = (lin % heads_all) / p.nh;
    const int g = h / (p.nh / p.nkv);
    const WindowKeys keys(p.win, i);
    const int n = kWindow ? keys.n : i + 1;
    const int row_base = b * p.S;
    const int col_q = h * kAttnHD, col_k = (p.nh + g) * kAttnHD, col_v = (p.nh + p.nkv + g) * kAttnHD;

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_qkv);
        tma_prefetch_desc(&tm_do);
        mbar_init(q_full, 1);
        for (int k = 0; k < 3; ++k) {
            mbar_init(&k_full[k], 1);
            mbar_init(&k_empty[k], 1);
        }
        for (int k = 0; k < 2; ++k) {
            mbar_init(&v_full[k], 1);
            mbar_init(&v_empty[k], 1);
            mbar_init(&s_full[k], 1);
            mbar_init(&s_empty[k], kAttnComputeThreads / 32);
        }
        mbar_init(dp_full, 1);
        mbar_init(ds_ready, kAttnComputeThreads / 32);
        mbar_init(final_bar, 1);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dep_wait();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tS = tmem_base, tdP = tmem_base + 256, tdQ = tmem_base + 384;   // two score buffers

    if (warp == 0) {
        if (lane == 0) {
            mbar_expect_tx(q_full, 2 * kAttnTileBytes);
            load_tile<kWindow>(sQ, &tm_qkv, q_full, col_q, b, p.S, i * kAttnTile);
            load_tile<kWindow>(sdO, &tm_do, q_full, col_q, b, p.S, i * kAttnTile);
            bool ok = true;
            int ks = 0;
            uint32_t kph = 0;
            for (int j = 0; j < n && ok; ++j) {
                const int slot = j & 1;
                const uint32_t ph = (j >> 1) & 1;
                const int kv_row = (kWindow ? keys.tile(j) : j) * kAttnTile;
                if (!mbar_wait(&k_empty[ks], kph ^ 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                mbar_expect_tx(&k_full[ks], kAttnTileBytes);
                load_tile<kWindow>(sK + ks * kAttnTileBytes, &tm_qkv, &k_full[ks], col_k, b, p.S, kv_row);
                if (!mbar_wait(&v_empty[slot], ph ^ 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                mbar_expect_tx(&v_full[slot], kAttnTileBytes);
                load_tile<kWindow>(sV + slot * kAttnTileBytes, &tm_qkv, &v_full[slot], col_v, b, p.S, kv_row);
                if (++ks == 3) {
                    ks = 0;
                    kph ^= 1;
                }
            }
            grid_dep_launch();
            if (!ok)
                for (int k = 0; k < 32; ++k) __nanosleep(50000);
        }
    } else if (warp == 1) {
        // ---------------- S = Q K^T, up to two steps ahead of the compute warps (kWindow: sinks' tiles as wide as there are sinks, all three products)
        const uint32_t idesc_kk = umma_idesc_bf16(128, 128, 0, 0);
        const uint64_t qd = umma_smem_desc_sw128(smem_u32(sQ), 0, 1024), kd = umma_smem_desc_sw128(smem_u32(sK), 0, 1024);
        const bool leader = elect_one();
        bool ok = mbar_wait_warp(q_full, 0, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
        int ks = 0;
        uint32_t kph = 0;
        for (int j = 0; j < n && ok; ++j) {
            const int buf = j & 1;
            if (!mbar_wait_warp(&k_full[ks], kph, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN) ||
                !mbar_wait_warp(&s_empty[buf], ((j >> 1) & 1) ^ 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
            tc_fence_after();
            if (leader) {
                issue_kk(tS + buf * 128, qd, kd + ks * kTileDesc, kWindow ? umma_idesc_bf16(128, keys.width(p.win, j), 0, 0) : idesc_kk);
                umma_commit(&s_full[buf]);
            }
            if (++ks == 3) {
                ks = 0;
                kph ^= 1;
            }
        }
    } else if (warp == 2) {
        // ---------------- dP = dO V^T, dQ += dS K (unscaled). Ordered behind S(j) by ds_ready(j), which the compute warps
        // give after they have seen S(j): the commit that frees K(j) therefore covers both its readers.
        const uint32_t idesc_kk = umma_idesc_bf16(128, 128, 0, 0), idesc_mn = umma_idesc_bf16(128, 128, 0, 1);
        const uint64_t dod = umma_smem_desc_sw128(smem_u32(sdO), 0, 1024), vd = umma_smem_desc_sw128(smem_u32(sV), 0, 1024);
        const uint64_t kd = umma_smem_desc_sw128(smem_u32(sK), kAttnSub, 1024);
        const bool leader = elect_one();
        bool ok = mbar_wait_warp(q_full, 0, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
        int ks = 0;            // ring slot and phase of the K tile of step j - 1
        uint32_t kph = 0;
        for (int j = 0; j <= n && ok; ++j) {
            const int slot = j & 1;
            if (j > 0) {
                if (!mbar_wait_warp(&k_full[ks], kph, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN) ||
                    !mbar_wait_warp(ds_ready, (j - 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                tc_fence_after();
                if (leader) {
                    issue_pv_g16<kWindow>(tdQ, tdP, kd + ks * kTileDesc, idesc_mn, j > 1, kWindow ? keys.width(p.win, j - 1) : kAttnTile);
                    umma_commit(&k_empty[ks]);
                    if (j == n) umma_commit(final_bar);
                }
                if (++ks == 3) {
                    ks = 0;
                    kph ^= 1;
                }
            }
            if (j < n) {
                if (!mbar_wait_warp(&v_full[slot], (j >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                tc_fence_after();
                if (leader) {
                    issue_kk(tdP, dod, vd + slot * kTileDesc, kWindow ? umma_idesc_bf16(128, keys.width(p.win, j), 0, 0) : idesc_kk);
                    umma_commit(dp_full);
                    umma_commit(&v_empty[slot]);
                }
            }
        }
    } else if (warp >= 4) {
        const int r = (warp & 3) * 32 + lane;  // q row inside the tile
        const int grp = (warp - 4) >> 2;       // which 32 of the step's 128 key columns
        const uint32_t lane_bits = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const long long vec = (static_cast<long long>(b) * p.nh + h) * p.S + i * kAttnTile + r;
        const bool there = !kWindow || i * kAttnTile + r < p.S;
        const float lse2 = there ? p.lse[vec] * 1.4426950408889634f : INFINITY;
        const float dl = there ? p.delta[vec] : 0.f;
        const int kb = grp * 32;   // first of this warp's 32 key columns
        const uint32_t tdPg = tdP + lane_bits + kb;
        bool ok = true;
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            const int buf = j & 1;
            // kWindow: the 32 columns this thread's query sees, a bit each: up to its own key, of the window or the sinks. (Past a sinks' tile's width the columns hold
            // anything; they are not seen, and dQ does not read what becomes of them.)
            const int kt = kWindow ? keys.tile(j) : j;
            const bool hides = kWindow && window_masks(p.win, i, kt);
            uint32_t seen = ~0u;
            if (hides) {
                const int last = (i - kt) * kAttnTile + r - kb;
                seen = bits_below(last + 1) & (~bits_below(last + 1 - p.win.window) | bits_below(p.win.sinks - kt * kAttnTile - kb));
            }
            const bool none = hides && !__any_sync(0xffffffffu, seen);
            if (!mbar_wait_warp(&s_full[buf], (j >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
            tc_fence_after();
            if (none) {
                mbar_arrive_warp(&s_empty[buf]);
                if (!mbar_wait_warp(dp_full, j & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                tc_fence_after();
                uint32_t zero[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) zero[e] = 0;
                tmem_st_32x16(tdPg, zero);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive_warp(ds_ready);
                continue;
            }
            uint32_t pr[32];
            tmem_ld_32x32(tS + buf * 128 + lane_bits + kb, pr);
            tmem_ld_wait();
            tc_fence_before();
            mbar_arrive_warp(&s_empty[buf]);
            if constexpr (kWindow) {
                window_prob_rows(pr, -lse2, p.scale_log2, hides, seen);
            } else {
                if (j == i) prob_rows<true>(pr, lse2, p.scale_log2, r, kb);
                else prob_rows<false>(pr, lse2, p.scale_log2, r, kb);
            }
            if (!mbar_wait_warp(dp_full, j & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
            tc_fence_after();
            uint32_t dp[32], dk[16];
            tmem_ld_32x32(tdPg, dp);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 2)
                if constexpr (kWindow) dk[e >> 1] = window_ds(pr[e], pr[e + 1], dp[e], dp[e + 1], -dl, -dl);
                else dk[e >> 1] = pack_bf16(__uint_as_float(pr[e]) * (__uint_as_float(dp[e]) - dl),
                                       __uint_as_float(pr[e + 1]) * (__uint_as_float(dp[e + 1]) - dl));
            tmem_st_32x16(tdPg, dk);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive_warp(ds_ready);
        }
        ok = ok && mbar_wait_warp(final_bar, 0, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
        const uint32_t stage = smem_u32(smem);
        if (ok) tc_fence_after();
        if constexpr (kWindow) {
            uint8_t* sub = smem + (grp >> 1) * kAttnSub;
            if (ok) window_stage(tdQ + lane_bits + kb, smem_u32(sub), r, (grp & 1) * 4, p.scale);
            window_store(tm_dqkv, sub, 1 + (grp >> 1), 256, (threadIdx.x & 255) == 128, ok, col_q + (grp >> 1) * 64, i * kAttnTile, b);
        } else {
            if (ok) stage_acc_chunk(tdQ + lane_bits, stage, r, grp);
            bar_sync_compute();
            if (ok) {
                const long long ld = static_cast<long long>(p.nh + 2 * p.nkv) * kAttnHD;
                __nv_bfloat16* dst0 = p.dqkv + (static_cast<long long>(row_base) + i * kAttnTile) * ld + col_q;
                __nv_bfloat16* const dst[2] = {dst0, nullptr};
                const float mul[2] = {p.scale, 0.f};
                write_staged<false, 2>(stage, dst, mul, ld, threadIdx.x - 128, p.rope ? p.rope + static_cast<long long>(i) * kAttnTile * 64 : nullptr);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// ---------------------------------------------------------------------------- both
// The first `dkdv_ctas` CTAs work on dK / dV, the others on dQ: the two need the same set-up, shared memory and registers, and neither reads
// what the other writes. As launches of their own each ended in a wave that leaves SMs idle, and a dK / dV part of few kv heads leaves
// them idle throughout; together the light CTAs of one fill up behind the heavy ones of the other. Forward, backward and both rotary embeddings, two
// launches and one: 8 x 384 tokens, 12 / 4 heads (96 and 288 CTAs) 73.9 -> 65.4 us; 7 x 256, 4 / 2 heads 45.3 -> 41.9; 3 x 2432, 32 / 8 heads
// 854 -> 837; 8192 tokens, 32 / 8 heads 2504 -> 2466. A chain of split heads (AttnBwdParams) waits only for CTAs of lower number, and dQ's CTAs wait
// for nobody: they leave their SMs to whatever part of the chain is not there yet.
template <bool kWindow>
__global__ void __launch_bounds__(kAttnBwdThreads, 1)
attn_bwd_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_do, const __grid_constant__ CUtensorMap tm_dqkv,
                const AttnBwdParams p, const int dkdv_ctas) {
    // no room to round the base up: tiles start on swizzle boundaries only if the shared window does (checked)
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023) {
        grid_dep_wait();
        if (threadIdx.x == 0) atomicCAS(p.status, 0, CAI_DEV_BAD_ARG);
        return;
    }
    const int cta = static_cast<int>(blockIdx.x);
    if (cta < dkdv_ctas) attn_dkdv<kWindow>(tm_qkv, tm_do, tm_dqkv, p, smem, cta);
    else attn_dq<kWindow>(tm_qkv, tm_do, tm_dqkv, p, smem, cta - dkdv_ctas);
}

constexpr int kAttnBwdSmem = 7 * kAttnTileBytes + 2048 + 256;
template <bool kWindow>
int configure_bwd(int dev) {
    static bool configured[64] = {};
    if (!configured[dev & 63]) {
        if (cudaFuncSetAttribute(attn_bwd_kernel<kWindow>, cudaFuncAttributeMaxDynamicSharedMemorySize, kAttnBwdSmem) != cudaSuccess) {
            set_last_error("cudaFuncSetAttribute(attn_bwd) failed");
            return CAI_K_CUDA;
        }
        configured[dev & 63] = true;
    }
    return CAI_K_OK;
}

// ---------------------------------------------------------------------------- the windowed form's row sums
// sum_d dO O has the rounding of O in it, and dS = P (dP - delta) is a difference: where a query sees few keys, what O was rounded by counts for more than what dS is. In
// roundings of the result, 1.41 being P's or dS's and the result's own, dq of a sequence's rows 0-5 was off by 1.8-2.1, of rows 6-15 by 1.6, of rows 32 on by 1.45-1.5.
// So delta of such rows is sum_j P dP, which it stands for, in fp32: of the first kFewRows of every sequence, and of all where the window and the sinks are no more than kFewKeys keys.
// dq is off by 1.3-1.5 then, wherever the row lies. A warp takes sixteen queries of a head and eight keys at a time, with the warp's own matrix instruction (a tile of
// 128 x 128 would be seen to an eighth and less). The order of the head's dimension inside a product is free: a lane takes eight of them in a row, of queries and of keys.
// In small grids the four warps of a CTA share the keys of one piece (`ways`): the time is one warp's chain of loads and exponentials (96 tokens, 8 / 2 heads, all rows so: 12.1 us a
// backward, one way 16.0; all rows so and from O alone, 4 x 4096, 16 / 8 heads, window 8 239 / 216, 3 x 1000, 9 / 3 heads, window 20 33.4 / 30.4, four ways 37.8). The other rows' sums are CTAs of the same launch, so that the chain is hidden behind their bytes: with the first 32 rows so, and from O alone, us
// of a backward: 2 x 128 tokens, 2 / 1 heads 10.1 / 9.7, 333, 8 / 1 heads 14.8 / 14.4, 8 x 128, 8 / 2 heads 14.7 / 14.2, 16 x 256, 16 / 4 heads 48.5 / 47.2, 4 x 4096, 16 / 8 heads
// the same within its noise of 1 %. With the first 96 rows so 17.4, 18.5 and 54 for the second to fourth. Three CTAs an SM: four of 128 registers spill (333 tokens: 16.4).
constexpr int kFewKeys = 24, kFewRows = 32;      // kFewRows: those that see up to kFewKeys, in whole pieces of sixteen
__device__ __forceinline__ void mma_16x8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The other rows', from O: those from `first` on of each sequence, walked as one array, eight times kUnroll of them a CTA. Sixteen lanes a row as in attn_delta_kernel; a warp
// that has eight pairs of rows adds them up together: a lane gives half of its sums away at each of the first steps.
template <int kUnroll>
__device__ __forceinline__ void window_row_sums_of_out(const __nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ dout, float* __restrict__ delta, int B, int S,
                                                       int nh, int first, unsigned cta) {
    const unsigned each = static_cast<unsigned>(S - first) * nh, total = each * B, skip = static_cast<unsigned>(first) * nh;
    const unsigned w0 = cta * (8u * kUnroll) + (threadIdx.x >> 4);
    const int sub = threadIdx.x & 15;
    uint4 a[kUnroll], d[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const unsigned w = w0 + 8u * i;
        a[i] = d[i] = make_uint4(0, 0, 0, 0);
        if (w < total) {
            const size_t off = static_cast<size_t>(w + (w / each + 1) * skip) * kAttnHD + sub * 8;
            a[i] = *reinterpret_cast<const uint4*>(out + off);
            d[i] = *reinterpret_cast<const uint4*>(dout + off);
        }
    }
    float s[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        uint64_t s2 = 0;
        const uint32_t x[4] = {a[i].x, a[i].y, a[i].z, a[i].w}, y[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) s2 = fma2(pair_of(bf16_lo(x[k]), bf16_hi(x[k])), pair_of(bf16_lo(y[k]), bf16_hi(y[k])), s2);
        const float2 v = floats_of(s2);
        s[i] = v.x + v.y;
    }
    // the lane's row of the kUnroll: bit by bit, as it gives the others away
    unsigned mine = 0;
    int o = 8;
#pragma unroll
    for (int half = kUnroll / 2; half > 0; half /= 2, o >>= 1) {
        const bool up = sub & o;
        mine += up ? half : 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float keep = up ? s[i + half] : s[i], give = up ? s[i] : s[i + half];
            s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    const int rest = o;
#pragma unroll
    for (; o > 0; o >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
    const unsigned w = w0 + 8u * mine;
    if (!(sub & (2 * rest - 1)) && w < total) {
        const unsigned b = w / each, in = w - b * each, at = in / nh, h = in - at * nh;
        delta[(static_cast<size_t>(b) * nh + h) * S + first + at] = s[0];
    }
}
__global__ void __launch_bounds__(128, 3)
attn_window_row_sums_kernel(const __nv_bfloat16* __restrict__ qkv, long long ld, const __nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ dout,
                            const float* __restrict__ lse, float* __restrict__ delta, int B, int S, int nh, int nkv, float scale_log2, AttnWindow win, int exact,
                            int ways, unsigned exact_ctas, int unroll) {
    __shared__ float sums[4][16];
    grid_dep_begin();
    if (blockIdx.x >= exact_ctas) {
        if (unroll == 8) window_row_sums_of_out<8>(out, dout, delta, B, S, nh, exact, blockIdx.x - exact_ctas);
        else window_row_sums_of_out<2>(out, dout, delta, B, S, nh, exact, blockIdx.x - exact_ctas);
        return;
    }
    // heads fastest: those of a kv head read the same keys
    const int pieces = (exact + 15) / 16, lane = threadIdx.x & 31, row = lane >> 2, part = lane & 3;
    const int warp = threadIdx.x >> 5, mine = ways == 4 ? warp : 0;
    const unsigned item = ways == 4 ? blockIdx.x : blockIdx.x * 4 + warp;      // the rows of all heads fit 30 bits
    if (item >= static_cast<unsigned>(pieces) * nh * B) return;
    const unsigned piece = item / nh;
    const int h = item - piece * nh, b = piece / pieces, q0 = (piece - b * pieces) * 16, g = h / (nh / nkv);
    const long long first = static_cast<long long>(b) * S;
    const int reach = q0 - win.window + 1, near = (reach > 0 ? reach : 0) & ~7, last = q0 + 15 < S - 1 ? q0 + 15 : S - 1;
    const int sinks = win.sinks < near ? win.sinks : near;
    // eight keys at a time, of the sinks and from `near` on; the first of them are asked for with the queries
    uint4 kk[4], vv[4];
    auto fetch = [&](int k0) {
        const int at = k0 + row;
        const __nv_bfloat16* k = qkv + (first + at) * ld + (nh + g) * kAttnHD + part * 8;
        const __nv_bfloat16* v = k + nkv * kAttnHD;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            kk[c] = vv[c] = make_uint4(0, 0, 0, 0);
            if (at < S) {
                kk[c] = *reinterpret_cast<const uint4*>(k + c * 32);
                vv[c] = *reinterpret_cast<const uint4*>(v + c * 32);
            }
        }
    };
    const int step = ways * 8;
    auto behind = [&](int k0) {      // the keys after these
        const int k1 = k0 + step;
        return k0 < near && k1 >= sinks ? near + mine * 8 : k1;
    };
    int k0 = mine * 8 < sinks ? mine * 8 : near + mine * 8;
    if (k0 <= last) fetch(k0);
    uint4 q[2][4], d[2][4];
    float lse_at[2], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int at = q0 + row + u * 8;
        const bool there = at < S;
        lse_at[u] = there ? lse[(static_cast<long long>(b) * nh + h) * S + at] : INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            q[u][c] = d[u][c] = make_uint4(0, 0, 0, 0);
            if (there) {
                q[u][c] = *reinterpret_cast<const uint4*>(qkv + (first + at) * ld + h * kAttnHD + c * 32 + part * 8);
                d[u][c] = *reinterpret_cast<const uint4*>(dout + ((first + at) * nh + h) * kAttnHD + c * 32 + part * 8);
            }
        }
    }
    while (k0 <= last) {
        float s[4] = {}, dp[4] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            mma_16x8(s, q[0][c].x, q[1][c].x, q[0][c].y, q[1][c].y, kk[c].x, kk[c].y);
            mma_16x8(s, q[0][c].z, q[1][c].z, q[0][c].w, q[1][c].w, kk[c].z, kk[c].w);
            mma_16x8(dp, d[0][c].x, d[1][c].x, d[0][c].y, d[1][c].y, vv[c].x, vv[c].y);
            mma_16x8(dp, d[0][c].z, d[1][c].z, d[0][c].w, d[1][c].w, vv[c].z, vv[c].w);
        }
        const int now = k0;
        k0 = behind(k0);
        if (k0 <= last) fetch(k0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = q0 + row + (e >> 1) * 8, j = now + part * 2 + (e & 1);
            if (j <= i && (j > i - win.window || j < win.sinks))
                sum[e >> 1] += fast_exp2(s[e] * scale_log2 - lse_at[e >> 1] * 1.4426950408889634f) * dp[e];
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], 1);
        sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], 2);
    }
    float* to = delta + (static_cast<long long>(b) * nh + h) * S + q0;
    if (ways == 4) {
        if (part == 0) {
            sums[warp][row] = sum[0];
            sums[warp][row + 8] = sum[1];
        }
        __syncthreads();
        if (threadIdx.x < 16 && q0 + threadIdx.x < S)
            to[threadIdx.x] = sums[0][threadIdx.x] + sums[1][threadIdx.x] + sums[2][threadIdx.x] + sums[3][threadIdx.x];
    } else if (part == 0) {
        if (q0 + row < S) to[row] = sum[0];
        if (q0 + row + 8 < S) to[row + 8] = sum[1];
    }
}

// ---------------------------------------------------------------------------- the windowed form's parts
// A key tile's parts added up, in order, to its bf16 rows of dK (times the scale) and dV: those of the window first, head part by head part, then
// those of the query tiles behind it. A thread takes four columns of a row, a warp eight rows of sixteen: a line of 128 bytes for each part of four columns, a sector of
// 32 for each row it writes. (No shared memory: these CTAs wait beside those of the gradients, which have all of it.)
constexpr int kJoinCtas = 32;       // of a tile
__global__ void __launch_bounds__(256)
attn_window_join_kernel(const AttnBwdParams p) {
    grid_dep_begin();
    const int lin = blockIdx.x / kJoinCtas, item = blockIdx.x % kJoinCtas * 256 + threadIdx.x;
    const int heads_all = p.nkv * p.B, j = lin / heads_all, g = lin % heads_all % p.nkv, b = lin % heads_all / p.nkv;
    const int nq = (p.S + kAttnTile - 1) / kAttnTile, near_last = window_last_query_tile(p.win, j, nq);
    const int far = j < p.cut.sink_tiles ? nq - 1 - near_last : 0;      // query tiles behind the window
    if (p.cut.head_parts * p.cut.near_parts == 1 && far <= 0) return;
    const int which = item >> 12, r = ((item >> 8) & 15) * 8 + ((item >> 2) & 7), c = ((item >> 5) & 7) * 4 + (item & 3);
    if (j * kAttnTile + r >= p.S) return;
    const float* at = p.partial + window_part_at(which, r, c);
    const int stride = heads_all * p.cut.head_parts;     // slots of one key tile, of one far part
    const int mine = (b * p.nkv + g) * p.cut.head_parts;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    // The head parts of each of `pieces`, from slot `first` on, four loads in flight (more of them, or more code, are slower where the kernel is short).
    auto add = [&](long long first, int pieces) {
        const int n = pieces * p.cut.head_parts;
        const float* piece = at + first * 32768;
        int k = 0;
#pragma unroll 1
        for (int done = 0; done < n; done += 4) {
            float4 a[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                a[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (done + u < n) a[u] = *reinterpret_cast<const float4*>(piece + k * 32768);
                if (++k == p.cut.head_parts) {
                    k = 0;
                    piece += stride * 32768ll;
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                s.x += a[u].x; s.y += a[u].y; s.z += a[u].z; s.w += a[u].w;
            }
        }
    };
    const int near = (near_last - j) / p.cut.near_tiles + 1;
    add(static_cast<long long>(j) * p.cut.near_parts * stride + mine, near < p.cut.near_parts ? near : p.cut.near_parts);
    if (far > 0 && j * kAttnTile + r < p.win.sinks)
        add(p.cut.near_slots + static_cast<long long>(j) * p.cut.far_parts * stride + mine, (far + p.cut.far_tiles - 1) / p.cut.far_tiles);
    const float mul = which ? 1.f : p.scale;
    *reinterpret_cast<uint2*>(p.dqkv + (static_cast<long long>(b) * p.S + j * kAttnTile + r) * p.ldq + (which ? p.nh + p.nkv + g : p.nh + g) * kAttnHD + c * 4) =
        make_uint2(pack_bf16(s.x * mul, s.y * mul), pack_bf16(s.z * mul, s.w * mul));
}

// Whole numbers only, so that host and device agree on every size. Cutting is worth it where one CTA's steps would outlast everybody's share of all steps
// by more than the second kernel costs, which is that of two steps and a little for each part it reads: dK / dV of a step cost about 5 / 4 of dQ's. us of a
// backward, whole tiles or cut by heads / by heads and query tiles: 4000 tokens, 1 head 63 / 51, 2 x 1500, 8 / 1 heads, window 100 38 / 35, 2000, 4 / 4 36 /
// 33, 5 x 60, 24 / 3 22 / 18.
AttnWindowParts window_parts(const AttnWindow& w, int B, int S, int nh, int nkv, int sms) {
    AttnWindowParts c = {};
    const int nq = (S + kAttnTile - 1) / kAttnTile, rep = nh / nkv;
    const long long groups = static_cast<long long>(B) * nkv;
    const int near_most = window_last_query_tile(w, 0, nq) + 1, far_most = nq - near_most;
    const int sink_all = (w.sinks + kAttnTile - 1) / kAttnTile;
    while (c.sink_tiles < sink_all && window_last_query_tile(w, c.sink_tiles, nq) + 1 < nq) ++c.sink_tiles;
    long long steps = 0;     // of one head, in quarters of a dQ step
    for (int j = 0; j < nq; ++j) steps += 9ll * (j < c.sink_tiles ? nq - j : window_last_query_tile(w, j, nq) - j + 1);
    const long long share = steps * B * nh / sms;
    long long best = -1;
    for (int heads = 1; heads <= rep; ++heads)
        for (int near = 1; rep % heads == 0 && near <= near_most; near *= 2) {
            const int tiles = (near_most + near - 1) / near;
            const long long longest = 5ll * tiles * (rep / heads), slots = groups * nq * heads * near;
            const long long cost = (longest > share ? longest : share) + (heads * near > 1 ? (c.sink_tiles ? 0 : 8) + slots / 8 : 0);
            if (best >= 0 && cost >= best) continue;
            best = cost;
            c.head_parts = heads;
            c.near_tiles = tiles;
            c.near_parts = (near_most + tiles - 1) / tiles;
        }
    const long long heads_all = groups * c.head_parts;
    if (c.sink_tiles) {
        // no shorter than a window, and no more of them than about one a SM
        long long tiles = (far_most * c.sink_tiles * heads_all + sms - 1) / sms;
        tiles = tiles > near_most ? tiles : near_most;
        c.far_tiles = static_cast<int>(tiles < far_most ? tiles : far_most);
        c.far_parts = (far_most + c.far_tiles - 1) / c.far_tiles;
    }
    c.near_ctas = static_cast<int>(nq * heads_all * c.near_parts);
    c.far_ctas = static_cast<int>(c.sink_tiles * heads_all * c.far_parts);
    c.near_slots = static_cast<int>(c.head_parts * c.near_parts > 1 ? c.near_ctas : c.sink_tiles * heads_all);
    return c;
}

}  // namespace cai

using namespace cai;

CAI_API int cai_flash_attn_bwd(const void* qkv, const void* out, const void* dout, const float* lse, float* delta,
                               void* dqkv, int B, int S, int nh, int nkv, int hd, float scale, void* stream) {
    return cai_flash_attn_bwd_parts(qkv, out, dout, lse, delta, dqkv, B, S, nh, nkv, hd, scale, 7, stream);
}

CAI_API int cai_flash_attn_bwd_parts(const void* qkv, const void* out, const void* dout, const float* lse, float* delta,
                                     void* dqkv, int B, int S, int nh, int nkv, int hd, float scale, int parts, void* stream) {
    return cai_flash_attn_bwd_rope(qkv, out, dout, lse, delta, dqkv, nullptr, B, S, nh, nkv, hd, scale, parts, stream);
}

CAI_API int cai_flash_attn_bwd_rope(const void* qkv, const void* out, const void* dout, const float* lse, float* delta, void* dqkv,
                                    const float* table, int B, int S, int nh, int nkv, int hd, float scale, int parts, void* stream) {
    if (hd != kAttnHD || S % kAttnTile || nkv <= 0 || nh % nkv) {
        set_last_error("flash_attn_bwd: needs head_dim 128, seq %% 128 == 0, heads %% kv_heads == 0");
        return CAI_K_BAD_ARG;
    }
    if (B <= 0 || S <= 0) return CAI_K_OK;
    if (reinterpret_cast<uintptr_t>(table) & 15) {
        set_last_error("flash_attn_bwd: the rotary table must start on 16 bytes");
        return CAI_K_BAD_ARG;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long ld = static_cast<long long>(nh + 2 * nkv) * hd;
    const long long ldo = static_cast<long long>(nh) * hd;
    CUtensorMap tm_qkv, tm_do;
    if (!encode_tmap_2d(&tm_qkv, qkv, static_cast<uint64_t>(B) * S, ld, ld, 64, kAttnTile, 2)) return CAI_K_BAD_ARG;
    if (!encode_tmap_2d(&tm_do, dout, static_cast<uint64_t>(B) * S, ldo, ldo, 64, kAttnTile, 2)) return CAI_K_BAD_ARG;
    const int dev = current_device();
    if (configure_bwd<false>(dev)) return CAI_K_CUDA;
    AttnBwdParams p = {};
    p.B = B; p.S = S; p.nh = nh; p.nkv = nkv;
    p.scale = scale;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.lse = lse;
    p.delta = delta;
    p.dqkv = static_cast<__nv_bfloat16*>(dqkv);
    p.status = status_words(dev);
    const int nq = S / kAttnTile;
    // Few kv groups per GPU (tensor parallelism): one CTA per query head instead of per kv group shortens the
    // longest CTA by the group size; the heads of a group then add into dK / dV in turn (chain counters).
    p.split_heads = 0;
    p.chain = nullptr;
    p.rope = reinterpret_cast<const float2*>(table);
    const size_t need = static_cast<size_t>(B) * nkv * nq;
    if ((parts & 2) && nh > nkv && static_cast<long long>(nq) * nkv * B < sm_count(dev) &&
        static_cast<long long>(nq) * nh * B <= sm_count(dev) && need <= kAttnChainSlots) {
        // the counters live in a device array of the library: nothing is allocated on this path. The first call
        // on a device resolves the array's address (which may load the module), so it should come before any
        // stream capture; later calls only enqueue work.
        static unsigned int* chain_ptr[64] = {};
        if (!chain_ptr[dev & 63] &&
            cudaGetSymbolAddress(reinterpret_cast<void**>(&chain_ptr[dev & 63]), g_attn_chain) != cudaSuccess) {
            set_last_error("attn_bwd: cannot resolve the chain counters");
            return CAI_K_CUDA;
        }
        // the row sums' kernel clears the slots where it runs first (it has 8 threads for each row of a head, a slot is 128 rows)
        if (!(parts & 1) && cudaMemsetAsync(chain_ptr[dev & 63], 0, need * sizeof(unsigned int), st) != cudaSuccess) return CAI_K_CUDA;
        p.split_heads = 1;
        p.chain = chain_ptr[dev & 63];
    }
    const long long rows = static_cast<long long>(B) * S * nh;
    if (parts & 1) {
        constexpr unsigned per_cta = 16u * kDeltaUnroll;
        launch_early(attn_delta_kernel, static_cast<unsigned>((rows + per_cta - 1) / per_cta), 256, 0, st,
                     static_cast<const __nv_bfloat16*>(out), static_cast<const __nv_bfloat16*>(dout), delta, static_cast<unsigned>(rows),
                     static_cast<unsigned>(S), static_cast<unsigned>(nh), (reinterpret_cast<uintptr_t>(out) & 15) == 0, p.chain,
                     static_cast<unsigned>(p.split_heads ? need : 0));
    }
    const long long kv_ctas = (parts & 2) ? static_cast<long long>(nq) * (p.split_heads ? nh : nkv) * B : 0;
    const long long q_ctas = (parts & 4) ? static_cast<long long>(nq) * nh * B : 0;
    if (kv_ctas + q_ctas)
        launch_early(attn_bwd_kernel<false>, static_cast<unsigned>(kv_ctas + q_ctas), kAttnBwdThreads, kAttnBwdSmem, st, tm_qkv, tm_do, tm_do, p,
                     static_cast<int>(kv_ctas));
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        set_last_error("attn_bwd launch failed: %s", cudaGetErrorString(e));
        return CAI_K_CUDA;
    }
    return CAI_K_OK;
}

CAI_API int cai_flash_attn_window_walk(int B, int S, int nh, int nkv, int window, int sinks, int sms, int* parts, int capacity) {
    if (!window_sizes_ok(B, S, nh, nkv, window, sinks) || sms <= 0) return 0;
    const AttnWindow w = {window < S ? window : S, sinks < S ? sinks : S};
    const AttnWindowParts c = window_parts(w, B, S, nh, nkv, sms);
    const int n = c.near_ctas + c.far_ctas;
    for (int lin = 0; lin < n && lin < capacity; ++lin) {
        const WindowPart t(w, c, B, S, nh, nkv, lin);
        const int v[8] = {t.j, t.b, t.g, t.h_first, t.heads, t.q_first, t.q_tiles, t.slot};
        for (int k = 0; k < 8; ++k) parts[lin * 8 + k] = v[k];
    }
    return n;
}
CAI_API int cai_flash_attn_window_keys(int S, int window, int sinks, int i, int* tiles, int capacity) {
    if (!window_sizes_ok(1, S, 1, 1, window, sinks) || i < 0 || i > (S - 1) / kAttnTile) return 0;
    const WindowKeys keys({window < S ? window : S, sinks < S ? sinks : S}, i);
    for (int k = 0; k < keys.n && k < capacity; ++k) {
        tiles[2 * k] = keys.tile(k);
        tiles[2 * k + 1] = keys.width({window < S ? window : S, sinks < S ? sinks : S}, k);
    }
    return keys.n;
}

CAI_API long long cai_flash_attn_window_bwd_scratch(int B, int S, int nh, int nkv, int window, int sinks) {
    if (!window_sizes_ok(B, S, nh, nkv, window, sinks)) return 0;
    const int sms = sm_count(current_device());
    const AttnWindowParts c = window_parts({window < S ? window : S, sinks < S ? sinks : S}, B, S, nh, nkv, sms > 0 ? sms : 148);
    return (static_cast<long long>(c.near_slots) + c.far_ctas) * 131072;
}

CAI_API int cai_flash_attn_window_bwd(const void* qkv, long long ld, const void* out, const void* dout, const float* lse, float* delta, void* dqkv,
                                      long long ldq, void* scratch, int B, int S, int nh, int nkv, int hd, float scale, int window, int sinks,
                                      void* stream) {
    if (!window_call_ok("flash_attn_window_bwd", qkv, ld, out, B, S, nh, nkv, hd, scale, window, sinks) ||
        !window_call_ok("flash_attn_window_bwd (gradient)", dqkv, ldq, dout, B, S, nh, nkv, hd, scale, window, sinks))
        return CAI_K_BAD_ARG;
    if (B == 0 || S == 0) return CAI_K_OK;
    if (!qkv || !out || !dout || !lse || !delta || !dqkv) {
        set_last_error("flash_attn_window_bwd: an address is null");
        return CAI_K_BAD_ARG;
    }
    if (reinterpret_cast<uintptr_t>(scratch) & 15) {
        set_last_error("flash_attn_window_bwd: the scratch has to start on 16 bytes");
        return CAI_K_BAD_ARG;
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long ldo = static_cast<long long>(nh) * hd;
    CUtensorMap tm_qkv, tm_do, tm_dqkv;
    if (!encode_tmap_3d(&tm_qkv, qkv, static_cast<uint64_t>(nh + 2 * nkv) * hd, S, B, ld, static_cast<uint64_t>(ld) * S, 64, kAttnTile, 2) ||
        !encode_tmap_3d(&tm_do, dout, ldo, S, B, ldo, static_cast<uint64_t>(ldo) * S, 64, kAttnTile, 2) ||
        !encode_tmap_3d(&tm_dqkv, dqkv, static_cast<uint64_t>(nh + 2 * nkv) * hd, S, B, ldq, static_cast<uint64_t>(ldq) * S, 64, kAttnTile, 2))
        return CAI_K_BAD_ARG;
    const int dev = current_device();
    if (configure_bwd<true>(dev)) return CAI_K_CUDA;
    AttnBwdParams p = {};
    p.B = B; p.S = S; p.nh = nh; p.nkv = nkv;
    p.scale = scale;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.lse = lse;
    p.delta = delta;
    p.dqkv = static_cast<__nv_bfloat16*>(dqkv);
    p.ldq = ldq;
    p.status = status_words(dev);
    p.win = {window < S ? window : S, sinks < S ? sinks : S};
    p.cut = window_parts(p.win, B, S, nh, nkv, sm_count(dev));
    p.partial = static_cast<float*>(scratch);
    if (!scratch && p.cut.near_slots + p.cut.far_ctas > 0) {
        set_last_error("flash_attn_window_bwd: needs the scratch that cai_flash_attn_window_bwd_scratch says");
        return CAI_K_BAD_ARG;
    }
    // rows below `exact` of each sequence from P and dP, the others from O
    const int exact = static_cast<long long>(p.win.window) + p.win.sinks <= kFewKeys || S < kFewRows ? S : kFewRows;
    const long long pieces = static_cast<long long>((exact + 15) / 16) * nh * B;
    const long long others = static_cast<long long>(S - exact) * nh * B;
    // Four ways where that leaves the other rows' CTAs beside them (16 x 256 tokens, 16 / 4 heads, whose 512 pieces would come first: 49.9 us, one way 48.5); of the
    // others few rows a CTA only where all CTAs are one wave (8 x 128, 8 / 2 heads: 15.5, eight a thread 15.0 with the four ways).
    const int sms = sm_count(dev), ways = pieces < (others ? 1 : 4) * sms ? 4 : 1, exact_ctas = static_cast<int>((pieces * ways + 3) / 4);
    const int unroll = others < 2 * 16 * sms ? 2 : 8;
    const int other_ctas = static_cast<int>((others + 8 * unroll - 1) / (8 * unroll));
    cudaError_t e = launch_early(attn_window_row_sums_kernel, exact_ctas + other_ctas, 128, 0, st, static_cast<const __nv_bfloat16*>(qkv), ld,
                                 static_cast<const __nv_bfloat16*>(out), static_cast<const __nv_bfloat16*>(dout), lse, delta, B, S, nh, nkv, p.scale_log2, p.win, exact,
                                 ways, static_cast<unsigned>(exact_ctas), unroll);
    const int kv_ctas = p.cut.near_ctas + p.cut.far_ctas;
    const long long q_ctas = static_cast<long long>((S + kAttnTile - 1) / kAttnTile) * nh * B;
    if (e == cudaSuccess)
        e = launch_early(attn_bwd_kernel<true>, static_cast<unsigned>(kv_ctas + q_ctas), kAttnBwdThreads, kAttnBwdSmem, st, tm_qkv, tm_do, tm_dqkv, p, kv_ctas);
    if (e == cudaSuccess && p.cut.near_slots + p.cut.far_ctas > 0) {
        const long long tiles = p.cut.head_parts * p.cut.near_parts > 1 ? (S + kAttnTile - 1) / kAttnTile : p.cut.sink_tiles;
        e = launch_early(attn_window_join_kernel, static_cast<unsigned>(tiles * nkv * B * kJoinCtas), 256, 0, st, p);
    }
    if (e != cudaSuccess) {
        set_last_error("flash_attn_window_bwd launch failed: %s", cudaGetErrorString(e));
        return CAI_K_CUDA;
    }
    return CAI_K_OK;
}
