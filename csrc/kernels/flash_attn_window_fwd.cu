// flash_attn_window_fwd.cu - causal grouped-query flash attention with a window and sinks, forward, for sm_100a, head_dim 128, sequences of any length.
//
//   s_ij = scale q_i . k_j where j <= i and (j > i - window or j < sinks), else -inf;   o_i = sum_j softmax(s_i)_j v_j;   lse_i = log sum_j exp(s_ij)
//
// One pass over the keys of a 128-row query tile, 64 at a time, with a running maximum and sum. Two CTAs share an SM (105 KB and half of the tensor memory each) and stay
// for the whole launch: each takes one (query tile, head, sequence) after the other, and the blocks of all of them are one stream, so that loads and scores
// run ahead over the end of a tile; with windows of few blocks a tile's beginning and end are most of it. Warp 0 loads by TMA, warp 1 issues the tcgen05
// products, warps 2-5 are the softmax, a thread a row. S = Q K^T lies in tensor memory for two blocks, so that the next block's scores are there
// when a block's softmax ends. P goes back over S in bf16 (its rounding is half a step, 2^-8 of a weight; the sum of the weights is that of the unrounded
// ones) and is the A operand of O += P V. The maximum is refreshed, and O rescaled, only when it grew by more than 2^8.
// The tensor map has the sequences apart: rows past a sequence's end come as zeros, never as the next one's.
// TMEM: S / P 0-63 and 64-127, O 128-255.
// Measured on a B200, us, one launch in a burst / back to back at the power limit (985 W, 1545-1597 MHz): 4 x 4096 tokens, 16 / 8 heads, window 1024, 4 sinks 153 / 163 (790 /
// 740 TFLOP/s of what is seen), 16384 tokens, window 4096 480 / 500 (1000 / 960); 333 tokens, 8 / 1 heads 8.2, 2 x 128, 2 / 1 heads 5.5. Tensor pipe, exponentials and issue
// slots are each near half busy: what a block takes is the chain from its scores to its P, which two CTAs overlap. 64 keys, although the scores' products run at 1.7 times the
// cycles per key (their operand reads fill shared memory's bandwidth), because tensor memory holds two blocks of scores only of that width: 128 keys at a time without the second
// 536 against 497-530 (8192 tokens, 32 / 8 heads). Two heads side by side in one CTA, sharing K and V: 588 against 494 (window 4096).
#include <math.h>

#include "attn_window.cuh"
#include "cai_kernels.h"
#include "host_common.h"

namespace cai {

// n / d for 0 <= n < 2^31: the product with floor(2^32 / d) is at most one short (n / 2^32 < 1 of what its last digits leave).
struct Divisor {
    int d;
    uint32_t m;
    Divisor() = default;
    explicit Divisor(int by) : d(by), m(by == 1 ? 0xffffffffu : static_cast<uint32_t>((1ull << 32) / static_cast<uint32_t>(by))) {}
    __host__ __device__ __forceinline__ int quotient(int n) const {
        const int q = static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * m) >> 32);
        return q + (n - q * d >= d);
    }
};

struct WindowFwdParams {
    int B, S, nh, nkv;
    float scale_log2;
    AttnWindow win;
    __nv_bfloat16* out;
    float* lse;
    int* status;
    int tiles, items;    // query tiles of a sequence; of all heads and sequences
    Divisor heads_all, heads, group;    // heads of all sequences, of one, of a kv head
};

constexpr int kWindowFwdThreads = 192;
constexpr int kBlock = 64, kBlockBytes = kBlock * kAttnHD * 2, kBlockSub = kBlockBytes / 2;   // of keys
constexpr int kStageBytes = 2048;       // of a softmax warp, for its output: 32 rows of 32 columns
constexpr int kWindowFwdSmem = 3 * kAttnTileBytes + 4 * kStageBytes + 1024 + 256;

// A warp's 32 finished rows of O, each lane with one, times `inv` to bf16, 32 columns at a time through 2 KB of shared memory, so that a store of the warp
// writes 64 bytes of each of eight rows; the first `rows` of them. `read`: told once they are out of tensor memory.
__device__ __forceinline__ void put_window_rows(uint32_t stage, uint32_t tO, float inv, __nv_bfloat16* out, long long ld, int lane, int rows, uint64_t* read) {
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        tmem_ld_32x32(tO + c * 32, v);
        tmem_ld_wait();
        if (c == 3) {
            tc_fence_before();
            mbar_arrive_warp(read);
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t o[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) o[t] = pack_bf16(__uint_as_float(v[j * 8 + 2 * t]) * inv, __uint_as_float(v[j * 8 + 2 * t + 1]) * inv);
            st_shared_v4(stage + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4), o[0], o[1], o[2], o[3]);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2), chunk = lane & 3;
            const uint4 w = ld_shared_v4(stage + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
            if (row < rows) *reinterpret_cast<uint4*>(out + row * ld + c * 32 + chunk * 8) = w;
        }
    }
}


// The blocks of 64 keys of query tile i, in ascending order: those of the sinks, then from the one with the first query's first key to the one with the last
// query.
struct WindowBlocks {
    int q0, sinks, lo, n;
    WindowBlocks() = default;
    __host__ __device__ WindowBlocks(const AttnWindow& w, int i, int S) {
        q0 = i * kAttnTile;
        const int reach = q0 - w.window + 1, end = q0 + kAttnTile < S ? q0 + kAttnTile : S, sink_blocks = (w.sinks + kBlock - 1) / kBlock;
        lo = reach > 0 ? reach / kBlock : 0;
        sinks = sink_blocks < lo ? sink_blocks : lo;
        n = sinks + (end + kBlock - 1) / kBlock - lo;
    }
    __host__ __device__ int block(int j) const { return j < sinks ? j : lo + j - sinks; }
};

// Item number `round` of CTA `cta` of `ctas`: rounds go to and fro, so that nobody gets the longest item of each.
__host__ __device__ __forceinline__ int item_of(int round, int cta, int ctas) { return round * ctas + ((round & 1) ? ctas - 1 - cta : cta); }
// An item: latest query tiles, which have the most keys, of every head first.
struct WindowTile {
    int tile, h, b;
    WindowTile() = default;
    __host__ __device__ __forceinline__ WindowTile(int item, int tiles, const Divisor& heads_all, const Divisor& heads) {
        const int row = heads_all.quotient(item), at = item - row * heads_all.d;
        tile = tiles - 1 - row;
        b = heads.quotient(at);
        h = at - b * heads.d;
    }
};

// The blocks of keys that a CTA takes, item after item.
struct WindowStream : WindowTile {
    int round;
    int u;                 // block of the item
    WindowBlocks keys;
    __device__ WindowStream(const WindowFwdParams& p) : round(-1), u(0) { keys.n = 0; next_item(p); }
    __device__ bool there() const { return keys.n > 0; }
    __device__ bool last() const { return u + 1 == keys.n; }
    __device__ int row() const { return keys.block(u) * kBlock; }
    __device__ void next_item(const WindowFwdParams& p) {
        ++round;
        const int item = item_of(round, blockIdx.x, gridDim.x);
        u = 0;
        keys.n = 0;
        if (item >= p.items) return;     // of the last round, which nothing follows
        static_cast<WindowTile&>(*this) = WindowTile(item, p.tiles, p.heads_all, p.heads);
        keys = WindowBlocks(p.win, tile, p.S);
    }
    __device__ void next(const WindowFwdParams& p) {
        if (++u == keys.n) next_item(p);
    }
};

// What the issuing warp has to know of it: how many blocks the item has left. (With the whole stream it spent 240 cycles a block on it, 700 an item, beside an idle
// pipe.)
struct WindowCount {
    int round, left, n, sinks;
    __device__ WindowCount(const WindowFwdParams& p) : round(-1) { next_item(p); }
    __device__ bool there() const { return left > 0; }
    __device__ bool first() const { return left == n; }
    // keys of block u of the item, as products take them
    __device__ int width(const WindowFwdParams& p, int u) const { return u < sinks ? seen_sinks(p.win, u * kBlock, kBlock) : kBlock; }
    __device__ void next_item(const WindowFwdParams& p) {
        ++round;
        const int item = item_of(round, blockIdx.x, gridDim.x);
        left = n = 0;
        if (item >= p.items) return;
        const WindowBlocks blocks(p.win, p.tiles - 1 - p.heads_all.quotient(item), p.S);
        left = n = blocks.n;
        sinks = blocks.sinks;
    }
    __device__ __forceinline__ void next(const WindowFwdParams& p) {
        if (--left == 0) next_item(p);
    }
};

__global__ void __launch_bounds__(kWindowFwdThreads, 2)
attn_window_fwd_kernel(const __grid_constant__ CUtensorMap tm, const WindowFwdParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;
    uint8_t* sK = smem + kAttnTileBytes;                     // block c of the stream in buffer c & 1
    uint8_t* sV = smem + kAttnTileBytes + 2 * kBlockBytes;   // likewise
    uint8_t* sO = smem + 3 * kAttnTileBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sO + 4 * kStageBytes);
    uint64_t* q_full = bars;
    uint64_t* k_first = bars + 1;    // the first two blocks of K
    uint64_t* kv_full = bars + 2;    // [2] V of block c and K of block c + 2
    uint64_t* done = bars + 4;       // [2] S of block c and P V of block c - 2 are computed: step c, in order, on barrier c & 1
    uint64_t* o_full = bars + 6;     // an item's last P V is done
    uint64_t* o_empty = bars + 7;    // its output has left tensor memory
    uint64_t* p_full = bars + 8;     // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 10);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm);
        for (int i = 0; i < 7; ++i) mbar_init(&bars[i], 1);
        for (int i = 7; i < 10; ++i) mbar_init(&bars[i], 4);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 256);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dep_wait();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            auto load_block = [&](uint8_t* dst, uint64_t* bar, const WindowStream& at, int head, int c) {
                tma_load_3d(dst + (c & 1) * kBlockBytes, &tm, bar, head * kAttnHD, at.row(), at.b);
                tma_load_3d(dst + (c & 1) * kBlockBytes + kBlockSub, &tm, bar, head * kAttnHD + 64, at.row(), at.b);
            };
            auto load_q = [&](const WindowStream& at) {
                mbar_expect_tx(q_full, kAttnTileBytes);
                for (int k = 0; k < 4; ++k)    // the tile's sub-tiles of 64 columns, 64 rows at a time
                    tma_load_3d(sQ + k * kBlockSub, &tm, q_full, at.h * kAttnHD + (k >> 1) * 64, at.tile * kAttnTile + (k & 1) * kBlock, at.b);
            };
            WindowStream cur(p), ahead = cur;      // block c, and the one whose K comes with its V
            load_q(cur);
            ahead.next(p);
            mbar_expect_tx(k_first, ahead.there() ? 2 * kBlockBytes : kBlockBytes);
            load_block(sK, k_first, cur, p.nh + p.group.quotient(cur.h), 0);
            if (ahead.there()) {
                load_block(sK, k_first, ahead, p.nh + p.group.quotient(ahead.h), 1);
                ahead.next(p);
            }
            bool ok = true;
            for (int c = 0; cur.there(); ++c) {
                // after step c nobody reads K of block c and V of block c - 2 any more, nor Q if the block is its item's last
                if (!mbar_wait(&done[c & 1], (c >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                mbar_expect_tx(&kv_full[c & 1], ahead.there() ? 2 * kBlockBytes : kBlockBytes);
                load_block(sV, &kv_full[c & 1], cur, p.nh + p.nkv + p.group.quotient(cur.h), c);
                if (ahead.there()) {
                    load_block(sK, &kv_full[c & 1], ahead, p.nh + p.group.quotient(ahead.h), c);
                    ahead.next(p);
                }
                const bool turn = cur.last();
                cur.next(p);
                if (turn && cur.there()) load_q(cur);
            }
            grid_dep_launch();
            if (!ok)
                for (int i = 0; i < 32; ++i) __nanosleep(50000);
        }
    } else if (warp == 1) {
        // S runs two blocks ahead: S of block c + 2 goes out behind P V of block c, whose P it overwrites (the pipe keeps their order). The issuing thread is at
        // most one MMA ahead of the pipe, which idles while the thread waits (some 200 cycles for a barrier that is satisfied already) or commits (100
        // to 150): a block has two waits and one commit.
        const uint32_t idesc_pv = umma_idesc_bf16(128, 128, 0, 1);
        const uint64_t qd = umma_smem_desc_sw128(smem_u32(sQ), 0, 1024), kd = umma_smem_desc_sw128(smem_u32(sK), 0, 1024);
        const uint64_t vd = umma_smem_desc_sw128(smem_u32(sV), kBlockSub, 1024);
        const uint32_t tS = tmem_base, tO = tmem_base + 128;
        const bool leader = elect_one();
        auto scores = [&](int slot, uint32_t idesc_qk) {
#pragma unroll
            for (int k = 0; k < kAttnHD / 16; ++k)
                umma_f16_ss(tS + slot * kBlock, qd + (((k >> 2) * kAttnSub + (k & 3) * 32) >> 4),
                            kd + ((slot * kBlockBytes + (k >> 2) * kBlockSub + (k & 3) * 32) >> 4), idesc_qk, k > 0 ? 1u : 0u);
        };
        // A sinks' block is as wide as there are sinks: 3 to 4 % of the products with windows of a thousand.
        constexpr uint32_t idesc_full = umma_idesc_bf16(128, kBlock, 0, 0);
        auto idesc_of = [&](const WindowCount& at, int u) { return u < at.sinks ? umma_idesc_bf16(128, at.width(p, u), 0, 0) : idesc_full; };
        uint32_t q_phase = 0, o_phase = 1;      // o_empty: nothing to wait for before the first item
        // the queries of the next item's first block
        auto queries = [&]() {
            const bool come = mbar_wait_warp(q_full, q_phase, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
            q_phase ^= 1;
            tc_fence_after();
            return come;
        };
        WindowCount cur(p), ahead = cur;
        bool ok = true;
        for (int k = 0; k < 2 && ahead.there() && ok; ++k) {
            ok = (!ahead.first() || queries()) && mbar_wait_warp(k_first, 0, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
            if (!ok) break;
            tc_fence_after();
            if (leader) {
                scores(k, idesc_of(ahead, ahead.n - ahead.left));
                umma_commit(&done[k]);
            }
            __syncwarp();
            ahead.next(p);
        }
        int c = 0;
        // P of block c and what its products read have come
        auto come = [&](bool first) {
            bool yes = mbar_wait_warp(&kv_full[c & 1], (c >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
            if (first) {      // the last item's output has to be out of O
                yes = yes && mbar_wait_warp(o_empty, o_phase, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
                o_phase ^= 1;
            }
            yes = yes && mbar_wait_warp(&p_full[c & 1], (c >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
            tc_fence_after();
            return yes;
        };
        auto weigh = [&](bool first) {
#pragma unroll
            for (int k = 0; k < kBlock / 16; ++k)
                umma_f16_ts(tO, tS + (c & 1) * kBlock + k * 8, vd + (((c & 1) * kBlockBytes + k * 2048) >> 4), idesc_pv, (!first || k > 0) ? 1u : 0u);
        };
        auto weigh_sinks = [&](bool first, int width) {
            for (int k = 0; k * 16 < width; ++k)
                umma_f16_ts(tO, tS + (c & 1) * kBlock + k * 8, vd + (((c & 1) * kBlockBytes + k * 2048) >> 4), idesc_pv, (!first || k > 0) ? 1u : 0u);
        };
        while (cur.there() && ok) {
            const int n = cur.n;
            int u = 0;
            // while the block two ahead is of the same item nothing else has to be known
            for (; u + 2 < n && u < cur.sinks; ++u, ++c) {
                if (!(ok = come(u == 0))) break;
                if (leader) {
                    weigh_sinks(u == 0, cur.width(p, u));
                    scores(c & 1, idesc_of(cur, u + 2));
                    umma_commit(&done[c & 1]);     // step c + 2
                }
                __syncwarp();
            }
            for (; u + 2 < n && ok; ++u, ++c) {
                if (!(ok = come(u == 0))) break;
                if (leader) {
                    weigh(u == 0);
                    scores(c & 1, idesc_full);
                    umma_commit(&done[c & 1]);
                }
                __syncwarp();
            }
            if (n > 2) ahead.next_item(p);
            for (; u < n && ok; ++u, ++c) {
                const bool more = ahead.there(), turn = more && ahead.first();
                if (!(ok = come(u == 0))) break;
                if (leader) {
                    if (u < cur.sinks) weigh_sinks(u == 0, cur.width(p, u));
                    else weigh(u == 0);
                    if (u + 1 == n) umma_commit(o_full);
                    if (more && !turn) scores(c & 1, idesc_of(ahead, ahead.n - ahead.left));
                    if (!turn) umma_commit(&done[c & 1]);
                }
                __syncwarp();
                if (turn) {
                    if (!(ok = queries())) break;
                    if (leader) {
                        scores(c & 1, idesc_of(ahead, 0));
                        umma_commit(&done[c & 1]);
                    }
                    __syncwarp();
                }
                if (more) ahead.next(p);
            }
            cur.next_item(p);
        }
    } else {
        const int r = (warp & 3) * 32 + lane;          // row inside the tile == TMEM lane
        const uint32_t lane_bits = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t tO = tmem_base + 128 + lane_bits;
        const uint32_t stage = smem_u32(sO + (warp - 2) * kStageBytes);
        const uint64_t scale2 = pair_of(p.scale_log2, p.scale_log2);
        bool ok = true;
        int c = 0;       // block of the stream
        for (WindowStream at(p); at.there() && ok; at.next_item(p)) {
            const int q0 = at.tile * kAttnTile;
            // A window may hide a whole row of a block, so that its maximum starts at the lowest finite number: exp2(-inf - m) is 0 then as well.
            float m_used = -3.4028234664e38f;
            uint64_t l2 = 0;
#pragma unroll 1
            for (int u = 0; u < at.keys.n; ++u, ++c) {
                // what does not need the scores comes before the wait for them
                const uint32_t tS = tmem_base + (c & 1) * kBlock + lane_bits;
                const int k0 = at.keys.block(u) * kBlock;
                const bool hides = k0 + kBlock > q0 || (q0 + kAttnTile - k0 > p.win.window && k0 + kBlock > p.win.sinks);
                uint32_t seen[2] = {~0u, ~0u};
                if (hides) {
                    // seen are the columns before < k <= last and those below `sink`; a bit each
                    const int last = r + q0 - k0, before = last - p.win.window, sink = p.win.sinks - k0;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        seen[h] = bits_below(last + 1 - h * 32) & (~bits_below(before + 1 - h * 32) | bits_below(sink - h * 32));
                }
                if (!mbar_wait_warp(&done[c & 1], (c >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                tc_fence_after();
                uint32_t sc[2][32];
                tmem_ld_32x32(tS, sc[0]);
                tmem_ld_32x32(tS + 32, sc[1]);
                tmem_ld_wait();
                if (hides) {
                    // Hidden scores become -inf here, so that one path serves all blocks below (a select at every exponential of every tile: 8192 tokens, 32 / 8
                    // heads, everything visible 808 -> 473 us).
#pragma unroll
                    for (int c2 = 0; c2 < 2; ++c2) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(seen[c2] & (1u << e))) sc[c2][e] = 0xff800000u;   // -inf
                    }
                }
                float mx[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t* v = &sc[i >> 2][(i & 3) * 8];
                    mx[i] = max3(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]));
                    mx[i] = max3(mx[i], __uint_as_float(v[3]), __uint_as_float(v[4]));
                    mx[i] = max3(mx[i], __uint_as_float(v[5]), __uint_as_float(v[6]));
                    mx[i] = fmaxf(mx[i], __uint_as_float(v[7]));
                }
                const float top = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
                const float m_new = fmaxf(m_used, top * p.scale_log2);
                if (__any_sync(0xffffffffu, m_new > m_used + 8.f)) {
                    const float alpha = fast_exp2(m_used - m_new);  // 0 on the first block
                    l2 = mul2(l2, pair_of(alpha, alpha));
                    if (u > 0) {
                        // O is complete up to the block before with step c + 1. (This warp has not given block c + 1, which step c + 3 needs: the barrier is in that
                        // phase or has just left it.)
                        if (!mbar_wait_warp(&done[(c + 1) & 1], ((c + 1) >> 1) & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN)) { ok = false; break; }
                        tc_fence_after();
#pragma unroll 1
                        for (int o = 0; o < 8; ++o) {
                            uint32_t v[16];
                            tmem_ld_32x16(tO + o * 16, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
                            tmem_st_32x16(tO + o * 16, v);
                        }
                        tmem_st_wait();
                    }
                    m_used = m_new;
                }
                const uint64_t m2 = pair_of(-m_used, -m_used);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t pk[16];
                    uint64_t s2 = 0;
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 x = floats_of(fma2(pair_of(__uint_as_float(sc[half][e]), __uint_as_float(sc[half][e + 1])), scale2, m2));
                        const float w0 = fast_exp2(x.x), w1 = fast_exp2(x.y);
                        s2 = add2(s2, pair_of(w0, w1));
                        pk[e >> 1] = pack_bf16(w0, w1);
                    }
                    l2 = add2(l2, s2);
                    tmem_st_32x16(tS + half * 16, pk);
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive_warp(&p_full[c & 1]);
            }
            ok = ok && mbar_wait_warp(o_full, at.round & 1, abort_flag, p.status, CAI_DEV_TIMEOUT_ATTN);
            if (!ok) break;
            tc_fence_after();
            const float2 ll = floats_of(l2);
            const float l = ll.x + ll.y, inv = 1.f / l;
            const long long ldo = static_cast<long long>(p.nh) * kAttnHD, row0 = static_cast<long long>(at.b) * p.S + q0 + (r & ~31);
            put_window_rows(stage, tO, inv, p.out + row0 * ldo + at.h * kAttnHD, ldo, lane, p.S - q0 - (r & ~31), o_empty);
            if (q0 + r < p.S) p.lse[(static_cast<long long>(at.b) * p.nh + at.h) * p.S + q0 + r] = (m_used + log2f(l)) * 0.6931471805599453f;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 256);
    }
}

}  // namespace cai

using namespace cai;

CAI_API int cai_flash_attn_window_blocks(int S, int window, int sinks, int i, int* blocks, int capacity) {
    if (!window_sizes_ok(1, S, 1, 1, window, sinks) || i < 0 || i > (S - 1) / kAttnTile) return 0;
    const AttnWindow w = {window < S ? window : S, sinks < S ? sinks : S};
    const WindowBlocks b(w, i, S);
    for (int k = 0; k < b.n && k < capacity; ++k) {
        blocks[2 * k] = b.block(k);
        blocks[2 * k + 1] = k < b.sinks ? seen_sinks(w, k * kBlock, kBlock) : kBlock;
    }
    return b.n;
}
CAI_API int cai_flash_attn_window_items(int B, int S, int nh, int ctas, int cta, int* items, int capacity) {
    if (!window_sizes_ok(B, S, nh, nh, 1, 0) || cta < 0 || cta >= ctas) return 0;
    const int tiles = (S + kAttnTile - 1) / kAttnTile, all = tiles * nh * B;
    const Divisor heads_all(nh * B), heads(nh);
    int n = 0;
    for (int round = 0;; ++round) {
        const int item = item_of(round, cta, ctas);
        if (item >= all) return n;
        if (n < capacity) {
            const WindowTile t(item, tiles, heads_all, heads);
            items[3 * n] = t.tile;
            items[3 * n + 1] = t.h;
            items[3 * n + 2] = t.b;
        }
        ++n;
    }
}

CAI_API int cai_flash_attn_window_fwd(const void* qkv, long long ld, void* out, float* lse, int B, int S, int nh, int nkv, int hd, float scale,
                                      int window, int sinks, void* stream) {
    if (!window_call_ok("flash_attn_window_fwd", qkv, ld, out, B, S, nh, nkv, hd, scale, window, sinks)) return CAI_K_BAD_ARG;
    if (B == 0 || S == 0) return CAI_K_OK;
    if (!qkv || !out || !lse) {
        set_last_error("flash_attn_window_fwd: an address is null");
        return CAI_K_BAD_ARG;
    }
    CUtensorMap tm;
    if (!encode_tmap_3d(&tm, qkv, static_cast<uint64_t>(nh + 2 * nkv) * hd, S, B, ld, static_cast<uint64_t>(ld) * S, 64, kBlock, 2)) return CAI_K_BAD_ARG;
    WindowFwdParams p;
    p.B = B; p.S = S; p.nh = nh; p.nkv = nkv;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.win = {window < S ? window : S, sinks < S ? sinks : S};
    p.out = static_cast<__nv_bfloat16*>(out);
    p.lse = lse;
    const int dev = current_device(), sms = sm_count(dev);
    p.status = status_words(dev);
    p.tiles = (S + kAttnTile - 1) / kAttnTile;
    p.items = static_cast<int>(static_cast<long long>(p.tiles) * nh * B);
    p.heads_all = Divisor(nh * B);
    p.heads = Divisor(nh);
    p.group = Divisor(nh / nkv);
    static bool configured[64] = {};
    if (!configured[dev & 63]) {
        if (cudaFuncSetAttribute(attn_window_fwd_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kWindowFwdSmem) != cudaSuccess ||
            cudaFuncSetAttribute(attn_window_fwd_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess) {
            set_last_error("cudaFuncSetAttribute(attn_window_fwd) failed");
            return CAI_K_CUDA;
        }
        configured[dev & 63] = true;
    }
    const cudaError_t e = launch_early(attn_window_fwd_kernel, p.items < 2 * sms ? p.items : 2 * sms, kWindowFwdThreads, kWindowFwdSmem,
                                       static_cast<cudaStream_t>(stream), tm, p);
    if (e != cudaSuccess) {
        set_last_error("flash_attn_window_fwd launch failed: %s", cudaGetErrorString(e));
        return CAI_K_CUDA;
    }
    return CAI_K_OK;
}
