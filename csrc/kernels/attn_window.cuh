// attn_window.cuh - what windowed attention's forward and backward kernels share: which tiles belong together, what is seen of them.
#pragma once

#include "attn_common.cuh"
#include "f32x2.cuh"
#include "sm100.cuh"

namespace cai {

// The lowest n of 32 bits, for any n.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }

// ---------------------------------------------------------------- a window and sinks
// Query q sees key k if k <= q and (k > q - window or k < sinks), with 1 <= window <= S and 0 <= sinks <= S.
struct AttnWindow {
    int window, sinks;
};
// How many of the `most` keys from k0 on are sinks, rounded up to 16.
__host__ __device__ inline int seen_sinks(const AttnWindow& w, int k0, int most) {
    const int n = (w.sinks - k0 + 15) / 16 * 16;
    return n < most ? n : most;
}
// The key tiles of query tile i, in ascending order: the sinks' tiles, then those from the one that holds the first query's first key up to the diagonal.
struct WindowKeys {
    int diag, near, n;
    __host__ __device__ WindowKeys(const AttnWindow& w, int i) {
        const int reach = i * kAttnTile - w.window + 1, lo = reach > 0 ? reach / kAttnTile : 0, sink_tiles = (w.sinks + kAttnTile - 1) / kAttnTile;
        diag = i;
        near = i - lo + 1;
        n = near + (sink_tiles < lo ? sink_tiles : lo);
    }
    __host__ __device__ int tile(int j) const { return j < n - near ? j : diag - (n - 1 - j); }
    // Of a sinks' tile only the first keys are seen: how many, up to what a product takes (16 at a time).
    __host__ __device__ int width(const AttnWindow& w, int j) const { return j < n - near ? seen_sinks(w, j * kAttnTile, kAttnTile) : kAttnTile; }
};
// The query tiles that key tile j is seen by through the window: j .. last.
__host__ __device__ inline int window_last_query_tile(const AttnWindow& w, int j, int tiles) {
    const long long last = (static_cast<long long>(j + 1) * kAttnTile + w.window - 2) / kAttnTile;
    return last < tiles ? static_cast<int>(last) : tiles - 1;
}
// Is something hidden between query tile i and key tile j <= i?
__device__ __forceinline__ bool window_masks(const AttnWindow& w, int i, int j) {
    return i == j || ((i - j + 1) * kAttnTile > w.window && (j + 1) * kAttnTile > w.sinks);
}

}  // namespace cai
