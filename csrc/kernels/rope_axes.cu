// rope_axes.cu - rotary embedding by the positions of several axes (time, height, width), in place on the q and k heads of a packed activation.
//
// Pair i of a head, its elements i and i + half, is turned by pos[axis(i)][token] * freqs[i]. The product is taken in 64 bits and brought to a part of
// one turn there: in 32 bits an angle of 10^5 radians is off by 0.004, as much as the result's rounding. A pair's angle is computed once per token, not
// once per head. Bound by memory, four bytes an element of q and k. Measured on a B200: 32768 tokens of 32 / 8 heads 101 us (6.7 TB/s: the rate of a copy), 5003 of
// 9 / 3 heads 4.9, 256 of 2 / 1 1.9.
#include "cai_kernels.h"
#include "host_common.h"
#include "norm_kernels.cuh"
#include "sm100.cuh"

namespace cai {

constexpr int kRopeThreads = 256, kRopeMostPairs = 2048;   // pairs of all tokens of a CTA
constexpr int kRopeItems = 4;                              // times eight pairs a thread has in flight

// k / d for k and d below 2^16: (k * ceil(2^32 / d)) >> 32.
struct SmallDiv {
    uint32_t d, m;
    SmallDiv() = default;
    explicit SmallDiv(uint32_t by) : d(by), m(by == 1 ? 0 : static_cast<uint32_t>(((1ull << 32) + by - 1) / by)) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t k) const { return m ? __umulhi(k, m) : k; }
};

struct RopeAxesParams {
    __nv_bfloat16* qkv;
    const double* freqs;
    const int* pos;
    long long ld, ldp;
    int T, half, tokens;            // tokens: of a CTA
    SmallDiv per_token, per_head;   // eight pairs each
    int axes, first[4], count[4];   // an axis' first pair, where they follow one another, and its number
    int interleaved, inverse;
};

__device__ __forceinline__ int rope_axis(const RopeAxesParams& p, int i) {
    if (p.interleaved) {
        const int a = i % p.axes, k = i / p.axes;
        const int n = a == 0 ? p.count[0] : a == 1 ? p.count[1] : a == 2 ? p.count[2] : p.count[3];
        return k < n ? a : 0;
    }
    return (i >= p.first[1]) + (i >= p.first[2]) + (i >= p.first[3]);
}

// The data of a CTA's first kRopeItems x 256 pieces is asked for before the angles are computed, which take about as long as it needs to come: read after
// them, 32768 tokens of 32 / 8 heads took 117 us. A thread computes one pair's angles, token after token.
__global__ void __launch_bounds__(kRopeThreads)
rope_axes_kernel(const RopeAxesParams p) {
    grid_dep_begin();
    // (cosine, sine) of the CTA's tokens and pairs; of eight pairs v, two and two: [token][two of the eight][v], so that neighbours read neighbours
    __shared__ float4 turn[kRopeMostPairs / 2];
    const long long t0 = static_cast<long long>(blockIdx.x) * p.tokens;
    const uint32_t tokens = static_cast<uint32_t>(min(static_cast<long long>(p.tokens), p.T - t0));
    const uint32_t items = tokens * p.per_token.d;
    __nv_bfloat16* at[kRopeItems];
    uint32_t cs[kRopeItems];
    uint4 a[kRopeItems], b[kRopeItems];
    auto fetch = [&](uint32_t k0) {
#pragma unroll
        for (int u = 0; u < kRopeItems; ++u) {
            const uint32_t k = k0 + u * kRopeThreads;
            if (k < items) {
                const uint32_t t = p.per_token(k), in = k - t * p.per_token.d, head = p.per_head(in), v = in - head * p.per_head.d;
                at[u] = p.qkv + (t0 + t) * p.ld + head * 2 * p.half + v * 8;
                cs[u] = t * (p.half >> 1) + v;
                a[u] = *reinterpret_cast<const uint4*>(at[u]);
                b[u] = *reinterpret_cast<const uint4*>(at[u] + p.half);
            }
        }
    };
    fetch(threadIdx.x);
    // as many tokens side by side as there are threads for whole sets of pairs
    const uint32_t beside = kRopeThreads / p.half, mine = threadIdx.x / p.half, i = threadIdx.x - mine * p.half;
    if (mine < beside) {
        const double turns_per_pos = p.freqs[i] * 0.15915494309189533577;
        const int* pos = p.pos + rope_axis(p, i) * p.ldp + t0;
        float2* out = reinterpret_cast<float2*>(turn) + ((i >> 1) & 3) * (p.half >> 2) + (i >> 3) * 2 + (i & 1);
        for (uint32_t t = mine; t < tokens; t += beside) {
            const double turns = pos[t] * turns_per_pos;
            float s, c;
            sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
            out[t * p.half] = make_float2(c, p.inverse ? -s : s);
        }
    }
    __syncthreads();
    for (uint32_t k0 = threadIdx.x;;) {
#pragma unroll
        for (int u = 0; u < kRopeItems; ++u) {
            if (k0 + u * kRopeThreads >= items) break;
            float x[8], y[8];
            unpack8(a[u], x);
            unpack8(b[u], y);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float4 q = turn[cs[u] + e * p.per_head.d];
                rope_rotate(x[2 * e], y[2 * e], q.x, q.y);
                rope_rotate(x[2 * e + 1], y[2 * e + 1], q.z, q.w);
            }
            *reinterpret_cast<uint4*>(at[u]) = pack8(x);
            *reinterpret_cast<uint4*>(at[u] + p.half) = pack8(y);
        }
        k0 += kRopeItems * kRopeThreads;
        if (k0 >= items) break;
        fetch(k0);
    }
}

}  // namespace cai

using namespace cai;

CAI_API int cai_rope_apply_axes(void* qkv, const double* freqs, const int* pos, long long ldp, int T, int nh, int nkv, int hd, long long ld, int axes,
                                int n0, int n1, int n2, int n3, int interleaved, int inverse, void* stream) {
    const int half = hd / 2, n[4] = {n0, n1, n2, n3};
    bool ok = hd > 0 && hd % 16 == 0 && hd <= 256 && axes >= 1 && axes <= 4 && T >= 0 && nh >= 0 && nkv >= 0 && nh <= 65535 && nkv <= 65535;
    int sum = 0;
    for (int a = 0; ok && a < 4; ++a) {
        ok = a < axes ? n[a] >= 0 && n[a] <= half : n[a] == 0;
        sum += n[a];
    }
    if (!ok || sum != half) {
        set_last_error("rope_apply_axes: needs a head dimension of a multiple of 16 up to 256 and one to four sections that add up to half of it (%d: %d, %d, "
                       "%d, %d)", hd, n0, n1, n2, n3);
        return CAI_K_BAD_ARG;
    }
    // every axis but the first has the pairs a, a + axes, a + 2 axes ..., as many as its section says
    for (int a = 1; interleaved && a < axes; ++a)
        if (n[a] > 0 && a + static_cast<long long>(axes) * (n[a] - 1) >= half) {
            set_last_error("rope_apply_axes: section %d of %d pairs does not fit every %d-th of %d pairs", a, n[a], axes, half);
            return CAI_K_BAD_ARG;
        }
    if ((ld & 7) || ld < static_cast<long long>(nh + nkv) * hd || (reinterpret_cast<uintptr_t>(qkv) & 15) || ldp < 0) {
        set_last_error("rope_apply_axes: rows have to start on 16 bytes and hold the q and k heads");
        return CAI_K_BAD_ARG;
    }
    if ((nh + nkv) * (half / 8) >= 65536) {
        set_last_error("rope_apply_axes: too many heads (%d)", nh + nkv);
        return CAI_K_BAD_ARG;
    }
    if (T == 0 || nh + nkv == 0) return CAI_K_OK;
    if (!qkv || !freqs || !pos) {
        set_last_error("rope_apply_axes: an address is null");
        return CAI_K_BAD_ARG;
    }
    RopeAxesParams p = {};
    p.qkv = static_cast<__nv_bfloat16*>(qkv);
    p.freqs = freqs; p.pos = pos;
    p.ld = ld; p.ldp = ldp;
    p.T = T; p.half = half;
    p.axes = axes;
    for (int a = 0, at = 0; a < 4; at += n[a++]) {
        p.first[a] = a < axes ? at : half;
        p.count[a] = n[a];
    }
    p.interleaved = interleaved; p.inverse = inverse;
    const int heads = nh + nkv;
    p.per_head = SmallDiv(half / 8);
    p.per_token = SmallDiv(heads * (half / 8));
    // one round of kRopeItems pieces a thread, or a token where one has more; fewer tokens where that leaves SMs without a CTA
    const int sms = sm_count(current_device()), most = kRopeMostPairs / half;
    p.tokens = kRopeItems * kRopeThreads / static_cast<int>(p.per_token.d);
    p.tokens = p.tokens < most ? p.tokens : most;
    if (static_cast<long long>(p.tokens) * 2 * sms > T) p.tokens = (T + 2 * sms - 1) / (2 * sms);
    p.tokens = p.tokens > 0 ? p.tokens : 1;
    const cudaError_t e = launch_early(rope_axes_kernel, static_cast<unsigned>((static_cast<long long>(T) + p.tokens - 1) / p.tokens), kRopeThreads, 0,
                                       static_cast<cudaStream_t>(stream), p);
    if (e != cudaSuccess) {
        set_last_error("rope_apply_axes launch failed: %s", cudaGetErrorString(e));
        return CAI_K_CUDA;
    }
    return CAI_K_OK;
}
