// rope_axes.cu - rotary embedding by the positions of several axes (time, height, width), in place on the q and k heads of a packed activation.
//
// Pair i of a head, its elements i and i + half, is turned by pos[axis(i)][token] * freqs[i]. The product is taken in 64 bits and brought to a part of
// one turn there: in 32 bits an angle of 10^5 radians is off by 0.004, as much as the result's rounding. A pair's angle is computed once per token, not
// once per head.
#include "cai_kernels.h"
#include "host_common.h"
#include "norm_kernels.cuh"
#include "sm100.cuh"

namespace cai {

struct RopeAxesParams {
    __nv_bfloat16* qkv;
    const double* freqs;
    const int* pos;
    long long ld, ldp;
    int T, heads, half, tokens;   // heads: those of q and k; tokens: of a CTA
    int axes, first[4];           // axis a's first pair, in order
    int count[4];
    int interleaved, inverse;
};

constexpr int kRopeThreads = 256, kRopeMostPairs = 2048;   // pairs of all tokens of a CTA

__device__ __forceinline__ int rope_axis(const RopeAxesParams& p, int i) {
    if (p.interleaved) {
        const int a = i % p.axes, k = i / p.axes;
        const int n = a == 0 ? p.count[0] : a == 1 ? p.count[1] : a == 2 ? p.count[2] : p.count[3];
        return k < n ? a : 0;
    }
    return (i >= p.first[1]) + (i >= p.first[2]) + (i >= p.first[3]);
}

__global__ void __launch_bounds__(kRopeThreads)
rope_axes_kernel(const RopeAxesParams p) {
    grid_dep_begin();
    __shared__ float2 turn[kRopeMostPairs];   // (cosine, sine) of the CTA's tokens and pairs
    const long long t0 = static_cast<long long>(blockIdx.x) * p.tokens;
    const int tokens = static_cast<int>(min(static_cast<long long>(p.tokens), p.T - t0));
    for (int k = threadIdx.x; k < tokens * p.half; k += kRopeThreads) {
        const int t = k / p.half, i = k - t * p.half;
        const double turns = p.pos[rope_axis(p, i) * p.ldp + t0 + t] * p.freqs[i] * 0.15915494309189533577;
        float s, c;
        sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
        turn[k] = make_float2(c, p.inverse ? -s : s);
    }
    __syncthreads();
    const int per = p.half >> 3, items = tokens * p.heads * per;
    for (int k = threadIdx.x; k < items; k += kRopeThreads) {
        const int t = k / (p.heads * per), in = k - t * p.heads * per, head = in / per, v = in - head * per;
        __nv_bfloat16* at = p.qkv + (t0 + t) * p.ld + head * 2 * p.half + v * 8;
        float a[8], b[8];
        unpack8(*reinterpret_cast<const uint4*>(at), a);
        unpack8(*reinterpret_cast<const uint4*>(at + p.half), b);
        const float2* cs = turn + t * p.half + v * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) rope_rotate(a[e], b[e], cs[e].x, cs[e].y);
        *reinterpret_cast<uint4*>(at) = pack8(a);
        *reinterpret_cast<uint4*>(at + p.half) = pack8(b);
    }
}

}  // namespace cai

using namespace cai;

CAI_API int cai_rope_apply_axes(void* qkv, const double* freqs, const int* pos, long long ldp, int T, int nh, int nkv, int hd, long long ld, int axes,
                                int n0, int n1, int n2, int n3, int interleaved, int inverse, void* stream) {
    const int half = hd / 2, n[4] = {n0, n1, n2, n3};
    bool ok = hd > 0 && hd % 16 == 0 && hd <= 256 && axes >= 1 && axes <= 4 && T >= 0 && nh >= 0 && nkv >= 0;
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
    if ((ld & 7) || ld < static_cast<long long>(nh + nkv) * hd || (reinterpret_cast<uintptr_t>(qkv) & 15) || (axes > 1 && ldp < T)) {
        set_last_error("rope_apply_axes: rows have to start on 16 bytes and hold the q and k heads, positions to lie axis by axis");
        return CAI_K_BAD_ARG;
    }
    if (T == 0 || nh + nkv == 0) return CAI_K_OK;
    RopeAxesParams p = {};
    p.qkv = static_cast<__nv_bfloat16*>(qkv);
    p.freqs = freqs; p.pos = pos;
    p.ld = ld; p.ldp = ldp;
    p.T = T; p.heads = nh + nkv; p.half = half;
    p.axes = axes;
    for (int a = 0, at = 0; a < 4; at += n[a++]) {
        p.first[a] = a < axes ? at : half;
        p.count[a] = n[a];
    }
    p.interleaved = interleaved; p.inverse = inverse;
    // about four times eight pairs a thread
    const int per = p.heads * (half / 8), most = kRopeMostPairs / half;
    p.tokens = (4 * kRopeThreads + per - 1) / per;
    p.tokens = p.tokens < most ? p.tokens : most;
    const cudaError_t e = launch_early(rope_axes_kernel, static_cast<unsigned>((static_cast<long long>(T) + p.tokens - 1) / p.tokens), kRopeThreads, 0,
                                       static_cast<cudaStream_t>(stream), p);
    if (e != cudaSuccess) {
        set_last_error("rope_apply_axes launch failed: %s", cudaGetErrorString(e));
        return CAI_K_CUDA;
    }
    return CAI_K_OK;
}
