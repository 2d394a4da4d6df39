// norm_e4m3.cu - RMSNorm in front of a block-scaled e4m3 product: the residual's addition, the norm and the quantiser in one pass.
//
//   h = bf16(x + residual)     rstd = (mean(h^2) + eps)^(-1/2)     y = h * rstd * g
//   s[row, b] = max |y| of the row's 128 columns b / 448 (1 where they are all zero)     q = e4m3(y / s)
//
// The norm is that of the rounded h, which is what the backward pass reads; q is rounded once, from y in fp32 (through a bf16 y, as the two kernels of
// their own do it, values next to a border of e4m3 are rounded twice).
#include <cuda_fp8.h>

#include "cai_kernels.h"
#include "host_common.h"
#include "norm_kernels.cuh"
#include "sm100.cuh"

namespace cai {

struct NormQuantParams {
    const __nv_bfloat16 *x, *residual, *g;
    long long ldx, ldr;
    __nv_bfloat16 *h, *y;       // null: not wanted
    __nv_fp8_storage_t* q;
    float *scale, *rstd;
    int rows, H, warps;         // warps: those that share a row
    float eps;
};

// A row is shared by p.warps warps, each lane holding kChunks times eight of its columns in registers, 256 columns of a warp apart: sixteen lanes hold one
// block of the quantiser. A CTA takes blockDim / (32 * p.warps) rows.
template <int kChunks>
__global__ void __launch_bounds__(256)
add_rmsnorm_quant_kernel(const NormQuantParams p) {
    grid_dep_begin();
    __shared__ float part[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int grp = warp / p.warps, sub = warp - grp * p.warps, groups = (blockDim.x >> 5) / p.warps;
    const long long row = static_cast<long long>(blockIdx.x) * groups + grp;
    const bool live = row < p.rows;
    const int col0 = sub * kChunks * 256 + lane * 8;
    uint4 v[kChunks];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        v[c] = make_uint4(0, 0, 0, 0);
        const int col = col0 + c * 256;
        if (live && col < p.H) v[c] = *reinterpret_cast<const uint4*>(p.x + row * p.ldx + col);
    }
    if (p.residual) {
        uint4 r[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            r[c] = make_uint4(0, 0, 0, 0);
            const int col = col0 + c * 256;
            if (live && col < p.H) r[c] = *reinterpret_cast<const uint4*>(p.residual + row * p.ldr + col);
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            float a[8], b[8];
            unpack8(v[c], a);
            unpack8(r[c], b);
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] += b[e];
            v[c] = pack8(a);
        }
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int col = col0 + c * 256;
        if (p.h && live && col < p.H) *reinterpret_cast<uint4*>(p.h + row * p.H + col) = v[c];
        float f[8];
        unpack8(v[c], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += f[e] * f[e];
    }
    ss = warp_sum(ss);
    if (p.warps > 1) {
        if (lane == 0) part[warp] = ss;
        __syncthreads();
        ss = 0.f;
        for (int k = 0; k < p.warps; ++k) ss += part[grp * p.warps + k];
    }
    const float rr = 1.f / sqrtf(ss / p.H + p.eps);
    if (live && sub == 0 && lane == 0) p.rstd[row] = rr;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int col = col0 + c * 256;
        const bool in = live && col < p.H;
        float f[8], gg[8];
        unpack8(v[c], f);
        unpack8(in ? *reinterpret_cast<const uint4*>(p.g + col) : make_uint4(0, 0, 0, 0), gg);
        float amax = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            f[e] = f[e] * rr * gg[e];
            amax = fmaxf(amax, fabsf(f[e]));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const float s = amax > 0.f ? amax / 448.f : 1.f, inv = 1.f / s;
        if (in) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                w[k] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * k] * inv, f[2 * k + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            *reinterpret_cast<uint2*>(p.q + row * p.H + col) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
            if (p.y) *reinterpret_cast<uint4*>(p.y + row * p.H + col) = pack8(f);
            if ((lane & 15) == 0) p.scale[row * (p.H >> 7) + (col >> 7)] = s;
        }
    }
}

}  // namespace cai

using namespace cai;

CAI_API int cai_add_rmsnorm_quant(const void* x, long long ldx, const void* residual, long long ldr, const void* g, void* h, void* y, void* q,
                                  float* scale, float* rstd, int rows, int H, float eps, void* stream) {
    if (H <= 0 || H % 128 || H > 16384 || rows < 0) {
        set_last_error("add_rmsnorm_quant: needs a multiple of 128 of at most 16384 columns (%d columns, %d rows)", H, rows);
        return CAI_K_BAD_ARG;
    }
    const auto off = [](const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; };
    if ((ldx & 7) || (residual && (ldr & 7)) || off(x) || off(residual) || off(g) || off(h) || off(y) || off(q)) {
        set_last_error("add_rmsnorm_quant: rows have to start on 16 bytes");
        return CAI_K_BAD_ARG;
    }
    if (rows == 0) return CAI_K_OK;
    NormQuantParams p = {};
    p.x = static_cast<const __nv_bfloat16*>(x);
    p.residual = static_cast<const __nv_bfloat16*>(residual);
    p.g = static_cast<const __nv_bfloat16*>(g);
    p.ldx = ldx; p.ldr = ldr;
    p.h = static_cast<__nv_bfloat16*>(h);
    p.y = static_cast<__nv_bfloat16*>(y);
    p.q = static_cast<__nv_fp8_storage_t*>(q);
    p.scale = scale; p.rstd = rstd;
    p.rows = rows; p.H = H; p.eps = eps;
    const int pieces = (H + 255) / 256;
    const int chunks = pieces <= 1 ? 1 : pieces <= 2 ? 2 : pieces <= 32 ? 4 : 8;
    p.warps = (pieces + chunks - 1) / chunks;
    const int groups = 8 / p.warps;
    const unsigned grid = static_cast<unsigned>((rows + groups - 1) / groups), threads = groups * p.warps * 32;
    const auto kernel = chunks == 1 ? add_rmsnorm_quant_kernel<1> : chunks == 2 ? add_rmsnorm_quant_kernel<2>
                        : chunks == 4 ? add_rmsnorm_quant_kernel<4> : add_rmsnorm_quant_kernel<8>;
    const cudaError_t e = launch_early(kernel, grid, threads, 0, static_cast<cudaStream_t>(stream), p);
    if (e != cudaSuccess) {
        set_last_error("add_rmsnorm_quant launch failed: %s", cudaGetErrorString(e));
        return CAI_K_CUDA;
    }
    return CAI_K_OK;
}
