// norm_e4m3.cu - RMSNorm in front of a block-scaled e4m3 product: the residual's addition, the norm and the quantiser in one pass.
//
//   h = bf16(x + residual)     rstd = (mean(h^2) + eps)^(-1/2)     y = h * rstd * g
//   s[row, b] = max |y| of the row's 128 columns b / 448 (1 where they are all zero)     q = e4m3(y / s)
//
// The norm is that of the rounded h, which is what the backward pass reads; q is rounded to e4m3 once, from y in fp32 times the reciprocal of s (through a bf16 y, as the two kernels of
// their own do it, values next to a border of e4m3 are rounded twice).
// Measured on a B200: 16384 x 4096 with residual and y 89 us (9 bytes an element, 6.8 TB/s: the rate of a copy), without either 48 (3 bytes, 4.2 TB/s:
// issue slots 69 % busy, DRAM 42 %; a CTA loads its rows and then computes, so that the two alternate, and each row reads and unpacks the gain anew), 8192 x 2048 24.7, 1777 x 1408 without either 3.8, 256 x 256 1.8, where a launch's own latencies are all there is.
#include <cuda_fp8.h>

#include "cai_kernels.h"
#include "f32x2.cuh"
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

__device__ __forceinline__ uint64_t bf16x2_pair(uint32_t v) { return pair_of(bf16_lo(v), bf16_hi(v)); }

// The scale of a block whose largest magnitude is `amax`. Where 1 / scale would leave fp32's range the block is near enough to zero for a scale that does not.
__device__ __forceinline__ float block_scale(float amax) { return amax > 0.f ? fmaxf(amax, 0x1p-100f) / 448.f : 1.f; }

// A row is shared by p.warps warps, each lane holding kChunks times eight of its columns in registers, 256 columns of a warp apart: sixteen lanes hold one
// block of the quantiser. A CTA takes blockDim / (32 * p.warps) rows. With the residual and y this is bound by its 9 bytes an element, without them, 3 bytes, more by
// its instructions: hence the arithmetic on pairs, and (kChunks = 4) the four blocks' maxima reduced together: a lane that gives two of its
// four away at the first step and one at the second is left with one, whose scale and reciprocal it computes for the sixteen.
template <int kChunks>
__global__ void __launch_bounds__(512, 2)
add_rmsnorm_quant_kernel(const NormQuantParams p) {
    grid_dep_begin();
    __shared__ float part[16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int grp = warp / p.warps, sub = warp - grp * p.warps, groups = (blockDim.x >> 5) / p.warps;
    const long long row = static_cast<long long>(blockIdx.x) * groups + grp;
    const bool live = row < p.rows;
    const int col0 = sub * kChunks * 256 + lane * 8;
    uint4 v[kChunks], g[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        v[c] = make_uint4(0, 0, 0, 0);
        const int col = col0 + c * 256;
        if (live && col < p.H) v[c] = *reinterpret_cast<const uint4*>(p.x + row * p.ldx + col);
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int col = col0 + c * 256;
        g[c] = col < p.H ? *reinterpret_cast<const uint4*>(p.g + col) : make_uint4(0, 0, 0, 0);
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
    uint64_t ss2 = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int col = col0 + c * 256;
        if (p.h && live && col < p.H) *reinterpret_cast<uint4*>(p.h + row * p.H + col) = v[c];
        const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint64_t f = bf16x2_pair(w[k]);
            ss2 = fma2(f, f, ss2);
        }
    }
    const float2 s01 = floats_of(ss2);
    float ss = warp_sum(s01.x + s01.y);
    if (p.warps > 1) {
        if (lane == 0) part[warp] = ss;
        __syncthreads();
        ss = 0.f;
        for (int k = 0; k < p.warps; ++k) ss += part[grp * p.warps + k];
    }
    const float rr = 1.f / sqrtf(ss / p.H + p.eps);
    if (live && sub == 0 && lane == 0) p.rstd[row] = rr;
    const uint64_t rr2 = pair_of(rr, rr);
    uint64_t y[kChunks][4];
    float amax[kChunks], inv[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w}, gw[4] = {g[c].x, g[c].y, g[c].z, g[c].w};
        amax[c] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            y[c][k] = mul2(mul2(bf16x2_pair(w[k]), rr2), bf16x2_pair(gw[k]));
            const float2 f = floats_of(y[c][k]);
            amax[c] = fmaxf(amax[c], fmaxf(fabsf(f.x), fabsf(f.y)));
        }
    }
    auto put_scale = [&](int c, float s) {
        const int col = sub * kChunks * 256 + c * 256 + (lane >> 4) * 128;
        if (live && col < p.H) p.scale[row * (p.H >> 7) + (col >> 7)] = s;
    };
    if constexpr (kChunks == 4) {
        // lane bit 3 decides which two of the four a lane keeps, bit 2 which one of them
        const bool b3 = lane & 8, b2 = lane & 4;
        const float k0 = fmaxf(b3 ? amax[2] : amax[0], __shfl_xor_sync(0xffffffffu, b3 ? amax[0] : amax[2], 8));
        const float k1 = fmaxf(b3 ? amax[3] : amax[1], __shfl_xor_sync(0xffffffffu, b3 ? amax[1] : amax[3], 8));
        float m = fmaxf(b2 ? k1 : k0, __shfl_xor_sync(0xffffffffu, b2 ? k0 : k1, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const float s = block_scale(m), one = 1.f / s;
        if (!(lane & 3)) put_scale((lane >> 2) & 3, s);
#pragma unroll
        for (int c = 0; c < 4; ++c) inv[c] = __shfl_sync(0xffffffffu, one, (lane & 16) + c * 4);
    } else {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax[c] = fmaxf(amax[c], __shfl_xor_sync(0xffffffffu, amax[c], o));
            const float s = block_scale(amax[c]);
            inv[c] = 1.f / s;
            if (!(lane & 15)) put_scale(c, s);
        }
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int col = col0 + c * 256;
        if (!live || col >= p.H) continue;
        const uint64_t inv2 = pair_of(inv[c], inv[c]);
        uint32_t w[4], yw[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            w[k] = __nv_cvt_float2_to_fp8x2(floats_of(mul2(y[c][k], inv2)), __NV_SATFINITE, __NV_E4M3);
            const float2 f = floats_of(y[c][k]);
            yw[k] = pack_bf16(f.x, f.y);
        }
        *reinterpret_cast<uint2*>(p.q + row * p.H + col) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
        if (p.y) *reinterpret_cast<uint4*>(p.y + row * p.H + col) = make_uint4(yw[0], yw[1], yw[2], yw[3]);
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
    if (!x || !g || !q || !scale || !rstd) {
        set_last_error("add_rmsnorm_quant: an address is null");
        return CAI_K_BAD_ARG;
    }
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
    // Four times eight columns a lane; fewer, on more warps, where the rows alone do not fill the SMs. A CTA has eight warps, sixteen where a row needs more.
    const int pieces = (H + 255) / 256, sms = sm_count(current_device());
    p.warps = (pieces + 3) / 4;
    while (p.warps < 8 && p.warps < pieces && static_cast<long long>(rows) * p.warps < 8 * sms) ++p.warps;
    const int chunks = (pieces + p.warps - 1) / p.warps;
    const int groups = p.warps > 8 ? 1 : 8 / p.warps;
    const unsigned grid = static_cast<unsigned>((rows + groups - 1) / groups), threads = groups * p.warps * 32;
    const auto kernel = chunks == 1 ? add_rmsnorm_quant_kernel<1> : chunks == 2 ? add_rmsnorm_quant_kernel<2> : chunks == 3 ? add_rmsnorm_quant_kernel<3>
                                                                                              : add_rmsnorm_quant_kernel<4>;
    const cudaError_t e = launch_early(kernel, grid, threads, 0, static_cast<cudaStream_t>(stream), p);
    if (e != cudaSuccess) {
        set_last_error("add_rmsnorm_quant launch failed: %s", cudaGetErrorString(e));
        return CAI_K_CUDA;
    }
    return CAI_K_OK;
}
