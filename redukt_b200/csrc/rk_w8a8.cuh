// Matrix product in 8-bit integers with a scale per token and per output channel.
//
//   s_t = max_k |x_tk| * (1 / 127) (1 for a zero row),  q_tk = clamp(round_half_away(x_tk * (1 / s_t)), +-127)
//   y_tn = float(sum_k q_tk w_nk) * (w_scale_n * s_t)
// Each f32 operation is correctly rounded and the sum is exact in int32, so every kernel here gives
// the same bits.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace rk {
namespace w8 {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

__device__ __forceinline__ int quant_one(float v, float inv) {
    float r = roundf(__fmul_rn(v, inv));
    r = (r != r) ? 0.0f : fminf(fmaxf(r, -127.0f), 127.0f);
    return (int)r;
}

__device__ __forceinline__ float row_scale(float amax) { return amax > 0.f ? __fmul_rn(amax, 1.f / 127.f) : 1.f; }

// One block per token: the row's largest magnitude (exact in any order), then its 8-bit values.
// The row's tail up to ld_q's multiple of 16 is not written.
template <class T>
__global__ void __launch_bounds__(256) k_quant_tokens(const T* __restrict__ x, uint32_t k, uint64_t ld_x, int8_t* __restrict__ q,
                                                      uint64_t ld_q, float* __restrict__ scale) {
    __shared__ float part[8];
    const uint64_t row = blockIdx.x;
    const T* xr = x + row * ld_x;
    float m = 0.f;
    for (uint32_t i = threadIdx.x; i < k; i += blockDim.x) m = fmaxf(m, fabsf(to_f32(xr[i])));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    m = part[0];
#pragma unroll
    for (int i = 1; i < 8; i++) m = fmaxf(m, part[i]);
    const float s = row_scale(m);
    const float inv = __fdiv_rn(1.f, s);
    for (uint32_t i = threadIdx.x; i < k; i += blockDim.x) q[row * ld_q + i] = (int8_t)quant_one(to_f32(xr[i]), inv);
    if (threadIdx.x == 0) scale[row] = s;
}

struct Args {
    const int8_t* a;
    const float* as;
    const int8_t* w;
    const float* ws;
    uint64_t ld_a, ld_w, ld_o;
    uint32_t m, n, k;
    void* out;
};

// 64 x 64 outputs per block, 4 x 4 per thread, dp4a over K in steps of 64 bytes.
template <class T>
__global__ void __launch_bounds__(256) k_w8a8_dp4a(Args a) {
    __shared__ int sa[64][17], sw[64][17];
    const uint32_t n0 = blockIdx.x * 64, m0 = blockIdx.y * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < a.k; k0 += 64) {
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const uint32_t r = i >> 4, c = k0 + (i & 15) * 4;
            uint32_t va = 0, vw = 0;
            for (int j = 0; j < 4; j++) {
                if (c + j >= a.k) break;
                if (m0 + r < a.m) va |= (uint32_t)(uint8_t)a.a[(m0 + r) * a.ld_a + c + j] << (8 * j);
                if (n0 + r < a.n) vw |= (uint32_t)(uint8_t)a.w[(n0 + r) * a.ld_w + c + j] << (8 * j);
            }
            sa[r][i & 15] = (int)va;
            sw[r][i & 15] = (int)vw;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 16; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(sa[ty + 16 * i][c], sw[tx + 16 * j][c], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const uint32_t r = m0 + ty + 16 * i, c = n0 + tx + 16 * j;
            if (r < a.m && c < a.n)
                put((T*)a.out + r * a.ld_o + c, __fmul_rn((float)acc[i][j], __fmul_rn(a.ws[c], a.as[r])));
        }
}

}  // namespace w8
}  // namespace rk
