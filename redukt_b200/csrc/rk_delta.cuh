// The gated delta rule over state slots, one token of each stream (whole requests: rk_delta_chunk.cuh).
//
// Per value head, S in R^{dv x dk} (a slot's state, f32, row-major), a_t = exp(g_t):
//   u_t = b_t (v_t - a_t S_{t-1} k_t),  S_t = a_t S_{t-1} + u_t k_t^T,  o_t = scale S_t q_t
// The output needs no second pass over the state: S_t q = a_t S_{t-1} q + u_t (k.q), so both row
// products S_{t-1} k and S_{t-1} q come from one read of S_{t-1}.  What bounds it is that read and the
// write of S_t: 256 streams x 16 heads of 128 x 128 move 540 MB in 83 us, 6.5 TB/s.  Eight lanes share a
// row, so a row's loads are 128 contiguous bytes each and a product is summed in three shuffles; a warp
// has eight rows in flight.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace rk {
namespace delta {

constexpr float kNormEps = 1e-6f;

struct Args {
    const void *q, *k, *v;
    const float *g, *beta;
    const uint32_t *cu, *slots, *fresh;   // cu: requests only; fresh may be NULL (no stream starts from zero)
    uint32_t n, n_rows;                   // requests or streams; rows of q, k, v
    uint32_t hk, hv, dv;
    uint64_t ld_q, ld_k, ld_v, ld_g, ld_o;
    float scale;
    int l2norm;
    float* state;
    uint32_t n_slots;
    uint64_t slot_stride;
    void* out;
    uint32_t* err;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Sum over the 8 lanes that share a state row; every lane gets the same bits.
template <class F>
__device__ __forceinline__ F sum8(F x) {
    x += __shfl_xor_sync(0xFFFFFFFFu, x, 4);
    x += __shfl_xor_sync(0xFFFFFFFFu, x, 2);
    x += __shfl_xor_sync(0xFFFFFFFFu, x, 1);
    return x;
}

constexpr int kWarps = 4;                 // warps per block
constexpr int kPass = 2;                  // row quads per warp: 4 rows at a time, twice
constexpr int kRows = kWarps * 4 * kPass; // state rows per block

// Eight lanes hold one state row: lane l of the eight holds its float4s l, l + 8, ... so each
// load of the eight is 128 contiguous bytes.
template <int DK, class T>
struct Rows {
    static constexpr int kF4 = DK / 32;   // float4s of a row per lane
    float4 s[kPass][kF4];

    __device__ __forceinline__ void load(const float* st, int row0, uint32_t dv, int grp, int l, bool zero) {
#pragma unroll
        for (int p = 0; p < kPass; p++)
#pragma unroll
            for (int i = 0; i < kF4; i++) {
                const uint32_t r = row0 + p * 4 + grp;
                s[p][i] = (zero || r >= dv) ? make_float4(0.f, 0.f, 0.f, 0.f)
                                            : *reinterpret_cast<const float4*>(st + (size_t)r * DK + 4 * (l + 8 * i));
            }
    }
    __device__ __forceinline__ void store(float* st, int row0, uint32_t dv, int grp, int l) const {
#pragma unroll
        for (int p = 0; p < kPass; p++)
#pragma unroll
            for (int i = 0; i < kF4; i++) {
                const uint32_t r = row0 + p * 4 + grp;
                if (r < dv) *reinterpret_cast<float4*>(st + (size_t)r * DK + 4 * (l + 8 * i)) = s[p][i];
            }
    }
    // One token: k and q are rows of DK elements, v and o of dv.
    __device__ __forceinline__ void token(const Args& a, const T* q, const T* k, const T* v, T* o, float g, float beta,
                                          int row0, int grp, int l) {
        // k.q in 64 bits: from zero state the output is u (k.q) alone, and a near-orthogonal pair
        // would leave it only the rounding errors of a 32-bit sum
        float kk[4 * kF4], qq[4 * kF4], k2 = 0.f, q2 = 0.f;
        double kqd = 0.0;
#pragma unroll
        for (int i = 0; i < 4 * kF4; i++) {
            const int c = 4 * (l + 8 * (i >> 2)) + (i & 3);
            kk[i] = to_f32(k[c]);
            qq[i] = to_f32(q[c]);
            k2 = fmaf(kk[i], kk[i], k2);
            q2 = fmaf(qq[i], qq[i], q2);
            kqd = fma((double)kk[i], (double)qq[i], kqd);
        }
        const float kq = (float)sum8(kqd);
        float rk = 1.f, rq = 1.f;
        if (a.l2norm) {
            rk = 1.f / sqrtf(sum8(k2) + kNormEps);
            rq = 1.f / sqrtf(sum8(q2) + kNormEps);
        }
        const float alpha = expf(g);
#pragma unroll
        for (int p = 0; p < kPass; p++) {
            float sk = 0.f, sq = 0.f;
#pragma unroll
            for (int i = 0; i < kF4; i++) {
                const float4 x = s[p][i];
                sk = fmaf(x.x, kk[4 * i], fmaf(x.y, kk[4 * i + 1], fmaf(x.z, kk[4 * i + 2], fmaf(x.w, kk[4 * i + 3], sk))));
                sq = fmaf(x.x, qq[4 * i], fmaf(x.y, qq[4 * i + 1], fmaf(x.z, qq[4 * i + 2], fmaf(x.w, qq[4 * i + 3], sq))));
            }
            sk = sum8(sk);
            sq = sum8(sq);
            const uint32_t r = row0 + p * 4 + grp;
            const float vr = r < a.dv ? to_f32(v[r]) : 0.f;
            const float u = beta * (vr - alpha * (rk * sk));
            const float ur = u * rk;   // the state is updated with the normalised key
#pragma unroll
            for (int i = 0; i < kF4; i++) {
                float4& x = s[p][i];
                x.x = fmaf(alpha, x.x, ur * kk[4 * i]);
                x.y = fmaf(alpha, x.y, ur * kk[4 * i + 1]);
                x.z = fmaf(alpha, x.z, ur * kk[4 * i + 2]);
                x.w = fmaf(alpha, x.w, ur * kk[4 * i + 3]);
            }
            if (l == 0 && r < a.dv) put(o + r, a.scale * rq * fmaf(alpha, sq, ur * kq));
        }
    }
};

// One token of each stream.  grid (ceil(dv / kRows), hv, streams).  Bound by the state's bytes.
template <int DK, class T>
__global__ void __launch_bounds__(kWarps * 32) k_delta_step(Args a) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = lane >> 3, l = lane & 7;
    const int row0 = (blockIdx.x * kWarps + warp) * 4 * kPass;
    const uint32_t h = blockIdx.y;
    const uint64_t b = blockIdx.z;
    const uint32_t slot = a.slots[b];
    T* o = (T*)a.out + b * a.ld_o + (uint64_t)h * a.dv;
    if (slot >= a.n_slots) {   // only this stream is rejected: its state is not touched
        for (uint32_t r = blockIdx.x * kRows + threadIdx.x; r < min(a.dv, (blockIdx.x + 1) * kRows); r += blockDim.x) put(o + r, 0.f);
        if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.err, 1u);
        return;
    }
    float* st = a.state + slot * a.slot_stride + (uint64_t)h * a.dv * DK;
    Rows<DK, T> R;
    R.load(st, row0, a.dv, grp, l, a.fresh && a.fresh[b]);
    const uint32_t hq = h / (a.hv / a.hk);
    R.token(a, (const T*)a.q + b * a.ld_q + (uint64_t)hq * DK, (const T*)a.k + b * a.ld_k + (uint64_t)hq * DK,
            (const T*)a.v + b * a.ld_v + (uint64_t)h * a.dv, o, a.g[b * a.ld_g + h], a.beta[b * a.ld_g + h], row0, grp, l);
    R.store(st, row0, a.dv, grp, l);
}

}  // namespace delta
}  // namespace rk
