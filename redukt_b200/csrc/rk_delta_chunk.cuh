// The gated delta rule over whole windows, 64 tokens at a time, on the warp-level tensor cores.
//
// With c_i the running sum of the log decays inside a chunk and S_0 the state before it:
//   A_ij = b_i e^{c_i - c_j} k_i.k_j  (j < i),   (I + A) U = b (V - e^{c} K S_0^T)
//   O = scale (e^{c} Q S_0^T + [e^{c_i - c_j} q_i.k_j]_{j <= i} U)
//   S_64 = e^{c_64} S_0 + sum_j e^{c_64 - c_j} u_j k_j^T
// Every exponent is a difference c_i - c_j with j <= i, so nothing overflows however strong the decay
// is.  c is summed in 64 bits and kept as two floats (times log2 e).
//
// Split: one block of 4 warps per (request, value head, 64 state rows); a state row depends on no
// other, so a warp keeps 16 of them in registers as mma accumulators for the whole request, and every
// product of the chain (X = S K^T, the solve, O, the update) turns accumulators straight into the next
// product's A operand.  Only K, Q, A and P pass through shared memory.  The triangular system is
// solved by 16-token blocks (their 16 x 16 diagonal blocks are inverted by substitution, the rest is
// subtracted), which stays accurate where the whole inverse would not (equal keys).
//
// Precision: an f32 operand is split into two f16 planes hi + lo after scaling its row by a power of
// two that puts the row's largest value in [2^14, 2^15): 22 bits of every value down to 2^-28 of that
// largest, and no overflow.  f32 x f32 is hi hi + hi lo + lo hi; a bf16 k or q is one f16 plane
// exactly, down to 2^-28 of its row's largest.  Sums are f32.
#pragma once
#include <cuda_fp16.h>

#include "rk_delta.cuh"
#include "rk_ptx.cuh"

namespace rk {
namespace delta {

constexpr int kC = 64;              // tokens per chunk
constexpr int kCWarps = 4;
constexpr int kCThreads = kCWarps * 32;
constexpr int kVRows = 16 * kCWarps;  // state rows per block

// Lower triangle of a 64 x 64 matrix by strips of 16 rows: strip r is 16 (r + 1) wide; a row's stride is
// an odd number of 16-byte units, so ldmatrix reads 8 rows without a bank conflict.
constexpr int kStripHalves = 16 * (24 + 40 + 56 + 72);
__device__ __forceinline__ int strip_at(int row, int col) {
    const int r = row >> 4;
    return 16 * (8 * r + 8 * r * (r + 1)) + (row & 15) * (16 * r + 24) + col;
}

constexpr int kDiagLd = 20;         // rows of 16 floats on 16 bytes, two columns apart in other banks

template <int DK, class T>
struct ChunkCfg {
    static constexpr bool kF32 = sizeof(T) == 4;
    static constexpr int KP = kF32 ? 2 : 1;     // planes of k and q
    static constexpr int LD = DK + 8;           // halves per row of a plane
    static constexpr int kMinBlocks = DK == 64 ? 3 : 2;
};

template <int DK, class T>
struct alignas(16) ChunkSmem {
    using Cfg = ChunkCfg<DK, T>;
    __half k[Cfg::KP][kC * Cfg::LD];
    __half q[Cfg::KP][kC * Cfg::LD];
    __half m[2][kStripHalves];          // A below the diagonal blocks, their inverses on them
    __half p[2][kStripHalves];
    float diag[kCWarps][16 * kDiagLd];  // a diagonal block, transposed: [column][row]
    float sk[kC], sq[kC];               // row scales of the planes, norms folded in
    float chi[kC], clo[kC];             // c * log2(e) in two floats
    float beta[kC];
    float ak[kC], cq[kC], wk[kC];       // factors of X, O and the update, per token
    float rf[kC];                       // e^{c_i - c_ref}, ref = the token before i's strip
    float cf[3][kC];                    // strip r + 1: e^{c_ref - c_j} times the key's scale
    float ascale[4][kC], pscale[4][kC]; // scales of a row of each 16 x 16 block of A and P
    float dblk[kCWarps];                // scale of each inverted block
    float gamma;
};

struct ChunkArgs {
    Args a;
    const uint32_t* blocks;       // (request, index) of each table block
    uint32_t block, merge;        // tokens per table block; table blocks per segment
    float *b_seg, *m_seg, *s_in;  // per segment and head: end state from zero, transition, start state
};

// A cut request: segments of block * merge tokens.  Over a segment a state row s becomes s M + b with M
// and b of that segment alone (M: what the rows of the identity become with v = 0; b: what zero
// becomes), so three launches replace the chain: the segments' M and b side by side, the start
// states one after the other (k_delta_scan, one small product per segment), the segments with
// outputs side by side.
// Number of a segment in the workspace: different for every (request, index / merge), and below
// n_rows / (block * merge) + n, because a request of l tokens has at most l / seg + 1 segments.
__device__ __forceinline__ uint64_t segment_id(const ChunkArgs& c, uint64_t first_row, uint32_t req, uint32_t seg_index) {
    return first_row / ((uint64_t)c.block * c.merge) + req + seg_index;
}

// 2^(14 - e) for a largest magnitude in [2^e, 2^(e+1)), and its inverse; finite for every m.
__device__ __forceinline__ float row_pow(float m, float& inv) {
    const int e = (int)(__float_as_uint(m) >> 23);
    const int s = min(268 - e, 253);
    inv = m > 0.f ? __uint_as_float((uint32_t)(254 - s) << 23) : 1.f;
    return m > 0.f ? __uint_as_float((uint32_t)s << 23) : 1.f;
}
// max that keeps a NaN out of the scale; the NaN itself stays in the value
__device__ __forceinline__ float amax(float m, float x) { return fmaxf(m, fabsf(x)); }
__device__ __forceinline__ float quad_max(float m) {
    m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    return fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
}

// two scaled values as one register of each plane
__device__ __forceinline__ uint32_t pack_hi(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const __half* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(tc::smem_u32(p)) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const __half* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(tc::smem_u32(p)) : "memory");
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// One row of DK values of type T to f16 planes: 8 lanes a row, lane l of the eight takes the 16-byte
// vectors l, l + 8, ...
template <int DK, class T>
struct RowLoad {
    static constexpr int N = 16 / sizeof(T), NV = DK / N / 8;
    uint4 raw[NV];
    __device__ __forceinline__ void load(const T* p, int l) {
#pragma unroll
        for (int i = 0; i < NV; i++) raw[i] = *reinterpret_cast<const uint4*>(p + (l + 8 * i) * N);
    }
    __device__ __forceinline__ void load_single(const T* p, int l) {   // any alignment
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < N; c++) reinterpret_cast<T*>(&raw[i])[c] = p[(l + 8 * i) * N + c];
    }
    __device__ __forceinline__ void clear_unless(bool live) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            raw[i].x = live ? raw[i].x : 0u;
            raw[i].y = live ? raw[i].y : 0u;
            raw[i].z = live ? raw[i].z : 0u;
            raw[i].w = live ? raw[i].w : 0u;
        }
    }
    __device__ __forceinline__ float get(int i, int c) const { return to_f32(reinterpret_cast<const T*>(&raw[i])[c]); }
    __device__ __forceinline__ void sums(float& m, float& ss) const {   // this lane's part
        m = ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < N; c++) {
                m = amax(m, get(i, c));
                ss = fmaf(get(i, c), get(i, c), ss);
            }
    }
    __device__ __forceinline__ void put(__half* hi, __half* lo, float s, int l) const {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            uint32_t h[N / 2], w[N / 2];
#pragma unroll
            for (int c = 0; c < N / 2; c++) {
                if constexpr (sizeof(T) == 4) split2(s * get(i, 2 * c), s * get(i, 2 * c + 1), h[c], w[c]);
                else h[c] = pack_hi(s * get(i, 2 * c), s * get(i, 2 * c + 1));
            }
            const int at = (l + 8 * i) * N;
            if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<uint2*>(hi + at) = make_uint2(h[0], h[1]);
                *reinterpret_cast<uint2*>(lo + at) = make_uint2(w[0], w[1]);
            } else {
                *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
            }
        }
    }
};

// Four rows of each 8-lane group: r, r + 4, r + 8, r + 12 of the warp's 16.
template <int DK, class T>
__device__ __forceinline__ void put_rows(RowLoad<DK, T> (&x)[4], __half* hi, __half* lo, int ld, float* scale, int row, int len, bool l2norm, int l) {
    float m[4], ss[4], s[4], inv[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[i].clear_unless(row + 4 * i < len);
        x[i].sums(m[i], ss[i]);
    }
#pragma unroll
    for (int o = 4; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < 4; i++) m[i] = fmaxf(m[i], __shfl_xor_sync(0xFFFFFFFFu, m[i], o));
    if (l2norm) {
#pragma unroll
        for (int o = 4; o; o >>= 1)
#pragma unroll
            for (int i = 0; i < 4; i++) ss[i] += __shfl_xor_sync(0xFFFFFFFFu, ss[i], o);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        s[i] = row_pow(m[i], inv[i]);
        if (l2norm) inv[i] *= 1.f / sqrtf(ss[i] + kNormEps);
        x[i].put(hi + (row + 4 * i) * ld, lo + (row + 4 * i) * ld, s[i], l);
        if (l == 0) scale[row + 4 * i] = inv[i];
    }
}

// Fills the chunk's shared operands: planes and scales of k and q, decay factors, A, its inverted
// diagonal blocks, and P.  All warps; ends with a barrier.
template <int DK, class T, bool kOut>
__device__ __forceinline__ void prepare_chunk(ChunkSmem<DK, T>& sm, const Args& a, uint64_t t0, int len, uint32_t h, uint32_t hq,
                                              bool wide) {
    using Cfg = ChunkCfg<DK, T>;
    constexpr int LD = Cfg::LD, KP = Cfg::KP;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = lane >> 3, l = lane & 7, g = lane >> 2, t = lane & 3;
    {
        const T* kp = (const T*)a.k + t0 * a.ld_k + (uint64_t)hq * DK;
        const T* qp = (const T*)a.q + t0 * a.ld_q + (uint64_t)hq * DK;
        const int row = warp * 16 + grp;
        RowLoad<DK, T> rk[4], rq[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {   // rows past the end read the last one and are cleared
            const uint32_t r = min(row + 4 * i, len - 1);
            if (wide) {
                rk[i].load(kp + r * a.ld_k, l);
                if (kOut) rq[i].load(qp + r * a.ld_q, l);
            } else {
                rk[i].load_single(kp + r * a.ld_k, l);
                if (kOut) rq[i].load_single(qp + r * a.ld_q, l);
            }
        }
        if (warp == 0) {   // tokens 2 lane, 2 lane + 1
            double c0 = 0.0, c1 = 0.0;
            float b0 = 0.f, b1 = 0.f;
            const int i0 = 2 * lane;
            if (i0 < len) {
                const float x = a.g[(t0 + i0) * a.ld_g + h];
                c0 = x < -1000.f ? -1000.0 : (double)x;   // e^-1000 is 0 in f32; -inf - -inf would be NaN
                b0 = a.beta[(t0 + i0) * a.ld_g + h];
            }
            if (i0 + 1 < len) {
                const float x = a.g[(t0 + i0 + 1) * a.ld_g + h];
                c1 = x < -1000.f ? -1000.0 : (double)x;
                b1 = a.beta[(t0 + i0 + 1) * a.ld_g + h];
            }
            double s = c0 + c1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xFFFFFFFFu, s, o);
                if (lane >= o) s += y;
            }
            const double e1 = s * 1.4426950408889634, e0 = (s - c1) * 1.4426950408889634;   // log2(e)
            sm.chi[i0] = (float)e0;
            sm.clo[i0] = (float)(e0 - (double)(float)e0);
            sm.chi[i0 + 1] = (float)e1;
            sm.clo[i0 + 1] = (float)(e1 - (double)(float)e1);
            sm.beta[i0] = b0;
            sm.beta[i0 + 1] = b1;
        }
        put_rows<DK, T>(rk, sm.k[0], sm.k[KP - 1], LD, sm.sk, row, len, a.l2norm, l);
        if (kOut) put_rows<DK, T>(rq, sm.q[0], sm.q[KP - 1], LD, sm.sq, row, len, a.l2norm, l);
    }
    __syncthreads();
    if (threadIdx.x < kC) {
        const int i = threadIdx.x, ref = (i & ~15) - 1;
        const float c = sm.chi[i] + sm.clo[i], e = exp2f(c);
        const float w = exp2f((sm.chi[kC - 1] - sm.chi[i]) + (sm.clo[kC - 1] - sm.clo[i]));
        sm.ak[i] = e * sm.sk[i];
        sm.wk[i] = w * sm.sk[i];
        if (kOut) sm.cq[i] = a.scale * e * sm.sq[i];
        if (i == kC - 1) sm.gamma = e;
        sm.rf[i] = ref < 0 ? 1.f : exp2f((sm.chi[i] - sm.chi[max(ref, 0)]) + (sm.clo[i] - sm.clo[max(ref, 0)]));
    } else {
        const int j = threadIdx.x - kC;
#pragma unroll
        for (int r = 1; r < 4; r++)
            if (j < 16 * r) sm.cf[r - 1][j] = sm.sk[j] * exp2f((sm.chi[16 * r - 1] - sm.chi[j]) + (sm.clo[16 * r - 1] - sm.clo[j]));
    }
    // Strip r of a product is rows 16 r .. 16 r + 15 against tokens 0 .. 16 r + 15.  Warp w does strip w of
    // K K^T and strip 3 - w of Q K^T, five 16 x 16 blocks for every warp: slot 0 the diagonal block of the
    // first, slot 1 that of the second, slots 2-4 the blocks beside them.
    const int rg = warp, rh = kCWarps - 1 - warp;
    float acc[5][2][4];
#pragma unroll
    for (int s = 0; s < 5; s++)
#pragma unroll
        for (int c = 0; c < 4; c++) acc[s][0][c] = acc[s][1][c] = 0.f;
    {
        const int arow = (lane & 7) + ((lane >> 3) & 1) * 8, acol = (lane >> 4) * 8;
        const int brow = (lane & 7) + (lane >> 4) * 8, bcol = ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int ks = 0; ks < DK / 16; ks++) {
            uint32_t fk[4], fkl[4], fq[4], fql[4];
            ldsm4(fk, &sm.k[0][(16 * rg + arow) * LD + ks * 16 + acol]);
            if (KP == 2) ldsm4(fkl, &sm.k[KP - 1][(16 * rg + arow) * LD + ks * 16 + acol]);
            if (kOut) {
                ldsm4(fq, &sm.q[0][(16 * rh + arow) * LD + ks * 16 + acol]);
                if (KP == 2) ldsm4(fql, &sm.q[KP - 1][(16 * rh + arow) * LD + ks * 16 + acol]);
            }
#pragma unroll
            for (int s = 0; s < 5; s++) {
                const bool key = s == 0 || (s > 1 && s - 2 < warp);
                if (!kOut && !key) continue;
                const int nb = s == 0 ? rg : s == 1 ? rh : s - 2 < warp ? s - 2 : s - 2 - warp;
                uint32_t fa[4], fl[4], fb[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    fa[c] = !kOut || key ? fk[c] : fq[c];
                    if (KP == 2) fl[c] = !kOut || key ? fkl[c] : fql[c];
                }
                const int off = (nb * 16 + brow) * LD + ks * 16 + bcol;
                ldsm4(fb, &sm.k[0][off]);
                if (KP == 2) {
                    uint32_t fw[4];
                    ldsm4(fw, &sm.k[KP - 1][off]);
                    mma_f16(acc[s][0], fa, fw[0], fw[1]);
                    mma_f16(acc[s][1], fa, fw[2], fw[3]);
                    mma_f16(acc[s][0], fl, fb[0], fb[1]);
                    mma_f16(acc[s][1], fl, fb[2], fb[3]);
                }
                mma_f16(acc[s][0], fa, fb[0], fb[1]);
                mma_f16(acc[s][1], fa, fb[2], fb[3]);
            }
        }
    }
    __syncthreads();   // the factors below
    {
        const int ig = 16 * rg + g, ih = 16 * rh + g;
        const float kg0 = sm.beta[ig] * sm.sk[ig], kg1 = sm.beta[ig + 8] * sm.sk[ig + 8];
        const float kh0 = kOut ? a.scale * sm.sq[ih] : 0.f, kh1 = kOut ? a.scale * sm.sq[ih + 8] : 0.f;
        // diagonal blocks: every pair's own exponent (column 8 n + 2 t + c of the block, rows g and g + 8)
#pragma unroll
        for (int s = 0; s < (kOut ? 2 : 1); s++) {
            const int i0 = s ? ih : ig, base = 16 * (s ? rh : rg);
            const float r0 = s ? kh0 : kg0, r1 = s ? kh1 : kg1;
            const float ch0 = sm.chi[i0], cl0 = sm.clo[i0], ch1 = sm.chi[i0 + 8], cl1 = sm.clo[i0 + 8];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int jj = 8 * n + 2 * t + c, j = base + jj;
                    const float kj = sm.sk[j], h = sm.chi[j], w = sm.clo[j];
                    const float e0 = exp2f((ch0 - h) + (cl0 - w)), e1 = exp2f((ch1 - h) + (cl1 - w));
                    const bool in0 = s ? jj <= g : jj < g, in1 = s ? jj <= g + 8 : jj < g + 8;
                    acc[s][n][c] = in0 ? acc[s][n][c] * (r0 * kj) * e0 : 0.f;
                    acc[s][n][2 + c] = in1 ? acc[s][n][2 + c] * (r1 * kj) * e1 : 0.f;
                    if (s == 0) {
                        sm.diag[warp][jj * kDiagLd + g] = acc[0][n][c];
                        sm.diag[warp][jj * kDiagLd + g + 8] = acc[0][n][2 + c];
                    }
                }
        }
        // the blocks beside them: a factor per row and one per column
        const float fg0 = kg0 * sm.rf[ig], fg1 = kg1 * sm.rf[ig + 8], fh0 = kh0 * sm.rf[ih], fh1 = kh1 * sm.rf[ih + 8];
#pragma unroll
        for (int s = 1; s < 5; s++) {
            const bool key = s > 1 && s - 2 < warp;
            if (!kOut && !key) continue;
            const int nb = s == 1 ? rh : key ? s - 2 : s - 2 - warp;
            const int r = key ? rg : rh, i0 = 16 * r + g;
            if (s > 1) {
                const float* cf = sm.cf[r - 1] + 16 * nb + 2 * t;
                const float r0 = key ? fg0 : fh0, r1 = key ? fg1 : fh1;
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        acc[s][n][c] *= r0 * cf[8 * n + c];
                        acc[s][n][2 + c] *= r1 * cf[8 * n + c];
                    }
            }
            float m0 = 0.f, m1 = 0.f, v0, v1;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    m0 = amax(m0, acc[s][n][c]);
                    m1 = amax(m1, acc[s][n][2 + c]);
                }
            const float p0 = row_pow(quad_max(m0), v0), p1 = row_pow(quad_max(m1), v1);
            float* sc = key ? sm.ascale[nb] : sm.pscale[nb];
            if (t == 0) {
                sc[i0] = v0;
                sc[i0 + 8] = v1;
            }
            __half* hi = key ? sm.m[0] : sm.p[0];
            __half* lo = key ? sm.m[1] : sm.p[1];
            const int at = strip_at(i0, 16 * nb + 2 * t), down = 8 * (16 * r + 24);
#pragma unroll
            for (int n = 0; n < 2; n++) {
                uint32_t x, y;
                split2(acc[s][n][0] * p0, acc[s][n][1] * p0, x, y);
                *reinterpret_cast<uint32_t*>(hi + at + 8 * n) = x;
                *reinterpret_cast<uint32_t*>(lo + at + 8 * n) = y;
                split2(acc[s][n][2] * p1, acc[s][n][3] * p1, x, y);
                *reinterpret_cast<uint32_t*>(hi + at + down + 8 * n) = x;
                *reinterpret_cast<uint32_t*>(lo + at + down + 8 * n) = y;
            }
        }
    }
    __syncwarp();
    {   // (I + A_ww)^-1 by forward substitution, lane c < 16 its column c (lanes 16.. repeat it)
        const int c = lane & 15;
        const float* at = sm.diag[warp];
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = i == c ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < 15; j++) {
            float col[16];
#pragma unroll
            for (int i = (j + 1) & ~3; i < 16; i += 4) {
                const float4 f = *reinterpret_cast<const float4*>(at + j * kDiagLd + i);
                col[i] = f.x, col[i + 1] = f.y, col[i + 2] = f.z, col[i + 3] = f.w;
            }
#pragma unroll
            for (int i = j + 1; i < 16; i++) x[i] = fmaf(-col[i], x[j], x[i]);
        }
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) m = amax(m, x[i]);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        float inv;
        const float s = row_pow(m, inv);
        if (lane == 0) sm.dblk[warp] = inv;
        if (lane < 16)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float y = x[i] * s;
                const __half hh = __float2half_rn(y);
                const int at0 = strip_at(16 * warp + i, 16 * warp + c);
                sm.m[0][at0] = hh;
                sm.m[1][at0] = __float2half_rn(y - __half2float(hh));
            }
    }
    __syncthreads();
}

// f32 accumulators of one 16-column group (two tiles) -> A operand planes, rows scaled; the inverse
// scales of rows g and g + 8 in inv.
__device__ __forceinline__ void to_planes(const float (&x)[4], const float (&y)[4], uint32_t (&hi)[4], uint32_t (&lo)[4], float (&inv)[2]) {
    float m0 = 0.f, m1 = 0.f;
#pragma unroll
    for (int c = 0; c < 2; c++) {
        m0 = amax(amax(m0, x[c]), y[c]);
        m1 = amax(amax(m1, x[2 + c]), y[2 + c]);
    }
    const float s0 = row_pow(quad_max(m0), inv[0]), s1 = row_pow(quad_max(m1), inv[1]);
    split2(x[0] * s0, x[1] * s0, hi[0], lo[0]);
    split2(x[2] * s1, x[3] * s1, hi[1], lo[1]);
    split2(y[0] * s0, y[1] * s0, hi[2], lo[2]);
    split2(y[2] * s1, y[3] * s1, hi[3], lo[3]);
}

// d0, d1 (16 columns) += planes x a 16 x 16 block of a strip matrix (rows i = columns of the result)
__device__ __forceinline__ void mma_block(float (&d0)[4], float (&d1)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                          const __half* bhi, const __half* blo, int ib, int jb, int lane) {
    const int row = 16 * ib + (lane & 7) + (lane >> 4) * 8, col = 16 * jb + ((lane >> 3) & 1) * 8;
    const int at = strip_at(row, col);
    uint32_t b[4], w[4];
    ldsm4(w, blo + at);
    mma_f16(d0, hi, w[0], w[1]);
    mma_f16(d1, hi, w[2], w[3]);
    ldsm4(b, bhi + at);
    mma_f16(d0, lo, b[0], b[1]);
    mma_f16(d1, lo, b[2], b[3]);
    mma_f16(d0, hi, b[0], b[1]);
    mma_f16(d1, hi, b[2], b[3]);
}

// grid (ceil(rows / 64), hv, requests or segments).
// kMode 0: whole requests, state from and to the slots.
// kMode 1: a segment's transition: rows below dv from zero state, rows dv .. dv + DK the identity with
//          v = 0; end states to b_seg and m_seg, no outputs.
// kMode 2: a segment from its start state in s_in, with outputs; the request's last one writes the slot.
template <int DK, class T, int kMode>
__global__ void __launch_bounds__(kCThreads, ChunkCfg<DK, T>::kMinBlocks) k_delta_chunk(ChunkArgs ca) {
    extern __shared__ uint8_t raw[];
    using Cfg = ChunkCfg<DK, T>;
    constexpr bool kOut = kMode != 1;
    constexpr int LD = Cfg::LD, KP = Cfg::KP, NT = DK / 8;
    ChunkSmem<DK, T>& sm = *reinterpret_cast<ChunkSmem<DK, T>*>(raw);
    const Args& a = ca.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t h = blockIdx.y, hq = h / (a.hv / a.hk);
    uint32_t req = blockIdx.z, index = 0;
    if (kMode != 0) {
        req = ca.blocks[2 * blockIdx.z];
        index = ca.blocks[2 * blockIdx.z + 1];
        if (req >= a.n || index % ca.merge) return;   // padding, or inside another block's segment
    }
    const uint32_t slot = a.slots[req];
    uint64_t t0 = min(a.cu[req], a.n_rows), t1 = min(a.cu[req + 1], a.n_rows);
    const uint64_t seg_head = kMode == 0 ? 0 : segment_id(ca, t0, req, index / ca.merge) * a.hv + h;
    bool last = true;
    if (kMode != 0) {
        const uint64_t seg = (uint64_t)ca.block * ca.merge, b = t0 + (uint64_t)index * ca.block;
        if (b >= t1) return;
        t0 = b;
        last = t1 <= t0 + seg;
        t1 = min(t1, t0 + seg);
        if (kMode == 1 && last) return;               // nothing starts from its end
    }
    const int row0 = blockIdx.x * kVRows + warp * 16;  // this warp's first state row
    if (slot >= a.n_slots) {   // only this request is rejected: zero outputs, no state touched
        if (kOut) {
            const uint32_t r0 = blockIdx.x * kVRows, w = min(a.dv, r0 + kVRows) - r0;
            for (uint64_t i = threadIdx.x; i < (t1 - t0) * w; i += kCThreads)
                put((T*)a.out + (t0 + i / w) * a.ld_o + (uint64_t)h * a.dv + r0 + i % w, 0.f);
            if (t1 > t0 && h == 0 && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.err, 1u);
        }
        return;
    }
    const bool ident = kMode == 1 && row0 >= (int)a.dv;
    const bool active = row0 < (int)a.dv + (kMode == 1 ? DK : 0);
    const uint64_t per_head = (uint64_t)a.dv * DK;
    float* st = a.state + slot * a.slot_stride + h * per_head;
    const float* src = kMode == 2 ? ca.s_in + seg_head * per_head : st;
    const bool zero = kMode == 1 || (kMode == 0 && a.fresh && a.fresh[req]);
    const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | (a.ld_q * sizeof(T)) | (a.ld_k * sizeof(T))) & 15) == 0;

    float S[NT][4];   // rows row0 + g and + 8, columns 8 n + 2 t, + 1
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int c = 8 * n + 2 * t;
        float2 x = make_float2(0.f, 0.f), y = x;
        if (active && !zero) {
            x = *reinterpret_cast<const float2*>(src + (uint64_t)(row0 + g) * DK + c);
            y = *reinterpret_cast<const float2*>(src + (uint64_t)(row0 + g + 8) * DK + c);
        }
        if (ident) {
            const int r = row0 + g - (int)a.dv;
            x = make_float2(c == r, c + 1 == r);
            y = make_float2(c == r + 8, c + 1 == r + 8);
        }
        S[n][0] = x.x, S[n][1] = x.y, S[n][2] = y.x, S[n][3] = y.y;
    }
    const T* vp = (const T*)a.v + (uint64_t)h * a.dv + row0 + g;
    T* op = (T*)a.out + (uint64_t)h * a.dv + row0 + g;

    for (uint64_t at = t0; at < t1; at += kC) {
        const int len = (int)min((uint64_t)kC, t1 - at);
        prepare_chunk<DK, T, kOut>(sm, a, at, len, h, hq, wide);
        if (at + kC < t1) {   // the next chunk's rows on their way to L2
            const uint64_t r = at + kC + (threadIdx.x >> 1);
            if (r < t1) {
                const char* kn = (const char*)((const T*)a.k + r * a.ld_k + (uint64_t)hq * DK);
                const char* qn = (const char*)((const T*)a.q + r * a.ld_q + (uint64_t)hq * DK);
#pragma unroll
                for (int b = 0; b < DK * (int)sizeof(T); b += 256) {
                    const int o = b + (threadIdx.x & 1) * 128;
                    if (o < DK * (int)sizeof(T)) {
                        prefetch_l2(kn + o);
                        if (kOut) prefetch_l2(qn + o);
                    }
                }
            }
        }
        if (active) {
            // X = S K^T and O = S Q^T over the 64 tokens; V meanwhile
            T V[8][4];
#pragma unroll
            for (int n = 0; n < 8; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int i = 8 * n + 2 * t + (c & 1);
                    V[n][c] = (i < len && !ident) ? vp[(at + i) * a.ld_v + (c >> 1) * 8] : T(0.f);
                }
            float X[8][4], O[8][4];
#pragma unroll
            for (int n = 0; n < 8; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) X[n][c] = O[n][c] = 0.f;
            float m0 = 0.f, m1 = 0.f;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                m0 = amax(amax(m0, S[n][0]), S[n][1]);
                m1 = amax(amax(m1, S[n][2]), S[n][3]);
            }
            float sv0, sv1;
            const float p0 = row_pow(quad_max(m0), sv0), p1 = row_pow(quad_max(m1), sv1);
            const int brow = (lane & 7) + (lane >> 4) * 8, bcol = ((lane >> 3) & 1) * 8;
#pragma unroll
            for (int ks = 0; ks < DK / 16; ks++) {
                uint32_t hi[4], lo[4];
                split2(S[2 * ks][0] * p0, S[2 * ks][1] * p0, hi[0], lo[0]);
                split2(S[2 * ks][2] * p1, S[2 * ks][3] * p1, hi[1], lo[1]);
                split2(S[2 * ks + 1][0] * p0, S[2 * ks + 1][1] * p0, hi[2], lo[2]);
                split2(S[2 * ks + 1][2] * p1, S[2 * ks + 1][3] * p1, hi[3], lo[3]);
#pragma unroll
                for (int nn = 0; nn < 4; nn++) {
                    const int off = (nn * 16 + brow) * LD + ks * 16 + bcol;
                    uint32_t b[4];
                    if (KP == 2) {
                        ldsm4(b, &sm.k[KP - 1][off]);
                        mma_f16(X[2 * nn], hi, b[0], b[1]);
                        mma_f16(X[2 * nn + 1], hi, b[2], b[3]);
                    }
                    ldsm4(b, &sm.k[0][off]);
                    mma_f16(X[2 * nn], lo, b[0], b[1]);
                    mma_f16(X[2 * nn + 1], lo, b[2], b[3]);
                    mma_f16(X[2 * nn], hi, b[0], b[1]);
                    mma_f16(X[2 * nn + 1], hi, b[2], b[3]);
                    if (kOut) {
                        if (KP == 2) {
                            ldsm4(b, &sm.q[KP - 1][off]);
                            mma_f16(O[2 * nn], hi, b[0], b[1]);
                            mma_f16(O[2 * nn + 1], hi, b[2], b[3]);
                        }
                        ldsm4(b, &sm.q[0][off]);
                        mma_f16(O[2 * nn], lo, b[0], b[1]);
                        mma_f16(O[2 * nn + 1], lo, b[2], b[3]);
                        mma_f16(O[2 * nn], hi, b[0], b[1]);
                        mma_f16(O[2 * nn + 1], hi, b[2], b[3]);
                    }
                }
            }
            // right-hand side b (V - e^c k-norm X), and the state's part of the output
#pragma unroll
            for (int n = 0; n < 8; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int i = 8 * n + 2 * t + (c & 1);
                    const float sv = c < 2 ? sv0 : sv1;
                    X[n][c] = sm.beta[i] * (to_f32(V[n][c]) - sm.ak[i] * (sv * X[n][c]));
                    if (kOut) O[n][c] = sm.cq[i] * (sv * O[n][c]);
                }
            // solve by blocks of 16 tokens; U takes the place of X
            uint32_t uh[4][4], ul[4][4];
            float us[4][2];
#pragma unroll
            for (int ib = 0; ib < 4; ib++) {
                float(&r0)[4] = X[2 * ib];
                float(&r1)[4] = X[2 * ib + 1];
                const int i = 16 * ib + 2 * t;
#pragma unroll
                for (int jb = 0; jb < ib; jb++) {
                    float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_block(d0, d1, uh[jb], ul[jb], sm.m[0], sm.m[1], ib, jb, lane);
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        r0[c] = fmaf(-(sm.ascale[jb][i + (c & 1)] * us[jb][c >> 1]), d0[c], r0[c]);
                        r1[c] = fmaf(-(sm.ascale[jb][i + 8 + (c & 1)] * us[jb][c >> 1]), d1[c], r1[c]);
                    }
                }
                uint32_t hi[4], lo[4];
                float inv[2];
                to_planes(r0, r1, hi, lo, inv);
                float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
                mma_block(d0, d1, hi, lo, sm.m[0], sm.m[1], ib, ib, lane);
                const float db = sm.dblk[ib];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    r0[c] = d0[c] * (db * inv[c >> 1]);
                    r1[c] = d1[c] * (db * inv[c >> 1]);
                }
                to_planes(r0, r1, uh[ib], ul[ib], us[ib]);
                if (kOut) {
#pragma unroll
                    for (int jb = 0; jb <= ib; jb++) {
                        float e0[4] = {0.f, 0.f, 0.f, 0.f}, e1[4] = {0.f, 0.f, 0.f, 0.f};
                        mma_block(e0, e1, uh[jb], ul[jb], sm.p[0], sm.p[1], ib, jb, lane);
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            O[2 * ib][c] = fmaf(sm.pscale[jb][i + (c & 1)] * us[jb][c >> 1], e0[c], O[2 * ib][c]);
                            O[2 * ib + 1][c] = fmaf(sm.pscale[jb][i + 8 + (c & 1)] * us[jb][c >> 1], e1[c], O[2 * ib + 1][c]);
                        }
                    }
                }
            }
            if (kOut) {
#pragma unroll
                for (int n = 0; n < 8; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int i = 8 * n + 2 * t + (c & 1);
                        if (i < len) put(op + (at + i) * a.ld_o + (c >> 1) * 8, O[n][c]);
                    }
            }
            // S = e^{c_64} S + sum_j (w_j u_j) k_j^T
            float n0 = 0.f, n1 = 0.f;
#pragma unroll
            for (int n = 0; n < 8; n++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float w = sm.wk[8 * n + 2 * t + c];
                    X[n][c] *= w;
                    X[n][2 + c] *= w;
                    n0 = amax(n0, X[n][c]);
                    n1 = amax(n1, X[n][2 + c]);
                }
            float iv0, iv1;
            const float q0 = row_pow(quad_max(n0), iv0), q1 = row_pow(quad_max(n1), iv1);
#pragma unroll
            for (int jb = 0; jb < 4; jb++) {
                split2(X[2 * jb][0] * q0, X[2 * jb][1] * q0, uh[jb][0], ul[jb][0]);
                split2(X[2 * jb][2] * q1, X[2 * jb][3] * q1, uh[jb][1], ul[jb][1]);
                split2(X[2 * jb + 1][0] * q0, X[2 * jb + 1][1] * q0, uh[jb][2], ul[jb][2]);
                split2(X[2 * jb + 1][2] * q1, X[2 * jb + 1][3] * q1, uh[jb][3], ul[jb][3]);
            }
            const float gamma = sm.gamma;
            const int trow = (lane & 7) + ((lane >> 3) & 1) * 8, tcol = (lane >> 4) * 8;
#pragma unroll
            for (int nn = 0; nn < NT / 2; nn++) {
                float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t b[4][4];
#pragma unroll
                for (int jb = 0; jb < 4; jb++) {
                    const int off = (16 * jb + trow) * LD + nn * 16 + tcol;
                    if (KP == 2) {
                        uint32_t w[4];
                        ldsm4t(w, &sm.k[KP - 1][off]);
                        mma_f16(d0, uh[jb], w[0], w[1]);
                        mma_f16(d1, uh[jb], w[2], w[3]);
                    }
                    ldsm4t(b[jb], &sm.k[0][off]);
                    mma_f16(d0, ul[jb], b[jb][0], b[jb][1]);
                    mma_f16(d1, ul[jb], b[jb][2], b[jb][3]);
                }
#pragma unroll
                for (int jb = 0; jb < 4; jb++) {
                    mma_f16(d0, uh[jb], b[jb][0], b[jb][1]);
                    mma_f16(d1, uh[jb], b[jb][2], b[jb][3]);
                }
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    S[2 * nn][c] = fmaf(gamma, S[2 * nn][c], (c < 2 ? iv0 : iv1) * d0[c]);
                    S[2 * nn + 1][c] = fmaf(gamma, S[2 * nn + 1][c], (c < 2 ? iv0 : iv1) * d1[c]);
                }
            }
        }
        __syncthreads();   // the shared operands are free again
    }
    if (!active || (kMode == 2 && !last)) return;   // only the last segment's end is the request's
    float* dst = st;
    int r = row0;
    if (kMode == 1) {
        dst = ident ? ca.m_seg + seg_head * (DK * DK) : ca.b_seg + seg_head * per_head;
        if (ident) r -= (int)a.dv;
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int c = 8 * n + 2 * t;
        *reinterpret_cast<float2*>(dst + (uint64_t)(r + g) * DK + c) = make_float2(S[n][0], S[n][1]);
        *reinterpret_cast<float2*>(dst + (uint64_t)(r + g + 8) * DK + c) = make_float2(S[n][2], S[n][3]);
    }
}

// Start states of a request's segments: S, S M_0 + b_0, ...  grid (ceil(dv / 8), hv, requests), DK threads:
// thread j owns column j of 8 state rows; bound by the L2 reads of M (DK^2 floats per segment and block).
constexpr int kScanRows = 8;
template <int DK>
__global__ void __launch_bounds__(DK) k_delta_scan(ChunkArgs ca) {
    __shared__ float4 rows[kScanRows][DK / 4];
    const Args& a = ca.a;
    const uint32_t h = blockIdx.y, req = blockIdx.z, slot = a.slots[req], j = threadIdx.x, r0 = blockIdx.x * kScanRows;
    const uint64_t t0 = min(a.cu[req], a.n_rows), t1 = min(a.cu[req + 1], a.n_rows), seg = (uint64_t)ca.block * ca.merge;
    if (slot >= a.n_slots || t0 >= t1) {   // a fresh request without tokens still leaves a zero state
        if (slot < a.n_slots && a.fresh && a.fresh[req])
            for (int r = 0; r < kScanRows; r++) a.state[slot * a.slot_stride + ((uint64_t)h * a.dv + r0 + r) * DK + j] = 0.f;
        return;
    }
    const uint64_t per_head = (uint64_t)a.dv * DK;
    const bool zero = a.fresh && a.fresh[req];
    float s[kScanRows];
#pragma unroll
    for (int r = 0; r < kScanRows; r++)
        s[r] = zero ? 0.f : a.state[slot * a.slot_stride + h * per_head + (uint64_t)(r0 + r) * DK + j];
    const uint32_t n_seg = (uint32_t)((t1 - t0 + seg - 1) / seg);
    for (uint32_t p = 0; p < n_seg; p++) {
        const uint64_t id = segment_id(ca, t0, req, p) * a.hv + h;
#pragma unroll
        for (int r = 0; r < kScanRows; r++) ca.s_in[id * per_head + (uint64_t)(r0 + r) * DK + j] = s[r];
        if (p + 1 == n_seg) break;
#pragma unroll
        for (int r = 0; r < kScanRows; r++) reinterpret_cast<float*>(rows[r])[j] = s[r];
        const float* m = ca.m_seg + id * (DK * DK) + j;
#pragma unroll
        for (int r = 0; r < kScanRows; r++) s[r] = ca.b_seg[id * per_head + (uint64_t)(r0 + r) * DK + j];
        __syncthreads();
#pragma unroll 8
        for (int k = 0; k < DK / 4; k++) {
            const float m0 = m[(4 * k) * DK], m1 = m[(4 * k + 1) * DK], m2 = m[(4 * k + 2) * DK], m3 = m[(4 * k + 3) * DK];
#pragma unroll
            for (int r = 0; r < kScanRows; r++) {
                const float4 x = rows[r][k];
                s[r] = fmaf(x.x, m0, fmaf(x.y, m1, fmaf(x.z, m2, fmaf(x.w, m3, s[r]))));
            }
        }
        __syncthreads();
    }
}

}  // namespace delta
}  // namespace rk
