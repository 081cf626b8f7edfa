// Plan of a ragged batch over state slots: token offsets, slots, per-token maps and block table
// from the requests' lengths, in one launch.
//
//   end_i = sum_{j<=i} len_j          cu = {0, min(end_i, max_tokens)}
//   keeps_i: request i names a slot that no earlier request names, and end_i <= max_tokens
//   new_i:   it names none, has tokens, and end_i <= max_tokens; the r-th new request takes the
//            r-th lowest slot that is neither in use nor named
//
// What bounds it: latency for a small batch (two block scans over at most 4,096 requests and slots
// held in shared memory), the stores of 8 bytes per token for a large one.  Every block runs the
// same scans over the same few inputs (36 KB at most, from L2) and then fills its own share of the
// token maps and of the block table, so no block waits for another and there is one launch.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace rk {
namespace plan {

constexpr int kThreads = 1024;
constexpr int kPer = 4;                          // requests (and slots) per thread
constexpr uint32_t kMax = kThreads * kPer;       // 4,096 requests and slots
constexpr uint32_t kNone = 0xFFFFFFFFu;

struct Args {
    const uint32_t* len;
    const uint32_t* want;
    const uint8_t* used;
    uint32_t n, n_slots, block, max_tokens, max_blocks;
    uint32_t *cu, *slot, *fresh;
    uint8_t* used_out;
    uint32_t *token_slot, *token_pos, *block_base, *blocks;
    uint32_t* err;
};

struct Smem {
    uint32_t cu[kMax + 1];
    uint32_t base[kMax + 1];
    uint32_t slot[kMax];
    uint32_t owner[kMax];      // lowest request that names the slot; later the ascending free list
    unsigned long long part[32];
    int bad;
};

// Exclusive prefix of `v` over the block's threads; the block's total in *total.
__device__ __forceinline__ unsigned long long scan_excl(unsigned long long v, Smem& sm, unsigned long long* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // `part` is free again
    if (lane == 31) sm.part[warp] = x;
    __syncthreads();
    unsigned long long w = sm.part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xFFFFFFFFu, w, o);
        if (lane >= o) w += y;
    }
    *total = __shfl_sync(0xFFFFFFFFu, w, 31);
    const unsigned long long before = __shfl_sync(0xFFFFFFFFu, w, warp ? warp - 1 : 0);
    return x - v + (warp ? before : 0ull);
}

// Largest i in [0, n) with cu[i] <= x; cu is non-decreasing and x < cu[n].
__device__ __forceinline__ uint32_t find(const uint32_t* cu, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (cu[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kThreads) k_plan(Args a) {
    extern __shared__ uint8_t raw[];
    Smem& sm = *reinterpret_cast<Smem*>(raw);
    const uint32_t t = threadIdx.x, i0 = t * kPer;
    uint32_t len[kPer], want[kPer];
    bool used[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const uint32_t i = i0 + j;
        len[j] = i < a.n ? a.len[i] : 0u;
        want[j] = i < a.n ? a.want[i] : kNone;
        used[j] = i >= a.n_slots || a.used[i] != 0;
        sm.owner[i] = kNone;
    }
    if (t == 0) sm.bad = 0;
    unsigned long long sum = 0, total;
#pragma unroll
    for (int j = 0; j < kPer; j++) sum += len[j];
    unsigned long long end = scan_excl(sum, sm, &total);  // its barriers also publish `owner`
    unsigned long long ends[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) ends[j] = end += len[j];
    // the lowest request that names a slot owns it, in any order of the atomics
#pragma unroll
    for (int j = 0; j < kPer; j++)
        if (want[j] < a.n_slots) atomicMin(&sm.owner[want[j]], i0 + j);
    __syncthreads();
    uint32_t cnt[kPer], blocks = 0, fresh = 0, spare = 0;
    bool keeps[kPer], isnew[kPer], taken[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const uint32_t i = i0 + j;
        const bool fits = ends[j] <= a.max_tokens;
        const uint32_t e = (uint32_t)(fits ? ends[j] : a.max_tokens);
        const unsigned long long b = ends[j] - len[j];
        const uint32_t l = e - (uint32_t)(b < a.max_tokens ? b : a.max_tokens);
        cnt[j] = (uint32_t)(((unsigned long long)l + a.block - 1) / a.block);
        blocks += cnt[j];
        keeps[j] = want[j] < a.n_slots && sm.owner[want[j]] == i && fits;
        isnew[j] = want[j] == kNone && len[j] > 0 && fits;
        fresh += isnew[j];
        taken[j] = used[j] || sm.owner[i] != kNone;
        spare += !taken[j];
        if (i <= a.n) sm.cu[i] = (uint32_t)(b < a.max_tokens ? b : a.max_tokens);
        if (i + 1 == a.n) sm.cu[a.n] = e;
    }
    // one scan for three counts: blocks in the high word, free slots and new requests below
    const unsigned long long mine = ((unsigned long long)blocks << 32) | (spare << 16) | fresh;
    const unsigned long long pre = scan_excl(mine, sm, &total);  // every read of `owner` is done
    uint32_t b = (uint32_t)(pre >> 32), f = (uint32_t)(pre >> 16) & 0xFFFFu, r = (uint32_t)pre & 0xFFFFu;
    const uint32_t r0 = r;
    const uint32_t n_free = (uint32_t)(total >> 16) & 0xFFFFu, n_new = (uint32_t)total & 0xFFFFu;
    uint32_t* free_list = sm.owner;
    uint32_t rank[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const uint32_t i = i0 + j;
        if (i <= a.n) sm.base[i] = b;
        b += cnt[j];
        if (i + 1 == a.n) sm.base[a.n] = b;
        rank[j] = f;
        if (!taken[j]) free_list[f++] = i;
    }
    __syncthreads();
    int bad = 0;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const uint32_t i = i0 + j;
        uint32_t s = keeps[j] ? want[j] : kNone;
        bool got = false;
        if (isnew[j]) {
            got = r < n_free;
            if (got) s = free_list[r];
            r++;
        }
        if (i < a.n) {
            sm.slot[i] = s;
            if (s == kNone && (len[j] > 0 || want[j] != kNone)) bad = 1;
            if (blockIdx.x == 0) {
                a.slot[i] = s;
                a.fresh[i] = got;
            }
        }
        if (blockIdx.x == 0 && i < a.n_slots)  // the lowest n_new free slots are given away
            a.used_out[i] = taken[j] || rank[j] < n_new;
    }
    (void)r0;
    if (bad) sm.bad = 1;
    __syncthreads();
    const uint32_t n_tokens = sm.cu[a.n], n_blocks = sm.base[a.n];
    if (blockIdx.x == 0) {
        for (uint32_t i = t; i <= a.n; i += kThreads) {
            a.cu[i] = sm.cu[i];
            a.block_base[i] = sm.base[i];
        }
        if (t == 0 && sm.bad) atomicOr(a.err, 1u);
    }
    // token maps: four tokens per thread and step, one search per step
    const unsigned long long stride = 4ull * kThreads * gridDim.x;
    for (unsigned long long k = 4ull * (blockIdx.x * kThreads + t); k < a.max_tokens; k += stride) {
        uint32_t q = (uint32_t)k;
        uint32_t rq = q < n_tokens ? find(sm.cu, a.n, q) : 0u;
        uint32_t s4[4], p4[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t x = q + j;
            if (x < n_tokens && x >= q) {
                while (sm.cu[rq + 1] <= x) rq++;
                s4[j] = sm.slot[rq];
                p4[j] = x - sm.cu[rq];
            } else {
                s4[j] = p4[j] = kNone;
            }
        }
        const bool whole = k + 4 <= a.max_tokens;
        if (whole && ((reinterpret_cast<uintptr_t>(a.token_slot) | reinterpret_cast<uintptr_t>(a.token_pos)) & 15) == 0) {
            *reinterpret_cast<uint4*>(a.token_slot + k) = make_uint4(s4[0], s4[1], s4[2], s4[3]);
            *reinterpret_cast<uint4*>(a.token_pos + k) = make_uint4(p4[0], p4[1], p4[2], p4[3]);
        } else {
            for (int j = 0; j < 4 && k + j < a.max_tokens; j++) {
                a.token_slot[k + j] = s4[j];
                a.token_pos[k + j] = p4[j];
            }
        }
    }
    for (unsigned long long k = blockIdx.x * kThreads + t; k < a.max_blocks; k += (unsigned long long)kThreads * gridDim.x) {
        uint32_t rq = kNone, at = kNone;
        if (k < n_blocks) {
            rq = find(sm.base, a.n, (uint32_t)k);
            at = (uint32_t)k - sm.base[rq];
        }
        a.blocks[2 * k] = rq;
        a.blocks[2 * k + 1] = at;
    }
}

}  // namespace plan
}  // namespace rk
