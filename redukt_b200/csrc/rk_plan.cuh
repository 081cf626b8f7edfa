// Plan of a ragged batch over state slots: token offsets, slots, per-token maps and block table
// from the requests' lengths, in one launch.
//
//   end_i = sum_{j<=i} len_j          cu = {0, min(end_i, max_tokens)}
//   keeps_i: request i names a slot that no earlier request names, and end_i <= max_tokens
//   new_i:   it names none, has tokens, and end_i <= max_tokens; the r-th new request takes the
//            r-th lowest slot that is neither in use nor named
//
// What bounds it: latency for a small batch (two block scans over at most 4,096 requests and slots held
// in shared memory: 8 requests take 6 us), the scans and the stores of 8 bytes per token for a large one
// (4,096 requests with 2.0 M tokens take 14 us, of which the stores alone would be 2.5).  Every block runs
// the same scans over the same few inputs (36 KB at most, from L2) and then fills its own share of the
// token maps and of the block table, so no block waits for another and there is one launch.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace rk {
namespace plan {

constexpr int kPer = 4;                          // requests (and slots) per thread
constexpr uint32_t kMax = 4096;                  // requests and slots: 1,024 threads; 256 serve 1,024 of them
constexpr uint32_t kNone = 0xFFFFFFFFu;

struct Args {
    const uint32_t* len;
    const uint32_t* want;
    const uint8_t* used;
    uint32_t n, n_slots, block, max_tokens, max_blocks;
    int shift;                   // log2(block) where block is a power of two, otherwise -1
    uint32_t *cu, *slot, *fresh;
    uint8_t* used_out;
    uint32_t *token_slot, *token_pos, *block_base, *blocks;
    uint32_t* err;
};

template <int kThreads>
struct Smem {
    static constexpr uint32_t kMax = kThreads * kPer;
    alignas(16) uint32_t cu[kMax + 4];
    alignas(16) uint32_t base[kMax + 4];
    alignas(16) uint32_t slot[kMax];
    alignas(16) uint32_t owner[kMax];      // lowest request that names the slot; later the ascending free list
    unsigned long long part[32];
    int bad;
};

// Exclusive prefix of `v` over the block's threads; the block's total in *total.
template <int kThreads>
__device__ __forceinline__ unsigned long long scan_excl(unsigned long long v, Smem<kThreads>& sm, unsigned long long* total) {
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
    unsigned long long w = lane < kThreads / 32 ? sm.part[lane] : 0ull;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xFFFFFFFFu, w, o);
        if (lane >= o) w += y;
    }
    *total = __shfl_sync(0xFFFFFFFFu, w, 31);
    const unsigned long long before = __shfl_sync(0xFFFFFFFFu, w, warp ? warp - 1 : 0);
    return x - v + (warp ? before : 0ull);
}

// Largest i in [lo, hi) with cu[i] <= x, by a whole warp, 32 probes a round; cu is non-decreasing,
// cu[lo] <= x < cu[hi].
__device__ __forceinline__ uint32_t find_warp(const uint32_t* cu, uint32_t lo, uint32_t hi, uint32_t x) {
    const uint32_t lane = threadIdx.x & 31;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;
        const uint32_t below = __popc(__ballot_sync(0xFFFFFFFFu, at < hi && cu[at] <= x));   // at least 1: cu[lo] <= x
        lo += (below - 1) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// The same, by one thread.
__device__ __forceinline__ uint32_t find(const uint32_t* cu, uint32_t lo, uint32_t hi, uint32_t x) {
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (cu[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads, 1) k_plan(Args a) {
    extern __shared__ uint8_t raw[];
    Smem<kThreads>& sm = *reinterpret_cast<Smem<kThreads>*>(raw);
    const uint32_t t = threadIdx.x, i0 = t * kPer;
    uint32_t len[kPer], want[kPer];
    bool used[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const uint32_t i = i0 + j;
        len[j] = i < a.n ? a.len[i] : 0u;
        want[j] = i < a.n ? a.want[i] : kNone;
        used[j] = i >= a.n_slots || a.used[i] != 0;
    }
    *reinterpret_cast<uint4*>(sm.owner + i0) = make_uint4(kNone, kNone, kNone, kNone);
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
    uint32_t begin[kPer], mine4[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const uint32_t i = i0 + j;
        const bool fits = ends[j] <= a.max_tokens;
        const uint32_t e = (uint32_t)(fits ? ends[j] : a.max_tokens);
        const unsigned long long b = ends[j] - len[j];
        const uint32_t l = e - (uint32_t)(b < a.max_tokens ? b : a.max_tokens);
        cnt[j] = l ? (a.shift >= 0 ? (l - 1) >> a.shift : (l - 1) / a.block) + 1 : 0u;
        blocks += cnt[j];
        keeps[j] = want[j] < a.n_slots && sm.owner[want[j]] == i && fits;
        isnew[j] = want[j] == kNone && len[j] > 0 && fits;
        fresh += isnew[j];
        taken[j] = used[j] || sm.owner[i] != kNone;
        spare += !taken[j];
        begin[j] = e - l;
    }
    // requests past the last have no tokens: their offset is the total, so cu[n] and base[n] come out right
    *reinterpret_cast<uint4*>(sm.cu + i0) = make_uint4(begin[0], begin[1], begin[2], begin[3]);
    if (t == kThreads - 1) sm.cu[kThreads * kPer] = (uint32_t)(ends[kPer - 1] <= a.max_tokens ? ends[kPer - 1] : a.max_tokens);
    // one scan for three counts: blocks in the high word, free slots and new requests below
    const unsigned long long mine = ((unsigned long long)blocks << 32) | (spare << 16) | fresh;
    const unsigned long long pre = scan_excl(mine, sm, &total);  // every read of `owner` is done
    uint32_t b = (uint32_t)(pre >> 32), f = (uint32_t)(pre >> 16) & 0xFFFFu, r = (uint32_t)pre & 0xFFFFu;
    const uint32_t n_free = (uint32_t)(total >> 16) & 0xFFFFu, n_new = (uint32_t)total & 0xFFFFu;
    uint32_t* free_list = sm.owner;
    uint32_t rank[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const uint32_t i = i0 + j;
        mine4[j] = b;
        b += cnt[j];
        rank[j] = f;
        if (!taken[j]) free_list[f++] = i;
    }
    *reinterpret_cast<uint4*>(sm.base + i0) = make_uint4(mine4[0], mine4[1], mine4[2], mine4[3]);
    if (t == kThreads - 1) sm.base[kThreads * kPer] = b;
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
    // Token maps: a warp fills one run of tokens, 128 at a time; the requests of a run's first and last token
    // bound every lane's search (to nothing, mostly).
    const uint32_t warps = gridDim.x * (kThreads / 32), lane = t & 31;
    const unsigned long long run = ((unsigned long long)a.max_tokens + 128ull * warps - 1) / (128ull * warps) * 128;
    const unsigned long long first = run * (blockIdx.x * (kThreads / 32) + (t >> 5));
    const bool wide = ((reinterpret_cast<uintptr_t>(a.token_slot) | reinterpret_cast<uintptr_t>(a.token_pos)) & 15) == 0;
    uint32_t lo = first < n_tokens ? find_warp(sm.cu, 0, a.n, (uint32_t)first) : 0u;
    for (unsigned long long c = first; c < first + run && c < a.max_tokens; c += 128) {
        uint32_t hi = lo;
        if (c < n_tokens) {
            const uint32_t last = (uint32_t)min(c + 127, (unsigned long long)n_tokens - 1);
            hi = sm.cu[lo + 1] > last ? lo : find_warp(sm.cu, lo, a.n, last);
        }
        const unsigned long long k = c + 4 * lane;
        uint32_t s4[4], p4[4];
        if (k + 4 <= n_tokens) {
            uint32_t rq = find(sm.cu, lo, hi + 1, (uint32_t)k), from = sm.cu[rq], to = sm.cu[rq + 1], sl = sm.slot[rq];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t x = (uint32_t)k + j;
                if (x >= to) {   // rare: a request ends inside the four
                    while (sm.cu[rq + 1] <= x) rq++;
                    from = sm.cu[rq], to = sm.cu[rq + 1], sl = sm.slot[rq];
                }
                s4[j] = sl;
                p4[j] = x - from;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s4[j] = p4[j] = kNone;
                if (k + j < n_tokens) {
                    const uint32_t rq = find(sm.cu, lo, hi + 1, (uint32_t)k + j);
                    s4[j] = sm.slot[rq];
                    p4[j] = (uint32_t)k + j - sm.cu[rq];
                }
            }
        }
        if (wide && k + 4 <= a.max_tokens) {
            *reinterpret_cast<uint4*>(a.token_slot + k) = make_uint4(s4[0], s4[1], s4[2], s4[3]);
            *reinterpret_cast<uint4*>(a.token_pos + k) = make_uint4(p4[0], p4[1], p4[2], p4[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (k + j < a.max_tokens) {
                    a.token_slot[k + j] = s4[j];
                    a.token_pos[k + j] = p4[j];
                }
        }
        lo = hi;
    }
    for (unsigned long long k = blockIdx.x * kThreads + t; k < a.max_blocks; k += (unsigned long long)kThreads * gridDim.x) {
        uint32_t rq = kNone, at = kNone;
        if (k < n_blocks) {
            rq = find(sm.base, 0, a.n, (uint32_t)k);
            at = (uint32_t)k - sm.base[rq];
        }
        a.blocks[2 * k] = rq;
        a.blocks[2 * k + 1] = at;
    }
}

}  // namespace plan
}  // namespace rk
