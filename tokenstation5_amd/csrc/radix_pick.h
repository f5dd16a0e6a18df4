// The k largest of n keys for one workgroup of 1024 threads: a radix descent, 8 bits a pass from the top, to
// the k-th largest key, then the indices above it and the first ones equal to it in
// ascending order. Deterministic: ties go to the lowest index.
#pragma once
#include "common.h"

namespace ts5hip {

constexpr int PICK_NT = 1024, PICK_NW = PICK_NT / 64;

struct PickLds {
    int hist[256];
    int wave_gt[PICK_NW], wave_eq[PICK_NW];
    uint64_t prefix;
    int left;
};

// key(i) for i < n: an unsigned key of BITS bits, larger first; 1 <= k <= n. emit(place, i)
// once for each of the k picked, places ascending with i.
template <int BITS, class Key, class Emit>
__device__ inline void radix_pick(PickLds &L, int n, int k, Key key, Emit emit) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t prefix = 0;
    int left = k;  // of the keys that share the prefix, as many are picked
    int shift = BITS;
    while (shift > 0) {
        shift -= 8;
        if (tid < 256) L.hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += PICK_NT) {
            const uint64_t x = key(i);
            if (shift + 8 >= BITS || x >> (shift + 8) == prefix) atomicAdd(&L.hist[(int)(x >> shift) & 255], 1);
        }
        __syncthreads();
        if (wave == 0) {  // lane l: digits 255 - 4 l down to 252 - 4 l
            int c[4], mine = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) c[j] = L.hist[255 - 4 * lane - j], mine += c[j];
            int before = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(before, o, 64);
                if (lane >= o) before += y;
            }
            before -= mine;  // keys with a larger digit
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (before < left && before + c[j] >= left) {
                    L.prefix = prefix << 8 | (uint64_t)(255 - 4 * lane - j);
                    L.left = left - before;
                }
                before += c[j];
            }
        }
        __syncthreads();
        prefix = L.prefix, left = L.left;
        __syncthreads();
    }
    // Each wave takes a run of indices: its counts, those of the waves before it, then the places.
    const int per = (n + PICK_NW * 64 - 1) / (PICK_NW * 64) * 64;
    const int i0 = wave * per, i1 = min(n, i0 + per);
    int gt = 0, eq = 0;
    for (int i = i0 + lane; i < i1; i += 64) {
        const uint64_t x = key(i);
        gt += x > prefix, eq += x == prefix;
    }
    gt = wave_sum(gt), eq = wave_sum(eq);
    if (lane == 0) L.wave_gt[wave] = gt, L.wave_eq[wave] = eq;
    __syncthreads();
    int place = 0, equal = 0;
    for (int w = 0; w < wave; w++) place += L.wave_gt[w], equal += L.wave_eq[w];
    place += min(equal, left);
    for (int i = i0; i < i1; i += 64) {
        const bool in = i + lane < i1;
        const uint64_t x = in ? key(i + lane) : 0;
        const uint64_t same = __ballot(in && x == prefix), below = (1ull << lane) - 1;
        const bool take = in && (x > prefix || (x == prefix && equal + __popcll(same & below) < left));
        const uint64_t taken = __ballot(take);
        if (take) emit(place + __popcll(taken & below), i + lane);
        place += __popcll(taken), equal += __popcll(same);
    }
}

// Order-preserving unsigned keys; -0 counts as 0.
__device__ inline uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline uint64_t order_key(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}

}  // namespace ts5hip
