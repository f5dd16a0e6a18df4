// The k largest of n keys for one workgroup of 1024 threads, ties to the lowest index, as ascending
// indices: a radix descent from the top digit to the k-th largest key, then the keys above it and the
// first ones equal to it. 12 bits a pass: one pass spreads an fp32 key's exponent and 3 bits
// over the bins, so that its LDS additions rarely meet, and few keys are left for the next (an fp64 key's first digit
// is its sign and exponent alone, which scores of one query share: that pass settles little and its additions meet);
// it ends once a bin is taken whole. The keys are staged in LDS, sixteen requests at a time, and a
// thread takes an odd number of neighbours there (an odd stride meets no bank twice), so that the
// last pass is counts and bit masks of its own keys instead of ballots; the picked
// indices go out through LDS in order. 32768 keys: 21 us (8-bit digits
// read from memory: 60). Deterministic.
#pragma once
#include <type_traits>

#include "common.h"

namespace ts5hip {

constexpr int PICK_NT = 1024, PICK_NW = PICK_NT / 64;
constexpr int PICK_BINS = 4096;

template <class T, int CAP>
struct PickLds {
    T key[CAP];
    int hist[PICK_BINS];
    uint32_t wave[PICK_NW];
    uint64_t prefix;
    int left, whole;
};

// Sum of v over the threads before this one; total: over all. Every thread calls it.
template <class L_>
__device__ inline uint32_t pick_scan(L_ &L, uint32_t v, uint32_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t x = v;  // the wave's inclusive sums by DPP: shifts within 16-lane rows, then the rows' last lanes on
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);   // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);   // row_shr:2
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xE, true);   // row_shr:4
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xC, true);   // row_shr:8
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    __syncthreads();
    if (lane == 63) L.wave[wave] = x;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PICK_NW; w++) {
        const uint32_t t = L.wave[w];
        before += w < wave ? t : 0, total += t;
    }
    return before + x - v;
}

// fetch(i) loads value i < n, key(i, value) makes an unsigned key T of it, larger first; 1 <= k <= n.
// emit(place, i) once for each of the k picked, places ascending with i. Past CAP keys they
// are staged again in every pass.
template <class T, int CAP, class Fetch, class Key, class Emit>
__device__ inline void radix_pick(PickLds<T, CAP> &L, int n, int k, Fetch fetch, Key key, Emit emit) {
    static_assert(CAP <= 32768, "16 bits count a chunk's keys, and 64 a thread's");
    constexpr int BITS = 8 * sizeof(T), AHEAD = sizeof(T) == 4 ? 16 : 8;
    const int tid = threadIdx.x;
    auto per = [](int m) { return ((m + PICK_NT - 1) / PICK_NT) | 1; };  // neighbours a thread
    auto stage = [&](int c0, auto counted) {  // keys c0 .. of the chunk; counted: their top digits too
        const int m = min(n - c0, CAP);
        __syncthreads();
        for (int i0 = tid; i0 < m; i0 += AHEAD * PICK_NT) {
            decltype(fetch(0)) v[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; j++) v[j] = fetch(c0 + min(i0 + j * PICK_NT, m - 1));
#pragma unroll
            for (int j = 0; j < AHEAD; j++) asm volatile("" : "+v"(v[j]));  // (no load of one waits for the use of another)
#pragma unroll
            for (int j = 0; j < AHEAD; j++)
                if (i0 + j * PICK_NT < m) {
                    const T x = key(c0 + i0 + j * PICK_NT, v[j]);
                    L.key[i0 + j * PICK_NT] = x;
                    if constexpr (decltype(counted)::value) atomicAdd(&L.hist[(int)(x >> (BITS - 12))], 1);
                }
        }
        __syncthreads();
    };
    T prefix = 0;   // of the k-th largest key, from bit `shift` on
    int left = k;   // of the keys with that prefix, as many are picked
    int shift = BITS;
    bool whole = false;
    while (shift > 0 && !whole) {
        const int width = min(12, shift), above = shift;
        shift -= width;
#pragma unroll
        for (int j = 0; j < PICK_BINS / PICK_NT; j++) L.hist[j * PICK_NT + tid] = 0;
        __syncthreads();
        for (int c0 = 0; c0 < n; c0 += CAP) {
            if (above == BITS) {
                stage(c0, std::true_type{});
                continue;
            }
            if (n > CAP) stage(c0, std::false_type{});
            const int m = min(n - c0, CAP), p = per(m), i1 = min(m, (tid + 1) * p);
#pragma unroll 4
            for (int i = tid * p; i < i1; i++) {
                const T x = L.key[i];
                if (x >> above == prefix)
                    atomicAdd(&L.hist[(int)(x >> shift) & ((1 << width) - 1)], 1);
            }
        }
        __syncthreads();
        int c[4];  // the thread's digits, from the largest down
        uint32_t mine = 0, total;
#pragma unroll
        for (int j = 0; j < 4; j++) c[j] = L.hist[PICK_BINS - 1 - 4 * tid - j], mine += (uint32_t)c[j];
        int before = (int)pick_scan(L, mine, total);  // keys with a larger digit
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (before < left && before + c[j] >= left) {
                L.prefix = (uint64_t)prefix << width | (uint64_t)(PICK_BINS - 1 - 4 * tid - j);
                L.left = left - before, L.whole = c[j] == left - before;
            }
            before += c[j];
        }
        __syncthreads();
        prefix = (T)L.prefix, left = L.left, whole = L.whole;
        __syncthreads();
    }
    // Per chunk: a thread's keys above and equal as bits, the counts before them, and the picked indices
    // over the keys in LDS.
    int gt0 = 0, eq0 = 0;
    for (int c0 = 0; c0 < n; c0 += CAP) {
        if (n > CAP) stage(c0, std::false_type{});
        const int m = min(n - c0, CAP), p = per(m), i0 = tid * p, i1 = min(m, i0 + p);
        uint64_t above = 0, equal = 0;
#pragma unroll 4
        for (int i = i0; i < i1; i++) {
            const T y = L.key[i] >> shift;
            above |= (uint64_t)(y > prefix) << (i - i0), equal |= (uint64_t)(y == prefix) << (i - i0);
        }
        uint32_t total;
        const uint32_t mine = (uint32_t)__popcll(above) | (uint32_t)__popcll(equal) << 16;
        const uint32_t before = pick_scan(L, mine, total);  // (its barriers: every key has been read)
        const int eq = eq0 + (int)(before >> 16);
        int place = (int)(before & 0xffff) + max(0, min(eq, left) - min(eq0, left));
        // (the equal ones that are still to be picked: all, none, or, for one thread, the lowest)
        const int room = left - eq;
        while (room > 0 && __popcll(equal) > room) equal &= ~(1ull << (63 - __clzll((long long)equal)));
        const uint64_t take = above | (room > 0 ? equal : 0);
#pragma unroll
        for (int w = 0; w < 2; w++)  // (32 bits at a time)
            for (uint32_t t = (uint32_t)(take >> (32 * w)); t; t &= t - 1)
                L.key[place++] = (T)(i0 + 32 * w + __ffs((int)t) - 1);
        __syncthreads();
        const int first = gt0 + min(eq0, left), gts = (int)(total & 0xffff), eqs = (int)(total >> 16);
        const int taken = gts + min(eq0 + eqs, left) - min(eq0, left);
        for (int i = tid; i < taken; i += PICK_NT) emit(first + i, c0 + (int)L.key[i]);
        gt0 += gts, eq0 += eqs;
        __syncthreads();
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
