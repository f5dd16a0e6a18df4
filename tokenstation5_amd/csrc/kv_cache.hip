// Rows of a KV cache moved: the keys of largest accumulated weight into another
// cache (eviction), and the accepted path of a tree of drafts to the front.
#include <algorithm>

#include "attn_rows.h"
#include "radix_pick.h"

namespace ts5hip {

struct EvictArgs {
    KvLayer kv, to;
    int HKV, n_ctx, n_ctx_out, n_keep, n_first, n_last;
    const int32_t *n_keys;
    const float *acc;  // [B][HKV][n_ctx]
    float *acc_out;    // [B][HKV][n_ctx_out]
    int32_t *kept;     // [B][HKV][n_keep]
    int32_t *n_out;    // [B] or null
};
__device__ inline int evict_count(const EvictArgs &a, int b) { return max(0, min(a.n_keys[b], a.n_ctx)); }

// The slots kept, ascending: the first and last ones, then those of the largest sums (NaN lowest),
// ties to the lowest slot. One workgroup a KV head: its passes over the keys in LDS bound it (4100 keys 8.3 us, 32768
// keys 21 us). grid (HKV, B).
__global__ __launch_bounds__(PICK_NT) void k_evict_pick(EvictArgs a) {
    __shared__ PickLds<uint32_t, 32768> L;
    const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, n = evict_count(a, b);
    int32_t *kept = a.kept + ((int64_t)b * a.HKV + kvh) * a.n_keep;
    if (kvh == 0 && tid == 0 && a.n_out) a.n_out[b] = min(n, a.n_keep);
    if (n <= a.n_keep) {
        for (int i = tid; i < a.n_keep; i += PICK_NT) kept[i] = i < n ? i : -1;
        return;
    }
    const float *acc = a.acc + ((int64_t)b * a.HKV + kvh) * a.n_ctx;
    radix_pick(
        L, n, a.n_keep, [&](int i) { return acc[i]; },
        [&](int i, float x) -> uint32_t {
            if (i < a.n_first || i >= n - a.n_last) return 0xffffffffu;
            return x != x ? 0u : order_key(x);
        },
        [&](int place, int i) { kept[place] = i; });
}

// K, V, scales and sums of the kept slots into the other cache; sums past them are zero. HBM bounds it (8 caches cut
// to 8192 keys of 8 heads of 128, q8: 285 MB read and written in 55 to 60 us). grid (row blocks, HKV, B).
constexpr int EVICT_ROWS = 32;
template <int HD, bool F16>
__global__ __launch_bounds__(256) void k_evict_copy(EvictArgs a) {
    constexpr int LPR = HD * (F16 ? 2 : 1) / 16, SW = HD / 64;  // 16-byte pieces, dwords of scales a row
    __shared__ int src[EVICT_ROWS];
    const int kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, r0 = blockIdx.x * EVICT_ROWS;
    const int64_t head = (int64_t)b * a.HKV + kvh, from = head * a.n_ctx, to = head * a.n_ctx_out;
    const int m = min(evict_count(a, b), a.n_keep), rows = min(EVICT_ROWS, m - r0);
    if (tid < EVICT_ROWS && r0 + tid < a.n_ctx_out) {
        const int r = r0 + tid;
        if (r < m) src[tid] = max(0, min(a.kept[head * a.n_keep + r], a.n_ctx - 1));  // (inside the cache, whatever came between)
        a.acc_out[to + r] = r < m ? a.acc[from + src[tid]] : 0.f;
    }
    __syncthreads();
    for (int e = tid; e < rows * LPR * 2; e += 256) {
        const int r = e / (2 * LPR), p = e % LPR;
        const bool v = e / LPR & 1;
        const uint4 *s = (const uint4 *)(v ? a.kv.v : a.kv.k) + (from + src[r]) * LPR + p;
        ((uint4 *)(v ? a.to.v : a.to.k))[(to + r0 + r) * LPR + p] = *s;
    }
    if constexpr (!F16) {
        for (int e = tid; e < rows * SW * 2; e += 256) {
            const int r = e / (2 * SW), p = e % SW;
            const bool v = e / SW & 1;
            const uint32_t *s = (const uint32_t *)(v ? a.kv.vs : a.kv.ks) + (from + src[r]) * SW + p;
            ((uint32_t *)(v ? a.to.vs : a.to.ks))[(to + r0 + r) * SW + p] = *s;
        }
    }
}

hipError_t launch_kv_evict(int B, int HKV, int HD, KvLayer kv, int kv_f16, int n_ctx, const int32_t *n_keys,
                           const float *acc, int n_keep, int n_first, int n_last, int n_ctx_out, KvLayer to,
                           float *acc_out, int32_t *kept, int32_t *n_out, hipStream_t s) {
    const EvictArgs a{kv, to, HKV, n_ctx, n_ctx_out, n_keep, n_first, n_last, n_keys, acc, acc_out, kept, n_out};
    hipLaunchKernelGGL(k_evict_pick, dim3(HKV, B), dim3(PICK_NT), 0, s, a);
    return rows_by_shape(HD, kv_f16, [&](auto hd, auto f16) {
        hipLaunchKernelGGL((k_evict_copy<decltype(hd)::value, decltype(f16)::value>),
                           dim3((n_ctx_out + EVICT_ROWS - 1) / EVICT_ROWS, HKV, B), dim3(256), 0, s, a);
        return hipGetLastError();
    });
}

// Rows slots[b][0 .. n) of each cache to slots slot0[b] .. + n - 1, in place: a workgroup holds all of
// a plane's rows in registers before it writes any, so the slots may overlap in
// any order. A row with a slot or place outside the cache is left out. grid (HKV, K and V, B).
template <int HD, bool F16>
__global__ __launch_bounds__(256) void k_kv_path(KvLayer kv, int HKV, int n_ctx, const int32_t *slots, int n,
                                                 const int32_t *slot0) {
    constexpr int LPR = HD * (F16 ? 2 : 1) / 16, SW = HD / 64, PER = KV_PATH_MAX * LPR / 256;
    constexpr int SPER = (KV_PATH_MAX * SW + 255) / 256;
    static_assert(PER * 256 == KV_PATH_MAX * LPR, "whole passes");
    const int b = blockIdx.z, v = blockIdx.y, tid = threadIdx.x, to = slot0[b];
    const int64_t head = ((int64_t)b * HKV + blockIdx.x) * n_ctx;
    uint4 *rows = (uint4 *)(v ? kv.v : kv.k);
    uint32_t *sc = (uint32_t *)(v ? kv.vs : kv.ks);
    auto ok = [&](int i, int64_t &from) {
        if (i >= n) return false;
        from = slots[(int64_t)b * n + i];
        return from >= 0 && from < n_ctx && (int64_t)to + i >= 0 && (int64_t)to + i < n_ctx;
    };
    uint4 w[PER];
    uint32_t x[SPER];
#pragma unroll
    for (int k = 0; k < PER; k++) {
        int64_t from;
        const int e = tid + 256 * k;
        w[k] = make_uint4(0, 0, 0, 0);
        if (ok(e / LPR, from)) w[k] = rows[(head + from) * LPR + e % LPR];
    }
    if constexpr (!F16) {
#pragma unroll
        for (int k = 0; k < SPER; k++) {
            int64_t from;
            const int e = tid + 256 * k;
            x[k] = 0;
            if (ok(e / SW, from)) x[k] = sc[(head + from) * SW + e % SW];
        }
    }
    wait_vmcnt<0>();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; k++) {
        int64_t from;
        const int e = tid + 256 * k;
        if (ok(e / LPR, from)) rows[(head + to + e / LPR) * LPR + e % LPR] = w[k];
    }
    if constexpr (!F16) {
#pragma unroll
        for (int k = 0; k < SPER; k++) {
            int64_t from;
            const int e = tid + 256 * k;
            if (ok(e / SW, from)) sc[(head + to + e / SW) * SW + e % SW] = x[k];
        }
    }
}

hipError_t launch_kv_path(int B, int HKV, int HD, KvLayer kv, int kv_f16, int n_ctx, const int32_t *slots, int n,
                          const int32_t *slot0, hipStream_t s) {
    return rows_by_shape(HD, kv_f16, [&](auto hd, auto f16) {
        hipLaunchKernelGGL((k_kv_path<decltype(hd)::value, decltype(f16)::value>), dim3(HKV, 2, B), dim3(256), 0, s, kv,
                           HKV, n_ctx, slots, n, slot0);
        return hipGetLastError();
    });
}

}  // namespace ts5hip
