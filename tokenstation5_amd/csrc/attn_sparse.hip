// Attention over the blocks of a cache that a bound on their scores picks for each query:
//  k_block_bounds  lowest and highest cached value of each dimension over a block's keys,
//                  rounded outwards to f16;
//  k_block_scores  for each block, the highest score that a key inside its bounds could have
//                  with any head of the KV head's group: max over heads of sum_d max(q_d lo_d,
//                  q_d hi_d). In fp64: a rounded score could pick another block, and another block
//                  is another output;
//  k_block_pick    the last block, the first, then the highest scores, ties to the lowest
//                  block, ascending;
//  k_attn_picked   attention over the picked blocks' keys (attn_rows.h), split over workgroups, of which
//                  few are joined by the last to finish, many by
//  k_picked_merge.
#include <algorithm>

#include "attn_rows.h"
#include "radix_pick.h"

namespace ts5hip {

// ---- bounds ----------------------------------------------------------------------------------------

// x to f16, down (up) to the next value where the nearest is above (below) it.
__device__ inline _Float16 f16_towards(float x, bool up) {
    const _Float16 h = (_Float16)x;
    const float y = (float)h;
    if (up ? !(y < x) : !(y > x)) return h;
    uint16_t b = __builtin_bit_cast(uint16_t, h);
    if ((b & 0x7fff) == 0) b = up ? 0x0001 : 0x8001;
    else b += ((b >> 15) == 0) == up ? 1 : -1;
    return __builtin_bit_cast(_Float16, b);
}

// A wave per block: LPR lanes a row, 16 bytes each. grid (ceil(blocks / 4), HKV, B) of the blocks that hold a cache's
// last n_new keys. HBM bounds it: 4 caches of 12288 to 16384 keys of 8 heads of 128, f16, 125 MB in 22 us; one block
// of each head 5.6 us, a launch and two round trips.
template <int HD, bool F16>
__global__ __launch_bounds__(256) void k_block_bounds(KvLayer kv, int HKV, int n_ctx, const int32_t *n_keys, int n_new,
                                                      int block, int n_blocks, _Float16 *bounds) {
    constexpr int VB = F16 ? 2 : 1, LPR = HD * VB / 16, RPW = 64 / LPR, V = 16 / VB;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kvh = blockIdx.y, b = blockIdx.z;
    const int n = max(0, min(n_keys[b], n_ctx));
    const int blk = max(n - n_new, 0) / block + (int)blockIdx.x * 4 + wave;
    if ((int64_t)blk * block >= n) return;
    const int64_t slot0 = ((int64_t)b * HKV + kvh) * n_ctx;
    const int first = blk * block, last = min(n, first + block), d0 = lane % LPR * V;
    float lo[V], hi[V];
#pragma unroll
    for (int j = 0; j < V; j++) lo[j] = INFINITY, hi[j] = -INFINITY;
    constexpr int AHEAD = 4;  // passes requested before the first is used (rows past the last: the last again)
    for (int r0 = first + lane / LPR; r0 < last; r0 += AHEAD * RPW) {
        u32x4 w[AHEAD];
        uint16_t sc[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const int64_t r = slot0 + min(r0 + k * RPW, last - 1);
            w[k] = *(const u32x4 *)(kv.k + (r * HD + d0) * VB);
            if constexpr (!F16) sc[k] = kv.ks[r * (HD / 32) + d0 / 32];
        }
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
#pragma unroll
            for (int j = 0; j < V; j++) {
                float x;
                if constexpr (F16) x = h2f((w[k][j / 2] >> (16 * (j & 1))) & 0xffff);
                else x = (float)(int8_t)(w[k][j / 4] >> (8 * (j & 3))) * h2f(sc[k]);
                lo[j] = fminf(lo[j], x), hi[j] = fmaxf(hi[j], x);  // (NaN: passed over)
            }
    }
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
        for (int j = 0; j < V; j++) {
            lo[j] = fminf(lo[j], __shfl_xor(lo[j], o, 64));
            hi[j] = fmaxf(hi[j], __shfl_xor(hi[j], o, 64));
        }
    if (lane < LPR) {
        _Float16 *p = bounds + (((int64_t)b * HKV + kvh) * n_blocks + blk) * 2 * HD + d0;
#pragma unroll
        for (int j = 0; j < V; j++) p[j] = f16_towards(lo[j], false), p[HD + j] = f16_towards(hi[j], true);
    }
}

hipError_t launch_block_bounds(int B, int HKV, int HD, KvLayer kv, int kv_f16, int n_ctx, const int32_t *n_keys,
                               int n_new, int block, void *bounds, hipStream_t s) {
    const int nb = (n_ctx + block - 1) / block, most = std::min(nb, (n_new + block - 1) / block + 1);
    const dim3 grid((most + 3) / 4, HKV, B);
    auto go = [&](auto hd, auto f16) {
        hipLaunchKernelGGL((k_block_bounds<decltype(hd)::value, decltype(f16)::value>), grid, dim3(256), 0, s, kv, HKV,
                           n_ctx, n_keys, n_new, block, nb, (_Float16 *)bounds);
        return hipGetLastError();
    };
    return rows_by_shape(HD, kv_f16, go);
}

// ---- scores and the pick ---------------------------------------------------------------------------

struct SparseArgs {
    const float *q;  // [B][H * HD]
    KvLayer kv;
    int n_ctx, H, HKV, per_batch, block, n_pick, n_split;
    const int32_t *n_keys;
    const _Float16 *bounds;  // [caches][HKV][n_blocks][2][HD]
    int n_blocks;
    float scale;
    double *scores;   // [B][HKV][n_blocks]
    int32_t *picked;  // [B][HKV][n_pick], -1 past the blocks there are
    float *part;      // [B][HKV][G][n_split][HD + 4]
    int *counters;    // [B * HKV], CTR_STRIDE ints apart, zero between launches
    float *out;
};
__device__ inline int sparse_count(const SparseArgs &a, int b) {
    const int n = max(0, min(a.n_keys[a.per_batch ? b : 0], a.n_ctx));  // (before b is added: no overflow)
    return a.per_batch ? n : min(n + b + 1, a.n_ctx);
}

template <int CTRL>
__device__ inline double dpp_f64(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    const uint32_t l = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, true);
    const uint32_t h = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
    return __longlong_as_double((long long)((uint64_t)h << 32 | l));
}

// HD / 8 lanes a block, 8 dims and four blocks a lane; a head's four sums over the lanes go together:
// two exchanges within a quad leave each of its lanes the quad's sum of one block, and only that goes
// on to the other quads. 16 queries over 14464 blocks in all of 8 heads of 128 (59 MB): 16 us, the bytes and
// the fp64 multiply-adds about even (30 us with a head's sum over all lanes by itself and q
// converted for each block). grid (ceil(n_blocks / blocks a workgroup), HKV, B).
template <int HD>
constexpr int score_blocks() { return 4 * 4 * 64 / (HD / 8); }
template <int HD>
__global__ __launch_bounds__(256) void k_block_scores(SparseArgs a) {
    constexpr int LPB = HD / 8, BPW = 64 / LPB;
    __shared__ __align__(16) float q[ROWS_MAX_G][HD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kvh = blockIdx.y, b = blockIdx.z;
    const int n = sparse_count(a, b), nb = (n + a.block - 1) / a.block, G = a.H / a.HKV;
    const int first = blockIdx.x * score_blocks<HD>();
    if (first >= nb - 1 || nb <= a.n_pick) return;  // the last block is read in any case, and so are all that fit
    for (int e = threadIdx.x; e < G * HD; e += 256) q[e / HD][e % HD] = a.q[((int64_t)b * a.H + kvh * G) * HD + e];
    const int64_t head = (int64_t)(a.per_batch ? b : 0) * a.HKV + kvh;
    const int d0 = lane % LPB * 8, blk0 = first + wave * 4 * BPW + lane / LPB;
    u32x4 lo[4], hi[4];
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const _Float16 *at = a.bounds + (head * a.n_blocks + min(blk0 + p * BPW, nb - 1)) * 2 * HD + d0;
        lo[p] = *(const u32x4 *)at, hi[p] = *(const u32x4 *)(at + HD);
    }
    __syncthreads();
    double best = -INFINITY;  // of block pass 2 * (lane & 1) + (lane >> 1 & 1)
    for (int g = 0; g < G; g++) {
        double x[8], s[4] = {0, 0, 0, 0};
        uint32_t neg[4];  // the halves whose query value takes the lowest
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float x0 = q[g][d0 + 2 * j], x1 = q[g][d0 + 2 * j + 1];
            x[2 * j] = x0, x[2 * j + 1] = x1;
            neg[j] = (x0 >= 0.f ? 0u : 0xffffu) | (x1 >= 0.f ? 0u : 0xffff0000u);
        }
#pragma unroll
        for (int p = 0; p < 4; p++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t w = (lo[p][j] & neg[j]) | (hi[p][j] & ~neg[j]);
                s[p] = fma(x[2 * j], (double)h2f(w & 0xffff), s[p]);
                s[p] = fma(x[2 * j + 1], (double)h2f(w >> 16), s[p]);
            }
        const bool odd = lane & 1, two = lane & 2;
        const double a0 = (odd ? s[2] : s[0]) + dpp_f64<0xB1>(odd ? s[0] : s[2]);  // quad_perm [1,0,3,2]
        const double a1 = (odd ? s[3] : s[1]) + dpp_f64<0xB1>(odd ? s[1] : s[3]);
        double t = (two ? a1 : a0) + dpp_f64<0x4E>(two ? a0 : a1);  // quad_perm [2,3,0,1]
        if constexpr (LPB == 8) {
            t += __shfl_xor(t, 4, 64);
        } else {
            t += dpp_f64<0x124>(t);  // row_ror:4
            t += dpp_f64<0x128>(t);  // row_ror:8
            if constexpr (LPB == 32) t += __shfl_xor(t, 16, 64);
        }
        if (!(t <= best)) best = t != t ? INFINITY : t;  // (NaN ranks first)
    }
    const int blk = blk0 + (2 * (lane & 1) + (lane >> 1 & 1)) * BPW;
    if (lane % LPB < 4 && blk < nb) a.scores[((int64_t)b * a.HKV + kvh) * a.n_blocks + blk] = best;
}

__global__ __launch_bounds__(PICK_NT) void k_block_pick(SparseArgs a) {
    __shared__ PickLds<uint64_t, 8192> L;
    const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int n = sparse_count(a, b), nb = (n + a.block - 1) / a.block;
    int32_t *out = a.picked + ((int64_t)b * a.HKV + kvh) * a.n_pick;
    if (nb <= a.n_pick) {
        for (int i = tid; i < a.n_pick; i += PICK_NT) out[i] = i < nb ? i : -1;
        return;
    }
    const double *sc = a.scores + ((int64_t)b * a.HKV + kvh) * a.n_blocks;
    if (tid == 0) out[a.n_pick - 1] = nb - 1;
    if (a.n_pick == 1) return;
    radix_pick(L, nb - 1, a.n_pick - 1, [&](int i) { return sc[i]; },
               [&](int i, double x) { return i == 0 ? ~(uint64_t)0 : order_key(x); },
               [&](int place, int i) { out[place] = i; });
}

// ---- attention over the picked blocks ----------------------------------------------------------------

// Units (KT tiles of 16 keys) of the picked blocks of query b, and a slice's share.
__device__ inline int sparse_units(const SparseArgs &a, int b, int KT) {
    const int nb = (sparse_count(a, b) + a.block - 1) / a.block;
    return (min(nb, a.n_pick) * (a.block / 16) + KT - 1) / KT;
}

// grid (n_split, HKV, B): one slice of the picked units for the G heads of a KV head, three workgroups a CU, each
// wave's next unit requested before this one is used. 16 queries over 4096 keys each (142 MB): 36 us; latency
// bounds it (the vector ALU is busy 45 % of the time). Up to FUSED_SPLITS slices
// the last workgroup joins them: partials of one launch go past the L2 and back, about 7 us behind 32
// slices, where a launch of its own takes 5 (one query: 13 against 10.4 us in all), but next to nothing
// behind 4 that end at different times (16 queries: 37 against 41 us).
constexpr int FUSED_SPLITS = 8;
template <int HD, bool F16, int KT, int NW, bool FUSED>
__global__ __launch_bounds__(64 * NW) void k_attn_picked(SparseArgs a) {
    __shared__ RowsLds<HD, NW> L;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rl = lane & 15, kq = lane >> 4;
    const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, G = a.H / a.HKV;
    RowsIn<HD, 1> in;  // requested before the counts that the keys' addresses wait for
    rows_request<HD, 1>(in, kq, [&](int, bool &ok) {
        ok = rl < G;
        return a.q + ((int64_t)b * a.H + kvh * G + min(rl, G - 1)) * HD;
    });
    const int n = sparse_count(a, b), units = sparse_units(a, b, KT), per = (units + a.n_split - 1) / a.n_split;
    const int u0 = split * per, u1 = min(units, u0 + per);
    if (FUSED && n == 0 && split == 0)  // no key: zeros
        for (int e = threadIdx.x; e < G * HD; e += 64 * NW) a.out[(((int64_t)b * a.HKV + kvh) * G) * HD + e] = 0.f;
    if (u0 >= u1) return;  // an empty slice: not counted, not joined
    const int tpb = a.block / 16, tiles = min((n + a.block - 1) / a.block, a.n_pick) * tpb;
    const int32_t *list = a.picked + ((int64_t)b * a.HKV + kvh) * a.n_pick;
    const RowsKv kv = rows_kv<HD, F16>(a.kv, ((int64_t)(a.per_batch ? b : 0) * a.HKV + kvh) * a.n_ctx, n);
    auto at = [&](int u, int (&kb)[KT]) {
#pragma unroll
        for (int t = 0; t < KT; t++) {
            const int tile = u * KT + t, i = tile < tiles && u < u1 ? tile : -1;
            kb[t] = i < 0 ? n : list[i / tpb] * a.block + i % tpb * 16;  // (none: zeros, no memory access)
        }
    };
    RowsUnit<HD, F16, KT> nxt;
    int kb[KT], kn[KT];
    at(u0 + wave, kn);
    rows_load<HD, F16, KT>(nxt, kv, kn, rl, kq);
    RowsQ<HD, 1> q;
    rows_query<HD, 1>(q, in, a.scale);
    RowsSum<HD, 1> sum;
    rows_clear<HD, 1>(sum);
    for (int u = u0 + wave; u < u1; u += NW) {
        const RowsUnit<HD, F16, KT> cur = nxt;
#pragma unroll
        for (int t = 0; t < KT; t++) kb[t] = kn[t];
        at(u + NW, kn);
        rows_load<HD, F16, KT>(nxt, kv, kn, rl, kq);
        rows_unit<HD, F16, KT, true, false>(cur, q, sum, kb, kq, [&](int key) { return rows_below(key, n); },
                                               [](int, const float (&)[4]) {});
    }
    // For the last workgroup, which may run on another XCD, the partials go past this one's L2, and only when they
    // are out does the workgroup count itself in.
    const int used = (units + per - 1) / per;
    const int64_t row0 = ((int64_t)b * a.HKV + kvh) * G;
    const __amdgpu_buffer_rsrc_t part = slice_rsrc(a.part + row0 * a.n_split * (HD + 4), (uint32_t)(G * a.n_split * (HD + 4) * 4));
    rows_combine<HD, NW>(L, sum, G, wave, rl, kq, [&](int r, int d, float4 o, float m, float l) {
        if (FUSED && used == 1) {
            *(float4 *)(a.out + (row0 + r) * HD + d) = rows_over(o, l);
            return;
        }
        const uint32_t at = (uint32_t)(r * a.n_split + split) * (HD + 4) * 4;
        constexpr int POLICY = FUSED ? BUF_SC1 : 0;
        if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, make_float2(m, l)), part, at, 0, POLICY);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), part, at + 16 + 4 * d, 0, POLICY);
    });
    if (!FUSED || used == 1) return;
    __shared__ RowsJoin J;
    __shared__ int last;
    wait_stores();
    __syncthreads();
    if (threadIdx.x == 0) {
        int *c = a.counters + (b * a.HKV + kvh) * CTR_STRIDE;
        last = atomicAdd(c, 1) == used - 1;
        if (last) st_dev(c, 0);
    }
    __syncthreads();
    if (!last) return;
    constexpr int TPR = HD / 4 * JOIN_SG;
    static_assert(64 * NW == 256, "rows_join's threads");
    for (int g0 = 0; g0 < G; g0 += 256 / TPR) {
        const int g = g0 + (int)threadIdx.x / TPR;
        float M, l;
        const float4 o = rows_join<HD, JOIN_SG>(J, used, M, l, [&](int s, int d, float2 &ml, float4 &x) {
            const uint32_t at = (uint32_t)(min(g, G - 1) * a.n_split + s) * (HD + 4) * 4;
            ml = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(part, at, 0, BUF_SC1));
            x = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(part, at + 16 + 4 * d, 0, BUF_SC1));
        });
        if (g < G && threadIdx.x % TPR < HD / 4)
            *(float4 *)(a.out + (row0 + g) * HD + 4 * (threadIdx.x % TPR)) = rows_over(o, l);
    }
}

template <int HD, int KT>
__global__ __launch_bounds__(256) void k_picked_merge(SparseArgs a, int64_t rows) {
    constexpr int TPR = HD / 4 * JOIN_SG;
    __shared__ RowsJoin J;
    const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR, at = min(row, rows - 1);
    const int units = sparse_units(a, (int)(at / a.H), KT), per = (units + a.n_split - 1) / a.n_split;
    const int used = units ? (units + per - 1) / per : 0;
    float M, l;
    const float4 o = rows_join<HD, JOIN_SG>(J, a.part + at * a.n_split * (HD + 4), used, M, l);
    if (row < rows && threadIdx.x % TPR < HD / 4)
        *(float4 *)(a.out + row * HD + 4 * (threadIdx.x % TPR)) = rows_over(o, l);
}

struct SparseScratch {
    int n_blocks, n_split;
    size_t scores, picked, part;
};
static SparseScratch sparse_scratch(int B, int H, int HKV, int HD, int n_ctx, int block, int n_pick, int n_cu) {
    SparseScratch p;
    p.n_blocks = (n_ctx + block - 1) / block;
    const int64_t keys = (int64_t)std::min(n_pick, p.n_blocks) * block;
    // Every workgroup a unit a wave at least; one round of two workgroups a CU.
    const int most = (int)std::min<int64_t>((keys + 63) / 64, ROWS_MAX_SPLIT);
    p.n_split = std::max(1, std::min(2 * n_cu / std::max(1, B * HKV), most));
    p.scores = align_up((size_t)B * HKV * p.n_blocks * sizeof(double), 256);
    p.picked = align_up((size_t)B * HKV * std::min(n_pick, p.n_blocks) * sizeof(int32_t), 256);
    p.part = (size_t)B * H * p.n_split * (HD + 4) * sizeof(float);
    return p;
}
size_t attn_sparse_scratch_bytes(int B, int H, int HKV, int HD, int n_ctx, int block, int n_pick, int n_cu) {
    const SparseScratch p = sparse_scratch(B, H, HKV, HD, n_ctx, block, n_pick, n_cu);
    return p.scores + p.picked + p.part;
}
hipError_t launch_attn_sparse(const float *q, int B, int H, int HKV, int HD, KvLayer kv, int kv_f16, int n_ctx,
                              const int32_t *n_keys, int per_batch, const void *bounds, int block, int n_pick,
                              float scale, void *scratch, int *counters, float *out, int32_t *picked, int n_cu, hipStream_t s) {
    const SparseScratch p = sparse_scratch(B, H, HKV, HD, n_ctx, block, n_pick, n_cu);
    uint8_t *base = (uint8_t *)scratch;
    SparseArgs a{};
    a.q = q, a.kv = kv, a.n_ctx = n_ctx, a.H = H, a.HKV = HKV, a.per_batch = per_batch, a.block = block;
    a.n_pick = picked ? n_pick : std::min(n_pick, p.n_blocks), a.n_split = p.n_split, a.n_keys = n_keys, a.bounds = (const _Float16 *)bounds;
    a.n_blocks = p.n_blocks, a.scale = scale, a.out = out;
    a.scores = (double *)base, a.picked = picked ? picked : (int32_t *)(base + p.scores);
    a.part = (float *)(base + p.scores + p.picked), a.counters = counters;
    return rows_by_shape(HD, kv_f16, [&](auto hd, auto f16) {
        constexpr int D = decltype(hd)::value, KT = D == 64 ? 2 : 1, NW = 4;
        constexpr bool F = decltype(f16)::value;
        hipLaunchKernelGGL(k_block_scores<D>, dim3((p.n_blocks + score_blocks<D>() - 1) / score_blocks<D>(), HKV, B), dim3(256),
                           0, s, a);
        hipLaunchKernelGGL(k_block_pick, dim3(HKV, B), dim3(PICK_NT), 0, s, a);
        if (p.n_split <= FUSED_SPLITS) {
            hipLaunchKernelGGL((k_attn_picked<D, F, KT, NW, true>), dim3(p.n_split, HKV, B), dim3(64 * NW), 0, s, a);
            return hipGetLastError();
        }
        hipLaunchKernelGGL((k_attn_picked<D, F, KT, NW, false>), dim3(p.n_split, HKV, B), dim3(64 * NW), 0, s, a);
        const int64_t rows = (int64_t)B * H;
        constexpr int RPW = 256 / (D / 4 * JOIN_SG);
        hipLaunchKernelGGL((k_picked_merge<D, KT>), dim3((unsigned)((rows + RPW - 1) / RPW)), dim3(256), 0, s, a, rows);
        return hipGetLastError();
    });
}

}  // namespace ts5hip
