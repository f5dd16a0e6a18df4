// Attention of several rows of queries over a KV cache, on the core of
// attn_rows.h: a tree of drafted tokens, a prompt chunk whose key weights are
// summed, and one query a cache whose scores are kept for that sum.
#include <algorithm>

#include "attn_rows.h"

namespace ts5hip {

struct RowsArgs {
    const float *q;  // [B][T][H * HD]
    KvLayer kv;      // B caches
    int n_ctx, H, HKV, T, n_split;
    int G, R, nrb;  // query heads a KV head, rows T * G, blocks of rows
    int least;      // keys a slice takes at least
    uint64_t g_m, nrb_m, split_m;  // rows_magic of G, nrb, n_split
    const int32_t *n_keys;  // per cache: the keys before the T tokens (tree), or all keys (one query)
    const uint64_t *mask;   // [B][T], tree
    int pos0;               // position of the first token (causal)
    int mode;
    float scale;
    float *part;    // [B][HKV][T * G][n_split][HD + 4]: m, l, -, -, O
    float *out;     // [B][T][H * HD]
    float *lse;     // [B][HKV][T * G] log2 of the sum of 2^score, or null
    float *scores;  // [B][HKV][G][stride] log2-domain scores (one query)
    int64_t stride;
    uint4 *planes;  // [HKV][row tile][HD / 32][2][64] the rows' fp16 planes, and then
    float *p2e;     // [HKV][row tile][16] their 2^e, or null (causal)
};
enum { ROWS_TREE = 0, ROWS_CAUSAL = 1, ROWS_ONE = 2 };

// The keys before the tokens (tree) or of the sequence, inside the cache whatever the caller's
// device memory holds.
__device__ inline int rows_count(const RowsArgs &a, int b) {
    if (a.mode == ROWS_CAUSAL) return a.pos0;
    return max(0, min(a.n_keys[b], a.mode == ROWS_TREE ? a.n_ctx - a.T : a.n_ctx));
}
// Keys that slices divide, and the keys of token t's row.
__device__ inline int rows_all(const RowsArgs &a, int n) { return a.mode == ROWS_ONE ? n : n + a.T; }
__device__ inline int rows_reach(const RowsArgs &a, int n, int t) { return a.mode == ROWS_CAUSAL ? n + t + 1 : rows_all(a, n); }

// The query head (and output) of row r of KV head kvh: token r / G, head r % G of the group.
__device__ inline int64_t rows_at(const RowsArgs &a, int b, int kvh, int r) {
    const int t = rows_div(r, a.g_m);
    return ((int64_t)b * a.T + t) * a.H + kvh * a.G + r - t * a.G;
}

// The infinite and NaN values of keys first .. kend - 1 that token t's rows take, onto dims d .. + 3 of a row:
// the products left them out there.
template <int HD, bool F16>
__device__ inline void rows_add_nonfinite(const RowsArgs &a, int b, int kvh, int t, int n, int first, int kend, int d,
                                          float4 &o) {
    const uint64_t own = a.mode == ROWS_TREE ? a.mask[(int64_t)b * a.T + t] & (~0ull >> (64 - a.T)) : 0;
    const int reach = a.mode == ROWS_CAUSAL ? n + t + 1 : n;
    for (int key = first; key < kend; key++) {
        if (key >= reach && !(key >= n && key - n < 64 && (own >> (key - n) & 1))) continue;
        const int64_t slot = ((int64_t)b * a.HKV + kvh) * a.n_ctx + key;
        o.x += rows_nonfinite<HD, F16>(a.kv, slot, d), o.y += rows_nonfinite<HD, F16>(a.kv, slot, d + 1);
        o.z += rows_nonfinite<HD, F16>(a.kv, slot, d + 2), o.w += rows_nonfinite<HD, F16>(a.kv, slot, d + 3);
    }
}

// grid (n_split, HKV, B): one slice of the keys for a KV head's R <= 16 rows,
// row r = G t + j being head j of token t. The waves take the slice's units in turn. ONE: one query a
// cache (16 of 12288 to 16384 keys, 32/8 heads of 128, q8: 504 MB in 120 us, 4.4 TB/s with the scores it
// writes); latency bounds it, the vector ALU is busy 45 % of the time.
template <int HD, bool F16, int KT, int NW, bool ONE>
__global__ __launch_bounds__(64 * NW, ONE && HD <= 128 ? 3 : 1) void k_attn_rows(RowsArgs a) {
    using S = RowsShape<HD, F16, KT>;
    __shared__ RowsLds<HD, NW> L;
    __shared__ int nonfinite;  // a masked unit left out infinite or NaN values
    if (!ONE && threadIdx.x == 0) nonfinite = 0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rl = lane & 15, kq = lane >> 4;
    const int R = a.R;
    const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    RowsIn<HD, 1> in;  // requested before the counts that the keys' addresses wait for
    rows_request<HD, 1>(in, kq, [&](int, bool &ok) {
        ok = rl < R;
        return a.q + rows_at(a, b, kvh, min(rl, R - 1)) * HD;
    });
    const int n = rows_count(a, b), chunk = rows_chunk(rows_all(a, n), a.n_split, a.split_m, a.least);
    const int kbeg = split * chunk, kend = min(kbeg + chunk, rows_reach(a, n, rows_div(R - 1, a.g_m)));
    if (kbeg >= kend) return;  // the merge reads no partial of this slice
    const int full = a.mode == ROWS_CAUSAL ? n + 1 : n;  // keys before it are every row's
    const RowsKv kv = rows_kv<HD, F16>(a.kv, ((int64_t)b * a.HKV + kvh) * a.n_ctx, kend);
    const int units = (kend - kbeg + S::UNIT - 1) / S::UNIT;
    RowsUnit<HD, F16, KT> nxt;
    auto at = [&](int u, int (&kb)[KT]) {
#pragma unroll
        for (int t = 0; t < KT; t++) kb[t] = kbeg + u * S::UNIT + 16 * t;
    };
    int kb[KT];
    at(wave, kb);
    rows_load<HD, F16, KT>(nxt, kv, kb, rl, kq);

    RowsQ<HD, 1> q;
    rows_query<HD, 1>(q, in, a.scale);
    // Keys before `seen` are the lane's row's, and then those of n + the set bits.
    const int t = rows_div(min(rl, R - 1), a.g_m), seen = rl >= R ? 0 : a.mode == ROWS_CAUSAL ? n + t + 1 : n;
    uint64_t bits = 0;
    if (!ONE && a.mode == ROWS_TREE) {
        const uint64_t m = a.mask[(int64_t)b * a.T + t] & (~0ull >> (64 - a.T));
        bits = rl < R ? m : 0;
    }
    if (!ONE && a.planes && split == 0 && wave == 0) {
        uint4 *p = a.planes + (int64_t)kvh * (HD / 32) * 2 * 64 + lane;
#pragma unroll
        for (int c = 0; c < HD / 32; c++) {
            p[(2 * c) * 64] = __builtin_bit_cast(uint4, q.h[0][c]);
            p[(2 * c + 1) * 64] = __builtin_bit_cast(uint4, q.l[0][c]);
        }
        if (kq == 0) a.p2e[(int64_t)kvh * 16 + rl] = q.p2e[0];
    }
    RowsSum<HD, 1> sum;
    rows_clear<HD, 1>(sum);
    if (!ONE) __syncthreads();  // the flag is set
    const int64_t row0 = ((int64_t)b * a.HKV + kvh) * R;
    if constexpr (ONE) {
        // One unit ahead in three waves a SIMD; two ahead in two waves is no faster (122 us), and in three it
        // spills (170 us).
        auto put = [&](int key, const float (&s)[4]) {
            if (rl < R && key < kend)
                *(float4 *)(a.scores + (row0 + rl) * a.stride + key) =
                    make_float4(s[0] * q.p2e[0], s[1] * q.p2e[0], s[2] * q.p2e[0], s[3] * q.p2e[0]);
        };
        auto seen4 = [&](int key) { return rows_below(key, kend); };
        for (int u = wave; u < units; u += NW) {
            const RowsUnit<HD, F16, KT> cur = nxt;
            at(u + NW, kb);
            rows_load<HD, F16, KT>(nxt, kv, kb, rl, kq);  // (past the slice: zeros, no memory access)
            at(u, kb);
            rows_unit<HD, F16, KT, true, false>(cur, q, sum, kb, kq, seen4, put);
        }
    } else {
        auto put = [](int, const float (&)[4]) {};
        for (int u = wave; u < units; u += NW) {
            const RowsUnit<HD, F16, KT> cur = nxt;
            int kn[KT];
            at(u, kb);
            at(u + NW, kn);
            rows_load<HD, F16, KT>(nxt, kv, kn, rl, kq);
            if (kb[0] + S::UNIT <= full)
                rows_unit<HD, F16, KT, false, false>(cur, q, sum, kb, kq, [](int) { return 15u; }, put);
            else if (rows_unit<HD, F16, KT, true, true>(
                         cur, q, sum, kb, kq,
                         [&](int key) { return rows_below(key, seen) | rows_window(bits, key - n); },
                         put))
                nonfinite = 1;
        }
    }
    rows_combine<HD, NW>(L, sum, R, wave, rl, kq, [&](int r, int d, float4 o, float m, float l) {
        const int t = rows_div(r, a.g_m);
        if (!ONE && nonfinite)
            rows_add_nonfinite<HD, F16>(a, b, kvh, t, n, kbeg + max(full - kbeg, 0) / S::UNIT * S::UNIT, kend, d, o);
        if (!ONE && a.n_split == 1) {
            *(float4 *)(a.out + rows_at(a, b, kvh, r) * HD + d) = rows_over(o, l);
            if (a.lse && d == 0) a.lse[row0 + r] = l == 0.f ? INFINITY : m + __log2f(l);
            return;
        }
        float *p = a.part + ((row0 + r) * a.n_split + split) * (HD + 4);
        if (d == 0) *(float4 *)p = make_float4(m, l, 0.f, 0.f);
        *(float4 *)(p + 4 + d) = o;
    });
}

// ---- many rows: the keys converted once for a workgroup --------------------------------------------------
// 64 NT rows, each of four waves 16 NT of them, over one slice of the keys in blocks of 16 NKT.
// The waves read a block's K and V while they compute the one before, convert a share of it each into the MFMA
// operands' own layout in LDS (16 bytes a lane, so that no read or write meets a bank twice:
// K [tile][chunk][lane], V hi and lo [tile pair][dim tile][lane]), and take all of it against
// their own rows. Each key is converted once for 64 NT rows instead of once for 16 NT, and two
// workgroups a CU fill each other's waits: waves that converted for themselves, one a SIMD, took 191 us where this
// takes 95 (4 trees of 64 tokens, 32/8 heads, up to 8192 keys). What bounds it: the matrix cores are busy for 34 % of the
// time and the vector ALU for 45 %, mostly in turn, as the two waves of a SIMD wait for their own chains.
// Eight waves with two blocks in LDS convert half as much a row and were slower (103 us), and so were higher
// priorities around the products (94 and 60 against 94 and 58 us).
template <int HD, bool F16, int NT_>
struct TileShape {
    static constexpr int NT = NT_, NKT = HD == 256 ? 2 : 4, KEYS = 16 * NKT, ROWS = 64 * NT;
    static constexpr int WPT = 4 / NKT;  // waves that share a key tile's conversion
    static constexpr int NC = HD / 32, NDT = HD / 16, CW = NC / WPT, DW = NDT / WPT;  // chunks and dims of a lane's share
    static constexpr int VB = F16 ? 2 : 1, KW = F16 ? 4 : 2, VW = DW * VB / 4;
};
template <int HD, bool F16>
struct TileLds {
    using S = TileShape<HD, F16, 1>;
    uint4 k[S::NKT][S::NC][64];
    uint2 vh[S::NKT / 2][S::NDT][64][2];
    uint2 vl[F16 ? 1 : S::NKT / 2][F16 ? 1 : S::NDT][64][2];
    __align__(16) float ks[F16 ? 1 : S::NKT][F16 ? 1 : S::NC][16];
    int nonfinite;
};

template <int HD, bool F16, int NT_>
__global__ __launch_bounds__(256, 2) void k_attn_tile(RowsArgs a) {
    using S = TileShape<HD, F16, NT_>;
    constexpr int NT = S::NT, NKT = S::NKT, NC = S::NC, NDT = S::NDT;
    __shared__ TileLds<HD, F16> L;
    if (threadIdx.x == 0) L.nonfinite = 0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rl = lane & 15, kq = lane >> 4;
    const int R = a.R;
    const int split = blockIdx.x, kvh = rows_div(blockIdx.y, a.nrb_m), r0 = ((int)blockIdx.y - kvh * a.nrb) * S::ROWS, b = blockIdx.z;
    const int w0 = r0 + 16 * NT * wave;  // the wave's first row
    RowsIn<HD, NT> in;  // requested before the counts that the keys' addresses wait for
    rows_request<HD, NT>(in, kq, [&](int qt, bool &ok) {
        const int r = w0 + 16 * qt + rl;
        ok = r < R;
        return a.q + rows_at(a, b, kvh, min(r, R - 1)) * HD;
    });
    const int n = rows_count(a, b), chunk = rows_chunk(rows_all(a, n), a.n_split, a.split_m, a.least);
    const int kbeg = split * chunk, kend = min(kbeg + chunk, rows_reach(a, n, rows_div(min(R, r0 + S::ROWS) - 1, a.g_m)));
    if (kbeg >= kend) return;  // the merge reads no partial of this slice
    const int full = a.mode == ROWS_CAUSAL ? n + rows_div(r0, a.g_m) + 1 : n;  // keys before it are every row's
    const RowsKv kv = rows_kv<HD, F16>(a.kv, ((int64_t)b * a.HKV + kvh) * a.n_ctx, kend);
    // The lane's share of a block: tile wave / WPT; K of key rl, chunks c0 ..; V of keys 4 kq .. + 3, dims
    // NDT rl + d0 ..; the K scale of key rl, chunk c0 + kq.
    const int tile = wave / S::WPT, c0 = wave % S::WPT * S::CW, d0 = wave % S::WPT * S::DW;
    uint32_t rk[S::CW][S::KW], rv[4][S::VW];
    uint16_t rks = 0, rvs[4];
    auto load = [&](int kb) {
        const int key = kb + 16 * tile;
#pragma unroll
        for (int c = 0; c < S::CW; c++)
            rows_words<S::KW>(kv.k, ((uint32_t)(key + rl) * HD + 32 * (c0 + c) + 8 * kq) * S::VB, rk[c]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            rows_words<S::VW>(kv.v, ((uint32_t)(key + 4 * kq + i) * HD + NDT * rl + d0) * S::VB, rv[i]);
            if constexpr (!F16)
                rvs[i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(
                    kv.vs, ((uint32_t)(key + 4 * kq + i) * NC + (NDT * rl + d0) / 32) * 2, 0, 0);
        }
        if constexpr (!F16)
            rks = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(kv.ks, ((uint32_t)(key + rl) * NC + c0 + kq % S::CW) * 2, 0, 0);
    };
    auto convert = [&](auto m) {
        constexpr bool masked = decltype(m)::value;
#pragma unroll
        for (int c = 0; c < S::CW; c++) L.k[tile][c0 + c][lane] = __builtin_bit_cast(uint4, rows_values<S::KW>(rk[c]));
        if constexpr (!F16) {
            if (kq < S::CW) L.ks[tile][c0 + kq][rl] = h2f(rks);
        }
        constexpr int PW = F16 ? 2 : 4;
        ar_h2 sc[2] = {};
        if constexpr (!F16) {
            sc[0] = __builtin_bit_cast(ar_h2, (uint32_t)rvs[0] | (uint32_t)rvs[1] << 16);
            sc[1] = __builtin_bit_cast(ar_h2, (uint32_t)rvs[2] | (uint32_t)rvs[3] << 16);
        }
        uint32_t any = 0;
#pragma unroll
        for (int d = 0; d < S::DW; d++) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int p = 0; p < 2; p++) {
                rows_value_pair<F16>(rv[2 * p][d / PW], rv[2 * p + 1][d / PW], d % PW, sc[p], hi[p], lo[p]);
                if constexpr (masked) {  // infinite and NaN values out: they are added where the rows are written
                    uint32_t keep = 0;
                    if ((hi[p] & 0x7c00u) != 0x7c00u) keep |= 0xffffu;
                    if ((hi[p] & 0x7c000000u) != 0x7c000000u) keep |= 0xffff0000u;
                    any |= ~keep, hi[p] &= keep, lo[p] &= keep;
                }
            }
            L.vh[tile / 2][d0 + d][lane][tile & 1] = make_uint2(hi[0], hi[1]);
            if constexpr (!F16) L.vl[tile / 2][d0 + d][lane][tile & 1] = make_uint2(lo[0], lo[1]);
        }
        if (masked && __builtin_amdgcn_ballot_w64(any != 0)) L.nonfinite = 1;
    };
    load(kbeg);

    RowsQ<HD, NT> q;
    rows_query<HD, NT>(q, in, a.scale);
    int seen[NT];       // keys before it are the row's
    uint64_t bits[NT];  // and then those of n + its set bits
#pragma unroll
    for (int qt = 0; qt < NT; qt++) {
        const int r = w0 + 16 * qt + rl, t = rows_div(min(r, R - 1), a.g_m);
        seen[qt] = r >= R ? 0 : a.mode == ROWS_CAUSAL ? n + t + 1 : n;
        bits[qt] = 0;
        if (a.mode == ROWS_TREE) {
            const uint64_t m = a.mask[(int64_t)b * a.T + t] & (~0ull >> (64 - a.T));
            bits[qt] = r < R ? m : 0;
        }
    }
    if (a.planes && split == 0) {
        const int tiles = (R + 15) / 16;
#pragma unroll
        for (int qt = 0; qt < NT; qt++) {
            const int row_tile = w0 / 16 + qt;
            if (row_tile >= tiles) break;
            uint4 *p = a.planes + ((int64_t)kvh * tiles + row_tile) * NC * 2 * 64 + lane;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                p[(2 * c) * 64] = __builtin_bit_cast(uint4, q.h[qt][c]);
                p[(2 * c + 1) * 64] = __builtin_bit_cast(uint4, q.l[qt][c]);
            }
            if (kq == 0) a.p2e[((int64_t)kvh * tiles + row_tile) * 16 + rl] = q.p2e[qt];
        }
    }
    RowsSum<HD, NT> sum;
    rows_clear<HD, NT>(sum);
    const int wfull = a.mode == ROWS_CAUSAL ? n + rows_div(w0, a.g_m) + 1 : n;  // every row of the wave's
    const int wreach = w0 < R ? rows_reach(a, n, rows_div(min(R, w0 + 16 * NT) - 1, a.g_m)) : 0;

    for (int kb = kbeg; kb < kend; kb += S::KEYS) {
        __syncthreads();  // every wave is done with the last block
        if (kb + S::KEYS > full) convert(std::true_type{});
        else convert(std::false_type{});
        load(kb + S::KEYS);  // (past the slice: zeros, no memory access)
        __syncthreads();
        if (kb >= wreach) continue;
        // 32 keys at a time (a whole block's scores and weights would take 32 registers more).
#pragma unroll 1
        for (int half = 0; half < NKT / 2; half++) {
            const int kh = kb + 32 * half;
            if (kh >= wreach) break;
            // S^T, two chunks of a tile at a time (so that other products lie between two on one
            // accumulator); the next two are read from LDS before these are used.
            float s[2][NT][4];
            {
                constexpr int STEPS = NC;
                ar_h8 ka[2][2];
                float4 k4[2][2];
                ar_f4 D[F16 ? 1 : 2][NT];
                auto fetch = [&](int step, int buf) {
                    const int t = 2 * half + step / (NC / 2), c = step % (NC / 2) * 2;
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        ka[buf][j] = __builtin_bit_cast(ar_h8, L.k[t][c + j][lane]);
                        if constexpr (!F16) k4[buf][j] = *(const float4 *)&L.ks[t][c + j][4 * kq];
                    }
                };
                fetch(0, 0);
#pragma unroll
                for (int step = 0; step < STEPS; step++) {
                    const int t = step / (NC / 2), c = step % (NC / 2) * 2, buf = step & 1;
                    if (step + 1 < STEPS) fetch(step + 1, buf ^ 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int plane = 0; plane < 2; plane++)
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int qt = 0; qt < NT; qt++) {
                                const bool first = plane == 0 && (!F16 || (c == 0 && j == 0));
                                ar_f4 &d = D[F16 ? 0 : j][qt];
                                if (first) d = ar_f4{0.f, 0.f, 0.f, 0.f};
                                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[buf][j], plane ? q.l[qt][c + j] : q.h[qt][c + j], d, 0, 0, 0);
                            }
                    if constexpr (F16) {
                        if (c + 2 == NC) {
#pragma unroll
                            for (int qt = 0; qt < NT; qt++)
#pragma unroll
                                for (int i = 0; i < 4; i++) s[t][qt][i] = D[0][qt][i];
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const float ks[4] = {k4[buf][j].x, k4[buf][j].y, k4[buf][j].z, k4[buf][j].w};
#pragma unroll
                            for (int qt = 0; qt < NT; qt++)
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    s[t][qt][i] = c + j == 0 ? ks[i] * D[j][qt][i] : fmaf(ks[i], D[j][qt][i], s[t][qt][i]);
                        }
                    }
                }
            }
            if (kh + 32 > wfull) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int qt = 0; qt < NT; qt++) {
                        const int key = kh + 16 * t + 4 * kq;
                        const uint32_t take = rows_below(key, seen[qt]) | rows_window(bits[qt], key - n);
#pragma unroll
                        for (int i = 0; i < 4; i++) s[t][qt][i] = take & 1u << i ? s[t][qt][i] : -INFINITY;
                    }
            }
            uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
            for (int qt = 0; qt < NT; qt++) {
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[t][qt][i]);
                const float m0 = rows_reference(sum, qt, max_xor32(max_xor16(mx)) * q.p2e[qt]);
                float l = 0.f;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[t][qt][2 * i], q.p2e[qt], -m0));
                        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[t][qt][2 * i + 1], q.p2e[qt], -m0));
                        l += p0 + p1;
                        rows_split(p0, p1, ph[qt][2 * t + i], pl[qt][2 * t + i]);
                    }
                sum.l[qt] += l;  // (the lane's share: its four keys of each tile)
            }
            // O^T, two dim tiles at a time, the next two's values read before.
            {
                constexpr int STEPS = NDT / 2;
                ar_h8 vh[2][2], vl[2][2];
                auto fetch = [&](int step, int buf) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        vh[buf][j] = *(const ar_h8 *)&L.vh[half][step * 2 + j][lane];
                        if constexpr (!F16) vl[buf][j] = *(const ar_h8 *)&L.vl[half][step * 2 + j][lane];
                    }
                };
                fetch(0, 0);
#pragma unroll
                for (int step = 0; step < STEPS; step++) {
                    const int d = step * 2, buf = step & 1;
                    if (step + 1 < STEPS) fetch(step + 1, buf ^ 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int term = 0; term < 3; term++) {  // Vh Ph, Vl Ph, Vh Pl
                        if (F16 && term == 1) continue;
#pragma unroll
                        for (int j = 0; j < 2; j++)
#pragma unroll
                            for (int qt = 0; qt < NT; qt++) {
                                const uint32_t *p = term == 2 ? pl[qt] : ph[qt];
                                const ar_h8 w = __builtin_bit_cast(ar_h8, u32x4{p[0], p[1], p[2], p[3]});
                                sum.o[qt][d + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(term == 1 ? vl[buf][j] : vh[buf][j], w,
                                                                                         sum.o[qt][d + j], 0, 0, 0);
                            }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int qt = 0; qt < NT; qt++) sum.l[qt] = add_xor32(add_xor16(sum.l[qt]));

    const bool extra = L.nonfinite;  // (set before a barrier that every wave has passed)
#pragma unroll
    for (int qt = 0; qt < NT; qt++) {
        const int r = w0 + 16 * qt + rl, t = rows_div(r, a.g_m);
        if (r >= R) continue;
        const int64_t row = ((int64_t)b * a.HKV + kvh) * R + r;
        float *p = a.n_split == 1 ? a.out + rows_at(a, b, kvh, r) * HD : a.part + (row * a.n_split + split) * (HD + 4) + 4;
        if (kq == 0) {
            if (a.n_split > 1) *(float4 *)(p - 4) = make_float4(sum.m[qt], sum.l[qt], 0.f, 0.f);
            else if (a.lse) a.lse[row] = sum.l[qt] == 0.f ? INFINITY : sum.m[qt] + __log2f(sum.l[qt]);
        }
        const float by = a.n_split > 1 ? 1.f : sum.l[qt] == 0.f ? 0.f : 1.0f / sum.l[qt];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int d = 0; d < NDT; d += 4)
                *(float4 *)(p + NDT * (4 * kq + i) + d) = make_float4(sum.o[qt][d][i] * by, sum.o[qt][d + 1][i] * by,
                                                                      sum.o[qt][d + 2][i] * by, sum.o[qt][d + 3][i] * by);
        if (extra) {  // (onto a quotient as onto its numerator)
#pragma unroll 1
            for (int dim = NDT * 4 * kq; dim < NDT * 4 * (kq + 1); dim += 4) {
                float4 o = *(const float4 *)(p + dim);
                rows_add_nonfinite<HD, F16>(a, b, kvh, t, n, kbeg + max(full - kbeg, 0) / S::KEYS * S::KEYS, kend, dim, o);
                *(float4 *)(p + dim) = o;
            }
        }
    }
}

// The slices' join, 256 / (HD / 4 x SG) rows a workgroup.
template <int HD, int SG>
__global__ __launch_bounds__(256) void k_rows_merge(RowsArgs a, int64_t rows) {
    constexpr int TPR = HD / 4 * SG;  // threads a row
    __shared__ RowsJoin J;
    const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR, at = min(row, rows - 1);
    const int d = 4 * ((int)threadIdx.x % (HD / 4)), R = a.R;
    const int b = (int)(at / ((int64_t)a.HKV * R)), kvh = (int)(at / R % a.HKV), r = (int)(at % R), t = rows_div(r, a.g_m);
    const int n = rows_count(a, b), chunk = rows_chunk(rows_all(a, n), a.n_split, a.split_m, a.least);
    const int used = (rows_reach(a, n, t) + chunk - 1) / chunk;
    float M, l;
    const float4 o = rows_join<HD, SG>(J, a.part + at * a.n_split * (HD + 4), used, M, l);
    if (row >= rows || threadIdx.x % TPR >= HD / 4) return;
    *(float4 *)(a.out + rows_at(a, b, kvh, r) * HD + d) = rows_over(o, l);
    if (a.lse && d == 0) a.lse[row] = l == 0.f ? INFINITY : M + __log2f(l);
}

// One query a cache: the join (the first workgroup of a KV head) and acc_out = acc + the group's
// weights 2^(score - lse). Scores read, sums read and written: 44 MB in 15 us (16 of 12288 to 16384 keys), 3 TB/s, so
// latency more than HBM: the slices' sums, then the scores (requested before those: the same time). grid (1 + key
// blocks of 1024, HKV, B).
template <int HD>
__global__ __launch_bounds__(256) void k_one_weights(RowsArgs a, const float *acc, float *acc_out) {
    __shared__ RowsJoin J;
    __shared__ float lse[ROWS_MAX_G];
    constexpr int TPR = HD / 4 * JOIN_SG;
    const int kvh = blockIdx.y, b = blockIdx.z, G = a.H / a.HKV, tid = threadIdx.x;
    const int n = rows_count(a, b), chunk = rows_chunk(n, a.n_split, a.split_m, a.least), used = (n + chunk - 1) / chunk;
    const int64_t head = (int64_t)b * a.HKV + kvh, row0 = head * G;
    if (blockIdx.x == 0) {
        for (int g0 = 0; g0 < G; g0 += 256 / TPR) {
            const int g = g0 + tid / TPR;
            float M, l;
            const float4 o = rows_join<HD, JOIN_SG>(J, a.part + (row0 + min(g, G - 1)) * a.n_split * (HD + 4), used, M, l);
            if (g < G && tid % TPR < HD / 4)
                *(float4 *)(a.out + (row0 + g) * HD + 4 * (tid % TPR)) = rows_over(o, l);
        }
        return;
    }
    const int k0 = ((int)blockIdx.x - 1) * 1024 + 4 * tid;
    if (k0 - 4 * tid >= n) return;
    {  // 16 lanes a head over the slices' m and l
        const int g = tid / 16, s0 = tid % 16;
        float m[ROWS_MAX_SPLIT / 16], l[ROWS_MAX_SPLIT / 16], M = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < ROWS_MAX_SPLIT / 16; i++) {
            const int s = s0 + 16 * i;
            const bool in = g < G && s < used;
            const float2 ml = *(const float2 *)(a.part + ((row0 + (in ? g : 0)) * a.n_split + (in ? s : 0)) * (HD + 4));
            m[i] = in ? ml.x : -INFINITY, l[i] = in ? ml.y : 0.f, M = fmaxf(M, m[i]);
        }
        M = row_max_dpp(M);
#pragma unroll
        for (int i = 0; i < ROWS_MAX_SPLIT / 16; i++)
            if (m[i] != -INFINITY || l[i] != l[i])  // (a slice of NaN scores has no maximum)
                sum = fmaf(__builtin_amdgcn_exp2f(m[i] - M), l[i], sum);
        sum = row_sum_dpp(sum);
        if (s0 == 0) lse[g] = sum == 0.f ? INFINITY : M + __log2f(sum);  // (every score minus infinity: no weights)
    }
    __syncthreads();
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    if (k0 >= n) return;
    for (int g = 0; g < G; g++) {
        const float4 s = *(const float4 *)(a.scores + (row0 + g) * a.stride + k0);
        w[0] += __builtin_amdgcn_exp2f(s.x - lse[g]), w[1] += __builtin_amdgcn_exp2f(s.y - lse[g]);
        w[2] += __builtin_amdgcn_exp2f(s.z - lse[g]), w[3] += __builtin_amdgcn_exp2f(s.w - lse[g]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (k0 + i < n) acc_out[head * a.n_ctx + k0 + i] = acc[head * a.n_ctx + k0 + i] + w[i];
}

// A prompt chunk's weights summed over its queries, for each key: a wave holds a unit's
// K and goes over every other row tile's planes (the next one's requested before this one's products),
// sums 2^(score - lse) in its lanes, and the workgroup adds lanes and waves in order at the end. Four
// waves with units of their own take the same row tiles: the L1 serves three of them
// (256 queries over 4096 keys: 25 us; waves that shared a unit instead read 540 MB of planes from the L2, 32 us).
// grid (blocks of PW_UNITS units, HKV).
constexpr int PW_UNITS = 4, PW_ROWS = 2;
template <int HD, bool F16, int KT>
__global__ __launch_bounds__(64 * PW_UNITS * PW_ROWS) void k_prompt_weights(RowsArgs a, const float *acc, float *acc_out) {
    using S = RowsShape<HD, F16, KT>;
    constexpr int NC = S::NC;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rl = lane & 15, kq = lane >> 4, kvh = blockIdx.y;
    const int G = a.H / a.HKV, R = a.T * G, tiles = (R + 15) / 16, n = a.pos0 + a.T;
    const int unit = wave % PW_UNITS, rows = wave / PW_UNITS, k0 = (blockIdx.x * PW_UNITS + unit) * S::UNIT;
    __shared__ float part[PW_ROWS][PW_UNITS][KT][16];
    const RowsKv kv = rows_kv<HD, F16>(a.kv, (int64_t)kvh * a.n_ctx, n);
    RowsUnit<HD, F16, KT> u;
    ar_h8 ka[KT][NC];
    float ks[KT][NC][4], w[KT][4];
#pragma unroll
    for (int t = 0; t < KT; t++) {
#pragma unroll
        for (int c = 0; c < NC; c++)
            rows_words<S::KW>(kv.k, ((uint32_t)(k0 + 16 * t + rl) * HD + 32 * c + 8 * kq) * S::VB, u.k[t][c]);
        if constexpr (!F16) rows_words<2 * NC>(kv.ks, (uint32_t)(k0 + 16 * t + 4 * kq) * NC * 2, u.ks[t]);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            ka[t][c] = rows_values<S::KW>(u.k[t][c]);
#pragma unroll
            for (int i = 0; i < 4; i++)
                ks[t][c][i] = F16 ? 1.f : h2f((u.ks[t][F16 ? 0 : (i * NC + c) / 2] >> (16 * (c & 1))) & 0xffff);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) w[t][i] = 0.f;
    }
    // The first row that sees key k0: token max(0, k0 - pos0).
    const int first = k0 < n ? max(0, k0 - a.pos0) * G / 16 : tiles;
    const uint4 *pl = a.planes + (int64_t)kvh * tiles * NC * 2 * 64 + lane;
    struct Tile {
        uint4 h[NC], l[NC];
        float p2e, lse;
    } nxt;
    auto request = [&](int tile) {
        const int at = min(tile, tiles - 1);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            nxt.h[c] = pl[((int64_t)at * NC * 2 + 2 * c) * 64];
            nxt.l[c] = pl[((int64_t)at * NC * 2 + 2 * c + 1) * 64];
        }
        nxt.p2e = a.p2e[((int64_t)kvh * tiles + at) * 16 + rl];
        nxt.lse = a.lse[(int64_t)kvh * R + min(16 * at + rl, R - 1)];
    };
    request(first + rows);
    for (int tile = first + rows; tile < tiles; tile += PW_ROWS) {
        ar_h8 qh[NC], ql[NC];
#pragma unroll
        for (int c = 0; c < NC; c++) qh[c] = __builtin_bit_cast(ar_h8, nxt.h[c]), ql[c] = __builtin_bit_cast(ar_h8, nxt.l[c]);
        const float p2e = nxt.p2e, lse = nxt.lse;
        request(tile + PW_ROWS);
        const int r = 16 * tile + rl;
        const int last = a.pos0 + rows_div(r, a.g_m);  // the last key the row sees
#pragma unroll
        for (int t = 0; t < KT; t++) {
            float s[4];
            if constexpr (F16) {
                ar_f4 D = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    D = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[t][c], qh[c], D, 0, 0, 0);
                    D = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[t][c], ql[c], D, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) s[i] = D[i];
            } else {
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    ar_f4 D = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[t][c], qh[c], ar_f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                    D = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[t][c], ql[c], D, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) s[i] = c == 0 ? ks[t][c][i] * D[i] : fmaf(ks[t][c][i], D[i], s[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[i], p2e, -lse));
                w[t][i] += k0 + 16 * t + 4 * kq + i <= last && r < R ? p : 0.f;
            }
        }
    }
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x = row_sum_dpp(w[t][i]);
            if (rl == 0) part[rows][unit][t][4 * kq + i] = x;
        }
    __syncthreads();
    const int e = threadIdx.x, key = blockIdx.x * PW_UNITS * S::UNIT + e;
    if (e < PW_UNITS * S::UNIT && key < n) {
        float x = 0.f;
#pragma unroll
        for (int r = 0; r < PW_ROWS; r++) x += part[r][e / S::UNIT][e % S::UNIT / 16][e % 16];
        acc_out[(int64_t)kvh * a.n_ctx + key] = acc[(int64_t)kvh * a.n_ctx + key] + x;
    }
}

// ---- host ----------------------------------------------------------------------------------------

// How the R rows that a KV head has of a sequence's tokens are shared out.
struct RowsPlan {
    bool tile;
    int per, nrb, least, n_split;  // rows a workgroup, blocks of rows, keys a slice takes at least, slices
};
static int rows_splits(int items, int keys, int slots, int least) {
    const int most = std::min((keys + least - 1) / least, ROWS_MAX_SPLIT);
    return std::max(1, std::min(slots / std::max(items, 1), most));
}

// Up to 16 rows go to k_attn_rows, whose waves split the keys (8 caches of 16384 keys, 16 rows: 61 us, 85 by
// k_attn_tile), more to k_attn_tile, whose waves split the rows (20 rows: 80 us, 130 by two row tiles a wave
// there). Its waves take one row tile each, or two past 64 rows where every workgroup has more than 384
// keys to go through: a key's conversion then serves twice the rows (64 tokens of 32/8 heads over 8 x 16384 keys 320 us,
// 405 by one tile, over 8 x 4096 98 and 110), but a block takes longer (1 x 4096 37 and 33 us, 1 x 700 25 and 18).
// Two workgroups a CU, but three of up to 32 rows of a q8 cache (two of their waves have none, and the keys' conversion
// bounds them: 20 rows over 8 x 16384 keys 80 us, 96 by two; f16 97 and 92, 64 rows over 8 x 4096 43 and 41, heads of
// 64 over 8 x 4096 14.7 and 13.4).
// A slice reads at least half as many bytes of keys and values as its rows' queries and partials take, and 128 keys.
// Where that is more than 64 keys and slices are more than the CUs, 64 keys more (64 rows over 4096 keys, 8 KV heads:
// 192 keys a slice 19.9 us with the join, 128 21.9, 256 21.0; over 1500 keys 16.8, 15.1, 19.3); where it is not and
// slices are at most half of the CUs, 64 (20 rows over 1500 keys 11.5 us, 12.9 by 128; over 3 x 1500 16.5 and 15.5).
// The same rules hold where they were not found, whole calls in us, two row tiles and one: f16, 32/8 heads of 128, 64
// tokens over 8 x 16384 keys 263 and 316, 8 x 4096 90 and 97 (32 tokens 62 and 56: the rule's worst), 1 x 4096 33 and 29;
// f16, 14/2 heads of 64, 64 tokens over 8 x 16384 80 and 86, 1 x 4096 17.2 and 16.0. Three workgroups a CU and two:
// 8/4 heads of 256, 16 to 64 tokens over 8 x 4096, q8 48 to 89 and 38 to 72, f16 44 to 85 and 37 to 60.
// `keys` is a tree's capacity, not its length, which is in device memory: a cache that is far from full is cut into longer
// slices than its keys are worth.
static RowsPlan rows_plan(int seqs, int R, int HD, int kv_f16, int keys, int n_cu) {  // seqs: caches x KV heads
    RowsPlan p;
    p.tile = R > 16;
    const bool two = HD <= 128 && R > 64 && (int64_t)seqs * ((R + 127) / 128) * keys > (int64_t)384 * 2 * n_cu;
    p.per = !p.tile ? 16 : two ? 128 : 64;
    p.nrb = (R + p.per - 1) / p.per;
    const int key = 2 * (kv_f16 ? 2 * HD : HD + HD / 16), worth = std::min(R, p.per) * (2 * HD + 4) * 4 / (2 * key);
    p.least = std::max(ROWS_MIN_KEYS, (worth + 63) / 64 * 64);
    const int64_t all = (int64_t)seqs * p.nrb * keys;
    if (p.tile && worth > 64 && all > (int64_t)p.least * n_cu) p.least += 64;
    if (p.tile && worth <= 64 && 2 * all <= (int64_t)ROWS_MIN_KEYS * n_cu) p.least = 64;
    p.n_split = rows_splits(seqs * p.nrb, keys, (!p.tile ? 1 : R <= 32 && HD == 128 && !kv_f16 ? 3 : 2) * n_cu, p.least);
    return p;
}

bool attn_rows_supported(int H, int HKV, int HD) {
    return HKV > 0 && H > 0 && H % HKV == 0 && (HD == 64 || HD == 128 || HD == 256) && H / HKV <= ROWS_MAX_G;
}

// The arguments that follow from the others.
static void rows_derive(RowsArgs &a, int n_split, int nrb, int least) {
    a.G = a.H / a.HKV, a.R = a.T * a.G, a.nrb = nrb, a.least = least, a.n_split = n_split;
    a.g_m = rows_magic(a.G), a.nrb_m = rows_magic(nrb), a.split_m = rows_magic(n_split);
}

// 16-key tiles a unit of k_attn_rows.
constexpr int rows_kt(int HD) { return HD == 64 ? 2 : 1; }
template <int HD, bool F16>
static hipError_t rows_launch(const RowsArgs &a, const RowsPlan &p, int B, hipStream_t s) {
    const dim3 grid(a.n_split, a.HKV * a.nrb, B);
    constexpr int NW = HD == 256 ? 4 : 8;
    if (!p.tile) hipLaunchKernelGGL((k_attn_rows<HD, F16, rows_kt(HD), NW, false>), grid, dim3(64 * NW), 0, s, a);
    else if (p.per == 64) hipLaunchKernelGGL((k_attn_tile<HD, F16, 1>), grid, dim3(256), 0, s, a);
    else if constexpr (HD <= 128) hipLaunchKernelGGL((k_attn_tile<HD, F16, 2>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}
template <int HD>
static hipError_t rows_launch_merge(const RowsArgs &a, int B, hipStream_t s) {
    const int64_t rows = (int64_t)B * a.H * a.T;
    const auto grid = [&](int tpr) { return dim3((unsigned)((rows + 256 / tpr - 1) / (256 / tpr))); };
    if (a.n_split <= 8) hipLaunchKernelGGL((k_rows_merge<HD, 1>), grid(HD / 4), dim3(256), 0, s, a, rows);
    else hipLaunchKernelGGL((k_rows_merge<HD, JOIN_SG>), grid(HD / 4 * JOIN_SG), dim3(256), 0, s, a, rows);
    return hipGetLastError();
}
static RowsPlan tree_plan(int B, int T, int H, int HKV, int HD, int kv_f16, int n_ctx, int n_cu) {
    return rows_plan(B * HKV, T * (H / HKV), HD, kv_f16, n_ctx, n_cu);
}
size_t attn_tree_scratch_bytes(int B, int T, int H, int HKV, int HD, int kv_f16, int n_ctx, int n_cu) {
    const int ns = tree_plan(B, T, H, HKV, HD, kv_f16, n_ctx, n_cu).n_split;
    return ns > 1 ? (size_t)B * T * H * ns * (HD + 4) * sizeof(float) : 0;
}
hipError_t launch_attn_tree(const float *q, int B, int T, int H, int HKV, int HD, KvLayer kv, int kv_f16, int n_ctx,
                            const int32_t *n_past, const uint64_t *mask, float scale, float *part, float *out, int n_cu,
                            hipStream_t s) {
    const RowsPlan p = tree_plan(B, T, H, HKV, HD, kv_f16, n_ctx, n_cu);
    RowsArgs a{};
    a.q = q, a.kv = kv, a.n_ctx = n_ctx, a.H = H, a.HKV = HKV, a.T = T, a.n_keys = n_past, a.mask = mask;
    a.mode = ROWS_TREE, a.scale = scale, a.part = part, a.out = out;
    rows_derive(a, p.n_split, p.nrb, p.least);
    return rows_by_shape(HD, kv_f16, [&](auto hd, auto f16) {
        const hipError_t e = rows_launch<decltype(hd)::value, decltype(f16)::value>(a, p, B, s);
        return e != hipSuccess || a.n_split == 1 ? e : rows_launch_merge<decltype(hd)::value>(a, B, s);
    });
}

// Two rounds of the three workgroups that a CU holds: sequences of different lengths leave less of the
// last one idle (16 of 12288 to 16384 keys: 121 us, 125 in one round, 132 in one and a third).
static int one_splits(int B, int HKV, int n_ctx, int n_cu) { return rows_splits(B * HKV, n_ctx, 6 * n_cu, ROWS_MIN_KEYS); }
static int64_t one_stride(int n_ctx) { return ((int64_t)n_ctx + 31) / 32 * 32; }
size_t attn_one_weights_scratch_bytes(int B, int H, int HKV, int HD, int n_ctx, int n_cu) {
    return (size_t)B * H * (one_stride(n_ctx) + (size_t)one_splits(B, HKV, n_ctx, n_cu) * (HD + 4)) * sizeof(float);
}
hipError_t launch_attn_one_weights(const float *q, int B, int H, int HKV, int HD, KvLayer kv, int kv_f16, int n_ctx,
                                   const int32_t *n_keys, float scale, void *scratch, float *out, const float *acc,
                                   float *acc_out, int n_cu, hipStream_t s) {
    RowsArgs a{};
    a.q = q, a.kv = kv, a.n_ctx = n_ctx, a.H = H, a.HKV = HKV, a.T = 1, a.n_keys = n_keys;
    a.mode = ROWS_ONE, a.scale = scale, a.out = out, a.stride = one_stride(n_ctx);
    a.scores = (float *)scratch, a.part = a.scores + (int64_t)B * H * a.stride;
    rows_derive(a, one_splits(B, HKV, n_ctx, n_cu), 1, ROWS_MIN_KEYS);
    return rows_by_shape(HD, kv_f16, [&](auto hd, auto f16) {
        constexpr int D = decltype(hd)::value;
        hipLaunchKernelGGL((k_attn_rows<D, decltype(f16)::value, rows_kt(D), 4, true>), dim3(a.n_split, HKV, B), dim3(256), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(k_one_weights<D>, dim3(1 + (n_ctx + 1023) / 1024, HKV, B), dim3(256), 0, s, a, acc,
                           acc_out);
        return hipGetLastError();
    });
}

struct PromptWeightsScratch {
    RowsPlan plan;
    size_t planes, p2e, lse, part, bytes;  // where each begins, and the end
};
static PromptWeightsScratch prompt_scratch(int nq, int H, int HKV, int HD, int kv_f16, int n_keys, int n_cu) {
    const size_t R = (size_t)nq * (H / HKV), tiles = (R + 15) / 16;
    PromptWeightsScratch p;
    p.plan = rows_plan(HKV, (int)R, HD, kv_f16, n_keys, n_cu);
    p.planes = 0;
    p.p2e = p.planes + align_up(HKV * tiles * HD / 32 * 2 * 64 * sizeof(uint4), 256);
    p.lse = p.p2e + align_up(HKV * tiles * 16 * sizeof(float), 256);
    p.part = p.lse + align_up(HKV * R * sizeof(float), 256);
    p.bytes = p.part + (p.plan.n_split > 1 ? (size_t)nq * H * p.plan.n_split * (HD + 4) * sizeof(float) : 0);
    return p;
}
size_t attn_prompt_weights_scratch_bytes(int nq, int H, int HKV, int HD, int kv_f16, int n_keys, int n_cu) {
    return prompt_scratch(nq, H, HKV, HD, kv_f16, n_keys, n_cu).bytes;
}
void attn_prompt_weights_layout(int nq, int H, int HKV, int HD, int kv_f16, int n_keys, int n_cu, size_t at[4]) {
    const PromptWeightsScratch p = prompt_scratch(nq, H, HKV, HD, kv_f16, n_keys, n_cu);
    at[0] = p.planes, at[1] = p.p2e, at[2] = p.lse, at[3] = p.part;
}
hipError_t launch_attn_prompt_weights(const float *q, int nq, int H, int HKV, int HD, KvLayer kv, int kv_f16, int n_ctx,
                                      int pos0, float scale, void *scratch, float *out, const float *acc,
                                      float *acc_out, int n_cu, hipStream_t s) {
    const PromptWeightsScratch p = prompt_scratch(nq, H, HKV, HD, kv_f16, pos0 + nq, n_cu);
    uint8_t *base = (uint8_t *)scratch;
    RowsArgs a{};
    a.q = q, a.kv = kv, a.n_ctx = n_ctx, a.H = H, a.HKV = HKV, a.T = nq, a.pos0 = pos0;
    a.mode = ROWS_CAUSAL, a.scale = scale, a.out = out;
    a.planes = (uint4 *)(base + p.planes), a.p2e = (float *)(base + p.p2e), a.lse = (float *)(base + p.lse);
    a.part = (float *)(base + p.part);
    rows_derive(a, p.plan.n_split, p.plan.nrb, p.plan.least);
    return rows_by_shape(HD, kv_f16, [&](auto hd, auto f16) {
        constexpr int D = decltype(hd)::value;
        constexpr bool F = decltype(f16)::value;
        hipError_t e = rows_launch<D, F>(a, p.plan, 1, s);
        if (e == hipSuccess && a.n_split > 1) e = rows_launch_merge<D>(a, 1, s);
        if (e != hipSuccess) return e;
        constexpr int KT = D == 256 ? 1 : 2, per = PW_UNITS * 16 * KT;
        hipLaunchKernelGGL((k_prompt_weights<D, F, KT>), dim3((pos0 + nq + per - 1) / per, HKV),
                           dim3(64 * PW_UNITS * PW_ROWS), 0, s, a, acc, acc_out);
        return hipGetLastError();
    });
}

}  // namespace ts5hip
