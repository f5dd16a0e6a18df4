// Attention of rows of queries over keys of one KV head on the matrix cores:
// the device core of the tree, key-weight and block-sparse attention kernels
// (attn_rows.hip, attn_sparse.hip). Head dimension 64, 128 or 256, a q8 or f16 cache.
//
// A row is one query head of one token; a wave holds 16 NT of them and takes
// units of 16 KT keys, its rows' running maximum, sum and output in
// registers:
//  * S^T (keys x rows) = K . Q^T on v_mfma_f32_16x16x32_f16: the rows as fp16 hi + lo
//    planes of q * scale * log2(e) * 2^-e (e per row keeps them in range: about 22
//    bits, the planes' products are exact and summed in fp32); q8: K as exact
//    integers, one product per 32-value scale group, then S += ks * R.
//  * online softmax per row in the log2 domain; the rows are the lanes'
//    columns. The reference is a running maximum less 7, so that weights go past
//    128 and their lo plane stays out of the fp16 subnormals; it follows the true
//    maximum only once that is 4 above it (weights to 2^11), so that the sums are rarely scaled.
//    A weight's planes end at 2^-24: beside its relative 2^-22 it is off by up to 2^-32 of the row's largest, which
//    shows only in a dim where the large weights all meet values of 0.
//  * O^T (dims x rows) += V^T . P^T. The D layout of S^T (lane: keys 4 kq .. + 3 of
//    each tile) is the B layout of P^T, so P stays in registers as hi + lo. For V^T
//    the lane in MFMA row m = lane & 15 and key group kq = lane >> 4 loads keys 4 kq ..
//    + 3, dims HD / 16 * m .. : tile dt takes dim HD / 16 * m + dt as its row m, so
//    the A operand is the lane's own data and V needs no transpose through LDS.
//    q8: v8 * vs is exact in 19 bits and goes in as fp16 hi + lo (Vh Ph + Vl Ph + Vh
//    Pl); values past fp16's range (65504) are infinite, as in an f16 cache.
// A workgroup's waves take units of a slice of the keys in turn and combine
// their (m, l, O) in LDS; slices combine through partials [HD + 4] floats long
// (m, l, -, -, O).
#pragma once
#include "attn_core.h"

namespace ts5hip {

typedef _Float16 ar_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 ar_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 ar_h2 __attribute__((ext_vector_type(2)));
typedef float ar_f2 __attribute__((ext_vector_type(2)));
typedef float ar_f4 __attribute__((ext_vector_type(4)));

constexpr float AR_LOG2E = 1.4426950408889634f;

// A unit of KT = 1 or 2 tiles of 16 keys: two make one value product of 32 keys,
// one leaves the registers for more rows, longer heads or more waves.
template <int HD, bool F16, int KT_>
struct RowsShape {
    static constexpr int KT = KT_;                       // 16-key tiles a unit
    static constexpr int UNIT = 16 * KT;
    static constexpr int NC = HD / 32;                   // 32-value chunks (q8 scale groups)
    static constexpr int NDT = HD / 16;                  // 16-dim output tiles = dims a lane holds of a value row
    static constexpr int VB = F16 ? 2 : 1;
    static constexpr int KW = F16 ? 4 : 2;               // dwords of 8 K values
    static constexpr int VW = NDT * VB / 4;              // dwords of a lane's V dims
};

// One KV head's keys [0, n) as bounded buffers: past n they read zeros.
struct RowsKv {
    __amdgpu_buffer_rsrc_t k, v, ks, vs;
};
template <int HD, bool F16>
__device__ inline RowsKv rows_kv(const KvLayer &kv, int64_t head_slot, int n) {
    constexpr int VB = F16 ? 2 : 1;
    RowsKv r;
    r.k = slice_rsrc(kv.k + head_slot * HD * VB, (uint32_t)n * HD * VB);
    r.v = slice_rsrc(kv.v + head_slot * HD * VB, (uint32_t)n * HD * VB);
    r.ks = r.k, r.vs = r.v;
    if constexpr (!F16) {
        r.ks = slice_rsrc(kv.ks + head_slot * (HD / 32), (uint32_t)n * (HD / 32) * 2);
        r.vs = slice_rsrc(kv.vs + head_slot * (HD / 32), (uint32_t)n * (HD / 32) * 2);
    }
    return r;
}

template <int N>
__device__ inline void rows_words(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t (&w)[N]) {
    static_assert(N == 1 || N == 2 || N % 4 == 0, "whole loads");
    if constexpr (N == 1) {
        w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
    } else if constexpr (N == 2) {
        const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
        w[0] = x[0], w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, off + 4 * i, 0, 0);
            w[i] = x[0], w[i + 1] = x[1], w[i + 2] = x[2], w[i + 3] = x[3];
        }
    }
}

// A unit's loads: tile t at key kb[t].
template <int HD, bool F16, int KT>
struct RowsUnit {
    using S = RowsShape<HD, F16, KT>;
    uint32_t k[KT][S::NC][S::KW];  // key rl of the tile, dims 32 c + 8 kq .. + 7
    uint32_t v[KT][4][S::VW];      // key 4 kq + i, dims NDT rl .. + NDT - 1
    uint32_t ks[KT][F16 ? 4 : 2 * S::NC];  // q8: keys 4 kq .. + 3, every group
    uint16_t vs[KT][4];            // q8: key 4 kq + i, the lane's dims' group
};
template <int HD, bool F16, int KT>
__device__ inline void rows_load(RowsUnit<HD, F16, KT> &u, const RowsKv &kv, const int (&kb)[KT],
                                 int rl, int kq) {
    using S = RowsShape<HD, F16, KT>;
#pragma unroll
    for (int t = 0; t < KT; t++) {
#pragma unroll
        for (int c = 0; c < S::NC; c++)
            rows_words<S::KW>(kv.k, ((uint32_t)(kb[t] + rl) * HD + 32 * c + 8 * kq) * S::VB, u.k[t][c]);
        if constexpr (!F16) rows_words<2 * S::NC>(kv.ks, (uint32_t)(kb[t] + 4 * kq) * S::NC * 2, u.ks[t]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t key = (uint32_t)(kb[t] + 4 * kq + i);
            rows_words<S::VW>(kv.v, (key * HD + S::NDT * rl) * S::VB, u.v[t][i]);
            if constexpr (!F16)
                u.vs[t][i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(kv.vs, key * S::NC * 2 + rl * S::NDT / 32 * 2, 0, 0);
        }
    }
}

// 8 int8 -> 8 exact fp16: 0x64xx is 1024 + xx, so (b + 128) in the low byte
// gives 1152 + b.
template <int N>
__device__ inline ar_h8 rows_values(const uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        return __builtin_bit_cast(ar_h8, u32x4{w[0], w[1], w[2], w[3]});
    } else {
        const ar_h2 k1152 = {(_Float16)1152.0f, (_Float16)1152.0f};
        ar_h2 h[4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t x = w[i] ^ 0x80808080u;
            h[2 * i] = __builtin_bit_cast(ar_h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - k1152;
            h[2 * i + 1] = __builtin_bit_cast(ar_h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - k1152;
        }
        return ar_h8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
    }
}

// Two fp32 as fp16 pairs hi + lo, x = hi + lo to about 22 bits.
__device__ inline void rows_split(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    const ar_f2 x = {x0, x1};
    const ar_h2 h = __builtin_convertvector(x, ar_h2);  // v_cvt_pk_f16_f32
    hi = __builtin_bit_cast(uint32_t, h);
    ar_f2 r;  // x - h: one instruction a half
    float r0, r1;
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(hi), "v"(x0));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(hi), "v"(x1));
    r[0] = r0, r[1] = r1;
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, ar_h2));
}

// The lane's rows (its MFMA columns), row 16 qt + rl of the wave's: B operands of dims
// 32 c + 8 kq .. + 7, and 2^e. row(qt, ok) is the row's address; a column without a row (not ok) has one to
// read from all the same, since a load under a branch would wait for the one before it, and zeros (which
// cost the matrix cores less power: copies of a row took 10 % longer).
template <int HD, int NT>
struct RowsQ {
    ar_h8 h[NT][HD / 32], l[NT][HD / 32];
    float p2e[NT];
};
template <int HD, int NT>
struct RowsIn {
    float4 x[NT][HD / 32][2];
    bool ok[NT];
};
template <int HD, int NT, class Row>
__device__ inline void rows_request(RowsIn<HD, NT> &in, int kq, Row row) {
#pragma unroll
    for (int qt = 0; qt < NT; qt++) {
        const float *p = row(qt, in.ok[qt]) + 8 * kq;
#pragma unroll
        for (int c = 0; c < HD / 32; c++)
            in.x[qt][c][0] = *(const float4 *)(p + 32 * c), in.x[qt][c][1] = *(const float4 *)(p + 32 * c + 4);
    }
}
// With WIDE, rows whose largest value is past fp32's range once it is scaled keep their 2^e all the same.
template <int HD, int NT, bool WIDE = false>
__device__ inline void rows_query(RowsQ<HD, NT> &q, const RowsIn<HD, NT> &in, float scale) {
    constexpr int NC = HD / 32;
    const float by = scale * AR_LOG2E;
#pragma unroll
    for (int qt = 0; qt < NT; qt++) {
        float amax = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float4 x = in.x[qt][c][k];
                // (fmaxf quiets each operand first: three instructions a value)
                asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(amax) : "v"(x.x), "v"(x.y));
                asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(amax) : "v"(x.z), "v"(x.w));
            }
        amax = max_xor32(max_xor16(amax));
        const float most = amax;
        amax *= fabsf(by);
        int e = amax > 0.f ? max(ilogbf(amax) - 13, -100) : 0;
        if (WIDE && amax == INFINITY && most < INFINITY && fabsf(by) < INFINITY) e = ilogbf(most) + ilogbf(by) - 12;
        const float sc = in.ok[qt] ? ldexpf(by, -e) : 0.f;  // (one rounding of q * by: the rest is a power of 2)
        q.p2e[qt] = ldexpf(1.0f, e);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            u32x4 h, l;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float4 x = in.x[qt][c][k];
                uint32_t h0, l0, h1, l1;
                rows_split(x.x * sc, x.y * sc, h0, l0);
                rows_split(x.z * sc, x.w * sc, h1, l1);
                h[2 * k] = h0, h[2 * k + 1] = h1, l[2 * k] = l0, l[2 * k + 1] = l1;
            }
            q.h[qt][c] = __builtin_bit_cast(ar_h8, h), q.l[qt][c] = __builtin_bit_cast(ar_h8, l);
        }
    }
}

template <int HD, int NT>
struct RowsSum {
    float m[NT], l[NT];    // (l: the lane's keys' share)
    ar_f4 o[NT][HD / 16];  // dim HD / 16 * (4 kq + i) + dt of row 16 qt + rl
};
template <int HD, int NT>
__device__ inline void rows_clear(RowsSum<HD, NT> &a) {
#pragma unroll
    for (int qt = 0; qt < NT; qt++) {
        a.m[qt] = -INFINITY, a.l[qt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < HD / 16; dt++) a.o[qt][dt] = ar_f4{0.f, 0.f, 0.f, 0.f};
    }
}

// S^T of a unit: s[t][i] (times 2^-e) of key 4 kq + i of tile t, row rl.
template <int HD, bool F16, int KT>
__device__ inline void rows_scores(const RowsUnit<HD, F16, KT> &u, const RowsQ<HD, 1> &q, float (&s)[KT][4]) {
    using S = RowsShape<HD, F16, KT>;
#pragma unroll
    for (int t = 0; t < KT; t++) {
        if constexpr (F16) {
            ar_f4 R = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < S::NC; c++) {
                const ar_h8 ka = rows_values<S::KW>(u.k[t][c]);
                R = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q.h[0][c], R, 0, 0, 0);
                R = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q.l[0][c], R, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) s[t][i] = R[i];
        } else {
#pragma unroll
            for (int c = 0; c < S::NC; c++) {
                const ar_h8 ka = rows_values<S::KW>(u.k[t][c]);
                float ks[4];
#pragma unroll
                for (int i = 0; i < 4; i++) ks[i] = h2f((u.ks[t][(i * S::NC + c) / 2] >> (16 * (c & 1))) & 0xffff);
                ar_f4 R = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q.h[0][c], ar_f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                R = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q.l[0][c], R, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) s[t][i] = c == 0 ? ks[i] * R[i] : fmaf(ks[i], R[i], s[t][i]);
            }
        }
    }
}

// The value products' A operand of tile dt: the lane's values dim NDT rl + dt of keys
// 4 kq .. + 3 of each tile; q8 as hi + lo of v8 * vs.
template <int HD, bool F16, int KT>
struct RowsScale {
    ar_h2 s[KT][2];
};
// The pair (key a, key b) of dim j of value dwords wa, wb, times their scales (q8).
template <bool F16>
__device__ inline void rows_value_pair(uint32_t wa, uint32_t wb, int j, ar_h2 sc, uint32_t &hi, uint32_t &lo) {
    if constexpr (F16) {
        hi = __builtin_amdgcn_perm(wb, wa, j & 1 ? 0x07060302u : 0x05040100u);
        lo = 0;
    } else {
        const ar_h2 k1152 = {(_Float16)1152.0f, (_Float16)1152.0f};
        const uint32_t b = __builtin_amdgcn_perm(wb ^ 0x80808080u, wa ^ 0x80808080u, 0x0c000c00u | (uint32_t)(4 + j) << 16 | (uint32_t)j);
        const ar_h2 v = __builtin_bit_cast(ar_h2, b | 0x64006400u) - k1152;
        const ar_h2 h = v * sc;
        hi = __builtin_bit_cast(uint32_t, h);
        lo = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(v, sc, -h));
    }
}
template <int HD, bool F16, int KT>
__device__ inline void rows_value_tile(const RowsUnit<HD, F16, KT> &u, const RowsScale<HD, F16, KT> &sc, int dt,
                                       uint32_t (&hi)[2 * KT],
                                       uint32_t (&lo)[2 * KT]) {
    constexpr int PW = F16 ? 2 : 4;  // dims a dword
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int p = 0; p < 2; p++)
            rows_value_pair<F16>(u.v[t][2 * p][dt / PW], u.v[t][2 * p + 1][dt / PW], dt % PW, sc.s[t][p], hi[2 * t + p],
                                 lo[2 * t + p]);
}
template <int KT>
struct RowsOp;
template <>
struct RowsOp<1> {
    using T = ar_h4;
    __device__ static T of(const uint32_t (&w)[2]) { return __builtin_bit_cast(T, u32x2{w[0], w[1]}); }
    __device__ static ar_f4 mfma(T a, T b, ar_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
};
template <>
struct RowsOp<2> {
    using T = ar_h8;
    __device__ static T of(const uint32_t (&w)[4]) { return __builtin_bit_cast(T, u32x4{w[0], w[1], w[2], w[3]}); }
    __device__ static ar_f4 mfma(T a, T b, ar_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// The rows' reference for weights of scores up to mx (log2 domain): raised, and the sums
// scaled, where some row's maximum is past it by ROWS_SLACK. Returns what scores are taken less.
constexpr float ROWS_SLACK = 4.f;
template <int HD, int NT>
__device__ inline float rows_reference(RowsSum<HD, NT> &a, int qt, float mx) {
    mx -= 7.f;
    if (__builtin_amdgcn_ballot_w64(mx > a.m[qt] + ROWS_SLACK)) {
        const float mn = fmaxf(a.m[qt], mx), alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(a.m[qt] - mn);
        a.m[qt] = mn, a.l[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < HD / 16; dt++) a.o[qt][dt] *= alpha;
    }
    return a.m[qt] == -INFINITY ? 0.f : a.m[qt];  // (no key yet: every weight is 0)
}

// Bits 0..3: which of keys key .. + 3 lie below n.
__device__ inline uint32_t rows_below(int key, int n) { return (1u << max(0, min(n - key, 4))) - 1u; }
// Bits 0..3: bits at .. at + 3 of x (at from -3 on; none past its end).
__device__ inline uint32_t rows_window(uint64_t x, int at) {
    const uint64_t r = x >> min(max(at, 0), 63), l = x << min(max(-at, 0), 63);
    return at >= 64 ? 0u : (uint32_t)(at >= 0 ? r : l) & 15u;
}

// One unit into the sums. With MASK, seen(key) has a bit for each of keys key .. + 3 that a
// row takes: bits, and no `a || b ? score : -inf` of a key at a time. The compiler (LLVM 22 of ROCm 7.2.0,
// structurizecfg, whatever the flags) moves an element of a product's vector, which costs nothing, out of the block that
// such a branch guards, and lanes that come to the block by b, not by a, get -inf: the score's register took b's
// shift and then -inf, and the block that had to bring the score back was empty (f16 scores are elements; q8's are sums).
// With SAN infinite and NaN values are left out (the product with a row that does not
// take their key would be NaN), and the unit says that it had some: they are added
// where the rows are written.
template <int HD, bool F16, int KT, bool MASK, bool SAN, class Seen, class Put>
__device__ inline bool rows_unit(const RowsUnit<HD, F16, KT> &u, const RowsQ<HD, 1> &q, RowsSum<HD, 1> &a,
                                 const int (&kb)[KT], int kq, Seen seen, Put put) {
    using S = RowsShape<HD, F16, KT>;
    using Op = RowsOp<KT>;
    float s[KT][4];
    rows_scores<HD, F16, KT>(u, q, s);
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < KT; t++) {
        const uint32_t take = MASK ? seen(kb[t] + 4 * kq) : 15u;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (MASK) s[t][i] = take & 1u << i ? s[t][i] : -INFINITY;
            mx = fmaxf(mx, s[t][i]);
        }
    }
#pragma unroll
    for (int t = 0; t < KT; t++) put(kb[t] + 4 * kq, s[t]);
    const float m0 = rows_reference(a, 0, max_xor32(max_xor16(mx)) * q.p2e[0]);
    float sum = 0.f;
    uint32_t whi[2 * KT], wlo[2 * KT];
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[t][2 * i], q.p2e[0], -m0));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[t][2 * i + 1], q.p2e[0], -m0));
            sum += p0 + p1;
            rows_split(p0, p1, whi[2 * t + i], wlo[2 * t + i]);
        }
    const typename Op::T ph = Op::of(whi), pl = Op::of(wlo);
    a.l[0] += sum;  // (the lane's share: its four keys of each tile)
    RowsScale<HD, F16, KT> sc;
    if constexpr (!F16) {
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int p = 0; p < 2; p++)
                sc.s[t][p] = __builtin_bit_cast(ar_h2, (uint32_t)u.vs[t][2 * p] | (uint32_t)u.vs[t][2 * p + 1] << 16);
    }
    // With SAN: whether any value is infinite or NaN, and then with those left out.
    bool bad = false;
    if constexpr (SAN) {
        uint32_t any = 0;  // bit 15 or 31: an exponent of all ones
#pragma unroll
        for (int dt = 0; dt < S::NDT; dt++) {
            uint32_t hi[2 * KT], lo[2 * KT];
            rows_value_tile<HD, F16, KT>(u, sc, dt, hi, lo);
#pragma unroll
            for (int w = 0; w < 2 * KT; w++) any |= (hi[w] & 0x7c007c00u) + 0x04000400u;
        }
        bad = __builtin_amdgcn_ballot_w64((any & 0x80008000u) != 0) != 0;
    }
    auto products = [&](auto clean) {
#pragma unroll
        for (int dt = 0; dt < S::NDT; dt++) {
            uint32_t hi[2 * KT], lo[2 * KT];
            rows_value_tile<HD, F16, KT>(u, sc, dt, hi, lo);
            if constexpr (decltype(clean)::value) {
#pragma unroll
                for (int w = 0; w < 2 * KT; w++) {
                    uint32_t keep = 0;
                    if ((hi[w] & 0x7c00u) != 0x7c00u) keep |= 0xffffu;
                    if ((hi[w] & 0x7c000000u) != 0x7c000000u) keep |= 0xffff0000u;
                    hi[w] &= keep, lo[w] &= keep;
                }
            }
            const typename Op::T vh = Op::of(hi), vl = Op::of(lo);
            a.o[0][dt] = Op::mfma(vh, ph, a.o[0][dt]);
            if constexpr (!F16) a.o[0][dt] = Op::mfma(vl, ph, a.o[0][dt]);
            a.o[0][dt] = Op::mfma(vh, pl, a.o[0][dt]);
        }
    };
    if (!SAN || !bad) products(std::false_type{});
    else products(std::true_type{});
    return SAN && bad;
}

// An infinite or NaN value as the products see it (fp16's range), else 0: dim d of slot `slot`.
template <int HD, bool F16>
__device__ inline float rows_nonfinite(const KvLayer &kv, int64_t slot, int d) {
    _Float16 h;
    if constexpr (F16) h = __builtin_bit_cast(_Float16, ((const uint16_t *)kv.v)[slot * HD + d]);
    else h = (_Float16)(float)kv.v[slot * HD + d] * __builtin_bit_cast(_Float16, kv.vs[slot * (HD / 32) + d / 32]);
    return (__builtin_bit_cast(uint16_t, h) & 0x7c00) == 0x7c00 ? (float)h : 0.f;
}

// The waves' sums of the workgroup's 16 rows, combined: emit(row, d, o, m, l) once
// for each row below `rows` and 4 dims from d on. Every thread calls it.
template <int HD, int NW>
struct RowsLds {
    __align__(16) float o[NW][16][HD + 4];
    float m[NW][16], l[NW][16];
};
template <int HD, int NW, class Emit>
__device__ inline void rows_combine(RowsLds<HD, NW> &L, const RowsSum<HD, 1> &a, int rows, int wave, int rl, int kq,
                                    Emit emit) {
    constexpr int NDT = HD / 16;
    const int nr = min(rows, 16);
    __syncthreads();
    const float sum = add_xor32(add_xor16(a.l[0]));
    if (rl < nr) {
        if (kq == 0) L.m[wave][rl] = a.m[0], L.l[wave][rl] = sum;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int d = 0; d < NDT; d += 4)
                *(float4 *)&L.o[wave][rl][NDT * (4 * kq + i) + d] =
                    make_float4(a.o[0][d][i], a.o[0][d + 1][i], a.o[0][d + 2][i], a.o[0][d + 3][i]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nr * (HD / 4); e += 64 * NW) {
        const int r = e / (HD / 4), d = 4 * (e % (HD / 4));
        float M = L.m[0][r];
#pragma unroll
        for (int w = 1; w < NW; w++) M = fmaxf(M, L.m[w][r]);
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float lw = L.l[w][r];
            const float x = lw != lw ? lw : L.m[w][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(L.m[w][r] - M);
            if (x == 0.f) continue;  // (a wave with no key of the row; NaN scores have no maximum)
            const float4 p = *(const float4 *)&L.o[w][r][d];
            l = fmaf(x, lw, l);
            o.x = fmaf(x, p.x, o.x), o.y = fmaf(x, p.y, o.y), o.z = fmaf(x, p.z, o.z), o.w = fmaf(x, p.w, o.w);
        }
        emit(r, d, o, M, l);
    }
}

// x / d for 0 <= x < 2^26, x d < 2^36, as one multiplication by m = rows_magic(d): m d is less than d above
// 2^36, so the error stays under x / 2^36 < 1 / d, and x m under 2^63.
__host__ inline uint64_t rows_magic(int d) { return ((1ull << 36) + d - 1) / d; }
__host__ __device__ inline int rows_div(int x, uint64_t m) { return (int)((uint64_t)(uint32_t)x * m >> 36); }

// Keys of each of n_split slices of n keys: at least `least`, and whole blocks of k_attn_tile (a slice that
// ended inside one would count the zeros behind it).
constexpr int ROWS_MIN_KEYS = 128;
constexpr int ROWS_MAX_SPLIT = 64;
__host__ __device__ inline int rows_chunk(int n, int n_split, uint64_t split_m, int least) {  // split_m = rows_magic(n_split)
    int c = rows_div(n + n_split - 1, split_m);
    c = c < least ? least : c;
    return (c + 63) / 64 * 64;
}

constexpr int ROWS_MAX_G = 16;  // query heads a KV head, where one row tile holds a query's

// sum_s 2^(m_s - M) (O_s, l_s) over the first `used` slices of a row's partials: HD / 4 x SG of a
// workgroup's 256 threads a row, 4 dims a thread and every SG-th slice, eight of them
// requested before the first is used (one at a time their latencies add up: 32 slices took 27 us, now
// 5); the SG parts join in LDS in order. Every thread of the workgroup calls it; the result is the SG = 0 part's.
constexpr int JOIN_SG = 4;
struct RowsJoin {
    __align__(16) float4 o[256];
    float2 ml[256];
};
// load(s, d, ml, x) loads slice s's m and l and its dims d .. + 3.
template <int HD, int SG, class Join, class Load>
__device__ inline float4 rows_join(Join &J, int used, float &M, float &l, Load load) {
    constexpr int L4 = HD / 4, AHEAD = 8;
    const int tid = threadIdx.x, sg = tid / L4 % SG, d = 4 * (tid % L4);
    M = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float m, float pl, float4 x) {
        const float mn = fmaxf(M, m);
        if (l != l || pl != pl) {  // a row of NaN scores has no maximum
            l = NAN, o = make_float4(NAN, NAN, NAN, NAN);
            return;
        }
        if (mn == -INFINITY) return;
        const float a = __builtin_amdgcn_exp2f(M - mn), w = __builtin_amdgcn_exp2f(m - mn);
        M = mn;
        if (a == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f), l = 0.f;  // (nothing yet: no 0 times an infinity)
        else o.x *= a, o.y *= a, o.z *= a, o.w *= a, l *= a;
        if (w == 0.f) return;
        l = fmaf(w, pl, l);
        o.x = fmaf(w, x.x, o.x), o.y = fmaf(w, x.y, o.y), o.z = fmaf(w, x.z, o.z), o.w = fmaf(w, x.w, o.w);
    };
    for (int s0 = sg; s0 < used; s0 += AHEAD * SG) {
        float2 ml[AHEAD];
        float4 x[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) load(min(s0 + i * SG, used - 1), d, ml[i], x[i]);
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (s0 + i * SG < used) add(ml[i].x, ml[i].y, x[i]);
    }
    if constexpr (SG > 1) {
        __syncthreads();
        J.o[tid] = o, J.ml[tid] = make_float2(M, l);
        __syncthreads();
        if (sg == 0) {
#pragma unroll
            for (int i = 1; i < SG; i++) add(J.ml[tid + i * L4].x, J.ml[tid + i * L4].y, J.o[tid + i * L4]);
        }
    }
    return o;
}
// Partials that an earlier launch wrote.
template <int HD, int SG>
__device__ inline float4 rows_join(RowsJoin &J, const float *p, int used, float &M, float &l) {
    return rows_join<HD, SG>(J, used, M, l, [&](int s, int d, float2 &ml, float4 &x) {
        const float *r = p + (int64_t)s * (HD + 4);
        ml = *(const float2 *)r, x = *(const float4 *)(r + 4 + d);
    });
}
// The row's output.
__device__ inline float4 rows_over(float4 o, float l) {
    const float inv = 1.0f / l;
    return l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// f(head dimension, whether f16) with both as constants.
template <class F>
static hipError_t rows_by_shape(int HD, int kv_f16, F f) {
    switch (HD * 2 + (kv_f16 ? 1 : 0)) {
    case 128: return f(std::integral_constant<int, 64>{}, std::false_type{});
    case 129: return f(std::integral_constant<int, 64>{}, std::true_type{});
    case 256: return f(std::integral_constant<int, 128>{}, std::false_type{});
    case 257: return f(std::integral_constant<int, 128>{}, std::true_type{});
    case 512: return f(std::integral_constant<int, 256>{}, std::false_type{});
    case 513: return f(std::integral_constant<int, 256>{}, std::true_type{});
    }
    return hipErrorInvalidValue;
}

}  // namespace ts5hip
