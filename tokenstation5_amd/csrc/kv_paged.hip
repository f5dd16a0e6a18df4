// Rows into and out of a cache in pages: the new tokens' q, k, v (bias, per-head norm, RoPE, then K and V rounded as
// the cache keeps them), and cached rows as fp32 or f16 values.
#include <algorithm>

#include "attn_core.h"

namespace ts5hip {

// A pool of pages, [page][KV head][slot][HD], and the sequences' tables.
struct PagedPool {
    KvLayer kv;
    const int32_t *table;  // [n_seq][n_table]
    int n_pages, lp, n_seq, n_table, HKV;  // lp: log2 of the page
};
// The slot of KV head 0 of token (seq, pos), or -1: the others follow a page's length apart.
__device__ inline int64_t paged_slot(const PagedPool &p, int seq, int pos) {
    if ((uint32_t)seq >= (uint32_t)p.n_seq || pos < 0 || pos >> p.lp >= p.n_table) return -1;
    const int page = p.table[(int64_t)seq * p.n_table + (pos >> p.lp)];
    if ((uint32_t)page >= (uint32_t)p.n_pages) return -1;
    return (((int64_t)page * p.HKV) << p.lp) + (pos & ((1 << p.lp) - 1));
}

// The largest |x| over groups of 8 lanes, in every lane: as bits, whose order is the numbers' with infinity and then NaN above.
template <int CTRL>
__device__ inline uint32_t max_dpp(uint32_t x) {
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xF, 0xF, false));
}
__device__ inline float amax8(const float (&x)[4]) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) m = max(m, __float_as_uint(x[k]) & 0x7fffffffu);
    m = max_dpp<0xB1>(m);                    // quad_perm [1,0,3,2]
    m = max_dpp<0x4E>(m);                    // quad_perm [2,3,0,1]
    return __uint_as_float(max_dpp<0x141>(m));  // row_half_mirror
}

// A row (one head of one token) takes HD / 4 lanes, 4 neighbouring values each; a thread takes the same head's row of TOK
// tokens, all requested before the places that they go to. Bytes bound it where there are many: 4096 tokens of 40/8 heads of
// 128 at 5.3 TB/s; a launch and three round trips where there are few (16 tokens 3.1 us).
// grid (rows of a token / those of a workgroup, tokens / TOK).
// Four tokens a thread from APPEND_MANY workgroups on (with rows that are not in a cache: 4096 tokens of 7 workgroups 40 us
// against 46, 2041 23.7 against 24.9; 2048 of 6 19.8 against 18.9, 700 of 7 10.9 against 9.6).
constexpr int APPEND_MANY = 13 * 1024;
struct AppendArgs {
    const float *qkv;  // [ntok][(H + 2 HKV) HD]
    const int32_t *seq, *pos;
    const float *bias, *q_norm, *k_norm, *rope_cs;  // the first three may be null
    float eps;
    int ntok, H, n_pos, n_rot, neox;
    float *q_out;
    PagedPool p;
};
template <int HD, bool F16, int TOK>
__global__ __launch_bounds__(256) void k_append_paged(AppendArgs a) {
    constexpr int LPR = HD / 4, RPW = 256 / LPR;
    __shared__ __align__(16) float rows[RPW][HD];
    const int row = threadIdx.x / LPR, d = 4 * (threadIdx.x % LPR);
    const int heads = a.H + 2 * a.p.HKV, hh = blockIdx.x * RPW + row, t0 = blockIdx.y * TOK;
    if (hh >= heads) return;  // (no barrier below: a row is inside one wave)
    const bool is_q = hh < a.H, is_k = !is_q && hh < a.H + a.p.HKV;
    float4 in[TOK];
#pragma unroll
    for (int i = 0; i < TOK; i++) in[i] = *(const float4 *)(a.qkv + ((int64_t)min(t0 + i, a.ntok - 1) * heads + hh) * HD + d);
    int at[TOK];
    int64_t slot0[TOK];
#pragma unroll
    for (int i = 0; i < TOK; i++) {
        const int t = min(t0 + i, a.ntok - 1);
        at[i] = a.pos[t];
        slot0[i] = paged_slot(a.p, a.seq[t], at[i]);
        if (t0 + i >= a.ntok || at[i] >= a.n_pos) slot0[i] = -1;  // left out
    }
    float4 bias = make_float4(0.f, 0.f, 0.f, 0.f), nw = bias;
    if (a.bias) bias = *(const float4 *)(a.bias + (int64_t)hh * HD + d);
    const float *norm = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
    if (norm) nw = *(const float4 *)(norm + d);
    const int half = a.n_rot / 2;
    const bool turned = (is_q || is_k) && d < a.n_rot;
    // The lane's four angles: of pairs d / 2 and d / 2 + 1, or of its own place in the lower or upper half.
    const bool low = d < half, quads = a.neox && half % 4 == 0;
    float4 cs[TOK][2];
    if (turned) {
#pragma unroll
        for (int i = 0; i < TOK; i++) {
            const float *c = a.rope_cs + (int64_t)(slot0[i] < 0 ? 0 : at[i]) * a.n_rot;  // half pairs (cos, sin)
            if (!a.neox) {
                cs[i][0] = make_float4(c[d], c[d + 1], 0.f, 0.f);
                if (d + 2 < a.n_rot) cs[i][0].z = c[d + 2], cs[i][0].w = c[d + 3];
            } else if (quads) {
                const float4 *q = (const float4 *)(c + 2 * (low ? d : d - half));
                cs[i][0] = q[0], cs[i][1] = q[1];
            } else {
                float2 x[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int e = d + k;
                    x[k] = e < a.n_rot ? *(const float2 *)(c + 2 * (e < half ? e : e - half)) : make_float2(1.f, 0.f);
                }
                cs[i][0] = make_float4(x[0].x, x[0].y, x[1].x, x[1].y), cs[i][1] = make_float4(x[2].x, x[2].y, x[3].x, x[3].y);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < TOK; i++) {
        if (slot0[i] < 0) continue;
        const int t = t0 + i;
        float4 x = in[i];
        if (a.bias) x.x += bias.x, x.y += bias.y, x.z += bias.z, x.w += bias.w;
        if (norm) {
            float ss = row_sum_dpp(x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w);
            if constexpr (HD >= 128) ss = add_xor16(ss);
            if constexpr (HD == 256) ss = add_xor32(ss);
            const float s = 1.0f / sqrtf(ss / (float)HD + a.eps);
            x.x = x.x * s * nw.x, x.y = x.y * s * nw.y, x.z = x.z * s * nw.z, x.w = x.w * s * nw.w;
        }
        if (turned) {
            if (!a.neox) {
                rope_pair(x.x, x.y, cs[i][0].x, cs[i][0].y);
                if (d + 2 < a.n_rot) rope_pair(x.z, x.w, cs[i][0].z, cs[i][0].w);
            } else {  // the other half's values through LDS
                *(float4 *)&rows[row][d] = x;
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                float v[4] = {x.x, x.y, x.z, x.w}, y[4];
                if (quads) {
                    const float4 o = *(const float4 *)&rows[row][low ? d + half : d - half];
                    y[0] = o.x, y[1] = o.y, y[2] = o.z, y[3] = o.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int e = d + k;
                        y[k] = e < a.n_rot ? rows[row][e < half ? e + half : e - half] : 0.f;
                    }
                }
                const float c[4] = {cs[i][0].x, cs[i][0].z, cs[i][1].x, cs[i][1].z};
                const float s[4] = {cs[i][0].y, cs[i][0].w, cs[i][1].y, cs[i][1].w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float lo = d + k < half ? v[k] : y[k], hi = d + k < half ? y[k] : v[k];
                    rope_pair(lo, hi, c[k], s[k]);
                    if (d + k < a.n_rot) v[k] = d + k < half ? lo : hi;
                }
                x = make_float4(v[0], v[1], v[2], v[3]);
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                __builtin_amdgcn_wave_barrier();  // (the next token's row takes this one's place)
            }
        }
        if (is_q) {
            *(float4 *)(a.q_out + ((int64_t)t * a.H + hh) * HD + d) = x;
            continue;
        }
        const int64_t slot = slot0[i] + ((int64_t)(is_k ? hh - a.H : hh - a.H - a.p.HKV) << a.p.lp);
        if constexpr (F16) {  // each value to the nearest half
            uint2 w;
            w.x = (uint32_t)f2h(x.x) | (uint32_t)f2h(x.y) << 16, w.y = (uint32_t)f2h(x.z) | (uint32_t)f2h(x.w) << 16;
            *(uint2 *)((uint16_t *)(is_k ? a.p.kv.k : a.p.kv.v) + slot * HD + d) = w;
        } else {  // per 32 values sc = f16(amax / 127), q = clamp(rint(v / sc), +-127); a NaN makes sc NaN, an infinity infinite
            const float v[4] = {x.x, x.y, x.z, x.w}, amax = amax8(v);
            const uint16_t sh = f2h(amax / 127.0f);
            const float sc = h2f(sh);
            uint32_t w = 0;
            if (sc > 0.f)
#pragma unroll
                for (int k = 0; k < 4; k++)  // (infinity / infinity is NaN: 127 with the value's sign)
                    w |= (uint32_t)((int)copysignf(fminf(127.f, rintf(fabsf(v[k]) / sc)), v[k]) & 0xff) << (8 * k);
            *(uint32_t *)((is_k ? a.p.kv.k : a.p.kv.v) + slot * HD + d) = w;
            if (d % 32 == 0) (is_k ? a.p.kv.ks : a.p.kv.vs)[slot * (HD / 32) + d / 32] = sh;
        }
    }
}

hipError_t launch_append_paged(const float *qkv, int ntok, const int32_t *seq, const int32_t *pos, int H, int HKV, int HD,
                               const float *bias, const float *q_norm, const float *k_norm, float eps,
                               const float *rope_cs, int n_pos, int n_rot, int neox, float *q_out, KvLayer kv, int kv_f16,
                               int n_pages, int page, const int32_t *table, int n_seq, int n_table, hipStream_t s) {
    AppendArgs a{};
    a.qkv = qkv, a.seq = seq, a.pos = pos, a.bias = bias, a.q_norm = q_norm, a.k_norm = k_norm, a.rope_cs = rope_cs;
    a.eps = eps, a.ntok = ntok, a.H = H, a.n_pos = n_pos, a.n_rot = n_rot, a.neox = neox, a.q_out = q_out;
    a.p = PagedPool{kv, table, n_pages, __builtin_ctz(page), n_seq, n_table, HKV};
    const int per = 1024 / HD, x = (H + 2 * HKV + per - 1) / per;
    auto go = [&](auto hd, auto f16) {
        constexpr int D = decltype(hd)::value;
        constexpr bool F = decltype(f16)::value;
        if ((int64_t)x * ntok >= APPEND_MANY) hipLaunchKernelGGL((k_append_paged<D, F, 4>), dim3(x, (ntok + 3) / 4), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_append_paged<D, F, 1>), dim3(x, ntok), dim3(256), 0, s, a);
        return hipGetLastError();
    };
    auto by_type = [&](auto hd) { return kv_f16 ? go(hd, std::true_type{}) : go(hd, std::false_type{}); };
    if (HD == 64) return by_type(std::integral_constant<int, 64>{});
    if (HD == 128) return by_type(std::integral_constant<int, 128>{});
    return by_type(std::integral_constant<int, 256>{});
}

// V values a thread of K and V each, READ_TOKENS tokens a workgroup. grid (tokens / READ_TOKENS). Bytes bound it: 48000 tokens of
// 8 KV heads of 128, q8 to f16, 62 us, 4.9 TB/s, a copy's rate.
constexpr int READ_TOKENS = 4;
template <int HD, bool F16, bool OUT16>
__global__ __launch_bounds__(256) void k_read_paged(int ntok, const int32_t *__restrict__ seq,
                                                    const int32_t *__restrict__ pos, void *__restrict__ k_out,
                                                    void *__restrict__ v_out, PagedPool p) {
    constexpr int V = OUT16 ? 8 : 4;  // 16 bytes of output
    const int width = p.HKV * HD;
    const int t0 = blockIdx.x * READ_TOKENS, per = width / V;
    int64_t slot0[READ_TOKENS];
#pragma unroll
    for (int i = 0; i < READ_TOKENS; i++) slot0[i] = t0 + i < ntok ? paged_slot(p, seq[t0 + i], pos[t0 + i]) : -1;
    for (int e = threadIdx.x; e < 2 * per; e += 256) {
        const bool v = e >= per;
        const int at = (v ? e - per : e) * V, h = at / HD, d = at % HD;
        const int8_t *src = v ? p.kv.v : p.kv.k;
        const uint16_t *scales = v ? p.kv.vs : p.kv.ks;
        uint32_t w[READ_TOKENS][F16 ? V / 2 : V / 4];
        uint16_t sc[READ_TOKENS];
#pragma unroll
        for (int i = 0; i < READ_TOKENS; i++) {
            const int64_t slot = max((int64_t)0, slot0[i]) + ((int64_t)h << p.lp);
            const uint32_t *s = (const uint32_t *)(src + (slot * HD + d) * (F16 ? 2 : 1));
#pragma unroll
            for (int k = 0; k < (F16 ? V / 2 : V / 4); k++) w[i][k] = s[k];
            if constexpr (!F16) sc[i] = scales[slot * (HD / 32) + d / 32];
        }
#pragma unroll
        for (int i = 0; i < READ_TOKENS; i++) {
            if (slot0[i] < 0) continue;  // left out
            float x[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                if constexpr (F16) x[k] = h2f(w[i][k / 2] >> (16 * (k & 1)) & 0xffff);
                else x[k] = (float)(int8_t)(w[i][k / 4] >> (8 * (k & 3))) * h2f(sc[i]);
            }
            const int64_t to = (int64_t)(t0 + i) * width + at;
            void *out = v ? v_out : k_out;
            if constexpr (OUT16) {
                uint4 o;
                uint32_t *q = (uint32_t *)&o;
#pragma unroll
                for (int k = 0; k < 4; k++) q[k] = (uint32_t)f2h(x[2 * k]) | (uint32_t)f2h(x[2 * k + 1]) << 16;
                *(uint4 *)((uint16_t *)out + to) = o;
            } else {
                *(float4 *)((float *)out + to) = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
    }
}

hipError_t launch_read_paged(int ntok, const int32_t *seq, const int32_t *pos, int HKV, int HD, KvLayer kv, int kv_f16,
                             int n_pages, int page, const int32_t *table, int n_seq, int n_table, int out16, void *k_out,
                             void *v_out, hipStream_t s) {
    const PagedPool p{kv, table, n_pages, __builtin_ctz(page), n_seq, n_table, HKV};
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((ntok + READ_TOKENS - 1) / READ_TOKENS), dim3(256), 0, s, ntok, seq, pos, k_out,
                           v_out, p);
        return hipGetLastError();
    };
    auto by_type = [&](auto hd) {
        constexpr int D = decltype(hd)::value;
        if (kv_f16) return out16 ? go(k_read_paged<D, true, true>) : go(k_read_paged<D, true, false>);
        return out16 ? go(k_read_paged<D, false, true>) : go(k_read_paged<D, false, false>);
    };
    if (HD == 64) return by_type(std::integral_constant<int, 64>{});
    if (HD == 128) return by_type(std::integral_constant<int, 128>{});
    return by_type(std::integral_constant<int, 256>{});
}

}  // namespace ts5hip
