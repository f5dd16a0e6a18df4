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

// Max over groups of 8 lanes, in every lane.
__device__ inline float max8(float v) {
    v = dpp_max<0xB1, 0xF, true>(v);     // quad_perm [1,0,3,2]
    v = dpp_max<0x4E, 0xF, true>(v);     // quad_perm [2,3,0,1]
    return dpp_max<0x141, 0xF, true>(v);  // row_half_mirror
}

// A row (one head of one token) takes HD / 4 lanes, 4 neighbouring values each. grid (rows of a token / those of a
// workgroup, tokens).
template <int HD, bool F16>
__global__ __launch_bounds__(256) void k_append_paged(const float *__restrict__ qkv, const int32_t *__restrict__ seq,
                                                      const int32_t *__restrict__ pos, int H,
                                                      const float *__restrict__ bias, const float *__restrict__ q_norm,
                                                      const float *__restrict__ k_norm, float eps,
                                                      const float *__restrict__ rope_cs, int n_pos, int n_rot, int neox,
                                                      float *__restrict__ q_out, PagedPool p) {
    constexpr int LPR = HD / 4, RPW = 256 / LPR;
    __shared__ __align__(16) float rows[RPW][HD];
    const int t = blockIdx.y, at = pos[t];
    const int64_t slot0 = paged_slot(p, seq[t], at);
    if (slot0 < 0 || at >= n_pos) return;  // left out
    const int row = threadIdx.x / LPR, d = 4 * (threadIdx.x % LPR);
    const int heads = H + 2 * p.HKV, hh = blockIdx.x * RPW + row;
    if (hh >= heads) return;  // (no barrier below: a row is inside one wave)
    const bool is_q = hh < H, is_k = !is_q && hh < H + p.HKV;
    float4 x = *(const float4 *)(qkv + ((int64_t)t * heads + hh) * HD + d);
    if (bias) {
        const float4 y = *(const float4 *)(bias + (int64_t)hh * HD + d);
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    const float *nw = is_q ? q_norm : is_k ? k_norm : nullptr;
    if (nw) {
        float ss = row_sum_dpp(x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w);
        if constexpr (HD >= 128) ss = add_xor16(ss);
        if constexpr (HD == 256) ss = add_xor32(ss);
        const float s = 1.0f / sqrtf(ss / (float)HD + eps);
        const float4 w = *(const float4 *)(nw + d);
        x.x = x.x * s * w.x, x.y = x.y * s * w.y, x.z = x.z * s * w.z, x.w = x.w * s * w.w;
    }
    if ((is_q || is_k) && d < n_rot) {
        const float *cs = rope_cs + (int64_t)at * n_rot;  // n_rot / 2 pairs (cos, sin)
        if (!neox) {
            rope_pair(x.x, x.y, cs[d], cs[d + 1]);
            if (d + 2 < n_rot) rope_pair(x.z, x.w, cs[d + 2], cs[d + 3]);
        } else {
            const int half = n_rot / 2;
            *(float4 *)&rows[row][d] = x;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = d + i;
                if (e < half) {
                    float y = rows[row][e + half];
                    rope_pair(v[i], y, cs[2 * e], cs[2 * e + 1]);
                } else if (e < n_rot) {
                    float y = rows[row][e - half];
                    rope_pair(y, v[i], cs[2 * (e - half)], cs[2 * (e - half) + 1]);
                }
            }
            x = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
    if (is_q) {
        *(float4 *)(q_out + ((int64_t)t * H + hh) * HD + d) = x;
        return;
    }
    const int kvh = is_k ? hh - H : hh - H - p.HKV;
    const int64_t slot = slot0 + ((int64_t)kvh << p.lp);
    if constexpr (F16) {  // each value to the nearest half
        uint2 w;
        w.x = (uint32_t)f2h(x.x) | (uint32_t)f2h(x.y) << 16, w.y = (uint32_t)f2h(x.z) | (uint32_t)f2h(x.w) << 16;
        *(uint2 *)((uint16_t *)(is_k ? p.kv.k : p.kv.v) + slot * HD + d) = w;
    } else {  // per 32 values sc = f16(amax / 127), q = clamp(rint(v / sc), +-127)
        const float amax = max8(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
        const uint16_t sh = f2h(amax / 127.0f);
        const float sc = h2f(sh), v[4] = {x.x, x.y, x.z, x.w};
        uint32_t w = 0;
        if (sc > 0.f)
#pragma unroll
            for (int i = 0; i < 4; i++)
                w |= (uint32_t)((int)fminf(127.f, fmaxf(-127.f, rintf(v[i] / sc))) & 0xff) << (8 * i);
        *(uint32_t *)((is_k ? p.kv.k : p.kv.v) + slot * HD + d) = w;
        if (d % 32 == 0) (is_k ? p.kv.ks : p.kv.vs)[slot * (HD / 32) + d / 32] = sh;
    }
}

hipError_t launch_append_paged(const float *qkv, int ntok, const int32_t *seq, const int32_t *pos, int H, int HKV, int HD,
                               const float *bias, const float *q_norm, const float *k_norm, float eps,
                               const float *rope_cs, int n_pos, int n_rot, int neox, float *q_out, KvLayer kv, int kv_f16,
                               int n_pages, int page, const int32_t *table, int n_seq, int n_table, hipStream_t s) {
    const PagedPool p{kv, table, n_pages, __builtin_ctz(page), n_seq, n_table, HKV};
    const int per = 1024 / HD;
    const dim3 grid((H + 2 * HKV + per - 1) / per, ntok);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, qkv, seq, pos, H, bias, q_norm, k_norm, eps, rope_cs, n_pos,
                           n_rot, neox, q_out, p);
        return hipGetLastError();
    };
    if (HD == 64) return kv_f16 ? go(k_append_paged<64, true>) : go(k_append_paged<64, false>);
    if (HD == 128) return kv_f16 ? go(k_append_paged<128, true>) : go(k_append_paged<128, false>);
    return kv_f16 ? go(k_append_paged<256, true>) : go(k_append_paged<256, false>);
}

// V values a thread of K and V each, READ_TOKENS tokens a workgroup. grid (tokens / READ_TOKENS).
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
