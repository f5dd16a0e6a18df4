// Attention of each sequence's newest tokens over a cache in pages: rows of queries on the core of attn_rows.h, the
// keys found tile by tile (16 of them, inside one page) through the sequence's table.
//
// Row (t, head) of sequence b takes keys max(0, L - window) .. L - 1, L = n_keys[b] - T + t + 1. The lengths are in
// device memory and may differ a hundredfold, so every workgroup computes the same plan from them: the shortest
// slice length L (in units of the core's keys) for which all sequences' slices together fit the launch's workgroups. A
// workgroup has one slice of one sequence and KV head and up to 16 rows; slices join through partials.
#include <algorithm>

#include "attn_rows.h"

namespace ts5hip {

struct PagedArgs {
    const float *q;        // [B][T][H * HD]
    KvLayer kv;            // [n_pages][HKV][page][HD]
    const int32_t *table;  // [B][n_table]
    int n_table, n_pages, lp;  // lp: log2 of the page
    int B, T, H, HKV, G, R, RT, window;  // R = T G rows a KV head in tiles of RT (16, or fewer in all)
    int cap;                // slices of all sequences, at most
    uint64_t g_m, hkv_m;    // rows_magic of G, HKV
    const int32_t *n_keys;  // [B]
    float scale;
    float *part;   // [HKV][row tile][cap][RT][HD + 4]: m, l, -, -, O
    int2 *plan;    // [B] each sequence's first slice and how many it has
    int *counters; // [B * HKV * row tiles], CTR_STRIDE ints apart, zero between launches
    float *out;    // [B][T][H * HD]
};

// A sequence's keys: [first, end) are some row's, counted from `first` (a multiple of 16).
struct PagedSpan {
    int first, end;
};
__device__ inline PagedSpan paged_span(const PagedArgs &a, int n) {
    PagedSpan s;
    s.end = max(0, min(n, a.n_table << a.lp));
    s.first = a.window ? max(0, s.end - a.T + 1 - a.window) & ~15 : 0;
    return s;
}
__device__ inline int paged_units(const PagedSpan &s, int unit) { return (s.end - s.first + unit - 1) / unit; }

// Inclusive sums over the wave's lanes.
__device__ inline int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);   // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);   // row_shr:2
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xE, true);   // row_shr:4
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xC, true);   // row_shr:8
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return x;
}
__device__ inline int wave_total(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// Slices of u units, `per` each; a sequence without a key has one, which writes its zeros.
__device__ inline int paged_slices(int u, int per) { return max(1, (u + per - 1) / per); }

// Slice j's sequence, its place among that sequence's slices, how many those are, and the units a slice has. b < 0:
// there is no such slice. Every lane of a wave calls it with the same j. Slices are whole rounds of NW waves.
struct PagedSlice {
    int b, at, used, per;
};
template <int UNIT, int NW, int LEAST>
__device__ inline PagedSlice paged_slice(const PagedArgs &a, int j) {
    const int lane = threadIdx.x & 63;
    auto units = [&](int b) { return b < a.B ? paged_units(paged_span(a, a.n_keys[b]), UNIT) : 0; };
    PagedSlice s;
    int sum = 0, u0 = units(lane);
    for (int b = 0; b < a.B; b += 64) sum += wave_total(b ? units(b + lane) : u0);
    // ceil(u / per) <= u / per + 1 summed over the sequences: this many units a slice always fit.
    auto whole = [](int per) { return max(LEAST, (per + NW - 1) / NW * NW); };
    s.per = whole((sum + a.cap - a.B - 1) / max(1, a.cap - a.B));
    if (a.B <= 64) {  // the fewest that fit
        int lo = whole((sum + a.cap - 1) / a.cap), hi = s.per;
        while (lo < hi) {  // (both whole rounds, and so is their middle)
            const int mid = (lo + hi) / 2 / NW * NW;
            if (wave_total(lane < a.B ? paged_slices(u0, mid) : 0) <= a.cap) hi = mid;
            else lo = mid + NW;
        }
        s.per = hi;
    }
    s.b = -1, s.at = 0, s.used = 0;
    int before = 0;
    for (int b = 0; b < a.B; b += 64) {
        const int mine = b + lane < a.B ? paged_slices(b ? units(b + lane) : u0, s.per) : 0, incl = before + wave_scan(mine);
        const uint64_t past = __builtin_amdgcn_ballot_w64(incl > j);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            s.b = b + l, s.used = __builtin_amdgcn_readlane(mine, l);
            s.at = j - (__builtin_amdgcn_readlane(incl, l) - s.used);
            break;
        }
        before = __builtin_amdgcn_readlane(incl, 63);
    }
    return s;
}

// A tile's 16 keys from `key` on, those below `end`, as bounded buffers: what is past them reads zeros. No page: all of it.
template <int HD, bool F16>
__device__ inline RowsKv paged_tile(const PagedArgs &a, int kvh, int page, int key, int end) {
    const bool ok = (uint32_t)page < (uint32_t)a.n_pages;
    const int n = ok ? max(0, min(end - key, 16)) : 0;
    const int64_t slot = (((int64_t)(ok ? page : 0) * a.HKV + kvh) << a.lp) + (key & ((1 << a.lp) - 1));
    return rows_kv<HD, F16>(a.kv, slot, n);
}
template <int HD, bool F16, int KT>
__device__ inline void paged_load(RowsUnit<HD, F16, KT> &u, int t, const RowsKv &kv, int rl, int kq) {
    using S = RowsShape<HD, F16, KT>;
#pragma unroll
    for (int c = 0; c < S::NC; c++) rows_words<S::KW>(kv.k, ((uint32_t)rl * HD + 32 * c + 8 * kq) * S::VB, u.k[t][c]);
    if constexpr (!F16) rows_words<2 * S::NC>(kv.ks, (uint32_t)(4 * kq) * S::NC * 2, u.ks[t]);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t key = (uint32_t)(4 * kq + i);
        rows_words<S::VW>(kv.v, (key * HD + S::NDT * rl) * S::VB, u.v[t][i]);
        if constexpr (!F16)
            u.vs[t][i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(kv.vs, key * S::NC * 2 + rl * S::NDT / 32 * 2, 0, 0);
    }
}

// Infinite and NaN values of a unit (as the products see them: fp16's range) replaced by zeros: the product with a row
// that does not take their key would be NaN. Whether the wave had any.
template <int HD, bool F16, int KT>
__device__ inline bool paged_clean(RowsUnit<HD, F16, KT> &u) {
    using S = RowsShape<HD, F16, KT>;
    uint32_t any = 0;
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const _Float16 sc = __builtin_bit_cast(_Float16, F16 ? (uint16_t)0 : u.vs[t][i]);
#pragma unroll
            for (int w = 0; w < S::VW; w++) {
                uint32_t x = u.v[t][i][w], out = 0;
                if constexpr (F16) {
                    out = ((x & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((x & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const _Float16 h = (_Float16)(float)(int8_t)(x >> (8 * k)) * sc;
                        out |= (__builtin_bit_cast(uint16_t, h) & 0x7c00) == 0x7c00 ? 0xffu << (8 * k) : 0u;
                    }
                }
                any |= out, u.v[t][i][w] = x & ~out;
            }
            if constexpr (!F16) u.vs[t][i] = (u.vs[t][i] & 0x7c00) == 0x7c00 ? 0 : u.vs[t][i];
        }
    return __builtin_amdgcn_ballot_w64(any != 0) != 0;
}

// A row's output.
template <int HD>
__device__ inline float *paged_out(const PagedArgs &a, int b, int kvh, int r) {
    const int t = rows_div(r, a.g_m);
    return a.out + (((int64_t)b * a.T + t) * a.H + kvh * a.G + r - t * a.G) * HD;
}

// grid (cap * HKV, row tiles): one slice of one sequence's keys for up to 16 rows of a KV head; the waves take its units
// in turn, each one's next requested before this one is used. With FUSED the last of a sequence's slices joins them.
template <int HD, bool F16, int KT, int NW, int LEAST, bool FUSED>
__global__ __launch_bounds__(64 * NW, HD <= 128 ? 2 : 1) void k_attn_paged(PagedArgs a) {
    using S = RowsShape<HD, F16, KT>;
    __shared__ RowsLds<HD, NW> L;
    __shared__ int nonfinite;  // a unit that not every row takes whole had infinite or NaN values: they are added at the end
    if (threadIdx.x == 0) nonfinite = 0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rl = lane & 15, kq = lane >> 4;
    const int j = rows_div(blockIdx.x, a.hkv_m), kvh = (int)blockIdx.x - j * a.HKV;
    const PagedSlice sl = paged_slice<S::UNIT, NW, LEAST>(a, j);
    if (sl.b < 0) return;
    const int b = sl.b, r0 = blockIdx.y * 16, rows = min(a.R - r0, 16);
    RowsIn<HD, 1> in;
    rows_request<HD, 1>(in, kq, [&](int, bool &ok) {
        const int r = r0 + min(rl, rows - 1), t = rows_div(r, a.g_m);
        ok = rl < rows;
        return a.q + (((int64_t)b * a.T + t) * a.H + kvh * a.G + r - t * a.G) * HD;
    });
    const PagedSpan sp = paged_span(a, a.n_keys[b]);
    const int units = paged_units(sp, S::UNIT), u0 = sl.at * sl.per, u1 = min(units, u0 + sl.per);
    if (!FUSED && kvh == 0 && blockIdx.y == 0 && sl.at == 0 && threadIdx.x == 0) a.plan[b] = make_int2(j, sl.used);

    // Pages of the wave's next 64 units, one a lane.
    const int32_t *table = a.table + (int64_t)b * a.n_table;
    int pages[KT];
    auto look = [&](int u) {
#pragma unroll
        for (int t = 0; t < KT; t++) {
            const int i = (sp.first + (u + lane * NW) * S::UNIT + 16 * t) >> a.lp;
            pages[t] = i < a.n_table ? table[i] : -1;
        }
    };
    RowsUnit<HD, F16, KT> nxt;
    int kb[KT], kn[KT];
    auto request = [&](int u, int i) {  // unit u, the wave's i-th
#pragma unroll
        for (int t = 0; t < KT; t++) {
            const int key = sp.first + u * S::UNIT + 16 * t, page = __builtin_amdgcn_readlane(pages[t], i & 63);
            const bool ok = u < u1 && (uint32_t)page < (uint32_t)a.n_pages;
            paged_load<HD, F16, KT>(nxt, t, paged_tile<HD, F16>(a, kvh, ok ? page : -1, key, sp.end), rl, kq);
            kn[t] = ok ? key : 0x7fffff00;  // (no page: no row takes its keys)
        }
    };
    look(u0 + wave);
    request(u0 + wave, 0);

    RowsQ<HD, 1> q;
    rows_query<HD, 1, true>(q, in, a.scale);
    // The lane's row takes keys [from, to); every row of the tile those of [all0, all1).
    const int t0 = rows_div(r0, a.g_m), t1 = rows_div(r0 + rows - 1, a.g_m), t = rows_div(r0 + min(rl, rows - 1), a.g_m);
    auto last = [&](int tt) { return sp.end - a.T + tt + 1; };
    const int to = rl < rows ? last(t) : 0, from = a.window ? max(0, last(t) - a.window) : 0;
    const int all1 = last(t0), all0 = a.window ? max(0, last(t1) - a.window) : 0;
    auto clean = [&](int key) { return key >= all0 && key + S::UNIT <= all1; };
    RowsSum<HD, 1> sum;
    rows_clear<HD, 1>(sum);
    __syncthreads();  // the flag is set
    for (int u = u0 + wave, i = 1; u < u1; u += NW, i++) {
        RowsUnit<HD, F16, KT> cur = nxt;
        bool whole = clean(sp.first + u * S::UNIT);
#pragma unroll
        for (int t = 0; t < KT; t++) kb[t] = kn[t], whole &= kn[t] != 0x7fffff00;
        if ((i & 63) == 0) look(u + NW);
        request(u + NW, i);
        if (!whole && paged_clean<HD, F16, KT>(cur)) nonfinite = 1;
        rows_unit<HD, F16, KT, true, false>(
            cur, q, sum, kb, kq, [&](int key) { return rows_below(key, to) & ~rows_below(key, from); },
            [](int, const float (&)[4]) {});
    }
    // The infinite and NaN values that were left out, of the keys that row r takes.
    auto add_nonfinite = [&](int r, int d, float4 &o) {
        const int end = last(rows_div(r0 + r, a.g_m)), begin = a.window ? max(0, end - a.window) : 0;
        for (int u = u0; u < u1; u++) {
            bool whole = clean(sp.first + u * S::UNIT);
            for (int key = sp.first + u * S::UNIT; key < sp.first + (u + 1) * S::UNIT; key++) {
                const int i = key >> a.lp, page = i < a.n_table ? table[i] : -1;
                if ((uint32_t)page >= (uint32_t)a.n_pages) whole = false;
            }
            if (whole) continue;
            for (int key = max(begin, sp.first + u * S::UNIT); key < min(end, sp.first + (u + 1) * S::UNIT); key++) {
                const int page = table[key >> a.lp];
                if ((uint32_t)page >= (uint32_t)a.n_pages) continue;
                const int64_t slot = (((int64_t)page * a.HKV + kvh) << a.lp) + (key & ((1 << a.lp) - 1));
                o.x += rows_nonfinite<HD, F16>(a.kv, slot, d), o.y += rows_nonfinite<HD, F16>(a.kv, slot, d + 1);
                o.z += rows_nonfinite<HD, F16>(a.kv, slot, d + 2), o.w += rows_nonfinite<HD, F16>(a.kv, slot, d + 3);
            }
        }
    };
    // For the last workgroup, which may run on another XCD, the partials go past this one's L2, and only when they
    // are out does the workgroup count itself in.
    float *parts = a.part + ((int64_t)(kvh * gridDim.y + blockIdx.y) * a.cap + j - sl.at) * a.RT * (HD + 4);  // the sequence's
    const uint32_t stride = (uint32_t)a.RT * (HD + 4) * 4;  // bytes from a slice to the next
    const __amdgpu_buffer_rsrc_t part = slice_rsrc(parts, (uint32_t)sl.used * stride);
    rows_combine<HD, NW>(L, sum, rows, wave, rl, kq, [&](int r, int d, float4 o, float m, float l) {
        if (nonfinite) add_nonfinite(r, d, o);
        if (sl.used == 1) {
            *(float4 *)(paged_out<HD>(a, b, kvh, r0 + r) + d) = rows_over(o, l);
            return;
        }
        const uint32_t at = (uint32_t)sl.at * stride + (uint32_t)r * (HD + 4) * 4;
        constexpr int POLICY = FUSED ? BUF_SC1 : 0;
        if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, make_float2(m, l)), part, at, 0, POLICY);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), part, at + 16 + 4 * d, 0, POLICY);
    });
    if (!FUSED || sl.used == 1) return;
    __shared__ RowsJoin J;
    __shared__ int is_last;
    wait_stores();
    __syncthreads();
    if (threadIdx.x == 0) {
        int *c = a.counters + ((b * a.HKV + kvh) * gridDim.y + blockIdx.y) * CTR_STRIDE;
        is_last = atomicAdd(c, 1) == sl.used - 1;
        if (is_last) st_dev(c, 0);
    }
    __syncthreads();
    if (!is_last) return;
    constexpr int TPR = HD / 4 * JOIN_SG;
    static_assert(64 * NW == 256, "rows_join's threads");
    for (int g0 = 0; g0 < rows; g0 += 256 / TPR) {
        const int g = g0 + (int)threadIdx.x / TPR;
        float M, l;
        const float4 o = rows_join<HD, JOIN_SG>(J, sl.used, M, l, [&](int s, int d, float2 &ml, float4 &x) {
            const uint32_t at = (uint32_t)s * stride + (uint32_t)min(g, rows - 1) * (HD + 4) * 4;
            ml = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(part, at, 0, BUF_SC1));
            x = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(part, at + 16 + 4 * d, 0, BUF_SC1));
        });
        if (g < rows && threadIdx.x % TPR < HD / 4)
            *(float4 *)(paged_out<HD>(a, b, kvh, r0 + g) + 4 * (threadIdx.x % TPR)) = rows_over(o, l);
    }
}

// The slices' join where few sequences have many: 256 / (HD / 4 x SG) rows a workgroup.
template <int HD>
__global__ __launch_bounds__(256) void k_paged_merge(PagedArgs a, int64_t rows) {
    constexpr int TPR = HD / 4 * JOIN_SG;
    __shared__ RowsJoin J;
    const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR, at = min(row, rows - 1);
    const int b = (int)(at / ((int64_t)a.HKV * a.R)), kvh = (int)(at / a.R % a.HKV), r = (int)(at % a.R);
    const int2 plan = a.plan[b];
    const int tiles = (a.R + 15) / 16;
    float M, l;
    const float4 o = rows_join<HD, JOIN_SG>(J, plan.y == 1 ? 0 : plan.y, M, l, [&](int s, int d, float2 &ml, float4 &x) {
        const float *p = a.part + (((int64_t)(kvh * tiles + r / 16) * a.cap + plan.x + s) * a.RT + r % 16) * (HD + 4);
        ml = *(const float2 *)p, x = *(const float4 *)(p + 4 + d);
    });
    if (plan.y == 1 || row >= rows || threadIdx.x % TPR >= HD / 4) return;
    *(float4 *)(paged_out<HD>(a, b, kvh, r) + 4 * (threadIdx.x % TPR)) = rows_over(o, l);
}

// ---- host ----------------------------------------------------------------------------------------

struct PagedPlan {
    int cap, tiles;
    bool fused;
    size_t part, plan;
};
static PagedPlan paged_plan(int B, int T, int H, int HKV, int HD, int n_cu) {
    PagedPlan p;
    const int R = T * (H / HKV);
    p.tiles = (R + 15) / 16;
    p.cap = std::max(2 * B, 3 * n_cu / std::max(1, HKV * p.tiles));
    p.fused = (int64_t)B * HKV * p.tiles <= 4096;
    p.part = align_up((size_t)p.cap * HKV * p.tiles * std::min(R, 16) * (HD + 4) * sizeof(float), 256);
    p.plan = (size_t)B * sizeof(int2);
    return p;
}
size_t attn_paged_scratch_bytes(int B, int T, int H, int HKV, int HD, int n_cu) {
    const PagedPlan p = paged_plan(B, T, H, HKV, HD, n_cu);
    return p.part + p.plan;
}
hipError_t launch_attn_paged(const float *q, int B, int T, int H, int HKV, int HD, KvLayer kv, int kv_f16, int n_pages,
                             int page, const int32_t *table, int n_table, const int32_t *n_keys, int window, float scale,
                             void *scratch, int *counters, float *out, int n_cu, hipStream_t s) {
    const PagedPlan p = paged_plan(B, T, H, HKV, HD, n_cu);
    PagedArgs a{};
    a.q = q, a.kv = kv, a.table = table, a.n_table = n_table, a.n_pages = n_pages, a.lp = __builtin_ctz(page);
    a.B = B, a.T = T, a.H = H, a.HKV = HKV, a.G = H / HKV, a.R = T * a.G, a.RT = std::min(a.R, 16), a.window = std::min(window, 1 << 30), a.cap = p.cap;
    a.g_m = rows_magic(a.G), a.hkv_m = rows_magic(HKV), a.n_keys = n_keys, a.scale = scale;
    a.part = (float *)scratch, a.plan = (int2 *)((uint8_t *)scratch + p.part), a.counters = counters, a.out = out;
    return rows_by_shape(HD, kv_f16, [&](auto hd, auto f16) {
        constexpr int D = decltype(hd)::value, KT = D == 64 ? 2 : 1, NW = 4, LEAST = 8 / KT;
        constexpr bool F = decltype(f16)::value;
        const dim3 grid(p.cap * HKV, p.tiles);
        if (p.fused) {
            hipLaunchKernelGGL((k_attn_paged<D, F, KT, NW, LEAST, true>), grid, dim3(64 * NW), 0, s, a);
            return hipGetLastError();
        }
        hipLaunchKernelGGL((k_attn_paged<D, F, KT, NW, LEAST, false>), grid, dim3(64 * NW), 0, s, a);
        const int64_t rows = (int64_t)B * HKV * a.R;
        constexpr int RPW = 256 / (D / 4 * JOIN_SG);
        hipLaunchKernelGGL(k_paged_merge<D>, dim3((unsigned)((rows + RPW - 1) / RPW)), dim3(256), 0, s, a, rows);
        return hipGetLastError();
    });
}

}  // namespace ts5hip
