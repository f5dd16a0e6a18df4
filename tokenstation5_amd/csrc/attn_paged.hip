// Attention of each sequence's newest tokens over a cache in pages: rows of queries on the core of attn_rows.h, the
// keys found tile by tile (16 of them, inside one page) through the sequence's table.
//
// Row (t, head) of sequence b takes keys max(0, L - window) .. L - 1, L = n_keys[b] - T + t + 1. The lengths are in
// device memory and may differ a hundredfold, so every workgroup computes the same plan from them: a slice length (in
// units of the core's keys) with which all sequences' slices together fit the launch's workgroups, up to 64 sequences (a
// lane each) the shortest such, past that one that always fits. A workgroup has one slice of one sequence and KV head and up
// to 32 rows; slices join through partials.
//
// What bounds it: f16 caches memory (16 sequences of 16384 keys, 32/8 heads of 128: 188 us, 5.7 TB/s). q8 caches no unit alone:
// the vector ALU, which turns int8 into fp16 planes, is busy for 51 % of the cycles and the matrix cores for 27 %, and the two
// waves a SIMD wait for data for 28 % of theirs (the same sequences 117 us, 4.9 TB/s; a contiguous cache 127). Several tokens
// the same: 58 %, 27 %, 31 % (8 sequences of 8192, 6 tokens, 40/8 heads 38.9 us and the join's 5.4; the bytes alone 29). Few or
// short sequences a chain of latencies, 4.1 us and the join's 2.1 for one key: the lengths, the plan, the table, the keys, the
// partials, the join.
//
// A wave has one unit in registers and requests the next one's keys once it has used this one's, and its values once it is
// done: with two or three units ahead nothing was faster (T = 1) and some 10 % slower.
#include <algorithm>

#include "attn_rows.h"

namespace ts5hip {

struct PagedArgs {
    const float *q;        // [B][T][H * HD]
    KvLayer kv;            // [n_pages][HKV][page][HD]
    const int32_t *table;  // [B][n_table]
    int n_table, n_pages, lp;  // lp: log2 of the page
    int B, T, H, HKV, G, R, RT, window;  // R = T G rows a KV head, in blocks of RT
    int cap;                // slices of all sequences, at most
    uint64_t g_m, hkv_m;    // rows_magic of G, HKV
    const int32_t *n_keys;  // [B]
    float scale;
    float *part;   // [HKV][row block][cap][RT][HD + 4]: m, l, -, -, O
    int2 *plan;    // [B] each sequence's first slice and how many it has
    int *counters; // [B * HKV * row blocks], CTR_STRIDE ints apart, zero between launches
    float *out;    // [B][T][H * HD]
};

// A sequence's keys: [first, end) are some row's, counted from `first` (a multiple of 32: whole units).
struct PagedSpan {
    int first, end;
};
__device__ inline PagedSpan paged_span(const PagedArgs &a, int n) {
    PagedSpan s;
    s.end = max(0, min(n, a.n_table << a.lp));
    s.first = a.window ? max(0, s.end - a.T + 1 - a.window) & ~31 : 0;
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

// Slice j's sequence, that one's count of keys, the slice's place among its slices, how many those are, and the units a
// slice has. b < 0: there is no such slice. Every lane of a wave calls it with the same j. Slices are whole rounds of NW waves.
struct PagedSlice {
    int b, n, at, used, per;
};
template <int UNIT, int NW, int LEAST>
__device__ inline PagedSlice paged_slice(const PagedArgs &a, int j) {
    const int lane = threadIdx.x & 63;
    auto count = [&](int b) { return b < a.B ? a.n_keys[b] : 0; };
    auto units = [&](int n) { return paged_units(paged_span(a, n), UNIT); };
    PagedSlice s;
    const int n0 = count(lane), u0 = units(n0);
    int sum = 0;
    for (int b = 0; b < a.B; b += 64) sum += wave_total(b ? units(count(b + lane)) : u0);
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
    s.b = -1, s.n = 0, s.at = 0, s.used = 0;
    int before = 0;
    for (int b = 0; b < a.B; b += 64) {
        const int n = b ? count(b + lane) : n0;
        const int mine = b + lane < a.B ? paged_slices(b ? units(n) : u0, s.per) : 0, incl = before + wave_scan(mine);
        const uint64_t past = __builtin_amdgcn_ballot_w64(incl > j);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            s.b = b + l, s.n = __builtin_amdgcn_readlane(n, l), s.used = __builtin_amdgcn_readlane(mine, l);
            s.at = j - (__builtin_amdgcn_readlane(incl, l) - s.used);
            break;
        }
        before = __builtin_amdgcn_readlane(incl, 63);
    }
    return s;
}

// A sequence's row of the table, which nothing writes while the kernel runs.
typedef const __attribute__((address_space(4))) int32_t *PagedTable;

// The page that a unit is in, as bounded buffers: what is past the sequence's keys reads zeros, and without a page
// all of it. `id` is the next page's, on its way.
template <int HD, bool F16>
struct PagedPage {
    RowsKv kv;
    int at, id;
    bool has;
    // The page of index `to` comes next. (A scalar load: as a vector load its value, wanted as a scalar, was waited for at
    // once, and with it every key and value on their way.)
    __device__ void look(const PagedArgs &a, PagedTable table, int to) { id = table[min(to, a.n_table - 1)]; }
    __device__ void turn(const PagedArgs &a, int kvh, int end, int to) {
        at = to, has = to < a.n_table && (uint32_t)id < (uint32_t)a.n_pages;
        // A wave also looks at the page past the sequence's last key, and the table may have one there: without max the count is
        // negative, and as a buffer's size it lets loads (the slot past all pages among them) run on for 4 GiB.
        // (readfirstlane: the compiler takes min and max as one vector instruction, and then each load as a loop over lanes
        // that might have buffers of their own)
        const int n = __builtin_amdgcn_readfirstlane(max(0, min(end - (to << a.lp), 1 << a.lp)));
        kv = rows_kv<HD, F16>(a.kv, ((int64_t)(has ? id : 0) * a.HKV + kvh) << a.lp, has ? n : 0);
    }
};
// The lane's byte offsets in a unit's keys, values and their scales.
template <int HD, bool F16, int KT>
struct PagedLane {
    using S = RowsShape<HD, F16, KT>;
    uint32_t k, v, ks, vs;
    __device__ PagedLane(int rl, int kq) {
        k = (rl * HD + 8 * kq) * S::VB, v = (4 * kq * HD + S::NDT * rl) * S::VB;
        ks = 4 * kq * (S::NC * 2), vs = ks + rl * S::NDT / 32 * 2;
    }
    // `x` as a sum of its own: the loads' distances from it are the instructions' then, where the compiler, which sees
    // disjoint bits, takes an instruction and a register for each.
    __device__ static uint32_t at(uint32_t lane, uint32_t x) {
        x += lane;
        asm("" : "+v"(x));
        return x;
    }
};
// A unit's keys and values, `slot` keys into its page (or past all pages: zeros).
template <int HD, bool F16, int KT>
__device__ inline void paged_load_k(RowsUnit<HD, F16, KT> &u, const RowsKv &kv, uint32_t slot, const PagedLane<HD, F16, KT> &l) {
    using S = RowsShape<HD, F16, KT>;
    const uint32_t k0 = l.at(l.k, slot * (HD * S::VB)), s0 = l.at(l.ks, slot * (S::NC * 2));
#pragma unroll
    for (int t = 0; t < KT; t++) {
#pragma unroll
        for (int c = 0; c < S::NC; c++) rows_words<S::KW>(kv.k, k0 + (16 * t * HD + 32 * c) * S::VB, u.k[t][c]);
        if constexpr (!F16) rows_words<2 * S::NC>(kv.ks, s0 + 16 * t * (S::NC * 2), u.ks[t]);
    }
}
template <int HD, bool F16, int KT>
__device__ inline void paged_load_v(RowsUnit<HD, F16, KT> &u, const RowsKv &kv, uint32_t slot, const PagedLane<HD, F16, KT> &l) {
    using S = RowsShape<HD, F16, KT>;
    const uint32_t v0 = l.at(l.v, slot * (HD * S::VB)), s0 = l.at(l.vs, slot * (S::NC * 2));
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            rows_words<S::VW>(kv.v, v0 + (16 * t + i) * HD * S::VB, u.v[t][i]);
            if constexpr (!F16)
                u.vs[t][i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(kv.vs, s0 + (16 * t + i) * (S::NC * 2), 0, 0);
        }
}

// A value's scale where it is used. (Opaque to the compiler, which otherwise packs two scales into a register where they are
// loaded, and so waits at the loop's end for the unit that it has just requested.)
__device__ inline uint32_t paged_scale(uint16_t s) {
    uint32_t x = s;
    asm("" : "+v"(x));
    return x;
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
            const uint16_t scale = F16 ? 0 : (uint16_t)paged_scale(u.vs[t][i]);
            const _Float16 sc = __builtin_bit_cast(_Float16, scale);
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
            if constexpr (!F16) u.vs[t][i] = (scale & 0x7c00) == 0x7c00 ? 0 : scale;
        }
    return __builtin_amdgcn_ballot_w64(any != 0) != 0;
}

// rows_value_tile with q8's pairs of keys from two dims a permutation: 6 instructions for 4 dims of both, not 8.
template <int HD, bool F16, int KT>
__device__ inline void paged_value_tile(const RowsUnit<HD, F16, KT> &u, const RowsScale<HD, F16, KT> &sc, int dt,
                                        uint32_t (&hi)[2 * KT], uint32_t (&lo)[2 * KT]) {
    if constexpr (F16) {
        rows_value_tile<HD, F16, KT>(u, sc, dt, hi, lo);
    } else {
        const ar_h2 k1152 = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const uint32_t both = __builtin_amdgcn_perm(u.v[t][2 * p + 1][dt / 4], u.v[t][2 * p][dt / 4],
                                                            dt & 2 ? 0x07030602u : 0x05010400u) ^ 0x80808080u;
                const uint32_t b = __builtin_amdgcn_perm(0x64646464u, both, dt & 1 ? 0x04030402u : 0x04010400u);
                const ar_h2 v = __builtin_bit_cast(ar_h2, b) - k1152, h = v * sc.s[t][p];
                hi[2 * t + p] = __builtin_bit_cast(uint32_t, h);
                lo[2 * t + p] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(v, sc.s[t][p], -h));
            }
    }
}

// One unit into the sums of NT row tiles, its keys and values converted once. Without `whole`, seen(qt, key) has a bit for each of
// keys key .. + 3 that the lane's row of tile qt takes. keys_done() comes where the unit's keys are used up.
// high(qt, c) and low(qt, c) are the planes of chunk c of row tile qt.
template <int HD, bool F16, int KT, int NT, class High, class Low, class Seen, class Done>
__device__ inline void paged_unit(const RowsUnit<HD, F16, KT> &u, const float (&p2e)[NT], High high, Low low,
                                  RowsSum<HD, NT> &a, const int (&kb)[KT], int kq, bool whole, Seen seen, Done keys_done) {
    using S = RowsShape<HD, F16, KT>;
    using Op = RowsOp<KT>;
    float s[NT][KT][4];
#pragma unroll
    for (int t = 0; t < KT; t++) {
        ar_f4 R[NT];
#pragma unroll
        for (int c = 0; c < S::NC; c++) {
            const ar_h8 ka = rows_values<S::KW>(u.k[t][c]);
            float ks[4];
            if constexpr (!F16)
#pragma unroll
                for (int i = 0; i < 4; i++) ks[i] = h2f((u.ks[t][(i * S::NC + c) / 2] >> (16 * (c & 1))) & 0xffff);
#pragma unroll
            for (int qt = 0; qt < NT; qt++) {
                if (!F16 || c == 0) R[qt] = ar_f4{0.f, 0.f, 0.f, 0.f};
                R[qt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, high(qt, c), R[qt], 0, 0, 0);
            }
#pragma unroll
            for (int qt = 0; qt < NT; qt++) R[qt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, low(qt, c), R[qt], 0, 0, 0);
            if constexpr (!F16)
#pragma unroll
                for (int qt = 0; qt < NT; qt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[qt][t][i] = c == 0 ? ks[i] * R[qt][i] : fmaf(ks[i], R[qt][i], s[qt][t][i]);
        }
        if constexpr (F16)
#pragma unroll
            for (int qt = 0; qt < NT; qt++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[qt][t][i] = R[qt][i];
    }
    keys_done();
    typename Op::T ph[NT], pl[NT];
#pragma unroll
    for (int qt = 0; qt < NT; qt++) {
        if (!whole) {
#pragma unroll
            for (int t = 0; t < KT; t++) {
                const uint32_t take = seen(qt, kb[t] + 4 * kq);
#pragma unroll
                for (int i = 0; i < 4; i++) s[qt][t][i] = take & 1u << i ? s[qt][t][i] : -INFINITY;
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[qt][t][i]);
        const float m0 = rows_reference(a, qt, max_xor32(max_xor16(mx)) * p2e[qt]);
        float sum = 0.f;
        uint32_t hi[2 * KT], lo[2 * KT];
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[qt][t][2 * i], p2e[qt], -m0));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(s[qt][t][2 * i + 1], p2e[qt], -m0));
                sum += p0 + p1;
                rows_split(p0, p1, hi[2 * t + i], lo[2 * t + i]);
            }
        a.l[qt] += sum;  // (the lane's share: its four keys of each tile)
        ph[qt] = Op::of(hi), pl[qt] = Op::of(lo);
    }
    RowsScale<HD, F16, KT> sc;
    if constexpr (!F16) {
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int p = 0; p < 2; p++)
                sc.s[t][p] = __builtin_bit_cast(ar_h2, paged_scale(u.vs[t][2 * p]) | paged_scale(u.vs[t][2 * p + 1]) << 16);
    }
#pragma unroll
    for (int dt = 0; dt < S::NDT; dt++) {
        uint32_t hi[2 * KT], lo[2 * KT];
        paged_value_tile<HD, F16, KT>(u, sc, dt, hi, lo);
        const typename Op::T vh = Op::of(hi), vl = Op::of(lo);
#pragma unroll
        for (int qt = 0; qt < NT; qt++) a.o[qt][dt] = Op::mfma(vh, ph[qt], a.o[qt][dt]);
        if constexpr (!F16)
#pragma unroll
            for (int qt = 0; qt < NT; qt++) a.o[qt][dt] = Op::mfma(vl, ph[qt], a.o[qt][dt]);
#pragma unroll
        for (int qt = 0; qt < NT; qt++) a.o[qt][dt] = Op::mfma(vh, pl[qt], a.o[qt][dt]);
    }
}

// A row's output.
template <int HD>
__device__ inline float *paged_out(const PagedArgs &a, int b, int kvh, int r) {
    const int t = rows_div(r, a.g_m);
    return a.out + (((int64_t)b * a.T + t) * a.H + kvh * a.G + r - t * a.G) * HD;
}

// What a kernel is made for: KT tiles of keys a unit (which does not end past a page), NT row tiles a wave, NW waves, EDGE:
// rows that do not take the same keys (several tokens, a window), FUSED: the last of a sequence's slices joins them.
template <int HD_, bool F16_, int KT_, int NT_, int NW_, bool EDGE_, bool FUSED_>
struct PagedForm {
    static constexpr int HD = HD_, KT = KT_, NT = NT_, NW = NW_, UNIT = 16 * KT, LEAST = 8 / KT < NW ? NW : 8 / KT;
    static constexpr bool F16 = F16_, EDGE = EDGE_, FUSED = FUSED_;
};

// RowsJoin of other workgroups.
template <int THREADS>
struct PagedJoin {
    __align__(16) float4 o[THREADS];
    float2 ml[THREADS];
};

// grid (cap * HKV, row blocks): one slice of one sequence's keys for up to 16 NT rows of a KV head; the waves take its units
// in turn.
template <class P>
__global__ __launch_bounds__(64 * P::NW, P::HD <= 128 ? 2 : 1) void k_attn_paged(PagedArgs a) {
    constexpr int HD = P::HD, NT = P::NT, KT = P::KT, NW = P::NW, UNIT = P::UNIT;
    constexpr bool F16 = P::F16, EDGE = P::EDGE, FUSED = P::FUSED;
    // LOW: the rows' planes go through LDS, where the low ones stay. HIGH: the high ones' chunks in registers: as many as do
    // not spill.
    constexpr bool LOW = NT > 1;
    constexpr int HIGH = LOW && !F16 && HD == 128 && KT == 2 ? 3 : HD / 32;
    __shared__ union {
        struct {
            uint4 high[LOW ? NT : 1][HD / 32][64], low[LOW ? NT : 1][HD / 32][64];
            float p2e[LOW ? NT : 1][16];
        } q;
        RowsLds<HD, NW> parts;
        PagedJoin<64 * NW> join;
    } L;
    __shared__ int nonfinite;  // a unit that not every row takes whole had infinite or NaN values: they are added at the end
    if (EDGE && threadIdx.x == 0) nonfinite = 0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rl = lane & 15, kq = lane >> 4;
    const int j = rows_div(blockIdx.x, a.hkv_m), kvh = (int)blockIdx.x - j * a.HKV;
    const PagedSlice sl = paged_slice<UNIT, NW, P::LEAST>(a, j);
    if (sl.b < 0) return;
    const int b = sl.b, r0 = blockIdx.y * a.RT, rows = min(a.R - r0, a.RT);
    constexpr int NQ = LOW ? 1 : NT;  // row tiles that a wave converts (LOW: wave w the w-th)
    RowsIn<HD, NQ> in;
    const int tile0 = LOW ? wave : 0;
    auto request_q = [&] {
        rows_request<HD, NQ>(in, kq, [&](int qt, bool &ok) {
            const int at = 16 * (tile0 + qt) + rl, r = r0 + min(at, rows - 1), t = rows_div(r, a.g_m);
            ok = at < rows;
            return a.q + (((int64_t)b * a.T + t) * a.H + kvh * a.G + r - t * a.G) * HD;
        });
    };
    if (tile0 < NT) request_q();
    const PagedSpan sp = paged_span(a, sl.n);
    const int units = paged_units(sp, UNIT), u0 = sl.at * sl.per, u1 = min(units, u0 + sl.per);
    if (!FUSED && kvh == 0 && blockIdx.y == 0 && sl.at == 0 && threadIdx.x == 0) a.plan[b] = make_int2(j, sl.used);

    // The wave's i-th unit, of a stretch of its own; its page is looked up one unit before.
    const PagedTable table = (PagedTable)(uintptr_t)(a.table + (int64_t)b * a.n_table);
    const int share = sl.per / NW, w0 = u0 + wave * share, mine = max(0, min(share, u1 - w0));
    auto key_of = [&](int i) { return sp.first + (w0 + i) * UNIT; };
    PagedPage<HD, F16> page;
    page.at = -1, page.look(a, table, key_of(0) >> a.lp);
    RowsUnit<HD, F16, KT> u;
    const PagedLane<HD, F16, KT> lanes(rl, kq);
    bool has;  // the unit has a page
    auto slot_of = [&](int i) { return i < mine ? (uint32_t)(key_of(i) & ((1 << a.lp) - 1)) : 1u << 20; };
    auto request_k = [&](int i) {
        const int to = key_of(i) >> a.lp;
        if (to != page.at) page.turn(a, kvh, sp.end, to);
        has = page.has;
        const int next = key_of(i + 1) >> a.lp;
        if (next != to) page.look(a, table, next);
        paged_load_k<HD, F16, KT>(u, page.kv, slot_of(i), lanes);
    };
    auto request_v = [&](int i) { paged_load_v<HD, F16, KT>(u, page.kv, slot_of(i), lanes); };
    request_k(0), request_v(0);

    RowsQ<HD, NT> q;
    if constexpr (LOW) {
        if (wave < NT) {
            RowsQ<HD, 1> mine;
            rows_query<HD, 1, true>(mine, in, a.scale);
#pragma unroll
            for (int c = 0; c < HD / 32; c++) {
                L.q.high[wave][c][lane] = __builtin_bit_cast(uint4, mine.h[0][c]);
                L.q.low[wave][c][lane] = __builtin_bit_cast(uint4, mine.l[0][c]);
            }
            if (kq == 0) L.q.p2e[wave][rl] = mine.p2e[0];
        }
        __syncthreads();
#pragma unroll
        for (int qt = 0; qt < NT; qt++) {
            q.p2e[qt] = L.q.p2e[qt][rl];
#pragma unroll
            for (int c = 0; c < HIGH; c++) q.h[qt][c] = __builtin_bit_cast(ar_h8, L.q.high[qt][c][lane]);
        }
    } else {
        rows_query<HD, NT, true>(q, in, a.scale);
    }
    // Token t's rows take keys [first(t), last(t)); every row of the workgroup those of [all0, all1).
    auto last = [&](int t) { return sp.end - a.T + t + 1; };
    auto first = [&](int t) { return a.window ? max(0, last(t) - a.window) : 0; };
    const int all1 = last(rows_div(r0, a.g_m)), all0 = first(rows_div(r0 + rows - 1, a.g_m));
    int to[NT];
#pragma unroll
    for (int qt = 0; qt < NT; qt++) {
        const int t = rows_div(r0 + min(16 * qt + rl, rows - 1), a.g_m);
        to[qt] = 16 * qt + rl < rows ? last(t) : 0;
    }
    auto inside = [&](int key) { return key >= all0 && key + UNIT <= all1; };
    RowsSum<HD, NT> sum;
    rows_clear<HD, NT>(sum);
    if (EDGE && !LOW) __syncthreads();  // the flag is set
    auto high = [&](int qt, int c) { return c < HIGH ? q.h[qt][c] : __builtin_bit_cast(ar_h8, L.q.high[LOW ? qt : 0][c][lane]); };
    auto low = [&](int qt, int c) { return LOW ? __builtin_bit_cast(ar_h8, L.q.low[LOW ? qt : 0][c][lane]) : q.l[qt][c]; };
    // The next unit's keys are requested once this one's are used, its values once all is.
    for (int i = 0; i < mine; i++) {
        const bool h = has, whole = h && inside(key_of(i));
        int kb[KT];
#pragma unroll
        for (int t = 0; t < KT; t++) kb[t] = h ? key_of(i) + 16 * t : 0x7fffff00;  // (no page: no row takes its keys)
        if constexpr (LOW) asm volatile("" ::: "memory");  // (the low planes are read again: registers are what LDS saves)
        if constexpr (EDGE)
            if (!whole && paged_clean<HD, F16, KT>(u)) nonfinite = 1;
        paged_unit<HD, F16, KT, NT>(
            u, q.p2e, high, low, sum, kb, kq, whole,
            [&](int qt, int key) {
                const uint32_t x = rows_below(key, to[qt]);
                return EDGE && a.window ? x & ~rows_below(key, to[qt] - a.window) : x;
            },
            [&] { request_k(i + 1); });
        request_v(i + 1);
    }

    // The infinite and NaN values that were left out, of the keys that row r takes.
    auto add_nonfinite = [&](int r, int d, float4 &o) {
        const int t = rows_div(r0 + r, a.g_m);
        for (int u = u0; u < u1; u++) {
            const int k0 = sp.first + u * UNIT;
            const int page = k0 >> a.lp < a.n_table ? table[k0 >> a.lp] : -1;
            if ((uint32_t)page >= (uint32_t)a.n_pages || inside(k0)) continue;
            for (int key = max(first(t), k0); key < min(last(t), k0 + UNIT); key++) {
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
#pragma unroll
    for (int qt = 0; qt < NT; qt++) {
        RowsSum<HD, 1> one;
        one.m[0] = sum.m[qt], one.l[0] = sum.l[qt];
#pragma unroll
        for (int dt = 0; dt < HD / 16; dt++) one.o[0][dt] = sum.o[qt][dt];
        if (16 * qt >= rows) break;
        rows_combine<HD, NW>(L.parts, one, rows - 16 * qt, wave, rl, kq, [&](int r, int d, float4 o, float m, float l) {
            r += 16 * qt;
            if (EDGE && nonfinite) add_nonfinite(r, d, o);
            if (sl.used == 1) {
                *(float4 *)(paged_out<HD>(a, b, kvh, r0 + r) + d) = rows_over(o, l);
                return;
            }
            const uint32_t at = (uint32_t)sl.at * stride + (uint32_t)r * (HD + 4) * 4;
            constexpr int POLICY = FUSED ? BUF_SC1 : 0;
            if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, make_float2(m, l)), part, at, 0, POLICY);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), part, at + 16 + 4 * d, 0, POLICY);
        });
    }
    if constexpr (FUSED) {
        if (sl.used == 1) return;
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
        auto join = [&](auto sg) {  // rows at a time: few slices leave each to a quarter of the threads
            constexpr int SG = decltype(sg)::value, TPR = HD / 4 * SG;
            for (int g0 = 0; g0 < rows; g0 += 64 * NW / TPR) {
                const int g = g0 + (int)threadIdx.x / TPR;
                float M, l;
                const float4 o = rows_join<HD, SG>(L.join, sl.used, M, l, [&](int s, int d, float2 &ml, float4 &x) {
                    const uint32_t at = (uint32_t)s * stride + (uint32_t)min(g, rows - 1) * (HD + 4) * 4;
                    ml = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(part, at, 0, BUF_SC1));
                    x = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(part, at + 16 + 4 * d, 0, BUF_SC1));
                });
                if (g < rows && threadIdx.x % TPR < HD / 4)
                    *(float4 *)(paged_out<HD>(a, b, kvh, r0 + g) + 4 * (threadIdx.x % TPR)) = rows_over(o, l);
            }
        };
        if (sl.used <= 8) join(std::integral_constant<int, 1>{});
        else join(std::integral_constant<int, JOIN_SG>{});
    }
}

// The slices' join where few sequences have many: 256 / (HD / 4 x SG) rows a workgroup.
template <int HD>
__global__ __launch_bounds__(256) void k_paged_merge(PagedArgs a, int64_t rows) {
    constexpr int TPR = HD / 4 * JOIN_SG;
    __shared__ RowsJoin J;
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (256 / TPR) + threadIdx.x / TPR, at = min(row, rows - 1);
    const int b = (int)(at / ((int64_t)a.HKV * a.R)), kvh = (int)(at / a.R % a.HKV), r = (int)(at % a.R);
    const int2 plan = a.plan[b];
    const int blocks = (a.R + a.RT - 1) / a.RT;
    float M, l;
    const float4 o = rows_join<HD, JOIN_SG>(J, plan.y == 1 ? 0 : plan.y, M, l, [&](int s, int d, float2 &ml, float4 &x) {
        const float *p = a.part + (((int64_t)(kvh * blocks + r / a.RT) * a.cap + plan.x + s) * a.RT + r % a.RT) * (HD + 4);
        ml = *(const float2 *)p, x = *(const float4 *)(p + 4 + d);
    });
    if (plan.y == 1 || row >= rows || threadIdx.x % TPR >= HD / 4) return;
    *(float4 *)(paged_out<HD>(a, b, kvh, r) + 4 * (threadIdx.x % TPR)) = rows_over(o, l);
}

// ---- host ----------------------------------------------------------------------------------------

struct PagedPlan {
    int nt, rt, blocks, nw, cap;  // row tiles a wave, rows a workgroup, blocks of them, waves a workgroup, slices in all
    bool fused;
    size_t part, plan;
};
static PagedPlan paged_plan(int B, int T, int H, int HKV, int HD, int n_cu) {
    PagedPlan p;
    const int R = T * (H / HKV);
    p.nt = R > 16 && HD <= 128 ? 2 : 1;  // (two share the keys' and values' conversions; heads of 256 have no registers for it)
    p.rt = std::min(R, 16 * p.nt);
    p.blocks = (R + p.rt - 1) / p.rt;
    const int items = B * HKV * p.blocks, slots = (HD <= 128 ? 2 : 1) * n_cu;
    // Few items want eight waves, which halve the slices to join (4 x 4096 keys 15.5 us against 17; two row tiles of 1 x 8192
    // 19 against 23, though of 1 x 700 16 against 13); with many items their long slices no longer even out (24 ragged sequences, 6
    // tokens: 107 against 81).
    p.nw = HD == 256 || (p.nt == 2 ? 2 * items >= n_cu : 8 * items >= slots) ? 4 : 8;
    // Two slices a sequence, which always fit, and whole rounds of the workgroups that run at once (40 ragged sequences 112 us
    // against 136 in one round and a quarter; three slices 4 % less here, but 64 x 2000 keys 69 against 61).
    auto cap = [&] {
        const int round = std::max(1, slots * 4 / p.nw / (HKV * p.blocks));
        return (2 * B + round - 1) / round * round;
    };
    p.cap = cap();
    // The last slice joins, a launch less, where sequences of one length leave its threads up to 8 loads each (64 x 128 keys 8 us
    // against 13, 1 x 32768 22.1 against 23.3, 1 x 700 9.9 against 11). With more its workgroup is the longer way (1 x 8192, 2
    // tokens 17.8 against 14.9; 8 ragged sequences of 4 tokens 38 against 23; two row tiles of them 22.7 against 13.9).
    p.fused = items <= 4096 && R <= 16 && (int64_t)p.cap / B * R * (HD / 4) <= 8 * 64 * p.nw;
    if (!p.fused && p.nt == 1 && HD <= 128) {
        p.nw = 8;
        p.cap = cap();
    }
    p.part = align_up((size_t)p.cap * HKV * p.blocks * p.rt * (HD + 4) * sizeof(float), 256);
    p.plan = (size_t)B * sizeof(int2);
    return p;
}
size_t attn_paged_scratch_bytes(int B, int T, int H, int HKV, int HD, int n_cu) {
    const PagedPlan p = paged_plan(B, T, H, HKV, HD, n_cu);
    return p.part + p.plan;
}
template <class P>
static hipError_t paged_launch(const PagedArgs &a, const PagedPlan &p, hipStream_t s) {
    hipLaunchKernelGGL(k_attn_paged<P>, dim3(p.cap * a.HKV, p.blocks), dim3(64 * P::NW), 0, s, a);
    if (P::FUSED) return hipGetLastError();
    const int64_t rows = (int64_t)a.B * a.HKV * a.R;
    constexpr int RPW = 256 / (P::HD / 4 * JOIN_SG);
    // (two dimensions: one has up to 2^32 threads, which 4096 sequences of 16 tokens of 256 heads of 256 pass)
    const int64_t groups = (rows + RPW - 1) / RPW, x = std::min<int64_t>(groups, 1 << 20);
    hipLaunchKernelGGL(k_paged_merge<P::HD>, dim3((unsigned)x, (unsigned)((groups + x - 1) / x)), dim3(256), 0, s, a, rows);
    return hipGetLastError();
}
// Two row tiles of q8 heads of 128 take 32 keys a unit if pages allow: half the value products' instructions (24 ragged
// sequences, 6 tokens: 81 us against 90; 1 x 8192 19 against 18). One row tile takes 16: 1 x 32768 keys 23.6 against 24.6 us,
// 8 x 8192 of 4 x 4 rows 36 against 42. Heads of 64 always 32 (24 ragged 17.7 against 18.8).
template <int D, bool F, int KT>
static hipError_t paged_by_rows(const PagedArgs &a, const PagedPlan &p, hipStream_t s) {
    constexpr int WIDE = D <= 128 ? 8 : 4;
    if constexpr (D <= 128)
        if (p.nt == 2) {
            if constexpr (D == 128 && !F)
                if (a.lp >= 5) {
                    if (p.nw == 8) return paged_launch<PagedForm<D, F, 2, 2, 8, true, false>>(a, p, s);
                    return paged_launch<PagedForm<D, F, 2, 2, 4, true, false>>(a, p, s);
                }
            if (p.nw == 8) return paged_launch<PagedForm<D, F, KT, 2, 8, true, false>>(a, p, s);
            return paged_launch<PagedForm<D, F, KT, 2, 4, true, false>>(a, p, s);
        }
    if (a.T > 1 || a.window) {
        if (p.fused && p.nw == 4) return paged_launch<PagedForm<D, F, KT, 1, 4, true, true>>(a, p, s);
        if (p.fused) return paged_launch<PagedForm<D, F, KT, 1, WIDE, true, true>>(a, p, s);
        return paged_launch<PagedForm<D, F, KT, 1, WIDE, true, false>>(a, p, s);
    }
    if (p.fused && p.nw == 4) return paged_launch<PagedForm<D, F, KT, 1, 4, false, true>>(a, p, s);
    if (p.fused) return paged_launch<PagedForm<D, F, KT, 1, WIDE, false, true>>(a, p, s);
    return paged_launch<PagedForm<D, F, KT, 1, WIDE, false, false>>(a, p, s);
}
hipError_t launch_attn_paged(const float *q, int B, int T, int H, int HKV, int HD, KvLayer kv, int kv_f16, int n_pages,
                             int page, const int32_t *table, int n_table, const int32_t *n_keys, int window, float scale,
                             void *scratch, int *counters, float *out, int n_cu, hipStream_t s) {
    const PagedPlan p = paged_plan(B, T, H, HKV, HD, n_cu);
    PagedArgs a{};
    a.q = q, a.kv = kv, a.table = table, a.n_table = n_table, a.n_pages = n_pages, a.lp = __builtin_ctz(page);
    a.B = B, a.T = T, a.H = H, a.HKV = HKV, a.G = H / HKV, a.R = T * a.G, a.RT = p.rt, a.window = std::min(window, 1 << 30);
    a.cap = p.cap, a.g_m = rows_magic(a.G), a.hkv_m = rows_magic(HKV), a.n_keys = n_keys, a.scale = scale;
    a.part = (float *)scratch, a.plan = (int2 *)((uint8_t *)scratch + p.part), a.counters = counters, a.out = out;
    return rows_by_shape(HD, kv_f16, [&](auto hd, auto f16) {
        constexpr int D = decltype(hd)::value;
        constexpr bool F = decltype(f16)::value;
        if constexpr (D == 64)
            if (page >= 32) return paged_by_rows<D, F, 2>(a, p, s);
        return paged_by_rows<D, F, 1>(a, p, s);
    });
}

}  // namespace ts5hip
