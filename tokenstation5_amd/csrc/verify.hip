// Drafted tokens judged by the target's and the draft's probabilities, with given random numbers: draft i is kept while
// r_i q_i(x_i) < p_i(x_i); after the first that is not, a token is drawn from max(p - q, 0), after the last one from p,
// as the first index whose cumulative weight passes u times their sum. What is emitted then has the target's
// distribution, whatever the draft's.
//
// All of it in fp64: a token is the first past a bound, and with fp32 weights about one draw in a thousand over 150000
// entries would be another one. Two launches:
//  k_verify_rows  the maximum of each slice of each row and the sum of its weights 2^((l - maximum) log2(e) / T);
//  k_verify_pick  joins the rows' slices, judges the drafts, and finds the slice and then the entry that the token is. Where
//                 that is drawn from p - q of two rows, a workgroup a slice judges (cheaper than a third launch) and sums
//                 that slice's weights, and the last one to finish goes on; else one workgroup does it all, from
//                 the sums there are (a draft's own entry is kept out of them, so that p without it is exact).
#include <algorithm>
#include <climits>

#include "common.h"
#include "kernels.h"

namespace ts5hip {

constexpr int VF_SLICE = 4096, VF_NT = 256, VP_NT = 512;  // entries of a slice, threads of k_verify_rows, of k_verify_pick
constexpr double VF_LOG2E = 1.4426950408889634;

struct VerifyPart {
    double sum;   // of the weights over the slice's own maximum's, less the row's draft
    float top;    // -inf: every entry is; NaN: no distribution (a NaN or plus infinity)
    int32_t best; // the first entry at the maximum
};
struct VerifyArgs {
    const float *logits, *draft;  // [B][T + 1][ld], [B][T][ld_draft] or null
    int64_t ld, ld_draft;
    int V, B, T, ns;              // ns: slices of a row
    const int32_t *drafts, *n_draft;  // [B][T], [B] or null
    const float *temp, *uni;      // [B], [B][T + 1]
    VerifyPart *parts;            // [B][2 T + 1][ns]: the target's rows, then the draft's
    double *sums;                 // [B][stride] of the slices of the row that is drawn from
    int sums_stride;
    int *counters;                // [B], CTR_STRIDE ints apart, zero between launches
    int32_t *tokens, *n_tokens;   // [B][T + 1], [B]
    float *logp;                  // [B][T + 1] or null
};
__device__ inline int vf_drafts(const VerifyArgs &a, int b) { return a.n_draft ? max(0, min(a.n_draft[b], a.T)) : a.T; }
__device__ inline bool vf_greedy(float t) { return !(t > 0.f); }

// 2^x, x <= 0 (minus infinity: 0): x = k + f with |f| <= 1/2, the polynomial of degree 10 that meets 2^f at the zeros of
// the 11th Chebyshev polynomial (off by 3.2e-16 at most), and k to the exponent.
__device__ inline double vf_exp2(double x) {
    x = fmax(x, -2000.0);  // (0; and where x is a product, a fused x - k would be its rounding error, of any size)
    const double k = __builtin_rint(x), f = x - k;
    double p = 7.072585949269223e-09;
    p = fma(p, f, 1.0208690299958306e-07);
    p = fma(p, f, 1.321544258792169e-06);
    p = fma(p, f, 1.5252657260200837e-05);
    p = fma(p, f, 0.0001540353044173605);
    p = fma(p, f, 0.0013333558230164974);
    p = fma(p, f, 0.009618129107606888);
    p = fma(p, f, 0.05550410866444772);
    p = fma(p, f, 0.24022650695910097);
    p = fma(p, f, 0.69314718055995);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)k);
}
// The weight of logit l where the maximum is m (finite). by = log2(e) / T, above 0, so that minus infinity weighs 0.
__device__ inline double vf_weight(float l, float m, double by) { return vf_exp2(((double)l - (double)m) * by); }
__device__ inline double vf_by(float temp) { return fmax(VF_LOG2E / (double)temp, 1e-300); }

// Lanes moved by DPP, a double as two halves; a lane without a source gets 0.
template <int CTRL, int ROW_MASK, int BANK_MASK>
__device__ inline double vf_dpp(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    const uint32_t l = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROW_MASK, BANK_MASK, true);
    const uint32_t h = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROW_MASK, BANK_MASK, true);
    return __longlong_as_double((long long)((uint64_t)h << 32 | l));
}
// The sum over each 16-lane row, in every lane of it.
__device__ inline double vf_row_sum(double x) {
    x += vf_dpp<0xB1, 0xF, 0xF>(x);   // quad_perm [1,0,3,2]
    x += vf_dpp<0x4E, 0xF, 0xF>(x);   // quad_perm [2,3,0,1]
    x += vf_dpp<0x141, 0xF, 0xF>(x);  // row_half_mirror
    return x + vf_dpp<0x140, 0xF, 0xF>(x);  // row_mirror
}
// Inclusive sums over the wave's lanes.
__device__ inline double vf_scan(double x) {
    x += vf_dpp<0x111, 0xF, 0xF>(x);  // row_shr:1
    x += vf_dpp<0x112, 0xF, 0xF>(x);  // row_shr:2
    x += vf_dpp<0x114, 0xF, 0xE>(x);  // row_shr:4
    x += vf_dpp<0x118, 0xF, 0xC>(x);  // row_shr:8
    x += vf_dpp<0x142, 0xA, 0xF>(x);  // row_bcast:15 into rows 1 and 3
    return x + vf_dpp<0x143, 0xC, 0xF>(x);  // row_bcast:31 into rows 2 and 3
}
__device__ inline double vf_lane(double x, int lane) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    const uint32_t l = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), h = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __longlong_as_double((long long)((uint64_t)h << 32 | l));
}
// The least over each 16-lane row, over the wave: in every lane.
template <int CTRL, int ROW_MASK>
__device__ inline int vf_dpp_min(int x) { return min(x, __builtin_amdgcn_update_dpp(x, x, CTRL, ROW_MASK, 0xF, false)); }
__device__ inline int vf_row_min(int x) {
    return vf_dpp_min<0x140, 0xF>(vf_dpp_min<0x141, 0xF>(vf_dpp_min<0x4E, 0xF>(vf_dpp_min<0xB1, 0xF>(x))));
}
__device__ inline int vf_wave_min(int x) {
    x = vf_dpp_min<0x143, 0xC>(vf_dpp_min<0x142, 0xA>(vf_row_min(x)));
    return __builtin_amdgcn_readlane(x, 63);
}

typedef float vf_f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows begin anywhere
// A thread's entries of a slice, of NT threads: x[4 j + i] is entry s0 + 4 (NT j + thread) + i; past the row: minus infinity.
template <int NT>
__device__ inline void vf_load(const float *row, int s0, int V, float (&x)[VF_SLICE / NT]) {
#pragma unroll
    for (int j = 0; j < VF_SLICE / NT / 4; j++) {
        const int e = s0 + 4 * (NT * j + (int)threadIdx.x);
        if (e + 4 <= V) {
            const vf_f4 v = *(const vf_f4 *)(row + e);
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 * j + i] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 * j + i] = e + i < V ? row[e + i] : -INFINITY;
        }
    }
}
template <int NT>
__device__ inline int vf_index(int s0, int k) { return s0 + 4 * (NT * (k / 4) + (int)threadIdx.x) + k % 4; }

// Sum over the workgroup, in every thread.
template <int NT>
__device__ inline double vf_block_sum(double v, double (&lds)[NT / WAVE]) {
    v = vf_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < NT / WAVE; w++) s += lds[w];
    return s;
}

// grid (slices, 2 T + 1 or T + 1 rows, B)
__global__ __launch_bounds__(VF_NT) void k_verify_rows(VerifyArgs a) {
    constexpr int PER = VF_SLICE / VF_NT;
    __shared__ double sums[4];
    __shared__ float tops[4];
    __shared__ int bests[4];
    __shared__ int bad;
    const int b = blockIdx.z, r = blockIdx.y, s0 = blockIdx.x * VF_SLICE, nd = vf_drafts(a, b);
    const float temp = a.temp[b];
    const bool target = r <= a.T;
    if (target ? r > nd : r - a.T - 1 >= nd || vf_greedy(temp)) return;  // not one of the sequence's rows
    const float *row = target ? a.logits + ((int64_t)b * (a.T + 1) + r) * a.ld
                              : a.draft + ((int64_t)b * a.T + r - a.T - 1) * a.ld_draft;
    float x[PER];
    vf_load<VF_NT>(row, s0, a.V, x);
    const int d = r < nd ? a.drafts[(int64_t)b * a.T + r] : -1;
    if (threadIdx.x == 0) bad = 0;
    float top = -INFINITY;
    bool no = false;
#pragma unroll
    for (int k = 0; k < PER; k++) top = fmaxf(top, x[k]), no |= x[k] != x[k];
    no |= top == INFINITY;
    top = wave_max_dpp(top);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    if (no) bad = 1;
    int best = INT_MAX;
#pragma unroll
    for (int k = PER - 1; k >= 0; k--) best = x[k] == top ? vf_index<VF_NT>(s0, k) : best;  // (ascending with k)
    best = vf_wave_min(best);
    if ((threadIdx.x & 63) == 0) bests[threadIdx.x >> 6] = best;
    double sum = 0.0;
    if (!vf_greedy(temp) && top != -INFINITY) {
        const double by = vf_by(temp);
        double w[PER];
#pragma unroll
        for (int k = 0; k < PER; k++) w[k] = vf_weight(x[k], top, by);
        if ((uint32_t)(d - s0) < (uint32_t)VF_SLICE) {
#pragma unroll
            for (int k = 0; k < PER; k++) w[k] = vf_index<VF_NT>(s0, k) == d ? 0.0 : w[k];
        }
#pragma unroll
        for (int k = 0; k < PER; k++) sum += w[k];
    }
    sum = vf_block_sum<VF_NT>(sum, sums);
    if (threadIdx.x == 0) {
        VerifyPart p;
        p.sum = sum, p.top = bad ? NAN : top, p.best = min(min(bests[0], bests[1]), min(bests[2], bests[3]));
        a.parts[((int64_t)b * (2 * a.T + 1) + r) * a.ns + blockIdx.x] = p;
    }
}

// A row's slices as one, by 16 lanes: in every one of them.
__device__ inline VerifyPart vf_join(const VerifyPart *p, int ns, double by) {
    constexpr int AHEAD = 4;
    const int lane = threadIdx.x & 15;
    float top = -INFINITY;
    double sum = 0.0;
    int best = INT_MAX, no = 0;
    for (int i0 = lane; i0 < ns; i0 += 16 * AHEAD) {  // (ascending: the first of equal maxima stays)
        VerifyPart x[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) x[k] = p[min(i0 + 16 * k, ns - 1)];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            if (i0 + 16 * k >= ns) break;
            no |= x[k].top != x[k].top;
            if (x[k].top > top) {
                sum = x[k].sum + (top == -INFINITY ? 0.0 : sum * vf_weight(top, x[k].top, by));
                top = x[k].top, best = x[k].best;
            } else if (x[k].top > -INFINITY) {
                sum += x[k].sum * vf_weight(x[k].top, top, by);
            }
        }
    }
    VerifyPart s;
    s.top = row_max_dpp(top);
    sum = top == -INFINITY ? 0.0 : sum * vf_weight(top, s.top, by);
    s.sum = vf_row_sum(sum), s.best = vf_row_min(top == s.top ? best : INT_MAX);
    if (vf_row_min(-no)) s.top = NAN;
    return s;
}
__device__ inline bool vf_has(const VerifyPart &p) { return p.top > -INFINITY; }  // (not NaN: a distribution)

// grid (slices with a draft model, else 1, B). Its time is a chain: the counts and drafts, the drafts' logits and the slices'
// sums, the slice, its weights.
constexpr int VF_MAX_DRAFTS = 63, VF_MAX_SLICES = 256;
__global__ __launch_bounds__(VP_NT) void k_verify_pick(VerifyArgs a) {
    __shared__ VerifyPart rows[2 * VF_MAX_DRAFTS + 1];
    __shared__ double lds[VP_NT / WAVE];
    __shared__ int drafts[VF_MAX_DRAFTS + 1], kept;
    __shared__ float draft_l[VF_MAX_DRAFTS + 1];  // their logits
    constexpr int PER = VF_SLICE / VP_NT, NW = VP_NT / WAVE;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float temp = a.temp[b];
    const int nd = vf_drafts(a, b);
    const float u_draw = a.uni[(int64_t)b * (a.T + 1) + a.T];
    const bool greedy = vf_greedy(temp), model = a.draft && !greedy;
    const double by = greedy ? 1.0 : vf_by(temp);
    const float *target = a.logits + (int64_t)b * (a.T + 1) * a.ld, *draft = a.draft + (int64_t)b * a.T * a.ld_draft;
    // Thread t < nd: draft t, its number and its logits.
    const int32_t d = tid < a.T ? a.drafts[(int64_t)b * a.T + tid] : -1;
    const float r = a.uni[(int64_t)b * (a.T + 1) + min(tid, a.T)];
    const bool inside = (uint32_t)d < (uint32_t)a.V;
    const float lp = inside ? target[tid * a.ld + d] : -INFINITY, lq = inside && a.draft ? draft[tid * a.ld_draft + d] : -INFINITY;
    if (tid < nd) drafts[tid] = d, draft_l[tid] = lp;
    const VerifyPart *parts = a.parts + (int64_t)b * (2 * a.T + 1) * a.ns;
    for (int i = tid / 16; i < nd + 1 + (model ? nd : 0); i += VP_NT / 16) {
        const VerifyPart p = vf_join(parts + (int64_t)(i <= nd ? i : a.T + i - nd) * a.ns, a.ns, by);
        if (tid % 16 == 0) rows[i] = p;
    }
    __syncthreads();
    double wp = 0.0, sp = 1.0;  // the draft's weight and its row's sum
    if (wave == 0) {
        bool ok = false;
        if (tid < nd && vf_has(rows[tid])) {
            const VerifyPart &p = rows[tid];
            if (greedy) {
                ok = d == p.best;
            } else if (inside) {
                wp = vf_weight(lp, p.top, by), sp = p.sum + wp;
                double q = 1.0;
                if (model) {
                    const VerifyPart &y = rows[nd + 1 + tid];
                    q = vf_has(y) ? vf_weight(lq, y.top, by) / y.sum : NAN;
                }
                ok = (double)r * q < wp / sp;
            }
        }
        const uint64_t no = __builtin_amdgcn_ballot_w64(!ok);
        if (tid == 0) kept = no ? min(nd, __ffsll((unsigned long long)no) - 1) : nd;
    }
    __syncthreads();
    const int m = kept;
    int32_t *tokens = a.tokens + (int64_t)b * (a.T + 1);
    float *logps = a.logp ? a.logp + (int64_t)b * (a.T + 1) : nullptr;
    if (blockIdx.x == 0) {  // the kept ones, and nothing behind the next
        if (tid < m) {
            tokens[tid] = d;
            if (logps) logps[tid] = greedy ? 0.f : (float)(((double)lp - (double)rows[tid].top) / (double)temp - log(sp));
        }
        if (tid > m && tid <= a.T) {
            tokens[tid] = -1;
            if (logps) logps[tid] = 0.f;
        }
    }
    const VerifyPart p = rows[m];
    if (!vf_has(p) || greedy) {
        if (blockIdx.x == 0 && tid == 0) {
            const bool has = vf_has(p);
            tokens[m] = has ? p.best : -1, a.n_tokens[b] = m + (has ? 1 : 0);
            if (logps) logps[m] = 0.f;
        }
        return;
    }
    // The token's weights: p of row m, less q where that row's draft was not kept.
    const int dm = m < nd ? drafts[m] : -1;
    const VerifyPart q = rows[model && m < nd ? nd + 1 + m : 0];
    const bool by_q = model && m < nd && vf_has(q);
    if (!by_q && blockIdx.x > 0) return;
    const float *row = target + (int64_t)m * a.ld, *qrow = draft + (int64_t)m * a.ld_draft;
    const float lm = m < nd ? draft_l[m] : -INFINITY;
    const double wm = vf_weight(lm, p.top, by), sum_p = p.sum + wm, inv_p = 1.0 / sum_p;
    int certain = !model ? dm : -1;  // (its entry is not drawn)
    double w[PER];
    auto weights = [&](int s0, bool less) {
        float x[PER];
        vf_load<VP_NT>(row, s0, a.V, x);
        if (less) {
            float y[PER];
            vf_load<VP_NT>(qrow, s0, a.V, y);
            const double inv_q = 1.0 / q.sum;
#pragma unroll
            for (int k = 0; k < PER; k++) {
                // (both products rounded: fused, equal rows would leave the rounding error of one, above 0 for half of the
                // entries, and the token would be drawn by those)
#pragma clang fp contract(off)
                const double pk = vf_weight(x[k], p.top, by) * inv_p, qk = vf_weight(y[k], q.top, by) * inv_q;
                w[k] = fmax(pk - qk, 0.0);
            }
        } else {
#pragma unroll
            for (int k = 0; k < PER; k++) {
                w[k] = vf_weight(x[k], p.top, by);
                w[k] = vf_index<VP_NT>(s0, k) == certain ? 0.0 : w[k];
            }
        }
    };
    double mine = 0.0;  // thread i: the weights of slice i
    if (by_q) {
        weights(blockIdx.x * VF_SLICE, true);
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < PER; k++) s += w[k];
        s = vf_block_sum<VP_NT>(s, lds);
        double *sums = a.sums + (int64_t)b * a.sums_stride;
        __shared__ int last;
        if (tid == 0) {
            __hip_atomic_store(sums + blockIdx.x, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            wait_stores();
            int *c = a.counters + b * CTR_STRIDE;
            last = atomicAdd(c, 1) == a.ns - 1;
            if (last) st_dev(c, 0);
        }
        __syncthreads();
        if (!last) return;
        if (tid < a.ns) mine = __hip_atomic_load(sums + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    const bool less = by_q && vf_block_sum<VP_NT>(mine, lds) > 0.0;  // (else they are equal: from p)
    if (!less) {
        mine = 0.0;
        if (tid < a.ns) {
            const VerifyPart x = parts[(int64_t)m * a.ns + tid];
            if (x.top > -INFINITY) mine = x.sum * vf_weight(x.top, p.top, by);
        }
        // The draft's own entry: not drawn where it was certain, unless there is no other (a number that is not below 1).
        if (!model && !(vf_block_sum<VP_NT>(mine, lds) > 0.0)) certain = -1;
        if (certain < 0 && (uint32_t)dm < (uint32_t)a.V && dm / VF_SLICE == tid) mine += wm;
    }
    // The slice: the first whose cumulative sum passes u of all; roundings may leave none: the last with a weight.
    __shared__ double before;
    __shared__ int firsts[NW], lasts[NW];
    double incl = vf_scan(mine);
    __syncthreads();
    if (lane == 63) lds[wave] = incl;
    __syncthreads();
    double base = 0.0, all = 0.0;
#pragma unroll
    for (int v = 0; v < NW; v++) base += v < wave ? lds[v] : 0.0, all += lds[v];
    incl += base;
    const double bound = (double)u_draw * all;
    auto pick = [&](int first, int last) {  // the least `first` there is, or the largest `last`
        first = vf_wave_min(first), last = -vf_wave_min(-last);
        if (lane == 0) firsts[wave] = first, lasts[wave] = last;
        __syncthreads();
        int f = INT_MAX, l = 0;
#pragma unroll
        for (int v = 0; v < NW; v++) f = min(f, firsts[v]), l = max(l, lasts[v]);
        return f != INT_MAX ? f : l;
    };
    const int slice = pick(mine > 0.0 && incl > bound ? tid : INT_MAX, mine > 0.0 ? tid : 0), s0 = slice * VF_SLICE;
    if (tid == slice) before = incl - mine;
    weights(s0, less);
    // Cumulative weights in the entries' order: groups j of 4 VP_NT, waves, lanes, four neighbours.
    __shared__ double tot[PER / 4][NW];
    double run[PER / 4];
#pragma unroll
    for (int j = 0; j < PER / 4; j++) {
        run[j] = vf_scan((w[4 * j] + w[4 * j + 1]) + (w[4 * j + 2] + w[4 * j + 3]));
        if (lane == 63) tot[j][wave] = run[j];
    }
    __syncthreads();
    base = before;
    int found = INT_MAX, positive = 0;
#pragma unroll
    for (int j = 0; j < PER / 4; j++) {
        double c = base;
#pragma unroll
        for (int v = 0; v < NW; v++) {
            c += v < wave ? tot[j][v] : 0.0;
            base += tot[j][v];
        }
        c += vf_dpp<0x138, 0xF, 0xF>(run[j]);  // wave_shr:1
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c += w[4 * j + i];
            const int e = vf_index<VP_NT>(s0, 4 * j + i);
            positive = w[4 * j + i] > 0.0 ? e : positive;
            found = w[4 * j + i] > 0.0 && c > bound ? min(found, e) : found;
        }
    }
    const int e = pick(found, positive);
    if (tid == 0) {
        tokens[m] = e, a.n_tokens[b] = m + 1;
        if (logps) logps[m] = (float)(((double)row[e] - (double)p.top) / (double)temp - log(sum_p));
    }
}

struct VerifyScratch {
    int ns, stride;
    size_t parts, sums;
};
static VerifyScratch verify_scratch(int V, int B, int T) {
    VerifyScratch s;
    s.ns = (V + VF_SLICE - 1) / VF_SLICE;
    s.stride = (s.ns + 15) / 16 * 16;  // whole 128-byte lines
    s.parts = align_up((size_t)B * (2 * T + 1) * s.ns * sizeof(VerifyPart), 256);
    s.sums = (size_t)B * s.stride * sizeof(double);
    return s;
}
int verify_max_vocab() { return VF_SLICE * VF_MAX_SLICES; }
int verify_max_drafts() { return VF_MAX_DRAFTS; }
size_t verify_scratch_bytes(int V, int B, int T) {
    const VerifyScratch s = verify_scratch(V, B, T);
    return s.parts + s.sums;
}
hipError_t launch_verify(const float *logits, int64_t ld, const float *draft, int64_t ld_draft, int V, int B, int T,
                         const int32_t *drafts, const int32_t *n_draft, const float *temp, const float *uni, void *scratch,
                         int *counters, int32_t *tokens, int32_t *n_tokens, float *logp, hipStream_t s) {
    const VerifyScratch p = verify_scratch(V, B, T);
    VerifyArgs a{};
    a.logits = logits, a.draft = draft, a.ld = ld, a.ld_draft = ld_draft, a.V = V, a.B = B, a.T = T, a.ns = p.ns;
    a.drafts = drafts, a.n_draft = n_draft, a.temp = temp, a.uni = uni;
    a.parts = (VerifyPart *)scratch, a.sums = (double *)((uint8_t *)scratch + p.parts), a.sums_stride = p.stride;
    a.counters = counters, a.tokens = tokens, a.n_tokens = n_tokens, a.logp = logp;
    hipLaunchKernelGGL(k_verify_rows, dim3(p.ns, T + 1 + (draft ? T : 0), B), dim3(VF_NT), 0, s, a);
    hipLaunchKernelGGL(k_verify_pick, dim3(draft ? p.ns : 1, B), dim3(VP_NT), 0, s, a);
    return hipGetLastError();
}

}  // namespace ts5hip
