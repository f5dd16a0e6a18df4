// Drafted tokens judged by the target's and the draft's probabilities, with given random numbers: draft i is kept while
// r_i q_i(x_i) < p_i(x_i); after the first that is not, a token is drawn from max(p - q, 0), after the last one from p,
// as the first index whose cumulative weight passes u times their sum. What is emitted then has the target's
// distribution, whatever the draft's.
//
// All of it in fp64: a token is the first past a bound, and with fp32 weights about one draw in a thousand over 150000
// entries would be another one. Two launches:
//  k_verify_rows  the maximum of each slice of each row and the sum of its weights 2^((l - maximum) log2(e) / T);
//  k_verify_pick  every workgroup of a sequence joins its rows' slices and judges the drafts (cheaper than a third
//                 launch), sums one slice's weights of the row the token is drawn from, and the last one to finish finds
//                 the slice and the entry.
#include <algorithm>
#include <climits>

#include "common.h"
#include "kernels.h"

namespace ts5hip {

constexpr int VF_NT = 256, VF_SLICE = 4096, VF_PER = VF_SLICE / VF_NT;  // 16 entries a thread, 4 neighbours at a time
constexpr double VF_LOG2E = 1.4426950408889634;

struct VerifyPart {
    double sum;   // of the weights, over the slice's own maximum's
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

// 2^x, x <= 0: x = k + f with |f| <= 1/2, the series of 2^f to its 13th term (under 2^-53), and k to the exponent.
__device__ inline double vf_exp2(double x) {
    x = fmax(x, -2000.0);  // (0; and where x is a product, a fused x - k would be its rounding error, of any size)
    const double k = __builtin_rint(x), f = (x - k) * 0.6931471805599453;
    double p = 1.0 / 6227020800.0;
    p = fma(p, f, 1.0 / 479001600.0);
    p = fma(p, f, 1.0 / 39916800.0);
    p = fma(p, f, 1.0 / 3628800.0);
    p = fma(p, f, 1.0 / 362880.0);
    p = fma(p, f, 1.0 / 40320.0);
    p = fma(p, f, 1.0 / 5040.0);
    p = fma(p, f, 1.0 / 720.0);
    p = fma(p, f, 1.0 / 120.0);
    p = fma(p, f, 1.0 / 24.0);
    p = fma(p, f, 1.0 / 6.0);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)k);
}
// The weight of logit l where the maximum is m; by = log2(e) / T.
__device__ inline double vf_weight(float l, float m, double by) {
    return l == -INFINITY ? 0.0 : vf_exp2(((double)l - (double)m) * by);
}

typedef float vf_f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows begin anywhere
// The thread's entries of a slice: x[4 j + i] is entry s0 + 4 (256 j + thread) + i; past the row: minus infinity.
__device__ inline void vf_load(const float *row, int s0, int V, float (&x)[VF_PER]) {
#pragma unroll
    for (int j = 0; j < VF_PER / 4; j++) {
        const int e = s0 + 4 * (VF_NT * j + (int)threadIdx.x);
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
__device__ inline int vf_index(int s0, int k) { return s0 + 4 * (VF_NT * (k / 4) + (int)threadIdx.x) + k % 4; }

// Sum over the workgroup, in thread 0.
__device__ inline double vf_block_sum(double v, double *lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

// grid (slices, 2 T + 1 or T + 1 rows, B)
__global__ __launch_bounds__(VF_NT) void k_verify_rows(VerifyArgs a) {
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
    float x[VF_PER];
    vf_load(row, s0, a.V, x);
    if (threadIdx.x == 0) bad = 0;
    float top = -INFINITY;
    bool no = false;
#pragma unroll
    for (int k = 0; k < VF_PER; k++) top = fmaxf(top, x[k]), no |= !(x[k] < INFINITY);
    top = wave_max_dpp(top);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    if (no) bad = 1;
    int best = INT_MAX;
#pragma unroll
    for (int k = VF_PER - 1; k >= 0; k--)
        if (x[k] == top) best = min(best, vf_index(s0, k));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, WAVE));
    if ((threadIdx.x & 63) == 0) bests[threadIdx.x >> 6] = best;
    double sum = 0.0;
    if (!vf_greedy(temp) && top != -INFINITY) {
        const double by = VF_LOG2E / (double)temp;
#pragma unroll
        for (int k = 0; k < VF_PER; k++) sum += vf_weight(x[k], top, by);
    }
    sum = vf_block_sum(sum, sums);
    if (threadIdx.x == 0) {
        VerifyPart p;
        p.sum = sum, p.top = bad ? NAN : top, p.best = min(min(bests[0], bests[1]), min(bests[2], bests[3]));
        a.parts[((int64_t)b * (2 * a.T + 1) + r) * a.ns + blockIdx.x] = p;
    }
}

// A row's slices as one, by a wave: in every lane.
__device__ inline VerifyPart vf_join(const VerifyPart *p, int ns, double by) {
    const int lane = threadIdx.x & 63;
    VerifyPart s;
    s.top = -INFINITY, s.sum = 0.0, s.best = INT_MAX;
    bool no = false;
    for (int i = lane; i < ns; i += WAVE) {  // (ascending: the first of equal maxima stays)
        const VerifyPart x = p[i];
        no |= x.top != x.top;
        if (x.top > s.top) {
            s.sum = x.sum + (s.top == -INFINITY ? 0.0 : s.sum * vf_exp2(((double)s.top - (double)x.top) * by));
            s.top = x.top, s.best = x.best;
        } else if (x.top > -INFINITY) {
            s.sum += x.sum * vf_exp2(((double)x.top - (double)s.top) * by);
        }
    }
    const float top = wave_max_dpp(s.top);
    s.sum = s.top == -INFINITY ? 0.0 : s.sum * vf_exp2(((double)s.top - (double)top) * by);
    if (s.top != top) s.best = INT_MAX;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        s.sum += __shfl_xor(s.sum, o, WAVE);
        s.best = min(s.best, __shfl_xor(s.best, o, WAVE));
    }
    s.top = __builtin_amdgcn_ballot_w64(no) ? NAN : top;
    return s;
}
__device__ inline bool vf_has(const VerifyPart &p) { return p.top > -INFINITY; }  // (not NaN: a distribution)

// grid (slices, B)
constexpr int VF_MAX_DRAFTS = 63, VF_MAX_SLICES = 256;
__global__ __launch_bounds__(VF_NT) void k_verify_pick(VerifyArgs a) {
    __shared__ VerifyPart rows[2 * VF_MAX_DRAFTS + 1];
    __shared__ double lds[4];
    __shared__ int kept;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nd = vf_drafts(a, b);
    const float temp = a.temp[b];
    const bool greedy = vf_greedy(temp), model = a.draft && !greedy;
    const double by = greedy ? 0.0 : VF_LOG2E / (double)temp;
    // Thread t < nd: draft t and its logits.
    const int32_t d = tid < nd ? a.drafts[(int64_t)b * a.T + tid] : -1;
    const bool inside = (uint32_t)d < (uint32_t)a.V;
    const float *target = a.logits + (int64_t)b * (a.T + 1) * a.ld, *draft = a.draft + (int64_t)b * a.T * a.ld_draft;
    const float lp = inside ? target[tid * a.ld + d] : -INFINITY, lq = inside && model ? draft[tid * a.ld_draft + d] : 0.f;
    const float r = tid < nd ? a.uni[(int64_t)b * (a.T + 1) + tid] : 0.f;
    const VerifyPart *parts = a.parts + (int64_t)b * (2 * a.T + 1) * a.ns;
    for (int i = wave; i < nd + 1 + (model ? nd : 0); i += VF_NT / WAVE) {
        const VerifyPart p = vf_join(parts + (int64_t)(i <= nd ? i : a.T + i - nd) * a.ns, a.ns, by);
        if (lane == 0) rows[i] = p;
    }
    __syncthreads();
    float logp = 0.f;
    if (wave == 0) {
        bool ok = false;
        if (tid < nd && vf_has(rows[tid])) {
            const VerifyPart &p = rows[tid];
            if (greedy) {
                ok = d == p.best;
            } else if (inside) {
                const double w = vf_weight(lp, p.top, by) / p.sum;
                const VerifyPart &q = rows[nd + 1 + (model ? tid : 0)];
                const double wq = !model ? 1.0 : vf_has(q) ? vf_weight(lq, q.top, by) / q.sum : NAN;
                ok = (double)r * wq < w;
                logp = (float)(((double)lp - (double)p.top) / (double)temp - log(p.sum));
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
            if (logps) logps[tid] = logp;
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
    // The token's weights: p, less q where the draft was not kept.
    const float *row = target + (int64_t)m * a.ld, *qrow = model && m < nd ? draft + (int64_t)m * a.ld_draft : nullptr;
    const VerifyPart q = rows[model && m < nd ? nd + 1 + m : 0];
    const bool by_q = qrow && vf_has(q);
    const int certain = !model && m < nd ? a.drafts[(int64_t)b * a.T + m] : -1;
    const double inv_p = 1.0 / p.sum, inv_q = by_q ? 1.0 / q.sum : 0.0;
    double w[VF_PER];
    auto weights = [&](int s0, bool plain) {
        float x[VF_PER];
        vf_load(row, s0, a.V, x);
#pragma unroll
        for (int k = 0; k < VF_PER; k++) w[k] = vf_weight(x[k], p.top, by) * inv_p;
        if (plain) return;
        if (by_q) {
            vf_load(qrow, s0, a.V, x);
#pragma unroll
            for (int k = 0; k < VF_PER; k++) w[k] = fmax(w[k] - vf_weight(x[k], q.top, by) * inv_q, 0.0);
        }
#pragma unroll
        for (int k = 0; k < VF_PER; k++)
            if (vf_index(s0, k) == certain) w[k] = 0.0;
    };
    auto sum_of = [&]() {
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < VF_PER; k++) s += w[k];
        return vf_block_sum(s, lds);
    };
    weights(blockIdx.x * VF_SLICE, false);
    const double mine = sum_of();
    double *sums = a.sums + (int64_t)b * a.sums_stride;
    __shared__ int last;
    if (tid == 0) {
        __hip_atomic_store(sums + blockIdx.x, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        wait_stores();
        int *c = a.counters + b * CTR_STRIDE;
        last = atomicAdd(c, 1) == a.ns - 1;
        if (last) st_dev(c, 0);
    }
    __syncthreads();
    if (!last) return;
    // The slice: the first whose cumulative sum passes u of all.
    __shared__ double slice[VF_MAX_SLICES];
    __shared__ double bound, before;
    __shared__ int chosen, entry, plain;
    if (tid < a.ns) slice[tid] = __hip_atomic_load(sums + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (tid == 0) {
        double all = 0.0;
        for (int i = 0; i < a.ns; i++) all += slice[i];
        plain = !(all > 0.0);  // (p and q equal up to rounding: the draft's row says nothing)
        if (plain) {
            all = 0.0;
            for (int i = 0; i < a.ns; i++) {
                const VerifyPart x = parts[(int64_t)m * a.ns + i];
                slice[i] = x.top == -INFINITY ? 0.0 : x.sum * vf_exp2(((double)x.top - (double)p.top) * by) * inv_p;
                all += slice[i];
            }
        }
        const double u = (double)a.uni[(int64_t)b * (a.T + 1) + a.T] * all;
        double run = 0.0;
        int at = -1;
        for (int i = 0; i < a.ns; i++) {
            if (slice[i] > 0.0) at = i, before = run;
            run += slice[i];
            if (run > u) break;
        }
        chosen = at, bound = u, entry = INT_MAX;
    }
    __syncthreads();
    const int s0 = chosen * VF_SLICE;
    weights(s0, plain);
    // Cumulative weights in the entries' order: groups j of 1024, waves, lanes, four neighbours.
    __shared__ double tot[VF_PER / 4][VF_NT / WAVE];
    double incl[VF_PER / 4];
#pragma unroll
    for (int j = 0; j < VF_PER / 4; j++) {
        double s = (w[4 * j] + w[4 * j + 1]) + (w[4 * j + 2] + w[4 * j + 3]);
#pragma unroll
        for (int o = 1; o < WAVE; o <<= 1) {
            const double y = __shfl_up(s, o, WAVE);
            if (lane >= o) s += y;
        }
        incl[j] = s;
        if (lane == 63) tot[j][wave] = s;
    }
    __syncthreads();
    const double u = bound;
    double base = before;
    int found = INT_MAX, positive = -1;
#pragma unroll
    for (int j = 0; j < VF_PER / 4; j++) {
#pragma unroll
        for (int v = 0; v < VF_NT / WAVE; v++) {
            if (v == wave) {
                const double prev = __shfl_up(incl[j], 1, WAVE);
                double c = base + (lane ? prev : 0.0);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    c += w[4 * j + i];
                    const int e = vf_index(s0, 4 * j + i);
                    if (w[4 * j + i] > 0.0) {
                        positive = e;
                        if (c > u) found = min(found, e);
                    }
                }
            }
            base += tot[j][v];
        }
    }
    // Roundings may leave no entry past the bound: then the slice's last with a weight.
    __shared__ int backup;
    if (tid == 0) backup = -1;
    __syncthreads();
    if (found != INT_MAX) atomicMin(&entry, found);
    if (positive >= 0) atomicMax(&backup, positive);
    __syncthreads();
    if (tid == 0) {
        const int e = entry != INT_MAX ? entry : backup;
        tokens[m] = e, a.n_tokens[b] = m + 1;
        if (logps) logps[m] = (float)(((double)row[e] - (double)p.top) / (double)temp - log(p.sum));
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
    hipLaunchKernelGGL(k_verify_pick, dim3(p.ns, B), dim3(VF_NT), 0, s, a);
    return hipGetLastError();
}

}  // namespace ts5hip
