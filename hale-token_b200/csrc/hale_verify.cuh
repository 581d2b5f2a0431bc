// hale_verify.cuh -- drafted tokens checked against a target's probabilities.
//
// For a sequence with n drafted tokens x_0 .. x_{n-1}, target logits rows
// 0 .. n and the draft's probabilities q_i, with p_i = softmax(logits_i / T):
//   x_i is kept while u_i q_i(x_i) < p_i(x_i); the first one that is not ends
//   the run and the next token is drawn from max(p_i - q_i, 0) instead; when
//   all are kept it is drawn from p_n.
// Tokens so drawn are distributed as tokens sampled from the target one by
// one. A draw takes the lowest index whose cumulated mass exceeds u times the
// whole. Where the border between two tokens lies depends on sums over the
// vocabulary, so exponentials and sums are formed in 64 bits: 32 would move
// the borders by about 1e-7 of the mass, and with 10^5 of them a draw in a
// thousand would land on a neighbour.
#pragma once

#include <cooperative_groups.h>

#include "hale_kv.cuh"

namespace hale {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyItems = 32;                             // logits a thread holds at a time
constexpr int kVerifyTile = kVerifyThreads * kVerifyItems;   // 8192
constexpr int kVerifyMaxDraft = 64;
constexpr int kVerifyCluster = 8;       // CTAs that draw one sequence's token
constexpr int kPickThreads = 512;
constexpr int kPickTile = 256;          // values of one warp step, 8 a lane
constexpr int kVerifyParts = 1 << 18;   // partial results the workspace holds

// Part of a row: largest value, its lowest index, and sum exp((x - max) / T).
struct VerifyPart {
    double sum;
    float top;
    int arg;
};

struct VerifyArgs {
    const void* logits;
    const float* probs;       // null: the draft gave no probabilities (q = 1 at the drafted token)
    const int32_t *draft, *n_draft;
    const float* u;
    size_t logits_stride, probs_stride;  // elements between rows
    int K, V, slice, slices;  // a row is cut into `slices` of `slice` values
    double per_t;             // 1 / T
    int greedy;
    VerifyPart* parts;        // [batch * (K + 1)][slices]
    int32_t *tokens, *count;
    float* logp;
    uint32_t* err;
};

// exp(x), x <= 0, to about 1e-11: 2^(k/64) from a table and the cubic Taylor
// polynomial on |r| <= ln 2 / 128. tab: 2^(j/64), j < 64. Below -700 it is 0
// (sums are at least 1).
__device__ __forceinline__ double verify_exp(double x, const double* tab) {
    const double k64 = 92.332482616893656877;  // 64 / ln 2
    const double magic = 6755399441055744.0;   // 1.5 * 2^52: the sum's low bits are the rounded integer
    const double t = fmax(x, -700.0) * k64, kd = t + magic;
    const long long k = __double_as_longlong(kd) - __double_as_longlong(magic);
    const double r = (t - (kd - magic)) * (1.0 / k64);
    const double p = __fma_rn(r, __fma_rn(r, __fma_rn(r, 1.0 / 6.0, 0.5), 1.0), 1.0);
    return x >= -700.0 ? __longlong_as_double(__double_as_longlong(p * tab[k & 63]) + ((k >> 6) << 52)) : 0.0;
}

__device__ __forceinline__ void verify_table(double* tab) {
    if (threadIdx.x < 64) tab[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Values i .. i+7 of a row (NaN as -inf), i a multiple of 8; past the end -inf.
template <int DT>
__device__ __forceinline__ void verify_load8(const void* row, int i, int V, bool vec, float (&x)[8]) {
    const float none = -__int_as_float(0x7f800000);
    if (vec && i + 8 <= V) {
        float a[4], b[4];
        load4<DT>(row, i, a);
        load4<DT>(row, i + 4, b);
#pragma unroll
        for (int e = 0; e < 4; e++) { x[e] = a[e]; x[4 + e] = b[e]; }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = i + e < V ? load1<DT>(row, i + e) : none;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = x[e] == x[e] ? x[e] : none;
}

template <int DT>
__device__ __forceinline__ const void* verify_row(const VerifyArgs& a, size_t row) {
    return static_cast<const char*>(a.logits) + row * a.logits_stride * (DT == 0 ? 4 : 2);
}

// One slice of one target row per CTA, read once: 32 values a thread stay in
// registers between the maximum and the sum. Bound by reading the logits; the
// 64-bit arithmetic of a value (9 operations) is issued beside the loads.
template <int DT>
__global__ void __launch_bounds__(kVerifyThreads) verify_stats_kernel(VerifyArgs a) {
    __shared__ double s_tab[64], s_sum[8];
    __shared__ float s_top[8];
    __shared__ int s_arg[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seq = blockIdx.y / (a.K + 1), i = blockIdx.y % (a.K + 1);
    if (a.n_draft && i > max(a.n_draft[seq], 0)) return;
    verify_table(s_tab);
    const void* row = verify_row<DT>(a, blockIdx.y);
    const bool vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
    const int begin = blockIdx.x * a.slice, end = min(a.V, begin + a.slice);
    const float none = -__int_as_float(0x7f800000);
    double sum = 0.0;
    float top = none;
    int arg = INT_MAX;
    for (int t0 = begin; t0 < end; t0 += kVerifyTile) {
        float x[kVerifyItems];
        float m = none;
#pragma unroll
        for (int g = 0; g < kVerifyItems / 8; g++) {
            float y[8];
            verify_load8<DT>(row, t0 + (g * kVerifyThreads + tid) * 8, end, vec, y);
#pragma unroll
            for (int e = 0; e < 8; e++) { x[8 * g + e] = y[e]; m = fmaxf(m, y[e]); }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        __syncthreads();
        if (lane == 0) s_top[warp] = m;
        __syncthreads();
        m = s_top[0];
#pragma unroll
        for (int w = 1; w < 8; w++) m = fmaxf(m, s_top[w]);
        if (a.greedy) {
            if (m > top) {
                int at = INT_MAX;
#pragma unroll
                for (int g = kVerifyItems / 8 - 1; g >= 0; g--)
#pragma unroll
                    for (int e = 7; e >= 0; e--)
                        if (x[8 * g + e] == m) at = t0 + (g * kVerifyThreads + tid) * 8 + e;
                at = __reduce_min_sync(0xffffffffu, at);
                if (lane == 0) s_arg[warp] = at;
                __syncthreads();
                arg = s_arg[0];
#pragma unroll
                for (int w = 1; w < 8; w++) arg = min(arg, s_arg[w]);
                __syncthreads();
            }
        }
        if (m == none) continue;  // nothing in this tile
        if (m > top) {
            if (top > none) sum *= verify_exp(((double)top - (double)m) * a.per_t, s_tab);
            top = m;
        }
        // the value's distance from the maximum, in f64: x / T - top / T
        const double shift = -(double)top * a.per_t;
        double part = 0.0;
#pragma unroll
        for (int e = 0; e < kVerifyItems; e++) {
            // the maximum counts as 1 even when it is infinite
            if (x[e] == top) part += 1.0;
            else if (x[e] > none) part += verify_exp(__fma_rn((double)x[e], a.per_t, shift), s_tab);
        }
        sum += part;
    }
    sum = warp_sum(sum);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        double s = 0.0;
#pragma unroll
        for (int w = 0; w < 8; w++) s += s_sum[w];
        VerifyPart p;
        p.sum = s;
        p.top = top;
        p.arg = arg;
        a.parts[(size_t)blockIdx.y * a.slices + blockIdx.x] = p;
    }
}

// One sequence per cluster of 8 CTAs: every CTA joins the rows' parts and
// makes the same decisions, then takes an eighth of the row that the next
// token is drawn from, notes the mass of each tile of 256 values, and the CTA
// that holds the drawn point searches its tile. The parts of a draw are joined
// through the cluster's shared memory: no workspace, no counters, a fixed
// order of every sum.
// Dynamic shared memory: mass of a CTA's tiles.
template <int DT>
__global__ void __cluster_dims__(kVerifyCluster, 1, 1) __launch_bounds__(kPickThreads)
    verify_pick_kernel(VerifyArgs a) {
    namespace cg = cooperative_groups;
    extern __shared__ double s_mass[];
    __shared__ double s_tab[64], s_total[kVerifyMaxDraft + 1], s_cta;
    __shared__ float s_top[kVerifyMaxDraft + 1];
    __shared__ int s_arg[kVerifyMaxDraft + 1], s_kept[kVerifyMaxDraft + 1];
    __shared__ int s_pick, s_at;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), seq = blockIdx.x / kVerifyCluster;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = kPickThreads / 32;
    const float none = -__int_as_float(0x7f800000);
    int n = a.K;
    if (a.n_draft) {
        n = a.n_draft[seq];
        if (n < 0 || n > a.K) {
            if (tid == 0 && rank == 0) raise_error(a.err, kErrBounds);
            n = min(max(n, 0), a.K);
        }
    }
    verify_table(s_tab);
    __syncthreads();
    const size_t row0 = (size_t)seq * (a.K + 1);
    const int32_t* draft = a.draft + (size_t)seq * a.K;
    const float* u = a.u + row0;
    for (int i = warp; i <= n; i += warps) {
        const VerifyPart* parts = a.parts + (row0 + i) * a.slices;
        float top = none;
        int arg = INT_MAX;
        for (int j = lane; j < a.slices; j += 32) {
            const float t = parts[j].top;
            if (t > top) { top = t; arg = parts[j].arg; }
        }
        float best = top;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
        arg = __reduce_min_sync(0xffffffffu, top == best ? arg : INT_MAX);
        double sum = 0.0;
        for (int j = lane; j < a.slices; j += 32) {
            const VerifyPart p = parts[j];
            if (p.top == best) sum += p.sum;
            else if (p.top > none) sum += p.sum * verify_exp(((double)p.top - (double)best) * a.per_t, s_tab);
        }
        sum = warp_sum(sum);
        if (lane == 0) {
            int kept = 0;
            if (i < n && best > none) {
                const int x = draft[i];
                if (x < 0 || x >= a.V) {
                    raise_error(a.err, kErrBounds);
                } else if (a.greedy) {
                    kept = x == arg;
                } else {
                    const float l = load1<DT>(verify_row<DT>(a, row0 + i), x);
                    const double p = l == best ? 1.0 : (l > none ? exp(((double)l - (double)best) * a.per_t) : 0.0);
                    const double q = a.probs ? (double)a.probs[((size_t)seq * a.K + i) * a.probs_stride + x] : 1.0;
                    kept = (double)u[i] * q < p / sum;
                }
            }
            s_top[i] = best;
            s_arg[i] = arg;
            s_total[i] = best > none ? sum : 0.0;
            s_kept[i] = kept;
        }
    }
    __syncthreads();
    int count = 0;
    while (count < n && s_kept[count]) count++;
    const float top = s_top[count];
    const bool refused = count < n;
    int token = -1;
    if (a.greedy) {
        if (top > none) token = s_arg[count];
    } else if (top > none) {
        // this CTA's share of the row, in tiles of 256 values
        const int tiles = (a.V + kPickTile - 1) / kPickTile;
        const int each = (tiles + kVerifyCluster - 1) / kVerifyCluster;
        const int first = min(tiles, rank * each), here = min(tiles, first + each) - first;
        const void* row = verify_row<DT>(a, row0 + count);
        const bool vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
        const float* q = refused && a.probs ? a.probs + ((size_t)seq * a.K + count) * a.probs_stride : nullptr;
        const bool qvec = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
        const int gone = refused && !a.probs ? draft[count] : -1;
        const double per_total = 1.0 / s_total[count], shift = -(double)top * a.per_t;
        bool rest = refused;  // the draft's probabilities are taken off
        // a lane's eight masses of a tile
        auto masses = [&](int tile, double (&w)[8]) {
            const int i = (first + tile) * kPickTile + 8 * lane;
            float x[8], y[8];
            verify_load8<DT>(row, i, a.V, vec, x);
            const bool off = rest && q;
            if (off) verify_load8<0>(q, i, a.V, qvec, y);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                double p = 0.0;
                if (x[e] == top) p = per_total;
                else if (x[e] > none) p = verify_exp(__fma_rn((double)x[e], a.per_t, shift), s_tab) * per_total;
                if (x[e] == none) p = 0.0;
                if (off && y[e] > none) p = fmax(p - (double)y[e], 0.0);
                if (rest && i + e == gone) p = 0.0;
                w[e] = p;
            }
        };
        double total = 0.0;
        for (int pass = 0; pass < 2; pass++) {
            for (int t = warp; t < here; t += warps) {
                double w[8], s = 0.0;
                masses(t, w);
#pragma unroll
                for (int e = 0; e < 8; e++) s += w[e];
                s = warp_sum(s);
                if (lane == 0) s_mass[t] = s;
            }
            __syncthreads();
            if (warp == 0) {
                double s = 0.0;
                for (int t = lane; t < here; t += 32) s += s_mass[t];
                s = warp_sum(s);
                if (lane == 0) s_cta = s;
            }
            cluster.sync();
            total = 0.0;
            for (int r = 0; r < kVerifyCluster; r++) total += *cluster.map_shared_rank(&s_cta, r);
            cluster.sync();
            // nothing left of p - q (rounding alone): the draw is from p
            if (total > 0.0 || !rest) break;
            rest = false;
        }
        // the CTA, then the tile, then the value where the cumulated mass
        // passes u * total; the last one with mass if rounding leaves none
        const double target = (double)u[a.K] * total;
        double before = 0.0, mine = 0.0;
        int pick = -1;
        for (int r = 0; r < kVerifyCluster; r++) {
            const double s = *cluster.map_shared_rank(&s_cta, r);
            if (s > 0.0) {
                pick = r;
                mine = before;
                if (before + s > target) break;
            }
            before += s;
        }
        cluster.sync();  // shared memory of the others is not read after this
        if (rank != pick) return;
        if (tid == 0) {
            double cum = mine, start = mine;
            int at = 0;
            for (int t = 0; t < here; t++) {
                if (s_mass[t] > 0.0) {
                    at = t;
                    start = cum;
                    if (cum + s_mass[t] > target) break;
                }
                cum += s_mass[t];
            }
            s_at = at;
            s_cta = start;
        }
        __syncthreads();
        if (warp == 0) {
            double w[8], s = 0.0;
            masses(s_at, w);
#pragma unroll
            for (int e = 0; e < 8; e++) s += w[e];
            double cum = s;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, cum, o);
                if (lane >= o) cum += y;
            }
            cum += s_cta - s;
            int found = INT_MAX, last = -1;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int i = (first + s_at) * kPickTile + 8 * lane + e;
                if (w[e] > 0.0) {
                    last = i;
                    if (found == INT_MAX && cum + w[e] > target) found = i;
                }
                cum += w[e];
            }
            found = __reduce_min_sync(0xffffffffu, found);
            last = __reduce_max_sync(0xffffffffu, last);
            if (lane == 0) s_pick = found == INT_MAX ? last : found;
        }
        __syncthreads();
        token = s_pick;
    }
    if (a.greedy || !(top > none)) {
        if (rank != 0) return;
    }
    // the kept tokens, the drawn one, -1 behind it
    for (int i = tid; i <= a.K; i += kPickThreads) {
        const int x = i < count ? draft[i] : (i == count ? token : -1);
        a.tokens[row0 + i] = x;
        if (a.logp) {
            float lp = 0.0f;
            if (x >= 0) {
                const float l = load1<DT>(verify_row<DT>(a, row0 + i), x);
                const double d = l == s_top[i] ? 0.0 : ((double)l - (double)s_top[i]) * a.per_t;
                lp = (float)(d - log(s_total[i]));
            }
            a.logp[row0 + i] = lp;
        }
    }
    if (tid == 0) a.count[seq] = count + (token >= 0);
}

}  // namespace hale
