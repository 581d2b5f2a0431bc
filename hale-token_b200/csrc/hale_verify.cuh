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
// vocabulary, so the row that is drawn from is summed in 64 bits: 32 would move
// its borders by about 1e-8 of the mass, and with 10^5 of them one draw in a
// thousand would land on a neighbour. The other rows only decide u q < p, a
// single border, for which exponentials in 32 bits do (2^-21 of p at most).
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

// The logit 600 T below a row's largest: what lies below it counts as that far
// below (1e-261, nothing next to a sum of at least 1).
__device__ __forceinline__ float verify_floor(float top, double per_t) {
    return fmaxf((float)((double)top - 600.0 / per_t), -0x1.fffffep127f);
}

// Weights exp((x - top) / T) of a row to about 1e-12: 2^(k/32) from a table and
// the Taylor polynomial to r^4 on |r| <= ln 2 / 64. With t = 32 (x - top) / (T
// ln 2) formed by one multiply-add, its rounded integer k falls out of the low
// bits of t + 1.5 2^52.
struct VerifyScale {
    double a, b;
    float floor;

    __device__ __forceinline__ VerifyScale(float top, double per_t) {
        a = per_t * 46.166241308446828384;  // 32 / ln 2
        b = -(double)top * a;
        floor = verify_floor(top, per_t);
    }
    // tab: 2^(j/32), j < 32. x at most the finite largest.
    __device__ __forceinline__ double weight(float x, const uint64_t* tab) const {
        const double magic = 6755399441055744.0;
        const double t = __fma_rn((double)fmaxf(x, floor), a, b), kd = t + magic, r = t - (kd - magic);
        const int k = __double2loint(kd);
        // Taylor's coefficients of exp(r ln 2 / 32)
        const double c1 = 0.021660849392498290192, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4;
        const double p = __fma_rn(r, __fma_rn(r, __fma_rn(r, __fma_rn(r, c4, c3), c2), c1), 1.0) *
                         __longlong_as_double((long long)tab[k & 31]);
        return __hiloint2double(__double2hiint(p) + ((k >> 5) << 20), __double2loint(p));
    }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int DT>
__device__ __forceinline__ const void* verify_row(const VerifyArgs& a, size_t row) {
    return static_cast<const char*>(a.logits) + row * a.logits_stride * (DT == 0 ? 4 : 2);
}

// Eight values of a row as they are stored, NaN and values past the end as
// -inf when they are taken out.
template <int DT>
struct VerifyRaw {
    uint4 v[DT == 0 ? 2 : 1];

    __device__ __forceinline__ void load(const void* row, int i, int end, bool vec) {
        if (vec && i + 8 <= end) {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(row) + (size_t)i * (DT == 0 ? 4 : 2));
#pragma unroll
            for (int j = 0; j < (DT == 0 ? 2 : 1); j++) v[j] = __ldg(p + j);
            return;
        }
        const uint32_t none = DT == 0 ? 0xff800000u : (DT == 1 ? 0xfc00u : 0xff80u);
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            w[e] = none;
            if (i + e < end)
                w[e] = DT == 0 ? reinterpret_cast<const uint32_t*>(row)[i + e] : reinterpret_cast<const uint16_t*>(row)[i + e];
        }
        if (DT == 0) {
            v[0] = make_uint4(w[0], w[1], w[2], w[3]);
            v[DT == 0 ? 1 : 0] = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
            v[0] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
        }
    }
    __device__ __forceinline__ float at(int e) const {
        const uint4 q = v[DT == 0 ? e / 4 : 0];
        const int k = DT == 0 ? e % 4 : e / 2;
        const uint32_t w = k == 0 ? q.x : k == 1 ? q.y : k == 2 ? q.z : q.w;
        const float x = DT == 0 ? __uint_as_float(w)
                      : DT == 1 ? half_bits_to_float((uint16_t)(e & 1 ? w >> 16 : w))
                                : __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
        return x == x ? x : -__int_as_float(0x7f800000);
    }
};

// One slice of one target row per CTA, read once: a thread keeps 32 values as
// they are stored, takes their maximum and then the sum of 32 exponentials in
// 32 bits; threads are joined at the end alone (sums in 64 bits). (x - top) /
// (T ln 2) is formed with both halves of the factor, so that far values are
// not all off in one direction. Bound by reading the logits.
template <int DT>
__global__ void __launch_bounds__(kVerifyThreads, DT == 0 ? 4 : 5) verify_stats_kernel(VerifyArgs a) {
    __shared__ double s_sum[8];
    __shared__ float s_top[8];
    __shared__ int s_arg[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seq = blockIdx.y / (a.K + 1), i = blockIdx.y % (a.K + 1);
    const void* row = verify_row<DT>(a, blockIdx.y);
    const bool vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
    const int begin = blockIdx.x * a.slice, end = min(a.V, begin + a.slice);
    const float none = -__int_as_float(0x7f800000), inf = __int_as_float(0x7f800000);
    if (a.n_draft && i > max(a.n_draft[seq], 0)) return;
    const double factor = a.per_t * 1.4426950408889634074;  // 1 / (T ln 2)
    const float hi = (float)factor, lo = (float)(factor - (double)hi), far = (float)fmin(600.0 / a.per_t, 1e38);
    float top = none;
    double sum = 0.0;
    int arg = INT_MAX;
    for (int t0 = begin; t0 < end; t0 += kVerifyTile) {
        VerifyRaw<DT> x[kVerifyItems / 8];
#pragma unroll
        for (int g = 0; g < kVerifyItems / 8; g++) x[g].load(row, t0 + (g * kVerifyThreads + tid) * 8, end, vec);
        float m = none;
#pragma unroll
        for (int g = 0; g < kVerifyItems / 8; g++)
#pragma unroll
            for (int e = 0; e < 8; e++) m = fmaxf(m, x[g].at(e));
        if (m == none) continue;
        if (m > top) {
            if (a.greedy) {
#pragma unroll
                for (int g = kVerifyItems / 8 - 1; g >= 0; g--)
#pragma unroll
                    for (int e = 7; e >= 0; e--)
                        if (x[g].at(e) == m) arg = t0 + (g * kVerifyThreads + tid) * 8 + e;
            }
            if (top > none) sum = m < inf ? sum * exp(((double)top - (double)m) * a.per_t) : 0.0;
            top = m;
        }
        float part = 0.0f;
        if (top < inf) {
            const float floor = fmaxf(top - far, -0x1.fffffep127f);
#pragma unroll
            for (int g = 0; g < kVerifyItems / 8; g++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float d = fmaxf(x[g].at(e), floor) - top;
                    part += exp2_fast(fmaf(d, hi, d * lo));
                }
        } else {  // infinite logits share everything
#pragma unroll
            for (int g = 0; g < kVerifyItems / 8; g++)
#pragma unroll
                for (int e = 0; e < 8; e++) part += x[g].at(e) == top ? 1.0f : 0.0f;
        }
        sum += (double)part;
    }
    // threads, then warps: the largest, its lowest place, the sums scaled to it
    auto join = [&](float best, float t, double s) {
        if (t == best) return s;
        return t > none && best < inf ? s * exp(((double)t - (double)best) * a.per_t) : 0.0;
    };
    float best = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    sum = warp_sum(join(best, top, sum));
    arg = __reduce_min_sync(0xffffffffu, top == best ? arg : INT_MAX);
    if (lane == 0) {
        s_top[warp] = best;
        s_sum[warp] = sum;
        s_arg[warp] = arg;
    }
    __syncthreads();
    if (warp == 0) {
        const float t = lane < 8 ? s_top[lane] : none;
        best = t;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
        double s = lane < 8 ? join(best, t, s_sum[lane]) : 0.0;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        arg = __reduce_min_sync(0xffffffffu, lane < 8 && t == best ? s_arg[lane] : INT_MAX);
        if (lane == 0) a.parts[(size_t)blockIdx.y * a.slices + blockIdx.x] = {s, best, arg};
    }
}

// One sequence per cluster of CTAs (8, fewer in large batches, so that all are
// there at once): every CTA joins the rows' parts and makes the same decisions,
// then takes its share of the row that the next token is drawn from, notes the
// mass of each tile of 256 values, and the CTA that holds the drawn point
// searches its tile. Against a draft's probabilities the row's sum is formed
// first, in 64 bits. The parts of a draw are joined through the cluster's
// shared memory: no workspace, no counters, a fixed order of every sum.
// Dynamic shared memory: mass of a CTA's tiles.
template <int DT>
__global__ void __launch_bounds__(kPickThreads, 2) verify_pick_kernel(VerifyArgs a) {
    namespace cg = cooperative_groups;
    extern __shared__ double s_mass[];
    __shared__ uint64_t s_tab[32];
    __shared__ double s_total[kVerifyMaxDraft + 1], s_cta;
    __shared__ float s_top[kVerifyMaxDraft + 1];
    __shared__ int s_arg[kVerifyMaxDraft + 1], s_kept[kVerifyMaxDraft + 1];
    __shared__ int s_pick, s_at;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), seq = blockIdx.x / ctas;
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
    if (tid < 32) s_tab[tid] = kExp2TabDev[tid];
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
            else if (p.top > none) sum += p.sum * exp(((double)p.top - (double)best) * a.per_t);
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
        const int each = (tiles + ctas - 1) / ctas;
        const int first = min(tiles, rank * each), here = min(tiles, first + each) - first;
        const void* row = verify_row<DT>(a, row0 + count);
        const bool vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
        const float* q = refused && a.probs ? a.probs + ((size_t)seq * a.K + count) * a.probs_stride : nullptr;
        const bool qvec = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
        const int gone = refused && !a.probs ? draft[count] : -1;
        double per_total = 1.0 / s_total[count];
        const bool certain = top == __int_as_float(0x7f800000);  // infinite logits share everything
        const VerifyScale f(certain ? 0.0f : top, a.per_t);
        bool rest = refused;  // the draft's probabilities are taken off
        // What this CTA's tiles hold, by phase: 0 the row's sum (p - q needs
        // it exactly), 1 the masses that are drawn from, 2 the drawn tile again.
        // One loop for all of them: the code is fetched once.
        int phase = rest && q ? 0 : 1;
        double w[8], total = 0.0, target = 0.0, before = 0.0;
        for (;;) {
            if (phase == 0) per_total = 1.0;
            const bool minus = rest && phase > 0;
            const int t1 = phase == 2 ? s_at + 1 : here;
            // a lane's eight values, the next tile's under way
            VerifyRaw<DT> x, x_next;
            VerifyRaw<0> y, y_next;
            auto fetch = [&](int t) {
                if (t >= t1) return;
                const int i = (first + t) * kPickTile + 8 * lane;
                x_next.load(row, i, a.V, vec);
                if (minus && q) y_next.load(q, i, a.V, qvec);
            };
            y_next.v[0] = y_next.v[1] = make_uint4(0, 0, 0, 0);
            fetch(phase == 2 ? s_at : warp);
            for (int t = phase == 2 ? s_at : warp; t < t1; t += warps) {
                x = x_next;
                y = y_next;
                fetch(t + warps);
                const int i = (first + t) * kPickTile + 8 * lane;
                double s = 0.0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    double p = certain ? (x.at(e) == top ? 1.0 : 0.0) : f.weight(x.at(e), s_tab);
                    // p - q, and nothing below 0, for a masked logit or (lookup drafts) the refused token
                    p = __fma_rn(p, per_total, -(double)fmaxf(y.at(e), 0.0f));
                    w[e] = p > 0.0 && x.at(e) > none && !(minus && i + e == gone) ? p : 0.0;
                    s += w[e];
                }
                if (phase < 2) {
                    s = warp_sum(s);
                    if (lane == 0) s_mass[t] = s;
                }
            }
            if (phase == 2) break;
            __syncthreads();
            if (warp == 0) {
                double s = 0.0;
                for (int t = lane; t < here; t += 32) s += s_mass[t];
                s = warp_sum(s);
                if (lane == 0) s_cta = s;
            }
            cluster.sync();
            total = 0.0;
            for (int r = 0; r < ctas; r++) total += *cluster.map_shared_rank(&s_cta, r);
            if (phase == 0 || (rest && !(total > 0.0))) {
                if (phase == 0) per_total = 1.0 / total;
                else rest = false;  // nothing left of p - q: the draw is from p
                phase = 1;
                cluster.sync();  // before s_cta is written again
                continue;
            }
            // the CTA, then the tile, then the value where the cumulated mass
            // passes u * total; the last one with mass if rounding leaves none
            target = (double)u[a.K] * total;
            int pick = -1;
            double sum = 0.0;
            for (int r = 0; r < ctas; r++) {
                const double s = *cluster.map_shared_rank(&s_cta, r);
                if (s > 0.0) {
                    pick = r;
                    before = sum;
                    if (sum + s > target) break;
                }
                sum += s;
            }
            cluster.sync();  // shared memory of the others is not read after this
            if (rank != pick) return;
            if (warp == 0) {
                int at = -1, last = 0;
                double base = before;
                for (int t0 = 0; t0 < here && at < 0; t0 += 32) {
                    const double mass = t0 + lane < here ? s_mass[t0 + lane] : 0.0;
                    double cum = mass;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double z = __shfl_up_sync(0xffffffffu, cum, o);
                        if (lane >= o) cum += z;
                    }
                    cum += base;
                    const unsigned hit = __ballot_sync(0xffffffffu, mass > 0.0 && cum > target);
                    const unsigned some = __ballot_sync(0xffffffffu, mass > 0.0);
                    if (hit | some) {
                        const int pick_lane = hit ? __ffs(hit) - 1 : 31 - __clz(some);
                        last = t0 + pick_lane;
                        before = __shfl_sync(0xffffffffu, cum - mass, pick_lane);
                        if (hit) at = last;
                    }
                    base = __shfl_sync(0xffffffffu, cum, 31);
                }
                if (lane == 0) s_at = last;
            }
            __syncthreads();
            phase = 2;
        }
        if (warp == 0) {
            double s = 0.0;
#pragma unroll
            for (int e = 0; e < 8; e++) s += w[e];
            double cum = s;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double z = __shfl_up_sync(0xffffffffu, cum, o);
                if (lane >= o) cum += z;
            }
            cum += before - s;
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
