// hale_kv_attn.cuh -- attention over the paged 8-bit cache (hale_kv.cuh).
//
// Row r of a sequence at position p, query head h over kv head h / group:
//   s_t = scale * ks_b(t) * sum_d q_d kc_td,   t = max(0, p - window + 1) .. p
//   out = sum_t softmax(s)_t vs_b(t) vc_t,     lse = log sum_t exp(s_t)
// with int8 codes kc, vc and one scale per block b of 16 tokens. The scales
// multiply whole scores and whole softmax weights, so the products run on the
// codes themselves.
//   - q is scaled by a power of two and rounded to an integer below 2^23, held
//     as three int8 digits in base 256 (off by at most 2^-23 of the row's
//     largest value, an f32's own last place there): q . kc is three int8
//     matrix products, exact in 32-bit integers.
//   - a softmax weight times its block's value scale, over the largest such
//     scale so far and times 2^14, is rounded to f16 (11 bits, the accuracy of
//     the result's own type or better); for f32 results to two f16 (22 bits).
// Maxima, sums and outputs are kept in 32 bits.
//
// Work is cut along rows, heads and the token axis alike. A segment is up to
// `rows` consecutive rows of one sequence; a tile is a segment with one kv
// head (its rows and the head's query heads are the tile's columns); a unit is
// one chunk of the tile's tokens. The units of all tiles, in order, are dealt
// out evenly: CTA c of G takes units [c W / G, (c + 1) W / G). A tile that
// falls into several CTAs is joined by the last of them to finish, in CTA
// order, so results do not depend on timing. Lengths are read on the device:
// nothing of this is known when the kernel is launched.
#pragma once

#include <type_traits>

#include "hale_kv.cuh"

namespace hale {

struct KvAttn {
    const void* q;
    void* out;
    float* lse;
    const int32_t *seqs, *positions;
    size_t q_stride, out_stride;
    int n, nh, group, window;
    int rows;      // most rows of a segment
    int heads;     // query heads of a tile (group, or a part of a very large one)
    int subs;      // tiles a kv head's group is cut into
    float scale;
    float* parts;        // [2 * gridDim][part_floats]
    int part_floats;
    unsigned* arrived;   // [gridDim], zero between calls
};

// Workspace of split tiles.
constexpr size_t kAttnPartBytes = (size_t)40 << 20;
constexpr int kAttnMaxGrid = 1024;

struct KvSegment {
    int row, rows, seq;
    int lo, hi;      // tokens any of its rows sees: [lo, hi)
    int c0, units;   // first chunk and number of chunks
};

// One past the last token row i sees, 0 for a row that sees nothing.
__device__ __forceinline__ int kv_row_end(const KvArgs& c, const KvAttn& a, int i, int seq) {
    const int p = a.positions[i];
    if (p < 0) return 0;
    if (seq >= c.n_seqs || p >= c.capacity()) {
        raise_error(c.err, kErrBounds);
        return 0;
    }
    return p + 1;
}

// The segment that starts at row i, if one does (else rows = 0). Rows of a
// negative sequence belong to none.
template <int CH>
__device__ __forceinline__ KvSegment kv_segment(const KvArgs& c, const KvAttn& a, int i) {
    KvSegment s;
    s.row = i;
    s.rows = 0;
    s.units = 0;
    s.seq = a.seqs ? a.seqs[i] : 0;
    if (s.seq < 0) return s;
    if (i % a.rows && (!a.seqs || a.seqs[i - 1] == s.seq)) return s;
    s.lo = INT_MAX;
    s.hi = 0;
    const int last = min(a.n, i - i % a.rows + a.rows);
    for (int j = i; j < last && (j == i || !a.seqs || a.seqs[j] == s.seq); j++) {
        const int end = kv_row_end(c, a, j, s.seq);
        s.hi = max(s.hi, end);
        if (end > 0) s.lo = min(s.lo, a.window > 0 ? max(0, end - a.window) : 0);
        s.rows++;
    }
    if (s.hi == 0) s.lo = 0;
    s.c0 = s.lo / CH;
    // a segment that sees nothing is still one unit: its rows are written
    s.units = max(1, (s.hi + CH - 1) / CH - s.c0);
    return s;
}

// The units a CTA owns, walked segment by segment.
template <int CH, int THREADS>
struct KvWalk {
    long long total, begin, end;  // units of all tiles; this CTA's
    int grid;                     // CTAs that have units
    long long base;               // units before the current segment
    KvSegment seg;

    __device__ __forceinline__ int owner(long long unit) const { return (int)(((unit + 1) * grid - 1) / total); }

    // All threads. False: nothing to do.
    __device__ bool start(const KvArgs& c, const KvAttn& a, KvSegment* s_seg, long long* s_sum) {
        constexpr int W = THREADS / 32;
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        const int tiles = c.nkv * a.subs;
        const int strip = (a.n + THREADS - 1) / THREADS, i0 = tid * strip, i1 = min(a.n, i0 + strip);
        long long mine = 0;
        KvSegment first;
        first.rows = 0;
        for (int i = i0; i < i1; i++) {
            const KvSegment s = kv_segment<CH>(c, a, i);
            if (s.rows) mine += (long long)s.units * tiles;
            if (s.rows && !first.rows) first = s;
        }
        long long x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) s_sum[warp] = x;
        __syncthreads();
        total = 0;
        long long before = 0;
#pragma unroll
        for (int w = 0; w < W; w++) {
            if (w < warp) before += s_sum[w];
            total += s_sum[w];
        }
        grid = (int)min((long long)gridDim.x, total);
        if ((int)blockIdx.x >= grid) return false;
        begin = total * blockIdx.x / grid;
        end = total * (blockIdx.x + 1) / grid;
        before += x - mine;
        if (begin >= before && begin < before + mine) {
            // this thread's strip holds the first unit
            for (int i = first.row;; i++) {
                const KvSegment s = i == first.row ? first : kv_segment<CH>(c, a, i);
                if (!s.rows) continue;
                const long long u = (long long)s.units * tiles;
                if (begin < before + u) {
                    *s_seg = s;
                    s_sum[W] = before;
                    break;
                }
                before += u;
            }
        }
        __syncthreads();
        seg = *s_seg;
        base = s_sum[W];
        return true;
    }

    // The next segment with units (there is one while base < end).
    __device__ void next(const KvArgs& c, const KvAttn& a) {
        base += (long long)seg.units * c.nkv * a.subs;
        int i = seg.row + seg.rows;
        while (i < a.n) {
            seg = kv_segment<CH>(c, a, i);
            if (seg.rows) return;
            i++;
        }
    }
};

// One CTA per (row, query head), four warps on alternating tokens, lanes over
// the head's dims; each warp keeps the running maximum, sum and weighted sum
// of a softmax in f32, joined at the end.
template <int DT>
__global__ void __launch_bounds__(128) kv_attention_kernel(KvArgs c, KvAttn a) {
    __shared__ float s_m[4], s_l[4], s_o[4][256];
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int seq = a.seqs ? a.seqs[row] : 0, head = h / a.group;
    if (seq < 0) return;
    int end = a.positions[row] + 1;
    if (seq >= c.n_seqs || end > c.capacity()) {
        if (threadIdx.x == 0) raise_error(c.err, kErrBounds);
        end = 0;
    }
    const int begin = a.window > 0 ? max(0, end - a.window) : 0;
    float q[8], o[8], m = -__int_as_float(0x7f800000), l = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int d = lane + 32 * i;
        q[i] = d < c.hd ? load1<DT>(a.q, (size_t)row * a.q_stride + (size_t)h * c.hd + d) : 0.0f;
        o[i] = 0.0f;
    }
    for (int t = begin + warp; t < end; t += 4) {
        const int page = c.page_of(c.table, seq, t), slot = c.slot(t);
        if (page < 0) {
            raise_error(c.err, kErrBounds);
            continue;
        }
        const size_t at = c.code_at(page, head, slot), sa = c.scale_at(page, head, slot);
        float s = 0.0f, v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = lane + 32 * i;
            const bool in = d < c.hd;
            s = fmaf(q[i], in ? (float)c.k[at + d] : 0.0f, s);
            v[i] = in ? (float)c.v[at + d] : 0.0f;
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= c.ks[sa] * a.scale;
        const float top = fmaxf(m, s), fix = expf(m - top), p = expf(s - top), f = p * c.vs[sa];
        l = l * fix + p;
        m = top;
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = fmaf(f, v[i], o[i] * fix);
    }
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int i = 0; i < 8; i++) s_o[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])), sum = 0.0f, f[4];
    const bool empty = !(top > -__int_as_float(0x7f800000)) && top == top;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        f[w] = empty || s_l[w] == 0.0f ? 0.0f : expf(s_m[w] - top);
        sum += f[w] * s_l[w];
    }
    for (int d = threadIdx.x; d < c.hd; d += 128) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) x += f[w] * s_o[w][d];
        store1<DT>(a.out, (size_t)row * a.out_stride + (size_t)h * c.hd + d, empty ? 0.0f : x / sum);
    }
    if (threadIdx.x == 0 && a.lse) a.lse[(size_t)row * a.nh + h] = empty ? -__int_as_float(0x7f800000) : top + logf(sum);
}

// ---------------------------------------------------------------------------
// small matrix pieces
// ---------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Bytes 0 and 2 (int8) of w as a pair of f16: 1024 + (byte ^ 0x80) is a f16
// whose low bits are the byte; 1152 is taken off again.
__device__ __forceinline__ uint32_t codes_even(uint32_t w) {
    const uint32_t x = (w & 0x00ff00ffu) ^ 0x64806480u, off = 0x64806480u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&off));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t codes_odd(uint32_t w) { return codes_even(w >> 8); }

// 16 (or 8) bytes that no one else will read again soon.
__device__ __forceinline__ uint4 load_stream16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load_stream8(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

constexpr float kWeightTop = 16384.0f;  // the largest weight as f16
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// Power of two that brings amax below 2^22.99 and to at least 2^21.99 (1 for 0
// and for values that are not finite).
__device__ __forceinline__ float kv_query_scale(float amax) {
    if (!(amax > 0.0f) || !(amax <= 0x1.fffffep127f)) return 1.0f;
    int e;
    const float f = frexpf(amax, &e);  // amax = f 2^e, f in [1/2, 1)
    // the digits reach 127 * 65793 < 2^23: f must stay below 0.996
    return ldexpf(1.0f, min(126, max(-126, (f < 0.99f ? 23 : 22) - e)));
}

// Four values as one register of each of the three digits of their integers:
// x = d0 65536 + d1 256 + d2, d1 and d2 in [-128, 127].
__device__ __forceinline__ void kv_query_digits(const float (&x)[4], uint32_t (&d)[3]) {
    d[0] = d[1] = d[2] = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int n = __float2int_rn(x[i]);
        const int lo = (int8_t)n, n1 = (n - lo) >> 8, mid = (int8_t)n1, hi = (n1 - mid) >> 8;
        d[0] |= (uint32_t)(hi & 0xff) << (8 * i);
        d[1] |= (uint32_t)(mid & 0xff) << (8 * i);
        d[2] |= (uint32_t)(lo & 0xff) << (8 * i);
    }
}

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------------------
// few columns: tokens x columns products fed from registers
//
// Four warps, each on its own 16 NB tokens of a unit. Keys: a lane loads 16
// consecutive dims of a token, which are (after a permutation of the dims that
// the query's fragment repeats) B fragments of 32 dims x 8 tokens as they
// stand: nothing between HBM and the tensor core. The A fragment's rows 0-7
// hold the columns' highest digits and rows 8-15 the middle ones, so a lane
// receives both sums of one column's score; a second product adds the lowest.
// The scores lie so that the weights are the B fragment of O^T = V^T P^T, an
// f16 product (weights span many orders of magnitude, which integers would cut
// off); V's A fragments are again bytes of a lane's own loads (four tokens,
// DP / 8 consecutive dims), paired by byte permutes and widened to f16.
// Every load is made, hidden tokens and dims past the head's included (at an
// address that is there): codes are finite whatever they are, and a hidden
// token's weight, like a missing dim of q, is 0.
constexpr int kFewWarps = 4, kFewThreads = 32 * kFewWarps;

template <int DP>
struct FewCfg {
    static constexpr int NB = DP <= 128 ? 2 : 1;         // blocks of 16 tokens a warp takes at a time
    static constexpr int TB = 16 * NB, CH = TB * kFewWarps;
    static constexpr int KC = DP / 64;                   // 64-dim pieces of a key row
    static constexpr int VW = DP / 32;                   // 32-bit words of a lane's dims of one value row
};

// HD: the head's dims where they are known (= DP), else 0.
template <int DT, int DP, int HD, int NT>
__global__ void __launch_bounds__(kFewThreads, DP <= 128 && NT == 1 ? 3 : 2) kv_attn_few_kernel(KvArgs c, KvAttn a) {
    using Cfg = FewCfg<DP>;
    constexpr int NB = Cfg::NB, CH = Cfg::CH, KC = Cfg::KC, VW = Cfg::VW, MT = DP / 16, COLS = 8 * NT;
    constexpr int SPLIT = DT == 0 ? 2 : 1;
    __shared__ KvSegment s_seg;
    __shared__ long long s_sum[kFewWarps + 1];
    __shared__ float s_m[kFewWarps][COLS], s_l[kFewWarps][COLS], s_f[COLS], s_inv[COLS];
    __shared__ int s_last;
    extern __shared__ __align__(16) float s_acc[];  // [kFewWarps][COLS][DP]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
    const int hd = HD ? HD : c.hd;
    const float none = -__int_as_float(0x7f800000);

    KvWalk<CH, kFewThreads> walk;
    if (!walk.start(c, a, &s_seg, s_sum)) return;
    long long unit = walk.begin;
    while (unit < walk.end) {
        while (unit >= walk.base + (long long)walk.seg.units * c.nkv * a.subs) walk.next(c, a);
        const KvSegment seg = walk.seg;
        const int tile = (int)((unit - walk.base) / seg.units), head = tile / a.subs, sub = tile % a.subs;
        const long long tile0 = walk.base + (long long)tile * seg.units, tile1 = tile0 + seg.units;
        const int u0 = seg.c0 + (int)(unit - tile0), u1 = seg.c0 + (int)(min(tile1, walk.end) - tile0);
        const int heads = min(a.heads, a.group - sub * a.heads), cols = seg.rows * heads;
        const int h0 = head * a.group + sub * a.heads;  // the tile's first query head

        // ---- the columns' queries, as B fragments, and what they see ----
        // (the integer product's k index runs over 16 t + 4 q4 + byte of a
        // 32-dim step: words 0, 1 and 2, 3 of a lane's 16 dims)
        uint32_t qf[3][NT][KC * 2][2];
        float qs[NT];
        int end[NT], begin[NT];
        int all_lo = 0, all_hi = INT_MAX;  // tokens every column sees
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int col = nt * 8 + g;
            const bool in = col < cols;
            const size_t at = in ? (size_t)(seg.row + col / heads) * a.q_stride + (size_t)(h0 + col % heads) * hd : 0;
            float x[KC][4][4];
            float amax = 0.0f;
#pragma unroll
            for (int p = 0; p < KC; p++) {
                const int d = 64 * p + 16 * q4;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    x[p][w][0] = x[p][w][1] = x[p][w][2] = x[p][w][3] = 0.0f;
                    if (in && d < hd) load4<DT>(a.q, at + d + 4 * w, x[p][w]);
#pragma unroll
                    for (int i = 0; i < 4; i++) amax = fmaxf(amax, fabsf(x[p][w][i]));
                }
            }
            bool wild = false;  // infinities and NaN have no digits
#pragma unroll
            for (int p = 0; p < KC; p++)
#pragma unroll
                for (int w = 0; w < 4; w++)
#pragma unroll
                    for (int i = 0; i < 4; i++) wild |= !(fabsf(x[p][w][i]) <= 0x1.fffffep127f);
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const unsigned wilds = __ballot_sync(0xffffffffu, wild);
            float up = kv_query_scale(amax);
#pragma unroll
            for (int p = 0; p < KC; p++)
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    uint32_t d[3];
#pragma unroll
                    for (int i = 0; i < 4; i++) x[p][w][i] *= up;
                    kv_query_digits(x[p][w], d);
#pragma unroll
                    for (int z = 0; z < 3; z++) qf[z][nt][2 * p + (w >> 1)][w & 1] = d[z];
                }
            if (wilds >> (4 * g) & 15u) up = __int_as_float(0x7fc00000);  // the column's scores become NaN
            qs[nt] = a.scale * kLog2e / up;
            end[nt] = begin[nt] = 0;
            if (in) {
                const int p = a.positions[seg.row + col / heads];
                end[nt] = p >= 0 && p < seg.hi ? p + 1 : 0;
                begin[nt] = a.window > 0 ? max(0, end[nt] - a.window) : 0;
                all_hi = min(all_hi, end[nt]);
                all_lo = max(all_lo, begin[nt]);
            }
        }
        all_hi = __reduce_min_sync(0xffffffffu, all_hi);
        all_lo = __reduce_max_sync(0xffffffffu, all_lo);

        float acc[MT][NT][4], m[NT], l[NT];
        float vtop = 0.0f, vinv = 0.0f;  // largest value scale so far, 2^14 over it
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt] = none;
            l[nt] = 0.0f;
#pragma unroll
            for (int i = 0; i < MT; i++) acc[i][nt][0] = acc[i][nt][1] = acc[i][nt][2] = acc[i][nt][3] = 0.0f;
        }
        const int32_t* row = c.table + (size_t)min(seg.seq, c.n_seqs - 1) * c.max_pages;
        // a page's codes and scales (at most 2^26 bytes), and this lane's place in a block
        const unsigned page_codes = (unsigned)(c.nkv * hd) << c.page_log2, page_scales = (unsigned)c.nkv << c.page_log2 >> 4;
        const int8_t* kbase = c.k + ((size_t)head << c.page_log2) * hd + (unsigned)(g * hd) + (HD ? 16 * q4 : 0);
        const int8_t* vbase = c.v + ((size_t)head << c.page_log2) * hd + (unsigned)(2 * q4 * hd) + (HD ? 4 * VW * g : 0);
        const float* ksbase = c.ks + ((size_t)head << c.page_log2 >> 4);
        const float* vsbase = c.vs + ((size_t)head << c.page_log2 >> 4);

        // ---- tokens ----
        uint4 kr[NB][2][KC];          // tokens g and g + 8 of each block
        uint32_t vr[NB][4][VW];       // tokens 2 q4, + 1, + 8, + 9
        float ks[NB], vs[NB], ks_next[NB], vs_next[NB];
        int page[NB], page_next[NB];
        // page of each block of unit u, -1: nothing of it is seen, or it is missing
        auto find = [&](int u, int (&pg)[NB]) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int t = u * CH + warp * Cfg::TB + 16 * b;
                pg[b] = -1;
                if (u < u1 && t < seg.hi && t + 16 > seg.lo) {
                    pg[b] = c.checked(row[t >> c.page_log2]);
                    if (pg[b] < 0 && lane == 0) raise_error(c.err, kErrBounds);
                }
            }
        };
        auto load_k = [&](int u, const int (&pg)[NB], float (&fk)[NB], float (&fv)[NB]) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int slot = c.slot(u * CH + warp * Cfg::TB + 16 * b);
                const unsigned pn = (unsigned)max(pg[b], 0);
                fk[b] = ksbase[(size_t)pn * page_scales + (slot >> 4)];
                fv[b] = vsbase[(size_t)pn * page_scales + (slot >> 4)];
                if (pg[b] < 0) fk[b] = fv[b] = 0.0f;
                const int8_t* src = kbase + (size_t)pn * page_codes + (unsigned)(slot * hd);
#pragma unroll
                for (int p = 0; p < KC; p++) {
                    const int d = HD ? 64 * p : min(64 * p + 16 * q4, hd - 16);
                    kr[b][0][p] = load_stream16(src + d);
                    kr[b][1][p] = load_stream16(src + 8 * hd + d);
                }
            }
        };
        auto load_v = [&](int u, const int (&pg)[NB]) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const int slot = c.slot(u * CH + warp * Cfg::TB + 16 * b);
                const int8_t* src = vbase + (size_t)(unsigned)max(pg[b], 0) * page_codes + (unsigned)(slot * hd);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int8_t* p = src + ((j & 1) + 8 * (j >> 1)) * hd;
                    if (VW == 2) {
                        const uint2 v = load_stream8(p);
                        vr[b][j][0] = v.x;
                        vr[b][j][1] = v.y;
                    } else {
#pragma unroll
                        for (int w = 0; w + 4 <= VW; w += 4) {
                            const uint4 v = load_stream16(p + (HD ? 4 * w : min(4 * VW * g + 4 * w, hd - 16)));
                            vr[b][j][w] = v.x;
                            vr[b][j][w + 1] = v.y;
                            vr[b][j][w + 2] = v.z;
                            vr[b][j][w + 3] = v.w;
                        }
                    }
                }
            }
        };
        find(u0, page);
        load_k(u0, page, ks, vs);
        load_v(u0, page);
        find(u0 + 1, page_next);
        // One step over the warp's tokens of unit u; WHOLE: every column sees
        // all of them and every page is there.
        auto step = [&](int u, auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            const int t0 = u * CH + warp * Cfg::TB;
            const bool more = u + 1 < u1;
            // q . kc, integers of at most 2^45, rounded to f32; [token half][token]
            float s[NB][NT][4];
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    int z[NT][4], lo[(NT + 1) / 2][4];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) z[nt][0] = z[nt][1] = z[nt][2] = z[nt][3] = 0;
#pragma unroll
                    for (int i = 0; i < (NT + 1) / 2; i++) lo[i][0] = lo[i][1] = lo[i][2] = lo[i][3] = 0;
#pragma unroll
                    for (int p = 0; p < KC; p++) {
                        const uint4 x = kr[b][j][p];
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            mma_s8(z[nt], qf[0][nt][2 * p][0], qf[1][nt][2 * p][0], qf[0][nt][2 * p][1], qf[1][nt][2 * p][1],
                                   x.x, x.y);
                            mma_s8(z[nt], qf[0][nt][2 * p + 1][0], qf[1][nt][2 * p + 1][0], qf[0][nt][2 * p + 1][1],
                                   qf[1][nt][2 * p + 1][1], x.z, x.w);
                        }
#pragma unroll
                        for (int i = 0; i < (NT + 1) / 2; i++) {  // the lowest digits of two sets of columns
                            constexpr int last = NT - 1;
                            const int n0 = 2 * i, n1 = NT == 1 ? 0 : (2 * i + 1 < last ? 2 * i + 1 : last);
                            mma_s8(lo[i], qf[2][n0][2 * p][0], qf[2][n1][2 * p][0], qf[2][n0][2 * p][1], qf[2][n1][2 * p][1],
                                   x.x, x.y);
                            mma_s8(lo[i], qf[2][n0][2 * p + 1][0], qf[2][n1][2 * p + 1][0], qf[2][n0][2 * p + 1][1],
                                   qf[2][n1][2 * p + 1][1], x.z, x.w);
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 2; e++)  // sums of digits are at most 2^22: 256 mid + lo fits 32 bits
                            s[b][nt][2 * j + e] = fmaf((float)z[nt][e], 65536.0f,
                                                       (float)(z[nt][2 + e] * 256 + lo[nt / 2][2 * (nt & 1) + e]));
                }
            if (more) load_k(u + 1, page_next, ks_next, vs_next);
            // score = s f in units of log 2
            float f[NB][NT], top[NT];
            bool hidden[NB][NT][4], raise = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                top[nt] = m[nt];
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    f[b][nt] = ks[b] * qs[nt];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int t = t0 + 16 * b + 8 * (e >> 1) + 2 * q4 + (e & 1);
                        hidden[b][nt][e] = !WHOLE && (page[b] < 0 || t >= end[nt] || t < begin[nt]);
                        const float y = s[b][nt][e] * f[b][nt];
                        top[nt] = fmaxf(top[nt], hidden[b][nt][e] ? none : y);
                    }
                }
                raise |= top[nt] > m[nt];
            }
            float vmax = vtop;
#pragma unroll
            for (int b = 0; b < NB; b++) vmax = fmaxf(vmax, vs[b]);
            if (__any_sync(0xffffffffu, raise || vmax > vtop)) {
                const float fix_v = vmax > 0.0f ? vtop / vmax : 1.0f;
                vtop = vmax;
                vinv = vmax > 0.0f ? kWeightTop / vmax : 0.0f;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float x = top[nt];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    const float fix = m[nt] == none ? 0.0f : exp2_fast(m[nt] - x);
                    m[nt] = x;
                    l[nt] *= fix;
                    // the outputs' columns are 2 q4 and 2 q4 + 1 of the lane
                    const float fix0 = __shfl_sync(0xffffffffu, fix, 8 * q4) * fix_v;
                    const float fix1 = __shfl_sync(0xffffffffu, fix, 8 * q4 + 4) * fix_v;
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        acc[i][nt][0] *= fix0;
                        acc[i][nt][1] *= fix1;
                        acc[i][nt][2] *= fix0;
                        acc[i][nt][3] *= fix1;
                    }
                }
            }
            // weights, and V^T P^T
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float fv = vs[b] * vinv;
                uint32_t pf[SPLIT][NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float base = m[nt] == none ? 0.0f : m[nt];
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        // one rounding between the product and its distance from the maximum
                        float p = exp2_fast(fmaf(s[b][nt][e], f[b][nt], -base));
                        if (hidden[b][nt][e]) p = 0.0f;
                        l[nt] += p;
                        w[e] = p * fv;
                    }
                    pf[0][nt][0] = pack_f16(w[0], w[1]);
                    pf[0][nt][1] = pack_f16(w[2], w[3]);
                    if (SPLIT == 2) {
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] -= __half2float(__float2half_rn(w[e]));
                        pf[SPLIT - 1][nt][0] = pack_f16(w[0], w[1]);
                        pf[SPLIT - 1][nt][1] = pack_f16(w[2], w[3]);
                    }
                }
#pragma unroll
                for (int i = 0; i < VW; i++) {
                    const uint32_t lo01 = __byte_perm(vr[b][0][i], vr[b][1][i], 0x5410), hi01 = __byte_perm(vr[b][0][i], vr[b][1][i], 0x7632);
                    const uint32_t lo23 = __byte_perm(vr[b][2][i], vr[b][3][i], 0x5410), hi23 = __byte_perm(vr[b][2][i], vr[b][3][i], 0x7632);
                    const uint32_t a0 = codes_even(lo01), a1 = codes_odd(lo01), a2 = codes_even(lo23), a3 = codes_odd(lo23);
                    const uint32_t b0 = codes_even(hi01), b1 = codes_odd(hi01), b2 = codes_even(hi23), b3 = codes_odd(hi23);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int z = 0; z < SPLIT; z++) {
                            mma_f16(acc[2 * i][nt], a0, a1, a2, a3, pf[z][nt][0], pf[z][nt][1]);
                            mma_f16(acc[2 * i + 1][nt], b0, b1, b2, b3, pf[z][nt][0], pf[z][nt][1]);
                        }
                }
            }
            if (more) {
                load_v(u + 1, page_next);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    page[b] = page_next[b];
                    ks[b] = ks_next[b];
                    vs[b] = vs_next[b];
                }
                find(u + 2, page_next);
            }
        };
        for (int u = u0; u < u1; u++) {
            const int t0 = u * CH + warp * Cfg::TB;
            bool whole = t0 >= all_lo && t0 + Cfg::TB <= all_hi;
#pragma unroll
            for (int b = 0; b < NB; b++) whole = whole && page[b] >= 0;
            if (whole) step(u, std::true_type{});
            else step(u, std::false_type{});
        }

        // ---- the four warps' parts joined ----
        const float unscale = vtop / kWeightTop;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float x = l[nt];
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            if (q4 == 0) {
                s_m[warp][nt * 8 + g] = m[nt];
                s_l[warp][nt * 8 + g] = x;
            }
        }
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int k = nt * 8 + 2 * q4 + e;
                float top = s_m[0][k];
#pragma unroll
                for (int w = 1; w < kFewWarps; w++) top = fmaxf(top, s_m[w][k]);
                // (a part that saw nothing is 0, or NaN where its scores were)
                const float mine = s_m[warp][k], fw = (mine == none ? 1.0f : exp2_fast(mine - top)) * unscale;
                float* dst = s_acc + ((size_t)warp * COLS + k) * DP + 4 * VW * g;
#pragma unroll
                for (int i = 0; i < MT; i++)
                    *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(acc[i][nt][e] * fw, acc[i][nt][e + 2] * fw);
            }
        if (tid < COLS) {
            float top = s_m[0][tid], sum = 0.0f;
#pragma unroll
            for (int w = 1; w < kFewWarps; w++) top = fmaxf(top, s_m[w][tid]);
#pragma unroll
            for (int w = 0; w < kFewWarps; w++) sum += (s_m[w][tid] == none ? 1.0f : exp2_fast(s_m[w][tid] - top)) * s_l[w][tid];
            s_f[tid] = top;
            s_inv[tid] = sum;
        }
        __syncthreads();
        const bool split = tile0 < walk.begin || tile1 > walk.end;
        const int quads = hd / 4;
        int c0 = 0, c1 = 0;
        if (split) {
            // this CTA's part to the workspace; the last to arrive joins them
            c0 = walk.owner(tile0);
            c1 = walk.owner(tile1 - 1);
            float* part = a.parts + ((size_t)2 * blockIdx.x + (tile0 >= walk.begin)) * a.part_floats;
            for (int i = tid; i < cols * quads; i += kFewThreads) {
                const int k = i / quads, d = 4 * (i - k * quads);
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kFewWarps; w++) {
                    const float4 y = *reinterpret_cast<const float4*>(s_acc + ((size_t)w * COLS + k) * DP + d);
                    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
                }
                __stcg(reinterpret_cast<float4*>(part + 2 * COLS + (size_t)k * hd + d), x);
            }
            if (tid < cols) {
                __stcg(part + tid, s_f[tid]);
                __stcg(part + COLS + tid, s_inv[tid]);
            }
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const unsigned before = atomicAdd(&a.arrived[c0], 1u);
                s_last = before == (unsigned)(c1 - c0);
                if (s_last) a.arrived[c0] = 0;
            }
            __syncthreads();
            if (s_last) __threadfence();
        }
        if (!split || s_last) {
            for (int i = tid; i < cols * quads; i += kFewThreads) {
                const int k = i / quads, d = 4 * (i - k * quads);
                float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum, top;
                if (!split) {
                    sum = s_inv[k];
                    top = s_f[k];
#pragma unroll
                    for (int w = 0; w < kFewWarps; w++) {
                        const float4 y = *reinterpret_cast<const float4*>(s_acc + ((size_t)w * COLS + k) * DP + d);
                        x[0] += y.x; x[1] += y.y; x[2] += y.z; x[3] += y.w;
                    }
                } else {
                    top = none;
                    for (int r = c0; r <= c1; r++)
                        top = fmaxf(top, __ldcg(a.parts + ((size_t)2 * r + (r == c0)) * a.part_floats + k));
                    sum = 0.0f;
                    for (int r = c0; r <= c1; r++) {
                        const float* part = a.parts + ((size_t)2 * r + (r == c0)) * a.part_floats;
                        const float mr = __ldcg(part + k), f = mr == none ? 1.0f : exp2_fast(mr - top);
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(part + 2 * COLS + (size_t)k * hd + d));
                        sum += f * __ldcg(part + COLS + k);
                        x[0] = fmaf(f, y.x, x[0]); x[1] = fmaf(f, y.y, x[1]);
                        x[2] = fmaf(f, y.z, x[2]); x[3] = fmaf(f, y.w, x[3]);
                    }
                }
                const bool empty = top == none && sum == 0.0f;  // nothing seen
                const int r = seg.row + k / heads, h = h0 + k % heads;
                const float inv = empty ? 0.0f : __fdiv_rn(1.0f, sum);
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = empty ? 0.0f : x[e] * inv;
                store4<DT>(a.out, (size_t)r * a.out_stride + (size_t)h * hd + d, x);
                if (d == 0 && a.lse) a.lse[(size_t)r * a.nh + h] = empty ? none : (top + log2f(sum)) * kLn2;
            }
        }
        __syncthreads();
        unit = min(tile1, walk.end);
    }
}

}  // namespace hale
