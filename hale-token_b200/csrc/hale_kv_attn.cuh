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
// out evenly over the CTAs. A tile that falls into several CTAs leaves its
// parts in the workspace, and a second, small kernel joins them in CTA order,
// so results do not depend on timing. (Joined by the last CTA to arrive, a
// tile's parts cost the same kernel a fence, a counter and 100 registers of
// its token loop.) Lengths are read on the device: nothing of this is known
// when the kernels are launched.
#pragma once

#include <type_traits>

#include "hale_kv.cuh"

namespace hale {

// A tile whose parts lie in the workspace: parts of CTAs c .. c + parts - 1
// (parts 0: none begins in CTA c).
struct KvSplit {
    int parts, cols, heads, row, h0;
};

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
    KvSplit* splits;     // [gridDim] the tile that begins in each CTA and is not finished there
};

// Workspace of split tiles.
constexpr size_t kAttnPartBytes = (size_t)40 << 20;
constexpr int kAttnMaxGrid = 1024;

struct KvSegment {
    int row, rows, seq;
    int lo, hi;      // tokens any of its rows sees: [lo, hi)
    int c0, units;   // first chunk; chunks, and COST units more
};

// COST: what beginning and ending a tile costs, in units. A tile's first COST
// units stand for it and hold no tokens, so that a CTA with many short tiles
// gets fewer tokens. (Few columns: preparing queries and joining warps takes
// 4 us where a unit of 128 tokens takes 2.5; without the charge 64 sequences
// of up to 8191 tokens took 138 us, CTAs with 12 tiles ending at 137 and the
// median at 101.)

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
template <int CH, int COST>
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
    s.units = max(1, (s.hi + CH - 1) / CH - s.c0) + COST;
    return s;
}

// The units a CTA owns, walked segment by segment: of `total` units CTA c gets
// `each`, the first `extra` CTAs one more. Units are counted in 32 bits (the
// host cuts calls that could have more into several).
template <int CH, int COST, int THREADS>
struct KvWalk {
    unsigned begin, end;   // this CTA's units
    unsigned each, extra;
    unsigned base;         // units before the current segment
    KvSegment seg;

    __device__ __forceinline__ unsigned owner(unsigned unit) const {
        const unsigned big = extra * (each + 1);
        return unit < big ? unit / (each + 1) : extra + (unit - big) / each;
    }

    // All threads. False: nothing to do.
    __device__ bool start(const KvArgs& c, const KvAttn& a, KvSegment* s_seg, unsigned* s_sum) {
        constexpr int W = THREADS / 32;
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        const int tiles = c.nkv * a.subs;
        const int strip = (a.n + THREADS - 1) / THREADS, i0 = tid * strip, i1 = min(a.n, i0 + strip);
        unsigned mine = 0;
        KvSegment first;
        first.rows = 0;
        for (int i = i0; i < i1; i++) {
            const KvSegment s = kv_segment<CH, COST>(c, a, i);
            if (s.rows) mine += (unsigned)(s.units * tiles);
            if (s.rows && !first.rows) first = s;
        }
        unsigned x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) s_sum[warp] = x;
        __syncthreads();
        unsigned total = 0, before = 0;
#pragma unroll
        for (int w = 0; w < W; w++) {
            if (w < warp) before += s_sum[w];
            total += s_sum[w];
        }
        if (blockIdx.x >= total) return false;
        const unsigned grid = min(gridDim.x, total);
        each = total / grid;
        extra = total - each * grid;
        begin = blockIdx.x * each + min(blockIdx.x, extra);
        end = begin + each + (blockIdx.x < extra);
        before += x - mine;
        if (begin >= before && begin < before + mine) {
            // this thread's strip holds the first unit
            for (int i = first.row;; i++) {
                const KvSegment s = i == first.row ? first : kv_segment<CH, COST>(c, a, i);
                if (!s.rows) continue;
                const unsigned u = (unsigned)(s.units * tiles);
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
        base += (unsigned)(seg.units * c.nkv * a.subs);
        int i = seg.row + seg.rows;
        while (i < a.n) {
            seg = kv_segment<CH, COST>(c, a, i);
            if (seg.rows) return;
            i++;
        }
    }
};

// ---------------------------------------------------------------------------
// small matrix pieces
// ---------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 load_shared8(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
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

// d = a b, or d += a b.
template <bool FIRST>
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    if (FIRST)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four dims of a row's result from the weighted sum x, the maximum and the sum
// of its weights; its lse beside the first.
template <int DT>
__device__ __forceinline__ void kv_finish(const KvAttn& a, int row, int head, int hd, int d, float (&x)[4], float top,
                                          float sum) {
    const float none = -__int_as_float(0x7f800000);
    const bool empty = top == none && sum == 0.0f;  // nothing seen (not: NaN scores, whose sum is NaN)
    const float inv = empty ? 0.0f : __fdiv_rn(1.0f, sum);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = empty ? 0.0f : x[e] * inv;
    store4<DT>(a.out, (size_t)row * a.out_stride + (size_t)head * hd + d, x);
    if (d == 0 && a.lse) a.lse[(size_t)row * a.nh + head] = empty ? none : (top + log2f(sum)) * kLn2;
}

// Split tiles joined, in CTA order: one CTA per possible tile, a warp per
// column, lanes over the dims; what a part counts is computed by the lanes
// over the parts while the first eight parts' values are under way.
constexpr int kJoinThreads = 256;

template <int DT>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(KvAttn a, int hd, int max_cols) {
    constexpr int BATCH = 8;
    const int lane = threadIdx.x & 31, c = blockIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const KvSplit t = a.splits[c];
    if (t.parts == 0) return;
    const float none = -__int_as_float(0x7f800000);
    const float* base = a.parts + (size_t)2 * c * a.part_floats;
    auto part = [&](int r) { return base + (size_t)(2 * r + (r == 0)) * a.part_floats; };
    for (int k = threadIdx.x >> 5; k < t.cols; k += kJoinThreads / 32) {
        for (int d = 4 * lane; d < (hd + 127) / 128 * 128; d += 128) {
            float4 y[BATCH];
            const bool in = d < hd;
            const size_t at = 2 * max_cols + (size_t)k * hd + d;
#pragma unroll
            for (int r = 0; r < BATCH; r++)
                y[r] = in && r < t.parts ? *reinterpret_cast<const float4*>(part(r) + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float top = none, sum = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int r = lane; r < t.parts; r += 32) top = fmaxf(top, part(r)[k]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            for (int r0 = 0; r0 < t.parts; r0 += 32) {
                const int r = r0 + lane;
                float w = 0.0f;
                if (r < t.parts) {
                    const float m = part(r)[k];
                    w = m == none ? 1.0f : exp2_fast(m - top);  // (a part that saw nothing is 0)
                    sum = fmaf(w, part(r)[max_cols + k], sum);
                }
                for (int i0 = 0; i0 < 32 && r0 + i0 < t.parts; i0 += BATCH) {
                    if (r0 + i0 > 0) {
#pragma unroll
                        for (int i = 0; i < BATCH; i++)
                            y[i] = in && r0 + i0 + i < t.parts ? *reinterpret_cast<const float4*>(part(r0 + i0 + i) + at)
                                                               : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
#pragma unroll
                    for (int i = 0; i < BATCH; i++) {
                        const float f = __shfl_sync(0xffffffffu, w, i0 + i);
                        x[0] = fmaf(f, y[i].x, x[0]); x[1] = fmaf(f, y[i].y, x[1]);
                        x[2] = fmaf(f, y[i].z, x[2]); x[3] = fmaf(f, y[i].w, x[3]);
                    }
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (in) kv_finish<DT>(a, t.row + k / t.heads, t.h0 + k % t.heads, hd, d, x, top, sum);
        }
    }
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
// Codes reach a warp through its own ring of stages in shared memory, filled
// by 16-byte asynchronous copies STAGES - 1 steps ahead: a warp waits for no
// other, and the bytes in flight do not depend on where its arithmetic stands.
// A token's 16-byte pieces are permuted (xor with bits of the token's number)
// so that the fragments' loads meet no bank twice. Whatever bytes lie in a
// hidden token or behind the head's dims, they are finite codes, and the
// token's weight, like a missing dim of q, is 0.
constexpr int kFewWarps = 4, kFewThreads = 32 * kFewWarps, kFewCost = 2;

template <int DP>
struct FewCfg {
    static constexpr int NB = DP <= 128 ? 2 : 1;         // blocks of 16 tokens a warp takes at a time
    static constexpr int TB = 16 * NB, CH = TB * kFewWarps;
    static constexpr int STAGES = 2;
    static constexpr int STAGE = 2 * TB * DP;            // bytes of a stage: keys, then values
    static constexpr int RING = STAGES * STAGE;          // of one warp
    static constexpr int PIECES = DP / 16;               // 16-byte pieces of a row
    static constexpr int KC = DP / 64;                   // 64-dim pieces of a key row
    static constexpr int VW = DP / 32;                   // 32-bit words of a lane's dims of one value row
};

// Where a token's piece i goes: i ^ swizzle. A key load reads pieces 4 p + 0..3
// of tokens g, g + 1: with 128-byte rows odd tokens move to the other half. A
// value load reads piece g of tokens 0, 2, 4, 6 (and g + 1 beside it).
template <int DP>
__device__ __forceinline__ int few_key_swizzle(int t) {
    return DP >= 128 ? (t & 1) << 2 : 0;
}
template <int DP>
__device__ __forceinline__ int few_value_swizzle(int t) {
    return DP >= 128 ? (t >> 1 & 3) << 1 : t >> 1 & 3;
}

// A block in a stage: its scales and its page (-1: nothing of it is seen).
struct alignas(16) FewBlock {
    float ks, vs;
    int page, unused;
};

// HD: the head's dims where they are known (= DP), else 0.
template <int DT, int DP, int HD, int NT>
__global__ void __launch_bounds__(kFewThreads, DP <= 128 && NT == 1 ? 3 : 2) kv_attn_few_kernel(KvArgs c, KvAttn a) {
    using Cfg = FewCfg<DP>;
    constexpr int NB = Cfg::NB, CH = Cfg::CH, KC = Cfg::KC, VW = Cfg::VW, MT = DP / 16, COLS = 8 * NT;
    constexpr int SPLIT = DT == 0 ? 2 : 1;
    __shared__ KvSegment s_seg;
    __shared__ unsigned s_sum[kFewWarps + 1];
    __shared__ float s_m[kFewWarps][COLS], s_l[kFewWarps][COLS], s_f[COLS], s_inv[COLS];
    __shared__ __align__(16) int8_t s_q[3][COLS][DP + 16];
    __shared__ int s_end[COLS];
    __shared__ FewBlock s_block[kFewWarps][Cfg::STAGES][NB];
    extern __shared__ __align__(128) int8_t s_ring[];  // [kFewWarps][RING]; between tiles the warps' sums
    float* s_acc = reinterpret_cast<float*>(s_ring);   // [kFewWarps][COLS][DP]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
    const uint32_t ring = smem_addr(s_ring) + warp * Cfg::RING;
    const int hd = HD ? HD : c.hd;
    const float none = -__int_as_float(0x7f800000);

    if (tid == 0) a.splits[blockIdx.x].parts = 0;
    KvWalk<CH, kFewCost, kFewThreads> walk;
    if (!walk.start(c, a, &s_seg, s_sum)) return;
    unsigned unit = walk.begin;
    while (unit < walk.end) {
        while (unit >= walk.base + (unsigned)(walk.seg.units * c.nkv * a.subs)) walk.next(c, a);
        const KvSegment seg = walk.seg;
        const int tile = (int)((unit - walk.base) / (unsigned)seg.units), head = tile / a.subs, sub = tile - head * a.subs;
        const unsigned tile0 = walk.base + (unsigned)(tile * seg.units), tile1 = tile0 + seg.units;
        const unsigned first = tile0 + kFewCost;  // the tile's first chunk
        if (walk.end <= first) return;             // this CTA's units end before it
        const unsigned from = max(unit, first);
        const int u0 = seg.c0 + (int)(from - first), u1 = seg.c0 + (int)(min(tile1, walk.end) - first);
        const int heads = min(a.heads, a.group - sub * a.heads), cols = seg.rows * heads;
        const int h0 = head * a.group + sub * a.heads;  // the tile's first query head

        // ---- the first tokens are under way while the queries are prepared ----
        // a page's codes (at most 2^26 bytes) and scales
        const unsigned page_codes = (unsigned)(c.nkv * hd) << c.page_log2, page_scales = (unsigned)c.nkv << c.page_log2 >> 4;
        // this lane's pieces: 32 / PIECES rows apart
        constexpr int PIECES = Cfg::PIECES, ROWS = 32 / PIECES;
        const int my_row = lane / PIECES, my_piece = lane % PIECES;
        const size_t my_at = ((size_t)head << c.page_log2) * hd + (unsigned)(my_row * hd + 16 * my_piece);
        const bool copies = HD || 16 * my_piece < hd;
        // (the swizzles are linear in a token's bits, and my_row and the steps share none)
        const uint32_t key_to = my_row * DP + 16 * (my_piece ^ few_key_swizzle<DP>(my_row));
        const uint32_t value_to = my_row * DP + 16 * (my_piece ^ few_value_swizzle<DP>(my_row));
        // where the fragments' tokens g and 2 q4 lie
        const uint32_t key_at[2] = {(uint32_t)(g * DP + 16 * (q4 ^ few_key_swizzle<DP>(g))),
                                    (uint32_t)(g * DP + 16 * ((4 + q4) ^ few_key_swizzle<DP>(g)))};
        const uint32_t value_at = 2 * q4 * DP + (VW == 2 ? 16 * ((g >> 1) ^ few_value_swizzle<DP>(2 * q4)) + 8 * (g & 1)
                                                         : 16 * ((VW / 4 * g) ^ few_value_swizzle<DP>(2 * q4)));
        const float* ksbase = c.ks + ((size_t)head << c.page_log2 >> 4);
        const float* vsbase = c.vs + ((size_t)head << c.page_log2 >> 4);

        // Pages of the warp's blocks: lane i holds that of block i of 32, a page
        // piece (PB blocks that lie in one page) an entry; the next 32 are
        // under way. -1: nothing of it is seen, or it is missing.
        constexpr int PB = HD ? NB : 1, PER = NB / PB;  // (a page of 16 tokens takes the kernels of any head size)
        const int32_t* row = c.table + (size_t)min(seg.seq, c.n_seqs - 1) * c.max_pages;
        auto find = [&](int u) {
            const int t = (u + lane / PER) * CH + warp * Cfg::TB + 16 * PB * (lane % PER);
            int pg = -1;
            if (u + lane / PER < u1 && t < seg.hi && t + 16 * PB > seg.lo) {
                pg = c.checked(row[t >> c.page_log2]);
                if (pg < 0) raise_error(c.err, kErrBounds);
            }
            return pg;
        };
        int pages = find(u0), pages_next = find(u0 + 32 / PER), pages_from = u0;
        // unit u's codes and scales into their stage
        auto fetch = [&](int u) {
            if (u < u1) {
                if (u - pages_from == 32 / PER) {
                    pages = pages_next;
                    pages_from = u;
                    pages_next = find(u + 32 / PER);
                }
                const int stage = (u - u0) % Cfg::STAGES;
                const uint32_t dst = ring + stage * Cfg::STAGE;
#pragma unroll
                for (int e = 0; e < PER; e++) {
                    const int pg = __shfl_sync(0xffffffffu, pages, (u - pages_from) * PER + e);
                    const int slot = c.slot(u * CH + warp * Cfg::TB + 16 * PB * e);
                    FewBlock* block = s_block[warp][stage] + PB * e;
                    if (lane < PB) block[lane].page = pg;
                    if (pg < 0) continue;
                    if (lane < 2 * PB) {
                        const size_t sa = (size_t)(unsigned)pg * page_scales + (slot >> 4) + (lane >> 1);
                        cp_async4(smem_addr(lane & 1 ? &block[lane >> 1].vs : &block[lane >> 1].ks), (lane & 1 ? vsbase : ksbase) + sa);
                    }
                    if (copies) {
                        const size_t at = (size_t)(unsigned)pg * page_codes + (unsigned)(slot * hd) + my_at;
                        const int8_t *kp = c.k + at, *vp = c.v + at;
#pragma unroll
                        for (int r = 0; r < 16 * PB; r += ROWS) {
                            cp_async16(dst + (16 * PB * e + r) * DP + (key_to ^ 16 * few_key_swizzle<DP>(r)), kp + r * hd);
                            cp_async16(dst + (Cfg::TB + 16 * PB * e + r) * DP + (value_to ^ 16 * few_value_swizzle<DP>(r)),
                                       vp + r * hd);
                        }
                    }
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < Cfg::STAGES - 1; i++) fetch(u0 + i);
        // ---- the columns' queries and what they see ----
        // A warp turns a column at a time into its digits; everyone then takes
        // its A fragments (rows g: column g) from shared memory. The integer
        // product's k index runs over 16 t + 4 q4 + byte of a 32-dim step:
        // words 0, 1 and 2, 3 of the 16 dims a lane's key pieces hold.
        for (int k = warp; k < COLS; k += kFewWarps) {
            float amax = 0.0f, x[(DP + 127) / 128][4];
            bool wild = false;  // infinities and NaN have no digits
            const size_t at = k < cols ? (size_t)(seg.row + k / heads) * a.q_stride + (size_t)(h0 + k % heads) * hd : 0;
#pragma unroll
            for (int v = 0; v < (DP + 127) / 128; v++) {
                const int d = 128 * v + 4 * lane;
                x[v][0] = x[v][1] = x[v][2] = x[v][3] = 0.0f;
                if (k < cols && d < hd) load4<DT>(a.q, at + d, x[v]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    amax = fmaxf(amax, fabsf(x[v][i]));
                    wild |= !(fabsf(x[v][i]) <= 0x1.fffffep127f);
                }
            }
            const float up = kv_query_scale(warp_max_abs(amax));
            wild = __any_sync(0xffffffffu, wild);
#pragma unroll
            for (int v = 0; v < (DP + 127) / 128; v++) {
                uint32_t d[3];
#pragma unroll
                for (int i = 0; i < 4; i++) x[v][i] *= up;
                kv_query_digits(x[v], d);
                if (128 * v + 4 * lane < DP) {
#pragma unroll
                    for (int z = 0; z < 3; z++) *reinterpret_cast<uint32_t*>(&s_q[z][k][128 * v + 4 * lane]) = d[z];
                }
            }
            if (lane == 0) {
                s_f[k] = wild ? __int_as_float(0x7fc00000) : a.scale * kLog2e / up;  // NaN: so are the column's scores
                int end = 0;
                if (k < cols) {
                    const int p = a.positions[seg.row + k / heads];
                    end = p >= 0 && p < seg.hi ? p + 1 : 0;
                }
                s_end[k] = end;
            }
        }
        __syncthreads();
        uint32_t qf[2][NT][KC * 2][2], qlo[(NT + 1) / 2][KC * 2][4];
        float qs[NT];
        int end[NT], begin[NT];
        int all_lo = 0, all_hi = INT_MAX;  // tokens every column sees
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int k = nt * 8 + g;
#pragma unroll
            for (int z = 0; z < 2; z++)
#pragma unroll
                for (int p = 0; p < KC; p++) {
                    const uint4 x = *reinterpret_cast<const uint4*>(&s_q[z][k][64 * p + 16 * q4]);
                    qf[z][nt][2 * p][0] = x.x;
                    qf[z][nt][2 * p][1] = x.y;
                    qf[z][nt][2 * p + 1][0] = x.z;
                    qf[z][nt][2 * p + 1][1] = x.w;
                }
            qs[nt] = s_f[k];
            end[nt] = s_end[k];
            begin[nt] = a.window > 0 ? max(0, end[nt] - a.window) : 0;
            if (k < cols) {
                all_hi = min(all_hi, end[nt]);
                all_lo = max(all_lo, begin[nt]);
            }
        }
        // the lowest digits of two sets of columns (of one: twice) as whole
        // operands; read by loads of their own, so that the second copy is no
        // register moved before every product
#pragma unroll
        for (int i = 0; i < (NT + 1) / 2; i++)
#pragma unroll
            for (int p = 0; p < KC; p++) {
                const uint32_t at = smem_addr(&s_q[2][16 * i + g][64 * p + 16 * q4]);
                const uint4 x = load_shared16(at), y = load_shared16(2 * i + 1 < NT ? at + 8 * (DP + 16) : at);
                const uint32_t quads[2][4] = {{x.x, y.x, x.y, y.y}, {x.z, y.z, x.w, y.w}};
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int e = 0; e < 4; e++) qlo[i][2 * p + h][e] = quads[h][e];
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
        int page[NB];
        float ks[NB], vs[NB];
        // One step over the warp's tokens of unit u; WHOLE: every column sees
        // all of them and every page is there.
        auto step = [&](int u, auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            const int t0 = u * CH + warp * Cfg::TB, stage = (u - u0) % Cfg::STAGES;
            const uint32_t keys = ring + stage * Cfg::STAGE, vals = keys + Cfg::TB * DP + value_at;
            // q . kc, integers of at most 2^45, rounded to f32; [token half][token]
            float s[NB][NT][4];
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    int z[NT][4], lo[(NT + 1) / 2][4];
#pragma unroll
                    for (int p = 0; p < KC; p++) {
                        const uint4 x = load_shared16(keys + (16 * b + 8 * j) * DP + 128 * (p / 2) + key_at[p & 1]);
#pragma unroll
                        for (int h = 0; h < 2; h++) {  // the two 32-dim steps of a piece
                            const uint32_t b0 = h ? x.z : x.x, b1 = h ? x.w : x.y;
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                const auto& hi = qf[0][nt][2 * p + h];
                                const auto& mid = qf[1][nt][2 * p + h];
                                if (p + h == 0) mma_s8<true>(z[nt], hi[0], mid[0], hi[1], mid[1], b0, b1);
                                else mma_s8<false>(z[nt], hi[0], mid[0], hi[1], mid[1], b0, b1);
                            }
#pragma unroll
                            for (int i = 0; i < (NT + 1) / 2; i++) {
                                const auto& q = qlo[i][2 * p + h];
                                if (p + h == 0) mma_s8<true>(lo[i], q[0], q[1], q[2], q[3], b0, b1);
                                else mma_s8<false>(lo[i], q[0], q[1], q[2], q[3], b0, b1);
                            }
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 2; e++)  // sums of digits are at most 2^22: 256 mid + lo fits 32 bits
                            s[b][nt][2 * j + e] = fmaf((float)z[nt][e], 65536.0f,
                                                       (float)(z[nt][2 + e] * 256 + lo[nt / 2][2 * (nt & 1) + e]));
                }
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
                uint32_t vr[4][VW];  // tokens 2 q4, + 1, + 8, + 9
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t src = vals + (16 * b + (j & 1) + 8 * (j >> 1)) * DP;
                    if (VW == 2) {
                        const uint2 v = load_shared8(src);
                        vr[j][0] = v.x;
                        vr[j][1] = v.y;
                    } else {
#pragma unroll
                        for (int w = 0; w + 4 <= VW; w += 4) {
                            const uint4 v = load_shared16(src + 4 * w);
                            vr[j][w] = v.x;
                            vr[j][w + 1] = v.y;
                            vr[j][w + 2] = v.z;
                            vr[j][w + 3] = v.w;
                        }
                    }
                }
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
                    const uint32_t lo01 = __byte_perm(vr[0][i], vr[1][i], 0x5410), hi01 = __byte_perm(vr[0][i], vr[1][i], 0x7632);
                    const uint32_t lo23 = __byte_perm(vr[2][i], vr[3][i], 0x5410), hi23 = __byte_perm(vr[2][i], vr[3][i], 0x7632);
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
        };
        for (int u = u0; u < u1; u++) {
            fetch(u + Cfg::STAGES - 1);
            cp_async_wait<Cfg::STAGES - 1>();
            __syncwarp();
            const int t0 = u * CH + warp * Cfg::TB, stage = (u - u0) % Cfg::STAGES;
            bool whole = t0 >= all_lo && t0 + Cfg::TB <= all_hi;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const FewBlock block = s_block[warp][stage][b];
                page[b] = block.page;
                ks[b] = block.ks;
                vs[b] = block.vs;
                whole = whole && page[b] >= 0;
            }
            if (!whole) {
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    // a block no row sees a token of: its scales may be anything
                    const int t = t0 + 16 * b;
                    if (page[b] < 0 || t >= seg.hi || t + 16 <= seg.lo) {
                        page[b] = -1;
                        ks[b] = vs[b] = 0.0f;
                    }
                }
            }
            if (whole) step(u, std::true_type{});
            else step(u, std::false_type{});
            __syncwarp();
        }
        cp_async_wait<0>();

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
        const bool split = first < walk.begin || tile1 > walk.end;
        const int quads = hd / 4;
        float* part = a.parts + ((size_t)2 * blockIdx.x + (first >= walk.begin)) * a.part_floats;
        for (int i = tid; i < cols * quads; i += kFewThreads) {
            const int k = i / quads, d = 4 * (i - k * quads);
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kFewWarps; w++) {
                const float4 y = *reinterpret_cast<const float4*>(s_acc + ((size_t)w * COLS + k) * DP + d);
                x[0] += y.x; x[1] += y.y; x[2] += y.z; x[3] += y.w;
            }
            if (split) *reinterpret_cast<float4*>(part + 2 * COLS + 4 * i) = make_float4(x[0], x[1], x[2], x[3]);
            else kv_finish<DT>(a, seg.row + k / heads, h0 + k % heads, hd, d, x, s_f[k], s_inv[k]);
        }
        if (split && tid < cols) {
            part[tid] = s_f[tid];
            part[COLS + tid] = s_inv[tid];
        }
        if (split && first >= walk.begin && tid == 0)
            a.splits[blockIdx.x] = {(int)walk.owner(tile1 - 1) - (int)blockIdx.x + 1, cols, heads, seg.row, h0};
        __syncthreads();
        unit = min(tile1, walk.end);
    }
}

// ---------------------------------------------------------------------------
// many columns: 64 of them per tile, codes widened to f16 once for all
//
// Four warps of 16 columns each. A unit of UT tokens arrives as codes by
// asynchronous copies (during the unit before it), is widened to f16 tiles in shared
// memory by all warps, and feeds both products from there: S = q K^T with q
// from shared memory, O += P V with P straight from S's registers. q is scaled
// by a power of two to at most 2^14: exact in f16 for f16 and (down to 2^-38
// of the row's largest value) bf16, two f16 (22 bits) for f32. Tiles lie in
// rows of 2 DP bytes whose 16-byte pieces are xor-ed with the row's number, so
// that the matrix loads meet no bank twice.
// Bound by instruction issue beside the matrix instructions (one m16n8k16 in 8
// cycles): a warp's unit of 64 tokens is 128 of them and about 1000 others,
// half of those the softmax.
// ---------------------------------------------------------------------------
constexpr int kManyWarps = 4, kManyThreads = 32 * kManyWarps, kManyCols = 16 * kManyWarps, kManyCost = 2;

template <int DT, int DP>
struct ManyCfg {
    static constexpr int SPLIT = DT == 0 ? 2 : 1;
    static constexpr int UT = DP <= 128 ? 64 : 32;        // tokens of a unit
    static constexpr int CODES = UT * DP;                 // bytes of a unit's keys (or values)
    static constexpr int QUERY = kManyCols * DP * 2;      // one f16 part of the queries
    static constexpr int TILE = UT * DP * 2;              // f16 keys (or values)
    static constexpr int SMEM = SPLIT * QUERY + 2 * TILE + 2 * CODES;
    static constexpr int PER_SM = SPLIT == 1 && DP <= 128 ? 3 : 2;
};

__device__ __forceinline__ void load_matrix(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void load_matrix_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void store_shared16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Four codes as four f16 in order.
__device__ __forceinline__ uint2 codes_f16(uint32_t w) {
    const uint32_t x = w ^ 0x80808080u, off = 0x64806480u;
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 o = *reinterpret_cast<const __half2*>(&off);
    const __half2 h0 = __hsub2(*reinterpret_cast<const __half2*>(&a), o), h1 = __hsub2(*reinterpret_cast<const __half2*>(&b), o);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
}
// Power of two that brings amax to at most 2^14 and at least 2^13.
__device__ __forceinline__ float kv_query_scale_f16(float amax) {
    if (!(amax > 0.0f) || !(amax <= 0x1.fffffep127f)) return 1.0f;
    int e;
    frexpf(amax, &e);
    return ldexpf(1.0f, min(126, max(-126, 14 - e)));
}

template <int DT, int DP>
__global__ void __launch_bounds__(kManyThreads, ManyCfg<DT, DP>::PER_SM) kv_attn_many_kernel(KvArgs c, KvAttn a) {
    using Cfg = ManyCfg<DT, DP>;
    constexpr int UT = Cfg::UT, SPLIT = Cfg::SPLIT, NB = UT / 16, ROW = 2 * DP;
    constexpr int PIECES = DP / 16;                     // 16-byte pieces of a row of codes
    constexpr int STEP = kManyThreads / PIECES;         // rows the CTA copies at once
    __shared__ KvSegment s_seg;
    __shared__ unsigned s_sum[kManyWarps + 1];
    __shared__ float s_up[kManyCols];
    __shared__ int s_end[kManyCols];
    __shared__ FewBlock s_block[2][NB];
    extern __shared__ __align__(128) int8_t s_many[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
    const int hd = c.hd;
    const float none = -__int_as_float(0x7f800000);
    const uint32_t s_q = smem_addr(s_many), s_k = s_q + SPLIT * Cfg::QUERY, s_v = s_k + Cfg::TILE, s_codes = s_v + Cfg::TILE;

    if (tid == 0) a.splits[blockIdx.x].parts = 0;
    KvWalk<UT, kManyCost, kManyThreads> walk;
    if (!walk.start(c, a, &s_seg, s_sum)) return;
    unsigned unit = walk.begin;
    while (unit < walk.end) {
        while (unit >= walk.base + (unsigned)(walk.seg.units * c.nkv * a.subs)) walk.next(c, a);
        const KvSegment seg = walk.seg;
        const int tile = (int)((unit - walk.base) / (unsigned)seg.units), head = tile / a.subs, sub = tile - head * a.subs;
        const unsigned tile0 = walk.base + (unsigned)(tile * seg.units), tile1 = tile0 + seg.units;
        const unsigned first = tile0 + kManyCost;  // the tile's first chunk
        if (walk.end <= first) return;             // this CTA's units end before it
        const unsigned from = max(unit, first);
        const int u0 = seg.c0 + (int)(from - first), u1 = seg.c0 + (int)(min(tile1, walk.end) - first);
        const int heads = min(a.heads, a.group - sub * a.heads), cols = seg.rows * heads;
        const int h0 = head * a.group + sub * a.heads;

        // ---- copies of a unit's codes: thread -> (row, piece), rows STEP apart ----
        const unsigned page_codes = (unsigned)(c.nkv * hd) << c.page_log2, page_scales = (unsigned)c.nkv << c.page_log2 >> 4;
        const int my_row = tid / PIECES, my_piece = tid % PIECES;
        const bool copies = 16 * my_piece < hd;
        const size_t my_at = ((size_t)head << c.page_log2) * hd + 16 * my_piece;
        const float* ksbase = c.ks + ((size_t)head << c.page_log2 >> 4);
        const float* vsbase = c.vs + ((size_t)head << c.page_log2 >> 4);
        const int32_t* row = c.table + (size_t)min(seg.seq, c.n_seqs - 1) * c.max_pages;
        // pages of 32 blocks by lane, the next 32 under way (as above)
        auto find = [&](int u) {
            const int t = u * UT + 16 * lane;
            int pg = -1;
            if (t < u1 * UT && t < seg.hi && t + 16 > seg.lo) {
                pg = c.checked(row[t >> c.page_log2]);
                if (pg < 0 && warp == 0) raise_error(c.err, kErrBounds);
            }
            return pg;
        };
        constexpr int HELD = 32 / NB;  // units whose pages are held
        int pages = find(u0), pages_next = find(u0 + HELD), pages_from = u0;
        auto fetch = [&](int u) {
            if (u < u1) {
                if (u - pages_from == HELD) {
                    pages = pages_next;
                    pages_from = u;
                    pages_next = find(u + HELD);
                }
                const int stage = (u - u0) & 1;
                const uint32_t dst = s_codes + 16 * tid;
#pragma unroll
                for (int r = 0; r < UT; r += STEP) {
                    // a warp's rows lie in one block
                    const int b = (r + my_row) >> 4;
                    const int pg = __shfl_sync(0xffffffffu, pages, (u - pages_from) * NB + b);
                    if (pg < 0 || !copies) continue;
                    const int slot = c.slot(u * UT + r + my_row);
                    const size_t at = (size_t)(unsigned)pg * page_codes + (unsigned)(slot * hd) + my_at;
                    cp_async16(dst + r * DP, c.k + at);
                    cp_async16(dst + Cfg::CODES + r * DP, c.v + at);
                }
                const int pg = __shfl_sync(0xffffffffu, pages, (u - pages_from) * NB + (tid & (NB - 1)));
                if (tid < NB) {
                    FewBlock& block = s_block[stage][tid];
                    block.page = pg;
                    if (pg >= 0) {
                        const size_t sa = (size_t)(unsigned)pg * page_scales + (c.slot(u * UT + 16 * tid) >> 4);
                        cp_async4(smem_addr(&block.ks), ksbase + sa);
                        cp_async4(smem_addr(&block.vs), vsbase + sa);
                    }
                }
            }
            cp_async_commit();
        };
        fetch(u0);

        // ---- queries: a warp widens its own 16 columns ----
        for (int k = 16 * warp; k < 16 * warp + 16; k++) {
            float amax = 0.0f, x[(DP + 127) / 128][4];
            bool wild = false;
            const size_t at = k < cols ? (size_t)(seg.row + k / heads) * a.q_stride + (size_t)(h0 + k % heads) * hd : 0;
#pragma unroll
            for (int v = 0; v < (DP + 127) / 128; v++) {
                const int d = 128 * v + 4 * lane;
                x[v][0] = x[v][1] = x[v][2] = x[v][3] = 0.0f;
                if (k < cols && d < hd) load4<DT>(a.q, at + d, x[v]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    amax = fmaxf(amax, fabsf(x[v][i]));
                    wild |= !(fabsf(x[v][i]) <= 0x1.fffffep127f);
                }
            }
            const float up = kv_query_scale_f16(warp_max_abs(amax));
            wild = __any_sync(0xffffffffu, wild);
#pragma unroll
            for (int v = 0; v < (DP + 127) / 128; v++) {
                const int d = 128 * v + 4 * lane;
                if (d >= DP) continue;
#pragma unroll
                for (int z = 0; z < SPLIT; z++) {
                    uint32_t w[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        float y0 = x[v][2 * i] * up, y1 = x[v][2 * i + 1] * up;
                        if (z) {
                            y0 -= __half2float(__float2half_rn(y0));
                            y1 -= __half2float(__float2half_rn(y1));
                        }
                        w[i] = pack_f16(y0, y1);
                    }
                    const uint32_t to = s_q + z * Cfg::QUERY + k * ROW + 16 * ((d >> 3) ^ (k & 7)) + 2 * (d & 7);
                    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(to), "r"(w[0]), "r"(w[1]) : "memory");
                }
            }
            if (lane == 0) {
                s_up[k] = wild ? __int_as_float(0x7fc00000) : a.scale * kLog2e / up;  // NaN: so are the column's scores
                int end = 0;
                if (k < cols) {
                    const int p = a.positions[seg.row + k / heads];
                    end = p >= 0 && p < seg.hi ? p + 1 : 0;
                }
                s_end[k] = end;
            }
        }
        __syncwarp();
        // a lane's columns of the products: 16 warp + g, + 8
        float qs[2], m[2], l[2], acc[DP / 8][4];
        int end[2], begin[2], all_lo = 0, all_hi = INT_MAX, any_hi = 0;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int k = 16 * warp + g + 8 * e;
            qs[e] = s_up[k];
            end[e] = s_end[k];
            begin[e] = a.window > 0 ? max(0, end[e] - a.window) : 0;
            m[e] = none;
            l[e] = 0.0f;
            if (k < cols) {
                all_hi = min(all_hi, end[e]);
                all_lo = max(all_lo, begin[e]);
                any_hi = max(any_hi, end[e]);
            }
        }
        all_hi = __reduce_min_sync(0xffffffffu, all_hi);
        all_lo = __reduce_max_sync(0xffffffffu, all_lo);
        any_hi = __reduce_max_sync(0xffffffffu, any_hi);
#pragma unroll
        for (int i = 0; i < DP / 8; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
        float vtop = 0.0f, vinv = 0.0f;

        for (int u = u0; u < u1; u++) {
            const int t0 = u * UT, stage = (u - u0) & 1;
            cp_async_wait<0>();
            __syncthreads();  // the codes are there, and no one reads the tiles any more
#pragma unroll
            for (int r = 0; r < UT; r += STEP) {
                const int t = r + my_row;
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const uint4 x = load_shared16(s_codes + v * Cfg::CODES + 16 * tid + r * DP);
                    const uint2 h0 = codes_f16(x.x), h1 = codes_f16(x.y), h2 = codes_f16(x.z), h3 = codes_f16(x.w);
                    const uint4 lo = make_uint4(h0.x, h0.y, h1.x, h1.y), hi = make_uint4(h2.x, h2.y, h3.x, h3.y);
                    const uint32_t to = (v ? s_v : s_k) + t * ROW;
                    store_shared16(to + 16 * ((2 * my_piece) ^ (t & 7)), lo);
                    store_shared16(to + 16 * ((2 * my_piece + 1) ^ (t & 7)), hi);
                }
            }
            __syncthreads();
            fetch(u + 1);
            if (t0 >= any_hi || t0 + UT <= seg.lo) continue;  // nothing of it for this warp's columns

            // ---- S = q K^T ----
            float s[UT / 8][4];
#pragma unroll
            for (int i = 0; i < UT / 8; i++) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
            for (int p = 0; p < DP / 16; p++) {
                uint32_t q[SPLIT][4];
#pragma unroll
                for (int z = 0; z < SPLIT; z++) {
                    const int r = 16 * warp + (lane & 15);
                    load_matrix(q[z], s_q + z * Cfg::QUERY + r * ROW + 16 * ((2 * p + (lane >> 4)) ^ (r & 7)));
                }
#pragma unroll
                for (int i = 0; i < UT / 16; i++) {
                    uint32_t k[4];
                    const int t = 16 * i + (lane & 7) + (lane >> 4 << 3);
                    load_matrix(k, s_k + t * ROW + 16 * ((2 * p + (lane >> 3 & 1)) ^ (t & 7)));
#pragma unroll
                    for (int z = 0; z < SPLIT; z++) {
                        mma_f16(s[2 * i], q[z][0], q[z][1], q[z][2], q[z][3], k[0], k[1]);
                        mma_f16(s[2 * i + 1], q[z][0], q[z][1], q[z][2], q[z][3], k[2], k[3]);
                    }
                }
            }
            // ---- softmax: score = s f in units of log 2 ----
            float ks[NB], vs[NB];
            int page[NB];
            bool whole = t0 >= all_lo && t0 + UT <= all_hi;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const FewBlock block = s_block[stage][b];
                const int t = t0 + 16 * b;
                const bool none_of_it = block.page < 0 || t >= seg.hi || t + 16 <= seg.lo;
                page[b] = none_of_it ? -1 : block.page;
                ks[b] = none_of_it ? 0.0f : block.ks;
                vs[b] = none_of_it ? 0.0f : block.vs;
                whole = whole && !none_of_it;
            }
            // softmax and second product; WHOLE: every column sees every token
            auto weigh = [&](auto whole_) {
            constexpr bool WHOLE = decltype(whole_)::value;
            auto hidden = [&](int i, int e) {  // token 8 i + 2 q4 + (e & 1)
                const int t = t0 + 8 * i + 2 * q4 + (e & 1);
                return !WHOLE && (page[i / 2] < 0 || t >= end[e >> 1] || t < begin[e >> 1]);
            };
            float top[2] = {m[0], m[1]}, vmax = vtop;
#pragma unroll
            for (int b = 0; b < NB; b++) vmax = fmaxf(vmax, vs[b]);
#pragma unroll
            for (int i = 0; i < UT / 8; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y = s[i][e] * (ks[i / 2] * qs[e >> 1]);
                    top[e >> 1] = fmaxf(top[e >> 1], hidden(i, e) ? none : y);
                }
            if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1] || vmax > vtop)) {
                const float fix_v = vmax > 0.0f ? vtop / vmax : 1.0f;
                vtop = vmax;
                vinv = vmax > 0.0f ? kWeightTop / vmax : 0.0f;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float x = top[e];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    const float fix = m[e] == none ? 0.0f : exp2_fast(m[e] - x);
                    m[e] = x;
                    l[e] *= fix;
#pragma unroll
                    for (int i = 0; i < DP / 8; i++) {
                        acc[i][2 * e] *= fix * fix_v;
                        acc[i][2 * e + 1] *= fix * fix_v;
                    }
                }
            }
            const float base[2] = {m[0] == none ? 0.0f : m[0], m[1] == none ? 0.0f : m[1]};
            // ---- O += P V, 16 tokens (a block) at a time ----
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float fv = vs[b] * vinv;
                uint32_t p[SPLIT][4];  // A fragment: (g, 2 q4), (g + 8, ..), (g, 2 q4 + 8), ..
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int i = 2 * b + j;
                        float x = exp2_fast(fmaf(s[i][e], ks[b] * qs[e >> 1], -base[e >> 1]));
                        if (hidden(i, e)) x = 0.0f;
                        l[e >> 1] += x;
                        w[e] = x * fv;
                    }
                    p[0][2 * j] = pack_f16(w[0], w[1]);
                    p[0][2 * j + 1] = pack_f16(w[2], w[3]);
                    if (SPLIT == 2) {
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] -= __half2float(__float2half_rn(w[e]));
                        p[SPLIT - 1][2 * j] = pack_f16(w[0], w[1]);
                        p[SPLIT - 1][2 * j + 1] = pack_f16(w[2], w[3]);
                    }
                }
#pragma unroll
                for (int i = 0; i < DP / 16; i++) {
                    uint32_t v[4];
                    const int t = 16 * b + (lane & 15);
                    load_matrix_t(v, s_v + t * ROW + 16 * ((2 * i + (lane >> 4)) ^ (t & 7)));
#pragma unroll
                    for (int z = 0; z < SPLIT; z++) {
                        mma_f16(acc[2 * i], p[z][0], p[z][1], p[z][2], p[z][3], v[0], v[1]);
                        mma_f16(acc[2 * i + 1], p[z][0], p[z][1], p[z][2], p[z][3], v[2], v[3]);
                    }
                }
            }
            };
            if (whole) weigh(std::true_type{});
            else weigh(std::false_type{});
        }
        cp_async_wait<0>();

        // ---- a warp's columns are its own: finished, or a part of a split tile ----
        const bool split = first < walk.begin || tile1 > walk.end;
        const float unscale = vtop / kWeightTop;
        float* part = a.parts + ((size_t)2 * blockIdx.x + (first >= walk.begin)) * a.part_floats;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float sum = l[e];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int k = 16 * warp + g + 8 * e;
#pragma unroll
            for (int i = 0; i < DP / 8; i++) {
                // a quad's lanes trade pairs, so that each holds four dims in a row
                const float x0 = acc[i][2 * e] * unscale, x1 = acc[i][2 * e + 1] * unscale;
                const float y0 = __shfl_xor_sync(0xffffffffu, x0, 1), y1 = __shfl_xor_sync(0xffffffffu, x1, 1);
                const int d = 8 * i + 2 * (q4 & 2);
                if (k >= cols || d >= hd || (q4 & 1) != (i & 1)) continue;
                float x[4] = {q4 & 1 ? y0 : x0, q4 & 1 ? y1 : x1, q4 & 1 ? x0 : y0, q4 & 1 ? x1 : y1};
                if (split) *reinterpret_cast<float4*>(part + 2 * kManyCols + (size_t)k * hd + d) = make_float4(x[0], x[1], x[2], x[3]);
                else kv_finish<DT>(a, seg.row + k / heads, h0 + k % heads, hd, d, x, m[e], sum);
            }
            if (split && q4 == 0 && k < cols) {
                part[k] = m[e];
                part[kManyCols + k] = sum;
            }
        }
        if (split && first >= walk.begin && tid == 0)
            a.splits[blockIdx.x] = {(int)walk.owner(tile1 - 1) - (int)blockIdx.x + 1, cols, heads, seg.row, h0};
        __syncthreads();
        unit = min(tile1, walk.end);
    }
}

}  // namespace hale
