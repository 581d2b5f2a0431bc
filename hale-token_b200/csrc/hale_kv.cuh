// hale_kv.cuh -- a paged key/value cache held in 8 bits: rows quantised into
// it and read back, attention over it, and the bookkeeping of its pages.
//
// One layer's keys (values alike) are int8 codes [page][kv head][token][dim];
// 16 consecutive tokens of a kv head share one f32 scale, and a code c stands
// for c * scale. The reference keeps f32 keys and values in one growing buffer
// per layer (src/model/attention.rs:59-85) and has no counterpart.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "hale_device.cuh"
#include "hale_kv_index.h"

namespace hale {

// One layer of a cache (pointers already at the layer) and its tables.
struct KvArgs : KvShape {
    int8_t *k, *v;
    float *ks, *vs;
    int32_t *table, *lens, *refs;
    uint32_t* err;
};

// Four consecutive values of a float type (DT 0 f32, 1 f16, 2 bf16) as f32;
// p at a multiple of four elements from a 16-byte boundary.
template <int DT>
__device__ __forceinline__ void load4(const void* p, size_t i, float (&x)[4]) {
    if (DT == 0) {
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
        if (DT == 1) {
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
            const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
            x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
        } else {
            x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
            x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
        }
    }
}

template <int DT>
__device__ __forceinline__ float load1(const void* p, size_t i) {
    if (DT == 0) return reinterpret_cast<const float*>(p)[i];
    const uint16_t h = reinterpret_cast<const uint16_t*>(p)[i];
    return DT == 1 ? half_bits_to_float(h) : __uint_as_float((uint32_t)h << 16);
}

// Rounded once, to nearest even, to the output's type.
template <int DT>
__device__ __forceinline__ void store1(void* p, size_t i, float x) {
    if (DT == 0) reinterpret_cast<float*>(p)[i] = x;
    else if (DT == 1) reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
    else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

template <int DT>
__device__ __forceinline__ void store4(void* p, size_t i, const float (&x)[4]) {
    if (DT == 0) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        uint2 v;
        if (DT == 1) {
            const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
            v = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
            const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
            v = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        }
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + i) = v;
    }
}

// ---------------------------------------------------------------------------
// rows into the cache
//
// The rows of one call that fall into one block of 16 tokens are written
// together: with a = the largest |x| of them (finite ones), want = a / 127,
// at least 2^-100 (so that no product below leaves the normal range), 0 when
// a = 0. A block whose first token is written starts anew, scale = want;
// otherwise scale = max(old scale, want), and the codes already there are
// rounded to the new scale when it grew. code = x / scale, rounded half to
// even on the exact quotient: the rounding does not depend on how a compiler
// or another program forms x / scale.
// ---------------------------------------------------------------------------

// |a| / 127 as the block's scale.
__device__ __forceinline__ float kv_want(float amax) {
    if (!(amax > 0.0f)) return 0.0f;
    return fmaxf(__fdiv_rn(amax, 127.0f), 0x1p-100f);
}

// x / s rounded half to even on the exact quotient, |x| <= 127 s(1 + 2^-23),
// inv = 1 / s rounded. q = rint(x * inv) is off by at most one; r = x - q s is
// exact in one fused step (q is the nearest integer or next to it, so r is a
// multiple of the operands' last place and fits), and comparing 2 |r| with s
// decides. NaN counts as 0.
__device__ __forceinline__ int kv_code(float x, float s, float inv) {
    if (!(fabsf(x) <= 0x1.fffffep127f)) return x != x ? 0 : (x > 0.0f ? 127 : -127);
    float q = rintf(__fmul_rn(x, inv));
    const float r = __fmaf_rn(-q, s, x), two = 2.0f * fabsf(r);
    if (two > s || (two == s && ((int)q & 1))) q += r > 0.0f ? 1.0f : -1.0f;
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// A code moved to a larger scale: c * from / to, rounded as above (the product
// has 31 bits and the quotient of two such numbers is never closer to a half
// than 2^-40 unless it is one, so 64-bit arithmetic rounds it right).
__device__ __forceinline__ int kv_recode(int c, float from, float to) {
    return (int)rint((double)c * (double)from / (double)to);
}

struct KvAppend {
    const void *k, *v;
    size_t k_stride, v_stride;  // elements between rows
    const int32_t *seqs, *positions;
    int n, rows_per_cta;
};

constexpr int kAppendRows = 32;  // most rows of one CTA

// (sequence, block) of row i, or -1 for a row to leave out.
__device__ __forceinline__ long long kv_row_key(const KvArgs& c, const KvAppend& a, int i) {
    const int s = a.seqs ? a.seqs[i] : 0, p = a.positions[i];
    if (s < 0 || p < 0) return -1;
    return ((long long)s << 32) | (unsigned)(p / kKvBlock);
}

// CTA x leads the blocks whose first row in the list is among its rows
// (rows_per_cta consecutive ones); it looks over the whole list for the other
// rows of those blocks (of two rows for one token the later one counts), then
// its warps take (block, head, keys or values) in turn, blockIdx.y splitting
// them over CTAs. A lane holds 4 NV dims of the block's 16 rows in registers:
// each value is read once, each code written once.
template <int DT, int NV>
__global__ void __launch_bounds__(256) kv_append_kernel(KvArgs c, KvAppend a) {
    __shared__ long long s_key[kAppendRows];
    __shared__ int s_first[kAppendRows], s_slot[kAppendRows][kKvBlock], s_late[kAppendRows];
    __shared__ int s_n;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r0 = blockIdx.x * a.rows_per_cta, r1 = min(a.n, r0 + a.rows_per_cta);
    if (tid < 32) {  // this CTA's candidates, in row order
        const int i = r0 + tid;
        long long key = -1;
        bool lead = false;
        if (i < r1) {
            key = kv_row_key(c, a, i);
            lead = key >= 0 && (i == 0 || kv_row_key(c, a, i - 1) != key);
        }
        const unsigned m = __ballot_sync(0xffffffffu, lead);
        if (lead) {
            const int at = __popc(m & ((1u << lane) - 1));
            s_key[at] = key;
            s_first[at] = i;
            s_late[at] = 0;
        }
        if (lane == 0) s_n = __popc(m);
    }
    for (int i = tid; i < kAppendRows * kKvBlock; i += 256) s_slot[i / kKvBlock][i % kKvBlock] = -1;
    __syncthreads();
    const int blocks = s_n;
    if (blocks == 0) return;
    auto look = [&](int i, int seq, int pos) {
        if (seq < 0 || pos < 0) return;
        const long long key = ((long long)seq << 32) | (unsigned)(pos / kKvBlock);
        for (int b = 0; b < blocks; b++) {
            if (s_key[b] != key) continue;
            if (i < s_first[b]) s_late[b] = 1;  // an earlier row leads this block
            else atomicMax(&s_slot[b][pos % kKvBlock], i);
        }
    };
    // four rows a load where both lists start on 16-byte boundaries
    const bool vec = ((reinterpret_cast<uintptr_t>(a.seqs) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0;
    const int n4 = vec ? a.n & ~3 : 0;
#pragma unroll 2
    for (int i = 4 * tid; i < n4; i += 4 * 256) {
        const int4 p = *reinterpret_cast<const int4*>(a.positions + i);
        const int4 s = a.seqs ? *reinterpret_cast<const int4*>(a.seqs + i) : make_int4(0, 0, 0, 0);
        look(i, s.x, p.x);
        look(i + 1, s.y, p.y);
        look(i + 2, s.z, p.z);
        look(i + 3, s.w, p.w);
    }
    for (int i = n4 + tid; i < a.n; i += 256) look(i, a.seqs ? a.seqs[i] : 0, a.positions[i]);
    __syncthreads();
    const int tasks = blocks * c.nkv * 2, step = 8 * gridDim.y;
    for (int t = warp + 8 * blockIdx.y; t < tasks; t += step) {
        const int b = t / (2 * c.nkv), head = (t >> 1) % c.nkv, is_v = t & 1;
        if (s_late[b]) continue;
        const int seq = (int)(s_key[b] >> 32);
        const long long pos = (s_key[b] & 0xffffffffll) * kKvBlock;
        const int page = c.page_of(c.table, seq, pos);
        if (page < 0) {
            if (lane == 0) raise_error(c.err, kErrBounds);
            continue;
        }
        const void* src = is_v ? a.v : a.k;
        const size_t stride = is_v ? a.v_stride : a.k_stride;
        int8_t* codes = (is_v ? c.v : c.k) + c.code_at(page, head, c.slot(pos));
        float* scale = (is_v ? c.vs : c.ks) + c.scale_at(page, head, c.slot(pos));
        float x[kKvBlock][NV][4];
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < kKvBlock; j++) {
            const int row = s_slot[b][j];
#pragma unroll
            for (int u = 0; u < NV; u++) {
                const int d = 4 * (lane + 32 * u);
                if (row >= 0 && d < c.hd) load4<DT>(src, (size_t)row * stride + (size_t)head * c.hd + d, x[j][u]);
                else x[j][u][0] = x[j][u][1] = x[j][u][2] = x[j][u][3] = 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < kKvBlock; j++)
#pragma unroll
            for (int u = 0; u < NV; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float m = fabsf(x[j][u][e]);
                    if (m <= 0x1.fffffep127f) amax = fmaxf(amax, m);  // NaN and infinities set no scale
                }
        amax = warp_max_abs(amax);
        float old = *scale;
        if (s_slot[b][0] >= 0 || !(old > 0.0f) || !(old <= 0x1.fffffep127f)) old = 0.0f;  // starts anew
        const float s = fmaxf(old, kv_want(amax));
        const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
        const bool grown = old > 0.0f && s > old;
        // x inv + 1.5 2^23 has the rounded quotient in its low byte; where the
        // remainder is half a code or more (a tie, a quotient rounded across
        // one, or no number) the lane's warp takes the careful path instead
        bool check = false;
        const float half = 0.5f * s;
#pragma unroll
        for (int j = 0; j < kKvBlock; j++) {
            if (s_slot[b][j] < 0) continue;
#pragma unroll
            for (int u = 0; u < NV; u++) {
                uint32_t t[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y = __fmaf_rn(x[j][u][e], inv, 12582912.0f);
                    check |= !(fabsf(__fmaf_rn(-(y - 12582912.0f), s, x[j][u][e])) < half);
                    t[e] = __float_as_uint(y);
                }
                const int d = 4 * (lane + 32 * u);
                if (d < c.hd)
                    *reinterpret_cast<uint32_t*>(codes + (size_t)j * c.hd + d) =
                        __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
            }
        }
        // the careful path, and codes that were there before; seldom, so kept
        // short (each pass of a kernel fetches its code anew)
        const bool again = __any_sync(0xffffffffu, check);
        if (again || grown) {
#pragma unroll 1
            for (int j = 0; j < kKvBlock; j++) {
                const int row = s_slot[b][j];
                if (row >= 0 ? !again : !grown) continue;
#pragma unroll 1
                for (int d = 4 * lane; d < c.hd; d += 128) {
                    uint32_t* at = reinterpret_cast<uint32_t*>(codes + (size_t)j * c.hd + d);
                    const uint32_t was = *at;
                    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (row >= 0) load4<DT>(src, (size_t)row * stride + (size_t)head * c.hd + d, y);
                    uint32_t w = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int q = row >= 0 ? kv_code(y[e], s, inv) : kv_recode((int8_t)(was >> (8 * e)), old, s);
                        w |= (uint32_t)(q & 0xff) << (8 * e);
                    }
                    *at = w;
                }
            }
        }
        __syncwarp();
        if (lane == 0) *scale = s;
    }
}

// Rows of the cache as the values they stand for: one warp per (row, head).
template <int DT>
__global__ void __launch_bounds__(256) kv_read_kernel(KvArgs c, const int32_t* __restrict__ seqs,
                                                      const int32_t* __restrict__ positions, int n, void* k_out,
                                                      void* v_out, size_t k_stride, size_t v_stride) {
    const size_t unit = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (unit >= (size_t)n * c.nkv) return;
    const int row = (int)(unit / c.nkv), head = (int)(unit % c.nkv);
    const int s = seqs ? seqs[row] : 0, p = positions[row];
    if (s < 0 || p < 0) return;
    const int page = c.page_of(c.table, s, p);
    if (page < 0) {
        if (lane == 0) raise_error(c.err, kErrBounds);
        return;
    }
    const int slot = c.slot(p);
    const size_t at = c.code_at(page, head, slot), sa = c.scale_at(page, head, slot);
    const float fk = c.ks[sa], fv = c.vs[sa];
    for (int d = 4 * lane; d < c.hd; d += 128) {
        const uint32_t wk = *reinterpret_cast<const uint32_t*>(c.k + at + d);
        const uint32_t wv = *reinterpret_cast<const uint32_t*>(c.v + at + d);
        float x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[e] = fmul((float)(int8_t)(wk >> (8 * e)), fk);
            y[e] = fmul((float)(int8_t)(wv >> (8 * e)), fv);
        }
        if (k_out) store4<DT>(k_out, (size_t)row * k_stride + (size_t)head * c.hd + d, x);
        if (v_out) store4<DT>(v_out, (size_t)row * v_stride + (size_t)head * c.hd + d, y);
    }
}

// ---------------------------------------------------------------------------
// pages
//
// refs[page] counts the table entries that name the page; 0 is a free page,
// so the free list is the table of counts itself and pages are handed out
// lowest number first: the result of a call depends on its arguments and the
// cache alone. The counting kernels are one CTA (the work is a scan of
// n_pages words); the pages themselves move in a second launch over the
// whole GPU.
// ---------------------------------------------------------------------------
constexpr int kPageThreads = 1024;
constexpr int kMaxListed = 16384;       // sequences named in one call
constexpr int kMaxKvSeqs = 1 << 18;
constexpr int kMaxKvPages = 1 << 20;

// Workspace of the page calls: pairs of pages to copy.
struct PagePairs {
    int32_t* count;
    int32_t *src, *dst;  // [kMaxKvPages / 2]
};

// Inclusive scan of v over the CTA (1024 threads); returns the thread's
// inclusive sum and sets the CTA's total.
__device__ __forceinline__ int cta_scan(int v, int* s_warp, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = s_warp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        s_warp[lane] = w;
    }
    __syncthreads();
    total = s_warp[31];
    return x + (warp ? s_warp[warp - 1] : 0);
}

// Sequences seqs[i] (NULL: i) get length new_lens[i]. First every shortened
// one gives up the pages behind its end. Then, in list order, each lengthened
// one gets the lowest free pages for its new tokens; when its last page is
// partly filled and shared it first gets its own copy of that page (the last
// sharer keeps the original). All or nothing: on a bad argument or too few
// free pages the error word is set and nothing changes.
// Dynamic shared memory: 2 n ints, n_seqs bits.
__global__ void __launch_bounds__(kPageThreads) kv_resize_kernel(KvArgs c, const int32_t* __restrict__ seqs,
                                                                 const int32_t* __restrict__ new_lens, int n,
                                                                 PagePairs out) {
    extern __shared__ int s_dyn[];
    int* s_off = s_dyn;        // [n] pages handed out before entry i
    int* s_last = s_dyn + n;   // [n] the partly filled last page of a growing entry, else -1
    unsigned* s_seen = reinterpret_cast<unsigned*>(s_dyn + 2 * n);
    __shared__ int s_warp[32];
    __shared__ int s_bad, s_pairs;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int pt = c.page_tokens();
    if (tid == 0) { s_bad = 0; s_pairs = 0; *out.count = 0; }
    for (int i = tid; i < (c.n_seqs + 31) / 32; i += kPageThreads) s_seen[i] = 0;
    __syncthreads();
    // arguments; every page that will be touched exists
    for (int i = tid; i < n; i += kPageThreads) {
        const int s = seqs ? seqs[i] : i, len = new_lens[i];
        s_last[i] = -1;
        if (s < 0 || s >= c.n_seqs || len < 0 || len > c.capacity()) { s_bad = 1; continue; }
        if (atomicOr(&s_seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) { s_bad = 1; continue; }
        const int old = c.lens[s];
        if (old < 0 || old > c.capacity()) { s_bad = 1; continue; }
        if (len > old && (old & (pt - 1))) {
            const int p = c.table[(size_t)s * c.max_pages + (old >> c.page_log2)];
            if (p < 0 || p >= c.n_pages) s_bad = 1;
            s_last[i] = p;
        }
    }
    __syncthreads();
    if (!s_bad) {
        for (int i = warp; i < n; i += 32) {
            const int s = seqs ? seqs[i] : i;
            const int from = (new_lens[i] + pt - 1) >> c.page_log2, to = (c.lens[s] + pt - 1) >> c.page_log2;
            for (int j = from + lane; j < to; j += 32) {
                const int p = c.table[(size_t)s * c.max_pages + j];
                if (p < 0 || p >= c.n_pages) s_bad = 1;
            }
        }
    }
    __syncthreads();
    if (s_bad) {
        if (tid == 0) raise_error(c.err, kErrBounds);
        return;
    }
    // counts of the pages given up (table entries stay until the end)
    for (int i = warp; i < n; i += 32) {
        const int s = seqs ? seqs[i] : i;
        const int from = (new_lens[i] + pt - 1) >> c.page_log2, to = (c.lens[s] + pt - 1) >> c.page_log2;
        for (int j = from + lane; j < to; j += 32) atomicSub(&c.refs[c.table[(size_t)s * c.max_pages + j]], 1);
    }
    __threadfence();
    __syncthreads();
    // demand of every entry, summed in list order
    int base = 0;
    for (int i0 = 0; i0 < n; i0 += kPageThreads) {
        const int i = i0 + tid;
        int want = 0;
        bool own = false;
        if (i < n) {
            const int s = seqs ? seqs[i] : i, len = new_lens[i], old = c.lens[s];
            if (len > old) want = ((len + pt - 1) >> c.page_log2) - ((old + pt - 1) >> c.page_log2);
            const int p = s_last[i];
            if (p >= 0) {
                const int shared = __ldcg(&c.refs[p]);
                if (shared > 1) {  // earlier entries of the list leave the page before this one
                    int before = 0;
                    for (int j = 0; j < i; j++) before += s_last[j] == p;
                    own = shared - before > 1;
                }
            }
            want += own;
        }
        int total;
        const int sum = cta_scan(want, s_warp, total);
        if (i < n) s_off[i] = (base + sum - want) | (own ? (int)0x80000000 : 0);
        base += total;
        __syncthreads();
    }
    const int demand = base;
    // enough free pages?
    int found = 0;
    for (int p0 = 0; p0 < c.n_pages && found < demand; p0 += 4 * kPageThreads) {
        int free = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int p = p0 + u * kPageThreads + tid;
            free += p < c.n_pages && __ldcg(&c.refs[p]) == 0;
        }
        int total;
        cta_scan(free, s_warp, total);
        found += total;
        __syncthreads();
    }
    if (found < demand) {
        for (int i = warp; i < n; i += 32) {
            const int s = seqs ? seqs[i] : i;
            const int from = (new_lens[i] + pt - 1) >> c.page_log2, to = (c.lens[s] + pt - 1) >> c.page_log2;
            for (int j = from + lane; j < to; j += 32) atomicAdd(&c.refs[c.table[(size_t)s * c.max_pages + j]], 1);
        }
        if (tid == 0) raise_error(c.err, kErrBounds);
        return;
    }
    // hand the lowest free pages out
    int given = 0;
    for (int p0 = 0; given < demand; p0 += kPageThreads) {
        const int p = p0 + tid;
        const int free = p < c.n_pages && __ldcg(&c.refs[p]) == 0;
        int total;
        const int g = given + cta_scan(free, s_warp, total) - free;
        if (free && g < demand) {
            int lo = 0, hi = n;  // the last entry whose offset is at most g
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if ((s_off[mid] & 0x7fffffff) <= g) lo = mid;
                else hi = mid;
            }
            const int own = s_off[lo] < 0, k = g - (s_off[lo] & 0x7fffffff);
            const int s = seqs ? seqs[lo] : lo, held = (c.lens[s] + pt - 1) >> c.page_log2;
            int* row = c.table + (size_t)s * c.max_pages;
            if (own && k == 0) {
                const int at = atomicAdd(&s_pairs, 1);
                out.src[at] = s_last[lo];
                out.dst[at] = p;
                atomicSub(&c.refs[s_last[lo]], 1);
                row[held - 1] = p;
            } else {
                row[held + k - own] = p;
            }
            c.refs[p] = 1;
        }
        given += total;
        __syncthreads();
    }
    // the entries given up, and the lengths
    for (int i = warp; i < n; i += 32) {
        const int s = seqs ? seqs[i] : i;
        const int from = (new_lens[i] + pt - 1) >> c.page_log2, to = (c.lens[s] + pt - 1) >> c.page_log2;
        for (int j = from + lane; j < to; j += 32) c.table[(size_t)s * c.max_pages + j] = -1;
        __syncwarp();
        if (lane == 0) c.lens[s] = new_lens[i];
    }
    if (tid == 0) *out.count = s_pairs;
}

// children[i] gives up its pages and shares parents[i]'s. One CTA per entry;
// each checks the whole list (a child once, never a parent), so that either
// all of them go ahead or none. Counts change by atomics on integers, whose
// order does not matter. Dynamic shared memory: n_seqs bits.
__global__ void __launch_bounds__(256) kv_fork_kernel(KvArgs c, const int32_t* __restrict__ parents,
                                                      const int32_t* __restrict__ children, int n) {
    extern __shared__ unsigned s_child[];
    const int tid = threadIdx.x;
    for (int i = tid; i < (c.n_seqs + 31) / 32; i += 256) s_child[i] = 0;
    __syncthreads();
    int bad = 0;
    for (int i = tid; i < n; i += 256) {
        const int s = children[i];
        if (s < 0 || s >= c.n_seqs) bad = 1;
        else if (atomicOr(&s_child[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) bad = 1;
    }
    bad = __syncthreads_or(bad);
    if (!bad)
        for (int i = tid; i < n; i += 256) {
            const int s = parents[i];
            if (s < 0 || s >= c.n_seqs || (s_child[s >> 5] >> (s & 31) & 1u)) bad = 1;
        }
    if (__syncthreads_or(bad)) {
        if (tid == 0 && blockIdx.x == 0) raise_error(c.err, kErrBounds);
        return;
    }
    const int parent = parents[blockIdx.x], child = children[blockIdx.x];
    const int32_t* from = c.table + (size_t)parent * c.max_pages;
    int32_t* to = c.table + (size_t)child * c.max_pages;
    for (int j = tid; j < c.max_pages; j += 256) {
        const int gone = to[j];
        int p = from[j];
        if (gone >= c.n_pages || p >= c.n_pages) raise_error(c.err, kErrBounds);
        if (gone >= 0 && gone < c.n_pages) atomicSub(&c.refs[gone], 1);
        if (p < 0 || p >= c.n_pages) p = -1;
        else atomicAdd(&c.refs[p], 1);
        to[j] = p;
    }
    if (tid == 0) c.lens[child] = c.lens[parent];
}

// The pages in use move to the front: with L of them, the k-th used page at L
// or above goes to the k-th free place below L. remap [2][n_pages]: the new
// number of every page (-1: it was free), and the old number of every page
// (-1 from L on).
__global__ void __launch_bounds__(kPageThreads) kv_compact_kernel(KvArgs c, int32_t* __restrict__ remap,
                                                                  int32_t* __restrict__ live, PagePairs out) {
    __shared__ int s_warp[32];
    const int tid = threadIdx.x;
    int32_t *to = remap, *from = remap + c.n_pages;
    int used = 0, total;
    for (int p = tid; p < c.n_pages; p += kPageThreads) used += c.refs[p] > 0;
    cta_scan(used, s_warp, total);
    const int L = total;
    int below = 0;
    for (int p = tid; p < L; p += kPageThreads) below += c.refs[p] > 0;
    __syncthreads();
    cta_scan(below, s_warp, total);
    const int kept = total, moved = L - kept;
    int base = 0;
    for (int p0 = 0; p0 < c.n_pages; p0 += kPageThreads) {
        const int p = p0 + tid;
        const int u = p < c.n_pages && c.refs[p] > 0;
        __syncthreads();
        const int rank = base + cta_scan(u, s_warp, total) - u;  // used pages before p
        if (p < c.n_pages) {
            to[p] = u && p < L ? p : -1;
            from[p] = u && p < L ? p : -1;
            if (!u && p < L) out.dst[p - rank] = p;
            if (u && p >= L) out.src[rank - kept] = p;
        }
        base += total;
    }
    __syncthreads();
    for (int i = tid; i < moved; i += kPageThreads) {
        const int s = out.src[i], d = out.dst[i];
        to[s] = d;
        from[d] = s;
        c.refs[d] = c.refs[s];
        c.refs[s] = 0;
    }
    if (tid == 0) {
        *out.count = moved;
        *live = L;
    }
}

// A list of pages to copy: every destination once, and never a source too
// (but a page onto itself, which is left alone). *count = n, or 0 with the
// error word set. Dynamic shared memory: n_pages bits.
__global__ void __launch_bounds__(kPageThreads) kv_check_pairs_kernel(KvArgs c, const int32_t* __restrict__ src,
                                                                      const int32_t* __restrict__ dst, int n,
                                                                      int32_t* count) {
    extern __shared__ unsigned s_dst[];
    const int tid = threadIdx.x;
    for (int i = tid; i < (c.n_pages + 31) / 32; i += kPageThreads) s_dst[i] = 0;
    __syncthreads();
    int bad = 0;
    for (int i = tid; i < n; i += kPageThreads) {
        const int d = dst[i], s = src[i];
        if (d < 0 || d >= c.n_pages || s < 0 || s >= c.n_pages) bad = 1;
        else if (atomicOr(&s_dst[d >> 5], 1u << (d & 31)) >> (d & 31) & 1u) bad = 1;
    }
    bad = __syncthreads_or(bad);
    if (!bad)
        for (int i = tid; i < n; i += kPageThreads)
            if (src[i] != dst[i] && (s_dst[src[i] >> 5] >> (src[i] & 31) & 1u)) bad = 1;
    bad = __syncthreads_or(bad);
    if (tid == 0) {
        *count = bad ? 0 : n;
        if (bad) raise_error(c.err, kErrBounds);
    }
}

// Pages src[i] -> dst[i] of every layer, codes and scales; remap, when given,
// also renumbers the table. A piece is one (pair, layer, keys or values);
// every thread keeps four 16-byte copies in flight.
__global__ void __launch_bounds__(256) kv_move_kernel(KvArgs c, int n_layers, const int32_t* __restrict__ count,
                                                      const int32_t* __restrict__ src,
                                                      const int32_t* __restrict__ dst,
                                                      const int32_t* __restrict__ remap) {
    const int tid = threadIdx.x;
    if (remap) {
        const size_t n = (size_t)c.n_seqs * c.max_pages;
        for (size_t i = (size_t)blockIdx.x * 256 + tid; i < n; i += (size_t)gridDim.x * 256) {
            const int p = c.table[i];
            if (p >= c.n_pages) raise_error(c.err, kErrBounds);
            else if (p >= 0) c.table[i] = remap[p];
        }
    }
    const size_t bytes = ((size_t)c.nkv << c.page_log2) * c.hd, scales = ((size_t)c.nkv << c.page_log2) / kKvBlock;
    const size_t vecs = bytes / 16, pieces = (size_t)*count * n_layers * 2;
    for (size_t i = blockIdx.x; i < pieces; i += gridDim.x) {
        const size_t pair = i / (2 * n_layers);
        const int layer = (int)(i / 2 % n_layers), s = src[pair], d = dst[pair];
        if (s == d) continue;
        const size_t first = (size_t)layer * c.n_pages;
        int8_t* codes = (i & 1) ? c.v : c.k;
        float* sc = (i & 1) ? c.vs : c.ks;
        const uint4* a = reinterpret_cast<const uint4*>(codes + (first + s) * bytes);
        uint4* b = reinterpret_cast<uint4*>(codes + (first + d) * bytes);
        size_t j = tid;
        for (; j + 3 * 256 < vecs; j += 4 * 256) {
            const uint4 x0 = __ldcs(a + j), x1 = __ldcs(a + j + 256), x2 = __ldcs(a + j + 512), x3 = __ldcs(a + j + 768);
            __stcs(b + j, x0);
            __stcs(b + j + 256, x1);
            __stcs(b + j + 512, x2);
            __stcs(b + j + 768, x3);
        }
        for (; j < vecs; j += 256) b[j] = a[j];
        for (size_t t = tid; t < scales; t += 256) sc[(first + d) * scales + t] = sc[(first + s) * scales + t];
    }
}

}  // namespace hale
