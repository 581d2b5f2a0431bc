// hale_serving.cu -- C ABI (include/hale_cuda.h) of the paged 8-bit key/value
// cache and of draft verification: argument checks and launches. The
// arithmetic lives in hale_kv.cuh and hale_verify.cuh.
#include "hale_host.h"

#include "hale_kv.cuh"
#include "hale_kv_attn.cuh"
#include "hale_verify.cuh"

#include <algorithm>
#include <cmath>

using namespace hale;

namespace {

// The calling thread's device while a call works on the context's.
struct OnDevice {
    int before = -1;
    cudaError_t err;
    explicit OnDevice(const hale_ctx* ctx) {
        int cur = 0;
        err = cudaGetDevice(&cur);
        if (err == cudaSuccess && cur != ctx->device) {
            err = cudaSetDevice(ctx->device);
            if (err == cudaSuccess) before = cur;
        }
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// Workspace of these calls: allocated once per context at its final size, so
// that a captured graph's addresses stay good for the context's life.
struct ServingWs {
    static constexpr size_t kPairsOff = 256;
    static constexpr size_t kPairsBytes = (size_t)kMaxKvPages / 2 * 4;
    static constexpr size_t kPartsOff = kPairsOff + 2 * kPairsBytes;
    static constexpr size_t kSplitsOff = kPartsOff + (size_t)kVerifyParts * sizeof(VerifyPart);
    static constexpr size_t kAttnOff = kSplitsOff + kAttnMaxGrid * sizeof(KvSplit);
    static constexpr size_t kTotal = kAttnOff + kAttnPartBytes;
    uint8_t* base;
    PagePairs pairs() const {
        return {reinterpret_cast<int32_t*>(base), reinterpret_cast<int32_t*>(base + kPairsOff),
                reinterpret_cast<int32_t*>(base + kPairsOff + kPairsBytes)};
    }
    VerifyPart* parts() const { return reinterpret_cast<VerifyPart*>(base + kPartsOff); }
    KvSplit* splits() const { return reinterpret_cast<KvSplit*>(base + kSplitsOff); }
    float* attn_parts() const { return reinterpret_cast<float*>(base + kAttnOff); }
};

hale_status serving_ws(hale_ctx* ctx, void* stream, ServingWs* out) {
    if (!ctx->serving_ws) {
        if (stream_capturing(stream))
            return fail(ctx, HALE_E_INVALID_ARGUMENT,
                        "the first such call on a context makes its workspace and cannot be captured; make one before");
        void* p = nullptr;
        CUDA_TRY(ctx, cudaMalloc(&p, ServingWs::kTotal));
        const cudaError_t e = cudaMemset(p, 0, ServingWs::kTotal);
        if (e != cudaSuccess) {
            cudaFree(p);
            return fail(ctx, HALE_E_CUDA, "clearing the workspace failed: %s", cudaGetErrorString(e));
        }
        CUDA_TRY(ctx, cudaStreamSynchronize(nullptr));
        ctx->serving_ws = p;
    }
    out->base = static_cast<uint8_t*>(ctx->serving_ws);
    return HALE_OK;
}

hale_status check_cache(hale_ctx* ctx, const hale_kv8* kv, const char* what) {
    if (!ctx) return fail(nullptr, HALE_E_INVALID_ARGUMENT, "%s: ctx is NULL", what);
    if (!kv) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: the cache is NULL", what);
    if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale || !kv->table || !kv->lens || !kv->refs)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: a buffer of the cache is NULL", what);
    if (!aligned16(kv->k) || !aligned16(kv->v))
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: the cache's codes must start on 16-byte boundaries", what);
    const uint32_t pt = kv->page_tokens;
    if (kv->head_dim == 0 || kv->head_dim % 16 || kv->head_dim > 256)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: head_dim %u (a multiple of 16 up to 256)", what, kv->head_dim);
    if (pt < HALE_KV8_BLOCK || pt > 256 || (pt & (pt - 1)))
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: page_tokens %u (16, 32, 64, 128 or 256)", what, pt);
    if (kv->n_layers == 0 || kv->n_layers > 65536 || kv->n_kv_heads == 0 || kv->n_kv_heads > 1024)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %u layers of %u kv heads", what, kv->n_layers, kv->n_kv_heads);
    if (kv->n_pages == 0 || kv->n_pages > (uint32_t)kMaxKvPages || kv->n_seqs == 0 || kv->n_seqs > (uint32_t)kMaxKvSeqs)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %u pages, %u sequences (up to 2^20 and 2^18)", what, kv->n_pages,
                    kv->n_seqs);
    if (kv->max_pages == 0 || (uint64_t)kv->max_pages * pt > 0x7fffff00ull)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %u pages of %u tokens a sequence (positions are 32-bit)", what,
                    kv->max_pages, pt);
    return HALE_OK;
}

KvArgs layer_args(const hale_ctx* ctx, const hale_kv8* kv, uint32_t layer) {
    KvArgs c{};
    const size_t tokens = (size_t)layer * kv->n_pages * kv->n_kv_heads * kv->page_tokens;
    c.k = kv->k + tokens * kv->head_dim;
    c.v = kv->v + tokens * kv->head_dim;
    c.ks = kv->k_scale + tokens / kKvBlock;
    c.vs = kv->v_scale + tokens / kKvBlock;
    c.table = kv->table;
    c.lens = kv->lens;
    c.refs = kv->refs;
    c.n_pages = (int)kv->n_pages;
    c.nkv = (int)kv->n_kv_heads;
    c.hd = (int)kv->head_dim;
    for (uint32_t p = kv->page_tokens; p > 1; p >>= 1) c.page_log2++;
    c.n_seqs = (int)kv->n_seqs;
    c.max_pages = (int)kv->max_pages;
    c.err = ctx->d_err;
    return c;
}

// Rows of heads * head_dim values, `stride` elements apart.
hale_status check_rows(hale_ctx* ctx, const char* what, const char* name, const void* p, hale_dtype dt, uint64_t stride,
                       uint64_t width) {
    const uint64_t el = dt == HALE_F32 ? 4 : 2;
    if (!p) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %s is NULL", what, name);
    if (stride < width || stride > (1ull << 40))
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: rows of %s are %llu elements apart, a row has %llu", what, name,
                    (unsigned long long)stride, (unsigned long long)width);
    if (!aligned16(p) || stride * el % 16)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: rows of %s must start on 16-byte boundaries", what, name);
    return HALE_OK;
}

constexpr uint32_t kMaxRows = 1u << 22;  // rows of one call

hale_status check_layer_rows(hale_ctx* ctx, const hale_kv8* kv, const char* what, uint32_t layer, hale_dtype dt,
                             const int32_t* positions, uint32_t n) {
    if (layer >= kv->n_layers)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: layer %u of %u", what, layer, kv->n_layers);
    if (!is_float(dt)) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: rows must be f32, f16 or bf16", what);
    if (n > kMaxRows) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %u rows (up to 2^22)", what, n);
    if (!positions) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: positions is NULL", what);
    return HALE_OK;
}

// CTAs of an attention launch: what the GPU holds at once, no more than there
// can be units of CH tokens, and no more than the workspace has parts for.
unsigned attn_grid(const hale_ctx* ctx, const KvArgs& c, const KvAttn& a, int per_sm, int chunk, int cost) {
    const uint64_t units = (uint64_t)a.n * c.nkv * a.subs * ((uint64_t)c.capacity() / chunk + 1 + cost);
    const uint64_t parts = kAttnPartBytes / 8 / a.part_floats;
    return (unsigned)std::min<uint64_t>({(uint64_t)ctx->sm_count * per_sm, units, parts, (uint64_t)kAttnMaxGrid});
}

// Rows of one launch: units are counted in 32 bits.
uint32_t attn_rows(const KvArgs& c, const KvAttn& a, int chunk, int cost) {
    const uint64_t row = (uint64_t)c.nkv * a.subs * ((uint64_t)c.capacity() / chunk + 1 + cost);
    const uint64_t rows = std::max<uint64_t>(1, 0x7fffffffull / row) / a.rows * a.rows;
    return (uint32_t)std::min<uint64_t>((uint64_t)a.n, std::max<uint64_t>(rows, (uint64_t)a.rows));
}

// Rows i .. i + n - 1 of a call.
template <int DT>
KvAttn attn_part(const KvAttn& a, uint32_t i, uint32_t n) {
    constexpr size_t el = DT == 0 ? 4 : 2;
    KvAttn b = a;
    b.q = static_cast<const char*>(a.q) + i * a.q_stride * el;
    b.out = static_cast<char*>(a.out) + i * a.out_stride * el;
    b.lse = a.lse ? a.lse + (size_t)i * a.nh : nullptr;
    b.seqs = a.seqs ? a.seqs + i : nullptr;
    b.positions = a.positions + i;
    b.n = (int)n;
    return b;
}

// The joining launch may begin while the CTAs before it finish (it waits for
// them itself).
template <int DT>
hale_status attn_join(hale_ctx* ctx, const KvAttn& a, int hd, int cols, unsigned grid, cudaStream_t st) {
    if (grid == 1) return HALE_OK;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kv_join_kernel<DT>, a, hd, cols));
    return check_launch(ctx, "kv_join");
}

template <int DT, int DP, int HD, int NT>
hale_status attn_few(hale_ctx* ctx, const KvArgs& c, KvAttn a, uint32_t run, cudaStream_t st) {
    constexpr int cols = 8 * NT;
    a.heads = std::min(a.group, cols);
    a.subs = (a.group + a.heads - 1) / a.heads;
    a.rows = (int)std::max<uint32_t>(1u, std::min<uint32_t>(run, (uint32_t)(cols / a.heads)));
    a.part_floats = cols * (2 + c.hd);
    const size_t smem = std::max((size_t)kFewWarps * cols * DP * 4, (size_t)kFewWarps * FewCfg<DP>::RING);
    CUDA_TRY(ctx, allow_smem(kv_attn_few_kernel<DT, DP, HD, NT>, smem));
    const uint32_t step = attn_rows(c, a, FewCfg<DP>::CH, kFewCost), n = (uint32_t)a.n;
    for (uint32_t i = 0; i < n; i += step) {
        const KvAttn b = attn_part<DT>(a, i, std::min(step, n - i));
        const unsigned grid = attn_grid(ctx, c, b, DP <= 128 && NT == 1 ? 3 : 2, FewCfg<DP>::CH, kFewCost);
        kv_attn_few_kernel<DT, DP, HD, NT><<<grid, kFewThreads, smem, st>>>(c, b);
        if (hale_status r = check_launch(ctx, "kv_attn_few")) return r;
        if (hale_status r = attn_join<DT>(ctx, b, c.hd, cols, grid, st)) return r;
    }
    return HALE_OK;
}

template <int DT, int DP>
hale_status attn_many(hale_ctx* ctx, const KvArgs& c, KvAttn a, uint32_t run, cudaStream_t st) {
    using Cfg = ManyCfg<DT, DP>;
    a.heads = std::min(a.group, kManyCols);
    a.subs = (a.group + a.heads - 1) / a.heads;
    a.rows = (int)std::max<uint32_t>(1u, std::min<uint32_t>(run, (uint32_t)(kManyCols / a.heads)));
    a.part_floats = kManyCols * (2 + c.hd);
    CUDA_TRY(ctx, allow_smem(kv_attn_many_kernel<DT, DP>, Cfg::SMEM));
    const uint32_t step = attn_rows(c, a, Cfg::UT, kManyCost), n = (uint32_t)a.n;
    for (uint32_t i = 0; i < n; i += step) {
        const KvAttn b = attn_part<DT>(a, i, std::min(step, n - i));
        const unsigned grid = attn_grid(ctx, c, b, Cfg::PER_SM, Cfg::UT, kManyCost);
        kv_attn_many_kernel<DT, DP><<<grid, kManyThreads, Cfg::SMEM, st>>>(c, b);
        if (hale_status r = check_launch(ctx, "kv_attn_many")) return r;
        if (hale_status r = attn_join<DT>(ctx, b, c.hd, kManyCols, grid, st)) return r;
    }
    return HALE_OK;
}

template <int DT>
hale_status attn_go(hale_ctx* ctx, const KvArgs& c, const KvAttn& a, uint32_t run, cudaStream_t st) {
    const uint64_t cols = (uint64_t)std::min<uint32_t>(run, (uint32_t)a.n) * a.group;
    // the kernels of a known head size take two blocks of 16 tokens from one page
    const int hd = c.page_log2 == 4 ? 0 : c.hd;
    if (cols <= 8) {
        switch (hd) {
        case 64: return attn_few<DT, 64, 64, 1>(ctx, c, a, run, st);
        case 128: return attn_few<DT, 128, 128, 1>(ctx, c, a, run, st);
        case 256: return attn_few<DT, 256, 256, 1>(ctx, c, a, run, st);
        default: return c.hd <= 128 ? attn_few<DT, 128, 0, 1>(ctx, c, a, run, st) : attn_few<DT, 256, 0, 1>(ctx, c, a, run, st);
        }
    }
    if (cols <= 16 && c.hd <= 128) {
        switch (hd) {
        case 64: return attn_few<DT, 64, 64, 2>(ctx, c, a, run, st);
        case 128: return attn_few<DT, 128, 128, 2>(ctx, c, a, run, st);
        default: return attn_few<DT, 128, 0, 2>(ctx, c, a, run, st);
        }
    }
    if (c.hd <= 64) return attn_many<DT, 64>(ctx, c, a, run, st);
    if (c.hd <= 128) return attn_many<DT, 128>(ctx, c, a, run, st);
    return attn_many<DT, 256>(ctx, c, a, run, st);
}

template <int DT>
void append_go(const KvArgs& c, const KvAppend& a, dim3 grid, cudaStream_t st) {
    if (c.hd <= 128) kv_append_kernel<DT, 1><<<grid, 256, 0, st>>>(c, a);
    else kv_append_kernel<DT, 2><<<grid, 256, 0, st>>>(c, a);
}

}  // namespace

extern "C" hale_status hale_kv8_append(hale_ctx* ctx, const hale_kv8* kv, uint32_t layer, const void* k, const void* v,
                                       hale_dtype dtype, uint64_t k_stride, uint64_t v_stride, const int32_t* seqs,
                                       const int32_t* positions, uint32_t n, void* stream) try {
    const char* what = "hale_kv8_append";
    hale_status r = check_cache(ctx, kv, what);
    if (r) return r;
    if (n == 0) return HALE_OK;
    const uint64_t width = (uint64_t)kv->n_kv_heads * kv->head_dim;
    if ((r = check_layer_rows(ctx, kv, what, layer, dtype, positions, n)) ||
        (r = check_rows(ctx, what, "k", k, dtype, k_stride, width)) ||
        (r = check_rows(ctx, what, "v", v, dtype, v_stride, width)))
        return r;
    // every CTA looks over the whole list: 2^18 rows are some milliseconds
    if (n > (1u << 18)) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %u rows (up to 2^18)", what, n);
    OnDevice on(ctx);
    CUDA_TRY(ctx, on.err);
    const KvArgs c = layer_args(ctx, kv, layer);
    KvAppend a{k, v, k_stride, v_stride, seqs, positions, (int)n, 1};
    // A CTA of one row keeps the heads of a decode step's rows apart (64 rows
    // of 8 heads: 128 CTAs). In long lists 15 of 16 such CTAs would lead no
    // block, and every one of them reads the whole list: 32 rows then.
    if (n > 1024) a.rows_per_cta = kAppendRows;
    const dim3 grid((n + a.rows_per_cta - 1) / a.rows_per_cta,
                    a.rows_per_cta == 1 ? std::min(64u, (2u * c.nkv + 7) / 8) : 1u);
    ProfScope ps(ctx, "kv8_append", S(stream));
    switch (dtype) {
    case HALE_F32: append_go<0>(c, a, grid, S(stream)); break;
    case HALE_F16: append_go<1>(c, a, grid, S(stream)); break;
    default: append_go<2>(c, a, grid, S(stream)); break;
    }
    return check_launch(ctx, "kv_append");
} catch (...) {
    return HALE_E_OUT_OF_MEMORY;
}

extern "C" hale_status hale_kv8_read(hale_ctx* ctx, const hale_kv8* kv, uint32_t layer, const int32_t* seqs,
                                     const int32_t* positions, uint32_t n, void* k_out, void* v_out, hale_dtype dtype,
                                     uint64_t k_stride, uint64_t v_stride, void* stream) try {
    const char* what = "hale_kv8_read";
    hale_status r = check_cache(ctx, kv, what);
    if (r) return r;
    if (n == 0) return HALE_OK;
    const uint64_t width = (uint64_t)kv->n_kv_heads * kv->head_dim;
    if ((r = check_layer_rows(ctx, kv, what, layer, dtype, positions, n))) return r;
    if (k_out && (r = check_rows(ctx, what, "k_out", k_out, dtype, k_stride, width))) return r;
    if (v_out && (r = check_rows(ctx, what, "v_out", v_out, dtype, v_stride, width))) return r;
    if (!k_out && !v_out) return HALE_OK;
    OnDevice on(ctx);
    CUDA_TRY(ctx, on.err);
    const KvArgs c = layer_args(ctx, kv, layer);
    const unsigned grid = (unsigned)(((uint64_t)n * c.nkv + 7) / 8);
    ProfScope ps(ctx, "kv8_read", S(stream));
    cudaStream_t st = S(stream);
    switch (dtype) {
    case HALE_F32: kv_read_kernel<0><<<grid, 256, 0, st>>>(c, seqs, positions, (int)n, k_out, v_out, k_stride, v_stride); break;
    case HALE_F16: kv_read_kernel<1><<<grid, 256, 0, st>>>(c, seqs, positions, (int)n, k_out, v_out, k_stride, v_stride); break;
    default: kv_read_kernel<2><<<grid, 256, 0, st>>>(c, seqs, positions, (int)n, k_out, v_out, k_stride, v_stride); break;
    }
    return check_launch(ctx, "kv_read");
} catch (...) {
    return HALE_E_OUT_OF_MEMORY;
}

extern "C" hale_status hale_kv8_attention(hale_ctx* ctx, const hale_kv8* kv, uint32_t layer, const void* q,
                                          hale_dtype dtype, uint64_t q_stride, const int32_t* seqs,
                                          const int32_t* positions, uint32_t n, uint32_t n_heads, float scale,
                                          uint32_t window, uint32_t run, void* out, uint64_t out_stride, float* lse,
                                          void* stream) try {
    const char* what = "hale_kv8_attention";
    hale_status r = check_cache(ctx, kv, what);
    if (r) return r;
    if (n == 0) return HALE_OK;
    if (n_heads == 0 || n_heads > 65535 || n_heads % kv->n_kv_heads)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %u query heads over %u kv heads", what, n_heads, kv->n_kv_heads);
    if (!std::isfinite(scale)) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: scale is not finite", what);
    if (run == 0) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: run is 0", what);
    const uint64_t width = (uint64_t)n_heads * kv->head_dim;
    if ((r = check_layer_rows(ctx, kv, what, layer, dtype, positions, n)) ||
        (r = check_rows(ctx, what, "q", q, dtype, q_stride, width)) ||
        (r = check_rows(ctx, what, "out", out, dtype, out_stride, width)))
        return r;
    OnDevice on(ctx);
    CUDA_TRY(ctx, on.err);
    const KvArgs c = layer_args(ctx, kv, layer);
    // a row's units are counted in 32 bits (no tile has fewer than 32 tokens a unit)
    if ((uint64_t)kv->n_kv_heads * (n_heads / kv->n_kv_heads / 8 + 1) * ((uint64_t)c.capacity() / 32 + 8) > 0x7fffffffull)
        return fail(ctx, HALE_E_UNSUPPORTED, "%s: sequences of %u pages over %u heads are too long", what, kv->max_pages, n_heads);
    KvAttn a{};
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.seqs = seqs;
    a.positions = positions;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.n = (int)n;
    a.nh = (int)n_heads;
    a.group = (int)(n_heads / kv->n_kv_heads);
    a.window = (int)std::min<uint32_t>(window, 0x7fffffffu);
    a.scale = scale;
    ServingWs ws;
    if ((r = serving_ws(ctx, stream, &ws))) return r;
    a.parts = ws.attn_parts();
    a.splits = ws.splits();
    ProfScope ps(ctx, "kv8_attention", S(stream));
    switch (dtype) {
    case HALE_F32: return attn_go<0>(ctx, c, a, run, S(stream));
    case HALE_F16: return attn_go<1>(ctx, c, a, run, S(stream));
    default: return attn_go<2>(ctx, c, a, run, S(stream));
    }
} catch (...) {
    return HALE_E_OUT_OF_MEMORY;
}

// CTAs of the copying launch: enough 16 KB in flight on every SM.
static unsigned move_grid(const hale_ctx* ctx) { return (unsigned)ctx->sm_count * 8; }

extern "C" hale_status hale_kv8_resize(hale_ctx* ctx, const hale_kv8* kv, const int32_t* seqs, const int32_t* new_lens,
                                       uint32_t n, void* stream) try {
    const char* what = "hale_kv8_resize";
    hale_status r = check_cache(ctx, kv, what);
    if (r) return r;
    if (n == 0) return HALE_OK;
    if (!new_lens) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: new_lens is NULL", what);
    if (n > kv->n_seqs || n > (uint32_t)kMaxListed)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %u sequences listed (the cache has %u; up to %d a call)", what, n,
                    kv->n_seqs, kMaxListed);
    OnDevice on(ctx);
    CUDA_TRY(ctx, on.err);
    ServingWs ws;
    if ((r = serving_ws(ctx, stream, &ws))) return r;
    const KvArgs c = layer_args(ctx, kv, 0);
    const size_t smem = (size_t)n * 8 + (kv->n_seqs + 31) / 32 * 4;
    CUDA_TRY(ctx, allow_smem(kv_resize_kernel, smem));
    {
        ProfScope ps(ctx, "kv8_resize", S(stream));
        kv_resize_kernel<<<1, kPageThreads, smem, S(stream)>>>(c, seqs, new_lens, (int)n, ws.pairs());
    }
    if ((r = check_launch(ctx, "kv_resize"))) return r;
    ProfScope ps(ctx, "kv8_move", S(stream));
    kv_move_kernel<<<move_grid(ctx), 256, 0, S(stream)>>>(c, (int)kv->n_layers, ws.pairs().count, ws.pairs().src,
                                                          ws.pairs().dst, nullptr);
    return check_launch(ctx, "kv_move");
} catch (...) {
    return HALE_E_OUT_OF_MEMORY;
}

extern "C" hale_status hale_kv8_fork(hale_ctx* ctx, const hale_kv8* kv, const int32_t* parents, const int32_t* children,
                                     uint32_t n, void* stream) try {
    const char* what = "hale_kv8_fork";
    hale_status r = check_cache(ctx, kv, what);
    if (r) return r;
    if (n == 0) return HALE_OK;
    if (!parents || !children) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: parents or children is NULL", what);
    if (n >= kv->n_seqs || n > (uint32_t)kMaxListed)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %u children (the cache has %u sequences; up to %d a call)", what, n,
                    kv->n_seqs, kMaxListed);
    OnDevice on(ctx);
    CUDA_TRY(ctx, on.err);
    const KvArgs c = layer_args(ctx, kv, 0);
    const size_t smem = (kv->n_seqs + 31) / 32 * 4;
    CUDA_TRY(ctx, allow_smem(kv_fork_kernel, smem));
    ProfScope ps(ctx, "kv8_fork", S(stream));
    kv_fork_kernel<<<n, 256, smem, S(stream)>>>(c, parents, children, (int)n);
    return check_launch(ctx, "kv_fork");
} catch (...) {
    return HALE_E_OUT_OF_MEMORY;
}

extern "C" hale_status hale_kv8_compact(hale_ctx* ctx, const hale_kv8* kv, int32_t* remap, int32_t* live,
                                        void* stream) try {
    const char* what = "hale_kv8_compact";
    hale_status r = check_cache(ctx, kv, what);
    if (r) return r;
    if (!remap || !live) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: remap or live is NULL", what);
    OnDevice on(ctx);
    CUDA_TRY(ctx, on.err);
    ServingWs ws;
    if ((r = serving_ws(ctx, stream, &ws))) return r;
    const KvArgs c = layer_args(ctx, kv, 0);
    {
        ProfScope ps(ctx, "kv8_compact", S(stream));
        kv_compact_kernel<<<1, kPageThreads, 0, S(stream)>>>(c, remap, live, ws.pairs());
    }
    if ((r = check_launch(ctx, "kv_compact"))) return r;
    ProfScope ps(ctx, "kv8_move", S(stream));
    kv_move_kernel<<<move_grid(ctx), 256, 0, S(stream)>>>(c, (int)kv->n_layers, ws.pairs().count, ws.pairs().src,
                                                          ws.pairs().dst, remap);
    return check_launch(ctx, "kv_move");
} catch (...) {
    return HALE_E_OUT_OF_MEMORY;
}

extern "C" hale_status hale_kv8_copy(hale_ctx* ctx, const hale_kv8* kv, const int32_t* src, const int32_t* dst, uint32_t n,
                                     void* stream) try {
    const char* what = "hale_kv8_copy";
    hale_status r = check_cache(ctx, kv, what);
    if (r) return r;
    if (n == 0) return HALE_OK;
    if (!src || !dst) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: src or dst is NULL", what);
    if (n > kv->n_pages) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %u pairs, the cache has %u pages", what, n, kv->n_pages);
    OnDevice on(ctx);
    CUDA_TRY(ctx, on.err);
    ServingWs ws;
    if ((r = serving_ws(ctx, stream, &ws))) return r;
    const KvArgs c = layer_args(ctx, kv, 0);
    const size_t smem = (kv->n_pages + 31) / 32 * 4;
    CUDA_TRY(ctx, allow_smem(kv_check_pairs_kernel, smem));
    {
        ProfScope ps(ctx, "kv8_copy", S(stream));
        kv_check_pairs_kernel<<<1, kPageThreads, smem, S(stream)>>>(c, src, dst, (int)n, ws.pairs().count);
    }
    if ((r = check_launch(ctx, "kv_check_pairs"))) return r;
    ProfScope ps(ctx, "kv8_move", S(stream));
    kv_move_kernel<<<move_grid(ctx), 256, 0, S(stream)>>>(c, (int)kv->n_layers, ws.pairs().count, src, dst, nullptr);
    return check_launch(ctx, "kv_move");
} catch (...) {
    return HALE_E_OUT_OF_MEMORY;
}

extern "C" hale_status hale_verify_drafts(hale_ctx* ctx, const void* logits, hale_dtype dtype, uint64_t logits_stride,
                                          const int32_t* draft_tokens, const float* draft_probs, uint64_t probs_stride,
                                          const int32_t* n_draft, uint32_t batch, uint32_t max_draft, uint32_t vocab,
                                          double temperature, const float* uniforms, int32_t* out_tokens, int32_t* out_n,
                                          float* out_logp, void* stream) try {
    const char* what = "hale_verify_drafts";
    if (!ctx) return fail(nullptr, HALE_E_INVALID_ARGUMENT, "%s: ctx is NULL", what);
    if (batch == 0) return HALE_OK;
    const bool greedy = !(temperature > 0.0);
    if (!logits || !out_tokens || !out_n || (max_draft && !draft_tokens) || (!greedy && !uniforms))
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: NULL buffer", what);
    if (!is_float(dtype)) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: logits must be f32, f16 or bf16", what);
    if (std::isnan(temperature) || std::isinf(temperature))
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: temperature is not finite", what);
    if (max_draft > (uint32_t)kVerifyMaxDraft)
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %u drafted tokens (up to %d)", what, max_draft, kVerifyMaxDraft);
    // a CTA notes the mass of each 256 values in shared memory: 2^22 values are 128 KB
    if (vocab == 0 || vocab > (1u << 22)) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: vocab %u out of range", what, vocab);
    if (logits_stride < vocab || (draft_probs && probs_stride < vocab) || logits_stride > (1ull << 40) ||
        probs_stride > (1ull << 40))
        return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: rows are closer together than the vocabulary is long", what);
    const uint64_t rows = (uint64_t)batch * (max_draft + 1);
    if (rows > 65535) return fail(ctx, HALE_E_INVALID_ARGUMENT, "%s: %llu rows of logits (up to 65535)", what,
                                  (unsigned long long)rows);
    OnDevice on(ctx);
    CUDA_TRY(ctx, on.err);
    ServingWs ws;
    hale_status r = serving_ws(ctx, stream, &ws);
    if (r) return r;
    VerifyArgs a{};
    a.logits = logits;
    a.probs = greedy ? nullptr : draft_probs;
    a.draft = draft_tokens;
    a.n_draft = n_draft;
    a.u = uniforms;
    a.logits_stride = logits_stride;
    a.probs_stride = probs_stride;
    a.K = (int)max_draft;
    a.V = (int)vocab;
    // slices of one register tile, larger ones where the parts would not fit
    uint32_t tiles = (vocab + kVerifyTile - 1) / kVerifyTile;
    const uint32_t most = std::max<uint32_t>(1u, (uint32_t)(kVerifyParts / rows));
    const uint32_t per = (tiles + most - 1) / most;
    a.slice = (int)(per * kVerifyTile);
    a.slices = (int)((tiles + per - 1) / per);
    a.per_t = greedy ? 1.0 : 1.0 / temperature;
    a.greedy = greedy;
    a.parts = ws.parts();
    a.tokens = out_tokens;
    a.count = out_n;
    a.logp = out_logp;
    a.err = ctx->d_err;
    const dim3 grid((unsigned)a.slices, (unsigned)rows);
    cudaStream_t st = S(stream);
    {
        ProfScope ps(ctx, "verify_stats", st);
        switch (dtype) {
        case HALE_F32: verify_stats_kernel<0><<<grid, kVerifyThreads, 0, st>>>(a); break;
        case HALE_F16: verify_stats_kernel<1><<<grid, kVerifyThreads, 0, st>>>(a); break;
        default: verify_stats_kernel<2><<<grid, kVerifyThreads, 0, st>>>(a); break;
        }
    }
    if ((r = check_launch(ctx, "verify_stats"))) return r;
    // clusters of 8 CTAs, of fewer where the GPU would not hold them all at once
    // (two CTAs an SM)
    const unsigned ctas = std::max(1u, std::min((unsigned)kVerifyCluster, 2u * ctx->sm_count / batch));
    const size_t smem = (((size_t)vocab + kPickTile - 1) / kPickTile / ctas + 1) * 8;
    ProfScope ps(ctx, "verify_pick", st);
    auto pick = dtype == HALE_F32 ? verify_pick_kernel<0> : dtype == HALE_F16 ? verify_pick_kernel<1> : verify_pick_kernel<2>;
    CUDA_TRY(ctx, allow_smem(pick, smem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(batch * ctas);
    cfg.blockDim = dim3(kPickThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute shape{};
    shape.id = cudaLaunchAttributeClusterDimension;
    shape.val.clusterDim = {ctas, 1, 1};
    cfg.attrs = &shape;
    cfg.numAttrs = 1;
    CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, pick, a));
    return check_launch(ctx, "verify_pick");
} catch (...) {
    return HALE_E_OUT_OF_MEMORY;
}
