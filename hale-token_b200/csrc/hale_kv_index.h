// hale_kv_index.h -- where a token of the paged 8-bit cache lies. Plain C++:
// the kernels and the host-side tests compile the same arithmetic.
#pragma once

#include <cstddef>
#include <cstdint>

#ifdef __CUDACC__
#define HALE_KV_HD __host__ __device__ __forceinline__
#else
#define HALE_KV_HD inline
#endif

namespace hale {

constexpr int kKvBlock = 16;  // tokens that share a scale

struct KvShape {
    int n_pages, nkv, hd, page_log2, n_seqs, max_pages;

    HALE_KV_HD int page_tokens() const { return 1 << page_log2; }
    // tokens a sequence can have
    HALE_KV_HD long long capacity() const { return (long long)max_pages << page_log2; }
    HALE_KV_HD int slot(long long pos) const { return (int)(pos & (page_tokens() - 1)); }
    // index of a token's first code and of its scale within a layer
    HALE_KV_HD size_t code_at(int page, int head, int slot) const {
        return ((((size_t)page * nkv + head) << page_log2) + slot) * hd;
    }
    HALE_KV_HD size_t scale_at(int page, int head, int slot) const {
        return ((((size_t)page * nkv + head) << page_log2) + slot) / kKvBlock;
    }
    HALE_KV_HD int checked(int page) const { return page >= 0 && page < n_pages ? page : -1; }
    // the page of a sequence's token, -1 when there is none or an argument is
    // out of range (the table is then not read)
    HALE_KV_HD int page_of(const int32_t* table, int seq, long long pos) const {
        if (seq < 0 || seq >= n_seqs || pos < 0 || pos >= capacity()) return -1;
        return checked(table[(size_t)seq * max_pages + (size_t)(pos >> page_log2)]);
    }
};

}  // namespace hale
