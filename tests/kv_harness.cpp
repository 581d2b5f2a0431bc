// Host build of the cache's index arithmetic (hale_kv_index.h) for
// test_kv8_cpu.py: reads "n_pages nkv hd page_log2 n_seqs max_pages seq pos
// head page" lines and prints "page code scale slot" of each; every table
// entry holds `page`.
#include <cstdio>
#include <vector>

#include "../hale-token_b200/csrc/hale_kv_index.h"

int main() {
    hale::KvShape s;
    int seq, head, page;
    long long pos;
    while (std::scanf("%d %d %d %d %d %d %d %lld %d %d", &s.n_pages, &s.nkv, &s.hd, &s.page_log2, &s.n_seqs, &s.max_pages,
                      &seq, &pos, &head, &page) == 10) {
        std::vector<int32_t> table((size_t)s.n_seqs * s.max_pages, page);
        const int p = s.page_of(table.data(), seq, pos), slot = s.slot(pos < 0 ? 0 : pos);
        std::printf("%d %zu %zu %d\n", p, s.code_at(p < 0 ? 0 : p, head, slot), s.scale_at(p < 0 ? 0 : p, head, slot), slot);
    }
    return 0;
}
