// Prints what the kernels make of row numbers, lengths, tables and windows from device memory, for
// sequences read from stdin: the clamps that keep their reads inside the buffers, run on the host.
#include <cstdio>
#include <vector>

#include "../telmo_amd/csrc/attn_common.hpp"

// As the entry points set it.
static void set_division(tg::AttnSeqs &s) {
    s.page_shift = 31;
    while ((1ull << (s.page_shift - 31)) < (uint64_t)s.page) s.page_shift++;
    s.page_mul = (uint32_t)(((1ull << s.page_shift) + s.page - 1) / s.page);
}

int main() {
    int batch, q_rows, k_rows, paged, width, page, pages;
    while (scanf("%d %d %d %d %d %d %d", &batch, &q_rows, &k_rows, &paged, &width, &page, &pages) == 7) {
        std::vector<int> qs(batch + 1), ks(batch + 1), lens(batch), table((size_t)batch * width);
        for (int &x : qs) scanf("%d", &x);
        for (int &x : ks) scanf("%d", &x);
        for (int &x : lens) scanf("%d", &x);
        for (int &x : table) scanf("%d", &x);
        tg::AttnSeqs s{};
        s.batch = batch, s.q_rows = q_rows, s.k_rows = k_rows;
        s.q_starts = qs.data(), s.k_starts = ks.data();
        if (paged) s.tables = table.data(), s.lengths = lens.data();
        s.ldt = width, s.width = width, s.page = page, s.pages = pages;
        set_division(s);
        for (int b = 0; b < batch; b++) {
            const tg::AttnSpan p = tg::span_of(s, b);
            printf("%d %d %d %d", p.q0, p.nq, p.k0, p.nk);
            if (paged)
                for (int j = 0, row; j < p.nk; j++) printf(" %d", tg::page_of(s, b, j, row));
            printf("\n");
        }
    }
    const int cases[][5] = {{0, 10, -1, -1, 0},          {5, 10, 2, 0, 0},  {-7, 10, 2, 3, 0},
                            {2147483647, 10, 0, 0, 99},  {5, 10, 2147483647, 2147483647, -4},
                            {-2147483647, 10, 2147483647, 0, 3}};
    for (const auto &c : cases) {
        const tg::AttnWindow w = tg::window_of(c[0], c[1], c[2], c[3], c[4]);
        printf("w %d %d %d\n", w.lo, w.hi, w.prefix);
    }
    // The division by multiplication, at the multiples of many page sizes and beside them.
    long wrong = 0, tried = 0;
    for (uint64_t page = 1; page <= 1u << 30; page += page / 97 + 1) {
        tg::AttnSeqs s{};
        s.page = (int)page;
        set_division(s);
        const uint64_t most = 0x7fffffffull / page;
        for (uint64_t n = 0; n <= most; n += n / 13 + 1)
            for (int d = -1; d <= 1; d++) {
                const uint64_t j = n * page + d;
                if (j > 0x7fffffffull) continue;
                wrong += (j * s.page_mul >> s.page_shift) != j / page, tried++;
            }
        wrong += (0x7fffffffull * s.page_mul >> s.page_shift) != most;
    }
    printf("d %ld %d\n", wrong, tried > 100000);
    return 0;
}
