// Prints what the kernels make of row numbers, lengths, tables and windows from device memory, for
// sequences read from stdin: the clamps that keep their reads inside the buffers, run on the host.
#include <cstdio>
#include <vector>

#include "../telmo_amd/csrc/attn_common.hpp"

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
        for (int b = 0; b < batch; b++) {
            const tg::AttnSpan p = tg::span_of(s, b);
            printf("%d %d %d %d", p.q0, p.nq, p.k0, p.nk);
            if (paged)
                for (int j = 0; j < p.nk; j++) printf(" %d", tg::page_of(s, b, j));
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
    return 0;
}
