// The scales that the product's workgroups read, checked against the rows of scales that there are: prints how many reads of
// how many lie past them, for workgroups of one to sixteen panels, four to a wavefront.
#include <cstdio>

#include "../telmo_amd/csrc/e4m3_product.hpp"

int main() {
    long past = 0, wrong = 0, tried = 0;
    for (size_t n = 1; n <= 5000; n++) {
        const size_t panels = tg::div_ceil(n, 16), rows = tg::div_ceil(n, 128);
        for (size_t width : {1, 2, 4, 8, 16})  // panels of a workgroup
            for (size_t panel0 = 0; panel0 < panels; panel0 += width)
                for (size_t panel = panel0; panel < panel0 + width; panel += 4) {
                    const size_t row = tg::e4m3_scale_row(panel, panels);
                    past += row >= rows;
                    wrong += panel < panels && row != panel * 16 / 128;
                    tried++;
                }
    }
    printf("%ld %ld %d\n", past, wrong, tried > 1000000);
    return 0;
}
