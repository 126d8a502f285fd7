// Attention over 16-bit rows by the tiles of attn_tile16.hpp.
#include "attn_tile16.hpp"

namespace tg {

namespace {

template <typename T, int D>
hipError_t launch_kind(const AttnArgs &a, int splits, hipStream_t s) {
    return a.seqs.tables ? launch_extra<T, T, D, true>(a, splits, s) : launch_extra<T, T, D, false>(a, splits, s);
}

template <typename T>
hipError_t launch_size(const AttnArgs &a, int splits, hipStream_t s) {
    if (a.d <= 64) return launch_kind<T, 64>(a, splits, s);
    if (a.d <= 128) return launch_kind<T, 128>(a, splits, s);
    return launch_kind<T, 256>(a, splits, s);
}

}  // namespace

hipError_t launch_attention16(const AttnArgs &a, int splits, hipStream_t s) {
    return a.type == F16 ? launch_size<_Float16>(a, splits, s) : launch_size<__bf16>(a, splits, s);
}

}  // namespace tg
