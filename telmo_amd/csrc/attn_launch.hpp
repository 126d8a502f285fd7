// The attention launchers behind launch_attention.
#pragma once

#include "tg_internal.hpp"

namespace tg {

// Workgroups of 256 threads that a grid holds.
constexpr size_t MAX_ATTN_BLOCKS = ((size_t)1 << 32) / 256 - 1;

// 16-bit rows; the keys in `splits` parts (a.work holds them) where that is more than one.
hipError_t launch_attention16(const AttnArgs &a, int splits, hipStream_t s);

// f32 rows; with position rows only heads of up to 128 (attention32_fits).
inline bool attention32_fits(const AttnArgs &a) { return !a.rel || a.d <= 128; }
// Tiles of 64 or 128 query rows.
hipError_t launch_attention32(const AttnArgs &a, int rows, int splits, hipStream_t s);

// Few query rows of any type, without position rows and documents.
inline bool attention_few_fits(const AttnArgs &a) {
    return !a.rel && !a.q_docs && (size_t)a.seqs.longest * (a.heads / a.kv_heads) <= 16;
}
hipError_t launch_attention_few(const AttnArgs &a, int splits, hipStream_t s);

}  // namespace tg
