// The product of rows and weights in e4m3 (kernels_e4m3.hip): its operands, and the workspace of the rounded rows.
#pragma once

#include <type_traits>

#include "tg_internal.hpp"

namespace tg {

// Weights in fragments: panels of 16 outputs, each its blocks of 128 inputs one after another (2 KB each); scales [outputs /
// 128, rounded up][blocks].
struct E4m3Panels {
    const uint8_t *values;
    const float *scales;
    size_t panels, blocks;
};
// The row of scales of a panel's outputs, eight panels each. Workgroups reach past the last panel, whose row stands for
// those that there are not.
__host__ __device__ inline size_t e4m3_scale_row(size_t panel, size_t panels) { return (panel < panels ? panel : panels - 1) / 8; }
inline size_t e4m3_weight_bytes(size_t n, size_t k) { return div_ceil(n, 16) * div_ceil(k, 128) * 2048; }

// Outputs: m rows of n, ld apart, of a type of rows. aligned: four of a row from a multiple of four on lie aligned.
struct E4m3Out {
    void *c;
    size_t ld, m, n;
    uint32_t type;
    bool aligned;
    EpiArgs epi;
};

// Rounded rows in fragments: tiles of 16 rows, each its blocks one after another; and 2^e of each row's block as a byte e
// + 127, those of four blocks a word: [quads of blocks][tiles][16 rows].
struct Rounded {
    uint8_t *values;
    uint32_t *powers;
    size_t tiles, blocks, quads;
};
// Tiles of 128 x 128 outputs that a call may have: as workgroups of 256 threads, or a quarter as many of 512, a launch's
// threads stay below 2^32. Their outputs in 16 bits fill a GPU's memory.
constexpr size_t E4M3_TILES = (size_t)1 << 23;
inline bool e4m3_fits(size_t m, size_t n) { return div_ceil(m, 128) * div_ceil(n, 128) <= E4M3_TILES; }
// Rows that are rounded as they are read, without a workspace.
constexpr size_t E4M3_FEW = 16;
inline size_t e4m3_work_bytes(size_t m, size_t k) {
    if (m <= E4M3_FEW) return 0;
    const size_t tiles = div_ceil(m, 16), blocks = div_ceil(k, 128);
    return tiles * blocks * 2048 + div_ceil(blocks, 4) * tiles * 64 + 1024;  // whole kilobytes of powers are copied
}
inline Rounded rounded_at(void *work, size_t m, size_t k) {
    Rounded r;
    r.tiles = div_ceil(m, 16), r.blocks = div_ceil(k, 128), r.quads = div_ceil(r.blocks, 4);
    r.values = static_cast<uint8_t *>(work);
    r.powers = reinterpret_cast<uint32_t *>(r.values + r.tiles * r.blocks * 2048);
    return r;
}

hipError_t launch_e4m3_weights(const uint8_t *src, size_t ld, size_t n, size_t k, uint8_t *out, hipStream_t s);
// type: of a. work: e4m3_work_bytes(m, k) bytes, 16-byte aligned.
hipError_t launch_e4m3_product(uint32_t type, const void *a, size_t lda, size_t k, const E4m3Panels &w, const E4m3Out &o,
                               void *work, hipStream_t s);

}  // namespace tg
