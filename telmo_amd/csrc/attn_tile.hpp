// What the tile kernels share: the order of workgroups, the tiles of keys that a range of queries needs,
// exchanges between a wavefront's halves, and where a tile's 16-byte chunks lie in LDS.
#pragma once

#include "attn_common.hpp"

namespace tg {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

// The greater (the sum) of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Where the 16-byte chunk c of a tile's row of CHUNKS chunks lies. K rows are read one chunk of 32 rows at a
// time and V rows 64 bytes of four rows at a time: either way the chunks of one read fall on different banks.
template <int CHUNKS>
__device__ __forceinline__ int k_place(int row, int c) {
    return row * CHUNKS + (c ^ (CHUNKS == 8 ? (row >> 1) & 7 : row & 15));
}
template <int CHUNKS>
__device__ __forceinline__ int v_place(int row, int c) {
    return row * CHUNKS + (c ^ (CHUNKS == 8 ? (row << 1) & 4 : (row & 3) << 2));
}

// Columns 32 x + (lane % 32) of eight rows of a 16-bit tile, the operand V' of 16 keys from row on, in the
// order in which the first product leaves the keys in a lane: rows 4 (lane / 32) + 0 .. 3, then those 8 on.
// Two reads of four rows each, transposed by the read.
template <int CHUNKS>
__device__ __forceinline__ s16x8 v_fragment(const void *tile, int row, int x, int lane) {
    const int r = row + (lane >> 5) * 4 + (lane & 15) / 4, c = x * 32 + (lane >> 4 & 1) * 16 + lane % 4 * 4;
    const short *v = static_cast<const short *>(tile);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4 *)(v + v_place<CHUNKS>(r, c / 8) * 8 + c % 8));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4 *)(v + v_place<CHUNKS>(r + 8, c / 8) * 8 + c % 8));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The key tiles that a range of query positions needs: those of the prefix, then those of the window.
template <int TILE_K>
struct Tiles {
    int front, start, count;
    __device__ __forceinline__ Tiles(const AttnWindow &first, const AttnWindow &last) {
        front = (first.prefix + TILE_K - 1) / TILE_K;
        start = first.lo / TILE_K > front ? first.lo / TILE_K : front;
        const int end = (last.hi + TILE_K - 1) / TILE_K;
        count = front + (end > start ? end - start : 0);
    }
    __device__ __forceinline__ int at(int n) const { return (n < front ? n : start + n - front) * TILE_K; }
};

// A workgroup's place in the call. Heads that share a key head are rows of one matrix: pair g r + x is head x
// of the group in query row r (g is 1 where each head has position rows of its own). Workgroups go round the
// 8 XCDs in turn: those of one head and part share an XCD and its L2, the rows with the most keys (the last
// ones of causal calls) first.
struct Place {
    int b, head, part, group;  // head: of k where the group shares a tile, of q otherwise
    int64_t pair0, pairs;      // the tile's first pair, the sequence's pairs
    AttnSpan sp;
    __device__ __forceinline__ bool find(const AttnArgs &a, int parts, int q_tiles, int groups, int heads, int tile_q) {
        const int id = blockIdx.x, in_xcd = id / 8;
        const int at = (in_xcd / q_tiles) * 8 + id % 8, tile = q_tiles - 1 - in_xcd % q_tiles;
        if (at >= groups) return false;
        part = at % parts;
        head = at / parts % heads;
        b = at / parts / heads;
        group = a.heads / heads;
        sp = span_of(a.seqs, b);
        pairs = (int64_t)(sp.nq < a.seqs.longest ? sp.nq : a.seqs.longest) * group;
        pair0 = (int64_t)tile * tile_q;
        return pair0 < pairs;
    }
};

}  // namespace tg
