// What the tile kernels share: the order of workgroups, the tiles of keys that a range of queries needs,
// exchanges between a wavefront's halves, and where a tile's 16-byte chunks lie in LDS.
#pragma once

#include "attn_common.hpp"

namespace tg {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

// Eight values as N bf16 parts that each cut eight bits off what is left: exact, and an infinity or NaN stays one.
template <int N>
__device__ __forceinline__ void cut_parts(const float *x, bf16x8 (&part)[N]) {
    for (int e = 0; e < 8; e++) {
        float left = x[e];
        for (int n = 0; n < N; n++) {
            const float cut = left - left == 0.0f ? __uint_as_float(__float_as_uint(left) & 0xffff0000u) : left;
            part[n][e] = (__bf16)cut;
            left = cut - cut == 0.0f ? left - cut : 0.0f;
        }
    }
}

// The greater (the sum) of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The same over the four lanes 16 apart.
__device__ __forceinline__ float max_quarters(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_quarters(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Values between the rows of a tile of 16-bit values in LDS. K rows are read 16 bytes of 16 rows at a time and V rows
// 64 bytes of four rows at a time: with 16 bytes (64 bytes) between the ends of the rows the pieces of one read fall on
// different banks, and all pieces that a lane reads lie at constants from one address.
template <int D>
constexpr int K_PITCH = D + 8;
template <int D>
constexpr int V_PITCH = D + 32;

// The lane's place in a tile of K: columns 8 (lane / 32) on of row lane % 32, the operand K of the first 32 rows and 16
// columns; and in a tile of V: where its transposing reads of the first 16 rows and 32 columns begin.
template <int D>
__device__ __forceinline__ int k_lane(int lane) {
    return (lane & 31) * K_PITCH<D> + (lane >> 5) * 8;
}
template <int D>
__device__ __forceinline__ int v_lane(int lane) {
    return ((lane >> 5) * 4 + (lane & 15) / 4) * V_PITCH<D> + (lane >> 4 & 1) * 16 + lane % 4 * 4;
}
// Columns 32 x + (lane % 32) of 16 rows from row 16 g on, the operand V', in the order in which the first product leaves
// the keys in a lane: rows 4 (lane / 32) + 0 .. 3, then those 8 on. Two reads of four rows each, transposed by the read.
template <int D>
__device__ __forceinline__ s16x8 v_fragment(const void *at, int g, int x) {
    const short *v = static_cast<const short *>(at) + g * 16 * V_PITCH<D> + x * 32;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)v);
    const s16x4 hi =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(v + 8 * V_PITCH<D>));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The end of a region without branches of N x PRODUCTS matrix products, each group of them fed by READS reads of LDS,
// of which the program has issued the first AHEAD groups' before the region: fixes the order that the next group's
// reads follow each group's products. Left to itself the compiler reads an operand just before the product that takes
// it and waits out LDS's latency every time.
template <int N, int READS, int AHEAD, int PRODUCTS = 1>
__device__ __forceinline__ void feed() {
#pragma unroll
    for (int n = 0; n < N; n++) {
        __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
        if (n + AHEAD < N) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
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

// The keys kb + bit that a query is shown, as bits: its window and prefix, without those that have no page, and with
// documents (DOCS) its own: the lane holds key kb + lane's document in `docs` and its query's in `doc`. The
// documents of a tile are few: each is compared once.
__device__ __forceinline__ uint64_t bits_below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }
template <bool DOCS, int TILE_K>
__device__ __forceinline__ uint64_t shown_bits(const AttnWindow &w, int kb, uint64_t homeless, int docs, int doc) {
    uint64_t bits = (bits_below(w.hi - kb) & ~bits_below(w.lo - kb)) | bits_below(w.prefix - kb);
    bits &= ~homeless;
    if (DOCS) {
        uint64_t mine = 0, left = bits_below(TILE_K);
        while (left) {
            const int d = __builtin_amdgcn_readlane(docs, __builtin_ctzll(left));
            const uint64_t same = __ballot(docs == d);
            if (doc == d) mine = same;
            left &= ~same;
        }
        bits &= doc < 0 ? 0 : mine;
    }
    return bits;
}
// Whether all of a tile's keys and the wavefront's queries are of one document.
__device__ __forceinline__ bool one_document(int docs, int doc) {
    const int first = __builtin_amdgcn_readfirstlane(docs);
    return first >= 0 && __all(docs == first && doc == first);
}
// All bits where the one is set, else none; and s where all are, else -infinity.
__device__ __forceinline__ uint32_t shown_mask(uint32_t bits, int bit) {
    return (uint32_t)((int32_t)(bits << (31 - bit)) >> 31);
}
__device__ __forceinline__ float shown_or_not(float s, uint32_t all) {
    return __uint_as_float((__float_as_uint(s) & all) | (0xff800000u & ~all));
}
__device__ __forceinline__ float shown_or_not(float s, uint32_t bits, int bit) {
    return shown_or_not(s, shown_mask(bits, bit));
}

// A workgroup's place in the call. Heads that share a key head are rows of one matrix: pair g r + x is head x
// of the group in query row r (g is 1 where each head has position rows of its own). Workgroups go round the
// 8 XCDs in turn, and here round the heads and parts: where those are a multiple of 8 all tiles of one share an XCD
// and its L2, otherwise they spread over all XCDs. The rows with the most keys (the last ones of causal calls) come
// first.
struct Place {
    int b, head, part, group;  // head: of k where the group shares a tile, of q otherwise
    int pair0, pairs;          // the tile's first pair, the sequence's pairs: 2^24 tiles of 128 at most
    AttnSpan sp;
    __device__ __forceinline__ bool find(const AttnArgs &a, int parts, int q_tiles, int groups, int heads, int tile_q) {
        const uint32_t tiles = blockIdx.x / (uint32_t)groups, at = blockIdx.x - tiles * (uint32_t)groups;
        const uint32_t set = at / (uint32_t)parts;
        const int tile = q_tiles - 1 - (int)tiles;
        part = (int)(at - set * (uint32_t)parts);
        b = (int)(set / (uint32_t)heads);
        head = (int)(set - (uint32_t)b * (uint32_t)heads);
        group = (int)((uint32_t)a.heads / (uint32_t)heads);
        sp = span_of(a.seqs, b);
        pairs = (sp.nq < a.seqs.longest ? sp.nq : a.seqs.longest) * group;
        pair0 = tile * tile_q;
        return pair0 < pairs;
    }
    // The query row of a pair, and its head in the group.
    __device__ __forceinline__ int row_of(int pair) const { return (int)((uint32_t)pair / (uint32_t)group); }
    __device__ __forceinline__ int head_of(int pair) const { return pair - row_of(pair) * group; }
};

// Where a thread's pieces of a tile of keys come from: pieces u = 0 .. PER - 1 are its column of rows row0 + u STEP
// of the tile. Offsets within a tile fit 32 bits (tile_strides_fit); the tile's own, and its pages', are scalars
// where STEP rows lie in one page. Rows past the last key are read as that one: they are hidden, and their values
// are some row's. Lane n of each wavefront looks up the tile's key n a tile ahead: its page and row in it, or its
// document.
template <typename T, int TILE_K, int PER, int STEP, bool PAGED>
struct KeyRows {
    static constexpr int64_t SIZE = sizeof(T);
    const char *k, *v;      // the head's first row
    uint32_t k_row, v_row;  // bytes between rows
    uint32_t column;        // bytes of the thread's column
    uint32_t k_off, v_off;  // bytes from the first of its rows to its piece
    int row0;
    int page, at;           // the lane's key's
    __device__ __forceinline__ KeyRows(const AttnArgs &a, const AttnSpan &sp, int kvh, int row0_, int col) {
        k = static_cast<const char *>(a.k) + ((PAGED ? 0 : sp.k0 * a.ldk) + kvh * a.hsk) * SIZE;
        v = static_cast<const char *>(a.v) + ((PAGED ? 0 : sp.k0 * a.ldv) + kvh * a.hsv) * SIZE;
        k_row = (uint32_t)(a.ldk * SIZE), v_row = (uint32_t)(a.ldv * SIZE);
        column = (uint32_t)(col * SIZE);
        row0 = row0_;
        k_off = row0 * k_row + column, v_off = row0 * v_row + column;
        page = at = 0;
    }
    // Looks up the keys of the tile at kb.
    __device__ __forceinline__ void look(const AttnArgs &a, const AttnSpan &sp, int b, int kb, int lane) {
        if (!PAGED) return;
        const int j = kb + lane % TILE_K;
        page = page_of(a.seqs, b, j < sp.nk ? j : sp.nk - 1, at);
    }
    // The keys of the tile that was looked up last that have no page.
    __device__ __forceinline__ uint64_t homeless() const { return PAGED ? __ballot(page < 0) : 0; }
    // f(u, key address, value address) for the tile at kb, the last one that was looked up.
    template <typename F>
    __device__ __forceinline__ void each(const AttnArgs &a, const AttnSpan &sp, int kb, F f) const {
        if (PAGED && a.seqs.page % STEP) {
#pragma unroll
            for (int u = 0; u < PER; u++) {
                const int p = __shfl(page, row0 + u * STEP), s = __shfl(at, row0 + u * STEP);
                const int64_t q = p < 0 ? 0 : p;
                f(u, k + q * (a.psk * SIZE) + ((uint64_t)(uint32_t)s * k_row + column),
                  v + q * (a.psv * SIZE) + ((uint64_t)(uint32_t)s * v_row + column));
            }
            return;
        }
        // STEP rows from key `first` (or from the last key, where they lie past it).
        const auto bases = [&](int u, int first, int64_t &kat, int64_t &vat) {
            if (PAGED) {
                const int p = __builtin_amdgcn_readlane(page, u * STEP), s = __builtin_amdgcn_readlane(at, u * STEP);
                const int64_t q = p < 0 ? 0 : p;
                kat = q * (a.psk * SIZE) + (uint64_t)(uint32_t)s * k_row;
                vat = q * (a.psv * SIZE) + (uint64_t)(uint32_t)s * v_row;
            } else {
                kat = (uint64_t)(uint32_t)first * k_row;
                vat = (uint64_t)(uint32_t)first * v_row;
            }
        };
        int64_t kat, vat;
        if (kb + TILE_K <= sp.nk) {
#pragma unroll
            for (int u = 0; u < PER; u++) {
                bases(u, kb + u * STEP, kat, vat);
                f(u, k + kat + k_off, v + vat + v_off);
            }
            return;
        }
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int first = kb + u * STEP, low = first < sp.nk ? first : sp.nk - 1;
            bases(u, low, kat, vat);
            const uint32_t row = first + row0 < sp.nk ? row0 : sp.nk - 1 - low;
            f(u, k + kat + (row * k_row + column), v + vat + (row * v_row + column));
        }
    }
};
// Whether offsets within a tile of keys fit 32 bits.
inline bool tile_strides_fit(const AttnArgs &a) {
    const int64_t most = INT32_MAX / 64 / 4;
    return a.ldk <= most && a.ldv <= most;
}

}  // namespace tg
