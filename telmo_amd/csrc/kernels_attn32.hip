// Attention over f32 rows on the matrix cores, tiles of 128 query rows by 32 keys, to f32's accuracy.
//
// The f32 matrix instructions run at a sixteenth of the 16-bit ones' rate, so each f32 operand is held as a sum of
// 16-bit ones. For the scores a row x of q, k or the position rows is scaled by a power of two to |x| < 2^15 and held
// as h + l in f16, 22 bits of each value within 2^-17 of the row's largest; three products h h', h l' and l h' leave out
// less than 2^-22 of such terms. Smaller values keep 2^-40 of the row's largest: where that can be more of a score than
// f32 sums lose (an outlier of q that meets zeros of k, with every other term far below it), the row is computed again
// by its definition. The weights
// and the values, which may not share a scale (a value is weighted by other rows' weights), are held as three bf16 each,
// 24 bits, and six products leave out less than 2^-23.
//
// The layout is that of the 16-bit kernel with 16 x 16 x 32 products: eight wavefronts of 16 queries each, a lane
// holding one query's scores with 8 of the 32 keys. Two wavefronts to a SIMD, so that one's splitting and exponentials
// run beside the other's products: 16 sequences of 750 rows of 8 heads of 128 with position rows take 307.5 us (180 TFLOP/s
// of f32, past the 154 that a large library product reaches on the f32 units), with four wavefronts of 32 queries,
// which read half as much LDS, 385. Bound by the splitting and the softmax on the vector units (43 % busy) in turn with
// the products (32 %). Tiles of 64 rows run the same with four wavefronts, for calls that leave CUs empty: there 32 keys
// take a workgroup 3.2 us and its start 10 (7 without position rows).
//
// Position rows: with T[c, i] = (q_i + w) r_c, the score of key j needs T[j - i, i]. The distances j - i of a
// wavefront's 16 queries and a tile's 32 keys lie in two blocks of 32 position rows, and the second one is the first
// of the next tile: each tile adds one product of 32 rows, kept in LDS as [query][64 distances], a ring of two blocks,
// from which a lane reads its own diagonal. Wavefronts whose queries are 32 apart use the same blocks tiles apart: LDS
// holds the last four. (q + w) r = (q + u) r + (w - u) r, the second part a number per position row, so one copy of
// the queries serves both products.
#include "attn_launch.hpp"
#include "attn_tile.hpp"

namespace tg {

namespace {

constexpr int TILE_K = 32;

// The power of two that brings a row whose largest magnitude is `top` below 2^15, and its inverse. Both stay
// normal numbers: a row of subnormals is scaled less, which loses nothing that f32 sums would keep.
struct Scale {
    float by, back;
};
__device__ __forceinline__ Scale scale_for(float top) {
    const int e = (int)(__float_as_uint(top) >> 23), s = 268 - e < 253 ? 268 - e : 253;
    return Scale{__uint_as_float((uint32_t)s << 23), __uint_as_float((uint32_t)(254 - s) << 23)};
}

// Eight values as sums of two f16 (three bf16) ones.
__device__ __forceinline__ void split2(const float *x, f16x8 &hi, f16x8 &lo) {
    f32x8 v, r;
    for (int e = 0; e < 8; e++) v[e] = x[e];
    hi = __builtin_convertvector(v, f16x8);
    for (int e = 0; e < 8; e++) r[e] = __builtin_fmaf((float)hi[e], -1.0f, v[e]);
    lo = __builtin_convertvector(r, f16x8);
}
struct Split3 {
    bf16x8 hi, mid, lo;
};
// Two values rounded to bf16 in one word, and what that leaves of them.
__device__ __forceinline__ uint32_t bf16_pair(float &a, float &b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
    a -= __uint_as_float(w << 16);
    b -= __uint_as_float(w & 0xffff0000u);
    return w;
}
__device__ __forceinline__ Split3 split3(const float *x) {
    u32x4 w[3];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float a = x[2 * e], b = x[2 * e + 1];
#pragma unroll
        for (int y = 0; y < 3; y++) w[y][e] = bf16_pair(a, b);
    }
    return Split3{__builtin_bit_cast(bf16x8, w[0]), __builtin_bit_cast(bf16x8, w[1]), __builtin_bit_cast(bf16x8, w[2])};
}

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Reductions over the CHUNKS neighbouring lanes that hold one row: quads, halves and whole rows of 16 lanes
// by the lane permutations that arithmetic instructions carry.
template <int CTRL>
__device__ __forceinline__ float lane_move(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
template <int CHUNKS>
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, lane_move<0xb1>(x));   // lanes 1 0 3 2
    x = fmaxf(x, lane_move<0x4e>(x));   // lanes 2 3 0 1
    x = fmaxf(x, lane_move<0x141>(x));  // mirrored in 8 lanes
    if (CHUNKS > 8) x = fmaxf(x, lane_move<0x140>(x));  // mirrored in 16
    if (CHUNKS > 16) x = fmaxf(x, __shfl_xor(x, 16));
    return x;
}
template <int CHUNKS>
__device__ __forceinline__ float row_sum(float x) {
    x += lane_move<0xb1>(x);
    x += lane_move<0x4e>(x);
    x += lane_move<0x141>(x);
    if (CHUNKS > 8) x += lane_move<0x140>(x);
    if (CHUNKS > 16) x += __shfl_xor(x, 16);
    return x;
}

// Values between the rows of a plane of V: its transposing reads take 32 bytes of eight rows at a time.
template <int D>
constexpr int V_STEP = D + 16;

template <int D, bool REL, int WAVES>
struct Shared {
    static constexpr int RING = WAVES / 2;  // blocks of position rows that the wavefronts use at a time
    _Float16 k[2][TILE_K * K_PITCH<D>];
    __bf16 v[3][TILE_K * V_STEP<D>];
    float k_back[TILE_K];
    _Float16 r[REL ? RING : 1][2][REL ? TILE_K * K_PITCH<D> : 8];
    float r_back[REL ? RING : 1][TILE_K], r_add[REL ? RING : 1][TILE_K];
    float terms[REL ? WAVES : 1][REL ? 16 * 64 : 1];  // per wavefront [query][64 distances], turned by 4 per query
};

// Columns 16 x + (lane % 16) of a plane's 32 rows, the operand V', in the order in which the score products leave the
// keys in a lane: rows 4 (lane / 16) + 0 .. 3 of the first 16 and of the last.
template <int D>
__device__ __forceinline__ bf16x8 v_columns(const __bf16 *at, int x) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(at + x * 16));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4 *)(at + 16 * V_STEP<D> + x * 16));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Eight values of a row of K or of position rows as they go into LDS.
struct Split2 {
    f16x8 hi, lo;
    float back, add;  // of the whole row: the scale's inverse, the product with wu
};
template <int CHUNKS>
__device__ __forceinline__ Split2 split_row(const float *x) {
    Split2 r;
    float top = 0.0f, y[8];
    for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e]));
    const Scale sc = scale_for(row_max<CHUNKS>(top));
    for (int e = 0; e < 8; e++) y[e] = x[e] * sc.by;
    split2(y, r.hi, r.lo);
    r.back = sc.back;
    r.add = 0.0f;
    return r;
}
// D: head size rounded up to 64, 128 or 256. EXTRA: scores are capped, biased or cut by documents.
template <int D, bool PAGED, bool EXTRA, bool REL, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void attn_tile32_kernel(
    const AttnArgs a, const AttnParts parts, const int q_tiles, const int groups) {
    constexpr int THREADS = 64 * WAVES, TILE_Q = 16 * WAVES, RING = Shared<D, REL, WAVES>::RING;
    // Where there are fewer pieces than threads, several threads handle each alike.
    constexpr int CHUNKS = D / 8, PIECES = TILE_K * CHUNKS, PER = PIECES > THREADS ? PIECES / THREADS : 1;
    constexpr int STEP = TILE_K / PER;
    constexpr int STEPS = D / 32;  // products along a row
    constexpr int AHEAD = 2;       // groups of operands on their way from LDS
    __shared__ __align__(16) Shared<D, REL, WAVES> sh;

    Place at;
    if (!at.find(a, parts.parts, q_tiles, groups, REL ? a.heads : a.kv_heads, TILE_Q)) return;
    const int part = at.part, b = at.b, group = at.group;
    const int kvh = REL ? at.head / (a.heads / a.kv_heads) : at.head;
    const AttnSpan sp = at.sp;
    const int pairs = at.pairs, pair0 = at.pair0;

    const int t = threadIdx.x, lane = t & 63, quarter = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);  // a scalar, and what follows from it
    const int prefix = a.prefix ? a.prefix[b] : 0;
    const int pair = pair0 + wave * 16 + col;
    const bool live = pair < pairs;
    const int r = live ? at.row_of(pair) : 0, h = at.head * group + (live ? at.head_of(pair) : 0);
    const int i = sp.shift() + r;
    const AttnWindow win = window_of(i, sp.nk, a.left, a.right, prefix);
    const int wave0 = pair0 + wave * 16, wave1 = wave0 + 15 < pairs - 1 ? wave0 + 15 : pairs - 1;
    const int pair1 = pair0 + TILE_Q - 1 < pairs - 1 ? pair0 + TILE_Q - 1 : pairs - 1;
    const auto window_at = [&](int p) {
        return window_of(sp.shift() + at.row_of(p), sp.nk, a.left, a.right, prefix);
    };
    const bool wave_live = wave0 < pairs;
    const AttnWindow w_first = window_at(wave_live ? wave0 : 0), w_last = window_at(wave_live ? wave1 : 0);
    const Tiles<TILE_K> tiles(window_at(pair0), window_at(pair1));
    const int n0 = (int)((int64_t)tiles.count * part / parts.parts);
    const int n1 = (int)((int64_t)tiles.count * (part + 1) / parts.parts);

    const int64_t row = (int64_t)sp.q0 + r;
    const int doc = a.q_docs ? (live ? a.q_docs[row] : -1) : 0;
    const float slope = EXTRA && a.slopes ? a.slopes[h] : 0.0f;

    // The lane's quarter of its query (plus u), split.
    f16x8 qh[STEPS], ql[STEPS];
    float q_back;
    {
        const float *q = static_cast<const float *>(a.q) + row * a.ldq + h * a.hsq;
        float x[STEPS][8], top = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int c = s * 32 + quarter * 8;
            const bool in = live && c < a.d;
            if (in) {
                load8(q + c, x[s]);
            } else {
                for (int e = 0; e < 8; e++) x[s][e] = 0.0f;
            }
            if (REL && a.rel_u && in)
                for (int e = 0; e < 8; e++) x[s][e] += a.rel_u[(int64_t)h * a.d + c + e];
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[s][e]));
        }
        const Scale sc = scale_for(max_quarters(top));
        q_back = sc.back;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            for (int e = 0; e < 8; e++) x[s][e] *= sc.by;
            split2(x[s], qh[s], ql[s]);
        }
    }

    // This thread's part of the tiles: rows row0 + u STEP, chunk c of each.
    const int row0 = t / CHUNKS % TILE_K, c = t % CHUNKS;
    const bool in_d = c * 8 < a.d;
    KeyRows<float, TILE_K, PER, STEP, PAGED> keys(a, sp, kvh, row0, in_d ? c * 8 : 0);
    const float *rp = REL ? a.rel + h * a.hsrel + (in_d ? c * 8 : 0) : nullptr;
    float kr[PER][8], vr[PER][8], rr[PER][8], wu[8];
    uint64_t homeless = 0;  // of the loaded tile's keys
    int doc_k = 0;          // the lane's key's document
    const auto look = [&](int kb) { keys.look(a, sp, b, kb, lane); };
    const auto load = [&](int kb) {
        homeless = keys.homeless();
        keys.each(a, sp, kb, [&](int u, const char *k, const char *v) {
            load8(reinterpret_cast<const float *>(k), kr[u]);
            load8(reinterpret_cast<const float *>(v), vr[u]);
        });
        if (EXTRA && a.q_docs) {
            const int j = kb + lane % TILE_K;
            doc_k = a.k_docs[sp.k0 + (j < sp.nk ? j : sp.nk - 1)];
        }
    };
    // Block n of position rows: distances 32 n - (the workgroup's first position) and on.
    const int first_i = sp.shift() + (int)pair0;
    const auto load_block = [&](int n, float(&x)[PER][8]) {
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int64_t distance = (int64_t)n * 32 - first_i + row0 + u * STEP;
            const int64_t at = distance < -a.rel_span ? 0 : distance > a.rel_span ? 2 * (int64_t)a.rel_span : distance + a.rel_span;
            load8(rp + at * a.ldrel, x[u]);
        }
    };
    // The columns that fill D up hold values of any kind: zeros in their place meet the queries' zeros.
    const auto fill = [&](float(&x)[PER][8]) {
        if (a.d < D)
#pragma unroll
            for (int u = 0; u < PER; u++)
                for (int e = 0; e < 8; e++) x[u][e] = in_d ? x[u][e] : 0.0f;
    };
    const auto split_block = [&](float(&x)[PER][8], Split2(&y)[PER]) {
        fill(x);
#pragma unroll
        for (int u = 0; u < PER; u++) {
            float add = 0.0f;
            for (int e = 0; e < 8; e++) add = __builtin_fmaf(wu[e], x[u][e], add);
            y[u] = split_row<CHUNKS>(x[u]);
            y[u].add = row_sum<CHUNKS>(add);
        }
    };
    const auto store_block = [&](int n, const Split2(&y)[PER]) {
        const int slot = n & (RING - 1);
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int brow = row0 + u * STEP, to = brow * K_PITCH<D> + c * 8;
            *reinterpret_cast<f16x8 *>(&sh.r[slot][0][to]) = y[u].hi;
            *reinterpret_cast<f16x8 *>(&sh.r[slot][1][to]) = y[u].lo;
            if (c == 0) {
                sh.r_back[slot][brow] = y[u].back;
                sh.r_add[slot][brow] = y[u].add;
            }
        }
    };
    // The three products of 32 rows (hi and lo, in LDS) with the queries: rows 16 x + 4 quarter + e in s[x][e].
    const int k_at = col * K_PITCH<D> + quarter * 8;
    const auto along = [&](const _Float16 *hi, const _Float16 *lo, f32x4(&s)[2]) {
        f16x8 xh[STEPS][2], xl[STEPS][2];
        const auto read = [&](int e) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                xl[e][x] = *reinterpret_cast<const f16x8 *>(lo + k_at + x * 16 * K_PITCH<D> + e * 32);
                xh[e][x] = *reinterpret_cast<const f16x8 *>(hi + k_at + x * 16 * K_PITCH<D> + e * 32);
            }
        };
        s[0] = s[1] = f32x4{};
#pragma unroll
        for (int e = 0; e < AHEAD; e++) read(e);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < STEPS; e++) {
            s[0] = mfma(xl[e][0], qh[e], s[0]);
            s[1] = mfma(xl[e][1], qh[e], s[1]);
            s[0] = mfma(xh[e][0], ql[e], s[0]);
            s[1] = mfma(xh[e][1], ql[e], s[1]);
            s[0] = mfma(xh[e][0], qh[e], s[0]);
            s[1] = mfma(xh[e][1], qh[e], s[1]);
            if (e + AHEAD < STEPS) read(e + AHEAD);
        }
        feed<STEPS, 4, AHEAD, 6>();
    };
    float widest = 0.0f;  // the largest inverse of a scale among the rows that the queries meet
    // T of block n for the wavefront's queries, into its ring of two blocks.
    const auto terms_of = [&](int n) {
        const int slot = n & (RING - 1);
        f32x4 s[2], back[2], add[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            back[x] = *reinterpret_cast<const f32x4 *>(&sh.r_back[slot][x * 16 + quarter * 4]);
            add[x] = *reinterpret_cast<const f32x4 *>(&sh.r_add[slot][x * 16 + quarter * 4]);
        }
        along(sh.r[slot][0], sh.r[slot][1], s);
#pragma unroll
        for (int x = 0; x < 2; x++) {
            f32x4 y;
            for (int e = 0; e < 4; e++) {
                y[e] = __builtin_fmaf(s[x][e], back[x][e] * q_back, add[x][e]);
                widest = fmaxf(widest, back[x][e]);
            }
            *reinterpret_cast<f32x4 *>(
                &sh.terms[wave][col * 64 + (((n & 1) * 32 + x * 16 + quarter * 4 + 4 * col) & 63)]) = y;
        }
    };
    // Where the term of the lane's key 16 x + 4 quarter + e lies when its block is an even one; the odd ones' lie 32 on
    // in the ring of 64, the bit of 32 turned over. Odd wavefronts' queries are 16 on from their block's.
    int term_at[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
        term_at[e] = col * 64 + ((e / 4 * 16 + 4 * quarter + e % 4 - (wave & 1) * 16 + 3 * col) & 63);

    f32x4 acc[D / 16] = {};
    float m = -INFINITY, l = 0.0f;
    const float mul = a.scale * LOG2E;

    // The loaded tile as it goes into LDS, split while the last products of the tile before run where the registers
    // hold both.
    constexpr bool EARLY = D <= 128;
    Split2 ks[PER], rs[PER];
    Split3 vs[PER];
    const auto split = [&]() {
        fill(kr);
#pragma unroll
        for (int u = 0; u < PER; u++) {
            ks[u] = split_row<CHUNKS>(kr[u]);
            vs[u] = split3(vr[u]);
        }
        if (REL) split_block(rr, rs);
    };

    if (REL) {
        for (int e = 0; e < 8; e++) {
            const int64_t x = (int64_t)h * a.d + c * 8 + e;
            wu[e] = in_d ? (a.rel_v ? a.rel_v[x] : 0.0f) - (a.rel_u ? a.rel_u[x] : 0.0f) : 0.0f;
        }
    }
    if (n0 < n1) {
        look(tiles.at(n0));
        load(tiles.at(n0));
        if (REL) load_block(tiles.at(n0) / TILE_K, rr);
        if (n0 + 1 < n1) look(tiles.at(n0 + 1));
        if (EARLY) split();
    }
    for (int n = n0; n < n1; n++) {
        const int kb = tiles.at(n), block = kb / TILE_K;
        if (REL && (n == n0 || tiles.at(n - 1) != kb - TILE_K)) {
            // The first tile of a run: the four blocks before its own, and T of each wavefront's first.
            float x[RING][PER][8];
#pragma unroll
            for (int y = 0; y < RING; y++) load_block(block - 1 - y, x[y]);
            __syncthreads();
#pragma unroll
            for (int y = 0; y < RING; y++) {
                Split2 z[PER];
                split_block(x[y], z);
                store_block(block - 1 - y, z);
            }
            __syncthreads();
            terms_of(block - 1 - wave / 2);
        }
        if (!EARLY) split();
        __syncthreads();  // every wavefront has read the last tile
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int krow = row0 + u * STEP, kto = krow * K_PITCH<D> + c * 8, vto = krow * V_STEP<D> + c * 8;
            *reinterpret_cast<f16x8 *>(&sh.k[0][kto]) = ks[u].hi;
            *reinterpret_cast<f16x8 *>(&sh.k[1][kto]) = ks[u].lo;
            *reinterpret_cast<bf16x8 *>(&sh.v[0][vto]) = vs[u].hi;
            *reinterpret_cast<bf16x8 *>(&sh.v[1][vto]) = vs[u].mid;
            *reinterpret_cast<bf16x8 *>(&sh.v[2][vto]) = vs[u].lo;
            if (c == 0) sh.k_back[krow] = ks[u].back;
        }
        if (REL) store_block(block, rs);
        const uint64_t hide = homeless;
        const int docs = doc_k;
        __syncthreads();
        if (n + 1 < n1) {
            load(tiles.at(n + 1));
            if (REL) load_block(tiles.at(n + 1) / TILE_K, rr);
        }
        if (n + 2 < n1) look(tiles.at(n + 2));

        float terms[8];
        if (REL) {
            const int n_block = block - wave / 2;
            terms_of(n_block);
#pragma unroll
            for (int e = 0; e < 8; e++) terms[e] = sh.terms[wave][term_at[e] ^ (n_block & 1) * 32];
        }
        f32x4 back[2], dots[2];
#pragma unroll
        for (int x = 0; x < 2; x++) back[x] = *reinterpret_cast<const f32x4 *>(&sh.k_back[x * 16 + quarter * 4]);
        along(sh.k[0], sh.k[1], dots);

        // Scores, and -infinity where the key is not shown, unless the whole tile is.
        const bool full = (kb >= w_last.lo && kb + TILE_K <= w_first.hi) || kb + TILE_K <= w_first.prefix;
        const bool same_doc = !EXTRA || !a.q_docs || one_document(docs, doc);
        const bool whole = full && !(PAGED && hide) && same_doc;
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float scale = back[e / 4][e % 4] * q_back;
            s[e] = REL ? __builtin_fmaf(dots[e / 4][e % 4], scale, terms[e]) : dots[e / 4][e % 4] * scale;
            widest = fmaxf(widest, whole ? back[e / 4][e % 4] : 0.0f);
        }
        const auto key_at = [&](int e) { return kb + e / 4 * 16 + 4 * quarter + e % 4; };
        if (EXTRA) scores_of<false, 8, true>(a, [&](int e) -> float & { return s[e]; }, key_at, h, slope, i);
        if (!whole) {
            const uint32_t bits =
                (uint32_t)(EXTRA && !same_doc ? shown_bits<true, TILE_K>(win, kb, hide, docs, doc)
                                              : shown_bits<false, TILE_K>(win, kb, hide, docs, doc)) >>
                4 * quarter;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t all = shown_mask(bits, e / 4 * 16 + e % 4);
                s[e] = shown_or_not(s[e], all);
                widest = fmaxf(widest, __uint_as_float(__float_as_uint(sh.k_back[e / 4 * 16 + 4 * quarter + e % 4]) & all));
            }
        }

        float top = s[0];
#pragma unroll
        for (int e = 1; e < 8; e++) top = fmaxf(top, s[e]);
        top = max_quarters(top);
        const float to_log2 = EXTRA ? LOG2E : mul;
        if (__any(top > m)) {
            const float mn = fmaxf(m, top);
            const float fade = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * to_log2);
            l *= fade;
#pragma unroll
            for (int x = 0; x < D / 16; x++) acc[x] *= fade;
            m = mn;
        }
        const float base = m == -INFINITY ? 0.0f : m;

        // The weights, then per 16 columns six products of three operands each.
        constexpr int COLUMNS = D / 16;
        bf16x8 vh[COLUMNS], vm[COLUMNS], vl[COLUMNS];
        const __bf16 *v_at = sh.v[0] + (quarter * 4 + col / 4) * V_STEP<D> + col % 4 * 4;
        const auto read_v = [&](int x) {
            vl[x] = v_columns<D>(v_at + 2 * TILE_K * V_STEP<D>, x);
            vh[x] = v_columns<D>(v_at, x);
            vm[x] = v_columns<D>(v_at + TILE_K * V_STEP<D>, x);
        };
#pragma unroll
        for (int x = 0; x < AHEAD; x++) read_v(x);
        __builtin_amdgcn_sched_barrier(0);
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = __builtin_amdgcn_exp2f((s[e] - base) * to_log2);
            l += p[e];
        }
        const Split3 ps = split3(p);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < COLUMNS; x += 2) {
            // Two columns' products in turn: none waits for the one before it.
#pragma unroll
            for (int y = x; y < x + 2; y++) acc[y] = mfma(vl[y], ps.hi, acc[y]);
#pragma unroll
            for (int y = x; y < x + 2; y++) acc[y] = mfma(vh[y], ps.lo, acc[y]);
#pragma unroll
            for (int y = x; y < x + 2; y++) acc[y] = mfma(vm[y], ps.mid, acc[y]);
#pragma unroll
            for (int y = x; y < x + 2; y++) acc[y] = mfma(vm[y], ps.hi, acc[y]);
#pragma unroll
            for (int y = x; y < x + 2; y++) acc[y] = mfma(vh[y], ps.mid, acc[y]);
#pragma unroll
            for (int y = x; y < x + 2; y++) acc[y] = mfma(vh[y], ps.hi, acc[y]);
            if (x + 2 < COLUMNS) read_v(x + 2), read_v(x + 3);
        }
        feed<COLUMNS / 2, 12, 1, 12>();
        if (EARLY && n + 1 < n1) split();
    }

    l = sum_quarters(l);
    // A pair of f16 is off by up to 2^-25 of its scale's inverse, and each of the other row's d values is at most 2^15 of
    // its own: both rows' errors move a score by d 2^-9 times the two inverses (twice that with position rows). Up to 2^-20,
    // or that much of the score where it is more than 1, is what f32 sums of d products lose.
    const float moved = (REL ? 2.0f : 1.0f) * 0x1p-9f * (float)a.d * q_back * max_quarters(widest) * a.scale;
    bool sound = !(moved > 0x1p-20f * fmaxf(1.0f, fabsf(EXTRA ? m : m * a.scale)));
    if (parts.parts > 1) {
        if (!live) return;
        if (!sound) acc[0][0] = NAN;  // for the joining wavefront, unless the part weighs nothing
        const size_t to = (size_t)part * parts.pairs + row * a.heads + h;
        if (quarter == 0) {
            parts.top[to] = EXTRA ? m : m * a.scale;
            parts.sum[to] = l;
        }
        float *o = parts.out + to * a.d;
#pragma unroll
        for (int x = 0; x < D / 16; x++) {
            const int oc = x * 16 + 4 * quarter;
            if (oc < a.d) *reinterpret_cast<f32x4 *>(o + oc) = acc[x];
        }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float *out = static_cast<float *>(a.out) + row * a.ldo + h * a.hso;
#pragma unroll
    for (int x = 0; x < D / 16; x++) {
        const int oc = x * 16 + 4 * quarter;
        const f32x4 o = acc[x] * inv;
        for (int y = 0; y < 4; y++) sound = sound && o[y] - o[y] == 0.0f;
        if (live && oc < a.d) *reinterpret_cast<f32x4 *>(out + oc) = o;
    }
    // An infinity or NaN among the operands, be it hidden, makes the split products NaN.
    unsigned long long again = __ballot(live && !sound);
    again |= again >> 32;
    again = (again | again >> 16) & 0xffff;
    while (again) {
        const int p = wave0 + __builtin_ctzll(again);
        again &= again - 1;
        attend_row<float>(a, b, at.head * group + at.head_of(p), at.row_of(p), lane);
    }
}

template <int D, bool PAGED, bool EXTRA, bool REL, int WAVES>
hipError_t launch_tile(const AttnArgs &a, int splits, hipStream_t s) {
    const int heads = REL ? a.heads : a.kv_heads;
    const size_t q_tiles = div_ceil((size_t)a.seqs.longest * (a.heads / heads), 16 * WAVES);
    const size_t groups = (size_t)a.seqs.batch * heads * splits, blocks = groups * q_tiles;
    if (q_tiles > INT32_MAX || blocks > MAX_ATTN_BLOCKS / 2) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((attn_tile32_kernel<D, PAGED, EXTRA, REL, WAVES>), dim3((unsigned)blocks), dim3(64 * WAVES), 0,
                       s, a, parts_of(a, splits), (int)q_tiles, (int)groups);
    return hipGetLastError();
}

template <int D, bool REL, int WAVES>
hipError_t launch_kind(const AttnArgs &a, int splits, hipStream_t s) {
    const bool extra = a.cap > 0.0f || a.slopes || a.table || a.q_docs;
    if (a.seqs.tables)
        return extra ? launch_tile<D, true, true, REL, WAVES>(a, splits, s)
                     : launch_tile<D, true, false, REL, WAVES>(a, splits, s);
    return extra ? launch_tile<D, false, true, REL, WAVES>(a, splits, s)
                 : launch_tile<D, false, false, REL, WAVES>(a, splits, s);
}

template <int WAVES>
hipError_t launch_size(const AttnArgs &a, int splits, hipStream_t s) {
    if (a.rel) return a.d <= 64 ? launch_kind<64, true, WAVES>(a, splits, s) : launch_kind<128, true, WAVES>(a, splits, s);
    if (a.d <= 64) return launch_kind<64, false, WAVES>(a, splits, s);
    if (a.d <= 128) return launch_kind<128, false, WAVES>(a, splits, s);
    return launch_kind<256, false, WAVES>(a, splits, s);
}

}  // namespace

hipError_t launch_attention32(const AttnArgs &a, int rows, int splits, hipStream_t s) {
    return rows == 64 ? launch_size<4>(a, splits, s) : launch_size<8>(a, splits, s);
}

}  // namespace tg
