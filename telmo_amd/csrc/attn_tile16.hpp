// Attention by 16-bit products on the matrix cores, tiles of 128 query rows by 64 keys: of 16-bit rows, and of rows of any
// type over a cache in e4m3.
//
// The query heads that share a key head are rows of one matrix: row g r + x is head x of the group in query
// row r. A workgroup takes 128 of them, a wavefront 32, and walks the keys 64 at a time through LDS. The
// products are S' = K Q' and O' = V' P', 32 x 32 x 16 each: in S' a lane holds the scores of one query (its
// column) with 32 of the 64 keys, so the softmax is arithmetic in the lane's registers and one exchange with
// the lane of the other half, and the same registers, rounded to 16 bits, are the operand P' of the second
// product, whose keys are taken in the order in which the lanes hold them. V' comes from LDS by transposing
// reads. The weights are rounded once to the rows' type, f16's scaled by 2^8 (as is their sum) so that weights
// down to 2^-22 of the largest are normal numbers.
//
// Bound by the wavefront's own chain: its exponentials, maxima and conversions take as long as its products, and
// two wavefronts to a SIMD overlap them only in part (matrix units 38 % busy, vector units 42 %, a chunk of 509
// rows of 32 heads over 32768 paged keys; with capped scores 36 % and 75 %). That chunk runs at 838 TFLOP/s, 8192
// causal rows with capped scores at 781, where a large library product reaches 1196. LDS carries each tile from
// memory to four wavefronts, double buffered; 256 rows and eight wavefronts, sharing each tile by twice as many,
// made the chunk 5 % faster but short and ragged calls 17 to 19 % slower. Wavefront priorities changed nothing.
#pragma once

#include "attn_launch.hpp"
#include "attn_tile.hpp"

namespace tg {

namespace {

constexpr int THREADS = 256, TILE_Q = 128;

// What a call does to its scores, in what it costs: a kernel of each kind, since the plain one folds the scale
// into the exponent and holds no choices in its loop.
enum Extra { PLAIN, CAPS, ALL };  // nothing; caps (fast_cap) and slopes; tables, documents and any caps too

template <typename T>
struct Half;
template <>
struct Half<_Float16> {
    typedef f16x8 v8;
    static constexpr float shift = 8.0f;
    static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Half<__bf16> {
    typedef bf16x8 v8;
    static constexpr float shift = 0.0f;
    static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

// What is multiplied, for rows of type T over keys of type C. Over e4m3 keys, which bf16 holds exactly with their power
// of two, rows and weights are sums of bf16 parts of eight bits each: all of f16's bits in two, of f32's in three.
template <typename T, typename C>
struct Parts16 {
    static constexpr bool BYTES = __is_same(C, e4m3), WIDE = __is_same(T, float);
    static constexpr int ROW = !BYTES || __is_same(T, __bf16) ? 1 : WIDE ? 3 : 2, WEIGHT = WIDE ? 3 : ROW;
};
template <typename T, typename C>
struct Multiplied {
    typedef T type;
};
template <typename T>
struct Multiplied<T, e4m3> {
    typedef __bf16 type;
};

// D: head size rounded up to 64, 128 or 256. C: the keys' type, T or (paged) e4m3. f32 rows take EXTRA ALL.
template <typename T, typename C, int D, bool PAGED, Extra EXTRA>
__global__ __launch_bounds__(THREADS, D == 256 || __is_same(T, float) ? 1 : 2) void attn_tile_kernel(const AttnArgs a, const AttnParts parts,
                                                                              const int q_tiles, const int groups) {
    typedef Parts16<T, C> Parts;
    typedef typename Multiplied<T, C>::type M;
    typedef typename Half<M>::v8 v8;
    constexpr bool BYTES = Parts::BYTES;
    constexpr int ROW = Parts::ROW, WEIGHT = Parts::WEIGHT;
    constexpr int TILE_K = D == 256 ? 32 : 64;  // keys of a tile: the output of 256 columns leaves registers for 32
    constexpr int HALVES = TILE_K / 32, N = TILE_K / 2;  // score products of a tile, scores of a lane
    constexpr int AHEAD = 4;  // operands on their way from LDS
    constexpr float NEAR = 1024.0f;
    constexpr int VALUES = 16 / sizeof(C);  // of a 16-byte piece
    constexpr int CHUNKS = D / VALUES, PER = TILE_K * CHUNKS / THREADS, STEP = THREADS / CHUNKS;
    __shared__ __align__(16) M k_tiles[2][TILE_K * K_PITCH<D>], v_tiles[2][TILE_K * V_PITCH<D>];

    Place at;
    if (!at.find(a, parts.parts, q_tiles, groups, a.kv_heads, TILE_Q)) return;
    const int part = at.part, kvh = at.head, b = at.b, group = at.group;
    const AttnSpan sp = at.sp;
    const int pairs = at.pairs, pair0 = at.pair0;

    const int t = threadIdx.x, lane = t & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);  // a scalar, and what follows from it
    const int prefix = a.prefix ? a.prefix[b] : 0;
    // The lane's query, and the first and last of the wavefront's and the workgroup's.
    const int pair = pair0 + wave * 32 + col;
    const bool live = pair < pairs;
    const int r = live ? at.row_of(pair) : 0, h = kvh * group + (live ? at.head_of(pair) : 0);
    const int i = sp.shift() + r;
    const AttnWindow win = window_of(i, sp.nk, a.left, a.right, prefix);
    const int wave0 = pair0 + wave * 32, wave1 = wave0 + 31 < pairs - 1 ? wave0 + 31 : pairs - 1;
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

    v8 qf[D / 16][ROW];
    const T *q = static_cast<const T *>(a.q) + row * a.ldq + h * a.hsq;
#pragma unroll
    for (int s = 0; s < D / 16; s++) {
        const int c = s * 16 + half * 8;
        if constexpr (ROW == 1) {
            qf[s][0] = live && c < a.d ? *reinterpret_cast<const v8 *>(q + c) : v8{};
        } else {
            float x[8] = {};
            if (live && c < a.d) load8(q + c, x);
            cut_parts(x, qf[s]);
        }
    }

    // This thread's part of the tiles: rows row0 + u STEP, chunk c of each.
    const int row0 = t / CHUNKS, c = t % CHUNKS;
    const bool in_d = c * VALUES < a.d;
    KeyRows<C, TILE_K, PER, STEP, PAGED> keys(a, sp, kvh, row0, in_d ? c * VALUES : 0);
    int k_exp = 0, v_exp = 0;  // of the lane's key of the loaded tile
    u32x4 kr[PER], vr[PER];
    uint64_t homeless = 0;  // of the loaded tile's keys
    int doc_k = 0;          // the lane's key's document
    const auto look = [&](int kb) { keys.look(a, sp, b, kb, lane); };
    const auto load = [&](int kb) {
        homeless = keys.homeless();
        if constexpr (BYTES) {
            const int p = keys.page < 0 ? 0 : keys.page;
            k_exp = a.k_exps[block_at(a, a.k_epage, p, keys.at) + kvh];
            v_exp = a.v_exps[block_at(a, a.v_epage, p, keys.at) + kvh];
        }
        keys.each(a, sp, kb, [&](int u, const char *k, const char *v) {
            kr[u] = *reinterpret_cast<const u32x4 *>(k);
            vr[u] = *reinterpret_cast<const u32x4 *>(v);
        });
        if (EXTRA == ALL && a.q_docs) {
            const int j = kb + lane;
            doc_k = a.k_docs[sp.k0 + (j < sp.nk ? j : sp.nk - 1)];
        }
        if (a.d < D)  // the columns that fill D up: values of any kind, but none that meets the queries' zeros
#pragma unroll
            for (int u = 0; u < PER; u++) kr[u] = in_d ? kr[u] : u32x4{};
    };

    f32x16 acc[D / 32] = {};
    float m = -INFINITY, l = 0.0f;
    const float mul = a.scale * LOG2E;
    // Plain scores are scaled and lowered by the base in one operation, the exponent's: off by half a step of base mul
    // for all keys of a tile alike, 2^-14 at most below NEAR. Past NEAR each tile comes through the gate and takes the
    // base off first, in f32 exactly wherever the weight is not nothing: rows of 10^4 have exponents of 10^9, whose
    // half step is far more than f16's weights can take.
    float off = Half<M>::shift, gate = -INFINITY;

    // Two tiles in LDS: while one is worked on, the next one, which left memory a tile ago, is written to the
    // other, and the one after it leaves memory.
    uint64_t hide = 0;  // of the tile that is worked on
    int docs = 0;
    const auto store = [&](int n) {
#pragma unroll
        for (int u = 0; u < PER; u++) {
            M *k = &k_tiles[n & 1][row0 * K_PITCH<D> + c * VALUES + u * STEP * K_PITCH<D>];
            M *v = &v_tiles[n & 1][row0 * V_PITCH<D> + c * VALUES + u * STEP * V_PITCH<D>];
            if constexpr (BYTES) {
                const float ks = two_to(__shfl(k_exp, row0 + u * STEP)), vs = two_to(__shfl(v_exp, row0 + u * STEP));
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const uint32_t k0 = kr[u][2 * x], k1 = kr[u][2 * x + 1], v0 = vr[u][2 * x], v1 = vr[u][2 * x + 1];
                    reinterpret_cast<u32x4 *>(k)[x] = u32x4{e4m3_widen<false>(k0, ks), e4m3_widen<true>(k0, ks),
                                                            e4m3_widen<false>(k1, ks), e4m3_widen<true>(k1, ks)};
                    reinterpret_cast<u32x4 *>(v)[x] = u32x4{e4m3_widen<false>(v0, vs), e4m3_widen<true>(v0, vs),
                                                            e4m3_widen<false>(v1, vs), e4m3_widen<true>(v1, vs)};
                }
            } else {
                *reinterpret_cast<u32x4 *>(k) = kr[u];
                *reinterpret_cast<u32x4 *>(v) = vr[u];
            }
        }
        hide = homeless;
        docs = doc_k;
        if (n + 1 < n1) load(tiles.at(n + 1));
        if (n + 2 < n1) look(tiles.at(n + 2));
    };
    if (n0 < n1) {
        look(tiles.at(n0));
        load(tiles.at(n0));
        if (n0 + 1 < n1) look(tiles.at(n0 + 1));
        store(n0);
        __syncthreads();
    }
    for (int n = n0; n < n1; n++) {
        const int kb = tiles.at(n);
        const M *ks = k_tiles[n & 1] + k_lane<D>(lane), *vs = v_tiles[n & 1] + v_lane<D>(lane);
        constexpr int SCORES = D / 16 * HALVES;  // products of K: of 16 columns and 32 keys each
        v8 kf[SCORES];
        f32x16 s[HALVES] = {};
        const auto k_fragment = [&](int e) {
            return *reinterpret_cast<const v8 *>(ks + e % HALVES * 32 * K_PITCH<D> + e / HALVES * 16);
        };
#pragma unroll
        for (int e = 0; e < AHEAD; e++) kf[e] = k_fragment(e);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < SCORES; e++) {
#pragma unroll
            for (int y = ROW - 1; y >= 0; y--)
                s[e % HALVES] = Half<M>::mfma(kf[e], qf[e / HALVES][y], s[e % HALVES]);
            if (e + AHEAD < SCORES) kf[e + AHEAD] = k_fragment(e + AHEAD);
        }
        feed<SCORES, 1, AHEAD, ROW>();

        // Scores, and -infinity where the key is not shown.
        const bool full = (kb >= w_last.lo && kb + TILE_K <= w_first.hi) || kb + TILE_K <= w_first.prefix;
        if (EXTRA)
            scores_of<!Parts::WIDE, N, EXTRA == ALL>(
                a, [&](int e) -> float & { return reinterpret_cast<float *>(&s[e / 16])[e % 16]; },
                [&](int e) { return kb + e / 16 * 32 + 8 * (e % 16 / 4) + 4 * half + e % 4; }, h, slope, i);
        const bool same_doc = EXTRA != ALL || !a.q_docs || one_document(docs, doc);
        if (!full || (PAGED && hide) || !same_doc) {
            const uint64_t bits = (EXTRA == ALL && !same_doc ? shown_bits<true, TILE_K>(win, kb, hide, docs, doc)
                                                             : shown_bits<false, TILE_K>(win, kb, hide, docs, doc)) >>
                                  4 * half;
#pragma unroll
            for (int e = 0; e < N; e++)
                s[e / 16][e % 16] = shown_or_not(s[e / 16][e % 16], (uint32_t)(bits >> e / 16 * 32), 8 * (e % 16 / 4) + e % 4);
        }

        float top = s[0][0];
#pragma unroll
        for (int e = 1; e < N; e++) top = fmaxf(top, s[e / 16][e % 16]);
        top = max_halves(top);
        if (__any(top > (EXTRA ? m : gate))) {
            const float mn = fmaxf(m, top);
            const float fade = m == -INFINITY ? 0.0f
                                              : __builtin_amdgcn_exp2f(EXTRA ? (m - mn) * LOG2E : (m - mn) * mul);
            l *= fade;
#pragma unroll
            for (int x = 0; x < D / 32; x++) acc[x] *= fade;
            m = gate = mn;
            if (!EXTRA) {
                const float base = m == -INFINITY ? 0.0f : m, far = base * mul;
                off = Half<M>::shift - far;
                if (__any(!(fabsf(far) < NEAR))) {
                    off = Half<M>::shift;
                    gate = -INFINITY;
#pragma unroll
                    for (int e = 0; e < N; e++) s[e / 16][e % 16] -= base;
                }
            }
        }
        const float base = m == -INFINITY ? 0.0f : m;
        v8 pf[N / 8][WEIGHT];
        // The first fragments of V are on their way while the weights are worked out.
        constexpr int PRODUCTS = N / 8 * (D / 32);
        s16x8 vf[PRODUCTS];
#pragma unroll
        for (int e = 0; e < AHEAD; e++) vf[e] = v_fragment<D>(vs, e / (D / 32), e % (D / 32));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < N / 8; g++) {
            f32x8 p;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = s[g / 2][(g % 2) * 8 + e];
                // The difference first where a bias can be the type's lowest value: its multiple is infinite.
                p[e] = __builtin_amdgcn_exp2f(EXTRA ? __builtin_fmaf(x - base, LOG2E, Half<M>::shift)
                                                    : __builtin_fmaf(x, mul, off));
                l += p[e];
            }
#pragma unroll
            for (int y = 0; y < WEIGHT; y++) {
                pf[g][y] = __builtin_convertvector(p, v8);
                if (y + 1 < WEIGHT) p -= __builtin_convertvector(pf[g][y], f32x8);
            }
        }
        if (n + 1 < n1) store(n + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < PRODUCTS; e++) {
#pragma unroll
            for (int y = WEIGHT - 1; y >= 0; y--)
                acc[e % (D / 32)] = Half<M>::mfma(__builtin_bit_cast(v8, vf[e]), pf[e / (D / 32)][y], acc[e % (D / 32)]);
            const int next = e + AHEAD;
            if (next < PRODUCTS) vf[next] = v_fragment<D>(vs, next / (D / 32), next % (D / 32));
        }
        feed<PRODUCTS, 2, AHEAD, WEIGHT>();
        __syncthreads();
    }

    l = sum_halves(l);
    if (parts.parts > 1) {
        if (!live) return;
        const size_t to = (size_t)part * parts.pairs + row * a.heads + h;
        if (half == 0) {
            parts.top[to] = EXTRA ? m : m * a.scale;
            parts.sum[to] = l;
        }
        float *o = parts.out + to * a.d;
#pragma unroll
        for (int x = 0; x < D / 32; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int oc = x * 32 + 8 * e + 4 * half;
                if (oc < a.d)
                    *reinterpret_cast<f32x4 *>(o + oc) =
                        f32x4{acc[x][4 * e], acc[x][4 * e + 1], acc[x][4 * e + 2], acc[x][4 * e + 3]};
            }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *out = static_cast<T *>(a.out) + row * a.ldo + h * a.hso;
    float worst = 0.0f;
#pragma unroll
    for (int x = 0; x < D / 32; x++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int oc = x * 32 + 8 * e + 4 * half;
            T o[4];
            for (int y = 0; y < 4; y++) {
                const float v = acc[x][4 * e + y] * inv;
                worst = fmaxf(worst, v - v == 0.0f ? 0.0f : 1.0f);
                o[y] = mean_to<T>(v);
            }
            if (live && oc < a.d) {
                if constexpr (Parts::WIDE) *reinterpret_cast<u32x4 *>(out + oc) = *reinterpret_cast<u32x4 *>(o);
                else *reinterpret_cast<u32x2 *>(out + oc) = *reinterpret_cast<u32x2 *>(o);
            }
        }
    // A NaN in the sum of weights comes from a shown score and is the result; one beside a sound sum may come
    // from a hidden key's value.
    unsigned long long again = __ballot(live && worst > 0.0f && l - l == 0.0f);
    again = (again | again >> 32) & 0xffffffffull;
    while (again) {
        const int p = wave0 + __builtin_ctzll(again);
        again &= again - 1;
        attend_row<T, C>(a, b, kvh * group + at.head_of(p), at.row_of(p), lane);
    }
}

template <typename T, typename C, int D, bool PAGED, Extra EXTRA>
hipError_t launch_tile(const AttnArgs &a, int splits, hipStream_t s) {
    const int group = a.heads / a.kv_heads;
    const size_t q_tiles = div_ceil((size_t)a.seqs.longest * group, TILE_Q);
    const size_t groups = (size_t)a.seqs.batch * a.kv_heads * splits, blocks = groups * q_tiles;
    if (q_tiles > INT32_MAX || blocks > MAX_ATTN_BLOCKS) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((attn_tile_kernel<T, C, D, PAGED, EXTRA>), dim3((unsigned)blocks), dim3(THREADS), 0, s, a,
                       parts_of(a, splits), (int)q_tiles, (int)groups);
    return hipGetLastError();
}

template <typename T, typename C, int D, bool PAGED>
hipError_t launch_extra(const AttnArgs &a, int splits, hipStream_t s) {
    if constexpr (__is_same(T, float)) {
        return launch_tile<T, C, D, PAGED, ALL>(a, splits, s);
    } else {
        if (a.table || a.q_docs || (a.cap > 0.0f && !fast_cap(a))) return launch_tile<T, C, D, PAGED, ALL>(a, splits, s);
        if (a.cap > 0.0f || a.slopes) return launch_tile<T, C, D, PAGED, CAPS>(a, splits, s);
        return launch_tile<T, C, D, PAGED, PLAIN>(a, splits, s);
    }
}

}  // namespace

}  // namespace tg
