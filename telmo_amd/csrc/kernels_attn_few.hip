// Attention of few query rows over many keys (single tokens over a cache): bound by reading the keys and values
// once.
//
// The rows of a sequence that share a key head (its new rows by the group's heads) are the 16 columns of
// 16 x 16 products. Nothing of the keys is used twice, so LDS does not hold them: each of a workgroup's
// wavefronts takes key tiles of its own and loads the operands of S' = K Q' from memory into registers as the
// matrix instructions want them (16 rows by 64 bytes a load), and V by whole rows (a load gives 16 lanes the
// 16 x 16 bytes of a row), two tiles under way at a time. V' wants keys side by side in a register: of 16-bit
// values, the eight rows that a lane holds are interleaved in registers; of f32 there is nothing to do. The
// output's columns are numbered so that a lane's loads are contiguous: product x of a piece holds its value x.
// The wavefronts' results are joined in LDS, and those of the parts by a second kernel.
//
// The products have time to spare, so the 16-bit weights are held as two numbers, f32's as they are on the f32
// matrix instructions.
//
// 32 sequences of 8192 keys, 8 key heads of 128 in bf16: 1.07 GB in 202 us, 5.3 TB/s (a large copy moves 4.8). The same
// call by the tiles of 128 rows takes 209, without parts 338; eight sequences of 750 f16 keys 14.7 (19.9), one of
// 100,000 keys and heads of 64 94 (114). One tile under way and twice the wavefronts: 140 for 128 us at lengths of
// up to 8192, two workgroups to a CU in fewer registers 120 to 137 for 113 to 134.
#include "attn_launch.hpp"
#include "attn_tile.hpp"

namespace tg {

namespace {

constexpr int COLS = 16;

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Memory of the GPU, said where the compiler would take an address for LDS's or memory's and wait for both.
template <typename T>
using Global = const __attribute__((address_space(1))) T *;

template <typename T, int D>
struct Few {
    static constexpr bool WIDE = sizeof(T) == 4;
    // Tiles whose operands are under way, and wavefronts: one on a SIMD where the operands fill its registers. Heads of 64
    // leave room for two wavefronts, heads of 256 for one tile of theirs.
    static constexpr int DEPTH = D == 256 ? 1 : 2, WAVES = D == 64 ? 8 : 4;
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int TILE = WIDE ? 16 : 32;             // keys of a tile
    static constexpr int CH = WIDE ? 4 : D == 64 ? 4 : 8;   // values of a lane's piece of a V row
    static constexpr int W = D / (16 * CH);                 // pieces of a V row
    static constexpr int VROWS = WIDE ? 4 : 8;              // V rows of a lane
    static constexpr int KS = WIDE ? D / 16 : D / 32;       // 16-byte pieces of a lane's part of a K row
    static constexpr int KT = TILE / 16;                    // K rows of a lane
    static constexpr int VW = CH * sizeof(T) / 4;           // words of a V piece
};

// D: head size rounded up to 64, 128 or 256. EXTRA: scores are capped or biased.
template <typename T, int D, bool PAGED, bool EXTRA>
__global__ __launch_bounds__((Few<T, D>::THREADS)) void attn_few_kernel(const AttnArgs a, const AttnParts parts) {
    typedef Few<T, D> F;
    constexpr int TILE = F::TILE, PITCH = D + 4, WAVES = F::WAVES, THREADS = F::THREADS;
    __shared__ __align__(16) float outs[WAVES][COLS][PITCH];
    __shared__ float tops[WAVES][COLS], sums[WAVES][COLS];
    __shared__ int again[COLS];

    const uint32_t set = blockIdx.x / (uint32_t)parts.parts;
    const int part = (int)(blockIdx.x - set * (uint32_t)parts.parts);
    const int b = (int)(set / (uint32_t)a.kv_heads), kvh = (int)set - b * a.kv_heads;
    const AttnSpan sp = span_of(a.seqs, b);
    const int group = (int)((uint32_t)a.heads / (uint32_t)a.kv_heads);
    const int pairs = (sp.nq < a.seqs.longest ? sp.nq : a.seqs.longest) * group;  // COLS at most
    if (pairs == 0) return;
    const auto row_of = [&](int pair) { return (int)((uint32_t)pair / (uint32_t)group); };

    const int t = threadIdx.x, lane = t & 63, quarter = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);  // a scalar, and what follows from it
    const int prefix = a.prefix ? a.prefix[b] : 0;
    const bool live = col < pairs;
    const int r = live ? row_of(col) : 0, h = kvh * group + (live ? col - r * group : 0);
    const int i = sp.shift() + r;
    const AttnWindow win = window_of(i, sp.nk, a.left, a.right, prefix);
    const AttnWindow w_first = window_of(sp.shift(), sp.nk, a.left, a.right, prefix);
    const AttnWindow w_last = window_of(sp.shift() + row_of(pairs - 1), sp.nk, a.left, a.right, prefix);
    const Tiles<TILE> tiles(w_first, w_last);
    const int n0 = (int)((int64_t)tiles.count * part / parts.parts) + wave;
    const int n1 = (int)((int64_t)tiles.count * (part + 1) / parts.parts);
    const int64_t row = (int64_t)sp.q0 + r;
    const float slope = EXTRA && a.slopes ? a.slopes[h] : 0.0f;

    u32x4 qf[F::KS];
    {
        const T *q = static_cast<const T *>(a.q) + row * a.ldq + h * a.hsq;
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int s = 0; s < F::KS; s++) {
            const int c = s * 4 * E + quarter * E;
            qf[s] = live && c < a.d ? *reinterpret_cast<const u32x4 *>(q + c) : u32x4{};
        }
    }

    const T *kbase = static_cast<const T *>(a.k) + kvh * a.hsk, *vbase = static_cast<const T *>(a.v) + kvh * a.hsv;
    const bool one_page = PAGED && a.seqs.page % TILE == 0;  // a tile lies in one page
    // A tile's operands in registers, two tiles' at a time.
    struct Operands {
        u32x4 k[F::KT][F::KS];
        uint32_t v[F::VROWS][F::W][F::VW];
        uint32_t hidden;  // keys that have no place
    } buf[F::DEPTH];
    // Lane n of a wavefront looks up the tile's key n (its first key, where the tile lies in one page).
    int page = 0, page_row = 0;
    const auto look = [&](int kb) {
        if (!PAGED) return;
        const int key = one_page ? kb : kb + lane % TILE;
        page = page_of(a.seqs, b, key < sp.nk ? key : sp.nk - 1, page_row);
    };
    // The wavefront's last tile. Past it loads read one row of it, and what they bring is hidden: two loads are always
    // under way, so that the compiler knows how many it need not wait for.
    const int last_tile = n1 - 1 - (n1 - 1 - n0) % WAVES;
    const auto tile_at = [&](int n) { return tiles.at(n < last_tile ? n : last_tile); };
    // The operands of tile n, which was looked up last, leave memory; the tile after it is looked up before they do,
    // so that waiting for its pages does not wait for them. Addresses first: the loads in one run.
    const auto load = [&](Operands &x, int n) {
        const int kb = tile_at(n);
        const bool real = n <= last_tile;
        int64_t kp[F::KT], vp[F::VROWS];  // offsets from the head's first value
        const auto key_of = [&](int key) { return !real ? 0 : kb + key < sp.nk ? key : sp.nk - 1 - kb; };  // within the tile
        const auto v_key = [&](int e) { return (e / 4) * 16 + quarter * 4 + e % 4; };
        x.hidden = 0;
        if (PAGED) {
            x.hidden = (uint32_t)__ballot(page < 0);
            const int64_t p = page < 0 ? 0 : page;
            const int64_t kat = p * a.psk + page_row * a.ldk, vat = p * a.psv + page_row * a.ldv;
            if (one_page) {
#pragma unroll
                for (int y = 0; y < F::KT; y++) kp[y] = kat + key_of(y * 16 + col) * a.ldk;
#pragma unroll
                for (int e = 0; e < F::VROWS; e++) vp[e] = vat + key_of(v_key(e)) * a.ldv;
            } else {
                const auto from = [&](int64_t offset, int lane_of) {
                    const int lo = __shfl((int)(uint32_t)offset, lane_of), hi = __shfl((int)(offset >> 32), lane_of);
                    return (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
                };
#pragma unroll
                for (int y = 0; y < F::KT; y++) kp[y] = from(kat, key_of(y * 16 + col));
#pragma unroll
                for (int e = 0; e < F::VROWS; e++) vp[e] = from(vat, key_of(v_key(e)));
            }
            look(tile_at(n + WAVES));
        } else {
            const int64_t k0 = (int64_t)(sp.k0 + kb) * a.ldk, v0 = (int64_t)(sp.k0 + kb) * a.ldv;
#pragma unroll
            for (int y = 0; y < F::KT; y++) kp[y] = k0 + key_of(y * 16 + col) * a.ldk;
#pragma unroll
            for (int e = 0; e < F::VROWS; e++) vp[e] = v0 + key_of(v_key(e)) * a.ldv;
        }
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int y = 0; y < F::KT; y++)
#pragma unroll
            for (int s = 0; s < F::KS; s++) {
                const int c = s * 4 * E + quarter * E;
                x.k[y][s] = *(Global<u32x4>)(kbase + kp[y] + (c < a.d ? c : 0));
            }
#pragma unroll
        for (int e = 0; e < F::VROWS; e++)
#pragma unroll
            for (int w = 0; w < F::W; w++) {
                // Rows past the last key and columns past d are read as others: weighted by zero, or not stored.
                const int c = w * 16 * F::CH + col * F::CH;
                if constexpr (F::VW == 4) {
                    const u32x4 y = *(Global<u32x4>)(vbase + vp[e] + (c < a.d ? c : 0));
                    for (int z = 0; z < 4; z++) x.v[e][w][z] = y[z];
                } else {
                    const u32x2 y = *(Global<u32x2>)(vbase + vp[e] + (c < a.d ? c : 0));
                    for (int z = 0; z < 2; z++) x.v[e][w][z] = y[z];
                }
            }
    };

    f32x4 acc[F::W][F::CH] = {};
    float m = -INFINITY, l = 0.0f;
    const float to_log2 = EXTRA ? LOG2E : a.scale * LOG2E;
    constexpr float SHIFT = __is_same(T, _Float16) ? 8.0f : 0.0f;  // weights below f16's normal numbers

    const auto work = [&](Operands &o, int n) {
        const int kb = tile_at(n);
        const bool real = n <= last_tile;
        const uint32_t hide = o.hidden;
        if (a.d < D) {  // zeros where the queries' zeros may meet a value of any kind
            constexpr int E = 16 / sizeof(T);
#pragma unroll
            for (int x = 0; x < F::KT; x++)
#pragma unroll
                for (int e = 0; e < F::KS; e++)
                    if (e * 4 * E + quarter * E >= a.d) o.k[x][e] = u32x4{};
        }
        f32x4 s[F::KT] = {};
#pragma unroll
        for (int e = 0; e < F::KS; e++)
#pragma unroll
            for (int x = 0; x < F::KT; x++) {
                if constexpr (F::WIDE) {
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        s[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(o.k[x][e][y]),
                                                                    __uint_as_float(qf[e][y]), s[x], 0, 0, 0);
                } else {
                    typedef T v8 __attribute__((ext_vector_type(8)));
                    s[x] = mfma16(__builtin_bit_cast(v8, o.k[x][e]), __builtin_bit_cast(v8, qf[e]), s[x]);
                }
            }

        const bool full = real && ((kb >= w_last.lo && kb + TILE <= w_first.hi) || kb + TILE <= w_first.prefix);
        constexpr int N = 4 * F::KT;
        if (EXTRA)
            scores_of<!F::WIDE, N, true>(
                a, [&](int e) -> float & { return reinterpret_cast<float *>(&s[e / 4])[e % 4]; },
                [&](int e) { return kb + e / 4 * 16 + quarter * 4 + e % 4; }, h, slope, i);
        if (!full || (PAGED && hide)) {
            const uint64_t homeless = !real || (one_page && hide) ? ~0ull : hide;
            const uint32_t bits = (uint32_t)shown_bits<false, TILE>(win, kb, homeless, 0, 0) >> 4 * quarter;
#pragma unroll
            for (int e = 0; e < N; e++) s[e / 4][e % 4] = shown_or_not(s[e / 4][e % 4], bits, e / 4 * 16 + e % 4);
        }
        float top = s[0][0];
#pragma unroll
        for (int e = 1; e < N; e++) top = fmaxf(top, s[e / 4][e % 4]);
        top = max_quarters(top);
        if (__any(top > m)) {
            const float mn = fmaxf(m, top);
            const float fade = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * to_log2);
            l *= fade;
#pragma unroll
            for (int w = 0; w < F::W; w++)
#pragma unroll
                for (int x = 0; x < F::CH; x++) acc[w][x] *= fade;
            m = mn;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float p[N];
#pragma unroll
        for (int e = 0; e < N; e++) {
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e / 4][e % 4] - base, to_log2, SHIFT));
            l += p[e];
        }
        if constexpr (F::WIDE) {
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int w = 0; w < F::W; w++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        acc[w][x] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(o.v[e][w][x]), p[e],
                                                                         acc[w][x], 0, 0, 0);
        } else {
            typedef T v8 __attribute__((ext_vector_type(8)));
            f32x8 pv;
#pragma unroll
            for (int e = 0; e < 8; e++) pv[e] = p[e];
            const v8 ph = __builtin_convertvector(pv, v8);
            const v8 pl = __builtin_convertvector(pv - __builtin_convertvector(ph, f32x8), v8);
#pragma unroll
            for (int w = 0; w < F::W; w++)
#pragma unroll
                for (int x = 0; x < F::CH; x++) {
                    u32x4 v;  // value x of the lane's eight rows
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        v[y] = __builtin_amdgcn_perm(o.v[2 * y + 1][w][x / 2], o.v[2 * y][w][x / 2],
                                                     x % 2 ? 0x07060302u : 0x05040100u);
                    acc[w][x] = mfma16(__builtin_bit_cast(v8, v), pl, acc[w][x]);
                    acc[w][x] = mfma16(__builtin_bit_cast(v8, v), ph, acc[w][x]);
                }
        }
    };

    if (n0 < n1) {
        look(tile_at(n0));
        load(buf[0], n0);
        if constexpr (F::DEPTH == 2) {
            load(buf[1], n0 + WAVES);
            for (int n = n0; n <= last_tile; n += 2 * WAVES) {
                work(buf[0], n);
                load(buf[0], n + 2 * WAVES);
                work(buf[1], n + WAVES);
                load(buf[1], n + 3 * WAVES);
            }
        } else {
            for (int n = n0; n <= last_tile; n += WAVES) {
                work(buf[0], n);
                if (n < last_tile) load(buf[0], n + WAVES);
            }
        }
    }

    // The wavefronts' parts: each thread adds up four values of a column.
    l = sum_quarters(l);
    if (t < COLS) again[t] = 0;
    if (quarter == 0) {
        tops[wave][col] = EXTRA ? m : m * a.scale;
        sums[wave][col] = l;
    }
#pragma unroll
    for (int w = 0; w < F::W; w++)
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int x = 0; x < F::CH; x += 4)
                *reinterpret_cast<f32x4 *>(&outs[wave][col][w * 16 * F::CH + (quarter * 4 + e) * F::CH + x]) =
                    f32x4{acc[w][x][e], acc[w][x + 1][e], acc[w][x + 2][e], acc[w][x + 3][e]};
    __syncthreads();
    for (int y = t; y < COLS * (D / 4); y += THREADS) {
        const int oc = y / (D / 4), c = y % (D / 4) * 4;
        if (oc >= pairs || c >= a.d) continue;
        float top = -INFINITY, sum = 0.0f;
        for (int w = 0; w < WAVES; w++) top = fmaxf(top, tops[w][oc]);
        const float base = top == -INFINITY ? 0.0f : top;
        f32x4 o = {};
        for (int w = 0; w < WAVES; w++) {
            const float weight = exp2f((tops[w][oc] - base) * LOG2E), part_sum = sums[w][oc];
            if (part_sum == 0.0f) continue;
            sum = __builtin_fmaf(weight, part_sum, sum);
            const f32x4 x = *reinterpret_cast<const f32x4 *>(&outs[w][oc][c]);
            for (int e = 0; e < 4; e++) o[e] = __builtin_fmaf(weight, x[e], o[e]);
        }
        const int pair_row = row_of(oc);
        const int64_t to_row = (int64_t)sp.q0 + pair_row;
        const int to_head = kvh * group + oc - pair_row * group;
        if (parts.parts > 1) {
            const size_t to = (size_t)part * parts.pairs + to_row * a.heads + to_head;
            if (c == 0) {
                parts.top[to] = top;
                parts.sum[to] = sum;
            }
            *reinterpret_cast<f32x4 *>(parts.out + to * a.d + c) = o;
            continue;
        }
        T *out = static_cast<T *>(a.out) + to_row * a.ldo + to_head * a.hso + c;
        bool sound = true;
        T v[4];
        for (int e = 0; e < 4; e++) {
            const float x = sum == 0.0f ? 0.0f : o[e] / sum;
            sound = sound && x - x == 0.0f;
            v[e] = mean_to<T>(x);
        }
        if constexpr (F::WIDE) *reinterpret_cast<u32x4 *>(out) = *reinterpret_cast<u32x4 *>(v);
        else *reinterpret_cast<u32x2 *>(out) = *reinterpret_cast<u32x2 *>(v);
        if (!sound && sum - sum == 0.0f) again[oc] = 1;
    }
    if (parts.parts > 1) return;
    // A hidden key's NaN or infinity beside a sound sum of weights, as in the tile kernels.
    __syncthreads();
    for (int x = wave; x < COLS; x += WAVES)
        if (again[x]) attend_row<T>(a, b, kvh * group + x - row_of(x) * group, row_of(x), lane);
}

template <typename T, int D, bool PAGED, bool EXTRA>
hipError_t launch_few(const AttnArgs &a, int splits, hipStream_t s) {
    const size_t blocks = (size_t)a.seqs.batch * a.kv_heads * splits;
    if (blocks > MAX_ATTN_BLOCKS / 2) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((attn_few_kernel<T, D, PAGED, EXTRA>), dim3((unsigned)blocks), dim3(Few<T, D>::THREADS), 0,
                       s, a, parts_of(a, splits));
    return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_kind(const AttnArgs &a, int splits, hipStream_t s) {
    const bool extra = a.cap > 0.0f || a.slopes || a.table;
    if (a.seqs.tables)
        return extra ? launch_few<T, D, true, true>(a, splits, s) : launch_few<T, D, true, false>(a, splits, s);
    return extra ? launch_few<T, D, false, true>(a, splits, s) : launch_few<T, D, false, false>(a, splits, s);
}

template <typename T>
hipError_t launch_size(const AttnArgs &a, int splits, hipStream_t s) {
    if (a.d <= 64) return launch_kind<T, 64>(a, splits, s);
    if (a.d <= 128) return launch_kind<T, 128>(a, splits, s);
    return launch_kind<T, 256>(a, splits, s);
}

}  // namespace

hipError_t launch_attention_few(const AttnArgs &a, int splits, hipStream_t s) {
    switch (a.type) {
        case F16: return launch_size<_Float16>(a, splits, s);
        case BF16: return launch_size<__bf16>(a, splits, s);
        default: return launch_size<float>(a, splits, s);
    }
}

}  // namespace tg
