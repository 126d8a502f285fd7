// Attention of few query rows (single tokens) over a cache in e4m3: bound by reading the keys and values once.
//
// The rows of a sequence that share a key head are the 16 columns of 16 x 16 x 32 products in bf16, which holds every
// value of e4m3 exactly, also times its block's power of two; the rows and the weights are sums of bf16 parts, as many as
// their type needs. Nothing of the keys is used twice, so LDS does not hold them: each wavefront takes tiles of 32 keys
// of its own and loads the operands of S' = K Q' as the products want them, 16 bytes of 16 rows (a piece is two
// operands, whose columns Q takes in the same order), and V by whole rows. V' wants eight keys side by side: bytes of
// eight rows, exchanged in registers before they are widened. K is widened with its row's power of two, which
// multiplies V's weights instead, exactly. The output's columns are numbered so that a lane's loads are contiguous.
// The wavefronts' results are joined in LDS, and those of the parts by a second kernel.
//
// 32 sequences of up to 8192 keys, 8 key heads of 128 and 32 heads in bf16: 279 MB in 70 us, 4.0 TB/s (a large copy 4.85, reads
// and writes), and 5 for the join. Eight sequences of 750 keys take 17 us a call, as over keys of 16 bits (15):
// page numbers, loads and sums wait for one another, not for bytes.
#include "attn_launch.hpp"
#include "attn_tile.hpp"

namespace tg {

namespace {

constexpr int COLS = 16, TILE = 32, WAVES = 4, THREADS = 64 * WAVES;

__device__ __forceinline__ f32x4 mfma(u32x4 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), b, c, 0, 0, 0);
}

// Memory of the GPU, said where the compiler would take an address for LDS's or memory's and wait for both.
template <typename T>
using Global = const __attribute__((address_space(1))) T *;

// bf16 parts of a row's values, and of a weight: rounded parts of eight bits each, 2^-18 (f32: 2^-27) of it left out.
template <typename T>
constexpr int ROW_PARTS = __is_same(T, float) ? 3 : __is_same(T, _Float16) ? 2 : 1;
template <typename T>
constexpr int WEIGHT_PARTS = __is_same(T, float) ? 3 : 2;

// D: head size rounded up to 64, 128 or 256. EXTRA: scores are capped or biased.
template <typename T, int D, bool EXTRA>
__global__ __launch_bounds__(THREADS) void attn8_few_kernel(const AttnArgs a, const AttnParts parts) {
    constexpr int PITCH = D + 4;
    constexpr int KS = D / 64;              // 16-byte pieces of a lane's part of a K row
    constexpr int KT = TILE / 16;           // K rows of a lane
    constexpr int VROWS = 8;                // V rows of a lane
    constexpr int CH = D / 16, VW = CH / 4; // values and words of a lane's piece of a V row
    constexpr int DEPTH = D == 256 ? 2 : 3; // tiles whose operands are under way
    constexpr int QP = ROW_PARTS<T>, WP = WEIGHT_PARTS<T>;
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

    // Columns 64 s + 16 quarter + 8 e of the lane's row: what the e-th operand of piece s of K holds.
    bf16x8 qf[KS][2][QP];
    {
        const T *q = static_cast<const T *>(a.q) + row * a.ldq + h * a.hsq;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int c = s * 64 + quarter * 16 + e * 8;
                float x[8] = {};
                if (live && c < a.d) load8(q + c, x);
                cut_parts(x, qf[s][e]);
            }
    }

    const char *kbase = static_cast<const char *>(a.k) + kvh * a.hsk, *vbase = static_cast<const char *>(a.v) + kvh * a.hsv;
    const int8_t *k_exps = a.k_exps + kvh, *v_exps = a.v_exps + kvh;
    const bool one_page = a.seqs.page % TILE == 0;  // a tile lies in one page
    // A tile's operands in registers, DEPTH tiles' at a time.
    struct Operands {
        u32x4 k[KT][KS];
        uint32_t v[VROWS][VW];
        int exps;         // the lane's: of key lane % 32, K's in the lower lanes and V's in the upper ones
        uint32_t hidden;  // keys that have no place
    } buf[DEPTH];
    // Lane n of a wavefront looks up the tile's key n % 32.
    int page = 0, page_row = 0;
    const auto look = [&](int kb) {
        const int key = kb + lane % TILE;
        page = page_of(a.seqs, b, key < sp.nk ? key : sp.nk - 1, page_row);
    };
    // The wavefront's last tile. Past it loads read one row of it, and what they bring is hidden: DEPTH tiles' loads are
    // always under way, so that the compiler knows how many it need not wait for.
    const int last_tile = n1 - 1 - (n1 - 1 - n0) % WAVES;
    const auto tile_at = [&](int n) { return tiles.at(n < last_tile ? n : last_tile); };
    // The operands of tile n, which was looked up last, leave memory; the tile after it is looked up before they do,
    // so that waiting for its pages does not wait for them. Addresses first: the loads in one run.
    const auto load = [&](Operands &x, int n) {
        const int kb = tile_at(n);
        const bool real = n <= last_tile;
        int64_t kp[KT], vp[VROWS];  // offsets from the head's first value
        const auto key_of = [&](int key) { return !real ? 0 : kb + key < sp.nk ? key : sp.nk - 1 - kb; };  // within the tile
        const auto v_key = [&](int e) { return (e / 4) * 16 + quarter * 4 + e % 4; };
        x.hidden = (uint32_t)__ballot(page < 0);
        const int p = page < 0 ? 0 : page;
        const int64_t exp_at = lane < TILE ? block_at(a, a.k_epage, p, page_row) : block_at(a, a.v_epage, p, page_row);
        const int8_t *const exp_of = (lane < TILE ? k_exps : v_exps) + exp_at;
        if (one_page) {  // all of the tile's keys follow its first
            const int first = __builtin_amdgcn_readlane(p, 0), at = __builtin_amdgcn_readlane(page_row, 0);
            const int64_t kat = first * a.psk + at * a.ldk, vat = first * a.psv + at * a.ldv;
#pragma unroll
            for (int y = 0; y < KT; y++) kp[y] = kat + key_of(y * 16 + col) * a.ldk;
#pragma unroll
            for (int e = 0; e < VROWS; e++) vp[e] = vat + key_of(v_key(e)) * a.ldv;
        } else {
            const int64_t kat = p * a.psk + page_row * a.ldk, vat = p * a.psv + page_row * a.ldv;
            const auto from = [&](int64_t offset, int lane_of) {
                const int lo = __shfl((int)(uint32_t)offset, lane_of), hi = __shfl((int)(offset >> 32), lane_of);
                return (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
            };
#pragma unroll
            for (int y = 0; y < KT; y++) kp[y] = from(kat, key_of(y * 16 + col));
#pragma unroll
            for (int e = 0; e < VROWS; e++) vp[e] = from(vat, key_of(v_key(e)));
        }
        look(tile_at(n + WAVES));
        x.exps = *(Global<int8_t>)exp_of;
#pragma unroll
        for (int y = 0; y < KT; y++)
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const int c = s * 64 + quarter * 16;
                x.k[y][s] = *(Global<u32x4>)(kbase + kp[y] + (c < a.d ? c : 0));
            }
        // Rows past the last key and columns past d are read as others: weighted by zero, or not stored.
        const int c = col * CH < a.d ? col * CH : 0;
#pragma unroll
        for (int e = 0; e < VROWS; e++) {
            if constexpr (VW == 4) {
                const u32x4 y = *(Global<u32x4>)(vbase + vp[e] + c);
                for (int z = 0; z < 4; z++) x.v[e][z] = y[z];
            } else if constexpr (VW == 2) {
                const u32x2 y = *(Global<u32x2>)(vbase + vp[e] + c);
                for (int z = 0; z < 2; z++) x.v[e][z] = y[z];
            } else {
                x.v[e][0] = *(Global<uint32_t>)(vbase + vp[e] + c);
            }
        }
    };

    f32x4 acc[CH] = {};
    float m = -INFINITY, l = 0.0f;
    const float to_log2 = EXTRA ? LOG2E : a.scale * LOG2E;

    const auto work = [&](Operands &o, int n) {
        const int kb = tile_at(n);
        const bool real = n <= last_tile;
        const uint32_t hide = o.hidden;
        if (a.d < D) {  // zeros where the queries' zeros may meet a value of any kind
#pragma unroll
            for (int x = 0; x < KT; x++)
#pragma unroll
                for (int s = 0; s < KS; s++)
                    if (s * 64 + quarter * 16 >= a.d) o.k[x][s] = u32x4{};
        }
        // Rows past the last key hold its values: their powers of two are its, too (their lanes looked it up).
        const float power = two_to(o.exps);
        f32x4 s[KT] = {};
#pragma unroll
        for (int x = 0; x < KT; x++) {
            const float up = __shfl(power, x * 16 + col);
#pragma unroll
            for (int y = 0; y < KS; y++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t lo = o.k[x][y][2 * e], hi = o.k[x][y][2 * e + 1];
                    const u32x4 k = {e4m3_widen<false>(lo, up), e4m3_widen<true>(lo, up), e4m3_widen<false>(hi, up),
                                     e4m3_widen<true>(hi, up)};
#pragma unroll
                    for (int z = QP - 1; z >= 0; z--) s[x] = mfma(k, qf[y][e][z], s[x]);
                }
        }

        const bool full = real && ((kb >= w_last.lo && kb + TILE <= w_first.hi) || kb + TILE <= w_first.prefix);
        constexpr int N = 4 * KT;
        if (EXTRA)
            scores_of<!__is_same(T, float), N, true>(
                a, [&](int e) -> float & { return reinterpret_cast<float *>(&s[e / 4])[e % 4]; },
                [&](int e) { return kb + e / 4 * 16 + quarter * 4 + e % 4; }, h, slope, i);
        if (!full || hide) {
            const uint32_t bits = (uint32_t)shown_bits<false, TILE>(win, kb, real ? hide : ~0ull, 0, 0) >> 4 * quarter;
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
            for (int x = 0; x < CH; x++) acc[x] *= fade;
            m = mn;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        f32x8 p;
#pragma unroll
        for (int e = 0; e < N; e++) {
            p[e] = __builtin_amdgcn_exp2f((s[e / 4][e % 4] - base) * to_log2);
            l += p[e];
            p[e] *= __shfl(power, TILE + e / 4 * 16 + quarter * 4 + e % 4);
        }
        bf16x8 w[WP];
#pragma unroll
        for (int z = 0; z < WP; z++) {
            w[z] = __builtin_convertvector(p, bf16x8);
            if (z + 1 < WP) p -= __builtin_convertvector(w[z], f32x8);
        }
        // Words of four rows' values of four columns become words of four columns' values of four rows.
#pragma unroll
        for (int y = 0; y < VW; y++) {
            uint32_t turned[2][4];
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const uint32_t v0 = o.v[4 * g][y], v1 = o.v[4 * g + 1][y], v2 = o.v[4 * g + 2][y], v3 = o.v[4 * g + 3][y];
                const uint32_t a01 = __builtin_amdgcn_perm(v1, v0, 0x05010400u), b01 = __builtin_amdgcn_perm(v1, v0, 0x07030602u);
                const uint32_t a23 = __builtin_amdgcn_perm(v3, v2, 0x05010400u), b23 = __builtin_amdgcn_perm(v3, v2, 0x07030602u);
                turned[g][0] = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
                turned[g][1] = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
                turned[g][2] = __builtin_amdgcn_perm(b23, b01, 0x05040100u);
                turned[g][3] = __builtin_amdgcn_perm(b23, b01, 0x07060302u);
            }
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const u32x4 v = {e4m3_widen<false>(turned[0][x], 1.0f), e4m3_widen<true>(turned[0][x], 1.0f),
                                 e4m3_widen<false>(turned[1][x], 1.0f), e4m3_widen<true>(turned[1][x], 1.0f)};
#pragma unroll
                for (int z = WP - 1; z >= 0; z--) acc[4 * y + x] = mfma(v, w[z], acc[4 * y + x]);
            }
        }
    };

    if (n0 < n1) {
        look(tile_at(n0));
#pragma unroll
        for (int x = 0; x < DEPTH; x++) load(buf[x], n0 + x * WAVES);
        for (int n = n0; n <= last_tile; n += DEPTH * WAVES)
#pragma unroll
            for (int x = 0; x < DEPTH; x++) {
                work(buf[x], n + x * WAVES);
                load(buf[x], n + (x + DEPTH) * WAVES);
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
    for (int e = 0; e < 4; e++)
#pragma unroll
        for (int x = 0; x < CH; x += 4)
            *reinterpret_cast<f32x4 *>(&outs[wave][col][(quarter * 4 + e) * CH + x]) =
                f32x4{acc[x][e], acc[x + 1][e], acc[x + 2][e], acc[x + 3][e]};
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
        if constexpr (sizeof(T) == 4) *reinterpret_cast<u32x4 *>(out) = *reinterpret_cast<u32x4 *>(v);
        else *reinterpret_cast<u32x2 *>(out) = *reinterpret_cast<u32x2 *>(v);
        if (!sound && sum - sum == 0.0f) again[oc] = 1;
    }
    if (parts.parts > 1) return;
    // A hidden key's NaN beside a sound sum of weights, as in the tile kernels.
    __syncthreads();
    for (int x = wave; x < COLS; x += WAVES)
        if (again[x]) attend_row<T, e4m3>(a, b, kvh * group + x - row_of(x) * group, row_of(x), lane);
}

template <typename T, int D, bool EXTRA>
hipError_t launch_few(const AttnArgs &a, int splits, hipStream_t s) {
    const size_t blocks = (size_t)a.seqs.batch * a.kv_heads * splits;
    if (blocks > MAX_ATTN_BLOCKS / 2) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((attn8_few_kernel<T, D, EXTRA>), dim3((unsigned)blocks), dim3(THREADS), 0, s, a,
                       parts_of(a, splits));
    return hipGetLastError();
}

template <typename T>
hipError_t launch_size(const AttnArgs &a, int splits, hipStream_t s) {
    const bool extra = a.cap > 0.0f || a.slopes || a.table;
    if (a.d <= 64) return extra ? launch_few<T, 64, true>(a, splits, s) : launch_few<T, 64, false>(a, splits, s);
    if (a.d <= 128) return extra ? launch_few<T, 128, true>(a, splits, s) : launch_few<T, 128, false>(a, splits, s);
    return extra ? launch_few<T, 256, true>(a, splits, s) : launch_few<T, 256, false>(a, splits, s);
}

}  // namespace

hipError_t launch_attention8_few(const AttnArgs &a, int splits, hipStream_t s) {
    switch (a.type) {
        case F16: return launch_size<_Float16>(a, splits, s);
        case BF16: return launch_size<__bf16>(a, splits, s);
        default: return launch_size<float>(a, splits, s);
    }
}

}  // namespace tg
