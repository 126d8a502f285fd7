// Attention over rows: out_i = sum_j p_ij v_j over the keys j that query i is shown, p_i their softmax of
//
//   s_ij = cap tanh(scale ((q_i + u) k_j + (q_i + w) r_c) / cap) - slope |j - i| + table[c'],
//
// c and c' the distance j - i clamped to the position rows' and the table's span; without cap, position
// rows, slopes or table those parts fall away. Shown are the keys of the query's own sequence in its
// window or prefix, in its document. A query that is shown nothing gets zeros.
//
// Statistics and sums are held in f32: one pass over the keys carries the running maximum m, the sum of
// exp(s - m) and the unnormalised output, both rescaled where m grows. Long keys of few rows are split over
// workgroups and the parts joined by a second kernel, in their order.
#include "attn_launch.hpp"
#include "attn_tile.hpp"

namespace tg {

namespace {

constexpr int ROW_WAVES = 4;

// C: the keys' type, T or e4m3.
template <typename T, typename C>
__global__ __launch_bounds__(64 * ROW_WAVES) void attn_rows_kernel(const AttnArgs a) {
    const int b = blockIdx.z, r = blockIdx.x * ROW_WAVES + (threadIdx.x >> 6);
    if (r < span_of(a.seqs, b).nq && r < a.seqs.longest) attend_row<T, C>(a, b, blockIdx.y, r, threadIdx.x & 63);
}

// The parts of a row and head, joined by one wavefront: with M the largest maximum, the sums and outputs of
// part p count e^(m_p - M) times. Lane p weighs part p; then each lane adds V values of all parts, in their order,
// STEP parts' loads on their way at a time. Bound by reading the parts: 509 rows of 32 heads of 128 in
// four parts, 34 MB, 11.6 us (2.9 TB/s); 32 single rows 4.9 us, mostly the latency of its loads in turn.
template <typename T, typename C, int V, int STEP>
__global__ __launch_bounds__(64 * ROW_WAVES) void attn_join_kernel(const AttnArgs a, const AttnParts parts) {
    typedef float fv __attribute__((ext_vector_type(V)));
    const int lane = threadIdx.x & 63, b = blockIdx.y;
    const AttnSpan sp = span_of(a.seqs, b);
    const uint32_t pair = blockIdx.x * ROW_WAVES + (threadIdx.x >> 6);
    const int r = (int)(pair / (uint32_t)a.heads), h = (int)(pair % (uint32_t)a.heads);
    if (r >= sp.nq || r >= a.seqs.longest) return;
    const size_t at = (size_t)(sp.q0 + r) * a.heads + h;
    const bool in = lane * V < a.d;
    const float *from = parts.out + at * a.d + (in ? lane * V : 0);
    const auto load = [&](int p, fv(&x)[STEP]) {
#pragma unroll
        for (int y = 0; y < STEP; y++)
            x[y] = *reinterpret_cast<const fv *>(
                from + (size_t)(p + y < parts.parts ? p + y : parts.parts - 1) * parts.pairs * a.d);
    };
    fv x[STEP];
    load(0, x);
    const float top = lane < parts.parts ? parts.top[lane * parts.pairs + at] : -INFINITY;
    const float sum = lane < parts.parts ? parts.sum[lane * parts.pairs + at] : 0.0f;
    float most = top;
    for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    // A part that was shown no key weighs nothing.
    const float weight = sum == 0.0f ? 0.0f : exp2f((top - (most == -INFINITY ? 0.0f : most)) * LOG2E);
    float l = weight * sum;
    for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
    fv acc = {};
    for (int p = 0; p < parts.parts; p += STEP) {
        if (p) load(p, x);
#pragma unroll
        for (int y = 0; y < STEP; y++) {
            const float w = p + y < parts.parts ? __shfl(weight, p + y) : 0.0f;
            if (w != 0.0f)
                for (int e = 0; e < V; e++) acc[e] = __builtin_fmaf(w, x[y][e], acc[e]);
        }
    }
    bool sound = true;
    if (in) {
        T *out = static_cast<T *>(a.out) + (int64_t)(sp.q0 + r) * a.ldo + h * a.hso + lane * V;
        for (int e = 0; e < V; e++) {
            const float y = l == 0.0f ? 0.0f : acc[e] / l;
            sound = sound && y - y == 0.0f;
            out[e] = mean_to<T>(y);
        }
    }
    // As the tile kernels do for rows that they finish themselves.
    if (!__all(sound) && (sizeof(T) == 4 || l - l == 0.0f)) attend_row<T, C>(a, b, h, r, lane);
}

template <typename T, typename C>
hipError_t launch_rows_of(const AttnArgs &a, hipStream_t s) {
    const size_t blocks = div_ceil((size_t)a.seqs.longest, ROW_WAVES);
    if (blocks > MAX_ATTN_BLOCKS) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)blocks, (unsigned)a.heads, (unsigned)a.seqs.batch);
    hipLaunchKernelGGL((attn_rows_kernel<T, C>), grid, dim3(64 * ROW_WAVES), 0, s, a);
    return hipGetLastError();
}
template <typename T>
hipError_t launch_rows(const AttnArgs &a, hipStream_t s) {
    return a.k_exps ? launch_rows_of<T, e4m3>(a, s) : launch_rows_of<T, T>(a, s);
}

template <typename T, typename C, int V, int STEP>
hipError_t launch_join_of(const AttnArgs &a, int splits, hipStream_t s) {
    const size_t blocks = div_ceil((size_t)a.seqs.longest * a.heads, ROW_WAVES);
    if (blocks > MAX_ATTN_BLOCKS) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((attn_join_kernel<T, C, V, STEP>), dim3((unsigned)blocks, (unsigned)a.seqs.batch),
                       dim3(64 * ROW_WAVES), 0, s, a, parts_of(a, splits));
    return hipGetLastError();
}
// The parts' loads on their way at a time, 4, 8 or 16: past the last part they repeat it, so not many more than there
// are (750 rows in five parts with 16 41.7 us, with 8 41.1; a chunk's four with 4 as with 16 within 1 us).
template <typename T, typename C, int V>
hipError_t launch_join_by(const AttnArgs &a, int splits, hipStream_t s) {
    return splits > 8   ? launch_join_of<T, C, V, 16>(a, splits, s)
           : splits > 4 ? launch_join_of<T, C, V, 8>(a, splits, s)
                        : launch_join_of<T, C, V, 4>(a, splits, s);
}
template <typename T>
hipError_t launch_join(const AttnArgs &a, int splits, hipStream_t s) {
    if (a.k_exps) return a.d > 128 ? launch_join_by<T, e4m3, 4>(a, splits, s) : launch_join_by<T, e4m3, 2>(a, splits, s);
    return a.d > 128 ? launch_join_by<T, T, 4>(a, splits, s) : launch_join_by<T, T, 2>(a, splits, s);
}

// How a call is spread: workgroups of `tile` query rows and heads, and how many parts the keys are cut into so that
// about `target` workgroups run, each with `least` keys or more. Without parts a chunk of 509 rows over 32768 keys takes
// 946 us (with 326), a minute's 750 f32 rows 84 (40), 2000 bf16 rows 52 (40). The targets, in us on either side:
//
//   TILES16    target 256, 512, 1024: the chunk 493, 326, 348; 100 rows over 32768 keys 137, 103, 113
//   TILES32    target 128, 256, 512: 750 rows with position rows 84, 40, 41; 4 x 750 98, 98, 119; 2000 rows 215, 135, 150
//   SMALL32    instead of TILES32, where that leaves half of the 256 CUs empty: 250 rows 33 (38), 128 rows 14.4 (16.2);
//              everywhere it would take 750 rows from 40 to 54 and 4 x 750 from 98 to 173
//   FEW        A CU holds one workgroup, whose start and end (page numbers, a cold pipeline, the wavefronts' sums)
//              nothing hides; but sequences differ in length, and more workgroups even that out. Target 256, 512, 1024,
//              2048: 16 sequences of 8192 keys and 8 key heads 102, 107, 119, 129, of up to 8192 keys (512 and 768)
//              42 to 78, 47 to 77. From one workgroup per CU on, a part more: 32 sequences of up to 8192 keys
//              110 to 134 us (114 to 150), 64 of up to 4096 108 to 136 (113 to 140), 32 of 8192 each 202 (195).
//              256 keys or more in a part (512): 2048 keys of one sequence 13.4 (15.2), eight of 750 in f32 21.6 (28.8)
//   FEW_ALONE  A single sequence's parts are alike: one round of workgroups, 32768 keys 31.5 (36.8). Heads of up to 64
//              take fewer registers and gain nothing (100,000 keys of 16 heads 97 against 89)
struct Spread {
    size_t tile, target, least;
};
constexpr Spread TILES16{128, 512, 256}, FEW{16, 512, 256}, FEW_ALONE{16, 256, 256};
constexpr Spread TILES32{128, 256, 128}, SMALL32{64, 256, 128};
constexpr size_t MOST_PARTS = 64;  // a lane of the joining wavefront each

size_t parts_for(const Spread &sp, size_t wgs, size_t keys) {
    size_t n = sp.target / (wgs ? wgs : 1);
    if (sp.tile == FEW.tile && wgs >= 256) n++;
    if (n > keys / sp.least) n = keys / sp.least;
    return n < 1 ? 1 : n > MOST_PARTS ? MOST_PARTS : n;
}

}  // namespace

size_t attention_work_bytes(size_t rows, size_t heads, size_t kv_heads, size_t d, size_t batch, size_t keys) {
    // The fewest workgroups that calls of these sizes have give the most parts.
    size_t n = 1;
    for (const Spread &sp : {TILES16, TILES32, SMALL32, FEW}) {
        const size_t tiles = div_ceil(rows * (heads / kv_heads), sp.tile), x = kv_heads * (tiles > batch ? tiles : batch);
        if (sp.tile == FEW.tile && rows * (heads / kv_heads) > FEW.tile * batch) continue;
        const size_t parts = parts_for(sp, x, keys);
        n = n > parts ? n : parts;
    }
    return n > 1 ? n * part_bytes(rows * heads, d) : 0;
}

hipError_t launch_attention(const AttnArgs &a, hipStream_t s) {
    const bool few = attention_few_fits(a);
    // LDS holds the blocks of position rows of heads of up to 128, and a tile's offsets fit 32 bits up to row strides
    // of 8 million values: what does not fit takes a wavefront per row.
    if (!few && (!tile_strides_fit(a) || (a.type == F32 && !attention32_fits(a)))) {
        switch (a.type) {
            case F16: return launch_rows<_Float16>(a, s);
            case BF16: return launch_rows<__bf16>(a, s);
            default: return launch_rows<float>(a, s);
        }
    }
    const size_t group = a.rel ? 1 : a.heads / a.kv_heads;
    // Workgroups with work: the longest sequence bounds each one's tiles, and the rows those of all. With the first bound
    // alone nine ragged sequences of 1124 f32 rows took 39.5 us (29.1), two of 2427 rows in f16 42.4 (35.7). Chunks over
    // pages keep to it: more parts than it gives made 8 ragged ones over 1520 keys slower (74 us for 58), 3 over 5837
    // too (32 for 28).
    const auto wgs_of = [&](const Spread &sp) {
        const size_t each = div_ceil((size_t)a.seqs.longest * group, sp.tile) * a.seqs.batch;
        const size_t all = div_ceil((size_t)a.seqs.q_rows * group, sp.tile) + a.seqs.batch;
        return (all < each && !a.seqs.tables ? all : each) * (a.heads / group);
    };
    size_t keys = a.seqs.tables ? (size_t)a.seqs.width * a.seqs.page
                  : !a.seqs.k_starts ? (size_t)(a.seqs.k_rows / a.seqs.batch)
                  : a.seqs.k_starts == a.seqs.q_starts ? (size_t)a.seqs.longest
                                                       : (size_t)a.seqs.k_rows;
    const size_t bytes = part_bytes((size_t)a.seqs.q_rows * a.heads, a.d);
    const auto parts = [&](const Spread &sp) {
        size_t reach = keys;
        if (a.left >= 0 && a.right >= 0 && !a.prefix) {  // no tile reaches further than its rows' windows
            const size_t most = (size_t)a.left + a.right + 1 + sp.tile;
            reach = reach < most ? reach : most;
        }
        size_t n = parts_for(sp, wgs_of(sp), reach);
        if (n * bytes > a.work_bytes) n = a.work_bytes / bytes;
        return n < 1 ? (size_t)1 : n;
    };
    const bool tiles32 = !few && a.type == F32 && !a.k_exps;
    Spread sp = few ? (a.seqs.batch == 1 && a.d > 64 ? FEW_ALONE : FEW) : tiles32 ? TILES32 : TILES16;
    size_t n = parts(sp);
    // f32 tiles of 64 rows where those of 128 leave half of the GPU's 256 CUs empty.
    if (tiles32 && wgs_of(sp) * n <= 128) {
        sp = SMALL32;
        n = parts(sp);
    }
    const hipError_t e = a.k_exps  ? (few ? launch_attention8_few(a, (int)n, s) : launch_attention8(a, (int)n, s))
                         : few     ? launch_attention_few(a, (int)n, s)
                         : tiles32 ? launch_attention32(a, (int)sp.tile, (int)n, s)
                                   : launch_attention16(a, (int)n, s);
    if (e != hipSuccess || n == 1) return e;
    switch (a.type) {
        case F16: return launch_join<_Float16>(a, (int)n, s);
        case BF16: return launch_join<__bf16>(a, (int)n, s);
        default: return launch_join<float>(a, (int)n, s);
    }
}

}  // namespace tg
