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

template <typename T>
__global__ __launch_bounds__(64 * ROW_WAVES) void attn_rows_kernel(const AttnArgs a) {
    const int b = blockIdx.z, r = blockIdx.x * ROW_WAVES + (threadIdx.x >> 6);
    if (r < span_of(a.seqs, b).nq && r < a.seqs.longest) attend_row<T>(a, b, blockIdx.y, r, threadIdx.x & 63);
}

// The parts of a row and head, joined by one wavefront: with M the largest maximum, the sums and outputs of
// part p count e^(m_p - M) times.
template <typename T>
__global__ __launch_bounds__(64 * ROW_WAVES) void attn_join_kernel(const AttnArgs a, const AttnParts parts) {
    const int lane = threadIdx.x & 63, b = blockIdx.z, h = blockIdx.y, r = blockIdx.x * ROW_WAVES + (threadIdx.x >> 6);
    const AttnSpan sp = span_of(a.seqs, b);
    if (r >= sp.nq || r >= a.seqs.longest) return;
    const size_t at = (size_t)(sp.q0 + r) * a.heads + h;
    float m = -INFINITY;
    for (int p = 0; p < parts.parts; p++) m = fmaxf(m, parts.top[p * parts.pairs + at]);
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, acc[4] = {};
    for (int p = 0; p < parts.parts; p++) {
        const size_t from = p * parts.pairs + at;
        const float w = exp2f((parts.top[from] - base) * LOG2E), sum = parts.sum[from];
        if (sum == 0.0f) continue;  // no key of this part was shown
        l = __builtin_fmaf(w, sum, l);
        for (int e = 0; e < 4; e++)
            if (e * 64 + lane < a.d) acc[e] = __builtin_fmaf(w, parts.out[from * a.d + e * 64 + lane], acc[e]);
    }
    T *out = static_cast<T *>(a.out) + (int64_t)(sp.q0 + r) * a.ldo + h * a.hso;
    bool sound = true;
    for (int e = 0; e < 4; e++)
        if (e * 64 + lane < a.d) {
            const float v = l == 0.0f ? 0.0f : acc[e] / l;
            sound = sound && v - v == 0.0f;
            out[e * 64 + lane] = (T)v;
        }
    // As the tile kernels do for rows that they finish themselves.
    if (!__all(sound) && (sizeof(T) == 4 || l - l == 0.0f)) attend_row<T>(a, b, h, r, lane);
}

template <typename T>
hipError_t launch_rows(const AttnArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)div_ceil((size_t)a.seqs.longest, ROW_WAVES), (unsigned)a.heads, (unsigned)a.seqs.batch);
    hipLaunchKernelGGL((attn_rows_kernel<T>), grid, dim3(64 * ROW_WAVES), 0, s, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_join(const AttnArgs &a, int splits, hipStream_t s) {
    const dim3 grid((unsigned)div_ceil((size_t)a.seqs.longest, ROW_WAVES), (unsigned)a.heads, (unsigned)a.seqs.batch);
    hipLaunchKernelGGL((attn_join_kernel<T>), grid, dim3(64 * ROW_WAVES), 0, s, a, parts_of(a, splits));
    return hipGetLastError();
}

// How a call is spread: workgroups of `tile` query rows and heads, and how many parts the keys are cut into so that
// about `target` workgroups run, each with `least` keys or more.
struct Spread {
    size_t tile, target, least;
};
constexpr Spread TILES{128, 512, 256}, FEW{16, 2048, 512};
constexpr size_t MOST_PARTS = 64;

size_t parts_for(const Spread &sp, size_t wgs, size_t keys) {
    size_t n = sp.target / (wgs ? wgs : 1);
    if (n > keys / sp.least) n = keys / sp.least;
    return n < 1 ? 1 : n > MOST_PARTS ? MOST_PARTS : n;
}

}  // namespace

size_t attention_work_bytes(size_t rows, size_t heads, size_t kv_heads, size_t d, size_t batch, size_t keys) {
    // The fewest workgroups that calls of these sizes have give the most parts.
    const auto parts = [&](const Spread &sp) {
        const size_t tiles = div_ceil(rows * (heads / kv_heads), sp.tile);
        return parts_for(sp, kv_heads * (tiles > batch ? tiles : batch), keys);
    };
    const size_t x = parts(TILES), y = rows * (heads / kv_heads) <= FEW.tile * batch ? parts(FEW) : 1;
    const size_t n = x > y ? x : y;
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
    const Spread &sp = few ? FEW : TILES;
    const size_t group = a.rel ? 1 : a.heads / a.kv_heads, tiles = div_ceil((size_t)a.seqs.longest * group, sp.tile);
    size_t keys = a.seqs.tables ? (size_t)a.seqs.width * a.seqs.page
                                : (size_t)(a.seqs.k_starts ? a.seqs.k_rows : a.seqs.k_rows / a.seqs.batch);
    if (a.left >= 0 && a.right >= 0 && !a.prefix) {  // no tile reaches further than its rows' windows
        const size_t reach = (size_t)a.left + a.right + 1 + sp.tile;
        keys = keys < reach ? keys : reach;
    }
    size_t n = parts_for(sp, tiles * (a.heads / group) * a.seqs.batch, keys);
    const size_t bytes = part_bytes((size_t)a.seqs.q_rows * a.heads, a.d);
    if (n * bytes > a.work_bytes) n = a.work_bytes / bytes;
    if (n < 1) n = 1;
    const hipError_t e = few                ? launch_attention_few(a, (int)n, s)
                         : a.type == F32 ? launch_attention32(a, (int)n, s)
                                         : launch_attention16(a, (int)n, s);
    if (e != hipSuccess || n == 1) return e;
    switch (a.type) {
        case F16: return launch_join<_Float16>(a, (int)n, s);
        case BF16: return launch_join<__bf16>(a, (int)n, s);
        default: return launch_join<float>(a, (int)n, s);
    }
}

}  // namespace tg
