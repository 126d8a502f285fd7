// Rotary positions, and new keys and values into their pages.
//
// A pair (x, y) of a head at position p becomes amplitude (x cos t - y sin t, y cos t + x sin t), t = p f
// for the pair's angle per position f. p f has no place in 32 bits (a position of a million times a
// frequency of one radian keeps 2^-4 radians), so the turns p f / 2 pi are a 64-bit product whose whole
// turns are dropped in 64 bits; what is left is exact enough in 32. A workgroup takes rows, works out
// each row's sines and cosines once into LDS and rotates all heads with them: the kernel moves x in and
// out and the 64-bit work is one pair in each head's place. Bound by memory: 16384 rows of 32 heads of 128 in
// bf16, half of each rotated, 268 MB in 64.4 us (4.2 TB/s; a large copy 4.8); eight rows take the time of a call,
// 7.5 us. Four rows to a workgroup keep 256 lanes busy with the pairs of heads of 128 in one step.
#include "attn_common.hpp"

namespace tg {

namespace {

constexpr int THREADS = 256;
constexpr int MAX_PAIRS = 128;  // pairs of a head of 256
constexpr int ROWS = 4;         // rows per workgroup at a time
constexpr size_t MAX_BLOCKS = 1 << 20;

inline size_t min_of(size_t a, size_t b) { return a < b ? a : b; }

// sin and cos of 2 pi turns, times amplitude.
__device__ __forceinline__ float2 turn(double turns, float amplitude) {
    const double whole = __builtin_rint(turns), rest = (turns - whole) * 4.0;  // quarter turns, |rest| <= 2
    const double quarter = __builtin_rint(rest);
    float s, c;
    sincospif((float)((rest - quarter) * 0.5), &s, &c);
    const int n = (int)quarter & 3;
    const float cs = n & 1 ? s : c, sn = n & 1 ? c : s;
    return make_float2(amplitude * (n == 1 || n == 2 ? -cs : cs), amplitude * (n >= 2 ? -sn : sn));
}

// n <= 8 values at p in 32 bits, in one piece where all eight are wanted and p is aligned.
template <typename T>
__device__ __forceinline__ void load_some(const T *p, int n, bool aligned, float *v) {
    if (n == 8 && aligned) {
        load8(p, v);
    } else {
        for (int e = 0; e < 8; e++) v[e] = e < n ? to_f32(p[e]) : 0.0f;
    }
}
template <typename U>
__device__ __forceinline__ void store_some(U *p, int n, bool aligned, const float *v) {
    if (n == 8 && aligned) {
        store8(p, v);
    } else {
        for (int e = 0; e < n; e++) p[e] = (U)v[e];
    }
}

// The pieces a head is worked in: eight pairs each, then eight of the values behind the rotated ones.
// A piece reads all that it overwrites before it writes, so out may be x.
__host__ __device__ inline int pair_pieces(int dim) { return (dim / 2 + 7) / 8; }
__host__ __device__ inline int pieces_of(int d, int dim) { return pair_pieces(dim) + (d - dim + 7) / 8; }

template <typename T, typename U>
__device__ __forceinline__ void rotate_piece(const T *x, U *out, int piece, int d, int dim, bool interleaved,
                                             const float2 *table) {
    const int half = dim / 2, turned = pair_pieces(dim);
    float v[8];
    if (piece >= turned) {
        const int c = dim + (piece - turned) * 8, n = d - c < 8 ? d - c : 8;
        load_some(x + c, n, dim % 8 == 0, v);
        store_some(out + c, n, dim % 8 == 0, v);
        return;
    }
    const int i = piece * 8, n = half - i < 8 ? half - i : 8;
    float w[8];
    if (interleaved) {
        const int m = 2 * n < 8 ? 2 * n : 8;
        load_some(x + 2 * i, m, true, v);
        load_some(x + 2 * i + 8, 2 * n - m, true, w);
        for (int e = 0; e < 8; e += 2) {
            const float2 s = e / 2 < n ? table[i + e / 2] : make_float2(0.0f, 0.0f);
            const float2 t = 4 + e / 2 < n ? table[i + 4 + e / 2] : make_float2(0.0f, 0.0f);
            const float a = v[e], b = v[e + 1], f = w[e], g = w[e + 1];
            v[e] = a * s.x - b * s.y, v[e + 1] = b * s.x + a * s.y;
            w[e] = f * t.x - g * t.y, w[e + 1] = g * t.x + f * t.y;
        }
        store_some(out + 2 * i, m, true, v);
        store_some(out + 2 * i + 8, 2 * n - m, true, w);
    } else {
        load_some(x + i, n, true, v);
        load_some(x + half + i, n, half % 8 == 0, w);
        for (int e = 0; e < 8; e++) {
            const float2 t = e < n ? table[i + e] : make_float2(0.0f, 0.0f);
            const float a = v[e], b = w[e];
            v[e] = a * t.x - b * t.y;
            w[e] = b * t.x + a * t.y;
        }
        store_some(out + i, n, true, v);
        store_some(out + half + i, n, half % 8 == 0, w);
    }
}

template <typename T, typename U>
__global__ __launch_bounds__(THREADS) void rotary_kernel(const T *x, int64_t ldx, int64_t hsx, U *out, int64_t ldo,
                                                         int64_t hso, size_t rows, int heads, int d,
                                                         const int32_t *positions, int64_t start, const RotaryArgs r) {
    __shared__ float2 table[ROWS][MAX_PAIRS];
    const int pairs = r.dim / 2, pieces = pieces_of(d, r.dim);
    for (size_t r0 = (size_t)blockIdx.x * ROWS; r0 < rows; r0 += (size_t)gridDim.x * ROWS) {
        const int n = rows - r0 < ROWS ? (int)(rows - r0) : ROWS;
        __syncthreads();
        for (int t = threadIdx.x; t < n * pairs; t += THREADS) {
            const size_t row = r0 + t / pairs;
            const double p = positions ? (double)positions[row] : (double)(start + (int64_t)row);
            table[t / pairs][t % pairs] = turn(p * r.turns[t % pairs], r.amplitude);
        }
        __syncthreads();
        for (int t = threadIdx.x; t < n * heads * pieces; t += THREADS) {
            const int at = t / (heads * pieces), h = t / pieces % heads;
            const int64_t row = (int64_t)r0 + at;
            rotate_piece(x + row * ldx + h * hsx, out + row * ldo + h * hso, t % pieces, d, r.dim, r.interleaved,
                         table[at]);
        }
    }
}

// The rows of all sequences, a page lookup per row. Four sequences' 6449 rows (2047, 1812, 1365, 1225) of 8 f32 heads of
// 128 into bf16 pages: 79 MB of reads and writes in 19.6 us (4.05 TB/s).
template <typename T, typename U>
__global__ __launch_bounds__(THREADS) void append_kernel(const T *k, int64_t ldk, int64_t hsk, const T *v,
                                                         int64_t ldv, int64_t hsv, U *ck, int64_t ldck, int64_t hsck,
                                                         int64_t psk, U *cv, int64_t ldcv, int64_t hscv, int64_t psv,
                                                         int heads, int d, const AttnSeqs q, const RotaryArgs r) {
    __shared__ float2 table[ROWS][MAX_PAIRS];
    __shared__ int page[ROWS], in_page[ROWS];
    const int b = blockIdx.y;
    const AttnSpan sp = span_of(q, b);
    const int pairs = r.dim / 2, k_pieces = pieces_of(d, r.dim), pieces = k_pieces + d / 8;
    const int rows = sp.nq < q.longest ? sp.nq : q.longest;
    // The length as it stands, also past the table: cut to it, new rows would take older ones' places.
    const int64_t first = (int64_t)q.lengths[b] - sp.nq;
    for (int r0 = blockIdx.x * ROWS; r0 < rows; r0 += gridDim.x * ROWS) {
        const int n = rows - r0 < ROWS ? rows - r0 : ROWS;
        __syncthreads();
        if ((int)threadIdx.x < n) {
            const int64_t pos = first + r0 + threadIdx.x;
            const bool held = pos >= 0 && pos < sp.nk;
            int at = 0;
            page[threadIdx.x] = held ? page_of(q, b, (int)pos, at) : -1;
            in_page[threadIdx.x] = at;
        }
        for (int t = threadIdx.x; t < n * pairs; t += THREADS)
            table[t / pairs][t % pairs] = turn((double)(first + r0 + t / pairs) * r.turns[t % pairs], r.amplitude);
        __syncthreads();
        for (int t = threadIdx.x; t < n * heads * pieces; t += THREADS) {
            const int at = t / (heads * pieces), h = t / pieces % heads, piece = t % pieces;
            if (page[at] < 0) continue;
            const int64_t row = (int64_t)sp.q0 + r0 + at;
            if (piece < k_pieces)
                rotate_piece(k + row * ldk + h * hsk, ck + page[at] * psk + in_page[at] * ldck + h * hsck, piece, d,
                             r.dim, r.interleaved, table[at]);
            else
                rotate_piece(v + row * ldv + h * hsv, cv + page[at] * psv + in_page[at] * ldcv + h * hscv,
                             piece - k_pieces, d, 0, false, table[at]);
        }
    }
}

template <typename T, typename U>
hipError_t rotary_to(const void *x, int64_t ldx, int64_t hsx, void *out, int64_t ldo, int64_t hso, size_t rows,
                     int heads, int d, const int32_t *positions, int64_t start, const RotaryArgs &r, hipStream_t s) {
    hipLaunchKernelGGL((rotary_kernel<T, U>), dim3((unsigned)min_of(div_ceil(rows, ROWS), MAX_BLOCKS)), dim3(THREADS), 0, s,
                       static_cast<const T *>(x), ldx, hsx, static_cast<U *>(out), ldo, hso, rows, heads, d, positions,
                       start, r);
    return hipGetLastError();
}

// f(T{}, U{}) for the stored types.
template <typename F>
hipError_t with_types(uint32_t type, uint32_t out_type, F f) {
    const auto to = [&](auto t) {
        switch (out_type) {
            case F16: return f(t, _Float16{});
            case BF16: return f(t, __bf16{});
            default: return f(t, float{});
        }
    };
    switch (type) {
        case F16: return to(_Float16{});
        case BF16: return to(__bf16{});
        default: return to(float{});
    }
}

}  // namespace

hipError_t launch_rotary(const void *x, uint32_t type, int64_t ldx, int64_t hsx, void *out, uint32_t out_type,
                         int64_t ldo, int64_t hso, size_t rows, int heads, int d, const int32_t *positions,
                         int64_t start, const RotaryArgs &r, hipStream_t s) {
    return with_types(type, out_type, [&](auto t, auto u) {
        return rotary_to<decltype(t), decltype(u)>(x, ldx, hsx, out, ldo, hso, rows, heads, d, positions, start, r, s);
    });
}

hipError_t launch_append(const void *k, int64_t ldk, int64_t hsk, const void *v, int64_t ldv, int64_t hsv,
                         uint32_t type, void *ck, int64_t ldck, int64_t hsck, int64_t psk, void *cv, int64_t ldcv,
                         int64_t hscv, int64_t psv, uint32_t cache_type, int heads, int d, const AttnSeqs &q,
                         const RotaryArgs &r, hipStream_t s) {
    return with_types(type, cache_type, [&](auto t, auto u) {
        using T = decltype(t);
        using U = decltype(u);
        const dim3 grid((unsigned)min_of(div_ceil((size_t)q.longest, ROWS), MAX_BLOCKS), (unsigned)q.batch);
        hipLaunchKernelGGL((append_kernel<T, U>), grid, dim3(THREADS), 0, s, static_cast<const T *>(k), ldk, hsk,
                           static_cast<const T *>(v), ldv, hsv, static_cast<U *>(ck), ldck, hsck, psk,
                           static_cast<U *>(cv), ldcv, hscv, psv, heads, d, q, r);
        return hipGetLastError();
    });
}

}  // namespace tg
