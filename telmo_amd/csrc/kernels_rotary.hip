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

// The same in 64 bits: Taylor's polynomials of sin and cos within an eighth of a turn, to 2^-45. Their coefficients are held
// in scalar registers: in vector ones they would cost a kernel one wavefront in four.
__device__ __forceinline__ double scalar(double x) {
    asm("" : "+s"(x));
    return x;
}
__device__ __forceinline__ double2 turn64(double turns, float amplitude) {
    const double whole = __builtin_rint(turns), rest = (turns - whole) * 4.0;  // quarter turns, |rest| <= 2
    const double quarter = __builtin_rint(rest), x = (rest - quarter) * 1.57079632679489661923, y = x * x;
    double s = scalar(1.0 / 6227020800.0), c = scalar(-1.0 / 87178291200.0);
    c = __builtin_fma(c, y, scalar(1.0 / 479001600.0));
    s = __builtin_fma(s, y, scalar(-1.0 / 39916800.0)), c = __builtin_fma(c, y, scalar(-1.0 / 3628800.0));
    s = __builtin_fma(s, y, scalar(1.0 / 362880.0)), c = __builtin_fma(c, y, scalar(1.0 / 40320.0));
    s = __builtin_fma(s, y, scalar(-1.0 / 5040.0)), c = __builtin_fma(c, y, scalar(-1.0 / 720.0));
    s = __builtin_fma(s, y, scalar(1.0 / 120.0)), c = __builtin_fma(c, y, scalar(1.0 / 24.0));
    s = __builtin_fma(s, y, scalar(-1.0 / 6.0)), c = __builtin_fma(c, y, -0.5);
    s = __builtin_fma(s * y, x, x), c = __builtin_fma(c, y, 1.0);
    const int n = (int)quarter & 3;
    const double cs = n & 1 ? s : c, sn = n & 1 ? c : s;
    return make_double2(amplitude * (n == 1 || n == 2 ? -cs : cs), amplitude * (n >= 2 ? -sn : sn));
}
// (x, y) turned, in the table's bits, and rounded once.
__device__ __forceinline__ void rotate(float &x, float &y, const float2 &t) {
    const float a = x, b = y;
    x = a * t.x - b * t.y;
    y = b * t.x + a * t.y;
}
__device__ __forceinline__ void rotate(float &x, float &y, const double2 &t) {
    const double a = x, b = y;
    x = (float)__builtin_fma(a, t.x, -(b * t.y));
    y = (float)__builtin_fma(b, t.x, a * t.y);
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

// put(first, n, whether `first` is a multiple of 8, n values in 32 bits) for the eights of a piece.
template <typename T, typename Turn, typename F>
__device__ __forceinline__ void with_piece(const T *x, int piece, int d, int dim, bool interleaved, const Turn *table, F put) {
    const int half = dim / 2, turned = pair_pieces(dim);
    float v[8];
    if (piece >= turned) {
        const int c = dim + (piece - turned) * 8, n = d - c < 8 ? d - c : 8;
        load_some(x + c, n, dim % 8 == 0, v);
        put(c, n, dim % 8 == 0, v);
        return;
    }
    const int i = piece * 8, n = half - i < 8 ? half - i : 8;
    float w[8];
    if (interleaved) {
        const int m = 2 * n < 8 ? 2 * n : 8;
        load_some(x + 2 * i, m, true, v);
        load_some(x + 2 * i + 8, 2 * n - m, true, w);
        for (int e = 0; e < 8; e += 2) {
            const Turn s = e / 2 < n ? table[i + e / 2] : Turn{}, t = 4 + e / 2 < n ? table[i + 4 + e / 2] : Turn{};
            rotate(v[e], v[e + 1], s);
            rotate(w[e], w[e + 1], t);
        }
        put(2 * i, m, true, v);
        put(2 * i + 8, 2 * n - m, true, w);
    } else {
        load_some(x + i, n, true, v);
        load_some(x + half + i, n, half % 8 == 0, w);
        for (int e = 0; e < 8; e++) {
            const Turn t = e < n ? table[i + e] : Turn{};
            rotate(v[e], w[e], t);
        }
        put(i, n, true, v);
        put(half + i, n, half % 8 == 0, w);
    }
}
template <typename T, typename U>
__device__ __forceinline__ void rotate_piece(const T *x, U *out, int piece, int d, int dim, bool interleaved,
                                             const float2 *table) {
    with_piece(x, piece, d, dim, interleaved, table, [&](int at, int n, bool aligned, const float *v) { store_some(out + at, n, aligned, v); });
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

// The same into pages of e4m3 values: a block of rows of a page has a power of two for each head, which is known when all of
// the block's new rows are. A workgroup takes a block of a sequence, a wavefront one head's keys or values in it at a time:
// first the largest of the new rows, rotated, then the block's exponent, and the rows that were there before in it where
// that grows, then the new rows again, rounded.
// The rotation is worked out in 64 bits: next to a border of e4m3 an f32 one rounds three times as many values to the other
// side as one of exact products and sums in f32 would (6 to 18 of 6.6 million instead of 1 to 7).
constexpr int TURNS = 2048;  // sines and cosines held at a time

// The older rows of a block, by one wavefront, times `down`.
__device__ __forceinline__ void lower_rows(uint8_t *rows8, int64_t ldc, int older, int d, int lane, float down) {
    for (int t = lane; t < older * (d / 16); t += 64) {
        uint32_t *to = reinterpret_cast<uint32_t *>(rows8 + t / (d / 16) * ldc + t % (d / 16) * 16);
        for (int e = 0; e < 4; e++) {
            const uint32_t y = to[e];
            to[e] = e4m3_pack(__builtin_amdgcn_cvt_f32_fp8(y, 0), __builtin_amdgcn_cvt_f32_fp8(y, 1),
                              __builtin_amdgcn_cvt_f32_fp8(y, 2), __builtin_amdgcn_cvt_f32_fp8(y, 3), down);
        }
    }
}

// Heads whose rotated part is whole pieces of 16 values, in blocks whose turns fit LDS. A lane takes a piece (two eights,
// of a rotated half each, or 16 in a row) of every 64 / pieces-th row, STEPS of them at a time, and keeps a block of as many
// in registers from the largest to the rounding; a longer block's rows are read again. No piece is cut, so that a step is
// loads and products without branches. Bound by memory: four sequences' 6449 rows (2047, 1812, 1365, 1225) of 8 heads of 128 in
// f32, keys rotated, blocks of 16, 66 MB in 18.3 us (3.6 TB/s); with four steps, and so half the wavefronts, 23, by cut pieces
// 25. Eight single rows take 6.
template <typename T, bool HALVES>
__global__ __launch_bounds__(THREADS) void append8_whole_kernel(const T *k, int64_t ldk, int64_t hsk, const T *v, int64_t ldv,
                                                                int64_t hsv, const Cache8 c, int heads, int d, const AttnSeqs q,
                                                                const RotaryArgs r) {
    constexpr int STEPS = 2;
    extern __shared__ double2 table[];  // of a block's rows
    const int b = blockIdx.y;
    const AttnSpan sp = span_of(q, b);
    const int rows = sp.nq < q.longest ? sp.nq : q.longest;
    if (rows <= 0) return;
    const int64_t first = (int64_t)q.lengths[b] - sp.nq;  // as it stands, also past the table
    const int64_t at = first < 0 ? 0 : first, end = first + rows < sp.nk ? first + rows : sp.nk;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, pairs = r.dim / 2, pieces = d / 16, apart = 64 / pieces;
    const int own = lane / pieces, piece = lane % pieces;  // the first row and the piece of it
    const bool busy = own < apart;
    for (int64_t block0 = (at / c.block + blockIdx.x) * c.block; block0 < end; block0 += (int64_t)gridDim.x * c.block) {
        const int64_t lo = block0 > at ? block0 : at, hi = end < block0 + c.block ? end : block0 + c.block;
        int row0;
        const int page = page_of(q, b, (int)block0, row0);
        if (page < 0) continue;
        const int older = (int)(lo - block0), n = (int)(hi - lo);
        const int64_t from = (int64_t)sp.q0 + (lo - first);  // the first new row
        if (pairs && (int)blockIdx.z * 4 < heads) {  // a workgroup of values alone needs no turns
            __syncthreads();
            for (int t = threadIdx.x; t < n * pairs; t += THREADS) table[t] = turn64((double)(lo + t / pairs) * r.turns[t % pairs], r.amplitude);
            __syncthreads();
        }
        for (int unit = blockIdx.z * 4 + wave; unit < 2 * heads; unit += gridDim.z * 4) {
            const bool key = unit < heads;
            const int h = key ? unit : unit - heads;
            const int64_t ld = key ? ldk : ldv, ldc = key ? c.ldk : c.ldv;
            uint8_t *rows8 = key ? c.k + page * c.psk + h * c.hsk : c.v + page * c.psv + h * c.hsv;
            rows8 += row0 * ldc;
            int8_t *exps = key ? c.k_exps + page * c.k_epage : c.v_exps + page * c.v_epage;
            exps += (int64_t)(row0 / c.block) * heads + h;
            const bool turned = key && piece * 16 < r.dim;
            const int a = turned && HALVES ? piece * 8 : piece * 16, z = turned && HALVES ? pairs + piece * 8 : a + 8;
            const T *x = (key ? k + h * hsk : v + h * hsv) + from * ld;
            float y[STEPS][16];
            const auto load = [&](int done) {
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    // Rows past the last and lanes past the last piece take a row that is there.
                    const int row = min(done + i * apart + own, n - 1);
                    load8(x + row * ld + a, y[i]);
                    load8(x + row * ld + z, y[i] + 8);
                }
                if (!turned) return;
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    const double2 *w = table + min(done + i * apart + own, n - 1) * pairs + piece * 8;
#pragma unroll
                    for (int e = 0; e < 8; e++) rotate(y[i][HALVES ? e : 2 * e], y[i][HALVES ? e + 8 : 2 * e + 1], w[e]);
                }
            };
            const int chunk = STEPS * apart;
            uint32_t top = 0;
            for (int done = 0; done < n; done += chunk) {
                load(done);
#pragma unroll
                for (int i = 0; i < STEPS; i++)
#pragma unroll
                    for (int e = 0; e < 16; e++) top = max(top, e4m3_size(y[i][e]));
            }
            for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
            int now = e4m3_exponent(top);
            if (older) {
                const int had = *exps;
                if (had >= now) now = had;
                else lower_rows(rows8, ldc, older, d, lane, two_to(had - now));
            }
            const float down = two_to(-now);
            for (int done = 0; done < n; done += chunk) {
                if (n > chunk) load(done);
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    const int row = done + i * apart + own;
                    if (row >= n || !busy) continue;
                    uint8_t *to = rows8 + (older + row) * ldc;
                    *reinterpret_cast<u32x2 *>(to + a) = u32x2{e4m3_pack(y[i][0], y[i][1], y[i][2], y[i][3], down), e4m3_pack(y[i][4], y[i][5], y[i][6], y[i][7], down)};
                    *reinterpret_cast<u32x2 *>(to + z) = u32x2{e4m3_pack(y[i][8], y[i][9], y[i][10], y[i][11], down), e4m3_pack(y[i][12], y[i][13], y[i][14], y[i][15], down)};
                }
            }
            if (lane == 0) *exps = (int8_t)now;
        }
    }
}

// Any rotated part and block: a table of as many rows' turns as fit, pieces that may be cut. What is read twice comes from
// the CU's cache the second time. The 6449 rows above in blocks of 64, whose turns are worked out twice for each set of four
// heads, take 37 us, and in blocks of 16 with 40 of the 128 values rotated 34.
template <typename T>
__global__ __launch_bounds__(THREADS) void append8_kernel(const T *k, int64_t ldk, int64_t hsk, const T *v, int64_t ldv,
                                                          int64_t hsv, const Cache8 c, int heads, int d, const AttnSeqs q,
                                                          const RotaryArgs r) {
    extern __shared__ double2 table[];  // of a block's rows, or TURNS
    const int b = blockIdx.y;
    const AttnSpan sp = span_of(q, b);
    const int rows = sp.nq < q.longest ? sp.nq : q.longest;
    if (rows <= 0) return;
    const int64_t first = (int64_t)q.lengths[b] - sp.nq;  // as it stands, also past the table
    const int64_t at = first < 0 ? 0 : first, end = first + rows < sp.nk ? first + rows : sp.nk;
    const int64_t step = (int64_t)gridDim.x * c.block;
    for (int64_t block0 = (at / c.block + blockIdx.x) * c.block; block0 < end; block0 += step) {
        // The positions of the block, those from lo to hi new.
        const int64_t lo = block0 > at ? block0 : at, hi = end < block0 + c.block ? end : block0 + c.block;
        int row0;
        const int page = page_of(q, b, (int)block0, row0);
        if (page < 0) continue;
        const int older = (int)(lo - block0), n = (int)(hi - lo);
        const int64_t from = (int64_t)sp.q0 + (lo - first);  // the first new row
        const int pairs = r.dim / 2;
        const int some = pairs ? min(n, TURNS / pairs) : n;  // rows whose turns fit the table
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const auto fill = [&](int done) {
            __syncthreads();
            for (int t = threadIdx.x; t < min(some, n - done) * pairs; t += THREADS)
                table[t] = turn64((double)(lo + done + t / pairs) * r.turns[t % pairs], r.amplitude);
            __syncthreads();
        };
        if (pairs && some == n && (int)blockIdx.z * 4 < heads) fill(0);  // a workgroup of values alone needs no turns
        for (int u0 = blockIdx.z * 4; u0 < 2 * heads; u0 += gridDim.z * 4) {
            // All wavefronts make the same steps: one past the last unit does the last one's again, and writes nothing.
            const int unit = min(u0 + wave, 2 * heads - 1);
            const bool mine = u0 + wave < 2 * heads, key = unit < heads;
            const int h = key ? unit : unit - heads, dim = key ? r.dim : 0;
            const T *x = key ? k + from * ldk + h * hsk : v + from * ldv + h * hsv;
            const int64_t ld = key ? ldk : ldv;
            const int64_t ldc = key ? c.ldk : c.ldv;
            uint8_t *rows8 = key ? c.k + page * c.psk + h * c.hsk : c.v + page * c.psv + h * c.hsv;
            rows8 += row0 * ldc;
            int8_t *exps = key ? c.k_exps + page * c.k_epage : c.v_exps + page * c.v_epage;
            exps += (int64_t)(row0 / c.block) * heads + h;
            const int pieces = pieces_of(d, dim), turned = pair_pieces(dim);
            // f(the block's row, first, n, aligned, values) for the eights of the wavefront's pieces.
            const auto each = [&](auto f) {
                for (int done = 0; done < n; done += some) {
                    if (pairs && some < n && u0 < heads) fill(done);
                    const int now = min(some, n - done);
                    const auto some_pieces = [&](int piece0, int count) {
                        for (int t = lane; t < now * count; t += 64) {
                            const int row = t / count;
                            with_piece(x + (done + row) * ld, piece0 + t % count, d, dim, r.interleaved, table + row * pairs,
                                       [&](int at, int n, bool aligned, const float *y) { f(done + row, at, n, aligned, y); });
                        }
                    };
                    // Pieces that are rotated, then the others: a wavefront does either at a time.
                    some_pieces(0, turned);
                    some_pieces(turned, pieces - turned);
                }
            };
            uint32_t top = 0;
            each([&](int, int, int count, bool, const float *y) {
                for (int e = 0; e < 8; e++)
                    if (e < count) top = max(top, e4m3_size(y[e]));
            });
            for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
            int now = e4m3_exponent(top);
            if (older) {
                const int had = *exps;
                if (had >= now) {
                    now = had;
                } else if (mine) {
                    lower_rows(rows8, ldc, older, d, lane, two_to(had - now));
                }
            }
            const float down = two_to(-now);
            each([&](int row, int at, int count, bool aligned, const float *y) {
                if (!mine) return;
                uint8_t *to = rows8 + (older + row) * ldc + at;
                const uint32_t a = e4m3_pack(y[0], y[1], y[2], y[3], down), b = e4m3_pack(y[4], y[5], y[6], y[7], down);
                if (count == 8 && aligned) {
                    *reinterpret_cast<u32x2 *>(to) = u32x2{a, b};
                } else {
                    for (int e = 0; e < count; e++) to[e] = (uint8_t)((e < 4 ? a : b) >> 8 * (e % 4));
                }
            });
            if (mine && lane == 0) *exps = (int8_t)now;
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

hipError_t launch_append8(const void *k, int64_t ldk, int64_t hsk, const void *v, int64_t ldv, int64_t hsv, uint32_t type,
                          const Cache8 &c, int heads, int d, const AttnSeqs &q, const RotaryArgs &r, hipStream_t s) {
    // The blocks that the longest sequence's rows reach into; heads are spread over workgroups as far as those leave the
    // GPU's 256 CUs without eight each.
    const size_t blocks = div_ceil((size_t)q.longest, (size_t)c.block) + 1, sets = div_ceil((size_t)heads * 2, 4);
    const size_t spread = div_ceil((size_t)2048, blocks * q.batch);
    const dim3 grid((unsigned)min_of(blocks, MAX_BLOCKS), (unsigned)q.batch, (unsigned)min_of(spread, sets));
    const auto launch = [&](auto t) {
        using T = decltype(t);
        const bool whole = r.dim % 16 == 0 && (size_t)c.block * (r.dim / 2) <= TURNS;
        const auto kernel = !whole ? append8_kernel<T> : r.interleaved ? append8_whole_kernel<T, false> : append8_whole_kernel<T, true>;
        const size_t turns = min_of((size_t)c.block * (r.dim / 2), TURNS) * sizeof(double2);
        hipLaunchKernelGGL(kernel, grid, dim3(THREADS), turns, s, static_cast<const T *>(k), ldk, hsk, static_cast<const T *>(v), ldv, hsv, c,
                           heads, d, q, r);
        return hipGetLastError();
    };
    switch (type) {
        case F16: return launch(_Float16{});
        case BF16: return launch(__bf16{});
        default: return launch(float{});
    }
}

}  // namespace tg
