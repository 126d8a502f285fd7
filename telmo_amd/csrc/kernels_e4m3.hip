// The product of rows and weights in eight bits: c = epi(a' w'^T), w' of e4m3 values with an f32 scale for each block of
// 128 outputs by 128 inputs, a' the rows rounded to e4m3 in groups of 128 inputs with a power of two each (e4m3.hpp):
//
//   c_ij = sum over blocks b of S[j / 128][b] sum over k in b of 2^e_ib a8_ik w8_jk
//
// S is one number for all of a wavefront's outputs, and one multiply-add per output adds a block to its f32 sum. The inner
// sum is made in one of two ways:
//
//   EXACT    the values are widened to bf16, which holds them exactly (the rows' with their power of two), and multiplied
//            16 x 16 x 32 at a time: products are exact and sums f32. Few rows, which are bound by the weights' bytes, and
//            all f32 outputs take this.
//   !EXACT   one instruction of 16 x 16 x 128 in e4m3, which takes the rows' powers of two as they are, at twice the rate.
//            It aligns its products before it adds them, and what lies 2^-13 below the largest of 32 of them is lost:
//            measured against 64 bits a sum of 128 is off by up to 2^-11.5 of its largest product, 1.1e-5 of the outputs'
//            norm where both sides are normal (EXACT 1e-7). That is too coarse for an f32 output, and a hundredth of what a
//            16-bit one is rounded by: many rows with 16-bit outputs take this.
//
// Operands lie in memory as the instruction takes them ("fragments"): for 16 rows (outputs) and a block of 128 inputs 2 KB
// in two halves of 64 lanes by 16 bytes, lane 16 g + r of half h holding the inputs 64 h + 16 g + [0, 16) of row r. Both
// sides number the inputs alike, so any such order gives the sum. Reads of LDS and copies to it are linear.
#include "e4m3.hpp"
#include "e4m3_product.hpp"

namespace tg {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A lane's 32 values of a fragment as the product takes them, widened times `up` where it is EXACT.
template <bool EXACT>
struct Operand {
    i32x8 v;
    __device__ __forceinline__ Operand(const i32x8 &bytes, float) : v(bytes) {}
};
template <>
struct Operand<true> {
    bf16x8 v[4];
    __device__ __forceinline__ Operand(const i32x8 &bytes, float up) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = (uint32_t)bytes[2 * i], hi = (uint32_t)bytes[2 * i + 1];
            v[i] = __builtin_bit_cast(bf16x8, u32x4{e4m3_widen<false>(lo, up), e4m3_widen<true>(lo, up),
                                                    e4m3_widen<false>(hi, up), e4m3_widen<true>(hi, up)});
        }
    }
};
// 16 outputs by 16 rows of one block of inputs; rows' powers of two, where they are not in a yet, in byte Q of each lane's
// word.
template <int Q>
__device__ __forceinline__ f32x4 block_product(const Operand<false> &w, const Operand<false> &a, uint32_t powers) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, a.v, f32x4{}, 0, 0, 0, 127, Q, (int)powers);
}
template <int Q>
__device__ __forceinline__ f32x4 block_product(const Operand<true> &w, const Operand<true> &a, uint32_t) {
    f32x4 sum = {};
#pragma unroll
    for (int i = 0; i < 4; i++) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], a.v[i], sum, 0, 0, 0);
    return sum;
}
// Byte q of a word of powers, e + 127 each, as 2^e.
__device__ __forceinline__ float power_of(uint32_t powers, int q) { return __uint_as_float((powers >> 8 * q & 255u) << 23); }
__device__ __forceinline__ i32x8 joined(i32x4 a, i32x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

__device__ __forceinline__ float max_of_quarters(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}

// Sixteen inputs of a row from k0 on in 32 bits, zeros past the last.
template <typename T>
__device__ __forceinline__ void load16(const T *row, size_t k0, size_t k, bool aligned, float *x) {
    if (aligned && k0 + 16 <= k) {
        if constexpr (sizeof(T) == 4) {
            for (int i = 0; i < 4; i++) {
                const f32x4 v = reinterpret_cast<const f32x4 *>(row + k0)[i];
                for (int e = 0; e < 4; e++) x[4 * i + e] = v[e];
            }
        } else {
            typedef T v8 __attribute__((ext_vector_type(8)));
            for (int i = 0; i < 2; i++) {
                const v8 v = reinterpret_cast<const v8 *>(row + k0)[i];
                for (int e = 0; e < 8; e++) x[8 * i + e] = (float)v[e];
            }
        }
    } else {
        for (int e = 0; e < 16; e++) x[e] = k0 + e < k ? (float)row[k0 + e] : 0.0f;
    }
}

// The lane's part of a fragment of the rows: row `row` (zeros where there is none) from input 128 b on, rounded under
// the exponent of the row's group, which the four lanes of a row find together.
template <typename T>
__device__ __forceinline__ i32x8 round_rows(const T *a, size_t lda, size_t row, bool real, size_t b, size_t k, bool aligned,
                                            int quarter, int &e) {
    float x[2][16] = {};
    if (real)
        for (int h = 0; h < 2; h++) load16(a + row * lda, b * 128 + h * 64 + quarter * 16, k, aligned, x[h]);
    uint32_t top = 0;
    for (int h = 0; h < 2; h++)
        for (int i = 0; i < 16; i++) {
            const uint32_t size = e4m3_size(x[h][i]);
            top = top > size ? top : size;
        }
    e = e4m3_exponent(__float_as_uint(max_of_quarters(__uint_as_float(top))));
    const float down = two_to(-e);
    i32x8 r;
    for (int h = 0; h < 2; h++)
        for (int i = 0; i < 4; i++)
            r[4 * h + i] = (int)e4m3_pack(x[h][4 * i], x[h][4 * i + 1], x[h][4 * i + 2], x[h][4 * i + 3], down);
    return r;
}

// The rows' fragments and, for each four blocks of inputs, the powers of two of 16 rows' blocks, a byte each.
template <typename T>
__global__ __launch_bounds__(256) void round_rows_kernel(const T *a, size_t lda, size_t m, size_t k, bool aligned, Rounded to) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t tiles = to.tiles;
    // A wavefront takes four blocks of 16 rows: one word of powers for each row.
    for (size_t u = (size_t)blockIdx.x * 4 + wave; u < tiles * to.quads; u += (size_t)gridDim.x * 4) {
        const size_t tile = u / to.quads, quad = u % to.quads, row = tile * 16 + (lane & 15);
        uint32_t powers = 0;
        for (int q = 0; q < 4; q++) {
            const size_t b = quad * 4 + q;
            if (b >= to.blocks) break;
            int e;
            const i32x8 r = round_rows(a, lda, row, row < m, b, k, aligned, lane >> 4, e);
            i32x4 *out = reinterpret_cast<i32x4 *>(to.values + (tile * to.blocks + b) * 2048 + lane * 16);
            out[0] = __builtin_shufflevector(r, r, 0, 1, 2, 3);
            out[64] = __builtin_shufflevector(r, r, 4, 5, 6, 7);
            powers |= (uint32_t)(e + 127) << 8 * q;
        }
        if (lane < 16) to.powers[(quad * tiles + tile) * 16 + lane] = powers;
    }
}

// Checkpoint weights (rows of k bytes, ld apart) into fragments; zeros past the last output and input.
__global__ __launch_bounds__(256) void weights_kernel(const uint8_t *src, size_t ld, size_t n, size_t k, size_t blocks,
                                                      size_t pieces, uint8_t *out) {
    for (size_t p = (size_t)blockIdx.x * 256 + threadIdx.x; p < pieces; p += (size_t)gridDim.x * 256) {
        const size_t lane = p % 64, half = p / 64 % 2, b = p / 128 % blocks, panel = p / 128 / blocks;
        const size_t o = panel * 16 + lane % 16, k0 = b * 128 + half * 64 + lane / 16 * 16;
        uint32_t w[4] = {};
        for (int e = 0; e < 16; e++)
            if (o < n && k0 + e < k) w[e / 4] |= (uint32_t)src[o * ld + k0 + e] << 8 * (e % 4);
        reinterpret_cast<u32x4 *>(out)[p] = u32x4{w[0], w[1], w[2], w[3]};
    }
}

// ------------------------------------------------------------------------------------------- outputs

// Four outputs of a row, from column n on, through the epilogue.
__device__ __forceinline__ void store4(const E4m3Out &o, size_t row, size_t n, f32x4 v) {
    float old[4] = {};
    const size_t at = row * o.ld + n;
    const int count = o.n - n < 4 ? (int)(o.n - n) : 4;
    const bool whole = count == 4 && o.aligned;
    const auto type = [&](auto t) {
        using U = decltype(t);
        typedef U u4 __attribute__((ext_vector_type(4)));
        U *c = static_cast<U *>(o.c) + at;
        if (o.epi.accumulate) {
            if (whole) {
                const u4 x = *reinterpret_cast<const u4 *>(c);
                for (int e = 0; e < 4; e++) old[e] = (float)x[e];
            } else {
                for (int e = 0; e < count; e++) old[e] = (float)c[e];
            }
        }
        u4 y;
        for (int e = 0; e < 4; e++)
            y[e] = (U)epilogue_vals(v[e], o.epi.bias != nullptr, o.epi.bias && e < count ? o.epi.bias[n + e] : 0.0f, o.epi.act,
                                    o.epi.scale, o.epi.accumulate, old[e]);
        if (whole) {
            *reinterpret_cast<u4 *>(c) = y;
        } else {
            for (int e = 0; e < count; e++) c[e] = y[e];
        }
    };
    if (o.type == F32) type(float{});
    else if (o.type == F16) type(_Float16{});
    else type(__bf16{});
}

// ------------------------------------------------------------------------------------- few rows

// MT x 16 rows by PN x 16 outputs of a workgroup, the blocks of inputs spread over its wavefronts, whose sums LDS joins in
// their order. FUSED: 16 rows at most, rounded as they are read; otherwise from their fragments.
constexpr int FEW_WAVES = 8;
template <typename T, int MT, int PN, bool FUSED>
__global__ __launch_bounds__(64 * FEW_WAVES) void few_kernel(const T *a, size_t lda, size_t k, bool aligned, Rounded in,
                                                             E4m3Panels w, E4m3Out o) {
    constexpr int SLOTS = MT * PN >= 8 ? 4 : 8;  // wavefronts' sums in LDS at a time
    __shared__ f32x4 sums[SLOTS][MT * PN][64];
    const int lane = threadIdx.x & 63, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int panel0 = blockIdx.x * PN, tile0 = blockIdx.y * MT;
    const int blocks = (int)w.blocks;
    f32x4 acc[MT][PN] = {};
    const int per = (blocks + FEW_WAVES - 1) / FEW_WAVES;
    const int b0 = wave * per, b1 = b0 + per < blocks ? b0 + per : blocks;
    const uint8_t *wp[PN];
    for (int p = 0; p < PN; p++) wp[p] = w.values + (size_t)min(panel0 + p, (int)w.panels - 1) * blocks * 2048 + lane * 16;
    const float *scale = w.scales + (size_t)(panel0 / 8) * blocks;
    for (int b = b0; b < b1; b++) {
        i32x8 wf[PN];
#pragma unroll
        for (int p = 0; p < PN; p++) {
            const i32x4 *at = reinterpret_cast<const i32x4 *>(wp[p] + (size_t)b * 2048);
            wf[p] = joined(at[0], at[64]);
        }
        const auto panel = [&](int p) { return Operand<true>(wf[p], 1.0f); };
        const float s = scale[b];
#pragma unroll
        for (int t = 0; t < MT; t++) {
            i32x8 af;
            float up;
            if constexpr (FUSED) {
                const size_t row = lane & 15;
                int e;
                af = round_rows(a, lda, row, row < o.m, b, k, aligned, quarter, e);
                up = two_to(e);
            } else {
                const size_t tile = min(tile0 + t, (int)in.tiles - 1);
                const i32x4 *at = reinterpret_cast<const i32x4 *>(in.values + (tile * blocks + b) * 2048 + lane * 16);
                af = joined(at[0], at[64]);
                up = power_of(in.powers[((size_t)(b / 4) * in.tiles + tile) * 16 + (lane & 15)], b % 4);
            }
            const Operand<true> rows(af, up);
#pragma unroll
            for (int p = 0; p < PN; p++) {
                const f32x4 part = block_product<0>(panel(p), rows, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[t][p][e] = __builtin_fmaf(part[e], s, acc[t][p][e]);
            }
        }
    }
    const auto put = [&](int slot) {
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int p = 0; p < PN; p++) sums[slot][t * PN + p][lane] = acc[t][p];
    };
    if (SLOTS == FEW_WAVES) {
        put(wave);
    } else {
        if (wave >= SLOTS) put(wave - SLOTS);
        __syncthreads();
        if (wave < SLOTS) {
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int p = 0; p < PN; p++) acc[t][p] += sums[wave][t * PN + p][lane];
            put(wave);
        }
    }
    __syncthreads();
    for (int y = threadIdx.x; y < MT * PN * 64; y += 64 * FEW_WAVES) {
        const int l = y % 64, t = y / 64 / PN, p = y / 64 % PN;
        const size_t row = (size_t)(tile0 + t) * 16 + (l & 15), n = (size_t)(panel0 + p) * 16 + (l >> 4) * 4;
        if (row >= o.m || n >= o.n) continue;
        f32x4 v = sums[0][t * PN + p][l];
        for (int s = 1; s < SLOTS; s++) v += sums[s][t * PN + p][l];
        store4(o, row, n, v);
    }
}

// ------------------------------------------------------------------------------------- many rows

__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}
// 64 lanes x 16 bytes from base + voff to LDS at lds. M0 holds the LDS address; a copy reads it without an interlock and
// needs one wait state after the write.
__device__ __forceinline__ void copy_to_lds(const uint8_t *base, uint32_t voff, uint32_t lds) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(voff), "s"(base) : "memory", "m0");
#pragma clang diagnostic pop
}
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Workgroups of WM x WN wavefronts of TM x TN tiles each. Two stages of a block of inputs in LDS: while one is worked on,
// the next is copied to the other.
template <int WM, int WN, int TM, int TN, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN, 2) void tile_kernel(Rounded in, E4m3Panels w, E4m3Out o, int m_tiles, int n_tiles) {
    constexpr int WAVES = WM * WN, RT = WM * TM, PT = WN * TN;  // row tiles and panels of the workgroup
    constexpr int CHUNKS = 2 * (RT + PT), STAGE = CHUNKS * 1024;
    static_assert(CHUNKS % WAVES == 0 && RT <= 16 && 8 % TN == 0, "");
    constexpr int CPW = CHUNKS / WAVES;
    __shared__ __align__(16) uint8_t smem[2 * STAGE + 2 * 1024];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM;
    // Neighbours in a grid of tiles, eight tile rows at a time, share an XCD's L2.
    int id = blockIdx.x;
    {
        const int total = m_tiles * n_tiles, each = total / 8, more = total % 8, xcd = id % 8, at = id / 8;
        id = xcd * each + min(xcd, more) + at;
    }
    const int band = id / (8 * n_tiles), in_band = id - band * 8 * n_tiles, high = min(8, m_tiles - band * 8);
    const int mt = band * 8 + in_band % high, nt = in_band / high;
    const int tile0 = mt * RT, panel0 = nt * PT;
    const int blocks = (int)w.blocks;

    const uint8_t *from[CPW];
#pragma unroll
    for (int c = 0; c < CPW; c++) {
        const int ch = wave + c * WAVES, x = ch / 2;
        from[c] = x < RT ? in.values + (size_t)min(tile0 + x, (int)in.tiles - 1) * blocks * 2048 + ch % 2 * 1024
                         : w.values + (size_t)min(panel0 + x - RT, (int)w.panels - 1) * blocks * 2048 + ch % 2 * 1024;
    }
    const uint32_t voff = lane * 16, lds0 = __builtin_amdgcn_readfirstlane(lds_address(smem));
    const auto issue = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < CPW; c++)
            copy_to_lds(from[c] + (size_t)b * 2048, voff, lds0 + (b & 1) * STAGE + (wave + c * WAVES) * 1024);
        if (b % 4 == 0 && wave == 0)  // 16 row tiles' powers of four blocks; what lies behind the last tile's is not used
            copy_to_lds(reinterpret_cast<const uint8_t *>(in.powers + ((size_t)(b / 4) * in.tiles + tile0) * 16), voff,
                        lds0 + 2 * STAGE + (b / 4 & 1) * 1024);
    };
    const float *scale = w.scales + (size_t)((panel0 + wn * TN) / 8) * blocks;

    f32x4 acc[TM][TN] = {};
    uint32_t powers[TM];
    const auto work = [&](auto q, int b) __attribute__((always_inline)) {
        const uint8_t *st = smem + (b & 1) * STAGE + lane * 16;
        const auto fragment = [&](int x) {
            return joined(*reinterpret_cast<const i32x4 *>(st + x * 2048), *reinterpret_cast<const i32x4 *>(st + x * 2048 + 1024));
        };
        if constexpr (q.value == 0)
#pragma unroll
            for (int t = 0; t < TM; t++)
                powers[t] = *reinterpret_cast<const uint32_t *>(smem + 2 * STAGE + (b / 4 & 1) * 1024 + ((wm * TM + t) * 16 + (lane & 15)) * 4);
        const float s = scale[b];
        const auto panel = [&](int p) { return Operand<EXACT>(fragment(RT + wn * TN + p), 1.0f); };
        static_assert(TN == 4, "");
        const Operand<EXACT> wf[TN] = {panel(0), panel(1), panel(2), panel(3)};
#pragma unroll
        for (int t = 0; t < TM; t++) {
            const Operand<EXACT> af(fragment(wm * TM + t), EXACT ? power_of(powers[t], q.value) : 1.0f);
            f32x4 part[TN];
#pragma unroll
            for (int p = 0; p < TN; p++) part[p] = block_product<q.value>(wf[p], af, powers[t]);
#pragma unroll
            for (int p = 0; p < TN; p++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[t][p][e] = __builtin_fmaf(part[p][e], s, acc[t][p][e]);
        }
    };
    issue(0);
    wait_copies();
    const auto step = [&](auto q, int b) __attribute__((always_inline)) {
        if (b >= blocks) return;
        __syncthreads();  // stage b is there, and the one before it has been read
        if (b + 1 < blocks) issue(b + 1);
        work(q, b);
        wait_copies();
    };
    for (int b = 0; b < blocks; b += 4) {
        step(std::integral_constant<int, 0>{}, b);
        step(std::integral_constant<int, 1>{}, b + 1);
        step(std::integral_constant<int, 2>{}, b + 2);
        step(std::integral_constant<int, 3>{}, b + 3);
    }
    // Two tiles' rows at a time go through the wavefront's own part of LDS, so that a row's outputs leave side by side.
    constexpr int PITCH = TN * 16 + 4;
    static_assert(WAVES * 32 * PITCH * 4 <= 2 * STAGE && TM % 2 == 0, "");
    __syncthreads();
    float *mine = reinterpret_cast<float *>(smem) + wave * 32 * PITCH;
#pragma unroll
    for (int t = 0; t < TM; t += 2) {
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int p = 0; p < TN; p++)
                *reinterpret_cast<f32x4 *>(mine + (x * 16 + (lane & 15)) * PITCH + p * 16 + (lane >> 4) * 4) = acc[t + x][p];
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int y = lane; y < 32 * TN * 4; y += 64) {
            const int r = y / (TN * 4), c = y % (TN * 4) * 4;
            const size_t row = (size_t)(tile0 + wm * TM + t) * 16 + r, n = (size_t)(panel0 + wn * TN) * 16 + c;
            if (row < o.m && n < o.n) store4(o, row, n, *reinterpret_cast<const f32x4 *>(mine + r * PITCH + c));
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <int WM, int WN, int TM, int TN, bool EXACT>
hipError_t launch_tiles(const Rounded &in, const E4m3Panels &w, const E4m3Out &o, hipStream_t s) {
    const size_t m_tiles = div_ceil(in.tiles, WM * TM), n_tiles = div_ceil(w.panels, WN * TN);
    if (m_tiles * n_tiles > INT32_MAX / 1024) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((tile_kernel<WM, WN, TM, TN, EXACT>), dim3((unsigned)(m_tiles * n_tiles)), dim3(64 * WM * WN), 0, s, in, w, o,
                       (int)m_tiles, (int)n_tiles);
    return hipGetLastError();
}

template <typename T, int MT, int PN, bool FUSED>
hipError_t launch_few(const T *a, size_t lda, size_t k, bool aligned, const Rounded &in, const E4m3Panels &w, const E4m3Out &o,
                      hipStream_t s) {
    const dim3 grid((unsigned)div_ceil(w.panels, PN), (unsigned)div_ceil(div_ceil(o.m, 16), MT));
    hipLaunchKernelGGL((few_kernel<T, MT, PN, FUSED>), grid, dim3(64 * FEW_WAVES), 0, s, a, lda, k, aligned, in, w, o);
    return hipGetLastError();
}

template <typename T>
hipError_t product(const T *a, size_t lda, size_t k, const E4m3Panels &w, const E4m3Out &o, const Rounded &in, hipStream_t s) {
    const bool aligned = reinterpret_cast<uintptr_t>(a) % 16 == 0 && lda * sizeof(T) % 16 == 0;
    if (!k) return launch_few<float, 4, 4, false>(nullptr, 0, k, aligned, in, w, o, s);  // the epilogue of empty sums
    if (o.m <= E4M3_FEW) {
        if (w.panels >= 1024) return launch_few<T, 1, 4, true>(a, lda, k, aligned, in, w, o, s);
        return launch_few<T, 1, 1, true>(a, lda, k, aligned, in, w, o, s);
    }
    const size_t units = in.tiles * in.quads, blocks = div_ceil(units, 4);
    hipLaunchKernelGGL((round_rows_kernel<T>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, s, a, lda, o.m,
                       k, aligned, in);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const size_t large = div_ceil(in.tiles, 16) * div_ceil(w.panels, 16), middle = div_ceil(in.tiles, 8) * div_ceil(w.panels, 8);
    if (large >= 256 && o.type != F32) return launch_tiles<2, 4, 8, 4, false>(in, w, o, s);
    if (middle >= 128 && o.type != F32) return launch_tiles<2, 2, 4, 4, false>(in, w, o, s);
    if (middle >= 128) return launch_tiles<2, 2, 4, 4, true>(in, w, o, s);
    return launch_few<float, 4, 4, false>(nullptr, 0, k, aligned, in, w, o, s);
}

}  // namespace

hipError_t launch_e4m3_weights(const uint8_t *src, size_t ld, size_t n, size_t k, uint8_t *out, hipStream_t s) {
    const size_t blocks = div_ceil(k, 128), pieces = div_ceil(n, 16) * blocks * 128, groups = div_ceil(pieces, 256);
    hipLaunchKernelGGL(weights_kernel, dim3((unsigned)(groups < 65536 ? groups : 65536)), dim3(256), 0, s, src, ld, n, k, blocks,
                       pieces, out);
    return hipGetLastError();
}

hipError_t launch_e4m3_product(uint32_t type, const void *a, size_t lda, size_t k, const E4m3Panels &w, const E4m3Out &o,
                               void *work, hipStream_t s) {
    const Rounded in = rounded_at(work, o.m, k);
    switch (type) {
        case F16: return product(static_cast<const _Float16 *>(a), lda, k, w, o, in, s);
        case BF16: return product(static_cast<const __bf16 *>(a), lda, k, w, o, in, s);
        default: return product(static_cast<const float *>(a), lda, k, w, o, in, s);
    }
}

}  // namespace tg
