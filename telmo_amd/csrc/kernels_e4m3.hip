// The product of rows and weights in eight bits: c = epi(a' w'^T), w' of e4m3 values with an f32 scale for each block of
// 128 outputs by 128 inputs, a' the rows rounded to e4m3 in groups of 128 inputs with a power of two each (e4m3.hpp):
//
//   c_ij = sum over blocks b of S[j / 128][b] sum over k in b of 2^e_ib a8_ik w8_jk
//
// S is one number for all of a wavefront's outputs. Its power of two is multiplied into the weights, which rounds nothing, so
// that no sum overflows that would not with the weights as they stand (8192^3 523 us; 515 with all of S applied afterwards);
// what is left of it, from 1 to 2, goes into the multiply-add per output that adds a block to its f32 sum. The inner sum is
// made in one of two ways:
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
#include <type_traits>

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
// Read-only memory that is read by scalar loads.
typedef const __attribute__((address_space(4))) float *Scalar;

// Product i of 16 outputs by 16 rows of a block of inputs (EXACT: of four), added to `sum`; powers of two, where they are not
// in w and a yet, as e + 127, the rows' each in its lanes.
__device__ __forceinline__ f32x4 block_product(const Operand<false> &w, const Operand<false> &a, uint32_t w_power, uint32_t power, int,
                                               f32x4 sum) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, a.v, sum, 0, 0, 0, (int)w_power, 0, (int)power);
}
__device__ __forceinline__ f32x4 block_product(const Operand<true> &w, const Operand<true> &a, uint32_t, uint32_t, int i, f32x4 sum) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], a.v[i], sum, 0, 0, 0);
}
// e + 127 as 2^e.
__device__ __forceinline__ float power_of(uint32_t power) { return __uint_as_float(power << 23); }
// A block's scale as 2^g, which the weights take (g + 127), and the rest. g stays where bf16 holds 448 2^g and 2^-9 2^g as
// normal numbers: a scale past that leaves more than 1 to 2, in products that are then far from f32's ends.
struct BlockScale {
    uint32_t power;
    float rest;
    __device__ __forceinline__ explicit BlockScale(float s) {
        power = min(max(__float_as_uint(s) >> 23 & 255u, 27u), 227u);
        rest = s * power_of(254u - power);
    }
};
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

// The lane's part of a fragment of the rows: 32 inputs of a row, rounded under the exponent of the row's group, which the
// four lanes of a row find together.
__device__ __forceinline__ i32x8 rounded(const float (&x)[2][16], int &e) {
    uint32_t top = 0;
    for (int h = 0; h < 2; h++)
        for (int i = 0; i < 16; i++) top = max(top, __float_as_uint(x[h][i]) & 0x7fffffffu);
    // Below 2^127 no value needs a bound, or a look at whether it is finite: three operations for each instead of nine.
    const bool plain = !__any(top >= 0x7f000000u);
    if (!plain) {
        top = 0;
        for (int h = 0; h < 2; h++)
            for (int i = 0; i < 16; i++) top = max(top, e4m3_size(x[h][i]));
    }
    e = e4m3_exponent(__float_as_uint(max_of_quarters(__uint_as_float(top))));
    const float down = two_to(-e);
    i32x8 r;
    for (int h = 0; h < 2; h++)
        for (int i = 0; i < 4; i++) {
            const float *y = x[h] + 4 * i;
            if (plain) {
                const int two = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * down, y[1] * down, 0, false);
                r[4 * h + i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * down, y[3] * down, two, true);
            } else {
                r[4 * h + i] = (int)e4m3_pack(y[0], y[1], y[2], y[3], down);
            }
        }
    return r;
}
// Of row `row` (zeros where there is none) from input 128 b on.
template <typename T>
__device__ __forceinline__ i32x8 round_rows(const T *a, size_t lda, size_t row, bool real, size_t b, size_t k, bool aligned,
                                            int quarter, int &e) {
    float x[2][16] = {};
    if (real)
        for (int h = 0; h < 2; h++) load16(a + row * lda, b * 128 + h * 64 + quarter * 16, k, aligned, x[h]);
    return rounded(x, e);
}
// The lane's inputs as they lie in memory: a block's can be on their way while the one before is worked on.
template <typename T>
struct Inputs {
    static constexpr int PIECE = 16 / sizeof(T);
    u32x4 v[2][16 / PIECE];
    __device__ __forceinline__ void load(const T *at) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 16 / PIECE; i++) v[h][i] = *reinterpret_cast<const u32x4 *>(at + h * 64 + i * PIECE);
    }
    __device__ __forceinline__ i32x8 round(int &e) const {
        float x[2][16];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                struct Piece {
                    T v[PIECE];
                };
                x[h][i] = (float)__builtin_bit_cast(Piece, v[h][i / PIECE]).v[i % PIECE];
            }
        return rounded(x, e);
    }
};

// The rows' fragments and powers of two, a wavefront for 16 rows of a block of inputs at a time.
template <typename T>
__global__ __launch_bounds__(256) void round_rows_kernel(const T *a, size_t lda, size_t m, size_t k, bool aligned, Rounded to) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (size_t u = (size_t)blockIdx.x * 4 + wave; u < to.tiles * to.blocks; u += (size_t)gridDim.x * 4) {
        const size_t tile = u / to.blocks, b = u % to.blocks, row = tile * 16 + (lane & 15);
        int e;
        const i32x8 r = round_rows(a, lda, row, row < m, b, k, aligned, lane >> 4, e);
        i32x4 *out = reinterpret_cast<i32x4 *>(to.values + u * 2048 + lane * 16);
        out[0] = __builtin_shufflevector(r, r, 0, 1, 2, 3);
        out[64] = __builtin_shufflevector(r, r, 4, 5, 6, 7);
        if (lane < 16) reinterpret_cast<uint8_t *>(to.powers + (b / 4 * to.tiles + tile) * 16 + lane)[b % 4] = (uint8_t)(e + 127);
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

// v / (1 + e^-v) to 2^-21 of itself from -87 on, where e^-v has a reciprocal that f32 holds as a normal number; 0 below, where
// it is less than 2^-119. The exponent's product with log2 e in two parts, of v cut where e^-v is nothing beside 1, the
// hardware's 2^x and reciprocal: the row kernels' SiLU, with their polynomial and division, takes 40 operations an output, as
// long as a product of 400 inputs.
__device__ __forceinline__ float silu(float v) {
    constexpr float L = 1.44269504088896340736f, REST = 1.92596299112661746887e-8f;  // log2 e = L + REST
    constexpr float LEAST = -87.0f;
    const float x = __builtin_amdgcn_fmed3f(v, LEAST, 128.0f);
    const float t = -L * x, low = __builtin_fmaf(-REST, x, __builtin_fmaf(-L, x, -t));
    const float e = __builtin_amdgcn_exp2f(t) * __builtin_fmaf(low, 0.69314718055994530942f, 1.0f);
    const float y = v * __builtin_amdgcn_rcpf(1.0f + e);  // for all: branches took longer (750 x 1024 -> 4096 0.5 us of 20)
    return v < LEAST ? -0.0f : y;
}
// The epilogue of a lane's rows of four outputs, from column n on. The bias is loaded and waited for once, and what the call
// says is held in scalar registers: waiting for a load of each row's own would wait for the store of the row before.
struct Outputs {
    const E4m3Out &o;
    size_t n;
    int count;  // outputs of the four that there are
    uint32_t type, act, accumulate;
    float scale;
    f32x4 bias;
    bool whole;  // every lane has four outputs or none, which lie aligned, and takes no old ones
    __device__ __forceinline__ Outputs(const E4m3Out &o_, size_t n_) : o(o_), n(n_) {
        count = n >= o.n ? 0 : o.n - n < 4 ? (int)(o.n - n) : 4;
        type = __builtin_amdgcn_readfirstlane(o.type);
        act = __builtin_amdgcn_readfirstlane(o.epi.act);
        accumulate = __builtin_amdgcn_readfirstlane(o.epi.accumulate);
        scale = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(o.epi.scale)));
        whole = o.aligned && o.n % 4 == 0 && !accumulate;
        bias = f32x4{};
        if (o.epi.bias)
            for (int e = 0; e < 4; e++) bias[e] = e < count ? o.epi.bias[n + e] : 0.0f;
        asm volatile("s_waitcnt vmcnt(0)" : "+v"(bias));
    }
    __device__ __forceinline__ f32x4 finished(f32x4 v) const {
        if (o.epi.bias) v += bias;
        if (act == ACT_RELU) {
            for (int e = 0; e < 4; e++) v[e] = v[e] > 0.0f ? v[e] : 0.0f;
        } else if (act == ACT_SILU) {
            for (int e = 0; e < 4; e++) v[e] = silu(v[e]);
        }
        return v * scale;
    }
    // f(row in type U) as the outputs' type wants it.
    template <typename F>
    __device__ __forceinline__ void typed(F f) const {
        if (type == F32) f(float{});
        else if (type == F16) f(_Float16{});
        else f(__bf16{});
    }
    // A row where `whole` holds.
    template <typename U>
    __device__ __forceinline__ void store_whole(size_t row, f32x4 v) const {
        typedef U u4 __attribute__((ext_vector_type(4)));
        v = finished(v);
        u4 y;
        for (int e = 0; e < 4; e++) y[e] = (U)v[e];
        if (row < o.m && count) *reinterpret_cast<u4 *>(static_cast<U *>(o.c) + row * o.ld + n) = y;
    }
    // Any row.
    __device__ __forceinline__ void store(size_t row, f32x4 v) const {
        if (row >= o.m) return;
        v = finished(v);
        typed([&](auto u) {
            using U = decltype(u);
            U *c = static_cast<U *>(o.c) + row * o.ld + n;
            for (int e = 0; e < count; e++) c[e] = (U)(accumulate ? (float)c[e] + v[e] : v[e]);
        });
    }
};

// ------------------------------------------------------------------------------------- few rows

// MT x 16 rows by PN x 16 outputs of a workgroup, the blocks of inputs spread over its wavefronts, whose sums LDS joins in
// their order. 16 rows at most are rounded as they are read, more come from their fragments.
//
// Bound by the weights' bytes: 16 rows of bf16 by 4096 x 16384 (68 MB) 16.8 us, 4.0 TB/s (a large copy 4.85). The rows' rounding
// is what a wavefront works longest on: with nine operations a value instead of three it took 19.5, and where each block
// waited for its rows 20.8. One row by 640 x 2560 takes the time of a call.
constexpr int FEW_WAVES = 8;
enum Source { FRAGMENTS, WHOLE, ANY };  // rows rounded before; rounded here, in whole aligned blocks of inputs, or not
template <typename T, int MT, int PN, Source FROM>
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
    const Scalar scale = (Scalar)(w.scales + e4m3_scale_row(panel0, w.panels) * blocks);
    // The next block's weights and rows are on their way while a block is multiplied (rows past the last are read as it).
    struct Block {
        i32x8 w[PN], rows[MT];
        uint32_t power[MT];
        float scale;
        Inputs<T> inputs;
    } now, next;
    const size_t row = lane & 15;
    const T *own = FROM == WHOLE ? a + (row < o.m ? row : o.m - 1) * lda + quarter * 16 : nullptr;
    const auto load = [&](int b) __attribute__((always_inline)) {
        if constexpr (FROM == WHOLE) next.inputs.load(own + (size_t)b * 128);
        if constexpr (FROM == FRAGMENTS)
#pragma unroll
            for (int t = 0; t < MT; t++) {
                const size_t tile = min(tile0 + t, (int)in.tiles - 1);
                const i32x4 *at = reinterpret_cast<const i32x4 *>(in.values + (tile * blocks + b) * 2048 + lane * 16);
                next.rows[t] = joined(at[0], at[64]);
                next.power[t] = reinterpret_cast<const uint8_t *>(in.powers + ((size_t)(b / 4) * in.tiles + tile) * 16 + row)[b % 4];
            }
#pragma unroll
        for (int p = 0; p < PN; p++) {
            const i32x4 *at = reinterpret_cast<const i32x4 *>(wp[p] + (size_t)b * 2048);
            next.w[p] = joined(at[0], at[64]);
        }
        next.scale = scale[b];
    };
    if (b0 < b1) load(b0);
    for (int b = b0; b < b1; b++) {
        now = next;
        load(b + 1 < b1 ? b + 1 : b);
        const BlockScale s(now.scale);
        const float w_up = power_of(s.power);
#pragma unroll
        for (int t = 0; t < MT; t++) {
            i32x8 af;
            float up;
            if constexpr (FROM == FRAGMENTS) {
                af = now.rows[t];
                up = power_of(now.power[t]);
            } else {
                int e;
                if constexpr (FROM == WHOLE) af = now.inputs.round(e);
                else af = round_rows(a, lda, row, row < o.m, b, k, aligned, quarter, e);
                up = two_to(e);
            }
            const Operand<true> rows(af, up);
#pragma unroll
            for (int p = 0; p < PN; p++) {
                const Operand<true> outs(now.w[p], w_up);
                f32x4 part = {};
#pragma unroll
                for (int i = 0; i < 4; i++) part = block_product(outs, rows, 0, 0, i, part);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[t][p][e] = __builtin_fmaf(part[e], s.rest, acc[t][p][e]);
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
        f32x4 v = sums[0][t * PN + p][l];
        for (int s = 1; s < SLOTS; s++) v += sums[s][t * PN + p][l];
        Outputs(o, (size_t)(panel0 + p) * 16 + (l >> 4) * 4).store((size_t)(tile0 + t) * 16 + (l & 15), v);
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
// The same of 64 lanes x 4 bytes.
__device__ __forceinline__ void copy_words_to_lds(const uint8_t *base, uint32_t voff, uint32_t lds) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(voff), "s"(base) : "memory", "m0");
#pragma clang diagnostic pop
}
// Until at most N of the wavefront's copies are on their way.
template <int N>
__device__ __forceinline__ void wait_copies() {
    static_assert(N < 64, "vmcnt holds 6 bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Workgroups of KG groups of WM x WN wavefronts of TM x TN tiles each. The groups share the outputs and take every KG-th
// block of inputs, and add up their sums in LDS. LDS holds two stages of a block for each group: while one is worked on, the
// next is copied to the other.
//
// 8192 x 8192 x 8192 into bf16 takes 40 us to round the rows (at the rate of a copy) and 480 by tiles of 256 x 256, 2290 TFLOP/s:
// a block of inputs is 2112 cycles of a CU's matrix instructions, and 192 KB that its wavefronts read from LDS and 64 KB that
// are copied there are 2048 of LDS, which the two share badly. 750 rows by 1024 x 4096 into f32, EXACT, take 20 us: 192 tiles
// for 256 CUs, eight blocks of inputs each, between a start and an end that nothing overlaps.
template <int WM, int WN, int TM, int TN, int KG, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN * KG, 2) void tile_kernel(Rounded in, E4m3Panels w, E4m3Out o, int m_tiles, int n_tiles) {
    constexpr int WAVES = WM * WN, RT = WM * TM, PT = WN * TN;     // wavefronts, row tiles and panels of a group
    constexpr int CHUNKS = 2 * (RT + PT), STAGE = (CHUNKS + 1) * 1024;  // fragments, and 16 row tiles' powers
    static_assert(CHUNKS % WAVES == 0 && RT <= 16 && 8 % TN == 0 && WAVES >= 4 && TM % KG == 0, "");
    constexpr int CPW = CHUNKS / WAVES;
    __shared__ __align__(16) uint8_t smem[2 * KG * STAGE];
    const int lane = threadIdx.x & 63, all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = all_waves / WAVES, wave = all_waves % WAVES, wm = wave % WM, wn = wave / WM;
    // Neighbours in a grid of tiles, eight tile rows at a time, share an XCD's L2.
    int id = blockIdx.x;
    {
        const int total = m_tiles * n_tiles, each = total / 8, more = total % 8, xcd = id % 8, at = id / 8;
        id = xcd * each + min(xcd, more) + at;
    }
    const int band = id / (8 * n_tiles), in_band = id - band * 8 * n_tiles, high = min(8, m_tiles - band * 8);
    const int mt = band * 8 + in_band % high, nt = in_band / high;
    const int tile0 = mt * RT, panel0 = nt * PT;
    const int blocks = (int)w.blocks, steps = (blocks + KG - 1) / KG;

    const uint8_t *from[CPW];
#pragma unroll
    for (int c = 0; c < CPW; c++) {
        const int ch = wave + c * WAVES, x = ch / 2;
        from[c] = x < RT ? in.values + (size_t)min(tile0 + x, (int)in.tiles - 1) * blocks * 2048 + ch % 2 * 1024
                         : w.values + (size_t)min(panel0 + x - RT, (int)w.panels - 1) * blocks * 2048 + ch % 2 * 1024;
    }
    uint8_t *const mine = smem + group * STAGE;
    const uint32_t voff = lane * 16, lds0 = __builtin_amdgcn_readfirstlane(lds_address(mine));
    // The group's block of a step (past the last block that one again) to a stage, with the powers of its quad of blocks: of
    // 16 row tiles, a quarter by each of four wavefronts; what lies behind the last tile's is not used. All wavefronts copy
    // alike, without a branch, which would leave the compiler to move the products out of their place.
    const auto issue = [&](int step, int stage) __attribute__((always_inline)) {
        const int b = min(step * KG + group, blocks - 1);
#pragma unroll
        for (int c = 0; c < CPW; c++)
            copy_to_lds(from[c] + (size_t)b * 2048, voff, lds0 + stage * KG * STAGE + (wave + c * WAVES) * 1024);
        copy_words_to_lds(reinterpret_cast<const uint8_t *>(in.powers + ((size_t)(b / 4) * in.tiles + tile0) * 16) + wave % 4 * 256,
                          lane * 4, lds0 + stage * KG * STAGE + CHUNKS * 1024 + wave % 4 * 256);
    };
    // A scalar load: one in a vector register would wait for the copies that left before it. A step's is loaded in the one before.
    const Scalar scale = (Scalar)(w.scales + e4m3_scale_row(panel0 + wn * TN, w.panels) * blocks);

    f32x4 acc[TM][TN] = {};
    const auto scale_of = [&](int step) { return scale[min(step * KG + group, blocks - 1)]; };
    const auto work = [&](int b, int stage, float scale_now) __attribute__((always_inline)) {
        const uint8_t *st = mine + stage * KG * STAGE + lane * 16;
        const auto fragment = [&](int x) {
            return joined(*reinterpret_cast<const i32x4 *>(st + x * 2048), *reinterpret_cast<const i32x4 *>(st + x * 2048 + 1024));
        };
        uint32_t powers[TM];
#pragma unroll
        for (int t = 0; t < TM; t++)
            powers[t] = mine[stage * KG * STAGE + CHUNKS * 1024 + ((wm * TM + t) * 16 + (lane & 15)) * 4 + (b & 3)];
        const BlockScale s(scale_now);
        const float w_up = power_of(s.power);
        const auto panel = [&](int p) { return Operand<EXACT>(fragment(RT + wn * TN + p), w_up); };
        static_assert(TN == 4, "");
        const Operand<EXACT> wf[TN] = {panel(0), panel(1), panel(2), panel(3)};
        // While a row tile is multiplied the next one's fragment is read (EXACT: widened, and the one after it read), and the
        // one before it added up.
        const auto rows = [&](const i32x8 &bytes, int t) { return Operand<EXACT>(bytes, EXACT ? power_of(powers[t]) : 1.0f); };
        constexpr int STEPS = EXACT ? 4 : 1;  // products of a block
        f32x4 part[2][TN];
        i32x8 bytes = fragment(wm * TM);
        Operand<EXACT> af = rows(bytes, 0);
        if (EXACT && TM > 1) bytes = fragment(wm * TM + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t <= TM; t++) {
            const int now = t < TM ? t : 0;
            const Operand<EXACT> multiplied = af;
            if (EXACT ? t + 2 < TM : t + 1 < TM) {
                const i32x8 next = fragment(wm * TM + t + (EXACT ? 2 : 1));
                if (EXACT) af = rows(bytes, t + 1);
                bytes = next;
                if (!EXACT) af = rows(bytes, t + 1);
            } else if (EXACT && t + 1 < TM) {
                af = rows(bytes, t + 1);
            }
#pragma unroll
            for (int i = 0; i < STEPS; i++)
#pragma unroll
                for (int p = 0; p < TN; p++) {
                    if (t < TM) part[t & 1][p] = block_product(wf[p], multiplied, s.power, powers[now], i, i ? part[t & 1][p] : f32x4{});
                    if (t > 0)
#pragma unroll
                        for (int e = 4 / STEPS * i; e < 4 / STEPS * (i + 1); e++)
                            acc[t - 1][p][e] = __builtin_fmaf(part[(t - 1) & 1][p][e], s.rest, acc[t - 1][p][e]);
                }
        }
#pragma unroll
        for (int t = 0; t < TM; t++) {
            if (t + (EXACT ? 2 : 1) < TM) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
            for (int p = 0; p < TN * STEPS; p++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (EXACT && t + 1 < TM) __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
                if (t > 0) __builtin_amdgcn_sched_group_barrier(0x002, 4 / STEPS, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    issue(0, 0);
    float scale_next = scale_of(0);
    wait_copies<0>();
    const auto step = [&](int i, int stage) __attribute__((always_inline)) {
        __syncthreads();  // the step's blocks are there, and the ones before them have been read
        issue(i + 1, stage ^ 1);
        const float scale_now = scale_next;
        scale_next = scale_of(i + 1);
        work(i * KG + group, stage, scale_now);
        wait_copies<0>();
    };
    const int whole = blocks / KG;  // steps in which every group has a block
    int i = 0;
    for (; i + 2 <= whole; i += 2) {
        step(i, 0);
        step(i + 1, 1);
    }
    if (i < whole) step(i++, 0);
    if (i < steps) {
        __syncthreads();
        if (i * KG + group < blocks) work(i * KG + group, i & 1, scale_next);
    }
    __syncthreads();
    // The groups' sums of a tile meet in one of them, a share of the tiles each.
    constexpr int SHARE = TM / KG;
    f32x4 sum[SHARE][TN];
    if constexpr (KG == 2) {
        f32x4 *const pass = reinterpret_cast<f32x4 *>(smem) + wave * SHARE * TN * 64 + lane;
        static_assert(2 * WAVES * SHARE * TN * 1024 <= 2 * KG * STAGE, "");
        constexpr int OTHER = WAVES * SHARE * TN * 64;
#pragma unroll
        for (int t = 0; t < SHARE; t++)
#pragma unroll
            for (int p = 0; p < TN; p++) {
                if (group == 0) pass[(t * TN + p) * 64] = acc[SHARE + t][p];
                else pass[OTHER + (t * TN + p) * 64] = acc[t][p];
            }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < SHARE; t++)
#pragma unroll
            for (int p = 0; p < TN; p++) {
                if (group == 0) sum[t][p] = acc[t][p] + pass[OTHER + (t * TN + p) * 64];
                else sum[t][p] = pass[(t * TN + p) * 64] + acc[SHARE + t][p];
            }
        __syncthreads();
    } else {
#pragma unroll
        for (int t = 0; t < TM; t++)
#pragma unroll
            for (int p = 0; p < TN; p++) sum[t][p] = acc[t][p];
    }
    // Two tiles' rows at a time go through the wavefront's own part of LDS, so that a row's outputs leave side by side.
    constexpr int PITCH = TN * 16 + 4, PAIR = SHARE < 2 ? SHARE : 2;
    static_assert(KG * WAVES * PAIR * 16 * PITCH * 4 <= 2 * KG * STAGE && SHARE % PAIR == 0, "");
    const Outputs outputs(o, (size_t)(panel0 + wn * TN) * 16 + lane % 16 * 4);
    static_assert(TN == 4, "a row's 64 outputs are 16 lanes'");
    float *const turned = reinterpret_cast<float *>(smem) + all_waves * PAIR * 16 * PITCH;
#pragma unroll
    for (int t = 0; t < SHARE; t += PAIR) {
#pragma unroll
        for (int x = 0; x < PAIR; x++)
#pragma unroll
            for (int p = 0; p < TN; p++)
                *reinterpret_cast<f32x4 *>(turned + (x * 16 + (lane & 15)) * PITCH + p * 16 + (lane >> 4) * 4) = sum[t + x][p];
        __builtin_amdgcn_wave_barrier();
        const size_t row = (size_t)(tile0 + wm * TM + group * SHARE + t) * 16 + lane / 16;
        const auto value = [&](int y) { return *reinterpret_cast<const f32x4 *>(turned + (y * 4 + lane / 16) * PITCH + lane % 16 * 4); };
        if (outputs.whole) {
            outputs.typed([&](auto u) {
#pragma unroll
                for (int y = 0; y < PAIR * 4; y++) outputs.template store_whole<decltype(u)>(row + y * 4, value(y));
            });
        } else {
#pragma unroll 1
            for (int y = 0; y < PAIR * 4; y++) outputs.store(row + y * 4, value(y));
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <int WM, int WN, int TM, int TN, int KG, bool EXACT>
hipError_t launch_tiles(const Rounded &in, const E4m3Panels &w, const E4m3Out &o, hipStream_t s) {
    const size_t m_tiles = div_ceil(in.tiles, WM * TM), n_tiles = div_ceil(w.panels, WN * TN);
    hipLaunchKernelGGL((tile_kernel<WM, WN, TM, TN, KG, EXACT>), dim3((unsigned)(m_tiles * n_tiles)), dim3(64 * WM * WN * KG), 0, s, in, w, o,
                       (int)m_tiles, (int)n_tiles);
    return hipGetLastError();
}

template <typename T, int MT, int PN, Source FROM>
hipError_t launch_few(const T *a, size_t lda, size_t k, bool aligned, const Rounded &in, const E4m3Panels &w, const E4m3Out &o,
                      hipStream_t s) {
    const dim3 grid((unsigned)div_ceil(w.panels, PN), (unsigned)div_ceil(div_ceil(o.m, 16), MT));
    hipLaunchKernelGGL((few_kernel<T, MT, PN, FROM>), grid, dim3(64 * FEW_WAVES), 0, s, a, lda, k, aligned, in, w, o);
    return hipGetLastError();
}

template <typename T>
hipError_t product(const T *a, size_t lda, size_t k, const E4m3Panels &w, const E4m3Out &o, const Rounded &in, hipStream_t s) {
    const bool aligned = reinterpret_cast<uintptr_t>(a) % 16 == 0 && lda * sizeof(T) % 16 == 0;
    if (!k) return launch_few<float, 2, 2, FRAGMENTS>(nullptr, 0, k, aligned, in, w, o, s);  // the epilogue of empty sums
    if (o.m <= E4M3_FEW) {
        // Each workgroup reads the rows again, and rounds them: two panels share that where they leave a workgroup to a CU, and
        // four where twice as many bytes of rows would be read (us, one panel, two and four): 16 rows of bf16 by 4096 x 4096 8.5
        // 9.6 12.4, by 4096 x 8192 14.3 10.6 14.1, by 4096 x 16384 24.8 16.6 20.5, by 1024 x 32768 22.6 13.1 11.7; of f32 by
        // 4096 x 4096 12.5 13.3 16.2, by 4096 x 8192 21.9 14.4 17.4, by 4096 x 16384 40.7 24.9 23.1; one row of bf16 by 8192 x
        // 8192 20.9 18.2 20.3.
        const auto launch = [&](auto pn) {
            constexpr int PN = decltype(pn)::value;
            if (aligned && k % 128 == 0) return launch_few<T, 1, PN, WHOLE>(a, lda, k, aligned, in, w, o, s);
            return launch_few<T, 1, PN, ANY>(a, lda, k, aligned, in, w, o, s);
        };
        if (w.panels * sizeof(T) >= 4096) return launch(std::integral_constant<int, 4>{});
        if (w.panels >= 512) return launch(std::integral_constant<int, 2>{});
        return launch(std::integral_constant<int, 1>{});
    }
    const size_t units = in.tiles * in.blocks, blocks = div_ceil(units, 4);
    hipLaunchKernelGGL((round_rows_kernel<T>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, s, a, lda, o.m,
                       k, aligned, in);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // Tiles of 128 x 128 by one group of wavefronts where those fill the 256 CUs twice over, by two groups where they fill
    // half of them, and blocks spread over eight wavefronts below that (us of a call; one group, two, 64 x 32 outputs and
    // 32 x 32 by eight wavefronts): 4000 rows by 4096 x 4096 145, 165, 206, 235; 1500 by 1024 x 4096 (384 tiles) 29.6,
    // 33.2, 39.6, 40.3; 2000 by 2048 x 2048 (256) 32.5, 29.9, 39.3, 42.1; 750 by 1024 x 4096 (192) 21.7, 20.3, 23.3, 24.4;
    // 256 by 4096 x 4096 (64) 44.0, 38.6, 21.0, 22.7; 750 by 4096 x 1024 (48) 46.2, 41.0, 22.3, 21.1; 64 by 4096 x 4096
    // 42.7, 37.6, 13.4, 11.2. 16-bit outputs: tiles of 256 x 256 where those fill the CUs.
    const size_t tiles = div_ceil(in.tiles, 8) * div_ceil(w.panels, 8);  // of 128 x 128
    if (o.type != F32) {
        if (div_ceil(in.tiles, 16) * div_ceil(w.panels, 16) >= 256) return launch_tiles<2, 4, 8, 4, 1, false>(in, w, o, s);
        if (tiles > 256) return launch_tiles<2, 2, 4, 4, 1, false>(in, w, o, s);
        if (tiles >= 96) return launch_tiles<2, 2, 4, 4, 2, false>(in, w, o, s);
    } else {
        if (tiles > 256) return launch_tiles<2, 2, 4, 4, 1, true>(in, w, o, s);
        if (tiles >= 128) return launch_tiles<2, 2, 4, 4, 2, true>(in, w, o, s);
    }
    if (div_ceil(in.tiles, 4) * div_ceil(w.panels, 2) >= 512) return launch_few<float, 4, 2, FRAGMENTS>(nullptr, 0, k, aligned, in, w, o, s);
    return launch_few<float, 2, 2, FRAGMENTS>(nullptr, 0, k, aligned, in, w, o, s);
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
