// What the attention, rotary and append kernels share: the stored types, where a sequence's rows lie,
// and which keys a query is shown.
#pragma once

#include "e4m3.hpp"
#include "tg_internal.hpp"

namespace tg {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(e4m3 x) { return e4m3_to_f32(x); }
// A weighted mean in the rows' type. Weights that were rounded up (sums of very many keys) take a mean of f16's largest
// values past 65520, which would round to infinity: a finite mean stays finite.
template <typename T>
__device__ __forceinline__ T mean_to(float x) {
    return (T)x;
}
template <>
__device__ __forceinline__ _Float16 mean_to<_Float16>(float x) {
    const float y = __builtin_amdgcn_fmed3f(x, -65504.0f, 65504.0f);
    return (_Float16)(x - x == 0.0f ? y : x);
}

// Eight values at p (16 bytes of a 16-bit type, 32 of f32; aligned to 16) in 32 bits, and back, rounded
// to nearest even.
__device__ __forceinline__ void load8(const float *p, float *v) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
    for (int i = 0; i < 4; i++) v[i] = a[i], v[i + 4] = b[i];
}
__device__ __forceinline__ void load8(const _Float16 *p, float *v) {
    const f16x8 a = *reinterpret_cast<const f16x8 *>(p);
    for (int i = 0; i < 8; i++) v[i] = (float)a[i];
}
__device__ __forceinline__ void load8(const __bf16 *p, float *v) {
    const bf16x8 a = *reinterpret_cast<const bf16x8 *>(p);
    for (int i = 0; i < 8; i++) v[i] = (float)a[i];
}
__device__ __forceinline__ void store8(float *p, const float *v) {
    *reinterpret_cast<f32x4 *>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4 *>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(_Float16 *p, const float *v) {
    f16x8 a;
    for (int i = 0; i < 8; i++) a[i] = (_Float16)v[i];
    *reinterpret_cast<f16x8 *>(p) = a;
}
__device__ __forceinline__ void store8(__bf16 *p, const float *v) {
    bf16x8 a;
    for (int i = 0; i < 8; i++) a[i] = (__bf16)v[i];
    *reinterpret_cast<bf16x8 *>(p) = a;
}

// Where sequence b's query and key rows lie. Row numbers from device memory are clamped to the buffers.
struct AttnSpan {
    int q0, nq;  // first query row, query rows
    int k0, nk;  // first key row (contiguous keys), keys
    __host__ __device__ inline int shift() const { return nk - nq; }  // the key position of query row 0
};
__host__ __device__ inline int clamp_to(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
__host__ __device__ inline AttnSpan span_of(const AttnSeqs &s, int b) {
    AttnSpan r;
    if (s.q_starts) {
        r.q0 = clamp_to(s.q_starts[b], 0, s.q_rows);
        r.nq = clamp_to(s.q_starts[b + 1], r.q0, s.q_rows) - r.q0;
    } else {
        r.nq = s.q_rows / s.batch;
        r.q0 = b * r.nq;
    }
    if (s.tables) {
        const int64_t held = (int64_t)s.width * s.page, most = 1 << 30;  // tiles past the last key count in 32 bits too
        r.k0 = 0;
        r.nk = s.pages ? clamp_to(s.lengths[b], 0, (int)(held < most ? held : most)) : 0;
    } else if (s.k_starts) {
        r.k0 = clamp_to(s.k_starts[b], 0, s.k_rows);
        r.nk = clamp_to(s.k_starts[b + 1], r.k0, s.k_rows) - r.k0;
    } else {
        r.nk = s.k_rows / s.batch;
        r.k0 = b * r.nk;
    }
    return r;
}

// The page that holds key position j of sequence b, or -1 where the table names none of the cache's, and the
// key's row in it.
__host__ __device__ inline int page_of(const AttnSeqs &s, int b, int j, int &row) {
    const int n = (int)((uint64_t)(uint32_t)j * s.page_mul >> s.page_shift);
    row = j - n * s.page;
    const int p = s.tables[(int64_t)b * s.ldt + n];
    return (unsigned)p < (unsigned)s.pages ? p : -1;
}

// Where the exponents of a row of an e4m3 page lie: those of its block, a head each.
__device__ __forceinline__ int64_t block_at(const AttnArgs &a, int64_t epage, int page, int row) {
    return page * epage + (int64_t)((uint64_t)(uint32_t)row * a.block_mul >> a.block_shift) * a.kv_heads;
}

// The keys that a query at position i is shown before documents are compared: lo <= j < hi, or j < prefix.
struct AttnWindow {
    int lo, hi, prefix;
    __host__ __device__ inline bool has(int j) const { return (j >= lo && j < hi) || j < prefix; }
};
__host__ __device__ inline AttnWindow window_of(int i, int nk, int32_t left, int32_t right, int prefix) {
    AttnWindow w;
    const int64_t lo = left < 0 ? 0 : (int64_t)i - left, hi = right < 0 ? nk : (int64_t)i + right + 1;
    w.lo = lo < 0 ? 0 : lo > nk ? nk : (int)lo;
    w.hi = hi < 0 ? 0 : hi > nk ? nk : (int)hi;
    w.prefix = clamp_to(prefix, 0, nk);
    return w;
}

constexpr float LOG2E = 1.44269504088896340736f;

// tanh to f32's accuracy: an odd polynomial below 0.3 (Taylor's, off by less than 2^-24 of x there), past it
// 1 - 2 / (e^2x + 1), whose absolute error of 2^-23 is relative to at least 0.29.
__device__ __forceinline__ float tanh_f32(float x) {
    const float a = fabsf(x), q = x * x;
    const float big = __builtin_copysignf(1.0f - 2.0f / (exp2f(2.0f * LOG2E * a) + 1.0f), x);
    float p = -1382.0f / 155925.0f;
    p = __builtin_fmaf(p, q, 62.0f / 2835.0f);
    p = __builtin_fmaf(p, q, -17.0f / 315.0f);
    p = __builtin_fmaf(p, q, 2.0f / 15.0f);
    p = __builtin_fmaf(p, q, -1.0f / 3.0f);
    return a < 0.3f ? __builtin_fmaf(x * q, p, x) : big;
}
// A product's score of head h at the distance key - query, with what the call does to scores.
__device__ __forceinline__ float score_of(const AttnArgs &a, float dot, int h, float slope, int distance) {
    float s = dot * a.scale;
    if (a.cap > 0.0f) s = a.cap * tanh_f32(s / a.cap);
    if (a.slopes) s -= slope * fabsf((float)distance);
    if (a.table)
        s += a.table[(int64_t)h * (2 * a.table_span + 1) + clamp_to(distance, -a.table_span, a.table_span) +
                     a.table_span];
    return s;
}

// Whether 16-bit rows take the hardware's reciprocal for their cap's tanh: it is off by 2^-22 absolutely, so the
// scores by at most 2^-14, an eighth of what f16's weights round away. The bound grows with the cap; larger ones take
// the tanh that is relative to the score, and so do caps so small that the factor before the score has no f32.
__host__ __device__ __forceinline__ float cap_factor(const AttnArgs &a) { return 2.0f * LOG2E * a.scale / a.cap; }
__host__ __device__ __forceinline__ bool fast_cap(const AttnArgs &a) {
    return a.cap <= 256.0f && cap_factor(a) < INFINITY;
}

// The same of a lane's N products, key_at(e) the e-th one's key: one kind of change after the other. FAST: fast_cap's
// where it holds, which a call without TABLE has seen to. TABLE: there may be a table.
template <bool FAST, int N, bool TABLE, typename S, typename F>
__device__ __forceinline__ void scores_of(const AttnArgs &a, S s, F key_at, int h, float slope, int i) {
    if (a.cap > 0.0f) {
        if (FAST && (!TABLE || fast_cap(a))) {
            const float into = cap_factor(a);
#pragma unroll
            for (int e = 0; e < N; e++)
                s(e) = __builtin_fmaf(-2.0f * a.cap,
                                      __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s(e) * into) + 1.0f), a.cap);
        } else {
#pragma unroll
            for (int e = 0; e < N; e++) s(e) = a.cap * tanh_f32(s(e) * a.scale / a.cap);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) s(e) *= a.scale;
    }
    if (a.slopes) {
#pragma unroll
        for (int e = 0; e < N; e++) s(e) = __builtin_fmaf(-slope, fabsf((float)(key_at(e) - i)), s(e));
    }
    if (TABLE && a.table) {
        const float *row = a.table + (int64_t)h * (2 * a.table_span + 1) + a.table_span;
#pragma unroll
        for (int e = 0; e < N; e++) s(e) += row[clamp_to(key_at(e) - i, -a.table_span, a.table_span)];
    }
}

// Row r of sequence b, head h, by one wavefront from the definition: a lane scores one key of 64 at a time,
// then the wavefront adds the weighted value rows of the keys that are shown, and of no others. The tile
// kernels multiply hidden keys' values by weights of zero, which makes a NaN of a NaN or an infinity: rows that
// come out of them not finite are computed again by this, slowly. C: the keys' type, e4m3 or T.
template <typename T, typename C = T>
__device__ void attend_row(const AttnArgs &a, int b, int h, int r, int lane) {
    const AttnSpan sp = span_of(a.seqs, b);
    const int64_t row = sp.q0 + r;
    const int kvh = h / (a.heads / a.kv_heads), i = sp.shift() + r;
    const T *q = static_cast<const T *>(a.q) + row * a.ldq + h * a.hsq;
    const AttnWindow win = window_of(i, sp.nk, a.left, a.right, a.prefix ? a.prefix[b] : 0);
    const int doc = a.q_docs ? a.q_docs[row] : 0;
    const float slope = a.slopes ? a.slopes[h] : 0.0f;
    float m = -INFINITY, l = 0.0f, acc[4] = {};
    for (int j0 = 0; j0 < sp.nk; j0 += 64) {
        const int j = j0 + lane;
        bool shown = j < sp.nk && win.has(j);
        int64_t kat = 0, vat = 0;
        float k_scale = 1.0f, v_scale = 1.0f;
        if (shown) {
            if (a.seqs.tables) {
                int at;
                const int p = page_of(a.seqs, b, j, at);
                shown = p >= 0;
                kat = p * a.psk + at * a.ldk;
                vat = p * a.psv + at * a.ldv;
                if (__is_same(C, e4m3) && shown) {
                    k_scale = two_to(a.k_exps[block_at(a, a.k_epage, p, at) + kvh]);
                    v_scale = two_to(a.v_exps[block_at(a, a.v_epage, p, at) + kvh]);
                }
            } else {
                kat = (int64_t)(sp.k0 + j) * a.ldk;
                vat = (int64_t)(sp.k0 + j) * a.ldv;
                if (a.q_docs) shown = doc >= 0 && a.k_docs[sp.k0 + j] == doc;
            }
        }
        float s = -INFINITY;
        if (shown) {
            const C *k = static_cast<const C *>(a.k) + kat + kvh * a.hsk;
            float dot = 0.0f;
            for (int c = 0; c < a.d; c++) {
                const float y = __is_same(C, e4m3) ? to_f32(k[c]) * k_scale : to_f32(k[c]);
                dot = __builtin_fmaf(to_f32(q[c]) + (a.rel_u ? a.rel_u[h * a.d + c] : 0.0f), y, dot);
            }
            if (a.rel) {
                const float *rr = a.rel + (clamp_to(j - i, -a.rel_span, a.rel_span) + a.rel_span) * a.ldrel + h * a.hsrel;
                float term = 0.0f;
                for (int c = 0; c < a.d; c++)
                    term = __builtin_fmaf(to_f32(q[c]) + (a.rel_v ? a.rel_v[h * a.d + c] : 0.0f), rr[c], term);
                dot += term;
            }
            s = score_of(a, dot, h, slope, j - i);
            shown = s != -INFINITY;
        }
        // A shown score of NaN or infinity makes the whole row NaN, whatever the other keys hold.
        if (__any(shown && !(s < INFINITY))) {
            l = NAN;
            break;
        }
        unsigned long long live = __ballot(shown);
        if (!live) continue;
        float top = s;
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
        const float p = shown ? expf(s - base) : 0.0f;
        const float fade = expf(m - base);
        l = l * fade + p;
        for (int e = 0; e < 4; e++) acc[e] *= fade;
        while (live) {
            const int t = __builtin_ctzll(live);
            live &= live - 1;
            const float w = __is_same(C, e4m3) ? __shfl(p * v_scale, t) : __shfl(p, t);
            const C *v = static_cast<const C *>(a.v) + __shfl(vat, t) + kvh * a.hsv;
            for (int e = 0; e < 4; e++)
                if (e * 64 + lane < a.d) acc[e] = __builtin_fmaf(w, to_f32(v[e * 64 + lane]), acc[e]);
        }
        m = mn;
    }
    for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
    T *out = static_cast<T *>(a.out) + row * a.ldo + h * a.hso;
    for (int e = 0; e < 4; e++)
        if (e * 64 + lane < a.d) out[e * 64 + lane] = mean_to<T>(l == 0.0f ? 0.0f : acc[e] / l);
}

// The parts of a call that splits its keys: per part, query row and head the score maximum, the sum of
// weights and the unnormalised output, in f32.
struct AttnParts {
    float *top, *sum, *out;  // [parts][rows x heads], [..], [parts][rows x heads][d]
    int parts;
    size_t pairs;  // rows x heads
};
inline size_t part_bytes(size_t pairs, size_t d) { return pairs * (d + 2) * sizeof(float); }
inline AttnParts parts_of(const AttnArgs &a, int parts) {
    AttnParts p;
    p.parts = parts;
    p.pairs = (size_t)a.seqs.q_rows * a.heads;
    p.out = static_cast<float *>(a.work);
    p.top = p.out + (size_t)parts * p.pairs * a.d;
    p.sum = p.top + (size_t)parts * p.pairs;
    return p;
}

}  // namespace tg
