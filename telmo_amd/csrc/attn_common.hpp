// What the attention, rotary and append kernels share: the stored types, where a sequence's rows lie,
// and which keys a query is shown.
#pragma once

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
        const int64_t held = (int64_t)s.width * s.page;
        r.k0 = 0;
        r.nk = clamp_to(s.lengths[b], 0, held < INT32_MAX ? (int)held : INT32_MAX);
    } else if (s.k_starts) {
        r.k0 = clamp_to(s.k_starts[b], 0, s.k_rows);
        r.nk = clamp_to(s.k_starts[b + 1], r.k0, s.k_rows) - r.k0;
    } else {
        r.nk = s.k_rows / s.batch;
        r.k0 = b * r.nk;
    }
    return r;
}

// The page that holds key position j of sequence b, or -1 where the table names none of the cache's.
__host__ __device__ inline int page_of(const AttnSeqs &s, int b, int j) {
    const int p = s.tables[(int64_t)b * s.ldt + j / s.page];
    return (unsigned)p < (unsigned)s.pages ? p : -1;
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

}  // namespace tg
