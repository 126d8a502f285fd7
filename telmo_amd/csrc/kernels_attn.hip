// Attention over rows: out_i = sum_j p_ij v_j over the keys j that query i is shown, p_i their softmax of
//
//   s_ij = cap tanh(scale ((q_i + u) k_j + (q_i + w) r_c) / cap) - slope |j - i| + table[c'],
//
// c and c' the distance j - i clamped to the position rows' and the table's span; without cap, position
// rows, slopes or table those parts fall away. Shown are the keys of the query's own sequence in its
// window or prefix, in its document. A query that is shown nothing gets zeros.
//
// Statistics and sums are held in f32: one pass over the keys carries the running maximum m, the sum of
// exp(s - m) and the unnormalised output, both rescaled where m grows.
#include "attn_common.hpp"

namespace tg {

namespace {

constexpr int ROW_WAVES = 4;

// One wavefront per query row and head: a lane scores one key of 64 at a time, then the wavefront adds
// the 64 weighted value rows, a lane holding every 64th value of the output.
template <typename T, int DMAX>
__global__ __launch_bounds__(64 * ROW_WAVES) void attn_rows_kernel(const AttnArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.z, h = blockIdx.y, r = blockIdx.x * ROW_WAVES + wave;
    const AttnSpan sp = span_of(a.seqs, b);
    __shared__ float qs[ROW_WAVES][2][DMAX];
    if (r >= sp.nq) return;
    const int64_t row = sp.q0 + r;
    const int kvh = h / (a.heads / a.kv_heads), i = sp.shift() + r;
    const T *q = static_cast<const T *>(a.q) + row * a.ldq + h * a.hsq;
    float *qu = qs[wave][0], *qw = qs[wave][1];
    for (int c = lane; c < a.d; c += 64) {
        const float x = to_f32(q[c]);
        qu[c] = a.rel_u ? x + a.rel_u[h * a.d + c] : x;
        qw[c] = a.rel_v ? x + a.rel_v[h * a.d + c] : x;
    }
    const AttnWindow win = window_of(i, sp.nk, a.left, a.right, a.prefix ? a.prefix[b] : 0);
    const int doc = a.q_docs ? a.q_docs[row] : 0;
    float m = -INFINITY, l = 0.0f, acc[DMAX / 64] = {};
    for (int j0 = 0; j0 < sp.nk; j0 += 64) {
        const int j = j0 + lane;
        bool shown = j < sp.nk && win.has(j);
        int64_t kat = 0, vat = 0;
        if (shown) {
            if (a.seqs.tables) {
                const int p = page_of(a.seqs, b, j);
                shown = p >= 0;
                kat = p * a.psk + (j % a.seqs.page) * a.ldk;
                vat = p * a.psv + (j % a.seqs.page) * a.ldv;
            } else {
                kat = (int64_t)(sp.k0 + j) * a.ldk;
                vat = (int64_t)(sp.k0 + j) * a.ldv;
                if (a.q_docs) shown = doc >= 0 && a.k_docs[sp.k0 + j] == doc;
            }
        }
        float s = -INFINITY;
        if (shown) {
            const T *k = static_cast<const T *>(a.k) + kat + kvh * a.hsk;
            float dot = 0.0f;
            for (int c = 0; c < a.d; c += 8) {
                float x[8];
                load8(k + c, x);
                for (int e = 0; e < 8; e++) dot = __builtin_fmaf(qu[c + e], x[e], dot);
            }
            if (a.rel) {
                const int at = clamp_to(j - i, -a.rel_span, a.rel_span) + a.rel_span;
                const float *rr = a.rel + at * a.ldrel + h * a.hsrel;
                float term = 0.0f;
                for (int c = 0; c < a.d; c++) term = __builtin_fmaf(qw[c], rr[c], term);
                dot += term;
            }
            s = dot * a.scale;
            if (a.cap > 0.0f) s = a.cap * tanhf(s / a.cap);
            if (a.slopes) s -= a.slopes[h] * fabsf((float)(j - i));
            if (a.table)
                s += a.table[(int64_t)h * (2 * a.table_span + 1) + clamp_to(j - i, -a.table_span, a.table_span) +
                             a.table_span];
        }
        unsigned long long live = __ballot(shown);
        if (!live) continue;
        float top = s;
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
        const float p = shown ? expf(s - base) : 0.0f;
        const float fade = expf(m - base);
        l = l * fade + p;
        for (int e = 0; e < DMAX / 64; e++) acc[e] *= fade;
        while (live) {
            const int t = __builtin_ctzll(live);
            live &= live - 1;
            const float w = __shfl(p, t);
            const T *v = static_cast<const T *>(a.v) + __shfl(vat, t) + kvh * a.hsv;
            for (int e = 0; e < DMAX / 64; e++)
                if (e * 64 + lane < a.d) acc[e] = __builtin_fmaf(w, to_f32(v[e * 64 + lane]), acc[e]);
        }
        m = mn;
    }
    for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
    T *out = static_cast<T *>(a.out) + row * a.ldo + h * a.hso;
    for (int e = 0; e < DMAX / 64; e++)
        if (e * 64 + lane < a.d) out[e * 64 + lane] = (T)(l == 0.0f ? 0.0f : acc[e] / l);
}

template <typename T>
hipError_t launch_rows(const AttnArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)div_ceil((size_t)a.seqs.longest, ROW_WAVES), (unsigned)a.heads, (unsigned)a.seqs.batch);
    if (a.d <= 64)
        hipLaunchKernelGGL((attn_rows_kernel<T, 64>), grid, dim3(64 * ROW_WAVES), 0, s, a);
    else if (a.d <= 128)
        hipLaunchKernelGGL((attn_rows_kernel<T, 128>), grid, dim3(64 * ROW_WAVES), 0, s, a);
    else
        hipLaunchKernelGGL((attn_rows_kernel<T, 256>), grid, dim3(64 * ROW_WAVES), 0, s, a);
    return hipGetLastError();
}

}  // namespace

size_t attention_work_bytes(size_t, size_t, size_t, size_t, size_t, size_t) { return 0; }

hipError_t launch_attention(const AttnArgs &a, hipStream_t s) {
    switch (a.type) {
        case F16: return launch_rows<_Float16>(a, s);
        case BF16: return launch_rows<__bf16>(a, s);
        default: return launch_rows<float>(a, s);
    }
}

}  // namespace tg
