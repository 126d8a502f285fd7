// A token of each row of logits l, by a given random number u: with w_i = e^((l_i - max) / temperature), the tokens in the
// order of falling logits (equal ones by their numbers) are cut after the first top_k, then before the first one whose
// predecessors' weights reach top_p of what is left, then before the first one with w < min_p; the first always stays. The
// token is the first one whose running sum exceeds u times the sum of those kept.
//
// Nothing is sorted but what lies next to a border. Weights are whole numbers of 2^-42 (the largest is 1), so that
// their sums do not depend on their order, and are added into bins of the logits: 32 for each factor of two of the
// weight, 64 factors, the last one for all that is smaller. Their running counts and sums say in which bin each border
// lies; that bin's tokens are then gathered, sorted and added up in 64 bits. A bin with more tokens than LDS sorts is first
// divided by its logits' bits, down to a single value, whose tokens differ in their numbers alone.
//
// Rows of up to WHOLE tokens are the work of one workgroup. Longer ones are read in parts by as many workgroups, each of
// which leaves its bins, counted from its own largest logit, for the row's workgroup to add up.
#include "tg_internal.hpp"

namespace tg {

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int BINS = 2048, PER_OCTAVE = 32;
constexpr int LIST = 4096;  // tokens that are sorted at a time
constexpr int PART_THREADS = 512, PART_VALUES = 64, PART = PART_THREADS * PART_VALUES;
constexpr double FIXED = 1024.0;  // added to a weight it leaves steps of 2^-42: 2^22 weights' sum fits 64 bits

// What a part of a row leaves: its bins' counts and sums, relative to its largest logit.
struct PartBins {
    uint64_t mass[BINS];
    uint32_t count[BINS];
    float top;  // -infinity: no token
    uint32_t pad[3];
};

template <typename T>
__device__ __forceinline__ float logit(const T *row, int i) {
    return (float)row[i];
}
// A logit as bits that order as it does, larger first: 0 for +infinity.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l);
    return ~(b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    const uint32_t o = ~key;
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// Zeros of either sign are one logit.
__device__ __forceinline__ float plain(float l) { return l == 0.0f ? 0.0f : l; }

// 2^t for t <= 0 to 2^-47 of itself: Taylor's polynomial of e^x for |x| <= ln 2 / 2.
__device__ __forceinline__ double exp2_64(double t) {
    if (!(t > -1080.0)) return 0.0;
    const double n = __builtin_rint(t), x = (t - n) * 0.69314718055994530942;
    double p = 1.0 / 39916800.0;
    p = __builtin_fma(p, x, 1.0 / 3628800.0);
    p = __builtin_fma(p, x, 1.0 / 362880.0);
    p = __builtin_fma(p, x, 1.0 / 40320.0);
    p = __builtin_fma(p, x, 1.0 / 5040.0);
    p = __builtin_fma(p, x, 1.0 / 720.0);
    p = __builtin_fma(p, x, 1.0 / 120.0);
    p = __builtin_fma(p, x, 1.0 / 24.0);
    p = __builtin_fma(p, x, 1.0 / 6.0);
    p = __builtin_fma(p, x, 0.5);
    p = __builtin_fma(p, x, 1.0);
    p = __builtin_fma(p, x, 1.0);
    return __builtin_ldexp(p, (int)n);
}

// The row's scale of weights: c = log2 e / temperature.
struct Weights {
    double c;
    float top;  // the largest logit
    double top_bin;
    __device__ __forceinline__ Weights(float temperature, float top_) : c(1.44269504088896340736 / temperature), top(top_) {
        top_bin = bin_edge(top);
    }
    __device__ __forceinline__ double bin_edge(float l) const { return __builtin_floor((double)l * (PER_OCTAVE * c)); }
    __device__ __forceinline__ double of(float l) const { return l == top ? 1.0 : exp2_64(((double)l - (double)top) * c); }
    __device__ __forceinline__ int bin(float l) const {
        if (l == top) return 0;
        const double b = top_bin - bin_edge(l);
        return b < BINS - 1 ? (int)b : BINS - 1;  // a difference of infinities too
    }
};

__device__ __forceinline__ uint64_t fixed(double w) {
    return (uint64_t)(__builtin_bit_cast(int64_t, w + FIXED) - __builtin_bit_cast(int64_t, FIXED));
}
__device__ __forceinline__ double unfixed(uint64_t m) { return (double)m * 0x1p-42; }
// A sum of a part's weights, times the part's largest one.
__device__ __forceinline__ uint64_t fixed_times(uint64_t m, double share) {
    return share == 1.0 ? m : (uint64_t)((double)m * share + 0.5);
}

__device__ __forceinline__ void count_in(const Weights &w, float l, uint32_t *count, uint64_t *mass) {
    const int b = w.bin(l);
    atomicAdd(&count[b], 1u);
    atomicAdd(reinterpret_cast<unsigned long long *>(&mass[b]), (unsigned long long)fixed(w.of(l)));
}

__device__ __forceinline__ float wave_max(float x) {
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

// Running sums of bins.
struct Bins {
    double mass[BINS];  // fixed weights while they are added
    uint32_t count[BINS];
    __device__ __forceinline__ uint64_t *fixed_mass() { return reinterpret_cast<uint64_t *>(mass); }
    __device__ __forceinline__ void clear() {
        __syncthreads();
        for (int b = threadIdx.x; b < BINS; b += THREADS) count[b] = 0, fixed_mass()[b] = 0;
        __syncthreads();
    }
};

// What all threads of a row's workgroup share.
struct Shared {
    Bins row;
    union {
        Bins part;            // what a bin of too many tokens is divided into, before
        uint64_t list[LIST];  // its tokens: logit's key and number
    };
    double wave_mass[WAVES];
    uint32_t wave_count[WAVES];
    float wave_top[WAVES];
    uint32_t listed, keys[2];
    int first;
};

// Running counts and sums of PER THREADS values: f(i, count, mass) gives a value, g(i, count, mass, the value's own mass)
// takes the sums with it.
template <int PER, typename F, typename G>
__device__ __forceinline__ void running(Shared &s, F f, G g) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint32_t c[PER], count = 0;
    double m[PER], mass = 0.0;
    for (int i = 0; i < PER; i++) {
        f(t * PER + i, c[i], m[i]);
        count += c[i];
        mass += m[i];
    }
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(count, o);
        const double y = __shfl_up(mass, o);
        if (lane >= o) count += x, mass += y;
    }
    __syncthreads();
    if (lane == 63) s.wave_count[wave] = count, s.wave_mass[wave] = mass;
    __syncthreads();
    count = __shfl_up(count, 1), mass = __shfl_up(mass, 1);
    if (lane == 0) count = 0, mass = 0.0;
    uint32_t before = 0;
    double base = 0.0;
    for (int x = 0; x < wave; x++) before += s.wave_count[x], base += s.wave_mass[x];
    count += before;
    mass += base;
    for (int i = 0; i < PER; i++) {
        count += c[i];
        mass += m[i];
        g(t * PER + i, count, mass, m[i]);
    }
}

// The least of the threads' numbers.
__device__ __forceinline__ int least(Shared &s, int x) {
    __syncthreads();
    if (threadIdx.x == 0) s.first = INT32_MAX;
    __syncthreads();
    for (int o = 32; o; o >>= 1) x = min(x, __shfl_xor(x, o));
    if ((threadIdx.x & 63) == 0 && x != INT32_MAX) atomicMin(&s.first, x);
    __syncthreads();
    return s.first;
}

// The first key from low to high where f(key) holds, high where none does; f holds from there on. By one wavefront.
template <typename F>
__device__ __forceinline__ uint32_t first_key(uint32_t low, uint32_t high, F f) {
    while (low < high) {
        // The lanes try 64 keys between them, the last one high - 1 at most.
        const uint32_t step = (high - low - 1) / 64 + 1;
        const uint64_t at = low + (uint64_t)step * (threadIdx.x & 63);
        const unsigned long long which = __ballot(at >= high || f((uint32_t)at));
        const int n = which ? __builtin_ctzll(which) : 64;
        if (n == 0) return low;
        const uint32_t last = low + step * (n - 1);  // does not hold
        const uint64_t next = (uint64_t)low + (uint64_t)step * n;
        high = next < high ? (uint32_t)next : high;
        low = last + 1;
        if (step == 1) return n < 64 ? high : low;
    }
    return low;
}

// Tokens that follow one another in the order: those with keys from low to high, and what comes before them.
struct Range {
    uint32_t low, high, count, before;
    double mass_before;
};

template <typename T>
struct Row {
    const T *logits;
    int n;
    Weights w;
    Shared &s;

    // f(logit, token) for the row's tokens; NaN and -infinity are none.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const float l = plain(logit(logits, i));
            if (l > -INFINITY) f(l, i);
        }
    }

    // Counts and fixed weights become running sums.
    __device__ __forceinline__ void sum(Bins &bins) const {
        __syncthreads();
        running<BINS / THREADS>(
            s, [&](int i, uint32_t &c, double &m) { c = bins.count[i], m = unfixed(bins.fixed_mass()[i]); },
            [&](int i, uint32_t c, double m, double) { bins.count[i] = c, bins.mass[i] = m; });
        __syncthreads();
    }

    // The first bin where f(bin, running count, running mass) holds, or the last one that has tokens; counts and masses
    // after r's.
    template <typename F>
    __device__ __forceinline__ int first_bin(const Bins &bins, F f, Range &r) const {
        int x = INT32_MAX;
        for (int i = BINS / THREADS - 1; i >= 0; i--) {
            const int b = threadIdx.x * (BINS / THREADS) + i;
            if (f(b, r.before + bins.count[b], r.mass_before + bins.mass[b])) x = b;
        }
        int b = least(s, x);
        if (b == INT32_MAX) {
            for (int i = BINS / THREADS - 1; i >= 0; i--)
                if (bins.count[threadIdx.x * (BINS / THREADS) + i] == bins.count[BINS - 1]) x = threadIdx.x * (BINS / THREADS) + i;
            b = least(s, x);
        }
        const uint32_t earlier = b ? bins.count[b - 1] : 0u;
        r.count = bins.count[b] - earlier;
        r.before += earlier;
        r.mass_before += b ? bins.mass[b - 1] : 0.0;
        return b;
    }

    // Where the weights below min_p begin: their first bin and key.
    struct Floor {
        int bin = BINS;
        uint32_t key = UINT32_MAX;
    };

    // The tokens of the row's first bin where f(whether it reaches the floor, running count, running mass) holds, or of a
    // part of it: LIST tokens at most, or more of a single logit.
    template <typename F>
    __device__ Range range_of(const Floor &floor, F f) const {
        Range r{0, 0, 0, 0, 0.0};
        const int bin = first_bin(s.row, [&](int b, uint32_t c, double m) { return f(b >= floor.bin, c, m); }, r);
        const uint32_t all = key_of(-INFINITY), start = key_of(w.top);
        if (threadIdx.x < 128) {  // a wavefront for either end
            const int b = bin + (threadIdx.x >> 6);
            const uint32_t key = b == 0 ? start : b == BINS ? all : first_key(start, all, [&](uint32_t k) { return w.bin(plain(logit_of(k))) >= b; });
            if ((threadIdx.x & 63) == 0) s.keys[threadIdx.x >> 6] = key;
        }
        __syncthreads();
        r.low = s.keys[0], r.high = s.keys[1] - 1;
        while (r.count > LIST && r.low < r.high) {
            int shift = 0;  // keys of a part: 2^shift
            while ((r.high - r.low) >> shift >= BINS) shift++;
            s.part.clear();
            each([&](float l, int) {
                const uint32_t key = key_of(l);
                if (key < r.low || key > r.high) return;
                const uint32_t b = (key - r.low) >> shift;
                atomicAdd(&s.part.count[b], 1u);
                atomicAdd(reinterpret_cast<unsigned long long *>(&s.part.fixed_mass()[b]), (unsigned long long)fixed(w.of(l)));
            });
            sum(s.part);
            const auto end_of = [&](int b) {
                const uint32_t low = r.low + ((uint32_t)b << shift);
                return (r.high - low) >> shift ? low + (1u << shift) - 1 : r.high;
            };
            const int b = first_bin(s.part, [&](int b, uint32_t c, double m) { return f(end_of(b) >= floor.key, c, m); }, r);
            r.high = end_of(b);
            r.low += (uint32_t)b << shift;
        }
        return r;
    }

    // The range's tokens in s.list, in order.
    __device__ void sort(const Range &r) const {
        __syncthreads();
        if (threadIdx.x == 0) s.listed = 0;
        __syncthreads();
        each([&](float l, int i) {
            const uint32_t key = key_of(l);
            if (key < r.low || key > r.high) return;
            const uint32_t at = atomicAdd(&s.listed, 1u);
            if (at < LIST) s.list[at] = (uint64_t)key << 32 | (uint32_t)i;
        });
        int size = 2;
        while (size < (int)r.count) size *= 2;
        for (int i = r.count + threadIdx.x; i < size; i += THREADS) s.list[i] = ~0ull;
        for (int block = 2; block <= size; block *= 2)
            for (int step = block / 2; step; step /= 2) {
                __syncthreads();
                for (int i = threadIdx.x; i < size / 2; i += THREADS) {
                    const int a = 2 * i - (i & (step - 1)), b = a + step;
                    const uint64_t x = s.list[a], y = s.list[b];
                    if ((x > y) == ((a & block) == 0)) s.list[a] = y, s.list[b] = x;
                }
            }
        __syncthreads();
    }

    // The first token of the range where f(rank, mass before, weight) holds: its place in the range (the range's count where
    // it holds nowhere), the mass before it and its weight.
    template <typename F>
    __device__ int first_token(const Range &r, F f, double &mass, double &weight) const {
        if (r.count > LIST) {  // of a single logit
            const double one = w.of(logit_of(r.low));
            int lo = 0, hi = (int)r.count;  // f does not hold before lo, and holds from hi on
            while (lo < hi) {
                const int mid = lo + (hi - lo) / 2;
                if (f(r.before + mid, r.mass_before + mid * one, one)) hi = mid;
                else lo = mid + 1;
            }
            mass = r.mass_before + lo * one;
            weight = one;
            return lo;
        }
        sort(r);
        int x = INT32_MAX;
        double found_mass = 0.0, found_weight = 0.0, end = 0.0;
        running<LIST / THREADS>(
            s,
            [&](int i, uint32_t &c, double &m) {
                c = 0;
                m = i < (int)r.count ? w.of(logit_of((uint32_t)(s.list[i] >> 32))) : 0.0;
            },
            [&](int i, uint32_t, double with, double own) {
                end = with;
                if (i < (int)r.count && x == INT32_MAX && f(r.before + i, r.mass_before + (with - own), own))
                    x = i, found_mass = r.mass_before + (with - own), found_weight = own;
            });
        const int at = least(s, x);
        const int who = at == INT32_MAX ? THREADS - 1 : at / (LIST / THREADS);
        if ((int)threadIdx.x == who) {
            s.wave_mass[0] = at == INT32_MAX ? r.mass_before + end : found_mass;
            s.wave_mass[1] = at == INT32_MAX ? 0.0 : found_weight;
        }
        __syncthreads();
        mass = s.wave_mass[0];
        weight = s.wave_mass[1];
        return at == INT32_MAX ? (int)r.count : at;
    }

    // The token at a place of a range: from the sorted list, or the place-th of a single logit's.
    __device__ int token_at(const Range &r, int place) const {
        if (r.count <= LIST) return (int)(uint32_t)s.list[place];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        uint32_t seen = 0;
        for (int i0 = 0; i0 < n && seen <= (uint32_t)place; i0 += THREADS) {
            const int i = i0 + threadIdx.x;
            const bool mine = i < n && key_of(plain(logit(logits, i))) == r.low;
            const unsigned long long which = __ballot(mine);
            __syncthreads();
            if (lane == 0) s.wave_count[wave] = (uint32_t)__builtin_popcountll(which);
            __syncthreads();
            uint32_t at = seen + (uint32_t)__builtin_popcountll(which & ((1ull << lane) - 1));
            for (int x = 0; x < wave; x++) at += s.wave_count[x];
            if (mine && at == (uint32_t)place) s.first = i;
            for (int x = 0; x < WAVES; x++) seen += s.wave_count[x];
        }
        __syncthreads();
        return s.first;
    }
};

// The row's options.
struct Chosen {
    float temperature, top_p, min_p;
    int top_k;
    __device__ __forceinline__ Chosen(const SampleArgs &a, int row) {
        temperature = a.temperatures ? a.temperatures[row] : a.temperature;
        top_k = a.top_ks ? a.top_ks[row] : a.top_k;
        top_p = a.top_ps ? a.top_ps[row] : a.top_p;
        min_p = a.min_ps ? a.min_ps[row] : a.min_p;
    }
    // A single token stays.
    __device__ __forceinline__ bool greedy() const { return !(temperature > 0.0f) || top_k == 1 || top_p <= 0.0f; }
};

template <typename T>
__device__ float row_top(const T *logits, int n, Shared &s) {
    float top = -INFINITY;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += THREADS) top = fmaxf(top, logit(logits, i));  // NaN is passed over
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) s.wave_top[threadIdx.x >> 6] = top;
    __syncthreads();
    top = s.wave_top[0];
    for (int x = 1; x < WAVES; x++) top = fmaxf(top, s.wave_top[x]);
    return plain(top);
}

template <typename T>
__global__ __launch_bounds__(THREADS) void sample_kernel(const SampleArgs a, const PartBins *parts, int part_count) {
    __shared__ Shared s;
    const int r = blockIdx.x;
    const T *logits = static_cast<const T *>(a.logits) + (int64_t)r * a.ld;
    const Chosen o(a, r);
    float top = -INFINITY;
    if (parts) {
        parts += (size_t)r * part_count;
        for (int p = 0; p < part_count; p++) top = fmaxf(top, parts[p].top);
    } else {
        top = row_top(logits, a.n, s);
    }
    const auto answer = [&](int token, float prob) {
        if (threadIdx.x == 0) {
            a.tokens[r] = token;
            if (a.probs) a.probs[r] = prob;
        }
    };
    if (!(top > -INFINITY)) return answer(-1, 0.0f);
    if (o.greedy()) {
        int x = INT32_MAX;
        for (int i = threadIdx.x; i < a.n && x == INT32_MAX; i += THREADS)
            if (plain(logit(logits, i)) == top) x = i;
        return answer(least(s, x), 1.0f);
    }
    const Row<T> row{logits, a.n, Weights(o.temperature, top), s};
    const Weights &w = row.w;
    s.row.clear();
    if (parts) {
        // A part's bins, counted from its own largest logit, lie `by` bins further on, the last one taking all past it.
        for (int p = 0; p < part_count; p++) {
            const PartBins &x = parts[p];
            if (!(x.top > -INFINITY)) continue;
            const double by = x.top == top ? 0.0 : w.top_bin - w.bin_edge(x.top), share = w.of(x.top);
            const int on = by < BINS - 1 ? (int)by : BINS - 1;
            for (int y = threadIdx.x; y < BINS; y += THREADS) {
                const uint32_t count = x.count[y];
                if (!count) continue;
                const int b = y + on < BINS - 1 ? y + on : BINS - 1;
                atomicAdd(&s.row.count[b], count);
                atomicAdd(reinterpret_cast<unsigned long long *>(&s.row.fixed_mass()[b]), (unsigned long long)fixed_times(x.mass[y], share));
            }
        }
    } else {
        row.each([&](float l, int) { count_in(w, l, s.row.count, s.row.fixed_mass()); });
    }
    row.sum(s.row);
    const uint32_t all = s.row.count[BINS - 1];
    uint32_t kept = o.top_k > 0 && (uint32_t)o.top_k < all ? (uint32_t)o.top_k : all;
    double mass = s.row.mass[BINS - 1], weight;
    if (kept < all) {
        const uint32_t k = kept;
        const Range x = row.range_of({}, [&](bool, uint32_t c, double) { return c > k; });
        row.first_token(x, [&](uint32_t rank, double, double) { return rank >= k; }, mass, weight);
    }
    if (o.top_p < 1.0f || o.min_p > 0.0f) {
        const double most = o.top_p < 1.0f ? (double)o.top_p * mass : INFINITY, least_weight = o.min_p;
        const uint32_t k = kept;
        typename Row<T>::Floor floor;
        if (o.min_p > 0.0f) {
            __syncthreads();
            if (threadIdx.x < 64) {
                const uint32_t end = key_of(-INFINITY);
                const uint32_t key = first_key(key_of(top), end, [&](uint32_t y) { return w.of(plain(logit_of(y))) < least_weight; });
                if (threadIdx.x == 0) s.keys[0] = key, s.first = key == end ? BINS : w.bin(plain(logit_of(key)));
            }
            __syncthreads();
            floor.bin = s.first, floor.key = s.keys[0];
        }
        const Range x = row.range_of(floor, [&](bool low, uint32_t c, double m) { return c > k || m > most || low; });
        const int at = row.first_token(
            x, [&](uint32_t rank, double before, double own) { return rank > 0 && (rank >= k || before >= most || own < least_weight); },
            mass, weight);
        kept = x.before + at;
    }
    const double target = (double)fminf(a.uniforms[r], 0x1.fffffep-1f) * mass;
    const Range x = row.range_of({}, [&](bool, uint32_t c, double m) { return m > target || c >= kept; });
    const uint32_t last = (kept < x.before + x.count ? kept : x.before + x.count) - 1;
    double before;
    const int at = row.first_token(
        x, [&](uint32_t rank, double sum, double own) { return rank >= last || sum + own > target; }, before, weight);
    answer(row.token_at(x, at), (float)(weight / mass));
}

// The bins of a part of a row: its logits stay in registers from the largest to the weights.
template <typename T>
__global__ __launch_bounds__(PART_THREADS) void parts_kernel(const SampleArgs a, PartBins *parts, int part_count) {
    __shared__ uint64_t mass[BINS];
    __shared__ uint32_t count[BINS];
    __shared__ float tops[PART_THREADS / 64];
    const int r = blockIdx.x / part_count, p = blockIdx.x % part_count;
    PartBins &out = parts[blockIdx.x];
    const Chosen o(a, r);
    const T *logits = static_cast<const T *>(a.logits) + (int64_t)r * a.ld + (int64_t)p * PART;
    const int n = min(a.n - p * PART, PART);
    float l[PART_VALUES];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PART_VALUES; i++) {
        const int at = i * PART_THREADS + threadIdx.x;
        l[i] = at < n ? plain(logit(logits, at)) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < PART_VALUES; i++) top = fmaxf(top, l[i]);
    for (int b = threadIdx.x; b < BINS; b += PART_THREADS) mass[b] = 0, count[b] = 0;
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int x = 0; x < PART_THREADS / 64; x++) top = fmaxf(top, tops[x]);
    if (threadIdx.x == 0) out.top = top;
    if (!(top > -INFINITY) || o.greedy()) return;
    const Weights w(o.temperature, top);
#pragma unroll
    for (int i = 0; i < PART_VALUES; i++)
        if (l[i] > -INFINITY) count_in(w, l[i], count, mass);
    __syncthreads();
    for (int b = threadIdx.x; b < BINS; b += PART_THREADS) out.mass[b] = mass[b], out.count[b] = count[b];
}

int part_count_of(size_t n) { return n <= SAMPLE_WHOLE ? 0 : (int)div_ceil(n, PART); }

}  // namespace

size_t sample_work_bytes(size_t rows, size_t n) { return rows * part_count_of(n) * sizeof(PartBins); }

hipError_t launch_sample(const SampleArgs &a, uint32_t type, int rows, void *work, hipStream_t s) {
    const int count = part_count_of((size_t)a.n);
    PartBins *parts = count ? static_cast<PartBins *>(work) : nullptr;
    const auto launch = [&](auto t) {
        using T = decltype(t);
        if (count) {
            hipLaunchKernelGGL((parts_kernel<T>), dim3((unsigned)(rows * count)), dim3(PART_THREADS), 0, s, a, parts, count);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        hipLaunchKernelGGL((sample_kernel<T>), dim3((unsigned)rows), dim3(THREADS), 0, s, a, (const PartBins *)parts, count);
        return hipGetLastError();
    };
    switch (type) {
        case F16: return launch(_Float16{});
        case BF16: return launch(__bf16{});
        default: return launch(float{});
    }
}

}  // namespace tg
