// A token of each row of logits l, by a given random number u: with w_i = e^((l_i - max) / temperature), the tokens in the
// order of falling logits (equal ones by their numbers) are cut after the first top_k, then before the first one whose
// predecessors' weights reach top_p of what is left, then before the first one with w < min_p; the first always stays. The
// token is the first one whose running sum exceeds u times the sum of those kept.
//
// Nothing is sorted but what lies next to a border. Tokens are counted and their weights added in bins of the logits: 32 for
// each factor of two of the weight, 64 factors, the last one (of weight 0 in these sums) for all that is smaller. The bin is
// floor y with y = 32 l log2 e / temperature, rounded once to steps of 2^-40, and a bin's sum is of 2^(y - floor y) - 1 in
// whole numbers of 2^-40, so that it depends neither on the order nor on the row's largest logit; one 64-bit atomic counts a
// token and adds its weight. The running counts and
// sums say in which bins each border and the drawn token can lie; the tokens of these bins are gathered in one pass,
// sorted, and added up in 64 bits. If they are more than LDS sorts, the borders are looked for one after the other, and a
// bin of too many tokens is first divided by its logits' bits, down to a single value, whose tokens differ in their
// numbers alone.
//
// Rows of up to WHOLE tokens are the work of one workgroup, which holds them in registers (so that they are read once).
// Longer ones are read in parts by as many workgroups, each of which leaves its bins, counted from its own largest logit, for
// the row's workgroup.
//
// 256 rows of 131072 f32 logits take 39 us for the parts (3.4 TB/s; 22 vector instructions for each logit, most of them in 64
// bits) and 56 us for the rows, half of it the second reading of the logits at 5 TB/s; with the rows read by a gathering
// after each border it was 129 us. A row of 8198 takes 14 us, no phase of it (load, count, sum, search, gather, sort, add) more
// than 3: waits for memory, LDS and instructions that nothing overlaps.
#include "tg_internal.hpp"

namespace tg {

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int BINS = 2048, PER_OCTAVE = 32;
constexpr int LIST = 4096;  // tokens that are sorted at a time
constexpr int WHOLE = (int)SAMPLE_WHOLE, WHOLE_VALUES = WHOLE / THREADS, SHORT_VALUES = 16;
constexpr int PART_THREADS = 256, PART_VALUES = 64, PART = PART_THREADS * PART_VALUES;
constexpr int COPIES = 2;     // of the bins that are counted: lanes next to each other add to different ones
constexpr int SUM_BITS = 49;  // of a counted bin; above them the count of up to 2^14 tokens, whose sum is below 2^48.5
static_assert(WHOLE <= COPIES << 14 && PART <= 1 << 14, "a bin's count and sum share 64 bits");
// Added to a weight it leaves steps of 2^-42. 2^22 weights' sum fits 64 bits, but for 2^22 ones, which come to 0: they are the
// whole row, in one bin, which is taken whatever its sum.
constexpr double FIXED = 1024.0;

// What a part of a row leaves: its bins, relative to its largest logit.
struct PartBins {
    uint64_t bins[BINS];
    float top;  // -infinity: no token
    uint32_t tokens, pad[2];
};

// Zeros of either sign are one logit.
__device__ __forceinline__ float plain(float l) { return l + 0.0f; }
// A logit as bits that order as it does, larger first: 0 for +infinity.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l);
    return ~(b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    const uint32_t o = ~key;
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

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

// 2^(f / 32) - 1 in steps of 2^-40 for the fraction f of a place, by Taylor's polynomial up to f^6 (the next term is below
// 2^-50).
struct Share {
    static constexpr double X = 0.69314718055994530942 / PER_OCTAVE;
    double p[6] = {X * X * X * X * X * X / 720.0, X * X * X * X * X / 120.0, X * X * X * X / 24.0, X * X * X / 6.0, X * X / 2.0, X};
    // In registers: as constants each would be moved there again for each logit.
    __device__ __forceinline__ Share() {
#pragma unroll
        for (int i = 0; i < 6; i++) asm("" : "+v"(p[i]));
    }
    __device__ __forceinline__ uint64_t operator()(double place) const {
        const double f = __builtin_amdgcn_fract(place);
        double s = p[0];
#pragma unroll
        for (int i = 1; i < 6; i++) s = __builtin_fma(s, f, p[i]);
        return __builtin_bit_cast(uint64_t, __builtin_fma(s, f, 0x1p12)) - __builtin_bit_cast(uint64_t, 0x1p12);
    }
};

// The scale of a row's weights, c = log2 e / temperature, and its bins. y - edge for l, with the edge floor y of the
// largest logit, lies in (-BINS + 1, 1) and is added to POINT in one rounding: steps of 2^-40, and the bin in the bits above.
constexpr double POINT = 0x1.8p12;
constexpr int POINT_BITS = 0x40b800;  // of POINT, the upper 24
struct Weights {
    double c, k, shift, edge;
    float top;  // the largest logit
    bool far;   // logits that differ from it lie in the last bin
    __device__ __forceinline__ Weights(float temperature, float top_) : c(1.44269504088896340736 / temperature), top(top_) {
        const double wide = PER_OCTAVE * c, y = (double)top * wide;
        far = !(__builtin_fabs(y) < 0x1p40);
        // f32 neighbours are 2^-24 apart at least: 2^14 bins with |y| brought down to 2^38. To infinity everything is far.
        k = top == INFINITY ? 0x1p-200 : __builtin_ldexp(wide, far ? 39 - __builtin_amdgcn_frexp_exp(y) : 0);
        edge = __builtin_floor((double)top * k);
        edge += __builtin_floor(__builtin_fma((double)top, k, POINT - edge) - POINT);
        edge = top == INFINITY ? INFINITY : edge;
        shift = top == INFINITY ? POINT - (BINS - 1) : POINT - edge;
    }
    __device__ __forceinline__ double of(float l) const { return l == top ? 1.0 : exp2_64(((double)l - (double)top) * c); }
    __device__ __forceinline__ double place(float l) const {
        return fmin(fmax(__builtin_fma((double)l, k, shift), POINT - (BINS - 1)), POINT + 1.0 - 0x1p-40);
    }
    static __device__ __forceinline__ uint32_t upper(double place) { return (uint32_t)(__builtin_bit_cast(uint64_t, place) >> 32); }
    static __device__ __forceinline__ int bin_of(double place) { return POINT_BITS - (int)(upper(place) >> 8); }
    __device__ __forceinline__ int bin(float l) const { return bin_of(place(l)); }
    // How much further on the bins lie that are counted from another, lower logit.
    __device__ __forceinline__ int further(const Weights &w) const {
        const double by = edge - w.edge;
        return w.top == top ? 0 : far || w.far || !(by < BINS - 1) ? BINS - 1 : (int)by;
    }
    __device__ __forceinline__ void count_in(float l, uint64_t *bins, const Share &share) const {
        const double at = place(l);
        atomicAdd(reinterpret_cast<unsigned long long *>(&bins[bin_of(at) * COPIES + (threadIdx.x & (COPIES - 1))]),
                  (unsigned long long)(share(at) + ((uint64_t)1 << SUM_BITS)));
    }
};

__device__ __forceinline__ uint64_t fixed(double w) {
    return (uint64_t)(__builtin_bit_cast(int64_t, w + FIXED) - __builtin_bit_cast(int64_t, FIXED));
}
__device__ __forceinline__ double unfixed(uint64_t m) { return (double)m * 0x1p-42; }

// N logits of each of X pieces from row[begin + first(piece)] on, wherever they lie; -infinity past the n-th of the row.
// The pieces start at multiples of N from a multiple of N.
template <int X, int N, typename T, typename F>
__device__ __forceinline__ void load(const T *row, int begin, int n, float (&l)[X][N], F first) {
    struct __attribute__((packed, aligned(sizeof(T)))) Piece {
        T v[N];
    };
    Piece p[X];
    float end[N];  // of the row's last, shorter piece
    const int last = n / N * N;
    if (n >= N) {
#pragma unroll
        for (int x = 0; x < X; x++) {
            const int at = begin + first(x);
            const uint32_t bytes = (uint32_t)(at < last ? at : 0) * (uint32_t)sizeof(T);
            p[x] = *reinterpret_cast<const Piece *>(reinterpret_cast<const char *>(row) + bytes);
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) end[i] = last + i < n ? plain((float)row[last + i]) : -INFINITY;
#pragma unroll
    for (int x = 0; x < X; x++) {
        const int at = begin + first(x);
#pragma unroll
        for (int i = 0; i < N; i++) l[x][i] = at < last ? plain((float)p[x].v[i]) : -INFINITY;
        if (at == last) {
#pragma unroll
            for (int i = 0; i < N; i++) l[x][i] = end[i];
        }
    }
}

// x of the lane before by a DPP control, `other` where there is none.
template <int CONTROL, int ROWS = 0xf, typename X>
__device__ __forceinline__ X from_lane(X x, X other) {
    if constexpr (sizeof(X) == 4) {
        return __builtin_bit_cast(X, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, other), __builtin_bit_cast(int, x), CONTROL, ROWS, 0xf, false));
    } else {
        const uint64_t a = __builtin_bit_cast(uint64_t, x), b = __builtin_bit_cast(uint64_t, other);
        return __builtin_bit_cast(X, (uint64_t)from_lane<CONTROL, ROWS>((uint32_t)a, (uint32_t)b) | (uint64_t)from_lane<CONTROL, ROWS>((uint32_t)(a >> 32), (uint32_t)(b >> 32)) << 32);
    }
}
// f over the lanes up to each.
template <typename X, typename F>
__device__ __forceinline__ X scan(X x, X none, F f) {
    x = f(from_lane<0x111>(x, none), x);
    x = f(from_lane<0x112>(x, none), x);
    x = f(from_lane<0x114>(x, none), x);
    x = f(from_lane<0x118>(x, none), x);
    x = f(from_lane<0x142, 0xa>(x, none), x);
    return f(from_lane<0x143, 0xc>(x, none), x);
}
__device__ __forceinline__ float wave_max(float x) {
    x = scan(x, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// The first of n <= 4096 numbers where f holds, n where none does; f holds from there on. By each wavefront for itself.
template <typename F>
__device__ __forceinline__ int first_of(int n, F f) {
    const int lane = threadIdx.x & 63;
    int low = 0;
    if (n > 64) {
        const int end = 64 * lane + 63;  // the last number of the lane's 64
        const unsigned long long which = __ballot(end >= n || f(end));
        low = 64 * (which ? (int)__builtin_ctzll(which) : 64);
    }
    const unsigned long long which = __ballot(low + lane >= n || f(low + lane));
    return min(low + (which ? (int)__builtin_ctzll(which) : 64), n);
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
    // The bin that has tokens where f(bin, running count, running mass) first holds, or the last one.
    template <typename F>
    __device__ __forceinline__ int first(F f) const {
        return with_tokens(first_of(BINS, [&](int x) { return f(x, count[x], mass[x]); }));
    }
    // Between bins without any, sums may grow by a rounding: then the bin before them.
    __device__ __forceinline__ int with_tokens(int b) const {
        if (b < BINS && count[b] > (b ? count[b - 1] : 0u)) return b;
        const uint32_t c = max(count[min(b, BINS - 1)], 1u);
        return first_of(BINS, [&](int x) { return count[x] >= c; });
    }
    // Two of them at a time.
    struct Border {
        uint32_t count;
        double mass;
        int bin;
        __device__ __forceinline__ bool past(int b, uint32_t c, double m) const { return c > count || m > mass || b >= bin; }
    };
    __device__ __forceinline__ void first(const Border &x, const Border &y, int &at_x, int &at_y) const {
        static_assert(BINS == 32 * 64, "half a wavefront's lanes look at every 64th bin");
        const int lane = threadIdx.x & 63, end = 64 * (lane & 31) + 63;
        const uint32_t c = count[end];
        const double m = mass[end];
        const unsigned long long which = __ballot(lane < 32 ? x.past(end, c, m) : y.past(end, c, m));
        const uint32_t low = (uint32_t)which, high = (uint32_t)(which >> 32);
        const int at_low = min(low ? __builtin_ctz(low) * 64 : BINS, BINS - 64), at_high = min(high ? __builtin_ctz(high) * 64 : BINS, BINS - 64);
        const unsigned long long of_x = __ballot(x.past(at_low + lane, count[at_low + lane], mass[at_low + lane]));
        const unsigned long long of_y = __ballot(y.past(at_high + lane, count[at_high + lane], mass[at_high + lane]));
        at_x = with_tokens(of_x ? at_low + (int)__builtin_ctzll(of_x) : BINS);
        at_y = with_tokens(of_y ? at_high + (int)__builtin_ctzll(of_y) : BINS);
    }
};

// What all threads of a row's workgroup share.
struct Shared {
    Bins row;
    union {
        uint64_t counted[BINS * COPIES];
        Bins part;  // what a bin of too many tokens is divided into, before
        struct {
            uint64_t list[LIST];  // its tokens: logit's key and number
            double before[LIST];  // the weights of those before in the list
        };
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
    count = scan(count, 0u, [](uint32_t a, uint32_t b) { return a + b; });
    mass = scan(mass, 0.0, [](double a, double b) { return a + b; });
    __syncthreads();
    if (lane == 63) s.wave_count[wave] = count, s.wave_mass[wave] = mass;
    __syncthreads();
    count = from_lane<0x138>(count, 0u), mass = from_lane<0x138>(mass, 0.0);
    uint32_t before = 0;
    double base = 0.0;
#pragma unroll
    for (int x = 0; x < WAVES - 1; x++) {
        const uint32_t c = s.wave_count[x];
        const double m = s.wave_mass[x];
        before += x < wave ? c : 0u, base += x < wave ? m : 0.0;
    }
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

// A row's logits: HELD of them in each thread's registers, or read again for each pass.
template <typename T, int HELD>
struct Logits {
    static constexpr int PIECE = 16 / sizeof(T), PIECES = (HELD ? HELD : 32) / PIECE;
    const T *row;
    int n;
    float held[HELD ? PIECES : 1][PIECE];

    __device__ __forceinline__ Logits(const T *row_, int n_) : row(row_), n(n_) {
        if constexpr (HELD > 0) read(held, 0);
    }
    __device__ __forceinline__ static int first(int piece) { return (piece * THREADS + (int)threadIdx.x) * PIECE; }
    __device__ __forceinline__ void read(float (&l)[PIECES][PIECE], int begin) const { load(row, begin, n, l, first); }
    // f(logit, token) for the row's tokens; NaN and -infinity are none.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        if constexpr (HELD > 0) {
            visit(held, 0, f);
        } else {
            for (int begin = 0; begin < n; begin += PIECES * THREADS * PIECE) {
                float l[PIECES][PIECE];
                read(l, begin);
                visit(l, begin, f);
            }
        }
    }
    // g(token) for the few tokens where f(logit) holds.
    template <typename F, typename G>
    __device__ __forceinline__ void each_of(F f, G g) const {
        const auto some = [&](const float (&l)[PIECES][PIECE], int begin) {
            static_assert(PIECES * PIECE <= 32, "a bit for each");
            uint32_t which = 0;
#pragma unroll
            for (int i = 0; i < PIECES * PIECE; i++) which |= f(l[i / PIECE][i % PIECE]) ? 1u << i : 0u;
            while (which) {
                const int i = __builtin_ctz(which);
                which &= which - 1;
                g(begin + first(i / PIECE) + i % PIECE);
            }
        };
        if constexpr (HELD > 0) {
            some(held, 0);
        } else {
            for (int begin = 0; begin < n; begin += PIECES * THREADS * PIECE) {
                float l[PIECES][PIECE];
                read(l, begin);
                some(l, begin);
            }
        }
    }
    template <typename F>
    __device__ __forceinline__ void visit(const float (&l)[PIECES][PIECE], int begin, F f) const {
#pragma unroll
        for (int x = 0; x < PIECES; x++)
#pragma unroll
            for (int y = 0; y < PIECE; y++)
                if (l[x][y] > -INFINITY) f(l[x][y], begin + first(x) + y);
    }
};

// Bins next to each other whose tokens are gathered: their place in the list, and the tokens and weights before them.
struct Span {
    int low, high, start = 0, count = 0;
    uint32_t before = 0;
    double mass_before = 0.0;
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

struct Drawn {
    int token;
    float prob;
};

// The first tokens of s.list in order.
__device__ __forceinline__ void sort_list(Shared &s, int count) {
    __syncthreads();
    if (count <= THREADS / 4) {  // four lanes count the tokens before one
        const int i = threadIdx.x / 4;
        const uint64_t own = i < count ? s.list[i] : 0;
        int place = 0;
        if (i < count)
            for (int y = threadIdx.x & 3; y < count; y += 4) place += s.list[y] < own;
        place += __shfl_xor(place, 1);
        place += __shfl_xor(place, 2);
        __syncthreads();
        if (i < count && (threadIdx.x & 3) == 0) s.list[place] = own;
        __syncthreads();
        return;
    }
    // Runs of 16, then twice as long ones from each two: a token's place is its own in its run and that in the other.
    constexpr int PER = LIST / THREADS, RUN = 16;
    static_assert(sizeof(s.before) == sizeof(s.list), "the runs go back and forth");
    uint64_t *from = s.list, *to = reinterpret_cast<uint64_t *>(s.before);
    for (int run = 1; run < count; run *= run == 1 ? RUN : 2) {
#pragma unroll
        for (int x = 0; x < PER; x++) {
            const int i = x * THREADS + threadIdx.x;
            if (i >= count) continue;
            const uint64_t own = from[i];
            int place;
            if (run == 1) {
                const int start = i & ~(RUN - 1), n = min(RUN, count - start);
                place = start;
                if (n == RUN) {
#pragma unroll
                    for (int y = 0; y < RUN; y++) place += from[start + y] < own;
                } else {
                    for (int y = 0; y < n; y++) place += from[start + y] < own;
                }
            } else {
                const int both = i & ~(2 * run - 1), other = (i & ~(run - 1)) == both ? both + run : both;
                int low = 0, high = max(min(run, count - other), 0);
                while (low < high) {
                    const int mid = (low + high) / 2;
                    if (from[other + mid] < own) low = mid + 1;
                    else high = mid;
                }
                place = both + (i & (run - 1)) + low;
            }
            to[place] = own;
        }
        __syncthreads();
        uint64_t *t = from;
        from = to, to = t;
    }
    if (from != s.list) {
        for (int i = threadIdx.x; i < count; i += THREADS) s.list[i] = from[i];
        __syncthreads();
    }
}

// The tokens of the spans in s.list, in order, and the weights before each.
template <typename T, int HELD>
__device__ __forceinline__ void gather(const Logits<T, HELD> &logits, const Weights &w, Shared &s, const Span &x, const Span &y, const Span &z, int count) {
    __syncthreads();  // the counted bins lie where the list does
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    const auto within = [](const Span &x, uint32_t upper) {
        return upper - ((uint32_t)(POINT_BITS - x.high) << 8) < (uint32_t)(x.high - x.low + 1) << 8;
    };
    logits.each_of([&](float l) {
        const uint32_t upper = Weights::upper(w.place(l));
        return (l > -INFINITY) & (within(x, upper) | within(y, upper) | within(z, upper));
    }, [&](int i) {
        const uint32_t at = atomicAdd(&s.listed, 1u);
        if (at < LIST) s.list[at] = (uint32_t)i;
    });
    // Their logits are read once more, all at a time.
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += THREADS) s.list[i] |= (uint64_t)key_of(plain((float)logits.row[(uint32_t)s.list[i]])) << 32;
    sort_list(s, count);
    const auto weight = [&](int i, uint32_t &c, double &m) { c = 0, m = i < count ? w.of(logit_of((uint32_t)(s.list[i] >> 32))) : 0.0; };
    const auto put = [&](int i, uint32_t, double with, double own) { s.before[i] = with - own; };
    if (count <= THREADS) running<1>(s, weight, put);
    else running<LIST / THREADS>(s, weight, put);
    __syncthreads();
}

template <typename T>
struct Row {
    const Logits<T, 0> logits;
    Weights w;
    Shared &s;

    // Counts and fixed weights become running sums.
    __device__ __forceinline__ void sum(Bins &bins) const {
        __syncthreads();
        running<BINS / THREADS>(
            s, [&](int i, uint32_t &c, double &m) { c = bins.count[i], m = unfixed(bins.fixed_mass()[i]); },
            [&](int i, uint32_t c, double m, double) { bins.count[i] = c, bins.mass[i] = m; });
        __syncthreads();
    }

    // The bin that has tokens where f(bin, running count, running mass) first holds, or the last one; counts and masses
    // after r's.
    template <typename F>
    __device__ __forceinline__ int first_bin(const Bins &bins, F f, Range &r) const {
        const int b = bins.first([&](int x, uint32_t c, double m) { return f(x, r.before + c, r.mass_before + m); });
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
        __syncthreads();  // all have the floor's key, and the ends of the range before
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
            logits.each([&](float l, int) {
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
        logits.each([&](float l, int i) {
            const uint32_t key = key_of(l);
            if (key < r.low || key > r.high) return;
            const uint32_t at = atomicAdd(&s.listed, 1u);
            if (at < LIST) s.list[at] = (uint64_t)key << 32 | (uint32_t)i;
        });
        sort_list(s, (int)r.count);
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
        for (int i0 = 0; i0 < logits.n && seen <= (uint32_t)place; i0 += THREADS) {
            const int i = i0 + threadIdx.x;
            const bool mine = i < logits.n && key_of(plain((float)logits.row[i])) == r.low;
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

// The borders one after the other, by their bins' tokens alone or parts of them.
template <typename T>
__device__ __noinline__ Drawn step_by_step(const T *logits, int n, Weights w, Shared &s, uint32_t k, uint32_t all, double u, double share, double least_weight) {
    const Row<T> row{Logits<T, 0>(logits, n), w, s};
    uint32_t kept = k;
    double mass = s.row.mass[BINS - 1], weight;
    if (k < all) {
        const Range x = row.range_of({}, [&](bool, uint32_t c, double) { return c > k; });
        row.first_token(x, [&](uint32_t rank, double, double) { return rank >= k; }, mass, weight);
    }
    if (share < INFINITY || least_weight > 0.0) {
        const double most = share * mass;
        typename Row<T>::Floor floor;
        if (least_weight > 0.0) {
            __syncthreads();
            if (threadIdx.x < 64) {
                const uint32_t end = key_of(-INFINITY);
                const uint32_t key = first_key(key_of(w.top), end, [&](uint32_t y) { return w.of(plain(logit_of(y))) < least_weight; });
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
    const double target = u * mass;
    const Range x = row.range_of({}, [&](bool, uint32_t c, double m) { return m > target || c >= kept; });
    const uint32_t last = (kept < x.before + x.count ? kept : x.before + x.count) - 1;
    double before;
    const int at = row.first_token(
        x, [&](uint32_t rank, double sum, double own) { return rank >= last || sum + own > target; }, before, weight);
    return {row.token_at(x, at), (float)(weight / mass)};
}

// The row's running counts and masses from its own counted bins or its parts'.
__device__ __forceinline__ void sum_bins(const Weights &w, float temperature, Shared &s, const PartBins *parts, int part_count) {
    constexpr int PER = BINS / THREADS;
    constexpr uint64_t SHARES = ((uint64_t)1 << SUM_BITS) - 1;
    uint32_t count[PER] = {}, tokens = 0;
    uint64_t share[PER] = {};
    const int first = threadIdx.x * PER;
    if (parts) {
        // A part's bins lie `on` further on, those of a part of no token past all. What falls past the last bin is known
        // from the tokens' number.
#pragma unroll 4
        for (int p = 0; p < part_count; p++) {
            const PartBins &x = parts[p];
            const int on = w.further(Weights(temperature, x.top));
            tokens += x.tokens;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int from = first + i - on;
                uint64_t v = x.bins[max(from, 0)];
                v = from >= 0 && first + i < BINS - 1 ? v : 0;
                count[i] += (uint32_t)(v >> SUM_BITS);
                share[i] += v & SHARES;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; i++) {
#pragma unroll
            for (int x = 0; x < COPIES; x++) {
                const uint64_t v = s.counted[(first + i) * COPIES + x];
                count[i] += (uint32_t)(v >> SUM_BITS);
                share[i] += v & SHARES;
            }
        }
    }
    // In units of the largest logit's own rounded weight: rows of one logit come out exactly.
    const uint64_t one = ((uint64_t)1 << 40) + Share()(w.place(w.top));
    const double unit = 0x1p-40 / ((double)one * 0x1p-40);
    running<PER>(
        s,
        [&](int i, uint32_t &c, double &m) {
            c = count[i - first];
            const uint64_t sum = ((uint64_t)c << 40) + share[i - first];
            m = i == BINS - 1 || !c ? 0.0 : i == 0 && sum == c * one ? (double)c : (double)sum * unit * exp2_64(i * (-1.0 / PER_OCTAVE));
        },
        [&](int i, uint32_t c, double m, double) { s.row.count[i] = parts && i == BINS - 1 ? tokens : c, s.row.mass[i] = m; });
    __syncthreads();
}

template <typename T, int HELD>
__global__ __launch_bounds__(THREADS) void sample_kernel(const SampleArgs a, const PartBins *parts, int part_count) {
    __shared__ Shared s;
    const int r = blockIdx.x;
    const Chosen o(a, r);
    const float uniform = a.uniforms[r];
    float top = -INFINITY;
    if constexpr (HELD == 0) {
        parts += (size_t)r * part_count;
        for (int p = threadIdx.x & 63; p < part_count; p += 64) top = fmaxf(top, parts[p].top);
        top = wave_max(top);
    }
    const Logits<T, HELD> logits(static_cast<const T *>(a.logits) + (int64_t)r * a.ld, a.n);
    if constexpr (HELD > 0) {
        for (int b = threadIdx.x; b < BINS * COPIES; b += THREADS) s.counted[b] = 0;
        logits.each([&](float l, int) { top = fmaxf(top, l); });
        top = wave_max(top);
        if ((threadIdx.x & 63) == 0) s.wave_top[threadIdx.x >> 6] = top;
        __syncthreads();
        top = wave_max(s.wave_top[threadIdx.x & (WAVES - 1)]);
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
        if constexpr (HELD > 0) {
            logits.each([&](float l, int i) { x = min(x, l == top ? i : INT32_MAX); });
        } else {
            int p = 0;
            while (parts[p].top != top) p++;
            for (int i = threadIdx.x; i < PART && p * PART + i < a.n && x == INT32_MAX; i += THREADS)
                if (plain((float)logits.row[p * PART + i]) == top) x = p * PART + i;
        }
        return answer(least(s, x), 1.0f);
    }
    const Weights w(o.temperature, top);
    if constexpr (HELD > 0) {
        const Share share;
        logits.each([&](float l, int) { w.count_in(l, s.counted, share); });
        __syncthreads();
    }
    sum_bins(w, o.temperature, s, HELD ? nullptr : parts, part_count);

    const uint32_t all = s.row.count[BINS - 1];
    const uint32_t k = o.top_k > 0 && (uint32_t)o.top_k < all ? (uint32_t)o.top_k : all;
    const bool cut_k = k < all, cut = o.top_p < 1.0f || o.min_p > 0.0f;
    const double u = (double)fminf(uniform, 0x1.fffffep-1f), share = o.top_p < 1.0f ? (double)o.top_p : INFINITY;
    const double least_weight = o.min_p;

    // The bins where the border of top_k lies, those where the next one can lie, given what stays before it, and those
    // where the token can lie.
    const auto count_to = [&](int b) { return b < 0 ? 0u : s.row.count[b]; };
    const auto mass_to = [&](int b) { return b < 0 ? 0.0 : s.row.mass[b]; };
    Span by_k{}, by_mass{}, drawn{};
    double low_mass = mass_to(BINS - 1), high_mass = low_mass;
    uint32_t low_kept = k, high_kept = k;
    if (cut_k) {
        by_k.low = by_k.high = s.row.first([&](int, uint32_t c, double) { return c > k; });
        low_mass = mass_to(by_k.low - 1), high_mass = mass_to(by_k.low);
    }
    const double low_k = low_mass, high_k = high_mass;
    if (cut) {
        int low_floor = BINS, high_floor = BINS;
        if (o.min_p > 0.0f) {  // the first bin below min_p, or the one before or after it where roundings decide
            const double past = fmaxf(-__log2f(o.min_p) * PER_OCTAVE, -4.0f);
            low_floor = past < BINS ? max((int)past - 1, 0) : BINS - 1;
            high_floor = past < BINS - 4 ? max((int)past + 3, 0) : BINS - 1;
        }
        s.row.first({k, share * low_k, low_floor}, {k, share * high_k, high_floor}, by_mass.low, by_mass.high);
        low_mass = mass_to(by_mass.low - 1), high_mass = mass_to(by_mass.high);
        low_kept = max(count_to(by_mass.low - 1), 1u), high_kept = min(count_to(by_mass.high), k);
    }
    s.row.first({low_kept - 1, u * low_mass, BINS}, {high_kept - 1, u * high_mass, BINS}, drawn.low, drawn.high);
    // Spans that overlap are one.
    const bool one_mass = !cut || by_mass.low <= drawn.high;
    if (one_mass) {
        if (cut) drawn.high = max(drawn.high, by_mass.high);
        by_mass = drawn;
    }
    const bool one_k = !cut_k || by_k.low <= by_mass.high;
    if (one_k) {
        if (cut_k) by_mass.high = max(by_mass.high, by_k.high);
        if (one_mass) drawn = by_mass;
        by_k = by_mass;
    }
    const auto place = [&](Span &x, int start) {
        x.start = start;
        x.before = count_to(x.low - 1);
        x.mass_before = mass_to(x.low - 1);
        x.count = (int)(count_to(x.high) - x.before);
    };
    place(drawn, 0);
    place(by_mass, one_mass ? 0 : drawn.count);
    place(by_k, one_k ? by_mass.start : by_mass.start + by_mass.count);
    const int listed = by_k.start + by_k.count;
    if (listed > LIST) {
        const Drawn x = step_by_step(logits.row, a.n, w, s, k, all, u, share, least_weight);
        return answer(x.token, x.prob);
    }
    gather(logits, w, s, drawn, by_mass, by_k, listed);
    const auto weight = [&](int i) { return w.of(logit_of((uint32_t)(s.list[i] >> 32))); };
    const auto mass_before = [&](const Span &x, int i) { return x.mass_before + (s.before[i] - s.before[x.start]); };
    const auto rank = [&](const Span &x, int i) { return x.before + (uint32_t)(i - x.start); };
    double mass = mass_to(BINS - 1);
    if (cut_k) mass = fmin(fmax(mass_before(by_k, by_k.start + (int)(k - by_k.before)), low_k), high_k);
    uint32_t kept = k;
    if (cut) {
        const double most = share * mass;
        const int i = by_mass.start + first_of(by_mass.count, [&](int i) {
            const uint32_t n = rank(by_mass, by_mass.start + i);
            return n > 0 && (n >= k || mass_before(by_mass, by_mass.start + i) >= most || weight(by_mass.start + i) < least_weight);
        });
        kept = rank(by_mass, i);
        mass = i == by_mass.start ? by_mass.mass_before : mass_before(by_mass, i - 1) + weight(i - 1);
        mass = fmin(fmax(mass, low_mass), high_mass);
    }
    const double target = u * mass;
    const uint32_t last = min(kept, drawn.before + (uint32_t)drawn.count) - 1;
    const int i = first_of(drawn.count, [&](int i) { return rank(drawn, i) >= last || mass_before(drawn, i) + weight(i) > target; });
    answer((int)(uint32_t)s.list[i], (float)(weight(i) / mass));
}

// The bins of a part of a row: its logits stay in registers from the largest to the weights.
template <typename T>
__global__ __launch_bounds__(PART_THREADS) void parts_kernel(const SampleArgs a, PartBins *parts, int part_count) {
    constexpr int PIECE = 16 / sizeof(T), PIECES = PART_VALUES / PIECE, PART_WAVES = PART_THREADS / 64;
    __shared__ __align__(16) uint64_t bins[BINS * COPIES];
    __shared__ float tops[PART_WAVES];
    __shared__ uint32_t tokens;
    const int r = blockIdx.x / part_count, p = blockIdx.x % part_count;
    PartBins &out = parts[blockIdx.x];
    const Chosen o(a, r);
    const T *logits = static_cast<const T *>(a.logits) + (int64_t)r * a.ld + (int64_t)p * PART;
    const int n = min(a.n - p * PART, PART);
    float l[PIECES][PIECE];
    float top = -INFINITY;
    load(logits, 0, n, l, [](int x) { return (x * PART_THREADS + (int)threadIdx.x) * PIECE; });
    for (int b = threadIdx.x; b < BINS * COPIES; b += PART_THREADS) bins[b] = 0;
    if (threadIdx.x == 0) tokens = 0;
#pragma unroll
    for (int x = 0; x < PIECES; x++)
#pragma unroll
        for (int y = 0; y < PIECE; y++) top = fmaxf(top, l[x][y]);  // NaN is passed over
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int x = 0; x < PART_WAVES; x++) top = fmaxf(top, tops[x]);
    if (!(top > -INFINITY) || o.greedy()) {
        if (threadIdx.x == 0) out.top = top, out.tokens = 0;
        return;
    }
    const Weights w(o.temperature, top);
    const Share share;
#pragma unroll
    for (int x = 0; x < PIECES; x++)
#pragma unroll
        for (int y = 0; y < PIECE; y++)
            if (l[x][y] > -INFINITY) w.count_in(l[x][y], bins, share);
    __syncthreads();
    uint32_t mine = 0;
    for (int b = threadIdx.x; b < BINS; b += PART_THREADS) {
        uint64_t v = 0;
        for (int x = 0; x < COPIES; x++) v += bins[b * COPIES + x];
        mine += (uint32_t)(v >> SUM_BITS);
        out.bins[b] = v;
    }
    for (int x = 32; x; x >>= 1) mine += __shfl_xor(mine, x);
    if ((threadIdx.x & 63) == 0) atomicAdd(&tokens, mine);
    __syncthreads();
    if (threadIdx.x == 0) out.top = top, out.tokens = tokens;
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
            hipLaunchKernelGGL((sample_kernel<T, 0>), dim3((unsigned)rows), dim3(THREADS), 0, s, a, (const PartBins *)parts, count);
        } else {
            const auto kernel = a.n <= SHORT_VALUES * THREADS ? sample_kernel<T, SHORT_VALUES> : sample_kernel<T, WHOLE_VALUES>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(THREADS), 0, s, a, (const PartBins *)nullptr, 0);
        }
        return hipGetLastError();
    };
    switch (type) {
        case F16: return launch(_Float16{});
        case BF16: return launch(__bf16{});
        default: return launch(float{});
    }
}

}  // namespace tg
