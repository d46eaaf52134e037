// tgbm_scores_sample: a class of every row, drawn from its scores by a random number that is given.
//
// The classes of a row in order, the best first and of equal scores the lower class: w = exp((score - best) / T) of each. Every cut keeps a front part of that
// order, and so the class that is drawn is the one where the sum of w passes u times the sum of what is kept. A sum over all classes decides which of two
// classes it is, so everything is 64 bits, and what many threads add up is added as whole numbers, whose sum has no order.
//
// 2048 x 65537 bfloat16 cut at a mass of 0.9: 248 us where the memory's share is 53. 47 vector instructions of a wavefront to a score of each lane, 18 of them its
// weight and place in 64 bits, take two thirds of that; the row is gone over four times (largest score, weights, cut, draw), behind the first from the last cache.
// 50000 x 1000: 195 us (39), 200000 x 100: 204 (16): about 1000 and 600 instructions of a row that its length has no part in. 256 x 128003 bfloat16 with settings of each row: 122 us (13).
// Rows of equal scores are one bucket's, and all of their additions go to one place: 1305 us for 50000 x 1000, 9.7 ms for 2048 x 65537, 3.6 for 1 x 128003.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "kernel_common.h"
#include "score_rules.h"

namespace tgbm {
namespace {

constexpr int kSampleBlock = 256;
typedef float Float4 __attribute__((ext_vector_type(4), aligned(4)));
constexpr float kNothing = -__builtin_inff();
constexpr float kGreedyBelow = 1e-6f;  // temperatures below take the best class
constexpr float kLargestBelowOne = 0x1.fffffep-1f;

// Scores in the order of unsigned integers, the two zeros being equal. No NaN comes here.
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(unsigned o) { return __uint_as_float(o ^ ((o >> 31) - 1u | 0x80000000u)); }
// A NaN is left out like -infinity.
__device__ __forceinline__ float without_nan(float v) { return fmaxf(v, kNothing); }

// What a row is drawn by.
struct RowSampling {
    float temperature, p, min_p, u;
    int k;        // INT_MAX: all
    bool greedy;  // the best class
    bool none;    // a number is NaN: no class
};
__device__ __forceinline__ RowSampling sampling_of(const tgbm_sampling &how, const float *u, long row) {
    RowSampling r;
    const float t = how.temperature != nullptr ? how.temperature[row] : how.temperature_all;
    const float p = how.p != nullptr ? how.p[row] : how.p_all;
    const float m = how.min_p != nullptr ? how.min_p[row] : how.min_p_all;
    const int k = how.k != nullptr ? how.k[row] : how.k_all;
    const float v = u[row];
    r.none = t != t || p != p || m != m || v != v;
    r.greedy = t < kGreedyBelow;
    r.temperature = r.greedy ? 1.f : fminf(t, 1e6f);
    r.p = p;
    r.min_p = fminf(fmaxf(m, 0.f), 1.f);
    r.u = fminf(fmaxf(v, 0.f), kLargestBelowOne);
    r.k = k <= 0 ? INT_MAX : k;
    return r;
}

// ------------------------------------------------------------------------------------------------------- few classes
// A thread holds its row's classes and puts them in order by a network of exchanges (Batcher's odd-even merge sort: 19 of 8, 63 of 16, 191 of 32). 500000 x 8: 18 us
// where every class was compared with every other one.
template <int E>
__device__ __forceinline__ void sort_down(unsigned long long (&key)[E]) {
#pragma unroll
    for (int p = 1; p < E; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < E; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < E && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const unsigned long long a = key[i + j], b = key[i + j + k];
                        const bool turn = a < b;
                        key[i + j] = turn ? b : a;
                        key[i + j + k] = turn ? a : b;
                    }
}
template <typename T, int E>
__global__ __launch_bounds__(kSampleBlock) void k_sample_few(tgbm_scores in, tgbm_score_rules rules, tgbm_sampling how, const float *u, int *classes, float *logp) {
    const long row = (long)blockIdx.x * kSampleBlock + threadIdx.x;
    if (row >= in.rows) return;
    const RowSampling r = sampling_of(how, u, row);
    const T *src = static_cast<const T *>(in.data) + (size_t)row * in.row_stride;
    float v[E];
#pragma unroll
    for (int c = 0; c < E; ++c) v[c] = c < in.classes ? score_to_float(src[(size_t)c * in.class_stride]) : kNothing;
    if (rules.bias != nullptr || rules.allowed != nullptr || rules.shown != nullptr) {
        unsigned times[E];
#pragma unroll
        for (int c = 0; c < E; ++c) times[c] = 0;
        if (rules.shown != nullptr) {
            long long b, e;
            shown_range(rules, row, &b, &e);
            for (long long i = b; i < e; i += 8) {  // (one by one every entry would be waited for: 64 x 23 with 300 shown classes a row, 206 us)
                int shown[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) shown[q] = i + q < e ? rules.shown[i + q] : -1;
#pragma unroll
                for (int q = 0; q < 8; ++q)
#pragma unroll
                    for (int c = 0; c < E; ++c) times[c] += shown[q] == c ? 1u : 0u;
            }
        }
        bool none;
        const unsigned *words = allowed_words(rules, row, 1, &none);
        const unsigned ok = none ? 0u : words != nullptr ? words[0] : ~0u;
#pragma unroll
        for (int c = 0; c < E; ++c)
            if (c < in.classes) v[c] = adjusted(v[c], rules.bias != nullptr ? rules.bias[c] : 0.f, times[c], ok >> c & 1u, rules);
    }
    unsigned long long key[E];
#pragma unroll
    for (int c = 0; c < E; ++c) key[c] = (unsigned long long)ordered(without_nan(v[c])) << 32 | (unsigned)~c;
    sort_down<E>(key);
    const float m = from_ordered((unsigned)(key[0] >> 32));
    if (m == kNothing || r.none) {
        classes[row] = -1;
        logp[row] = r.none ? __builtin_nanf("") : kNothing;
        return;
    }
    const double by = 1.0 / (double)r.temperature;
    const int k = r.greedy ? 1 : r.k;
    double w[E], sum = 0;
#pragma unroll
    for (int c = 0; c < E; ++c) {
        const float x = from_ordered((unsigned)(key[c] >> 32));
        const double e = x == m ? 1.0 : exp(((double)x - (double)m) * by);
        w[c] = x > kNothing && c < k && e >= (double)r.min_p ? e : 0.0;
        sum += w[c];
    }
    double kept = sum;
    if (r.p < 1.f) {
        const double most = (double)r.p * sum;
        double front = 0;
        kept = 0;
#pragma unroll
        for (int c = 0; c < E; ++c) {
            const double its = w[c];
            if (c > 0 && !(front < most)) w[c] = 0;
            front += its;
            kept += w[c];
        }
    }
    const double target = (double)r.u * kept;
    double front = 0, its = 0;
    int drawn = -1;
#pragma unroll
    for (int c = 0; c < E; ++c) {
        if (w[c] > 0 && front <= target) {
            drawn = (int)~(unsigned)key[c];
            its = w[c];
        }
        front += w[c];
    }
    classes[row] = drawn;
    logp[row] = r.greedy ? 0.f : (float)log(its / kept);
}

// ------------------------------------------------------------------------------------------------------- from a list
// Rows whose best classes are listed in order, as top leaves them, up to 128 of a row.
// (of all lanes: one that does not take part hands nothing on)
struct WaveSumD {
    double v;
    template <int CTRL, int ROWS>
    __device__ __forceinline__ void at() { v += __longlong_as_double(dpp_ll<CTRL, ROWS>(__double_as_longlong(v))); }
};
__device__ __forceinline__ double wave_scan_d(double v) {  // inclusive
    WaveSumD s{v};
    wave_scan_steps(s);
    return s.v;
}
__device__ __forceinline__ double from_below_d(double v) { return __longlong_as_double(dpp_ll<kDppWaveShr1>(__double_as_longlong(v))); }  // (0 in lane 0)
__device__ __forceinline__ double read_lane_d(double v, int lane) { return __longlong_as_double(read_lane_ll(__double_as_longlong(v), lane)); }
// L lanes to a row, whose scores are in order: two that follow one another to each lane, -infinity behind the last. class_of(i): of the lane's.
template <int L, typename Class>
__device__ __forceinline__ void draw_ordered(const float (&x)[2], const RowSampling &r, bool on, Class class_of, int *cls, float *logp) {
    const int lane = lane_id() % L, first_lane = lane_id() / L * L;
    const float m = __shfl(x[0], first_lane);
    const double by = 1.0 / (double)r.temperature;
    double w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const double e = x[i] == m ? 1.0 : exp(((double)x[i] - (double)m) * by);
        w[i] = x[i] > kNothing && e >= (double)r.min_p && 2 * lane + i < (r.greedy ? 1 : r.k) ? e : 0.0;
    }
    WaveSumD scan{w[0] + w[1]};
    scan.at<kDppRowShr + 1, 0xf>();
    scan.at<kDppRowShr + 2, 0xf>();
    scan.at<kDppRowShr + 4, 0xf>();
    scan.at<kDppRowShr + 8, 0xf>();
    if constexpr (L >= 32) scan.at<kDppBcast15, 0xa>();
    if constexpr (L == 64) scan.at<kDppBcast31, 0xc>();
    const double upto1 = scan.v, below = from_below_d(upto1), front0 = lane == 0 ? 0.0 : below, front1 = front0 + w[0];
    const auto of_lane = [&](double d, int l) { return __longlong_as_double(((long long)__shfl((int)(__double_as_longlong(d) >> 32), first_lane + l) << 32) |
                                                                           (unsigned)__shfl((int)(unsigned)__double_as_longlong(d), first_lane + l)); };
    const auto last_of = [&](bool is) {  // the row's last lane where it is so, -1: there is none
        const unsigned long long who = __ballot(is) >> first_lane & (L == 64 ? ~0ull : (1ull << L % 64) - 1);
        return 63 - (who != 0 ? __clzll((long long)who) : 64);
    };
    double kept = of_lane(upto1, L - 1);
    if (r.p < 1.f) {  // (all lanes of a row, but not all rows: what they read of each other is the row's own)
        const double most = (double)r.p * kept;
        const int last0 = max(0, last_of(w[0] > 0 && (front0 < most || lane == 0))), last1 = last_of(w[1] > 0 && front1 < most);
        // the sum up to the last one that is kept
        const double even = of_lane(front1, last0), odd = of_lane(upto1, last0);
        kept = last1 == last0 ? odd : even;
    }
    const double target = (double)r.u * kept;
    const int l0 = max(0, last_of(w[0] > 0 && (front0 <= target || lane == 0))), l1 = last_of(w[1] > 0 && front1 <= target);
    const int l = l0 > l1 ? l0 : l1, i = l1 == l ? 1 : 0;
    if (!on || lane != l) return;
    if (m == kNothing || r.none) {
        *cls = -1;
        *logp = r.none ? __builtin_nanf("") : kNothing;
    } else {
        *cls = class_of(i);
        *logp = r.greedy ? 0.f : (float)log((i ? w[1] : w[0]) / kept);
    }
}
template <int L>
__global__ __launch_bounds__(kSampleBlock) void k_sample_listed(const float *values, const int *listed, int k, int rows, tgbm_sampling how, const float *u, int *classes,
                                                                float *logp) {
    const long at_row = (long)blockIdx.x * (kSampleBlock / L) + threadIdx.x / L;
    const bool on = at_row < rows;  // (all lanes stay: one that does not take part hands nothing on)
    const long row = on ? at_row : rows - 1;
    const int lane = lane_id() % L;
    float x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = 2 * lane + i < k ? values[(size_t)row * k + 2 * lane + i] : kNothing;
    draw_ordered<L>(x, sampling_of(how, u, row), on, [&](int i) { return listed[(size_t)row * k + 2 * lane + i]; }, classes + row, logp + row);
}

// A wavefront's row of up to 128 classes, put in order by a bitonic sort, two that follow one another to a lane at the end.
constexpr int kSorted = 128;
__device__ __forceinline__ unsigned long long shfl_xor_u64(unsigned long long v, int mask) {
    return (unsigned long long)(unsigned)__shfl_xor((int)(v >> 32), mask) << 32 | (unsigned)__shfl_xor((int)(unsigned)v, mask);
}
__device__ __forceinline__ void sort_wave_down(unsigned long long (&key)[2]) {
    const int lane = lane_id();
#pragma unroll
    for (int run = 2; run <= kSorted; run *= 2) {
        const bool down = (2 * lane & run) == 0;  // (run 128: all)
#pragma unroll
        for (int d = run / 2; d >= 2; d /= 2) {
            const bool lower = (lane & d / 2) == 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const unsigned long long other = shfl_xor_u64(key[i], d / 2);
                key[i] = (other > key[i]) == (lower == down) ? other : key[i];
            }
        }
        const bool turn = (key[1] > key[0]) == down;
        const unsigned long long a = turn ? key[1] : key[0], b = turn ? key[0] : key[1];
        key[0] = a;
        key[1] = b;
    }
}
__device__ __forceinline__ void draw_sorted(const float *scores, int n, const RowSampling &r, int *cls, float *logp) {
    unsigned long long key[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = lane_id() + 64 * i;
        key[i] = c < n ? (unsigned long long)ordered(without_nan(scores[c])) << 32 | (unsigned)~c : 0;
    }
    sort_wave_down(key);
    // (what is no class has the least key, which is no score's)
    const float x[2] = {key[0] != 0 ? from_ordered((unsigned)(key[0] >> 32)) : kNothing, key[1] != 0 ? from_ordered((unsigned)(key[1] >> 32)) : kNothing};
    draw_ordered<64>(x, r, true, [&](int i) { return (int)~(unsigned)key[i]; }, cls, logp);
}

// ------------------------------------------------------------------------------------------------------- any rows
// Rows' adjusted scores as 32-bit numbers, classes side by side: what goes by other ways than a row's own scores (classes that were shown, rows side by
// side). A tile of 64 x 64.
constexpr int kLaid = 64;
template <typename T>
__global__ __launch_bounds__(kSampleBlock) void k_lay_out(tgbm_scores in, tgbm_score_rules rules, float *out, long pitch) {
    __shared__ float tile[kLaid][kLaid + 1];
    const long row0 = (long)blockIdx.y * kLaid;
    const int c0 = (int)blockIdx.x * kLaid, lane = lane_id();
    const bool columns = in.row_stride == 1 && in.class_stride != 1;
    for (int i = wave_id(); i < kLaid; i += kSampleBlock / 64) {
        const long row = columns ? row0 + lane : row0 + i;
        const int c = columns ? c0 + i : c0 + lane;
        float s = kNothing;
        if (row < in.rows && c < in.classes) s = score_to_float(static_cast<const T *>(in.data)[(size_t)c * in.class_stride + (size_t)row * in.row_stride]);
        tile[columns ? lane : i][columns ? i : lane] = s;
    }
    __syncthreads();
    for (int i = wave_id(); i < kLaid; i += kSampleBlock / 64) {
        const long row = row0 + i;
        const int c = c0 + lane;
        if (row >= in.rows || c >= in.classes) continue;
        bool none;
        const unsigned *words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
        const bool ok = !none && (words == nullptr || (words[c / 32] >> (c % 32) & 1u));
        out[(size_t)row * pitch + c] = adjusted(tile[i][lane], rules.bias != nullptr ? rules.bias[c] : 0.f, 0, ok, rules);
    }
}
// The classes that a row was shown: counted in LDS, kShownClasses of them at a time, and whoever takes a count away stores.
constexpr int kShownClasses = 8192;
template <typename T>
__global__ __launch_bounds__(kSampleBlock) void k_lay_shown(tgbm_scores in, tgbm_score_rules rules, float *out, long pitch) {
    __shared__ unsigned times[kShownClasses];
    const long row = blockIdx.x;
    const int c0 = (int)blockIdx.y * kShownClasses, size = min(in.classes - c0, kShownClasses);
    long long b, e;
    shown_range(rules, row, &b, &e);
    if (b >= e) return;
    auto each = [&](auto f) {
        for (long long i = b + threadIdx.x; i < e; i += kSampleBlock) {
            const int c = rules.shown[i] - c0;
            if ((unsigned)c < (unsigned)size) f(c);
        }
    };
    each([&](int c) { times[c] = 0; });
    __syncthreads();
    each([&](int c) { atomicAdd(&times[c], 1u); });
    __syncthreads();
    bool none;
    const unsigned *words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
    each([&](int i) {
        const unsigned n = atomicExch(&times[i], 0u);
        if (n == 0) return;
        const int c = c0 + i;
        const bool ok = !none && (words == nullptr || (words[c / 32] >> (c % 32) & 1u));
        const float s = score_to_float(static_cast<const T *>(in.data)[(size_t)c * in.class_stride + (size_t)row * in.row_stride]);
        out[(size_t)row * pitch + c] = adjusted(s, rules.bias != nullptr ? rules.bias[c] : 0.f, n, ok, rules);
    });
}

// A score's place on the scale that sums are kept by: P parts to a halving of w, 64 halvings; its bucket is the nearest whole number. What is further down than that
// (2^-64 of the best class) is nothing beside a random number's last place, 2^-24, whatever there is of it.
template <int P>
struct Scale {
    static constexpr int kBuckets = 64 * P;
    static constexpr double kOfE = P * 1.44269504088896340736;  // parts to a factor of e
};
constexpr double kToWhole = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the nearest whole number

// 2^(-h / P), h in [-1/2, 1/2], plus `magic` = 2^(52 - bits): its last 52 bits are the power of two times 2^bits, rounded. Taylor's series, up to where the next term
// is below 2^-48 of the whole; 2^-46 is what a whole number of a row of 2^16 classes is rounded by (weight_bits).
template <int P>
__device__ __forceinline__ unsigned long long part_of_two(double h, double magic) {
    constexpr double a = -0.69314718055994530942 / P, c2 = a * a / 2, c3 = c2 * a / 3, c4 = c3 * a / 4, c5 = c4 * a / 5, c6 = c5 * a / 6, c7 = c6 * a / 7;
    static_assert(P == 32 || P == 8);
    double e = P == 32 ? __builtin_fma(h, c5, c4) : __builtin_fma(h, __builtin_fma(h, __builtin_fma(h, c7, c6), c5), c4);
    e = __builtin_fma(h, e, c3);
    e = __builtin_fma(h, e, c2);
    e = __builtin_fma(h, e, a);
    e = __builtin_fma(h, e, 1.0);
    return (unsigned long long)__double_as_longlong(e + magic) & 0xfffffffffffffull;
}

// What is shared by the G threads that work on a row, a workgroup or a wavefront of several.
template <int G>
constexpr int parts_of() { return G == 64 ? 8 : 32; }
template <int G>
constexpr int listed_of() { return G == 64 ? 64 : 256; }
template <int G>
constexpr int chosen_of() { return G == 64 ? 1 : G == 256 ? 512 : 2048; }
template <int G>
struct alignas(16) DrawShared {
    unsigned long long chosen[chosen_of<G>()];
    unsigned long long mass[Scale<parts_of<G>()>::kBuckets + 1];  // (the last one takes what does not count)
    unsigned long long key[listed_of<G>()], weight[listed_of<G>()], front[listed_of<G>()];
    double part[G / 64];
    float part_f[G / 64];
    int part_i[G / 64];
    unsigned long long best, least, most;
    int listed, count;
};
template <int G>
__device__ __forceinline__ void group_sync() {
    if constexpr (G == 64) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    else __syncthreads();
}
template <int G>
__device__ __forceinline__ int in_group() { return G == 64 ? lane_id() : (int)threadIdx.x; }

// A group's work on a row. Row: row.each(f) calls f(scores, their first class) for the thread's vectors; what is no class is -infinity there, NaNs stay what they
// are and are to be let fall by comparisons.
template <int G, typename Row>
struct Draw {
    static constexpr int V = Row::V, P = parts_of<G>(), kBuckets = Scale<P>::kBuckets, kEach = kBuckets / G, kListed = listed_of<G>();
    DrawShared<G> &sh;
    Row &row;
    double best, by, step;  // (the place of a score is (best - score) * by; step: 1 / by)
    double magic;
    float least = -FLT_MAX;      // the least score that is kept
    unsigned long long cut = 0;  // the last one of the order that is kept, as a key
    double last_place = kBuckets - 0.5;

    static __device__ __forceinline__ unsigned long long key_of(float x, int c) { return (unsigned long long)ordered(x) << 32 | (unsigned)~c; }
    __device__ __forceinline__ double place_of(float x) const { return (best - (double)x) * by; }
    static __device__ __forceinline__ int bucket_of(double place) { return (int)__double_as_longlong(place + kToWhole); }
    __device__ __forceinline__ unsigned long long weight_of(double place) const { return part_of_two<P>(place - ((place + kToWhole) - kToWhole), magic); }
    // A score below which none has a place up to `place`; the other way: above which none has one from there on.
    __device__ __forceinline__ float score_below(double place) const {
        const double x = best - place * step;
        return __double2float_rd(x - 0x1p-49 * (fabs(x) + fabs(best)));
    }
    __device__ __forceinline__ float score_above(double place) const {
        const double x = best - place * step;
        return __double2float_ru(x + 0x1p-49 * (fabs(x) + fabs(best)));
    }
    int chosen = -1;  // how many there are, once all that is kept lies in the list of them

    // Lists all that is kept and whose score is `bound` or more, if there is room for them. A row of 128003 classes is gone over six times where a count and a mass cut it,
    // two or three times with the list.
    __device__ __forceinline__ void choose(float bound) {
        if (G == 64 || chosen >= 0) return;
        bound = fmaxf(bound, least);
        group_sync<G>();
        if (in_group<G>() == 0) sh.count = 0;
        group_sync<G>();
        row.each([&](const float (&x)[V], int c) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < V; ++j) any |= x[j] >= bound;
            if (!__any(any)) return;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const unsigned long long who = __ballot(x[j] >= bound);
                if (who == 0) continue;
                const int first = __ffsll((long long)who) - 1;
                int to = 0;
                if (lane_id() == first) to = atomicAdd(&sh.count, __popcll(who));
                to = read_lane(to, first) + lanes_below(who);
                if (x[j] >= bound && to < chosen_of<G>()) sh.chosen[to] = key_of(x[j], c + j);
            }
        });
        group_sync<G>();
        const int n = sh.count;
        chosen = n <= chosen_of<G>() ? n : -1;
        least = chosen >= 0 ? bound : least;
    }
    // f(place, bucket, key) for those that are kept and whose score is from lo to hi
    template <typename F>
    __device__ __forceinline__ void kept(float lo, float hi, F f) {
        lo = fmaxf(lo, least);
        if (G > 64 && chosen >= 0) {
            for (int i = in_group<G>(); i < chosen; i += G) {
                const unsigned long long key = sh.chosen[i];
                const float x = from_ordered((unsigned)(key >> 32));
                if (x >= lo && x <= hi && key >= cut) {
                    const double s = place_of(x);
                    if (s <= last_place) f(s, bucket_of(s), key);
                }
            }
            return;
        }
        row.each([&](const float (&x)[V], int c) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < V; ++j) any |= x[j] >= lo && x[j] <= hi;
            if (!any) return;
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (x[j] >= lo && x[j] <= hi) {
                    const double s = place_of(x[j]);
                    const unsigned long long key = key_of(x[j], c + j);
                    if (s <= last_place && key >= cut) f(s, bucket_of(s), key);
                }
        });
    }

    // Exclusive sums over the threads, in their order, and the sum of all.
    __device__ __forceinline__ double scan(double v, double *all) {
        const double upto = wave_scan_d(v);
        if constexpr (G == 64) {
            *all = read_lane_d(upto, 63);
            return from_below_d(upto);
        }
        group_sync<G>();
        if (lane_id() == 63) sh.part[wave_id()] = upto;
        group_sync<G>();
        double before = 0, sum = 0;
#pragma unroll
        for (int w = 0; w < G / 64; ++w) {
            if (w == wave_id()) before = sum;
            sum += sh.part[w];
        }
        *all = sum;
        return before + from_below_d(upto);
    }
    __device__ __forceinline__ void clear() {
        group_sync<G>();
        for (int i = in_group<G>(); i < kBuckets; i += G) sh.mass[i] = 0;
        clear_list();
    }
    __device__ __forceinline__ void clear_list() {
        group_sync<G>();
        if (in_group<G>() == 0) {
            sh.listed = 0;
            sh.best = 0;
            sh.least = ~0ull;
            sh.most = 0;
        }
        group_sync<G>();
    }

    // Whether the order up to `before` leaves the next one in what is looked for: up to a target, or below it.
    static __device__ __forceinline__ bool within(double before, double target, bool below) { return below ? before < target : before <= target; }

    // The buckets' sums, those in front of the thread's, and the sum of all. first, ratio: what the whole numbers of the thread's first bucket count, and each
    // bucket's next to the one before.
    __device__ __forceinline__ double sums(double first, double ratio, double (&mass)[kEach], double *all) {
        double mine = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            mass[i] = (double)sh.mass[in_group<G>() * kEach + i] * first;
            first *= ratio;
            mine += mass[i];
        }
        return scan(mine, all);
    }
    // The bucket where the sum passes the target, and the sum in front of it (the first one, where roundings leave none).
    __device__ __forceinline__ void find(const double (&mass)[kEach], double before, double target, bool below, int *bucket, double *front) {
        int at = -1;
        double its = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (mass[i] > 0 && within(before, target, below)) {
                at = in_group<G>() * kEach + i;
                its = before;
            }
            before += mass[i];
        }
        const unsigned long long who = __ballot(at >= 0);
        const int lane = who != 0 ? 63 - __clzll((long long)who) : 0;
        at = read_lane(at, lane);
        its = read_lane_d(its, lane);
        if constexpr (G > 64) {
            group_sync<G>();
            if (lane_id() == 0) {
                sh.part_i[wave_id()] = at;
                sh.part[wave_id()] = its;
            }
            group_sync<G>();
#pragma unroll
            for (int w = 0; w < G / 64; ++w)
                if (const int other = sh.part_i[w]; other >= 0) {
                    at = other;
                    its = sh.part[w];
                }
            group_sync<G>();
        }
        *bucket = __builtin_amdgcn_readfirstlane(at >= 0 ? at : 0);
        *front = at >= 0 ? its : 0.0;
    }

    struct Found {
        unsigned long long key;
        double before, weight;  // in the bucket's unit
    };
    static constexpr int kKeyBits = P == 32 ? 11 : 9;
    // The one of a bucket where its sum passes the target (in its unit). weight(place): of one.
    template <typename Weight>
    __device__ __forceinline__ Found resolve(int bucket, double target, bool below, Weight weight) {
        const float low = score_below(bucket + 0.5), high = score_above(bucket - 0.5);
        unsigned long long lo = 0, hi = ~0ull;
        double front = 0;
        for (;;) {
            clear_list();
            kept(low, high, [&](double s, int b, unsigned long long key) {
                if (b != bucket || key < lo || key > hi) return;
                const int to = atomicAdd(&sh.listed, 1);
                if (to < kListed) {
                    sh.key[to] = key;
                    sh.weight[to] = weight(s);
                    sh.front[to] = 0;
                }
            });
            group_sync<G>();
            const int n = sh.listed;
            if (n <= kListed) return among(n, front, target, below);
            // too many for a list: by parts of the keys between the least and the largest of them
            kept(low, high, [&](double, int b, unsigned long long key) {
                if (b != bucket || key < lo || key > hi) return;
                atomicMin(&sh.least, key);
                atomicMax(&sh.most, key);
            });
            group_sync<G>();
            lo = sh.least;
            hi = sh.most;
            const int width = 64 - __clzll((long long)(hi - lo)), shift = width > kKeyBits ? width - kKeyBits : 0;
            static_assert(kBuckets == 1 << kKeyBits);
            clear();
            kept(low, high, [&](double s, int b, unsigned long long key) {
                if (b == bucket && key >= lo && key <= hi) atomicAdd(&sh.mass[(hi - key) >> shift], weight(s));
            });
            group_sync<G>();
            double mass[kEach], all;
            const double before = sums(1.0, 1.0, mass, &all);
            int part;
            double its;
            find(mass, front + before, target, below, &part, &its);
            front = part == 0 ? front : its;
            hi -= (unsigned long long)part << shift;
            const unsigned long long span = (1ull << shift) - 1;
            lo = hi - lo > span ? hi - span : lo;
        }
    }
    // The same among n listed ones, which are put in order by what is in front of each.
    __device__ __forceinline__ Found among(int n, double front, double target, bool below) {
        constexpr int kShares = G / kListed;
        const int share = in_group<G>() / kListed;
        if (const int j = in_group<G>() % kListed; j < n) {
            const unsigned long long mine = sh.key[j];
            unsigned long long sum = 0;
            for (int o = share; o < n; o += kShares) sum += sh.key[o] > mine ? sh.weight[o] : 0ull;
            atomicAdd(&sh.front[j], sum);
        }
        group_sync<G>();
        // (the first one always is; a larger sum in front comes later in the order, and no two are equal)
        for (int j = in_group<G>(); j < n; j += G)
            if (sh.front[j] != 0 && within(front + (double)sh.front[j], target, below)) atomicMax(&sh.best, sh.front[j]);
        group_sync<G>();
        const unsigned long long its = sh.best;
        for (int j = in_group<G>(); j < n; j += G)
            if (sh.front[j] == its) sh.listed = j;
        group_sync<G>();
        const int j = sh.listed;
        return Found{sh.key[j], front + (double)its, (double)sh.weight[j]};
    }

    // Leaves the k best. The k-th of the threads' own best scores is a bound: only what reaches it is looked at one by one.
    __device__ __forceinline__ void keep_best(int k, float mine) {
        double mass[kEach], all, front;
        int bucket;
        float bound = least;
        if (k <= G) {
            clear();
            if (mine >= least && place_of(mine) <= last_place) atomicAdd(&sh.mass[bucket_of(place_of(mine))], 1ull);
            group_sync<G>();
            const double before = sums(1.0, 1.0, mass, &all);
            if (all >= (double)k) {
                find(mass, before, (double)(k - 1), false, &bucket, &front);
                bound = fmaxf(bound, score_below(bucket + 0.5));
                choose(bound);
            }
        }
        clear();
        kept(bound, __builtin_inff(), [&](double, int b, unsigned long long) { atomicAdd(&sh.mass[b], 1ull); });
        group_sync<G>();
        const double before = sums(1.0, 1.0, mass, &all);
        if (all <= (double)k) {  // (all that reach the bound: it is the cut)
            least = bound;
            return;
        }
        find(mass, before, (double)(k - 1), false, &bucket, &front);
        const unsigned long long key = resolve(bucket, (double)(k - 1) - front, false, [](double) { return 1ull; }).key;
        cut = key;
        least = from_ordered((unsigned)(key >> 32));
    }
    // The weights of what is kept, into the buckets.
    __device__ __forceinline__ void add_up(bool all_kept) {
        clear();
        if (!all_kept) {
            kept(least, __builtin_inff(), [&](double s, int b, unsigned long long) { atomicAdd(&sh.mass[b], weight_of(s)); });
        } else {
            row.each([&](const float (&x)[V], int) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const double s = __builtin_fmin(place_of(x[j]), (double)kBuckets), at = s + kToWhole;
                    atomicAdd(&sh.mass[(int)__double_as_longlong(at)], part_of_two<P>(s - (at - kToWhole), magic));
                }
            });
        }
        group_sync<G>();
    }
};

template <int G>
__device__ __forceinline__ float block_max(float v, float *part) {
    v = wave_max_f(v);
    if constexpr (G == 64) return v;
    group_sync<G>();
    if (lane_id() == 0) part[wave_id()] = v;
    group_sync<G>();
#pragma unroll
    for (int w = 0; w < G / 64; ++w) v = fmaxf(v, part[w]);
    return v;
}
template <int G>
__device__ __forceinline__ int block_min(int v, int *part) {
    v = wave_min_i(v);
    if constexpr (G == 64) return v;
    group_sync<G>();
    if (lane_id() == 0) part[wave_id()] = v;
    group_sync<G>();
#pragma unroll
    for (int w = 0; w < G / 64; ++w) v = min(v, part[w]);
    return v;
}
template <int G>
__device__ __forceinline__ int block_sum(int v, int *part) {
    v = wave_sum_i(v);
    if constexpr (G == 64) return v;
    group_sync<G>();
    if (lane_id() == 0) part[wave_id()] = v;
    group_sync<G>();
    v = 0;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) v += part[w];
    return v;
}

template <int G>
__device__ __forceinline__ float block_sum_f(float v, float *part) {
    for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
    group_sync<G>();
    if (lane_id() == 0) part[wave_id()] = v;
    group_sync<G>();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) v += part[w];
    return v;
}

// The class of the n-th (from 0) score that is m, by bisection.
template <int G, typename Row>
__device__ __forceinline__ int nth_class(Row &row, float m, int n, int classes, int *part) {
    int lo = -1, hi = classes - 1;
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        int count = 0;
        row.each([&](const float (&x)[Row::V], int c) {
#pragma unroll
            for (int j = 0; j < Row::V; ++j) count += x[j] == m && c + j <= mid ? 1 : 0;
        });
        if (block_sum<G>(count, part) > n) hi = mid;
        else lo = mid;
    }
    return hi;
}

// A row's draw, its largest score being m, a number. False: min_p cuts.
template <int G, typename Row>
__device__ __forceinline__ bool begin_draw(Draw<G, Row> &d, const RowSampling &r, float m, int bits) {
    d.best = (double)m;
    constexpr int P = parts_of<G>();
    d.by = Scale<P>::kOfE / (double)r.temperature;
    d.step = (double)r.temperature * (1.0 / Scale<P>::kOfE);
    d.magic = __longlong_as_double((long long)(1023 + 52 - bits) << 52);
    if (r.min_p == 0.f) return true;
    d.last_place = fmin(d.last_place, -log2((double)r.min_p) * P);
    d.least = fmaxf(d.least, d.score_below(d.last_place));
    return false;
}

// What a bucket's whole numbers count: 2^(-b / P - bits).
template <int P>
__device__ __forceinline__ double unit_of(int b, int bits) {
    const double one = __longlong_as_double((long long)(1023 - bits) << 52);
    if constexpr (P == 32) return exp2(-(double)b / P) * one;
    constexpr double kPart[8] = {1.0, 0.91700404320467123174, 0.84089641525371454303, 0.77110541270397041180, 0.70710678118654752440, 0.64841977732550483296, 0.59460355750136053336,
                                 0.54525386633262882960};
    double part = kPart[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) part = b % 8 == i ? kPart[i] : part;
    return part * __longlong_as_double((long long)(1023 - b / 8) << 52) * one;
}
template <int P>
__device__ __forceinline__ constexpr double next_unit() { return P == 32 ? 0.97857206208770013451 : 0.91700404320467123174; }  // 2^(-1 / P)

// The draw, the weights of all that is kept being in their buckets.
template <int G, typename Row>
__device__ __forceinline__ void end_draw(Draw<G, Row> &d, const RowSampling &r, int classes, int bits, int *cls, float *logp) {
    constexpr int P = parts_of<G>();
    DrawShared<G> &sh = d.sh;
    const auto weight = [&](double s) { return d.weight_of(s); };
    double mass[Draw<G, Row>::kEach], all;
    const auto unit = [&](int b) { return unit_of<P>(b, bits); };
    const double before = d.sums(unit(in_group<G>() * Draw<G, Row>::kEach), next_unit<P>(), mass, &all);
    double kept = all, front;
    int bucket;
    if (r.p < 1.f) {
        const double most = fmax((double)r.p, 0.0) * all;
        d.find(mass, before, most, true, &bucket, &front);
        const double its = unit(bucket);
        // The draw is among those up to here. A bucket's weights are nearly the same: its whole numbers say how many they are.
        float count = 0.f;
        if (G > 64 && d.chosen < 0) {
#pragma unroll
            for (int i = 0; i < Draw<G, Row>::kEach; ++i) {
                const int b = in_group<G>() * Draw<G, Row>::kEach + i;
                if (b <= bucket) count += (float)sh.mass[b];
            }
            count = block_sum_f<G>(count, sh.part_f) * (float)unit_of<P>(0, bits);
            // (more of them cost as much to list as they save: 2048 x 65537, 2300 of a row kept: 249 us, 279 with the list)
            if (count < fminf(0.95f * chosen_of<G>(), (float)classes / 128.f)) d.choose(d.score_below(bucket + 0.5));
        }
        const auto last = d.resolve(bucket, (most - front) / its, true, weight);
        kept = front + (last.before + last.weight) * its;
    }
    const double target = (double)r.u * kept;
    d.find(mass, before, target, false, &bucket, &front);
    const double its = unit(bucket);
    const auto drawn = d.resolve(bucket, (target - front) / its, false, weight);
    if (in_group<G>() == 0) {
        *cls = (int)~(unsigned)drawn.key;
        *logp = (float)log(drawn.weight * its / kept);
    }
}

// The draw of a row by a workgroup. bits: of a whole number that stands for a w of one, so that the sum of a row's has room in 63.
template <int G, typename Row>
__device__ __forceinline__ void draw_row(Row &row, const RowSampling &r, int classes, int bits, DrawShared<G> &sh, int *cls, float *logp) {
    constexpr int V = Row::V;
    float mine = kNothing;
    row.each([&](const float (&x)[V], int) {
#pragma unroll
        for (int j = 0; j < V; ++j) mine = fmaxf(mine, x[j]);
    });
    const float m = block_max<G>(mine, sh.part_f);
    if (m == kNothing || r.none) {
        if (in_group<G>() == 0) {
            *cls = -1;
            *logp = r.none ? __builtin_nanf("") : kNothing;
        }
        return;
    }
    if (r.greedy) {
        int first = INT_MAX;
        row.each([&](const float (&x)[V], int c) {
#pragma unroll
            for (int j = 0; j < V; ++j) first = x[j] == m ? min(first, c + j) : first;
        });
        first = block_min<G>(first, sh.part_i);
        if (in_group<G>() == 0) {
            *cls = first;
            *logp = 0.f;
        }
        return;
    }
    if (m == __builtin_inff()) {  // (infinite scores share alike)
        int count = 0;
        row.each([&](const float (&x)[V], int) {
#pragma unroll
            for (int j = 0; j < V; ++j) count += x[j] == m ? 1 : 0;
        });
        int n = min(block_sum<G>(count, sh.part_i), r.k);
        if (r.p < 1.f) n = max(1, (int)ceil((double)fmaxf(r.p, 0.f) * n));
        const int c = nth_class<G>(row, m, (int)((double)r.u * n), classes, sh.part_i);
        if (in_group<G>() == 0) {
            *cls = c;
            *logp = (float)-log((double)n);
        }
        return;
    }
    Draw<G, Row> d{sh, row};
    bool all_kept = begin_draw(d, r, m, bits);
    if (!all_kept) d.choose(d.least);
    if (r.k < classes) {
        d.keep_best(r.k, mine);
        all_kept = all_kept && d.cut == 0 && d.least == -FLT_MAX;
    }
    d.add_up(all_kept);
    end_draw(d, r, classes, bits, cls, logp);
}

// A row's scores, classes side by side, with bias and allowed sets, read by vectors of 16 bytes as often as they are gone over. (Scores that stay in registers want
// every loop over them to be written out, and there are a dozen: the compiler did not find registers for it.)
template <typename T, int G, bool RULES>
struct ScoreRow {
    static constexpr int V = 16 / (int)sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    const T *src;
    const float *bias;
    const unsigned *words;
    int begin, classes;  // from where to where
    bool none;

    __device__ __forceinline__ Vec read(int c) const {
        if (c + V <= classes) return *reinterpret_cast<const Vec *>(src + c);
        Vec v = (T)kNothing;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < classes) v[j] = src[c + j];
        return v;
    }
    template <typename F>
    __device__ __forceinline__ void give(const Vec &v, int c, F f) {
        float x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = score_to_float(v[j]);
        if constexpr (RULES) {
            if (bias != nullptr) {
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    if (c + j + 4 <= classes) {
                        const Float4 b = *reinterpret_cast<const Float4 *>(bias + c + j);
#pragma unroll
                        for (int q = 0; q < 4; ++q) x[j + q] += b[q];
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q) x[j + q] += c + j + q < classes ? bias[c + j + q] : 0.f;
                    }
                }
            }
            if (none || words != nullptr) {
                const unsigned ok = none ? 0u : words[c / 32] >> (c % 32);
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] = ok >> j & 1u ? x[j] : kNothing;
            }
        }
        f(x, c);
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) {
        // (the next vectors are on their way while one is worked on)
        constexpr int kStep = G * V;
        int c = begin + (int)threadIdx.x * V;
        Vec a = (T)kNothing, b = (T)kNothing;
        if (c < classes) a = read(c);
        if (c + kStep < classes) b = read(c + kStep);
        for (; c < classes; c += kStep) {
            const Vec now = a;
            a = b;
            if (c + 2 * kStep < classes) b = read(c + 2 * kStep);
            give(now, c, f);
        }
    }
};

template <typename T, int G, bool RULES>
__device__ __forceinline__ ScoreRow<T, G, RULES> row_of(const tgbm_scores &in, const tgbm_score_rules &rules, long row, int begin, int end) {
    ScoreRow<T, G, RULES> scores;
    scores.src = static_cast<const T *>(in.data) + (size_t)row * in.row_stride;
    scores.begin = begin;
    scores.classes = end;
    scores.bias = rules.bias;
    scores.words = nullptr;
    scores.none = false;
    if constexpr (RULES) scores.words = allowed_words(rules, row, (in.classes + 31) / 32, &scores.none);
    return scores;
}
// (128 registers a lane are a few too few for all that a row may need: 1 to 37 are spilled)
template <typename T, int G, bool RULES>
__global__ __launch_bounds__(G, 4) void k_sample_rows(tgbm_scores in, tgbm_score_rules rules, tgbm_sampling how, const float *u, int *classes, float *logp, int bits) {
    __shared__ DrawShared<G> sh;
    const long row = blockIdx.x;
    auto scores = row_of<T, G, RULES>(in, rules, row, 0, in.classes);
    draw_row<G>(scores, sampling_of(how, u, row), in.classes, bits, sh, classes + row, logp + row);
}

// Few long rows: parts of a row by a workgroup each, in four launches. The largest score; the weights' buckets, added up over the parts as the whole numbers that they
// are, and where a number of classes cuts how many there are in each; the scores of the buckets where the cuts and the draw can be; the draw among those. One workgroup
// to a row took 58 us for 1 x 128003 bfloat16, 116 for 8 of them, 167 for 256 with settings of each row.
// Where it pays hangs on the length first (bfloat16, us by parts and by whole rows). Cut at a mass of 0.9: 64 x 16384 33 and 23, 64 x 32768 42 and 34, 256 x 32768 56 and 37,
// 1 x 65536 36 and 43, 64 x 65536 56 and 50, 64 x 100000 63 and 98, 384 x 128003 154 and 241. With settings of each row: 256 x 32768 61 and 44, 64 x 65536 61 and 83,
// 256 x 128003 137 and 235, 384 x 128003 172 and 198. Beyond that many rows the chip is full either way, and whole rows launch once (512 x 32768 72 and 49).
// (A least probability or a count alone leave so little of a row that it does not pay up to 250 000 classes: 256 x 128003 62 and 34, 92 and 46.)
constexpr int kSplitBlock = 512, kSplitParts = 64, kSplitRows = 384, kSplitLeast = 65536, kSplitListed = chosen_of<kSplitBlock>();
struct SplitRow {
    unsigned long long mass[Scale<parts_of<kSplitBlock>()>::kBuckets];
    unsigned long long listed[kSplitListed];
    unsigned times[Scale<parts_of<kSplitBlock>()>::kBuckets];  // (of rows whose number of classes is cut)
    float most[kSplitParts];
    int count, first, unused[2];  // first: the first class of the largest score, where that is the answer
};
__device__ __forceinline__ void part_of_row(int classes, int *begin, int *end) {
    const int size = ((classes - 1) / (int)gridDim.x + 64) / 64 * 64;
    *begin = min((int)blockIdx.x * size, classes);
    *end = min(*begin + size, classes);
}
__device__ __forceinline__ float most_of(const SplitRow &s, int parts) { return wave_max_f(lane_id() < parts ? s.most[lane_id()] : kNothing); }
// (rows that have no draw of this kind: the last launch goes over them by itself)
__device__ __forceinline__ bool goes_by_parts(const RowSampling &r, float m) { return !r.none && !r.greedy && m > kNothing && m < __builtin_inff(); }

template <typename T, bool RULES>
__global__ __launch_bounds__(kSplitBlock, 4) void k_split_most(tgbm_scores in, tgbm_score_rules rules, SplitRow *splits) {
    __shared__ float part_f[kSplitBlock / 64];
    SplitRow &s = splits[blockIdx.y];
    int begin, end;
    part_of_row(in.classes, &begin, &end);
    auto scores = row_of<T, kSplitBlock, RULES>(in, rules, blockIdx.y, begin, end);
    float mine = kNothing;
    scores.each([&](const float (&x)[decltype(scores)::V], int) {
#pragma unroll
        for (int j = 0; j < decltype(scores)::V; ++j) mine = fmaxf(mine, x[j]);
    });
    const float m = block_max<kSplitBlock>(mine, part_f);
    if (threadIdx.x == 0) {
        s.most[blockIdx.x] = m;
        if (blockIdx.x == 0) {
            s.count = 0;
            s.first = INT_MAX;
        }
    }
    constexpr int kBuckets = Scale<parts_of<kSplitBlock>()>::kBuckets;
    for (int i = (int)(blockIdx.x * kSplitBlock + threadIdx.x); i < kBuckets; i += (int)gridDim.x * kSplitBlock) {
        s.mass[i] = 0;
        s.times[i] = 0;
    }
}
template <typename T, bool RULES>
__global__ __launch_bounds__(kSplitBlock, 4) void k_split_add(tgbm_scores in, tgbm_score_rules rules, tgbm_sampling how, const float *u, SplitRow *splits, int bits) {
    __shared__ DrawShared<kSplitBlock> sh;
    const RowSampling r = sampling_of(how, u, blockIdx.y);
    SplitRow &s = splits[blockIdx.y];
    const float m = most_of(s, gridDim.x);
    if (!goes_by_parts(r, m)) return;
    int begin, end;
    part_of_row(in.classes, &begin, &end);
    auto scores = row_of<T, kSplitBlock, RULES>(in, rules, blockIdx.y, begin, end);
    Draw<kSplitBlock, decltype(scores)> d{sh, scores};
    const bool all_kept = begin_draw(d, r, m, bits);
    unsigned *const times = reinterpret_cast<unsigned *>(sh.chosen);
    if (r.k < in.classes) {
        for (int i = threadIdx.x; i <= d.kBuckets; i += kSplitBlock) times[i] = 0;
        d.clear();
        d.kept(d.least, __builtin_inff(), [&](double place, int bucket, unsigned long long) {
            atomicAdd(&sh.mass[bucket], d.weight_of(place));
            atomicAdd(&times[bucket], 1u);
        });
        __syncthreads();
    } else {
        d.add_up(all_kept);
    }
    for (int i = threadIdx.x; i < d.kBuckets; i += kSplitBlock)
        if (sh.mass[i] != 0) {
            atomicAdd(&s.mass[i], sh.mass[i]);
            if (r.k < in.classes) atomicAdd(&s.times[i], times[i]);
        }
}
// The bucket where the number of classes is cut, -1 where there are no more than that, and how many there are in front of it.
template <typename D>
__device__ __forceinline__ int cut_of_times(D &d, const SplitRow &s, int k, double *front) {
    d.clear();
    for (int i = threadIdx.x; i < d.kBuckets; i += kSplitBlock) d.sh.mass[i] = s.times[i];
    __syncthreads();
    double mass[D::kEach], all;
    const double before = d.sums(1.0, 1.0, mass, &all);
    if (all <= (double)k) return -1;
    int bucket;
    d.find(mass, before, (double)(k - 1), false, &bucket, front);
    return bucket;
}
template <typename T, bool RULES>
__global__ __launch_bounds__(kSplitBlock, 4) void k_split_list(tgbm_scores in, tgbm_score_rules rules, tgbm_sampling how, const float *u, SplitRow *splits, int bits) {
    __shared__ DrawShared<kSplitBlock> sh;
    const RowSampling r = sampling_of(how, u, blockIdx.y);
    SplitRow &s = splits[blockIdx.y];
    const float m = most_of(s, gridDim.x);
    if (!(goes_by_parts(r, m) || (r.greedy && !r.none && m > kNothing))) return;
    int begin, end;
    part_of_row(in.classes, &begin, &end);
    auto scores = row_of<T, kSplitBlock, RULES>(in, rules, blockIdx.y, begin, end);
    using D = Draw<kSplitBlock, decltype(scores)>;
    if (r.greedy) {
        int its = INT_MAX;
        scores.each([&](const float (&x)[D::V], int c) {
#pragma unroll
            for (int j = 0; j < D::V; ++j) its = x[j] == m ? min(its, c + j) : its;
        });
        its = wave_min_i(its);
        if (lane_id() == 0 && its != INT_MAX) atomicMin(&s.first, its);
        return;
    }
    D d{sh, scores};
    begin_draw(d, r, m, bits);
    double front = 0;
    const int last_bucket = r.k < in.classes ? cut_of_times(d, s, r.k, &front) : -1;
    d.clear();
    for (int i = threadIdx.x; i < d.kBuckets; i += kSplitBlock) sh.mass[i] = last_bucket < 0 || i <= last_bucket ? s.mass[i] : 0;
    __syncthreads();
    double mass[D::kEach], all;
    const double before = d.sums(unit_of<D::P>(threadIdx.x * D::kEach, bits), next_unit<D::P>(), mass, &all);
    const auto of = [&](int bucket) { return (double)s.mass[bucket] * unit_of<D::P>(bucket, bits); };
    // Sums are known but for the part of a bucket that is cut: from where to where the cut by mass and the draw can be.
    double least = last_bucket < 0 ? all : all - of(last_bucket), most = all;
    int cut_first = 0, cut_last = -1, first, last;
    if (r.p < 1.f) {
        const double p = fmax((double)r.p, 0.0);
        d.find(mass, before, p * least * (1.0 - 0x1p-40), true, &cut_first, &front);
        least = fmax(front - 0x1p-40 * all, 0.0);
        d.find(mass, before, p * most * (1.0 + 0x1p-40), true, &cut_last, &front);
        most = front + of(cut_last);
    }
    d.find(mass, before, (double)r.u * least * (1.0 - 0x1p-40), false, &first, &front);
    d.find(mass, before, (double)r.u * most * (1.0 + 0x1p-40), false, &last, &front);
    const int from = min(first, min(cut_last < 0 ? first : cut_first, last_bucket < 0 ? first : last_bucket)), to = max(last, max(cut_last, last_bucket));
    d.kept(d.score_below(to + 0.5), d.score_above(from - 0.5), [&](double, int b, unsigned long long key) {
        if ((b < first || b > last) && (b < cut_first || b > cut_last) && b != last_bucket) return;
        const int at = atomicAdd(&s.count, 1);
        if (at < kSplitListed) s.listed[at] = key;
    });
}
template <typename T, bool RULES>
__global__ __launch_bounds__(kSplitBlock, 4) void k_split_draw(tgbm_scores in, tgbm_score_rules rules, tgbm_sampling how, const float *u, const SplitRow *splits, int parts, int *classes,
                                                               float *logp, int bits) {
    __shared__ DrawShared<kSplitBlock> sh;
    const long row = blockIdx.x;
    const RowSampling r = sampling_of(how, u, row);
    const SplitRow &s = splits[row];
    const float m = most_of(s, parts);
    auto scores = row_of<T, kSplitBlock, RULES>(in, rules, row, 0, in.classes);
    if (r.greedy && !r.none && m > kNothing) {
        if (threadIdx.x == 0) {
            classes[row] = s.first;
            logp[row] = 0.f;
        }
        return;
    }
    if (!goes_by_parts(r, m) || s.count > kSplitListed) {
        draw_row<kSplitBlock>(scores, r, in.classes, bits, sh, classes + row, logp + row);
        return;
    }
    Draw<kSplitBlock, decltype(scores)> d{sh, scores};
    begin_draw(d, r, m, bits);
    d.chosen = s.count;  // (not all that is kept, but all of the buckets that are looked into)
    for (int i = threadIdx.x; i < d.chosen; i += kSplitBlock) sh.chosen[i] = s.listed[i];
    double front = 0;
    const int last_bucket = r.k < in.classes ? cut_of_times(d, s, r.k, &front) : -1;
    if (last_bucket >= 0) {
        const unsigned long long key = d.resolve(last_bucket, (double)(r.k - 1) - front, false, [](double) { return 1ull; }).key;
        d.cut = key;
        d.least = from_ordered((unsigned)(key >> 32));
    }
    d.clear();
    for (int i = threadIdx.x; i < d.kBuckets; i += kSplitBlock) sh.mass[i] = last_bucket < 0 || i < last_bucket ? s.mass[i] : 0;
    __syncthreads();
    if (last_bucket >= 0) {
        d.kept(d.least, __builtin_inff(), [&](double place, int b, unsigned long long) {
            if (b == last_bucket) atomicAdd(&sh.mass[b], d.weight_of(place));
        });
        __syncthreads();
    }
    end_draw(d, r, in.classes, bits, classes + row, logp + row);
}

// A row in LDS, adjusted, for a wavefront; behind its classes -infinity up to a multiple of four.
struct LdsRow {
    static constexpr int V = 4;
    const float *scores;
    int classes;
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int c = lane_id() * 4; c < classes; c += 256) {
            const float4 v = *reinterpret_cast<const float4 *>(scores + c);
            const float x[4] = {v.x, v.y, v.z, v.w};
            f(x, c);
        }
    }
};

// Rows of a middle length: a wavefront to a row, whose adjusted scores lie in LDS. COLUMNS: the rows lie side by side, and a workgroup brings as many as it has
// wavefronts; else each brings its own. A class that was shown has a bit, and its cell holds how often first; whoever takes the bit away puts the score there.
// LDS of a wavefront: DrawShared (unless its row is SORTED), pitch cells, with lists pitch / 32 + 1 words of bits.
template <typename T, bool COLUMNS, bool RULES, bool SORTED>
__global__ __launch_bounds__(COLUMNS ? 1024 : 256, SORTED ? 8 : 4) void k_sample_middle(tgbm_scores in, tgbm_score_rules rules, tgbm_sampling how, const float *u, int *classes, float *logp, int bits,
                                                                       int pitch, int of_wave) {
    constexpr int kWaves = COLUMNS ? 16 : 4;
    extern __shared__ __align__(16) char lds[];
    const auto shared_of = [&](int w) { return reinterpret_cast<DrawShared<64> *>(lds + (size_t)w * of_wave); };
    const auto cells_of = [&](int w) { return reinterpret_cast<unsigned *>(lds + (size_t)w * of_wave + (SORTED ? 0 : sizeof(DrawShared<64>))); };
    const auto bits_of = [&](int w) { return cells_of(w) + pitch; };
    static_assert(sizeof(DrawShared<64>) % 16 == 0);
    const int lane = lane_id(), wave = wave_id(), n = in.classes;
    const long row0 = (COLUMNS ? tile_of_block(blockIdx.x, gridDim.x) : (long)blockIdx.x) * kWaves;
    if (row0 >= in.rows) return;
    // who brings what: r: the row of the tile, at, step: its classes
    const int r = COLUMNS ? (int)threadIdx.x % 16 : wave, at = COLUMNS ? (int)threadIdx.x / 16 : lane, step = 64;
    const long row = row0 + r;
    const bool on = row < in.rows;
    if (!COLUMNS && !on) return;
    const auto sync = [&] { group_sync<COLUMNS ? 1024 : 64>(); };
    unsigned *const cell = cells_of(r), *const bit_of = bits_of(r);
    const T *src = static_cast<const T *>(in.data) + (size_t)(on ? row : 0) * in.row_stride;
    bool none = false;
    const unsigned *words = nullptr;
    long long b = 0, e = 0;
    if constexpr (RULES) {
        if (on) words = allowed_words(rules, row, (n + 31) / 32, &none);
        if (rules.shown != nullptr) {
            for (int i = at; i < (n + 31) / 32; i += step) bit_of[i] = 0;
            sync();
            if (on) shown_range(rules, row, &b, &e);
            for (long long i = b + at; i < e; i += step) {
                const int c = rules.shown[i];
                if ((unsigned)c >= (unsigned)n) continue;
                cell[c] = 0;
                atomicOr(&bit_of[c / 32], 1u << (c % 32));
            }
            sync();
            for (long long i = b + at; i < e; i += step) {
                const int c = rules.shown[i];
                if ((unsigned)c < (unsigned)n) atomicAdd(&cell[c], 1u);
            }
        }
    }
    const auto one = [&](int c, T v) {
        float s = score_to_float(v);
        if constexpr (RULES) {
            if (rules.bias != nullptr) s += rules.bias[c];
            if (none || (words != nullptr && !(words[c / 32] >> (c % 32) & 1u))) s = kNothing;
            if (rules.shown != nullptr && (bit_of[c / 32] >> (c % 32) & 1u)) return;
        }
        cell[c] = __float_as_uint(s);
    };
    if (on) {
        // (eight loads of a thread are on their way together)
        for (int c = at; c < n; c += 8 * step) {
            T v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = src[(size_t)min(c + i * step, n - 1) * in.class_stride];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i * step < n) one(c + i * step, v[i]);
        }
        if (at < (-n & 3)) cell[n + at] = __float_as_uint(kNothing);
    }
    if constexpr (RULES) {
        if (rules.shown != nullptr) {
            sync();
            for (long long i = b + at; i < e; i += step) {
                const int c = rules.shown[i];
                if ((unsigned)c >= (unsigned)n) continue;
                const unsigned bit = 1u << (c % 32);
                if (!(atomicAnd(&bit_of[c / 32], ~bit) & bit)) continue;  // (another mention of the class has come first)
                const bool ok = !none && (words == nullptr || words[c / 32] & bit);
                cell[c] = __float_as_uint(adjusted(score_to_float(src[(size_t)c * in.class_stride]), rules.bias != nullptr ? rules.bias[c] : 0.f, cell[c], ok, rules));
            }
        }
    }
    sync();
    const long its = row0 + wave;
    if (its >= in.rows) return;
    LdsRow scores{reinterpret_cast<const float *>(cells_of(wave)), n};
    if constexpr (SORTED) draw_sorted(scores.scores, n, sampling_of(how, u, its), classes + its, logp + its);
    else draw_row<64>(scores, sampling_of(how, u, its), n, bits, *shared_of(wave), classes + its, logp + its);
}

// ------------------------------------------------------------------------------------------------------- how a call goes
enum Way { kFew, kFromList, kMiddle, kRows, kLaidOut };
constexpr int kFewClasses = 32;
constexpr int kListShort = 64, kListLong = 8192;
constexpr int kMiddleRows = 2048, kMiddleColumns = 1024;  // (16 rows' LDS holds 1050)
constexpr size_t kLaidBytes = (size_t)128 << 20;  // (half of what the last cache holds)

Way way_of(const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how) {
    // (a thread that goes through a long list alone: 24 x 26 with 300 shown classes a row, 172 us)
    if (in.classes <= kFewClasses) return rules.shown == nullptr || rules.n_shown <= 32ll * in.rows ? kFew : kMiddle;
    // top's lists where they are short, or the rows long: with more best classes shorter rows' scores overflow them (10343 x 3310, rows side by side, k 120: 1086 us).
    // Two or three launches more: not for few rows (200 x 100, k 20: 22 us, 11 without), and up to 128 classes only for the shortest lists (200000 x 100, k 20: 181 us,
    // 232 without; k 40: 243, 222). A count that cuts nothing is none.
    const bool columns = rows_side_by_side(in), middle = in.classes <= (columns ? kMiddleColumns : kMiddleRows), sorted = in.classes <= kSorted;
    const int listed = how.k == nullptr && how.k_all < in.classes && !(middle && in.rows <= (sorted ? 16384 : 256)) ? how.k_all : 0;
    if (listed >= 1 && (listed <= (sorted ? kListShort / 2 : kListShort) || (listed <= kTopMost && !columns && in.classes > kListLong))) return kFromList;
    if (middle) return kMiddle;
    return rules.shown != nullptr || rows_side_by_side(in) ? kLaidOut : kRows;
}
int middle_pitch(int classes) { return (classes + 3) / 4 * 4; }
int middle_lds(int classes) { return (int)(((classes <= kSorted ? 0 : sizeof(DrawShared<64>)) + sizeof(unsigned) * (middle_pitch(classes) + (classes + 31) / 32) + 15) / 16 * 16); }
// values, classes and what top leaves beside them, in front of its own workspace
size_t list_bytes(size_t rows, size_t k) { return (sizeof(float) * rows * (2 * k + 1) + 15) / 16 * 16; }
long laid_pitch(int classes) { return ((long)classes + 3) / 4 * 4; }
int laid_rows(int classes, int rows) { return (int)std::max<long>(1, std::min<long>(rows, (long)(kLaidBytes / sizeof(float)) / laid_pitch(classes))); }

tgbm_sampling take(tgbm_sampling how, int first) {
    if (how.temperature != nullptr) how.temperature += first;
    if (how.p != nullptr) how.p += first;
    if (how.min_p != nullptr) how.min_p += first;
    if (how.k != nullptr) how.k += first;
    return how;
}

template <typename T>
void sample_few(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp) {
    const unsigned blocks = (unsigned)((in.rows - 1) / kSampleBlock + 1);
    if (in.classes <= 8) k_sample_few<T, 8><<<blocks, kSampleBlock, 0, s>>>(in, rules, how, u, classes, logp);
    else if (in.classes <= 16) k_sample_few<T, 16><<<blocks, kSampleBlock, 0, s>>>(in, rules, how, u, classes, logp);
    else k_sample_few<T, 32><<<blocks, kSampleBlock, 0, s>>>(in, rules, how, u, classes, logp);
}

// Bits of a whole number that stands for a w of one: the sum of a row's, of which w is at most 1.05 in a bucket, has room in 63. 50 up to 2^11 classes, 45 at 2^16, 39 at 2^22: a weight is
// rounded by 2^-40 of itself at most, where a random number's last place is 2^-24.
int weight_bits(int classes) {
    int log_classes = 0;
    while ((1 << log_classes) < classes) ++log_classes;
    return std::min(50, 61 - log_classes);
}

template <typename T, bool COLUMNS, bool RULES, bool SORTED>
void sample_middle(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp) {
    constexpr int kWaves = COLUMNS ? 16 : 4;
    static LdsOptIn opt_in;
    opt_in({reinterpret_cast<const void *>(&k_sample_middle<T, COLUMNS, RULES, SORTED>)});
    // (rows' cells begin four banks apart, so that sixteen rows of four classes are stored at once)
    const int of_wave = COLUMNS ? (middle_lds(in.classes) + 239) / 256 * 256 + 16 : middle_lds(in.classes);
    const unsigned tiles = (unsigned)((in.rows - 1) / kWaves + 1);
    k_sample_middle<T, COLUMNS, RULES, SORTED><<<COLUMNS ? blocks_of_tiles(tiles) : tiles, 64 * kWaves, of_wave * kWaves, s>>>(in, rules, how, u, classes, logp,
                                                                                                                              weight_bits(in.classes), middle_pitch(in.classes), of_wave);
}
template <typename T, bool COLUMNS, bool RULES>
void sample_middle(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp) {
    // (sums of up to 128 weights: 200000 x 100 cut at a mass of 0.9, 442 us by buckets)
    if (in.classes <= kSorted) sample_middle<T, COLUMNS, RULES, true>(s, in, rules, how, u, classes, logp);
    else sample_middle<T, COLUMNS, RULES, false>(s, in, rules, how, u, classes, logp);
}
template <typename T>
void sample_middle(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp) {
    const bool some = rules.bias != nullptr || rules.allowed != nullptr || rules.shown != nullptr;
    if (rows_side_by_side(in)) (some ? sample_middle<T, true, true> : sample_middle<T, true, false>)(s, in, rules, how, u, classes, logp);
    else (some ? sample_middle<T, false, true> : sample_middle<T, false, false>)(s, in, rules, how, u, classes, logp);
}

// Few long rows go by parts.
bool goes_by_splits(int classes, int rows) { return rows <= kSplitRows && classes >= kSplitLeast; }
size_t split_bytes(int classes, int rows) { return goes_by_splits(classes, rows) ? sizeof(SplitRow) * (size_t)rows : 0; }

template <typename T, bool RULES>
void sample_rows(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp, void *room) {
    if (goes_by_splits(in.classes, in.rows)) {
        const int bits = weight_bits(in.classes), parts = std::min({kSplitParts, in.classes / 4096, std::max(2, 1024 / in.rows)});
        const dim3 grid((unsigned)parts, (unsigned)in.rows);
        SplitRow *splits = static_cast<SplitRow *>(room);
        k_split_most<T, RULES><<<grid, kSplitBlock, 0, s>>>(in, rules, splits);
        k_split_add<T, RULES><<<grid, kSplitBlock, 0, s>>>(in, rules, how, u, splits, bits);
        k_split_list<T, RULES><<<grid, kSplitBlock, 0, s>>>(in, rules, how, u, splits, bits);
        k_split_draw<T, RULES><<<in.rows, kSplitBlock, 0, s>>>(in, rules, how, u, splits, parts, classes, logp, bits);
        return;
    }
    // Threads of a row's workgroup. 256 for a few vectors each (cut at a mass of 0.9, us with 256 and 512: 20000 x 4096 float32 353 and 460, 300 x 4096 17 and 15); 1024 where each CU has a row at
    // most, and that is long (us with 512 and 1024: 256 x 5000 float32 14 and 16, 256 x 16384 bfloat16 25 and 26, with k 500 33 and 24, 256 x 32768 39 and 37, with k 500 50 and 27;
    // 384 x 32768, more rows than CUs, 47 and 61).
    const int bits = weight_bits(in.classes), vectors = (in.classes - 1) / (16 / (int)sizeof(T)) + 1;
    if (vectors <= 4 * 256) k_sample_rows<T, 256, RULES><<<in.rows, 256, 0, s>>>(in, rules, how, u, classes, logp, bits);
    else if (in.rows > 256 || in.classes < 16384) k_sample_rows<T, 512, RULES><<<in.rows, 512, 0, s>>>(in, rules, how, u, classes, logp, bits);
    else k_sample_rows<T, 1024, RULES><<<in.rows, 1024, 0, s>>>(in, rules, how, u, classes, logp, bits);
}
template <typename T>
void sample_rows(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp, void *room) {
    if (rules.bias != nullptr || rules.allowed != nullptr) sample_rows<T, true>(s, in, rules, how, u, classes, logp, room);
    else sample_rows<T, false>(s, in, rules, how, u, classes, logp, room);
}

template <typename T>
void sample_laid_out(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp,
                     float *room) {
    const long pitch = laid_pitch(in.classes);
    const int most = laid_rows(in.classes, in.rows);
    for (int row = 0; row < in.rows; row += std::min(most, in.rows - row)) {
        tgbm_scores part = in;
        tgbm_score_rules r = rules;
        take_rows(part, r, row, std::min(most, in.rows - row));
        k_lay_out<T><<<dim3((in.classes - 1) / kLaid + 1, (part.rows - 1) / kLaid + 1), kSampleBlock, 0, s>>>(part, r, room, pitch);
        if (rules.shown != nullptr) k_lay_shown<T><<<dim3(part.rows, (in.classes - 1) / kShownClasses + 1), kSampleBlock, 0, s>>>(part, r, room, pitch);
        const tgbm_scores laid{room, 1, pitch, TGBM_F32, in.classes, part.rows};
        sample_rows<float>(s, laid, tgbm_score_rules{}, take(how, row), u + row, classes + row, logp + row, room + (size_t)most * pitch);
    }
}

template <typename T>
void sample(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp,
            void *workspace) {
    switch (way_of(in, rules, how)) {
        case kFew: return sample_few<T>(s, in, rules, how, u, classes, logp);
        case kMiddle: return sample_middle<T>(s, in, rules, how, u, classes, logp);
        case kRows: return sample_rows<T>(s, in, rules, how, u, classes, logp, workspace);
        case kLaidOut: return sample_laid_out<T>(s, in, rules, how, u, classes, logp, static_cast<float *>(workspace));
        case kFromList: {
            const size_t n = (size_t)in.rows, k = (size_t)how.k_all;
            float *values = static_cast<float *>(workspace), *lse = values + n * k;
            int *listed = reinterpret_cast<int *>(lse + n);
            launch_scores_top(s, in, rules, how.k_all, 1.f, values, listed, lse, static_cast<char *>(workspace) + list_bytes(n, k));
            const auto blocks = [&](int lanes) { return (unsigned)((in.rows - 1) / (kSampleBlock / lanes) + 1); };
            if (k <= 32) k_sample_listed<16><<<blocks(16), kSampleBlock, 0, s>>>(values, listed, how.k_all, in.rows, how, u, classes, logp);
            else if (k <= 64) k_sample_listed<32><<<blocks(32), kSampleBlock, 0, s>>>(values, listed, how.k_all, in.rows, how, u, classes, logp);
            else k_sample_listed<64><<<blocks(64), kSampleBlock, 0, s>>>(values, listed, how.k_all, in.rows, how, u, classes, logp);
        }
    }
}

}  // namespace

size_t scores_sample_workspace(const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how) {
    return workspace_of_slices(in.rows, [&](int rows) -> size_t {
        switch (way_of(in, rules, how)) {
            case kFromList: return list_bytes((size_t)rows, (size_t)how.k_all) + scores_top_workspace(rows_side_by_side(in), in.classes, rows, how.k_all);
            case kLaidOut: {
                // (as many rows as are laid out at a time, or what is left of them, may go by parts of a row)
                const int most = laid_rows(in.classes, rows);
                return sizeof(float) * (size_t)most * laid_pitch(in.classes) + std::max(split_bytes(in.classes, most), split_bytes(in.classes, rows % most));
            }
            case kRows: return split_bytes(in.classes, rows);
            default: return 0;
        }
    });
}

void launch_scores_sample(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp,
                          void *workspace) {
    for (int row = 0; row < in.rows; row += std::min(kSliceRows, in.rows - row)) {
        tgbm_scores part = in;
        tgbm_score_rules r = rules;
        take_rows(part, r, row, std::min(kSliceRows, in.rows - row));
        const tgbm_sampling h = take(how, row);
        if (in.type == TGBM_F32) sample<float>(s, part, r, h, u + row, classes + row, logp + row, workspace);
        else if (in.type == TGBM_F16) sample<_Float16>(s, part, r, h, u + row, classes + row, logp + row, workspace);
        else sample<__bf16>(s, part, r, h, u + row, classes + row, logp + row, workspace);
    }
}

}  // namespace tgbm
