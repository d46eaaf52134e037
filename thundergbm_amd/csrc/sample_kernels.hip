// tgbm_scores_sample: a class of every row, drawn from its scores by a random number that is given.
//
// The classes of a row in order, the best first and of equal scores the lower class: w = exp((score - best) / T) of each. Every cut keeps a front part of that
// order, and so the class that is drawn is the one where the sum of w passes u times the sum of what is kept. A sum over all classes decides which of two
// classes it is, so everything is 64 bits, and what many threads add up is added as whole numbers, whose sum has no order.
#include <cfloat>
#include <climits>

#include "kernel_common.h"
#include "score_rules.h"

namespace tgbm {
namespace {

constexpr int kSampleBlock = 256;
constexpr float kNothing = -__builtin_inff();
constexpr float kGreedyBelow = 1e-6f;  // temperatures below take the best class
constexpr float kLargestBelowOne = 0x1.fffffep-1f;

// Scores in the order of unsigned integers, the two zeros being equal. No NaN comes here.
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
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
// A thread holds its row's classes: the sum of those in front of each is what counts, no order is made.
template <typename T, int E>
__global__ __launch_bounds__(kSampleBlock) void k_sample_few(tgbm_scores in, tgbm_score_rules rules, tgbm_sampling how, const float *u, int *classes, float *logp) {
    const long row = (long)blockIdx.x * kSampleBlock + threadIdx.x;
    if (row >= in.rows) return;
    const RowSampling r = sampling_of(how, u, row);
    const T *src = static_cast<const T *>(in.data) + (size_t)row * in.row_stride;
    float v[E];
#pragma unroll
    for (int c = 0; c < E; ++c) v[c] = c < in.classes ? score_to_float(src[(size_t)c * in.class_stride]) : kNothing;
    unsigned times[E];
#pragma unroll
    for (int c = 0; c < E; ++c) times[c] = 0;
    if (rules.shown != nullptr) {
        long long b, e;
        shown_range(rules, row, &b, &e);
        for (long long i = b; i < e; ++i) {
            const int shown = rules.shown[i];
#pragma unroll
            for (int c = 0; c < E; ++c) times[c] += shown == c ? 1u : 0u;
        }
    }
    bool none;
    const unsigned *words = allowed_words(rules, row, 1, &none);
    const unsigned ok = none ? 0u : words != nullptr ? words[0] : ~0u;
    float m = kNothing;
#pragma unroll
    for (int c = 0; c < E; ++c)
        if (c < in.classes) {
            v[c] = without_nan(adjusted(v[c], rules.bias != nullptr ? rules.bias[c] : 0.f, times[c], ok >> c & 1u, rules));
            m = fmaxf(m, v[c]);
        }
    if (m == kNothing || r.none) {
        classes[row] = -1;
        logp[row] = r.none ? __builtin_nanf("") : kNothing;
        return;
    }
    const double by = 1.0 / (double)r.temperature;
    double w[E], sum = 0;
    int rank[E];
#pragma unroll
    for (int c = 0; c < E; ++c) {
        rank[c] = 0;
#pragma unroll
        for (int o = 0; o < E; ++o)
            if (o != c) rank[c] += (o < c ? v[o] >= v[c] : v[o] > v[c]) ? 1 : 0;
        const double x = v[c] == m ? 1.0 : exp(((double)v[c] - (double)m) * by);
        w[c] = v[c] > kNothing && rank[c] < (r.greedy ? 1 : r.k) && x >= (double)r.min_p ? x : 0.0;
        sum += w[c];
    }
    double front[E], kept = 0;
#pragma unroll
    for (int c = 0; c < E; ++c) {
        front[c] = 0;
#pragma unroll
        for (int o = 0; o < E; ++o) front[c] += rank[o] < rank[c] ? w[o] : 0.0;
    }
#pragma unroll
    for (int c = 0; c < E; ++c) {
        if (r.p < 1.f && rank[c] > 0 && !(front[c] < (double)r.p * sum)) w[c] = 0;
        kept += w[c];
    }
    const double target = (double)r.u * kept;
    int best = -1, best_rank = -1;
    double its = 0;
#pragma unroll
    for (int c = 0; c < E; ++c)
        if (w[c] > 0 && front[c] <= target && rank[c] > best_rank) {
            best = c;
            best_rank = rank[c];
            its = w[c];
        }
    classes[row] = best;
    logp[row] = r.greedy ? 0.f : (float)log(its / kept);
}

// ------------------------------------------------------------------------------------------------------- from a list
// Rows whose best classes are listed in order, as top leaves them: a wavefront takes a row's k of up to 128.
__device__ __forceinline__ double shfl_up_d(double v, int d) { return __longlong_as_double(shfl_up_ll(__double_as_longlong(v), d)); }
__device__ __forceinline__ double read_lane_d(double v, int lane) { return __longlong_as_double(read_lane_ll(__double_as_longlong(v), lane)); }
__device__ __forceinline__ double wave_scan_d(double v) {  // inclusive
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double o = shfl_up_d(v, d);
        if (lane_id() >= d) v += o;
    }
    return v;
}
__global__ __launch_bounds__(kSampleBlock) void k_sample_listed(const float *values, const int *listed, int k, int rows, tgbm_sampling how, const float *u, int *classes,
                                                                float *logp) {
    const long row = (long)blockIdx.x * (kSampleBlock / 64) + wave_id();
    if (row >= rows) return;
    const RowSampling r = sampling_of(how, u, row);
    const int lane = lane_id();
    const float *v = values + (size_t)row * k;
    float x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = 2 * lane + i < k ? v[2 * lane + i] : kNothing;
    const float m = read_lane(x[0], 0);
    if (m == kNothing || r.none) {
        if (lane == 0) {
            classes[row] = -1;
            logp[row] = r.none ? __builtin_nanf("") : kNothing;
        }
        return;
    }
    double w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const double e = x[i] == m ? 1.0 : exp(((double)x[i] - (double)m) / (double)r.temperature);
        w[i] = x[i] > kNothing && e >= (double)r.min_p && 2 * lane + i < (r.greedy ? 1 : r.k) ? e : 0.0;
    }
    const double upto1 = wave_scan_d(w[0] + w[1]), sum = read_lane_d(upto1, 63);
    const double up = shfl_up_d(upto1, 1);  // (of all lanes: one that does not take part hands nothing on)
    const double front0 = lane == 0 ? 0.0 : up, front1 = front0 + w[0];
    double kept = sum;
    if (r.p < 1.f) {
        const double most = (double)r.p * sum;
        const bool in0 = w[0] > 0 && (front0 < most || lane == 0), in1 = w[1] > 0 && front1 < most;
        const int last0 = 63 - __clzll((long long)__ballot(in0)), which1 = __any(in1) ? 63 - __clzll((long long)__ballot(in1)) : -1;
        // the sum up to the last one that is kept
        kept = which1 == last0 ? read_lane_d(upto1, last0) : read_lane_d(front1, last0);
    }
    const double target = (double)r.u * kept;
    const unsigned long long at0 = __ballot(w[0] > 0 && (front0 <= target || lane == 0)), at1 = __ballot(w[1] > 0 && front1 <= target);
    const int l0 = 63 - __clzll((long long)at0), l1 = at1 != 0 ? 63 - __clzll((long long)at1) : -1;
    const int l = l0 > l1 ? l0 : l1, i = l1 == l ? 1 : 0;
    if (lane == l) {
        classes[row] = listed[(size_t)row * k + 2 * l + i];
        logp[row] = r.greedy ? 0.f : (float)log((i ? w[1] : w[0]) / kept);
    }
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

// A score's place on the scale that sums are kept by: 32 parts to a halving of w, 64 halvings; its bucket is the nearest whole number. What is further down than that
// (2^-64 of the best class) is nothing beside a random number's last place, 2^-24, whatever there is of it.
constexpr int kParts = 32, kBuckets = 64 * kParts;
constexpr double kPartsOfE = kParts * 1.44269504088896340736;  // parts to a factor of e
constexpr double kToWhole = 6755399441055744.0;                // 1.5 * 2^52: the sum's low word is the nearest whole number

// 2^(-h / 32), h in [-1/2, 1/2], plus `magic` = 2^(52 - bits): its last 52 bits are the power of two times 2^bits, rounded. Taylor's series: the sixth term is below
// 2^-48 of the whole, 2^-46 is what a whole number of a row of 2^16 classes is rounded by.
__device__ __forceinline__ unsigned long long part_of_two(double h, double magic) {
    constexpr double a = -0.69314718055994530942 / kParts, c2 = a * a / 2, c3 = c2 * a / 3, c4 = c3 * a / 4, c5 = c4 * a / 5;
    double e = __builtin_fma(h, c5, c4);
    e = __builtin_fma(h, e, c3);
    e = __builtin_fma(h, e, c2);
    e = __builtin_fma(h, e, a);
    e = __builtin_fma(h, e, 1.0);
    return (unsigned long long)__double_as_longlong(e + magic) & 0xfffffffffffffull;
}

constexpr int kListed = 256;
template <int BLOCK>
struct DrawShared {
    unsigned long long mass[kBuckets + 1];  // (the last one takes what does not count)
    unsigned long long key[kListed], weight[kListed], front[kListed];
    double part[BLOCK / 64];
    float part_f[BLOCK / 64];
    int part_i[BLOCK / 64];
    unsigned long long best, least, most;
    double before;
    int listed, bucket;
};

// One workgroup's work on a row. Row: row.each(f) calls f(scores, their first class) for the thread's vectors; what is no class or NaN is -infinity there.
template <int BLOCK, typename Row>
struct Draw {
    static constexpr int V = Row::V, kEach = kBuckets / BLOCK;
    DrawShared<BLOCK> &sh;
    Row &row;
    double best, by;  // (the place of a score is (best - score) * by)
    double magic;
    float least = -FLT_MAX;      // the least score that is kept
    unsigned long long cut = 0;  // the last one of the order that is kept, as a key
    double last_place = kBuckets - 0.5;

    static __device__ __forceinline__ unsigned long long key_of(float x, int c) { return (unsigned long long)ordered(x) << 32 | (unsigned)~c; }
    __device__ __forceinline__ double place_of(float x) const { return (best - (double)x) * by; }
    static __device__ __forceinline__ int bucket_of(double place) { return (int)__double_as_longlong(place + kToWhole); }
    __device__ __forceinline__ unsigned long long weight_of(double place) const { return part_of_two(place - ((place + kToWhole) - kToWhole), magic); }
    // A score below which none has a place up to `place`; the other way: above which none has one from there on.
    __device__ __forceinline__ float score_below(double place) const {
        const double x = best - place / by;
        return __double2float_rd(x - 0x1p-49 * (fabs(x) + fabs(best)));
    }
    __device__ __forceinline__ float score_above(double place) const {
        const double x = best - place / by;
        return __double2float_ru(x + 0x1p-49 * (fabs(x) + fabs(best)));
    }
    // f(place, bucket, key) for those that are kept and whose score is from lo to hi
    template <typename F>
    __device__ __forceinline__ void kept(float lo, float hi, F f) {
        lo = fmaxf(lo, least);
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
        __syncthreads();
        if (lane_id() == 63) sh.part[wave_id()] = upto;
        __syncthreads();
        double before = 0, sum = 0;
#pragma unroll
        for (int w = 0; w < BLOCK / 64; ++w) {
            if (w == wave_id()) before = sum;
            sum += sh.part[w];
        }
        *all = sum;
        const double up = shfl_up_d(upto, 1);
        return lane_id() == 0 ? before : before + up;
    }
    __device__ __forceinline__ void clear() {
        __syncthreads();
        for (int i = threadIdx.x; i < kBuckets; i += BLOCK) sh.mass[i] = 0;
        clear_list();
    }
    __device__ __forceinline__ void clear_list() {
        __syncthreads();
        if (threadIdx.x == 0) {
            sh.bucket = 0;
            sh.listed = 0;
            sh.best = 0;
            sh.least = ~0ull;
            sh.most = 0;
        }
        __syncthreads();
    }

    // Whether the order up to `before` leaves the next one in what is looked for: up to a target, or below it.
    static __device__ __forceinline__ bool within(double before, double target, bool below) { return below ? before < target : before <= target; }

    // The buckets' sums, those in front of the thread's, and the sum of all. unit(b): what a bucket's whole numbers count.
    template <typename Unit>
    __device__ __forceinline__ double sums(Unit unit, double (&mass)[kEach], double *all) {
        double mine = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int b = threadIdx.x * kEach + i;
            const unsigned long long m = sh.mass[b];
            mass[i] = m != 0 ? (double)m * unit(b) : 0.0;
            mine += mass[i];
        }
        return scan(mine, all);
    }
    // The bucket where the sum passes the target, and the sum in front of it.
    __device__ __forceinline__ void find(const double (&mass)[kEach], double before, double target, bool below, int *bucket, double *front) {
        __syncthreads();
        if (threadIdx.x == 0) sh.bucket = 0;
        __syncthreads();
        int at = -1;
        double its = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (mass[i] > 0 && within(before, target, below)) {
                at = threadIdx.x * kEach + i;
                its = before;
            }
            before += mass[i];
        }
        if (at >= 0) atomicMax(&sh.bucket, at);
        __syncthreads();
        *bucket = sh.bucket;
        if (at == *bucket) sh.before = its;
        else if (*bucket == 0 && threadIdx.x == 0) sh.before = 0;  // (roundings may leave none: the first one then)
        __syncthreads();
        *front = sh.before;
    }

    struct Found {
        unsigned long long key;
        double before, weight;  // in the bucket's unit
    };
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
            __syncthreads();
            const int n = sh.listed;
            if (n <= kListed) return among(n, front, target, below);
            // too many for a list: by parts of the keys between the least and the largest of them
            kept(low, high, [&](double, int b, unsigned long long key) {
                if (b != bucket || key < lo || key > hi) return;
                atomicMin(&sh.least, key);
                atomicMax(&sh.most, key);
            });
            __syncthreads();
            lo = sh.least;
            hi = sh.most;
            const int width = 64 - __clzll((long long)(hi - lo)), shift = width > 11 ? width - 11 : 0;
            static_assert(kBuckets == 1 << 11);
            clear();
            kept(low, high, [&](double s, int b, unsigned long long key) {
                if (b == bucket && key >= lo && key <= hi) atomicAdd(&sh.mass[(hi - key) >> shift], weight(s));
            });
            __syncthreads();
            double mass[kEach], all;
            const double before = sums([](int) { return 1.0; }, mass, &all);
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
        constexpr int kShares = BLOCK / kListed > 0 ? BLOCK / kListed : 1;
        const int share = threadIdx.x / kListed;
        for (int j = threadIdx.x % kListed; j < n; j += BLOCK < kListed ? BLOCK : kListed) {
            const unsigned long long mine = sh.key[j];
            unsigned long long sum = 0;
            for (int o = share; o < n; o += kShares) sum += sh.key[o] > mine ? sh.weight[o] : 0ull;
            atomicAdd(&sh.front[j], sum);
        }
        __syncthreads();
        // (the first one always is; a larger sum in front comes later in the order, and no two are equal)
        for (int j = threadIdx.x; j < n; j += BLOCK)
            if (sh.front[j] != 0 && within(front + (double)sh.front[j], target, below)) atomicMax(&sh.best, sh.front[j]);
        __syncthreads();
        const unsigned long long its = sh.best;
        for (int j = threadIdx.x; j < n; j += BLOCK)
            if (sh.front[j] == its) sh.listed = j;
        __syncthreads();
        const int j = sh.listed;
        return Found{sh.key[j], front + (double)its, (double)sh.weight[j]};
    }

    // Leaves the k best. The k-th of the threads' own best scores is a bound: only what reaches it is looked at one by one.
    __device__ __forceinline__ void keep_best(int k) {
        double mass[kEach], all, front;
        int bucket;
        const auto ones = [](int) { return 1.0; };
        float bound = least;
        if (k <= BLOCK) {
            float mine = kNothing;
            row.each([&](const float (&x)[V], int) {
#pragma unroll
                for (int j = 0; j < V; ++j) mine = fmaxf(mine, x[j]);
            });
            clear();
            if (mine >= least && place_of(mine) <= last_place) atomicAdd(&sh.mass[bucket_of(place_of(mine))], 1ull);
            __syncthreads();
            const double before = sums(ones, mass, &all);
            if (all >= (double)k) {
                find(mass, before, (double)(k - 1), false, &bucket, &front);
                bound = fmaxf(bound, score_below(bucket + 0.5));
            }
        }
        clear();
        kept(bound, __builtin_inff(), [&](double, int b, unsigned long long) { atomicAdd(&sh.mass[b], 1ull); });
        __syncthreads();
        const double before = sums(ones, mass, &all);
        if (all <= (double)k) {  // (all that reach the bound: it is the cut)
            least = bound;
            return;
        }
        find(mass, before, (double)(k - 1), false, &bucket, &front);
        const unsigned long long key = resolve(bucket, (double)(k - 1) - front, false, [](double) { return 1ull; }).key;
        cut = key;
        const unsigned o = (unsigned)(key >> 32);
        least = __uint_as_float(o ^ ((o >> 31) - 1u | 0x80000000u));
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
                    atomicAdd(&sh.mass[(int)__double_as_longlong(at)], part_of_two(s - (at - kToWhole), magic));
                }
            });
        }
        __syncthreads();
    }
};

template <int BLOCK>
__device__ __forceinline__ float block_max(float v, float *part) {
    v = wave_max_f(v);
    __syncthreads();
    if (lane_id() == 0) part[wave_id()] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) v = fmaxf(v, part[w]);
    return v;
}
template <int BLOCK>
__device__ __forceinline__ int block_min(int v, int *part) {
    v = wave_min_i(v);
    __syncthreads();
    if (lane_id() == 0) part[wave_id()] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) v = min(v, part[w]);
    return v;
}
template <int BLOCK>
__device__ __forceinline__ int block_sum(int v, int *part) {
    v = wave_sum_i(v);
    __syncthreads();
    if (lane_id() == 0) part[wave_id()] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < BLOCK / 64; ++w) v += part[w];
    return v;
}

// The class of the n-th (from 0) score that is m, by bisection.
template <int BLOCK, typename Row>
__device__ __forceinline__ int nth_class(Row &row, float m, int n, int classes, int *part) {
    int lo = -1, hi = classes - 1;
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        int count = 0;
        row.each([&](const float (&x)[Row::V], int c) {
#pragma unroll
            for (int j = 0; j < Row::V; ++j) count += x[j] == m && c + j <= mid ? 1 : 0;
        });
        if (block_sum<BLOCK>(count, part) > n) hi = mid;
        else lo = mid;
    }
    return hi;
}

// The draw of a row by a workgroup. bits: of a whole number that stands for a w of one, so that the sum of a row's has room in 63.
template <int BLOCK, typename Row>
__device__ __forceinline__ void draw_row(Row &row, const RowSampling &r, int classes, int bits, DrawShared<BLOCK> &sh, int *cls, float *logp) {
    constexpr int V = Row::V;
    float m = kNothing;
    row.each([&](const float (&x)[V], int) {
#pragma unroll
        for (int j = 0; j < V; ++j) m = fmaxf(m, x[j]);
    });
    m = block_max<BLOCK>(m, sh.part_f);
    if (m == kNothing || r.none) {
        if (threadIdx.x == 0) {
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
        first = block_min<BLOCK>(first, sh.part_i);
        if (threadIdx.x == 0) {
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
        int n = min(block_sum<BLOCK>(count, sh.part_i), r.k);
        if (r.p < 1.f) n = max(1, (int)ceil((double)fmaxf(r.p, 0.f) * n));
        const int c = nth_class<BLOCK>(row, m, (int)((double)r.u * n), classes, sh.part_i);
        if (threadIdx.x == 0) {
            *cls = c;
            *logp = (float)-log((double)n);
        }
        return;
    }
    Draw<BLOCK, Row> d{sh, row};
    d.best = (double)m;
    d.by = kPartsOfE / (double)r.temperature;
    d.magic = __longlong_as_double((long long)(1023 + 52 - bits) << 52);
    bool all_kept = true;
    if (r.min_p > 0.f) {
        d.last_place = fmin(d.last_place, -log2((double)r.min_p) * kParts);
        d.least = fmaxf(d.least, d.score_below(d.last_place));
        all_kept = false;
    }
    if (r.k < classes) {
        d.keep_best(r.k);
        all_kept = all_kept && d.cut == 0 && d.least == -FLT_MAX;
    }
    const auto weight = [&](double s) { return d.weight_of(s); };
    double mass[Draw<BLOCK, Row>::kEach], all;
    d.add_up(all_kept);
    const double one = __longlong_as_double((long long)(1023 - bits) << 52);
    const auto unit = [&](int b) { return exp2(-(double)b / kParts) * one; };
    const double before = d.sums(unit, mass, &all);
    double kept = all, front;
    int bucket;
    if (r.p < 1.f) {
        const double most = fmax((double)r.p, 0.0) * all;
        d.find(mass, before, most, true, &bucket, &front);
        const double its = unit(bucket);
        const auto last = d.resolve(bucket, (most - front) / its, true, weight);
        kept = front + (last.before + last.weight) * its;
    }
    const double target = (double)r.u * kept;
    d.find(mass, before, target, false, &bucket, &front);
    const double its = unit(bucket);
    const auto drawn = d.resolve(bucket, (target - front) / its, false, weight);
    if (threadIdx.x == 0) {
        *cls = (int)~(unsigned)drawn.key;
        *logp = (float)log(drawn.weight * its / kept);
    }
}

// A row's scores, classes side by side, with bias and allowed sets. N vectors of 16 bytes to a thread, which stay in registers as they were read; longer rows (N is
// 0) are read as often as they are gone over.
template <typename T, int BLOCK, int N, bool RULES>
struct ScoreRow {
    static constexpr int V = 16 / (int)sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    const T *src;
    const float *bias;
    const unsigned *words;
    int classes;
    bool none;
    Vec held[N > 0 ? N : 1];

    __device__ __forceinline__ Vec read(int c) const {
        if (c + V <= classes) return *reinterpret_cast<const Vec *>(src + c);
        Vec v = (T)kNothing;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < classes) v[j] = src[c + j];
        return v;
    }
    __device__ __forceinline__ void load() {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (i * BLOCK + (int)threadIdx.x) * V;
            held[i] = c < classes ? read(c) : (Vec)(T)kNothing;
        }
    }
    template <typename F>
    __device__ __forceinline__ void give(const Vec &v, int c, F f) {
        float x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = score_to_float(v[j]);
        if constexpr (RULES) {
            if (bias != nullptr) {
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] += bias[min(c + j, classes - 1)];
            }
            if (none || words != nullptr) {
                const unsigned ok = none ? 0u : words[c / 32] >> (c % 32);
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] = ok >> j & 1u ? x[j] : kNothing;
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = without_nan(x[j]);
        f(x, c);
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) {
        if constexpr (N > 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                // (one vector at a time, unpacked anew wherever it is looked at: the compiler would keep all of them)
                __builtin_amdgcn_sched_barrier(0);
                typedef unsigned Words __attribute__((ext_vector_type(4)));
                Words w = __builtin_bit_cast(Words, held[i]);
                asm volatile("" : "+v"(w));
                const int c = (i * BLOCK + (int)threadIdx.x) * V;
                if (c < classes) give(__builtin_bit_cast(Vec, w), c, f);
            }
        } else {
            for (int c = (int)threadIdx.x * V; c < classes; c += BLOCK * V) give(read(c), c, f);
        }
    }
};

template <typename T, int BLOCK, int N, bool RULES>
__global__ __launch_bounds__(BLOCK, BLOCK == 1024 ? 4 : 4) void k_sample_rows(tgbm_scores in, tgbm_score_rules rules, tgbm_sampling how, const float *u, int *classes, float *logp, int bits) {
    __shared__ DrawShared<BLOCK> sh;
    const long row = blockIdx.x;
    const RowSampling r = sampling_of(how, u, row);
    ScoreRow<T, BLOCK, N, RULES> scores;
    scores.src = static_cast<const T *>(in.data) + (size_t)row * in.row_stride;
    scores.classes = in.classes;
    scores.bias = rules.bias;
    scores.words = nullptr;
    scores.none = false;
    if constexpr (RULES) scores.words = allowed_words(rules, row, (in.classes + 31) / 32, &scores.none);
    scores.load();
    draw_row<BLOCK>(scores, r, in.classes, bits, sh, classes + row, logp + row);
}

// ------------------------------------------------------------------------------------------------------- how a call goes
enum Way { kFew, kFromList, kRows, kLaidOut };
constexpr int kFewClasses = 32;
constexpr size_t kLaidBytes = (size_t)128 << 20;  // (half of what the last cache holds)

Way way_of(const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how) {
    if (in.classes <= kFewClasses) return kFew;
    if (how.k == nullptr && how.k_all >= 1 && how.k_all <= kTopMost) return kFromList;
    return rules.shown != nullptr || rows_side_by_side(in) ? kLaidOut : kRows;
}
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

template <typename T, bool RULES>
void sample_rows(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp) {
    int log_classes = 0;
    while ((1 << log_classes) < in.classes) ++log_classes;
    const int bits = std::min(50, 61 - log_classes), vectors = (in.classes - 1) / (16 / (int)sizeof(T)) + 1;
    if (vectors <= 4 * 256) k_sample_rows<T, 256, 0, RULES><<<in.rows, 256, 0, s>>>(in, rules, how, u, classes, logp, bits);
    else if (getenv("B1") == nullptr) k_sample_rows<T, 512, 0, RULES><<<in.rows, 512, 0, s>>>(in, rules, how, u, classes, logp, bits);
    else k_sample_rows<T, 1024, 0, RULES><<<in.rows, 1024, 0, s>>>(in, rules, how, u, classes, logp, bits);
}
template <typename T>
void sample_rows(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp) {
    if (rules.bias != nullptr || rules.allowed != nullptr) sample_rows<T, true>(s, in, rules, how, u, classes, logp);
    else sample_rows<T, false>(s, in, rules, how, u, classes, logp);
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
        sample_rows<float>(s, laid, tgbm_score_rules{}, take(how, row), u + row, classes + row, logp + row);
    }
}

template <typename T>
void sample(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how, const float *u, int *classes, float *logp,
            void *workspace) {
    switch (way_of(in, rules, how)) {
        case kFew: return sample_few<T>(s, in, rules, how, u, classes, logp);
        case kRows: return sample_rows<T>(s, in, rules, how, u, classes, logp);
        case kLaidOut: return sample_laid_out<T>(s, in, rules, how, u, classes, logp, static_cast<float *>(workspace));
        case kFromList: {
            const size_t n = (size_t)in.rows, k = (size_t)how.k_all;
            float *values = static_cast<float *>(workspace), *lse = values + n * k;
            int *listed = reinterpret_cast<int *>(lse + n);
            launch_scores_top(s, in, rules, how.k_all, 1.f, values, listed, lse, static_cast<char *>(workspace) + list_bytes(n, k));
            k_sample_listed<<<(in.rows - 1) / (kSampleBlock / 64) + 1, kSampleBlock, 0, s>>>(values, listed, how.k_all, in.rows, how, u, classes, logp);
        }
    }
}

}  // namespace

size_t scores_sample_workspace(const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_sampling &how) {
    return workspace_of_slices(in.rows, [&](int rows) -> size_t {
        switch (way_of(in, rules, how)) {
            case kFromList: return list_bytes((size_t)rows, (size_t)how.k_all) + scores_top_workspace(rows_side_by_side(in), in.classes, rows, how.k_all);
            case kLaidOut: return sizeof(float) * (size_t)laid_rows(in.classes, rows) * laid_pitch(in.classes);
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
