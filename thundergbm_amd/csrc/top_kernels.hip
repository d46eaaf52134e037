// tgbm_scores_top: the k best classes of every row, and the logarithm of the sum of the exponentials, in one read of the scores.
//
// A group of wavefronts holds a row, or a chunk of it, in registers. The k-th largest of the threads' own maxima is a lower
// bound of the k-th largest score: the k threads above it hold one such score each. Any bound that between k and a few more
// maxima reach will do, so it is found by bisection over the maxima (ballots, no memory), and what reaches it - about as many
// scores, a thread rarely holds two of the best - goes to a short list in LDS, which is put in order by counting. Equal scores
// are told apart by their class, so that the list stays short where many are equal. Rows that go by chunks leave k scores of
// each, and a launch of its own makes the same choice among those.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "kernel_common.h"
#include "score_rules.h"

namespace tgbm {
namespace {

constexpr int kTopBlock = 256;
constexpr float kNothing = -__builtin_inff();  // the score of what is not listed

// Scores in the order of unsigned integers, the two zeros being equal. No NaN comes here.
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(unsigned o) { return __uint_as_float(o ^ ((o >> 31) - 1u | 0x80000000u)); }
constexpr unsigned kLeast = 0x00800000u;  // ordered(-FLT_MAX): the least that is listed

__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }
template <int W>
__device__ __forceinline__ void group_sync() {
    if constexpr (W == 1) wave_fence();
    else __syncthreads();
}

template <int W>
struct TopList {
    static constexpr int kRoom = W == 1 ? 256 : 1024;
    unsigned long long entry[kRoom];  // ordered score, then the complement of the place: larger is better
    unsigned best[W == 1 ? 1 : W * 64];
    int first[W == 1 ? 1 : W * 64];
    float part_max[W], part_sum[W];
    int part[W];
    int count, exact, at_most;
    unsigned bound;
};

template <int M>
__device__ __forceinline__ int count_from(const unsigned (&b)[M], unsigned least) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < M; ++j) n += __popcll(__ballot(b[j] >= least));
    return n;
}
template <int M>
__device__ __forceinline__ int count_up_to(const int (&f)[M], int most) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < M; ++j) n += __popcll(__ballot(f[j] <= most));
    return n;
}

// A bound that k to `limit` of the maxima reach, or all of them where they are fewer; *exact: there is none, more than
// that many are equal to the bound, and fewer than k lie above it.
template <int M>
__device__ __forceinline__ unsigned find_bound(const unsigned (&b)[M], int k, int limit, int *exact) {
    *exact = 0;
    unsigned lo = kLeast, hi = 0xff800001u;  // (one past infinity)
    if (count_from(b, lo) <= limit) return lo;
    while (hi - lo > 1) {
        const unsigned mid = lo + (hi - lo) / 2;
        const int n = count_from(b, mid);
        if (n >= k) {
            lo = mid;
            if (n <= limit) return lo;
        } else {
            hi = mid;
        }
    }
    *exact = 1;
    return lo;
}

// The need-th smallest of the places.
template <int M>
__device__ __forceinline__ int find_place(const int (&f)[M], int need) {
    int lo = -1, hi = INT_MAX - 1;
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (count_up_to(f, mid) >= need) hi = mid;
        else lo = mid;
    }
    return hi;
}

// The same over all scores of the group.
template <int W>
__device__ __forceinline__ int group_sum(int n, TopList<W> &sh) {
    n = wave_sum_i(n);
    if constexpr (W == 1) return n;
    __syncthreads();
    sh.part[wave_id()] = n;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < W; ++w) all += sh.part[w];
    return all;
}

// The candidates of the group's k best: sh.entry, as many as are returned, the same in all threads. at(i): the place of v[i],
// which ascends with i. Every thread of the group comes here.
template <int W, int E, typename At>
__device__ __forceinline__ int list_candidates(const float (&v)[E], At at, int k, TopList<W> &sh) {
    const int lane = lane_id(), t = W == 1 ? lane : (int)threadIdx.x;
    float best = kNothing;
#pragma unroll
    for (int i = 0; i < E; ++i) best = fmaxf(best, v[i]);
    const int limit = k + max(4, k / 4);
    unsigned bound;
    int exact, at_most = INT_MAX;
    if constexpr (W == 1) {
        const unsigned b[1] = {ordered(best)};
        bound = find_bound(b, k, limit, &exact);
    } else {
        sh.best[t] = ordered(best);
        if (t == 0) sh.count = 0;
        __syncthreads();
        if (wave_id() == 0) {
            unsigned b[W];
#pragma unroll
            for (int j = 0; j < W; ++j) b[j] = sh.best[j * 64 + lane];
            int e;
            const unsigned found = find_bound(b, k, limit, &e);
            if (lane == 0) {
                sh.bound = found;
                sh.exact = e;
            }
        }
        __syncthreads();
        bound = sh.bound;
        exact = sh.exact;
    }
    if (exact) {  // (the same in all threads)
        const float equal = from_ordered(bound);
        int first = INT_MAX;
#pragma unroll
        for (int i = E - 1; i >= 0; --i) first = v[i] == equal ? at(i) : first;
        if (best != equal) first = INT_MAX;
        if constexpr (W == 1) {
            const unsigned b[1] = {ordered(best)};
            const int f[1] = {first};
            at_most = find_place(f, k - count_from(b, bound + 1));
        } else {
            sh.first[t] = first;
            __syncthreads();
            if (wave_id() == 0) {
                unsigned b[W];
                int f[W];
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    b[j] = sh.best[j * 64 + lane];
                    f[j] = sh.first[j * 64 + lane];
                }
                const int place = find_place(f, k - count_from(b, bound + 1));
                if (lane == 0) sh.at_most = place;
            }
            __syncthreads();
            at_most = sh.at_most;
        }
    }
    const float least = from_ordered(bound);
    unsigned mine = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) mine |= (v[i] >= least && (v[i] > least || at(i) <= at_most) ? 1u : 0u) << i;
    int scan = wave_scan_i(__popc(mine));
    int total = __shfl(scan, 63), begin = scan - __popc(mine);
    if constexpr (W > 1) {
        int base = 0;
        if (lane == 0) base = atomicAdd(&sh.count, total);
        begin += __shfl(base, 0);
    }
    auto put = [&] {
        int to = begin;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (mine >> i & 1u) {
                if (to < TopList<W>::kRoom) sh.entry[to] = (unsigned long long)ordered(v[i]) << 32 | (unsigned)~at(i);
                ++to;
            }
    };
    put();
    group_sync<W>();
    if constexpr (W > 1) total = sh.count;
    if (total <= TopList<W>::kRoom) return total;
    // The best scores lie together in few threads: the exact k-th one by bisection over all of them.
    unsigned lo = bound, hi = 0xff800001u;
    auto count = [&](unsigned from) {
        const float f = from_ordered(from);
        int n = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) n += v[i] >= f ? 1 : 0;
        return group_sum<W>(n, sh);
    };
    while (hi - lo > 1) {
        const unsigned mid = lo + (hi - lo) / 2;
        if (count(mid) >= k) lo = mid;
        else hi = mid;
    }
    const int need = k - (lo == 0xff800000u ? 0 : count(lo + 1));
    const float equal = from_ordered(lo);
    int p_lo = -1, p_hi = INT_MAX - 1;
    while (p_hi - p_lo > 1) {
        const int mid = p_lo + (p_hi - p_lo) / 2;
        int n = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) n += v[i] == equal && at(i) <= mid ? 1 : 0;
        if (group_sum<W>(n, sh) >= need) p_hi = mid;
        else p_lo = mid;
    }
    mine = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) mine |= (v[i] > equal || (v[i] == equal && at(i) <= p_hi) ? 1u : 0u) << i;
    scan = wave_scan_i(__popc(mine));
    begin = scan - __popc(mine);
    total = __shfl(scan, 63);
    if constexpr (W > 1) {
        __syncthreads();
        sh.part[wave_id()] = total;
        __syncthreads();
        total = 0;
        for (int w = 0; w < W; ++w) {
            if (w < wave_id()) begin += sh.part[w];
            total += sh.part[w];
        }
    }
    put();
    group_sync<W>();
    return total;
}

// Where a row's (or a chunk's) best classes go.
struct TopOut {
    float *values;  // [][k]
    int *classes;
    float *lse;     // [] of rows, or the largest score and the sum of chunks
};

// The candidates in order. class_at(place): the class.
template <int W, typename Class>
__device__ __forceinline__ void write_best(const TopList<W> &sh, int found, int k, size_t slot, const TopOut &out, Class class_at) {
    const int t = W == 1 ? lane_id() : (int)threadIdx.x;
    for (int j = t; j < found; j += 64 * W) {
        const unsigned long long e = sh.entry[j];
        int better = 0;
        for (int o = 0; o < found; ++o) better += sh.entry[o] > e ? 1 : 0;
        if (better < k) {
            out.values[slot * k + better] = from_ordered((unsigned)(e >> 32));
            out.classes[slot * k + better] = class_at((int)~(unsigned)e);
        }
    }
    for (int j = found + t; j < k; j += 64 * W) {
        out.values[slot * k + j] = kNothing;
        out.classes[slot * k + j] = -1;
    }
}

// The largest of the group's scores (0 where it is no number) and the sum of exp((v - it) / temperature). A NaN makes the sum
// NaN, an infinity makes it infinite.
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float reference_of(float m) { return fabsf(m) <= FLT_MAX ? m : 0.f; }
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// A sum to the reference `from` as one to `to`; an infinite one stays infinite.
__device__ __forceinline__ float rescaled(float sum, float from, float to, float by) {
    return sum <= FLT_MAX ? sum * exp2_of((from - to) * by) : sum;
}

template <int W, int E>
__device__ __forceinline__ void sum_exponentials(const float (&v)[E], float by, TopList<W> &sh, float *reference, float *sum) {
    float m = kNothing;
#pragma unroll
    for (int i = 0; i < E; ++i) m = fmaxf(m, v[i]);
    m = reference_of(wave_max_f(m));
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += exp2_of((v[i] - m) * by);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if constexpr (W > 1) {
        if (lane_id() == 0) {
            sh.part_max[wave_id()] = s > 0.f || s != s ? m : kNothing;
            sh.part_sum[wave_id()] = s;
        }
        __syncthreads();
        m = kNothing;
        for (int w = 0; w < W; ++w) m = fmaxf(m, sh.part_max[w]);
        m = reference_of(m);
        s = 0.f;
        for (int w = 0; w < W; ++w)
            if (sh.part_max[w] > kNothing) s += rescaled(sh.part_sum[w], sh.part_max[w], m, by);
    }
    *reference = m;
    *sum = s;
}
// (a sum that nothing adds to has no reference: log(0) + 0)
__device__ __forceinline__ float log_sum(float m, float s, float temperature) {
    return s > 0.f || s != s ? m / temperature + __builtin_amdgcn_logf(s) * kLn2 : kNothing;
}

// Classes side by side: E scores of a thread, by vectors of 16 bytes.
template <typename T>
struct Vector {
    static constexpr int kOf = 16 / (int)sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// A group of W wavefronts takes chunk `tile % chunks` of a row; with W = 1 there are four groups to a workgroup. LDS behind the
// lists: how often the classes of the chunk were shown, where there are lists.
template <typename T, int W, int E>
__global__ __launch_bounds__(W == 1 ? kTopBlock : 64 * W) void k_top_rows(tgbm_scores in, tgbm_score_rules rules, int k, float temperature, TopOut out,
                                                                          int chunks, int chunk, long tiles, bool whole) {
    constexpr int kGroups = W == 1 ? kTopBlock / 64 : 1;
    __shared__ TopList<W> lists[kGroups];
    extern __shared__ unsigned shown_times[];
    constexpr int V = Vector<T>::kOf;
    const int t = W == 1 ? lane_id() : (int)threadIdx.x, group = W == 1 ? wave_id() : 0;
    TopList<W> &sh = lists[group];
    unsigned *times = shown_times + (size_t)group * chunk;
    const float by = kLog2e / temperature;
    for (long tile = (long)blockIdx.x * kGroups + group; tile < tiles; tile += (long)gridDim.x * kGroups) {
        const long row = tile / chunks;
        const int c0 = (int)(tile % chunks) * chunk, c1 = min(in.classes, c0 + chunk);
        bool counted = false;
        if (rules.shown != nullptr) {
            long long b, e;
            shown_range(rules, row, &b, &e);
            counted = b < e;  // (the same for the group)
            if (counted) {
                for (int c = t; c < chunk; c += 64 * W) times[c] = 0;
                group_sync<W>();
                for (long long i = b + t; i < e; i += 64 * W) {
                    const int c = rules.shown[i];
                    if (c >= c0 && c < c1) atomicAdd(&times[c - c0], 1u);
                }
                group_sync<W>();
            }
        }
        bool none;
        const unsigned *words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
        const T *src = static_cast<const T *>(in.data) + (size_t)row * in.row_stride;
        float v[E];
#pragma unroll
        for (int g = 0; g < E / V; ++g) {
            const int c = c0 + (g * 64 * W + t) * V;
            typename Vector<T>::type x;
            if (c + V <= c1) {
                x = *reinterpret_cast<const typename Vector<T>::type *>(src + c);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] = c + j < c1 ? src[c + j] : (T)kNothing;
            }
            unsigned ok = none ? 0u : ~0u;
            if (words != nullptr && c < c1) ok = words[c / 32] >> (c % 32);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float s = score_to_float(x[j]);
                if (c + j < c1)
                    s = adjusted(s, rules.bias != nullptr ? rules.bias[c + j] : 0.f, counted ? times[c + j - c0] : 0u, ok >> j & 1u, rules);
                v[g * V + j] = s;
            }
        }
        float m, s;
        sum_exponentials<W>(v, by, sh, &m, &s);
        if (t == 0) {
            if (whole) {
                out.lse[row] = log_sum(m, s, temperature);
            } else {
                out.lse[tile * 2] = m;
                out.lse[tile * 2 + 1] = s;
            }
        }
        const int found = list_candidates<W>(v, [&](int i) { return c0 + ((i / V) * 64 * W + t) * V + i % V; }, k, sh);
        write_best(sh, found, k, (size_t)tile, out, [](int place) { return place; });
        group_sync<W>();
    }
}

// Rows side by side: a workgroup brings `rows` rows of a chunk of at most 64 * E classes into LDS, class by class, and its
// wavefronts take a row each.
constexpr int kColumnBlock = 512;
template <typename T, int E>
__global__ __launch_bounds__(kColumnBlock) void k_top_columns(tgbm_scores in, tgbm_score_rules rules, int k, float temperature, TopOut out, int chunks,
                                                              int chunk, int row_bits, long tiles, bool whole) {
    __shared__ TopList<1> lists[kColumnBlock / 64];
    extern __shared__ unsigned cell[];  // [chunk][rows + 1]
    const int rows = 1 << row_bits, pitch = rows + 1;
    const float by = kLog2e / temperature;
    const int r = threadIdx.x & (rows - 1), slot = threadIdx.x >> row_bits, slots = kColumnBlock >> row_bits;
    for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long row0 = tile / chunks * rows, row = row0 + r;
        const int c0 = (int)(tile % chunks) * chunk, c1 = min(in.classes, c0 + chunk);
        if (rules.shown != nullptr) {
            for (int i = threadIdx.x; i < chunk * pitch; i += kColumnBlock) cell[i] = 0;
            __syncthreads();
            long long b = 0, e = 0;
            if (row < in.rows) shown_range(rules, row, &b, &e);
            for (long long i = b + slot; i < e; i += slots) {
                const int c = rules.shown[i];
                if (c >= c0 && c < c1) atomicAdd(&cell[(c - c0) * pitch + r], 1u);
            }
            __syncthreads();
        }
        if (row < in.rows) {
            bool none;
            const unsigned *words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
            const T *src = static_cast<const T *>(in.data);
            for (int c = c0 + slot; c < c1; c += slots) {
                const float z = score_to_float(src[(size_t)c * in.class_stride + row]);
                unsigned *at = cell + (c - c0) * pitch + r;
                const bool ok = !none && (words == nullptr || (words[c / 32] >> (c % 32) & 1u));
                *at = __float_as_uint(adjusted(z, rules.bias != nullptr ? rules.bias[c] : 0.f, rules.shown != nullptr ? *at : 0u, ok, rules));
            }
        }
        __syncthreads();
        TopList<1> &sh = lists[wave_id()];
        for (int q = wave_id(); q < rows && row0 + q < in.rows; q += kColumnBlock / 64) {
            float v[E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int c = i * 64 + lane_id();
                v[i] = c < c1 - c0 ? __uint_as_float(cell[c * pitch + q]) : kNothing;
            }
            const size_t out_at = (size_t)(row0 + q) * chunks + tile % chunks;
            float m, s;
            sum_exponentials<1>(v, by, sh, &m, &s);
            if (lane_id() == 0) {
                if (whole) {
                    out.lse[row0 + q] = log_sum(m, s, temperature);
                } else {
                    out.lse[out_at * 2] = m;
                    out.lse[out_at * 2 + 1] = s;
                }
            }
            const int found = list_candidates<1>(v, [&](int i) { return c0 + i * 64 + lane_id(); }, k, sh);
            write_best(sh, found, k, out_at, out, [](int place) { return place; });
            wave_fence();
        }
        __syncthreads();
    }
}

// Few classes: a thread holds its row's and counts, for every one of them, those that are better.
template <typename T, int E>
__global__ __launch_bounds__(kTopBlock) void k_top_few(tgbm_scores in, tgbm_score_rules rules, int k, float temperature, TopOut out) {
    const float by = kLog2e / temperature;
    for (long row = (long)blockIdx.x * kTopBlock + threadIdx.x; row < in.rows; row += (long)gridDim.x * kTopBlock) {
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
                v[c] = adjusted(v[c], rules.bias != nullptr ? rules.bias[c] : 0.f, times[c], ok >> c & 1u, rules);
                m = fmaxf(m, v[c]);
            }
        m = reference_of(m);
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < E; ++c) s += exp2_of((v[c] - m) * by);
        out.lse[row] = log_sum(m, s, temperature);
        int listed = 0;
#pragma unroll
        for (int c = 0; c < E; ++c) {
            int better = 0;
#pragma unroll
            for (int o = 0; o < E; ++o) better += v[o] > v[c] || (v[o] == v[c] && o < c) ? 1 : 0;
            const bool in_list = v[c] > kNothing;
            listed += in_list ? 1 : 0;
            if (in_list && better < k) {
                out.values[row * k + better] = v[c];
                out.classes[row * k + better] = c;
            }
        }
        for (int j = listed; j < k; ++j) {
            out.values[row * k + j] = kNothing;
            out.classes[row * k + j] = -1;
        }
    }
}

// `per_join` parts of a row become one: places among them ascend with the class wherever scores are equal.
template <int W, int E>
__global__ __launch_bounds__(W == 1 ? kTopBlock : 64 * W) void k_top_join(int parts, int per_join, int joins, long tiles, int k, float temperature, TopOut in,
                                                                          TopOut out) {
    constexpr int kGroups = W == 1 ? kTopBlock / 64 : 1;
    __shared__ TopList<W> lists[kGroups];
    const int t = W == 1 ? lane_id() : (int)threadIdx.x, group = W == 1 ? wave_id() : 0;
    TopList<W> &sh = lists[group];
    const float by = kLog2e / temperature;
    for (long tile = (long)blockIdx.x * kGroups + group; tile < tiles; tile += (long)gridDim.x * kGroups) {
        const int first = (int)(tile % joins) * per_join, mine = min(parts - first, per_join), count = mine * k;
        const size_t from = (size_t)(tile / joins) * parts + first;
        const float *values = in.values + from * k;
        const int *classes = in.classes + from * k;
        float v[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int at = i * 64 * W + t;
            v[i] = at < count ? values[at] : kNothing;
        }
        // (every wavefront for itself: a part has one sum)
        const float *sums = in.lse + from * 2;
        float m = kNothing;
        for (int c = lane_id(); c < mine; c += 64) m = fmaxf(m, sums[c * 2 + 1] > 0.f ? sums[c * 2] : kNothing);
        m = reference_of(wave_max_f(m));
        float s = 0.f;
        for (int c = lane_id(); c < mine; c += 64) {
            const float part = sums[c * 2 + 1];
            if (part != 0.f) s += rescaled(part, sums[c * 2], m, by);
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
        if (t == 0) {
            if (joins == 1) {
                out.lse[tile] = log_sum(m, s, temperature);
            } else {
                out.lse[tile * 2] = m;
                out.lse[tile * 2 + 1] = s;
            }
        }
        const int found = list_candidates<W>(v, [&](int i) { return i * 64 * W + t; }, k, sh);
        write_best(sh, found, k, (size_t)tile, out, [&](int place) { return classes[place]; });
        group_sync<W>();
    }
}

int blocks_of(long groups) { return (int)std::max(1l, std::min(groups, 1l << 20)); }

// How a call goes: chunks of a row, and the classes of one.
struct TopPlan {
    bool few, columns;
    int chunks, chunk;
    int waves;     // classes side by side: wavefronts of a group
    int row_bits;  // rows side by side
    int per_thread;
};
constexpr int kFewClasses = 32;
constexpr int kJoinMost = 16384;  // scores that a join takes
constexpr int kGroupsWanted = 512;

TopPlan plan_top(bool columns, int classes, int rows, int k) {
    TopPlan p{};
    p.columns = columns;
    p.few = classes <= kFewClasses;
    p.chunks = 1;
    p.chunk = classes;
    if (p.few) return p;
    const int most = columns ? 1024 : 16384, least = columns ? 1024 : 2048;
    long tiles = columns ? (rows + 15) / 16 : rows;
    long chunks = (classes - 1) / most + 1;
    chunks = std::max(chunks, std::min<long>((classes - 1) / least + 1, kGroupsWanted / std::max(1l, tiles)));
    chunks = std::min(chunks, std::max<long>((classes - 1) / most + 1, kJoinMost / k));  // (one join, where it is a choice)
    p.chunk = (int)(((classes - 1) / chunks + 32) / 32 * 32);
    p.chunks = (classes - 1) / p.chunk + 1;
    if (columns) {
        p.per_thread = 1;
        while (p.per_thread * 64 < p.chunk) p.per_thread *= 2;
        p.row_bits = 4;
        while (p.row_bits < 7 && (64l * p.per_thread << (p.row_bits + 1)) <= 16384) ++p.row_bits;
    } else {
        p.waves = p.chunk <= 2048 ? 1 : p.chunk <= 8192 ? 4 : 8;
        p.per_thread = p.waves > 1 ? 32 : p.chunk <= 512 ? 8 : p.chunk <= 1024 ? 16 : 32;
    }
    return p;
}

template <typename T, int W, int E>
void top_rows(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    constexpr int kGroups = W == 1 ? kTopBlock / 64 : 1;
    const long tiles = (long)in.rows * p.chunks;
    const size_t lds = rules.shown != nullptr ? sizeof(unsigned) * (size_t)p.chunk * kGroups : 0;
    if (lds > 32 * 1024) {
        static LdsOptIn opt_in;
        opt_in({reinterpret_cast<const void *>(&k_top_rows<T, W, E>)});
    }
    k_top_rows<T, W, E><<<blocks_of((tiles - 1) / kGroups + 1), W == 1 ? kTopBlock : 64 * W, lds, s>>>(in, rules, k, temperature, out, p.chunks, p.chunk, tiles,
                                                                                                    p.chunks == 1);
}

template <typename T, int E>
void top_columns(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    const long tiles = ((long)((in.rows - 1) >> p.row_bits) + 1) * p.chunks;
    const size_t lds = sizeof(unsigned) * (size_t)p.chunk * ((1 << p.row_bits) + 1);
    static LdsOptIn opt_in;
    opt_in({reinterpret_cast<const void *>(&k_top_columns<T, E>)});
    k_top_columns<T, E><<<blocks_of(tiles), kColumnBlock, lds, s>>>(in, rules, k, temperature, out, p.chunks, p.chunk, p.row_bits, tiles, p.chunks == 1);
}

template <typename T>
void top(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    if (p.few) {
        const int blocks = blocks_of(((long)in.rows - 1) / kTopBlock + 1);
        if (in.classes <= 8) k_top_few<T, 8><<<blocks, kTopBlock, 0, s>>>(in, rules, k, temperature, out);
        else if (in.classes <= 16) k_top_few<T, 16><<<blocks, kTopBlock, 0, s>>>(in, rules, k, temperature, out);
        else k_top_few<T, 32><<<blocks, kTopBlock, 0, s>>>(in, rules, k, temperature, out);
    } else if (p.columns) {
        if (p.per_thread <= 1) top_columns<T, 1>(s, p, in, rules, k, temperature, out);
        else if (p.per_thread == 2) top_columns<T, 2>(s, p, in, rules, k, temperature, out);
        else if (p.per_thread == 4) top_columns<T, 4>(s, p, in, rules, k, temperature, out);
        else if (p.per_thread == 8) top_columns<T, 8>(s, p, in, rules, k, temperature, out);
        else top_columns<T, 16>(s, p, in, rules, k, temperature, out);
    } else if (p.waves == 8) {
        top_rows<T, 8, 32>(s, p, in, rules, k, temperature, out);
    } else if (p.waves == 4) {
        top_rows<T, 4, 32>(s, p, in, rules, k, temperature, out);
    } else if (p.per_thread == 32) {
        top_rows<T, 1, 32>(s, p, in, rules, k, temperature, out);
    } else if (p.per_thread == 16) {
        top_rows<T, 1, 16>(s, p, in, rules, k, temperature, out);
    } else {
        top_rows<T, 1, 8>(s, p, in, rules, k, temperature, out);
    }
}

template <int W, int E>
void join(hipStream_t s, int parts, int per_join, int joins, int rows, int k, float temperature, const TopOut &in, const TopOut &out) {
    constexpr int kGroups = W == 1 ? kTopBlock / 64 : 1;
    const long tiles = (long)rows * joins;
    k_top_join<W, E><<<blocks_of((tiles - 1) / kGroups + 1), W == 1 ? kTopBlock : 64 * W, 0, s>>>(parts, per_join, joins, tiles, k, temperature, in, out);
}

size_t part_bytes(size_t parts, int k) { return sizeof(float) * parts * (2 * (size_t)k + 2); }
TopOut parts_at(void *p, size_t parts, int k) {
    TopOut o;
    o.values = static_cast<float *>(p);
    o.classes = reinterpret_cast<int *>(o.values + parts * k);
    o.lse = reinterpret_cast<float *>(o.classes + parts * k);
    return o;
}
int parts_of_a_join(int k) { return std::max(2, kJoinMost / k); }

}  // namespace

size_t scores_top_workspace(bool columns, int classes, int rows, int k) {
    const TopPlan p = plan_top(columns, classes, rows, k);
    size_t bytes = 0;
    for (int parts = p.chunks; parts > 1; parts = (parts - 1) / parts_of_a_join(k) + 1) bytes += part_bytes((size_t)rows * parts, k);
    return bytes;
}

void launch_scores_top(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, float *values, int *classes, float *lse,
                       void *workspace) {
    const TopPlan p = plan_top(rows_side_by_side(in), in.classes, in.rows, k);
    const TopOut out{values, classes, lse};
    char *room = static_cast<char *>(workspace);
    auto next = [&](int parts) {
        if (parts == 1) return out;
        const TopOut o = parts_at(room, (size_t)in.rows * parts, k);
        room += part_bytes((size_t)in.rows * parts, k);
        return o;
    };
    TopOut now = next(p.chunks);
    if (in.type == TGBM_F32) top<float>(s, p, in, rules, k, temperature, now);
    else if (in.type == TGBM_F16) top<_Float16>(s, p, in, rules, k, temperature, now);
    else top<__bf16>(s, p, in, rules, k, temperature, now);
    for (int parts = p.chunks; parts > 1;) {
        const int per_join = std::min(parts, parts_of_a_join(k)), joins = (parts - 1) / per_join + 1, count = per_join * k;
        const TopOut to = next(joins);
        if (count <= 256) join<1, 4>(s, parts, per_join, joins, in.rows, k, temperature, now, to);
        else if (count <= 1024) join<1, 16>(s, parts, per_join, joins, in.rows, k, temperature, now, to);
        else if (count <= 4096) join<4, 16>(s, parts, per_join, joins, in.rows, k, temperature, now, to);
        else join<8, 32>(s, parts, per_join, joins, in.rows, k, temperature, now, to);
        now = to;
        parts = joins;
    }
}

}  // namespace tgbm
