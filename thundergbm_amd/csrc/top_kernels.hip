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

// What a group of W wavefronts shares. The list of candidates is elsewhere (Places).
template <int W>
struct TopShared {
    unsigned best[W == 1 ? 1 : W * 64];
    int first[W == 1 ? 1 : W * 64];
    float part_max[W], part_sum[W];
    int part[W];
    int count, exact, at_most;
    unsigned bound;
};

// The list: candidate e is the ordered score base[2 * e * stride] and the complement of its place behind it; larger is better.
struct Places {
    unsigned *base;
    int stride, room;
    __device__ __forceinline__ void put(int e, unsigned score, int place) const {
        base[(size_t)(2 * e) * stride] = score;
        base[(size_t)(2 * e + 1) * stride] = (unsigned)~place;
    }
    __device__ __forceinline__ unsigned score(int e) const { return base[(size_t)(2 * e) * stride]; }
    __device__ __forceinline__ unsigned place(int e) const { return base[(size_t)(2 * e + 1) * stride]; }
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
    if (count_from(b, kLeast) <= limit) return kLeast;
    // bisection between the least and the largest of them
    float most = kNothing, least = -kNothing;
#pragma unroll
    for (int j = 0; j < M; ++j) {
        most = fmaxf(most, from_ordered(b[j]));
        least = fminf(least, b[j] >= kLeast ? from_ordered(b[j]) : -kNothing);
    }
    unsigned lo = ordered(-wave_max_f(-least)), hi = ordered(wave_max_f(most)) + 1;
    if (count_from(b, hi - 1) > limit) lo = hi - 1;  // (many are the largest)
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

// Over all threads of the group.
template <int W>
__device__ __forceinline__ int group_sum(int n, TopShared<W> &sh) {
    n = wave_sum_i(n);
    if constexpr (W == 1) return n;
    __syncthreads();
    sh.part[wave_id()] = n;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < W; ++w) all += sh.part[w];
    return all;
}

// Where the scores of a thread lie: v[i] at base + i / V * step + i % V, the last of N at `extra` where it is apart from them.
template <int N, int V, bool EXTRA>
struct Layout {
    int base, step, extra;
    __device__ __forceinline__ int at(int i) const { return EXTRA && i == N - 1 ? extra : base + i / V * step + i % V; }
    // (with a constant i: at(i) <= most without a register for every at(i))
    __device__ __forceinline__ bool up_to(int i, int most) const { return EXTRA && i == N - 1 ? extra <= most : base <= most - (i / V * step + i % V); }
};

// Keeps the compiler from working out all of a loop's conditions or addresses ahead of it, in registers that it does not have.
__device__ __forceinline__ unsigned one_by_one(unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
}

__device__ __forceinline__ float one_by_one(float v) {
    asm volatile("" : "+v"(v));
    return v;
}

template <int E>
__device__ __forceinline__ float best_of(const float (&v)[E]) {
    float best = kNothing;
#pragma unroll
    for (int i = 0; i < E; ++i) best = fmaxf(best, v[i]);
    return best;
}

// Writes the scores that `mine` marks (bit i: v[i]) behind those of the threads before, and returns how many the group has, the
// list's room being there or not.
template <int W, int E, typename At>
__device__ __forceinline__ int put_marked(const float (&v)[E], unsigned mine, At at, TopShared<W> &sh, const Places &list) {
    const int scan = wave_scan_i(__popc(mine));
    int total = __shfl(scan, 63), to = scan - __popc(mine);
    if constexpr (W > 1) {
        int base = 0;
        if (lane_id() == 0) base = atomicAdd(&sh.count, total);
        to += __shfl(base, 0);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        mine = one_by_one(mine);
        if (mine >> i & 1u) {
            if (to < list.room) list.put(to, ordered(one_by_one(v[i])), at.at(i));
            ++to;
        }
    }
    group_sync<W>();
    if constexpr (W > 1) total = sh.count;
    return total;
}

// The candidates of the group's k best, as many as are returned, the same in all threads. at: a Layout, whose places
// ascend with i; best: the thread's largest. Every thread of the group comes here. The list holds at least k.
template <int W, int E, typename At>
__device__ __forceinline__ int list_candidates(const float (&v)[E], float best, At at, int k, TopShared<W> &sh, const Places &list) {
    const int lane = lane_id(), t = W == 1 ? lane : (int)threadIdx.x;
    const int limit = k + max(4, k / 4);
    unsigned bound;
    int exact;
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
    const float least = from_ordered(bound);
    unsigned mine = 0;
    if (!exact) {  // (the same in all threads)
#pragma unroll
        for (int i = 0; i < E; ++i) mine |= (v[i] >= least ? 1u : 0u) << i;
    } else {
        int first = INT_MAX, at_most;
#pragma unroll
        for (int i = E - 1; i >= 0; --i) first = v[i] == least ? i : first;
        first = best == least ? at.at(first) : INT_MAX;
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
#pragma unroll
        for (int i = 0; i < E; ++i) mine |= (v[i] > least || (v[i] == least && at.up_to(i, at_most)) ? 1u : 0u) << i;
    }
    const int total = put_marked<W>(v, mine, at, sh, list);
    if (total <= list.room) return total;
    // The best scores lie together in few threads: the exact k-th one by bisection over all of them.
    unsigned lo = bound, hi = 0xff800001u;  // (one past infinity)
    while (hi - lo > 1) {
        const unsigned mid = lo + (hi - lo) / 2;
        const float f = from_ordered(mid);
        int n = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) n += v[i] >= f ? 1 : 0;
        if (group_sum<W>(n, sh) >= k) lo = mid;
        else hi = mid;
    }
    const float equal = from_ordered(lo);
    int above = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) above += v[i] > equal ? 1 : 0;
    const int need = k - group_sum<W>(above, sh);
    int p_lo = -1, p_hi = INT_MAX - 1;
    while (p_hi - p_lo > 1) {
        const int mid = p_lo + (p_hi - p_lo) / 2;
        const float now = one_by_one(equal);
        int n = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) n += v[i] == now && at.up_to(i, mid) ? 1 : 0;
        if (group_sum<W>(n, sh) >= need) p_hi = mid;
        else p_lo = mid;
    }
    mine = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) mine |= (v[i] > equal || (v[i] == equal && at.up_to(i, p_hi)) ? 1u : 0u) << i;
    if constexpr (W > 1) {
        __syncthreads();
        if (t == 0) sh.count = 0;
        __syncthreads();
    }
    return put_marked<W>(v, mine, at, sh, list);
}

// Where a row's (or a chunk's) best classes go.
struct TopOut {
    float *values;  // [][k]
    int *classes;
    float *lse;     // [] of rows, or the largest score and the sum of chunks
};

// The candidates in order. class_at(place): the class.
template <int W, typename Class>
__device__ __forceinline__ void write_best(const Places &list, int found, int k, size_t slot, const TopOut &out, Class class_at) {
    const int t = W == 1 ? lane_id() : (int)threadIdx.x;
    for (int j = t; j < found; j += 64 * W) {
        const unsigned score = list.score(j), place = list.place(j);
        int better = 0;
        for (int o = 0; o < found; ++o) {
            const unsigned s = list.score(o);
            better += s > score || (s == score && list.place(o) > place) ? 1 : 0;
        }
        if (better < k) {
            out.values[slot * k + better] = from_ordered(score);
            out.classes[slot * k + better] = class_at((int)~place);
        }
    }
    for (int j = found + t; j < k; j += 64 * W) {
        out.values[slot * k + j] = kNothing;
        out.classes[slot * k + j] = -1;
    }
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float reference_of(float m) { return fabsf(m) <= FLT_MAX ? m : 0.f; }
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// A sum to the reference `from` as one to `to`; an infinite one stays infinite.
__device__ __forceinline__ float rescaled(float sum, float from, float to, float by) {
    return sum <= FLT_MAX ? sum * exp2_of((from - to) * by) : sum;
}

// The largest of the group's scores (0 where it is no number) and the sum of exp((v - it) / temperature). A NaN makes the sum
// NaN, an infinity makes it infinite. best: the thread's largest.
template <int W, int E>
__device__ __forceinline__ void sum_exponentials(const float (&v)[E], float best, float by, TopShared<W> &sh, float *reference, float *sum) {
    float m = reference_of(wave_max_f(best));
    float part[4] = {0.f, 0.f, 0.f, 0.f};
    if (fabsf(m) < 1e30f) {
        // one multiply-add for the argument; what the product m * by was rounded by is put right in the sum
        const float shift = m * by, off = __builtin_fmaf(m, by, -shift);
#pragma unroll
        for (int i = 0; i < E; ++i) part[i % 4] += exp2_of(__builtin_fmaf(v[i], by, -shift));
        const float s = (part[0] + part[1]) + (part[2] + part[3]);
        part[0] = s <= FLT_MAX ? __builtin_fmaf(s, -off * kLn2, s) : s;
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) part[i % 4] += exp2_of((v[i] - m) * by);
        part[0] = (part[0] + part[1]) + (part[2] + part[3]);
    }
    float s = part[0];
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

// Classes side by side: E scores of a thread, by vectors of 16 bytes, which need not lie on such an address.
template <typename T>
struct Vector {
    static constexpr int kOf = 16 / (int)sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};
typedef float Float4 __attribute__((ext_vector_type(4), aligned(4)));

// LDS of a group's lists of shown classes: a bit for each class of the chunk, and how often where the bit is set.
template <int W>
__device__ __forceinline__ void count_shown(const tgbm_score_rules &rules, long long b, long long e, int c0, int c1, int chunk, unsigned *bits, unsigned *times) {
    const int t = W == 1 ? lane_id() : (int)threadIdx.x;
    for (int w = t; w < chunk / 32; w += 64 * W) bits[w] = 0;
    group_sync<W>();
    for (long long i = b + t; i < e; i += 64 * W) {
        const int c = rules.shown[i];
        if (c < c0 || c >= c1) continue;
        times[c - c0] = 0;
        atomicOr(&bits[(c - c0) / 32], 1u << ((c - c0) % 32));
    }
    group_sync<W>();
    for (long long i = b + t; i < e; i += 64 * W) {
        const int c = rules.shown[i];
        if (c >= c0 && c < c1) atomicAdd(&times[c - c0], 1u);
    }
    group_sync<W>();
}

// A group of W wavefronts takes chunk `tile % chunks` (a multiple of 32 classes) of a row; with W = 1 there are four groups to a
// workgroup. A thread has E scores in whole vectors, and one of what is left behind the last vector. RULES: there may be any. LDS: the lists of candidates,
// then, where classes were shown, bits and times.
template <typename T, int W, int E, bool RULES>
__global__ __launch_bounds__(W == 1 ? kTopBlock : 64 * W, 6) void k_top_rows(tgbm_scores in, tgbm_score_rules rules, int k, float temperature, TopOut out,
                                                                          int chunks, int chunk, long tiles, bool whole) {
    constexpr int kGroups = W == 1 ? kTopBlock / 64 : 1, kRoom = W == 1 ? 256 : 1024;
    __shared__ TopShared<W> shared[kGroups];
    __shared__ unsigned candidates[kGroups][2 * kRoom];
    extern __shared__ unsigned shown_lds[];
    constexpr int V = Vector<T>::kOf, N = E + 1, kStep = 64 * W * V;
    const int t = W == 1 ? lane_id() : (int)threadIdx.x, group = W == 1 ? wave_id() : 0;
    TopShared<W> &sh = shared[group];
    const Places list{candidates[group], 1, kRoom};
    unsigned *bits = shown_lds + (size_t)group * (chunk + chunk / 32), *times = bits + chunk / 32;
    const float by = kLog2e / temperature;
    for (long tile = (long)blockIdx.x * kGroups + group; tile < tiles; tile += (long)gridDim.x * kGroups) {
        const long row = tile / chunks;
        const int c0 = (int)(tile % chunks) * chunk, size = min(in.classes - c0, chunk), whole_size = size / V * V;
        // (a thread's places are worked out where they are used, not kept over the tiles)
        const Layout<N, V, true> at{(int)one_by_one((unsigned)t * V), kStep, (int)one_by_one((unsigned)(whole_size + t))};
        const T *src = static_cast<const T *>(in.data) + (size_t)row * in.row_stride + c0;
        float v[N];
        {
            typename Vector<T>::type x[E / V];
#pragma unroll
            for (int g = 0; g < E / V; ++g) {
                x[g] = (T)kNothing;
                if (at.base < whole_size - g * kStep) x[g] = *reinterpret_cast<const typename Vector<T>::type *>(src + at.base + g * kStep);
            }
            v[E] = t < size - whole_size ? score_to_float(src[at.extra]) : kNothing;
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = score_to_float(x[i / V][i % V]);
        }
        if constexpr (RULES) {
            if (rules.bias != nullptr) {
                const float *bias = rules.bias + c0;
#pragma unroll
                for (int g = 0; g < E / V; ++g)
                    if (at.base < whole_size - g * kStep) {
#pragma unroll
                        for (int j = 0; j < V; j += 4) {
                            const Float4 b = *reinterpret_cast<const Float4 *>(bias + at.base + g * kStep + j);
#pragma unroll
                            for (int q = 0; q < 4; ++q) v[g * V + j + q] += b[q];
                        }
                    }
                if (t < size - whole_size) v[E] += bias[at.extra];
            }
            bool none;
            const unsigned *words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
            if (rules.shown != nullptr) {
                long long b, e;
                shown_range(rules, row, &b, &e);
                if (b < e) {  // (the same for the group)
                    count_shown<W>(rules, b, e, c0, c0 + size, chunk, bits, times);
                    unsigned held = 0;
#pragma unroll
                    for (int g = 0; g < E / V; ++g) {
                        const int c = at.base + g * kStep;
                        if (c < whole_size) held |= (bits[c / 32] >> (c % 32) & ((1u << V) - 1u)) << (g * V);
                    }
                    if (t < size - whole_size) held |= (bits[at.extra / 32] >> (at.extra % 32) & 1u) << E;
                    // few of a thread's scores are: one at a time, from the start (its register has no number that a loop can use)
                    while (__any(held != 0)) {
                        const bool now = held != 0;
                        const int i = now ? __ffs((int)held) - 1 : 0;
                        float s = 0.f;
                        if (now) {
                            const int c = at.at(i);
                            s = adjusted(score_to_float(src[c]), rules.bias != nullptr ? rules.bias[c0 + c] : 0.f, times[c], true, rules);
                        }
                        held &= held - 1;
#pragma unroll
                        for (int j = 0; j < N; ++j) v[j] = now && j == i ? s : v[j];
                    }
                }
            }
            if (words != nullptr || none) {
#pragma unroll
                for (int g = 0; g < E / V; ++g) {
                    const int c = at.base + g * kStep;
                    const unsigned ok = words != nullptr && c < whole_size ? words[(c0 + c) / 32] >> (c % 32) : 0u;
#pragma unroll
                    for (int j = 0; j < V; ++j) v[g * V + j] = ok >> j & 1u ? v[g * V + j] : kNothing;
                }
                const bool ok = words != nullptr && t < size - whole_size && (words[(c0 + at.extra) / 32] >> (at.extra % 32) & 1u);
                v[E] = ok ? v[E] : kNothing;
            }
        }
        const float best = best_of(v);
        float m, s;
        sum_exponentials<W>(v, best, by, sh, &m, &s);
        if (t == 0) {
            if (whole) {
                out.lse[row] = log_sum(m, s, temperature);
            } else {
                out.lse[tile * 2] = m;
                out.lse[tile * 2 + 1] = s;
            }
        }
        const int found = list_candidates<W>(v, best, at, k, sh, list);
        write_best<W>(list, found, k, (size_t)tile, out, [&](int p) { return c0 + p; });
        group_sync<W>();
    }
}

// Rows side by side: a workgroup brings `rows` rows of a chunk (a multiple of 32, at most 64 * E classes) into LDS, class by class, eight
// classes of a row to a thread at a time, and its wavefronts take a row each. A row's column is its list of candidates once
// its scores are in registers. LDS: [tile_classes][rows + 1] scores, then, where classes were shown, [rows][chunk / 32] bits.
constexpr int kColumnBlock = 1024;
template <typename T, int E, bool RULES>
__global__ __launch_bounds__(kColumnBlock, 8) void k_top_columns(tgbm_scores in, tgbm_score_rules rules, int k, float temperature, TopOut out, int chunks,
                                                                 int chunk, int row_bits, int tile_classes, long tiles, bool whole) {
    __shared__ TopShared<1> sh;  // (nothing of it is used by one wavefront)
    extern __shared__ unsigned cell[];
    const int rows = 1 << row_bits, pitch = rows + 1;
    unsigned *const bits = cell + (size_t)tile_classes * pitch;
    const float by = kLog2e / temperature;
    const int r = threadIdx.x & (rows - 1), slot = threadIdx.x >> row_bits, slots = kColumnBlock >> row_bits;
    const T *src = static_cast<const T *>(in.data);
    for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long row0 = tile / chunks * rows, row = row0 + r;
        const int c0 = (int)(tile % chunks) * chunk, c1 = min(in.classes, c0 + chunk);
        unsigned *const my_bits = bits + r * (chunk / 32);
        bool counted = false;
        if constexpr (RULES) {
            counted = rules.shown != nullptr;
            if (counted) {
                for (int i = threadIdx.x; i < rows * (chunk / 32); i += kColumnBlock) bits[i] = 0;
                __syncthreads();
                long long b = 0, e = 0;
                if (row < in.rows) shown_range(rules, row, &b, &e);
                for (long long i = b + slot; i < e; i += slots) {
                    const int c = rules.shown[i] - c0;
                    if (c < 0 || c >= c1 - c0) continue;
                    cell[c * pitch + r] = 0;
                    atomicOr(&my_bits[c / 32], 1u << (c % 32));
                }
                __syncthreads();
                for (long long i = b + slot; i < e; i += slots) {
                    const int c = rules.shown[i] - c0;
                    if (c >= 0 && c < c1 - c0) atomicAdd(&cell[c * pitch + r], 1u);
                }
                __syncthreads();
            }
        }
        if (row < in.rows) {
            bool none = false;
            const unsigned *words = RULES ? allowed_words(rules, row, (in.classes + 31) / 32, &none) : nullptr;
            for (int c = slot * 8; c < c1 - c0; c += slots * 8) {
                const T *from = src + (size_t)(c0 + c) * in.class_stride + row;
                unsigned *to = cell + c * pitch + r;
                float z[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] = c + j < c1 - c0 ? score_to_float(from[(size_t)j * in.class_stride]) : kNothing;
                if constexpr (!RULES) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (c + j < c1 - c0) to[j * pitch] = __float_as_uint(z[j]);
                } else {
                    unsigned ok = none ? 0u : words != nullptr ? words[(c0 + c) / 32] >> ((c0 + c) % 32) : ~0u;
                    unsigned held = counted ? my_bits[c / 32] >> (c % 32) & 0xffu : 0u;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (c + j < c1 - c0) {
                            const float s = rules.bias != nullptr ? z[j] + rules.bias[c0 + c + j] : z[j];
                            if (!(held >> j & 1u)) to[j * pitch] = __float_as_uint(ok >> j & 1u ? s : kNothing);
                        }
                    while (held != 0) {
                        const int j = __ffs((int)held) - 1;
                        held &= held - 1;
                        to[j * pitch] = __float_as_uint(adjusted(score_to_float(from[(size_t)j * in.class_stride]), rules.bias != nullptr ? rules.bias[c0 + c + j] : 0.f,
                                                                 to[j * pitch], ok >> j & 1u, rules));
                    }
                }
            }
        }
        __syncthreads();
        for (int q = wave_id(); q < rows && row0 + q < in.rows; q += kColumnBlock / 64) {
            const int lane = (int)one_by_one((unsigned)lane_id());  // (places are worked out where they are used)
            const unsigned *from = cell + lane * pitch + q;
            float v[E];
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = lane < c1 - c0 - i * 64 ? __uint_as_float(from[i * 64 * pitch]) : kNothing;
            const size_t out_at = (size_t)(row0 + q) * chunks + tile % chunks;
            const float best = best_of(v);
            float m, s;
            sum_exponentials<1>(v, best, by, sh, &m, &s);
            if (lane_id() == 0) {
                if (whole) {
                    out.lse[row0 + q] = log_sum(m, s, temperature);
                } else {
                    out.lse[out_at * 2] = m;
                    out.lse[out_at * 2 + 1] = s;
                }
            }
            wave_fence();
            const Places list{cell + q, pitch, tile_classes / 2};
            const int found = list_candidates<1>(v, best, Layout<E, 1, false>{lane, 64, 0}, k, sh, list);
            write_best<1>(list, found, k, out_at, out, [&](int p) { return c0 + p; });
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
    constexpr int kRoom = W == 1 ? 256 : 1024;
    __shared__ TopShared<W> shared[kGroups];
    __shared__ unsigned candidates[kGroups][2 * kRoom];
    const int t = W == 1 ? lane_id() : (int)threadIdx.x, group = W == 1 ? wave_id() : 0;
    TopShared<W> &sh = shared[group];
    const Places list{candidates[group], 1, kRoom};
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
        const int found = list_candidates<W>(v, best_of(v), Layout<E, 1, false>{(int)one_by_one((unsigned)t), 64 * W, 0}, k, sh, list);
        write_best<W>(list, found, k, (size_t)tile, out, [&](int p) { return classes[p]; });
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
    int tile_classes;
    int per_thread;
};
constexpr int kFewClasses = 32;
constexpr int kRowScores = 24;  // classes side by side: the most that a thread has in whole vectors
constexpr int kJoinMost = 16384;  // scores that a join takes
constexpr int kGroupsWanted = 512;

TopPlan plan_top(bool columns, int classes, int rows, int k) {
    TopPlan p{};
    p.columns = columns;
    p.few = classes <= kFewClasses;
    p.chunks = 1;
    p.chunk = classes;
    if (p.few) return p;
    const int most = columns ? 1024 : 8 * 64 * kRowScores, least = columns ? 1024 : 64 * kRowScores;
    long tiles = columns ? (rows + 15) / 16 : rows;
    long chunks = (classes - 1) / most + 1;
    chunks = std::max(chunks, std::min<long>((classes - 1) / least + 1, kGroupsWanted / std::max(1l, tiles)));
    chunks = std::min(chunks, std::max<long>((classes - 1) / most + 1, kJoinMost / k));  // (one join, where it is a choice)
    p.chunk = (int)(((classes - 1) / chunks + 32) / 32 * 32);
    p.chunks = (classes - 1) / p.chunk + 1;
    if (columns) {
        p.per_thread = 1;
        while (p.per_thread * 64 < p.chunk) p.per_thread *= 2;
        p.tile_classes = std::max(p.chunk, 2 * kTopMost);  // (a list's room)
        p.row_bits = 4;
        while (p.row_bits < 6 && (p.tile_classes << (p.row_bits + 1)) <= 16384) ++p.row_bits;
    } else {
        p.waves = p.chunk <= 64 * kRowScores ? 1 : p.chunk <= 256 * kRowScores ? 4 : 8;
        p.per_thread = p.waves > 1 ? kRowScores : p.chunk <= 512 ? 8 : p.chunk <= 1024 ? 16 : kRowScores;
    }
    return p;
}

template <typename T, int W, int E, bool RULES>
void top_rows(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    constexpr int kGroups = W == 1 ? kTopBlock / 64 : 1;
    const long tiles = (long)in.rows * p.chunks;
    const size_t lds = rules.shown != nullptr ? sizeof(unsigned) * (size_t)(p.chunk + p.chunk / 32) * kGroups : 0;
    if (lds > 32 * 1024) {
        static LdsOptIn opt_in;
        opt_in({reinterpret_cast<const void *>(&k_top_rows<T, W, E, RULES>)});
    }
    k_top_rows<T, W, E, RULES><<<blocks_of((tiles - 1) / kGroups + 1), W == 1 ? kTopBlock : 64 * W, lds, s>>>(in, rules, k, temperature, out, p.chunks, p.chunk,
                                                                                                           tiles, p.chunks == 1);
}

template <typename T, int E, bool RULES>
void top_columns(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    const long tiles = ((long)((in.rows - 1) >> p.row_bits) + 1) * p.chunks;
    const size_t lds = sizeof(unsigned) * ((size_t)p.tile_classes * ((1 << p.row_bits) + 1) + (rules.shown != nullptr ? (size_t)p.chunk / 32 << p.row_bits : 0));
    static LdsOptIn opt_in;
    opt_in({reinterpret_cast<const void *>(&k_top_columns<T, E, RULES>)});
    k_top_columns<T, E, RULES><<<blocks_of(tiles), kColumnBlock, lds, s>>>(in, rules, k, temperature, out, p.chunks, p.chunk, p.row_bits, p.tile_classes, tiles,
                                                                      p.chunks == 1);
}

template <typename T, bool RULES>
void top(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    if (p.few) {
        const int blocks = blocks_of(((long)in.rows - 1) / kTopBlock + 1);
        if (in.classes <= 8) k_top_few<T, 8><<<blocks, kTopBlock, 0, s>>>(in, rules, k, temperature, out);
        else if (in.classes <= 16) k_top_few<T, 16><<<blocks, kTopBlock, 0, s>>>(in, rules, k, temperature, out);
        else k_top_few<T, 32><<<blocks, kTopBlock, 0, s>>>(in, rules, k, temperature, out);
    } else if (p.columns) {
        constexpr bool kRules = RULES || sizeof(T) != 4;
        if (p.per_thread <= 2) top_columns<T, 2, kRules>(s, p, in, rules, k, temperature, out);
        else if (p.per_thread == 4) top_columns<T, 4, kRules>(s, p, in, rules, k, temperature, out);
        else if (p.per_thread == 8) top_columns<T, 8, kRules>(s, p, in, rules, k, temperature, out);
        else top_columns<T, 16, kRules>(s, p, in, rules, k, temperature, out);
    } else if (p.waves == 8) {
        top_rows<T, 8, kRowScores, RULES>(s, p, in, rules, k, temperature, out);
    } else if (p.waves == 4) {
        top_rows<T, 4, kRowScores, RULES>(s, p, in, rules, k, temperature, out);
    } else if (p.per_thread == kRowScores) {
        top_rows<T, 1, kRowScores, RULES>(s, p, in, rules, k, temperature, out);
    } else if (p.per_thread == 16) {
        top_rows<T, 1, 16, RULES>(s, p, in, rules, k, temperature, out);
    } else {
        top_rows<T, 1, 8, RULES>(s, p, in, rules, k, temperature, out);
    }
}

template <typename T>
void top_any(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    if (rules.bias != nullptr || rules.allowed != nullptr || rules.shown != nullptr) top<T, true>(s, p, in, rules, k, temperature, out);
    else top<T, false>(s, p, in, rules, k, temperature, out);
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
    if (in.type == TGBM_F32) top_any<float>(s, p, in, rules, k, temperature, now);
    else if (in.type == TGBM_F16) top_any<_Float16>(s, p, in, rules, k, temperature, now);
    else top_any<__bf16>(s, p, in, rules, k, temperature, now);
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
