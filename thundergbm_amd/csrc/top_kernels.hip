// tgbm_scores_top: the k best classes of every row, and the logarithm of the sum of the exponentials, in one read of the scores.
//
// A group of wavefronts holds a row, or a chunk of it, in registers. The k-th largest of the threads' own maxima is a lower
// bound of the k-th largest score: the k threads above it hold one such score each. Any bound that between k and a few more
// maxima reach will do, so it is found by bisection over the maxima (ballots, no memory). Only the threads whose maximum reaches it, about k of
// them, can hold a score that does: they lay theirs out in LDS, and what reaches the bound - a thread rarely holds two of the best - is listed
// and put in order by counting. Equal scores are told apart by their class, so that no more than k threads are left where
// many are equal. Where the list overflows all the same, the k-th score is bisected among those laid out. Rows that go by chunks
// leave k scores of each, and a launch of its own makes the same choice among those.
//
// 2048 x 65537 bfloat16, k 64: 88 us by the profiler and 9 for the join of three parts a row, 92 together where calls follow one another (the memory's share is
// 54); 877 vector instructions of a wavefront, three quarters of that time, for 48 scores of a lane: an exponential of each, three looks at it (largest, sum, bound),
// the search and the list. 50021 x 1000 float32, rows side by side, k 10, sets and lists: 106 us where the memory's share is 42; 806 vector and 510
// scalar instructions to a row of 16 scores a lane, most of them the same whatever the scores: the search, the list and its order. What a longer list costs
// short rows stands at kFewBestRows and in k_top_rows.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

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

// What a group of W wavefronts shares.
template <int W>
struct TopShared {
    unsigned best[W == 1 ? 1 : W * 64];
    int first[W == 1 ? 1 : W * 64];
    float part_max[W], part_sum[W];
    int part[W];
    int threads, listed, exact, at_most;
    unsigned bound;
};
constexpr int kListRoom = 192;                            // candidates: more than kTopMost
constexpr int kMostThreads = kTopMost + kTopMost / 4;       // that lay their scores out
__host__ __device__ constexpr int candidates_wanted(int k) { return k + (k / 4 > 4 ? k / 4 : 4); }

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

// Where the scores of thread t lie: score i at t * V + i / V * step + i % V, the last of N at extra + t where it is apart from them.
template <int N_, int V, bool EXTRA>
struct Layout {
    static constexpr int N = N_;
    int step, extra;
    __device__ __forceinline__ int at(int t, int i) const { return EXTRA && i == N - 1 ? extra + t : t * V + i / V * step + i % V; }
};
// As the former, or one by one: score i of thread t at t + i * 64 * W.
template <int N_, int V, int W>
struct DealtLayout {
    static constexpr int N = N_;
    int extra;
    bool dealt;
    __device__ __forceinline__ int at(int t, int i) const { return dealt ? t + i * 64 * W : Layout<N, V, true>{64 * W * V, extra}.at(t, i); }
};
// One wavefront, whose lanes count as several threads each, thread t = lane + 64 * part: lane + 64 * (part * N + i).
template <int N_>
struct LaneParts {
    static constexpr int N = N_;
    __device__ __forceinline__ int at(int t, int i) const { return (t & 63) + ((t >> 6) * N + i) * 64; }
};

// Keeps the compiler from working out all of a loop's conditions or addresses ahead of it, in registers that it does not have.
__device__ __forceinline__ unsigned one_by_one(unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
}

// A thread's scores: as they are worked out,
template <int N>
struct Held {
    float v[N];
    __device__ __forceinline__ float operator[](int i) const { return v[i]; }
    __device__ __forceinline__ void look_again() {}
    // N words of 32 bits, and a score of those
    static constexpr int kWords = N;
    __device__ __forceinline__ unsigned word(int i) const { return __float_as_uint(v[i]); }
    static __device__ __forceinline__ float score_of(const unsigned *words, int i) { return __uint_as_float(words[i]); }
};
// or as they were read, two of 16 bits to a register, and unpacked wherever they are looked at.
template <typename T, int E>
struct HeldPairs {
    unsigned pair[E / 2];
    float last;
    static constexpr int kWords = E / 2 + 1;
    static __device__ __forceinline__ float half(unsigned pair, int i) {
        if constexpr (std::is_same<T, __bf16>::value) return __uint_as_float(i % 2 ? pair & 0xffff0000u : pair << 16);
        else return (float)__builtin_bit_cast(_Float16, (unsigned short)(pair >> (i % 2 * 16)));
    }
    __device__ __forceinline__ float operator[](int i) const { return i == E ? last : half(pair[i / 2], i); }
    __device__ __forceinline__ unsigned word(int i) const { return i == E / 2 ? __float_as_uint(last) : pair[i]; }
    static __device__ __forceinline__ float score_of(const unsigned *words, int i) { return i == E ? __uint_as_float(words[E / 2]) : half(words[i / 2], i); }
    // (the compiler is not to keep what it has unpacked so far)
    __device__ __forceinline__ void look_again() {
#pragma unroll
        for (int i = 0; i < E / 2; ++i) asm volatile("" : "+v"(pair[i]));
    }
};

template <int N, typename Scores>
__device__ __forceinline__ float best_of(const Scores &v) {
    float best = kNothing;
#pragma unroll
    for (int i = 0; i < N; ++i) best = fmaxf(best, v[i]);
    return best;
}

// Where a row's (or a chunk's) best classes go.
struct TopOut {
    float *values;  // [][k]
    int *classes;
    float *lse;     // [] of rows, or the largest score and the sum of chunks
};

// LDS of a group: the candidates, ordered score in front of the complement of the place (larger is better), and how many of them are
// better; the scores of the threads that reach the bound, the words of the q-th of them from q * kWords on, and who they are.
template <int W, typename Scores>
struct LaidOut {
    static constexpr int kRoom = kListRoom, kWords = Scores::kWords;
    static constexpr int kThreads = W == 1 ? 64 : kMostThreads;
    __align__(16) unsigned word[kThreads * kWords];
    unsigned short owner[kThreads];
    unsigned long long key[kListRoom];
    int better[W == 1 ? 1 : kListRoom];

    __device__ __forceinline__ void put(int q, int t, const Scores &v, int) {
        owner[q] = (unsigned short)t;
#pragma unroll
        for (int i = 0; i < kWords; ++i) word[q * kWords + i] = v.word(i);
    }
    template <typename At>
    __device__ __forceinline__ float get(int q, int i, const At &) const { return Scores::score_of(word + q * kWords, i); }
    template <typename At>
    __device__ __forceinline__ int place(int q, int i, const At &at) const { return at.at(owner[q], i); }
    __device__ __forceinline__ float laid_out(int q, int i, int) const { return Scores::score_of(word + q * kWords, i); }
    __device__ __forceinline__ void list(int to, float s, int p) {
        key[to] = (unsigned long long)ordered(s) << 32 | (unsigned)~p;
        if constexpr (W > 1) better[to] = 0;
    }
    __device__ __forceinline__ unsigned long long listed(int j) const { return key[j]; }
};
// A row's column of a tile holds the scores already, by their places.
struct ColumnLists {
    static constexpr int kRoom = 160;
    unsigned char owner[kMostThreads];
    unsigned short entry[kRoom];
};
struct Column {
    static constexpr int kRoom = ColumnLists::kRoom;
    const unsigned *column;
    int pitch, lines;
    ColumnLists &lists;
    __device__ __forceinline__ float at_line(int p) const { return __uint_as_float(column[p * pitch]); }
    template <typename Scores>
    __device__ __forceinline__ void put(int q, int t, const Scores &, int) { lists.owner[q] = (unsigned char)t; }
    template <typename At>
    __device__ __forceinline__ float get(int q, int i, const At &at) const {
        const int p = at.at(lists.owner[q], i);
        return p < lines ? at_line(p) : kNothing;
    }
    template <typename At>
    __device__ __forceinline__ int place(int q, int i, const At &at) const { return at.at(lists.owner[q], i); }
    __device__ __forceinline__ float laid_out(int, int, int p) const { return at_line(p); }
    __device__ __forceinline__ void list(int to, float, int p) { lists.entry[to] = (unsigned short)p; }
    __device__ __forceinline__ unsigned long long listed(int j) const {
        const int p = lists.entry[j];
        return (unsigned long long)ordered(at_line(p)) << 32 | (unsigned)~p;
    }
};

// The k best of the group's scores go to `slot` of the output, in order. v: M times N scores, each N of them a thread's to the
// choice (M is 1 but for one wavefront); best: the largest of each; at: where they lie, ascending with i; room: LDS of the group; class_at(place): the class; meanwhile():
// what the last of several wavefronts does while the first one looks for the bound, behind a barrier. Every thread of the group comes here.
template <int W, int M, int N, typename Scores, typename At, typename Room, typename Class, typename Meanwhile>
__device__ __forceinline__ void write_top(Scores &v, const float (&best)[M], const At &at, int k, TopShared<W> &sh, Room &room, size_t slot,
                                          const TopOut &out, Class class_at, Meanwhile meanwhile) {
    static_assert(M == 1 || W == 1);
    const int lane = lane_id(), t = W == 1 ? lane : (int)threadIdx.x;
    unsigned bound;
    int exact, at_most = INT_MAX;
    if constexpr (W == 1) {
        unsigned b[M];
#pragma unroll
        for (int j = 0; j < M; ++j) b[j] = ordered(best[j]);
        bound = find_bound(b, k, candidates_wanted(k), &exact);
    } else {
        sh.best[t] = ordered(best[0]);
        if (t == 0) sh.threads = sh.listed = 0;
        __syncthreads();
        if (wave_id() == 0) {
            unsigned b[W];
#pragma unroll
            for (int j = 0; j < W; ++j) b[j] = sh.best[j * 64 + lane];
            int e;
            const unsigned found = find_bound(b, k, candidates_wanted(k), &e);
            if (lane == 0) {
                sh.bound = found;
                sh.exact = e;
            }
        }
        if (wave_id() == W - 1) meanwhile();
        __syncthreads();
        bound = sh.bound;
        exact = sh.exact;
    }
    const float least = from_ordered(bound);
    int first[M];
#pragma unroll
    for (int j = 0; j < M; ++j) first[j] = INT_MAX;
    if (exact) {  // (the same in all threads)
        v.look_again();
#pragma unroll
        for (int j = 0; j < M; ++j) {
#pragma unroll
            for (int i = N - 1; i >= 0; --i) first[j] = v[j * N + i] == least ? i : first[j];
            first[j] = best[j] == least ? at.at(t + 64 * j, first[j]) : INT_MAX;
        }
        if constexpr (W == 1) {
            unsigned b[M];
#pragma unroll
            for (int j = 0; j < M; ++j) b[j] = ordered(best[j]);
            at_most = find_place(first, k - count_from(b, bound + 1));
        } else {
            sh.first[t] = first[0];
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
    // the candidates: a bit for each score that reaches the bound
    v.look_again();
    constexpr int kWords = (M * N + 31) / 32;
    unsigned mine[kWords];
#pragma unroll
    for (int w = 0; w < kWords; ++w) mine[w] = 0;
    if (!exact) {
#pragma unroll
        for (int i = M * N - 1; i >= 0; --i) mine[i / 32] = mine[i / 32] + mine[i / 32] + (v[i] >= least ? 1u : 0u);
    } else {
#pragma unroll
        for (int i = M * N - 1; i >= 0; --i)
            mine[i / 32] = mine[i / 32] + mine[i / 32] + (v[i] > least || (v[i] == least && at.at(t + 64 * (i / N), i % N) <= at_most) ? 1u : 0u);
    }
    // their threads - at most candidates_wanted(k), or k where the bound is exact - lay their scores out and list what reaches it
    int listed = 0, threads = 0;
#pragma unroll
    for (int j = 0; j < M; ++j) {
        unsigned bits[(N + 31) / 32];
        int count = 0;
#pragma unroll
        for (int w = 0; w < (N + 31) / 32; ++w) {
            if constexpr (M == 1) bits[w] = mine[w];
            else bits[w] = mine[j * N / 32] >> (j * N % 32) & ((1u << N) - 1u);  // (M is 1 where N does not divide 32)
            count += __popc(bits[w]);
        }
        const unsigned long long who = __ballot(count != 0);
        if (who == 0) continue;
        const int scan = wave_scan_i(count), total = read_lane(scan, 63);
        int q = threads + lanes_below(who), to = listed + scan - count;
        if constexpr (W == 1) {
            threads += __popcll(who);
            listed += total;
        } else {
            int q0 = 0, to0 = 0;
            if (lane == 0) {
                q0 = atomicAdd(&sh.threads, __popcll(who));
                to0 = atomicAdd(&sh.listed, total);
            }
            q += __shfl(q0, 0);
            to += __shfl(to0, 0);
        }
        if (count != 0) {
            room.put(q, t + 64 * j, v, j * N);
            wave_fence();
#pragma unroll
            for (int w = 0; w < (N + 31) / 32; ++w)
                while (bits[w] != 0) {
                    const int i = __ffs((int)bits[w]) - 1 + w * 32, p = at.at(t + 64 * j, i);
                    bits[w] &= bits[w] - 1;
                    if (to < Room::kRoom) room.list(to, room.laid_out(q, i, p), p);
                    ++to;
                }
        }
    }
    group_sync<W>();
    if constexpr (W > 1) {
        listed = sh.listed;
        threads = sh.threads;
    }
    if (listed > Room::kRoom) {  // (the same in all threads)
        // The best scores lie together in few threads: the exact k-th one by bisection over all that were laid out.
        const int entries = threads * N;
        auto value = [&](int e) { return room.get(e / N, e % N, at); };
        auto place = [&](int e) { return room.place(e / N, e % N, at); };
        auto count = [&](auto is) {
            int n = 0;
            for (int e = t; e < entries; e += 64 * W) n += is(e) ? 1 : 0;
            return group_sum<W>(n, sh);
        };
        unsigned lo = bound, hi = 0xff800001u;  // (one past infinity)
        while (hi - lo > 1) {
            const unsigned mid = lo + (hi - lo) / 2;
            const float f = from_ordered(mid);
            if (count([&](int e) { return value(e) >= f; }) >= k) lo = mid;
            else hi = mid;
        }
        const float equal = from_ordered(lo);
        const int need = k - count([&](int e) { return value(e) > equal; });
        int p_lo = -1, p_hi = INT_MAX - 1;
        while (p_hi - p_lo > 1) {
            const int mid = p_lo + (p_hi - p_lo) / 2;
            if (count([&](int e) { return value(e) == equal && place(e) <= mid; }) >= need) p_hi = mid;
            else p_lo = mid;
        }
        if constexpr (W > 1) {
            __syncthreads();
            if (t == 0) sh.listed = 0;
            __syncthreads();
        }
        listed = 0;
        for (int e0 = 0; e0 < entries; e0 += 64 * W) {
            const int e = e0 + t;
            float x = kNothing;
            bool is = false;
            if (e < entries) {
                x = value(e);
                is = x > equal || (x == equal && place(e) <= p_hi);
            }
            const unsigned long long which = __ballot(is);
            if (which == 0) continue;
            int to = listed;
            if constexpr (W == 1) {
                listed += __popcll(which);
            } else {
                if (lane == 0) to = atomicAdd(&sh.listed, __popcll(which));
                to = __shfl(to, 0);
            }
            to += lanes_below(which);
            if (is && to < Room::kRoom) room.list(to, x, place(e));
        }
        group_sync<W>();
        if constexpr (W > 1) listed = sh.listed;
    }
    float *const values = out.values + slot * k;
    int *const classes = out.classes + slot * k;
    auto write = [&](unsigned long long key, int rank) {
        if (rank < k) {
            values[rank] = from_ordered((unsigned)(key >> 32));
            classes[rank] = class_at((int)~(unsigned)key);
        }
    };
    if constexpr (W == 1) {
        for (int j0 = 0; j0 < listed; j0 += 64) {
            const unsigned long long mine_key = room.listed(min(j0 + lane, listed - 1));
            int rank = 0;
            if (listed <= 64) {
                for (int o = 0; o < listed; ++o) rank += (unsigned long long)read_lane_ll((long long)mine_key, o) > mine_key ? 1 : 0;
            } else {
                for (int o = 0; o < listed; ++o) rank += room.listed(o) > mine_key ? 1 : 0;
            }
            if (j0 + lane < listed) write(mine_key, rank);
        }
    } else {
        // the threads beyond the candidates compare as well
        const int lines = max((listed + 63) / 64, 1), parts = W / lines, part = wave_id() / lines, j = (wave_id() - part * lines) * 64 + lane;
        if (j < listed && part < parts) {
            const unsigned long long mine_key = room.listed(j);
            int rank = 0;
            for (int o = part; o < listed; o += parts) rank += room.listed(o) > mine_key ? 1 : 0;
            atomicAdd(&room.better[j], rank);
        }
        __syncthreads();
        if (t < listed) write(room.listed(t), room.better[t]);
    }
    for (int j = listed + t; j < k; j += 64 * W) {
        values[j] = kNothing;
        classes[j] = -1;
    }
}

// Over a wavefront, the same in every lane.
struct WaveSumF {
    float v;
    template <int CTRL, int ROWS>
    __device__ __forceinline__ void at() { v += __int_as_float(dpp_i<CTRL, ROWS>(0, __float_as_int(v))); }
};
__device__ __forceinline__ float wave_sum_f(float v) {
    WaveSumF s{v};
    wave_scan_steps(s);
    return read_lane(s.v, 63);
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float reference_of(float m) { return fabsf(m) <= FLT_MAX ? m : 0.f; }
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// A sum to the reference `from` as one to `to`; an infinite one stays infinite.
__device__ __forceinline__ float rescaled(float sum, float from, float to, float by) {
    return sum <= FLT_MAX ? sum * exp2_of((from - to) * by) : sum;
}

// Up to here half a step of max / temperature (in powers of two) is 2^-9 at most, and a factor of 1 - off ln 2 stands for 2^-off within 1e-6. Far beyond, that factor
// becomes negative.
constexpr float kShiftMost = 65536.f;

// The largest of a wavefront's scores (0 where it is no number) and the sum of exp((v - it) / temperature). A NaN makes the sum
// NaN, an infinity makes it infinite. best: the thread's largest.
template <int E, typename Scores>
__device__ __forceinline__ void sum_exponentials(const Scores &v, float best, float by, float *reference, float *sum) {
    float m = reference_of(wave_max_f(best));
    float part[4] = {0.f, 0.f, 0.f, 0.f};
    const float shift = m * by;
    if (fabsf(shift) < kShiftMost) {
        // one multiply-add for the argument; what the product m * by was rounded by is put right in the sum
        const float off = __builtin_fmaf(m, by, -shift);
#pragma unroll
        for (int i = 0; i < E; ++i) part[i % 4] += exp2_of(__builtin_fmaf(v[i], by, -shift));
        const float s = (part[0] + part[1]) + (part[2] + part[3]);
        part[0] = s <= FLT_MAX ? __builtin_fmaf(s, -off * kLn2, s) : s;
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) part[i % 4] += exp2_of((v[i] - m) * by);
        part[0] = (part[0] + part[1]) + (part[2] + part[3]);
    }
    *reference = m;
    *sum = wave_sum_f(part[0]);
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

// A group of W wavefronts takes a chunk (a multiple of 32 classes) of a row; with W = 1 there are four groups to a
// workgroup. A thread has E scores in whole vectors, and one of what is left behind the last vector. RULES: there may be any. LDS: the lists of candidates,
// then, where classes were shown, bits and times.
template <typename T, int E, bool RULES>
constexpr bool held_in_pairs() { return sizeof(T) == 2 && !RULES && E > 24; }
template <typename T, int W, int E, bool RULES>
constexpr int waves_of_top_rows() { return held_in_pairs<T, E, RULES>() ? 6 : E > 24 ? 4 : W == 1 ? 5 : 6; }
template <typename T, int W, int E, bool RULES>
__global__ __launch_bounds__(W == 1 ? kTopBlock : 64 * W, (waves_of_top_rows<T, W, E, RULES>())) void k_top_rows(tgbm_scores in, tgbm_score_rules rules, int k, float temperature, TopOut out,
                                                                          int chunks, int chunk, bool whole) {
    constexpr int kGroups = W == 1 ? kTopBlock / 64 : 1;
    constexpr int V = Vector<T>::kOf, N = E + 1, kStep = 64 * W * V;
    constexpr bool kPairs = held_in_pairs<T, E, RULES>();
    // Short rows: vectors leave most threads without a score. Where too few are left to choose a bound among, all of their scores would be candidates: they are
    // dealt out one by one then, through LDS (100 000 x 200 bfloat16, k 20: 78 us, 447 without; k 5, where enough are left: 59, 53). Four wavefronts always do:
    // 100 000 x 200 float32, k 64: 331 us, 1550 without; 13 333 x 1500, k 128: 282, 309; k 64: 54, 52.
    constexpr bool kSpread = E == 8;
    __shared__ __align__(16) float spread[kSpread && W > 1 ? 64 * W * E : 4];
    __shared__ TopShared<W> shared[kGroups];
    using Scores = typename std::conditional<held_in_pairs<T, E, RULES>(), HeldPairs<T, E>, Held<N>>::type;
    __shared__ LaidOut<W, Scores> rooms[kGroups];
    extern __shared__ unsigned shown_lds[];
    const int t = W == 1 ? lane_id() : (int)threadIdx.x, group = W == 1 ? wave_id() : 0;
    TopShared<W> &sh = shared[group];
    unsigned *bits = shown_lds + (size_t)group * (chunk + chunk / 32), *times = bits + chunk / 32;
    const float by = kLog2e / temperature;
    const int part = blockIdx.y;
    const long row = (long)blockIdx.x * kGroups + group;
    if (W == 1 && row >= in.rows) return;
    {
        const size_t out_at = (size_t)row * chunks + part;
        const int c0 = part * chunk, size = min(in.classes - c0, chunk), whole_size = size / V * V;
        const Layout<N, V, true> at{kStep, whole_size};
        const bool dealt = kSpread && (W > 1 || whole_size * 4 < candidates_wanted(k) * V * 5);
        const typename std::conditional<kSpread, DealtLayout<N, V, W>, Layout<N, V, true>>::type choice_at = [&] {
            if constexpr (kSpread) return DealtLayout<N, V, W>{whole_size, dealt};
            else return at;
        }();
        const int base = (int)one_by_one((unsigned)t * V);  // (places are worked out where they are used, not kept over the tiles)
        const T *src = static_cast<const T *>(in.data) + (size_t)row * in.row_stride + c0;
        Scores held_scores;
        {
            typename Vector<T>::type x[E / V];
#pragma unroll
            for (int g = 0; g < E / V; ++g) {
                x[g] = (T)kNothing;
                if (base < whole_size - g * kStep) x[g] = *reinterpret_cast<const typename Vector<T>::type *>(src + base + g * kStep);
            }
            const float last = t < size - whole_size ? score_to_float(src[whole_size + t]) : kNothing;
            if constexpr (kPairs) {
                held_scores.last = last;
                typedef unsigned Words __attribute__((ext_vector_type(4)));
#pragma unroll
                for (int i = 0; i < E / 2; ++i) held_scores.pair[i] = __builtin_bit_cast(Words, x[i / 4])[i % 4];
            } else {
                held_scores.v[E] = last;
#pragma unroll
                for (int i = 0; i < E; ++i) held_scores.v[i] = score_to_float(x[i / V][i % V]);
            }
        }
        if constexpr (RULES) {
            auto &v = held_scores.v;
            if (rules.bias != nullptr) {
                const float *bias = rules.bias + c0;
#pragma unroll
                for (int g = 0; g < E / V; ++g)
                    if (base < whole_size - g * kStep) {
#pragma unroll
                        for (int j = 0; j < V; j += 4) {
                            const Float4 b = *reinterpret_cast<const Float4 *>(bias + base + g * kStep + j);
#pragma unroll
                            for (int q = 0; q < 4; ++q) v[g * V + j + q] += b[q];
                        }
                    }
                if (t < size - whole_size) v[E] += bias[whole_size + t];
            }
            bool none;
            const unsigned *words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
            if (rules.shown != nullptr) {
                long long b, e;
                shown_range(rules, row, &b, &e);
                if (b < e) {  // (the same for the group)
                    count_shown<W>(rules, b, e, c0, c0 + size, chunk, bits, times);
                    // few of a thread's scores are: one at a time, from the start (its register has no number that a loop can use)
#pragma unroll
                    for (int w = 0; w < (N + 23) / 24; ++w) {  // (24 scores are whole vectors)
                        unsigned held = 0;
#pragma unroll
                        for (int i = w * 24; i < (w * 24 + 24 < E ? w * 24 + 24 : E); i += V) {
                            const int c = base + i / V * kStep;
                            if (c < whole_size) held |= (bits[c / 32] >> (c % 32) & ((1u << V) - 1u)) << (i - w * 24);
                        }
                        if (w == E / 24 && t < size - whole_size) held |= (bits[(whole_size + t) / 32] >> ((whole_size + t) % 32) & 1u) << (E - w * 24);
                        while (__any(held != 0)) {
                            const bool now = held != 0;
                            const int i = now ? __ffs((int)held) - 1 + w * 24 : 0;
                            float s = 0.f;
                            if (now) {
                                const int c = at.at(t, i);
                                s = adjusted(score_to_float(src[c]), rules.bias != nullptr ? rules.bias[c0 + c] : 0.f, times[c], true, rules);
                            }
                            held &= held - 1;
#pragma unroll
                            for (int j = w * 24; j < (w * 24 + 24 < N ? w * 24 + 24 : N); ++j) v[j] = now && j == i ? s : v[j];
                        }
                    }
                }
            }
            if (words != nullptr || none) {
#pragma unroll
                for (int g = 0; g < E / V; ++g) {
                    const int c = base + g * kStep;
                    const unsigned ok = words != nullptr && c < whole_size ? words[(c0 + c) / 32] >> (c % 32) : 0u;
#pragma unroll
                    for (int j = 0; j < V; ++j) v[g * V + j] = ok >> j & 1u ? v[g * V + j] : kNothing;
                }
                const bool ok = words != nullptr && t < size - whole_size && (words[(c0 + whole_size + t) / 32] >> ((whole_size + t) % 32) & 1u);
                v[E] = ok ? v[E] : kNothing;
            }
        }
        if constexpr (kSpread) if (dealt) {
            auto &v = held_scores.v;
            float *const of_row = W > 1 ? spread : reinterpret_cast<float *>(rooms[group].word);  // (the lists come later)
#pragma unroll
            for (int g = 0; g < E / V; ++g)
                if (base < whole_size - g * kStep) {
#pragma unroll
                    for (int j = 0; j < V; j += 4) *reinterpret_cast<float4 *>(of_row + base + g * kStep + j) = float4{v[g * V + j], v[g * V + j + 1], v[g * V + j + 2], v[g * V + j + 3]};
                }
            if (t < size - whole_size) of_row[whole_size + t] = v[E];
            group_sync<W>();
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = t + i * 64 * W < size ? of_row[t + i * 64 * W] : kNothing;
            v[E] = kNothing;
            group_sync<W>();
        }
        const float best[1] = {best_of<N>(held_scores)};
        float m, s;
        held_scores.look_again();
        sum_exponentials<N>(held_scores, best[0], by, &m, &s);
        auto leave = [&](float reference, float sum) {
            if (whole) {
                out.lse[row] = log_sum(reference, sum, temperature);
            } else {
                out.lse[out_at * 2] = reference;
                out.lse[out_at * 2 + 1] = sum;
            }
        };
        if (lane_id() == 0) {
            if constexpr (W == 1) {
                leave(m, s);
            } else {
                sh.part_max[wave_id()] = m;
                sh.part_sum[wave_id()] = s;
            }
        }
        write_top<W, 1, N>(held_scores, best, choice_at, k, sh, rooms[group], out_at, out, [&](int p) { return c0 + p; }, [&] {
            const bool in = lane_id() < W;
            const float its_max = in ? sh.part_max[lane_id()] : 0.f, its_sum = in ? sh.part_sum[lane_id()] : 0.f;
            const float all = reference_of(wave_max_f(its_sum > 0.f ? its_max : kNothing));
            const float sum = wave_sum_f(its_sum != 0.f ? rescaled(its_sum, its_max, all, by) : 0.f);
            if (lane_id() == 0) leave(all, sum);
        });
    }
}

// Rows side by side: a workgroup brings `rows` rows of a chunk (a multiple of 32, at most 64 * E classes) into LDS, class by class, eight
// classes of a row to a thread at a time, and its wavefronts take a row each. M: parts of a lane's scores that count as threads, so that
// there are more of them than best classes. LDS: [chunk][rows + 1] scores, then, where classes were shown, [rows][chunk / 32] bits: such a
// class's cell holds how often first; whoever takes its bit away puts the score there.
constexpr int kColumnBlock = 1024;
template <typename T, int E, int M, bool RULES>
__global__ __launch_bounds__(kColumnBlock, 8) void k_top_columns(tgbm_scores in, tgbm_score_rules rules, int k, float temperature, TopOut out, int chunks,
                                                                 int chunk, int row_bits, bool whole) {
    __shared__ TopShared<1> sh;  // (nothing of it is used by one wavefront)
    __shared__ ColumnLists lists[kColumnBlock / 64];
    extern __shared__ unsigned cell[];
    const int rows = 1 << row_bits, pitch = rows + 1;
    unsigned *const bits = cell + (size_t)chunk * pitch;
    const float by = kLog2e / temperature;
    const int r = threadIdx.x & (rows - 1), slot = threadIdx.x >> row_bits, slots = kColumnBlock >> row_bits;
    const long row_tiles = ((in.rows - 1) >> row_bits) + 1;
    const int part = blockIdx.y;
    const long tile = tile_of_block(blockIdx.x, gridDim.x);
    if (tile >= row_tiles) return;
    {
        const long row0 = tile << row_bits, row = row0 + r;
        const int c0 = part * chunk, size = min(in.classes - c0, chunk);
        const T *src = static_cast<const T *>(in.data) + (size_t)c0 * in.class_stride + row;
        unsigned *const my_bits = bits + r * (chunk / 32);
        bool none = false;
        const unsigned *words = nullptr;
        const float *bias = rules.bias != nullptr ? rules.bias + c0 : nullptr;
        long long b = 0, e = 0;
        if constexpr (RULES) {
            if (row < in.rows) words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
            if (words != nullptr) words += c0 / 32;
            if (rules.shown != nullptr) {
                for (int i = threadIdx.x; i < rows * (chunk / 32); i += kColumnBlock) bits[i] = 0;
                __syncthreads();
                if (row < in.rows) shown_range(rules, row, &b, &e);
                for (long long i = b + slot; i < e; i += slots) {
                    const int c = rules.shown[i] - c0;
                    if (c < 0 || c >= size) continue;
                    cell[c * pitch + r] = 0;
                    atomicOr(&my_bits[c / 32], 1u << (c % 32));
                }
                __syncthreads();
                for (long long i = b + slot; i < e; i += slots) {
                    const int c = rules.shown[i] - c0;
                    if (c >= 0 && c < size) atomicAdd(&cell[c * pitch + r], 1u);
                }
            }
        }
        if (row < in.rows) {
            for (int c = slot * 8; c < size; c += slots * 8) {
                const T *from = src + (size_t)c * in.class_stride;
                unsigned *to = cell + c * pitch + r;
                unsigned held = 0, ok = ~0u;
                if constexpr (RULES) {
                    ok = none ? 0u : words != nullptr ? words[c / 32] >> (c % 32) : ~0u;
                    held = rules.shown != nullptr ? my_bits[c / 32] >> (c % 32) & 0xffu : 0u;
                }
                if (c + 8 <= size) {
                    float z[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[j] = score_to_float(from[(size_t)j * in.class_stride]);
                    if constexpr (RULES) {
                        if (bias != nullptr) {
#pragma unroll
                            for (int j = 0; j < 8; j += 4) {
                                const Float4 more = *reinterpret_cast<const Float4 *>(bias + c + j);
#pragma unroll
                                for (int q = 0; q < 4; ++q) z[j + q] += more[q];
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) z[j] = ok >> j & 1u ? z[j] : kNothing;
                        if (held == 0) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) to[j * pitch] = __float_as_uint(z[j]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (!(held >> j & 1u)) to[j * pitch] = __float_as_uint(z[j]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) to[j * pitch] = __float_as_uint(z[j]);
                    }
                } else {
                    for (int j = 0; c + j < size; ++j) {
                        float z = score_to_float(from[(size_t)j * in.class_stride]);
                        if (bias != nullptr) z += bias[c + j];
                        if (!(held >> j & 1u)) to[j * pitch] = __float_as_uint(ok >> j & 1u ? z : kNothing);
                    }
                }
            }
        }
        if constexpr (RULES) {
            if (rules.shown != nullptr) {
                __syncthreads();
                for (long long i = b + slot; i < e; i += slots) {
                    const int c = rules.shown[i] - c0;
                    if (c < 0 || c >= size) continue;
                    const unsigned bit = 1u << (c % 32);
                    if (!(atomicAnd(&my_bits[c / 32], ~bit) & bit)) continue;  // (another mention of the class has come first)
                    const bool ok = !none && (words == nullptr || words[c / 32] & bit);
                    unsigned *to = cell + c * pitch + r;
                    *to = __float_as_uint(adjusted(score_to_float(src[(size_t)c * in.class_stride]), bias != nullptr ? bias[c] : 0.f, *to, ok, rules));
                }
            }
        }
        __syncthreads();
        for (int q = wave_id(); q < rows && row0 + q < in.rows; q += kColumnBlock / 64) {
            const int lane = (int)one_by_one((unsigned)lane_id());  // (places are worked out where they are used)
            const unsigned *from = cell + lane * pitch + q;
            Held<E> v;
            float best[M];
#pragma unroll
            for (int i = 0; i < E; ++i) v.v[i] = lane < size - i * 64 ? __uint_as_float(from[i * 64 * pitch]) : kNothing;
            float largest = kNothing;
#pragma unroll
            for (int j = 0; j < M; ++j) {
                best[j] = kNothing;
#pragma unroll
                for (int i = 0; i < E / M; ++i) best[j] = fmaxf(best[j], v[j * (E / M) + i]);
                largest = fmaxf(largest, best[j]);
            }
            const size_t out_at = (size_t)(row0 + q) * chunks + part;
            float m, s;
            sum_exponentials<E>(v, largest, by, &m, &s);
            if (lane_id() == 0) {
                if (whole) {
                    out.lse[row0 + q] = log_sum(m, s, temperature);
                } else {
                    out.lse[out_at * 2] = m;
                    out.lse[out_at * 2 + 1] = s;
                }
            }
            Column column{cell + q, pitch, size, lists[wave_id()]};
            write_top<1, M, E / M>(v, best, LaneParts<E / M>{}, k, sh, column, out_at, out, [&](int p) { return c0 + p; }, [] {});
            wave_fence();
        }
    }
}

// Few classes: a thread holds its row's and counts, for every one of them, those that are better.
template <typename T, int E>
__global__ __launch_bounds__(kTopBlock) void k_top_few(tgbm_scores in, tgbm_score_rules rules, int k, float temperature, TopOut out) {
    const float by = kLog2e / temperature;
    const long row = (long)blockIdx.x * kTopBlock + threadIdx.x;
    if (row < in.rows) {
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
__global__ __launch_bounds__(W == 1 ? kTopBlock : 64 * W) void k_top_join(int parts, int per_join, int joins, int rows, int k, float temperature, TopOut in,
                                                                          TopOut out) {
    constexpr int kGroups = W == 1 ? kTopBlock / 64 : 1;
    __shared__ TopShared<W> shared[kGroups];
    __shared__ LaidOut<W, Held<E>> rooms[kGroups];
    const int t = W == 1 ? lane_id() : (int)threadIdx.x, group = W == 1 ? wave_id() : 0;
    TopShared<W> &sh = shared[group];
    const float by = kLog2e / temperature;
    const int part = blockIdx.y;
    const long row = (long)blockIdx.x * kGroups + group;
    if (W == 1 && row >= rows) return;
    {
        const int first = part * per_join, mine = min(parts - first, per_join), count = mine * k;
        const size_t from = (size_t)row * parts + first, tile = (size_t)row * joins + part;
        const float *values = in.values + from * k;
        const int *classes = in.classes + from * k;
        Held<E> v;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int at = i * 64 * W + t;
            v.v[i] = at < count ? values[at] : kNothing;
        }
        auto join_sums = [&] {  // (by one wavefront)
            const float *sums = in.lse + from * 2;
            float m = kNothing;
            for (int c = lane_id(); c < mine; c += 64) m = fmaxf(m, sums[c * 2 + 1] > 0.f ? sums[c * 2] : kNothing);
            m = reference_of(wave_max_f(m));
            float s = 0.f;
            for (int c = lane_id(); c < mine; c += 64) {
                const float its = sums[c * 2 + 1];
                if (its != 0.f) s += rescaled(its, sums[c * 2], m, by);
            }
            s = wave_sum_f(s);
            if (lane_id() == 0) {
                if (joins == 1) {
                    out.lse[row] = log_sum(m, s, temperature);
                } else {
                    out.lse[tile * 2] = m;
                    out.lse[tile * 2 + 1] = s;
                }
            }
        };
        if constexpr (W == 1) join_sums();
        const float best[1] = {best_of<E>(v)};
        write_top<W, 1, E>(v, best, Layout<E, 1, false>{64 * W, 0}, k, sh, rooms[group], tile, out, [&](int p) { return classes[p]; }, join_sums);
    }
}

// How a call goes: chunks of a row, and the classes of one.
struct TopPlan {
    bool few, columns;
    int chunks, chunk;
    int waves;     // classes side by side: wavefronts of a group
    int row_bits;  // rows side by side
    int per_thread;
    int parts;  // of a lane's scores, rows side by side
};
constexpr int kFewClasses = 32;
// With up to so many best classes the maxima of 64 lanes give a bound that few scores reach: with more the lists overflow, and rows go by the 256
// maxima of four wavefronts (classes side by side; 20 000 x 1000 float32, k 40: 31 us, with four 57; 48: 110, 61; 64: 341, 76), or of a lane's scores in four parts
// (rows side by side; k 26: 30 us, in parts 35; 32: 52, 37; 64: 1206, 76).
constexpr int kFewBestRows = 42, kFewBest = 28;
// Classes side by side: the most scores that a thread has in whole vectors. Looking for the bound, the list and its order cost about as much as
// the scores of 24, so rows that fill them go by 48.
constexpr int kRowScores = 24, kRowScoresWide = 48;
constexpr int kJoinMost = 16384;  // scores that a join takes
constexpr int kGroupsWanted = 512;

TopPlan plan_top(bool columns, int classes, int rows, int k) {
    TopPlan p{};
    p.columns = columns;
    p.few = classes <= kFewClasses;
    p.chunks = 1;
    p.chunk = classes;
    if (p.few) return p;
    const int most = columns ? 1024 : 8 * 64 * kRowScoresWide, least = columns ? 1024 : 64 * kRowScores;
    long tiles = columns ? (rows + 15) / 16 : rows;
    long chunks = (classes - 1) / most + 1;
    chunks = std::max(chunks, std::min<long>((classes - 1) / least + 1, kGroupsWanted / std::max(1l, tiles)));
    chunks = std::min(chunks, std::max<long>((classes - 1) / most + 1, kJoinMost / k));  // (one join, where it is a choice)
    p.chunk = (int)(((classes - 1) / chunks + 32) / 32 * 32);
    p.chunks = (classes - 1) / p.chunk + 1;
    if (columns) {
        p.per_thread = 1;
        while (p.per_thread * 64 < p.chunk) p.per_thread *= 2;
        p.per_thread = std::max(p.per_thread, 2);
        p.row_bits = 4;
        while (p.row_bits < 6 && (p.chunk << (p.row_bits + 1)) <= 16384) ++p.row_bits;
    } else if (k > kFewBestRows && p.chunk <= 64 * kRowScores) {
        p.waves = 4;
        p.per_thread = 8;
    } else {
        p.waves = p.chunk <= 64 * kRowScores ? 1 : p.chunk <= 256 * kRowScores ? 4 : 8;
        p.per_thread = p.chunk > 512 * kRowScores ? kRowScoresWide : p.waves > 1 ? kRowScores : p.chunk <= 512 ? 8 : p.chunk <= 1024 ? 16 : kRowScores;
    }
    p.parts = columns && k > kFewBest ? std::min(4, p.per_thread) : 1;
    return p;
}

template <typename T, int W, int E, bool RULES>
void top_rows(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    constexpr int kGroups = W == 1 ? kTopBlock / 64 : 1;
    const size_t lds = rules.shown != nullptr ? sizeof(unsigned) * (size_t)(p.chunk + p.chunk / 32) * kGroups : 0;
    if (lds > 32 * 1024) {
        static LdsOptIn opt_in;
        opt_in({reinterpret_cast<const void *>(&k_top_rows<T, W, E, RULES>)});
    }
    const dim3 grid((unsigned)((in.rows - 1) / kGroups + 1), (unsigned)p.chunks);
    k_top_rows<T, W, E, RULES><<<grid, W == 1 ? kTopBlock : 64 * W, lds, s>>>(in, rules, k, temperature, out, p.chunks, p.chunk, p.chunks == 1);
}

template <typename T, int E, int M, bool RULES>
void top_columns(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    const size_t lds = sizeof(unsigned) * ((size_t)p.chunk * ((1 << p.row_bits) + 1) + (rules.shown != nullptr ? (size_t)p.chunk / 32 << p.row_bits : 0));
    static LdsOptIn opt_in;
    opt_in({reinterpret_cast<const void *>(&k_top_columns<T, E, M, RULES>)});
    const dim3 grid(blocks_of_tiles((unsigned)((in.rows - 1) >> p.row_bits) + 1), (unsigned)p.chunks);
    k_top_columns<T, E, M, RULES><<<grid, kColumnBlock, lds, s>>>(in, rules, k, temperature, out, p.chunks, p.chunk, p.row_bits, p.chunks == 1);
}
template <typename T, int E, bool RULES>
void top_columns(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    if (p.parts == 1) top_columns<T, E, 1, RULES>(s, p, in, rules, k, temperature, out);
    else top_columns<T, E, E < 4 ? E : 4, RULES>(s, p, in, rules, k, temperature, out);
}

template <typename T, bool RULES>
void top(hipStream_t s, const TopPlan &p, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, const TopOut &out) {
    if (p.few) {
        const unsigned blocks = (unsigned)((in.rows - 1) / kTopBlock + 1);
        if (in.classes <= 8) k_top_few<T, 8><<<blocks, kTopBlock, 0, s>>>(in, rules, k, temperature, out);
        else if (in.classes <= 16) k_top_few<T, 16><<<blocks, kTopBlock, 0, s>>>(in, rules, k, temperature, out);
        else k_top_few<T, 32><<<blocks, kTopBlock, 0, s>>>(in, rules, k, temperature, out);
    } else if (p.columns) {
        constexpr bool kRules = RULES || sizeof(T) != 4;
        if (p.per_thread <= 2) top_columns<T, 2, kRules>(s, p, in, rules, k, temperature, out);
        else if (p.per_thread == 4) top_columns<T, 4, kRules>(s, p, in, rules, k, temperature, out);
        else if (p.per_thread == 8) top_columns<T, 8, kRules>(s, p, in, rules, k, temperature, out);
        else top_columns<T, 16, kRules>(s, p, in, rules, k, temperature, out);
    } else if (p.waves == 8 && p.per_thread == kRowScoresWide) {
        top_rows<T, 8, kRowScoresWide, RULES>(s, p, in, rules, k, temperature, out);
    } else if (p.waves == 8) {
        top_rows<T, 8, kRowScores, RULES>(s, p, in, rules, k, temperature, out);
    } else if (p.waves == 4 && p.per_thread == 8) {
        top_rows<T, 4, 8, RULES>(s, p, in, rules, k, temperature, out);
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
    const dim3 grid((unsigned)((rows - 1) / kGroups + 1), (unsigned)joins);
    k_top_join<W, E><<<grid, W == 1 ? kTopBlock : 64 * W, 0, s>>>(parts, per_join, joins, rows, k, temperature, in, out);
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
    return workspace_of_slices(rows, [&](int slice) {
        const TopPlan p = plan_top(columns, classes, slice, k);
        size_t bytes = 0;
        for (int parts = p.chunks; parts > 1; parts = (parts - 1) / parts_of_a_join(k) + 1) bytes += part_bytes((size_t)slice * parts, k);
        return bytes;
    });
}

static void launch_slice(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, float *values, int *classes, float *lse,
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
        if (k > kFewBest && count <= 1024) join<4, 4>(s, parts, per_join, joins, in.rows, k, temperature, now, to);
        else if (count <= 256) join<1, 4>(s, parts, per_join, joins, in.rows, k, temperature, now, to);
        else if (count <= 1024) join<1, 16>(s, parts, per_join, joins, in.rows, k, temperature, now, to);
        else if (count <= 4096) join<4, 16>(s, parts, per_join, joins, in.rows, k, temperature, now, to);
        else join<8, 32>(s, parts, per_join, joins, in.rows, k, temperature, now, to);
        now = to;
        parts = joins;
    }
}

// (a launch has fewer than 2^32 threads in a direction: very many rows go by slices, which share the workspace one after the other)
void launch_scores_top(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, float *values, int *classes, float *lse,
                       void *workspace) {
    for (int row = 0; row < in.rows; row += std::min(kSliceRows, in.rows - row)) {
        tgbm_scores part = in;
        tgbm_score_rules r = rules;
        take_rows(part, r, row, std::min(kSliceRows, in.rows - row));
        launch_slice(s, part, r, k, temperature, values + (size_t)row * k, classes + (size_t)row * k, lse + row, workspace);
    }
}

}  // namespace tgbm
