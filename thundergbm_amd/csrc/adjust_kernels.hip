// tgbm_scores_adjust. One read and one write of every score, by 16 bytes of a thread (8 of 16-bit scores whose rows lie side by side); memory bounds it.
//
// Shown classes are counted in LDS, by integers, while the scores that a workgroup has asked for are on their way, and whoever holds a score looks up
// its count: no score is stored twice, so `out` may be `in`. A workgroup takes rows' tiles of 64 x 128 classes, or up to 4096 (8192 of 16 bits) classes of a
// row. Storing the shown classes' scores behind the others, which touches their lines again, took 150 us where this takes 106 (100003 x 500
// float32, 64 sets, 20 shown classes a row: 3.8 TB/s of the 5 that a copy reaches; rows do not begin at 16 bytes there, which costs 7 us) and 81 where it
// takes 58 (512 x 65537 bfloat16, a set for each row, 1500 shown classes a row).
#include <algorithm>
#include <type_traits>

#include "kernel_common.h"
#include "score_rules.h"

namespace tgbm {
namespace {

constexpr int kAdjustBlock = 256;

template <typename T, int N>
struct ScoreVector {  // side by side, on any address of a score
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
typedef float Float4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ bool is_in_set(const unsigned *words, bool none, int c) { return !none && (words == nullptr || (words[c / 32] >> (c % 32) & 1u)); }

// ------------------------------------------------------------------------------------------------------- shown classes
// The score of class c of a row that was shown it `times` times.
template <typename T>
__device__ __forceinline__ void store_adjusted(const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_scores &out, long row, int c, unsigned times) {
    bool none;
    const unsigned *words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
    const float z = score_to_float(static_cast<const T *>(in.data)[(size_t)c * in.class_stride + (size_t)row * in.row_stride]);
    static_cast<T *>(const_cast<void *>(out.data))[(size_t)c * out.class_stride + (size_t)row * out.row_stride] =
        (T)adjusted(z, rules.bias != nullptr ? rules.bias[c] : 0.f, times, is_in_set(words, none, c), rules);
}

// The lists of the 64 rows of a tile of kTileClasses classes that begin at c0, as counts in LDS, [classes][rows]: of 16 bits, or, where a list is longer
// than those go, of 32 bits for half of the classes at a time.
constexpr int kTileRows = 64, kTileClasses = 128;
struct TileLists {
    static constexpr int kKept = 8, kLongest = 65535;
    __align__(16) unsigned counts[kTileRows * kTileClasses / 2];
    long long begin[kTileRows];
    int before[kTileRows + 1], narrow;  // before: entries of the rows before

    // whether counts of 16 bits do (all threads of the workgroup come here)
    __device__ __forceinline__ bool look(const tgbm_score_rules &rules, long row0, int rows) {
        if (threadIdx.x < 64) {
            long long b = 0, e = 0;
            if (row0 + threadIdx.x < rows) shown_range(rules, row0 + threadIdx.x, &b, &e);
            const bool fit = __all(e - b <= kLongest);
            const int sum = wave_scan_i(fit ? (int)(e - b) : 0);
            begin[threadIdx.x] = b;
            before[threadIdx.x + 1] = sum;
            if (threadIdx.x == 0) {
                before[0] = 0;
                narrow = fit ? 1 : 0;
            }
        }
        clear();
        __syncthreads();
        return narrow != 0;
    }
    __device__ __forceinline__ void clear() {
        const uint4 zero = {0, 0, 0, 0};
        for (int i = threadIdx.x; i < kTileRows * kTileClasses / 8; i += kAdjustBlock) reinterpret_cast<uint4 *>(counts)[i] = zero;
    }
    // behind look(), and in front of a barrier
    __device__ __forceinline__ void count(const tgbm_score_rules &rules, int c0, int c1) {
        const int n = before[kTileRows];
        auto entry = [&](int i, int *r) {
            *r = 0;
#pragma unroll
            for (int d = kTileRows / 2; d > 0; d >>= 1)
                if (before[*r + d] <= i) *r += d;
            return rules.shown[begin[*r] + (i - before[*r])] - c0;
        };
        auto add = [&](int c, int r) {
            if ((unsigned)c >= (unsigned)(c1 - c0)) return;
            const int cell = c * kTileRows + r;
            atomicAdd(&counts[cell / 2], 1u << cell % 2 * 16);
        };
        int c[kKept], r[kKept];
#pragma unroll
        for (int u = 0; u < kKept; ++u) {
            c[u] = -1;
            if ((int)threadIdx.x + u * kAdjustBlock < n) c[u] = entry(threadIdx.x + u * kAdjustBlock, &r[u]);
        }
#pragma unroll
        for (int u = 0; u < kKept; ++u)
            if ((int)threadIdx.x + u * kAdjustBlock < n) add(c[u], r[u]);
        for (int i = threadIdx.x + kKept * kAdjustBlock; i < n; i += kAdjustBlock) {
            int of;
            const int cls = entry(i, &of);
            add(cls, of);
        }
    }
    // how often class c0 + c was shown to rows 4 * quad to 4 * quad + 3
    __device__ __forceinline__ uint2 of(int c, int quad) const { return reinterpret_cast<const uint2 *>(counts)[c * (kTileRows / 4) + quad]; }
    // Long lists: the scores of classes [c0, c1), as many as there are counts of 32 bits, behind clear() and a barrier. Four threads go through a row's list.
    template <typename T>
    __device__ __forceinline__ void store_long(const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_scores &out, long row0, int c0, int c1) {
        const int r = threadIdx.x % kTileRows, slot = threadIdx.x / kTileRows;
        const bool on = row0 + r < in.rows;
        long long b = 0, e = 0;
        if (on) shown_range(rules, row0 + r, &b, &e);
#pragma unroll 1
        for (long long i = b + slot; i < e; i += kAdjustBlock / kTileRows) {
            const int c = rules.shown[i];
            if (c >= c0 && c < c1) atomicAdd(&counts[(c - c0) * kTileRows + r], 1u);
        }
        __syncthreads();
        if (on) {
#pragma unroll 1
            for (int c = c0 + slot; c < c1; c += kAdjustBlock / kTileRows) store_adjusted<T>(in, rules, out, row0 + r, c, counts[(c - c0) * kTileRows + r]);
        }
    }
};

// ---------------------------------------------------------------------------------------------- bias and allowed sets
// Rows side by side: a wavefront takes 32 classes of 4 << quad_bits rows, four rows to a thread, 64 >> quad_bits classes side by side. ok: a bit for each of
// the 32 classes, of each of the four rows.
__device__ __forceinline__ void allowed_of_rows(const tgbm_score_rules &rules, long row, int rows, int classes, int g, unsigned (&ok)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) ok[j] = ~0u;
    if (rules.allowed == nullptr) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        bool none;
        const unsigned *words = allowed_words(rules, std::min(row + j, (long)rows - 1), (classes + 31) / 32, &none);
        ok[j] = none ? 0u : words != nullptr ? words[g / 32] : ~0u;
    }
}
// ALONG: out is in the same order.
template <typename T, bool ALONG>
__global__ __launch_bounds__(kAdjustBlock) void k_adjust_columns(tgbm_scores in, tgbm_score_rules rules, tgbm_scores out, int quad_bits) {
    using V = typename ScoreVector<T, 4>::type;
    static_assert(kAdjustBlock / 64 * 32 == kTileClasses);
    const long tile = tile_of_block(blockIdx.x, gridDim.x);
    const int lane = threadIdx.x & 63, step = 64 >> quad_bits;
    const int g = ((int)blockIdx.y * (kAdjustBlock / 64) + (int)(threadIdx.x >> 6)) * 32, end = std::min(g + 32, in.classes);
    const long row = ((tile << quad_bits) + (lane & ((1 << quad_bits) - 1))) * 4;
    const int live = (int)std::min(4l, in.rows - row);
    if (g >= in.classes || live <= 0) return;
    unsigned ok[4];
    allowed_of_rows(rules, row, in.rows, in.classes, g, ok);
    int c = g + (lane >> quad_bits);
    const T *from = static_cast<const T *>(in.data) + (size_t)c * in.class_stride + row;
    T *to = static_cast<T *>(const_cast<void *>(out.data)) + (size_t)c * out.class_stride + (size_t)row * out.row_stride;
    if (ALONG && live == 4) {
        constexpr int kAtOnce = 8;
        for (; c < end; c += kAtOnce * step) {
            V x[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                if (c + u * step < end) x[u] = *reinterpret_cast<const V *>(from);
                from += (size_t)step * in.class_stride;
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                if (c + u * step < end) {
                    const float bias = rules.bias != nullptr ? rules.bias[c + u * step] : 0.f;
                    V v;
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = (T)(ok[j] >> (c + u * step - g) & 1u ? score_to_float(x[u][j]) + bias : -__builtin_inff());
                    *reinterpret_cast<V *>(to) = v;
                }
                to += (size_t)step * out.class_stride;
            }
        }
    } else {
        for (; c < end; c += step) {
            const float bias = rules.bias != nullptr ? rules.bias[c] : 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < live) to[(size_t)j * out.row_stride] = (T)(ok[j] >> (c - g) & 1u ? score_to_float(from[j]) + bias : -__builtin_inff());
            from += (size_t)step * in.class_stride;
            to += (size_t)step * out.class_stride;
        }
    }
}

// Rows side by side, with lists: a tile's are counted in LDS while its scores are on their way, and a thread takes the counts of four rows of a class with
// the scores.
template <typename T, bool ALONG>
__global__ __launch_bounds__(kAdjustBlock) void k_adjust_tiles(tgbm_scores in, tgbm_score_rules rules, tgbm_scores out) {
    using V = typename ScoreVector<T, 4>::type;
    constexpr int kQuads = kTileRows / 4, kStep = 64 / kQuads, kEach = 32 / kStep;
    __shared__ __align__(16) TileLists lists;
    const long tile = tile_of_block(blockIdx.x, gridDim.x);
    const int lane = threadIdx.x & 63, first = (int)blockIdx.y * kTileClasses, last = std::min(in.classes, first + kTileClasses);
    const int g = first + (int)(threadIdx.x >> 6) * 32, c = g + lane / kQuads, end = std::min(g + 32, last);
    const long row = tile * kTileRows + lane % kQuads * 4;
    const int live = (int)std::min(4l, std::max(0l, in.rows - row));
    V x[kEach];
    const T *from = static_cast<const T *>(in.data) + (size_t)c * in.class_stride + row;
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
        if (c + u * kStep < end) {
            if (live == 4) {
                x[u] = *reinterpret_cast<const V *>(from);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < live) x[u][j] = from[j];
            }
        }
        from += (size_t)kStep * in.class_stride;
    }
    const bool mine = g < end && live > 0, narrow = lists.look(rules, tile * kTileRows, in.rows);
    if (!narrow) {
        for (int half = first; half < last; half += kTileClasses / 2) {
            lists.store_long<T>(in, rules, out, tile * kTileRows, half, std::min(last, half + kTileClasses / 2));
            __syncthreads();
            lists.clear();
            __syncthreads();
        }
        return;
    }
    lists.count(rules, first, last);
    __syncthreads();
    if (!mine) return;
    unsigned ok[4];
    allowed_of_rows(rules, row, in.rows, in.classes, g, ok);
    T *to = static_cast<T *>(const_cast<void *>(out.data)) + (size_t)c * out.class_stride + (size_t)row * out.row_stride;
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
        const int cu = c + u * kStep;
        if (cu < end) {
            const float bias = rules.bias != nullptr ? rules.bias[cu] : 0.f;
            float s[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] = score_to_float(x[u][j]) + bias;
            const uint2 times = lists.of(cu - first, lane % kQuads);
            unsigned held = (times.x & 0xffffu ? 1u : 0u) | (times.x >> 16 ? 2u : 0u) | (times.y & 0xffffu ? 4u : 0u) | (times.y >> 16 ? 8u : 0u);
            while (held != 0) {  // (few are shown: one at a time)
                const int at = __ffs((int)held) - 1;
                held &= held - 1;
                float its = at == 0 ? s[0] : at == 1 ? s[1] : at == 2 ? s[2] : s[3];
                its = held_back(its, (at < 2 ? times.x : times.y) >> at % 2 * 16 & 0xffffu, rules);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] = at == j ? its : s[j];
            }
            V v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (T)(ok[j] >> (cu - g) & 1u ? s[j] : -__builtin_inff());
            if (ALONG && live == 4) {
                *reinterpret_cast<V *>(to) = v;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < live) to[(size_t)j * out.row_stride] = v[j];
            }
        }
        to += (size_t)kStep * out.class_stride;
    }
}

// Classes side by side: 2^row_bits threads to a row, kRowVectors vectors of 16 bytes to each of them. LISTS: a bit in LDS says that a class was shown, and
// a word how often; the row's threads go through its list while the scores are on their way.
constexpr int kRowVectors = 4;
template <int CELLS>
struct ShownTimes {
    static constexpr int kKept = 8;
    unsigned bits[CELLS / 32];
    unsigned times[CELLS];

    // of classes [c0, c0 + size) of a row whose cells begin at `first`, by its per_row threads. All threads of the workgroup come here.
    __device__ __forceinline__ void count(const tgbm_score_rules &rules, long row, bool on, int c0, int size, int first, int at, int per_row) {
#pragma unroll
        for (int i = 0; i < CELLS / 32; i += kAdjustBlock)
            if (i + (int)threadIdx.x < CELLS / 32) bits[i + threadIdx.x] = 0;
        long long b = 0, e = 0;
        if (on) shown_range(rules, row, &b, &e);
        int kept[kKept];  // (-1: none of these classes; a list is gone through twice, and every load is waited for)
#pragma unroll
        for (int u = 0; u < kKept; ++u) {
            const long long i = b + at + u * per_row;
            const int c = i < e ? rules.shown[i] - c0 : -1;
            kept[u] = (unsigned)c < (unsigned)size ? first + c : -1;
        }
        auto each = [&](auto f) {
#pragma unroll
            for (int u = 0; u < kKept; ++u)
                if (kept[u] >= 0) f(kept[u]);
            for (long long i = b + at + kKept * per_row; i < e; i += per_row) {
                const int c = rules.shown[i] - c0;
                if ((unsigned)c < (unsigned)size) f(first + c);
            }
        };
        __syncthreads();
        each([&](int cell) {
            times[cell] = 0;
            atomicOr(&bits[cell / 32], 1u << cell % 32);
        });
        __syncthreads();
        each([&](int cell) { atomicAdd(&times[cell], 1u); });
        __syncthreads();
    }
};

template <typename T, bool ALONG, bool LISTS>
__global__ __launch_bounds__(kAdjustBlock) void k_adjust_rows(tgbm_scores in, tgbm_score_rules rules, tgbm_scores out, int row_bits) {
    constexpr int kOf = 16 / (int)sizeof(T);
    using V = typename ScoreVector<T, kOf>::type;
    __shared__ typename std::conditional<LISTS, ShownTimes<kRowVectors * kOf * kAdjustBlock>, char>::type shown;
    const int per_row = 1 << row_bits, at = threadIdx.x & (per_row - 1), step = per_row * kOf, group = threadIdx.x >> row_bits;
    const long row = (long)blockIdx.x * (kAdjustBlock >> row_bits) + group;
    const bool on = row < in.rows;
    const int c0 = (int)blockIdx.y * kRowVectors * step, c1 = on ? std::min(in.classes, c0 + kRowVectors * step) : c0, whole = c0 + (c1 - c0) / kOf * kOf;
    const T *src = static_cast<const T *>(in.data) + (size_t)row * in.row_stride;
    T *dst = static_cast<T *>(const_cast<void *>(out.data)) + (size_t)row * out.row_stride;
    const int c = c0 + at * kOf, first = group * kRowVectors * step - c0;  // (first + a class: its cell)
    V x[kRowVectors];
    if constexpr (ALONG) {
#pragma unroll
        for (int u = 0; u < kRowVectors; ++u)
            if (c + u * step < whole) x[u] = *reinterpret_cast<const V *>(src + c + u * step);
    }
    if constexpr (LISTS) shown.count(rules, row, on, c0, c1 - c0, first + c0, at, per_row);
    if (!on) return;
    bool none;
    const unsigned *words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
    if constexpr (ALONG) {
#pragma unroll
        for (int u = 0; u < kRowVectors; ++u) {
            const int cu = c + u * step;
            if (cu >= whole) break;
            const unsigned ok = none ? 0u : words != nullptr ? words[cu / 32] >> (cu % 32) : ~0u;
            float s[kOf];
#pragma unroll
            for (int j = 0; j < kOf; j += 4) {
                Float4 bias = {0.f, 0.f, 0.f, 0.f};
                if (rules.bias != nullptr) bias = *reinterpret_cast<const Float4 *>(rules.bias + cu + j);
#pragma unroll
                for (int q = 0; q < 4; ++q) s[j + q] = score_to_float(x[u][j + q]) + bias[q];
            }
            if constexpr (LISTS) {
                // few are: one at a time (a register has no number that a loop can use)
                unsigned held = shown.bits[(first + cu) / 32] >> ((first + cu) % 32) & ((1u << kOf) - 1u);
                while (held != 0) {
                    const int i = __ffs((int)held) - 1;
                    held &= held - 1;
                    float its = s[0];
#pragma unroll
                    for (int j = 1; j < kOf; ++j) its = i == j ? s[j] : its;
                    its = held_back(its, shown.times[first + cu + i], rules);
#pragma unroll
                    for (int j = 0; j < kOf; ++j) s[j] = i == j ? its : s[j];
                }
            }
            V v;
#pragma unroll
            for (int j = 0; j < kOf; ++j) v[j] = (T)(ok >> j & 1u ? s[j] : -__builtin_inff());
            *reinterpret_cast<V *>(dst + cu) = v;
        }
    }
    for (int o = (ALONG ? whole : c0) + at; o < c1; o += per_row) {
        unsigned times = 0;
        if constexpr (LISTS) times = shown.bits[(first + o) / 32] >> ((first + o) % 32) & 1u ? shown.times[first + o] : 0u;
        dst[(size_t)o * out.class_stride] = (T)adjusted(score_to_float(src[o]), rules.bias != nullptr ? rules.bias[o] : 0.f, times, is_in_set(words, none, o), rules);
    }
}

// Long lists: a workgroup takes a row and kTableClasses classes, counts them in LDS, and whoever takes a count away stores. A thread keeps its
// first entries: the list is gone through three times, and every load is waited for.
constexpr int kTableClasses = 8192, kKept = 8;
template <typename T>
__global__ __launch_bounds__(kAdjustBlock) void k_adjust_long_lists(tgbm_scores in, tgbm_score_rules rules, tgbm_scores out) {
    __shared__ unsigned times[kTableClasses];
    const long row = blockIdx.x;
    const int c0 = (int)blockIdx.y * kTableClasses, size = std::min(in.classes - c0, kTableClasses);
    long long b, e;
    shown_range(rules, row, &b, &e);
    if (b >= e) return;
    int kept[kKept];  // (-1: none of this workgroup's)
#pragma unroll
    for (int u = 0; u < kKept; ++u) {
        const long long i = b + threadIdx.x + u * kAdjustBlock;
        const int c = i < e ? rules.shown[i] - c0 : -1;
        kept[u] = (unsigned)c < (unsigned)size ? c : -1;
    }
    auto each = [&](auto f) {
#pragma unroll
        for (int u = 0; u < kKept; ++u)
            if (kept[u] >= 0) f(kept[u]);
        for (long long i = b + threadIdx.x + kKept * kAdjustBlock; i < e; i += kAdjustBlock) {
            const int c = rules.shown[i] - c0;
            if ((unsigned)c < (unsigned)size) f(c);
        }
    };
    each([&](int c) { times[c] = 0; });
    __syncthreads();
    each([&](int c) { atomicAdd(&times[c], 1u); });
    __syncthreads();
    each([&](int c) {
        const unsigned n = atomicExch(&times[c], 0u);
        if (n != 0) store_adjusted<T>(in, rules, out, row, c0 + c, n);
    });
}

template <typename T, bool ALONG>
void adjust_slice(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_scores &out) {
    const bool columns = rows_side_by_side(in);
    if (!columns) {
        constexpr int kOf = 16 / (int)sizeof(T);
        int row_bits = 2;
        while (row_bits < 8 && (kRowVectors * kOf << row_bits) < in.classes) ++row_bits;
        const dim3 grid((in.rows - 1) / (kAdjustBlock >> row_bits) + 1, (in.classes - 1) / (kRowVectors * kOf << row_bits) + 1);
        if (rules.shown != nullptr) k_adjust_rows<T, ALONG, true><<<grid, kAdjustBlock, 0, s>>>(in, rules, out, row_bits);
        else k_adjust_rows<T, ALONG, false><<<grid, kAdjustBlock, 0, s>>>(in, rules, out, row_bits);
        return;
    }
    const bool lists = rules.shown != nullptr;
    // Every tile of 128 classes goes through its rows' lists. For many classes a second launch that goes through them once costs less, and stores the shown
    // classes' scores again (it cannot where the scores are gone by then). 20011 x 1000, 150 shown classes a row: 82 us by tiles, 156 that way; 400: 169, 244;
    // 2000 x 5000: 150: 38, 31; 2000 x 20000: 20: 76, 85; 50: 87, 87.
    constexpr long long kVisits = 1 << 19;  // classes times shown classes of a row
    const bool tiles = lists && (in.data == out.data || rules.n_shown <= in.rows * kVisits / in.classes);
    const int quad_bits = tiles ? 4 : in.rows <= 32 ? 2 : in.rows <= 128 ? 4 : 6;
    const dim3 grid(blocks_of_tiles((in.rows - 1) / (4 << quad_bits) + 1), (in.classes - 1) / kTileClasses + 1);
    if (tiles) {
        k_adjust_tiles<T, ALONG><<<grid, kAdjustBlock, 0, s>>>(in, rules, out);
        return;
    }
    k_adjust_columns<T, ALONG><<<grid, kAdjustBlock, 0, s>>>(in, rules, out, quad_bits);
    if (lists) k_adjust_long_lists<T><<<dim3(in.rows, (in.classes - 1) / kTableClasses + 1), kAdjustBlock, 0, s>>>(in, rules, out);
}

template <typename T>
void adjust(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_scores &out) {
    const bool along = rows_side_by_side(in) ? out.row_stride == 1 : out.class_stride == 1;
    for (int row = 0; row < in.rows; row += std::min(kSliceRows, in.rows - row)) {
        tgbm_scores from = in, to = out;
        tgbm_score_rules r = rules, unused = tgbm_score_rules{};
        take_rows(from, r, row, std::min(kSliceRows, in.rows - row));
        take_rows(to, unused, row, from.rows);
        if (along) adjust_slice<T, true>(s, from, r, to);
        else adjust_slice<T, false>(s, from, r, to);
    }
}

}  // namespace

void launch_scores_adjust(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_scores &out) {
    if (in.type == TGBM_F32) adjust<float>(s, in, rules, out);
    else if (in.type == TGBM_F16) adjust<_Float16>(s, in, rules, out);
    else adjust<__bf16>(s, in, rules, out);
}

}  // namespace tgbm
