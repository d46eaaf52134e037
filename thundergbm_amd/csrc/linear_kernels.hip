// tgbm_rows_quantise and tgbm_scores_linear: rows of numbers in 8 bits with a scale each, and class scores as their product with a row of weights for every
// class.
//
// q = rint(x / scale), scale = max |x| / 127. A score is (sum of q_x q_w) * scale_x * scale_w + bias: the sum is whole numbers of 32 bits, which 2^16 features
// cannot leave, and exact; three operations of 32 bits and one rounding to the scores' type are behind it.
//
// Rows are brought to a common form first, kChunk features at a time with zeros behind the last: where a row of features is zero it does not matter what
// the weights' rows hold there.
//
// 8192 x 8192 x 32000: 1.85 ms, 2.32 POP/s (the library's 8-bit product of 8192^3: 2.13). The matrix units are busy 62 % of the cycles, and the clock is at 1.53 GHz: power bounds
// it. 1 x 4096 x 32000: 25 us of the kernel for 131 MB, 5.2 TB/s. 100003 x 200 x 500 float32: 88 us, of which the rows' quantisation takes 24, where the memory's share is 55.
#include <algorithm>

#include "kernel_common.h"
#include "score_rules.h"

namespace tgbm {
namespace {

constexpr int kLinearBlock = 256;
constexpr int kChunk = 128;

typedef int Int4 __attribute__((ext_vector_type(4)));

// What a row's largest magnitude makes of it. most: its bits; an infinity or a NaN among the numbers is the largest of all, and the row has no scale.
__device__ __forceinline__ float scale_of(unsigned most) { return most < 0x7f800000u ? __uint_as_float(most) / 127.f : __builtin_nanf(""); }
__device__ __forceinline__ int whole_of(float v, float scale) { return scale > 0.f ? (int)fminf(fmaxf(rintf(v / scale), -127.f), 127.f) : 0; }

// Whole numbers of several, as bytes. A product with 1 / scale is off by 127 * 2^-23 at most, roundings of the inverse, the product and the quotient that is meant
// together: only where it lies that near to half a step, one in 12 000, does the quotient itself have to be rounded (65537 x 1024: 83 us with a division for
// every number).
constexpr float kNearHalf = 0.5f - 0x1p-14f, kSmallScale = 0x1p-100f;
template <int N, typename T>
__device__ __forceinline__ void whole_of_all(const T &v, float scale, float inverse, unsigned (&bytes)[N / 4]) {
    constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: the sum's last byte is the whole number
    unsigned word[N];
    bool near = !(scale > kSmallScale);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float x = score_to_float(v[j]), by = x * inverse, sum = by + kMagic;
        word[j] = __float_as_uint(sum);
        near |= fabsf(by - (sum - kMagic)) > kNearHalf;
    }
    if (near) {
#pragma unroll
        for (int j = 0; j < N; ++j) word[j] = (unsigned)whole_of(score_to_float(v[j]), scale);
    }
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
        const unsigned low = __builtin_amdgcn_perm(word[j * 4 + 1], word[j * 4], 0x0c0c0400), high = __builtin_amdgcn_perm(word[j * 4 + 3], word[j * 4 + 2], 0x0c0c0400);
        bytes[j] = high << 16 | low;
    }
}

// G threads take a row (a workgroup takes several rows, or one), N vectors of 16 bytes each, which stay in registers. `pad` bytes from the row's begin on are
// written: zeros behind its features.
template <typename T, int G, int N>
__global__ __launch_bounds__(G > kLinearBlock ? G : kLinearBlock) void k_quantise(const T *x, long long pitch, int rows, int features, signed char *q, long long q_pitch, int pad, float *scales) {
    constexpr int kBlock = G > kLinearBlock ? G : kLinearBlock, V = 16 / (int)sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    typedef signed char Out __attribute__((ext_vector_type(16 / sizeof(T)), aligned(1)));
    __shared__ unsigned part[kBlock / 64];
    const long row = (long)blockIdx.x * (kBlock / G) + threadIdx.x / G;
    const int t = threadIdx.x % G;
    const bool on = row < rows;  // (all threads stay for the others)
    const T *from = x + (size_t)(on ? row : 0) * pitch;
    Vec v[N];
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = (i * G + t) * V;
        v[i] = (T)0.f;
        if (at + V <= features) {
            v[i] = *reinterpret_cast<const Vec *>(from + at);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (at + j < features) v[i][j] = from[at + j];
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) most = max(most, __float_as_uint(score_to_float(v[i][j])) & 0x7fffffffu);
#pragma unroll
    for (int d = (G < 64 ? G : 64) / 2; d > 0; d /= 2) most = max(most, (unsigned)__shfl_xor((int)most, d));
    if constexpr (G > 64) {
        if (lane_id() == 0) part[wave_id()] = most;
        __syncthreads();
        constexpr int kWaves = G / 64;
        const int first = wave_id() / kWaves * kWaves;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = max(most, part[first + w]);
    }
    if (!on) return;
    const float scale = scale_of(most);
    if (t == 0) scales[row] = scale;
    signed char *to = q + (size_t)row * q_pitch;
    const float inverse = 1.f / scale;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = (i * G + t) * V;
        unsigned bytes[V / 4];
        whole_of_all<V>(v[i], scale, inverse, bytes);
        const Out o = __builtin_bit_cast(Out, bytes);
        if (at + V <= pad) {
            *reinterpret_cast<Out *>(to + at) = o;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (at + j < pad) to[at + j] = o[j];
        }
    }
    // (a padding that is longer than what a launch is chosen for; of 2^31 bytes nearly, a place as an int would go round)
    for (unsigned i = N * G * V + t; i < (unsigned)pad; i += G) to[i] = 0;
}

// Longer rows: a workgroup reads its row twice.
template <typename T>
__global__ __launch_bounds__(1024) void k_quantise_long(const T *x, long long pitch, int features, signed char *q, long long q_pitch, int pad, float *scales) {
    __shared__ unsigned part[16];
    const T *row = x + (size_t)blockIdx.x * pitch;
    unsigned most = 0;
    for (int i = threadIdx.x; i < features; i += 1024) most = max(most, __float_as_uint(score_to_float(row[i])) & 0x7fffffffu);
    for (int d = 32; d > 0; d /= 2) most = max(most, (unsigned)__shfl_xor((int)most, d));
    if (lane_id() == 0) part[wave_id()] = most;
    __syncthreads();
    for (int w = 0; w < 16; ++w) most = max(most, part[w]);
    const float scale = scale_of(most);
    if (threadIdx.x == 0) scales[blockIdx.x] = scale;
    signed char *to = q + (size_t)blockIdx.x * q_pitch;
    for (unsigned i = threadIdx.x; i < (unsigned)pad; i += 1024) to[i] = (signed char)(i < (unsigned)features ? whole_of(score_to_float(row[i]), scale) : 0);
}

// Rows of whole numbers, moved to rows of `pad` bytes, 16 of them to a thread.
__global__ __launch_bounds__(kLinearBlock) void k_pack(const signed char *x, long long pitch, int rows, int features, signed char *to, int pad) {
    typedef Int4 Loose __attribute__((aligned(1)));
    const int parts = pad / 16;
    const long at = (long)blockIdx.x * kLinearBlock + threadIdx.x, row = at / parts;
    const int f = (int)(at - row * parts) * 16;
    if (row >= rows) return;
    const signed char *from = x + (size_t)row * pitch + f;
    Int4 v = {0, 0, 0, 0};
    if (f + 16 <= features) {
        v = *reinterpret_cast<const Loose *>(from);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (f + j < features) v[j / 4] |= (int)((unsigned)(unsigned char)from[j] << j % 4 * 8);
    }
    *reinterpret_cast<Int4 *>(to + (size_t)row * pad + f) = v;
}
void pack(hipStream_t s, const signed char *x, long long pitch, int rows, int features, signed char *to, int pad) {
    const int most = std::max(1, (1 << 30) / pad);  // (a launch has fewer than 2^32 threads in a direction)
    for (int row = 0; row < rows; row += std::min(most, rows - row)) {
        const int n = std::min(most, rows - row);
        k_pack<<<(unsigned)(((long)n * (pad / 16) - 1) / kLinearBlock + 1), kLinearBlock, 0, s>>>(x + (size_t)row * pitch, pitch, n, features, to + (size_t)row * pad, pad);
    }
}

struct Rows8 {
    const signed char *data;
    const float *scale;
    long long pitch;
    int rows;
};
typedef int Int16 __attribute__((ext_vector_type(16)));
typedef float Float4 __attribute__((ext_vector_type(4), aligned(4)));

// (as three operations, whichever kernel does it)
__device__ __forceinline__ float score_of(int sum, float x_scale, float w_scale, float bias) {
#pragma clang fp contract(off)
    return (float)sum * x_scale * w_scale + bias;
}

// What a tile's lines and columns are: `lines` follow one another in the scores' memory. In one order of the scores those are the classes, in the other the rows.
struct Product {
    Rows8 lines, columns;
    const float *bias;
    int features;
    void *out;
    long long column_stride;
};

__device__ __forceinline__ void to_lds(const signed char *from, signed char *to) {  // 16 bytes of each lane, to 16 bytes behind the lane below's
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}

// LDS of a workgroup: two stages, and in their place, when they are done with, 32 columns of each wavefront's scores on their way out and the scales.
template <typename O, int LINES>
__host__ __device__ constexpr int line_pitch() { return LINES + 16 / (int)sizeof(O); }
template <typename O, int BL, int BC, int WL, int WC>
__host__ __device__ constexpr int lds_of_scores() { return (int)sizeof(O) * WL * WC * 32 * line_pitch<O, BL / WL>(); }
template <typename O, int BL, int BC, int WL, int WC>
constexpr size_t lds_of_tiles() { return std::max(2 * (BL + BC) * kChunk, lds_of_scores<O, BL, BC, WL, WC>() + 2 * (BL + BC) * (int)sizeof(float)); }

// BL lines x BC columns to a workgroup of WL * WC wavefronts. Two stages of kChunk bytes of every line and column in LDS: while the wavefronts work on one the
// other one is on its way there. A line's 16-byte parts lie in an order that goes by the line, so that the lanes of a read, which look at the same part of
// 32 lines, find them in different banks. CLASSES: the lines are classes.
template <typename O, int BL, int BC, int WL, int WC, bool CLASSES>
__global__ __launch_bounds__(64 * WL * WC, 2) void k_linear_tiles(Product p, int line_tiles, int column_tiles) {
    constexpr int kWaves = WL * WC, kL = BL / WL / 32, kC = BC / WC / 32, kStage = (BL + BC) * kChunk;
    extern __shared__ __align__(16) signed char lds[];
    // Neighbouring tiles on one die, by columns of kBand tiles of lines
    constexpr int kBand = 8;
    const int tiles = line_tiles * column_tiles, tile = (int)tile_of_block(blockIdx.x, gridDim.x);
    if (tile >= tiles) return;
    const int band = tile / (kBand * column_tiles), in_band = tile - band * kBand * column_tiles, high = min(kBand, line_tiles - band * kBand);
    const int l0 = (band * kBand + in_band % high) * BL, c0 = in_band / high * BC;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
    const int chunks = (p.features + kChunk - 1) / kChunk, whole = (p.features + 15) / 16 * 16;

    // a wavefront brings eight lines at a time
    constexpr int kLoadL = BL / 8 / kWaves, kLoadC = BC / 8 / kWaves;
    static_assert(kLoadL % 2 == 0 && kLoadC % 2 == 0);
    // (the order of a line's parts: in 64 banks, the 16 lines that a quarter of a wavefront reads have each their own)
    const auto part_of = [&](int i) { return (lane % 8) ^ (lane / 16 + i % 2 * 4); };
    const signed char *const of_l = p.lines.data + (size_t)l0 * p.lines.pitch, *const of_c = p.columns.data + (size_t)c0 * p.columns.pitch;
    unsigned at_l[kLoadL], at_c[kLoadC];  // (from a tile's first line: 256 lines of up to 2^17 bytes)
#pragma unroll
    for (int i = 0; i < kLoadL; ++i) at_l[i] = (unsigned)min((wave * kLoadL + i) * 8 + lane / 8, p.lines.rows - 1 - l0) * (unsigned)p.lines.pitch + part_of(i) * 16;
#pragma unroll
    for (int i = 0; i < kLoadC; ++i) at_c[i] = (unsigned)min((wave * kLoadC + i) * 8 + lane / 8, p.columns.rows - 1 - c0) * (unsigned)p.columns.pitch + part_of(i) * 16;
    auto bring = [&](int chunk, int stage) {
        signed char *to = lds + stage * kStage;
        // weights may end with their features: what is read instead, a line's begin, meets zeros
        const int f = chunk * kChunk;
        unsigned back[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) back[i] = f + part_of(i) * 16 >= whole ? f + part_of(i) * 16 : 0;
#pragma unroll
        for (int i = 0; i < kLoadL; ++i) to_lds(of_l + (at_l[i] + f - (CLASSES ? back[i % 2] : 0u)), to + (wave * kLoadL + i) * 8 * kChunk);
#pragma unroll
        for (int i = 0; i < kLoadC; ++i) to_lds(of_c + (at_c[i] + f - (CLASSES ? 0u : back[i % 2])), to + (BL + (wave * kLoadC + i) * 8) * kChunk);
    };
    const int wl = wave / WC * (BL / WL), wc = wave % WC * (BC / WC);
    Int16 sum[kL][kC] = {};
    bring(0, 0);
    for (int chunk = 0; chunk < chunks; ++chunk) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const signed char *stage = lds + (chunk & 1) * kStage;
        Int4 a[4][kL], b[4][kC];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = lane % 32 * kChunk + (((k * 2 + lane / 32) ^ (lane / 2 % 8)) * 16);
#pragma unroll
            for (int i = 0; i < kL; ++i) a[k][i] = *reinterpret_cast<const Int4 *>(stage + (wl + i * 32) * kChunk + at);
#pragma unroll
            for (int j = 0; j < kC; ++j) b[k][j] = *reinterpret_cast<const Int4 *>(stage + (BL + wc + j * 32) * kChunk + at);
        }
        __builtin_amdgcn_sched_barrier(0);
        bring(min(chunk + 1, chunks - 1), (chunk + 1) & 1);  // (once more at the end: a branch would wait for the reads)
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < kC; ++j)
#pragma unroll
                for (int i = 0; i < kL; ++i) sum[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[k][i], b[k][j], sum[i][j], 0, 0, 0);
    }
    // The scores, 32 columns of a wavefront at a time, by way of LDS: a column's lines are stored side by side.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    constexpr int kPitch = line_pitch<O, BL / WL>(), kThreads = 64 * kWaves;
    O *const mine = reinterpret_cast<O *>(lds) + wave * 32 * kPitch;
    float *const l_scale = reinterpret_cast<float *>(lds + lds_of_scores<O, BL, BC, WL, WC>()), *const l_bias = l_scale + BL, *const c_scale = l_bias + BL, *const c_bias = c_scale + BC;
    for (int i = threadIdx.x; i < BL; i += kThreads) {
        const int l = min(l0 + i, p.lines.rows - 1);
        l_scale[i] = p.lines.scale[l];
        if (CLASSES) l_bias[i] = p.bias != nullptr ? p.bias[l] : 0.f;
    }
    for (int i = threadIdx.x; i < BC; i += kThreads) {
        const int c = min(c0 + i, p.columns.rows - 1);
        c_scale[i] = p.columns.scale[c];
        if (!CLASSES) c_bias[i] = p.bias != nullptr ? p.bias[c] : 0.f;
    }
    __syncthreads();
    typedef O Four __attribute__((ext_vector_type(4)));
    constexpr int kOf = 16 / (int)sizeof(O), kLanes = BL / WL / kOf;  // lanes that store a column
    typedef O Vec __attribute__((ext_vector_type(16 / sizeof(O))));
    typedef O Loose __attribute__((ext_vector_type(16 / sizeof(O)), aligned(sizeof(O))));
#pragma unroll
    for (int j = 0; j < kC; ++j) {
        const float by = c_scale[wc + j * 32 + lane % 32], of_column = CLASSES ? 0.f : c_bias[wc + j * 32 + lane % 32];
#pragma unroll
        for (int i = 0; i < kL; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at = i * 32 + g * 8 + lane / 32 * 4;
                const float4 its = *reinterpret_cast<const float4 *>(l_scale + wl + at);
                const float4 bias = CLASSES ? *reinterpret_cast<const float4 *>(l_bias + wl + at) : float4{of_column, of_column, of_column, of_column};
                Four z;
                const auto score = [&](int q, float s, float more) { return (O)(CLASSES ? score_of(sum[i][j][g * 4 + q], by, s, more) : score_of(sum[i][j][g * 4 + q], s, by, more)); };
                z[0] = score(0, its.x, bias.x);
                z[1] = score(1, its.y, bias.y);
                z[2] = score(2, its.z, bias.z);
                z[3] = score(3, its.w, bias.w);
                *reinterpret_cast<Four *>(mine + lane % 32 * kPitch + at) = z;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int step = 0; step < 32 * kLanes / 64; ++step) {
            const int c = step * (64 / kLanes) + lane / kLanes, col = c0 + wc + j * 32 + c, at = lane % kLanes * kOf, line = l0 + wl + at;
            if (col >= p.columns.rows || line >= p.lines.rows) continue;
            O *to = static_cast<O *>(p.out) + (size_t)col * p.column_stride + line;
            const Vec v = *reinterpret_cast<const Vec *>(mine + c * kPitch + at);
            if (line + kOf <= p.lines.rows) {
                *reinterpret_cast<Loose *>(to) = v;
            } else {
#pragma unroll
                for (int q = 0; q < kOf; ++q)
                    if (line + q < p.lines.rows) to[q] = v[q];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Scores of one or of four classes that lie side by side, in the type that they have.
struct ScoreOut {
    void *data;
    long long class_stride, row_stride;
    int type;
    template <typename O>
    __device__ __forceinline__ void as(const float (&z)[4], int cls, int row, int classes) const {
        typedef O Four __attribute__((ext_vector_type(4), aligned(sizeof(O))));
        O *to = static_cast<O *>(data) + (size_t)cls * class_stride + (size_t)row * row_stride;
        if (class_stride == 1 && cls + 4 <= classes) {
            *reinterpret_cast<Four *>(to) = Four{(O)z[0], (O)z[1], (O)z[2], (O)z[3]};
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (cls + q < classes) to[(size_t)q * class_stride] = (O)z[q];
        }
    }
    __device__ __forceinline__ void four(const float (&z)[4], int cls, int row, int classes) const {
        if (type == TGBM_F32) as<float>(z, cls, row, classes);
        else if (type == TGBM_F16) as<_Float16>(z, cls, row, classes);
        else as<__bf16>(z, cls, row, classes);
    }
};

// Few rows: the rows' features in LDS, `slice` of them at a time, and 16 * A classes to a wavefront, whose weights go from memory to the product; S wavefronts share
// the features. T: of the rows, which are quantised on the way into LDS if they are floating ones (all of their features at once then).
constexpr int few_block(int shares) { return shares > 4 ? 64 * shares : kLinearBlock; }
// (Two wavefronts to a SIMD at least: with more than 256 registers the compiler puts sums into the accumulation registers.)
template <typename T, int A, int R, int S>
__global__ __launch_bounds__(few_block(S), S > 8 ? 4 : 2) void k_linear_few(const T *x, const float *x_scales, long long x_pitch, int rows, Rows8 w, int features, const float *bias, ScoreOut out, int slice) {
    constexpr bool kQuantise = sizeof(T) > 1;
    constexpr int kBlock = few_block(S), kTiles = kBlock / 64 / S;
    __shared__ Int4 shared[S > 1 ? kTiles * (S - 1) * A * R : 1][64];
    __shared__ float scale_of_row[16 * R];
    __shared__ unsigned most_of_row[kQuantise ? 16 * R : 1];
    extern __shared__ __align__(16) signed char of_x[];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), share = wave % S, tile = wave / S;
    const int c0 = ((int)blockIdx.x * kTiles + tile) * 16 * A, r0 = (int)blockIdx.y * 16 * R, live = min(rows - r0, 16 * R), pitch = slice + 16;
    const int chunks = (features + kChunk - 1) / kChunk, whole = (features + 15) / 16 * 16;
    x += (size_t)r0 * x_pitch;
    const signed char *of_class[A];
#pragma unroll
    for (int i = 0; i < A; ++i) of_class[i] = w.data + (size_t)min(c0 + i * 16 + lane % 16, w.rows - 1) * w.pitch;
    Int4 sum[A][R] = {};
    // (what the scores want besides is on its way from the start)
    float w_scale[A][4], w_bias[A][4];
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int cls = min(c0 + i * 16 + lane / 16 * 4 + q, w.rows - 1);
            w_scale[i][q] = w.scale[cls];
            w_bias[i][q] = bias != nullptr ? bias[cls] : 0.f;
        }
    constexpr int kAtOnce = A * R > 2 ? 2 : 4;
    Int4 a[kAtOnce][2][A];
    const auto bring = [&](int c) {
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = min(c + s * S, chunks - 1) * kChunk + h * 64 + lane / 16 * 16;
#pragma unroll
                for (int i = 0; i < A; ++i) a[s][h][i] = *reinterpret_cast<const Int4 *>(of_class[i] + (at >= whole ? 0 : at));
            }
    };
    for (int f0 = 0; f0 < features; f0 += slice) {
        const int first = f0 / kChunk + share, last = min(chunks, (f0 + slice) / kChunk);
        bring(first);
        if (f0 != 0) __syncthreads();
        if constexpr (kQuantise) {
            // all threads go over the rows' vectors, twice: the second time they come from near
            constexpr int V = 16 / (int)sizeof(T);
            typedef T Loose __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
            typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T))));
            const int parts = chunks * kChunk / V;
            const auto each = [&](auto f) {
#pragma unroll 2
                for (int i = threadIdx.x; i < live * parts; i += kBlock) {
                    const int r = i / parts, at = (i - r * parts) * V;
                    const T *row = x + (size_t)r * x_pitch;
                    Vec v = (T)0.f;
                    if (at + V <= features) {
                        v = *reinterpret_cast<const Loose *>(row + at);
                    } else {
#pragma unroll
                        for (int j = 0; j < V; ++j)
                            if (at + j < features) v[j] = row[at + j];
                    }
                    f(r, at, v);
                }
            };
            if ((int)threadIdx.x < live) most_of_row[threadIdx.x] = 0;
            __syncthreads();
            each([&](int r, int, const Vec &v) {
                unsigned most = 0;
#pragma unroll
                for (int j = 0; j < V; ++j) most = max(most, __float_as_uint(score_to_float(v[j])) & 0x7fffffffu);
                atomicMax(&most_of_row[r], most);
            });
            __syncthreads();
            each([&](int r, int at, const Vec &v) {
                const float scale = scale_of(most_of_row[r]);
                unsigned bytes[V / 4];
                whole_of_all<V>(v, scale, 1.f / scale, bytes);
                typedef unsigned Words __attribute__((ext_vector_type(V / 4)));
                *reinterpret_cast<Words *>(of_x + r * pitch + at) = __builtin_bit_cast(Words, bytes);
            });
            if ((int)threadIdx.x < live) scale_of_row[threadIdx.x] = scale_of(most_of_row[threadIdx.x]);
        } else {
            const int parts = (last * kChunk - f0) / 16;
            for (int i = threadIdx.x; i < live * parts; i += kBlock) {
                const int r = i / parts, at = (i - r * parts) * 16;
                *reinterpret_cast<Int4 *>(of_x + r * pitch + at) = *reinterpret_cast<const Int4 *>(x + (size_t)r * x_pitch + f0 + at);
            }
            if (f0 == 0 && (int)threadIdx.x < live) scale_of_row[threadIdx.x] = x_scales[r0 + threadIdx.x];
        }
        __syncthreads();
        const signed char *of_row[R];
#pragma unroll
        for (int j = 0; j < R; ++j) of_row[j] = of_x + min(j * 16 + lane % 16, live - 1) * pitch + lane / 16 * 16;
        for (int c = first; c < last; c += kAtOnce * S) {
            if (c != first) bring(c);
#pragma unroll
            for (int s = 0; s < kAtOnce; ++s)
                if (c + s * S < last) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        Int4 b[R];
#pragma unroll
                        for (int j = 0; j < R; ++j) b[j] = *reinterpret_cast<const Int4 *>(of_row[j] + (c + s * S) * kChunk - f0 + h * 64);
#pragma unroll
                        for (int i = 0; i < A; ++i)
#pragma unroll
                            for (int j = 0; j < R; ++j) sum[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s][h][i], b[j], sum[i][j], 0, 0, 0);
                    }
                }
        }
    }
    if constexpr (S > 1) {
        if (share > 0) {
#pragma unroll
            for (int i = 0; i < A; ++i)
#pragma unroll
                for (int j = 0; j < R; ++j) shared[((tile * (S - 1) + share - 1) * A + i) * R + j][lane] = sum[i][j];
        }
        __syncthreads();
        if (share > 0) return;
#pragma unroll
        for (int s = 0; s < S - 1; ++s)
#pragma unroll
            for (int i = 0; i < A; ++i)
#pragma unroll
                for (int j = 0; j < R; ++j) sum[i][j] += shared[((tile * (S - 1) + s) * A + i) * R + j][lane];
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int r = j * 16 + lane % 16;
        if (r >= live) continue;
        const float by = scale_of_row[r];
#pragma unroll
        for (int i = 0; i < A; ++i) {
            const int cls = c0 + i * 16 + lane / 16 * 4;
            float z[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) z[q] = score_of(sum[i][j][q], by, w_scale[i][q], w_bias[i][q]);
            out.four(z, cls, r0 + r, w.rows);
        }
    }
}

constexpr size_t kPackedBytes = (size_t)512 << 20;  // of a slice's features

constexpr long long kPitchMost = 1 << 17;  // places in a tile are 32 bits
bool lies_well(const tgbm_rows &r) {
    return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.pitch % 16 == 0 && r.pitch <= kPitchMost && (r.features % 16 == 0 || r.padded);
}
long long pad_of(int features) { return ((long long)features + kChunk - 1) / kChunk * kChunk; }
bool packs_weights(const tgbm_rows &w) { return !lies_well(w); }
bool packs_features(const tgbm_rows &x) { return x.type != TGBM_I8 || !lies_well(x) || x.features % kChunk != 0; }
int packed_rows(const tgbm_rows &x) { return (int)std::max<long long>(1, std::min<long long>(x.rows, (long long)(kPackedBytes / (size_t)pad_of(x.features)))); }
size_t in_lines(size_t bytes) { return (bytes + 127) / 128 * 128; }

template <typename O, int BL, int BC, int WL, int WC, bool CLASSES>
void linear_tiles(hipStream_t s, const Product &p) {
    const int line_tiles = (p.lines.rows - 1) / BL + 1, column_tiles = (p.columns.rows - 1) / BC + 1;
    static LdsOptIn opt_in;
    opt_in({reinterpret_cast<const void *>(&k_linear_tiles<O, BL, BC, WL, WC, CLASSES>)});
    k_linear_tiles<O, BL, BC, WL, WC, CLASSES><<<blocks_of_tiles((unsigned)(line_tiles * column_tiles)), 64 * WL * WC, lds_of_tiles<O, BL, BC, WL, WC>(), s>>>(p, line_tiles,
                                                                                                                                                       column_tiles);
}

// Rows in LDS: as many of their features as fit, all of them where the rows are quantised on the way. Every workgroup does that again: it pays where they are few
// (1 x 4096 x 32000: 25 us, 27 with a launch before; 2 rows: 28 both; 16 x 1024 x 4000: 11, 15; 16 x 1024 x 32000: 20, 14).
constexpr int kFewLds = 64 * 1024, kFusedMost = 16 * 1024;
constexpr long long kFusedWork = 200000000;
bool quantised_on_the_way(const tgbm_rows &x, const tgbm_rows &w) {
    const long long numbers = (long long)x.rows * pad_of(x.features);
    return x.type != TGBM_I8 && x.rows <= 16 && numbers <= kFusedMost && numbers * w.rows <= kFusedWork;
}

template <typename T, int A, int R, int S>
void linear_few(hipStream_t s, const T *x, const float *scale, long long pitch, int rows, const Rows8 &w, int features, const float *bias, const ScoreOut &out) {
    constexpr int kOf = few_block(S) / 64 / S * 16 * A;
    const int live = std::min(rows, 16 * R), slice = std::min((int)pad_of(features), (kFewLds / live - 16) / kChunk * kChunk);
    static LdsOptIn opt_in;
    opt_in({reinterpret_cast<const void *>(&k_linear_few<T, A, R, S>)});
    k_linear_few<T, A, R, S><<<dim3((w.rows - 1) / kOf + 1, (rows - 1) / (16 * R) + 1), few_block(S), live * (slice + 16), s>>>(x, scale, pitch, rows, w, features, bias, out, slice);
}
template <typename T, int A, int R>
void linear_few(hipStream_t s, const T *x, const float *scale, long long pitch, int rows, const Rows8 &w, int features, const float *bias, const ScoreOut &out) {
    const long waves = (long)((w.rows - 1) / (16 * A) + 1) * ((rows - 1) / (16 * R) + 1);
    // More wavefronts share the features where there are few of them (1 x 4096 x 32000, 2000 wavefronts of 16 classes: 26 us, 30 where four share; 8 x 65536 x 100: 62 us
    // with four, 45 with sixteen). Where a wavefront has several sums, sixteen of them have too few registers: 24 x 8192 x 1000 takes 24 us with sixteen and 18 with eight,
    // 100 x 8192 x 500 33 and 26, 64 x 65536 x 100 235 and 250 (with the weights in the last cache), and the sixteen's scratch of 604 bytes a lane is 320 MB of the device's memory.
    constexpr long kFull = A * R > 1 ? 1024 : 4096;
    if (waves >= kFull || features <= 2 * kChunk) linear_few<T, A, R, 1>(s, x, scale, pitch, rows, w, features, bias, out);
    else if (waves >= std::min(kFull / 2, 1024l) || features <= 4 * kChunk) linear_few<T, A, R, 2>(s, x, scale, pitch, rows, w, features, bias, out);
    else if (waves >= 128 || features <= 16 * kChunk) linear_few<T, A, R, 4>(s, x, scale, pitch, rows, w, features, bias, out);
    else linear_few<T, A, R, (A * R > 1 ? 8 : 16)>(s, x, scale, pitch, rows, w, features, bias, out);
}

// Large tiles; the lines behind the last whole one go by small tiles where they would make a round of their own on the chip's 256 CUs (2048 x 4096 x 65537: 565 us, 550
// that way).
template <typename O, bool CLASSES>
void linear_large(hipStream_t s, Product p) {
    const int columns = (p.columns.rows - 1) / 256 + 1, whole = p.lines.rows / 256, rest = p.lines.rows % 256;
    const auto rounds = [&](long lines) { return (lines * columns + 255) / 256; };
    if (rest == 0 || rest > 128 || whole == 0 || rounds(whole + 1) == rounds(whole)) return linear_tiles<O, 256, 256, 2, 4, CLASSES>(s, p);
    p.lines.rows = whole * 256;
    linear_tiles<O, 256, 256, 2, 4, CLASSES>(s, p);
    p.lines.data += (size_t)p.lines.rows * p.lines.pitch;
    p.lines.scale += p.lines.rows;
    if (CLASSES && p.bias != nullptr) p.bias += p.lines.rows;
    p.out = static_cast<O *>(p.out) + p.lines.rows;
    p.lines.rows = rest;
    linear_tiles<O, 128, 128, 2, 2, CLASSES>(s, p);
}

template <typename O>
void linear_tiles(hipStream_t s, const Rows8 &x, const Rows8 &w, int features, const float *bias, const ScoreOut &out, long tiles) {
    const bool large = tiles >= 2048 && features > 4 * kChunk;
    if (out.class_stride == 1) {
        const Product p{w, x, bias, features, out.data, out.row_stride};
        if (large) linear_large<O, true>(s, p);
        else linear_tiles<O, 128, 128, 2, 2, true>(s, p);
    } else {
        const Product p{x, w, bias, features, out.data, out.class_stride};
        if (large) linear_large<O, false>(s, p);
        else linear_tiles<O, 128, 128, 2, 2, false>(s, p);
    }
}

// The scores of rows in 8 bits.
void linear(hipStream_t s, const Rows8 &x, const Rows8 &w, int features, const float *bias, ScoreOut out) {
    constexpr int kMost = 1 << 20;  // rows of a launch
    for (int r = 0; r < x.rows; r += std::min(kMost, x.rows - r)) {
        Rows8 part = x;
        part.data += (size_t)r * x.pitch;
        part.scale += r;
        part.rows = std::min(kMost, x.rows - r);
        const long tiles = (long)((w.rows - 1) / 128 + 1) * ((part.rows - 1) / 128 + 1);
        if (part.rows <= 16) linear_few<signed char, 1, 1>(s, part.data, part.scale, part.pitch, part.rows, w, features, bias, out);
        else if (part.rows <= 32) linear_few<signed char, 2, 2>(s, part.data, part.scale, part.pitch, part.rows, w, features, bias, out);
        else if (tiles < 32) linear_few<signed char, 1, 4>(s, part.data, part.scale, part.pitch, part.rows, w, features, bias, out);
        else if (out.type == TGBM_F32) linear_tiles<float>(s, part, w, features, bias, out, tiles);
        else if (out.type == TGBM_F16) linear_tiles<_Float16>(s, part, w, features, bias, out, tiles);
        else linear_tiles<__bf16>(s, part, w, features, bias, out, tiles);
        out.data = static_cast<char *>(out.data) + (out.type == TGBM_F32 ? 4 : 2) * (size_t)part.rows * out.row_stride;
    }
}

}  // namespace

namespace {
template <typename T, int G, int N>
void quantise(hipStream_t s, const tgbm_rows &x, signed char *q, long long q_pitch, int pad, float *scale) {
    constexpr int kBlock = G > kLinearBlock ? G : kLinearBlock;
    k_quantise<T, G, N><<<(x.rows - 1) / (kBlock / G) + 1, kBlock, 0, s>>>(static_cast<const T *>(x.data), x.pitch, x.rows, x.features, q, q_pitch, pad, scale);
}
template <typename T>
void quantise(hipStream_t s, const tgbm_rows &x, signed char *q, long long q_pitch, int pad, float *scale) {
    const int vectors = (x.features - 1) / (16 / (int)sizeof(T)) + 1;
    if (vectors <= 16) quantise<T, 8, 2>(s, x, q, q_pitch, pad, scale);
    else if (vectors <= 64) quantise<T, 16, 4>(s, x, q, q_pitch, pad, scale);
    else if (vectors <= 256) quantise<T, 64, 4>(s, x, q, q_pitch, pad, scale);
    else if (vectors <= 1024) quantise<T, 256, 4>(s, x, q, q_pitch, pad, scale);
    else if (vectors <= 4096) quantise<T, 1024, 4>(s, x, q, q_pitch, pad, scale);
    else k_quantise_long<T><<<x.rows, 1024, 0, s>>>(static_cast<const T *>(x.data), x.pitch, x.features, q, q_pitch, pad, scale);
}
}  // namespace

// (a launch has fewer than 2^32 threads in a direction: very many rows go by slices)
void launch_rows_quantise(hipStream_t s, const tgbm_rows &x, signed char *q, long long q_pitch, int pad, float *scale) {
    constexpr int kMost = 1 << 20;
    const size_t size = x.type == TGBM_F32 ? 4 : 2;
    for (int row = 0; row < x.rows; row += std::min(kMost, x.rows - row)) {
        tgbm_rows part = x;
        part.data = static_cast<const char *>(x.data) + size * (size_t)row * x.pitch;
        part.rows = std::min(kMost, x.rows - row);
        signed char *to = q + (size_t)row * q_pitch;
        if (x.type == TGBM_F32) quantise<float>(s, part, to, q_pitch, pad, scale + row);
        else if (x.type == TGBM_F16) quantise<_Float16>(s, part, to, q_pitch, pad, scale + row);
        else quantise<__bf16>(s, part, to, q_pitch, pad, scale + row);
    }
}

size_t scores_linear_workspace(const tgbm_rows &x, const tgbm_rows &w) {
    const size_t pad = (size_t)pad_of(x.features);
    size_t bytes = packs_weights(w) ? in_lines(pad * w.rows) : 0;
    if (packs_features(x) && !quantised_on_the_way(x, w)) bytes += in_lines(pad * packed_rows(x)) + (x.type != TGBM_I8 ? sizeof(float) * (size_t)packed_rows(x) : 0);
    return bytes;
}

void launch_scores_linear(hipStream_t s, const tgbm_rows &x, const tgbm_rows &w, const float *bias, const tgbm_scores &out, void *workspace) {
    const int pad = (int)pad_of(x.features);
    signed char *room = static_cast<signed char *>(workspace);
    Rows8 weights{static_cast<const signed char *>(w.data), w.scale, w.pitch, w.rows};
    if (packs_weights(w)) {
        pack(s, weights.data, w.pitch, w.rows, w.features, room, pad);
        weights.data = room;
        weights.pitch = pad;
        room += in_lines((size_t)pad * w.rows);
    }
    ScoreOut to{const_cast<void *>(out.data), out.class_stride, out.row_stride, out.type};
    if (quantised_on_the_way(x, w)) {
        if (x.type == TGBM_F32) linear_few<float, 1, 1>(s, static_cast<const float *>(x.data), nullptr, x.pitch, x.rows, weights, x.features, bias, to);
        else if (x.type == TGBM_F16) linear_few<_Float16, 1, 1>(s, static_cast<const _Float16 *>(x.data), nullptr, x.pitch, x.rows, weights, x.features, bias, to);
        else linear_few<__bf16, 1, 1>(s, static_cast<const __bf16 *>(x.data), nullptr, x.pitch, x.rows, weights, x.features, bias, to);
        return;
    }
    const int most = packs_features(x) ? packed_rows(x) : x.rows;
    for (int row = 0; row < x.rows; row += std::min(most, x.rows - row)) {
        tgbm_rows part = x;
        const size_t size = x.type == TGBM_I8 ? 1 : x.type == TGBM_F32 ? 4 : 2;
        part.data = static_cast<const char *>(x.data) + size * (size_t)row * x.pitch;
        part.rows = std::min(most, x.rows - row);
        Rows8 features{static_cast<const signed char *>(part.data), x.type == TGBM_I8 ? x.scale + row : nullptr, x.pitch, part.rows};
        if (packs_features(x)) {
            if (x.type == TGBM_I8) {
                pack(s, features.data, x.pitch, part.rows, x.features, room, pad);
            } else {
                float *scale = reinterpret_cast<float *>(room + in_lines((size_t)pad * most));
                launch_rows_quantise(s, part, room, pad, pad, scale);
                features.scale = scale;
            }
            features.data = room;
            features.pitch = pad;
        }
        linear(s, features, weights, x.features, bias, to);
        to.data = static_cast<char *>(to.data) + (out.type == TGBM_F32 ? 4 : 2) * (size_t)part.rows * out.row_stride;
    }
}

}  // namespace tgbm
