// tgbm_scores_adjust. One read and one write of every score; the lists of shown classes are counted in LDS, a tile of
// classes at a time, with integer additions (their order does not change a count).
#include <algorithm>

#include "device_api.h"
#include "score_rules.h"

namespace tgbm {
namespace {

constexpr int kAdjustBlock = 256;
constexpr int kTileRows = 64;     // rows side by side: a wavefront's lanes are rows,
constexpr int kTileClasses = 128;  // and a workgroup takes so many classes
constexpr int kRowClasses = 8192;  // classes side by side: classes of a row that a workgroup takes

// Rows side by side. Tiles are row tiles * class tiles, and a workgroup takes every gridDim.x-th one.
template <typename T>
__global__ __launch_bounds__(kAdjustBlock) void k_adjust_columns(tgbm_scores in, tgbm_score_rules rules, tgbm_scores out, int class_tiles, long tiles) {
    __shared__ unsigned times[kTileClasses * kTileRows];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long row = tile / class_tiles * kTileRows + lane;
        const int c0 = (int)(tile % class_tiles) * kTileClasses;
        const int c1 = row < in.rows ? min(in.classes, c0 + kTileClasses) : c0;
        if (rules.shown != nullptr) {
            for (int i = threadIdx.x; i < kTileClasses * kTileRows; i += kAdjustBlock) times[i] = 0;
            __syncthreads();
            // four threads a row
            long long b = 0, e = 0;
            if (row < in.rows) shown_range(rules, row, &b, &e);
            for (long long i = b + wave; i < e; i += kAdjustBlock / 64) {
                const int c = rules.shown[i];
                if (c >= c0 && c < c1) atomicAdd(&times[(c - c0) * kTileRows + lane], 1u);
            }
            __syncthreads();
        }
        if (row < in.rows) {
            bool none;
            const unsigned *words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
            const T *src = static_cast<const T *>(in.data);
            T *dst = static_cast<T *>(const_cast<void *>(out.data));
            for (int c = c0 + wave; c < c1; c += kAdjustBlock / 64) {
                const float z = score_to_float(src[(size_t)c * in.class_stride + row]);
                const bool ok = !none && (words == nullptr || (words[c / 32] >> (c % 32) & 1u));
                const float v = adjusted(z, rules.bias != nullptr ? rules.bias[c] : 0.f,
                                         rules.shown != nullptr ? times[(c - c0) * kTileRows + lane] : 0u, ok, rules);
                dst[(size_t)c * out.class_stride + (size_t)row * out.row_stride] = (T)v;
            }
        }
        __syncthreads();  // (the counts are cleared for the next tile)
    }
}

// Classes side by side. Short rows share a workgroup: 2^row_bits threads each, up to eight classes a thread. Tiles are
// row groups * chunks, and a workgroup takes every gridDim.x-th one.
template <typename T>
__global__ __launch_bounds__(kAdjustBlock) void k_adjust_rows(tgbm_scores in, tgbm_score_rules rules, tgbm_scores out, int row_bits, int chunks,
                                                              long tiles) {
    __shared__ unsigned times_of[kRowClasses];
    const int per_row = 1 << row_bits, at = threadIdx.x & (per_row - 1), slot = threadIdx.x >> row_bits;
    unsigned *times = times_of + (size_t)slot * min(in.classes, kRowClasses);
    for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long row = tile / chunks * (kAdjustBlock >> row_bits) + slot;
        const int c0 = (int)(tile % chunks) * kRowClasses;
        const int c1 = row < in.rows ? min(in.classes, c0 + kRowClasses) : c0;
        if (rules.shown != nullptr) {
            long long b = 0, e = 0;
            if (row < in.rows) shown_range(rules, row, &b, &e);
            for (int c = c0 + at; c < c1; c += per_row) times[c - c0] = 0;
            __syncthreads();
            for (long long i = b + at; i < e; i += per_row) {
                const int c = rules.shown[i];
                if (c >= c0 && c < c1) atomicAdd(&times[c - c0], 1u);
            }
            __syncthreads();
        }
        if (row < in.rows) {
            bool none;
            const unsigned *words = allowed_words(rules, row, (in.classes + 31) / 32, &none);
            const T *src = static_cast<const T *>(in.data) + (size_t)row * in.row_stride;
            T *dst = static_cast<T *>(const_cast<void *>(out.data)) + (size_t)row * out.row_stride;
            for (int c = c0 + at; c < c1; c += per_row) {
                const float z = score_to_float(src[c]);
                const bool ok = !none && (words == nullptr || (words[c / 32] >> (c % 32) & 1u));
                const float v = adjusted(z, rules.bias != nullptr ? rules.bias[c] : 0.f, rules.shown != nullptr ? times[c - c0] : 0u, ok, rules);
                dst[(size_t)c * out.class_stride] = (T)v;
            }
        }
        __syncthreads();  // (the counts are cleared for the next tile)
    }
}

unsigned grid_of(long tiles) { return (unsigned)std::min(tiles, 1l << 20); }

template <typename T>
void adjust(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_scores &out) {
    if (rows_side_by_side(in)) {
        const int class_tiles = (in.classes - 1) / kTileClasses + 1;
        const long tiles = (long)class_tiles * ((in.rows - 1) / kTileRows + 1);
        k_adjust_columns<T><<<grid_of(tiles), kAdjustBlock, 0, s>>>(in, rules, out, class_tiles, tiles);
    } else {
        int row_bits = 3;
        while (row_bits < 8 && (8 << row_bits) < in.classes) ++row_bits;
        const int chunks = (in.classes - 1) / kRowClasses + 1;
        const long tiles = (long)chunks * ((in.rows - 1) / (kAdjustBlock >> row_bits) + 1);
        k_adjust_rows<T><<<grid_of(tiles), kAdjustBlock, 0, s>>>(in, rules, out, row_bits, chunks, tiles);
    }
}

}  // namespace

void launch_scores_adjust(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_scores &out) {
    if (in.type == TGBM_F32) adjust<float>(s, in, rules, out);
    else if (in.type == TGBM_F16) adjust<_Float16>(s, in, rules, out);
    else adjust<__bf16>(s, in, rules, out);
}

}  // namespace tgbm
