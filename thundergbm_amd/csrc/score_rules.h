// What a class score becomes before an answer, for the kernels of adjust and top: bias, then the penalty of classes that the
// row was shown, then the classes that are not allowed. Every step is one 32-bit operation with one rounding, in this order:
// which of two classes is the better one must not hang on how a kernel groups its arithmetic.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "class_scores.h"

namespace tgbm {
namespace {

// Tiles of rows whose neighbours share cache lines with them. Workgroups go to the eight dies in turn; here a die gets tiles that follow one another, so
// that the shared lines are read into, and put together in, one L2 (where there are enough tiles to fill the dies that way).
constexpr unsigned kDies = 8, kTilesForDies = 256;
inline unsigned blocks_of_tiles(unsigned tiles) { return tiles < kTilesForDies ? tiles : (tiles + kDies - 1) / kDies * kDies; }
__device__ __forceinline__ long tile_of_block(unsigned block, unsigned blocks) {
    return blocks < kTilesForDies ? block : (block % kDies) * (blocks / kDies) + block / kDies;
}

template <typename T>
__device__ __forceinline__ float score_to_float(T v);
template <>
__device__ __forceinline__ float score_to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float score_to_float<_Float16>(_Float16 v) { return (float)v; }
template <>
__device__ __forceinline__ float score_to_float<__bf16>(__bf16 v) { return (float)v; }

// times: how often the row was shown the class, at least once
__device__ __forceinline__ float held_back(float s, unsigned times, const tgbm_score_rules &rules) {
#pragma clang fp contract(off)
    const float a = s > 0.f ? s / rules.repetition : s * rules.repetition;
    const float b = rules.frequency * (float)times;
    return a - b - rules.presence;
}

__device__ __forceinline__ float adjusted(float s, float bias, unsigned times, bool allowed, const tgbm_score_rules &rules) {
#pragma clang fp contract(off)
    s = s + bias;
    if (times != 0) s = held_back(s, times, rules);
    return allowed ? s : -__builtin_inff();
}

// The set of allowed classes of a row: its words, or nullptr for all classes. A number that is no set's allows nothing, which
// *none says.
__device__ __forceinline__ const unsigned *allowed_words(const tgbm_score_rules &rules, long row, int words, bool *none) {
    *none = false;
    if (rules.allowed == nullptr) return nullptr;
    long set = rules.allowed_sets == 1 ? 0 : row;
    if (rules.allowed_set != nullptr) {
        set = rules.allowed_set[row];
        if (set < 0) return nullptr;
        *none = set >= rules.allowed_sets;
        if (*none) return nullptr;
    }
    return rules.allowed + (size_t)set * words;
}

// The row's part of the list of shown classes, whatever shown_begin holds: a part that does not lie in the list is cut.
__device__ __forceinline__ void shown_range(const tgbm_score_rules &rules, long row, long long *begin, long long *end) {
    long long b = rules.shown_begin[row], e = rules.shown_begin[row + 1];
    b = b < 0 ? 0 : b;
    e = e > rules.n_shown ? rules.n_shown : e;
    *begin = b;
    *end = e < b ? b : e;
}

}  // namespace
}  // namespace tgbm
