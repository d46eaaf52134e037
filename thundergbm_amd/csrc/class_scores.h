// Operators on class scores that lie on the GPU: adjusting them before an answer, the best classes of every row, and the
// loss against a teacher's top scores (the tgbm_scores_* entry points). Launchers are stream-ordered, allocate nothing and
// never synchronise; the entry points (scores_api.hip) have checked the arguments. None has a counterpart in the reference,
// whose answers are its arg-max and its softmax over the raw scores (multiclass_obj.cu:44-88) and whose multi-class loss
// knows labels only (multiclass_obj.cu:6-35).
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/thundergbm.h"
#include "common.h"

namespace tgbm {

constexpr int kClassesMost = 1 << 22;  // (the tiles of a row are one direction of a launch: at most 65 535)
constexpr int kSliceRows = 1 << 22;  // rows of a launch
constexpr int kTopMost = 128;      // classes that top lists
constexpr int kTeacherMost = 128;  // entries of a teacher's row

// Whether the arguments of an entry point can be worked on; if not, why not is said on stderr (scores_api.hip).
bool scores_ok(const char *entry, const char *what, const tgbm_scores *s);
bool rules_ok(const char *entry, const tgbm_score_rules *rules, int rows);

inline bool rows_side_by_side(const tgbm_scores &s) { return !(s.class_stride == 1 && (s.rows == 1 || s.row_stride != 1)); }

// Rows [first, first + rows) of the scores, and the rules for them.
inline void take_rows(tgbm_scores &s, tgbm_score_rules &rules, int first, int rows) {
    const size_t size = s.type == TGBM_F32 ? 4 : 2;
    s.data = static_cast<const char *>(s.data) + size * (size_t)first * (size_t)s.row_stride;
    // (a set for each row: the later rows' sets)
    if (rules.allowed != nullptr && rules.allowed_set == nullptr && rules.allowed_sets > 1) {
        rules.allowed += (size_t)first * ((s.classes + 31) / 32);
        rules.allowed_sets = std::max(2, rules.allowed_sets - first);  // (one would be everybody's)
    }
    if (rules.allowed_set != nullptr) rules.allowed_set += first;
    if (rules.shown_begin != nullptr) rules.shown_begin += first;
    s.rows = rows;
}

// The workspace of a call that goes by slices of rows: what of(rows) says for a whole slice, or for the last one, which may be split over
// the chip in another way.
template <typename Of>
size_t workspace_of_slices(int rows, Of of) {
    const int last = rows % kSliceRows;
    return std::max(of(std::min(rows, kSliceRows)), rows > kSliceRows && last > 0 ? of(last) : (size_t)0);
}

void launch_scores_adjust(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, const tgbm_scores &out);

size_t scores_top_workspace(bool columns, int classes, int rows, int k);
void launch_scores_top(hipStream_t s, const tgbm_scores &in, const tgbm_score_rules &rules, int k, float temperature, float *values, int *classes, float *lse,
                       void *workspace);

// row_of (may be null): the teacher's row, and the loss's, of every row of the scores, the labels and the pairs.
size_t scores_distill_workspace(int classes, int rows, int entries);
void launch_scores_distill(hipStream_t s, const tgbm_scores &in, const tgbm_teacher &teacher, const float *labels, float temperature, float weight,
                           float *loss, void *pairs, long pair_stride, const int *row_of, void *workspace);

}  // namespace tgbm
