// extern "C" layer of the operators on class scores (part 3 of include/thundergbm.h). Nothing here throws or aborts: what
// cannot be done is said on stderr and returned.
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "class_scores.h"

using namespace tgbm;

namespace {

int refused(const char *entry, const char *fmt, ...) {
    char text[256];
    va_list args;
    va_start(args, fmt);
    std::vsnprintf(text, sizeof(text), fmt, args);
    va_end(args);
    std::fprintf(stderr, "%s: %s\n", entry, text);
    std::fflush(stderr);
    return 1;
}

int launched(const char *entry) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    std::fprintf(stderr, "%s: launch failed: %s\n", entry, hipGetErrorString(e));
    std::fflush(stderr);
    return 2;
}

// 0 when the array can be worked on
int check_scores(const char *entry, const char *what, const tgbm_scores *s) {
    if (s == nullptr) return refused(entry, "%s is null", what);
    if (s->type != TGBM_F32 && s->type != TGBM_F16 && s->type != TGBM_BF16) return refused(entry, "%s: unknown type %d", what, s->type);
    if (s->classes < 1 || s->classes > kClassesMost) return refused(entry, "%s: %d classes", what, s->classes);
    if (s->rows < 0) return refused(entry, "%s: %d rows", what, s->rows);
    if (s->rows > 0 && s->data == nullptr) return refused(entry, "%s: null data", what);
    const bool columns = s->row_stride == 1 && (s->classes == 1 || s->class_stride >= s->rows);
    const bool rows = s->class_stride == 1 && (s->rows <= 1 || s->row_stride >= s->classes);
    const bool one_row = s->rows <= 1 && s->class_stride >= 1;
    if (!columns && !rows && !one_row)
        return refused(entry, "%s: strides %lld and %lld of %d classes and %d rows: one of them is 1, the other one at least as long", what, s->class_stride,
                       s->row_stride, s->classes, s->rows);
    return 0;
}

// Whether two arrays of one type and the same sizes share an element. Parts of one larger array may lie between each other's lines: they have its strides.
bool overlap(const tgbm_scores &a, const tgbm_scores &b) {
    const long long size = a.type == TGBM_F32 ? 4 : 2;
    const auto bytes = [&](const tgbm_scores &s) { return ((s.classes - 1) * s.class_stride + (s.rows - 1) * s.row_stride + 1) * size; };
    const char *first = static_cast<const char *>(a.data), *second = static_cast<const char *>(b.data);
    if (first + bytes(a) <= second || second + bytes(b) <= first) return false;
    if (a.class_stride != b.class_stride || a.row_stride != b.row_stride) return true;
    const bool columns = rows_side_by_side(a);
    if ((columns ? a.classes : a.rows) == 1) return true;  // (one line, whose pitch says nothing)
    const long long pitch = columns ? a.class_stride : a.row_stride, width = columns ? a.rows : a.classes;
    const long long apart = (first < second ? second - first : first - second) % (pitch * size);
    return apart < width * size || apart > (pitch - width) * size;
}

int check_rules(const char *entry, const tgbm_score_rules *r, int rows) {
    if (r == nullptr) return refused(entry, "rules is null");
    if (r->allowed != nullptr) {
        if (r->allowed_sets < 1) return refused(entry, "%d allowed sets", r->allowed_sets);
        if (r->allowed_set == nullptr && r->allowed_sets != 1 && r->allowed_sets < rows)
            return refused(entry, "%d allowed sets for %d rows, and no allowed_set", r->allowed_sets, rows);
    } else if (r->allowed_set != nullptr) {
        return refused(entry, "allowed_set without allowed");
    }
    if (r->shown != nullptr) {
        if (r->shown_begin == nullptr) return refused(entry, "shown without shown_begin");
        if (r->n_shown < 0) return refused(entry, "n_shown is %lld", r->n_shown);
        if (!(r->repetition > 0.f) || !std::isfinite(r->repetition)) return refused(entry, "repetition is %g: a number above 0 is wanted", r->repetition);
        if (!std::isfinite(r->frequency) || !std::isfinite(r->presence)) return refused(entry, "frequency %g, presence %g", r->frequency, r->presence);
    } else if (r->shown_begin != nullptr && r->n_shown != 0) {
        return refused(entry, "shown_begin without shown");
    }
    return 0;
}

int check_temperature(const char *entry, float t) {
    return t >= 1e-6f && t <= 1e6f ? 0 : refused(entry, "temperature is %g: 1e-6 to 1e6 is wanted", t);
}

int check_sampling(const char *entry, const tgbm_sampling *h) {
    if (h == nullptr) return refused(entry, "how is null");
    const float t = h->temperature_all;
    if (h->temperature == nullptr && !(t == 0.f || (t >= 1e-6f && t <= 1e6f))) return refused(entry, "temperature is %g: 0 or 1e-6 to 1e6 is wanted", t);
    if (h->p == nullptr && !(h->p_all > 0.f && h->p_all <= 1.f)) return refused(entry, "p is %g: above 0 and up to 1 is wanted", h->p_all);
    if (h->min_p == nullptr && !(h->min_p_all >= 0.f && h->min_p_all <= 1.f)) return refused(entry, "min_p is %g: 0 to 1 is wanted", h->min_p_all);
    if (h->k == nullptr && h->k_all < 0) return refused(entry, "k is %d: 0 or more is wanted", h->k_all);
    return 0;
}

int check_rows(const char *entry, const char *what, const tgbm_rows *r, bool whole_numbers, bool floating) {
    if (r == nullptr) return refused(entry, "%s is null", what);
    const bool is_floating = r->type == TGBM_F32 || r->type == TGBM_F16 || r->type == TGBM_BF16;
    if (!(is_floating && floating) && !(r->type == TGBM_I8 && whole_numbers)) return refused(entry, "%s: type %d", what, r->type);
    if (r->rows < 0) return refused(entry, "%s: %d rows", what, r->rows);
    if (r->features < 1 || r->features > kFeaturesMost) return refused(entry, "%s: %d features: 1 to %d are wanted", what, r->features, kFeaturesMost);
    if (r->rows > 1 ? r->pitch < r->features : r->pitch < 0) return refused(entry, "%s: a pitch of %lld for %d features", what, r->pitch, r->features);
    if (r->rows > 0 && r->data == nullptr) return refused(entry, "%s: null data", what);
    if (r->type == TGBM_I8 && r->rows > 0 && r->scale == nullptr) return refused(entry, "%s: no scales", what);
    return 0;
}

// (a single row's pitch says nothing but whether what is behind it can be read)
tgbm_rows with_pitch(tgbm_rows r) {
    if (r.pitch < r.features) {
        r.pitch = r.features;
        r.padded = 0;
    }
    return r;
}

}  // namespace

namespace tgbm {
bool scores_ok(const char *entry, const char *what, const tgbm_scores *s) { return check_scores(entry, what, s) == 0; }
bool rules_ok(const char *entry, const tgbm_score_rules *rules, int rows) { return check_rules(entry, rules, rows) == 0; }
bool sampling_ok(const char *entry, const tgbm_sampling *how) { return check_sampling(entry, how) == 0; }
bool rows_ok(const char *entry, const char *what, const tgbm_rows *rows) { return check_rows(entry, what, rows, false, true) == 0; }
}  // namespace tgbm

extern "C" int tgbm_scores_adjust(const tgbm_scores *in, const tgbm_score_rules *rules, const tgbm_scores *out, void *stream) {
    const char *entry = "tgbm_scores_adjust";
    int rc = check_scores(entry, "in", in);
    if (rc == 0) rc = check_scores(entry, "out", out);
    if (rc == 0) rc = check_rules(entry, rules, in->rows);
    if (rc != 0) return rc;
    if (out->type != in->type || out->classes != in->classes || out->rows != in->rows) return refused(entry, "out is not of in's type and sizes");
    if (in->data == out->data && (in->class_stride != out->class_stride || in->row_stride != out->row_stride))
        return refused(entry, "out is in's memory with other strides");
    if (in->rows == 0) return 0;
    if (in->data != out->data && overlap(*in, *out)) return refused(entry, "out overlaps in");
    launch_scores_adjust(static_cast<hipStream_t>(stream), *in, *rules, *out);
    return launched(entry);
}

extern "C" size_t tgbm_scores_top_workspace(const tgbm_scores *in, int k) {
    if (check_scores("tgbm_scores_top_workspace", "in", in) != 0 || k < 1 || k > kTopMost || in->rows == 0) return 0;
    return scores_top_workspace(rows_side_by_side(*in), in->classes, in->rows, k);
}

extern "C" int tgbm_scores_top(const tgbm_scores *in, const tgbm_score_rules *rules, int k, float temperature, float *values, int *classes, float *lse,
                               void *workspace, size_t workspace_bytes, void *stream) {
    const char *entry = "tgbm_scores_top";
    int rc = check_scores(entry, "in", in);
    if (rc == 0) rc = check_rules(entry, rules, in->rows);
    if (rc == 0) rc = check_temperature(entry, temperature);
    if (rc != 0) return rc;
    if (k < 1 || k > kTopMost) return refused(entry, "k is %d: 1 to %d is wanted", k, kTopMost);
    if (in->rows == 0) return 0;
    if (values == nullptr || classes == nullptr || lse == nullptr) return refused(entry, "an output is null");
    const size_t needed = scores_top_workspace(rows_side_by_side(*in), in->classes, in->rows, k);
    if (needed > workspace_bytes || (needed > 0 && workspace == nullptr)) return refused(entry, "%zu bytes of workspace, %zu are needed", workspace_bytes, needed);
    launch_scores_top(static_cast<hipStream_t>(stream), *in, *rules, k, temperature, values, classes, lse, workspace);
    return launched(entry);
}

extern "C" size_t tgbm_scores_distill_workspace(const tgbm_scores *in, int entries) {
    if (check_scores("tgbm_scores_distill_workspace", "in", in) != 0 || entries < 1 || entries > kTeacherMost || in->rows == 0) return 0;
    return scores_distill_workspace(in->classes, in->rows, entries);
}

extern "C" int tgbm_scores_distill(const tgbm_scores *in, const tgbm_teacher *teacher, const float *labels, float temperature, float weight, float *loss,
                                   float *pairs, long long pair_stride, void *workspace, size_t workspace_bytes, void *stream) {
    const char *entry = "tgbm_scores_distill";
    if (const int rc = check_scores(entry, "in", in)) return rc;
    if (in->type != TGBM_F32) return refused(entry, "in: float scores are wanted");
    if (in->rows > 1 && in->row_stride != 1) return refused(entry, "in: the rows of a class lie side by side");
    if (teacher == nullptr) return refused(entry, "teacher is null");
    if (teacher->type != TGBM_F32 && teacher->type != TGBM_F16 && teacher->type != TGBM_BF16) return refused(entry, "teacher: unknown type %d", teacher->type);
    if (teacher->entries < 1 || teacher->entries > kTeacherMost)
        return refused(entry, "teacher: %d entries: 1 to %d are wanted", teacher->entries, kTeacherMost);
    if (!(temperature >= 1e-3f && temperature <= 1e3f)) return refused(entry, "temperature is %g: 1e-3 to 1e3 is wanted", temperature);
    if (!(weight >= 0.f && weight <= 1.f)) return refused(entry, "weight is %g: 0 to 1 is wanted", weight);
    if (labels == nullptr && weight != 1.f && in->rows > 0) return refused(entry, "weight is %g, and there are no labels", weight);
    if (pairs != nullptr && in->classes > 1 && pair_stride < in->rows) return refused(entry, "pair_stride is %lld for %d rows", pair_stride, in->rows);
    if (in->rows == 0) return 0;
    if (teacher->classes == nullptr || teacher->scores == nullptr) return refused(entry, "teacher: null entries");
    if (loss == nullptr && pairs == nullptr) return refused(entry, "there is no output");
    const size_t needed = scores_distill_workspace(in->classes, in->rows, teacher->entries);
    if (needed > workspace_bytes || (needed > 0 && workspace == nullptr)) return refused(entry, "%zu bytes of workspace, %zu are needed", workspace_bytes, needed);
    launch_scores_distill(static_cast<hipStream_t>(stream), *in, *teacher, labels, temperature, weight, loss, pairs, pair_stride, nullptr, workspace);
    return launched(entry);
}

extern "C" size_t tgbm_scores_sample_workspace(const tgbm_scores *in, const tgbm_score_rules *rules, const tgbm_sampling *how) {
    const char *entry = "tgbm_scores_sample_workspace";
    if (check_scores(entry, "in", in) != 0 || check_rules(entry, rules, in->rows) != 0 || check_sampling(entry, how) != 0 || in->rows == 0) return 0;
    return scores_sample_workspace(*in, *rules, *how);
}

extern "C" int tgbm_scores_sample(const tgbm_scores *in, const tgbm_score_rules *rules, const tgbm_sampling *how, const float *u, int *classes, float *logp,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    const char *entry = "tgbm_scores_sample";
    int rc = check_scores(entry, "in", in);
    if (rc == 0) rc = check_rules(entry, rules, in->rows);
    if (rc == 0) rc = check_sampling(entry, how);
    if (rc != 0) return rc;
    if (in->rows == 0) return 0;
    if (u == nullptr) return refused(entry, "u is null");
    if (classes == nullptr || logp == nullptr) return refused(entry, "an output is null");
    const size_t needed = scores_sample_workspace(*in, *rules, *how);
    if (needed > workspace_bytes || (needed > 0 && workspace == nullptr)) return refused(entry, "%zu bytes of workspace, %zu are needed", workspace_bytes, needed);
    if (needed > 0 && reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return refused(entry, "the workspace does not begin at 16 bytes");
    launch_scores_sample(static_cast<hipStream_t>(stream), *in, *rules, *how, u, classes, logp, workspace);
    return launched(entry);
}

extern "C" int tgbm_rows_quantise(const tgbm_rows *x, signed char *q, long long q_pitch, int q_width, float *scale, void *stream) {
    const char *entry = "tgbm_rows_quantise";
    if (const int rc = check_rows(entry, "x", x, false, true)) return rc;
    if (q_width < x->features || q_pitch < q_width) return refused(entry, "q: %d of %lld bytes a row for %d features", q_width, q_pitch, x->features);
    if (x->rows == 0) return 0;
    if (q == nullptr || scale == nullptr) return refused(entry, "an output is null");
    launch_rows_quantise(static_cast<hipStream_t>(stream), with_pitch(*x), q, q_pitch, q_width, scale);
    return launched(entry);
}

extern "C" size_t tgbm_scores_linear_workspace(const tgbm_rows *x, const tgbm_rows *weights) {
    const char *entry = "tgbm_scores_linear_workspace";
    if (check_rows(entry, "x", x, true, true) != 0 || check_rows(entry, "weights", weights, true, false) != 0 || x->rows == 0 || weights->rows == 0) return 0;
    return scores_linear_workspace(with_pitch(*x), with_pitch(*weights));
}

extern "C" int tgbm_scores_linear(const tgbm_rows *x, const tgbm_rows *weights, const float *bias, const tgbm_scores *out, void *workspace, size_t workspace_bytes,
                                  void *stream) {
    const char *entry = "tgbm_scores_linear";
    int rc = check_rows(entry, "x", x, true, true);
    if (rc == 0) rc = check_rows(entry, "weights", weights, true, false);
    if (rc == 0) rc = check_scores(entry, "out", out);
    if (rc != 0) return rc;
    if (x->features != weights->features) return refused(entry, "%d features of x, %d of the weights", x->features, weights->features);
    if (out->classes != weights->rows || out->rows != x->rows)
        return refused(entry, "out has %d classes and %d rows, the weights have %d and x has %d", out->classes, out->rows, weights->rows, x->rows);
    if (x->rows == 0) return 0;
    const tgbm_rows x_ = with_pitch(*x), w_ = with_pitch(*weights);
    const size_t needed = scores_linear_workspace(x_, w_);
    if (needed > workspace_bytes || (needed > 0 && workspace == nullptr)) return refused(entry, "%zu bytes of workspace, %zu are needed", workspace_bytes, needed);
    if (needed > 0 && reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return refused(entry, "the workspace does not begin at 16 bytes");
    launch_scores_linear(static_cast<hipStream_t>(stream), x_, w_, bias, *out, workspace);
    return launched(entry);
}
