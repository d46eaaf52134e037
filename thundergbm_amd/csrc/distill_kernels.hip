// tgbm_scores_distill: the loss of class scores against a teacher's best scores, and the gradient pairs of a boosting round.
//
// A row's classes fall into those that the teacher names, at most kTeacherMost, and the others. Of the others only the largest
// score and the sum of the exponentials below it count (the softmax's denominator, and their part of it, kept to a reference
// of their own so that it keeps its precision when it is tiny), so a tile of [classes][rows] scores in LDS is enough: the
// named ones are replaced by marks there, what belongs to them stands in a list of [entries][rows], and one pass over the tile
// gives the sums, a second one the pairs. Scores are read once, pairs written once. Classes beyond a tile go by chunks: one
// launch leaves each chunk's sums, a second one adds them up and writes the pairs, which reads the scores a second time. Up to 32
// classes a thread holds its whole row.
//
// Memory bounds it where there are pairs to write: 120011 x 1000, 32 bfloat16 entries and labels, 384 us, 3.8 TB/s (370 us of 120064 rows: with others the
// 128 bytes that 16 rows' pairs of a class are straddle lines). 500000 x 8, five float16 entries and labels: 20 us, 3.4 TB/s. The loss alone is bound by
// the tiles' barriers: 200000 x 100, ten entries, 41 us, 2.4 TB/s. Few rows wait for their chunks' sums: 24 x 50021, 100 entries, 11 and 18 us. The second
// launch works its own chunk's sums out once more on the way to its marks: 20000 x 5000, 32 entries and labels, takes 483 us where bytes alone take 241.
#include <algorithm>
#include <cfloat>

#include "device_api.h"
#include "score_rules.h"

namespace tgbm {
namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kNone = -__builtin_inff();

// Marks in the tile: NaNs that no score is left as (a score that is NaN becomes the one of the hardware).
constexpr unsigned kNaN = 0x7fc00000u, kMark = 0xffc00000u;
__device__ __forceinline__ bool is_mark(unsigned v) { return v - kMark < (unsigned)kTeacherMost; }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log_of(float x) { return __builtin_amdgcn_logf(x) * kLn2; }
// Whether q (log q - log p) counts in the loss: below the least normal number it is 1e-38 times a logarithm, and log_of takes such a q for 0.
__device__ __forceinline__ bool counts_in_loss(float q) { return !(q < FLT_MIN); }  // (a NaN does)
__device__ __forceinline__ float reference_of(float m) { return fabsf(m) <= FLT_MAX ? m : 0.f; }

// Of a sum of exponentials: 0 is one of scores that are all -inf, no class has any probability then; one that is infinite or NaN has
// such a score, and the whole row becomes NaN.
__device__ __forceinline__ float inverse_of(float sum) { return sum == 0.f ? 0.f : sum <= FLT_MAX ? 1.f / sum : __builtin_nanf(""); }

// What the classes of a row, or of a chunk of it, add up to. Sums are those of exp((z - max) / T), and with 1 of exp(z - max).
struct RowSums {
    float other_max, other_sum, other_sum1;  // of the classes that are not named
    float named_max, named_sum, named_sum1;
    float cross, mass;  // sum of q (log q - (z - named_max) / T), and of q, over the named classes
    float label;        // the label's score, where it is one of the classes
};

// What the call is about.
struct DistillCall {
    tgbm_scores in;
    tgbm_teacher teacher;
    const float *labels;  // nullptr: the teacher alone
    float temperature, weight;
    float *loss;
    GHPair *pairs;
    long pair_stride;
    const int *row_of;  // rows may lie in another order than the teacher's
};

__device__ __forceinline__ float teacher_at(const tgbm_teacher &t, size_t at) {
    if (t.type == TGBM_F32) return static_cast<const float *>(t.scores)[at];
    if (t.type == TGBM_F16) return (float)static_cast<const _Float16 *>(t.scores)[at];
    return (float)static_cast<const __bf16 *>(t.scores)[at];
}
__device__ __forceinline__ int label_of(const DistillCall &call, long row) {  // -1: none
    if (call.labels == nullptr) return -1;
    const float y = call.labels[row];
    return y >= 0.f && y < (float)call.in.classes && y == floorf(y) ? (int)y : -1;
}

// What turns a row's scores into pairs. Every probability is an exponential to one of the two references times a factor: with
// e = exp((z - max) / T), e1 = exp(z - max): p = e * p_by, the gradient is e * g_by + e1 * g1_by, less b at the label; a named
// class's is aT * (mass * p - q). mass: of the teacher altogether, entries and rest, as the derivative of -sum q log p is (sum q) p - q over T: 1, but
// where what is left over has no class to go to, or the entries have more than 1 together.
struct RowFactors {
    float other_max, other_p, other_p1, other_g;
    float named_max, named_p, named_p1;
    float a, b, aT, mass;  // a: the weight, times the mass for the hessian
};

// sum: of all classes; any: the teacher names a class; given: the sum of all entries' q; label < 0: none. Returns the loss as well.
__device__ __forceinline__ RowFactors factors_of(const RowSums &sum, bool any, float given, bool has_rest, int label, float temperature, float weight, float *loss) {
    const float by = kLog2e / temperature;
    const bool others = sum.other_sum != 0.f, named = sum.named_sum != 0.f;
    const float higher = reference_of(fmaxf(others ? sum.other_max : kNone, named ? sum.named_max : kNone));
    const float other_up = others ? exp2_of((sum.other_max - higher) * by) : 0.f, named_up = named ? exp2_of((sum.named_max - higher) * by) : 0.f;
    const float Z = sum.other_sum * other_up + sum.named_sum * named_up, inv = inverse_of(Z);
    RowFactors f;
    f.a = !any ? 0.f : given <= FLT_MAX ? weight : __builtin_nanf("");
    f.b = label >= 0 ? 1.f - weight : 0.f;
    f.aT = f.a * temperature;
    const bool takes = has_rest && others && any;
    const float rest = takes ? fmaxf(0.f, 1.f - given) : 0.f;  // the teacher's mass on the other classes
    f.mass = !has_rest ? 1.f : takes ? fmaxf(given, 1.f) : given;
    f.other_max = sum.other_max;
    f.named_max = sum.named_max;
    f.other_p = other_up * inv;
    f.named_p = named_up * inv;
    f.other_g = f.aT * (f.mass * f.other_p - (rest != 0.f ? rest / sum.other_sum : 0.f));
    f.other_p1 = f.named_p1 = 0.f;
    float log_Z1 = 0.f;
    if (label >= 0) {
        const float other_up1 = others ? exp2_of((sum.other_max - higher) * kLog2e) : 0.f, named_up1 = named ? exp2_of((sum.named_max - higher) * kLog2e) : 0.f;
        const float Z1 = sum.other_sum1 * other_up1 + sum.named_sum1 * named_up1, inv1 = inverse_of(Z1);
        f.other_p1 = other_up1 * inv1;
        f.named_p1 = named_up1 * inv1;
        log_Z1 = Z1 != 0.f ? log_of(Z1) : 0.f;
    }
    float value = 0.f;
    if (f.a != 0.f) {  // (or NaN)
        const float log_Z = Z != 0.f ? log_of(Z) : 0.f;
        // log p of a named class is (z - named_max) / T less log Z + (higher - named_max) / T
        float soft = sum.mass != 0.f ? sum.cross + sum.mass * (log_Z + (higher - sum.named_max) / temperature) : 0.f;
        if (rest != 0.f) soft += rest * (log_of(rest) - (log_of(sum.other_sum) + (sum.other_max - higher) / temperature - log_Z));
        value = f.a * temperature * temperature * soft;
    }
    if (f.b != 0.f) value += f.b * (log_Z1 - (sum.label - higher));
    *loss = value;
    f.a *= f.mass;
    return f;
}

// g and h from p, p1 and the gradient before the label's part.
__device__ __forceinline__ GHPair pair_of(const RowFactors &f, float p, float p1, float g, bool is_label) {
    const float h = 2.f * (f.a * (p * (1.f - p)) + f.b * (p1 * (1.f - p1)));
    return GHPair{g + f.b * (p1 - (is_label ? 1.f : 0.f)), h < 1e-16f ? 1e-16f : h};  // (NaN stays)
}

// ------------------------------------------------------------------------------------------------------ few classes
constexpr int kFewBlock = 256;
template <int C>
__global__ __launch_bounds__(kFewBlock) void k_distill_few(DistillCall call) {
    const long row = (long)blockIdx.x * kFewBlock + threadIdx.x;
    if (row >= call.in.rows) return;
    const int classes = call.in.classes, K = call.teacher.entries;
    const size_t given_row = (size_t)(call.row_of != nullptr ? call.row_of[row] : row);
    const float by = kLog2e / call.temperature;
    const bool hard = call.labels != nullptr;
    const float *from = static_cast<const float *>(call.in.data) + row;
    float z[C], q[C];
#pragma unroll
    for (int c = 0; c < C; ++c) z[c] = c < classes ? from[(size_t)c * call.in.class_stride] : kNone;
    // the teacher: what the entries of a class add up to
    const int *named = call.teacher.classes + given_row * K;
    float top = kNone;
    unsigned there = 0;  // (bit c: class c is named)
    for (int j = 0; j < K; ++j) {
        const int c = named[j];
        const float t = teacher_at(call.teacher, given_row * K + j);
        if ((unsigned)c < (unsigned)classes && t != kNone) {
            top = fmaxf(top, t);
            there |= 1u << c;
        }
    }
    top = reference_of(top);
#pragma unroll
    for (int c = 0; c < C; ++c) q[c] = 0.f;
    float sum_q = 0.f;
    for (int j = 0; j < K; ++j) {
        const int c = named[j];
        const float t = teacher_at(call.teacher, given_row * K + j);
        const float e = (unsigned)c < (unsigned)classes && t != kNone ? exp2_of((t - top) * by) : 0.f;
        sum_q += e;
#pragma unroll
        for (int o = 0; o < C; ++o) q[o] += o == c ? e : 0.f;
    }
    const bool rest = call.teacher.lse != nullptr, any = there != 0;
    const float scale = rest ? exp2_of((top / call.temperature - call.teacher.lse[given_row]) * kLog2e) : any ? 1.f / sum_q : 0.f;
    RowSums s{};
    const int label = label_of(call, row);
    float mo = kNone, mn = kNone;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        q[c] *= scale;
        if (there >> c & 1u) mn = fmaxf(mn, z[c]);
        else mo = fmaxf(mo, z[c]);
        s.label = c == label ? z[c] : s.label;
    }
    s.other_max = reference_of(mo);
    s.named_max = reference_of(mn);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const bool is_named = there >> c & 1u;
        const float d = z[c] - (is_named ? s.named_max : s.other_max), e = exp2_of(d * by), e1 = hard ? exp2_of(d * kLog2e) : 0.f;
        s.named_sum += is_named ? e : 0.f;
        s.other_sum += is_named || c >= classes ? 0.f : e;
        s.named_sum1 += is_named ? e1 : 0.f;
        s.other_sum1 += is_named || c >= classes ? 0.f : e1;
        if (is_named && counts_in_loss(q[c])) {
            s.cross += q[c] * (log_of(q[c]) - d / call.temperature);
            s.mass += q[c];
        }
    }
    float value;
    const RowFactors f = factors_of(s, any, any ? sum_q * scale : 0.f, rest, label, call.temperature, call.weight, &value);
    if (call.loss != nullptr) call.loss[given_row] = value;
    if (call.pairs == nullptr) return;
    GHPair *to = call.pairs + row;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const bool is_named = there >> c & 1u;
        const float d = z[c] - (is_named ? f.named_max : f.other_max), e = exp2_of(d * by), e1 = hard ? exp2_of(d * kLog2e) : 0.f;
        const float p = e * (is_named ? f.named_p : f.other_p), p1 = e1 * (is_named ? f.named_p1 : f.other_p1);
        if (c < classes) *to = pair_of(f, p, p1, is_named ? f.aT * (f.mass * p - q[c]) : e * f.other_g, c == label);
        to += call.pair_stride;
    }
}

// ----------------------------------------------------------------------------------------------------- more classes
enum DistillPart { DISTILL_WHOLE, DISTILL_SUMS, DISTILL_PAIRS };

// R rows of a workgroup of B threads, thread = slot * R + row.
template <int R, int B>
struct Rows {
    static constexpr int kSlots = B / R, kWaves = B / 64, kLanes = R < 64 ? R : 64;  // kLanes: rows of a wavefront
    static_assert(R <= 64);
    static constexpr int kMostValues = 6;
    float part[kMostValues][kWaves][kLanes], all[kMostValues][kLanes];

    // Sums over a row's threads (largest of the first MAXIMA), the same in all of them: over lanes, then over wavefronts.
    template <int N, int MAXIMA>
    __device__ __forceinline__ void reduce(float (&v)[N]) {
        static_assert(N <= kMostValues && N * kLanes <= B);
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int d = kLanes; d < 64; d <<= 1) {
                const float o = __shfl_xor(v[k], d);
                v[k] = k < MAXIMA ? fmaxf(v[k], o) : v[k] + o;
            }
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = threadIdx.x & (kLanes - 1);
        if (lane < kLanes) {
#pragma unroll
            for (int k = 0; k < N; ++k) part[k][wave][lane] = v[k];
        }
        __syncthreads();
        if (threadIdx.x < N * kLanes) {
            const int k = threadIdx.x / kLanes;
            float x = part[k][0][r];
            for (int w = 1; w < kWaves; ++w) x = k < MAXIMA ? fmaxf(x, part[k][w][r]) : x + part[k][w][r];
            all[k][r] = x;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = all[k][r];
    }
};

// LDS: [chunk][R] scores; then of the entries [K][R + 1]: their classes, q, and scores.
template <int R, int B, DistillPart PART>
__global__ __launch_bounds__(B, 8) void k_distill(DistillCall call, RowSums *__restrict__ sums, int chunks, int chunk) {
    using Group = Rows<R, B>;
    constexpr int kSlots = Group::kSlots, kPitch = R + 1;
    __shared__ Group group;
    __shared__ RowFactors factors[R];
    __shared__ float label_score[R];
    extern __shared__ unsigned cell[];
    const int K = call.teacher.entries;
    int *const class_of = reinterpret_cast<int *>(cell + (size_t)chunk * R);
    float *const q_of = reinterpret_cast<float *>(class_of + K * kPitch), *const z_of = q_of + K * kPitch;
    const int r = threadIdx.x % R, slot = threadIdx.x / R;
    const long tile = tile_of_block(blockIdx.x, gridDim.x);
    const long row0 = tile * R, row = row0 + r;
    if (row0 >= call.in.rows) return;
    const bool on = row < call.in.rows, hard = call.labels != nullptr;
    const int c0 = blockIdx.y * chunk, size = min(call.in.classes - c0, chunk);
    const float by = kLog2e / call.temperature;
    const float *from = static_cast<const float *>(call.in.data) + (size_t)c0 * call.in.class_stride + row;
    const auto given_of = [&](long i) { return (size_t)(call.row_of != nullptr ? call.row_of[i] : i); };

    if (on) {
        for (int c = slot; c < size; c += 8 * kSlots) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c + j * kSlots < size ? from[(size_t)(c + j * kSlots) * call.in.class_stride] : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j * kSlots < size) cell[(c + j * kSlots) * R + r] = v[j] == v[j] ? __float_as_uint(v[j]) : kNaN;
        }
    }
    // the entries: their scores for now, -1 for the class of one that is left out
    for (int i = threadIdx.x; i < R * K; i += B) {
        const int of = i / K, j = i - of * K;
        int c = -1;
        float t = kNone;
        if (row0 + of < call.in.rows) {
            const size_t at = given_of(row0 + of) * K + j;
            c = call.teacher.classes[at];
            t = teacher_at(call.teacher, at);
        }
        class_of[j * kPitch + of] = (unsigned)c < (unsigned)call.in.classes && t != kNone ? c : -1;
        q_of[j * kPitch + of] = t;
    }
    if (threadIdx.x < R) label_score[threadIdx.x] = 0.f;
    __syncthreads();
    float first[2] = {kNone, kNone};  // the largest, and whether there is one (NaN is an entry)
    for (int j = slot; j < K; j += kSlots)
        if (class_of[j * kPitch + r] >= 0) {
            first[0] = fmaxf(first[0], q_of[j * kPitch + r]);
            first[1] = 1.f;
        }
    group.template reduce<2, 2>(first);
    const bool any = first[1] == 1.f;
    // q = exp((t - top) / T) * scale: below the row's best entry before anything is rounded, as what all scores have in common may be large over T
    const float top = reference_of(first[0]);
    float scale;
    if (call.teacher.lse != nullptr) {
        scale = on ? exp2_of((top / call.temperature - call.teacher.lse[given_of(row)]) * kLog2e) : 0.f;
    } else {
        float s[1] = {0.f};
        for (int j = slot; j < K; j += kSlots)
            if (class_of[j * kPitch + r] >= 0) s[0] += exp2_of((q_of[j * kPitch + r] - top) * by);
        group.template reduce<1, 0>(s);
        scale = any ? 1.f / s[0] : 0.f;
    }
    float given = 0.f;
    for (int j = slot; j < K; j += kSlots) {
        const int c = class_of[j * kPitch + r] - c0;
        if (c + c0 < 0) continue;
        const float q = exp2_of((q_of[j * kPitch + r] - top) * by) * scale;
        given += q;
        q_of[j * kPitch + r] = q;
        if (c >= 0 && c < size) z_of[j * kPitch + r] = __uint_as_float(cell[c * R + r]);
        else class_of[j * kPitch + r] = -1;  // (another chunk's)
    }
    __syncthreads();
    for (int j = slot; j < K; j += kSlots) {
        const int c = class_of[j * kPitch + r] - c0;
        if (c >= 0) cell[c * R + r] = kMark + j;
    }
    __syncthreads();
    bool twice = false;
    for (int j = slot; j < K; j += kSlots) {
        const int c = class_of[j * kPitch + r] - c0;
        twice |= c >= 0 && cell[c * R + r] != kMark + j;
    }
    if (__syncthreads_or(twice)) {  // a class that several entries name belongs to the first of them
        for (int j = slot; j < K; j += kSlots) {
            const int c = class_of[j * kPitch + r] - c0;
            if (c >= 0) atomicMin(&cell[c * R + r], kMark + j);
        }
        __syncthreads();
        for (int j = slot; j < K; j += kSlots) {
            const int c = class_of[j * kPitch + r] - c0;
            if (c < 0 || cell[c * R + r] != kMark + j) continue;
            float q = q_of[j * kPitch + r];
            for (int o = j + 1; o < K; ++o)
                if (class_of[o * kPitch + r] == c + c0) q += q_of[o * kPitch + r];
            q_of[j * kPitch + r] = q;  // (nobody else reads it: the others' sums are of other classes)
        }
        __syncthreads();
        for (int j = slot; j < K; j += kSlots) {
            const int c = class_of[j * kPitch + r] - c0;
            if (c >= 0 && cell[c * R + r] != kMark + j) class_of[j * kPitch + r] = -1;
        }
    }
    // the sums
    float most[3] = {kNone, kNone, given};
    if (on) {
#pragma unroll 4
        for (int i = slot; i < size; i += kSlots) {
            const unsigned v = cell[i * R + r];
            most[0] = fmaxf(most[0], is_mark(v) ? kNone : __uint_as_float(v));
        }
    }
    for (int j = slot; j < K; j += kSlots)
        if (class_of[j * kPitch + r] >= 0) most[1] = fmaxf(most[1], z_of[j * kPitch + r]);
    group.template reduce<3, 2>(most);
    given = most[2];
    RowSums sum{};
    sum.other_max = reference_of(most[0]);
    sum.named_max = reference_of(most[1]);
    float s[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (on) {
#pragma unroll 4
        for (int i = slot; i < size; i += kSlots) {
            const unsigned v = cell[i * R + r];
            const float d = is_mark(v) ? kNone : __uint_as_float(v) - sum.other_max;
            s[0] += exp2_of(d * by);
            if (hard) s[1] += exp2_of(d * kLog2e);
        }
    }
    const int label = on ? label_of(call, row) : -1;
    for (int j = slot; j < K; j += kSlots) {
        const int c = class_of[j * kPitch + r];
        if (c < 0) continue;
        const float z = z_of[j * kPitch + r], d = z - sum.named_max, q = q_of[j * kPitch + r];
        s[2] += exp2_of(d * by);
        if (hard) s[3] += exp2_of(d * kLog2e);
        if (counts_in_loss(q)) {
            s[4] += q * (log_of(q) - d / call.temperature);
            s[5] += q;
        }
        if (c == label) label_score[r] = z;
    }
    if (slot == 0 && label >= c0 && label < c0 + size && !is_mark(cell[(label - c0) * R + r])) label_score[r] = __uint_as_float(cell[(label - c0) * R + r]);
    group.template reduce<6, 0>(s);
    sum.other_sum = s[0];
    sum.other_sum1 = s[1];
    sum.named_sum = s[2];
    sum.named_sum1 = s[3];
    sum.cross = s[4];
    sum.mass = s[5];
    sum.label = label_score[r];
    if constexpr (PART == DISTILL_SUMS) {
        if (on && slot == 0) sums[row * chunks + blockIdx.y] = sum;
        return;
    }
    if constexpr (PART == DISTILL_PAIRS) {
        // all chunks' sums: a row's threads share them out
        const RowSums *its = sums + row * chunks;
        float m[2] = {kNone, kNone};
        if (on)
            for (int p = slot; p < chunks; p += kSlots) {
                if (its[p].other_sum != 0.f) m[0] = fmaxf(m[0], its[p].other_max);
                if (its[p].named_sum != 0.f) m[1] = fmaxf(m[1], its[p].named_max);
            }
        group.template reduce<2, 2>(m);
        sum.other_max = reference_of(m[0]);
        sum.named_max = reference_of(m[1]);
        float a[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, l[1] = {0.f};
        if (on)
            for (int p = slot; p < chunks; p += kSlots) {
                const RowSums c = its[p];
                if (c.other_sum != 0.f) {
                    a[0] += c.other_sum * exp2_of((c.other_max - sum.other_max) * by);
                    a[1] += c.other_sum1 * exp2_of((c.other_max - sum.other_max) * kLog2e);
                }
                if (c.named_sum != 0.f) {
                    const float d = c.named_max - sum.named_max;
                    a[2] += c.named_sum * exp2_of(d * by);
                    a[3] += c.named_sum1 * exp2_of(d * kLog2e);
                }
                if (c.mass != 0.f) {
                    a[4] += c.cross - c.mass * ((c.named_max - sum.named_max) / call.temperature);
                    a[5] += c.mass;
                }
                if (label >= p * chunk && label < (p + 1) * chunk) l[0] = c.label;
            }
        group.template reduce<6, 0>(a);
        group.template reduce<1, 0>(l);
        sum.other_sum = a[0];
        sum.other_sum1 = a[1];
        sum.named_sum = a[2];
        sum.named_sum1 = a[3];
        sum.cross = a[4];
        sum.mass = a[5];
        sum.label = l[0];
    }
    if (slot == 0) {
        float value;
        factors[r] = factors_of(sum, any, given, call.teacher.lse != nullptr, label, call.temperature, call.weight, &value);
        if (call.loss != nullptr && on && blockIdx.y == 0) call.loss[given_of(row)] = value;
    }
    if (call.pairs == nullptr) return;
    __syncthreads();
    if (!on) return;
    const RowFactors f = factors[r];
    GHPair *const to = call.pairs + (size_t)c0 * call.pair_stride + row;
#pragma unroll 2
    for (int i = slot; i < size; i += kSlots) {
        const unsigned v = cell[i * R + r];
        const bool named = is_mark(v);
        float z = __uint_as_float(v), q = 0.f;
        if (named) {
            z = z_of[(v - kMark) * kPitch + r];
            q = q_of[(v - kMark) * kPitch + r];
        }
        const float d = z - (named ? f.named_max : f.other_max), e = exp2_of(d * by), e1 = hard ? exp2_of(d * kLog2e) : 0.f;
        const float p = e * (named ? f.named_p : f.other_p), p1 = e1 * (named ? f.named_p1 : f.other_p1);
        to[(size_t)i * call.pair_stride] = pair_of(f, p, p1, named ? f.aT * (f.mass * p - q) : e * f.other_g, c0 + i == label);
    }
}

// How a call goes: rows of a workgroup, chunks of the classes.
struct DistillPlan {
    int rows, threads, chunks, chunk;  // rows 0: few classes
    size_t lds;
};
constexpr int kFewClasses = 32;
constexpr size_t kMostBytes = 144 * 1024;  // one workgroup a CU,
constexpr size_t kTileBytes = 72 * 1024;   // or two
constexpr size_t kSmallBytes = 36 * 1024, kMediumBytes = 48 * 1024;
constexpr int kManyRows = 16384;

DistillPlan plan_distill(int classes, int rows, int entries) {
    DistillPlan p{};
    p.chunks = 1;
    p.chunk = classes;
    if (classes <= kFewClasses) return p;
    auto bytes = [&](int chunk, int r) { return sizeof(float) * ((size_t)r * chunk + 3 * (size_t)entries * (r + 1)); };
    p.rows = rows <= 2 ? 1 : rows <= 8 ? 4 : 16;
    // Much of a workgroup's time goes by at barriers, where another one's work fills in: as many threads as four, three or two workgroups a CU (that LDS has
    // room for) need to have their loads on their way. 166 666 x 120, 10 entries: 73 us with 32 rows and 256 threads, 183 with 16 and 1024; 100 000 x 200, 32
    // entries: 76 with 16 and 256, 129 with 16 and 1024; 40 000 x 500: 70 with 16 and 512, 79 with 16 and 1024; 20 000 x 1000: 67, 65.
    p.threads = 1024;
    const bool many = rows >= kManyRows;
    if (many && bytes(classes, 32) <= kSmallBytes) {
        p.rows = 32;
        p.threads = 256;
    } else if (many && bytes(classes, 16) <= kMediumBytes) {
        p.threads = bytes(classes, 16) <= kSmallBytes ? 256 : 512;
    }
    const long row_tiles = ((long)rows - 1) / p.rows + 1;
    long chunks = 1;
    if (bytes(classes, p.rows) > kMostBytes) chunks = (classes - 1) / (long)((kTileBytes / sizeof(float) - 3 * (size_t)entries * (p.rows + 1)) / p.rows) + 1;
    // few rows: their classes are shared out over the chip, 512 at least to a workgroup (24 x 50021: 29 us; 256 at least: 41, more sums to add up for each)
    if (row_tiles < 128 && classes > 2048) chunks = std::max(chunks, std::min<long>(512 / row_tiles, (classes - 1) / 512 + 1));
    p.chunk = (int)((classes - 1) / chunks + 1);
    p.chunks = (classes - 1) / p.chunk + 1;
    p.lds = bytes(p.chunk, p.rows);
    return p;
}

template <int R, int B, DistillPart PART>
void distill_part(hipStream_t s, const DistillPlan &p, const DistillCall &call, RowSums *sums) {
    static LdsOptIn opt_in;
    opt_in({reinterpret_cast<const void *>(&k_distill<R, B, PART>)});
    const unsigned tiles = (unsigned)((call.in.rows - 1) / R + 1);
    // (the loss alone needs one chunk's workgroup to add up)
    const dim3 grid(blocks_of_tiles(tiles), PART == DISTILL_PAIRS && call.pairs == nullptr ? 1 : p.chunks);
    k_distill<R, B, PART><<<grid, B, p.lds, s>>>(call, sums, p.chunks, p.chunk);
}

template <int R, int B>
void distill_rows(hipStream_t s, const DistillPlan &p, const DistillCall &call, RowSums *sums) {
    if constexpr (B == 1024) {  // (tiles of fewer threads hold all classes)
        if (p.chunks > 1) {
            distill_part<R, B, DISTILL_SUMS>(s, p, call, sums);
            distill_part<R, B, DISTILL_PAIRS>(s, p, call, sums);
            return;
        }
    }
    distill_part<R, B, DISTILL_WHOLE>(s, p, call, nullptr);
}

}  // namespace

size_t scores_distill_workspace(int classes, int rows, int entries) {
    return workspace_of_slices(rows, [&](int slice) {
        const DistillPlan p = plan_distill(classes, slice, entries);
        return p.chunks == 1 ? 0 : sizeof(RowSums) * (size_t)slice * p.chunks;
    });
}

void launch_scores_distill(hipStream_t s, const tgbm_scores &in, const tgbm_teacher &teacher, const float *labels, float temperature, float weight,
                           float *loss, void *pairs, long pair_stride, const int *row_of, void *workspace) {
    RowSums *sums = static_cast<RowSums *>(workspace);
    const size_t score = teacher.type == TGBM_F32 ? 4 : 2;
    for (int row = 0; row < in.rows; row += std::min(kSliceRows, in.rows - row)) {
        DistillCall call{in, teacher, weight == 1.f ? nullptr : labels, temperature, weight, loss, static_cast<GHPair *>(pairs), pair_stride, row_of};
        call.in.data = static_cast<const float *>(in.data) + row;
        call.in.rows = std::min(kSliceRows, in.rows - row);
        if (call.labels != nullptr) call.labels += row;
        if (call.pairs != nullptr) call.pairs += row;
        if (row_of != nullptr) {
            call.row_of += row;
        } else {
            const size_t first = (size_t)row * teacher.entries;
            call.teacher.classes += first;
            call.teacher.scores = static_cast<const char *>(teacher.scores) + first * score;
            if (teacher.lse != nullptr) call.teacher.lse += row;
            if (loss != nullptr) call.loss += row;
        }
        const DistillPlan p = plan_distill(in.classes, call.in.rows, teacher.entries);
        const unsigned few = (unsigned)((call.in.rows - 1) / kFewBlock + 1);
        switch (p.rows) {
            case 0:
                if (in.classes <= 8) k_distill_few<8><<<few, kFewBlock, 0, s>>>(call);
                else if (in.classes <= 16) k_distill_few<16><<<few, kFewBlock, 0, s>>>(call);
                else k_distill_few<32><<<few, kFewBlock, 0, s>>>(call);
                break;
            case 1: distill_rows<1, 1024>(s, p, call, sums); break;
            case 4: distill_rows<4, 1024>(s, p, call, sums); break;
            case 32: distill_rows<32, 256>(s, p, call, sums); break;
            default:
                if (p.threads == 256) distill_rows<16, 256>(s, p, call, sums);
                else if (p.threads == 512) distill_rows<16, 512>(s, p, call, sums);
                else distill_rows<16, 1024>(s, p, call, sums);
                break;
        }
    }
}

}  // namespace tgbm
