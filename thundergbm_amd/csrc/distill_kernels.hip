// tgbm_scores_distill: the loss of class scores against a teacher's best scores, and the gradient pairs of a boosting round.
//
// A row's classes fall into those that the teacher names, at most kTeacherMost, and the others. Of the others only the largest
// score and the sum of the exponentials below it count (the softmax's denominator, and their part of it, kept to a reference
// of their own so that it keeps its precision when it is tiny), so a tile of [classes][rows] scores in LDS is enough: the
// named ones are replaced by marks there, what belongs to them stands in a list of [entries][rows], and one pass over the tile
// gives the sums, a second one the pairs. Scores are read once, pairs written once. Classes beyond a tile go by chunks: one
// launch leaves each chunk's sums, a second one adds them up and writes the pairs, which reads the scores a second time.
#include <algorithm>
#include <cfloat>

#include "device_api.h"
#include "score_rules.h"

namespace tgbm {
namespace {

constexpr int kDistillBlock = 256;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kNone = -__builtin_inff();

// Marks in the tile: NaNs that no score is left as (a score that is NaN becomes the one of the hardware).
constexpr unsigned kNaN = 0x7fc00000u, kMark = 0xffc00000u;
__device__ __forceinline__ bool is_mark(unsigned v) { return v >= kMark && v < kMark + kTeacherMost; }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log_of(float x) { return __builtin_amdgcn_logf(x) * kLn2; }
__device__ __forceinline__ float reference_of(float m) { return fabsf(m) <= FLT_MAX ? m : 0.f; }

// Of a sum of exponentials: 0 is one of scores that are all -inf, no class has any probability then; one that is infinite or NaN has
// such a score, and the whole row becomes NaN.
__device__ __forceinline__ float inverse_of(float sum) { return sum == 0.f ? 0.f : sum <= FLT_MAX ? 1.f / sum : __builtin_nanf(""); }

// What a chunk leaves of a row.
struct ChunkSums {
    float other_max, other_sum, other_sum1;  // of the classes that are not named: largest score, sums of exp((z - it) / T) and exp(z - it)
    float named_max, named_sum, named_sum1;
    float cross, mass;  // sum of q (log q - (z - named_max) / T) and of q over the chunk's named classes
    float label;        // z - max(other_max, named_max) of the label, if it is one of the chunk's (else 0)
    float has_label;
};

enum DistillPart { DISTILL_WHOLE, DISTILL_SUMS, DISTILL_PAIRS };

__device__ __forceinline__ float teacher_at(const tgbm_teacher &t, size_t at) {
    if (t.type == TGBM_F32) return static_cast<const float *>(t.scores)[at];
    if (t.type == TGBM_F16) return (float)static_cast<const _Float16 *>(t.scores)[at];
    return (float)static_cast<const __bf16 *>(t.scores)[at];
}

// Sum, or largest, over the threads of a row (thread = slot * R + row): over the lanes of each wavefront, then over the wavefronts.
template <int R, bool MAX>
__device__ __forceinline__ float over_slots(float v, float *room) {
    if constexpr (R == kDistillBlock) return v;
    constexpr int kRows = R < 64 ? R : 64;  // of a wavefront
    for (int d = kRows; d < 64; d <<= 1) {
        const float o = __shfl_xor(v, d);
        v = MAX ? fmaxf(v, o) : v + o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) < kRows) room[(threadIdx.x >> 6) * 64 + (threadIdx.x & (kRows - 1))] = v;
    __syncthreads();
    constexpr int kStep = R > 64 ? R / 64 : 1;  // wavefronts that hold the same rows
    const int first = R > 64 ? (threadIdx.x >> 6) % kStep : 0;
    float all = room[first * 64 + (threadIdx.x & (kRows - 1))];
#pragma unroll
    for (int w = first + kStep; w < kDistillBlock / 64; w += kStep) {
        const float o = room[w * 64 + (threadIdx.x & (kRows - 1))];
        all = MAX ? fmaxf(all, o) : all + o;
    }
    return all;
}

// R rows of a workgroup, kDistillBlock / R threads for each. tile: chunk classes; LDS: [chunk][R] scores, [entries][R] pairs of q and z.
template <int R, DistillPart PART>
__global__ __launch_bounds__(kDistillBlock) void k_distill(tgbm_scores in, tgbm_teacher teacher, const float *__restrict__ labels, float temperature, float weight,
                                                           float *__restrict__ loss, GHPair *__restrict__ pairs, long pair_stride,
                                                           const int *__restrict__ row_of, ChunkSums *__restrict__ sums, int chunks, int chunk,
                                                           long tiles) {
    extern __shared__ unsigned cell[];  // [chunk][R]
    __shared__ float room[kDistillBlock];
    constexpr int kSlots = kDistillBlock / R;
    const int K = teacher.entries;
    float *const q_of = reinterpret_cast<float *>(cell + (size_t)chunk * R);  // [K][R]
    float *const z_of = q_of + (size_t)K * R;
    const int r = threadIdx.x % R, slot = threadIdx.x / R;
    const float by1 = kLog2e, by = kLog2e / temperature;
    const bool hard = labels != nullptr;
    for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        if (PART == DISTILL_PAIRS && pairs == nullptr && tile % chunks != 0) continue;  // (the loss alone)
        const long row = tile / chunks * R + r;
        const bool on = row < in.rows;
        const int c0 = (int)(tile % chunks) * chunk, c1 = min(in.classes, c0 + chunk);
        const float *z = static_cast<const float *>(in.data) + row;
        // rows may lie in another order than the teacher's
        const size_t given = on ? (size_t)(row_of != nullptr ? row_of[row] : row) : 0;
        if (on)
            for (int c = c0 + slot; c < c1; c += kSlots) {
                const float v = z[(size_t)c * in.class_stride];
                cell[(c - c0) * R + r] = v == v ? __float_as_uint(v) : kNaN;
            }
        // the teacher's entries: q
        const int *named = teacher.classes + given * K;
        auto entry = [&](int j, int *c) {  // its score over the temperature; -inf: left out
            *c = on ? named[j] : -1;
            const float t = on ? teacher_at(teacher, given * K + j) / temperature : kNone;
            return (unsigned)*c < (unsigned)in.classes ? t : kNone;
        };
        float top = kNone, any = 0.f;
        int c;
        for (int j = slot; j < K; j += kSlots) {
            const float t = entry(j, &c);
            top = fmaxf(top, t);
            any = t != kNone ? 1.f : any;  // (NaN is an entry)
        }
        any = over_slots<R, true>(any, room);
        float norm;  // log of what the exponentials are divided by
        if (teacher.lse != nullptr) {
            norm = on ? teacher.lse[given] : 0.f;
        } else {
            top = reference_of(over_slots<R, true>(top, room));
            float s = 0.f;
            for (int j = slot; j < K; j += kSlots) s += exp2_of((entry(j, &c) - top) * kLog2e);
            norm = top + log_of(over_slots<R, false>(s, room));
        }
        float mass = 0.f;
        bool twice = false;
        for (int j = slot; j < K; j += kSlots) {
            const float t = entry(j, &c);
            const bool there = t != kNone;
            const float q = there ? exp2_of((t - norm) * kLog2e) : 0.f;
            mass += q;
            const bool mine = there && c >= c0 && c < c1;
            q_of[j * R + r] = q;
            z_of[j * R + r] = mine ? __uint_as_float(cell[(c - c0) * R + r]) : kNone;
        }
        mass = over_slots<R, false>(mass, room);  // (and all entries have read their scores)
        for (int j = slot; j < K; j += kSlots) {
            const bool mine = entry(j, &c) != kNone && c >= c0 && c < c1;
            if (mine) cell[(c - c0) * R + r] = kMark + j;
        }
        __syncthreads();
        for (int j = slot; j < K; j += kSlots) {
            const bool mine = entry(j, &c) != kNone && c >= c0 && c < c1;
            if (mine && cell[(c - c0) * R + r] != kMark + j) twice = true;
        }
        if (__syncthreads_or(twice)) {  // a class that several entries name belongs to the first of them
            for (int j = slot; j < K; j += kSlots) {
                const bool mine = entry(j, &c) != kNone && c >= c0 && c < c1;
                if (mine) atomicMin(&cell[(c - c0) * R + r], kMark + j);
            }
            __syncthreads();
            for (int j = slot; j < K; j += kSlots) {
                const bool mine = entry(j, &c) != kNone && c >= c0 && c < c1;
                if (!mine || cell[(c - c0) * R + r] != kMark + j) continue;
                float q = q_of[j * R + r];
                for (int o = j + 1; o < K; ++o) {
                    int co;
                    if (entry(o, &co) != kNone && co == c) q += q_of[o * R + r];
                }
                q_of[j * R + r] = q;  // (read by nobody else: the others' sums take entries behind their own of other classes)
            }
            __syncthreads();
        }
        // the sums
        ChunkSums sum{};
        float m = kNone;
        if (on)
            for (int i = slot; i < c1 - c0; i += kSlots) {
                const unsigned v = cell[i * R + r];
                if (!is_mark(v)) m = fmaxf(m, __uint_as_float(v));
            }
        sum.other_max = reference_of(over_slots<R, true>(m, room));
        float s = 0.f, s1 = 0.f;
        if (on)
            for (int i = slot; i < c1 - c0; i += kSlots) {
                const unsigned v = cell[i * R + r];
                if (is_mark(v)) continue;
                const float d = __uint_as_float(v) - sum.other_max;
                s += exp2_of(d * by);
                if (hard) s1 += exp2_of(d * by1);
            }
        sum.other_sum = over_slots<R, false>(s, room);
        if (hard) sum.other_sum1 = over_slots<R, false>(s1, room);
        // (the first of a class's entries stands for it)
        auto owner = [&](int j, int *c) { return entry(j, c) != kNone && *c >= c0 && *c < c1 && cell[(*c - c0) * R + r] == kMark + j; };
        m = kNone;
        for (int j = slot; j < K; j += kSlots)
            if (owner(j, &c)) m = fmaxf(m, z_of[j * R + r]);
        sum.named_max = reference_of(over_slots<R, true>(m, room));
        s = s1 = 0.f;
        float cross = 0.f, part = 0.f;
        for (int j = slot; j < K; j += kSlots) {
            if (!owner(j, &c)) continue;
            const float d = z_of[j * R + r] - sum.named_max, q = q_of[j * R + r];
            s += exp2_of(d * by);
            if (hard) s1 += exp2_of(d * by1);
            if (q != 0.f) {
                cross += q * (log_of(q) - d / temperature);
                part += q;
            }
        }
        sum.named_sum = over_slots<R, false>(s, room);
        if (hard) sum.named_sum1 = over_slots<R, false>(s1, room);
        sum.cross = over_slots<R, false>(cross, room);
        sum.mass = over_slots<R, false>(part, room);
        const float y = hard && on ? labels[row] : -1.f;
        const int label = y >= 0.f && y < (float)in.classes && y == floorf(y) ? (int)y : -1;
        if (label >= c0 && label < c1) {
            const unsigned v = cell[(label - c0) * R + r];
            sum.has_label = 1.f;
            const float higher = fmaxf(sum.other_sum > 0.f ? sum.other_max : kNone, sum.named_sum > 0.f ? sum.named_max : kNone);
            sum.label = (is_mark(v) ? z_of[(v - kMark) * R + r] : __uint_as_float(v)) - reference_of(higher);
        }
        if constexpr (PART == DISTILL_SUMS) {
            if (on && slot == 0) sums[row * chunks + tile % chunks] = sum;
            __syncthreads();
            continue;
        }
        // all chunks' sums
        ChunkSums all = sum;
        if constexpr (PART == DISTILL_PAIRS) {
            all = ChunkSums{};
            float mo = kNone, mn = kNone;
            if (on)
                for (int p = 0; p < chunks; ++p) {
                    const ChunkSums &a = sums[row * chunks + p];
                    if (a.other_sum != 0.f) mo = fmaxf(mo, a.other_max);
                    if (a.named_sum != 0.f) mn = fmaxf(mn, a.named_max);
                }
            all.other_max = reference_of(mo);
            all.named_max = reference_of(mn);
            const float higher = reference_of(fmaxf(mo, mn));
            if (on)
                for (int p = 0; p < chunks; ++p) {
                    const ChunkSums &a = sums[row * chunks + p];
                    if (a.other_sum != 0.f) {
                        all.other_sum += a.other_sum * exp2_of((a.other_max - all.other_max) * by);
                        all.other_sum1 += a.other_sum1 * exp2_of((a.other_max - all.other_max) * by1);
                    }
                    if (a.named_sum != 0.f) {
                        const float d = a.named_max - all.named_max;
                        all.named_sum += a.named_sum * exp2_of(d * by);
                        all.named_sum1 += a.named_sum1 * exp2_of(d * by1);
                    }
                    if (a.mass != 0.f) {
                        all.cross += a.cross - a.mass * ((a.named_max - all.named_max) / temperature);
                        all.mass += a.mass;
                    }
                    if (a.has_label != 0.f) {
                        const float own = fmaxf(a.other_sum > 0.f ? a.other_max : kNone, a.named_sum > 0.f ? a.named_max : kNone);
                        all.has_label = 1.f;
                        all.label = a.label + (reference_of(own) - higher);
                    }
                }
        }
        // the row: every probability is an exponential to one of the two references times a factor
        const float no_other = all.other_sum == 0.f ? 1.f : 0.f, no_named = all.named_sum == 0.f ? 1.f : 0.f;
        const float higher = reference_of(fmaxf(no_other != 0.f ? kNone : all.other_max, no_named != 0.f ? kNone : all.named_max));
        const float other_up = no_other != 0.f ? 0.f : exp2_of((all.other_max - higher) * by), named_up = no_named != 0.f ? 0.f : exp2_of((all.named_max - higher) * by);
        const float Z = all.other_sum * other_up + all.named_sum * named_up;
        const float invZ = inverse_of(Z);
        const float a = any == 0.f ? 0.f : mass <= FLT_MAX ? weight : __builtin_nanf(""), b = label >= 0 ? 1.f - weight : 0.f;
        float rest = 0.f;  // the teacher's mass on the other classes
        if (teacher.lse != nullptr && no_other == 0.f && any != 0.f) rest = fmaxf(0.f, 1.f - mass);
        const float named_factor = named_up * invZ;                               // p = exp((z - named_max) / T) * it
        const float other_factor = other_up * invZ;                               // p = exp((z - other_max) / T) * it
        const float target_factor = rest != 0.f ? rest / all.other_sum : 0.f;       // the teacher's share, likewise
        float named_factor1 = 0.f, other_factor1 = 0.f, log_Z1 = 0.f;
        if (hard) {
            const float other_up1 = no_other != 0.f ? 0.f : exp2_of((all.other_max - higher) * by1);
            const float named_up1 = no_named != 0.f ? 0.f : exp2_of((all.named_max - higher) * by1);
            const float Z1 = all.other_sum1 * other_up1 + all.named_sum1 * named_up1;
            const float invZ1 = inverse_of(Z1);
            named_factor1 = named_up1 * invZ1;
            other_factor1 = other_up1 * invZ1;
            log_Z1 = Z1 != 0.f ? log_of(Z1) : 0.f;
        }
        if (loss != nullptr && on && slot == 0 && tile % chunks == 0) {
            float value = 0.f;
            if (a != 0.f) {  // (or NaN)
                const float log_Z = Z != 0.f ? log_of(Z) : 0.f;
                // log p of a named class = (z - named_max) / T - [log Z + (higher - named_max) / T]
                float soft = all.mass != 0.f ? all.cross + all.mass * (log_Z + (higher - all.named_max) / temperature) : 0.f;
                if (rest > 0.f || rest != rest)
                    soft += rest * (log_of(rest) - (log_of(all.other_sum) + (all.other_max - higher) / temperature - log_Z));
                value = a * temperature * temperature * soft;
            }
            if (b != 0.f && all.has_label != 0.f) value += b * (log_Z1 - all.label);
            loss[given] = value;
        }
        if (pairs != nullptr) {
            const float aT = a * temperature;
            auto put = [&](int c, float p, float target, float p1) {
                const float g = aT * (p - target) + b * (p1 - (c == label ? 1.f : 0.f));
                const float h = a * (p * (1.f - p)) + b * (p1 * (1.f - p1));
                pairs[(size_t)c * pair_stride + row] = GHPair{g, 2.f * h < 1e-16f ? 1e-16f : 2.f * h};  // (NaN stays)
            };
            if (on)
                for (int i = slot; i < c1 - c0; i += kSlots) {
                    const unsigned v = cell[i * R + r];
                    if (is_mark(v)) {
                        const int j = (int)(v - kMark);
                        const float d = z_of[j * R + r] - all.named_max;
                        put(c0 + i, exp2_of(d * by) * named_factor, q_of[j * R + r], hard ? exp2_of(d * by1) * named_factor1 : 0.f);
                    } else {
                        const float d = __uint_as_float(v) - all.other_max, e = exp2_of(d * by);
                        put(c0 + i, e * other_factor, e * target_factor, hard ? exp2_of(d * by1) * other_factor1 : 0.f);
                    }
                }
        }
        __syncthreads();  // (the tile is the next one's)
    }
}

// How a call goes: rows of a workgroup, chunks of the classes.
struct DistillPlan {
    int rows, chunks, chunk;
    size_t lds;
};
constexpr size_t kTileBytes = 76 * 1024;  // two workgroups a CU

DistillPlan plan_distill(int classes, int rows, int entries) {
    auto bytes = [&](int chunk, int r) { return sizeof(float) * (size_t)r * ((size_t)chunk + 2 * (size_t)entries); };
    DistillPlan p{};
    p.rows = 1;
    for (int kind : {4, 16})
        if (kind / 2 < rows) p.rows = kind;
    for (int kind : {64, 256})
        if (kind / 2 < rows && bytes(classes, kind) <= kTileBytes) p.rows = kind;
    const long fit = (long)(kTileBytes / sizeof(float) / p.rows) - 2 * entries;
    const long row_tiles = ((long)rows - 1) / p.rows + 1;
    long chunks = bytes(classes, p.rows) <= kTileBytes ? 1 : (classes - 1) / fit + 1;
    if (row_tiles < 256 && classes > 4096) chunks = std::max(chunks, std::min<long>(512 / row_tiles, (classes - 1) / 1024 + 1));
    p.chunk = (int)((classes - 1) / chunks + 1);
    p.chunks = (classes - 1) / p.chunk + 1;
    p.lds = bytes(p.chunk, p.rows);
    return p;
}

template <int R, DistillPart PART>
void distill(hipStream_t s, const DistillPlan &p, const tgbm_scores &in, const tgbm_teacher &teacher, const float *labels, float temperature, float weight,
             float *loss, GHPair *pairs, long pair_stride, const int *row_of, ChunkSums *sums) {
    static LdsOptIn opt_in;
    opt_in({reinterpret_cast<const void *>(&k_distill<R, PART>)});
    const long tiles = (((long)in.rows - 1) / R + 1) * p.chunks;
    k_distill<R, PART><<<(unsigned)std::min(tiles, 1l << 20), kDistillBlock, p.lds, s>>>(in, teacher, labels, temperature, weight, loss, pairs, pair_stride, row_of,
                                                                                       sums, p.chunks, p.chunk, tiles);
}

template <int R>
void distill_rows(hipStream_t s, const DistillPlan &p, const tgbm_scores &in, const tgbm_teacher &teacher, const float *labels, float temperature, float weight,
                  float *loss, GHPair *pairs, long pair_stride, const int *row_of, ChunkSums *sums) {
    if (p.chunks == 1) {
        distill<R, DISTILL_WHOLE>(s, p, in, teacher, labels, temperature, weight, loss, pairs, pair_stride, row_of, nullptr);
    } else {
        distill<R, DISTILL_SUMS>(s, p, in, teacher, labels, temperature, weight, nullptr, nullptr, 0, row_of, sums);
        distill<R, DISTILL_PAIRS>(s, p, in, teacher, labels, temperature, weight, loss, pairs, pair_stride, row_of, sums);
    }
}

}  // namespace

size_t scores_distill_workspace(int classes, int rows, int entries) {
    const DistillPlan p = plan_distill(classes, rows, entries);
    return p.chunks == 1 ? 0 : sizeof(ChunkSums) * (size_t)rows * p.chunks;
}

void launch_scores_distill(hipStream_t s, const tgbm_scores &in, const tgbm_teacher &teacher, const float *labels, float temperature, float weight,
                           float *loss, void *pairs, long pair_stride, const int *row_of, void *workspace) {
    const DistillPlan p = plan_distill(in.classes, in.rows, teacher.entries);
    if (weight == 1.f) labels = nullptr;
    GHPair *gh = static_cast<GHPair *>(pairs);
    ChunkSums *sums = static_cast<ChunkSums *>(workspace);
    switch (p.rows) {
        case 1: distill_rows<1>(s, p, in, teacher, labels, temperature, weight, loss, gh, pair_stride, row_of, sums); break;
        case 4: distill_rows<4>(s, p, in, teacher, labels, temperature, weight, loss, gh, pair_stride, row_of, sums); break;
        case 16: distill_rows<16>(s, p, in, teacher, labels, temperature, weight, loss, gh, pair_stride, row_of, sums); break;
        case 64: distill_rows<64>(s, p, in, teacher, labels, temperature, weight, loss, gh, pair_stride, row_of, sums); break;
        default: distill_rows<256>(s, p, in, teacher, labels, temperature, weight, loss, gh, pair_stride, row_of, sums); break;
    }
}

}  // namespace tgbm
