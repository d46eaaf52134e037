// tgbm_rows_quantise and tgbm_scores_linear: rows of numbers in 8 bits with a scale each, and class scores as their product with a row of weights for every
// class.
//
// q = rint(x / scale), scale = max |x| / 127. A score is (sum of q_x q_w) * scale_x * scale_w + bias: the sum is whole numbers of 32 bits, which 2^16 features
// cannot leave, and exact; three operations of 32 bits and one rounding to the scores' type are behind it.
//
// Rows are brought to a common form first, kChunk features at a time with zeros behind the last: where a row of features is zero it does not matter what
// the weights' rows hold there.
#include "kernel_common.h"
#include "score_rules.h"

namespace tgbm {
namespace {

constexpr int kLinearBlock = 256;
constexpr int kChunk = 128;

typedef int Int4 __attribute__((ext_vector_type(4)));

template <int BLOCK>
__device__ __forceinline__ unsigned block_max_u(unsigned v, unsigned *part) {
    for (int d = 32; d > 0; d /= 2) v = max(v, (unsigned)__shfl_xor((int)v, d));
    if (lane_id() == 0) part[wave_id()] = v;
    __syncthreads();
    for (int w = 0; w < BLOCK / 64; ++w) v = max(v, part[w]);
    return v;
}

// A workgroup takes a row. `pad` bytes from the row's begin on are written: zeros behind its features.
template <typename T>
__global__ __launch_bounds__(kLinearBlock) void k_quantise(const T *x, long long pitch, int features, signed char *q, long long q_pitch, int pad, float *scales) {
    __shared__ unsigned part[kLinearBlock / 64];
    const T *row = x + (size_t)blockIdx.x * pitch;
    unsigned most = 0;
    for (int i = threadIdx.x; i < features; i += kLinearBlock) most = max(most, __float_as_uint(score_to_float(row[i])) & 0x7fffffffu);
    most = block_max_u<kLinearBlock>(most, part);
    const bool fine = most < 0x7f800000u;  // (an infinity or a NaN among them: the row has no scale)
    const float scale = fine ? __uint_as_float(most) / 127.f : __builtin_nanf("");
    if (threadIdx.x == 0) scales[blockIdx.x] = scale;
    signed char *to = q + (size_t)blockIdx.x * q_pitch;
    for (int i = threadIdx.x; i < pad; i += kLinearBlock) {
        float v = 0.f;
        if (i < features && scale > 0.f) v = fminf(fmaxf(rintf(score_to_float(row[i]) / scale), -127.f), 127.f);
        to[i] = (signed char)(int)v;
    }
}

// Rows of whole numbers, moved to rows of `pad` bytes.
__global__ __launch_bounds__(kLinearBlock) void k_pack(const signed char *x, long long pitch, int features, signed char *to, int pad) {
    const signed char *row = x + (size_t)blockIdx.x * pitch;
    for (int i = threadIdx.x; i < pad; i += kLinearBlock) to[(size_t)blockIdx.x * pad + i] = i < features ? row[i] : (signed char)0;
}

// 64 classes x 64 rows to a workgroup, 16 classes to a wavefront. Every operand row's next kChunk bytes at a time.
constexpr int kTile = 64;
struct Rows8 {
    const signed char *data;
    const float *scale;
    long long pitch;
    int rows;
};
template <typename O>
__global__ __launch_bounds__(kLinearBlock) void k_linear(Rows8 x, Rows8 w, int features, const float *bias, O *out, long long class_stride, long long row_stride) {
    __shared__ __align__(16) signed char ws[kTile][kChunk + 16], xs[kTile][kChunk + 16];
    const int c0 = blockIdx.x * kTile, r0 = blockIdx.y * kTile, lane = lane_id(), wave = wave_id();
    const int whole = (features + 15) / 16 * 16;
    Int4 sum[4] = {};
    for (int f0 = 0; f0 < features; f0 += kChunk) {
        __syncthreads();
        for (int i = threadIdx.x; i < kTile * kChunk / 16; i += kLinearBlock) {
            const int row = i / (kChunk / 16), f = i % (kChunk / 16) * 16;
            const Int4 zero = {0, 0, 0, 0};
            // (what lies behind the features of a weights' row meets zeros)
            *reinterpret_cast<Int4 *>(&ws[row][f]) =
                c0 + row < w.rows && f0 + f < whole ? *reinterpret_cast<const Int4 *>(w.data + (size_t)(c0 + row) * w.pitch + f0 + f) : zero;
            *reinterpret_cast<Int4 *>(&xs[row][f]) = r0 + row < x.rows ? *reinterpret_cast<const Int4 *>(x.data + (size_t)(r0 + row) * x.pitch + f0 + f) : zero;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kChunk; k += 64) {
            const Int4 a = *reinterpret_cast<const Int4 *>(&ws[wave * 16 + lane % 16][k + lane / 16 * 16]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const Int4 b = *reinterpret_cast<const Int4 *>(&xs[j * 16 + lane % 16][k + lane / 16 * 16]);
                sum[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, sum[j], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int row = r0 + j * 16 + lane % 16;
        if (row >= x.rows) continue;
        const float by = x.scale[row];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = c0 + wave * 16 + lane / 16 * 4 + i;
            if (c >= w.rows) continue;
            float z = (float)sum[j][i] * by * w.scale[c];
            if (bias != nullptr) z += bias[c];
            out[(size_t)c * class_stride + (size_t)row * row_stride] = (O)z;
        }
    }
}

constexpr size_t kPackedBytes = (size_t)512 << 20;  // of a slice's features

bool lies_well(const tgbm_rows &r) {
    return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.pitch % 16 == 0 && (r.features % 16 == 0 || r.padded);
}
long long pad_of(int features) { return ((long long)features + kChunk - 1) / kChunk * kChunk; }
bool packs_weights(const tgbm_rows &w) { return !lies_well(w); }
bool packs_features(const tgbm_rows &x) { return x.type != TGBM_I8 || !lies_well(x) || x.features % kChunk != 0; }
int packed_rows(const tgbm_rows &x) { return (int)std::max<long long>(1, std::min<long long>(x.rows, (long long)(kPackedBytes / (size_t)pad_of(x.features)))); }
size_t in_lines(size_t bytes) { return (bytes + 127) / 128 * 128; }

template <typename O>
void linear(hipStream_t s, const Rows8 &x, const Rows8 &w, int features, const float *bias, const tgbm_scores &out, int row0) {
    O *to = static_cast<O *>(const_cast<void *>(out.data)) + (size_t)row0 * out.row_stride;
    constexpr int kMost = 65535 * kTile;  // (a direction of a launch)
    for (int r = 0; r < x.rows; r += std::min(kMost, x.rows - r)) {
        Rows8 part = x;
        part.data += (size_t)r * x.pitch;
        part.scale += r;
        part.rows = std::min(kMost, x.rows - r);
        k_linear<O><<<dim3((w.rows - 1) / kTile + 1, (part.rows - 1) / kTile + 1), kLinearBlock, 0, s>>>(part, w, features, bias, to + (size_t)r * out.row_stride,
                                                                                                         out.class_stride, out.row_stride);
    }
}

}  // namespace

void launch_rows_quantise(hipStream_t s, const tgbm_rows &x, signed char *q, long long q_pitch, int pad, float *scale) {
    if (x.type == TGBM_F32) k_quantise<float><<<x.rows, kLinearBlock, 0, s>>>(static_cast<const float *>(x.data), x.pitch, x.features, q, q_pitch, pad, scale);
    else if (x.type == TGBM_F16) k_quantise<_Float16><<<x.rows, kLinearBlock, 0, s>>>(static_cast<const _Float16 *>(x.data), x.pitch, x.features, q, q_pitch, pad, scale);
    else k_quantise<__bf16><<<x.rows, kLinearBlock, 0, s>>>(static_cast<const __bf16 *>(x.data), x.pitch, x.features, q, q_pitch, pad, scale);
}

size_t scores_linear_workspace(const tgbm_rows &x, const tgbm_rows &w) {
    const size_t pad = (size_t)pad_of(x.features);
    size_t bytes = packs_weights(w) ? in_lines(pad * w.rows) : 0;
    if (packs_features(x)) bytes += in_lines(pad * packed_rows(x)) + (x.type != TGBM_I8 ? sizeof(float) * (size_t)packed_rows(x) : 0);
    return bytes;
}

void launch_scores_linear(hipStream_t s, const tgbm_rows &x, const tgbm_rows &w, const float *bias, const tgbm_scores &out, void *workspace) {
    const int pad = (int)pad_of(x.features);
    signed char *room = static_cast<signed char *>(workspace);
    Rows8 weights{static_cast<const signed char *>(w.data), w.scale, w.pitch, w.rows};
    if (packs_weights(w)) {
        k_pack<<<w.rows, kLinearBlock, 0, s>>>(weights.data, w.pitch, w.features, room, pad);
        weights.data = room;
        weights.pitch = pad;
        room += in_lines((size_t)pad * w.rows);
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
                k_pack<<<part.rows, kLinearBlock, 0, s>>>(features.data, x.pitch, x.features, room, pad);
            } else {
                float *scale = reinterpret_cast<float *>(room + in_lines((size_t)pad * most));
                launch_rows_quantise(s, part, room, pad, pad, scale);
                features.scale = scale;
            }
            features.data = room;
            features.pitch = pad;
        }
        if (out.type == TGBM_F32) linear<float>(s, features, weights, x.features, bias, out, row);
        else if (out.type == TGBM_F16) linear<_Float16>(s, features, weights, x.features, bias, out, row);
        else linear<__bf16>(s, features, weights, x.features, bias, out, row);
    }
}

}  // namespace tgbm
