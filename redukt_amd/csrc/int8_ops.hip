// int8_ops.hip — int8 codes of activation rows and the product of codes (redukt_ops.h).
#include <hip/hip_runtime.h>

#include "op_common.h"

// The recipe's scale, inverse and scaled value are each rounded to f32: nothing is fused.
#pragma clang fp contract(off)

namespace rdk {
namespace {

constexpr int kWave = 64;
constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;

typedef int i32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- codes

__device__ __forceinline__ int8_t code_of(float v, float inv) {
    float t = roundf(v * inv);
    if (t < -127.0f) t = -127.0f;
    if (t > 127.0f) t = 127.0f;
    return t != t ? (int8_t)0 : (int8_t)(int)t;
}

// |v| into a running maximum that a NaN never enters.
__device__ __forceinline__ float fold_abs(float m, float v) {
    const float a = fabsf(v);
    return a > m ? a : m;
}

// One workgroup a row: the row's maximum, then its codes from a second read.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_quantize_rows(redukt_quantize_rows a) {
    __shared__ float wm[kWaves];
    const uint32_t r = blockIdx.x;
    const T* x = (const T*)a.x + (int64_t)r * a.x_stride;
    float m = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kBlock) m = fold_abs(m, (float)x[c]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fold_abs(m, __shfl_xor(m, o, kWave));
    if (threadIdx.x % kWave == 0) wm[threadIdx.x / kWave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; w++) m = fold_abs(m, wm[w]);
    const float scale = m > 0.0f ? m / 127.0f : 1.0f;
    const float inv = 1.0f / scale;
    int8_t* q = a.codes + (int64_t)r * a.codes_stride;
    for (uint32_t c = threadIdx.x; c < a.cols; c += kBlock) q[c] = code_of((float)x[c], inv);
    if (threadIdx.x == 0) a.scales[r] = scale;
}

// ---------------------------------------------------------------- product

// v_mfma_i32_16x16x64_i8: lane l holds 16 consecutive codes of row l % 16, the columns 16 (l / 16)
// + [0, 16); of the result, column l % 16 of rows 4 (l / 16) + [0, 4).
__device__ __forceinline__ i32x4 mma8(const i32x4& a, const i32x4& b, const i32x4& c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// Codes of any alignment: 64 x 64 outputs a workgroup, 64 columns at a time staged byte by byte
// with zeros outside the operands.
constexpr int kTile = 64, kPitch = kTile + 16;
template <typename T>
__global__ __launch_bounds__(kBlock) void k_int8_bytes(redukt_int8_matmul a) {
    __shared__ __attribute__((aligned(16))) int8_t sx[kTile * kPitch], sw[kTile * kPitch];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t i0 = blockIdx.y * kTile, j0 = blockIdx.x * kTile;
    i32x4 acc[4] = {};
    for (uint32_t c0 = 0; c0 < a.k; c0 += kTile) {
        for (int e = threadIdx.x; e < kTile * kTile; e += kBlock) {
            const uint32_t r = e / kTile, c = c0 + e % kTile;
            sx[r * kPitch + e % kTile] = i0 + r < a.m && c < a.k ? a.x[(int64_t)(i0 + r) * a.x_stride + c] : 0;
            sw[r * kPitch + e % kTile] = j0 + r < a.n && c < a.k ? a.w[(int64_t)(j0 + r) * a.w_stride + c] : 0;
        }
        __syncthreads();
        const i32x4 fx = *(const i32x4*)(sx + (16 * wave + lane % 16) * kPitch + 16 * (lane / 16));
#pragma unroll
        for (int t = 0; t < 4; t++)
            acc[t] = mma8(fx, *(const i32x4*)(sw + (16 * t + lane % 16) * kPitch + 16 * (lane / 16)), acc[t]);
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const uint32_t j = j0 + 16 * t + lane % 16;
        if (j >= a.n) continue;
        const float ws = a.w_scales[j], bias = a.bias ? a.bias[j] : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t i = i0 + 16 * wave + 4 * (lane / 16) + e;
            if (i >= a.m) continue;
            const float y = (float)acc[t][e] * (a.x_scales[i] * ws);
            ((T*)a.out)[(int64_t)i * a.out_stride + j] = (T)(a.bias ? y + bias : y);
        }
    }
}

const void* by_type(uint32_t dtype, const void* bf16, const void* f16, const void* f32) {
    return dtype == REDUKT_OP_BF16 ? bf16 : dtype == REDUKT_OP_F16 ? f16 : f32;
}

}  // namespace
}  // namespace rdk

using namespace rdk;

extern "C" {

int32_t redukt_op_quantize_rows(const redukt_quantize_rows* a, void* stream) {
    if (!a || a->dtype > REDUKT_OP_F32 || a->rows >= (1u << 31) || a->cols >= (1u << 31)) return BACKEND_INVALID_ARGUMENT;
    if (a->rows == 0) return BACKEND_OK;
    if (!a->scales || !op_aligned(a->scales, 4)) return BACKEND_INVALID_ARGUMENT;
    if (a->cols && (!a->x || !a->codes || !op_aligned(a->x, op_elem_bytes(a->dtype)))) return BACKEND_INVALID_ARGUMENT;
    if (a->rows > 1 && a->cols && (a->codes_stride < (int64_t)a->cols || (a->x_stride != 0 && a->x_stride < (int64_t)a->cols)))
        return BACKEND_INVALID_ARGUMENT;
    OpDevice dev(a->scales);
    if (!dev.ok) return BACKEND_INVALID_ARGUMENT;
    redukt_quantize_rows k = *a;
    const void* fn = by_type(a->dtype, (const void*)k_quantize_rows<__bf16>, (const void*)k_quantize_rows<_Float16>,
                             (const void*)k_quantize_rows<float>);
    return op_launch(fn, dim3(a->rows), dim3(kBlock), 0, stream, k);
}

int32_t redukt_op_int8_matmul(const redukt_int8_matmul* a, void* stream) {
    if (!a || a->dtype > REDUKT_OP_F32 || a->m >= (1u << 31) || a->n >= (1u << 31) || a->k > 131000)
        return BACKEND_INVALID_ARGUMENT;
    if (a->m == 0 || a->n == 0) return BACKEND_OK;
    if (!a->out || !op_aligned(a->out, op_elem_bytes(a->dtype)) || (a->m > 1 && a->out_stride < (int64_t)a->n))
        return BACKEND_INVALID_ARGUMENT;
    if (!a->x_scales || !a->w_scales || !op_aligned(a->x_scales, 4) || !op_aligned(a->w_scales, 4) || !op_aligned(a->bias, 4))
        return BACKEND_INVALID_ARGUMENT;
    if (a->k && (!a->x || !a->w)) return BACKEND_INVALID_ARGUMENT;
    if ((a->m > 1 && a->x_stride != 0 && a->x_stride < (int64_t)a->k) ||
        (a->n > 1 && a->w_stride != 0 && a->w_stride < (int64_t)a->k))
        return BACKEND_INVALID_ARGUMENT;
    OpDevice dev(a->out);
    if (!dev.ok) return BACKEND_INVALID_ARGUMENT;
    redukt_int8_matmul k = *a;
    const void* fn = by_type(a->dtype, (const void*)k_int8_bytes<__bf16>, (const void*)k_int8_bytes<_Float16>,
                             (const void*)k_int8_bytes<float>);
    const dim3 grid((a->n + kTile - 1) / kTile, (a->m + kTile - 1) / kTile);
    if (grid.y > 65535) return BACKEND_INVALID_ARGUMENT;
    return op_launch(fn, grid, dim3(kBlock), 0, stream, k);
}

}  // extern "C"
