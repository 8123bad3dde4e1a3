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

// v / scale to the nearest whole number, halves away from zero, as an int in [-127, 127]; NaN gives 0.  Adding the largest f32
// below 1/2 with v's sign and dropping the fraction rounds so: the sum of a half and it is a tie, which goes up to the even 1 (and
// so on up to 2^22), and that of the largest value below a half stays below 1.  The conversion saturates, and takes NaN to 0.
__device__ __forceinline__ int code_of(float v, float inv) {
    const float t = v * inv;
    const float h = t + __builtin_copysignf(0x1.fffffep-2f, t);
    int q;
    asm("v_cvt_i32_f32 %0, %1" : "=v"(q) : "v"(h));
    return min(max(q, -127), 127);
}

// |v| into a running maximum that a NaN never enters.
__device__ __forceinline__ float fold_abs(float m, float v) {
    const float a = fabsf(v);
    return a > m ? a : m;
}

// WAVES waves a row (one: a row each).  V elements a load: 16 bytes where the rows are aligned, else one.  Of a row, kHeld loads a
// lane stay in registers between the maximum and the codes, so it is read once; what is longer is read again.
// Bound by the bytes: 8,191 x 4,096 in bf16, 100 MB, 19 to 22 us (4.6 to 5.3 TB/s, as a large copy); one row of 768 is the launch, 2 us.
template <typename T, int V, int WAVES>
__global__ __launch_bounds__(kBlock) void k_quantize_rows(redukt_quantize_rows a) {
    constexpr int kHeld = 4, kLanes = WAVES * kWave, kSpan = kLanes * V;
    __shared__ float wm[kWaves];
    const int lane = threadIdx.x % kLanes;
    const uint32_t group = blockIdx.y * gridDim.x + blockIdx.x, r = WAVES == 1 ? group * kWaves + threadIdx.x / kWave : group;
    if (r >= a.rows) return;                   // (whole waves, and none of a shared row)
    const T* const x = (const T*)a.x + (int64_t)r * a.x_stride;
    int8_t* const q = a.codes + (int64_t)r * a.codes_stride;
    typedef T vec __attribute__((ext_vector_type(V)));
    typedef int8_t codes __attribute__((ext_vector_type(V)));
    const uint32_t whole = a.cols / V * V, c0 = lane * V;
    vec held[kHeld];
    float m = 0.0f;
#pragma unroll
    for (int u = 0; u < kHeld; u++) {
        held[u] = vec{};
        if (c0 + u * kSpan < whole) held[u] = *(const vec*)(x + c0 + u * kSpan);
    }
#pragma unroll
    for (int u = 0; u < kHeld; u++)
#pragma unroll
        for (int e = 0; e < V; e++) m = fold_abs(m, (float)held[u][e]);
    for (uint32_t c = c0 + kHeld * kSpan; c < whole; c += kSpan) {
        const vec v = *(const vec*)(x + c);
#pragma unroll
        for (int e = 0; e < V; e++) m = fold_abs(m, (float)v[e]);
    }
    if (V > 1 && whole + lane < a.cols) m = fold_abs(m, (float)x[whole + lane]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fold_abs(m, __shfl_xor(m, o, kWave));
    if constexpr (WAVES > 1) {
        if (threadIdx.x % kWave == 0) wm[threadIdx.x / kWave] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; w++) m = fold_abs(m, wm[w]);
    }
    float scale = m / 127.0f;
    if (scale == 0.0f) scale = 1.0f;           // (also where the quotient rounds to 0: its inverse would make 127 of every value)
    const float inv = 1.0f / scale;
    const auto store = [&](uint32_t c, const vec& v) {
        codes y;
#pragma unroll
        for (int e = 0; e < V; e++) y[e] = (int8_t)code_of((float)v[e], inv);
        *(codes*)(q + c) = y;
    };
#pragma unroll
    for (int u = 0; u < kHeld; u++)
        if (c0 + u * kSpan < whole) store(c0 + u * kSpan, held[u]);
    for (uint32_t c = c0 + kHeld * kSpan; c < whole; c += kSpan) store(c, *(const vec*)(x + c));
    if (V > 1 && whole + lane < a.cols) q[whole + lane] = (int8_t)code_of((float)x[whole + lane], inv);
    if (lane == 0) a.scales[r] = scale;
}

// ---------------------------------------------------------------- product
//
// out[i][j] = (sum_c x[i][c] w[j][c]) (x_scales[i] w_scales[j]) + bias[j].  Sums of codes are exact, so the order of the
// columns is free and every kernel gives the same bits.  The channels are the matrix instructions' left operand, so a lane
// holds neighbouring channels of one token.

// v_mfma_i32_16x16x64_i8: lane l holds 16 consecutive codes of row l % 16, the columns 16 (l / 16)
// + [0, 16); of the result, column l % 16 of rows 4 (l / 16) + [0, 4).
__device__ __forceinline__ i32x4 mma8(const i32x4& a, const i32x4& b, const i32x4& c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float scaled(const redukt_int8_matmul& a, int sum, uint32_t i, uint32_t j) {
    const float y = (float)sum * (a.x_scales[i] * a.w_scales[j]);
    return a.bias ? y + a.bias[j] : y;
}

// Codes of any alignment: 64 x 64 outputs a workgroup, 64 columns at a time staged byte by byte
// with zeros outside the operands.  For odd sizes and strides, not for speed: 16-byte accesses need rows that begin on 16 bytes
// (100 tokens of 4,096 x 1,530: 92 us; of 4,096 x 1,536, by the kernels below, 5).
constexpr int kTile = 64, kPitch = kTile + 16;
template <typename T>
__global__ __launch_bounds__(kBlock) void k_int8_bytes(redukt_int8_matmul a) {
    __shared__ __attribute__((aligned(16))) int8_t sx[kTile * kPitch], sw[kTile * kPitch];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t tiles = (a.n + kTile - 1) / kTile, i0 = blockIdx.x / tiles * kTile, j0 = blockIdx.x % tiles * kTile;
    i32x4 acc[4] = {};
    for (uint32_t c0 = 0; c0 < a.k; c0 += kTile) {
        for (int e = threadIdx.x; e < kTile * kTile; e += kBlock) {
            const uint32_t r = e / kTile, c = c0 + e % kTile;
            sx[r * kPitch + e % kTile] = i0 + r < a.m && c < a.k ? a.x[(int64_t)(i0 + r) * a.x_stride + c] : 0;
            sw[r * kPitch + e % kTile] = j0 + r < a.n && c < a.k ? a.w[(int64_t)(j0 + r) * a.w_stride + c] : 0;
        }
        __syncthreads();
        const i32x4 fw = *(const i32x4*)(sw + (16 * wave + lane % 16) * kPitch + 16 * (lane / 16));
#pragma unroll
        for (int t = 0; t < 4; t++)
            acc[t] = mma8(fw, *(const i32x4*)(sx + (16 * t + lane % 16) * kPitch + 16 * (lane / 16)), acc[t]);
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const uint32_t i = i0 + 16 * t + lane % 16;
        if (i >= a.m) continue;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t j = j0 + 16 * wave + 4 * (lane / 16) + e;
            if (j < a.n) ((T*)a.out)[(int64_t)i * a.out_stride + j] = (T)scaled(a, acc[t][e], i, j);
        }
    }
}

// Few tokens (up to 16, of many channels up to 3: redukt_op_int8_matmul): the weights are read once, straight into registers, and
// nothing else costs much (one token of 50,280 x 768: 38.6 MB in 10.3 us, 3.7 TB/s with the launch; of 8,192 x 8,192 67 MB in 12.7,
// 5.3).  Workgroups begin at different columns: rows of a power of two put the same columns into the same channel of a cache, where all
// would wait at once (8,192 x 8,192: 17.6 -> 13.8 us).  Of a workgroup's eight waves `split` share 16 channels, each taking every
// split-th line of 128 columns; their sums meet in LDS.
struct Int8Few {
    redukt_int8_matmul a;
    uint32_t split;
};

template <typename T>
__global__ __launch_bounds__(512) void k_int8_few(Int8Few f) {
    __shared__ i32x4 part[8][kWave];
    const redukt_int8_matmul& a = f.a;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l16 = lane % 16, g4 = lane / 16;
    const uint32_t split = f.split, j0 = (blockIdx.x * (8 / split) + wave / split) * 16;
    const uint32_t lines = (a.k + 127) / 128;
    const int8_t* const w = a.w + (int64_t)min(j0 + l16, a.n - 1) * a.w_stride;
    const int8_t* const x = a.x + (int64_t)min((uint32_t)l16, a.m - 1) * a.x_stride;
    i32x4 acc = {};
    if (j0 < a.n) {
        const uint32_t rot = blockIdx.x * 4 % lines;
        for (uint32_t turn = wave % split; turn < lines; turn += split) {
            const uint32_t c = turn + rot - (turn + rot >= lines ? lines : 0);
            // (columns past k: the last ones again, against zeros)
            uint32_t at[2];
            i32x4 fw[2], fx[2];
#pragma unroll
            for (int s = 0; s < 2; s++) {
                at[s] = 128 * c + 64 * s + 16 * g4;
                fw[s] = *(const i32x4*)(w + min(at[s], a.k - 16));
                fx[s] = *(const i32x4*)(x + min(at[s], a.k - 16));
            }
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const i32x4 z = {};
                acc = mma8(at[s] < a.k ? fw[s] : z, fx[s], acc);
            }
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave % split) return;
    for (uint32_t s = 1; s < split; s++) acc += part[wave + s][lane];
    if ((uint32_t)l16 >= a.m) return;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t j = j0 + 4 * g4 + e;
        if (j < a.n) ((T*)a.out)[(int64_t)l16 * a.out_stride + j] = (T)scaled(a, acc[e], l16, j);
    }
}

// Many tokens: tiles of TN channels by TM tokens, KC columns at a time from memory straight into one of STAGES LDS buffers while
// the matrix cores work on another.  A wave takes (TN / WN) x (TM / WM) outputs in 32 x 32 tiles.
//
// A row of KC codes is KC / 16 pieces of 16 bytes; piece c of row r stands at place c ^ (r / 2 % 8) (KC 128) or c ^ (r % 16)
// (KC 256), so that the 16 rows that 16 lanes read a piece of meet no bank twice.  The loads write LDS in lane order, so the
// lane picks the piece that belongs to its place.
//
// Tiles of 256 x 256 are bound by the matrix cores and the LDS reads beside them: 8,192 of 8,192 x 4,096 in 249 us, 2.2 POP/s (the
// library's int8 product 250).  The smaller ones by the columns on their way: 64 of 8,192 x 8,192 in 14.0, 67 MB at 4.8 TB/s; 100 of
// 4,096 x 1,536 in 5.1, the launch and twelve steps.
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) unsigned char lds_u8;
typedef __attribute__((address_space(3))) void lds_void;

__device__ __forceinline__ i32x16 mma32(const i32x4& a, const i32x4& b, const i32x16& c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

template <int KC>
__device__ __forceinline__ int place_of(int row, int c) {
    return KC == 128 ? c ^ (row / 2 % 8) : c ^ (row % 16);
}

// ROWS rows of a tile into `to`, 1 KB a wave and request; `at` is the lane's place in the operand, stride the bytes of a row.
template <int KC, int ROWS, int WAVES>
__device__ __forceinline__ void stage_rows(__amdgpu_buffer_rsrc_t from, lds_u8* __restrict__ to, uint32_t at, uint32_t stride, int wave) {
#pragma unroll
    for (int u = 0; u < ROWS * KC / 1024 / WAVES; u++)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void*)(to + (u * WAVES + wave) * 1024), 16,
                                                 (int)(at + u * (WAVES * 1024 / KC) * stride), 0, 0, 0);
}

template <int KC>
__device__ __forceinline__ i32x4 piece(const lds_u8* rows, int row, int c) {
    return *(const __attribute__((address_space(3))) i32x4*)(rows + row * KC + place_of<KC>(row, c) * 16);
}

template <int KC, int NI, int NJ>
__device__ __forceinline__ void multiply(const lds_u8* __restrict__ w, const lds_u8* __restrict__ x, i32x16 (&acc)[NI][NJ], int rw, int rx, int lane) {
    // (the next fragments are asked for before the products of these; 128 of 768 x 4,096: 10.8 -> 9.7 us)
    i32x4 fw[2][NI], fx[2][NJ];
    const auto load = [&](int s) {
#pragma unroll
        for (int i = 0; i < NI; i++) fw[s % 2][i] = piece<KC>(w, rw + 32 * i + lane % 32, 2 * s + lane / 32);
#pragma unroll
        for (int j = 0; j < NJ; j++) fx[s % 2][j] = piece<KC>(x, rx + 32 * j + lane % 32, 2 * s + lane / 32);
    };
    load(0);
#pragma unroll
    for (int s = 0; s < KC / 32; s++) {
        if (s + 1 < KC / 32) load(s + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[i][j] = mma32(fw[s % 2][i], fx[s % 2][j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

struct Int8Tiles {
    redukt_int8_matmul a;
    uint32_t tiles_m, tiles_n;
    uint32_t wide;             // rows of out take 16-byte stores
};

// All but this wave's last N loads into LDS are done, and what it read from LDS is there; then the workgroup meets.  (__syncthreads
// would wait for every load.)
template <int N>
__device__ __forceinline__ void wait_and_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0070);        // vmcnt(N) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename T, int TM, int TN, int WM, int WN, int KC, int STAGES>
__global__ __launch_bounds__(64 * WM * WN) void k_int8_tiles(Int8Tiles f) {
    constexpr int W = WM * WN, NI = TN / WN / 32, NJ = TM / WM / 32, kStage = (TM + TN) * KC;
    constexpr int kPending = (STAGES - 2) * kStage / 1024 / W;     // requests of the stages behind the next one
    static_assert(kPending < 64 && TM * KC / 1024 % W == 0 && TN * KC / 1024 % W == 0, "");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[STAGES][kStage];
    const redukt_int8_matmul& a = f.a;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    // Workgroups go round the eight XCDs in turn: an XCD takes neighbouring tiles, eight of the tokens' by four of the
    // channels' at a time, whose rows its L2 then holds once.
    const uint32_t total = f.tiles_m * f.tiles_n, per = (total + 7) / 8, t = blockIdx.x % 8 * per + blockIdx.x / 8;
    if (blockIdx.x / 8 >= per || t >= total) return;
    const uint32_t band = 8 * f.tiles_n, m0 = t / band * 8, high = min(f.tiles_m - m0, 8u);
    const uint32_t i0 = (m0 + t % band % high) * TM, j0 = t % band / high * TN;

    const uint32_t xs = (uint32_t)a.x_stride, ws = (uint32_t)a.w_stride;
    const auto rx = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x + (size_t)i0 * xs), (short)0,
                                                      (int)((min(a.m - i0, (uint32_t)TM) - 1) * xs + a.k), 0x00020000);
    const auto rw = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + (size_t)j0 * ws), (short)0,
                                                      (int)((min(a.n - j0, (uint32_t)TN) - 1) * ws + a.k), 0x00020000);
    constexpr int kPieces = KC / 16, kRows = 64 / kPieces;         // rows of one request
    const int row = wave * kRows + lane / kPieces;
    const uint32_t col = place_of<KC>(row, lane % kPieces) * 16;
    static_assert(W * kRows % 16 == 0, "a lane's rows have one order of pieces");
    // (rows past the tile and columns past k are out of the buffers' bounds and come as zeros)
    const auto stage = [&](lds_u8* __restrict__ to, uint32_t c) {
        const bool in = c + col < a.k;
        stage_rows<KC, TN, W>(rw, to, in ? row * ws + col + c : 0x80000000u, ws, wave);
        stage_rows<KC, TM, W>(rx, to + TN * KC, in ? row * xs + col + c : 0x80000000u, xs, wave);
    };
    const int rj = wave / WN * (TM / WM), ri = wave % WN * (TN / WN);
    i32x16 acc[NI][NJ] = {};
    // A step's columns are waited for (with those behind them still under way); then every wave is done with the buffer of the
    // columns before them, which takes the ones STAGES - 1 further on (past k: zeros, without a request to memory).
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) stage((lds_u8*)lds[s], s * KC);
    for (uint32_t c = 0; c < a.k; c += STAGES * KC) {
#pragma unroll
        for (int s = 0; s < STAGES; s++) {
            if (c + s * KC >= a.k) break;
            wait_and_meet<kPending>();
            stage((lds_u8*)lds[(s + STAGES - 1) % STAGES], c + (s + STAGES - 1) * KC);
            multiply<KC, NI, NJ>((const lds_u8*)lds[s], (const lds_u8*)lds[s] + TN * KC, acc, ri, rj, lane);
        }
    }
    wait_and_meet<0>();                        // (zeros may still be on their way)

    // 32 tokens of a wave's channels at a time through LDS, so that a row of them is stored as whole lines.
    constexpr int CH = TN / WN, kRow = CH * sizeof(T), kOuts = kRow / 16, kPer = 16 / sizeof(T);
    static_assert(32 * kRow * W <= STAGES * kStage, "");
    unsigned char* const mine = &lds[0][0] + wave * 32 * kRow;
    typedef T out4 __attribute__((ext_vector_type(4)));
    typedef T out16 __attribute__((ext_vector_type(kPer)));
    float sw[NI][4][4], bias[NI][4][4];
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t j = min(j0 + ri + 32 * i + 8 * g + 4 * (lane / 32) + e, a.n - 1);
                sw[i][g][e] = a.w_scales[j];
                bias[i][g][e] = a.bias ? a.bias[j] : 0.0f;
            }
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const uint32_t i_row = i0 + rj + 32 * j;
        const float sx = a.x_scales[min(i_row + lane % 32, a.m - 1)];
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                out4 v;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y = (float)acc[i][j][4 * g + e] * (sx * sw[i][g][e]);
                    v[e] = (T)(a.bias ? y + bias[i][g][e] : y);
                }
                const int at = (32 * i + 8 * g + 4 * (lane / 32)) * (int)sizeof(T), r = lane % 32;
                *(out4*)(mine + r * kRow + ((at / 16 ^ r % kOuts) * 16) + at % 16) = v;
            }
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
        for (int u = 0; u < 32 * kOuts / kWave; u++) {
            const int id = u * kWave + lane, r = id / kOuts, p = id % kOuts;
            const out16 v = *(const out16*)(mine + r * kRow + ((p ^ r % kOuts) * 16));
            const uint32_t i = i_row + r, c = j0 + ri + p * kPer;
            if (i >= a.m || c >= a.n) continue;
            T* const o = (T*)a.out + (int64_t)i * a.out_stride + c;
            if (f.wide && c + kPer <= a.n) {
                *(out16*)o = v;
            } else {
#pragma unroll
                for (int e = 0; e < kPer; e++)
                    if (c + e < a.n) o[e] = v[e];
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

#define OP_BY_TYPE(dtype, fn, ...) \
    ((dtype) == REDUKT_OP_BF16 ? (const void*)fn<__bf16 __VA_OPT__(, ) __VA_ARGS__> \
     : (dtype) == REDUKT_OP_F16 ? (const void*)fn<_Float16 __VA_OPT__(, ) __VA_ARGS__> \
                                : (const void*)fn<float __VA_OPT__(, ) __VA_ARGS__>)

template <int WAVES>
const void* quantize_wide_fn(uint32_t dtype) {
    return dtype == REDUKT_OP_BF16  ? (const void*)k_quantize_rows<__bf16, 8, WAVES>
           : dtype == REDUKT_OP_F16 ? (const void*)k_quantize_rows<_Float16, 8, WAVES>
                                    : (const void*)k_quantize_rows<float, 4, WAVES>;
}

constexpr int64_t kMaxStride = 1 << 22;      // 256 rows stay within 32-bit offsets
constexpr uint32_t kGridX = 1 << 20;         // workgroups along x; more of them go along y

int32_t few(const redukt_int8_matmul& a, void* stream) {
    const uint32_t groups = (a.n + 15) / 16, lines = (a.k + 127) / 128;
    uint32_t split = 1;
    while (split < 8 && split * 2 <= lines && groups * split < 2048) split *= 2;
    Int8Few k{a, split};
    const uint32_t per = 8 / split, grid = (groups + per - 1) / per;
    if (!op_grid_ok(grid, 512)) return BACKEND_INVALID_ARGUMENT;
    return op_launch(OP_BY_TYPE(a.dtype, k_int8_few), dim3(grid), dim3(512), 0, stream, k);
}

template <int TM, int TN, int WM, int WN, int KC, int STAGES>
int32_t tiles(const redukt_int8_matmul& a, void* stream) {
    const bool wide = op_aligned(a.out, 16) && a.out_stride * op_elem_bytes(a.dtype) % 16 == 0;
    Int8Tiles k{a, (a.m + TM - 1) / TM, (a.n + TN - 1) / TN, wide};
    const uint64_t total = (uint64_t)k.tiles_m * k.tiles_n, grid = (total + 7) / 8 * 8;
    if (!op_grid_ok(grid, 64 * WM * WN)) return BACKEND_INVALID_ARGUMENT;
    return op_launch(OP_BY_TYPE(a.dtype, k_int8_tiles, TM, TN, WM, WN, KC, STAGES), dim3((uint32_t)grid), dim3(64 * WM * WN), 0, stream, k);
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
    const int size = (int)op_elem_bytes(a->dtype), v = 16 / size;
    const bool wide = op_aligned(a->x, 16) && op_aligned(a->codes, v) && (a->rows == 1 || (a->x_stride * size % 16 == 0 && a->codes_stride % v == 0));
    // A row that four loads a lane of one wave cover is that wave's; longer ones take four waves.
    const bool one = a->cols <= 4u * kWave * (wide ? v : 1);
    const void* fn = !wide ? (one ? OP_BY_TYPE(a->dtype, k_quantize_rows, 1, 1) : OP_BY_TYPE(a->dtype, k_quantize_rows, 1, 4))
                     : one ? quantize_wide_fn<1>(a->dtype) : quantize_wide_fn<4>(a->dtype);
    const uint32_t groups = one ? (a->rows + kWaves - 1) / kWaves : a->rows, x = groups < kGridX ? groups : kGridX;
    return op_launch(fn, dim3(x, (groups + x - 1) / x), dim3(kBlock), 0, stream, k);
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
    const bool aligned = op_aligned(a->x, 16) && op_aligned(a->w, 16) && a->x_stride % 16 == 0 && a->w_stride % 16 == 0 &&
                         a->k % 16 == 0 && a->k > 0 && a->x_stride <= kMaxStride && a->w_stride <= kMaxStride;
    if (!aligned) {
        redukt_int8_matmul k = *a;
        const uint64_t grid = (uint64_t)((a->n + kTile - 1) / kTile) * ((a->m + kTile - 1) / kTile);
        if (!op_grid_ok(grid, kBlock)) return BACKEND_INVALID_ARGUMENT;
        return op_launch(OP_BY_TYPE(a->dtype, k_int8_bytes), dim3((uint32_t)grid), dim3(kBlock), 0, stream, k);
    }
    // Every kernel gives the same bits, so the choice is by time alone (us, on either side of each edge; n and k after m).  Up to
    // 16 tokens: weights straight into registers (16 of 4,096 x 4,096: 8.3, tiles 9.5; 8 of 768 x 4,096: 6.9 and 9.0), up to 3 where the
    // channels alone give every CU a tile (2 of 8,192 x 8,192: 14.1, tiles 14.7; 8: 16.0 and 14.5; 8 of 50,280 x 768: 13.4 and 11.9).
    if (a->m <= (a->n >= 8192 ? 3 : 16)) return few(*a, stream);
    // Tiles of 256 once they fill the CUs (8,192 of 8,192 x 4,096: 249, tiles of 128: 291; 2,048 of 4,096 x 1,536, 128 tiles: 27.8 and
    // 20.9), of 128 once they nearly do (4,096 of 768 x 768, 192 tiles: 10.3, tiles of 64: 10.8; 1,000 of 1,536 x 768, 96 tiles:
    // 9.4 and 7.0), else of 64, by 32 channels where half of the CUs would have none (64 of 8,192 x 8,192: 13.2, by 64
    // 14.8; 128 of 4,096 x 4,096 8.0 and 8.1; 100 of 4,096 x 1,536 5.0 both).  Where no CU has
    // two workgroups, each keeps more columns on their way (1,024 of 4,096 x 4,096, 256 tiles of 128: 28.2 with two stages, 25.3 with three;
    // 2,048 of 4,096 x 1,536, 512 tiles: 21.4 and 25.3; 128 of 8,192 x 8,192, 256 of 64: 26.3 with two of 256 columns, 17.6 with four
    // of 128; 512 of 4,096 x 4,096, 512 of 64: 16.4 and 17.8).
    const auto count = [&](uint32_t t) { return (uint64_t)((a->m + t - 1) / t) * ((a->n + t - 1) / t); };
    if (count(256) >= 256) return tiles<256, 256, 2, 4, 128, 2>(*a, stream);
    if (count(128) > 256) return tiles<128, 128, 2, 2, 128, 2>(*a, stream);
    if (count(128) >= 192) return tiles<128, 128, 2, 2, 128, 3>(*a, stream);
    if (count(64) <= 128) return tiles<64, 32, 2, 1, 128, 6>(*a, stream);
    if (count(64) <= 256) return tiles<64, 64, 2, 2, 128, 4>(*a, stream);
    return tiles<64, 64, 2, 2, 256, 2>(*a, stream);
}

}  // extern "C"
