// delta_ops.hip — the gated delta rule on caller tensors (redukt_ops.h).
//
// A value head's state S [dk][dv] takes a token (k, q, v, g, beta) as
//     S <- a S + k d^T,   d = beta (v - a S^T k),   o = scale S^T q,   a = e^g.
// Columns of S do not meet, so any split over dv is free; S^T k and S^T q sum over dk.
#include <hip/hip_runtime.h>

#include "mfma_common.h"
#include "op_common.h"

// (mfma_common.h turns contraction off for the step kernels' bit-exact arithmetic)
#pragma clang fp contract(fast)

namespace rdk {
namespace {

constexpr float kUnitEps = 1e-6f;      // added to the sum of squares that k and q are divided by

// What normalizes a row of this sum of squares; NaN where the sum is not finite (1 / sqrt(inf) = 0 would make zeros of a finite row).
__device__ __forceinline__ float unit_factor(float sum) { return rsqrtf(sum + kUnitEps) + 0.0f * sum; }

struct DeltaArgs {
    redukt_delta_rows r;
    const float* in;           // states read (null: zeros)
    float* states;             // states written (null: none)
    uint32_t n_slots;
    const int32_t* slots;
    const int32_t* cu;         // null: one row an entry
    uint32_t n;                // entries
};

// v summed over the lanes that differ in bits 3, 4 and 5, the same bits in every one of them.
__device__ __forceinline__ float rows_sum(float v) {
    v += __shfl_xor(v, 8, kWave);
    v += __shfl_xor(v, 16, kWave);
    v += __shfl_xor(v, 32, kWave);
    return v;
}

// One wave keeps 32 columns of one head's state in registers: lane 8 rg + c the rows rg DK/8
// + [0, DK/8) of columns 4 c + [0, 4), so each load of the wave takes whole 128-byte lines.
// Both sums over dk are formed from the state as it is read (S'^T q = a S^T q + (k.q) d), in one
// exchange between the eight row groups, so the state is read and written once.
// Bound by those bytes: 500 entries of 32 heads of 128 x 128, 2.1 GB, take 395 us (5.4 TB/s; a large copy moves 5.2, and some of
// a pool stays in cache); 100 of 16 heads 34 us (6.3, mostly from cache).  One entry of a small model is the launch, 4 us.
template <typename T, int DK>
__global__ __launch_bounds__(256) void k_delta_step(DeltaArgs a) {
    constexpr int R = DK / 8;
    const redukt_delta_rows& r = a.r;
    const int lane = threadIdx.x % kWave, rg = lane / 8, c4 = (lane % 8) * 4;
    const uint32_t blocks = r.dv / 32;
    const uint64_t id = (uint64_t)blockIdx.x * (blockDim.x / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t i = (uint32_t)(id / (r.hv * blocks));
    if (i >= a.n) return;
    const uint32_t hb = (uint32_t)(id % (r.hv * blocks)), h = hb / blocks, col = hb % blocks * 32 + c4;
    const uint32_t hq = h / (r.hv / r.hk);
    const int slot = entry_slot(a.slots, a.n_slots, i, true, lane);
    if (slot == kSkip) return;
    T* const out = (T*)r.out + (int64_t)i * r.out_stride + (size_t)h * r.dv + col;
    if (slot == kBad) {
        for (int j = 0; j < 4; j++) out[j] = (T)__builtin_nanf("");
        return;
    }
    float* const state = a.states + (((size_t)slot * r.hv + h) * DK + rg * R) * r.dv + col;
    float4 S[R];
#pragma unroll
    for (int e = 0; e < R; e++) S[e] = *(const float4*)(state + (size_t)e * r.dv);
    float k[R], q[R], v[4];
    op_load((const T*)r.k + (int64_t)i * r.k_stride + hq * DK + rg * R, k);
    op_load((const T*)r.q + (int64_t)i * r.q_stride + hq * DK + rg * R, q);
    op_load((const T*)r.v + (int64_t)i * r.v_stride + h * r.dv + col, v);
    const float decay = expf(r.g[(int64_t)i * r.g_stride + h]), beta = r.beta[(int64_t)i * r.beta_stride + h];
    float4 sk = make_float4(0, 0, 0, 0), sq = make_float4(0, 0, 0, 0);
    float kk = 0, qq = 0, kq = 0;
#pragma unroll
    for (int e = 0; e < R; e++) {
        sk.x += k[e] * S[e].x, sk.y += k[e] * S[e].y, sk.z += k[e] * S[e].z, sk.w += k[e] * S[e].w;
        sq.x += q[e] * S[e].x, sq.y += q[e] * S[e].y, sq.z += q[e] * S[e].z, sq.w += q[e] * S[e].w;
        kk += k[e] * k[e], qq += q[e] * q[e], kq += k[e] * q[e];
    }
    sk.x = rows_sum(sk.x), sk.y = rows_sum(sk.y), sk.z = rows_sum(sk.z), sk.w = rows_sum(sk.w);
    sq.x = rows_sum(sq.x), sq.y = rows_sum(sq.y), sq.z = rows_sum(sq.z), sq.w = rows_sum(sq.w);
    kq = rows_sum(kq);
    float uk = 1.0f, uq = r.scale;
    if (r.flags & REDUKT_DELTA_NORMALIZE) {
        uk = unit_factor(rows_sum(kk));
        uq *= unit_factor(rows_sum(qq));
    }
    // d carries the key's factor, so that the rows of k enter as they are
    const float ak = decay * uk;
    const float4 d = make_float4(beta * (v[0] - ak * sk.x) * uk, beta * (v[1] - ak * sk.y) * uk, beta * (v[2] - ak * sk.z) * uk,
                                 beta * (v[3] - ak * sk.w) * uk);
#pragma unroll
    for (int e = 0; e < R; e++) {
        S[e].x = decay * S[e].x + k[e] * d.x;
        S[e].y = decay * S[e].y + k[e] * d.y;
        S[e].z = decay * S[e].z + k[e] * d.z;
        S[e].w = decay * S[e].w + k[e] * d.w;
        *(float4*)(state + (size_t)e * r.dv) = S[e];
    }
    if (rg == 0) {
        typedef T out4 __attribute__((ext_vector_type(4)));
        *(out4*)out = out4{(T)(uq * (decay * sq.x + kq * d.x)), (T)(uq * (decay * sq.y + kq * d.y)),
                           (T)(uq * (decay * sq.z + kq * d.z)), (T)(uq * (decay * sq.w + kq * d.w))};
    }
}

const void* delta_step_fn(uint32_t dtype, uint32_t dk) {
    static const void* const fns[3][2] = {
        {(const void*)k_delta_step<__bf16, 64>, (const void*)k_delta_step<__bf16, 128>},
        {(const void*)k_delta_step<_Float16, 64>, (const void*)k_delta_step<_Float16, 128>},
        {(const void*)k_delta_step<float, 64>, (const void*)k_delta_step<float, 128>},
    };
    return fns[dtype][dk == 128];
}

// ---------------------------------------------------------------- sequences in chunks
//
// C = 64 tokens at a time, with G the running sum of g within the chunk, c = C - 1 its last
// token, u_i and p_i the factors that normalize k_i and q_i (the scale in p_i):
//     A_ij = beta_i u_i u_j e^(G_i - G_j) k_i.k_j (j < i),      T = (I + A)^-1 diag(beta)
//     P_ij = p_i u_j e^(G_i - G_j) q_i.k_j (j <= i)
//     X = V - diag(u_i e^G_i) K S
//     O = diag(p_i e^G_i) Q S + (P T) X
//     S <- e^G_c S + K^T (diag(u_i e^(G_c - G_i)) T) X
// P T, diag() T and the diagonals need no state: k_delta_prep makes them for all chunks side by
// side.  k_delta_chunks goes through a sequence's chunks in order with the state in registers, 16
// columns a wave.
//
// Arithmetic.  The products run on the bf16 matrix cores.  Keys and queries in bf16 are their
// own operand (f16: two limbs, f32: three, exact); S, X and diag() T are f32 split into three
// limbs of 8 bits, and products of limbs are kept down to 2^-24 of the whole, so the state is as
// exact as f32 sums are (two limbs leave about 4e-6).  P T, and S and X where only a 16-bit output
// comes of them, are two limbs (2^-17 against an output's half step of 2^-8 or 2^-11).  A third one of
// P T and X there takes the outputs' error before their rounding from 3.7e-6 to 0.7e-6, and both forms are
// off by 1.7e-3 behind it in bf16; but 6 KB more a chunk go through L1: 8,192 tokens 259 -> 293 us, 37 ragged
// prompts 183 -> 191.  G is summed in 64 bits: the decays are e to small differences of sums that may be large.
//
// What is not finite.  A matrix product would spread one over rows it does not reach by the rule
// (0 times it), so rows of X from a column's first such value on are taken as zeros, and the column's
// outputs from there on and its state become NaN; k_delta_prep marks the tokens from the first whose
// key, g or beta is not finite (g = -inf is).
//
// Layout.  The 16 x 16 result tile of an MFMA has column l % 16, rows 4 (l / 16) + r in lane l;
// its right operand wants column l % 16 and eight consecutive inner indices 8 (l / 16) + j.
// Rows of a pair of result tiles (2 s, 2 s + 1) stand for the indices
//     32 s + 8 (row / 4) + 4 (tile % 2) + row % 4,                                      (*)
// so a lane's eight results of the pair are eight consecutive inner indices of the next product:
// S, X and D go from result to right operand without an exchange between lanes.  Left operands
// take their rows in the same order.  (At dk 64 a wave has one tile of S, 16 indices in their own
// order, and multiplies it 16 inner indices at a time.)

constexpr int kChunk = 64;
constexpr int kTri = 6;                    // 16 x 32 fragments of a lower triangle of 64
constexpr int kFrag = 1024;                // bytes of one fragment's limb: 64 lanes of 8 bf16

template <typename T> struct Limbs;
template <> struct Limbs<__bf16> { static constexpr int in = 1, out = 2; };
template <> struct Limbs<_Float16> { static constexpr int in = 2, out = 2; };
template <> struct Limbs<float> { static constexpr int in = 3, out = 3; };

// What k_delta_prep leaves of a chunk and value head: the fragments of diag() T in three limbs, of P T in LO, and
// f32 vectors [64]: u_i e^G_i, p_i e^G_i, and e^G_c in every place.
constexpr int kVecs = 3;
constexpr int unit_bytes(int out_limbs) { return kTri * (3 + out_limbs) * kFrag + kVecs * kChunk * 4; }

// The index that row `row` of result tile `tile` stands for (*).
__device__ __forceinline__ int tile_index(int tile, int row) {
    return 32 * (tile / 2) + 8 * (row / 4) + 4 * (tile % 2) + row % 4;
}

template <int N>
struct Split {
    bf16x8 l[N];
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// a and b rounded to bf16, in the low and the high half of a word.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// v, or bf16's largest finite value with its sign where v is beyond that: what the first limb of v is rounded from.  (f32's values from
// 3.3962e38 on would round to infinity, and their rests with them; so the rest is what is beyond, and still exact in two limbs.  Of an
// infinity the rest is one, of a NaN a NaN.)  For values that may be so large.
__device__ __forceinline__ float within_bf16(float v) { return __builtin_amdgcn_fmed3f(v, -0x1.fep127f, 0x1.fep127f); }

// Eight f32 as N bf16 limbs: each the rounded rest of those before it (the differences are exact).
template <int N, bool WIDE = false>
__device__ __forceinline__ Split<N> split8(const float (&v)[8]) {
    u32x4 w[N];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float a = v[2 * j], b = v[2 * j + 1];
#pragma unroll
        for (int n = 0; n < N; n++) {
            const uint32_t p = WIDE && n == 0 ? pack_bf16(within_bf16(a), within_bf16(b)) : pack_bf16(a, b);
            w[n][j] = p;
            if (n + 1 < N) {
                a -= __builtin_bit_cast(float, p << 16);
                b -= __builtin_bit_cast(float, p & 0xffff0000u);
            }
        }
    }
    Split<N> o;
#pragma unroll
    for (int n = 0; n < N; n++) o.l[n] = __builtin_bit_cast(bf16x8, w[n]);
    return o;
}

// Eight elements of an operand in memory as limbs (exactly).
template <typename T>
__device__ __forceinline__ Split<Limbs<T>::in> load_limbs(const T* p) {
    if constexpr (sizeof(T) == 2 && Limbs<T>::in == 1) {
        return {{*(const bf16x8*)p}};
    } else {
        float v[8];
        op_load(p, v);
        return split8<Limbs<T>::in>(v);
    }
}

// c += a b, with the products of limbs i and j kept for i + j < K.
template <int K, int NA, int NB>
__device__ __forceinline__ f32x4 mma_limbs(const Split<NA>& a, const Split<NB>& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < NA; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
            if (i + j < K) c = mma(a.l[i], b.l[j], c);
    return c;
}

template <int N>
__device__ __forceinline__ Split<N> as_split(const bf16x8 (&v)[N]) {
    Split<N> o;
#pragma unroll
    for (int n = 0; n < N; n++) o.l[n] = v[n];
    return o;
}

struct ChunkArgs {
    DeltaArgs d;
    unsigned char* ws;         // units: (value head, chunk slot)
    uint32_t slots;            // chunk slots
    uint32_t per;              // value heads of a workgroup of k_delta_prep
};

// Sequence i's rows, within [0, rows].
__device__ __forceinline__ uint32_t row_of(const ChunkArgs& a, uint32_t i) {
    return min((uint32_t)max(a.d.cu[i], 0), a.d.r.rows);
}

// The sequence that is the pos-th by length, longest first (n <= 64; every lane of the wave takes part).  Workgroups that wait for a
// CU start in this order, so that no long sequence begins last (37 of 3 to 932 tokens: 203 -> 194 us).  More than 64 sequences, which
// one wave does not hold, start in the order of their numbers.
__device__ __forceinline__ uint32_t by_length(const ChunkArgs& a, uint32_t pos, int lane) {
    const bool in = (uint32_t)lane < a.d.n;
    const uint32_t b = in ? row_of(a, lane) : 0, len = in ? max(row_of(a, lane + 1), b) - b : 0;
    uint32_t rank = 0;
    for (uint32_t j = 0; j < a.d.n; j++) {
        const uint32_t x = __builtin_amdgcn_readlane(len, j);
        rank += x > len || (x == len && (int)j < lane);
    }
    return __builtin_ctzll(__ballot(in && rank == pos));
}

// Chunk c of the sequence that starts at row b and is the i-th has slot b / 64 + i + c: slots of one sequence
// are consecutive, those of the next begin after them, and rows / 64 + n slots are enough.
__device__ __forceinline__ uint32_t first_chunk(uint32_t b, uint32_t i) { return b / kChunk + i; }

__device__ __forceinline__ f32x4 mma4(float a, float b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

constexpr int kPitchA = kChunk + 4;        // f32 rows of the 64 x 64 matrices in LDS

// A buffer descriptor: loads past `bytes` give zeros, stores there are dropped.
__device__ __forceinline__ auto rows_rsrc(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}

// One element as its bits, a register each (a conversion, or a packing, would wait for the load), and its value.
template <typename T, typename R>
__device__ __forceinline__ uint32_t buffer_bits(R rsrc, uint32_t at) {
    if constexpr (sizeof(T) == 4) return __builtin_amdgcn_raw_buffer_load_b32(rsrc, (int)at, 0, 0);
    else return __builtin_amdgcn_raw_buffer_load_b16(rsrc, (int)at, 0, 0);
}
template <typename T>
__device__ __forceinline__ float of_bits(uint32_t v) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, v);
    else return (float)__builtin_bit_cast(T, (unsigned short)v);
}

// The index of row `row` of tile `tile` of the state: (*) where a wave has a pair of tiles.
template <int DK>
__device__ __forceinline__ int state_index(int tile, int row) {
    return DK == 128 ? tile_index(tile, row) : 16 * tile + row;
}

// a[0] b0 + a[1] b1 with three limbs each, as four chains of sums.
__device__ __forceinline__ f32x4 mma_four(const bf16x8 (&a)[2][3], const Split<3>& b0, const Split<3>& b1) {
    f32x4 x = mma(a[0][0], b0.l[0], f32x4{}), z = mma(a[1][0], b1.l[0], f32x4{});
    f32x4 y = mma(a[0][1], b0.l[0], f32x4{}), w = mma(a[1][1], b1.l[0], f32x4{});
    x = mma(a[0][0], b0.l[1], x), z = mma(a[1][0], b1.l[1], z);
    y = mma(a[0][1], b0.l[1], y), w = mma(a[1][1], b1.l[1], w);
    x = mma(a[0][0], b0.l[2], x), z = mma(a[1][0], b1.l[2], z);
    y = mma(a[0][2], b0.l[0], y), w = mma(a[1][2], b1.l[0], w);
    return (x + z) + (y + w);
}

template <int V>
struct Int {
    static constexpr int value = V;
};

// 4 NW f32 of a lane (16 NW inner indices of a product) as N limbs.
template <int NW, int N>
struct Part {
    typedef __bf16 vec __attribute__((ext_vector_type(4 * NW)));
    vec l[N];
};

template <int NW, int N, bool WIDE>
__device__ __forceinline__ Part<NW, N> split_part(const float (&v)[4 * NW]) {
    typedef uint32_t words __attribute__((ext_vector_type(2 * NW)));
    words w[N];
#pragma unroll
    for (int j = 0; j < 2 * NW; j++) {
        float a = v[2 * j], b = v[2 * j + 1];
#pragma unroll
        for (int n = 0; n < N; n++) {
            const uint32_t p = WIDE && n == 0 ? pack_bf16(within_bf16(a), within_bf16(b)) : pack_bf16(a, b);
            w[n][j] = p;
            a -= __builtin_bit_cast(float, p << 16);
            b -= __builtin_bit_cast(float, p & 0xffff0000u);
        }
    }
    Part<NW, N> o;
#pragma unroll
    for (int n = 0; n < N; n++) o.l[n] = __builtin_bit_cast(typename Part<NW, N>::vec, w[n]);
    return o;
}

__device__ __forceinline__ f32x4 mma_part(const bf16x8& a, const bf16x8& b, const f32x4& c) { return mma(a, b, c); }
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mma_part(const bf16x4& a, const bf16x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, a), __builtin_bit_cast(i16x4, b), c, 0, 0, 0);
}

// Fragment x of the lower triangle at m (f32 [64][kPitchA], natural order), its rows times f, with N limbs to `to`: fragment
// x is tile 0, 1, 2, 2, 3, 3 and inner indices 32 s + [0, 32) with s = 0, 0, 0, 1, 0, 1.
template <int N>
__device__ __forceinline__ void store_fragment(const float* m, const float* f, unsigned char* to, int x, int lane) {
    const int tile = x < 2 ? x : 2 + (x - 2) / 2, s = x < 2 ? 0 : (x - 2) % 2, row = tile_index(tile, lane % 16);
    float v[8];
    op_load(m + row * kPitchA + 32 * s + 8 * (lane / 16), v);
    const float scale = f ? f[row] : 1.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] *= scale;
    const Split<N> y = split8<N, true>(v);
#pragma unroll
    for (int n = 0; n < N; n++) *(bf16x8*)(to + (x * N + n) * kFrag + lane * 16) = y.l[n];
}

// v moved between lanes by the DPP control CTRL, 0 where a lane has no source or its row is not in ROWS.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The sum of the lanes up to each one: within rows of 16, then the rows' last lanes into those behind them.
__device__ __forceinline__ double prefix_sum(double v) {
    v = dpp_add<0x111, 0xF>(v);                // row_shr 1, 2, 4, 8
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);                // row_bcast 15 into rows 1 and 3
    return dpp_add<0x143, 0xC>(v);             // row_bcast 31 into rows 2 and 3
}

// 2^x by the hardware (1 ulp; what is below 2^-126 becomes 0).
__device__ __forceinline__ float exp2_hw(double x) { return __builtin_amdgcn_exp2f((float)x); }

template <typename T, int DK>
struct PrepLds {
    static constexpr int PK = DK + 16 / sizeof(T);     // rows of odd multiples of 16 bytes: 16 neighbouring ones meet no bank twice
    static constexpr int kRows = 2 * kChunk * PK * sizeof(T), kMatrices = 2 * kChunk * kPitchA * 4;
    __attribute__((aligned(16))) unsigned char m[kRows > kMatrices ? kRows : kMatrices];      // k and q, then A and T
    double g[kChunk];
    float b[kChunk], u[kChunk], p[kChunk], w[kChunk];
};

// Four waves make the units of one chunk, `len` rows from t0 on, and of `per` value heads of one key head.  (I + A)^-1 is solved by
// blocks: 16 by substitution, all four of a chunk side by side in one wave, then 32 and 64 by products, which keeps it as exact as
// substitution (a product of powers of A would not be, where keys are alike and the powers are large).
// A barrier that prepare() passes for its first head.  They are counted as they are written, because waves that have no part in it
// (k_delta_chunks) meet its four waves at each of them: every wave must pass it exactly once, in no loop and under no condition.
#define PREP_MEET() (__syncthreads(), (void)__COUNTER__)
constexpr int kPrepFirst = __COUNTER__;
template <typename T, int DK>
__device__ __forceinline__ void prepare(const ChunkArgs& a, PrepLds<T, DK>& lds, uint32_t slot, uint32_t t0, uint32_t len, uint32_t h0,
                                        uint32_t per) {
    constexpr int LI = Limbs<T>::in, LO = Limbs<T>::out, KS = DK / 32, SZ = sizeof(T), PK = PrepLds<T, DK>::PK;
    constexpr int kLoads = kChunk * DK * SZ / 16 / 256;
    double* const sG = lds.g;
    float *const sB = lds.b, *const sU = lds.u, *const sP = lds.p, *const sW = lds.w;
    T* const sK = (T*)lds.m;
    T* const sQ = sK + kChunk * PK;
    float* const sA = (float*)lds.m;
    float* const sT = sA + kChunk * kPitchA;
    const redukt_delta_rows& r = a.d.r;
    const int lane = threadIdx.x % kWave, wave = wave_index(), g4 = lane / 16, l16 = lane % 16;
    const uint32_t hq = h0 / (r.hv / r.hk);

    float g0 = 0.0f, beta = 0.0f;              // of token `lane` and one value head, in wave 0
    const auto load_gates = [&](uint32_t h) {
        if (wave == 0 && (uint32_t)lane < len) {
            g0 = r.g[(int64_t)(t0 + lane) * r.g_stride + h];
            beta = r.beta[(int64_t)(t0 + lane) * r.beta_stride + h];
        }
    };
    const auto put_gates = [&]() {
        if (wave == 0) {
            // (a token whose g or beta is not finite is marked by a NaN beta; decays are kept as logarithms to base 2)
            const bool bad = !(g0 < __builtin_inff()) || !(fabsf(beta) < __builtin_inff());
            sG[lane] = prefix_sum(bad ? 0.0 : (double)fmaxf(g0, -1e5f) * 1.4426950408889634);
            sB[lane] = bad ? __builtin_nanf("") : beta;
        }
    };
    {   // rows past the chunk's end as zeros
        const uint32_t ks = (uint32_t)r.k_stride * SZ, qs = (uint32_t)r.q_stride * SZ;
        const auto rk = rows_rsrc((const unsigned char*)r.k + (size_t)t0 * ks + (size_t)hq * DK * SZ, (len - 1) * ks + DK * SZ);
        const auto rq = rows_rsrc((const unsigned char*)r.q + (size_t)t0 * qs + (size_t)hq * DK * SZ, (len - 1) * qs + DK * SZ);
        load_gates(h0);
        u32x4 kv[kLoads], qv[kLoads];
        constexpr int kPer = DK * SZ / 16;     // 16 bytes each
#pragma unroll
        for (int u = 0; u < kLoads; u++) {
            const int id = u * 256 + threadIdx.x;
            kv[u] = __builtin_amdgcn_raw_buffer_load_b128(rk, (int)(id / kPer * ks + id % kPer * 16), 0, 0);
            qv[u] = __builtin_amdgcn_raw_buffer_load_b128(rq, (int)(id / kPer * qs + id % kPer * 16), 0, 0);
        }
        put_gates();
#pragma unroll
        for (int u = 0; u < kLoads; u++) {
            const int id = u * 256 + threadIdx.x;
            *(u32x4*)((unsigned char*)sK + id / kPer * (PK * SZ) + id % kPer * 16) = kv[u];
            *(u32x4*)((unsigned char*)sQ + id / kPer * (PK * SZ) + id % kPer * 16) = qv[u];
        }
    }
    PREP_MEET();

    // k.k and q.k: wave w the tiles (w, 0 .. w)
    f32x4 kk[4] = {}, qk[4] = {};
    float k2 = 0.0f, q2 = 0.0f;                // this lane's part of the sums of squares of row 16 w + l16
    const bool norm = (r.flags & REDUKT_DELTA_NORMALIZE) != 0;
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const int col = 32 * s + 8 * g4;
        float kr[8], qr[8];
        op_load(sK + (16 * wave + l16) * PK + col, kr);
        op_load(sQ + (16 * wave + l16) * PK + col, qr);
#pragma unroll
        for (int x = 0; x < 8; x++) k2 += kr[x] * kr[x], q2 += qr[x] * qr[x];
        const Split<LI> kl = split8<LI>(kr), ql = split8<LI, LI == 3>(qr);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j > wave) break;
            const Split<LI> kj = load_limbs(sK + (16 * j + l16) * PK + col);
            kk[j] = mma_limbs<3>(kl, kj, kk[j]);
            qk[j] = mma_limbs<3>(ql, kj, qk[j]);
        }
    }
    k2 += __shfl_xor(k2, 16, kWave), q2 += __shfl_xor(q2, 16, kWave);
    k2 += __shfl_xor(k2, 32, kWave), q2 += __shfl_xor(q2, 32, kWave);
    if (g4 == 0) {
        // (a key's sum that is not finite marks the token: 0 x it is NaN)
        sU[16 * wave + l16] = norm ? unit_factor(k2) : 1.0f + 0.0f * k2;
        sP[16 * wave + l16] = r.scale * (norm ? unit_factor(q2) : 1.0f);
    }
    PREP_MEET();                               // k and q are done with; sU, sP are written

    int here = threadIdx.x;
    for (uint32_t h = h0; h < h0 + per; h++) {
        asm volatile("" : "+v"(here));          // (addresses are made anew for each head: kept, they would take 80 registers)
        const int lane = here % kWave, g4 = lane / 16, l16 = lane % 16;
        if (h > h0) {
            __syncthreads();                   // the last head's fragments have been read
            put_gates();
            __syncthreads();
        }
        if (h + 1 < h0 + per) load_gates(h + 1);
        unsigned char* const unit = a.ws + ((size_t)h * a.slots + slot) * unit_bytes(LO);
        // from the first token `past` whose key, g or beta is not finite on there are no rows
        const uint64_t bads = __ballot(sU[lane] != sU[lane] || sB[lane] != sB[lane]);
        const int past = bads ? __builtin_ctzll(bads) : kChunk;
        f32x4 vp[4] = {};
        {
            double gi[4];
            float bi[4], pi[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int ti = 16 * wave + 4 * g4 + x;
                gi[x] = sG[ti];
                bi[x] = ti < past ? sB[ti] * sU[ti] : 0.0f;
                pi[x] = ti < past ? sP[ti] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int tj = 16 * j + l16;
                if (j > wave) {
#pragma unroll
                    for (int x = 0; x < 4; x++) sA[(16 * wave + 4 * g4 + x) * kPitchA + tj] = 0.0f;
                    continue;
                }
                const double gj = sG[tj];
                const float uj = tj < past ? sU[tj] : 0.0f;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    // (from a token that is not finite on the products are not looked at, and nothing before it is reached)
                    const int ti = 16 * wave + 4 * g4 + x;
                    const float w = exp2_hw(gi[x] - gj) * uj;
                    const bool in = tj <= ti && ti < past;
                    sA[ti * kPitchA + tj] = in && tj < ti ? bi[x] * w * kk[j][x] : 0.0f;
                    vp[j][x] = in ? pi[x] * w * qk[j][x] : 0.0f;
                }
            }
        }
        PREP_MEET();
        if (wave == 0) {   // the diagonal blocks: column l16 of block g4 of (I + A)^-1 by substitution
            const float* A = sA + (16 * g4) * kPitchA + 16 * g4;
            float t[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float v0 = i == l16 ? 1.0f : 0.0f, v1 = 0.0f;
#pragma unroll
                for (int j = 0; j < i; j++) {
                    if (j % 2) v1 -= A[i * kPitchA + j] * t[j];
                    else v0 -= A[i * kPitchA + j] * t[j];
                }
                t[i] = v0 + v1;
            }
            float* D = sT + (16 * g4) * kPitchA + 16 * g4 + l16;
#pragma unroll
            for (int i = 0; i < 16; i++) D[i * kPitchA] = t[i];
        } else if (wave == 1) {
            float* const vec = (float*)(unit + kTri * (3 + LO) * kFrag);
            const double last = sG[kChunk - 1];
            const float eg = exp2_hw(sG[lane]), u = sU[lane];
            sW[lane] = lane < past ? u * exp2_hw(last - sG[lane]) : 0.0f;
            vec[lane] = lane < past ? u * eg : __builtin_nanf("");
            vec[kChunk + lane] = sP[lane] * eg;
            vec[2 * kChunk + lane] = exp2_hw(last);
        }
        PREP_MEET();
        // [[T1, 0], [-T2 A21 T1, T2]]: from blocks of 16 to 32
        // (inner indices in the order 4 g + s: a lane's left elements are neighbours, and no bank is met twice on the right)
        const auto at = [&](const float* m, int tr, int tc, int row, int col) { return m[(16 * tr + row) * kPitchA + 16 * tc + col]; };
        if (wave < 2) {
            const int i = 2 * wave + 1, j = 2 * wave;
            f32x4 m = {}, y = {};
#pragma unroll
            for (int s = 0; s < 4; s++) m = mma4(at(sA, i, j, l16, 4 * g4 + s), at(sT, j, j, 4 * g4 + s, l16), m);
#pragma unroll
            for (int s = 0; s < 4; s++) y = mma4(at(sT, i, i, l16, 4 * g4 + s), m[s], y);
#pragma unroll
            for (int x = 0; x < 4; x++) sT[(16 * i + 4 * g4 + x) * kPitchA + 16 * j + l16] = -y[x];
        } else {   // the upper blocks within 32, which the fragments cover
            const int i = 2 * (wave - 2);
#pragma unroll
            for (int x = 0; x < 4; x++) sT[(16 * i + 4 * g4 + x) * kPitchA + 16 * (i + 1) + l16] = 0.0f;
        }
        PREP_MEET();
        {   // from 32 to 64: wave w block (2 + w / 2, w % 2)
            const int i = wave / 2, j = wave % 2;
            f32x4 y = {};
#pragma unroll
            for (int p = 0; p < 2; p++) {
                if (p > i) break;
                f32x4 m = {};
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    if (q < j) continue;
#pragma unroll
                    for (int s = 0; s < 4; s++) m = mma4(at(sA, 2 + p, q, l16, 4 * g4 + s), at(sT, q, j, 4 * g4 + s, l16), m);
                }
#pragma unroll
                for (int s = 0; s < 4; s++) y = mma4(at(sT, 2 + i, 2 + p, l16, 4 * g4 + s), m[s], y);
            }
            PREP_MEET();                           // A is done with: P takes its place
#pragma unroll
            for (int x = 0; x < 4; x++) sT[(32 + 16 * i + 4 * g4 + x) * kPitchA + 16 * j + l16] = -y[x];
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int x = 0; x < 4; x++) sA[(16 * wave + 4 * g4 + x) * kPitchA + 16 * k + l16] = vp[k][x];
        }
        PREP_MEET();
        // P (I + A)^-1 by tiles (row, column), whose products' lengths are row - column + 1: five for each wave
        const uint32_t tiles = (uint32_t)(0xFA5400E8009D000Cull >> 16 * wave) & 0xFFFF;      // 4 row + column, a nibble each
        f32x4 y[4] = {};
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (q > 1 && wave < 3) break;
            const int i = tiles >> (4 * q + 2) & 3, j = tiles >> 4 * q & 3;
            for (int k = j; k <= i; k++) {
#pragma unroll
                for (int s = 0; s < 4; s++) y[q] = mma4(at(sA, i, k, l16, 4 * g4 + s), at(sT, k, j, 4 * g4 + s, l16), y[q]);
            }
        }
        PREP_MEET();                               // P and (I + A)^-1 have been read: their columns take beta
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (q > 1 && wave < 3) break;
            const int i = tiles >> (4 * q + 2) & 3, j = tiles >> 4 * q & 3;
            const float bj = 16 * j + l16 < past ? sB[16 * j + l16] : 0.0f;
#pragma unroll
            for (int x = 0; x < 4; x++) sA[(16 * i + 4 * g4 + x) * kPitchA + 16 * j + l16] = y[q][x] * bj;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j > (wave | 1)) break;             // (what is above is not looked at, but within 32, where it is zeros)
            const float bj = 16 * j + l16 < past ? sB[16 * j + l16] : 0.0f;
#pragma unroll
            for (int x = 0; x < 4; x++) sT[(16 * wave + 4 * g4 + x) * kPitchA + 16 * j + l16] *= bj;
        }
        PREP_MEET();
        for (int x = wave; x < 2 * kTri; x += 4) {
            if (x < kTri) store_fragment<3>(sT, sW, unit, x, lane);
            else store_fragment<LO>(sA, nullptr, unit + kTri * 3 * kFrag, x - kTri, lane);
        }
    }
}

constexpr int kPrepBarriers = __COUNTER__ - kPrepFirst - 1;
#undef PREP_MEET

// A workgroup a chunk and `per` value heads, for all chunks and heads side by side.
// Bound by the chain of its steps, with four workgroups a CU beside each other: of 128 chunks of 32 heads, two to a key head, 50 us,
// 12,000 cycles of a workgroup go to the request of its rows and their way to LDS, 4,000 to k.k and q.k, and 23,500 to each head (A and P
// with their decays 6,000, the substitution 5,400, 32 and 64 3,500, P T and the strengths 5,500, the fragments' stores 2,600).  It
// moves 200 MB in that time, 4 TB/s, three quarters of what a copy moves.
template <typename T, int DK>
__global__ __launch_bounds__(256, Limbs<T>::in == 1 ? 4 : Limbs<T>::in == 2 ? 3 : 2) void k_delta_prep(ChunkArgs a) {
    __shared__ PrepLds<T, DK> lds;
    const uint32_t slots_h = a.d.r.hv / a.per, slot = blockIdx.x / slots_h, h0 = blockIdx.x % slots_h * a.per;
    uint32_t lo = 0, hi = a.d.n - 1;           // the last sequence that starts at this slot or before
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (first_chunk(row_of(a, mid), mid) <= slot) lo = mid;
        else hi = mid - 1;
    }
    const uint32_t b = row_of(a, lo), e = row_of(a, lo + 1), first = first_chunk(b, lo);
    if (slot < first) return;
    const uint64_t t0 = (uint64_t)b + (uint64_t)(slot - first) * kChunk;
    if (t0 < e) prepare<T, DK>(a, lds, slot, (uint32_t)t0, min(e - (uint32_t)t0, (uint32_t)kChunk), h0, a.per);
}

// One workgroup takes 16 NC columns of one head's state through a sequence.  Waves 0 to 3 carry the state: each owns a
// quarter of its rows and of a chunk's tokens, so the chain of a chunk (S -> X -> D -> S) is a quarter as long as one
// wave's would be; partial sums of K S, and X and D as limbs, pass between them through LDS, three barriers a chunk.
// Waves 4 to 7 make the outputs of the same tokens from the limbs of S and X that they find there, beside the chain
// instead of in it.  Every left operand is read by one wave only, straight from memory into registers, a chunk
// ahead of its use; K^T comes from the rows of K by LDS, transposed as it is read.
// Bound by the chunk's chain and by what a CU's L1 takes in beside it: 64 KB a chunk at dk 128 in bf16 (K, Q, T and P T), 1.7 us.  Of
// 215 us for 128 chunks of 256 column tiles the chain alone, its operands standing still in registers, is 156; with the fragments of
// K^T from memory too, 80 KB a chunk, it was 250.
//
// ALONE: sequences of one chunk at most, whose units waves 0 to 3 make first, each column tile's workgroup the same ones.
template <typename T, int DK, int NC, bool ALONE>
__global__ __launch_bounds__(512, 2) void k_delta_chunks(ChunkArgs a) {
    constexpr int LI = Limbs<T>::in, LO = Limbs<T>::out, NW = DK / 64, SZ = sizeof(T);
    constexpr int KF = 4 * NW;                 // a lane's inner indices of one wave's rows of the state
    __shared__ __attribute__((aligned(16))) f32x4 sR[NC][4][3][kWave];       // partial K S: [tile of tokens][of the other waves]
    constexpr bool kRaw = LI == 2 && NC == 4;  // (in f16 two limbs of K would be 1 KB too many beside four column tiles)
    __shared__ __attribute__((aligned(16))) unsigned char sK[4][kRaw ? 1 : LI][kChunk * 16 * NW * 2];     // each wave's columns of K
    __shared__ __attribute__((aligned(16))) unsigned char sS[NC][4][LO][kWave * KF * 2], sX[NC][2][3][kFrag], sD[NC][2][3][kFrag];
    __shared__ __attribute__((aligned(16))) int sBad[NC][16][4];
    const redukt_delta_rows& r = a.d.r;
    const int lane = threadIdx.x % kWave, wave = wave_index() % 4, g4 = lane / 16, l16 = lane % 16;
    // the workgroups that read one key head's chunks are neighbours of one XCD
    const uint32_t group = r.hv / r.hk, cols = (r.dv / 16 + NC - 1) / NC;
    const XcdTile w = xcd_tile(blockIdx.x, group * cols, a.d.n * r.hk);
    if (!w.live) return;
    const uint32_t i = a.d.n > 1 && a.d.n <= kWave ? by_length(a, w.unit / r.hk, lane) : w.unit / r.hk;
    const uint32_t hq = w.unit % r.hk, h = hq * group + w.part / cols;
    const uint32_t col0 = w.part % cols * (16 * NC) + l16;
    const int slot = entry_slot(a.d.slots, a.d.n_slots, i, a.d.states != nullptr, lane);
    if (slot == kSkip) return;
    const uint32_t b = row_of(a, i), e = max(row_of(a, i + 1), b);
    if (slot == kBad) {
        T* const out = (T*)r.out + (size_t)h * r.dv;
        for (uint32_t t = b + threadIdx.x / 16; t < e; t += 32)
            for (uint32_t col = col0; col < min(col0 - l16 + 16 * NC, r.dv); col += 16)
                out[(int64_t)t * r.out_stride + col] = (T)__builtin_nanf("");
        return;
    }
    // (of a head's last workgroup a column tile may be past dv: it takes column l16 along and stores nothing)
    const auto live = [&](int nc) { return col0 + 16 * nc < r.dv; };
    const auto col_of = [&](int nc) { return live(nc) ? col0 + 16 * nc : (uint32_t)l16; };
    const uint32_t chunks = (e - b + kChunk - 1) / kChunk, first = first_chunk(b, i);
    if constexpr (ALONE) {
        __shared__ PrepLds<T, DK> lds;
        if (chunks) {
            if (wave_index() < 4) {
                prepare<T, DK>(a, lds, first, b, e - b, h, 1);
                __builtin_amdgcn_s_waitcnt(0x0f70);                    // vmcnt(0): the unit is written before it is read
            } else {
                for (int x = 0; x < kPrepBarriers; x++) __syncthreads();       // prepare()'s
            }
            __syncthreads();
        }
    }
    typedef T vecK __attribute__((ext_vector_type(KF)));
    // Rows of a chunk by buffer accesses, whose bounds end the chunk (they count the vector offset only, so the
    // scalar one stays 0): a pointer that moves on by a chunk, and the bytes of the chunk's rows.
    struct Rows {
        const unsigned char* p;
        uint32_t stride, width;
        __device__ __forceinline__ auto rsrc(uint32_t rows) const { return rows_rsrc(p, (rows - 1) * stride + width); }
        __device__ __forceinline__ void step(uint32_t chunks) { p += (size_t)(chunks * kChunk) * stride; }
    };
    const auto rows_of = [&](const void* p, int64_t stride, uint32_t first_col, uint32_t width) {
        return Rows{(const unsigned char*)p + ((size_t)b * (uint32_t)stride + first_col) * SZ, (uint32_t)stride * SZ, width * SZ};
    };
    const auto loadK = [&](auto rsrc, uint32_t off) {
        if constexpr (KF * SZ == 8) {
            return __builtin_bit_cast(vecK, __builtin_amdgcn_raw_buffer_load_b64(rsrc, (int)off, 0, 0));
        } else if constexpr (KF * SZ == 16) {
            return __builtin_bit_cast(vecK, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off, 0, 0));
        } else {
            struct { u32x4 v[2]; } x = {{__builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off, 0, 0),
                                        __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off + 16, 0, 0)}};
            return __builtin_bit_cast(vecK, x);
        }
    };
    const auto limbs = [&](const vecK& x, auto wide) {
        Part<NW, LI> o;
        if constexpr (LI == 1) {
            o.l[0] = __builtin_bit_cast(typename Part<NW, LI>::vec, x);
        } else {
            float v[KF];
#pragma unroll
            for (int j = 0; j < KF; j++) v[j] = (float)x[j];
            o = split_part<NW, LI, wide.value && LI == 3>(v);
        }
        return o;
    };
    const unsigned char* unit = a.ws + ((size_t)h * a.slots + first) * unit_bytes(LO);
    const auto get = [&](const unsigned char (&from)[3][kFrag], auto n_) {
        constexpr int N = decltype(n_)::value;
        Split<N> o;
#pragma unroll
        for (int n = 0; n < N; n++) o.l[n] = *(const bf16x8*)(from[n] + lane * 16);
        return o;
    };
    // Fragments of the workspace, by their number from p on.  Of a triangle, the first is this wave's tile and tokens [0, 32), the
    // second tokens [32, 64): zeros for waves 0 and 1, by a buffer without bytes.
    const int f0 = wave < 2 ? wave : 2 * wave - 2;
    const auto frag = [&](const unsigned char* p, uint32_t bytes, int first) {
        return __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rows_rsrc(p, bytes), lane * 16, first * kFrag, 0));
    };
    const uint32_t frag1 = wave < 2 ? 0 : unit_bytes(LO);
    const uint32_t row4 = tile_index(wave, 4 * g4);        // the first of a lane's four tokens
    const auto bad_of = [&](int nc) {                      // the column's first token that is not finite
        const int4 v = *(const int4*)sBad[nc][l16];
        return min(min(v.x, v.y), min(v.z, v.w));
    };

    if (wave_index() < 4) {
        __builtin_amdgcn_s_setprio(3);
        const size_t at = ((size_t)slot * r.hv + h) * DK * r.dv;
        int here = lane;
        const auto state_at = [&](int nc, int p, int x) {
            const uint32_t c = col0 - l16 + here % 16 + 16 * nc;
            return at + (size_t)state_index<DK>(NW * wave + p, 4 * (here / 16) + x) * r.dv + (c < r.dv ? c : here % 16);
        };
        f32x4 S[NC][NW];
#pragma unroll
        for (int nc = 0; nc < NC; nc++)
#pragma unroll
            for (int p = 0; p < NW; p++)
#pragma unroll
                for (int x = 0; x < 4; x++) S[nc][p][x] = a.d.in ? a.d.in[state_at(nc, p, x)] : 0.0f;
        Rows rk = rows_of(r.k, r.k_stride, hq * DK, DK), rv = rows_of(r.v, r.v_stride, h * r.dv, r.dv);
        vecK kf[4];                            // tiles wave, wave + 1, .. (mod 4)
        bf16x8 tf[2][3];
        uint32_t vv[NC][4];
        f32x4 kd;
        float keep;
        uint32_t k_at[4];
#pragma unroll
        for (int o = 0; o < 4; o++) k_at[o] = tile_index((wave + o) % 4, l16) * rk.stride + (4 * KF * wave + KF * g4) * SZ;
        const auto load_k = [&](uint32_t rows) {           // all tokens, the columns of this wave's rows of the state
            const auto rsrc = rk.rsrc(rows);
#pragma unroll
            for (int o = 0; o < 4; o++) kf[o] = loadK(rsrc, k_at[o]);
        };
        const auto load_v = [&](uint32_t rows) {
            const auto rsrc = rv.rsrc(rows);
#pragma unroll
            for (int nc = 0; nc < NC; nc++)
#pragma unroll
                for (int x = 0; x < 4; x++) vv[nc][x] = buffer_bits<T>(rsrc, (row4 + x) * rv.stride + col_of(nc) * SZ);
            kd = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rows_rsrc(unit, unit_bytes(LO)), (int)row4 * 4,
                                                                                 kTri * (3 + LO) * kFrag, 0));
        };
        const auto load_t = [&]() {
#pragma unroll
            for (int n = 0; n < 3; n++) tf[0][n] = frag(unit, unit_bytes(LO), f0 * 3 + n);
#pragma unroll
            for (int n = 0; n < 3; n++) tf[1][n] = frag(unit, frag1, f0 * 3 + 3 + n);
        };
        const auto load_keep = [&]() {
            keep = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rows_rsrc(unit, unit_bytes(LO)), lane * 4,
                                                                                  kTri * (3 + LO) * kFrag + 2 * kChunk * 4, 0));
        };
        // K^T for the last step: this wave's columns of K, which it holds as rows, go through LDS and come back transposed, 4 tokens x
        // 16 columns by 16 lanes.  A row's pieces of KF columns stand at place (piece ^ row / 8 % 4).
        Part<NW, LI> kl[4];                    // the limbs of kf
        const auto split_k = [&]() {
#pragma unroll
            for (int o = 0; o < 4; o++) {
                const int row = tile_index((wave + o) % 4, l16), at = row * (NW * 32) + (g4 ^ row / 8 % 4) * (KF * 2);
                kl[o] = limbs(kf[o], Int<0>());      // (a key with such an element is not finite: its sum of squares is not)
                if constexpr (kRaw) {
                    *(vecK*)(sK[wave][0] + at) = kf[o];
                } else {
#pragma unroll
                    for (int n = 0; n < LI; n++) *(typename Part<NW, LI>::vec*)(sK[wave][n] + at) = kl[o].l[n];
                }
            }
        };
        // Where the chain's length counts most, a chunk's K is requested as the chunk before begins, and split beside its last products; else
        // it is split as its own chunk begins (us late and early: 8,192 tokens of 32 heads of 128, 275 and 266; 37 ragged prompts with four
        // tiles, 192 and 196; 12 sequences of heads of 64, 194 and 198).
        constexpr bool kEarly = DK == 128 && NC < 4;
        const auto get_kt = [&](int p, int s, int n) {       // row l16 of tile p, the tokens 32 s + 8 g4 + [0, 8)
            typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
            const unsigned char* const at = sK[wave][n] + (32 * s + 8 * g4 + l16 / 4) * (NW * 32) + (l16 % 4 ^ g4) * (KF * 2) + 8 * p;
            struct { i16x4 v[2]; } x = {{__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at),
                                        __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at + 4 * NW * 32))}};
            return __builtin_bit_cast(bf16x8, x);
        };
        // The four rows of this wave's tile that a lane holds, as half of a right operand's fragment.
        const auto put = [&](unsigned char (*to)[3][kFrag], const f32x4& v) {
            const float x[4] = {v[0], v[1], v[2], v[3]};
            const Part<1, 3> y = split_part<1, 3, true>(x);
#pragma unroll
            for (int n = 0; n < 3; n++)
                *(typename Part<1, 3>::vec*)(to[wave / 2][n] + lane * 16 + wave % 2 * 8) = y.l[n];
        };
        uint32_t left = e - b;                 // rows from this chunk's first on
        if (chunks) {
            const uint32_t rows = min(left, (uint32_t)kChunk);
            load_k(rows);
            load_v(rows);
            load_t();
            load_keep();
            if (kEarly) split_k();
        }
        for (uint32_t c = 0; c < chunks; c++) {
            // (the last chunk requests itself again instead of one past the end)
            const uint32_t on = left > kChunk ? 1 : 0;
            left -= on * kChunk;
            const uint32_t rows = min(left, (uint32_t)kChunk);
            rk.step(on), rv.step(on);
            unit += on * unit_bytes(LO);
            f32x4 X[NC];
            if (kEarly) load_k(rows);
            else split_k();
#pragma unroll
            for (int nc = 0; nc < NC; nc++) {
                float v[KF];
#pragma unroll
                for (int j = 0; j < KF; j++) v[j] = S[nc][j / 4][j % 4];
                const Part<NW, 3> x = split_part<NW, 3, true>(v);
#pragma unroll
                for (int n = 0; n < LO; n++) *(typename Part<NW, 3>::vec*)(sS[nc][wave][n] + lane * (KF * 2)) = x.l[n];
                f32x4 y[4] = {};
#pragma unroll
                for (int j = 0; j < 3; j++)
#pragma unroll
                    for (int n = 0; n < LI; n++)
                        if (n + j < 3) {
#pragma unroll
                            for (int o = 0; o < 4; o++) y[o] = mma_part(kl[o].l[n], x.l[j], y[o]);
                        }
                X[nc] = y[0];
#pragma unroll
                for (int o = 1; o < 4; o++) sR[nc][(wave + o) % 4][3 - o][lane] = y[o];
            }
            if (!kEarly) load_k(rows);
            __syncthreads();                   // A: S and partial sums are there
#pragma unroll
            for (int nc = 0; nc < NC; nc++) {
#pragma unroll
                for (int o = 1; o < 4; o++) X[nc] += sR[nc][wave][o - 1][lane];
                uint32_t top = 0;
                f32x4 x;
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const float v = of_bits<T>(vv[nc][y]) - kd[y] * X[nc][y];
                    x[y] = v;
                    top = max(top, __builtin_bit_cast(uint32_t, v) & 0x7fffffffu);
                }
                int bad = kChunk;              // this tile's first token in this column that is not finite
                if (__any(top >= 0x7f800000u)) {
#pragma unroll
                    for (int y = 3; y >= 0; y--)
                        if (!(fabsf(x[y]) < __builtin_inff())) bad = row4 + y, x[y] = 0.0f;
                    bad = min(bad, __shfl_xor(bad, 16, kWave));
                    bad = min(bad, __shfl_xor(bad, 32, kWave));
                }
                sBad[nc][l16][wave] = bad;     // (the same from all four lanes of a column)
                put(sX[nc], x);
            }
            load_v(rows);
            __syncthreads();                   // B: X is there
#pragma unroll
            for (int nc = 0; nc < NC; nc++) {
                const int bad = bad_of(nc);
                f32x4 D = mma_four(tf, get(sX[nc][0], Int<3>()), get(sX[nc][1], Int<3>()));
                if (__any(bad < kChunk)) {
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        if ((int)row4 + y >= bad) D[y] = __builtin_nanf("");
                }
                put(sD[nc], D);
            }
            load_t();
            Split<LI> ktf[NW][2];
#pragma unroll
            for (int f = 0; f < NW * 2; f++) {
                if constexpr (kRaw) {
                    typedef T eight __attribute__((ext_vector_type(8)));
                    const eight k = __builtin_bit_cast(eight, get_kt(f / 2, f % 2, 0));
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) v[j] = (float)k[j];
                    ktf[f / 2][f % 2] = split8<LI>(v);
                } else {
#pragma unroll
                    for (int n = 0; n < LI; n++) ktf[f / 2][f % 2].l[n] = get_kt(f / 2, f % 2, n);
                }
            }
            __syncthreads();                   // C: D is there
#pragma unroll
            for (int nc = 0; nc < NC; nc++) {
                const Split<3> x0 = get(sD[nc][0], Int<3>()), x1 = get(sD[nc][1], Int<3>());
                if (kEarly && nc == 0) split_k();
#pragma unroll
                for (int p = 0; p < NW; p++) {
#pragma unroll
                    for (int y = 0; y < 4; y++) S[nc][p][y] *= keep;
                }
#pragma unroll
                for (int n = 0; n < LI; n++)
#pragma unroll
                    for (int j = 0; j < 3 - n; j++)
#pragma unroll
                        for (int p = 0; p < NW; p++) S[nc][p] = mma(ktf[p][0].l[n], x0.l[j], S[nc][p]);
#pragma unroll
                for (int n = 0; n < LI; n++)
#pragma unroll
                    for (int j = 0; j < 3 - n; j++)
#pragma unroll
                        for (int p = 0; p < NW; p++) S[nc][p] = mma(ktf[p][1].l[n], x1.l[j], S[nc][p]);
            }
            load_keep();
        }
        if (a.d.states) {
            asm volatile("" : "+v"(here));     // (the addresses are made anew: kept from the start, they would take 16 registers)
#pragma unroll
            for (int nc = 0; nc < NC; nc++)
#pragma unroll
                for (int p = 0; p < NW; p++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (live(nc)) a.d.states[state_at(nc, p, x)] = S[nc][p][x];
        }
    } else {
        Rows rq = rows_of(r.q, r.q_stride, hq * DK, DK), ro = rows_of(r.out, r.out_stride, h * r.dv, r.dv);
        vecK qf[4];
        bf16x8 pf[2][LO];
        f32x4 qd;
        const uint32_t q_at = tile_index(wave, l16) * rq.stride + KF * g4 * SZ;
        const auto load_q = [&](uint32_t rows) {           // this wave's tokens, all columns
            const auto rsrc = rq.rsrc(rows);
#pragma unroll
            for (int s = 0; s < 4; s++) qf[s] = loadK(rsrc, q_at + 4 * KF * s * SZ);
        };
        const auto load_p = [&]() {
#pragma unroll
            for (int n = 0; n < LO; n++) pf[0][n] = frag(unit, unit_bytes(LO), kTri * 3 + f0 * LO + n);
#pragma unroll
            for (int n = 0; n < LO; n++) pf[1][n] = frag(unit, frag1, kTri * 3 + f0 * LO + LO + n);
            qd = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rows_rsrc(unit, unit_bytes(LO)), (int)row4 * 4,
                                                                                 kTri * (3 + LO) * kFrag + kChunk * 4, 0));
        };
        uint32_t left = e - b;
        if (chunks) {
            load_q(min(left, (uint32_t)kChunk));
            load_p();
        }
        for (uint32_t c = 0; c < chunks; c++) {
            const auto to = ro.rsrc(min(left, (uint32_t)kChunk));
            const uint32_t on = left > kChunk ? 1 : 0;
            left -= on * kChunk;
            rq.step(on), ro.step(1);
            unit += on * unit_bytes(LO);
            // What is read here stands still until the next A (X) and until the chain's first step behind C (S), so the work lies where
            // the chain's own is long: Q S beside the second step, P X beside the fourth and first.
            f32x4 O[NC], Q[NC][2] = {};
            __syncthreads();                   // A
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const Part<NW, LI> q = limbs(qf[s], Int<1>());
#pragma unroll
                for (int nc = 0; nc < NC; nc++)
#pragma unroll
                    for (int j = 0; j < LO; j++) {
                        const auto x = *(const typename Part<NW, LI>::vec*)(sS[nc][s][j] + lane * (KF * 2));
#pragma unroll
                        for (int n = 0; n < LI; n++)
                            if (n + j < LO) Q[nc][s % 2] = mma_part(q.l[n], x, Q[nc][s % 2]);
                    }
            }
            load_q(min(left, (uint32_t)kChunk));
            __syncthreads();                   // B
            __syncthreads();                   // C
#pragma unroll
            for (int nc = 0; nc < NC; nc++) {
                const int bad = bad_of(nc);
                O[nc] = mma_limbs<LO>(as_split<LO>(pf[0]), get(sX[nc][0], Int<LO>()), f32x4{});
                const f32x4 y = mma_limbs<LO>(as_split<LO>(pf[1]), get(sX[nc][1], Int<LO>()), f32x4{});
#pragma unroll
                for (int z = 0; z < 4; z++) O[nc][z] = qd[z] * (Q[nc][0][z] + Q[nc][1][z]) + (O[nc][z] + y[z]);
                if (__any(bad < kChunk)) {
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        if ((int)row4 + y >= bad) O[nc][y] = __builtin_nanf("");
                }
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const int o = (int)((row4 + y) * ro.stride + (live(nc) ? (col0 + 16 * nc) * SZ : 0x80000000u));
                    const T v = (T)(float)O[nc][y];
                    if constexpr (SZ == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned int, v), to, o, 0, 0);
                    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), to, o, 0, 0);
                }
            }
            load_p();
        }
    }
}

const void* delta_prep_fn(uint32_t dtype, uint32_t dk) {
    static const void* const fns[3][2] = {
        {(const void*)k_delta_prep<__bf16, 64>, (const void*)k_delta_prep<__bf16, 128>},
        {(const void*)k_delta_prep<_Float16, 64>, (const void*)k_delta_prep<_Float16, 128>},
        {(const void*)k_delta_prep<float, 64>, (const void*)k_delta_prep<float, 128>},
    };
    return fns[dtype][dk == 128];
}

template <typename T, int NC, bool ALONE = false>
const void* delta_chunks_of(uint32_t dk) {
    return dk == 128 ? (const void*)k_delta_chunks<T, 128, NC, ALONE> : (const void*)k_delta_chunks<T, 64, NC, ALONE>;
}

const void* delta_alone_fn(uint32_t dtype, uint32_t dk) {
    return dtype == REDUKT_OP_BF16  ? delta_chunks_of<__bf16, 1, true>(dk)
           : dtype == REDUKT_OP_F16 ? delta_chunks_of<_Float16, 1, true>(dk)
                                    : delta_chunks_of<float, 1, true>(dk);
}

// NC 1, 2, or 4, the last with 16-bit elements only (in f32 its limbs do not fit LDS).
const void* delta_chunks_fn(uint32_t dtype, uint32_t dk, uint32_t nc) {
    if (dtype == REDUKT_OP_F32) return nc == 1 ? delta_chunks_of<float, 1>(dk) : delta_chunks_of<float, 2>(dk);
    if (dtype == REDUKT_OP_F16)
        return nc == 1 ? delta_chunks_of<_Float16, 1>(dk) : nc == 2 ? delta_chunks_of<_Float16, 2>(dk) : delta_chunks_of<_Float16, 4>(dk);
    return nc == 1 ? delta_chunks_of<__bf16, 1>(dk) : nc == 2 ? delta_chunks_of<__bf16, 2>(dk) : delta_chunks_of<__bf16, 4>(dk);
}

uint64_t chunk_slots(const redukt_delta_rows& a, uint32_t n_seq) { return (uint64_t)a.rows / kChunk + n_seq; }

uint64_t units_bytes(const redukt_delta_rows& a, uint32_t n_seq) {
    return chunk_slots(a, n_seq) * a.hv * unit_bytes(a.dtype == REDUKT_OP_F32 ? 3 : 2);
}

int32_t launch_chunks(ChunkArgs& k, void* stream) {
    const redukt_delta_rows& r = k.d.r;
    // Two value heads of one key head share its products where workgroups still fill the CUs twice over (129 chunks of 32 heads,
    // two to a key head: 304 -> 289 us with k_delta_chunks).
    if (r.hv / r.hk % 2 == 0 && chunk_slots(r, k.d.n) * r.hv >= 1024) k.per = 2;
    const uint64_t prep = chunk_slots(r, k.d.n) * (r.hv / k.per);
    // NC column tiles a workgroup read a chunk's operands once for all of them, but a chunk then takes longer: worth it once there are
    // workgroups waiting for a CU.  Ragged sequences of 16 heads of 128 columns, us with 1, 2 and 4 tiles: 5 of them (640 tiles) 88, 94
    // and 138; 10 (1,280) 96, 78 and 97; 20 (2,560) 153, 118 and 107; 37 (4,736) 296, 230 and 196.
    const uint64_t all = (uint64_t)k.d.n * r.hv * (r.dv / 16);
    // No sequence of 64 rows in all has a second chunk: the preparation goes into the same launch, once for each column tile, while all
    // workgroups are on the CUs at once, one on each, or two at dk 64 with 16-bit elements (us in two launches and one, bf16: 12 heads of
    // 64 columns, 48 tiles, 13.5 and 12.2, ten such sequences, 480 tiles, 17.5 and 16.0, twelve, 576, 20.1 and 25.0; 32 heads of 128,
    // 256 tiles, 16.3 and 14.6, 40, 320 tiles, 19.6 and 25.2).
    const bool alone = r.rows <= kChunk && all <= (r.dk == 64 && r.dtype != REDUKT_OP_F32 ? 512 : 256);
    const uint32_t NC = all >= 2048 && r.dtype != REDUKT_OP_F32 ? 4 : all >= 1024 ? 2 : 1;
    const uint64_t cols = (r.dv / 16 + NC - 1) / NC, units = (uint64_t)k.d.n * r.hk;
    const uint64_t grid = (units + kXcds - 1) / kXcds * kXcds * (r.hv / r.hk) * cols;
    if (!op_grid_ok(prep, 256) || !op_grid_ok(grid, 512)) return BACKEND_INVALID_ARGUMENT;
    k.slots = (uint32_t)chunk_slots(r, k.d.n);
    if (alone) return op_launch(delta_alone_fn(r.dtype, r.dk), dim3((uint32_t)grid), dim3(512), 0, stream, k);
    if (r.rows) {
        const int32_t rc = op_launch(delta_prep_fn(r.dtype, r.dk), dim3((uint32_t)prep), dim3(256), 0, stream, k);
        if (rc != BACKEND_OK) return rc;
    }
    return op_launch(delta_chunks_fn(r.dtype, r.dk, NC), dim3((uint32_t)grid), dim3(512), 0, stream, k);
}

bool sizes_ok(const redukt_delta_rows* a) {
    return a && a->dtype <= REDUKT_OP_F32 && a->hk > 0 && a->hv > 0 && a->hv <= 4096 && a->hv % a->hk == 0 &&
           (a->dk == 64 || a->dk == 128) && a->dv > 0 && a->dv % 32 == 0 && a->dv <= 256 && a->rows < (1u << 31) &&
           (a->flags & ~REDUKT_DELTA_NORMALIZE) == 0;
}

constexpr int64_t kMaxStride = 1 << 22;      // a chunk's 64 rows stay within 32-bit offsets

bool rows_ok(const redukt_delta_rows* a) {
    const int64_t per = 16 / op_elem_bytes(a->dtype);
    const void* const ptrs[] = {a->q, a->k, a->v, a->out};
    const int64_t strides[] = {a->q_stride, a->k_stride, a->v_stride, a->out_stride};
    const int64_t width[] = {(int64_t)a->hk * a->dk, (int64_t)a->hk * a->dk, (int64_t)a->hv * a->dv,
                             (int64_t)a->hv * a->dv};
    for (int i = 0; i < 4; i++) {
        if (!ptrs[i] || !op_aligned(ptrs[i], 16) || strides[i] % per) return false;
        if (a->rows > 1 && (strides[i] < width[i] || strides[i] > kMaxStride)) return false;
    }
    return a->g && a->beta && op_aligned(a->g, 4) && op_aligned(a->beta, 4) &&
           (a->rows <= 1 || (a->g_stride >= 0 && a->beta_stride >= 0));
}

// The rows with a step from one to the next that is a row's width where there is one row only.
redukt_delta_rows stepped(redukt_delta_rows a) {
    if (a.rows == 1) {
        a.q_stride = a.k_stride = (int64_t)a.hk * a.dk;
        a.v_stride = a.out_stride = (int64_t)a.hv * a.dv;
    }
    return a;
}

int32_t launch_step(DeltaArgs& k, void* stream) {
    const uint64_t waves = (uint64_t)k.n * k.r.hv * (k.r.dv / 32);
    if (!op_grid_ok((waves + 3) / 4, 256)) return BACKEND_INVALID_ARGUMENT;
    return op_launch(delta_step_fn(k.r.dtype, k.r.dk), dim3((uint32_t)((waves + 3) / 4)), dim3(256), 0, stream, k);
}

}  // namespace
}  // namespace rdk

using namespace rdk;

extern "C" {

int32_t redukt_op_delta_step(const redukt_delta_rows* a, float* states, uint32_t n_slots, const int32_t* slots,
                             void* stream) {
    if (!sizes_ok(a) || a->rows > kMaxOpRows) return BACKEND_INVALID_ARGUMENT;
    if (a->rows == 0) return BACKEND_OK;
    if (!rows_ok(a) || !states || !op_aligned(states, 16) || !op_aligned(slots, 4)) return BACKEND_INVALID_ARGUMENT;
    if (n_slots >= (1u << 31) || (!slots && a->rows > n_slots)) return BACKEND_INVALID_ARGUMENT;
    OpDevice dev(a->out);
    if (!dev.ok) return BACKEND_INVALID_ARGUMENT;
    DeltaArgs k{stepped(*a), states, states, n_slots, slots, nullptr, a->rows};
    return launch_step(k, stream);
}

uint64_t redukt_op_delta_chunk_workspace(const redukt_delta_rows* a, uint32_t n_seq) {
    if (!sizes_ok(a) || n_seq > kMaxOpRows) return 0;
    return units_bytes(*a, n_seq);
}

int32_t redukt_op_delta_chunk(const redukt_delta_rows* a, const int32_t* cu, uint32_t n_seq, const float* state_in,
                              float* state_out, uint32_t n_slots, const int32_t* slots, void* workspace,
                              uint64_t workspace_bytes, void* stream) {
    if (!sizes_ok(a) || n_seq > kMaxOpRows) return BACKEND_INVALID_ARGUMENT;
    if (n_seq == 0) return BACKEND_OK;
    if ((a->rows && !rows_ok(a)) || !cu || !op_aligned(cu, 4) || !op_aligned(slots, 4) || !op_aligned(state_in, 16) ||
        !op_aligned(state_out, 16))
        return BACKEND_INVALID_ARGUMENT;
    if (state_in || state_out) {
        if (n_slots >= (1u << 31) || (!slots && n_seq > n_slots)) return BACKEND_INVALID_ARGUMENT;
        if (state_in && state_out && !apart(state_in, state_out, (size_t)n_slots * a->hv * a->dk * a->dv * 4))
            return BACKEND_INVALID_ARGUMENT;
    } else if (slots) {
        return BACKEND_INVALID_ARGUMENT;
    }
    if (a->rows == 0 && !state_out) return BACKEND_OK;
    const uint64_t need = redukt_op_delta_chunk_workspace(a, n_seq);
    if (need && (!workspace || !op_aligned(workspace, 16) || workspace_bytes < need)) return BACKEND_INVALID_ARGUMENT;
    OpDevice dev(cu);
    if (!dev.ok) return BACKEND_INVALID_ARGUMENT;
    ChunkArgs k{{stepped(*a), state_in, state_out, n_slots, slots, cu, n_seq}, (unsigned char*)workspace, 0, 1};
    return launch_chunks(k, stream);
}

}  // extern "C"
