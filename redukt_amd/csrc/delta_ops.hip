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

struct DeltaArgs {
    redukt_delta_rows r;
    const float* in;           // states read (null: zeros)
    float* states;             // states written (null: none)
    uint32_t n_slots;
    const int32_t* slots;
    const int32_t* cu;         // null: one row an entry
    uint32_t n;                // entries
};

// What becomes of entry i: its slot, or kSkip (padded, nothing is touched) or kBad (out of range, or named
// by an earlier entry while states are written).  Every lane of the wave takes part.
constexpr int kSkip = -1, kBad = -2;
__device__ __forceinline__ int entry_slot(const int32_t* slots, uint32_t n_slots, uint32_t i, bool writes, int lane) {
    if (!slots) return (int)i;
    const int s = __builtin_amdgcn_readfirstlane(slots[i]);
    if (s == -1) return kSkip;
    if (s < 0 || (uint32_t)s >= n_slots) return kBad;
    if (!writes) return s;
    bool earlier = false;
    for (uint32_t c = lane; c < i; c += kWave) earlier |= slots[c] == s;
    return __any(earlier) ? kBad : s;
}

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
// exchange between the eight row groups.
template <typename T, int DK>
__global__ __launch_bounds__(256) void k_delta_rows(DeltaArgs a) {
    constexpr int R = DK / 8;
    const redukt_delta_rows& r = a.r;
    const int lane = threadIdx.x % kWave, rg = lane / 8, c4 = (lane % 8) * 4;
    const uint32_t blocks = r.dv / 32;
    const uint64_t id = (uint64_t)blockIdx.x * (blockDim.x / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t i = (uint32_t)(id / (r.hv * blocks));
    if (i >= a.n) return;
    const uint32_t hb = (uint32_t)(id % (r.hv * blocks)), h = hb / blocks, col = hb % blocks * 32 + c4;
    const uint32_t hq = h / (r.hv / r.hk);
    uint32_t t0 = i, t1 = i + 1;
    if (a.cu) {
        t0 = min((uint32_t)max(a.cu[i], 0), r.rows);
        t1 = min((uint32_t)max(a.cu[i + 1], 0), r.rows);
    }
    const int slot = entry_slot(a.slots, a.n_slots, i, a.states != nullptr, lane);
    if (slot == kSkip) return;
    T* out = (T*)r.out + (size_t)h * r.dv + col;
    if (slot == kBad) {
        for (uint32_t t = t0 + rg; t < t1; t += 8)
            for (int j = 0; j < 4; j++) out[(int64_t)t * r.out_stride + j] = (T)__builtin_nanf("");
        return;
    }
    const size_t at = (((size_t)slot * r.hv + h) * DK + rg * R) * r.dv + col;
    float4 S[R];
#pragma unroll
    for (int e = 0; e < R; e++) S[e] = a.in ? *(const float4*)(a.in + at + (size_t)e * r.dv) : make_float4(0, 0, 0, 0);
    for (uint32_t t = t0; t < t1; t++) {
        float k[R], q[R], v[4];
        op_load((const T*)r.k + (int64_t)t * r.k_stride + hq * DK + rg * R, k);
        op_load((const T*)r.q + (int64_t)t * r.q_stride + hq * DK + rg * R, q);
        op_load((const T*)r.v + (int64_t)t * r.v_stride + h * r.dv + col, v);
        const float decay = expf(r.g[(int64_t)t * r.g_stride + h]), beta = r.beta[(int64_t)t * r.beta_stride + h];
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
            uk = rsqrtf(rows_sum(kk) + kUnitEps);
            uq *= rsqrtf(rows_sum(qq) + kUnitEps);
        }
        // d carries the key's factor, so that the rows of k enter as they are
        const float ak = decay * uk;
        const float4 d = make_float4(beta * (v[0] - ak * sk.x) * uk, beta * (v[1] - ak * sk.y) * uk,
                                     beta * (v[2] - ak * sk.z) * uk, beta * (v[3] - ak * sk.w) * uk);
#pragma unroll
        for (int e = 0; e < R; e++) {
            S[e].x = decay * S[e].x + k[e] * d.x;
            S[e].y = decay * S[e].y + k[e] * d.y;
            S[e].z = decay * S[e].z + k[e] * d.z;
            S[e].w = decay * S[e].w + k[e] * d.w;
        }
        if (rg == 0) {
            T* o = out + (int64_t)t * r.out_stride;
            o[0] = (T)(uq * (decay * sq.x + kq * d.x));
            o[1] = (T)(uq * (decay * sq.y + kq * d.y));
            o[2] = (T)(uq * (decay * sq.z + kq * d.z));
            o[3] = (T)(uq * (decay * sq.w + kq * d.w));
        }
    }
    if (a.states) {
#pragma unroll
        for (int e = 0; e < R; e++) *(float4*)(a.states + at + (size_t)e * r.dv) = S[e];
    }
}

const void* delta_rows_fn(uint32_t dtype, uint32_t dk) {
    static const void* const fns[3][2] = {
        {(const void*)k_delta_rows<__bf16, 64>, (const void*)k_delta_rows<__bf16, 128>},
        {(const void*)k_delta_rows<_Float16, 64>, (const void*)k_delta_rows<_Float16, 128>},
        {(const void*)k_delta_rows<float, 64>, (const void*)k_delta_rows<float, 128>},
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
// comes of them, are two limbs (2^-17 against an output's half step of 2^-8 or 2^-11).  G is
// summed in 64 bits: the decays are e to small differences of sums that may be large.
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
// S, X and D go from result to right operand within a lane, without LDS and without an exchange.
// Left operands take their rows in the same order.

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

// Eight f32 as N bf16 limbs: each the rounded rest of those before it (the differences are exact).
template <int N>
__device__ __forceinline__ Split<N> split8(const float (&v)[8]) {
    u32x4 w[N];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float a = v[2 * j], b = v[2 * j + 1];
#pragma unroll
        for (int n = 0; n < N; n++) {
            const uint32_t p = pack_bf16(a, b);
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

template <int N>
__device__ __forceinline__ Split<N> split_pair(const f32x4& a, const f32x4& b) {
    const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return split8<N>(v);
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

// c[m] += a(m) b for four row tiles m, limb by limb so that the tiles' sums overlap.
template <int K, int NB, typename A, typename C>
__device__ __forceinline__ void mma_rows(A&& a, const Split<NB>& b, C&& c) {
    const decltype(a(0)) x[4] = {a(0), a(1), a(2), a(3)};
    constexpr int NA = sizeof(x[0]) / sizeof(bf16x8);
#pragma unroll
    for (int i = 0; i < NA; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
            if (i + j < K) {
#pragma unroll
                for (int m = 0; m < 4; m++) c[m] = mma(x[m].l[i], b.l[j], c[m]);
            }
}

constexpr int kt_bytes(int dk, int in_limbs) { return dk / 16 * 2 * in_limbs * kFrag; }

template <int N>
__device__ __forceinline__ Split<N> as_split(const bf16x8 (&v)[N]) {
    Split<N> o;
#pragma unroll
    for (int n = 0; n < N; n++) o.l[n] = v[n];
    return o;
}

struct ChunkArgs {
    DeltaArgs d;
    unsigned char* ws;         // units: (chunk slot, value head)
    unsigned char* kt;         // fragments of k^T: (chunk slot, key head)
};

// Sequence i's rows, within [0, rows].
__device__ __forceinline__ uint32_t row_of(const ChunkArgs& a, uint32_t i) {
    return min((uint32_t)max(a.d.cu[i], 0), a.d.r.rows);
}

// Chunk c of the sequence that starts at row b and is the i-th has slot b / 64 + i + c: slots of one sequence
// are consecutive, those of the next begin after them, and rows / 64 + n slots are enough.
__device__ __forceinline__ uint32_t first_chunk(uint32_t b, uint32_t i) { return b / kChunk + i; }

__device__ __forceinline__ f32x4 mma4(float a, float b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

constexpr int kPitchA = kChunk + 4;        // f32 rows of the 64 x 64 matrices in LDS

// Fragments of the lower triangle at m (f32 [64][kPitchA], natural order), its rows times f, with N limbs to `to`: fragment
// x is tile 0, 1, 2, 2, 3, 3 and inner indices 32 s + [0, 32) with s = 0, 0, 0, 1, 0, 1.
template <int N>
__device__ __forceinline__ void store_triangle(const float* m, const float* f, unsigned char* to, int wave, int lane) {
    for (int x = wave; x < kTri; x += 4) {
        const int tile = x < 2 ? x : 2 + (x - 2) / 2, s = x < 2 ? 0 : (x - 2) % 2, row = tile_index(tile, lane % 16);
        float v[8];
        op_load(m + row * kPitchA + 32 * s + 8 * (lane / 16), v);
        const float scale = f ? f[row] : 1.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= scale;
        const Split<N> y = split8<N>(v);
#pragma unroll
        for (int n = 0; n < N; n++) *(bf16x8*)(to + (x * N + n) * kFrag + lane * 16) = y.l[n];
    }
}

// One workgroup a chunk and value head: its unit, and with a key head's first value head the fragments of k^T.
template <typename T, int DK>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 2 : 3) void k_delta_prep(ChunkArgs a) {
    constexpr int LI = Limbs<T>::in, LO = Limbs<T>::out, KS = DK / 32;
    __shared__ __attribute__((aligned(16))) float sA[kChunk * kPitchA], sT[kChunk * kPitchA];
    __shared__ double sG[kChunk];
    __shared__ float sB[kChunk], sU[kChunk], sP[kChunk], sW[kChunk];
    const redukt_delta_rows& r = a.d.r;
    const int lane = threadIdx.x % kWave, wave = wave_index(), g4 = lane / 16, l16 = lane % 16;
    const uint32_t slot = blockIdx.x / r.hv, h = blockIdx.x % r.hv, group = r.hv / r.hk, hq = h / group;
    uint32_t lo = 0, hi = a.d.n - 1;       // the last sequence that starts at this slot or before
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (first_chunk(row_of(a, mid), mid) <= slot) lo = mid;
        else hi = mid - 1;
    }
    const uint32_t b = row_of(a, lo), e = row_of(a, lo + 1), first = first_chunk(b, lo);
    if (slot < first) return;
    const uint64_t t0_ = (uint64_t)b + (uint64_t)(slot - first) * kChunk;
    if (t0_ >= e) return;
    const uint32_t t0 = (uint32_t)t0_, len = min(e - t0, (uint32_t)kChunk);

    // k.k and q.k: wave w the tiles (w, 0 .. w)
    f32x4 kk[4] = {}, qk[4] = {};
    float k2[4] = {}, q2 = 0.0f;           // this lane's part of the sums of squares: rows l16 of the column tiles, of the query tile
    const T* kp = (const T*)r.k + (size_t)hq * DK;
    const T* qp = (const T*)r.q + (size_t)hq * DK;
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const int col = 32 * s + 8 * g4;
        Split<LI> kf[4], qf;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j > wave) break;
            const uint32_t t = 16 * j + l16;
            float v[8] = {};
            if (t < len) op_load(kp + (int64_t)(t0 + t) * r.k_stride + col, v);
            kf[j] = split8<LI>(v);
#pragma unroll
            for (int x = 0; x < 8; x++) k2[j] += v[x] * v[x];
        }
        {
            const uint32_t t = 16 * wave + l16;
            float v[8] = {};
            if (t < len) op_load(qp + (int64_t)(t0 + t) * r.q_stride + col, v);
            qf = split8<LI>(v);
#pragma unroll
            for (int x = 0; x < 8; x++) q2 += v[x] * v[x];
        }
        Split<LI> own = kf[0];
#pragma unroll
        for (int j = 1; j < 4; j++)
            if (j == wave) own = kf[j];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j > wave) break;
            kk[j] = mma_limbs<3>(own, kf[j], kk[j]);
            qk[j] = mma_limbs<3>(qf, kf[j], qk[j]);
        }
    }
    const bool norm = (r.flags & REDUKT_DELTA_NORMALIZE) != 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (j > wave) break;
        float v = k2[j];
        v += __shfl_xor(v, 16, kWave);
        v += __shfl_xor(v, 32, kWave);
        // (a sum that is not finite stays one: 0 x it is NaN)
        if (j == wave && g4 == 0) sU[16 * wave + l16] = norm ? rsqrtf(v + kUnitEps) + 0.0f * v : 1.0f + 0.0f * v;
    }
    q2 += __shfl_xor(q2, 16, kWave);
    q2 += __shfl_xor(q2, 32, kWave);
    if (g4 == 0) sP[16 * wave + l16] = r.scale * (norm ? rsqrtf(q2 + kUnitEps) : 1.0f);

    unsigned char* unit = a.ws + ((size_t)slot * r.hv + h) * unit_bytes(LO);
    float* vec = (float*)(unit + kTri * (3 + LO) * kFrag);
    if (h % group == 0) {
        // row (*) of k^T's tile p, the tokens 32 s + 8 g + [0, 8)
        unsigned char* const kt = a.kt + ((size_t)slot * r.hk + hq) * kt_bytes(DK, LI);
        for (int f = wave; f < DK / 16 * 2; f += 4) {
            const T* const col = kp + tile_index(f / 2, l16);
            float v[8];
#pragma unroll
            for (int x = 0; x < 8; x++) {
                const uint32_t t = 32 * (f % 2) + 8 * g4 + x;
                v[x] = t < len ? (float)col[(int64_t)(t0 + t) * r.k_stride] : 0.0f;
            }
            const Split<LI> y = split8<LI>(v);
#pragma unroll
            for (int n = 0; n < LI; n++) *(bf16x8*)(kt + (f * LI + n) * kFrag + lane * 16) = y.l[n];
        }
    }
    __syncthreads();                       // sU and sP are written
    if (wave == 0) {
        const bool in = (uint32_t)lane < len;
        const float g0 = in ? r.g[(int64_t)(t0 + lane) * r.g_stride + h] : 0.0f;
        const float beta = in ? r.beta[(int64_t)(t0 + lane) * r.beta_stride + h] : 0.0f, u = sU[lane];
        const bool bad = !(g0 < __builtin_inff()) || !(fabsf(beta) < __builtin_inff()) || u != u;
        const uint64_t bads = __ballot(bad);
        const bool past = bads && lane >= __builtin_ctzll(bads);       // from the first such token on
        double g = past ? 0.0 : (double)fmaxf(g0, -1e5f);
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const double v = __shfl_up(g, o, kWave);
            if (lane >= o) g += v;
        }
        const double last = __shfl(g, kWave - 1, kWave);
        sG[lane] = g;
        sB[lane] = past ? __builtin_nanf("") : beta;
        const float eg = expf((float)g);
        sW[lane] = in && !past ? u * expf((float)(last - g)) : 0.0f;
        vec[lane] = past ? __builtin_nanf("") : u * eg;
        vec[kChunk + lane] = sP[lane] * eg;
        vec[2 * kChunk + lane] = expf((float)last);
    }
    __syncthreads();
    f32x4 vp[4] = {};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int tj = 16 * j + l16;
        const float bj = sB[tj];
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const int ti = 16 * wave + 4 * g4 + x;
            float va = 0.0f;
            if (j <= wave && tj <= ti && bj == bj && sB[ti] == sB[ti]) {
                const float w = expf((float)(sG[ti] - sG[tj])) * sU[tj];
                va = tj < ti ? sB[ti] * sU[ti] * w * kk[j][x] : 0.0f;
                vp[j][x] = sP[ti] * w * qk[j][x];
            }
            sA[ti * kPitchA + tj] = va;
        }
    }
    __syncthreads();
    {   // the diagonal blocks: column l16 of (I + A)^-1 by substitution
        const float* A = sA + (16 * wave) * kPitchA + 16 * wave;
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
        float* D = sT + (16 * wave) * kPitchA + 16 * wave + l16;
        if (g4 == 0) {
#pragma unroll
            for (int i = 0; i < 16; i++) D[i * kPitchA] = t[i];
        }
    }
    __syncthreads();
    // [[T1, 0], [-T2 A21 T1, T2]]: from blocks of 16 to 32
    auto at = [&](const float* m, int tr, int tc, int row, int col) { return m[(16 * tr + row) * kPitchA + 16 * tc + col]; };
    if (wave < 2) {
        const int i = 2 * wave + 1, j = 2 * wave;
        f32x4 m = {}, y = {};
#pragma unroll
        for (int s = 0; s < 4; s++) m = mma4(at(sA, i, j, l16, 4 * s + g4), at(sT, j, j, 4 * s + g4, l16), m);
#pragma unroll
        for (int s = 0; s < 4; s++) y = mma4(at(sT, i, i, l16, 4 * g4 + s), m[s], y);
#pragma unroll
        for (int x = 0; x < 4; x++) sT[(16 * i + 4 * g4 + x) * kPitchA + 16 * j + l16] = -y[x];
    } else {   // the upper blocks within 32, which the fragments cover
        const int i = 2 * (wave - 2);
#pragma unroll
        for (int x = 0; x < 4; x++) sT[(16 * i + 4 * g4 + x) * kPitchA + 16 * (i + 1) + l16] = 0.0f;
    }
    __syncthreads();
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
                for (int s = 0; s < 4; s++)
                    m = mma4(at(sA, 2 + p, q, l16, 4 * s + g4), at(sT, q, j, 4 * s + g4, l16), m);
            }
#pragma unroll
            for (int s = 0; s < 4; s++) y = mma4(at(sT, 2 + i, 2 + p, l16, 4 * g4 + s), m[s], y);
        }
        __syncthreads();               // A is done with: P takes its place, and its columns take beta with T's
#pragma unroll
        for (int x = 0; x < 4; x++) sT[(32 + 16 * i + 4 * g4 + x) * kPitchA + 16 * j + l16] = -y[x];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int x = 0; x < 4; x++) sA[(16 * wave + 4 * g4 + x) * kPitchA + 16 * k + l16] = vp[k][x];
    }
    __syncthreads();
    f32x4 y[4] = {};                   // rows 16 wave of P (I + A)^-1
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (j > wave) break;
#pragma unroll
        for (int k = j; k < 4; k++) {
            if (k > wave) break;
#pragma unroll
            for (int s = 0; s < 4; s++) y[j] = mma4(at(sA, wave, k, l16, 4 * s + g4), at(sT, k, j, 4 * s + g4, l16), y[j]);
        }
    }
    // diag() T, and P T once every wave has read P: columns times beta (0 from a token that is not finite on)
    const auto beta_of = [&](int t) { const float v = sB[t]; return v == v ? v : 0.0f; };
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float bj = beta_of(16 * j + l16);
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const int at_ = (16 * wave + 4 * g4 + x) * kPitchA + 16 * j + l16;
            sA[at_] = y[j][x] * bj;
            sT[at_] = j <= (wave | 1) ? sT[at_] * bj : 0.0f;
        }
    }
    __syncthreads();
    store_triangle<3>(sT, sW, unit, wave, lane);
    store_triangle<LO>(sA, nullptr, unit + kTri * 3 * kFrag, wave, lane);
}

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

// One workgroup of four waves takes 16 NC columns of one head's state through a sequence.  A wave owns a quarter of the
// state's rows and of a chunk's tokens, so the chain of a chunk (S -> X -> D -> S) is a quarter as long as one
// wave's would be; S, X and D pass between the waves as limbs through LDS, three barriers a chunk.  Every left operand is read
// by one wave only, straight from memory into registers, a chunk ahead of its use.
template <typename T, int DK, int NC>
__global__ __launch_bounds__(256, 2) void k_delta_chunks(ChunkArgs a) {
    constexpr int LI = Limbs<T>::in, LO = Limbs<T>::out, KS = DK / 32, NW = DK / 64, SZ = sizeof(T);
    __shared__ __attribute__((aligned(16))) unsigned char sS[NC][KS][3][kFrag], sX[NC][2][3][kFrag], sD[NC][2][3][kFrag];
    __shared__ __attribute__((aligned(16))) int sBad[NC][16][4];
    const redukt_delta_rows& r = a.d.r;
    const int lane = threadIdx.x % kWave, wave = wave_index(), g4 = lane / 16, l16 = lane % 16;
    // the workgroups that read one key head's chunks are neighbours of one XCD
    const uint32_t group = r.hv / r.hk, cols = (r.dv / 16 + NC - 1) / NC;
    const XcdTile w = xcd_tile(blockIdx.x, group * cols, a.d.n * r.hk);
    if (!w.live) return;
    const uint32_t i = w.unit / r.hk, hq = w.unit % r.hk, h = hq * group + w.part / cols;
    const uint32_t col0 = w.part % cols * (16 * NC) + l16;
    const int slot = entry_slot(a.d.slots, a.d.n_slots, i, a.d.states != nullptr, lane);
    if (slot == kSkip) return;
    const uint32_t b = row_of(a, i), e = max(row_of(a, i + 1), b);
    if (slot == kBad) {
        T* const out = (T*)r.out + (size_t)h * r.dv;
        for (uint32_t t = b + threadIdx.x / 16; t < e; t += 16)
            for (uint32_t col = col0; col < min(col0 - l16 + 16 * NC, r.dv); col += 16)
                out[(int64_t)t * r.out_stride + col] = (T)__builtin_nanf("");
        return;
    }
    // (of a head's last workgroup a column tile may be past dv: it takes column l16 along and stores nothing)
    const auto live = [&](int nc) { return col0 + 16 * nc < r.dv; };
    const auto col_of = [&](int nc) { return live(nc) ? col0 + 16 * nc : (uint32_t)l16; };
    const size_t at = ((size_t)slot * r.hv + h) * DK * r.dv;
    f32x4 S[NC][NW];
#pragma unroll
    for (int nc = 0; nc < NC; nc++)
#pragma unroll
        for (int p = 0; p < NW; p++)
#pragma unroll
            for (int x = 0; x < 4; x++)
                S[nc][p][x] = a.d.in ? a.d.in[at + (size_t)tile_index(NW * wave + p, 4 * g4 + x) * r.dv + col_of(nc)] : 0.0f;
    const uint32_t chunks = (e - b + kChunk - 1) / kChunk, first = first_chunk(b, i);
    typedef T vec8 __attribute__((ext_vector_type(8), aligned(16)));
    vec8 kf[KS], qf[KS];
    bf16x8 tf[2][3], pf[2][LO], ktf[NW][2][LI];
    uint32_t vv[NC][4];
    f32x4 kd, qd;
    float keep;
    // Rows of a chunk by buffer accesses, whose bounds end the chunk (they count the vector offset only, so the
    // scalar one stays 0).
    const uint32_t ks = (uint32_t)r.k_stride * SZ, qs = (uint32_t)r.q_stride * SZ, vs = (uint32_t)r.v_stride * SZ,
                   os = (uint32_t)r.out_stride * SZ;
    const uint32_t row = tile_index(wave, l16), row4 = tile_index(wave, 4 * g4);
    const auto rows_in = [&](uint32_t c) { return min(e - b - c * kChunk, (uint32_t)kChunk); };
    const auto rsrc_of = [&](const void* p, uint32_t c, uint32_t stride, uint32_t first_col, uint32_t width) {
        return rows_rsrc((const unsigned char*)p + (size_t)(b + c * kChunk) * stride + (size_t)first_col * SZ,
                         (rows_in(c) - 1) * stride + width * SZ);
    };
    const auto load8 = [&](auto rsrc, uint32_t off) {
        if constexpr (SZ == 2) {
            return __builtin_bit_cast(vec8, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off, 0, 0));
        } else {
            struct { u32x4 v[2]; } x = {{__builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off, 0, 0),
                                        __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off + 16, 0, 0)}};
            return __builtin_bit_cast(vec8, x);
        }
    };
    const auto unit_of = [&](uint32_t c) { return a.ws + ((size_t)(first + c) * r.hv + h) * unit_bytes(LO); };
    const auto load_kq = [&](uint32_t c) {
        const auto rk = rsrc_of(r.k, c, ks, hq * DK, DK);
        const auto rq = rsrc_of(r.q, c, qs, hq * DK, DK);
#pragma unroll
        for (int s = 0; s < KS; s++) {
            kf[s] = load8(rk, row * ks + (32 * s + 8 * g4) * SZ);
            qf[s] = load8(rq, row * qs + (32 * s + 8 * g4) * SZ);
        }
    };
    const auto load_v = [&](uint32_t c) {
        const auto rv = rsrc_of(r.v, c, vs, h * r.dv, r.dv);
#pragma unroll
        for (int nc = 0; nc < NC; nc++)
#pragma unroll
            for (int x = 0; x < 4; x++) vv[nc][x] = buffer_bits<T>(rv, (row4 + x) * vs + col_of(nc) * SZ);
        const float* const vec = (const float*)(unit_of(c) + kTri * (3 + LO) * kFrag);
        kd = *(const f32x4*)(vec + row4);
        qd = *(const f32x4*)(vec + kChunk + row4);
    };
    // fragment 0 is this wave's tile and tokens [0, 32), 1 tokens [32, 64) (waves 2 and 3 only)
    const int f0 = wave < 2 ? wave : 2 * wave - 2, f1 = wave < 2 ? wave : f0 + 1;
    const auto load_tp = [&](uint32_t c) {
        const unsigned char* const u = unit_of(c);
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int f = s ? f1 : f0;
#pragma unroll
            for (int n = 0; n < 3; n++) tf[s][n] = *(const bf16x8*)(u + (f * 3 + n) * kFrag + lane * 16);
#pragma unroll
            for (int n = 0; n < LO; n++) pf[s][n] = *(const bf16x8*)(u + (kTri * 3 + f * LO + n) * kFrag + lane * 16);
        }
    };
    const auto load_kt = [&](uint32_t c) {
        const unsigned char* const u = a.kt + ((size_t)(first + c) * r.hk + hq) * kt_bytes(DK, LI) + wave * (NW * 2 * LI * kFrag);
#pragma unroll
        for (int f = 0; f < NW * 2; f++)
#pragma unroll
            for (int n = 0; n < LI; n++) ktf[f / 2][f % 2][n] = *(const bf16x8*)(u + (f * LI + n) * kFrag + lane * 16);
        keep = ((const float*)(unit_of(c) + kTri * (3 + LO) * kFrag))[2 * kChunk];
    };
    // The four rows of tile `tile` that this lane holds, as half of a right operand's fragment.
    const auto put = [&](unsigned char (*to)[3][kFrag], int tile, const f32x4& v) {
        float a0 = v[0], a1 = v[1], a2 = v[2], a3 = v[3];
#pragma unroll
        for (int n = 0; n < 3; n++) {
            const uint32_t p = pack_bf16(a0, a1), q = pack_bf16(a2, a3);
            *(uint2*)(to[tile / 2][n] + lane * 16 + tile % 2 * 8) = make_uint2(p, q);
            a0 -= __builtin_bit_cast(float, p << 16), a1 -= __builtin_bit_cast(float, p & 0xffff0000u);
            a2 -= __builtin_bit_cast(float, q << 16), a3 -= __builtin_bit_cast(float, q & 0xffff0000u);
        }
    };
    const auto get = [&](const unsigned char (&from)[3][kFrag]) {
        Split<3> o;
#pragma unroll
        for (int n = 0; n < 3; n++) o.l[n] = *(const bf16x8*)(from[n] + lane * 16);
        return o;
    };
    const auto limbs = [&](const vec8& x) {
        if constexpr (LI == 1) {
            return Split<1>{{__builtin_bit_cast(bf16x8, x)}};
        } else {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = (float)x[j];
            return split8<LI>(v);
        }
    };
    const auto put_state = [&]() {
#pragma unroll
        for (int nc = 0; nc < NC; nc++)
#pragma unroll
            for (int p = 0; p < NW; p++) put(sS[nc], NW * wave + p, S[nc][p]);
    };
    if (chunks) {
        load_kq(0);
        load_v(0);
        load_tp(0);
        load_kt(0);
        put_state();
    }
    for (uint32_t c = 0; c < chunks; c++) {
        // (the last chunk requests itself again instead of one past the end)
        const uint32_t next = min(c + 1, chunks - 1);
        __syncthreads();                   // S is there
        f32x4 X[NC][2] = {}, O[NC][2] = {};
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const Split<LI> kl = limbs(kf[s]), ql = limbs(qf[s]);
#pragma unroll
            for (int nc = 0; nc < NC; nc++) {
                const Split<3> x = get(sS[nc][s]);
                X[nc][s % 2] = mma_limbs<3>(kl, x, X[nc][s % 2]);
                O[nc][s % 2] = mma_limbs<LO>(ql, x, O[nc][s % 2]);
            }
        }
        load_kq(next);
        bool any_bad = false;
#pragma unroll
        for (int nc = 0; nc < NC; nc++) {
            uint32_t top = 0;
            f32x4 x;
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const float v = of_bits<T>(vv[nc][y]) - kd[y] * (X[nc][0][y] + X[nc][1][y]);
                x[y] = v;
                O[nc][0][y] = qd[y] * (O[nc][0][y] + O[nc][1][y]);
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
            if (lane < 16) sBad[nc][l16][wave] = bad;
            put(sX[nc], wave, x);
        }
        load_v(next);
        __syncthreads();                   // X is there
        f32x4 D[NC] = {};
        int bad[NC];
#pragma unroll
        for (int nc = 0; nc < NC; nc++) {
            const int4 v = *(const int4*)sBad[nc][l16];
            bad[nc] = min(min(v.x, v.y), min(v.z, v.w));
            any_bad |= bad[nc] < kChunk;
            const Split<3> x = get(sX[nc][0]);
            D[nc] = mma_limbs<3>(as_split<3>(tf[0]), x, D[nc]);
            O[nc][0] = mma_limbs<LO>(as_split<LO>(pf[0]), x, O[nc][0]);
        }
        if (wave >= 2) {
#pragma unroll
            for (int nc = 0; nc < NC; nc++) {
                const Split<3> x = get(sX[nc][1]);
                D[nc] = mma_limbs<3>(as_split<3>(tf[1]), x, D[nc]);
                O[nc][0] = mma_limbs<LO>(as_split<LO>(pf[1]), x, O[nc][0]);
            }
        }
        load_tp(next);
        if (__any(any_bad)) {
#pragma unroll
            for (int nc = 0; nc < NC; nc++)
#pragma unroll
                for (int y = 0; y < 4; y++)
                    if ((int)row4 + y >= bad[nc]) O[nc][0][y] = D[nc][y] = __builtin_nanf("");
        }
#pragma unroll
        for (int nc = 0; nc < NC; nc++) put(sD[nc], wave, D[nc]);
        __syncthreads();                   // D is there
#pragma unroll
        for (int nc = 0; nc < NC; nc++) {
#pragma unroll
            for (int p = 0; p < NW; p++)
#pragma unroll
                for (int y = 0; y < 4; y++) S[nc][p][y] *= keep;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const Split<3> x = get(sD[nc][s]);
#pragma unroll
                for (int p = 0; p < NW; p++) S[nc][p] = mma_limbs<3>(as_split<LI>(ktf[p][s]), x, S[nc][p]);
            }
        }
        load_kt(next);
        put_state();
        const auto ro = rsrc_of(r.out, c, os, h * r.dv, r.dv);
#pragma unroll
        for (int nc = 0; nc < NC; nc++)
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const int o = (int)((row4 + y) * os + (live(nc) ? (col0 + 16 * nc) * SZ : 0x80000000u));
                const T v = (T)(float)O[nc][0][y];
                if constexpr (SZ == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned int, v), ro, o, 0, 0);
                else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), ro, o, 0, 0);
            }
    }
    if (a.d.states) {
#pragma unroll
        for (int nc = 0; nc < NC; nc++)
#pragma unroll
            for (int p = 0; p < NW; p++)
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if (live(nc))
                        a.d.states[at + (size_t)tile_index(NW * wave + p, 4 * g4 + x) * r.dv + col0 + 16 * nc] = S[nc][p][x];
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

template <int NC>
const void* delta_chunks_fn(uint32_t dtype, uint32_t dk) {
    static const void* const fns[3][2] = {
        {(const void*)k_delta_chunks<__bf16, 64, NC>, (const void*)k_delta_chunks<__bf16, 128, NC>},
        {(const void*)k_delta_chunks<_Float16, 64, NC>, (const void*)k_delta_chunks<_Float16, 128, NC>},
        {(const void*)k_delta_chunks<float, 64, NC>, (const void*)k_delta_chunks<float, 128, NC>},
    };
    return fns[dtype][dk == 128];
}

uint64_t chunk_slots(const redukt_delta_rows& a, uint32_t n_seq) { return (uint64_t)a.rows / kChunk + n_seq; }

#ifndef KNC
#define KNC 1
#endif
uint64_t units_bytes(const redukt_delta_rows& a, uint32_t n_seq) {
    return chunk_slots(a, n_seq) * a.hv * unit_bytes(a.dtype == REDUKT_OP_F32 ? 3 : 2);
}

int32_t launch_chunks(ChunkArgs& k, void* stream) {
    const redukt_delta_rows& r = k.d.r;
    const uint64_t prep = chunk_slots(r, k.d.n) * r.hv;
    constexpr uint32_t NC = KNC;
    const uint64_t cols = (r.dv / 16 + NC - 1) / NC, units = (uint64_t)k.d.n * r.hk;
    const uint64_t grid = (units + kXcds - 1) / kXcds * kXcds * (r.hv / r.hk) * cols;
    if (prep > 0x7fffffffu || grid > 0x7fffffffu) return BACKEND_INVALID_ARGUMENT;
    k.kt = k.ws + units_bytes(r, k.d.n);
    if (r.rows) {
        const int32_t rc = op_launch(delta_prep_fn(r.dtype, r.dk), dim3((uint32_t)prep), dim3(256), 0, stream, k);
        if (rc != BACKEND_OK) return rc;
    }
    return op_launch(delta_chunks_fn<NC>(r.dtype, r.dk), dim3((uint32_t)grid), dim3(256), 0, stream, k);
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

// Whether two pools of n bytes are the same one or have nothing in common.
bool apart(const void* a, const void* b, size_t n) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x == y || (x < y ? y - x : x - y) >= n;
}

// The rows with a step from one to the next that is a row's width where there is one row only.
redukt_delta_rows stepped(redukt_delta_rows a) {
    if (a.rows == 1) {
        a.q_stride = a.k_stride = (int64_t)a.hk * a.dk;
        a.v_stride = a.out_stride = (int64_t)a.hv * a.dv;
    }
    return a;
}

int32_t launch_rows(DeltaArgs& k, void* stream) {
    const uint64_t waves = (uint64_t)k.n * k.r.hv * (k.r.dv / 32);
    if ((waves + 3) / 4 > 0x7fffffffu) return BACKEND_INVALID_ARGUMENT;
    return op_launch(delta_rows_fn(k.r.dtype, k.r.dk), dim3((uint32_t)((waves + 3) / 4)), dim3(256), 0, stream, k);
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
    return launch_rows(k, stream);
}

uint64_t redukt_op_delta_chunk_workspace(const redukt_delta_rows* a, uint32_t n_seq) {
    if (!sizes_ok(a) || n_seq > kMaxOpRows) return 0;
    const int limbs = a->dtype == REDUKT_OP_F32 ? 3 : a->dtype == REDUKT_OP_F16 ? 2 : 1;
    return units_bytes(*a, n_seq) + chunk_slots(*a, n_seq) * a->hk * kt_bytes(a->dk, limbs);
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
    ChunkArgs k{{stepped(*a), state_in, state_out, n_slots, slots, cu, n_seq}, (unsigned char*)workspace, nullptr};
    return launch_chunks(k, stream);
}

}  // extern "C"
