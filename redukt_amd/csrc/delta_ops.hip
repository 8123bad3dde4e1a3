// delta_ops.hip — the gated delta rule on caller tensors (redukt_ops.h).
//
// A value head's state S [dk][dv] takes a token (k, q, v, g, beta) as
//     S <- a S + k d^T,   d = beta (v - a S^T k),   o = scale S^T q,   a = e^g.
// Columns of S do not meet, so any split over dv is free; S^T k and S^T q sum over dk.
#include <hip/hip_runtime.h>

#include "op_common.h"

namespace rdk {
namespace {

constexpr int kWave = 64;
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

bool sizes_ok(const redukt_delta_rows* a) {
    return a && a->dtype <= REDUKT_OP_F32 && a->hk > 0 && a->hv > 0 && a->hv <= 4096 && a->hv % a->hk == 0 &&
           (a->dk == 64 || a->dk == 128) && a->dv > 0 && a->dv % 32 == 0 && a->dv <= 256 && a->rows < (1u << 31) &&
           (a->flags & ~REDUKT_DELTA_NORMALIZE) == 0;
}

bool rows_ok(const redukt_delta_rows* a) {
    const int64_t per = 16 / op_elem_bytes(a->dtype);
    const void* const ptrs[] = {a->q, a->k, a->v, a->out};
    const int64_t strides[] = {a->q_stride, a->k_stride, a->v_stride, a->out_stride};
    const int64_t width[] = {(int64_t)a->hk * a->dk, (int64_t)a->hk * a->dk, (int64_t)a->hv * a->dv,
                             (int64_t)a->hv * a->dv};
    for (int i = 0; i < 4; i++) {
        if (!ptrs[i] || !op_aligned(ptrs[i], 16) || strides[i] % per) return false;
        if (a->rows > 1 && strides[i] < width[i] && (i == 3 || strides[i] != 0)) return false;
    }
    return a->g && a->beta && op_aligned(a->g, 4) && op_aligned(a->beta, 4) &&
           (a->rows <= 1 || (a->g_stride >= 0 && a->beta_stride >= 0));
}

// Whether two pools of n bytes are the same one or have nothing in common.
bool apart(const void* a, const void* b, size_t n) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x == y || (x < y ? y - x : x - y) >= n;
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
    DeltaArgs k{*a, states, states, n_slots, slots, nullptr, a->rows};
    return launch_rows(k, stream);
}

uint64_t redukt_op_delta_chunk_workspace(const redukt_delta_rows* a, uint32_t n_seq) {
    (void)a, (void)n_seq;
    return 0;
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
    DeltaArgs k{*a, state_in, state_out, n_slots, slots, cu, n_seq};
    return launch_rows(k, stream);
}

}  // extern "C"
