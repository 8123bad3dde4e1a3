// scan_ops.hip — the selective scan on caller tensors (redukt_ops.h): one token, whole sequences, gradients.
//
// A channel's state h [n] takes a token (x, dt, z; B, C of its group) as
//     h <- e^(s a) h + s x B,   y = C . h + d x,   out = y silu(z),   s = softplus(dt + dt_bias).
// Channels do not meet, and neither do the n parts of a state but in C . h.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "op_common.h"

#pragma clang fp contract(fast)

namespace rdk {
namespace {

// ---------------------------------------------------------------- lanes
//
// Four lanes share a channel, each with S = n / 4 parts of its state; a wave has 16 channels, a workgroup 64.  What a token costs
// apart from its state (the softplus, the gate, loads and stores) is shared out the other way round: of four tokens in turn, each lane
// of the quad does one.  Values go from a lane to its quad by DPP moves, and four tokens' partial sums come back as
// each lane's own token's sum.

constexpr int kBlock = 256;
constexpr int kBlockCh = 64;               // channels of a workgroup

template <int S> struct Parts { typedef float vec __attribute__((ext_vector_type(S))); };

template <int J>
__device__ __forceinline__ float quad_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), J * 0x55, 0xf, 0xf, true));
}
__device__ __forceinline__ float quad_xor1(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xb1, 0xf, 0xf, true));
}
__device__ __forceinline__ float quad_xor2(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4e, 0xf, 0xf, true));
}

// The quad's sum of v, (0 + 1) + (2 + 3), in all four lanes.
__device__ __forceinline__ float quad_sum(float v) {
    v += quad_xor1(v);
    return v + quad_xor2(v);
}

// Lane q of the quad gets the quad's sum of p[q], in quad_sum's order.
__device__ __forceinline__ float quad_sums(const float (&p)[4], int q) {
    const bool odd = q & 1, high = q & 2;
    const float s01 = (odd ? p[1] : p[0]) + quad_xor1(odd ? p[0] : p[1]);
    const float s23 = (odd ? p[3] : p[2]) + quad_xor1(odd ? p[2] : p[3]);
    return (high ? s23 : s01) + quad_xor2(high ? s01 : s23);
}

// ---------------------------------------------------------------- functions

constexpr float kLog2e = 0x1.715476p+0f, kLog2eRest = 0x1.4ae0cp-26f, kLn2 = 0x1.62e43p-1f;

// e^v for v <= 0: the power's argument in two parts, so its rounding does not grow with |v|.
__device__ __forceinline__ float exp_down(float v) {
    v = fmaxf(v, -200.0f);                     // (e^-inf, without inf - inf in the rest; of NaN as well, which callers keep)
    const float t = v * kLog2e, rest = fmaf(v, kLog2e, -t) + v * kLog2eRest, e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, rest * kLn2, e);
}

// ln(1 + e) for e in [0, 1], as 2 artanh(w) = 2 (w + w^3 / 3 + ...) with w = e / (2 + e) <= 1/3: the series' tail as a polynomial of
// degree 3 in w^2, fitted so that its largest relative error on [0, 1/3] is least (4.5e-9).
__device__ __forceinline__ float log_1p(float e) {
    const float w = e * __builtin_amdgcn_rcpf(2.0f + e), w2 = w * w;
    float p = 0x1.1ed7bep-3f;
    p = fmaf(p, w2, 0x1.1ebd0ep-3f);
    p = fmaf(p, w2, 0x1.99d208p-3f);
    p = fmaf(p, w2, 0x1.555502p-2f);
    return 2.0f * fmaf(w * w2, p, w);
}

// ln(1 + e^v), and its derivative.
struct Step {
    float s, slope;
};
__device__ __forceinline__ Step softplus(float v) {
    const float e = exp_down(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.0f + e);
    return {(v <= 0.0f ? 0.0f : v) + log_1p(e), v > 0.0f ? r : e * r};     // (s of NaN is NaN)
}

// 1 / (1 + e^-v); of NaN a number, times which it stays NaN.
__device__ __forceinline__ float sigmoid(float v) {
    const float e = exp_down(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.0f + e);
    return v > 0.0f ? r : e * r;
}

__device__ __forceinline__ float power(float s, float a2) { return __builtin_amdgcn_exp2f(s * a2); }

// ---------------------------------------------------------------- one token

struct ScanArgs {
    redukt_scan_rows r;
    const float* in;           // states read (null: zeros)
    float* states;             // states written (null: none)
    uint32_t n_slots;
    const int32_t* slots;
    const int32_t* cu;         // null: one row an entry
    uint32_t n;                // entries
    float* ws;                 // pieces: states [places][channels][n], then the sums of their time steps [places][channels]
    uint32_t pieces;           // places
    uint16_t joined;           // the first states of all pieces are in ws (k_scan_join)
    uint16_t spread;           // which place a piece has (place_of)
};

// A lane's parts of its channel's a (times log2 e), and d and dt_bias.
template <int S>
struct Channel {
    float a2[S], d, bias;
};

template <int S>
__device__ __forceinline__ Channel<S> channel_of(const redukt_scan_rows& r, uint32_t ch, int q) {
    Channel<S> k;
    const float* const a = r.a + (size_t)ch * (4 * S) + q * S;
#pragma unroll
    for (int i = 0; i < S; i++) k.a2[i] = a[i] * kLog2e;
    k.d = r.d ? r.d[ch] : 0.0f;
    k.bias = r.dt_bias ? r.dt_bias[ch] : 0.0f;
    return k;
}

template <int S>
__device__ __forceinline__ void load_state(const float* p, float (&h)[S]) {
    const typename Parts<S>::vec v = *(const typename Parts<S>::vec*)p;
#pragma unroll
    for (int i = 0; i < S; i++) h[i] = v[i];
}

template <int S>
__device__ __forceinline__ void store_state(float* p, const float (&h)[S]) {
    typename Parts<S>::vec v;
#pragma unroll
    for (int i = 0; i < S; i++) v[i] = h[i];
    *(typename Parts<S>::vec*)p = v;
}

// A wave takes 64 channels of an entry, 16 at a time with their states' loads side by side (NB 4), or 16 (NB 1, while there are too few waves
// for the device otherwise).  With NB 4 each lane of a quad does one of the four channels' softplus and gate.
// Bound by the states' bytes, read and written once: 1,000 entries of 1,536 channels of 16, 206 MB, 33 us in a row of calls on the same states
// (in part from cache) and 46 where states change from call to call (4.5 TB/s; a large copy moves 5.2).  One entry is the launch, 3.3 us.
template <typename T, int S, int NB>
__global__ __launch_bounds__(kBlock) void k_scan_step(ScanArgs a) {
    constexpr int N = 4 * S, kWide = 16 * NB;
    const redukt_scan_rows& r = a.r;
    const int lane = threadIdx.x % kOpWave, q = lane % 4;
    const uint32_t blocks = (r.channels + kWide - 1) / kWide;
    const uint64_t id = (uint64_t)blockIdx.x * (kBlock / kOpWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kOpWave);
    const uint32_t i = (uint32_t)(id / blocks), ch0 = (uint32_t)(id % blocks) * kWide;
    if (i >= a.n) return;
    // (the lane's own channel, for which it does what a quad shares out)
    const uint32_t own = ch0 + lane / 4 + (NB == 4 ? 16 * q : 0), ch = min(own, r.channels - 1);
    const bool in = own < r.channels && (NB == 4 || q == 0);
    const uint32_t g = ch0 / (r.channels / r.groups) * N + q * S;
    const T* const pb = (const T*)r.b + (int64_t)i * r.b_stride + g;
    const T* const pc = (const T*)r.c + (int64_t)i * r.c_stride + g;
    const T x0 = ((const T*)r.x)[(int64_t)i * r.x_stride + ch], t0 = ((const T*)r.dt)[(int64_t)i * r.dt_stride + ch];
    const T z0 = r.z ? ((const T*)r.z)[(int64_t)i * r.z_stride + ch] : x0;
    const float d = r.d ? r.d[ch] : 0.0f, bias = r.dt_bias ? r.dt_bias[ch] : 0.0f;
    T b0[S], c0[S];
#pragma unroll
    for (int e = 0; e < S; e++) b0[e] = pb[e], c0[e] = pc[e];
    float k[NB][S];
#pragma unroll
    for (int j = 0; j < NB; j++) load_state<S>(r.a + (size_t)min(ch0 + 16 * j + lane / 4, r.channels - 1) * N + q * S, k[j]);
    const int slot = entry_slot(a.slots, a.n_slots, i, true, lane);
    if (slot == kSkip) return;
    T* const out = (T*)r.out + (int64_t)i * r.out_stride + ch;
    if (slot == kBad) {
        if (in) *out = (T)__builtin_nanf("");
        return;
    }
    float* const state = a.states + (size_t)slot * r.channels * N + q * S;
    float h[NB][S];
#pragma unroll
    for (int j = 0; j < NB; j++) load_state<S>(state + (size_t)min(ch0 + 16 * j + lane / 4, r.channels - 1) * N, h[j]);
    const float x = (float)x0, s = softplus((float)t0 + bias).s, u = s * x;
    float p[4] = {};
    const auto block = [&](auto J) {
        constexpr int j = J.value;
        if constexpr (j < NB) {
            const float sj = NB == 4 ? quad_lane<j>(s) : s, uj = NB == 4 ? quad_lane<j>(u) : u;
#pragma unroll
            for (int e = 0; e < S; e++) {
                h[j][e] = fmaf(power(sj, k[j][e] * kLog2e), h[j][e], uj * (float)b0[e]);
                p[j] = fmaf((float)c0[e], h[j][e], p[j]);
            }
        }
    };
    block(std::integral_constant<int, 0>()), block(std::integral_constant<int, 1>());
    block(std::integral_constant<int, 2>()), block(std::integral_constant<int, 3>());
    float y = fmaf(d, x, NB == 4 ? quad_sums(p, q) : quad_sum(p[0]));
    if (r.z) {
        const float z = (float)z0;
        y *= z * sigmoid(z);
    }
#pragma unroll
    for (int j = 0; j < NB; j++)
        if (ch0 + 16 * j + lane / 4 < r.channels) store_state<S>(state + (size_t)(ch0 + 16 * j + lane / 4) * N, h[j]);
    if (in) *out = (T)y;
}

// ---------------------------------------------------------------- sequences in pieces
//
// A sequence is cut into pieces of 64 tokens (32 where a state has many parts).  With h_p the state before piece p and S_p the sum of its
// time steps, the state after it is e^(S_p a) h_p + l_p, where l_p is what its tokens make of a state of zeros.  k_scan_pieces makes l_p and S_p
// of all pieces side by side; then each piece's first state is joined from those before it, and k_scan_run goes through the piece once more
// from there and writes the outputs.  Both go by the sequence's own tokens alone, so its bits do not depend on the call around it.

template <int S> constexpr int kPiece = S <= 4 ? 64 : 32;
constexpr int kSpan = 16;                  // tokens of a request: four a lane

// Sequence i's rows: cu[i] to cu[i + 1], within [0, rows].  With `ends` the rows before the first and behind the last one are
// sequences 0 and n + 1 of their own, which nothing belongs to.
struct Bounds {
    const int32_t* cu;
    uint32_t n, rows;
    bool ends;
    __device__ __forceinline__ uint32_t count() const { return ends ? n + 2 : n; }
    __device__ __forceinline__ uint32_t at(uint32_t j) const {
        if (ends) {
            if (j == 0) return 0;
            if (j == n + 2) return rows;
            j--;
        }
        return min((uint32_t)max(cu[j], 0), rows);
    }
};

// A piece: rows [t0, t0 + len) are number `index` of `count` pieces of sequence seq.  Sequence i's pieces
// have the slots from rows / P + i on (its first row's), so those of one are consecutive, those of the next begin after them, and
// rows / P + n slots are enough.  len is 0 in the slot of a sequence without rows (index 0, count 0) and in unused ones (index > 0).
// Row `begin` is the sequence's first one.
struct Piece {
    uint32_t seq, t0, len, index, count, begin;
};

template <int P>
__device__ __forceinline__ Piece piece_of(const Bounds& m, uint32_t slot) {
    uint32_t lo = 0, hi = m.count() - 1;       // the last sequence that starts at this slot or before
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (m.at(mid) / P + mid <= slot) lo = mid;
        else hi = mid - 1;
    }
    const uint32_t b = m.at(lo), e = max(m.at(lo + 1), b), first = b / P + lo;
    Piece k{lo, 0, 0, slot - first, (e - b + P - 1) / P, b};
    if (slot < first) k.index = ~0u, k.count = 0;          // (boundaries that decrease)
    if (k.index < k.count) {
        k.t0 = b + k.index * P;
        k.len = min(e - k.t0, (uint32_t)P);
    }
    return k;
}

// The place in ws of the first piece of sequence `seq`, whose first row is `begin`.  Only sequences of two pieces and more have places there, so
// where there are many sequences they are given out by rows alone: with more than P rows a sequence's two places for each P of them are as many
// as its pieces at least, from floor(2 begin / P) on, so those of sequences that follow each other do not meet and 2 rows / P are enough.
template <int P>
__device__ __forceinline__ uint32_t place_of(const ScanArgs& a, uint32_t begin, uint32_t seq) {
    return __builtin_amdgcn_readfirstlane(a.spread ? 2 * begin / P : begin / P + seq);      // (a wave has one sequence)
}

// Rows of B (or C) of a piece in LDS, as f32.
template <typename T, int N>
__device__ __forceinline__ void stage(float* to, const void* from, int64_t stride, uint32_t t0, uint32_t len, uint32_t g) {
    const T* const p = (const T*)from + (int64_t)t0 * stride + g * N;
    for (uint32_t e = threadIdx.x; e < len * N; e += kBlock) to[e] = (float)p[(e / N) * (uint32_t)stride + e % N];
}

// Of 16 tokens in a row, those that are this lane's (4 g + q) of one array.  Tokens past the piece are its last one again.
template <typename T>
struct Tokens {
    T v[kSpan / 4];
};

template <typename T>
__device__ __forceinline__ Tokens<T> fetch(const T* p, uint32_t stride, uint32_t t, uint32_t len, int q) {
    Tokens<T> k;
#pragma unroll
    for (int g = 0; g < kSpan / 4; g++) k.v[g] = p[min(t + 4 * g + q, len - 1) * stride];
    return k;
}

template <int S>
__device__ __forceinline__ void parts(const float* p, float (&v)[S]) {
    load_state<S>(p, v);
}

// The state after `upto` pieces from h, by what k_scan_pieces left of them.
template <int S>
__device__ __forceinline__ void join(const ScanArgs& a, const Channel<S>& k, uint32_t ch, int q, uint32_t first, uint32_t upto, float (&h)[S]) {
    const float* const sums = a.ws + (size_t)a.pieces * a.r.channels * (4 * S);
#pragma unroll 4
    for (uint32_t p = 0; p < upto; p++) {
        const size_t at = (size_t)(first + p) * a.r.channels + ch;
        float l[S];
        load_state<S>(a.ws + at * (4 * S) + q * S, l);
        const float s = sums[at];
#pragma unroll
        for (int e = 0; e < S; e++) h[e] = fmaf(power(s, k.a2[e]), h[e], l[e]);
    }
}

template <int S>
__device__ __forceinline__ void first_state(const ScanArgs& a, int slot, uint32_t ch, int q, float (&h)[S]) {
    if (a.in) {
        load_state<S>(a.in + ((size_t)slot * a.r.channels + ch) * (4 * S) + q * S, h);
    } else {
#pragma unroll
        for (int e = 0; e < S; e++) h[e] = 0.0f;
    }
}

// l_p and S_p of a piece that is not its sequence's last.  In the last one's place of ws goes the sequence's first state, which
// k_scan_run may otherwise find overwritten by the last state (the pools may be one).
template <typename T, int S>
__global__ __launch_bounds__(kBlock) void k_scan_pieces(ScanArgs a) {
    constexpr int N = 4 * S, P = kPiece<S>;
    __shared__ __attribute__((aligned(16))) float sb[P * N];
    const redukt_scan_rows& r = a.r;
    const int lane = threadIdx.x % kOpWave, q = lane % 4;
    const uint32_t blocks = (r.channels + kBlockCh - 1) / kBlockCh, ch0 = blockIdx.x % blocks * kBlockCh, slot = blockIdx.x / blocks;
    const Piece m = piece_of<P>(Bounds{a.cu, a.n, r.rows, false}, slot);
    if (m.len == 0 || m.count == 1) return;
    const int st = entry_slot(a.slots, a.n_slots, m.seq, a.states != nullptr, lane);
    if (st < 0) return;
    const uint32_t at = ch0 + threadIdx.x / 4;
    const bool in = at < r.channels;
    const uint32_t ch = in ? at : r.channels - 1;
    const size_t place = (size_t)(place_of<P>(a, m.begin, m.seq) + m.index) * r.channels + ch;
    float* const mine = a.ws + place * N + q * S;
    float h[S];
    if (m.index + 1 == m.count) {
        first_state<S>(a, st, ch, q, h);
        if (in) store_state<S>(mine, h);
        return;
    }
    stage<T, N>(sb, r.b, r.b_stride, m.t0, m.len, ch0 / (r.channels / r.groups));
    const Channel<S> k = channel_of<S>(r, ch, q);
    const T* const px = (const T*)r.x + (int64_t)m.t0 * r.x_stride + ch;
    const T* const pt = (const T*)r.dt + (int64_t)m.t0 * r.dt_stride + ch;
    const uint32_t xs = (uint32_t)r.x_stride, ts = (uint32_t)r.dt_stride;
    Tokens<T> x = fetch(px, xs, 0, P, q), t = fetch(pt, ts, 0, P, q);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < S; e++) h[e] = 0.0f;
    float sum = 0.0f;
    for (int t0 = 0; t0 < P; t0 += kSpan) {
        const Tokens<T> x1 = x, t1 = t;
        if (t0 + kSpan < P) x = fetch(px, xs, t0 + kSpan, P, q), t = fetch(pt, ts, t0 + kSpan, P, q);
#pragma unroll
        for (int g = 0; g < kSpan / 4; g++) {
            const float s = softplus((float)t1.v[g] + k.bias).s, u = s * (float)x1.v[g];
            sum += s;
            const auto token = [&](auto J) {
                const float sj = quad_lane<J.value>(s), uj = quad_lane<J.value>(u);
                float b[S];
                parts<S>(sb + (t0 + 4 * g + J.value) * N + q * S, b);
#pragma unroll
                for (int e = 0; e < S; e++) h[e] = fmaf(power(sj, k.a2[e]), h[e], uj * b[e]);
            };
            token(std::integral_constant<int, 0>()), token(std::integral_constant<int, 1>());
            token(std::integral_constant<int, 2>()), token(std::integral_constant<int, 3>());
        }
    }
    sum = quad_sum(sum);
    if (!in) return;
    store_state<S>(mine, h);
    if (q == 0) a.ws[(size_t)a.pieces * r.channels * N + place] = sum;
}

// The first states of all pieces of a sequence, in the places of what k_scan_pieces left there: a quad a channel.  A workgroup is one
// wave: what it waits for is the way through its CU (8,192 tokens of 1,536 channels, gradients: 20 us with four waves).
constexpr int kJoinCh = 16;
template <int S>
__global__ __launch_bounds__(kOpWave) void k_scan_join(ScanArgs a) {
    constexpr int N = 4 * S, P = kPiece<S>;
    const redukt_scan_rows& r = a.r;
    const int lane = threadIdx.x, q = lane % 4;
    const uint32_t blocks = (r.channels + kJoinCh - 1) / kJoinCh, i = blockIdx.x / blocks;
    const uint32_t ch = blockIdx.x % blocks * kJoinCh + lane / 4;
    const Bounds m{a.cu, a.n, r.rows, false};
    const uint32_t b = m.at(i), e = max(m.at(i + 1), b), count = (e - b + P - 1) / P, first = place_of<P>(a, b, i);
    if (count < 2) return;
    const int st = entry_slot(a.slots, a.n_slots, i, a.states != nullptr, lane);
    if (st < 0 || ch >= r.channels) return;
    const Channel<S> k = channel_of<S>(r, ch, q);
    const float* const sums = a.ws + (size_t)a.pieces * r.channels * N;
    float h[S];
    first_state<S>(a, st, ch, q, h);
    constexpr int kAhead = 8;
    for (uint32_t p0 = 0; p0 < count; p0 += kAhead) {
        float l[kAhead][S], s[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) {     // (the last piece's are not needed, and neither is what lies behind it)
            const size_t at = (size_t)(first + min(p0 + u, count - 1)) * r.channels + ch;
            load_state<S>(a.ws + at * N + q * S, l[u]);
            s[u] = sums[at];
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (p0 + u >= count) break;
            store_state<S>(a.ws + ((size_t)(first + p0 + u) * r.channels + ch) * N + q * S, h);
#pragma unroll
            for (int v = 0; v < S; v++) h[v] = fmaf(power(s[u], k.a2[v]), h[v], l[u][v]);
        }
    }
}

// Outputs of a piece, and the last state from the last one.
template <typename T, int S>
__global__ __launch_bounds__(kBlock) void k_scan_run(ScanArgs a) {
    constexpr int N = 4 * S, P = kPiece<S>;
    __shared__ __attribute__((aligned(16))) float sb[P * N], sc[P * N];
    const redukt_scan_rows& r = a.r;
    const int lane = threadIdx.x % kOpWave, q = lane % 4;
    const uint32_t blocks = (r.channels + kBlockCh - 1) / kBlockCh, ch0 = blockIdx.x % blocks * kBlockCh, slot = blockIdx.x / blocks;
    const Piece m = piece_of<P>(Bounds{a.cu, a.n, r.rows, false}, slot);
    if (m.len == 0 && (m.index || m.count || !a.states)) return;
    const int st = entry_slot(a.slots, a.n_slots, m.seq, a.states != nullptr, lane);
    if (st == kSkip) return;
    const uint32_t at = ch0 + threadIdx.x / 4;
    const bool in = at < r.channels;
    const uint32_t ch = in ? at : r.channels - 1;
    T* const po = (T*)r.out + (int64_t)m.t0 * r.out_stride + ch;
    const uint32_t os = (uint32_t)r.out_stride;
    if (st == kBad) {
        for (uint32_t t = q; in && t < m.len; t += 4) po[t * os] = (T)__builtin_nanf("");
        return;
    }
    float h[S];
    if (m.len == 0) {                          // a sequence without rows hands its first state on
        first_state<S>(a, st, ch, q, h);
        if (in) store_state<S>(a.states + ((size_t)st * r.channels + ch) * N + q * S, h);
        return;
    }
    const T* const px = (const T*)r.x + (int64_t)m.t0 * r.x_stride + ch;
    const T* const pt = (const T*)r.dt + (int64_t)m.t0 * r.dt_stride + ch;
    const T* const pz = r.z ? (const T*)r.z + (int64_t)m.t0 * r.z_stride + ch : px;
    const uint32_t xs = (uint32_t)r.x_stride, ts = (uint32_t)r.dt_stride, zs = r.z ? (uint32_t)r.z_stride : xs;
    Tokens<T> x = fetch(px, xs, 0, m.len, q), t = fetch(pt, ts, 0, m.len, q), z = fetch(pz, zs, 0, m.len, q);
    const uint32_t gr = ch0 / (r.channels / r.groups);
    stage<T, N>(sb, r.b, r.b_stride, m.t0, m.len, gr);
    stage<T, N>(sc, r.c, r.c_stride, m.t0, m.len, gr);
    const Channel<S> k = channel_of<S>(r, ch, q);
    if (m.count == 1) {
        first_state<S>(a, st, ch, q, h);
    } else {
        const uint32_t first = place_of<P>(a, m.begin, m.seq);
        load_state<S>(a.ws + ((size_t)(first + (a.joined ? m.index : m.count - 1)) * r.channels + ch) * N + q * S, h);
        if (!a.joined) join<S>(a, k, ch, q, first, m.index, h);
    }
    __syncthreads();
    for (uint32_t t0 = 0; t0 < m.len; t0 += kSpan) {
        const Tokens<T> x1 = x, t1 = t, z1 = z;
        if (t0 + kSpan < m.len) {
            x = fetch(px, xs, t0 + kSpan, m.len, q);
            t = fetch(pt, ts, t0 + kSpan, m.len, q);
            z = fetch(pz, zs, t0 + kSpan, m.len, q);
        }
        const auto span = [&](auto WHOLE) {
#pragma unroll
            for (int g = 0; g < kSpan / 4; g++) {
                const float xv = (float)x1.v[g], s = softplus((float)t1.v[g] + k.bias).s, u = s * xv;
                float p[4];
                const auto token = [&](auto J) {
                    p[J.value] = 0.0f;
                    if (!WHOLE.value && t0 + 4 * g + J.value >= m.len) return;
                    const float sj = quad_lane<J.value>(s), uj = quad_lane<J.value>(u);
                    float b[S], c[S];
                    parts<S>(sb + (t0 + 4 * g + J.value) * N + q * S, b);
                    parts<S>(sc + (t0 + 4 * g + J.value) * N + q * S, c);
#pragma unroll
                    for (int e = 0; e < S; e++) {
                        h[e] = fmaf(power(sj, k.a2[e]), h[e], uj * b[e]);
                        p[J.value] = fmaf(c[e], h[e], p[J.value]);
                    }
                };
                token(std::integral_constant<int, 0>()), token(std::integral_constant<int, 1>());
                token(std::integral_constant<int, 2>()), token(std::integral_constant<int, 3>());
                float y = fmaf(k.d, xv, quad_sums(p, q));
                if (r.z) {
                    const float zv = (float)z1.v[g];
                    y *= zv * sigmoid(zv);
                }
                const uint32_t to = t0 + 4 * g + q;
                if (in && (WHOLE.value || to < m.len)) po[to * os] = (T)y;
            }
        };
        if (t0 + kSpan <= m.len) span(std::true_type());
        else span(std::false_type());
    }
    if (a.states && in && m.index + 1 == m.count) store_state<S>(a.states + ((size_t)st * r.channels + ch) * N + q * S, h);
}

// ---------------------------------------------------------------- gradients
//
// With dy = dout silu(z) and G_t the gradient of the state after token t,
//     G_t = dy_t C_t + e^(s_(t+1) a) G_(t+1)          dC_t = sum over channels of dy h_t       dB_t = sum over channels of G s x
//     dx = s sum_n G B + dy d                         ds = sum_n G (a e^(s a) h_(t-1) + x B)   da = sum over tokens of G s e^(s a) h_(t-1)
//     dz = dout y silu'(z),  ddt = ds softplus'.
// What goes back over a piece's first token is R = e^(s_t0 a) G_t0, and R_p = r_p + e^(S_p a) R_(p+1), where r_p comes of the piece alone:
// the same joining as of the states, from the other end.  k_scan_grad_pieces makes l_p, S_p and r_p, going forward (r_p = sum of
// dy_t C_t e^((s_t0 + ... + s_t) a)).  k_scan_grad_run then goes through a piece forward, keeping the states every L tokens, and backward over
// these, L at a time: once more forward with the powers and e^(s a) h_(t-1) of all L tokens in registers, then backward.
//
// Bound by the vector unit as well: k_scan_grad_run issues 135 vector instructions for a token of 16 channels of 16 parts, a fifth of them to sum dB
// and dC over channels.  8,192 tokens of 1,536 channels in bf16: pieces 71 us, joining 18, k_scan_grad_run 236, the sums over workgroups and
// pieces 9 (the bytes alone would take 35).

// Pieces are as long as scan_chunk's, or (SHORT) half of that in calls too small to fill the device with those.
template <int S, bool SHORT> constexpr int kGradPiece = SHORT ? kPiece<S> / 2 : kPiece<S>;

struct GradArgs {
    ScanArgs a;                // in: the first states; states: null
    redukt_scan_grads g;
    const float* dlast;        // null: zeros
    float* dfirst;             // null: not wanted
    float* back;               // r_p [places][channels][n] (joined: R_(p+1))
    float* bc;                 // dB, dC of a workgroup's channels: [parts][rows][2 n]
    float* tok;                // da, then dd and ddt_bias of a piece: [slots][channels][n], [slots][channels][2]
    uint32_t slots;            // of pieces
    uint32_t per;              // blocks of 64 channels of a workgroup
    uint32_t parts, parts_g;   // workgroups along the channels, of all groups and of one
};

template <typename T, int S, bool SHORT>
__global__ __launch_bounds__(kBlock) void k_scan_grad_pieces(GradArgs ga) {
    constexpr int N = 4 * S, P = kGradPiece<S, SHORT>;
    __shared__ __attribute__((aligned(16))) float sb[P * N], sc[P * N];
    const ScanArgs& a = ga.a;
    const redukt_scan_rows& r = a.r;
    const int lane = threadIdx.x % kOpWave, q = lane % 4;
    const uint32_t blocks = (r.channels + kBlockCh - 1) / kBlockCh, ch0 = blockIdx.x % blocks * kBlockCh, slot = blockIdx.x / blocks;
    const Piece m = piece_of<P>(Bounds{a.cu, a.n, r.rows, true}, slot);
    if (m.len == 0 || m.count == 1 || m.seq == 0 || m.seq == a.n + 1) return;
    const uint32_t at = ch0 + threadIdx.x / 4;
    const bool in = at < r.channels;
    const uint32_t ch = in ? at : r.channels - 1;
    const uint32_t gr = ch0 / (r.channels / r.groups);
    stage<T, N>(sb, r.b, r.b_stride, m.t0, m.len, gr);
    stage<T, N>(sc, r.c, r.c_stride, m.t0, m.len, gr);
    const Channel<S> k = channel_of<S>(r, ch, q);
    const T* const px = (const T*)r.x + (int64_t)m.t0 * r.x_stride + ch;
    const T* const pt = (const T*)r.dt + (int64_t)m.t0 * r.dt_stride + ch;
    const T* const pd = (const T*)ga.g.dout + (int64_t)m.t0 * ga.g.dout_stride + ch;
    const T* const pz = r.z ? (const T*)r.z + (int64_t)m.t0 * r.z_stride + ch : px;
    const uint32_t xs = (uint32_t)r.x_stride, ts = (uint32_t)r.dt_stride, ds = (uint32_t)ga.g.dout_stride, zs = r.z ? (uint32_t)r.z_stride : xs;
    __syncthreads();
    float h[S], w[S], back[S];
#pragma unroll
    for (int e = 0; e < S; e++) h[e] = 0.0f, w[e] = 1.0f, back[e] = 0.0f;
    float sum = 0.0f;
    for (uint32_t t0 = 0; t0 < m.len; t0 += kSpan) {
        const Tokens<T> x = fetch(px, xs, t0, m.len, q), t = fetch(pt, ts, t0, m.len, q), z = fetch(pz, zs, t0, m.len, q),
                        d = fetch(pd, ds, t0, m.len, q);
#pragma unroll
        for (int g = 0; g < kSpan / 4; g++) {
            if (t0 + 4 * g >= m.len) break;
            const float s = softplus((float)t.v[g] + k.bias).s, u = s * (float)x.v[g];
            float dy = (float)d.v[g];
            if (r.z) {
                const float zv = (float)z.v[g];
                dy *= zv * sigmoid(zv);
            }
            if (t0 + 4 * g + q < m.len) sum += s;
            const auto token = [&](auto J) {
                const uint32_t tok = t0 + 4 * g + J.value;
                if (tok >= m.len) return;
                const float sj = quad_lane<J.value>(s), uj = quad_lane<J.value>(u), dj = quad_lane<J.value>(dy);
                float b[S], c[S];
                parts<S>(sb + tok * N + q * S, b);
                parts<S>(sc + tok * N + q * S, c);
#pragma unroll
                for (int e = 0; e < S; e++) {
                    const float f = power(sj, k.a2[e]);
                    h[e] = fmaf(f, h[e], uj * b[e]);
                    w[e] *= f;
                    back[e] = fmaf(w[e], dj * c[e], back[e]);
                }
            };
            token(std::integral_constant<int, 0>()), token(std::integral_constant<int, 1>());
            token(std::integral_constant<int, 2>()), token(std::integral_constant<int, 3>());
        }
    }
    sum = quad_sum(sum);
    if (!in) return;
    const size_t place = (size_t)(place_of<P>(a, m.begin, m.seq) + m.index) * r.channels + ch;
    store_state<S>(a.ws + place * N + q * S, h);
    store_state<S>(ga.back + place * N + q * S, back);
    if (q == 0) a.ws[(size_t)a.pieces * r.channels * N + place] = sum;
}

// R_(p+1) of piece p, from the pieces behind it.
template <int S>
__device__ __forceinline__ void join_back(const GradArgs& g, const Channel<S>& k, uint32_t ch, int q, const Piece& m, uint32_t first, float (&R)[S]) {
    const redukt_scan_rows& r = g.a.r;
    const float* const sums = g.a.ws + (size_t)g.a.pieces * r.channels * (4 * S);
#pragma unroll 4
    for (uint32_t p = m.count - 1; p > m.index; p--) {
        const size_t at = (size_t)(first + p) * r.channels + ch;
        float l[S];
        load_state<S>(g.back + at * (4 * S) + q * S, l);
        const float s = sums[at];
#pragma unroll
        for (int e = 0; e < S; e++) R[e] = fmaf(power(s, k.a2[e]), R[e], l[e]);
    }
}

template <int S>
__device__ __forceinline__ void state_or_zeros(const float* pool, uint32_t seq, uint32_t channels, uint32_t ch, int q, float (&h)[S]) {
#pragma unroll
    for (int e = 0; e < S; e++) h[e] = 0.0f;
    if (pool) load_state<S>(pool + ((size_t)seq * channels + ch) * (4 * S) + q * S, h);
}

// The first states of all pieces of a sequence (blockIdx.y 0), or what comes back behind them (1), in place.
template <int S, bool SHORT>
__global__ __launch_bounds__(kOpWave) void k_scan_grad_join(GradArgs ga) {
    constexpr int N = 4 * S, P = kGradPiece<S, SHORT>;
    const redukt_scan_rows& r = ga.a.r;
    const int lane = threadIdx.x, q = lane % 4;
    const uint32_t blocks = (r.channels + kJoinCh - 1) / kJoinCh, i = blockIdx.x / blocks + 1;
    const uint32_t ch = blockIdx.x % blocks * kJoinCh + lane / 4;
    const Bounds m{ga.a.cu, ga.a.n, r.rows, true};
    const uint32_t b = m.at(i), e = max(m.at(i + 1), b), count = (e - b + P - 1) / P, first = place_of<P>(ga.a, b, i);
    if (count < 2 || ch >= r.channels) return;
    const bool backward = blockIdx.y;
    const Channel<S> k = channel_of<S>(r, ch, q);
    const float* const sums = ga.a.ws + (size_t)ga.a.pieces * r.channels * N;
    float* const pool = backward ? ga.back : ga.a.ws;
    float h[S];
    state_or_zeros<S>(backward ? ga.dlast : ga.a.in, i - 1, r.channels, ch, q, h);
    constexpr int kAhead = S <= 4 ? 16 : 4;
    const auto piece = [&](uint32_t p) { return (size_t)(first + (backward ? count - 1 - p : p)) * r.channels + ch; };
    for (uint32_t p0 = 0; p0 < count; p0 += kAhead) {
        float l[kAhead][S], s[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const size_t at = piece(min(p0 + u, count - 1));
            load_state<S>(pool + at * N + q * S, l[u]);
            s[u] = sums[at];
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (p0 + u >= count) break;
            store_state<S>(pool + piece(p0 + u) * N + q * S, h);
#pragma unroll
            for (int v = 0; v < S; v++) h[v] = fmaf(power(s[u], k.a2[v]), h[v], l[u][v]);
        }
    }
}

// (A bit cast straight from a vector's element reads the first one, whichever is meant: the words are copied first.)
template <typename X>
__device__ __forceinline__ float both(const X& x) {
    const uint32_t lo = x[0], hi = x[1];
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

template <int CTRL>
__device__ __forceinline__ float row_move(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
constexpr int kRor8 = 0x128, kShl4 = 0x104;

// v[i] and v[i + S], i < S, summed over the wave's 16 channels (a quad's place in the sums is one channel), and put into to[q S + ...] and
// to[N + q S + ...].  Each exchange adds two halves of the wave and leaves each half with half of the values: lanes 32 apart share out the
// two kinds, lanes 16 and then 8 apart the parts; what is left is added over lanes 4 apart, and the lower of them writes.
template <int S>
__device__ __forceinline__ void sum_channels(float (&v)[2 * S], float* to, int lane, bool add) {
    constexpr int N = 4 * S;
    const int q = lane % 4;
    float w[S];
#pragma unroll
    for (int i = 0; i < S; i++) {
        const auto x = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v[i]), __builtin_bit_cast(uint32_t, v[i + S]), false, false);
        w[i] = both(x);
    }
    float y[S / 2];
#pragma unroll
    for (int i = 0; i < S / 2; i++) {
        const auto x = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, w[i]), __builtin_bit_cast(uint32_t, w[i + S / 2]), false, false);
        y[i] = both(x);
    }
    constexpr int R = S >= 4 ? S / 4 : 1;
    const bool high = lane & 8;
    float z[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        if constexpr (S >= 4) z[i] = (high ? y[i + R] : y[i]) + row_move<kRor8>(high ? y[i] : y[i + R]);
        else z[i] = y[i] + row_move<kRor8>(y[i]);
        z[i] += row_move<kShl4>(z[i]);
    }
    if (lane & 4 || (S == 2 && high)) return;
    float* const p = to + (lane & 32 ? N : 0) + q * S + (lane & 16 ? S / 2 : 0) + (S >= 4 && high ? R : 0);
#pragma unroll
    for (int i = 0; i < R; i++) p[i] = add ? p[i] + z[i] : z[i];
}

// L.  (With 16 of a state of 16 parts a wave has the registers of a SIMD to itself: 8,192 tokens of 1,536 channels 467 us, with 8 358.)
constexpr int kBack = 8;

template <typename T, int S, bool SHORT>
__global__ __launch_bounds__(kBlock) void k_scan_grad_run(GradArgs ga) {
    constexpr int N = 4 * S, P = kGradPiece<S, SHORT>, L = kBack, W = kBlock / kOpWave;
    __shared__ __attribute__((aligned(16))) float sb[P * N], sc[P * N], kept[W][P / L][kOpWave * S], sums[W][P * 2 * N];
    const ScanArgs& a = ga.a;
    const redukt_scan_rows& r = a.r;
    const redukt_scan_grads& d = ga.g;
    const int lane = threadIdx.x % kOpWave, q = lane % 4, wave = threadIdx.x / kOpWave;
    const uint32_t part = blockIdx.x % ga.parts, slot = blockIdx.x / ga.parts, gr = part / ga.parts_g;
    const uint32_t per_g = r.channels / r.groups, blocks_g = (per_g + kBlockCh - 1) / kBlockCh;
    const uint32_t block0 = part % ga.parts_g * ga.per, block1 = min(block0 + ga.per, blocks_g);
    const Piece m = piece_of<P>(Bounds{a.cu, a.n, r.rows, true}, slot);
    const bool none = m.len == 0 || m.seq == 0 || m.seq == a.n + 1;
    const uint32_t first = place_of<P>(a, m.begin, m.seq);
    float* const tok_a = ga.tok;
    float* const tok_d = ga.tok + (size_t)ga.slots * r.channels * N;
    if (!none) {
        stage<T, N>(sb, r.b, r.b_stride, m.t0, m.len, gr);
        stage<T, N>(sc, r.c, r.c_stride, m.t0, m.len, gr);
        __syncthreads();
    }
    for (uint32_t block = block0; block < block1; block++) {
        const uint32_t at = block * kBlockCh + threadIdx.x / 4;
        const bool in = at < per_g;
        const uint32_t ch = gr * per_g + (in ? at : per_g - 1);
        const size_t mine = (size_t)slot * r.channels + ch;
        float G[S], da[S], dd = 0.0f, dbias = 0.0f;
#pragma unroll
        for (int e = 0; e < S; e++) da[e] = 0.0f;
        T* const qx = (T*)d.dx + (int64_t)m.t0 * d.dx_stride + ch;
        T* const qt = (T*)d.ddt + (int64_t)m.t0 * d.ddt_stride + ch;
        T* const qz = (T*)d.dz + (int64_t)m.t0 * d.dz_stride + ch;
        const uint32_t dxs = (uint32_t)d.dx_stride, dts = (uint32_t)d.ddt_stride, dzs = (uint32_t)d.dz_stride;
        if (none) {
            for (uint32_t t = q; in && t < m.len; t += 4) {
                qx[t * dxs] = (T)0.0f;
                qt[t * dts] = (T)0.0f;
                if (r.z) qz[t * dzs] = (T)0.0f;
            }
            // (a sequence without rows hands the gradient of its last state back)
            if (in && ga.dfirst && m.index == 0 && m.count == 0 && m.seq > 0 && m.seq <= a.n) {
                state_or_zeros<S>(ga.dlast, m.seq - 1, r.channels, ch, q, G);
                store_state<S>(ga.dfirst + ((size_t)(m.seq - 1) * r.channels + ch) * N + q * S, G);
            }
        } else {
            const Channel<S> k = channel_of<S>(r, ch, q);
            float h[S];
            if (a.joined && m.count > 1) {
                const size_t place = (size_t)(first + m.index) * r.channels + ch;
                load_state<S>(a.ws + place * N + q * S, h);
                load_state<S>(ga.back + place * N + q * S, G);
            } else {
                state_or_zeros<S>(a.in, m.seq - 1, r.channels, ch, q, h);
                state_or_zeros<S>(ga.dlast, m.seq - 1, r.channels, ch, q, G);
                join<S>(a, k, ch, q, first, m.index, h);
                join_back<S>(ga, k, ch, q, m, first, G);
            }
            if (!in) {
#pragma unroll
                for (int e = 0; e < S; e++) G[e] = 0.0f;
            }
            const T* const px = (const T*)r.x + (int64_t)m.t0 * r.x_stride + ch;
            const T* const pt = (const T*)r.dt + (int64_t)m.t0 * r.dt_stride + ch;
            const T* const pd = (const T*)d.dout + (int64_t)m.t0 * d.dout_stride + ch;
            const T* const pz = r.z ? (const T*)r.z + (int64_t)m.t0 * r.z_stride + ch : px;
            const uint32_t xs = (uint32_t)r.x_stride, ts = (uint32_t)r.dt_stride, ds = (uint32_t)d.dout_stride, zs = r.z ? (uint32_t)r.z_stride : xs;
            const uint32_t back = (m.len + L - 1) / L;
            float* const keep = &kept[wave][0][lane * S];
            // The states before each L tokens but the first ones.
            store_state<S>(keep, h);
            for (uint32_t l = 0; l + 1 < back; l++) {
                float s[L / 4], u[L / 4];
#pragma unroll
                for (int g = 0; g < L / 4; g++) {
                    const uint32_t t = l * L + 4 * g + q;
                    s[g] = softplus((float)pt[t * ts] + k.bias).s;
                    u[g] = s[g] * (float)px[t * xs];
                }
#pragma unroll
                for (int g = 0; g < L / 4; g++) {
                    const auto token = [&](auto J) {
                        const float sj = quad_lane<J.value>(s[g]), uj = quad_lane<J.value>(u[g]);
                        float b[S];
                        parts<S>(sb + (l * L + 4 * g + J.value) * N + q * S, b);
#pragma unroll
                        for (int e = 0; e < S; e++) h[e] = fmaf(power(sj, k.a2[e]), h[e], uj * b[e]);
                    };
                    token(std::integral_constant<int, 0>()), token(std::integral_constant<int, 1>());
                    token(std::integral_constant<int, 2>()), token(std::integral_constant<int, 3>());
                }
                store_state<S>(keep + (l + 1) * (kOpWave * S), h);
            }
            for (uint32_t l = back; l-- > 0;) {
                const uint32_t t0 = l * L;
                const auto span = [&](auto WHOLE) {
                    float s[L / 4], slope[L / 4], x[L / 4], u[L / 4], dy[L / 4], f[L][S], w[L][S];
                    load_state<S>(keep + l * (kOpWave * S), h);
                    T tx[L / 4], tt[L / 4], tz[L / 4], td[L / 4];
#pragma unroll
                    for (int g = 0; g < L / 4; g++) {
                        const uint32_t t = WHOLE.value ? t0 + 4 * g + q : min(t0 + 4 * g + q, m.len - 1);
                        tx[g] = px[t * xs], tt[g] = pt[t * ts], tz[g] = pz[t * zs], td[g] = pd[t * ds];
                    }
#pragma unroll
                    for (int g = 0; g < L / 4; g++) {
                        const uint32_t t = t0 + 4 * g + q;
                        const bool live = WHOLE.value || t < m.len;
                        const Step st = softplus((float)tt[g] + k.bias);
                        s[g] = st.s, slope[g] = st.slope, x[g] = (float)tx[g], u[g] = s[g] * x[g];
                        float p[4];
                        const auto token = [&](auto J) {
                            p[J.value] = 0.0f;
                            if (!WHOLE.value && t0 + 4 * g + J.value >= m.len) return;
                            const float sj = quad_lane<J.value>(s[g]), uj = quad_lane<J.value>(u[g]);
                            float b[S], c[S];
                            parts<S>(sb + (t0 + 4 * g + J.value) * N + q * S, b);
                            parts<S>(sc + (t0 + 4 * g + J.value) * N + q * S, c);
#pragma unroll
                            for (int e = 0; e < S; e++) {
                                f[4 * g + J.value][e] = power(sj, k.a2[e]);
                                w[4 * g + J.value][e] = f[4 * g + J.value][e] * h[e];
                                h[e] = fmaf(uj, b[e], w[4 * g + J.value][e]);
                                p[J.value] = fmaf(c[e], h[e], p[J.value]);
                            }
                        };
                        token(std::integral_constant<int, 0>()), token(std::integral_constant<int, 1>());
                        token(std::integral_constant<int, 2>()), token(std::integral_constant<int, 3>());
                        dy[g] = (float)td[g];
                        if (r.z) {
                            const float y = fmaf(k.d, x[g], quad_sums(p, q)), z = (float)tz[g], sg = sigmoid(z);
                            if (in && live) qz[t * dzs] = (T)(dy[g] * y * (sg * fmaf(z, 1.0f - sg, 1.0f)));
                            dy[g] *= z * sg;
                        }
                        if (!in) dy[g] = 0.0f;           // (and with it G: a lane without a channel of its own adds nothing to dB and dC)
                    }
#pragma unroll
                    for (int g = L / 4 - 1; g >= 0; g--) {
                        float p[4], k4[4];
                        const auto token = [&](auto J) {
                            constexpr int j = J.value;
                            p[j] = k4[j] = 0.0f;
                            if (!WHOLE.value && t0 + 4 * g + j >= m.len) return;
                            const float sj = quad_lane<j>(s[g]), uj = quad_lane<j>(u[g]), dj = quad_lane<j>(dy[g]);
                            float b[S], c[S], v[2 * S];
                            parts<S>(sb + (t0 + 4 * g + j) * N + q * S, b);
                            parts<S>(sc + (t0 + 4 * g + j) * N + q * S, c);
#pragma unroll
                            for (int e = 0; e < S; e++) {
                                const float wv = w[4 * g + j][e];
                                G[e] = fmaf(dj, c[e], G[e]);
                                v[e] = G[e] * uj;
                                v[S + e] = dj * fmaf(uj, b[e], wv);
                                p[j] = fmaf(G[e], b[e], p[j]);
                                const float gw = G[e] * wv;
                                k4[j] = fmaf(gw, k.a2[e], k4[j]);
                                da[e] = fmaf(gw, sj, da[e]);
                                G[e] *= f[4 * g + j][e];
                            }
                            sum_channels<S>(v, &sums[wave][(t0 + 4 * g + j) * 2 * N], lane, block != block0);
                        };
                        token(std::integral_constant<int, 3>()), token(std::integral_constant<int, 2>());
                        token(std::integral_constant<int, 1>()), token(std::integral_constant<int, 0>());
                        const float into = quad_sums(p, q), up = quad_sums(k4, q) * kLn2;
                        const uint32_t t = t0 + 4 * g + q;
                        const bool live = WHOLE.value || t < m.len;
                        const float ddt = fmaf(x[g], into, up) * slope[g];
                        if (live) dd = fmaf(dy[g], x[g], dd), dbias += ddt;
                        if (in && live) {
                            qx[t * dxs] = (T)fmaf(s[g], into, dy[g] * k.d);
                            qt[t * dts] = (T)ddt;
                        }
                    }
                };
                if (t0 + L <= m.len) span(std::true_type());
                else span(std::false_type());
            }
            if (in && ga.dfirst && m.index == 0) store_state<S>(ga.dfirst + ((size_t)(m.seq - 1) * r.channels + ch) * N + q * S, G);
            dd = quad_sum(dd), dbias = quad_sum(dbias);
        }
        if (in) {
            store_state<S>(tok_a + mine * N + q * S, da);
            if (q < 2) tok_d[mine * 2 + q] = q ? dbias : dd;
        }
    }
    if (m.len == 0) return;
    __syncthreads();
    float* const to = ga.bc + ((size_t)part * r.rows + m.t0) * (2 * N);
    for (uint32_t e = threadIdx.x; e < m.len * 2 * N; e += kBlock) {
        float v = 0.0f;
        if (!none) {
#pragma unroll
            for (int w = 0; w < W; w++) v += sums[w][e];
        }
        to[e] = v;
    }
}

// dB and dC of a token and group: the sum over the workgroups that had its channels.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_scan_grad_rows(GradArgs ga) {
    const redukt_scan_rows& r = ga.a.r;
    const uint64_t id = (uint64_t)blockIdx.x * kBlock + threadIdx.x;
    const uint32_t wide = 2 * r.n, row_wide = wide * r.groups, t = (uint32_t)(id / row_wide), e = (uint32_t)(id % row_wide);
    if (t >= r.rows) return;
    const uint32_t gr = e / wide, i = e % wide;
    float v = 0.0f;
#pragma unroll 4
    for (uint32_t p = 0; p < ga.parts_g; p++) v += ga.bc[((size_t)(gr * ga.parts_g + p) * r.rows + t) * wide + i];
    if (i < r.n) ((T*)ga.g.db)[(int64_t)t * ga.g.db_stride + gr * r.n + i] = (T)v;
    else ((T*)ga.g.dc)[(int64_t)t * ga.g.dc_stride + gr * r.n + i - r.n] = (T)v;
}

// da, dd and ddt_bias: the sums over the pieces, 64 columns a workgroup, every fourth piece a wave.
__global__ __launch_bounds__(kBlock) void k_scan_grad_columns(GradArgs ga) {
    __shared__ float half[kBlock];
    const redukt_scan_rows& r = ga.a.r;
    const uint64_t wide = (uint64_t)r.channels * r.n, narrow = (uint64_t)r.channels * 2;
    const uint64_t col = (uint64_t)blockIdx.x * kOpWave + threadIdx.x % kOpWave;
    const bool in = col < wide + narrow, of_a = col < wide;
    const float* const from = of_a ? ga.tok + col : ga.tok + (uint64_t)ga.slots * wide + (col - wide);
    const uint64_t step = of_a ? wide : narrow;
    float v = 0.0f;
    if (in) {
#pragma unroll 8
        for (uint32_t p = threadIdx.x / kOpWave; p < ga.slots; p += kBlock / kOpWave) v += from[p * step];
    }
    half[threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.x >= kOpWave || !in) return;
    v = half[threadIdx.x] + half[threadIdx.x + 64] + (half[threadIdx.x + 128] + half[threadIdx.x + 192]);
    if (of_a) {
        ga.g.da[col] = v;
    } else {
        const uint64_t c = col - wide;
        float* const to = c % 2 ? ga.g.ddt_bias : ga.g.dd;
        if (to) to[c / 2] = v;
    }
}

// ---------------------------------------------------------------- launches

#define SCAN_BY_N(T, n, fn, ...) \
    ((n) == 8    ? (const void*)fn<T, 2 __VA_OPT__(, ) __VA_ARGS__> \
     : (n) == 16 ? (const void*)fn<T, 4 __VA_OPT__(, ) __VA_ARGS__> \
     : (n) == 32 ? (const void*)fn<T, 8 __VA_OPT__(, ) __VA_ARGS__> \
                 : (const void*)fn<T, 16 __VA_OPT__(, ) __VA_ARGS__>)
#define SCAN_FN(r, fn, ...) \
    ((r).dtype == REDUKT_OP_BF16  ? SCAN_BY_N(__bf16, (r).n, fn __VA_OPT__(, ) __VA_ARGS__) \
     : (r).dtype == REDUKT_OP_F16 ? SCAN_BY_N(_Float16, (r).n, fn __VA_OPT__(, ) __VA_ARGS__) \
                                  : SCAN_BY_N(float, (r).n, fn __VA_OPT__(, ) __VA_ARGS__))

const void* join_fn(uint32_t n) {
    return n == 8 ? (const void*)k_scan_join<2> : n == 16 ? (const void*)k_scan_join<4> : n == 32 ? (const void*)k_scan_join<8> : (const void*)k_scan_join<16>;
}
template <bool SHORT>
const void* grad_join_fn(uint32_t n) {
    return n == 8    ? (const void*)k_scan_grad_join<2, SHORT>
           : n == 16 ? (const void*)k_scan_grad_join<4, SHORT>
           : n == 32 ? (const void*)k_scan_grad_join<8, SHORT>
                     : (const void*)k_scan_grad_join<16, SHORT>;
}

uint32_t piece_rows(uint32_t n) { return n <= 16 ? kPiece<4> : kPiece<16>; }

constexpr int64_t kMaxStride = 1 << 22;      // a piece's rows stay within 32-bit offsets
constexpr uint32_t kJoinHere = 32;           // pieces that each piece joins by itself

bool sizes_ok(const redukt_scan_rows* a) {
    return a && a->dtype <= REDUKT_OP_F32 && a->rows < (1u << 31) && a->channels > 0 && a->channels <= (1u << 20) && a->groups > 0 &&
           a->channels % a->groups == 0 && (a->groups == 1 || a->channels / a->groups % kBlockCh == 0) &&
           (a->n == 8 || a->n == 16 || a->n == 32 || a->n == 64);
}

// Whether p holds rows of `width` elements that a call may go through.
bool row_ok(const redukt_scan_rows* a, const void* p, int64_t stride, int64_t width) {
    return p && op_aligned(p, op_elem_bytes(a->dtype)) && (a->rows <= 1 || (stride >= width && stride <= kMaxStride));
}

bool rows_ok(const redukt_scan_rows* a, bool outputs) {
    const int64_t bc = (int64_t)a->groups * a->n;
    return row_ok(a, a->x, a->x_stride, a->channels) && row_ok(a, a->dt, a->dt_stride, a->channels) &&
           (!a->z || row_ok(a, a->z, a->z_stride, a->channels)) && row_ok(a, a->b, a->b_stride, bc) && row_ok(a, a->c, a->c_stride, bc) &&
           (!outputs || row_ok(a, a->out, a->out_stride, a->channels));
}

bool layer_ok(const redukt_scan_rows* a) {
    return a->a && op_aligned(a->a, 16) && op_aligned(a->d, 4) && op_aligned(a->dt_bias, 4);
}

// The rows with steps that are a row's width where there is one row only.
redukt_scan_rows stepped(redukt_scan_rows a) {
    if (a.rows == 1) {
        a.x_stride = a.dt_stride = a.z_stride = a.out_stride = a.channels;
        a.b_stride = a.c_stride = (int64_t)a.groups * a.n;
    }
    return a;
}

uint64_t chunk_pieces(const redukt_scan_rows& a, uint32_t n_seq) { return (uint64_t)a.rows / piece_rows(a.n) + n_seq; }
// Places in ws: by sequences, or by rows alone where that takes fewer (65,536 tokens of as many sequences, 1,536 channels of 16: 6.9 GB and 214 MB).
bool chunk_spread(const redukt_scan_rows& a, uint32_t n_seq) { return 2ull * a.rows / piece_rows(a.n) < chunk_pieces(a, n_seq); }
uint64_t chunk_places(const redukt_scan_rows& a, uint32_t n_seq) { return chunk_spread(a, n_seq) ? 2ull * a.rows / piece_rows(a.n) : chunk_pieces(a, n_seq); }
uint64_t chunk_floats(const redukt_scan_rows& a, uint32_t n_seq) { return chunk_places(a, n_seq) * a.channels * (a.n + 1ull); }

struct GradPlan {
    uint32_t piece, per, parts_g, parts;
    bool small, spread;
    uint64_t pieces, places, bc, tok, bytes;
};

GradPlan grad_plan(const redukt_scan_rows& a, uint32_t n_seq) {
    GradPlan p;
    const uint32_t blocks = (a.channels / a.groups + kBlockCh - 1) / kBlockCh;
    p.piece = piece_rows(a.n);
    // Shorter pieces while there are less than one and a half workgroups a CU of the others (us with short and long ones: 512 tokens of
    // 1,536 channels, 216 workgroups, 43.8 and 52.4; four segments of 1,030 in all and 768 channels, 240, 49.9 and 55.3; 2,048 of 768, 396, 73.9
    // and 74.0; the four segments of 1,536, 480, 79.0 and 70.8).
    p.small = ((uint64_t)a.rows / p.piece + n_seq) * blocks * a.groups < 384;
    if (p.small) p.piece /= 2;
    p.pieces = (uint64_t)a.rows / p.piece + n_seq + 2;
    // A workgroup takes up to four blocks of channels one after the other, whose dB and dC it adds, while there are workgroups enough without.
    p.per = 4;
    while (p.per > 1 && p.pieces * a.groups * ((blocks + p.per - 1) / p.per) < 1024) p.per /= 2;
    p.parts_g = (blocks + p.per - 1) / p.per;
    p.parts = p.parts_g * a.groups;
    p.spread = 2ull * a.rows / p.piece < p.pieces;
    p.places = p.spread ? 2ull * a.rows / p.piece : p.pieces;
    const uint64_t states = p.places * a.channels * a.n;
    p.bc = (uint64_t)p.parts * a.rows * 2 * a.n;
    p.tok = p.pieces * a.channels * (a.n + 2ull);
    p.bytes = 4 * (states + p.places * a.channels + states + p.tok + p.bc + 12);
    return p;
}

uint64_t round4(uint64_t floats) { return (floats + 3) / 4 * 4; }

}  // namespace
}  // namespace rdk

using namespace rdk;

extern "C" {

int32_t redukt_op_scan_step(const redukt_scan_rows* a, float* states, uint32_t n_slots, const int32_t* slots, void* stream) {
    if (!sizes_ok(a) || a->rows > kMaxOpRows) return BACKEND_INVALID_ARGUMENT;
    if (a->rows == 0) return BACKEND_OK;
    if (!rows_ok(a, true) || !layer_ok(a) || !states || !op_aligned(states, 16) || !op_aligned(slots, 4)) return BACKEND_INVALID_ARGUMENT;
    if (n_slots >= (1u << 31) || (!slots && a->rows > n_slots)) return BACKEND_INVALID_ARGUMENT;
    // (us with 16 and 64 channels a wave, 1,536 channels: 20 entries 5.6 and 6.1, 40 5.1 and 4.7, 400 22.8 and 16.3)
    const bool few = (uint64_t)a->rows * ((a->channels + 63) / 64) < 768;
    const uint32_t wide = few ? 16 : 64;
    const uint64_t grid = ((uint64_t)a->rows * ((a->channels + wide - 1) / wide) + 3) / 4;
    if (!op_grid_ok(grid, kBlock)) return BACKEND_INVALID_ARGUMENT;
    OpDevice dev(a->out);
    if (!dev.ok) return BACKEND_INVALID_ARGUMENT;
    ScanArgs k{stepped(*a), states, states, n_slots, slots, nullptr, a->rows, nullptr, 0, 0, 0};
    return op_launch(few ? SCAN_FN(k.r, k_scan_step, 1) : SCAN_FN(k.r, k_scan_step, 4), dim3((uint32_t)grid), dim3(kBlock), 0, stream, k);
}

uint64_t redukt_op_scan_chunk_workspace(const redukt_scan_rows* a, uint32_t n_seq) {
    if (!sizes_ok(a) || n_seq > kMaxOpRows || a->rows <= piece_rows(a->n)) return 0;
    return 4 * chunk_floats(*a, n_seq);
}

int32_t redukt_op_scan_chunk(const redukt_scan_rows* a, const int32_t* cu, uint32_t n_seq, const float* state_in, float* state_out,
                             uint32_t n_slots, const int32_t* slots, void* workspace, uint64_t workspace_bytes, void* stream) {
    if (!sizes_ok(a) || n_seq > kMaxOpRows) return BACKEND_INVALID_ARGUMENT;
    if (n_seq == 0) return BACKEND_OK;
    if ((a->rows && !rows_ok(a, true)) || !layer_ok(a) || !cu || !op_aligned(cu, 4) || !op_aligned(slots, 4) || !op_aligned(state_in, 16) ||
        !op_aligned(state_out, 16))
        return BACKEND_INVALID_ARGUMENT;
    if (state_in || state_out) {
        if (n_slots >= (1u << 31) || (!slots && n_seq > n_slots)) return BACKEND_INVALID_ARGUMENT;
        if (state_in && state_out && !apart(state_in, state_out, (size_t)n_slots * a->channels * a->n * 4)) return BACKEND_INVALID_ARGUMENT;
    } else if (slots) {
        return BACKEND_INVALID_ARGUMENT;
    }
    if (a->rows == 0 && !state_out) return BACKEND_OK;
    const uint64_t need = redukt_op_scan_chunk_workspace(a, n_seq);
    if (need && (!workspace || !op_aligned(workspace, 16) || workspace_bytes < need)) return BACKEND_INVALID_ARGUMENT;
    const uint64_t pieces = chunk_pieces(*a, n_seq), blocks = (a->channels + kBlockCh - 1) / kBlockCh, joins = (a->channels + kJoinCh - 1) / kJoinCh;
    if (!op_grid_ok(pieces * blocks, kBlock) || !op_grid_ok(n_seq * joins, kOpWave)) return BACKEND_INVALID_ARGUMENT;
    OpDevice dev(cu);
    if (!dev.ok) return BACKEND_INVALID_ARGUMENT;
    // No sequence has more pieces than the rows fill; few of them are joined by each piece itself, which saves a launch.
    ScanArgs k{stepped(*a), state_in, state_out, n_slots, slots, cu, n_seq, (float*)workspace, (uint32_t)chunk_places(*a, n_seq),
               a->rows > kJoinHere * piece_rows(a->n), chunk_spread(*a, n_seq)};
    const dim3 grid((uint32_t)(pieces * blocks));
    if (need) {
        int32_t rc = op_launch(SCAN_FN(k.r, k_scan_pieces), grid, dim3(kBlock), 0, stream, k);
        if (rc == BACKEND_OK && k.joined) rc = op_launch(join_fn(k.r.n), dim3((uint32_t)(n_seq * joins)), dim3(kOpWave), 0, stream, k);
        if (rc != BACKEND_OK) return rc;
    }
    return op_launch(SCAN_FN(k.r, k_scan_run), grid, dim3(kBlock), 0, stream, k);
}

uint64_t redukt_op_scan_grad_workspace(const redukt_scan_rows* a, uint32_t n_seq) {
    if (!sizes_ok(a) || n_seq > kMaxOpRows) return 0;
    return grad_plan(*a, n_seq).bytes;
}

int32_t redukt_op_scan_grad(const redukt_scan_rows* a, const redukt_scan_grads* g, const int32_t* cu, uint32_t n_seq, const float* state_in,
                            const float* dstate_out, float* dstate_in, void* workspace, uint64_t workspace_bytes, void* stream) {
    if (!sizes_ok(a) || !g || n_seq > kMaxOpRows) return BACKEND_INVALID_ARGUMENT;
    const int64_t bc = (int64_t)a->groups * a->n;
    if (a->rows && (!rows_ok(a, false) || !row_ok(a, g->dout, g->dout_stride, a->channels) || !row_ok(a, g->dx, g->dx_stride, a->channels) ||
                    !row_ok(a, g->ddt, g->ddt_stride, a->channels) || (a->z && !row_ok(a, g->dz, g->dz_stride, a->channels)) ||
                    !row_ok(a, g->db, g->db_stride, bc) || !row_ok(a, g->dc, g->dc_stride, bc)))
        return BACKEND_INVALID_ARGUMENT;
    if (!layer_ok(a) || !g->da || !op_aligned(g->da, 16) || !op_aligned(g->dd, 4) || !op_aligned(g->ddt_bias, 4) || !a->d != !g->dd ||
        !a->dt_bias != !g->ddt_bias || !a->z != !g->dz)
        return BACKEND_INVALID_ARGUMENT;
    if (!cu || !op_aligned(cu, 4) || !op_aligned(state_in, 16) || !op_aligned(dstate_out, 16) || !op_aligned(dstate_in, 16))
        return BACKEND_INVALID_ARGUMENT;
    const GradPlan p = grad_plan(*a, n_seq);
    if (!workspace || !op_aligned(workspace, 16) || workspace_bytes < p.bytes) return BACKEND_INVALID_ARGUMENT;
    const uint64_t blocks = (a->channels + kBlockCh - 1) / kBlockCh, joins = (a->channels + kJoinCh - 1) / kJoinCh, sums = ((uint64_t)a->rows * a->groups * 2 * a->n + kBlock - 1) / kBlock;
    const uint64_t columns = ((uint64_t)a->channels * (a->n + 2) + kOpWave - 1) / kOpWave;
    if (!op_grid_ok(p.pieces * blocks, kBlock) || !op_grid_ok(sums, kBlock) || !op_grid_ok(n_seq * joins, kOpWave))
        return BACKEND_INVALID_ARGUMENT;
    OpDevice dev(cu);
    if (!dev.ok) return BACKEND_INVALID_ARGUMENT;
    GradArgs k{};
    k.a = ScanArgs{stepped(*a), state_in, nullptr, n_seq, nullptr, cu, n_seq, (float*)workspace, (uint32_t)p.places, a->rows > kJoinHere * p.piece, p.spread};
    k.g = *g;
    if (a->rows == 1) {
        k.g.dout_stride = k.g.dx_stride = k.g.ddt_stride = k.g.dz_stride = a->channels;
        k.g.db_stride = k.g.dc_stride = bc;
    }
    k.dlast = dstate_out, k.dfirst = dstate_in;
    const uint64_t states = p.places * a->channels * a->n;
    k.back = k.a.ws + round4(states + p.places * a->channels);
    k.tok = k.back + states;
    k.bc = k.tok + round4(p.tok);
    k.slots = (uint32_t)p.pieces;
    k.per = p.per, k.parts = p.parts, k.parts_g = p.parts_g;
    if (a->rows > p.piece) {
        const void* const fn = p.small ? SCAN_FN(k.a.r, k_scan_grad_pieces, true) : SCAN_FN(k.a.r, k_scan_grad_pieces, false);
        int32_t rc = op_launch(fn, dim3((uint32_t)(p.pieces * blocks)), dim3(kBlock), 0, stream, k);
        if (rc == BACKEND_OK && k.a.joined && n_seq)
            rc = op_launch(p.small ? grad_join_fn<true>(a->n) : grad_join_fn<false>(a->n), dim3((uint32_t)(n_seq * joins), 2), dim3(kOpWave), 0, stream, k);
        if (rc != BACKEND_OK) return rc;
    }
    int32_t rc = op_launch(p.small ? SCAN_FN(k.a.r, k_scan_grad_run, true) : SCAN_FN(k.a.r, k_scan_grad_run, false), dim3((uint32_t)(p.pieces * p.parts)), dim3(kBlock), 0,
                           stream, k);
    if (rc == BACKEND_OK && a->rows) {
        const void* const fn = a->dtype == REDUKT_OP_BF16  ? (const void*)k_scan_grad_rows<__bf16>
                               : a->dtype == REDUKT_OP_F16 ? (const void*)k_scan_grad_rows<_Float16>
                                                           : (const void*)k_scan_grad_rows<float>;
        rc = op_launch(fn, dim3((uint32_t)sums), dim3(kBlock), 0, stream, k);
    }
    if (rc == BACKEND_OK) rc = op_launch((const void*)k_scan_grad_columns, dim3((uint32_t)columns), dim3(kBlock), 0, stream, k);
    return rc;
}

}  // extern "C"
