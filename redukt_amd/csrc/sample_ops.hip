// sample_ops.hip — tokens drawn from rows of logits (redukt_ops.h).
//
// Weights are whole numbers, W = e^((l - max) / T) in steps of 2^-42, so their sums are exact in 64-bit integers: they have no order,
// may be added by atomics, and the drawn token depends on nothing but the row.
#include <hip/hip_runtime.h>

#include "op_common.h"

#pragma clang fp contract(off)

namespace rdk {
namespace {

constexpr double kOne = 0x1p42;
constexpr double kLeast = -29.9;           // ln 2^-43 = -29.81: e to less than this is no whole step
constexpr uint32_t kBins = 2048;           // of (max - l) / T, linear, down to kLeast
constexpr uint32_t kList = 1024;           // elements that are put in order by comparing each with all
constexpr uint32_t kCoarse = 512;          // bins of the threads' largest logits
constexpr uint32_t kFewK = 512;            // top_k that the list takes in general
constexpr uint32_t kMaxVocab = 1u << 20;   // 2^20 weights of 2^42 stay below 2^63

// Logits' order as that of unsigned numbers.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);         // (-0 is 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float value_of(uint32_t key) { return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// Where the kept part of a row's order (larger values first, equal ones by index) ends: its last element.
struct Cut {
    uint32_t key, index;
    __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= index); }
};

struct SampleArgs {
    redukt_sample a;
    uint32_t aligned;          // rows begin on 16 bytes
};

// An element of the list: its place in the order of values as one word (the larger comes first), and its weight.
struct __attribute__((aligned(16))) Listed {
    uint64_t order, w;
    __device__ __forceinline__ uint32_t key() const { return (uint32_t)(order >> 32); }
    __device__ __forceinline__ uint32_t index() const { return ~(uint32_t)order; }
};
__device__ __forceinline__ uint64_t order_of(uint32_t key, uint32_t index) { return (uint64_t)key << 32 | (uint32_t)~index; }

template <int THREADS>
struct SampleLds {
    Listed list[kList];
    union {
        uint64_t weight[kBins];
        uint32_t count[kBins];
    };
    uint64_t wave_sum[THREADS / kOpWave];
    float wave_max[THREADS / kOpWave];
    uint32_t listed, least, most, bin, found_key, found_index, kept;
    uint64_t before, sum;
    Listed sorted[kList];
};

// A row of logits, VEC neighbouring ones of a sweep over the row a thread.  Passes of the general way read it again (from L2: with every
// one of them unrolled over 64 logits in registers, they spill).
template <typename T, int THREADS>
struct Row {
    static constexpr int VEC = 16 / sizeof(T), kSweep = THREADS * VEC;
    typedef T vec __attribute__((ext_vector_type(VEC)));
    const T* p;
    uint32_t n, sweeps;
    bool aligned;

    __device__ __forceinline__ vec load(uint32_t s) const {
        const uint32_t i = s * kSweep + threadIdx.x * VEC;
        vec v;
        if (aligned && i + VEC <= n) return *(const vec*)(p + i);
#pragma unroll
        for (int e = 0; e < VEC; e++) v[e] = i + e < n ? p[i + e] : (T)(-__builtin_inff());
        return v;
    }
    // fn(sweep, first index, values) for every sweep, by all threads.
    template <typename F>
    __device__ __forceinline__ void each(F&& fn) const {
        vec next = load(0);
        for (uint32_t s = 0; s < sweeps; s++) {
            const vec v = next;
            if (s + 1 < sweeps) next = load(s + 1);
            fn(s, s * kSweep + threadIdx.x * VEC, v);
        }
    }
};

// The row's measure: what its values mean once the largest one is known.
struct Scale {
    float most;
    float bins;                // bins a unit of logits
    double inv;                // 1 / T
    // Where l is below the largest, in bins: falls with l, and is below kBins for all that weigh anything (kLeast leaves 6 bins to
    // spare for the rounding).  NaN and -inf are nowhere.
    __device__ __forceinline__ float place(float l) const { return l == most ? 0.0f : (most - l) * bins; }
    __device__ __forceinline__ bool live(float l) const { return place(l) < (float)kBins; }
    __device__ __forceinline__ uint32_t bin(float l) const { return (uint32_t)place(l); }
    __device__ __forceinline__ uint64_t weight(float l) const {
        if (l == most) return (uint64_t)kOne;
        const double x = ((double)l - (double)most) * inv;
        return x >= kLeast ? (uint64_t)__builtin_rint(exp(x) * kOne) : 0;
    }
};

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kOpWave);
    return v;
}

// v summed over the lanes up to this one.
__device__ __forceinline__ uint64_t wave_upto(uint64_t v, int lane) {
#pragma unroll
    for (int o = 1; o < kOpWave; o <<= 1) {
        const uint64_t x = __shfl_up(v, o, kOpWave);
        if (lane >= o) v += x;
    }
    return v;
}

template <int THREADS>
__device__ __forceinline__ uint64_t block_sum(SampleLds<THREADS>& l, uint64_t v) {
    v = wave_sum(v);
    __syncthreads();
    if (threadIdx.x % kOpWave == 0) l.wave_sum[threadIdx.x / kOpWave] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int w = 0; w < THREADS / kOpWave; w++) s += l.wave_sum[w];
    return s;
}

// Whether an element that `before` comes before (elements, or their weight) is kept: `need` elements, or weights below `target`.
struct Want {
    bool by_weight;
    uint64_t need;
    double target;
    __device__ __forceinline__ bool keeps(uint64_t before) const { return by_weight ? before == 0 || (double)before < target : before < need; }
};

// The bin that the last kept element is in, into l.bin, and what is before the bin into l.before.  `value` holds a bin's elements or
// weight.  Everything fits below `want`'s limit: l.bin stays kBins.
template <int THREADS, typename V>
__device__ __forceinline__ void find_bin(SampleLds<THREADS>& l, const V* value, const Want& want) {
    constexpr int kPer = kBins / THREADS;
    const int lane = threadIdx.x % kOpWave, wave = threadIdx.x / kOpWave;
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) mine += value[threadIdx.x * kPer + i];
    const uint64_t upto = wave_upto(mine, lane);
    if (threadIdx.x == 0) l.bin = kBins;
    if (lane == kOpWave - 1) l.wave_sum[wave] = upto;
    __syncthreads();
    uint64_t before = upto - mine, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / kOpWave; w++) {
        if (w < wave) before += l.wave_sum[w];
        all += l.wave_sum[w];
    }
    // (the last bin with elements whose first one may be kept; and behind it something is not)
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const uint64_t v = value[threadIdx.x * kPer + i];
        if (v && want.keeps(before) && (!want.keeps(before + v) || before + v == all)) l.bin = threadIdx.x * kPer + i, l.before = before;
        before += v;
    }
    __syncthreads();
}

// The last kept element: in bin l.bin, behind l.before elements or weights.  `in` says who takes part.
template <typename R, int THREADS, typename In>
__device__ __forceinline__ Cut find_cut(SampleLds<THREADS>& l, const R& row, const Scale& m, const Want& want, In&& in) {
    const uint32_t bin = l.bin;
    const uint64_t before = l.before;
    if (threadIdx.x == 0) l.listed = 0, l.least = ~0u, l.most = 0;
    __syncthreads();
    row.each([&](uint32_t, uint32_t i0, const typename R::vec& v) {
#pragma unroll
        for (int e = 0; e < R::VEC; e++) {
            const float x = (float)v[e];
            if (!m.live(x) || m.bin(x) != bin || !in(key_of(x), i0 + e)) continue;
            const uint32_t key = key_of(x), at = atomicAdd(&l.listed, 1u);
            if (at < kList) l.list[at] = Listed{order_of(key, i0 + e), want.by_weight ? m.weight(x) : 1};
            atomicMin(&l.least, key);
            atomicMax(&l.most, key);
        }
    });
    __syncthreads();
    const uint32_t n = l.listed;
    if (n <= kList) {
        // Each element looks at all others for what comes before it.
        for (uint32_t t = threadIdx.x; t < n; t += THREADS) {
            const Listed me = l.list[t];
            uint64_t sum = before, rank = 0;
            for (uint32_t j = 0; j < n; j++)
                if (l.list[j].order > me.order) sum += l.list[j].w, rank++;
            if (want.keeps(sum) && (rank + 1 == n || !want.keeps(sum + me.w))) l.found_key = me.key(), l.found_index = me.index();
        }
        __syncthreads();
        return {l.found_key, l.found_index};
    }
    // Many elements of (nearly) one value: the key is searched for between the least and the largest of them, then the number of
    // those that have it, in the order of their indexes.
    uint32_t lo = l.least, hi = l.most;
    const auto from = [&](uint32_t key) {      // what the elements from `key` on add to `before`
        uint64_t s = 0;
        row.each([&](uint32_t, uint32_t i0, const typename R::vec& v) {
#pragma unroll
            for (int e = 0; e < R::VEC; e++) {
                const float x = (float)v[e];
                if (!m.live(x) || m.bin(x) != bin || key_of(x) < key || !in(key_of(x), i0 + e)) continue;
                s += want.by_weight ? m.weight(x) : 1;
            }
        });
        return before + block_sum(l, s);
    };
    while (lo < hi) {                          // the largest key whose followers are not kept: those from it on are enough
        const uint32_t mid = hi - (hi - lo) / 2;
        if (!want.keeps(from(mid))) lo = mid;
        else hi = mid - 1;
    }
    const uint64_t above = lo == ~0u ? before : from(lo + 1);
    // Of those with the key, by sweeps of the row: as long as what came before still leaves one to keep.
    uint64_t done = above;
    uint32_t last = 0;
    const int lane = threadIdx.x % kOpWave, wave = threadIdx.x / kOpWave;
    row.each([&](uint32_t, uint32_t i0, const typename R::vec& v) {
        uint64_t w[R::VEC], mine = 0;
#pragma unroll
        for (int e = 0; e < R::VEC; e++) {
            const float x = (float)v[e];
            const bool hit = key_of(x) == lo && m.live(x) && m.bin(x) == bin && in(lo, i0 + e);
            w[e] = !hit ? 0 : want.by_weight ? m.weight(x) : 1;
            mine += w[e];
        }
        const uint64_t upto = wave_upto(mine, lane);
        __syncthreads();
        if (lane == kOpWave - 1) l.wave_sum[wave] = upto;
        __syncthreads();
        uint64_t s = done + upto - mine, all = 0;
#pragma unroll
        for (int k = 0; k < THREADS / kOpWave; k++) {
            if (k < wave) s += l.wave_sum[k];
            all += l.wave_sum[k];
        }
#pragma unroll
        for (int e = 0; e < R::VEC; e++)
            if (w[e]) {
                if (want.keeps(s)) last = max(last, i0 + e);
                s += w[e];
            }
        done += all;
    });
    if (threadIdx.x == 0) l.found_index = 0;
    __syncthreads();
    atomicMax(&l.found_index, last);
    __syncthreads();
    return {lo, l.found_index};
}

// The limit that a running sum of kept weights passes at the drawn token: u of the whole sum (u of 1 or more: just below it; below 0 or
// NaN: 0).
__device__ __forceinline__ double limit_of(float u, uint64_t sum) {
    const double limit = (u > 0.0f ? (double)u : 0.0) * (double)sum;
    return limit < (double)sum ? limit : (double)sum * 0.9999999999999999;
}

// How many neighbouring threads share each of n elements: 1 to 16.
template <int THREADS>
__device__ __forceinline__ uint32_t sharers(uint32_t n) {
    uint32_t share = 16;
    while (share > 1 && n * share > THREADS) share /= 2;
    return share;
}

__device__ __forceinline__ uint64_t shared_sum(uint64_t v, uint32_t share) {
    for (uint32_t o = 1; o < share; o <<= 1) v += __shfl_xor(v, o, kOpWave);
    return v;
}

// Where everything that may be kept is in the list (n > 0 elements; top_k and top_p of them, `all` the sum that top_p is of if top_k keeps
// all): each element looks at all others for its place in the order of values, and those that are kept at each other once more in that of
// indexes.
template <int THREADS>
__device__ __forceinline__ void draw_listed(SampleLds<THREADS>& l, uint32_t n, uint64_t top_k, bool by_p, double top_p, uint64_t all, double least, float u,
                                            int32_t* token) {
    constexpr uint64_t kMark = 1ull << 53;     // an element counts as this beside its weight: 1,024 weights stay below it
    constexpr int kPer = kList / THREADS > 1 ? kList / THREADS : 1;
    uint32_t share = sharers<THREADS>(n), sub = threadIdx.x % share;
    Listed me[kPer];
    uint64_t before[kPer];
    uint32_t rank[kPer];
    if (threadIdx.x == 0) l.kept = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const uint32_t t = i * (THREADS / share) + threadIdx.x / share;
        rank[i] = ~0u;
        if (t >= n) continue;                  // (a shared element's threads all go or stay)
        me[i] = l.list[t];
        uint64_t sum = 0;
#pragma unroll 8
        for (uint32_t j = sub; j < n; j += share) sum += l.list[j].order > me[i].order ? l.list[j].w + kMark : 0;
        sum = shared_sum(sum, share);
        if (sub != 0) continue;
        rank[i] = (uint32_t)(sum / kMark);
        before[i] = sum % kMark;
        if (rank[i] + 1 == (top_k < n ? (uint32_t)top_k : n)) l.sum = before[i] + me[i].w;
    }
    __syncthreads();
    const Want want{true, 0, top_p * (double)(top_k == ~0ull ? all : l.sum)};
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        if (rank[i] >= top_k || rank[i] == ~0u || (by_p && !want.keeps(before[i])) || (double)me[i].w < least) continue;
        l.sorted[rank[i]] = me[i];
        atomicMax(&l.kept, rank[i] + 1);
    }
    __syncthreads();
    const uint32_t m = l.kept;
#pragma unroll
    for (int i = 0; i < kPer; i++)
        if (rank[i] + 1 == m) l.before = before[i] + me[i].w;        // (all kept weights)
    __syncthreads();
    const double limit = limit_of(u, l.before);
    share = sharers<THREADS>(m), sub = threadIdx.x % share;
    for (uint32_t t = threadIdx.x / share; t < m; t += THREADS / share) {
        const Listed e = l.sorted[t];
        uint64_t upto = 0;
#pragma unroll 8
        for (uint32_t j = sub; j < m; j += share) upto += (uint32_t)l.sorted[j].order >= (uint32_t)e.order ? l.sorted[j].w : 0;      // (indexes are inverted)
        upto = shared_sum(upto, share);
        if (sub == 0 && (double)upto > limit && !((double)(upto - e.w) > limit)) *token = (int32_t)e.index();
    }
}

// The coarse bin (kCoarse of them, in l.count) that the top_k-th of the threads' largest logits is in, or kCoarse if there are not so many.
template <int THREADS>
__device__ __forceinline__ uint32_t coarse_bin(SampleLds<THREADS>& l, uint32_t top_k, int lane) {
    constexpr int kPer = kCoarse / kOpWave;
    if (threadIdx.x < kOpWave) {
        uint32_t c[kPer], mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) mine += c[i] = l.count[lane * kPer + i];
        uint32_t upto = mine;
#pragma unroll
        for (int o = 1; o < kOpWave; o <<= 1) {
            const uint32_t x = __shfl_up(upto, o, kOpWave);
            if (lane >= o) upto += x;
        }
        const uint64_t hit = __ballot(upto >= top_k);
        if (lane == 0) l.bin = kCoarse;
        if (hit && lane == (int)__builtin_ctzll(hit)) {
            uint32_t before = upto - mine, bin = lane * kPer;
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                before += c[i];
                if (before < top_k) bin++;
            }
            l.bin = bin;
        }
    }
    __syncthreads();
    return l.bin;
}

// HELD: sweeps that stay in registers, which hold the whole row; 0: none.
//
// With top_k the way is short.  Each thread has the largest of its logits; the top_k-th logit is no further down than the top_k-th of
// these, and there are few others so far up: they are listed from registers and put in order by comparing each with all.  So a row is
// read once.
template <typename T, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void k_sample(SampleArgs s) {
    typedef Row<T, THREADS> R;
    constexpr int VEC = R::VEC, kWaves = THREADS / kOpWave;
    __shared__ SampleLds<THREADS> l;
    extern __shared__ uint64_t cells[];        // [sweeps][waves]: kept weights
    const redukt_sample& a = s.a;
    const int lane = threadIdx.x % kOpWave, wave = threadIdx.x / kOpWave;
    const uint32_t r = blockIdx.x;
    const R row{(const T*)a.logits + (int64_t)r * a.logits_stride, a.vocab, (a.vocab + R::kSweep - 1) / R::kSweep, s.aligned != 0};

    const float temperature = a.temperatures ? a.temperatures[r] : a.temperature, u = a.u[r];
    const int32_t top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    const float top_p = a.top_ps ? a.top_ps[r] : a.top_p, min_p = a.min_ps ? a.min_ps[r] : a.min_p;

    float mine = -__builtin_inff();
    typename R::vec held[HELD ? HELD : 1];
    const auto fold = [&](const typename R::vec& v) {
#pragma unroll
        for (int e = 0; e < VEC; e++) mine = (float)v[e] > mine ? (float)v[e] : mine;        // (NaN is none)
    };
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++)
            if ((uint32_t)i < row.sweeps) held[i] = row.load(i);
#pragma unroll
        for (int i = 0; i < HELD; i++)
            if ((uint32_t)i < row.sweeps) fold(held[i]);
    } else {
        row.each([&](uint32_t, uint32_t, const typename R::vec& v) { fold(v); });
    }
    Scale m;
    m.most = mine;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m.most = fmaxf(m.most, __shfl_xor(m.most, o, kOpWave));
    if (lane == 0) l.wave_max[wave] = m.most;
    if (threadIdx.x == 0) l.found_index = ~0u;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; w++) m.most = fmaxf(m.most, l.wave_max[w]);
    if (m.most == -__builtin_inff()) {         // nothing to draw from
        if (threadIdx.x == 0) a.tokens[r] = -1;
        return;
    }
    if (!(temperature > 0.0f)) {               // the first of the largest
        row.each([&](uint32_t, uint32_t i0, const typename R::vec& v) {
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if ((float)v[e] == m.most) atomicMin(&l.found_index, i0 + e);
        });
        __syncthreads();
        if (threadIdx.x == 0) a.tokens[r] = (int32_t)l.found_index;
        return;
    }
    m.inv = 1.0 / (double)temperature;
    m.bins = (float)((kBins - 1) / -kLeast * m.inv);
    const bool by_k = top_k > 0 && (uint32_t)top_k < a.vocab, by_p = top_p < 1.0f, by_min = min_p > 0.0f;
    const double least = by_min ? (double)fminf(min_p, 1.0f) * kOne : 0.0;

    if constexpr (HELD > 0) {
        if (by_k && top_k <= (int)kFewK) {
            for (uint32_t i = threadIdx.x; i < kCoarse; i += THREADS) l.count[i] = 0;
            if (threadIdx.x == 0) l.listed = 0;
            __syncthreads();
            if (m.live(mine)) atomicAdd(&l.count[m.bin(mine) / (kBins / kCoarse)], 1u);
            __syncthreads();
            const uint32_t bin = coarse_bin(l, (uint32_t)top_k, lane);
            if (bin < kCoarse) {
                // (what is a little further down may be listed too, but nothing less: the bin's end as a logit, with room for roundings)
                float from = m.most - (float)((bin + 1) * (kBins / kCoarse)) / m.bins * 1.0001f;
                if (!(from < m.most)) from = m.most;
                // (counted first, so that a wave asks for its places in the list once)
                uint32_t hits = 0;
#pragma unroll
                for (int i = 0; i < HELD; i++) {
                    if ((uint32_t)i >= row.sweeps) continue;
#pragma unroll
                    for (int e = 0; e < VEC; e++) hits += __popcll(__ballot((float)held[i][e] >= from));
                }
                uint32_t at = 0;
                if (lane == 0 && hits) at = atomicAdd(&l.listed, hits);
                at = __builtin_amdgcn_readfirstlane(at);
                if (hits && at + hits <= kList) {
#pragma unroll
                    for (int i = 0; i < HELD; i++) {
                        if ((uint32_t)i >= row.sweeps) continue;
#pragma unroll
                        for (int e = 0; e < VEC; e++) {
                            const bool hit = (float)held[i][e] >= from;
                            const uint64_t all = __ballot(hit);
                            if (!all) continue;
                            const uint32_t to = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
                            if (hit) l.list[to].order = order_of(key_of((float)held[i][e]), (uint32_t)i * R::kSweep + threadIdx.x * VEC + e);
                            at += __popcll(all);
                        }
                    }
                }
                __syncthreads();
                const uint32_t n = l.listed;
                if (n <= kList) {
                    for (uint32_t t = threadIdx.x; t < n; t += THREADS) l.list[t].w = m.weight(value_of(l.list[t].key()));
                    __syncthreads();
                    draw_listed(l, n, (uint64_t)top_k, by_p, (double)top_p, 0, least, u, a.tokens + r);
                    return;
                }
            }
            __syncthreads();
        }
    }
    Cut cut{0, ~0u};                           // everything
    if (by_k || by_p) {
        // The bin that the cut is in: by elements, or by weight where only that counts.
        uint64_t sum = 0;
        for (uint32_t i = threadIdx.x; i < kBins; i += THREADS) {
            if (by_k) l.count[i] = 0;
            else l.weight[i] = 0;
        }
        if (threadIdx.x == 0) l.listed = 0;
        __syncthreads();
        row.each([&](uint32_t, uint32_t, const typename R::vec& v) {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float x = (float)v[e];
                if (!m.live(x)) continue;
                if (by_k) {
                    atomicAdd(&l.count[m.bin(x)], 1u);
                } else if (const uint64_t w = m.weight(x)) {
                    sum += w;
                    atomicAdd((unsigned long long*)&l.weight[m.bin(x)], (unsigned long long)w);
                }
            }
        });
        if (!by_k) sum = block_sum(l, sum);
        __syncthreads();
        const Want want{!by_k, (uint64_t)top_k, (double)top_p * (double)sum};
        if (by_k) find_bin(l, l.count, want);
        else find_bin(l, l.weight, want);
        // What may be kept, if it fits the list.
        const uint32_t bin = l.bin;
        row.each([&](uint32_t, uint32_t i0, const typename R::vec& v) {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float x = (float)v[e];
                if (!(m.place(x) < (float)(bin + 1))) continue;
                const uint32_t at = atomicAdd(&l.listed, 1u);
                if (at < kList) l.list[at] = Listed{order_of(key_of(x), i0 + e), m.weight(x)};
            }
        });
        __syncthreads();
        if (l.listed <= kList) {
            draw_listed(l, l.listed, by_k ? (uint64_t)top_k : ~0ull, by_p, (double)top_p, sum, least, u, a.tokens + r);
            return;
        }
        __syncthreads();                       // (find_cut begins the list anew)
        cut = find_cut(l, row, m, want, [](uint32_t, uint32_t) { return true; });
    }
    if (by_k && by_p) {
        for (uint32_t i = threadIdx.x; i < kBins; i += THREADS) l.weight[i] = 0;
        __syncthreads();
        uint64_t sum = 0;
        row.each([&](uint32_t, uint32_t i0, const typename R::vec& v) {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float x = (float)v[e];
                if (!m.live(x) || !cut.keeps(key_of(x), i0 + e)) continue;
                const uint64_t w = m.weight(x);
                sum += w;
                if (w) atomicAdd((unsigned long long*)&l.weight[m.bin(x)], (unsigned long long)w);
            }
        });
        sum = block_sum(l, sum);
        const Want want{true, 0, (double)top_p * (double)sum};
        __syncthreads();
        find_bin(l, l.weight, want);
        const Cut upto = cut;
        cut = find_cut(l, row, m, want, [&](uint32_t k, uint32_t i) { return upto.keeps(k, i); });
    }
    // Kept weights, by sweep and wave, and their sum.
    const auto kept = [&](float x, uint32_t i) {
        if (!m.live(x) || !cut.keeps(key_of(x), i)) return (uint64_t)0;
        const uint64_t w = m.weight(x);
        return (double)w >= least ? w : 0;
    };
    uint64_t sum = 0;
    row.each([&](uint32_t sweep, uint32_t i0, const typename R::vec& v) {
        uint64_t w = 0;
#pragma unroll
        for (int e = 0; e < VEC; e++) w += kept((float)v[e], i0 + e);
        w = wave_sum(w);
        if (lane == 0) cells[sweep * kWaves + wave] = w;
        sum += w;
    });
    __syncthreads();
    if (lane == 0) l.wave_sum[wave] = sum;
    __syncthreads();
    if (wave != 0) return;
    sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) sum += l.wave_sum[w];
    const double limit = limit_of(u, sum);
    uint64_t before = 0;
    uint32_t cell = 0;
    for (uint32_t c0 = 0; c0 < row.sweeps * kWaves; c0 += kOpWave) {
        const uint32_t c = c0 + lane;
        const uint64_t w = c < row.sweeps * kWaves ? cells[c] : 0, upto = wave_upto(w, lane);
        const uint64_t hit = __ballot((double)(before + upto) > limit);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            cell = c0 + at;
            before += __shfl(upto - w, at, kOpWave);
            break;
        }
        before += __shfl(upto, kOpWave - 1, kOpWave);
    }
    const uint32_t i0 = cell / kWaves * R::kSweep + (cell % kWaves * kOpWave + lane) * VEC;
    uint64_t w[VEC], own = 0;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        w[e] = i0 + e < a.vocab ? kept((float)row.p[i0 + e], i0 + e) : 0;
        own += w[e];
    }
    const uint64_t upto = wave_upto(own, lane);
    const uint64_t hit = __ballot((double)(before + upto) > limit);
    if (!hit || lane != (int)__builtin_ctzll(hit)) return;
    uint64_t to = before + upto;
    uint32_t token = i0;
#pragma unroll
    for (int e = VEC - 1; e >= 0; e--) {       // (from behind: the first index whose sum is over)
        if ((double)to > limit && w[e]) token = i0 + e;
        to -= w[e];
    }
    a.tokens[r] = (int32_t)token;
}

template <typename T>
int32_t launch(SampleArgs& k, void* stream) {
    constexpr int VEC = 16 / sizeof(T);
    const uint32_t v = k.a.vocab;
    // A thread has at least a few loads of a row, but no fewer than 256 threads share one; up to 64 logits a thread stay in registers.
    const uint32_t threads = v <= 4096 ? 256 : 1024, sweeps = (v + threads * VEC - 1) / (threads * VEC);
    if (!op_grid_ok(k.a.rows, threads)) return BACKEND_INVALID_ARGUMENT;
    const void* const fn = threads == 256         ? (const void*)k_sample<T, 256, 16 / VEC>
                           : sweeps <= 64u / VEC ? (const void*)k_sample<T, 1024, 64 / VEC>
                                                 : (const void*)k_sample<T, 1024, 0>;
    return op_launch(fn, dim3(k.a.rows), dim3(threads), sweeps * (threads / kOpWave) * 8, stream, k);
}

}  // namespace
}  // namespace rdk

using namespace rdk;

extern "C" {

int32_t redukt_op_sample(const redukt_sample* a, void* stream) {
    if (!a || a->dtype > REDUKT_OP_F32 || a->rows >= (1u << 31) || a->vocab == 0 || a->vocab > kMaxVocab) return BACKEND_INVALID_ARGUMENT;
    if (a->rows == 0) return BACKEND_OK;
    if (!a->logits || !a->u || !a->tokens || !op_aligned(a->logits, op_elem_bytes(a->dtype)) || !op_aligned(a->u, 4) || !op_aligned(a->tokens, 4) ||
        !op_aligned(a->temperatures, 4) || !op_aligned(a->top_ks, 4) || !op_aligned(a->top_ps, 4) || !op_aligned(a->min_ps, 4))
        return BACKEND_INVALID_ARGUMENT;
    if (a->rows > 1 && a->logits_stride != 0 && a->logits_stride < (int64_t)a->vocab) return BACKEND_INVALID_ARGUMENT;
    OpDevice dev(a->tokens);
    if (!dev.ok) return BACKEND_INVALID_ARGUMENT;
    SampleArgs k{*a, op_aligned(a->logits, 16) && (a->rows == 1 || a->logits_stride * op_elem_bytes(a->dtype) % 16 == 0)};
    return a->dtype == REDUKT_OP_BF16 ? launch<__bf16>(k, stream) : a->dtype == REDUKT_OP_F16 ? launch<_Float16>(k, stream) : launch<float>(k, stream);
}

}  // extern "C"
