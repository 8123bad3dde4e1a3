// sample_ops.hip — tokens drawn from rows of logits (redukt_ops.h).
//
// Weights are whole numbers, W = e^((l - max) / T) in steps of 2^-42, so their sums are exact in 64-bit integers: they have no order,
// may be added by atomics, and the drawn token depends on nothing but the row.
#include <hip/hip_runtime.h>

#include "op_common.h"

#pragma clang fp contract(fast)

namespace rdk {
namespace {

constexpr double kOne = 0x1p42;
constexpr double kLeast = -29.9;           // ln 2^-43 = -29.81: e to less than this is no whole step
constexpr uint32_t kBins = 2048;           // of (max - l) / T, linear, down to kLeast
constexpr uint32_t kList = 1024;           // elements that are put in order in LDS
constexpr int kPowerBits = 7, kPowers = 1 << kPowerBits;
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
    double powers[kPowers];    // 2^(i / kPowers)
    Listed list[kList], sorted[kList];
    union {
        uint64_t weight[kBins];
        uint32_t count[kBins];
    };
    uint64_t wave_sum[THREADS / kOpWave];
    float wave_max[THREADS / kOpWave];
    uint32_t listed, least, most, bin, found_key, found_index, kept;
    uint64_t before, sum;
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

    __device__ __forceinline__ vec load(uint32_t s) const { return at(s * kSweep + threadIdx.x * VEC); }
    __device__ __forceinline__ vec at(uint32_t i) const {
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
    float most, half;          // the largest, and half of it
    float bins;                // bins a unit of logits, at most half of f32's range (of less than a T of 2e-37; what weighs anything is below 30 T)
    float half_bins;           // twice that: bins a unit of half logits
    double steps;              // kPowers log2(e) / T: steps of 2^(1 / kPowers) a unit of logits
    const double* powers;
    // Where l is below the largest, in bins: falls with l, and is below kBins for all that weigh anything (kLeast leaves 6 bins to
    // spare for the rounding).  NaN and -inf are nowhere.  It goes by half of the difference, which has no overflow.
    __device__ __forceinline__ float place(float l) const { return l == most ? 0.0f : fmaf(l, -0.5f, half) * half_bins; }
    __device__ __forceinline__ bool live(float l) const { return place(l) < (float)kBins; }
    __device__ __forceinline__ uint32_t bin(float l) const { return (uint32_t)place(l); }
    // 2^42 e^((l - most) / T) to the nearest whole number, of a live l.  The power's argument in steps of 2^(1 / 128) is a whole number (added
    // to 1.5 * 2^52 it stands in the sum's last bits) and a rest of at most half a step, |rest ln 2 / 128| <= 0.0028; of its power's series five
    // terms leave 1.4e-15.  Adding 2^52 leaves the whole number in the last bits again.
    __device__ __forceinline__ uint64_t weight(float l) const {
        if (l == most) return (uint64_t)kOne;
        constexpr double kWhole = 0x1.8p52, kRest = 0x1.62e42fefa39efp-1 / kPowers;
        const double x = ((double)l - (double)most) * steps, whole = x + kWhole;
        const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, whole);
        const double r = (x - (whole - kWhole)) * kRest;
        const double p = 1.0 + r * (1.0 + r * (0.5 + r * (1.0 / 6.0 + r * (1.0 / 24.0))));
        const double w = __builtin_ldexp(powers[k & (kPowers - 1)] * p, (k >> kPowerBits) + 42);
        return x >= kLeast * (kPowers * 0x1.71547652b82fep+0) ? __builtin_bit_cast(uint64_t, w + 0x1p52) & 0xfffffffffffffull : 0;
    }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or_0(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_or_0(uint64_t v) {
    return (uint64_t)dpp_or_0<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp_or_0<CTRL, ROWS>((uint32_t)v);
}

// v summed over the lanes up to this one: within rows of 16 by moves of 1, 2, 4 and 8 lanes, then a row's last lane into the next row, and
// lane 31 into the upper half.
template <typename V>
__device__ __forceinline__ V wave_upto(V v) {
    v += dpp_or_0<0x111, 0xf>(v);
    v += dpp_or_0<0x112, 0xf>(v);
    v += dpp_or_0<0x114, 0xf>(v);
    v += dpp_or_0<0x118, 0xf>(v);
    v += dpp_or_0<0x142, 0xa>(v);
    v += dpp_or_0<0x143, 0xc>(v);
    return v;
}

__device__ __forceinline__ uint32_t from_lane(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int lane) { return (uint64_t)from_lane((uint32_t)(v >> 32), lane) << 32 | from_lane((uint32_t)v, lane); }

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) { return from_lane(wave_upto(v), kOpWave - 1); }

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
    const uint64_t upto = wave_upto(mine);
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
        const uint64_t upto = wave_upto(mine);
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

// What draw_listed keeps in the bins' place.
constexpr uint32_t kFine = 256;            // its bins
struct Ordered {
    uint32_t first[kFine + 1];             // elements of a bin, then the place of its first one
    uint32_t place[kList];                 // an element's bin, and behind 16 bits its number there
    uint64_t weight[kFine];                // kept weights by index
};
static_assert(sizeof(Ordered) <= kBins * 8, "");

// Where everything that may be kept is in the list (n elements, none further than `reach` below the largest; top_k and top_p of them, `all` the
// sum that top_p is of if top_k keeps all).  Elements go to 256 bins by value, and within a bin each looks at the others for its place.  From there
// one wave goes on without waiting for others: sums along the order say who is kept, their weights go to 256 bins by index, and the bin that the
// limit falls into is looked through.  (1,000 rows of 1,000 logits by workgroups of 256: 21 us, with each element against all others 130.)
template <int THREADS>
__device__ __forceinline__ void draw_listed(SampleLds<THREADS>& l, const Scale& m, uint32_t n, float reach, uint32_t vocab, uint64_t top_k, bool by_p, double top_p,
                                            uint64_t all, uint64_t least, float u, int32_t* token) {
    constexpr uint32_t kPer = kFine / kOpWave;
    Ordered& o = *(Ordered*)l.weight;
    const int lane = threadIdx.x % kOpWave;
    const float fine = (float)(kFine - 1) / reach;
    for (uint32_t i = threadIdx.x; i < kFine; i += THREADS) o.first[i] = 0, o.weight[i] = 0;
    if (threadIdx.x == 0) l.kept = 0;
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < n; t += THREADS) {
        const float v = value_of(l.list[t].key());
        const uint32_t bin = v == m.most ? 0u : (uint32_t)fminf((m.most - v) * fine, (float)(kFine - 1));
        l.list[t].w = m.weight(v);
        o.place[t] = bin | atomicAdd(&o.first[bin], 1u) << 16;
    }
    __syncthreads();
    if (threadIdx.x < kOpWave) {
        uint32_t c[kPer], mine = 0;
#pragma unroll
        for (uint32_t i = 0; i < kPer; i++) mine += c[i] = o.first[lane * kPer + i];
        uint32_t before = wave_upto(mine) - mine;
#pragma unroll
        for (uint32_t i = 0; i < kPer; i++) {
            o.first[lane * kPer + i] = before;
            before += c[i];
        }
        if (lane == 0) o.first[kFine] = n;
    }
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < n; t += THREADS) l.sorted[o.first[o.place[t] & 0xffff] + (o.place[t] >> 16)] = l.list[t];
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < n; t += THREADS) {
        const uint32_t bin = o.place[t] & 0xffff, first = o.first[bin], end = o.first[bin + 1], at = first + (o.place[t] >> 16);
        const Listed me = l.sorted[at];
        uint32_t rank = first;
        for (uint32_t j = first; j < end; j++) rank += l.sorted[j].order > me.order;
        l.list[rank] = me;                     // (all are in `sorted`)
    }
    __syncthreads();
    if (threadIdx.x >= kOpWave) return;
    // In order now: a lane takes `per` neighbouring ones.
    const uint32_t per = (n + kOpWave - 1) / kOpWave, t0 = lane * per, t1 = min(t0 + per, n);
    uint64_t sum = 0;
    for (uint32_t t = t0; t < t1; t++) sum += t < top_k ? l.list[t].w : 0;
    uint64_t upto = wave_upto(sum);
    const Want want{true, 0, top_p * (double)(top_k == ~0ull ? all : from_lane(upto, kOpWave - 1))};
    const uint32_t wide = (vocab + kFine - 1) / kFine;
    uint64_t before = upto - sum;
    sum = 0;
    for (uint32_t t = t0; t < t1; t++) {
        const Listed e = l.list[t];
        const bool kept = t < top_k && (!by_p || want.keeps(before)) && e.w >= least;
        before += e.w;
        if (kept) {
            sum += e.w;
            atomicAdd((unsigned long long*)&o.weight[e.index() / wide], (unsigned long long)e.w);
        } else {
            l.list[t].w = 0;
        }
    }
    sum = wave_sum(sum);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const double limit = limit_of(u, sum);
    uint64_t w[kPer], mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPer; i++) mine += w[i] = o.weight[lane * kPer + i];
    upto = wave_upto(mine);
    const int at = __builtin_ctzll(__ballot((double)upto > limit) | 1ull << 63);        // (the last lane's is)
    before = upto - mine;
    uint32_t bin = lane * kPer;
#pragma unroll
    for (uint32_t i = 0; i + 1 < kPer; i++)
        if (bin == lane * kPer + i && !((double)(before + w[i]) > limit)) before += w[i], bin++;
    before = from_lane(before, at), bin = from_lane(bin, at);
    for (uint32_t t = t0; t < t1; t++)
        if (l.list[t].w && l.list[t].index() / wide == bin) l.sorted[atomicAdd(&l.kept, 1u)] = l.list[t];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const uint32_t few = l.kept;
    for (uint32_t t = lane; t < few; t += kOpWave) {
        const Listed e = l.sorted[t];
        uint64_t s = before;
        for (uint32_t j = 0; j < few; j++) s += l.sorted[j].index() <= e.index() ? l.sorted[j].w : 0;
        if ((double)s > limit && !((double)(s - e.w) > limit)) *token = (int32_t)e.index();
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
        const uint32_t upto = wave_upto(mine);
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

// HELD: sweeps whose loads go out together; WHOLE: they cover the row.
//
// With top_k the way is short.  Each thread has the largest of its logits; the top_k-th logit is no further down than the top_k-th of
// these, and there are few others so far up: they are listed and put in order.  A row is read once, and of it again what the threads read
// that have such a logit.
// Bound by the steps of a row, one after the other: 50,280 logits in f32 take 1,024 threads 24,000 cycles, 5,700 of them to read the row, 3,400 for
// its largest values, 6,000 to list what may be kept, 8,000 to order it and draw.  One row 10.5 us; 1,000 in bf16, 100 MB, two workgroups a CU, 38
// (2.6 TB/s), in f32 61 (3.3).  Without top_k all weights are formed, in 64 bits: 1,000 rows 81 us, and with top_p, whose sums by bin are atomics
// in LDS, 211.
template <typename T, int THREADS, int HELD, bool WHOLE>
__global__ __launch_bounds__(THREADS, 4) void k_sample(SampleArgs s) {
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
    for (uint32_t s0 = 0; s0 < (WHOLE ? 1 : row.sweeps); s0 += HELD) {
        typename R::vec held[HELD];
#pragma unroll
        for (int i = 0; i < HELD; i++)
            if (s0 + i < row.sweeps) held[i] = row.load(s0 + i);
#pragma unroll
        for (int i = 0; i < HELD; i++)
            if (s0 + i < row.sweeps) {
#pragma unroll
                for (int e = 0; e < VEC; e++) mine = (float)held[i][e] > mine ? (float)held[i][e] : mine;        // (NaN is none)
            }
    }
    Scale m;
    m.most = mine;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m.most = fmaxf(m.most, __shfl_xor(m.most, o, kOpWave));
    if (lane == 0) l.wave_max[wave] = m.most;
    if (threadIdx.x == 0) l.found_index = ~0u;
    if (threadIdx.x < kPowers) l.powers[threadIdx.x] = exp2((double)threadIdx.x / kPowers);
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
    const double inverse = 1.0 / (double)temperature;
    m.half = 0.5f * m.most;
    m.bins = fminf((float)((kBins - 1) / -kLeast * inverse), 0x1p126f);
    m.half_bins = 2.0f * m.bins;
    m.steps = kPowers * 0x1.71547652b82fep+0 * inverse;
    m.powers = l.powers;
    const bool by_k = top_k > 0 && (uint32_t)top_k < a.vocab, by_p = top_p < 1.0f, by_min = min_p > 0.0f;
    const uint64_t least = by_min ? (uint64_t)__builtin_ceil((double)fminf(min_p, 1.0f) * kOne) : 1;       // (the limit is exact, and weights are whole)

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
            // The threads that have one, and then all threads over what those read: a row's other logits are not looked at again.
            if (threadIdx.x == 0) l.kept = 0;
            __syncthreads();
            uint32_t* const who = (uint32_t*)l.sorted;
            const uint64_t some = __ballot(mine >= from);
            uint32_t to = 0;
            if (lane == 0 && some) to = atomicAdd(&l.kept, (uint32_t)__popcll(some));
            to = from_lane(to, 0) + __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0));
            if (mine >= from) who[to] = threadIdx.x;
            __syncthreads();
            constexpr uint32_t kAbreast = THREADS / 4;
            const uint32_t many = l.kept;
            for (uint32_t j0 = 0; j0 < many; j0 += kAbreast) {
                const uint32_t j = j0 + threadIdx.x % kAbreast, first = who[min(j, many - 1)] * VEC;
                // (four loads at once, in a row's first part where they would pass its end)
                for (uint32_t s0 = wave * kOpWave / kAbreast; s0 < row.sweeps; s0 += 16) {
                    typename R::vec v[4];
                    uint32_t i[4], hits = 0;
                    const bool vectors = row.aligned && a.vocab >= (uint32_t)VEC;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        i[k] = (s0 + 4 * k) * R::kSweep + first;
                        if (vectors) v[k] = *(const typename R::vec*)(row.p + (i[k] + VEC <= a.vocab ? i[k] : 0));
                    }
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        if (!vectors || i[k] + VEC > a.vocab) v[k] = row.at(min(i[k], a.vocab));      // (-inf behind the row)
#pragma unroll
                        for (int e = 0; e < VEC; e++) hits += (float)v[k][e] >= from;
                    }
                    if (j >= many) hits = 0;
                    // (places in the list for a whole wave at once: an atomic a logit costs more than all else here)
                    const uint32_t upto = wave_upto(hits), all = from_lane(upto, kOpWave - 1);
                    uint32_t at = 0;
                    if (lane == 0 && all) at = atomicAdd(&l.listed, all);
                    at = from_lane(at, 0) + upto - hits;
                    if (!hits || at + hits > kList) continue;
#pragma unroll
                    for (int k = 0; k < 4; k++)
#pragma unroll
                        for (int e = 0; e < VEC; e++)
                            if ((float)v[k][e] >= from) l.list[at++].order = order_of(key_of((float)v[k][e]), i[k] + e);
                }
            }
            __syncthreads();
            const uint32_t n = l.listed;
            if (n <= kList) {
                draw_listed(l, m, n, m.most - from, a.vocab, (uint64_t)top_k, by_p, (double)top_p, 0, least, u, a.tokens + r);
                return;
            }
        }
        __syncthreads();
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
            uint32_t hits = 0;                 // (places for a whole wave at once, as above)
#pragma unroll
            for (int e = 0; e < VEC; e++) hits += m.place((float)v[e]) < (float)(bin + 1);
            const uint32_t upto = wave_upto(hits), all = from_lane(upto, kOpWave - 1);
            uint32_t at = 0;
            if (lane == 0 && all) at = atomicAdd(&l.listed, all);
            at = from_lane(at, 0) + upto - hits;
            if (!hits || at + hits > kList) return;
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (m.place((float)v[e]) < (float)(bin + 1)) l.list[at++].order = order_of(key_of((float)v[e]), i0 + e);
        });
        __syncthreads();
        if (l.listed <= kList) {
            draw_listed(l, m, l.listed, (float)(bin + 1) / m.bins, a.vocab, by_k ? (uint64_t)top_k : ~0ull, by_p, (double)top_p, sum, least, u, a.tokens + r);
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
    const bool whole = cut.key == 0;
    const auto kept = [&](float x, uint32_t i) {
        if (!m.live(x) || !(whole || cut.keeps(key_of(x), i))) return (uint64_t)0;
        const uint64_t w = m.weight(x);
        return w >= least ? w : 0;
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
        const uint64_t w = c < row.sweeps * kWaves ? cells[c] : 0, upto = wave_upto(w);
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
    const uint64_t upto = wave_upto(own);
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
    // With more rows than CUs two workgroups share one, and one works while the other waits for its single wave (us with 1,024 and 512 threads:
    // 200 rows of 50,280 in bf16 13.8 and 15.2, 300 24.5 and 17.9, 1,000 53 and 38, 1,000 of 1,000 40 and 21; one row in f32 10.5 and 12.6).
    // A row's loads go out all at once where 16 vectors of a thread cover it (64 registers; in f32 32 of them spill), else by turns.
    const uint32_t threads = k.a.rows <= 256 ? 1024 : 512, sweeps = (v + threads * VEC - 1) / (threads * VEC);
    if (!op_grid_ok(k.a.rows, threads)) return BACKEND_INVALID_ARGUMENT;
    const void* const fn = threads == 1024 ? sweeps <= 64u / VEC ? (const void*)k_sample<T, 1024, 64 / VEC, true> : (const void*)k_sample<T, 1024, 64 / VEC, false>
                           : sweeps <= 16  ? (const void*)k_sample<T, 512, 16, true>
                                           : (const void*)k_sample<T, 512, 64 / VEC, false>;
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
