// The next token of a row of logits by temperature, top-k, top-p and min-p
// from a given random number (tmh_sample). The reference samples on the host.
//
// With the candidates by falling logit (equal ones by rising index) and
// weights w = e^((x - highest) / t), each cut keeps a prefix of that order, so
// what is left is the shortest of three prefixes, and only its sum S matters:
// the token is the first whose running sum passes u·S. No row is sorted.
// A histogram over y = (highest - x) · log2 e / t holds the count and the sum
// of weights of each bin; the bin in which a count or a sum is reached is
// looked up in it, and only that bin's few candidates are put in order.
//
// Weights are exp2 in f64, summed as integers of 2^-shift (shift = 62 less the
// bits of n: 45 at a vocabulary of 131071), so a sum is the same in any order
// and the ids do not depend on how the work falls; a weight below half that
// step counts as none.
#include "../../include/tensomite_hip.h"
#include "tmh_device.h"
#include "tmh_internal.h"

namespace tmh {

namespace {

typedef unsigned long long u64;

struct Sample {
    const float* x;
    uint32_t ldx, n, shift;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* ids;
};

constexpr uint32_t THREADS = 1024, WAVES = THREADS / 64;
constexpr uint32_t BINS = 4096;  // of y, four a thread
constexpr uint32_t ZOOM = 1024;  // of keys, one a thread
constexpr uint32_t LIST = 2048;  // candidates put in order at once, two a thread
constexpr uint32_t PAIRS = 256;  // of which so many by comparing each with each

// Rising keys for falling values; -0 and 0 are one value.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t w = __float_as_uint(x + 0.0f);
    return w & 0x80000000u ? w : w ^ 0x7fffffffu;
}

__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key : key ^ 0x7fffffffu);
}

// 2^-y for y from 0 to 64: the exponent, and 2^f by its Taylor polynomial to
// f^11 for f within half of 0 (off by less than 2^-46 of it).
__device__ __forceinline__ double exp2_minus(double y) {
    const double k = __builtin_rint(y);
    const double f = (k - y) * 0.6931471805599453;
    double p = 1.0 / 39916800.0;
    p = __builtin_fma(p, f, 1.0 / 3628800.0);
    p = __builtin_fma(p, f, 1.0 / 362880.0);
    p = __builtin_fma(p, f, 1.0 / 40320.0);
    p = __builtin_fma(p, f, 1.0 / 5040.0);
    p = __builtin_fma(p, f, 1.0 / 720.0);
    p = __builtin_fma(p, f, 1.0 / 120.0);
    p = __builtin_fma(p, f, 1.0 / 24.0);
    p = __builtin_fma(p, f, 1.0 / 6.0);
    p = __builtin_fma(p, f, 0.5);
    p = __builtin_fma(p, f, 1.0);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, -(int)k);
}

// A row's measure: its highest value, and y's scale, end and bins.
struct Measure {
    float highest, scale, cut, per_y;
    double exact;  // the scale in f64
    uint32_t shift;

    // y in f32 falls as x rises, so bins stand in the candidates' order, and
    // y above cut is a weight of none. NaN and -inf are not within it.
    __device__ __forceinline__ float y(float x) const { return x == highest ? 0.0f : (highest - x) * scale; }
    __device__ __forceinline__ bool within(float y) const { return y <= cut; }
    __device__ __forceinline__ uint32_t bin(float y) const { return min((uint32_t)(y * per_y), BINS - 1u); }
    __device__ __forceinline__ double part(float x) const {
        return x == highest ? 1.0 : exp2_minus(((double)highest - (double)x) * exact);
    }
    __device__ __forceinline__ u64 weight(double part) const {
        return (u64)__builtin_rint(__builtin_ldexp(part, (int)shift));
    }
};

// Where a count or a sum is reached: the bin, what stands before it, how many
// it holds; then the candidate, and the sum through it.
struct Found {
    uint32_t bin, count_before, count, index;
    u64 sum_before, sum;
};

struct Lds {
    u64 sums[BINS];
    u64 zoom_sums[ZOOM];
    u64 list[LIST];  // key, then index
    u64 weights[LIST];
    uint32_t counts[BINS];
    uint32_t zoom_counts[ZOOM];
    u64 wave_sum[WAVES];
    uint32_t wave_count[WAVES];
    float wave_low[WAVES], wave_high[WAVES];
    uint32_t wave_index[WAVES];
    Found found;
    uint32_t listed, low, high;
};

// Replaces count and sum by what the threads before this one hold of them;
// all and total are everyone's.
__device__ __forceinline__ void scan(Lds& l, uint32_t& count, u64& sum, uint32_t& all, u64& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t c = count;
    u64 s = sum;
#pragma unroll
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t oc = __shfl_up(c, d, 64);
        const u64 os = __shfl_up(s, d, 64);
        if (lane >= d) c += oc, s += os;
    }
    __syncthreads();
    if (lane == 63u) l.wave_count[wave] = c, l.wave_sum[wave] = s;
    __syncthreads();
    uint32_t cb = 0;
    u64 sb = 0;
    all = 0, total = 0;
    for (uint32_t w = 0; w < WAVES; ++w) {
        if (w == wave) cb = all, sb = total;
        all += l.wave_count[w], total += l.wave_sum[w];
    }
    count = cb + c - count;
    sum = sb + s - sum;
}

// What is looked for: the candidate at place `target` (from 0), or the first
// whose running sum passes `target`.
struct Target {
    bool by_sum;
    u64 target;
    __device__ __forceinline__ bool in(uint32_t count_before, uint32_t count, u64 sum_before, u64 sum) const {
        return by_sum ? sum_before <= target && target - sum_before < sum
                      : count_before <= target && target - count_before < count;
    }
};

// The bin of a histogram, PER a thread, that the target is in, when `count`
// and `sum` stand before the first bin; into l.found.
template <uint32_t PER>
__device__ __forceinline__ void find_bin(Lds& l, const uint32_t* counts, const u64* sums, Target t, uint32_t count,
                                         u64 sum) {
    uint32_t c = 0, all;
    u64 s = 0, total;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) c += counts[threadIdx.x * PER + i], s += sums[threadIdx.x * PER + i];
    scan(l, c, s, all, total);
    c += count, s += sum;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t bc = counts[threadIdx.x * PER + i];
        const u64 bs = sums[threadIdx.x * PER + i];
        if (t.in(c, bc, s, bs))
            l.found.bin = threadIdx.x * PER + i, l.found.count_before = c, l.found.count = bc, l.found.sum_before = s;
        c += bc, s += bs;
    }
    __syncthreads();
}

// The target among the listed candidates, which l.found's bin holds.
__device__ __forceinline__ void find_listed(Lds& l, const Measure& m, Target t) {
    const uint32_t n = l.listed, count = l.found.count_before;
    const u64 sum = l.found.sum_before;
    if (n > PAIRS) {  // a bitonic sort of the next power of two
        uint32_t size = 2u * PAIRS;
        while (size < n) size <<= 1;
        for (uint32_t i = n + threadIdx.x; i < size; i += THREADS) l.list[i] = ~0ull;
        for (uint32_t k = 2; k <= size; k <<= 1)
            for (uint32_t d = k >> 1; d > 0; d >>= 1) {
                __syncthreads();
                if (threadIdx.x < size / 2u) {
                    const uint32_t i = 2u * threadIdx.x - (threadIdx.x & (d - 1u));
                    const u64 a = l.list[i], b = l.list[i + d];
                    if ((a > b) == ((i & k) == 0)) l.list[i] = b, l.list[i + d] = a;
                }
            }
        __syncthreads();
    }
    for (uint32_t i = threadIdx.x; i < LIST; i += THREADS)
        l.weights[i] = i < n ? m.weight(m.part(value_of((uint32_t)(l.list[i] >> 32)))) : 0;
    __syncthreads();
    if (n > PAIRS) {
        const uint32_t at = 2u * threadIdx.x;
        uint32_t c = at < n ? min(2u, n - at) : 0, all;
        const u64 first = l.weights[at], second = l.weights[at + 1u];
        u64 s = first + second, total;
        scan(l, c, s, all, total);
        c += count, s += sum;
        if (at < n && t.in(c, 1, s, first)) l.found.index = (uint32_t)l.list[at], l.found.sum = s + first;
        c += 1u, s += first;
        if (at + 1u < n && t.in(c, 1, s, second)) l.found.index = (uint32_t)l.list[at + 1u], l.found.sum = s + second;
    } else {
        // four threads a candidate, each comparing it with a quarter of them
        const uint32_t i = threadIdx.x >> 2;
        const u64 mine = i < n ? l.list[i] : 0;
        uint32_t c = 0;
        u64 s = 0;
        if (i < n)
            for (uint32_t j = threadIdx.x & 3u; j < n; j += 4u)
                if (l.list[j] < mine) c += 1u, s += l.weights[j];
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) c += __shfl_xor(c, d, 64), s += __shfl_xor(s, d, 64);
        c += count, s += sum;
        if ((threadIdx.x & 3u) == 0 && i < n && t.in(c, 1, s, l.weights[i]))
            l.found.index = (uint32_t)mine, l.found.sum = s + l.weights[i];
    }
    __syncthreads();
}

// Lists the candidates with keys from low to high.
__device__ __forceinline__ void list_keys(Lds& l, const Measure& m, const float* row, uint32_t n, uint32_t low,
                                          uint32_t high) {
    if (threadIdx.x == 0) l.listed = 0;
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < n; j += THREADS) {
        const float x = row[j];
        const uint32_t key = key_of(x);
        if (m.within(m.y(x)) && key >= low && key <= high) {
            const uint32_t at = atomicAdd(&l.listed, 1u);
            if (at < LIST) l.list[at] = (u64)key << 32 | j;
        }
    }
    __syncthreads();
}

// The candidate that the target is in, and the sum through it, into l.found.
__device__ __forceinline__ void find(Lds& l, const Measure& m, const float* row, uint32_t n, Target t) {
    find_bin<BINS / THREADS>(l, l.counts, l.sums, t, 0, 0);
    const uint32_t bin = l.found.bin;
    // the keys of the bin
    if (threadIdx.x == 0) l.low = ~0u, l.high = 0;
    __syncthreads();
    uint32_t low = ~0u, high = 0;
    for (uint32_t j = threadIdx.x; j < n; j += THREADS) {
        const float x = row[j], y = m.y(x);
        if (m.within(y) && m.bin(y) == bin) low = min(low, key_of(x)), high = max(high, key_of(x));
    }
    if (low <= high) atomicMin(&l.low, low), atomicMax(&l.high, high);
    __syncthreads();
    low = l.low, high = l.high;
    // more than the list holds: histograms of ever fewer keys
    while (l.found.count > LIST && low < high) {
        uint32_t shift = 0;
        while (((high - low) >> shift) >= ZOOM) ++shift;
        l.zoom_counts[threadIdx.x] = 0, l.zoom_sums[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < n; j += THREADS) {
            const float x = row[j];
            const uint32_t key = key_of(x);
            if (m.within(m.y(x)) && key >= low && key <= high) {
                atomicAdd(&l.zoom_counts[(key - low) >> shift], 1u);
                atomicAdd(&l.zoom_sums[(key - low) >> shift], m.weight(m.part(x)));
            }
        }
        __syncthreads();
        find_bin<1>(l, l.zoom_counts, l.zoom_sums, t, l.found.count_before, l.found.sum_before);
        low += l.found.bin << shift;
        high = min(high, low + (1u << shift) - 1u);
    }
    if (l.found.count <= LIST) {
        list_keys(l, m, row, n, low, high);
        find_listed(l, m, t);
        return;
    }
    // one value more often than the list holds: by index
    const u64 weight = m.weight(m.part(value_of(low)));
    const u64 place = t.by_sum ? (t.target - l.found.sum_before) / weight : t.target - l.found.count_before;
    if (threadIdx.x == 0) l.found.sum = l.found.sum_before + (place + 1u) * weight;
    uint32_t before = 0;
    for (uint32_t base = 0; base < n; base += THREADS) {
        const uint32_t j = base + threadIdx.x;
        const bool is = j < n && key_of(row[j]) == low;
        uint32_t c = is ? 1u : 0u, all;
        u64 s = 0, total;
        scan(l, c, s, all, total);
        if (is && before + c == place) l.found.index = j;
        before += all;
    }
    __syncthreads();
}

// One row by one workgroup.
__global__ __launch_bounds__(1024) void k_sample(Sample a) {
    extern __shared__ u64 lds_words[];
    Lds& l = *reinterpret_cast<Lds*>(lds_words);
    const uint32_t r = blockIdx.x, n = a.n, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const float* row = a.x + (size_t)r * a.ldx;
    const float temperature = a.temperature ? a.temperature[r] : 1.0f;
    // the highest value, its first index, and the lowest but -inf
    float high = -INFINITY, low = INFINITY;
    uint32_t index = ~0u;
    for (uint32_t j = threadIdx.x; j < n; j += THREADS) {
        const float x = row[j];
        if (x == x && (index == ~0u || x > high)) high = x, index = j;
        if (x > -INFINITY) low = fminf(low, x);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const float oh = __shfl_xor(high, d, 64);
        const uint32_t oi = __shfl_xor(index, d, 64);
        low = fminf(low, __shfl_xor(low, d, 64));
        if (oi != ~0u && (index == ~0u || oh > high || (oh == high && oi < index))) high = oh, index = oi;
    }
    if (lane == 0) l.wave_high[wave] = high, l.wave_index[wave] = index, l.wave_low[wave] = low;
#pragma unroll
    for (uint32_t i = 0; i < BINS / THREADS; ++i) l.counts[threadIdx.x + i * THREADS] = 0, l.sums[threadIdx.x + i * THREADS] = 0;
    __syncthreads();
    for (uint32_t w = 0; w < WAVES; ++w) {
        const float oh = l.wave_high[w];
        const uint32_t oi = l.wave_index[w];
        low = fminf(low, l.wave_low[w]);
        if (oi != ~0u && (index == ~0u || oh > high || (oh == high && oi < index))) high = oh, index = oi;
    }
    if (!(temperature > 0.0f) || high == -INFINITY) {
        if (threadIdx.x == 0) {
            const float first = row[0];
            a.ids[r] = first != first || index == ~0u ? 0 : (int32_t)index;
        }
        return;
    }
    Measure m;
    m.highest = high;
    m.exact = 1.4426950408889634 / (double)temperature;
    m.scale = (float)m.exact;
    m.shift = a.shift;
    m.cut = (float)(a.shift + 2u);
    const float range = fminf((high - low) * m.scale, m.cut);
    m.per_y = range > 0.0f ? fminf((float)BINS / range, 1e30f) : 0.0f;
    const float least = a.min_p ? a.min_p[r] : 0.0f;
    const bool cut_least = !(least <= 0.0f);
    u64 kept = 0;  // the sum of weights of at least `least`
    for (uint32_t j = threadIdx.x; j < n; j += THREADS) {
        const float x = row[j], y = m.y(x);
        if (m.within(y)) {
            const double part = m.part(x);
            const u64 weight = m.weight(part);
            atomicAdd(&l.counts[m.bin(y)], 1u);
            atomicAdd(&l.sums[m.bin(y)], weight);
            if (part >= (double)least) kept += weight;
        }
    }
    __syncthreads();
    uint32_t count = 0, all, none = 0, ignore;
    u64 sum = 0, total, everyone;
#pragma unroll
    for (uint32_t i = 0; i < BINS / THREADS; ++i) count += l.counts[threadIdx.x + i * THREADS], sum += l.sums[threadIdx.x + i * THREADS];
    scan(l, count, sum, all, total);
    // the prefix that stays: the shortest of three
    const int32_t k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    if (k > 0 && (uint32_t)k < all) {
        find(l, m, row, n, Target{false, (u64)k - 1u});
        total = l.found.sum;
    }
    if (!(p >= 1.0f)) {
        const double reach = (double)p * (double)total;
        find(l, m, row, n, Target{true, reach > 0.0 ? (u64)__builtin_ceil(reach) - 1u : 0});
        total = min(total, l.found.sum);
    }
    if (cut_least) {
        scan(l, none, kept, ignore, everyone);
        total = min(total, everyone);
    }
    total = max(total, (u64)1 << a.shift);
    const double passes = (double)a.u[r] * (double)total;
    find(l, m, row, n, Target{true, passes > 0.0 ? min((u64)passes, total - 1u) : passes == passes ? 0 : total - 1u});
    if (threadIdx.x == 0) a.ids[r] = (int32_t)l.found.index;
}

int code(hipError_t e) { return e == hipErrorOutOfMemory ? TMH_ERROR_OUT_OF_MEMORY : (int)e; }

}  // namespace

}  // namespace tmh

extern "C" {

int tmh_sample(uint64_t x, uint32_t ldx, uint32_t rows, uint32_t n, uint64_t temperature, uint64_t top_k,
               uint64_t top_p, uint64_t min_p, uint64_t u, uint64_t ids) {
    using namespace tmh;
    if (n == 0 || n > 1u << 24 || ldx < n) return TMH_ERROR_SHAPE;
    if (rows == 0) return TMH_SUCCESS;
    if (!x || !u || !ids) return TMH_ERROR_INVALID_VALUE;
    if (rows > 0x7fffffffu) return TMH_ERROR_SHAPE;
    DeviceContext ctx;
    const int err = device_context(&ctx, true);
    if (err) return err;
    uint32_t bits = 0;
    while (n >> bits) ++bits;
    Sample a{(const float*)x, ldx, n, 62u - bits, (const float*)temperature, (const int32_t*)top_k,
             (const float*)top_p, (const float*)min_p, (const float*)u, (int32_t*)ids};
    TMH_LAUNCH(k_sample, dim3(rows), dim3(THREADS), sizeof(Lds), ctx.stream, a);
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) note_launch(ctx.index, 1, false);
    return code(e);
}

}  // extern "C"
