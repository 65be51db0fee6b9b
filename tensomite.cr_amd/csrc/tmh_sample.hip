// The next token of a row of logits by temperature, top-k, top-p and min-p
// from a given random number (tmh_sample). The reference samples on the host.
//
// With the candidates by falling logit (equal ones by rising index) and
// weights w = e^((x - highest) / t), each cut keeps a prefix of that order, so
// what is left is the shortest of three prefixes, and only its sum S matters:
// the token is the first whose running sum passes u·S. No row is sorted.
// A histogram over y = (highest - x) · log2 e / t holds the count and the sum
// of weights of each bin; the bin in which a count or a sum is reached is
// looked up in it, and only few candidates are put in order: those through the
// cut's bin where they are few, else those of that one bin.
//
// Weights are exp2 in f64, summed as integers of 2^-shift (shift = 62 less the
// bits of n, at most 50: 45 at a vocabulary of 131071), so a sum is the same in
// any order and the ids do not depend on how the work falls; a weight below
// half that step counts as none.
//
// Three launches: chunks' highest and lowest values, chunks' histograms added
// to their row's, then a workgroup a row. A row of 131072 takes about 30 vector
// operations a value for its weights and is read three times, from the caches
// after the first; rows are cut in chunks until there is one for each compute
// unit.
#include "../../include/tensomite_hip.h"
#include "tmh_device.h"
#include "tmh_internal.h"

#include <algorithm>

namespace tmh {

namespace {

typedef unsigned long long u64;

constexpr uint32_t THREADS = 1024, WAVES = THREADS / 64;
constexpr uint32_t BINS = 2048;  // of y, two a thread
constexpr uint32_t ZOOM = 1024;  // of keys, one a thread
constexpr uint32_t LIST = 2048;  // candidates put in order at once, two a thread
constexpr uint32_t PAIRS = 256;  // of which so many by comparing each with each

// A chunk's highest value that is a number and its first index (or ~0), and
// its lowest value but -inf.
struct Extent {
    float high, low;
    uint32_t index;
    __device__ __forceinline__ void take(const Extent& o) {
        low = fminf(low, o.low);
        if (o.index != ~0u && (index == ~0u || o.high > high || (o.high == high && o.index < index)))
            high = o.high, index = o.index;
    }
};

// A row's histogram.
struct Histogram {
    u64 sums[BINS];
    u64 least;  // the sum of the weights that min_p leaves
    uint32_t counts[BINS];
};

struct Sample {
    const float* x;
    uint32_t ldx, n, shift;
    uint32_t chunk, chunks;  // values of a chunk, chunks of a row
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* ids;
    Extent* extents;  // [rows, chunks]
    Histogram* rows;
};

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
    double exact, one;  // the scale in f64; 2^shift

    __device__ __forceinline__ Measure(const Extent& e, float temperature, uint32_t shift) {
        highest = e.high;
        exact = 1.4426950408889634 / (double)temperature;
        scale = (float)exact;
        cut = (float)(shift + 2u);
        one = (double)((u64)1 << shift);
        const float range = fminf((e.high - e.low) * scale, cut);
        per_y = range > 0.0f ? fminf((float)BINS / range, 1e30f) : 0.0f;
    }
    // y in f32 falls as x rises, so bins stand in the candidates' order, and
    // y above cut is a weight of none. NaN and -inf are not within it.
    __device__ __forceinline__ float y(float x) const { return x == highest ? 0.0f : (highest - x) * scale; }
    __device__ __forceinline__ bool within(float y) const { return y <= cut; }
    __device__ __forceinline__ uint32_t bin(float y) const { return min((uint32_t)(y * per_y), BINS - 1u); }
    __device__ __forceinline__ double part(float x) const {
        return x == highest ? 1.0 : exp2_minus(((double)highest - (double)x) * exact);
    }
    // to the nearest integer of 2^-shift, at most 2^50, in the low bits of a
    // number of 2^52
    __device__ __forceinline__ u64 weight(double part) const {
        return (u64)__builtin_bit_cast(long long, part * one + 4503599627370496.0) & 0xfffffffffffffull;
    }
    // The first key whose bin is `bin` or after it (keys not within cut are
    // after all bins), by 64 keys a round.
    __device__ __forceinline__ uint32_t first_key(uint32_t bin_from) const {
        const uint32_t lane = threadIdx.x & 63u;
        uint32_t low = key_of(highest), high = 0xff800000u;  // -inf's
        while (low < high) {
            const uint32_t step = (high - low - 1u) / 64u + 1u;
            const u64 at = (u64)low + (u64)step * lane;
            bool past = at >= high;
            if (!past) {
                const float v = y(value_of((uint32_t)at));
                past = !within(v) || bin(v) >= bin_from;
            }
            const uint64_t ones = __ballot(past);
            const uint32_t first = ones ? (uint32_t)__ffsll((unsigned long long)ones) - 1u : 64u;
            if (first == 0) return low;
            high = (uint32_t)min((u64)high, (u64)low + (u64)step * first);
            low = low + step * (first - 1u) + 1u;
        }
        return low;
    }
};

// Where a count or a sum is reached: the bin, what stands before it, how many
// it holds; then the candidate, and the sum through it.
struct Found {
    uint32_t bin, count_before, count, index;
    u64 sum_before, sum;
};

struct Lds {
    u64 zoom_sums[ZOOM];
    u64 list[LIST];     // key, then index
    u64 sorted[LIST];
    u64 through[LIST];  // sums through the sorted
    uint32_t zoom_counts[ZOOM];
    u64 wave_sum[WAVES];
    uint32_t wave_count[WAVES];
    Found found;
    uint32_t listed;
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

// A thread's bins of a histogram, and what the threads before it hold.
template <uint32_t PER>
struct Bins {
    uint32_t counts[PER], count_before;
    u64 sums[PER], sum_before;

    // The bin that the target is in, into l.found.
    __device__ __forceinline__ void find(Lds& l, Target t) const {
        uint32_t c = count_before;
        u64 s = sum_before;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            if (t.in(c, counts[i], s, sums[i])) {
                l.found.bin = threadIdx.x * PER + i;
                l.found.count_before = c, l.found.count = counts[i], l.found.sum_before = s;
            }
            c += counts[i], s += sums[i];
        }
        __syncthreads();
    }
};

// Lists the candidates with values from `low` to `high`: all of them into
// l.listed, LIST at most into the list.
__device__ __forceinline__ void list_values(Lds& l, const float* row, uint32_t n, float low, float high) {
    if (threadIdx.x == 0) l.listed = 0;
    __syncthreads();
    const auto take = [&](float x, uint32_t j) {
        if (x >= low && x <= high) {
            const uint32_t at = atomicAdd(&l.listed, 1u);
            if (at < LIST) l.list[at] = (u64)key_of(x) << 32 | j;
        }
    };
    constexpr uint32_t AHEAD = 8;
    uint32_t j = threadIdx.x;
    for (; j + (AHEAD - 1u) * THREADS < n; j += AHEAD * THREADS) {
        float x[AHEAD];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) x[i] = row[j + i * THREADS];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) take(x[i], j + i * THREADS);
    }
    for (; j < n; j += THREADS) take(row[j], j);
    __syncthreads();
}

// Puts the list (at most LIST) in order, with the sums through each, `sum`
// standing before the first.
__device__ __forceinline__ void sort_list(Lds& l, const Measure& m, u64 sum) {
    const uint32_t n = l.listed;
    if (n > PAIRS) {  // a bitonic sort of the next power of two
        uint32_t size = 2u * PAIRS;
        while (size < n) size <<= 1;
        for (uint32_t i = threadIdx.x; i < size; i += THREADS) l.sorted[i] = i < n ? l.list[i] : ~0ull;
        for (uint32_t k = 2; k <= size; k <<= 1)
            for (uint32_t d = k >> 1; d > 0; d >>= 1) {
                __syncthreads();
                if (threadIdx.x < size / 2u) {
                    const uint32_t i = 2u * threadIdx.x - (threadIdx.x & (d - 1u));
                    const u64 a = l.sorted[i], b = l.sorted[i + d];
                    if ((a > b) == ((i & k) == 0)) l.sorted[i] = b, l.sorted[i + d] = a;
                }
            }
    } else {
        // four threads a candidate, each comparing it with a quarter of them
        const uint32_t i = threadIdx.x >> 2;
        const u64 mine = i < n ? l.list[i] : 0;
        uint32_t c = 0;
        if (i < n)
            for (uint32_t j = threadIdx.x & 3u; j < n; j += 4u) c += l.list[j] < mine ? 1u : 0u;
        c += __shfl_xor(c, 1, 64);
        c += __shfl_xor(c, 2, 64);
        if ((threadIdx.x & 3u) == 0 && i < n) l.sorted[c] = mine;
    }
    __syncthreads();
    const uint32_t at = 2u * threadIdx.x;
    u64 w[2];
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i)
        w[i] = at + i < n ? m.weight(m.part(value_of((uint32_t)(l.sorted[at + i] >> 32)))) : 0;
    uint32_t none = 0, all;
    u64 before = w[0] + w[1], total;
    scan(l, none, before, all, total);
    l.through[at] = sum + before + w[0];
    l.through[at + 1u] = sum + before + w[0] + w[1];
    __syncthreads();
}

// The target among the sorted, `count` and `sum` standing before the first.
__device__ __forceinline__ void find_sorted(Lds& l, Target t, uint32_t count, u64 sum) {
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {
        const uint32_t at = 2u * threadIdx.x + i;
        if (at < l.listed) {
            const u64 before = at ? l.through[at - 1u] : sum, through = l.through[at];
            if (t.in(count + at, 1, before, through - before)) l.found.index = (uint32_t)l.sorted[at], l.found.sum = through;
        }
    }
    __syncthreads();
}

// The candidate that the target is in, and the sum through it, into l.found;
// the target's bin is there.
__device__ __forceinline__ void find_in_bin(Lds& l, const Measure& m, const float* row, uint32_t n, Target t) {
    uint32_t low = m.first_key(l.found.bin), high = m.first_key(l.found.bin + 1u) - 1u;
    // more than the list holds: histograms of ever fewer keys
    while (l.found.count > LIST && low < high) {
        uint32_t shift = 0;
        while (((high - low) >> shift) >= ZOOM) ++shift;
        __syncthreads();
        l.zoom_counts[threadIdx.x] = 0, l.zoom_sums[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < n; j += THREADS) {
            const float x = row[j];
            const uint32_t key = key_of(x);
            if (key >= low && key <= high) {
                atomicAdd(&l.zoom_counts[(key - low) >> shift], 1u);
                atomicAdd(&l.zoom_sums[(key - low) >> shift], m.weight(m.part(x)));
            }
        }
        __syncthreads();
        Bins<1> bins;
        uint32_t all;
        u64 total;
        bins.counts[0] = bins.count_before = l.zoom_counts[threadIdx.x];
        bins.sums[0] = bins.sum_before = l.zoom_sums[threadIdx.x];
        scan(l, bins.count_before, bins.sum_before, all, total);
        bins.count_before += l.found.count_before, bins.sum_before += l.found.sum_before;
        bins.find(l, t);
        low += l.found.bin << shift;
        high = min(high, low + (1u << shift) - 1u);
    }
    const uint32_t count = l.found.count_before;
    const u64 sum = l.found.sum_before;
    if (l.found.count <= LIST) {
        list_values(l, row, n, value_of(high), value_of(low));
        sort_list(l, m, sum);
        find_sorted(l, t, count, sum);
        return;
    }
    // one value more often than the list holds: by index
    const u64 weight = m.weight(m.part(value_of(low)));
    const u64 place = t.by_sum ? (t.target - sum) / weight : t.target - count;
    uint32_t before = 0;
    for (uint32_t base = 0; base < n; base += THREADS) {
        const uint32_t j = base + threadIdx.x;
        const bool is = j < n && key_of(row[j]) == low;
        uint32_t c = is ? 1u : 0u, all;
        u64 s = 0, total;
        scan(l, c, s, all, total);
        if (is && before + c == place) l.found.index = j, l.found.sum = sum + (place + 1u) * weight;
        before += all;
    }
    __syncthreads();
}

// The highest and lowest values of chunk blockIdx.x of row blockIdx.y, whose
// share of the row's histogram it clears.
__global__ __launch_bounds__(1024) void k_sample_extent(Sample a) {
    __shared__ Extent waves[WAVES];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const float* row = a.x + (size_t)blockIdx.y * a.ldx;
    const uint32_t from = blockIdx.x * a.chunk, to = min(from + a.chunk, a.n);
    Extent e{-INFINITY, INFINITY, ~0u};
    const auto take = [&](float x, uint32_t j) {
        if (x == x && (e.index == ~0u || x > e.high)) e.high = x, e.index = j;
        if (x > -INFINITY) e.low = fminf(e.low, x);
    };
    constexpr uint32_t AHEAD = 8;
    uint32_t j = from + threadIdx.x;
    for (; j + (AHEAD - 1u) * THREADS < to; j += AHEAD * THREADS) {
        float x[AHEAD];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) x[i] = row[j + i * THREADS];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) take(x[i], j + i * THREADS);
    }
    for (; j < to; j += THREADS) take(row[j], j);
    Histogram& h = a.rows[blockIdx.y];
    for (uint32_t b = blockIdx.x * THREADS + threadIdx.x; b < BINS; b += a.chunks * THREADS) h.sums[b] = 0, h.counts[b] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) h.least = 0;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        Extent o;
        o.high = __shfl_xor(e.high, d, 64);
        o.low = __shfl_xor(e.low, d, 64);
        o.index = __shfl_xor(e.index, d, 64);
        e.take(o);
    }
    if (lane == 0) waves[wave] = e;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < WAVES; ++w) e.take(waves[w]);
        a.extents[(size_t)blockIdx.y * a.chunks + blockIdx.x] = e;
    }
}

// A row's extent from its chunks', and whether it is to be sampled at all.
__device__ __forceinline__ bool row_extent(const Sample& a, uint32_t r, float temperature, Extent& e) {
    e = a.extents[(size_t)r * a.chunks];
    for (uint32_t c = 1; c < a.chunks; ++c) e.take(a.extents[(size_t)r * a.chunks + c]);
    return temperature > 0.0f && e.high > -INFINITY;
}

// The histogram of chunk blockIdx.x of row blockIdx.y, added to the row's.
__global__ __launch_bounds__(1024) void k_sample_histogram(Sample a) {
    __shared__ u64 sums[BINS];
    __shared__ uint32_t counts[BINS];
    __shared__ u64 least_sum;
    const uint32_t r = blockIdx.y;
    const float* row = a.x + (size_t)r * a.ldx;
    const float temperature = a.temperature ? a.temperature[r] : 1.0f;
    Extent e;
    if (!row_extent(a, r, temperature, e)) return;
    const Measure m(e, temperature, a.shift);
    const float least = a.min_p ? a.min_p[r] : 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < BINS / THREADS; ++i) sums[threadIdx.x + i * THREADS] = 0, counts[threadIdx.x + i * THREADS] = 0;
    if (threadIdx.x == 0) least_sum = 0;
    __syncthreads();
    u64 kept = 0;
    const auto take = [&](float x) {
        const float y = m.y(x);
        if (m.within(y)) {
            const double part = m.part(x);
            const u64 weight = m.weight(part);
            atomicAdd(&counts[m.bin(y)], 1u);
            atomicAdd(&sums[m.bin(y)], weight);
            if (part >= (double)least) kept += weight;
        }
    };
    const uint32_t from = blockIdx.x * a.chunk, to = min(from + a.chunk, a.n);
    constexpr uint32_t AHEAD = 4;
    uint32_t j = from + threadIdx.x;
    for (; j + (AHEAD - 1u) * THREADS < to; j += AHEAD * THREADS) {
        float x[AHEAD];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) x[i] = row[j + i * THREADS];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) take(x[i]);
    }
    for (; j < to; j += THREADS) take(row[j]);
    if (!(least <= 0.0f)) {
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) kept += __shfl_xor(kept, d, 64);
        if ((threadIdx.x & 63u) == 0) atomicAdd(&least_sum, kept);
    }
    __syncthreads();
    Histogram& h = a.rows[r];
    if (threadIdx.x == 0 && least_sum) atomicAdd(&h.least, least_sum);
#pragma unroll
    for (uint32_t i = 0; i < BINS / THREADS; ++i) {
        const uint32_t b = threadIdx.x + i * THREADS;
        if (a.chunks == 1u) {
            h.counts[b] = counts[b], h.sums[b] = sums[b];
        } else if (counts[b]) {
            atomicAdd(&h.counts[b], counts[b]);
            if (sums[b]) atomicAdd(&h.sums[b], sums[b]);
        }
    }
}

// One row by one workgroup: the cuts and the choice.
__global__ __launch_bounds__(1024) void k_sample(Sample a) {
    extern __shared__ u64 lds_words[];
    Lds& l = *reinterpret_cast<Lds*>(lds_words);
    const uint32_t r = blockIdx.x, n = a.n;
    const float* row = a.x + (size_t)r * a.ldx;
    const float temperature = a.temperature ? a.temperature[r] : 1.0f;
    Extent e;
    if (!row_extent(a, r, temperature, e)) {
        if (threadIdx.x == 0) {
            const float first = row[0];
            a.ids[r] = first != first || e.index == ~0u ? 0 : (int32_t)e.index;
        }
        return;
    }
    const Measure m(e, temperature, a.shift);
    constexpr uint32_t PER = BINS / THREADS;
    const Histogram& h = a.rows[r];
    Bins<PER> bins;
    bins.count_before = 0, bins.sum_before = 0;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        bins.counts[i] = h.counts[threadIdx.x * PER + i], bins.sums[i] = h.sums[threadIdx.x * PER + i];
        bins.count_before += bins.counts[i], bins.sum_before += bins.sums[i];
    }
    const float least = a.min_p ? a.min_p[r] : 0.0f, p = a.top_p ? a.top_p[r] : 1.0f, u = a.u[r];
    const int32_t k = a.top_k ? a.top_k[r] : 0;
    const u64 least_sum = h.least;
    uint32_t all;
    u64 total;
    scan(l, bins.count_before, bins.sum_before, all, total);
    // what is wanted of the histogram; where the candidates through a cut's
    // bin fit the list, of them, in order, from then on
    bool listed = false;
    const auto find = [&](Target t, bool cut) {
        if (!listed) {
            bins.find(l, t);
            if (!cut || l.found.count_before + l.found.count > LIST) {
                find_in_bin(l, m, row, n, t);
                return;
            }
            list_values(l, row, n, value_of(m.first_key(l.found.bin + 1u) - 1u), m.highest);
            sort_list(l, m, 0);
            listed = true;
        }
        find_sorted(l, t, 0, 0);
    };
    // the prefix that stays: the shortest of three
    if (k > 0 && (uint32_t)k < all) {
        find(Target{false, (u64)k - 1u}, true);
        total = l.found.sum;
    }
    if (!(p >= 1.0f)) {
        const double reach = (double)p * (double)total;
        find(Target{true, reach > 0.0 ? (u64)__builtin_ceil(reach) - 1u : 0}, true);
        total = min(total, l.found.sum);
    }
    if (!(least <= 0.0f)) total = min(total, least_sum);
    total = max(total, (u64)1 << a.shift);
    const double passes = (double)u * (double)total;
    find(Target{true, passes > 0.0 ? min((u64)passes, total - 1u) : passes == passes ? 0 : total - 1u}, false);
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
    if (rows > 65535u) return TMH_ERROR_SHAPE;
    DeviceContext ctx;
    const int err = device_context(&ctx, true);
    if (err) return err;
    uint32_t bits = 0;
    while (n >> bits) ++bits;
    // a chunk for each compute unit, of four values a thread or more
    constexpr uint32_t LEAST = 4u * THREADS;
    const uint32_t chunks = std::max(1u, std::min((uint32_t)ctx.compute_units / rows, (n + LEAST - 1u) / LEAST));
    const uint32_t chunk = (n + chunks - 1u) / chunks;
    const size_t extents = ((size_t)rows * chunks * sizeof(Extent) + 255u) & ~(size_t)255u;
    Workspace work(ctx.index, extents + (size_t)rows * sizeof(Histogram));
    if (work.status) return work.status;
    Sample a{(const float*)x, ldx, n, std::min(62u - bits, 50u), chunk, (n + chunk - 1u) / chunk,
             (const float*)temperature, (const int32_t*)top_k, (const float*)top_p, (const float*)min_p,
             (const float*)u, (int32_t*)ids, (Extent*)work.memory, (Histogram*)(work.memory + extents)};
    const dim3 grid(a.chunks, rows);
    TMH_LAUNCH(k_sample_extent, grid, dim3(THREADS), 0, ctx.stream, a);
    TMH_LAUNCH(k_sample_histogram, grid, dim3(THREADS), 0, ctx.stream, a);
    TMH_LAUNCH(k_sample, dim3(rows), dim3(THREADS), sizeof(Lds), ctx.stream, a);
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) note_launch(ctx.index, 1, false);
    return code(e);
}

}  // extern "C"
