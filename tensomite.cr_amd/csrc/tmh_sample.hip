// The next token of a row of logits by temperature, top-k, top-p and min-p
// from a given random number (tmh_sample). The reference samples on the host.
//
// With the candidates by falling logit (equal ones by rising index) and
// weights w = e^((x - highest) / t), each cut keeps a prefix of that order, so
// what is left is the shortest of three prefixes, and only its sum S matters:
// the token is the first whose running sum passes u·S. No row is sorted.
// A histogram over y = (highest - x) · log2 e / t holds the count and the sum
// of weights of each bin; the bin in which a count or a sum is reached is
// looked up in it, and only few candidates are taken further: those through the
// cut's bin where they fit the LDS, else those of that one bin.
//
// Weights are exp2 in f64, to 2^-48 of each, and summed as integers, so a sum is
// the same in any order and the ids do not depend on how the work falls. A bin
// counts in units of its own, 2^-shift of the power of two above its weights
// (shift = 62 less the bits of n, at most 50: 45 at a vocabulary of 131071);
// sums over bins are in units of 2^-60 of the whole sum or less. Weights below
// 2^-80 count as none.
//
// Rows of ordinary length go a workgroup each, in one launch. Few long ones go in
// three, cut in chunks until there is one for each compute unit: chunks' highest
// and lowest values; their histograms, added to the row's, with each chunk's first
// candidates; then a workgroup a row. Temperatures count as 1e-38 at least. Lists
// are bounded where they are written, not by what was counted alone: a row that
// another stream writes meanwhile gives some id, and nothing past an array.
//
// Measured: 200 rows of 50257 with cuts 49 us (the first pass 6, at 6.7 TB/s; the
// histogram 13, its vector operations, about 30 a value; 5 for each list taken from
// the row; latencies the rest); 32 of 131072 with top-p 36 (7, 17 and 12); one of
// 49152 with top-k 40 and top-p 20.7 (4, 8 and 8).
#include "../../include/tensomite_hip.h"
#include "tmh_device.h"
#include "tmh_internal.h"

#include <algorithm>

namespace tmh {

namespace {

typedef unsigned long long u64;

constexpr uint32_t THREADS = 1024, WAVES = THREADS / 64;
constexpr uint32_t BINS = 2048;  // of y, two a thread
constexpr uint32_t ZOOM = 1024;  // finer ones, of keys, one a thread
constexpr uint32_t LIST = 4096;  // candidates held in LDS
constexpr uint32_t FEW = 64;     // of which so many are put in order, one a lane
constexpr uint32_t FIRST = 512;  // a chunk's first candidates, for the row's list

// v of the lane `CTRL` says, 0 where there is none or the row is not in MASK.
template <int CTRL, int MASK>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, MASK, 0xF, true);
}

// v of the lane n before this one among its sixteen, in a ring.
template <int N>
__device__ __forceinline__ uint32_t ring(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x120 + N, 0xF, 0xF, false);
}

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
    template <int N>
    __device__ __forceinline__ void take_ring() {
        Extent o;
        o.high = __uint_as_float(ring<N>(__float_as_uint(high)));
        o.low = __uint_as_float(ring<N>(__float_as_uint(low)));
        o.index = ring<N>(index);
        take(o);
    }
    // every sixteen lanes'
    __device__ __forceinline__ void take_sixteen() {
        take_ring<8>();
        take_ring<4>();
        take_ring<2>();
        take_ring<1>();
    }
    __device__ __forceinline__ void take_wave() {
        take_sixteen();
#pragma unroll
        for (int d = 16; d <= 32; d <<= 1) {
            Extent o;
            o.high = __shfl_xor(high, d, 64);
            o.low = __shfl_xor(low, d, 64);
            o.index = __shfl_xor(index, d, 64);
            take(o);
        }
    }
};

// A row's histogram.
struct Histogram {
    u64 sums[BINS];  // each in its bin's units
    uint32_t counts[BINS];
    u64 rough;        // their sum in the highest's units, each cut to whole ones
    u64 least;        // of the weights that min_p leaves in the bin of its border
    uint32_t border;  // that bin, or BINS: min_p leaves all
};

// A chunk's first candidates: all of its bins before `end`.
struct First {
    uint32_t count, end;
    u64 list[FIRST];  // key, then index
};

struct Sample {
    const float* x;
    uint32_t ldx, n, shift;
    uint32_t chunk, chunks, count;  // values of a chunk, chunks of a row, rows
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* ids;
    Extent* extents;  // [rows, chunks]
    Histogram* rows;
    First* firsts;  // [rows, chunks]
};

// A row's settings.
struct Settings {
    float temperature, top_p, min_p, u;
    int32_t top_k;
    __device__ __forceinline__ Settings(const Sample& a, uint32_t r)
        : temperature(a.temperature ? a.temperature[r] : 1.0f),
          top_p(a.top_p ? a.top_p[r] : 1.0f),
          min_p(a.min_p ? a.min_p[r] : 0.0f),
          u(a.u[r]),
          top_k(a.top_k ? a.top_k[r] : 0) {}
};

// Rising keys for falling values; -0 and 0 are one value.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t w = __float_as_uint(x + 0.0f);
    return w & 0x80000000u ? w : w ^ 0x7fffffffu;
}

__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key : key ^ 0x7fffffffu);
}

constexpr uint32_t MINUS_INFINITY = 0xff800000u;  // its key

// v · 2^-by, by of either sign: shifted, and cut where bits fall out.
__device__ __forceinline__ u64 scale_down(u64 v, int by) {
    return by >= 64 ? 0 : by >= 0 ? v >> by : v << -by;
}

// 2^-y for y from 0 to 64: the exponent, and 2^f by its Taylor polynomial to
// f^11 for f within half of 0 (off by less than 2^-46 of it).
__device__ __forceinline__ double exp2_minus(double y) {
    constexpr double ROUND = 6755399441055744.0;  // 1.5 · 2^52: what is added to it is rounded to integers
    const double shifted = y + ROUND;
    const double f = (shifted - ROUND - y) * 0.6931471805599453;
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
    return __builtin_bit_cast(double, __builtin_bit_cast(u64, p) - (__builtin_bit_cast(u64, shifted) << 52));
}

// A number that is the same on every lane, in a scalar register.
__device__ __forceinline__ float uniform(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(v)));
}
__device__ __forceinline__ double uniform(double v) {
    const u64 w = __builtin_bit_cast(u64, v);
    return __builtin_bit_cast(double, (u64)(uint32_t)__builtin_amdgcn_readfirstlane((int)(w >> 32)) << 32 |
                                          (uint32_t)__builtin_amdgcn_readfirstlane((int)w));
}

// A row's measure: y = (highest - x) / t in units of log 2, and its bins. Finite
// candidates no further than FLT_MAX and 2^-80 of the weight from the highest are
// within it, or where that is infinite all that are; NaN and -inf are not.
struct Measure {
    float top, highest, lowest, scale, per_y;  // the highest as it is, and FLT_MAX at most
    double exact, bin_y, bin_x;  // the scale in f64; a bin's y and x
    double series[6];            // (-exact · ln 2)^k / k!, k from 1
    uint32_t shift;

    __device__ __forceinline__ Measure(const Extent& e, float temperature, uint32_t bits) {
        constexpr float MOST = 3.4028234663852886e38f;
        exact = uniform(1.4426950408889634 / (double)fminf(fmaxf(temperature, 1e-38f), MOST));
        scale = uniform((float)exact);
        const float span = (e.high - e.low) * scale;  // infinite or none where the highest is infinite
        const float end = span <= 80.0f ? span : 80.0f;
        top = uniform(e.high), highest = uniform(fminf(e.high, MOST));
        lowest = uniform(e.high > MOST   ? e.high
                         : span <= 80.0f ? e.low
                                         : (float)fmax((double)e.low, (double)e.high - fmin(80.0 / exact, (double)MOST)));
        shift = bits;
        per_y = uniform(end > 0.0f ? fminf((float)BINS / end, 1e30f) : 0.0f);
        bin_y = uniform(end > 0.0f ? 1.0 / (double)per_y : 0.0);
        bin_x = uniform(bin_y / exact);
        const double ln = -0.6931471805599453 * exact;
        series[0] = ln;
#pragma unroll
        for (int k = 1; k < 6; ++k) series[k] = series[k - 1] * ln * (1.0 / (k + 1));
#pragma unroll
        for (int k = 0; k < 6; ++k) series[k] = uniform(series[k]);
    }
    __device__ __forceinline__ bool within(float x) const { return x >= lowest; }
    // The bin of a candidate: rises as x falls, so bins stand in their order.
    __device__ __forceinline__ uint32_t bin(float x) const {
        return min((uint32_t)((highest - fminf(x, highest)) * scale * per_y), BINS - 1u);
    }
    // Where a bin begins, about: any number of f64 near there would do.
    __device__ __forceinline__ double begin(uint32_t bin) const { return __builtin_fma((double)bin, -bin_x, (double)highest); }
    // A bin's unit is 2^-(shift + power). A weight is that at the bin's beginning
    // times e^-(begin - x) / t, whose exponent (at most 80 / BINS in units of log 2)
    // Taylor's polynomial to the sixth power takes to within 2^-48 of it.
    __device__ __forceinline__ uint32_t power(uint32_t bin) const { return (uint32_t)((double)bin * bin_y); }
    __device__ __forceinline__ double weight_of_begin(uint32_t bin, double begin) const {
        return exp2_minus(((double)highest - begin) * exact - (double)power(bin)) * (double)((u64)1 << shift);
    }
    __device__ __forceinline__ double scaled(float x, double begin, double weight_of_begin) const {
        const double d = begin - (double)fminf(x, highest);
        double p = series[5];
#pragma unroll
        for (int k = 4; k >= 0; --k) p = __builtin_fma(p, d, series[k]);
        return weight_of_begin * __builtin_fma(p, d, 1.0);
    }
    __device__ __forceinline__ double scaled(float x, uint32_t bin) const {
        const double b = begin(bin);
        return scaled(x, b, weight_of_begin(bin, b));
    }
    // To the nearest integer (at most 2^50), in the low bits of a number of 2^52,
    // whose own bits are BIAS.
    static constexpr u64 BIAS = 0x4330000000000000ull;
    static __device__ __forceinline__ u64 biased(double scaled) {
        return (u64)__builtin_bit_cast(long long, scaled + 4503599627370496.0);
    }
    __device__ __forceinline__ u64 weight(float x, uint32_t bin) const { return biased(scaled(x, bin)) - BIAS; }
    __device__ __forceinline__ u64 weight(float x) const { return weight(x, bin(x)); }
    // Whether the weight of x is at least `least` of the highest's.
    __device__ __forceinline__ bool reaches(float x, float least) const {
        if (!within(x)) return false;
        const uint32_t b = bin(x);
        return scaled(x, b) >= __builtin_ldexp((double)least, (int)(shift + power(b)));
    }
    // The first key (of a value not above the highest) for which `past` is true,
    // by 64 keys a round, by one wave (sixteen at once would wait for each other);
    // past is false, then true, and -inf's key is past.
    template <class PAST>
    __device__ __forceinline__ uint32_t search(uint32_t low, uint32_t high, PAST past) const {
        const uint32_t lane = threadIdx.x & 63u;
        while (low < high) {
            const uint32_t step = (high - low - 1u) / 64u + 1u;
            const u64 at = (u64)low + (u64)step * lane;
            const uint64_t ones = __ballot(at >= high || past((uint32_t)at));
            const uint32_t n = ones ? (uint32_t)__ffsll((unsigned long long)ones) - 1u : 64u;
            if (n == 0) return low;
            high = (uint32_t)min((u64)high, (u64)low + (u64)step * n);
            low = low + step * (n - 1u) + 1u;
        }
        return low;
    }
    // The first key whose bin is `from` or after it (keys not within are after all
    // bins): near where the bin should begin, else among all.
    __device__ __forceinline__ uint32_t first_key(uint32_t from) const {
        const auto past = [&](uint32_t key) {
            const float x = value_of(key);
            return !within(x) || bin(x) >= from;
        };
        const uint32_t first = key_of(top), guess = key_of(highest - (float)from / per_y / scale);
        uint32_t low = max(first, guess - min(guess, 2048u)), high = min(MINUS_INFINITY, guess + 2047u);
        const bool near = low < high && (low == first || !past(low)) && (high == MINUS_INFINITY || past(high));
        if (!__all(near)) low = first, high = MINUS_INFINITY;
        return search(low, high, past);
    }
    // The first key whose weight is below `least` of the highest's.
    __device__ __forceinline__ uint32_t first_below(float least) const {
        return search(key_of(top), MINUS_INFINITY, [&](uint32_t key) { return !reaches(value_of(key), least); });
    }
    // The bin of a key, BINS where it is not within.
    __device__ __forceinline__ uint32_t bin_of_key(uint32_t key) const {
        const float x = value_of(key);
        return key < MINUS_INFINITY && within(x) ? bin(x) : BINS;
    }
};

// Where a count or a sum is reached: the bin, what stands before it and what it
// holds (`own`: in its units); then the candidate, and the sum through it.
struct Found {
    uint32_t bin, count_before, count, index;
    u64 sum_before, sum_of, own, sum;
};

struct Lds {
    u64 zoom_sums[ZOOM];
    u64 list[LIST];  // key, then index
    u64 few[FEW];    // those of them the target is among
    u64 weights[FEW], sums_before[FEW];
    uint32_t counts_before[FEW];
    uint32_t zoom_counts[ZOOM];
    u64 wave_sum[WAVES];
    uint32_t wave_count[WAVES];
    Extent waves[WAVES];
    Found found;
    uint32_t listed, picked;
    uint32_t keys[2];  // the first of a bin, and of the next
};

// One step of the wave's running sums.
template <int CTRL, int MASK>
__device__ __forceinline__ void scan_step(uint32_t& c, u64& s) {
    c += dpp<CTRL, MASK>(c);
    s += (u64)dpp<CTRL, MASK>((uint32_t)(s >> 32)) << 32 | dpp<CTRL, MASK>((uint32_t)s);
}

// Running sums of the wave's lanes.
__device__ __forceinline__ void scan_wave(uint32_t& c, u64& s) {
    scan_step<0x111, 0xF>(c, s);  // 1, 2, 4 and 8 lanes back within each 16
    scan_step<0x112, 0xF>(c, s);
    scan_step<0x114, 0xF>(c, s);
    scan_step<0x118, 0xF>(c, s);
    scan_step<0x142, 0xA>(c, s);  // lane 15's to the next 16, lane 31's to the upper half
    scan_step<0x143, 0xC>(c, s);
}

// Replaces count and sum by what the threads before this one hold of them;
// all and total are everyone's.
__device__ __forceinline__ void scan(u64* wave_sum, uint32_t* wave_count, uint32_t& count, u64& sum, uint32_t& all, u64& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t c = count;
    u64 s = sum;
    scan_wave(c, s);
    __syncthreads();
    if (lane == 63u) wave_count[wave] = c, wave_sum[wave] = s;
    __syncthreads();
    uint32_t cb = 0;
    u64 sb = 0;
    all = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) {
        if (w == wave) cb = all, sb = total;
        all += wave_count[w], total += wave_sum[w];
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
    u64 sums[PER], own[PER], sum_before;

    // The bin that the target is in, into l.found.
    __device__ __forceinline__ void find(Lds& l, Target t) const {
        uint32_t c = count_before;
        u64 s = sum_before;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            if (t.in(c, counts[i], s, sums[i])) {
                l.found.bin = threadIdx.x * PER + i;
                l.found.count_before = c, l.found.count = counts[i];
                l.found.sum_before = s, l.found.sum_of = sums[i], l.found.own = own[i];
            }
            c += counts[i], s += sums[i];
        }
        __syncthreads();
    }
};

// The bin of the finer histogram that the target is in, into l.found.
__device__ __forceinline__ void find_zoomed(Lds& l, Target t, uint32_t count, u64 sum) {
    Bins<1> bins;
    uint32_t all;
    u64 total;
    bins.counts[0] = bins.count_before = l.zoom_counts[threadIdx.x];
    bins.sums[0] = bins.own[0] = bins.sum_before = l.zoom_sums[threadIdx.x];
    scan(l.wave_sum, l.wave_count, bins.count_before, bins.sum_before, all, total);
    bins.count_before += count, bins.sum_before += sum;
    bins.find(l, t);
}

struct alignas(4) Values {
    float v[4];
};

// A row, or a chunk of it, in memory: each() hands every value with its index to
// `take`, over the workgroup, four a load (of any alignment), AHEAD loads a
// thread in flight.
struct InMemory {
    const float* row;
    uint32_t from, to;
    static constexpr uint32_t STEP = 4u * THREADS;

    // the end of its whole fours
    __device__ __forceinline__ uint32_t whole() const { return to - (to - from) % 4u; }
    template <uint32_t AHEAD>
    __device__ __forceinline__ void load(Values (&x)[AHEAD], uint32_t j, uint32_t end) const {
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i)
            if (j + i * STEP < end) x[i] = *reinterpret_cast<const Values*>(row + j + i * STEP);
    }
    template <uint32_t AHEAD, class TAKE>
    __device__ __forceinline__ void each(TAKE take) const {
        const uint32_t end = whole();
        for (uint32_t j = from + 4u * threadIdx.x; j < end; j += AHEAD * STEP) {
            Values x[AHEAD];
            load<AHEAD>(x, j, end);
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i) {
                if (j + i * STEP >= end) break;
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) take(x[i].v[k], j + i * STEP + k);
            }
        }
        if (threadIdx.x < to - end) take(row[end + threadIdx.x], end + threadIdx.x);
    }
};

// The first keys of a bin and of the next, into l.keys, by a wave each.
__device__ __forceinline__ void find_keys(Lds& l, const Measure& m, uint32_t bin) {
    const uint32_t wave = threadIdx.x >> 6;
    if (wave < 2u) {
        const uint32_t key = m.first_key(bin + wave);
        if ((threadIdx.x & 63u) == 0) l.keys[wave] = key;
    }
    __syncthreads();
}

// Lists the candidates with values from `low` to `high`: all of them counted in
// l.listed, LIST at most in the list. A lane counts what 32 values hold, a wave
// takes its places at once, and then they are written.
__device__ __forceinline__ void list_values(Lds& l, const InMemory& row, float low, float high) {
    constexpr uint32_t AHEAD = 8;
    const float NONE = __builtin_nanf("");
    const auto put = [&](uint32_t at, float v, uint32_t j) {
        if (at < LIST) l.list[at] = (u64)key_of(v) << 32 | j;
    };
    if (threadIdx.x == 0) l.listed = 0;
    __syncthreads();
    const uint32_t end = row.whole();
    for (uint32_t j = row.from + 4u * threadIdx.x; j < end; j += AHEAD * InMemory::STEP) {
        Values x[AHEAD];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) x[i] = Values{{NONE, NONE, NONE, NONE}};
        row.load<AHEAD>(x, j, end);
        uint32_t mine = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4u * AHEAD; ++i) mine += x[i / 4u].v[i % 4u] >= low && x[i / 4u].v[i % 4u] <= high ? 1u : 0u;
        if (!__any(mine != 0)) continue;
        // the lanes here are the wave's first ones
        uint32_t through = mine;
        u64 none = 0;
        scan_wave(through, none);
        const int last = 63 - __clzll((long long)__ballot(true));
        uint32_t at = 0;
        if ((threadIdx.x & 63u) == 0) at = atomicAdd(&l.listed, (uint32_t)__builtin_amdgcn_readlane((int)through, last));
        at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + through - mine;
#pragma unroll
        for (uint32_t i = 0; i < 4u * AHEAD; ++i) {
            const float v = x[i / 4u].v[i % 4u];
            if (v >= low && v <= high) put(at++, v, j + i / 4u * InMemory::STEP + i % 4u);
        }
    }
    if (threadIdx.x < row.to - end) {
        const float v = row.row[end + threadIdx.x];
        if (v >= low && v <= high) put(atomicAdd(&l.listed, 1u), v, end + threadIdx.x);
    }
    __syncthreads();
}

// Lists the candidates through bin `last` from what the chunks' lists hold; false
// where one of them ends before that.
__device__ __forceinline__ bool list_firsts(Lds& l, const Measure& m, const First* chunks, uint32_t n, uint32_t last) {
    const uint32_t lane = threadIdx.x & 63u;
    bool all = true;
    for (uint32_t c = lane; c < n; c += 64u) all &= chunks[c].end > last;
    if (!__all(all)) return false;
    if (threadIdx.x == 0) l.listed = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n * FIRST; i += THREADS) {
        const First& f = chunks[i / FIRST];
        if (i % FIRST >= f.count) continue;
        const u64 c = f.list[i % FIRST];
        if (m.bin(value_of((uint32_t)(c >> 32))) > last) continue;
        const uint32_t at = atomicAdd(&l.listed, 1u);
        if (at < LIST) l.list[at] = c;
    }
    __syncthreads();
    return true;
}

// Candidates one a lane of the first wave, with what stands before each in their
// order, which all waves find. Their weights are in units of 2^-FINE, or where
// they are of one bin in its.
constexpr int FINE = 56;
struct Few {
    u64 mine, weight, sum;
    uint32_t n, count;

    __device__ __forceinline__ Few(Lds& l, const u64* from, uint32_t size, const Measure& m, bool one_bin,
                                   uint32_t before, u64 sum_before)
        : mine(~0ull), weight(0), sum(0), n(size), count(0) {
        const uint32_t lane = threadIdx.x & 63u;
        if (threadIdx.x < 64u) {
            if (lane < n) {
                mine = from[lane];
                const float x = value_of((uint32_t)(mine >> 32));
                const uint32_t bin = m.bin(x);
                weight = scale_down(m.weight(x, bin), one_bin ? 0 : (int)(m.shift + m.power(bin)) - FINE);
            }
            l.weights[lane] = weight, l.sums_before[lane] = sum_before, l.counts_before[lane] = before;
        }
        __syncthreads();
        if (lane < n) {
            const u64 of = from[lane];
            for (uint32_t j = threadIdx.x >> 6; j < n; j += WAVES)
                if (from[j] < of) count += 1u, sum += l.weights[j];
            if (count) atomicAdd(&l.counts_before[lane], count), atomicAdd(&l.sums_before[lane], sum);
        }
        __syncthreads();
        sum = l.sums_before[lane], count = l.counts_before[lane];
    }
    static __device__ __forceinline__ u64 one(u64 v, uint32_t lane) {
        return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), (int)lane) << 32 |
               (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane);
    }
    // The index of the candidate that the target is in, and the sum through it.
    __device__ __forceinline__ uint32_t find(Target t, u64& through) const {
        const uint64_t is = __ballot((threadIdx.x & 63u) < n && t.in(count, 1, sum, weight));
        const uint32_t lane = is ? (uint32_t)__ffsll((unsigned long long)is) - 1u : 0u;
        through = one(sum + weight, lane);
        return (uint32_t)one(mine, lane);
    }
};

// The candidate that the target is in among the listed that `is` holds for, n of
// them, FEW at most, with count and sum before them; and the sum through it.
template <class IS>
__device__ __forceinline__ void find_few(Lds& l, const Measure& m, Target t, uint32_t n, uint32_t count, u64 sum, IS is) {
    const uint32_t listed = l.listed;
    if (threadIdx.x == 0) l.picked = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < listed; i += THREADS) {
        if (!is(l.list[i])) continue;
        const uint32_t at = atomicAdd(&l.picked, 1u);
        if (at < FEW) l.few[at] = l.list[i];
    }
    __syncthreads();
    const Few few(l, l.few, min(n, FEW), m, true, count, sum);
    if (threadIdx.x < 64u) {
        u64 through;
        const uint32_t index = few.find(t, through);
        if (threadIdx.x == 0) l.found.index = index, l.found.sum = through;
    }
    __syncthreads();
}

// The candidate that the target is in among the listed (at most LIST) with keys
// from low to high, which are as many and have as much before them as l.found
// says, and the sum through it, into l.found: by histograms of ever fewer keys
// and indices until a wave can put what is left in order.
__device__ __forceinline__ void find_listed(Lds& l, const Measure& m, Target t, uint32_t key_low, uint32_t key_high) {
    const uint32_t listed = l.listed;
    u64 low = (u64)key_low << 32, high = (u64)key_high << 32 | 0xffffffffu, sum = l.found.sum_before;
    uint32_t n = l.found.count, count = l.found.count_before;
    while (n > FEW && low < high) {
        uint32_t shift = 0;
        while (((high - low) >> shift) >= ZOOM) ++shift;
        __syncthreads();
        l.zoom_counts[threadIdx.x] = 0, l.zoom_sums[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < listed; i += THREADS) {
            const u64 c = l.list[i];
            if (c >= low && c <= high) {
                atomicAdd(&l.zoom_counts[(uint32_t)((c - low) >> shift)], 1u);
                atomicAdd(&l.zoom_sums[(uint32_t)((c - low) >> shift)], m.weight(value_of((uint32_t)(c >> 32))));
            }
        }
        __syncthreads();
        find_zoomed(l, t, count, sum);
        count = l.found.count_before, sum = l.found.sum_before, n = l.found.count;
        low += (u64)l.found.bin << shift;
        high = min(high, low + ((u64)1 << shift) - 1u);
    }
    find_few(l, m, t, n, count, sum, [&](u64 c) { return c >= low && c <= high; });
}

// The candidate that the target is in among those of the value of `key`, by index:
// more of them than the list holds.
__device__ __forceinline__ void find_equal(Lds& l, const Measure& m, const InMemory& row, Target t, uint32_t key) {
    const u64 sum = l.found.sum_before, weight = m.weight(value_of(key));
    const u64 place = t.by_sum ? (t.target - sum) / weight : t.target - l.found.count_before;
    uint32_t before = 0;
    for (uint32_t base = 0; base < row.to; base += THREADS) {
        const uint32_t j = base + threadIdx.x;
        const bool is = j < row.to && key_of(row.row[j]) == key;
        uint32_t c = is ? 1u : 0u, all;
        u64 s = 0, total;
        scan(l.wave_sum, l.wave_count, c, s, all, total);
        if (is && before + c == place) l.found.index = j, l.found.sum = sum + (place + 1u) * weight;
        before += all;
    }
    __syncthreads();
}

// The candidate that the target is in, and the sum through it, into l.found;
// the target's bin is there, in common units and its own, `finer` bits below
// those. `listed`: the bin's candidates are.
__device__ __forceinline__ void find_in_bin(Lds& l, const Measure& m, const InMemory& row, Target t, int finer, bool listed) {
    const uint32_t bin = l.found.bin;
    const u64 common_before = l.found.sum_before, common = l.found.sum_of;
    if (t.by_sum) t.target = min(scale_down(t.target - common_before, -finer), l.found.own - 1u);
    if (listed && l.found.count <= FEW) {
        const uint32_t n = l.found.count, count = l.found.count_before;
        find_few(l, m, t, n, count, 0, [&](u64 c) { return m.bin(value_of((uint32_t)(c >> 32))) == bin; });
    } else {
        __syncthreads();
        if (threadIdx.x == 0) l.found.sum_before = 0;
        find_keys(l, m, bin);
        uint32_t low = l.keys[0], high = l.keys[1] - 1u;
        // more than the list holds: histograms of ever fewer keys
        while (l.found.count > LIST && low < high) {
            uint32_t shift = 0;
            while (((high - low) >> shift) >= ZOOM) ++shift;
            __syncthreads();
            l.zoom_counts[threadIdx.x] = 0, l.zoom_sums[threadIdx.x] = 0;
            __syncthreads();
            row.each<4>([&](float x, uint32_t) {
                const uint32_t key = key_of(x);
                if (key >= low && key <= high) {
                    atomicAdd(&l.zoom_counts[(key - low) >> shift], 1u);
                    atomicAdd(&l.zoom_sums[(key - low) >> shift], m.weight(x));
                }
            });
            __syncthreads();
            find_zoomed(l, t, l.found.count_before, l.found.sum_before);
            low += l.found.bin << shift;
            high = min(high, low + (1u << shift) - 1u);
        }
        if (l.found.count <= LIST) {
            if (!listed) list_values(l, row, value_of(high), value_of(low));
            find_listed(l, m, t, low, high);
        } else {
            find_equal(l, m, row, t, low);
        }
    }
    if (threadIdx.x == 0) l.found.sum = common_before + min(scale_down(l.found.sum, finer), common);
    __syncthreads();
}

// The highest and lowest values of a row or chunk, into `waves`: every wave's.
__device__ __forceinline__ void find_extent(Extent* waves, const InMemory& row) {
    Extent e{-INFINITY, INFINITY, ~0u};
    row.each<4>([&](float x, uint32_t j) {
        if (x == x && (e.index == ~0u || x > e.high)) e.high = x, e.index = j;
        if (x > -INFINITY) e.low = fminf(e.low, x);
    });
    e.take_wave();
    if ((threadIdx.x & 63u) == 0) waves[threadIdx.x >> 6] = e;
    __syncthreads();
}

// Whether a row is to be sampled at all, and what it has if not: its highest
// value's index, as tmh_argmax chooses it.
__device__ __forceinline__ bool sampled(float temperature, const Extent& e) {
    return temperature > 0.0f && e.high > -INFINITY;
}

__device__ __forceinline__ void take_highest(const Sample& a, uint32_t r, const Extent& e) {
    if (threadIdx.x != 0) return;
    const float first = a.x[(size_t)r * a.ldx];
    a.ids[r] = first != first || e.index == ~0u ? 0 : (int32_t)e.index;
}

// What a histogram is made in, in LDS.
struct Counting {
    Histogram h;
    double begins[BINS];  // the weights at the bins' beginnings
    uint32_t below;        // the first key whose weight is below min_p

    // The histogram of a row or chunk.
    __device__ __forceinline__ void count(const Measure& m, const InMemory& row, float least) {
        constexpr uint32_t PER = BINS / THREADS;
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            const uint32_t b = threadIdx.x + i * THREADS;
            h.sums[b] = 0, h.counts[b] = 0, begins[b] = m.weight_of_begin(b, m.begin(b));
        }
        if (threadIdx.x < 64u) {
            const uint32_t key = least <= 0.0f ? MINUS_INFINITY : m.first_below(least);
            if (threadIdx.x == 0) h.least = 0, h.rough = 0, below = key, h.border = m.bin_of_key(key);
        }
        __syncthreads();
        const uint32_t border = h.border;
        const float first_below = value_of(below);
        u64 kept = 0;
        row.each<4>([&](float x, uint32_t) {
            if (m.within(x)) {
                const uint32_t bin = m.bin(x);
                const u64 weight = m.biased(m.scaled(x, m.begin(bin), begins[bin]));
                atomicAdd(&h.counts[bin], 1u);
                atomicAdd(&h.sums[bin], weight);
                if (bin == border && x > first_below) kept += weight - m.BIAS;
            }
        });
        if (border < BINS) add(h.least, kept);
        __syncthreads();
        u64 rough = 0;
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) {
            const uint32_t b = threadIdx.x + i * THREADS;
            const u64 sum = h.sums[b] - h.counts[b] * m.BIAS;  // modulo 2^64
            h.sums[b] = sum;
            rough += scale_down(sum, (int)m.power(b));
        }
        add(h.rough, rough);
        __syncthreads();
    }
    static __device__ __forceinline__ void add(u64& to, u64 v) {
        uint32_t none = 0;
        scan_wave(none, v);
        if ((threadIdx.x & 63u) == 63u) atomicAdd(&to, v);
    }
};

// A row's histogram: this thread's bins of it, and what is the whole row's.
struct Whole {
    static constexpr uint32_t PER = BINS / THREADS;
    u64 own[PER], rough, least;
    uint32_t counts[PER], border;

    __device__ __forceinline__ Whole(const Histogram& h) : rough(h.rough), least(h.least), border(h.border) {
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) own[i] = h.sums[threadIdx.x * PER + i], counts[i] = h.counts[threadIdx.x * PER + i];
    }
};

// The cuts and the choice of row r from its histogram, by a workgroup.
__device__ __forceinline__ void choose(const Sample& a, uint32_t r, Lds& l, const Settings& set, const Measure& m,
                                       const InMemory& row, const Whole& h, const First* firsts, uint32_t chunks) {
    constexpr uint32_t PER = Whole::PER;
    // Common units of 2^-common: the sum of all weights, less than twice what it
    // roughly is, stays below 2^62 of them. A bin's own are finer by so many bits.
    const int bits = 65 - __clzll((long long)h.rough), common = 62 + (int)m.shift - bits;
    const auto finer = [&](uint32_t bin) { return (int)(m.shift + m.power(bin)) - common; };
    Bins<PER> bins;
    bins.count_before = 0, bins.sum_before = 0;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        bins.counts[i] = h.counts[i], bins.own[i] = h.own[i];
        bins.sums[i] = scale_down(h.own[i], finer(threadIdx.x * PER + i));
        bins.count_before += bins.counts[i], bins.sum_before += bins.sums[i];
    }
    uint32_t all;
    u64 total;
    scan(l.wave_sum, l.wave_count, bins.count_before, bins.sum_before, all, total);
    // the prefix that stays is the shortest of three: the sums through the
    // k-th, through the first to reach p, and of weights of at least min_p
    const bool cut_k = set.top_k > 0 && (uint32_t)set.top_k < all, cut_p = !(set.top_p >= 1.0f);
    u64 least_sum = ~0ull;
    if (h.border < BINS) {
        if (threadIdx.x == h.border / PER) {
            u64 before = bins.sum_before;
#pragma unroll
            for (uint32_t i = 0; i < PER; ++i) before += threadIdx.x * PER + i < h.border ? bins.sums[i] : 0;
            l.found.sum = before + scale_down(h.least, finer(h.border));
        }
        __syncthreads();
        least_sum = l.found.sum;
    }
    const Target kth{false, (u64)set.top_k - 1u};
    // the first to reach p of a sum, the first to pass u of it
    const auto reach = [&](double of) {
        const double sum = (double)set.top_p * of;
        return Target{true, sum > 0.0 ? (u64)__builtin_ceil(sum) - 1u : 0};
    };
    const auto choice = [&](u64 of) {
        const double sum = (double)set.u * (double)of;
        return Target{true, sum > 0.0 ? min((u64)sum, of - 1u) : sum == sum ? 0 : of - 1u};
    };
    bool listed = false;
    if (cut_k || cut_p) {
        bins.find(l, cut_k ? kth : reach((double)total));
        if (l.found.count_before + l.found.count <= LIST) {
            // the candidates through the cut's bin: of them from here on
            listed = true;
            if (chunks == 0 || !list_firsts(l, m, firsts, chunks, l.found.bin)) {
                find_keys(l, m, l.found.bin);
                list_values(l, row, value_of(l.keys[1] - 1u), m.top);
            }
            if (l.listed <= FEW) {
                const Few few(l, l.list, l.listed, m, false, 0, 0);
                if (threadIdx.x < 64u) {
                    // in units of 2^-FINE
                    u64 through, left = ~0ull;
                    double of = __builtin_ldexp((double)total, FINE - common);
                    if (cut_k) few.find(kth, left), of = (double)left;
                    if (cut_p) few.find(reach(of), through), left = min(left, through);
                    if (least_sum != ~0ull)
                        left = min(left, (u64)fmin(__builtin_ldexp((double)least_sum, FINE - common), 9.0e18));
                    const uint32_t index = few.find(choice(max(left, (u64)1 << FINE)), through);
                    if (threadIdx.x == 0) a.ids[r] = (int32_t)index;
                }
                return;
            }
        }
    }
    const auto find = [&](Target t) {
        bins.find(l, t);
        find_in_bin(l, m, row, t, finer(l.found.bin), listed);
    };
    if (cut_k) find(kth), total = l.found.sum;
    if (cut_p) find(reach((double)total)), total = min(total, l.found.sum);
    total = min(total, least_sum);
    // the highest always stays
    find(choice(max(total, scale_down((u64)1 << m.shift, (int)m.shift - common))));
    if (threadIdx.x == 0) a.ids[r] = (int32_t)l.found.index;
}

// The highest and lowest values of chunk blockIdx.y of row blockIdx.x, whose
// share of the row's histogram it clears. Rows stand first in the grid, up to
// a multiple of eight: a row's chunks then meet on one XCD, whose L2 holds the
// row for the later launches.
__global__ __launch_bounds__(1024) void k_sample_extent(Sample a) {
    __shared__ Extent waves[WAVES];
    const uint32_t r = blockIdx.x, chunk = blockIdx.y;
    if (r >= a.count) return;
    find_extent(waves, InMemory{a.x + (size_t)r * a.ldx, chunk * a.chunk, min(chunk * a.chunk + a.chunk, a.n)});
    Histogram& h = a.rows[r];
    for (uint32_t b = chunk * THREADS + threadIdx.x; b < BINS; b += a.chunks * THREADS) h.sums[b] = 0, h.counts[b] = 0;
    if (threadIdx.x == 0) {
        if (chunk == 0) h.least = 0, h.rough = 0;
        Extent e = waves[0];
        for (uint32_t w = 1; w < WAVES; ++w) e.take(waves[w]);
        a.extents[(size_t)r * a.chunks + chunk] = e;
    }
}

// A row's extent from its chunks' or its waves'.
__device__ __forceinline__ Extent join_extents(const Extent* parts, uint32_t count) {
    Extent e{-INFINITY, INFINITY, ~0u};
    if (count <= 16u) {
        if ((threadIdx.x & 15u) < count) e = parts[threadIdx.x & 15u];
        e.take_sixteen();
        return e;
    }
    for (uint32_t c = threadIdx.x & 63u; c < count; c += 64u) e.take(parts[c]);
    e.take_wave();
    return e;
}

// The histogram of chunk blockIdx.y of row blockIdx.x, added to the row's, and
// where a cut may come the chunk's first candidates.
__global__ __launch_bounds__(1024) void k_sample_histogram(Sample a) {
    __shared__ Counting counting;
    __shared__ u64 wave_sum[WAVES];
    __shared__ uint32_t wave_count[WAVES], end, listed;
    constexpr uint32_t PER = BINS / THREADS;
    const uint32_t r = blockIdx.x, chunk = blockIdx.y;
    if (r >= a.count) return;
    const Settings set(a, r);
    const Extent e = join_extents(a.extents + (size_t)r * a.chunks, a.chunks);
    if (!sampled(set.temperature, e)) return;
    const Measure m(e, set.temperature, a.shift);
    const InMemory part{a.x + (size_t)r * a.ldx, chunk * a.chunk, min(chunk * a.chunk + a.chunk, a.n)};
    counting.count(m, part, set.min_p);
    Histogram& h = a.rows[r];
    if (threadIdx.x == 0) {
        atomicAdd(&h.rough, counting.h.rough);
        if (counting.h.least) atomicAdd(&h.least, counting.h.least);
        if (chunk == 0) h.border = counting.h.border;
        end = BINS, listed = 0;
    }
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t b = threadIdx.x + i * THREADS;
        if (counting.h.counts[b]) {
            atomicAdd(&h.counts[b], counting.h.counts[b]);
            if (counting.h.sums[b]) atomicAdd(&h.sums[b], counting.h.sums[b]);
        }
    }
    if (set.top_k <= 0 && set.top_p >= 1.0f) return;
    uint32_t count = 0, all;
    u64 none = 0, total;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) count += counting.h.counts[threadIdx.x * PER + i];
    scan(wave_sum, wave_count, count, none, all, total);
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t b = threadIdx.x * PER + i, of = counting.h.counts[b];
        if (count <= FIRST && count + of > FIRST) end = b;
        count += of;
    }
    __syncthreads();
    First& first = a.firsts[(size_t)r * a.chunks + chunk];
    const uint32_t before = end;
    part.each<2>([&](float x, uint32_t j) {
        if (!m.within(x) || m.bin(x) >= before) return;
        const uint32_t at = atomicAdd(&listed, 1u);
        if (at < FIRST) first.list[at] = (u64)key_of(x) << 32 | j;
    });
    __syncthreads();
    if (threadIdx.x == 0) first.count = listed, first.end = before;
}

// A row from its histogram.
__global__ __launch_bounds__(1024) void k_sample_choose(Sample a) {
    __shared__ Lds l;
    const uint32_t r = blockIdx.x;
    const Settings set(a, r);
    const Extent e = join_extents(a.extents + (size_t)r * a.chunks, a.chunks);
    if (!sampled(set.temperature, e)) {
        take_highest(a, r, e);
        return;
    }
    const Whole h(a.rows[r]);
    const Measure m(e, set.temperature, a.shift);
    choose(a, r, l, set, m, InMemory{a.x + (size_t)r * a.ldx, 0, a.n}, h, a.firsts + (size_t)r * a.chunks, a.chunks);
}

// A whole row by one workgroup.
__global__ __launch_bounds__(1024) void k_sample_row(Sample a) {
    extern __shared__ u64 lds_words[];
    Counting& counting = *reinterpret_cast<Counting*>(lds_words);
    Lds& l = *reinterpret_cast<Lds*>(&counting + 1);
    const uint32_t r = blockIdx.x;
    const InMemory row{a.x + (size_t)r * a.ldx, 0, a.n};
    const Settings set(a, r);
    find_extent(l.waves, row);
    const Extent e = join_extents(l.waves, WAVES);
    if (!sampled(set.temperature, e)) {
        take_highest(a, r, e);
        return;
    }
    const Measure m(e, set.temperature, a.shift);
    counting.count(m, row, set.min_p);
    choose(a, r, l, set, m, row, Whole(counting.h), nullptr, 0);
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
    Sample a{(const float*)x, ldx, n, std::min(62u - bits, 50u), n, 1, rows, (const float*)temperature,
             (const int32_t*)top_k, (const float*)top_p, (const float*)min_p, (const float*)u, (int32_t*)ids, nullptr,
             nullptr};
    // a chunk for each compute unit, of four values a thread or more
    constexpr uint32_t LEAST = 4u * THREADS, LDS = sizeof(Counting) + sizeof(Lds);
    const uint32_t chunks = std::min((uint32_t)ctx.compute_units / rows, (n + LEAST - 1u) / LEAST);
    // One launch where a workgroup is through a row before three are (us, one launch
    // and three: 1 x 16384 18.5 and 21.6, 1 x 32768 24.2 and 22.1; 32 x 32768 25.6
    // and 27.6, 32 x 50000 32.0 and 29.7; 100 x 50000 33.2 and 36.7)
    if (chunks <= 1u || n <= 24576u + 512u * rows) {
        TMH_LAUNCH(k_sample_row, dim3(rows), dim3(THREADS), LDS, ctx.stream, a);
    } else {
        a.chunk = (n + chunks - 1u) / chunks;
        a.chunks = (n + a.chunk - 1u) / a.chunk;
        const size_t extents = ((size_t)rows * a.chunks * sizeof(Extent) + 255u) & ~(size_t)255u;
        const size_t histograms = (size_t)rows * sizeof(Histogram);
        Workspace work(ctx.index, extents + histograms + (size_t)rows * a.chunks * sizeof(First));
        if (work.status) return work.status;
        a.extents = (Extent*)work.memory;
        a.rows = (Histogram*)(work.memory + extents);
        a.firsts = (First*)(work.memory + extents + histograms);
        const dim3 grid((rows + 7u) / 8u * 8u, a.chunks);
        TMH_LAUNCH(k_sample_extent, grid, dim3(THREADS), 0, ctx.stream, a);
        TMH_LAUNCH(k_sample_histogram, grid, dim3(THREADS), 0, ctx.stream, a);
        TMH_LAUNCH(k_sample_choose, dim3(rows), dim3(THREADS), 0, ctx.stream, a);
    }
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) note_launch(ctx.index, 1, false);
    return code(e);
}

}  // extern "C"
