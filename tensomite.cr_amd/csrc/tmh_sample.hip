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
// Few rows go in three launches: chunks' highest and lowest values, chunks'
// histograms added to their row's, then a workgroup a row; rows are cut in chunks
// until there is one for each compute unit. Many rows go a workgroup each, in one
// launch. The weights' vector operations, about 40 a value, bound the histogram;
// latencies, scans and the passes over the row the rest.
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
    __device__ __forceinline__ void take_wave() {
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
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
    u64 rough;       // their sum in the highest's units, each cut to whole ones
    u64 least;       // of the weights that min_p leaves in the bin of its border
    uint32_t counts[BINS];
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

// A row's measure: its highest value, and y's scale, end and bins.
struct Measure {
    float highest, scale, cut, per_y;
    double exact, bin_y;  // the scale in f64; a bin's y
    uint32_t shift;

    __device__ __forceinline__ Measure(const Extent& e, float temperature, uint32_t bits) {
        highest = e.high;
        exact = 1.4426950408889634 / (double)temperature;
        scale = (float)exact;
        cut = fminf((e.high - e.low) * scale, 80.0f);  // the lowest's
        shift = bits;
        per_y = cut > 0.0f ? fminf((float)BINS / cut, 1e30f) : 0.0f;
        bin_y = cut > 0.0f ? 1.0 / (double)per_y : 0.0;
    }
    // y in f32 falls as x rises, so bins stand in the candidates' order; y above
    // cut is a weight of none, or no candidate's. NaN and -inf are not within it.
    __device__ __forceinline__ float y(float x) const { return x == highest ? 0.0f : (highest - x) * scale; }
    __device__ __forceinline__ bool within(float y) const { return y <= cut; }
    __device__ __forceinline__ uint32_t bin(float y) const { return min((uint32_t)(y * per_y), BINS - 1u); }
    // A bin's unit is 2^-(shift + power). A weight is that at the bin's beginning
    // times 2^-rest, the rest of y (at most 80 / BINS) by its Taylor polynomial
    // to the sixth power, off by less than 2^-48 of it.
    __device__ __forceinline__ uint32_t power(uint32_t bin) const { return (uint32_t)((double)bin * bin_y); }
    __device__ __forceinline__ double begin(uint32_t bin) const {
        return exp2_minus((double)bin * bin_y - (double)power(bin)) * (double)((u64)1 << shift);
    }
    __device__ __forceinline__ double scaled(float x, uint32_t bin, double begin) const {
        const double y = x == highest ? 0.0 : ((double)highest - (double)x) * exact;
        const double rest = __builtin_fma((double)bin, -bin_y, y);
        double p = 0.00015403530393381608;  // (-ln 2)^k / k!
        p = __builtin_fma(p, rest, -0.0013333558146428443);
        p = __builtin_fma(p, rest, 0.009618129107628477);
        p = __builtin_fma(p, rest, -0.05550410866482158);
        p = __builtin_fma(p, rest, 0.2402265069591007);
        p = __builtin_fma(p, rest, -0.6931471805599453);
        p = __builtin_fma(p, rest, 1.0);
        return begin * p;
    }
    // to the nearest integer (at most 2^50), in the low bits of a number of 2^52
    static __device__ __forceinline__ u64 whole(double scaled) {
        return (u64)__builtin_bit_cast(long long, scaled + 4503599627370496.0) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 weight(float x, uint32_t bin) const { return whole(scaled(x, bin, begin(bin))); }
    __device__ __forceinline__ u64 weight(float x) const { return weight(x, bin(y(x))); }
    // Whether the weight of x is at least `least` of the highest's.
    __device__ __forceinline__ bool reaches(float x, float least) const {
        const float v = y(x);
        if (!within(v)) return false;
        const uint32_t b = bin(v);
        return scaled(x, b, begin(b)) >= __builtin_ldexp((double)least, (int)(shift + power(b)));
    }
    // The first key (of a value not above the highest) for which `past` is true,
    // by 64 keys a round; past is false, then true, and -inf's key is past.
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
    // The first key whose bin is `from` or after it (keys not within cut are
    // after all bins): near where the bin should begin, else among all.
    __device__ __forceinline__ uint32_t first_key(uint32_t from) const {
        const auto past = [&](uint32_t key) {
            const float v = y(value_of(key));
            return !within(v) || bin(v) >= from;
        };
        const uint32_t first = key_of(highest), guess = key_of(highest - (float)from / per_y / scale);
        uint32_t low = max(first, guess - min(guess, 2048u)), high = min(MINUS_INFINITY, guess + 2047u);
        const bool near = low < high && (low == first || !past(low)) && (high == MINUS_INFINITY || past(high));
        if (!__all(near)) low = first, high = MINUS_INFINITY;
        return search(low, high, past);
    }
    // The first key whose weight is below `least` of the highest's.
    __device__ __forceinline__ uint32_t first_below(float least) const {
        return search(key_of(highest), MINUS_INFINITY, [&](uint32_t key) { return !reaches(value_of(key), least); });
    }
    // The bin of a key, BINS where it is not within cut.
    __device__ __forceinline__ uint32_t bin_of_key(uint32_t key) const {
        const float v = y(value_of(key));
        return key < MINUS_INFINITY && within(v) ? bin(v) : BINS;
    }
};

// Where a count or a sum is reached: the bin, what stands before it and what it
// holds; then the candidate, and the sum through it.
struct Found {
    uint32_t bin, count_before, count, index;
    u64 sum_before, sum_of, sum;
};

struct Lds {
    u64 zoom_sums[ZOOM];
    u64 list[LIST];  // key, then index
    u64 few[FEW];    // those of them the target is among
    uint32_t zoom_counts[ZOOM];
    u64 wave_sum[WAVES];
    uint32_t wave_count[WAVES];
    Extent waves[WAVES];
    Found found;
    uint32_t listed, picked;
};

// v of the lane `CTRL` says, 0 where there is none or the row is not in MASK.
template <int CTRL, int MASK>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, MASK, 0xF, true);
}

// One step of the wave's running sums.
template <int CTRL, int MASK>
__device__ __forceinline__ void scan_step(uint32_t& c, u64& s) {
    c += dpp<CTRL, MASK>(c);
    s += (u64)dpp<CTRL, MASK>((uint32_t)(s >> 32)) << 32 | dpp<CTRL, MASK>((uint32_t)s);
}

// Replaces count and sum by what the threads before this one hold of them;
// all and total are everyone's.
__device__ __forceinline__ void scan(Lds& l, uint32_t& count, u64& sum, uint32_t& all, u64& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t c = count;
    u64 s = sum;
    scan_step<0x111, 0xF>(c, s);  // 1, 2, 4 and 8 lanes back within each 16
    scan_step<0x112, 0xF>(c, s);
    scan_step<0x114, 0xF>(c, s);
    scan_step<0x118, 0xF>(c, s);
    scan_step<0x142, 0xA>(c, s);  // lane 15's to the next 16, lane 31's to the upper half
    scan_step<0x143, 0xC>(c, s);
    __syncthreads();
    if (lane == 63u) l.wave_count[wave] = c, l.wave_sum[wave] = s;
    __syncthreads();
    uint32_t cb = 0;
    u64 sb = 0;
    all = 0, total = 0;
#pragma unroll
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
                l.found.count_before = c, l.found.count = counts[i];
                l.found.sum_before = s, l.found.sum_of = sums[i];
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
    bins.sums[0] = bins.sum_before = l.zoom_sums[threadIdx.x];
    scan(l, bins.count_before, bins.sum_before, all, total);
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

    template <uint32_t AHEAD, class TAKE>
    __device__ __forceinline__ void each(TAKE take) const {
        constexpr uint32_t STEP = 4u * THREADS;
        uint32_t j = from + 4u * threadIdx.x;
        for (; j + (AHEAD - 1u) * STEP + 4u <= to; j += AHEAD * STEP) {
            Values x[AHEAD];
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i) x[i] = *reinterpret_cast<const Values*>(row + j + i * STEP);
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) take(x[i].v[k], j + i * STEP + k);
        }
        for (; j + 4u <= to; j += STEP) {
            const Values x = *reinterpret_cast<const Values*>(row + j);
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) take(x.v[k], j + k);
        }
        for (; j < to; ++j) take(row[j], j);
    }
};

// Lists the candidates with values from `low` to `high`: all of them counted in
// l.listed, LIST at most in the list.
__device__ __forceinline__ void list_values(Lds& l, const InMemory& row, float low, float high) {
    if (threadIdx.x == 0) l.listed = 0;
    __syncthreads();
    row.each<8>([&](float x, uint32_t j) {
        if (x >= low && x <= high) {
            const uint32_t at = atomicAdd(&l.listed, 1u);
            if (at < LIST) l.list[at] = (u64)key_of(x) << 32 | j;
        }
    });
    __syncthreads();
}

// Candidates one a lane of a wave, with what stands before each in their order.
// Their weights are in units of 2^-FINE, or where they are of one bin in its.
constexpr int FINE = 56;
struct Few {
    u64 mine, weight, sum;
    uint32_t n, count;

    __device__ __forceinline__ Few(const u64* from, uint32_t size, const Measure& m, bool one_bin, uint32_t before,
                                   u64 sum_before)
        : mine(~0ull), weight(0), sum(sum_before), n(size), count(before) {
        const uint32_t lane = threadIdx.x & 63u;
        if (lane < n) {
            mine = from[lane];
            const float x = value_of((uint32_t)(mine >> 32));
            const uint32_t bin = m.bin(m.y(x));
            weight = scale_down(m.weight(x, bin), one_bin ? 0 : (int)(m.shift + m.power(bin)) - FINE);
        }
        for (uint32_t j = 0; j < n; ++j) {
            const bool less = one(mine, j) < mine;
            count += less ? 1u : 0u;
            sum += less ? one(weight, j) : 0;
        }
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

// The candidate that the target is in among the listed (at most LIST) with keys
// from low to high, which are as many and have as much before them as l.found
// says, and the sum through it, into l.found: by histograms of ever fewer keys
// and indices until a wave can put what is left in order.
__device__ __forceinline__ void find_listed(Lds& l, const Measure& m, Target t, uint32_t key_low, uint32_t key_high) {
    const uint32_t listed = l.listed;
    u64 low = (u64)key_low << 32, high = (u64)key_high << 32 | 0xffffffffu, sum = l.found.sum_before;
    uint32_t n = l.found.count, count = l.found.count_before;
    while (n > FEW) {
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
    if (threadIdx.x == 0) l.picked = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < listed; i += THREADS) {
        const u64 c = l.list[i];
        if (c >= low && c <= high) l.few[atomicAdd(&l.picked, 1u)] = c;
    }
    __syncthreads();
    if (threadIdx.x < 64u) {
        const Few few(l.few, n, m, true, count, sum);
        u64 through;
        const uint32_t index = few.find(t, through);
        if (threadIdx.x == 0) l.found.index = index, l.found.sum = through;
    }
    __syncthreads();
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
        scan(l, c, s, all, total);
        if (is && before + c == place) l.found.index = j, l.found.sum = sum + (place + 1u) * weight;
        before += all;
    }
    __syncthreads();
}

// The candidate that the target is in, and the sum through it, into l.found;
// the target's bin is there, and its sum in its own units in `held`, `finer` bits
// below the common ones. `listed`: the bin's candidates are.
__device__ __forceinline__ void find_in_bin(Lds& l, const Measure& m, const InMemory& row, Target t, u64 held, int finer,
                                            bool listed) {
    uint32_t low = m.first_key(l.found.bin), high = m.first_key(l.found.bin + 1u) - 1u;
    const u64 common_before = l.found.sum_before, common = l.found.sum_of;
    __syncthreads();
    if (threadIdx.x == 0) l.found.sum_before = 0;
    if (t.by_sum) t.target = min(scale_down(t.target - common_before, -finer), held - 1u);
    __syncthreads();
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

    __device__ __forceinline__ void clear(const Measure& m) {
#pragma unroll
        for (uint32_t i = 0; i < BINS / THREADS; ++i) {
            const uint32_t b = threadIdx.x + i * THREADS;
            h.sums[b] = 0, h.counts[b] = 0, begins[b] = m.begin(b);
        }
        if (threadIdx.x == 0) h.least = 0, h.rough = 0;
        __syncthreads();
    }
    // The histogram of a row or chunk.
    __device__ __forceinline__ void count(const Measure& m, const InMemory& row, float least) {
        const uint32_t below = least <= 0.0f ? MINUS_INFINITY : m.first_below(least), border = m.bin_of_key(below);
        clear(m);
        u64 kept = 0;
        row.each<4>([&](float x, uint32_t) {
            const float y = m.y(x);
            if (m.within(y)) {
                const uint32_t bin = m.bin(y);
                const u64 weight = m.whole(m.scaled(x, bin, begins[bin]));
                atomicAdd(&h.counts[bin], 1u);
                atomicAdd(&h.sums[bin], weight);
                if (bin == border && key_of(x) < below) kept += weight;
            }
        });
        if (border < BINS) add(h.least, kept);
        __syncthreads();
        u64 rough = 0;
#pragma unroll
        for (uint32_t i = 0; i < BINS / THREADS; ++i) {
            const uint32_t b = threadIdx.x + i * THREADS;
            rough += scale_down(h.sums[b], (int)m.power(b));
        }
        add(h.rough, rough);
        __syncthreads();
    }
    static __device__ __forceinline__ void add(u64& to, u64 v) {
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
        if ((threadIdx.x & 63u) == 0) atomicAdd(&to, v);
    }
};

// The cuts and the choice of row r from its histogram, by a workgroup.
__device__ __forceinline__ void choose(const Sample& a, uint32_t r, Lds& l, const Measure& m, const InMemory& row,
                                       const Histogram& h) {
    constexpr uint32_t PER = BINS / THREADS;
    // Common units of 2^-common: the sum of all weights, less than twice what it
    // roughly is, stays below 2^62 of them. A bin's own are finer by so many bits.
    const int bits = 65 - __clzll((long long)h.rough), common = 62 + (int)m.shift - bits;
    const auto finer = [&](uint32_t bin) { return (int)(m.shift + m.power(bin)) - common; };
    Bins<PER> bins;
    bins.count_before = 0, bins.sum_before = 0;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t b = threadIdx.x * PER + i;
        bins.counts[i] = h.counts[b], bins.sums[i] = scale_down(h.sums[b], finer(b));
        bins.count_before += bins.counts[i], bins.sum_before += bins.sums[i];
    }
    const float least = a.min_p ? a.min_p[r] : 0.0f, p = a.top_p ? a.top_p[r] : 1.0f, u = a.u[r];
    const int32_t k = a.top_k ? a.top_k[r] : 0;
    uint32_t all;
    u64 total;
    scan(l, bins.count_before, bins.sum_before, all, total);
    // the prefix that stays is the shortest of three: the sums through the
    // k-th, through the first to reach p, and of weights of at least min_p
    const bool cut_k = k > 0 && (uint32_t)k < all, cut_p = !(p >= 1.0f);
    u64 least_sum = ~0ull;
    if (!(least <= 0.0f)) {
        const uint32_t border = m.bin_of_key(m.first_below(least));
        if (border < BINS) {
            __syncthreads();
            if (threadIdx.x == border / PER) {
                u64 before = bins.sum_before;
#pragma unroll
                for (uint32_t i = 0; i < PER; ++i) before += threadIdx.x * PER + i < border ? bins.sums[i] : 0;
                l.found.sum = before + scale_down(h.least, finer(border));
            }
            __syncthreads();
            least_sum = l.found.sum;
        }
    }
    const Target kth{false, (u64)k - 1u};
    // the first to reach p of a sum, the first to pass u of it
    const auto reach = [&](double of) {
        const double sum = (double)p * of;
        return Target{true, sum > 0.0 ? (u64)__builtin_ceil(sum) - 1u : 0};
    };
    const auto choice = [&](u64 of) {
        const double sum = (double)u * (double)of;
        return Target{true, sum > 0.0 ? min((u64)sum, of - 1u) : sum == sum ? 0 : of - 1u};
    };
    bool listed = false;
    if (cut_k || cut_p) {
        bins.find(l, cut_k ? kth : reach((double)total));
        if (l.found.count_before + l.found.count <= LIST) {
            // the candidates through the cut's bin: of them from here on
            listed = true;
            list_values(l, row, value_of(m.first_key(l.found.bin + 1u) - 1u), m.highest);
            if (l.listed <= FEW) {
                if (threadIdx.x < 64u) {
                    // in units of 2^-FINE
                    const Few few(l.list, l.listed, m, false, 0, 0);
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
        const uint32_t bin = l.found.bin;
        find_in_bin(l, m, row, t, h.sums[bin], finer(bin), listed);
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
    for (uint32_t c = threadIdx.x & 63u; c < count; c += 64u) e.take(parts[c]);
    e.take_wave();
    return e;
}

// The histogram of chunk blockIdx.y of row blockIdx.x, added to the row's.
__global__ __launch_bounds__(1024) void k_sample_histogram(Sample a) {
    __shared__ Counting counting;
    const uint32_t r = blockIdx.x, chunk = blockIdx.y;
    if (r >= a.count) return;
    const float temperature = a.temperature ? a.temperature[r] : 1.0f;
    const Extent e = join_extents(a.extents + (size_t)r * a.chunks, a.chunks);
    if (!sampled(temperature, e)) return;
    const Measure m(e, temperature, a.shift);
    counting.count(m, InMemory{a.x + (size_t)r * a.ldx, chunk * a.chunk, min(chunk * a.chunk + a.chunk, a.n)},
                   a.min_p ? a.min_p[r] : 0.0f);
    Histogram& h = a.rows[r];
    if (threadIdx.x == 0) {
        atomicAdd(&h.rough, counting.h.rough);
        if (counting.h.least) atomicAdd(&h.least, counting.h.least);
    }
#pragma unroll
    for (uint32_t i = 0; i < BINS / THREADS; ++i) {
        const uint32_t b = threadIdx.x + i * THREADS;
        if (counting.h.counts[b]) {
            atomicAdd(&h.counts[b], counting.h.counts[b]);
            if (counting.h.sums[b]) atomicAdd(&h.sums[b], counting.h.sums[b]);
        }
    }
}

// A row from its histogram.
__global__ __launch_bounds__(1024) void k_sample_choose(Sample a) {
    __shared__ Lds l;
    const uint32_t r = blockIdx.x;
    const float temperature = a.temperature ? a.temperature[r] : 1.0f;
    const Extent e = join_extents(a.extents + (size_t)r * a.chunks, a.chunks);
    if (!sampled(temperature, e)) {
        take_highest(a, r, e);
        return;
    }
    const Measure m(e, temperature, a.shift);
    choose(a, r, l, m, InMemory{a.x + (size_t)r * a.ldx, 0, a.n}, a.rows[r]);
}

// A whole row by one workgroup: where there is a row for each compute unit or
// nearly, chunks would gain nothing.
__global__ __launch_bounds__(1024) void k_sample_row(Sample a) {
    extern __shared__ u64 lds_words[];
    Counting& counting = *reinterpret_cast<Counting*>(lds_words);
    Lds& l = *reinterpret_cast<Lds*>(&counting + 1);
    const uint32_t r = blockIdx.x;
    const InMemory row{a.x + (size_t)r * a.ldx, 0, a.n};
    find_extent(l.waves, row);
    const float temperature = a.temperature ? a.temperature[r] : 1.0f;
    const Extent e = join_extents(l.waves, WAVES);
    if (!sampled(temperature, e)) {
        take_highest(a, r, e);
        return;
    }
    const Measure m(e, temperature, a.shift);
    counting.count(m, row, a.min_p ? a.min_p[r] : 0.0f);
    choose(a, r, l, m, row, counting.h);
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
    if (chunks <= 1u) {
        TMH_LAUNCH(k_sample_row, dim3(rows), dim3(THREADS), LDS, ctx.stream, a);
    } else {
        a.chunk = (n + chunks - 1u) / chunks;
        a.chunks = (n + a.chunk - 1u) / a.chunk;
        const size_t extents = ((size_t)rows * a.chunks * sizeof(Extent) + 255u) & ~(size_t)255u;
        Workspace work(ctx.index, extents + (size_t)rows * sizeof(Histogram));
        if (work.status) return work.status;
        a.extents = (Extent*)work.memory;
        a.rows = (Histogram*)(work.memory + extents);
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
