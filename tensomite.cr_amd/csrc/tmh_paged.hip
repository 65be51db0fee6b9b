// A key/value cache in pages that sequences share: the write of new keys and
// values (tmh_rope_write_paged) and the attention of new tokens over them
// (tmh_attention_paged). The reference has no counterpart.
//
// Attention of a query row q at position p, over its visible positions j:
//
//   s_j = scale · q·k_j      e_j = exp(s_j - max s)      o = Σ e_j v_j / Σ e_j
//
// in one pass over the keys, with a running maximum and sum. Scores are kept
// in units of log 2 (the scale times log2 e goes into q), so the exponential
// is the hardware's exp2.
#include "../../include/tensomite_hip.h"
#include "tmh_device.h"
#include "tmh_internal.h"

#include <algorithm>
#include <cmath>

namespace tmh {

namespace {

// n / d for n below 2^31 by a multiplication (d from 1 on).
struct Divider {
    uint32_t d, mul, shift;
    explicit Divider(uint32_t by) : d(by), mul(0), shift(0) {
        while (((uint64_t)1 << shift) < by) ++shift;
        mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - by)) / by + 1u);
    }
    __device__ __forceinline__ uint32_t divide(uint32_t n) const { return (__umulhi(mul, n) + n) >> shift; }
};

// A call's sequences and the cache they are in.
struct Paged {
    const int32_t* table;
    const int32_t* starts;
    const int32_t* lengths;
    uint32_t table_width, sequences, tokens;
    uint32_t max_new, max_length;
    uint32_t pages, kv_heads, width;
    Divider page;  // by the page size
    int32_t* errors;
};

// The thread's wave, in a scalar register: what follows from it stays in them.
__device__ __forceinline__ uint32_t wave_index() {
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
}

struct Sequence {
    uint32_t first, count, length;  // its first row, new tokens and positions
};

__device__ __forceinline__ void report(int32_t* errors, int32_t value, int32_t limit) {
    if (atomicAdd(&errors[0], 1) == 0) {
        errors[1] = value;
        errors[2] = limit;
    }
}

// Reads sequence s; false when its numbers do not fit the call.
__device__ __forceinline__ bool read_sequence(const Paged& a, uint32_t s, Sequence& q) {
    const int32_t first = a.starts[s], end = a.starts[s + 1u], length = a.lengths[s];
    q.first = (uint32_t)first;
    q.count = (uint32_t)(end - first);
    q.length = (uint32_t)length;
    return first >= 0 && end >= first && (uint32_t)end <= a.tokens && length >= end - first && q.count <= a.max_new &&
           q.length <= a.max_length && (length == 0 || a.page.divide(q.length - 1u) < a.table_width);
}

// The sequence that row t falls in: how many end at or before it (uniform
// over the wave, every lane active).
__device__ __forceinline__ uint32_t sequence_of(const Paged& a, uint32_t t) {
    uint32_t s = 0;
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t i = 0; i < a.sequences; i += 64u) {
        const bool before = i + lane < a.sequences && a.starts[i + lane + 1u] <= (int32_t)t;
        s += (uint32_t)__popcll(__ballot(before));
    }
    return s;
}

// The cache row (of `width` elements) of position p of sequence s and kv head
// h; a page out of range is reported and false.
__device__ __forceinline__ bool cache_row(const Paged& a, uint32_t s, uint32_t p, uint32_t h, uint32_t& row) {
    const uint32_t at = a.page.divide(p);
    const uint32_t id = (uint32_t)a.table[(size_t)s * a.table_width + at];
    if (id >= a.pages) {
        report(a.errors, (int32_t)id, (int32_t)a.pages);
        return false;
    }
    row = (id * a.kv_heads + h) * a.page.d + (p - at * a.page.d);
    return true;
}

// Four values of the cache's element type.
struct alignas(4) Four {
    float v[4];
};
template <uint32_t KIND>
struct Element;
template <>
struct Element<TMH_CACHE_F32> {
    typedef float type;
};
template <>
struct Element<TMH_CACHE_F16> {
    typedef _Float16 type;
};
template <>
struct Element<TMH_CACHE_BF16> {
    typedef __bf16 type;
};

template <uint32_t KIND>
__device__ __forceinline__ void store_four(void* base, size_t at, const float (&v)[4]) {
    typedef typename Element<KIND>::type T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (T)v[i];  // the nearest, ties to even
    *reinterpret_cast<T4*>((T*)base + at) = o;
}

// ------------------------------------------------------------- the cache write

struct WritePaged {
    Paged p;
    const float* x;
    uint32_t ldx, heads;
    const float* cos;
    const float* sin;
    uint32_t table_rows;
    float* q_dst;
    void* keys;
    void* values;
};

// A token's items, four columns of a head's first half with their partners
// in the second, over workgroups blockIdx.y of 256 threads; blockIdx.x is the
// token. Bytes bound it: 16-byte loads, the token's sequence found by a ballot (5504
// tokens of 8 sequences, 32 heads of 64 each of q, k and v, into bf16: 225 MB in
// 46 us, 4.9 TB/s; one token 2 us, the launch).
template <uint32_t KIND>
__global__ __launch_bounds__(256) void k_rope_write_paged(WritePaged a) {
    const uint32_t t = blockIdx.x;
    const uint32_t s = sequence_of(a.p, t);
    if (s >= a.p.sequences || (int32_t)t < a.p.starts[0]) return;
    Sequence q;
    const bool fits = read_sequence(a.p, s, q);
    const uint32_t i = t - q.first;
    const uint32_t pos = q.length - q.count + i;
    if (!fits || i >= q.count || pos >= a.table_rows) {
        if (threadIdx.x == 0 && blockIdx.y == 0)
            report(a.p.errors, (int32_t)(fits ? pos : s), (int32_t)(fits ? a.table_rows : a.p.sequences));
        return;
    }
    const uint32_t width = a.p.width, half = width >> 1, per = width >> 3;
    const uint32_t item = blockIdx.y * 256u + threadIdx.x;
    const uint32_t unit = item / per, col = (item % per) * 4u;
    if (unit >= a.heads + 2u * a.p.kv_heads) return;
    const float* src = a.x + (size_t)t * a.ldx + (size_t)unit * width + col;
    Four lo = *reinterpret_cast<const Four*>(src), hi = *reinterpret_cast<const Four*>(src + half);
    if (unit < a.heads + a.p.kv_heads) {
        const size_t at = (size_t)pos * width + col;
        const Four cl = *reinterpret_cast<const Four*>(a.cos + at), ch = *reinterpret_cast<const Four*>(a.cos + at + half);
        const Four sl = *reinterpret_cast<const Four*>(a.sin + at), sh = *reinterpret_cast<const Four*>(a.sin + at + half);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // as the host: the partner of a first-half column times -1, two
            // products and their sum, each rounded
            const float l = lo.v[j] * cl.v[j] + hi.v[j] * -1.0f * sl.v[j];
            const float h = hi.v[j] * ch.v[j] + lo.v[j] * sh.v[j];
            lo.v[j] = l;
            hi.v[j] = h;
        }
    }
    if (unit < a.heads) {
        float* dst = a.q_dst + ((size_t)t * a.heads + unit) * width + col;
        *reinterpret_cast<Four*>(dst) = lo;
        *reinterpret_cast<Four*>(dst + half) = hi;
        return;
    }
    uint32_t row;
    const bool key = unit < a.heads + a.p.kv_heads;
    if (!cache_row(a.p, s, pos, unit - a.heads - (key ? 0u : a.p.kv_heads), row)) return;
    void* base = key ? a.keys : a.values;
    store_four<KIND>(base, (size_t)row * width + col, lo.v);
    store_four<KIND>(base, (size_t)row * width + col + half, hi.v);
}

// ------------------------------------------------------------------- attention

struct AttendPaged {
    Paged p;
    const float* q;
    uint32_t ldq, heads;
    Divider group;  // by the query heads of a kv head
    const void* keys;
    const void* values;
    uint32_t window, sinks;
    float scale;  // times log2 e
    float* dst;
    uint32_t ld_dst;
    // Tiles of keys that one workgroup takes; where a row has more, its parts
    // (unscaled outputs; the reference score and the sum of weights) go to
    // part and the join kernels add them. `splits` parts a row have room.
    // The parts of few rows stand by sequence, kv head and row, `room` rows
    // each; those of other rows (room 0) by token and head.
    uint32_t share, splits, room;
    uint32_t row_tile;  // query rows of a tile of more than few
    uint32_t alone;     // k_attend_tile takes sequences of few rows too
    float* part;
    float2* part_sums;
};

constexpr uint32_t KEYS = 64;      // positions of a tile of keys
constexpr uint32_t FEW_TILE = 16;  // query rows of a tile of few rows
constexpr uint32_t FEW_ROWS = 32;  // the most query rows of a kv head that are few
constexpr uint32_t MOST_GROUPS = (1u << 24) - 1u;  // workgroups of 256 threads that a launch can have

// The tiles of keys that positions [lo, hi] see: `early` of the sinks, then
// those from the window's first, `from`, on.
struct Span {
    uint32_t early, from, tiles;
    __device__ __forceinline__ uint32_t key(uint32_t tile) const {
        return tile < early ? tile * KEYS : from + (tile - early) * KEYS;
    }
};

__device__ __forceinline__ uint32_t window_start(const AttendPaged& a, uint32_t pos) {
    return a.window && pos >= a.window ? pos - a.window + 1u : 0u;
}

__device__ __forceinline__ Span span_of(const AttendPaged& a, uint32_t lo, uint32_t hi) {
    Span s;
    s.from = window_start(a, lo) / KEYS * KEYS;
    s.early = min(a.sinks / KEYS + (a.sinks % KEYS ? 1u : 0u), s.from / KEYS);
    s.tiles = s.early + (hi - s.from) / KEYS + 1u;
    return s;
}

__device__ __forceinline__ bool sees(const AttendPaged& a, uint32_t pos, uint32_t j) {
    return j <= pos && (a.window == 0u || pos - j < a.window || j < a.sinks);
}

// A tile of a sequence's query rows of one kv head: row r is new token
// r / group, query head kh * group + r % group.
struct Rows {
    uint32_t s, kh, first, count;  // the tile's first row, and rows
    Sequence sq;
    uint32_t lo, hi;  // positions of its first and last row
    Span span;
    uint32_t parts, begin, end;  // its parts, and the tiles of keys of this one

    __device__ __forceinline__ uint32_t token(const AttendPaged& a, uint32_t r) const {
        return sq.first + a.group.divide(r);
    }
    __device__ __forceinline__ uint32_t head(const AttendPaged& a, uint32_t r) const {
        return kh * a.group.d + r - a.group.divide(r) * a.group.d;
    }
    __device__ __forceinline__ uint32_t position(const AttendPaged& a, uint32_t r) const {
        return sq.length - sq.count + a.group.divide(r);
    }
    // The rows from `from` on (a multiple of `size`), `size` at most; part
    // `part` of theirs. False when there are none.
    __device__ __forceinline__ bool set(const AttendPaged& a, uint32_t from, uint32_t size, uint32_t part) {
        const uint32_t all = sq.count * a.group.d;
        if (from >= all) return false;
        first = from;
        count = min(size, all - from);
        lo = position(a, from);
        hi = position(a, from + count - 1u);
        span = span_of(a, lo, hi);
        parts = (span.tiles + a.share - 1u) / a.share;
        if (part >= parts) return false;
        // even parts, so that none is a remainder
        begin = (uint32_t)((uint64_t)span.tiles * part / parts);
        end = (uint32_t)((uint64_t)span.tiles * (part + 1u) / parts);
        return true;
    }
    // Where row r's parts stand.
    __device__ __forceinline__ size_t place(const AttendPaged& a, uint32_t r) const {
        return (a.room ? ((size_t)s * a.p.kv_heads + kh) * a.room + r : (size_t)token(a, r) * a.heads + head(a, r)) *
               a.splits;
    }
    // Whether position pos sees any key of the part.
    __device__ __forceinline__ bool sees_any(const AttendPaged& a, uint32_t pos) const {
        for (uint32_t tile = begin; tile < end; ++tile) {
            const uint32_t k = span.key(tile);
            if (k <= pos && (a.window == 0u || pos < k + KEYS || pos - (k + KEYS - 1u) < a.window || k < a.sinks)) return true;
        }
        return false;
    }
    // The cache row to read for position j: j's, or where no row of the tile
    // sees j that of the last position, so that pages of hidden positions
    // alone are never touched; a page out of range is reported, and page 0's.
    __device__ __forceinline__ uint32_t cache_row_for(const AttendPaged& a, uint32_t j) const {
        const bool some = j <= hi && (j >= window_start(a, lo) || j < a.sinks);
        uint32_t row = 0;
        cache_row(a.p, s, some ? j : hi, kh, row);
        return row;
    }
};

// The plain form of one query row over the tiles of keys [begin, end), by a
// workgroup of 256 threads: a thread per key and quarter of its columns for
// the scores, a thread per column for the values; hidden positions are not
// read. The kernels below give it the rows whose results are not finite: what
// is not a number or not finite among hidden positions reaches the
// matrix cores' sums (0 times NaN), as do infinities split into parts.
// Returns column threadIdx.x of the sums, with the reference score and the
// sum of weights.
template <uint32_t KIND>
__device__ __forceinline__ float plain_row(const AttendPaged& a, uint32_t s, uint32_t kh, uint32_t pos,
                                                     const float* q, const Span& span, uint32_t begin, uint32_t end,
                                                     float& top, float& total) {
    typedef typename Element<KIND>::type T;
    __shared__ float weight[KEYS];
    __shared__ uint32_t rows[KEYS];
    const uint32_t width = a.p.width, quarter = width / 4u;
    float out = 0.0f;
    top = -INFINITY, total = 0.0f;
    for (uint32_t tile = begin; tile < end; ++tile) {
        const uint32_t j = span.key(tile) + threadIdx.x / 4u;
        float score = 0.0f;
        uint32_t row = 0;
        const bool seen = sees(a, pos, j) && cache_row(a.p, s, j, kh, row);
        if (seen) {
            const uint32_t c0 = threadIdx.x % 4u * quarter;
            const T* k = (const T*)a.keys + (size_t)row * width + c0;
            for (uint32_t c = 0; c < quarter; ++c) score += q[c0 + c] * a.scale * (float)k[c];
        }
        score += __shfl_xor(score, 1, 64);
        score += __shfl_xor(score, 2, 64);
        __syncthreads();  // the last tile's weights have been read
        if (threadIdx.x % 4u == 0) {
            weight[threadIdx.x / 4u] = seen ? score : -INFINITY;
            rows[threadIdx.x / 4u] = seen ? row : ~0u;
        }
        __syncthreads();
        const float mine = weight[threadIdx.x & 63u];
        const bool is = rows[threadIdx.x & 63u] != ~0u;
        float best = mine;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) best = fmaxf(best, __shfl_xor(best, d, 64));
        const float higher = fmaxf(top, best);
        const float ref = higher == -INFINITY ? 0.0f : higher;
        const float keep = __builtin_amdgcn_exp2f(top - ref);
        const float e = is ? __builtin_amdgcn_exp2f(mine - ref) : 0.0f;
        float sum = e;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
        top = higher;
        total = total * keep + sum;
        __syncthreads();
        if (threadIdx.x < 64u) weight[threadIdx.x] = e;
        __syncthreads();
        out *= keep;
        if (threadIdx.x < width)
            for (uint32_t k = 0; k < KEYS; ++k)
                if (rows[k] != ~0u) out += weight[k] * (float)((const T*)a.values)[(size_t)rows[k] * width + threadIdx.x];
    }
    return out;
}

// Writes a row's result, or its part: column c of `width`.
__device__ __forceinline__ void put_column(const AttendPaged& a, const Rows& w, uint32_t r, uint32_t part, uint32_t c,
                                           float sum, float top, float total) {
    if (w.parts == 1u) {
        a.dst[(size_t)w.token(a, r) * a.ld_dst + w.head(a, r) * a.p.width + c] = sum / total;
        return;
    }
    const size_t at = w.place(a, r) + part;
    a.part[at * a.p.width + c] = sum;
    if (c == 0) a.part_sums[at] = make_float2(top, total);
}

// The tile's rows whose bit is set in `which`, by the plain form.
template <uint32_t KIND>
__device__ __forceinline__ void plain_rows(const AttendPaged& a, const Rows& w, uint32_t part, const uint32_t* which) {
    for (uint32_t i = 0; i < w.count; ++i) {
        if (!(which[i / 32u] >> i % 32u & 1u)) continue;
        const uint32_t r = w.first + i;
        float top, total;
        const float* q = a.q + (size_t)w.token(a, r) * a.ldq + w.head(a, r) * a.p.width;
        const float sum = plain_row<KIND>(a, w.s, w.kh, w.position(a, r), q, w.span, w.begin, w.end, top, total);
        if (threadIdx.x < a.p.width) put_column(a, w, r, part, threadIdx.x, sum, top, total);
    }
}

// ------------------------------------------------------- on the matrix cores
//
// The matrix cores multiply 16-bit numbers exactly and add in f32, so f32
// accuracy takes numbers in parts: an f32 number is the sum of three bf16
// ones (its 24 bits cut in eights, exactly), or of two f16 ones to 2^-22 of
// it. An F16 or BF16 cache is one part as it stands; the queries and the
// weights of the softmax have PARTS parts of its type, and an F32 cache three
// of bf16, of whose products with theirs those down to 2^-16 of the first are
// taken (three more would add 2^-24 and less).

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

template <uint32_t KIND>
struct Split {
    static constexpr uint32_t PARTS = KIND == TMH_CACHE_F16 ? 2 : 3;        // of f32 numbers
    static constexpr uint32_t CACHE_PARTS = KIND == TMH_CACHE_F32 ? 3 : 1;  // of the cache's
    static constexpr uint32_t BYTES = KIND == TMH_CACHE_F32 ? 4 : 2;
};

// Eight numbers of each part, as a matrix operand holds them.
template <uint32_t N>
struct Operand {
    u32x4 part[N];
};

// Parts of the numbers v0 and v1, at pair `at` of the operand. Cutting rounds
// toward zero; what it leaves goes to the next part. f16 (v below 65536): two
// times 11 bits, at least 2^-25 absolute.
template <uint32_t KIND>
__device__ __forceinline__ void split_pair(Operand<Split<KIND>::PARTS>& o, int at, float v0, float v1) {
    if constexpr (KIND == TMH_CACHE_F16) {
        const float h0 = __uint_as_float(__float_as_uint(v0) & 0xffffe000u);
        const float h1 = __uint_as_float(__float_as_uint(v1) & 0xffffe000u);
        o.part[0][at] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(h0, h1));
        o.part[1][at] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(v0 - h0, v1 - h1));
    } else {
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const uint32_t w0 = __float_as_uint(v0), w1 = __float_as_uint(v1);
            o.part[p][at] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
            v0 -= __uint_as_float(w0 & 0xffff0000u);
            v1 -= __uint_as_float(w1 & 0xffff0000u);
        }
    }
}

// Eight bytes of LDS a lane, turned: lanes 4r .. 4r + 3 of 16 name row r of four
// rows of 16 numbers, and lane c gets column c of them.
__device__ __forceinline__ uint64_t read_turned(const uint8_t* at) {
    return __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(const lds_byte*)at));
}

template <uint32_t KIND>
__device__ __forceinline__ f32x4 multiply16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (KIND == TMH_CACHE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The products of a cache operand's parts and another's, smallest first.
template <uint32_t KIND>
__device__ __forceinline__ f32x4 multiply_parts16(const Operand<Split<KIND>::CACHE_PARTS>& a,
                                                  const Operand<Split<KIND>::PARTS>& b, f32x4 c) {
    constexpr int LAST = (int)Split<KIND>::PARTS - 1;
#pragma unroll
    for (int order = LAST; order >= 0; --order)
#pragma unroll
        for (int p = 0; p < (int)Split<KIND>::CACHE_PARTS; ++p)
            if (order - p >= 0) c = multiply16<KIND>(a.part[p], b.part[order - p], c);
    return c;
}

// Scores are compared with a row's reference, the highest when it was last
// set; weights are 2^(score - reference + HEADROOM), and the reference is set
// anew once a score passes it by SLACK. Weights stay below 2^(HEADROOM + SLACK),
// within f16, and those down to 2^-24 of the reference's have all their bits.
constexpr float HEADROOM = 6.0f, SLACK = 8.0f;
constexpr float NO_REFERENCE = -3.0e38f;

// A power of two that brings the largest magnitude of a row to be split into
// f16 parts to 2^13 .. 2^14; none where it is from 2^-3 to 2^13, at which the
// parts' 2^-25 is 2^-22 of it already.
__device__ __forceinline__ float power_for(float largest) {
    const int e = (int)(__float_as_uint(largest) >> 23) - 127;
    if (largest == 0.0f || e > 127 || (e >= -3 && e < 13)) return 1.0f;
    return __uint_as_float((uint32_t)(min(13 - e, 126) + 127) << 23);
}

// ---------------------------------------------------------------- few query rows

// Decode steps and chunks of a few tokens: up to FEW_TILE query rows of a kv
// head against a share of the keys. Reading the cache bounds it, so the four
// waves take 32 positions each in turn, nothing shared: keys go from memory to
// the operand's registers, values through the wave's own LDS (direct loads,
// then transposed reads), a step ahead where there is room. Scores are taken
// transposed, keys down and queries across: a lane then holds weights of one
// query and of eight keys, which is what the second product wants of it, with
// the keys in the order 4g..4g+3, 16+4g..16+4g+3 for lane group g.
// Measured: 376832 positions of 8 kv heads of 128, f16, 270 us, 5.7 TB/s; 48
// windows of 1024, f32, 84 us, 4.8 TB/s; 8 sequences of 2048 and less with 32 kv
// heads of 64, bf16, 19 us, 4.7 TB/s; 512 positions of 3 kv heads 7.5 us, all of it
// latency (a page looked up, keys read, the waves' sums joined).
template <uint32_t KIND, uint32_t W>
struct Few {
    static constexpr uint32_t BYTES = Split<KIND>::BYTES;
    static constexpr uint32_t CHUNKS = W * BYTES / 16u;         // 16-byte chunks of a row
    static constexpr uint32_t STAGE = 32u * W * BYTES;          // values of one step
    // a step ahead, where two workgroups' then fit a compute unit's LDS and
    // registers (48 windows of 1024, f32, 128 wide: 101 us with it, 96 without)
    static constexpr uint32_t STAGES = STAGE <= 8192u ? 2 : 1;
    static constexpr uint32_t LOADS = STAGE / 1024u;
    static constexpr uint32_t EIGHT = BYTES / 2u;               // 16-byte pieces of eight numbers
    static constexpr uint32_t STEPS = W / 32u;                  // of the score's product
    static constexpr uint32_t OUT = 4u * FEW_TILE * (W + 4u) * 4u;
    static constexpr uint32_t LDS = 4u * STAGE * STAGES > OUT ? 4u * STAGE * STAGES : OUT;
    // Where a chunk of a row stands in it, so that what is read at once falls
    // on different banks: four rows by four lane groups of one column's 64
    // bytes (f32), or sixteen rows of 32 bytes (f16, bf16).
    static __device__ __forceinline__ constexpr uint32_t swizzle(uint32_t chunk, uint32_t row) {
        return BYTES == 4u ? chunk ^ ((row >> 2 & (CHUNKS / 4u - 1u) & 3u) << 2) : chunk ^ (row & (CHUNKS - 1u) & 7u);
    }
};

template <uint32_t KIND, uint32_t W>
__device__ __forceinline__ void attend_few(const AttendPaged& a, uint32_t row_tiles, uint32_t block, uint8_t* lds) {
    typedef Few<KIND, W> F;
    constexpr uint32_t CP = Split<KIND>::CACHE_PARTS, NP = Split<KIND>::PARTS;
    __shared__ float tops[4][FEW_TILE], totals[4][FEW_TILE];
    __shared__ uint32_t redo;
    const uint32_t lane = threadIdx.x & 63u, wave = wave_index(), col = lane & 15u, group = lane >> 4;
    Rows w;
    uint32_t b = block;
    w.kh = b % a.p.kv_heads, b /= a.p.kv_heads;
    const uint32_t row_tile = b % row_tiles;
    b /= row_tiles;
    w.s = b % a.p.sequences;
    const uint32_t part = b / a.p.sequences;
    if (!read_sequence(a.p, w.s, w.sq)) {
        if (b < a.p.sequences && w.kh == 0 && row_tile == 0 && threadIdx.x == 0)
            report(a.p.errors, (int32_t)w.s, (int32_t)a.p.sequences);
        return;
    }
    if (w.sq.count * a.group.d > FEW_ROWS || !w.set(a, row_tile * FEW_TILE, FEW_TILE, part)) return;
    const uint32_t width = a.p.width;

    // this lane's query: rows past the tile's repeat its last
    const uint32_t r = w.first + min(col, w.count - 1u);
    const uint32_t pos = w.position(a, r);
    const float* q = a.q + (size_t)w.token(a, r) * a.ldq + w.head(a, r) * width;
    Operand<NP> query[F::STEPS];
    float power = 1.0f, undo = 1.0f;
    {
        float v[F::STEPS][8];
        float largest = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < F::STEPS; ++k) {
            const uint32_t c = k * 32u + group * 8u;
            const Four* from = reinterpret_cast<const Four*>(q + (c < width ? c : 0u));
            const Four lo = from[0], hi = from[1];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k][j] = j < 4 ? lo.v[j & 3] : hi.v[j & 3];
        }
#pragma unroll
        for (uint32_t k = 0; k < F::STEPS; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[k][j] = k * 32u + group * 8u < width ? v[k][j] * a.scale : 0.0f;
                largest = fmaxf(largest, fabsf(v[k][j]));
            }
        if (KIND == TMH_CACHE_F16) {
            largest = fmaxf(largest, __shfl_xor(largest, 16, 64));
            largest = fmaxf(largest, __shfl_xor(largest, 32, 64));
            power = power_for(largest);
            undo = 1.0f / power;
        }
#pragma unroll
        for (uint32_t k = 0; k < F::STEPS; ++k)
#pragma unroll
            for (int j = 0; j < 8; j += 2) split_pair<KIND>(query[k], j / 2, v[k][j] * power, v[k][j + 1] * power);
    }

    uint8_t* stage = lds + wave * F::STAGE * F::STAGES;
    const uint32_t stage_at = lds_address(stage);
    const size_t row_bytes = (size_t)width * F::BYTES;
    // step i of this wave: 32 positions, two steps a tile of keys
    const uint32_t steps = 2u * (w.end - w.begin);
    const auto first_key = [&](uint32_t i) { return w.span.key(w.begin + i / 2u) + (i & 1u) * 32u; };
    // the step's keys, 8 columns of rows col and 16 + col each (where a row is
    // narrower than W its first columns stand in, taken for 0); its values
    const auto load = [&](uint32_t i, uint32_t buffer, u32x4 (&key)[2][F::STEPS][F::EIGHT]) {
        const uint32_t mine = w.cache_row_for(a, first_key(i) + (lane & 31u));
#pragma unroll
        for (uint32_t t = 0; t < 2u; ++t) {
            const uint8_t* from = (const uint8_t*)a.keys + (size_t)__shfl(mine, t * 16u + col, 64) * row_bytes;
#pragma unroll
            for (uint32_t k = 0; k < F::STEPS; ++k) {
                const uint32_t c = k * 32u + group * 8u;
#pragma unroll
                for (uint32_t e = 0; e < F::EIGHT; ++e)
                    key[t][k][e] = *(const u32x4*)(from + (c < width ? c : 0u) * F::BYTES + e * 16u);
            }
        }
#pragma unroll
        for (uint32_t l = 0; l < F::LOADS; ++l) {
            const uint32_t slot = l * 64u + lane, row = slot / F::CHUNKS;
            const uint32_t at = F::swizzle(slot % F::CHUNKS, row) * 16u;
            const uint8_t* from = (const uint8_t*)a.values + (size_t)__shfl(mine, row, 64) * row_bytes;
            lds_load16(from + (at < row_bytes ? at : 0u), stage_at + buffer * F::STAGE + l * 1024u);
        }
    };

    float ref = NO_REFERENCE, total = 0.0f;
    f32x4 out[W / 16u];
#pragma unroll
    for (uint32_t d = 0; d < W / 16u; ++d) out[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 key[2][F::STEPS][F::EIGHT], next[2][F::STEPS][F::EIGHT];
    if (F::STAGES == 2u && wave < steps) load(wave, 0, key);
    uint32_t buffer = 0;
    for (uint32_t i = wave; i < steps; i += 4u) {
        if (F::STAGES == 1u) load(i, 0, key);
        wait_vm_lds<0>();
        asm volatile("" ::: "memory");
        const bool more = F::STAGES == 2u && i + 4u < steps;
        if (more) load(i + 4u, buffer ^ 1u, next);

        f32x4 score[2];
#pragma unroll
        for (uint32_t t = 0; t < 2u; ++t) {
            score[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t k = 0; k < F::STEPS; ++k) {
                Operand<CP> o;
                if (width < W && k * 32u + group * 8u >= width)
#pragma unroll
                    for (uint32_t e = 0; e < F::EIGHT; ++e) key[t][k][e] = u32x4{0u, 0u, 0u, 0u};
                if constexpr (KIND == TMH_CACHE_F32) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        split_pair<KIND>(o, j, __uint_as_float(key[t][k][j / 2][j % 2 * 2]),
                                         __uint_as_float(key[t][k][j / 2][j % 2 * 2 + 1]));
                } else {
                    o.part[0] = key[t][k][0];
                }
                score[t] = multiply_parts16<KIND>(o, query[k], score[t]);
            }
        }
        const uint32_t k0 = first_key(i);
        const bool whole = k0 + 31u <= w.lo && (a.window == 0u || w.hi - k0 < a.window || k0 + 31u < a.sinks);
        float best = -INFINITY;
#pragma unroll
        for (uint32_t t = 0; t < 2u; ++t)
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                if (KIND == TMH_CACHE_F16) score[t][j] *= undo;
                if (!whole && !sees(a, pos, k0 + t * 16u + group * 4u + j)) score[t][j] = -INFINITY;
                best = fmaxf(best, score[t][j]);
            }
        if (__any(best > ref + SLACK)) {
            best = fmaxf(best, __shfl_xor(best, 16, 64));
            best = fmaxf(best, __shfl_xor(best, 32, 64));
            if (best > ref + SLACK) {
                const float keep = __builtin_amdgcn_exp2f(ref - best);
                ref = best;
                total *= keep;
#pragma unroll
                for (uint32_t d = 0; d < W / 16u; ++d) out[d] *= keep;
            }
        }
        const float zero = ref - HEADROOM;
        Operand<NP> weight;
        float sum = 0.0f;
#pragma unroll
        for (uint32_t t = 0; t < 2u; ++t) {
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                score[t][j] = __builtin_amdgcn_exp2f(score[t][j] - zero);
                sum += score[t][j];
            }
            split_pair<KIND>(weight, (int)t * 2, score[t][0], score[t][1]);
            split_pair<KIND>(weight, (int)t * 2 + 1, score[t][2], score[t][3]);
        }
        total += sum;
        const uint8_t* from = stage + buffer * F::STAGE;
#pragma unroll
        for (uint32_t d = 0; d < W / 16u; ++d) {
            Operand<CP> o;
            if constexpr (KIND == TMH_CACHE_F32) {
                float v[8];
#pragma unroll
                for (uint32_t j = 0; j < 8u; ++j) {
                    const uint32_t row = group * 4u + j % 4u + j / 4u * 16u;
                    v[j] = *(const float*)(from + row * W * 4u + F::swizzle(d * 4u + col / 4u, row) * 16u + col % 4u * 4u);
                }
#pragma unroll
                for (int j = 0; j < 8; j += 2) split_pair<KIND>(o, j / 2, v[j], v[j + 1]);
            } else {
                // 4 rows of 16 columns a lane group, turned: 4 rows of a column a lane
                const uint32_t row = group * 4u + col / 4u;
                const uint8_t* at = from + row * W * 2u + F::swizzle(d * 2u + col % 4u / 2u, row) * 16u + col % 2u * 8u;
                const uint64_t early = read_turned(at), late = read_turned(at + 16u * W * 2u);
                o.part[0] = u32x4{(uint32_t)early, (uint32_t)(early >> 32), (uint32_t)late, (uint32_t)(late >> 32)};
            }
            out[d] = multiply_parts16<KIND>(o, weight, out[d]);
        }
        if (more) {
#pragma unroll
            for (uint32_t t = 0; t < 2u; ++t)
#pragma unroll
                for (uint32_t k = 0; k < F::STEPS; ++k)
#pragma unroll
                    for (uint32_t e = 0; e < F::EIGHT; ++e) key[t][k][e] = next[t][k][e];
            buffer ^= 1u;
        }
    }

    // the four waves' sums, brought to one reference and added
    total += __shfl_xor(total, 16, 64);
    total += __shfl_xor(total, 32, 64);
    if (group == 0) tops[wave][col] = ref, totals[wave][col] = total;
    if (threadIdx.x == 0) redo = 0;
    __syncthreads();
    {
        const float top = fmaxf(fmaxf(tops[0][col], tops[1][col]), fmaxf(tops[2][col], tops[3][col]));
        const float keep = __builtin_amdgcn_exp2f(ref - top);
        float* to = (float*)lds + (wave * FEW_TILE + col) * (W + 4u) + group * 4u;
#pragma unroll
        for (uint32_t d = 0; d < W / 16u; ++d) *(f32x4*)(to + d * 16u) = out[d] * keep;
    }
    __syncthreads();
    const uint32_t c = threadIdx.x % W;
    for (uint32_t i = threadIdx.x / W; i < w.count; i += 256u / W) {
        if (c >= width) break;
        const float top = fmaxf(fmaxf(tops[0][i], tops[1][i]), fmaxf(tops[2][i], tops[3][i]));
        float sum = 0.0f, all = 0.0f;
#pragma unroll
        for (uint32_t v = 0; v < 4u; ++v) {
            sum += ((const float*)lds)[(v * FEW_TILE + i) * (W + 4u) + c];
            all += totals[v][i] * __builtin_amdgcn_exp2f(tops[v][i] - top);
        }
        const uint32_t row = w.first + i;
        if (!(fabsf(sum) < INFINITY) || !(all < INFINITY) || (all == 0.0f && w.sees_any(a, w.position(a, row))))
            atomicOr(&redo, 1u << i);
        put_column(a, w, row, part, c, sum, top - HEADROOM, all);
    }
    __syncthreads();
    const uint32_t again = redo;
    if (again) plain_rows<KIND>(a, w, part, &again);
}

template <uint32_t KIND, uint32_t W>
__global__ __launch_bounds__(256) void k_attend_few(AttendPaged a, uint32_t row_tiles) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    attend_few<KIND, W>(a, row_tiles, blockIdx.x, lds);
}

// --------------------------------------------------------------- more query rows

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <uint32_t KIND>
__device__ __forceinline__ f32x16 multiply32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (KIND == TMH_CACHE_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <uint32_t KIND>
__device__ __forceinline__ f32x16 multiply_parts32(const Operand<Split<KIND>::CACHE_PARTS>& a,
                                                   const Operand<Split<KIND>::PARTS>& b, f32x16 c) {
    constexpr int LAST = (int)Split<KIND>::PARTS - 1;
#pragma unroll
    for (int order = LAST; order >= 0; --order)
#pragma unroll
        for (int p = 0; p < (int)Split<KIND>::CACHE_PARTS; ++p)
            if (order - p >= 0) c = multiply32<KIND>(a.part[p], b.part[order - p], c);
    return c;
}

// Prompts and chunks: Tile's ROWS query rows of a kv head, 32 a wave, against a
// share of the keys, KT positions staged into LDS at a time for the four waves.
// Products and the softmax's vector operations (about eleven a score, most of them
// the exponential and the cutting in parts) bound it together: a wave has one or
// the other, and the other waves of its SIMD fill in. Scores are transposed as
// above; a lane then holds, of each 32 keys, 4h..4h+3 of every eight for its half h
// of the wave, which are the keys its second operand is given. F16 and BF16 tiles
// come by direct loads into one of two buffers while the other is used; F32 ones are
// split in parts on the way through registers, once for the four waves.
// Measured: 512 tokens at the end of 30000, 32 heads of 128 over 8, bf16: 575 us, 434
// TFLOP/s of attention and three times that of products; a prompt of 2048, 32 heads
// of 64, f16: 52 us, 330 TFLOP/s and twice that.
// Rows up to 64 columns wide go 64 a workgroup, whose waves have half of the keys
// of a step each (2048-token prompt, 32 heads of 64, f16: 53 us; 128 rows: 72).
template <uint32_t KIND, uint32_t W>
struct Tile {
    static constexpr uint32_t SHARES = W <= 64u ? 2 : 1;  // of a step's keys, by wave
    static constexpr uint32_t ROWS = 128u / SHARES;       // query rows of a workgroup
    static constexpr bool F32 = KIND == TMH_CACHE_F32;
    static constexpr uint32_t KT = W == 256u || (F32 && W == 128u) ? 32 : 64;
    static constexpr uint32_t CHUNKS = W / 8u;  // of 8 columns: 16 bytes of LDS a part
    static constexpr uint32_t PART = KT * W * 2u;
    static constexpr uint32_t PARTS = Split<KIND>::CACHE_PARTS;
    static constexpr uint32_t STAGE = 2u * PARTS * PART;  // keys, then values
    static constexpr uint32_t LDS = F32 ? STAGE : 2u * STAGE;
    static constexpr uint32_t LOADS = KT * CHUNKS / 256u;  // chunks a thread brings of keys, and of values
    static __device__ __forceinline__ constexpr uint32_t swizzle(uint32_t chunk, uint32_t row) {
        return chunk ^ (row & (CHUNKS - 1u) & 7u);
    }
};

// Sets w (its kv head is set) to part `part` of row tile `tile` of the sequences
// with more than few rows; a sequence's last rows, which see the most, stand
// first. Uniform over the wave, every lane active.
__device__ __forceinline__ bool find_row_tile(const AttendPaged& a, uint32_t tile, uint32_t part, Rows& w) {
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t i = 0; i < a.p.sequences; i += 64u) {
        Sequence sq{};
        uint32_t tiles = 0;
        if (i + lane < a.p.sequences && read_sequence(a.p, i + lane, sq) && (a.alone || sq.count * a.group.d > FEW_ROWS))
            tiles = (sq.count * a.group.d + a.row_tile - 1u) / a.row_tile;
        uint32_t through = tiles;
#pragma unroll
        for (uint32_t d = 1; d < 64u; d <<= 1) {
            const uint32_t o = __shfl_up(through, d, 64);
            if (lane >= d) through += o;
        }
        const uint64_t past = __ballot(through > tile);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            w.s = i + (uint32_t)at;
            w.sq.first = __builtin_amdgcn_readlane(sq.first, at);
            w.sq.count = __builtin_amdgcn_readlane(sq.count, at);
            w.sq.length = __builtin_amdgcn_readlane(sq.length, at);
            return w.set(a, (__builtin_amdgcn_readlane(through, at) - 1u - tile) * a.row_tile, a.row_tile, part);
        }
        tile -= __builtin_amdgcn_readlane(through, 63);
    }
    return false;
}

template <uint32_t KIND, uint32_t W>
__device__ __forceinline__ void attend_tile(const AttendPaged& a, uint32_t block, uint8_t* lds) {
    typedef Tile<KIND, W> T;
    constexpr uint32_t CP = Split<KIND>::CACHE_PARTS, NP = Split<KIND>::PARTS, KT = T::KT, SHARES = T::SHARES;
    __shared__ uint32_t redo[T::ROWS / 32u], cache_rows[2][KT];
    const uint32_t lane = threadIdx.x & 63u, wave = wave_index(), col = lane & 31u, half = lane >> 5;
    const uint32_t rows_of = wave % (4u / SHARES), keys_of = wave / (4u / SHARES);  // the wave's 32 rows, its share of the keys
    Rows w;
    uint32_t b = block;
    w.kh = b % a.p.kv_heads, b /= a.p.kv_heads;
    const uint32_t part = b % a.splits;
    if (!find_row_tile(a, b / a.splits, part, w)) {
        if (a.alone && block == 0 && threadIdx.x == 0 && !read_sequence(a.p, 0, w.sq)) report(a.p.errors, 0, 1);
        return;
    }
    const uint32_t width = a.p.width;
    const size_t row_bytes = (size_t)width * Split<KIND>::BYTES;

    // this lane's query (rows past the tile's repeat its last), and the
    // positions of the wave's
    const uint32_t r = w.first + min(rows_of * 32u + col, w.count - 1u);
    const uint32_t pos = w.position(a, r);
    const bool idle = rows_of * 32u >= w.count;
    const uint32_t lo = w.position(a, w.first + min(rows_of * 32u, w.count - 1u));
    const uint32_t hi = w.position(a, w.first + min(rows_of * 32u + 31u, w.count - 1u));
    Operand<NP> query[W / 16u];
    float power = 1.0f, undo = 1.0f;
    {
        const float* q = a.q + (size_t)w.token(a, r) * a.ldq + w.head(a, r) * width;
        float v[W / 16u][8];
        float largest = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < W / 16u; ++k) {
            const uint32_t c = k * 16u + half * 8u;
            const Four* from = reinterpret_cast<const Four*>(q + (c < width ? c : 0u));
            const Four lo4 = from[0], hi4 = from[1];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[k][j] = c < width ? (j < 4 ? lo4.v[j & 3] : hi4.v[j & 3]) * a.scale : 0.0f;
                largest = fmaxf(largest, fabsf(v[k][j]));
            }
        }
        if (KIND == TMH_CACHE_F16) {
            largest = fmaxf(largest, __shfl_xor(largest, 32, 64));
            power = power_for(largest);
            undo = 1.0f / power;
        }
#pragma unroll
        for (uint32_t k = 0; k < W / 16u; ++k)
#pragma unroll
            for (int j = 0; j < 8; j += 2) split_pair<KIND>(query[k], j / 2, v[k][j] * power, v[k][j + 1] * power);
    }

    // step i: KT positions. A thread brings chunk at % CHUNKS of rows at /
    // CHUNKS for at = threadIdx.x + 256 l (where a row is narrower than W its
    // first columns stand in). One wave in turn looks up the pages of a step's
    // rows, two steps ahead.
    constexpr uint32_t PER = KEYS / KT;
    const uint32_t steps = PER * (w.end - w.begin);
    const auto first_key = [&](uint32_t i) { return w.span.key(w.begin + i / PER) + i % PER * KT; };
    const auto get_rows = [&](uint32_t i, uint32_t (&rows)[T::LOADS]) {
#pragma unroll
        for (uint32_t l = 0; l < T::LOADS; ++l) rows[l] = cache_rows[i & 1u][(threadIdx.x + l * 256u) / T::CHUNKS];
    };
    const auto load_direct = [&](uint32_t i) {
        uint32_t rows[T::LOADS];
        get_rows(i, rows);
        const uint32_t to = lds_address(lds + (i & 1u) * T::STAGE + wave * 1024u);
#pragma unroll
        for (uint32_t l = 0; l < T::LOADS; ++l) {
            const uint32_t at = threadIdx.x + l * 256u;
            const uint32_t c = T::swizzle(at % T::CHUNKS, at / T::CHUNKS) * 16u;
            const size_t from = (size_t)rows[l] * row_bytes + (c < row_bytes ? c : 0u);
            lds_load16((const uint8_t*)a.keys + from, to + l * 4096u);
            lds_load16((const uint8_t*)a.values + from, to + T::PART + l * 4096u);
        }
    };
    f32x4 held[T::F32 ? T::LOADS : 1][2][2];
    const auto load_held = [&](uint32_t i) {
        uint32_t rows[T::LOADS];
        get_rows(i, rows);
#pragma unroll
        for (uint32_t l = 0; l < T::LOADS; ++l) {
            const uint32_t c = (threadIdx.x + l * 256u) % T::CHUNKS * 32u;
            const size_t from = (size_t)rows[l] * row_bytes + (c < row_bytes ? c : 0u);
            held[l][0][0] = *(const f32x4*)((const uint8_t*)a.keys + from);
            held[l][0][1] = *(const f32x4*)((const uint8_t*)a.keys + from + 16u);
            held[l][1][0] = *(const f32x4*)((const uint8_t*)a.values + from);
            held[l][1][1] = *(const f32x4*)((const uint8_t*)a.values + from + 16u);
        }
    };
    const auto store_held = [&]() {
#pragma unroll
        for (uint32_t l = 0; l < T::LOADS; ++l) {
            const uint32_t at = threadIdx.x + l * 256u, row = at / T::CHUNKS;
#pragma unroll
            for (uint32_t v = 0; v < 2u; ++v) {
                Operand<NP> o;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    split_pair<KIND>(o, j, held[l][v][j / 2][j % 2 * 2], held[l][v][j / 2][j % 2 * 2 + 1]);
#pragma unroll
                for (uint32_t p = 0; p < CP; ++p)
                    *(u32x4*)(lds + (v * CP + p) * T::PART + row * W * 2u + T::swizzle(at % T::CHUNKS, row) * 16u) = o.part[p];
            }
        }
    };

    // In units of the scores times power: zero is what weights count from (the
    // reference less HEADROOM), limit the score that sets the reference anew.
    float zero = 0.0f, limit = -INFINITY, total = 0.0f;
    const bool scaled = __any(undo != 1.0f);
    f32x16 out[W / 32u];
#pragma unroll
    for (uint32_t d = 0; d < W / 32u; ++d) out[d] = f32x16{} * 0.0f;
    if (threadIdx.x < T::ROWS / 32u) redo[threadIdx.x] = 0;
    if (threadIdx.x < 2u * KT && threadIdx.x / KT < steps)
        cache_rows[threadIdx.x / KT][threadIdx.x % KT] = w.cache_row_for(a, first_key(threadIdx.x / KT) + threadIdx.x % KT);
    lds_sync();
    if constexpr (T::F32)
        load_held(0);
    else
        load_direct(0);
    // 32 keys from position kg, rows 32 g .. of a stage: whether none of the wave's
    // rows sees any; their scores; their weights and values
    const auto hidden = [&](uint32_t kg) { return idle || kg > hi || (kg >= a.sinks && kg + 32u <= window_start(a, lo)); };
    const auto multiply = [&](const uint8_t* stage, uint32_t g, f32x16& score) {
        // ahead of other waves' vector operations (512 tokens at the end of 30000,
        // bf16, 128 wide: 612 us, 596 with it)
        __builtin_amdgcn_s_setprio(1);
        score = f32x16{} * 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < W / 16u; ++k) {
            Operand<CP> o;
            const uint32_t row = g * 32u + col;
#pragma unroll
            for (uint32_t p = 0; p < CP; ++p)
                o.part[p] = *(const u32x4*)(stage + p * T::PART + row * W * 2u + T::swizzle(k * 2u + half, row) * 16u);
            score = multiply_parts32<KIND>(o, query[k], score);
        }
        __builtin_amdgcn_s_setprio(0);
    };
    const auto weigh = [&](const uint8_t* stage, uint32_t g, uint32_t kg, f32x16& score) {
        const bool whole = kg + 31u <= lo && (a.window == 0u || hi - kg < a.window || kg + 31u < a.sinks);
        if (!whole) {
#pragma unroll
            for (uint32_t j = 0; j < 16u; ++j)
                if (!sees(a, pos, kg + j / 4u * 8u + half * 4u + j % 4u)) score[j] = -INFINITY;
        }
        float best = score[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) best = fmaxf(best, score[j]);
        if (__any(best > limit)) {
            best = fmaxf(best, __shfl_xor(best, 32, 64));
            if (best > limit) {
                const float keep = limit == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((zero - best) * undo + HEADROOM);
                zero = best - HEADROOM * power;
                limit = best + SLACK * power;
                total *= keep;
#pragma unroll
                for (uint32_t d = 0; d < W / 32u; ++d) out[d] *= keep;
            }
        }
        score -= zero;
        if (KIND == TMH_CACHE_F16 && scaled) {
            asm volatile("");  // a branch: most rows have no power
#pragma unroll
            for (int j = 0; j < 16; ++j) score[j] *= undo;
        }
        Operand<NP> weight[2];
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const float e0 = __builtin_amdgcn_exp2f(score[j]), e1 = __builtin_amdgcn_exp2f(score[j + 1]);
            sum += e0;
            sum += e1;
            split_pair<KIND>(weight[j / 8], j % 8 / 2, e0, e1);
        }
        total += sum;
#pragma unroll
        for (uint32_t d = 0; d < W / 32u; ++d)
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c) {
                // keys 16c + 4 half .. + 3 and 8 further; 16 columns a lane group
                Operand<CP> o;
                const uint32_t row = g * 32u + c * 16u + half * 4u + col % 16u / 4u;
                const uint32_t chunk = d * 4u + col / 16u * 2u + col % 4u / 2u;
#pragma unroll
                for (uint32_t p = 0; p < CP; ++p) {
                    const uint8_t* from = stage + (CP + p) * T::PART + col % 2u * 8u;
                    const uint64_t early = read_turned(from + row * W * 2u + T::swizzle(chunk, row) * 16u);
                    const uint64_t late = read_turned(from + (row + 8u) * W * 2u + T::swizzle(chunk, row + 8u) * 16u);
                    o.part[p] = u32x4{(uint32_t)early, (uint32_t)(early >> 32), (uint32_t)late, (uint32_t)(late >> 32)};
                }
                out[d] = multiply_parts32<KIND>(o, weight[c], out[d]);
            }
    };
    for (uint32_t i = 0; i < steps; ++i) {
        const uint8_t* stage = lds;
        if constexpr (T::F32) {
            lds_sync();  // the last step's tile has been read
            store_held();
            lds_sync();
            if (i + 1u < steps) load_held(i + 1u);
        } else {
            // this step's tile has landed, and every wave is past the last's
            wait_vm_lds<0>();
            lds_sync();
            if (i + 1u < steps) load_direct(i + 1u);
            stage = lds + (i & 1u) * T::STAGE;
        }
        const bool looks = i + 2u < steps && wave == (i & 3u);
        uint32_t ahead = 0;
        if (looks) ahead = w.cache_row_for(a, first_key(i + 2u) + lane % KT);
#pragma unroll
        for (uint32_t g0 = 0; g0 < KT / 32u; g0 += SHARES) {
            const uint32_t g = g0 + keys_of, kg = first_key(i) + g * 32u;
            if (hidden(kg)) continue;
            f32x16 score;
            multiply(stage, g, score);
            weigh(stage, g, kg, score);
        }
        if (looks && lane < KT) cache_rows[i & 1u][lane] = ahead;
    }

    total += __shfl_xor(total, 32, 64);
    float top = limit == -INFINITY ? -INFINITY : zero * undo;
    if constexpr (SHARES == 2u) {
        // the rows' other half of the keys
        float* other = (float*)lds + (rows_of * 64u + lane) * (W / 2u + 4u);
        lds_sync();
        if (keys_of == 1u) {
#pragma unroll
            for (uint32_t d = 0; d < W / 32u; ++d)
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e)
                    *(f32x4*)(other + d * 16u + e * 4u) =
                        f32x4{out[d][e * 4u], out[d][e * 4u + 1u], out[d][e * 4u + 2u], out[d][e * 4u + 3u]};
            *(f32x4*)(other + W / 2u) = f32x4{top, total, 0.0f, 0.0f};
        }
        lds_sync();
        if (keys_of == 0u) {
            const f32x4 sums = *(const f32x4*)(other + W / 2u);
            const float best = fmaxf(top, sums[0]), ref = best == -INFINITY ? 0.0f : best;
            const float mine = __builtin_amdgcn_exp2f(top - ref), theirs = __builtin_amdgcn_exp2f(sums[0] - ref);
            top = best;
            total = total * mine + sums[1] * theirs;
#pragma unroll
            for (uint32_t d = 0; d < W / 32u; ++d)
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) {
                    const f32x4 o = *(const f32x4*)(other + d * 16u + e * 4u);
#pragma unroll
                    for (uint32_t j = 0; j < 4u; ++j) out[d][e * 4u + j] = out[d][e * 4u + j] * mine + o[j] * theirs;
                }
        }
    }
    const uint32_t mine = rows_of * 32u + col;
    if (keys_of == 0u && mine < w.count) {
        bool finite = total < INFINITY && (total > 0.0f || !w.sees_any(a, pos));
        const float by = w.parts == 1u ? 1.0f / total : 1.0f;
        const size_t at = w.place(a, r) + part;
        float* to = w.parts == 1u ? a.dst + (size_t)w.token(a, r) * a.ld_dst + w.head(a, r) * width : a.part + at * width;
        if (w.parts > 1u && half == 0) a.part_sums[at] = make_float2(top, total);
#pragma unroll
        for (uint32_t d = 0; d < W / 32u; ++d)
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) {
                const uint32_t c = d * 32u + e * 8u + half * 4u;
                if (c >= width) continue;
                Four o;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    finite &= fabsf(out[d][e * 4u + j]) < INFINITY;
                    o.v[j] = out[d][e * 4u + j] * by;
                }
                *reinterpret_cast<Four*>(to + c) = o;
            }
        if (!finite) atomicOr(&redo[mine / 32u], 1u << mine % 32u);
    }
    __syncthreads();
    uint32_t any = 0;
#pragma unroll
    for (uint32_t i = 0; i < T::ROWS / 32u; ++i) any |= redo[i];
    if (any) plain_rows<KIND>(a, w, part, redo);
}

// One sequence, of more rows than few. Registers for three waves a SIMD where LDS
// has room for as many (1024 tokens after 3000, 9 heads of 64, bf16: 61 us with two
// waves, 53 with three; the batch below, whose workgroups are shorter, loses by it).
template <uint32_t KIND, uint32_t W>
__global__ __launch_bounds__(256, W <= 64u && KIND != TMH_CACHE_F32 ? 3 : 1) void k_attend_tile(AttendPaged a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    attend_tile<KIND, W>(a, blockIdx.x, lds);
}

// A batch with sequences of both kinds: row tiles in the first `tiles`
// workgroups, few rows behind them, so that each fills what the other leaves
// (chunks and decode steps of 12 sequences, f32, 9 heads of 64: two launches in
// turn 36.5 us, 24.4 so).
template <uint32_t KIND, uint32_t W>
__global__ __launch_bounds__(256) void k_attend_mixed(AttendPaged more, AttendPaged few, uint32_t tiles, uint32_t row_tiles) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    if (blockIdx.x < tiles)
        attend_tile<KIND, W>(more, blockIdx.x, lds);
    else
        attend_few<KIND, W>(few, row_tiles, blockIdx.x - tiles, lds);
}

// Joins the parts of row r, by a wave: each part brought to the highest reference
// and added. The parts wait in L2 or memory, so latency bounds it: a load takes
// 64 / (width / 4) parts, and eight loads go out before the first is used (256 rows
// of up to 4 parts 4 us, 16384 of 4 parts of 128 columns 14).
__device__ __forceinline__ void join_row(const AttendPaged& a, const Rows& w, uint32_t r, f32x4* lanes) {
    const uint32_t lane = threadIdx.x & 63u, width = a.p.width, quads = width / 4u;
    const size_t at = w.place(a, r);
    // lane: columns 4 (lane % quads) .. + 3 of part lane / quads of each load
    constexpr uint32_t AHEAD = 8;
    const uint32_t each = 64u / quads, mine = lane / quads, col = lane % quads * 4u;
    float top = -INFINITY, total = 0.0f;
    f32x4 out{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t z0 = 0; z0 < w.parts; z0 += AHEAD * each) {
        Four part[AHEAD];
        float2 sums[AHEAD];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            const uint32_t z = z0 + i * each + mine;
            if (z0 + i * each >= w.parts) break;
            const size_t from = at + (mine < each && z < w.parts ? z : z0);
            part[i] = *reinterpret_cast<const Four*>(a.part + from * width + col);
            sums[i] = a.part_sums[from];
            if (mine >= each || z >= w.parts) sums[i] = make_float2(-INFINITY, 0.0f);
        }
        float best = top;
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i)
            if (z0 + i * each < w.parts) best = fmaxf(best, sums[i].x);
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) best = fmaxf(best, __shfl_xor(best, d, 64));
        const float ref = best == -INFINITY ? 0.0f : best;
        const float keep = __builtin_amdgcn_exp2f(top - ref);
        top = best;
        total *= keep;
        out *= keep;
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            const uint32_t z = z0 + i * each + mine;
            if (mine >= each || z >= w.parts) continue;
            const float by = __builtin_amdgcn_exp2f(sums[i].x - ref);
            total += sums[i].y * by;
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] += part[i].v[j] * by;
        }
    }
    // the lanes of a column, and one column's of every part's sum
    lanes[lane] = out;
    if (lane % quads != 0) total = 0.0f;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) total += __shfl_xor(total, d, 64);
    if (lane < quads) {
        for (uint32_t e = 1; e < each; ++e) out += lanes[lane + e * quads];
        Four o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o.v[j] = out[j] / total;
        *reinterpret_cast<Four*>(a.dst + (size_t)w.token(a, r) * a.ld_dst + w.head(a, r) * width + col) = o;
    }
}

// Joins the rows that came in parts: a sixteenth of a row tile, a quarter of that a
// wave, in the first JOINS `groups` workgroups; then few rows, a wave a row, by
// sequence, kv head and row, `count` of them.
constexpr uint32_t JOINS = 16;
__global__ __launch_bounds__(256) void k_attend_join(AttendPaged more, AttendPaged few, uint32_t groups, uint32_t count) {
    __shared__ f32x4 lanes[4][64];
    const uint32_t wave = wave_index();
    Rows w;
    if (blockIdx.x < JOINS * groups) {
        const uint32_t b = blockIdx.x / JOINS, rows = more.row_tile / (4u * JOINS);
        w.kh = b % more.p.kv_heads;
        if (!find_row_tile(more, b / more.p.kv_heads, 0, w) || w.parts == 1u) return;
        const uint32_t from = (blockIdx.x % JOINS * 4u + wave) * rows;
        for (uint32_t i = from; i < min(from + rows, w.count); ++i) join_row(more, w, w.first + i, lanes[wave]);
        return;
    }
    uint32_t b = (blockIdx.x - JOINS * groups) * 4u + wave;
    if (b >= count) return;
    const uint32_t r = b % few.room;
    b /= few.room;
    w.kh = b % few.p.kv_heads;
    w.s = b / few.p.kv_heads;
    if (!read_sequence(few.p, w.s, w.sq)) return;
    const uint32_t rows = w.sq.count * few.group.d;
    if (rows > FEW_ROWS || r >= rows || !w.set(few, r / FEW_TILE * FEW_TILE, FEW_TILE, 0) || w.parts == 1u) return;
    join_row(few, w, r, lanes[wave]);
}

// A call's launches: `few` and `more` are its sequences of few rows and of more.
struct Launch {
    AttendPaged few, more;
    uint32_t row_tiles;               // of few rows, the most of a sequence and kv head
    uint32_t few_groups, more_groups;  // row tiles times kv heads; 0 where there are none
    hipStream_t stream;
};

template <uint32_t KIND, uint32_t W>
void launch_width(const Launch& l) {
    constexpr uint32_t lds_few = Few<KIND, W>::LDS, lds_more = Tile<KIND, W>::LDS;
    const uint32_t few = l.few_groups * l.few.splits, more = l.more_groups * l.more.splits;
    if (!more) {
        TMH_LAUNCH((k_attend_few<KIND, W>), dim3(few), dim3(256), lds_few, l.stream, l.few, l.row_tiles);
    } else if (!few) {
        TMH_LAUNCH((k_attend_tile<KIND, W>), dim3(more), dim3(256), lds_more, l.stream, l.more);
    } else {
        TMH_LAUNCH((k_attend_mixed<KIND, W>), dim3(more + few), dim3(256), std::max(lds_few, lds_more), l.stream, l.more,
                   l.few, more, l.row_tiles);
    }
}

template <uint32_t KIND>
void launch_attention_paged(const Launch& l) {
    const uint32_t width = l.few.p.width;
    if (width <= 32u)
        launch_width<KIND, 32>(l);
    else if (width <= 64u)
        launch_width<KIND, 64>(l);
    else if (width <= 128u)
        launch_width<KIND, 128>(l);
    else
        launch_width<KIND, 256>(l);
}

// Tiles of keys that a row tile of `tokens` new tokens sees, at most.
uint64_t most_tiles(const AttendPaged& a, uint32_t tokens) {
    const uint64_t all = ((uint64_t)a.p.max_length + KEYS - 1u) / KEYS;
    if (a.window == 0u) return all;
    return std::min<uint64_t>(all, ((uint64_t)a.sinks + KEYS - 1u) / KEYS + ((uint64_t)a.window + tokens + KEYS) / KEYS + 1u);
}

// Shares of at most `tiles` tiles of keys: no more than `parts`, of at least
// `least` tiles each.
void set_shares(AttendPaged& a, uint64_t tiles, uint64_t parts, uint32_t least) {
    a.share = (uint32_t)std::max<uint64_t>(least, (tiles + parts - 1u) / parts);
    a.splits = (uint32_t)std::max<uint64_t>(1u, (tiles + a.share - 1u) / a.share);
}

int check_paged(uint32_t tokens, uint32_t kind, uint32_t pages, uint32_t page_size, uint32_t kv_heads, uint32_t width,
                uint32_t table_width, uint32_t sequences) {
    if (kind != TMH_CACHE_F32 && kind != TMH_CACHE_F16 && kind != TMH_CACHE_BF16) return TMH_ERROR_DTYPE;
    if (width == 0 || width % 8u != 0 || width > 256u || kv_heads == 0 || kv_heads > 65535u) return TMH_ERROR_SHAPE;
    if (pages == 0 || page_size == 0 || table_width == 0) return TMH_ERROR_SHAPE;
    if (tokens > MOST_GROUPS || sequences > 0x7ffffffeu || (uint64_t)sequences * table_width > 0x7fffffffull ||
        (uint64_t)pages * kv_heads > 0x7fffffffull || (uint64_t)pages * kv_heads * page_size > 0x7fffffffull)
        return TMH_ERROR_SHAPE;
    return TMH_SUCCESS;
}

int code(hipError_t e) { return e == hipErrorOutOfMemory ? TMH_ERROR_OUT_OF_MEMORY : (int)e; }

}  // namespace

}  // namespace tmh

extern "C" {

int tmh_rope_write_paged(uint64_t x, uint32_t ldx, uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t width,
                         uint64_t cos, uint64_t sin, uint32_t table_rows, uint32_t kind, uint32_t pages,
                         uint32_t page_size, uint64_t page_table, uint32_t table_width, uint32_t sequences,
                         uint64_t starts, uint64_t lengths, uint64_t q_dst, uint64_t keys, uint64_t values) {
    using namespace tmh;
    int err = check_paged(tokens, kind, pages, page_size, kv_heads, width, table_width, sequences);
    if (err) return err;
    const uint64_t units = (uint64_t)heads + 2ull * kv_heads;
    if (heads == 0 || heads > 65535u || ldx < units * width || table_rows == 0) return TMH_ERROR_SHAPE;
    if (tokens == 0 || sequences == 0) return TMH_SUCCESS;
    if (!x || !cos || !sin || !page_table || !starts || !lengths || !q_dst || !keys || !values || keys % 16u != 0 ||
        values % 16u != 0)
        return TMH_ERROR_INVALID_VALUE;
    DeviceContext ctx;
    if ((err = device_context(&ctx, true)) != TMH_SUCCESS) return err;
    WritePaged a{{(const int32_t*)page_table, (const int32_t*)starts, (const int32_t*)lengths, table_width, sequences,
                  tokens, tokens, 0x7fffffffu, pages, kv_heads, width, Divider(page_size), ctx.errors},
                 (const float*)x, ldx, heads, (const float*)cos, (const float*)sin, table_rows, (float*)q_dst,
                 (void*)keys, (void*)values};
    const dim3 grid(tokens, (uint32_t)((units * (width / 8u) + 255u) / 256u));
    if (kind == TMH_CACHE_F32)
        TMH_LAUNCH(k_rope_write_paged<TMH_CACHE_F32>, grid, dim3(256), 0, ctx.stream, a);
    else if (kind == TMH_CACHE_F16)
        TMH_LAUNCH(k_rope_write_paged<TMH_CACHE_F16>, grid, dim3(256), 0, ctx.stream, a);
    else
        TMH_LAUNCH(k_rope_write_paged<TMH_CACHE_BF16>, grid, dim3(256), 0, ctx.stream, a);
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) note_launch(ctx.index, 1, true);
    return code(e);
}

int tmh_attention_paged(uint64_t q, uint32_t ldq, uint32_t tokens, uint32_t heads, uint32_t kind, uint64_t keys,
                        uint64_t values, uint32_t pages, uint32_t page_size, uint32_t kv_heads, uint32_t width,
                        uint64_t page_table, uint32_t table_width, uint32_t sequences, uint64_t starts,
                        uint64_t lengths, uint32_t max_new, uint32_t max_length, uint32_t window, uint32_t sinks,
                        float scale, uint64_t dst, uint32_t ld_dst) {
    using namespace tmh;
    int err = check_paged(tokens, kind, pages, page_size, kv_heads, width, table_width, sequences);
    if (err) return err;
    if (heads == 0 || heads > 65535u || heads % kv_heads != 0 || ldq < heads * width || ld_dst < heads * width)
        return TMH_ERROR_SHAPE;
    if ((uint64_t)tokens * heads > 0x7fffffffull || max_new > 0x7fffffffu || max_length > 0x7fffffffu ||
        window > 0x7fffffffu || sinks > 0x7fffffffu)
        return TMH_ERROR_SHAPE;
    if (tokens == 0 || sequences == 0) return TMH_SUCCESS;
    if (!q || !page_table || !starts || !lengths || !dst || !keys || !values || keys % 16u != 0 || values % 16u != 0)
        return TMH_ERROR_INVALID_VALUE;
    DeviceContext ctx;
    if ((err = device_context(&ctx, true)) != TMH_SUCCESS) return err;
    const uint32_t group = heads / kv_heads;
    AttendPaged a{{(const int32_t*)page_table, (const int32_t*)starts, (const int32_t*)lengths, table_width, sequences,
                   tokens, max_new, max_length, pages, kv_heads, width, Divider(page_size), ctx.errors},
                  (const float*)q, ldq, heads, Divider(group), (const void*)keys, (const void*)values, window, sinks,
                  (float)((double)scale * 1.4426950408889634), (float*)dst, ld_dst, 0, 1, 0, 128, 0, nullptr, nullptr};
    Launch l{a, a, 0, 0, 0, ctx.stream};
    AttendPaged &few = l.few, &more = l.more;
    const uint64_t rows = std::max<uint64_t>(1u, (uint64_t)max_new * group);
    const bool has_more = rows > FEW_ROWS;
    more.row_tile = width <= 64u ? 64 : 128;
    more.alone = has_more && sequences == 1u;  // the usual prompt
    few.room = (uint32_t)std::min<uint64_t>(FEW_ROWS, rows);
    l.row_tiles = (few.room + FEW_TILE - 1u) / FEW_TILE;
    uint64_t few_groups = 0, more_groups = 0;
    if (!more.alone) {
        // As many workgroups as run at once by their registers, no more: four a
        // compute unit up to 64 columns, two to 128, one above (4 sequences of up to
        // 131072, 8 kv heads of 128, f16: 275 us with two a compute unit, 290 with
        // four; 4 of 4000, 5 of 256: 24 with one, 33 with more). A share's time goes
        // with its tiles, the join's with the parts, their sum is least at a root
        // (20000 positions, 8 kv heads of 128, f16, 313 tiles: 27.4 us in 16 parts, 23.6
        // in 32, 27.1 in 63). Shares are four tiles at least, one step a wave, and
        // eight are one share: a second launch costs more than it gains (512
        // positions, 3 kv heads of 64: 7.9 us in one launch, 10.1 in two; 2000: 11.9 with
        // shares of eight tiles, 10.2 of four).
        few_groups = (uint64_t)sequences * kv_heads * l.row_tiles;
        const uint64_t at_once = (width <= 64u ? 4u : width <= 128u ? 2u : 1u) * (uint64_t)ctx.compute_units;
        const uint64_t tiles = most_tiles(a, FEW_ROWS);
        const uint64_t parts = std::min(at_once / few_groups, (uint64_t)(2.0 * std::sqrt((double)tiles)));
        set_shares(few, tiles, std::max<uint64_t>(parts, 1u), tiles <= 8u ? 8u : 4u);
    }
    if (has_more) {
        // Row tiles of all sequences, at most; and about, a sequence's last half full.
        const uint64_t all = (uint64_t)tokens * group, ends = std::min<uint64_t>(sequences, all / (FEW_ROWS + 1u));
        more_groups = (all / more.row_tile + ends) * kv_heads;
        uint64_t about = (all / more.row_tile + (ends + 1u) / 2u) * kv_heads;
        if (more.alone) about = more_groups = (all + more.row_tile - 1u) / more.row_tile * kv_heads;
        // Again as many as run at once (beside few rows two a compute unit at most),
        // and no second round of a few (1024 tokens after 3000, 9 heads of 64, 144 row
        // tiles: f16 48.0 us in 4 parts, 43.1 in 5, 52.2 in 6; f32 95.9 in 2, 75.0 in 3,
        // 99.4 in 4). Row tiles see from 1 - f of the tiles to all: of p parts they
        // have p (1 - f / 2) + 1 / 2 on average, p where that is less than one apart.
        // Prompts, f near 1, are even enough in three (1500 tokens, 16 heads of 128, f16:
        // 60.5 us whole, 53.0, 49.9, 59.5 in 2, 3, 4), and where one round would leave
        // them whole their last tiles would run on alone, so that two are taken if row
        // tiles are few or long (4096 tokens, 8 heads of 256, f16: 335 us whole, 252 in
        // 3; but 1500 tokens, 32 heads of 64, 38 whole, 73 in 3). Shares as above; eight
        // tiles are one: a prompt of 512, f16, 15.2 us in one launch, 16.6 in two.
        const bool f32 = kind == TMH_CACHE_F32, narrow = width <= 32u || (width <= 64u && !f32);
        const uint64_t each = narrow ? (more.alone ? 3u : 2u) : width <= 64u || (width <= 128u && !f32) ? 2u : 1u;
        const uint64_t at_once = each * ctx.compute_units, tiles = most_tiles(a, more.row_tile);
        const double f = std::min(1.0, (double)max_new / std::max(1.0, (double)max_length));
        const auto parts_for = [&](uint64_t groups) {
            const double p = (double)groups / (double)std::max<uint64_t>(about, 1u);
            return f * p < 1.0 ? p : (p - 0.5) / (1.0 - f / 2.0);
        };
        double parts = parts_for(at_once);
        if (f > 0.9) {
            if (parts < 2.0 && (4u * about <= 3u * at_once || (about <= at_once && tiles >= 48u))) parts = parts_for(2u * at_once);
            parts = std::min(parts, 3.0);
        }
        set_shares(more, tiles, (uint64_t)std::max(parts, 1.0), tiles <= 8u ? 8u : 4u);
    }
    if (few_groups * few.splits + more_groups * more.splits > MOST_GROUPS || more_groups > MOST_GROUPS / (2u * JOINS))
        return TMH_ERROR_SHAPE;
    l.few_groups = (uint32_t)few_groups, l.more_groups = (uint32_t)more_groups;
    const size_t few_parts = few.splits > 1u ? (size_t)sequences * kv_heads * few.room * few.splits : 0;
    const size_t more_parts = more.splits > 1u ? (size_t)tokens * heads * more.splits : 0;
    const size_t sums = ((few_parts + more_parts) * sizeof(float2) + 255u) & ~(size_t)255u;
    Workspace work(ctx.index, sums + (few_parts + more_parts) * width * sizeof(float));
    if (work.status) return work.status;
    few.part_sums = (float2*)work.memory;
    few.part = (float*)(work.memory + sums);
    more.part_sums = few.part_sums + few_parts;
    more.part = few.part + few_parts * width;
    if (kind == TMH_CACHE_F32)
        launch_attention_paged<TMH_CACHE_F32>(l);
    else if (kind == TMH_CACHE_F16)
        launch_attention_paged<TMH_CACHE_F16>(l);
    else
        launch_attention_paged<TMH_CACHE_BF16>(l);
    hipError_t e = hipGetLastError();
    const uint32_t groups = more_parts ? l.more_groups : 0u, count = few_parts ? sequences * kv_heads * few.room : 0u;
    if (e == hipSuccess && (groups || count)) {
        TMH_LAUNCH(k_attend_join, dim3(JOINS * groups + (count + 3u) / 4u), dim3(256), 0, ctx.stream, more, few, groups, count);
        e = hipGetLastError();
    }
    if (e == hipSuccess) note_launch(ctx.index, 1, true);
    return code(e);
}

}  // extern "C"
