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
// token. Bytes bound it: 16-byte loads and stores, the token's sequence found
// by one ballot.
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
        if (threadIdx.x == 0 && blockIdx.y == 0) report(a.p.errors, (int32_t)(fits ? pos : s), (int32_t)(fits ? a.table_rows : a.p.sequences));
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
    uint32_t ldq, heads, group;
    const void* keys;
    const void* values;
    uint32_t window, sinks;
    float scale;  // times log2 e
    float* dst;
    uint32_t ld_dst;
};

constexpr uint32_t KEYS = 64;  // positions of a tile of keys

// The tiles of keys that positions [lo, hi] see: `early` of the sinks, then
// those from the window's first, `from`, on.
struct Span {
    uint32_t early, from, tiles;
    __device__ __forceinline__ uint32_t key(uint32_t tile) const {
        return tile < early ? tile * KEYS : from + (tile - early) * KEYS;
    }
};

__device__ __forceinline__ Span span_of(const AttendPaged& a, uint32_t lo, uint32_t hi) {
    Span s;
    const uint32_t low = a.window && lo >= a.window ? lo - a.window + 1u : 0u;
    s.from = low / KEYS * KEYS;
    s.early = min((a.sinks + KEYS - 1u) / KEYS, s.from / KEYS);
    s.tiles = s.early + (hi - s.from) / KEYS + 1u;
    return s;
}

__device__ __forceinline__ bool sees(const AttendPaged& a, uint32_t pos, uint32_t j) {
    return j <= pos && (a.window == 0u || pos - j < a.window || j < a.sinks);
}

// One query row by one workgroup: the plain form, a thread per key and
// quarter of its columns for the scores, a thread per column for the values.
template <uint32_t KIND>
__global__ __launch_bounds__(256) void k_attend_row(AttendPaged a) {
    typedef typename Element<KIND>::type T;
    __shared__ float weight[KEYS];
    __shared__ uint32_t rows[KEYS];
    const uint32_t t = blockIdx.x / a.heads, h = blockIdx.x % a.heads, kh = h / a.group;
    const uint32_t s = sequence_of(a.p, t);
    if (s >= a.p.sequences || (int32_t)t < a.p.starts[0]) return;
    Sequence sq;
    const bool fits = read_sequence(a.p, s, sq);
    const uint32_t i = t - sq.first;
    if (!fits || i >= sq.count) {
        if (threadIdx.x == 0 && h == 0) report(a.p.errors, (int32_t)s, (int32_t)a.p.sequences);
        return;
    }
    const uint32_t pos = sq.length - sq.count + i, width = a.p.width, quarter = width / 4u;
    const float* q = a.q + (size_t)t * a.ldq + h * width;
    const Span span = span_of(a, pos, pos);
    float top = -INFINITY, total = 0.0f, out = 0.0f;
    for (uint32_t tile = 0; tile < span.tiles; ++tile) {
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
            rows[threadIdx.x / 4u] = seen ? row : 0xffffffffu;
        }
        __syncthreads();
        float best = weight[threadIdx.x & 63u];
        const float mine = best;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) best = fmaxf(best, __shfl_xor(best, d, 64));
        const float higher = fmaxf(top, best);
        const float ref = higher == -INFINITY ? 0.0f : higher;
        const float keep = __builtin_amdgcn_exp2f(top - ref);
        float e = rows[threadIdx.x & 63u] != 0xffffffffu ? __builtin_amdgcn_exp2f(mine - ref) : 0.0f;
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
                if (rows[k] != 0xffffffffu) out += weight[k] * (float)((const T*)a.values)[(size_t)rows[k] * width + threadIdx.x];
    }
    if (threadIdx.x < width) a.dst[(size_t)t * a.ld_dst + h * width + threadIdx.x] = out / total;
}

int check_paged(uint32_t tokens, uint32_t kind, uint32_t pages, uint32_t page_size, uint32_t kv_heads, uint32_t width,
                uint32_t table_width, uint32_t sequences) {
    if (kind != TMH_CACHE_F32 && kind != TMH_CACHE_F16 && kind != TMH_CACHE_BF16) return TMH_ERROR_DTYPE;
    if (width == 0 || width % 8u != 0 || width > 256u || kv_heads == 0 || kv_heads > 65535u) return TMH_ERROR_SHAPE;
    if (pages == 0 || page_size == 0 || table_width == 0) return TMH_ERROR_SHAPE;
    if (tokens > 0x7fffffffu || sequences > 0x7ffffffeu || (uint64_t)sequences * table_width > 0x7fffffffull ||
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
    AttendPaged a{{(const int32_t*)page_table, (const int32_t*)starts, (const int32_t*)lengths, table_width, sequences,
                   tokens, max_new, max_length, pages, kv_heads, width, Divider(page_size), ctx.errors},
                  (const float*)q, ldq, heads, heads / kv_heads, (const void*)keys, (const void*)values, window, sinks,
                  (float)((double)scale * 1.4426950408889634), (float*)dst, ld_dst};
    const dim3 grid(tokens * heads);
    if (kind == TMH_CACHE_F32)
        TMH_LAUNCH(k_attend_row<TMH_CACHE_F32>, grid, dim3(256), 0, ctx.stream, a);
    else if (kind == TMH_CACHE_F16)
        TMH_LAUNCH(k_attend_row<TMH_CACHE_F16>, grid, dim3(256), 0, ctx.stream, a);
    else
        TMH_LAUNCH(k_attend_row<TMH_CACHE_BF16>, grid, dim3(256), 0, ctx.stream, a);
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) note_launch(ctx.index, 1, true);
    return code(e);
}

}  // extern "C"
