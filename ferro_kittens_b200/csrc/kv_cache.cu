// The key/value cache in 4 bits, for sm_100a: quantising tokens as they are written, reading rows back, and
// attention of a sequence's newest tokens over its rows. No counterpart in the reference, whose attention
// reads whole bf16 planes (examples/src/flash_forward.rs:151-158); the format is stated in the header.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fk_host.h"
#include "fk_ptx.cuh"

namespace fk {
namespace cache {

enum NoteCode : uint32_t {
    kBadSlot = 0x501,    // a slot outside the cache
    kBadPage = 0x502,    // a page table entry outside the cache
    kBadLength = 0x503,  // a length past the page table
};

/// The first bad index of a launch goes into the caller's status words.
__device__ __forceinline__ void note(uint32_t* status, uint32_t code, uint32_t where, uint32_t value) {
    if (status && atomicCAS(status, 0u, code) == 0u) {
        status[1] = blockIdx.x;
        status[2] = where;
        status[3] = value;
    }
}

/// n / d for n < 2^31 by one wide multiply: m = ceil(2^(31 + s) / d) with 2^(s - 1) < d <= 2^s errs by less
/// than 2^-31 of n, so the floor is exact.
struct Divider {
    uint32_t multiplier, shift, divisor;
    __host__ __device__ Divider() : multiplier(0), shift(0), divisor(0) {}
    explicit Divider(uint32_t d) : multiplier(0), shift(31), divisor(d) {
        while ((1ull << (shift - 31)) < d) ++shift;
        multiplier = static_cast<uint32_t>(((1ull << shift) + d - 1) / d);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
        return static_cast<uint32_t>((static_cast<uint64_t>(n) * multiplier) >> shift);
    }
};

// ---------------------------------------------------------------- the two element types

template <bool BF16>
struct Element;

template <>
struct Element<true> {
    static constexpr uint32_t kNaN = 0x7fffu;
    static constexpr uint32_t kMagic = 0x43004300u;  // 128: a code in the low mantissa bits reads as 128 + code
    static __device__ __forceinline__ float low(uint32_t pair) { return __uint_as_float(pair << 16); }
    static __device__ __forceinline__ float high(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }
    static __device__ __forceinline__ uint32_t min_nan(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    /// The bits of the largest value of the type not above x >= 0.
    static __device__ __forceinline__ uint32_t truncate(float x) { return __float_as_uint(x) >> 16; }
    static __device__ __forceinline__ uint32_t minus_magic(uint32_t x) {
        uint32_t d;
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(0x3f803f80u), "r"(0xc300c300u));
        return d;
    }
    static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
        uint32_t d;
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
        return d;
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};

template <>
struct Element<false> {
    static constexpr uint32_t kNaN = 0x7fffu;
    static constexpr uint32_t kMagic = 0x64006400u;  // 1024
    static __device__ __forceinline__ float low(uint32_t pair) {
        return __half2float(__ushort_as_half(static_cast<unsigned short>(pair & 0xffffu)));
    }
    static __device__ __forceinline__ float high(uint32_t pair) {
        return __half2float(__ushort_as_half(static_cast<unsigned short>(pair >> 16)));
    }
    static __device__ __forceinline__ uint32_t min_nan(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    static __device__ __forceinline__ uint32_t truncate(float x) {
        return __half_as_ushort(__float2half_rz(x));
    }
    static __device__ __forceinline__ uint32_t minus_magic(uint32_t x) {
        uint32_t d;
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0xe400e400u));
        return d;
    }
    static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
        uint32_t d;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
        return d;
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t d;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
        return d;
    }
};

/// The 8 x 8 matrix of nibbles held one row a lane by eight neighbouring lanes, transposed (its own inverse):
/// halves, bytes, then nibbles change places with the lane 4, 2 and 1 away.
__device__ __forceinline__ uint32_t transpose_nibbles(uint32_t x, uint32_t lane) {
    uint32_t y = __shfl_xor_sync(0xffffffffu, x, 4);
    x = __byte_perm(x, y, (lane & 4u) ? 0x3276u : 0x5410u);
    y = __shfl_xor_sync(0xffffffffu, x, 2);
    x = __byte_perm(x, y, (lane & 2u) ? 0x3715u : 0x6240u);
    y = __shfl_xor_sync(0xffffffffu, x, 1);
    return (lane & 1u) ? (x & 0xf0f0f0f0u) | ((y >> 4) & 0x0f0f0f0fu) : (x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u);
}

// ---------------------------------------------------------------- writing and reading

constexpr uint32_t kRowThreads = 256;

struct RowArguments {
    const void* tensor[2];  // k, v (the source of a write, the destination of a read)
    uint32_t* codes[2];
    uint32_t* params[2];
    int64_t token_stride[2], head_stride[2];  // bytes
    const void* slots;
    uint32_t slots_wide;
    uint32_t tokens, rows;  // rows = tokens * kv_heads
    uint64_t capacity;      // pages * page_size
    uint32_t page_size;
    Divider heads, page;
    uint32_t clear_skipped;
};

/// The cache row of token `token`'s head `head`, or false for a slot that is negative or outside the cache.
__device__ __forceinline__ bool cache_row(const RowArguments& args, uint32_t token, uint32_t head, uint64_t& row,
                                          uint32_t* status) {
    const int64_t slot = args.slots_wide ? static_cast<const int64_t*>(args.slots)[token]
                                         : static_cast<const int32_t*>(args.slots)[token];
    if (slot < 0) return false;
    if (static_cast<uint64_t>(slot) >= args.capacity) {
        note(status, kBadSlot, token, static_cast<uint32_t>(slot));
        return false;
    }
    const uint32_t page = args.page.quotient(static_cast<uint32_t>(slot));
    const uint32_t place = static_cast<uint32_t>(slot) - page * args.page_size;
    row = (static_cast<uint64_t>(page) * args.heads.divisor + head) * args.page_size + place;
    return true;
}

/// Where a row's word of natural order `block` (channels 8 * block + 0..7) sits: the keys' matrix [4][D / 32].
template <int D>
__device__ __forceinline__ uint32_t key_word(uint32_t block) {
    return (block & 3u) * (D / 32) + (block >> 2);
}
/// Where the transposed word of lane `block` sits: the values' matrix [8][D / 64] of words.
template <int D>
__device__ __forceinline__ uint32_t value_word(uint32_t block) {
    return (block & 7u) * (D / 64) + (block >> 3);
}

// One lane holds 8 channels (16 bytes) of a row, D / 8 lanes a row; a group's smallest and largest value are
// found together, as the minimum of packed pairs (x, -x) over its G / 8 lanes.
template <int D, int G, bool BF16>
__global__ void __launch_bounds__(kRowThreads) write_kernel(const __grid_constant__ RowArguments args,
                                                            uint32_t* status) {
    using E = Element<BF16>;
    constexpr uint32_t kLanes = D / 8;
    const uint32_t which = blockIdx.y;
    const uint32_t lane = threadIdx.x & 31u, block = threadIdx.x % kLanes;
    const uint32_t step = gridDim.x * (kRowThreads / kLanes);
    for (uint32_t first = blockIdx.x * (kRowThreads / kLanes); first < args.rows; first += step) {
        const uint32_t index = first + threadIdx.x / kLanes;
        uint4 x = make_uint4(0, 0, 0, 0);
        uint64_t row = 0;
        bool kept = index < args.rows;
        if (kept) {
            const uint32_t token = args.heads.quotient(index), head = index - token * args.heads.divisor;
            kept = cache_row(args, token, head, row, status);
            if (kept)
                x = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(args.tensor[which]) +
                                                          token * args.token_stride[which] +
                                                          head * args.head_stride[which]) +
                           block);
        }
        const uint32_t words[4] = {x.x, x.y, x.z, x.w};
        // {smallest, -largest} of the group, NaN if it holds one.
        uint32_t least = words[0], most = words[0] ^ 0x80008000u;
#pragma unroll
        for (uint32_t i = 1; i < 4; ++i) {
            least = E::min_nan(least, words[i]);
            most = E::min_nan(most, words[i] ^ 0x80008000u);
        }
        uint32_t ends = E::min_nan(__byte_perm(least, most, 0x5410), __byte_perm(least, most, 0x7632));
#pragma unroll
        for (uint32_t mask = 1; mask < G / 8; mask *= 2)
            ends = E::min_nan(ends, __shfl_xor_sync(0xffffffffu, ends, mask));
        const float low = E::low(ends), high = -E::high(ends);
        // Half the span: the span itself may pass fp32's range. `lost` is what its rounding left out, exactly
        // (the error of a sum is a float).
        const float a = 0.5f * high, b = 0.5f * low;
        const float half_span = a - b;
        const float b_part = half_span - a;
        const float lost = (a - (half_span - b_part)) - (b + b_part);
        const bool finite = half_span < __uint_as_float(0x7f800000u);  // false for NaN as well
        uint32_t scale_bits = finite ? E::truncate(__fdiv_rn(half_span, 7.5f)) : 0u;
        float scale = E::low(scale_bits);
        // The quotient's rounding may have carried it over a value of the type: 7.5 * scale is exact.
        if (finite && (7.5f * scale > half_span || (7.5f * scale == half_span && lost < 0.0f))) {
            --scale_bits;
            scale = E::low(scale_bits);
        }
        const uint32_t low_bits = finite ? (ends & 0xffffu) : E::kNaN;
        // Tiny spans are lifted by 2^100 so that 1 / scale stays finite, huge ones halved so that x - low does
        // (the products are exact).
        const float lift = scale > 0x1p100f ? 0.5f : scale < 0x1p-100f && scale > 0.0f ? 0x1p100f : 1.0f;
        const float step_size = scale * lift, origin = -low * lift;
        const bool coded = finite && scale > 0.0f;
        const float inverse = coded ? __fdiv_rn(1.0f, step_size) : 0.0f;
        const float half_step = coded ? 0.5f * step_size : __uint_as_float(0x7f800000u);
        uint32_t word = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            const float value = (i & 1u) ? E::high(words[i / 2]) : E::low(words[i / 2]);
            const float lifted = value * lift;
            const float t = coded ? lifted + origin : 0.0f;
            // What rounding left out of t, exactly.
            const float o_part = t - lifted;
            const float t_lost = coded ? (lifted - (t - o_part)) + (origin - o_part) : 0.0f;
            const float guess = fminf(rintf(t * inverse), 15.0f);
            // Where t stands against the guess's borders: the remainder is exact.
            const float r = __fmaf_rn(-guess, step_size, t);
            int code = static_cast<int>(guess);
            if ((r - half_step) + t_lost >= 0.0f) ++code;
            else if ((r + half_step) + t_lost < 0.0f) --code;
            code = min(max(code, 0), 15);
            word |= static_cast<uint32_t>(code) << (4 * i);
        }
        uint32_t at;
        if (which == 0) {
            at = key_word<D>(block);
        } else {
            word = transpose_nibbles(word, lane);
            at = value_word<D>(block);
        }
        if (kept) {
            args.codes[which][row * (D / 8) + at] = word;
            if (block % (G / 8) == 0) args.params[which][row * (D / G) + block / (G / 8)] = scale_bits | (low_bits << 16);
        }
    }
}

// The same lanes the other way: a code in the low mantissa bits of a power of two, less that power, is exact,
// and one fused multiply-add in the cache's type rounds low + code * scale once.
template <int D, int G, bool BF16>
__global__ void __launch_bounds__(kRowThreads) read_kernel(const __grid_constant__ RowArguments args,
                                                           uint32_t* status) {
    using E = Element<BF16>;
    constexpr uint32_t kLanes = D / 8;
    const uint32_t which = blockIdx.y;
    const uint32_t lane = threadIdx.x & 31u, block = threadIdx.x % kLanes;
    const uint32_t step = gridDim.x * (kRowThreads / kLanes);
    for (uint32_t first = blockIdx.x * (kRowThreads / kLanes); first < args.rows; first += step) {
        const uint32_t index = first + threadIdx.x / kLanes;
        const bool inside = index < args.rows;
        uint32_t word = 0, pair = 0;
        uint4* destination = nullptr;
        bool kept = false;
        if (inside) {
            const uint32_t token = args.heads.quotient(index), head = index - token * args.heads.divisor;
            uint64_t row = 0;
            kept = cache_row(args, token, head, row, status);
            if (kept) {
                word = args.codes[which][row * (D / 8) + (which == 0 ? key_word<D>(block) : value_word<D>(block))];
                pair = args.params[which][row * (D / G) + block / (G / 8)];
            }
            destination = reinterpret_cast<uint4*>(static_cast<uint8_t*>(const_cast<void*>(args.tensor[which])) +
                                                   token * args.token_stride[which] + head * args.head_stride[which]) +
                          block;
        }
        if (which == 1) word = transpose_nibbles(word, lane);
        const uint32_t scale = __byte_perm(pair, 0, 0x1010), low = __byte_perm(pair, 0, 0x3232);
        uint32_t y[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t codes = ((word >> (8 * i)) & 0xfu) | ((word >> (8 * i) << 12) & 0xf0000u);
            y[i] = E::fma(E::minus_magic(codes | E::kMagic), scale, low);
        }
        if (inside && (kept || args.clear_skipped)) *destination = kept ? make_uint4(y[0], y[1], y[2], y[3]) : make_uint4(0, 0, 0, 0);
    }
}

// ---------------------------------------------------------------- attention

struct AttentionArguments {
    const uint8_t* k_codes;
    const uint32_t* k_params;
    const uint8_t* v_codes;
    const uint32_t* v_params;
    const uint8_t* q;
    int64_t q_batch_stride, q_token_stride, q_head_stride;  // bytes
    void* out;
    float* lse;
    const int32_t* lengths;
    const int32_t* table;
    int64_t table_stride;
    uint32_t table_pages, pages, page_size;
    uint32_t batch, queries, heads, kv_heads;
    float scale;
    uint32_t window, sinks;
    Divider page;
};

constexpr uint32_t kAttentionThreads = 128;

// One block per (query row, sequence), a warp per token in turn with a running maximum and sum of its own.
template <int D, int G, bool BF16>
__global__ void __launch_bounds__(kAttentionThreads) attention_kernel(const __grid_constant__ AttentionArguments args,
                                                                      uint32_t* status) {
    using E = Element<BF16>;
    constexpr uint32_t kWarps = kAttentionThreads / 32, kEach = D / 32;
    __shared__ float sums[kWarps][D];
    __shared__ float peaks[kWarps], totals[kWarps];
    const uint32_t b = blockIdx.y, query = blockIdx.x / args.heads, head = blockIdx.x % args.heads;
    const uint32_t kv_head = head / (args.heads / args.kv_heads);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t capacity = static_cast<uint64_t>(args.table_pages) * args.page_size;
    int64_t length = max(args.lengths[b], 0);
    if (static_cast<uint64_t>(length) > capacity) {
        if (threadIdx.x == 0) note(status, kBadLength, b, static_cast<uint32_t>(length));
        length = static_cast<int64_t>(capacity);
    }
    const int64_t at = length - args.queries + query;
    const uint16_t* q = reinterpret_cast<const uint16_t*>(args.q + b * args.q_batch_stride +
                                                          query * args.q_token_stride + head * args.q_head_stride);
    float mine[kEach], sum[kEach];
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
        mine[e] = E::low(q[lane + 32 * e]) * args.scale;
        sum[e] = 0.0f;
    }
    float peak = -INFINITY, total = 0.0f;
    for (int64_t j = warp; j <= at; j += kWarps) {
        if (args.window && j <= at - static_cast<int64_t>(args.window) && j >= static_cast<int64_t>(args.sinks)) continue;
        const uint32_t entry = args.page.quotient(static_cast<uint32_t>(j));
        const uint32_t page = args.table ? static_cast<uint32_t>(args.table[b * args.table_stride + entry]) : b;
        if (page >= args.pages) {
            if (lane == 0) note(status, kBadPage, b, page);
            continue;
        }
        const uint64_t row = (static_cast<uint64_t>(page) * args.kv_heads + kv_head) * args.page_size +
                             (static_cast<uint32_t>(j) - entry * args.page_size);
        float score = 0.0f, v[kEach];
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) {
            const uint32_t d = lane + 32 * e, run = d / 8;
            const uint32_t kn = key_word<D>(run) * 8 + d % 8, vn = (d % 8) * (D / 8) + run;
            const uint32_t kc = (args.k_codes[row * (D / 2) + kn / 2] >> (4 * (kn & 1))) & 15u;
            const uint32_t vc = (args.v_codes[row * (D / 2) + vn / 2] >> (4 * (vn & 1))) & 15u;
            const uint32_t kp = args.k_params[row * (D / G) + d / G], vp = args.v_params[row * (D / G) + d / G];
            score += mine[e] * fmaf(static_cast<float>(kc), E::low(kp), E::high(kp));
            v[e] = fmaf(static_cast<float>(vc), E::low(vp), E::high(vp));
        }
#pragma unroll
        for (uint32_t mask = 16; mask > 0; mask >>= 1) score += __shfl_xor_sync(0xffffffffu, score, mask);
        const float higher = fmaxf(peak, score);
        const float keep = higher == peak ? 1.0f : __expf(peak - higher), weight = __expf(score - higher);
        peak = higher;
        total = total * keep + weight;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) sum[e] = fmaf(weight, v[e], sum[e] * keep);
    }
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) sums[warp][lane + 32 * e] = sum[e];
    if (lane == 0) {
        peaks[warp] = peak;
        totals[warp] = total;
    }
    __syncthreads();
    float top = peaks[0], all = 0.0f, y = 0.0f;
    for (uint32_t w = 1; w < kWarps; ++w) top = fmaxf(top, peaks[w]);
    const uint64_t place = (static_cast<uint64_t>(b) * args.queries + query) * args.heads + head;
    for (uint32_t w = 0; w < kWarps; ++w) {
        const float share = peaks[w] == -INFINITY ? 0.0f : __expf(peaks[w] - top);
        all += totals[w] * share;
        if (threadIdx.x < D) y += sums[w][threadIdx.x] * share;
    }
    if (threadIdx.x < D)
        static_cast<uint16_t*>(args.out)[place * D + threadIdx.x] =
            static_cast<uint16_t>(E::pack(all == 0.0f ? 0.0f : y / all, 0.0f));
    if (threadIdx.x == 0 && args.lse) args.lse[place] = all == 0.0f ? -INFINITY : top + logf(all);
}

}  // namespace cache
}  // namespace fk

// ------------------------------------------------------------------ C ABI

using namespace fk;

/// What every entry asks of the cache itself.
static int check_cache(const fk_cache_t* cache) {
    if (!cache) return fk_fail(FK_ERR_INVALID, "the cache is null");
    if (!cache->k_codes || !cache->k_params || !cache->v_codes || !cache->v_params)
        return fk_fail(FK_ERR_INVALID, "a cache buffer is null");
    if (cache->element != FK_BF16 && cache->element != FK_F16)
        return fk_fail(FK_ERR_INVALID, "a cache is of bf16 or fp16 values, not element type %u", cache->element);
    if (cache->head_dim != 64 && cache->head_dim != 128)
        return fk_fail(FK_ERR_SHAPE, "head_dim %u is neither 64 nor 128", cache->head_dim);
    if ((cache->group != 32 && cache->group != 64 && cache->group != 128) || cache->group > cache->head_dim)
        return fk_fail(FK_ERR_SHAPE, "groups of %u do not divide a head of %u into groups of 32, 64 or 128", cache->group,
                       cache->head_dim);
    if (cache->pages == 0 || cache->page_size == 0 || cache->kv_heads == 0)
        return fk_fail(FK_ERR_SHAPE, "a cache of %u pages x %u tokens x %u heads is empty", cache->pages,
                       cache->page_size, cache->kv_heads);
    const unsigned __int128 rows =
        static_cast<unsigned __int128>(cache->pages) * cache->page_size * cache->kv_heads;
    if (rows >= (1ull << 31))
        return fk_fail(FK_ERR_SHAPE, "%u pages x %u tokens x %u heads is more than 2^31 - 1 rows", cache->pages,
                       cache->page_size, cache->kv_heads);
    if ((reinterpret_cast<uintptr_t>(cache->k_codes) | reinterpret_cast<uintptr_t>(cache->k_params) |
         reinterpret_cast<uintptr_t>(cache->v_codes) | reinterpret_cast<uintptr_t>(cache->v_params)) & 15u)
        return fk_fail(FK_ERR_ALIGNMENT, "cache buffers must be 16-byte aligned");
    return FK_OK;
}

/// `call(D, G, BF16)` with the cache's sizes and type as compile-time constants.
template <typename Call>
static int for_cache(const fk_cache_t* cache, Call call) {
#define FK_CACHE_CASE(D, G)                                                                     \
    if (cache->head_dim == D && cache->group == G)                                              \
        return cache->element == FK_BF16 ? call(std::integral_constant<int, D>{},               \
                                                std::integral_constant<int, G>{}, std::true_type{})  \
                                         : call(std::integral_constant<int, D>{},               \
                                                std::integral_constant<int, G>{}, std::false_type{});
    FK_CACHE_CASE(128, 128)
    FK_CACHE_CASE(128, 64)
    FK_CACHE_CASE(128, 32)
    FK_CACHE_CASE(64, 64)
    FK_CACHE_CASE(64, 32)
#undef FK_CACHE_CASE
    return fk_fail(FK_ERR_SHAPE, "no kernel for heads of %u in groups of %u", cache->head_dim, cache->group);
}

static int move_rows(bool write, const fk_cache_t* cache, const void* k, const void* v, int64_t k_token_stride,
                     int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, const void* slots,
                     uint32_t slot_bytes, uint32_t tokens, int clear_skipped, void* stream, uint32_t* device_status) {
    const int checked = check_cache(cache);
    if (checked != FK_OK) return checked;
    if (slot_bytes != 4 && slot_bytes != 8)
        return fk_fail(FK_ERR_INVALID, "slots are integers of 4 or 8 bytes, not %u", slot_bytes);
    if (tokens == 0) return FK_OK;
    if (!k || !v || !slots) return fk_fail(FK_ERR_INVALID, "an operand pointer is null");
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u)
        return fk_fail(FK_ERR_ALIGNMENT, "keys and values must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(slots) % slot_bytes)
        return fk_fail(FK_ERR_ALIGNMENT, "slots must be aligned to their %u bytes", slot_bytes);
    const int64_t strides[4] = {k_token_stride, k_head_stride, v_token_stride, v_head_stride};
    for (const int64_t stride : strides)
        if (stride % 8)
            return fk_fail(FK_ERR_ALIGNMENT, "a stride of %lld elements is no multiple of 8: rows move 16 bytes at a time",
                           static_cast<long long>(stride));
    if (static_cast<uint64_t>(tokens) * cache->kv_heads >= (1ull << 31))
        return fk_fail(FK_ERR_SHAPE, "%u tokens x %u heads is more than 2^31 - 1 rows", tokens, cache->kv_heads);
    DeviceFacts facts;
    const int known = device_facts(&facts);
    if (known != FK_OK) return known;
    cache::RowArguments args;
    args.tensor[0] = k;
    args.tensor[1] = v;
    args.codes[0] = static_cast<uint32_t*>(cache->k_codes);
    args.codes[1] = static_cast<uint32_t*>(cache->v_codes);
    args.params[0] = static_cast<uint32_t*>(cache->k_params);
    args.params[1] = static_cast<uint32_t*>(cache->v_params);
    args.token_stride[0] = 2 * k_token_stride;
    args.token_stride[1] = 2 * v_token_stride;
    args.head_stride[0] = 2 * k_head_stride;
    args.head_stride[1] = 2 * v_head_stride;
    args.slots = slots;
    args.slots_wide = slot_bytes == 8;
    args.tokens = tokens;
    args.rows = tokens * cache->kv_heads;
    args.capacity = static_cast<uint64_t>(cache->pages) * cache->page_size;
    args.page_size = cache->page_size;
    args.heads = cache::Divider(cache->kv_heads);
    args.page = cache::Divider(cache->page_size);
    args.clear_skipped = clear_skipped != 0;
    return for_cache(cache, [&](auto dim, auto group, auto bf16) {
        const uint32_t rows_a_block = cache::kRowThreads / (dim / 8);
        const uint32_t blocks = (args.rows + rows_a_block - 1) / rows_a_block;
        const uint32_t most = static_cast<uint32_t>(facts.sm_count) * 4;  // half of what fits; k and v are grid rows
        const dim3 grid(blocks < most ? blocks : most, 2);
        if (write)
            cache::write_kernel<dim, group, bf16>
                <<<grid, cache::kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(args, device_status);
        else
            cache::read_kernel<dim, group, bf16>
                <<<grid, cache::kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(args, device_status);
        FK_CUDA(cudaGetLastError());
        return static_cast<int>(FK_OK);
    });
}

extern "C" int fk_cache_write(const fk_cache_t* cache, const void* k, const void* v, int64_t k_token_stride,
                              int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                              const void* slots, uint32_t slot_bytes, uint32_t tokens, void* stream,
                              uint32_t* device_status) {
    return move_rows(true, cache, k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride, slots, slot_bytes,
                     tokens, 0, stream, device_status);
}

extern "C" int fk_cache_read(const fk_cache_t* cache, void* k, void* v, int64_t k_token_stride,
                             int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                             const void* slots, uint32_t slot_bytes, uint32_t tokens, int clear_skipped, void* stream,
                             uint32_t* device_status) {
    return move_rows(false, cache, k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride, slots, slot_bytes,
                     tokens, clear_skipped, stream, device_status);
}

extern "C" uint64_t fk_cache_attention_workspace_bytes(uint32_t sm_count) { return 16ull * sm_count; }

extern "C" int fk_cache_attention(const fk_cache_t* cache, const void* q, int64_t q_batch_stride,
                                  int64_t q_token_stride, int64_t q_head_stride, void* out, float* lse,
                                  const int32_t* lengths, const int32_t* table, int64_t table_stride,
                                  uint32_t table_pages, uint32_t batch, uint32_t queries, uint32_t heads, float scale,
                                  uint32_t window, uint32_t sinks, void* workspace, uint64_t workspace_bytes,
                                  void* stream, uint32_t* device_status) {
    const int checked = check_cache(cache);
    if (checked != FK_OK) return checked;
    if (heads == 0 || heads % cache->kv_heads)
        return fk_fail(FK_ERR_SHAPE, "%u query heads do not divide over %u kv heads", heads, cache->kv_heads);
    if (batch == 0 || queries == 0) return FK_OK;
    if (!q || !out || !lengths || !workspace) return fk_fail(FK_ERR_INVALID, "an operand pointer is null");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15u)
        return fk_fail(FK_ERR_ALIGNMENT, "queries, output and workspace must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(table)) & 3u)
        return fk_fail(FK_ERR_ALIGNMENT, "lse, lengths and table must be 4-byte aligned");
    const int64_t strides[3] = {q_batch_stride, q_token_stride, q_head_stride};
    for (const int64_t stride : strides)
        if (stride % 8)
            return fk_fail(FK_ERR_ALIGNMENT, "a stride of %lld elements is no multiple of 8: rows move 16 bytes at a time",
                           static_cast<long long>(stride));
    if (!table && batch > cache->pages)
        return fk_fail(FK_ERR_SHAPE, "%u sequences without a table own a page each, and the cache has %u", batch,
                       cache->pages);
    if (table && table_pages == 0) return fk_fail(FK_ERR_SHAPE, "the page table has no columns");
    const uint32_t columns = table ? table_pages : 1;
    const uint64_t capacity = static_cast<uint64_t>(columns) * cache->page_size;
    if (capacity >= (1ull << 31))
        return fk_fail(FK_ERR_SHAPE, "%u pages of %u tokens are more than 2^31 - 1 tokens a sequence", columns,
                       cache->page_size);
    DeviceFacts facts;
    const int known = device_facts(&facts);
    if (known != FK_OK) return known;
    if (workspace_bytes < fk_cache_attention_workspace_bytes(facts.sm_count))
        return fk_fail(FK_ERR_SHAPE, "a workspace of %llu bytes is under the %llu of this device",
                       static_cast<unsigned long long>(workspace_bytes),
                       static_cast<unsigned long long>(fk_cache_attention_workspace_bytes(facts.sm_count)));
    cache::AttentionArguments args;
    args.k_codes = static_cast<const uint8_t*>(cache->k_codes);
    args.k_params = static_cast<const uint32_t*>(cache->k_params);
    args.v_codes = static_cast<const uint8_t*>(cache->v_codes);
    args.v_params = static_cast<const uint32_t*>(cache->v_params);
    args.q = static_cast<const uint8_t*>(q);
    args.q_batch_stride = 2 * q_batch_stride;
    args.q_token_stride = 2 * q_token_stride;
    args.q_head_stride = 2 * q_head_stride;
    args.out = out;
    args.lse = lse;
    args.lengths = lengths;
    args.table = table;
    args.table_stride = table_stride;
    args.table_pages = columns;
    args.pages = cache->pages;
    args.page_size = cache->page_size;
    args.batch = batch;
    args.queries = queries;
    args.heads = heads;
    args.kv_heads = cache->kv_heads;
    args.scale = scale;
    args.window = window;
    args.sinks = sinks;
    args.page = cache::Divider(cache->page_size);
    return for_cache(cache, [&](auto dim, auto group, auto bf16) {
        cache::attention_kernel<dim, group, bf16>
            <<<dim3(queries * heads, batch), cache::kAttentionThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                args, device_status);
        FK_CUDA(cudaGetLastError());
        return static_cast<int>(FK_OK);
    });
}
