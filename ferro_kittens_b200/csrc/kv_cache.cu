// The key/value cache in 4 bits, for sm_100a: quantising tokens as they are written, reading rows back, and
// attention of a sequence's newest tokens over its rows. No counterpart in the reference, whose attention
// reads whole bf16 planes (examples/src/flash_forward.rs:151-158); the format is stated in the header.
//
// All three are bound by memory on paper. Shares below are of a plain copy's rate, 6.55 TB/s.

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <type_traits>

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

/// Everything before this launch on its stream is done and seen (see `launch`). Since the kernel has begun by then, nothing it reads counts
/// as constant for its lifetime: no load here is a non-coherent one.
__device__ __forceinline__ void wait_for_earlier_launches() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
/// The first bad index of a launch goes into the caller's status words: code, its upper half, where it stands, its lower half.
__device__ __forceinline__ void note(uint32_t* status, uint32_t code, uint32_t where, uint64_t value) {
    if (status && atomicCAS(status, 0u, code) == 0u) {
        status[1] = static_cast<uint32_t>(value >> 32);
        status[2] = where;
        status[3] = static_cast<uint32_t>(value);
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
    static __device__ __forceinline__ uint32_t max_nan(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    /// The smaller magnitude of each pair (the signs mean nothing).
    static __device__ __forceinline__ uint32_t min_magnitude(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    /// What of a sum's size a value must have, not to lie below its last bit: 2^-15 (8 significant bits of 24), made 2^-14.
    static constexpr float kVanishes = 0x1p-14f;
    static __device__ __forceinline__ bool finite(uint32_t pair) {
        return (pair & 0x7f80u) != 0x7f80u && (pair & 0x7f800000u) != 0x7f800000u;
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
    static __device__ __forceinline__ uint32_t max_nan(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    static __device__ __forceinline__ uint32_t min_magnitude(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("min.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    static constexpr float kVanishes = 0x1p-11f;
    static __device__ __forceinline__ bool finite(uint32_t pair) {
        return (pair & 0x7c00u) != 0x7c00u && (pair & 0x7c000000u) != 0x7c000000u;
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

/// Whether a group's parameters give finite values to weigh, their middle, low + 8 * scale, among them (that of written ones lies
/// between the smallest and the largest value).
template <bool BF16>
__device__ __forceinline__ bool usable_params(uint32_t pair) {
    using E = Element<BF16>;
    return E::finite(pair) && fabsf(fmaf(8.0f, E::low(pair), E::high(pair))) < __uint_as_float(0x7f800000u);
}

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

constexpr uint32_t kRowThreads = 128;

struct RowArguments {
    const void* tensor[2];  // k, v (the source of a write, the destination of a read)
    uint32_t* codes[2];
    uint32_t* params[2];
    int64_t token_stride[2], head_stride[2];  // bytes
    const void* slots;
    uint32_t slots_wide;
    uint32_t rows;          // tokens * kv_heads
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
        note(status, kBadSlot, token, static_cast<uint64_t>(slot));
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

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float one_if_ge(float a, float b) {
    float y;
    asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

/// {smallest, -largest} of a group together, NaN if it holds one: 8 channels (`x`) in each of G / 8 neighbouring lanes.
template <int G, bool BF16>
__device__ __forceinline__ uint32_t group_ends(const uint4 x) {
    using E = Element<BF16>;
    const uint32_t least = E::min_nan(E::min_nan(x.x, x.y), E::min_nan(x.z, x.w));
    const uint32_t most = E::max_nan(E::max_nan(x.x, x.y), E::max_nan(x.z, x.w)) ^ 0x80008000u;
    uint32_t ends = E::min_nan(__byte_perm(least, most, 0x5410), __byte_perm(least, most, 0x7632));
#pragma unroll
    for (uint32_t mask = 1; mask < G / 8; mask *= 2) ends = E::min_nan(ends, __shfl_xor_sync(0xffffffffu, ends, mask));
    return ends;
}

/// The group's scale in the low half and its smallest value in the high one, of its ends.
template <bool BF16>
__device__ __forceinline__ uint32_t group_params(uint32_t ends) {
    using E = Element<BF16>;
    const float low = E::low(ends), high = -E::high(ends);
    // Half the span (the span itself may pass fp32's range), and what its rounding left out, exactly (the error of a sum is
    // a float).
    const float a = 0.5f * high, b = 0.5f * low;
    const float half_span = a - b;
    const float b_part = half_span - a;
    const float lost = (a - (half_span - b_part)) - (b + b_part);
    const bool finite = half_span < __uint_as_float(0x7f800000u);  // false for NaN as well
    // The scale: half_span / 7.5 with a little added, cut to the type, is right or one too large, which 7.5 times it, exact,
    // tells.
    uint32_t scale_bits = E::truncate(half_span * (0x1.111112p-3f * (1.0f + 0x1p-21f)));
    const float product = 7.5f * E::low(scale_bits);
    if (product > half_span || (product == half_span && lost < 0.0f)) --scale_bits;
    return finite ? scale_bits | (ends << 16) : E::kNaN << 16;
}

/// The codes of 8 channels whose group has the parameters `params` and the largest value `high`.
template <bool BF16>
__device__ __forceinline__ uint32_t group_codes(const uint4 x, uint32_t params, float high) {
    using E = Element<BF16>;
    const uint32_t words[4] = {x.x, x.y, x.z, x.w};
    const float scale = E::low(params), low = E::high(params);
    const float half_step = 0.5f * scale, span = high - low;
    // A guess that is never above the code and at most one below: the quotient's error is under 2^-18. The remainder t -
    // guess * scale is exact, and a half step or more of it is one more.
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number
    const float inverse = rcp_approx(scale);
    const float2 origin2 = make_float2(-low, -low), inverse2 = make_float2(inverse, inverse);
    const float2 bias2 = make_float2(-0x1p-17f, -0x1p-17f), magic2 = make_float2(kMagic, kMagic);
    const float2 minus_magic2 = make_float2(-kMagic, -kMagic), minus_scale2 = make_float2(-scale, -scale);
    float2 code[4];
    float nearest = 0.0f;  // the largest remainder
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const float2 t = __fadd2_rn(make_float2(E::low(words[i]), E::high(words[i])), origin2);
        const float2 guess = __fadd2_rn(__fadd2_rn(__ffma2_rn(t, inverse2, bias2), magic2), minus_magic2);
        const float2 rest = __ffma2_rn(guess, minus_scale2, t);
        code[i] = __fadd2_rn(guess, make_float2(one_if_ge(rest.x, half_step), one_if_ge(rest.y, half_step)));
        nearest = fmaxf(nearest, fmaxf(rest.x, rest.y));
    }
    // t is exact but where a value or the smallest one all but vanishes in it: there its rounding may have made a half step of the
    // remainder. (Of one channel's, while another's may lie above half a step, by what the guess is low: so the largest remainder
    // says where none can be.) Where the scale was cut short (of a span of a few subnormals) codes pass 15, and far scales leave fp32's range
    // in t or in 1 / scale. All these go the long way, far scales lifted by 2^100 or halved (exactly).
    uint32_t small = E::min_magnitude(E::min_magnitude(words[0], words[1]), E::min_magnitude(words[2], words[3]));
    small = E::min_magnitude(small, __byte_perm(small, params, 0x7632));  // with its other half, and the smallest value
    const float vanishing = fminf(fabsf(E::low(small)), fabsf(E::high(small)));
    const bool far = scale < 0x1p-100f || scale > 0x1p100f;
    if (scale > 0.0f && ((nearest >= half_step && vanishing < span * E::kVanishes) || span >= 15.5f * scale || far)) {
        const float lift = scale > 0x1p100f ? 0.5f : scale < 0x1p-100f ? 0x1p100f : 1.0f;
        const float step = scale * lift, origin = -low * lift, lifted_half = 0.5f * step;
        const float lifted_inverse = __frcp_rn(step);
#pragma unroll 1
        for (uint32_t i = 0; i < 8; ++i) {
            const uint32_t pair = i < 4 ? (i < 2 ? words[0] : words[1]) : (i < 6 ? words[2] : words[3]);
            const float lifted = ((i & 1u) ? E::high(pair) : E::low(pair)) * lift;
            const float t = lifted + origin, o_part = t - lifted;
            const float t_lost = (lifted - (t - o_part)) + (origin - o_part);
            float c = fminf(rintf(t * lifted_inverse), 15.0f);
            const float rest = __fmaf_rn(c, -step, t);
            if ((rest - lifted_half) + t_lost >= 0.0f) c += 1.0f;
            else if ((rest + lifted_half) + t_lost < 0.0f) c -= 1.0f;
            c = fminf(c, 15.0f);
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (k == i) ((k & 1u) ? code[k / 2].y : code[k / 2].x) = c;
        }
    }
    // Four codes make a whole number under 2^16, which a sum with 2^23 leaves in the low bits.
    const float2 shift2 = make_float2(256.0f, 256.0f);
    const float2 front = __ffma2_rn(code[1], shift2, code[0]), back = __ffma2_rn(code[3], shift2, code[2]);
    const uint32_t first = __float_as_uint(__fmaf_rn(front.y, 16.0f, front.x) + 8388608.0f);
    const uint32_t last = __float_as_uint(__fmaf_rn(back.y, 16.0f, back.x) + 8388608.0f);
    return scale > 0.0f ? __byte_perm(first, last, 0x5410) : 0u;  // no span, or NaN: every code is 0
}

// One lane holds 8 channels (16 bytes) of a row's key and of its value, D / 8 lanes a row, ROWS rows of its own at a time: slots,
// then rows, of all of them are on their way before the first is worked on. The group's ends meet by shuffles of packed pairs;
// everything behind them is on packed fp32 pairs, without a division, and exact (see above). What bounds it is the issue of
// instructions (0.81 a cycle and scheduler, 175 a warp for 8 channels of its lanes): 150001 tokens of 8 heads of 64 fp16 values take 116 us, 53 %
// of the copy rate; 8191 tokens of 8 heads of 128 bf16 values 16 us.
template <int D, int G, int ROWS, bool BF16>
__global__ void __launch_bounds__(kRowThreads) write_kernel(const __grid_constant__ RowArguments args,
                                                            uint32_t* status) {
    constexpr uint32_t kLanes = D / 8, kAtATime = kRowThreads / kLanes;
    wait_for_earlier_launches();
    const uint32_t lane = threadIdx.x & 31u, block = threadIdx.x % kLanes;
    const uint32_t first = blockIdx.x * (kAtATime * ROWS) + threadIdx.x / kLanes;
    uint4 x[ROWS][2];
    uint64_t row[ROWS];
    bool kept[ROWS];
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) {
        const uint32_t index = min(first + r * kAtATime, args.rows - 1);
        const uint32_t token = args.heads.quotient(index), head = index - token * args.heads.divisor;
#pragma unroll
        for (uint32_t which = 0; which < 2; ++which)
            x[r][which] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(args.tensor[which]) +
                                                                token * args.token_stride[which] +
                                                                head * args.head_stride[which]) +
                                 block);
        kept[r] = first + r * kAtATime < args.rows && cache_row(args, token, head, row[r], status);
    }
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) {
        // Even lanes work out the key group's parameters, odd ones the value group's.
        const uint32_t ends[2] = {group_ends<G, BF16>(x[r][0]), group_ends<G, BF16>(x[r][1])};
        const uint32_t own = group_params<BF16>((lane & 1u) ? ends[1] : ends[0]);
        const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 1);
        const uint32_t params[2] = {(lane & 1u) ? other : own, (lane & 1u) ? own : other};
#pragma unroll
        for (uint32_t which = 0; which < 2; ++which) {
            uint32_t word = group_codes<BF16>(x[r][which], params[which], -Element<BF16>::high(ends[which]));
            if (which == 1) word = transpose_nibbles(word, lane);
            if (kept[r]) {
                args.codes[which][row[r] * (D / 8) + (which == 0 ? key_word<D>(block) : value_word<D>(block))] = word;
                if (block % (G / 8) == 0) args.params[which][row[r] * (D / G) + block / (G / 8)] = params[which];
            }
        }
    }
}

// The same lanes the other way: a code in the low mantissa bits of a power of two, less that power, is exact,
// and one fused multiply-add in the cache's type rounds low + code * scale once. 65536 tokens of 8 heads of 128 bf16 values take
// 59 us, 90 % of the copy rate (four fifths of the bytes are writes). Two rows a thread and blocks of 128 threads: with non-coherent
// loads 64 us, against 71 with 256 threads, 75 with one row, 74 and 87 with four and eight (registers that hold rows in flight cost
// threads).
template <int D, int G, int ROWS, bool BF16>
__global__ void __launch_bounds__(kRowThreads) read_kernel(const __grid_constant__ RowArguments args,
                                                           uint32_t* status) {
    using E = Element<BF16>;
    constexpr uint32_t kLanes = D / 8, kAtATime = kRowThreads / kLanes;
    wait_for_earlier_launches();
    const uint32_t lane = threadIdx.x & 31u, block = threadIdx.x % kLanes;
    const uint32_t first = blockIdx.x * (kAtATime * ROWS) + threadIdx.x / kLanes;
    uint32_t word[ROWS][2], pair[ROWS][2];
    bool kept[ROWS];
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) {
        const uint32_t index = min(first + r * kAtATime, args.rows - 1);
        const uint32_t token = args.heads.quotient(index), head = index - token * args.heads.divisor;
        uint64_t row = 0;
        kept[r] = cache_row(args, token, head, row, status);
        if (!kept[r]) row = 0;
#pragma unroll
        for (uint32_t which = 0; which < 2; ++which) {
            word[r][which] = args.codes[which][row * (D / 8) + (which == 0 ? key_word<D>(block) : value_word<D>(block))];
            pair[r][which] = args.params[which][row * (D / G) + block / (G / 8)];
            if (!kept[r]) word[r][which] = pair[r][which] = 0;  // reads as zeros
        }
    }
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) {
        const uint32_t index = first + r * kAtATime;
        const uint32_t token = args.heads.quotient(index), head = index - token * args.heads.divisor;
        word[r][1] = transpose_nibbles(word[r][1], lane);
#pragma unroll
        for (uint32_t which = 0; which < 2; ++which) {
            const uint32_t scale = __byte_perm(pair[r][which], 0, 0x1010), low = __byte_perm(pair[r][which], 0, 0x3232);
            uint32_t y[4];  // channels (i, i + 4)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                y[i] = E::fma(E::minus_magic(((word[r][which] >> (4 * i)) & 0x000f000fu) | E::kMagic), scale, low);
            if (index < args.rows && (kept[r] || args.clear_skipped))
                __stcs(reinterpret_cast<uint4*>(static_cast<uint8_t*>(const_cast<void*>(args.tensor[which])) +
                                                token * args.token_stride[which] + head * args.head_stride[which]) +
                           block,
                       make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410),
                                  __byte_perm(y[0], y[1], 0x7632), __byte_perm(y[2], y[3], 0x7632)));
        }
    }
}

// ---------------------------------------------------------------- attention

struct AttentionArguments {
    const uint8_t* codes[2];  // keys, values
    const uint8_t* params[2];
    const uint8_t* q;
    int64_t q_batch_stride, q_token_stride, q_head_stride;  // bytes
    uint16_t* out;
    float* lse;
    const int32_t* lengths;
    const int32_t* table;
    int64_t table_stride;
    uint32_t table_pages, pages, page_size;
    uint32_t batch, queries, heads, kv_heads;
    uint32_t rows, row_tiles;  // query rows of a (sequence, kv head): queries * heads / kv_heads
    float scale;
    int32_t window, sinks;
    Divider page, ratio, unit, tiles;  // by page_size, heads / kv_heads, a unit's tokens, row_tiles
    uint32_t segment_cost;  // what beginning and ending a segment takes, in units
    uint32_t copying;       // warps that copy: 1, 2 (a side each) or 4 (every other run of a side each)
    uint32_t* arrivals;    // workspace: a counter for each block, then the partial results
    float* partials;
};

constexpr uint32_t kWarpTokens = 32;
constexpr uint32_t kStages = 3;
constexpr uint32_t kMostBlocksPerSm = 3;
constexpr uint32_t kMostRows = 16;
/// Floats of one block's part of a segment: rows of outputs, then (peak, total) of each row.
constexpr uint32_t kPartialFloats = kMostRows * (128 + 2);
/// How far (in powers of two) a score may lie above its row's reference before the reference is moved: weights reach 2^kSlack.
constexpr float kSlack = 6.0f;
/// Each group of channels has a power of two, `fit`, that brings its value scales into [kLeast, kMost) for the product with the codes:
/// weight * scale * fit is under 2^15. A weight loses bits to fp16's subnormals under 2^-14 only, and errs by at most 2^-24 there, as its
/// scale's product with the row's largest weight, 1 or more. Tokens of scales outside the window are multiplied in fp32.
constexpr float kLeast = 0.5f, kMost = 512.0f;
constexpr int32_t kFitBiased = 254 + 4;  // less a scale's biased exponent: that of the power that brings it into [2^4, 2^5)
constexpr int32_t kMostFit = 253;        // biased exponents of powers whose inverses are normal numbers, too
/// That many tokens of 32 outside the window move it: their scales' mean exponent to 2^4. (32 sequences of up to 30000 tokens take 137 us,
/// 196 with one token in 32 outside.)
constexpr uint32_t kManyFar = 8;
constexpr int32_t kFarthest = 80;  // how far (in powers of two) a scale may lie above the window's middle, for fp32's range
constexpr uint32_t kStallFull = 0x504;  // a computing warp waiting for a stage of tokens
constexpr uint32_t kStallFree = 0x505;  // a copying warp waiting for a stage to be free

template <int D, int G, int NT>
struct AttentionShape {
    static constexpr uint32_t kGroups = D / G;
    static constexpr uint32_t kRows = 8 * NT;
    // One row tile's queries stay in registers; of more, the fragments, the groups' sums and what makes powers of two of the rows'
    // scores lie in shared memory.
    static constexpr bool kSharedQueries = NT > 1;
    static constexpr uint32_t kQueryBytes = kSharedQueries ? kRows * D * 2 + kRows * kGroups * 4 + kRows * 4 : 0;
    // For each computing warp: its tokens in each stage. The merge of the warps' results lies over the piece's last stage, which
    // is given back after it, or (where rows are more than fit there) beside.
    static constexpr uint32_t kCodeBytes = kWarpTokens * D / 2;
    static constexpr uint32_t kParamBytes = kWarpTokens * kGroups * 4;
    static constexpr uint32_t kStageBytes = 2 * kCodeBytes + 2 * kParamBytes;
    static constexpr uint32_t kPitch = D + 4;  // floats of a merged row: the four columns of a fragment fall in other banks
    static constexpr uint32_t kMergeBytes = kRows * kPitch * 4 + kRows * 8;
    static constexpr bool kMergeInRing = kMergeBytes <= kStageBytes;
    static constexpr uint32_t kScratchBytes = kMergeInRing ? 0 : kMergeBytes;
    static constexpr uint32_t kWarpBytes = kStages * kStageBytes + kScratchBytes;
    // Registers a thread: 128, or 168 where a lane holds more outputs or groups.
    static constexpr uint32_t kMostThreads = 32 * (D * NT <= 128 && kGroups <= 2 ? 16 : 12);
    /// Computing warps of each of `share` blocks on an SM: 228 KiB, of which every block takes 1 KiB, and its static part.
    static constexpr uint32_t most_warps(uint32_t share, uint32_t copying) {
        const uint32_t by_memory = (228 * 1024 / share - 2048 - kQueryBytes) / kWarpBytes, by_threads = kMostThreads / 32 / share - copying;
        return by_threads < by_memory ? by_threads : by_memory;
    }
    // A block alone on its SM has four copying warps, which need few registers: theirs go to the computing warps.
    static constexpr uint32_t kCopyingAlone = 4;
    static constexpr uint32_t kCopyingRegisters = 56;
    static constexpr uint32_t kLaunchRegisters = 65536 / kMostThreads / 8 * 8;
    static constexpr uint32_t kComputingRegisters =
        (kLaunchRegisters * kMostThreads - kCopyingRegisters * 32 * kCopyingAlone) / (kMostThreads - 32 * kCopyingAlone) / 8 * 8;
    static_assert(most_warps(1, kCopyingAlone) * 32 == kMostThreads - 32 * kCopyingAlone && kMostThreads % 128 == 0,
                  "registers change hands between whole warpgroups");
    static constexpr uint32_t shared_bytes(uint32_t warps) { return kQueryBytes + warps * kWarpBytes; }
};

/// What of a sequence is read: its tokens, less those between the sinks and the window that no query row sees.
struct Extent {
    int32_t length, first;  // tokens; the first query's position (0 if it lies before the first token)
    int32_t start;          // the first token that some row's window reaches
    int32_t kept, skipped;  // tokens read before the gap, and the gap's length, both multiples of 16: parameters are copied by 16 bytes
    __device__ __forceinline__ int32_t visible() const { return length - skipped; }
    __device__ __forceinline__ int32_t token(int32_t at) const { return at < kept ? at : at + skipped; }
};

__device__ __forceinline__ Extent extent_of(const AttentionArguments& args, uint32_t b, int32_t length, uint32_t* status) {
    Extent e;
    e.length = max(length, 0);
    const int32_t capacity = static_cast<int32_t>(args.table_pages * args.page_size);
    if (e.length > capacity) {
        note(status, kBadLength, b, static_cast<uint32_t>(e.length));
        e.length = capacity;
    }
    e.first = max(e.length - static_cast<int32_t>(args.queries), 0);
    e.start = args.window ? max(e.first + 1 - args.window, 0) : 0;
    e.kept = min((min(args.sinks, e.start) + 15) & ~15, e.start & ~15);
    e.skipped = (e.start & ~15) - e.kept;
    return e;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
        "l"(src), "r"(bytes), "r"(bar)
        : "memory");
}
/// BYTES of a row's parameters.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
/// The barrier's phase also waits for this thread's copy_async so far (one more arrival, made when they have landed).
__device__ __forceinline__ void copy_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
/// A rendezvous of the block's first `threads` threads, the warps that compute.
__device__ __forceinline__ void sync_computing(uint32_t threads) {
    asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
}

/// D[16, 8] += A[16, 16] . B[16, 8] in fp16 with fp32 sums.
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
    return d;
}
/// (x & mask) | more in one instruction, which the compiler otherwise makes two of where both are constants.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t more) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(mask), "r"(more));
    return d;
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ float power_of_two(int32_t biased) { return __int_as_float(biased << 23); }

template <int WORDS>
__device__ __forceinline__ void load_words(uint32_t (&w)[WORDS], const void* from) {
    if constexpr (WORDS == 8) {
        const uint4 x = static_cast<const uint4*>(from)[0], y = static_cast<const uint4*>(from)[1];
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w, w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
    } else if constexpr (WORDS == 4) {
        const uint4 x = *static_cast<const uint4*>(from);
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (WORDS == 2) {
        const uint2 x = *static_cast<const uint2*>(from);
        w[0] = x.x, w[1] = x.y;
    } else {
        w[0] = *static_cast<const uint32_t*>(from);
    }
}

/// One more at `counter`: what the block wrote before its last rendezvous comes first for whoever counts on, and what those that
/// counted before wrote comes first for this block's next one.
__device__ __forceinline__ uint32_t arrive(uint32_t* counter) {
    uint32_t before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    return before;
}

/// A piece of a segment (of its first row's tile), and if blocks share the segment, in how many parts and which block keeps count.
struct Cut {
    uint32_t b, kv_head, first_row, parts, owner;
};

/// Four channels of a row's output, and with the first its normaliser.
template <int D, bool BF16>
__device__ __forceinline__ void finish_row(const AttentionArguments& args, const Cut& piece, uint32_t row, uint32_t d, float4 y,
                                           float2 stat) {
    using E = Element<BF16>;
    const uint32_t r = piece.first_row + row, t = args.ratio.quotient(r);
    const uint64_t place = (static_cast<uint64_t>(piece.b) * args.queries + t) * args.heads +
                           piece.kv_head * args.ratio.divisor + (r - t * args.ratio.divisor);
    const bool empty = stat.y == 0.0f;
    const float inverse = empty ? 0.0f : __fdividef(1.0f, stat.y);
    if (empty) y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    *reinterpret_cast<uint2*>(args.out + place * D + d) =
        make_uint2(E::pack(y.x * inverse, y.y * inverse), E::pack(y.z * inverse, y.w * inverse));
    if (d == 0 && args.lse) args.lse[place] = empty ? -INFINITY : (stat.x + log2f(stat.y)) * 0.6931471805599453f;
}

// Attention. Of one sequence and kv head (a segment), for up to 8 NT of its query rows: with key codes c, scale s, low l of each
// group g of channels, values alike (c', s', l'), and F = scale * log2(e),
//   x_j = sum_g (s_jg * sum_{d in g} q_d c_jd + l_jg * sum_{d in g} q_d),  p_j = 2^(F (x_j - x_ref)),
//   O_d = (sum_j (p_j s'_jg) (c'_jd - 8) + sum_j p_j (l'_jg + 8 s'_jg)) / sum_j p_j
// so that the matrix instructions only ever see codes, which are exact fp16 subnormals as they lie in the cache, and no code is
// ever multiplied out. Scores and outputs are computed transposed (tokens, then channels, are the rows of the m16n8k16
// fragments, query rows the columns): eight rows fill the instruction, a lane holds two tokens' parameters, and a code that is
// unpacked once serves all of them. Sums, references and the l terms are fp32; p s' is rounded to fp16 (relative 2^-11, of terms
// that count from the middle of the codes, or 2^-24 of s' and the row's largest p: see kLeast), queries are of a power of two for each
// row.
//
// A block computes with most of its warps, each 32 tokens of a unit at a time, and copies with the rest through a ring of stages
// on barriers (bulk copies of a page's run at a time; every wait is bounded). The units of all sequences, heads and row tiles
// form one line, cut evenly over the blocks on the device, since the lengths live there: a block's share may begin and end inside
// a segment. Warps' parts of a piece meet in shared memory, blocks' parts of a segment in the workspace, where the block that
// comes last adds them up in the order of the line: the same bits every time.
//
// What bounds it: for an SM's part of the copy rate (23 bytes a cycle) the 16 tokens of a warp's step, 2304 bytes of a 128-wide
// head in groups of 64, may take 98 cycles. All told a step is 363 warp instructions, 91 cycles of the four schedulers; 157 of
// them are masks, shifts and permutes on the ALU, which takes one every other cycle: 78 cycles; 16 are matrix products of 8 cycles: 33.
// Four warps a scheduler, all of them on dependent chains (masks, products, exponentials, products), issue in 63 % of the cycles
// and keep the ALU busy for 54 %: the kernel is bound by latency and issue, not by memory (49 % of its peak under the profiler). Of
// 128-wide heads in groups of 64, one query a sequence: 32 ragged sequences of up to 30000 tokens, 8 kv heads with 8 query heads
// each, 137 us (64 % of the copy rate); one of 131072 tokens 45 us (51 %); 48 of up to 4096 tokens 46 us (39 %); one
// of 777 with 4 query heads each 14 us, all of it beginnings and ends: lengths, queries, first copies, merging.
// Tried and slower or no faster: parameters widened to floats in shared memory (its wavefronts are then 80 % of what it can do),
// every warp sending its own copies (a bulk copy takes its warp some 150 cycles), small runs copied 16 bytes a lane, 2 or 4
// stages instead of 3, the next piece's queries held in registers (spills). Tiles of 32 rows missed the tolerance: they left no
// registers to centre the codes in.
template <int D, int G, int NT, bool BF16, bool ALONE>
__global__ void __launch_bounds__(AttentionShape<D, G, NT>::kMostThreads, 1)
    attention_kernel(const __grid_constant__ AttentionArguments args, uint32_t* status) {
    using E = Element<BF16>;
    using Shape = AttentionShape<D, G, NT>;
    constexpr uint32_t kGroups = Shape::kGroups, kRows = Shape::kRows, kPitch = Shape::kPitch;
    constexpr uint32_t kKeyWords = D / 32, kValueWords = D / 64, kTiles = D / 16;
    extern __shared__ __align__(16) uint8_t shared[];
    __shared__ uint64_t barriers[2 * kStages];  // of each stage: it is full; it is free again
    __shared__ uint32_t bad_pages[kStages];     // whether a stage has places whose page lies outside the cache
    __shared__ uint32_t stop_flag, complete[2];
    __shared__ Cut cuts[2];              // the parts of segments that are cut over blocks: the one this share begins in, ends in
    // The first warps compute, the last ones copy.
    const uint32_t warps = blockDim.x / 32 - args.copying, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t unit_tokens = warps * kWarpTokens;
    uint8_t* const ring = shared + Shape::kQueryBytes;
    const uint32_t stage_bytes = warps * Shape::kStageBytes, value_codes = warps * Shape::kCodeBytes;

    wait_for_earlier_launches();
    int32_t length_here = lane < args.batch ? args.lengths[lane] : 0;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(barriers + 2 * i), args.copying);
            mbar_init(smem_u32(barriers + 2 * i + 1), warps);
        }
        stop_flag = cuts[0].parts = cuts[1].parts = 0;
    }
    fence_mbarrier_init();

    // ---- this block's share: units of unit_tokens tokens, sequence by sequence, (kv head, row tile) by (kv head,
    // row tile), cut evenly over the blocks whatever the lengths are. A segment, one sequence's units of one (kv
    // head, row tile), begins with args.segment_cost units of no work: what beginning and ending it takes. Every warp
    // goes through the lengths by itself.
    const uint32_t segments = args.kv_heads * args.row_tiles;  // of one sequence
    const auto cost_of = [&](const Extent& e) {
        return max(args.unit.quotient(static_cast<uint32_t>(e.visible()) + unit_tokens - 1), 1u) + args.segment_cost;
    };
    uint32_t mine = lane < args.batch ? cost_of(extent_of(args, lane, length_here, status)) : 0, total = mine;
    for (uint32_t i = lane + 32; i < args.batch; i += 32) total += cost_of(extent_of(args, i, args.lengths[i], status));
    total = __reduce_add_sync(0xffffffffu, total) * segments;
    const uint32_t blocks = min(gridDim.x, max(total / 2, 1u));
    if (blockIdx.x >= blocks) return;
    // The first `longer` blocks take a unit more than the others.
    const uint32_t share = total / blocks, longer = total - share * blocks;
    const auto block_of = [&](uint32_t place) {
        const uint32_t behind = longer * (share + 1);
        return place < behind ? place / (share + 1) : longer + (place - behind) / share;
    };
    uint32_t at = blockIdx.x * share + min(blockIdx.x, longer);
    const uint32_t end = at + share + (blockIdx.x < longer ? 1 : 0);
    uint32_t b = 0, before = 0;
    for (uint32_t chunk = 0;; chunk += 32) {
        if (chunk) {
            length_here = chunk + lane < args.batch ? args.lengths[chunk + lane] : 0;
            mine = chunk + lane < args.batch ? cost_of(extent_of(args, chunk + lane, length_here, nullptr)) : 0;
        }
        uint32_t sum = mine * segments;
#pragma unroll
        for (uint32_t d = 1; d < 32; d *= 2) {
            const uint32_t other = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += other;
        }
        // The lane whose sequence the share begins in: the first whose sum passes it.
        const uint32_t past = __ballot_sync(0xffffffffu, at < before + sum);
        if (past) {
            const uint32_t found = __ffs(past) - 1;
            b = chunk + found;
            before += __shfl_sync(0xffffffffu, sum - mine * segments, found);
            length_here = __shfl_sync(0xffffffffu, length_here, found);
            break;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }

    __syncthreads();
    const StallSite site{status, &stop_flag, 0};
    bool live = true;  // until a wait gives up: nothing is waited for after that

    Extent extent = extent_of(args, b, length_here, nullptr);
    uint32_t cost = cost_of(extent);
    uint32_t segment = (at - before) / cost;
    uint32_t offset = (at - before) - segment * cost;  // of `at` in its segment
    uint32_t stage = 0, parity = 0;
    // The piece at hand: units [from, to) of the segment (b, kv_head, rows from first_row).
    uint32_t length = 0, from = 0, to = 0, kv_head = 0, first_row = 0;
    const auto units_of = [&](uint32_t its_cost) { return its_cost - args.segment_cost; };
    const auto find_piece = [&]() {
        while (at < end) {
            length = min(cost - offset, end - at);  // of the share that lies in this segment
            from = offset > args.segment_cost ? offset - args.segment_cost : 0;
            to = offset + length > args.segment_cost ? offset + length - args.segment_cost : 0;
            if (from < to) {
                kv_head = args.tiles.quotient(segment);
                first_row = (segment - kv_head * args.row_tiles) * kRows;
                return true;
            }
            at += length;  // only the segment's beginning lies in this share
        }
        return false;
    };
    const auto next_piece = [&]() {
        at += length;
        if (at >= end) return false;
        offset = 0;
        if (++segment == segments) {
            segment = 0;
            ++b;
            extent = extent_of(args, b, args.lengths[b], nullptr);
            cost = cost_of(extent);
        }
        return find_piece();
    };

    const auto page_at = [&](int32_t place) {
        return args.table ? static_cast<uint32_t>(args.table[b * args.table_stride + args.page.quotient(extent.token(place))]) : b;
    };
    const auto next_stage = [&]() {
        stage = stage == kStages - 1 ? 0 : stage + 1;
        parity ^= stage == 0;
    };

    if (warp >= warps) {
        if constexpr (ALONE) setmaxnreg_dec<Shape::kCopyingRegisters>();
        // ---- copies: tokens that follow each other in a page are one run, copied in bulk, codes and parameters. (Parameters
        // of runs that do not begin and end on 16 bytes go token by token.) Lane r works out run r of a unit; the pages of the
        // next unit's runs are asked for before the present one's are copied, by one thread after another's numbers.
        const uint32_t side = (warp - warps) & 1u;
        const bool first_copying = warp == warps;
        const uint32_t own_runs = args.copying < 4 ? 0xffffffffu : warp - warps < 2 ? 0x55555555u : 0xaaaaaaaau;
        struct Run {
            uint32_t entry, inside, at, length;  // page of the sequence, place in it, place in the unit, tokens
        };
        const auto run_of = [&](uint32_t unit, uint32_t r, Run& run) {
            const int32_t place = static_cast<int32_t>(unit * unit_tokens);
            const int32_t count = min(extent.visible() - place, static_cast<int32_t>(unit_tokens));
            // Before the gap between sinks and window, and behind it, tokens follow each other.
            const int32_t front = max(min(extent.kept - place, count), 0);
            uint32_t base = 0;
#pragma unroll
            for (uint32_t part = 0; part < 2; ++part) {
                const uint32_t tokens = static_cast<uint32_t>(part ? max(count - front, 0) : front);
                if (tokens == 0) continue;
                const uint32_t begin = static_cast<uint32_t>(part ? place + front + extent.skipped : place);
                const uint32_t first = args.page.quotient(begin), runs = args.page.quotient(begin + tokens - 1) - first + 1;
                if (r < base + runs) {
                    run.entry = first + (r - base);
                    const uint32_t page_begin = run.entry * args.page_size, start = max(begin, page_begin);
                    run.inside = start - page_begin;
                    run.length = min(begin + tokens - start, args.page_size - run.inside);
                    run.at = start - begin + (part ? front : 0);
                    return true;
                }
                base += runs;
            }
            return false;
        };
        const auto page_of = [&](const Run& run) {
            return args.table ? static_cast<uint32_t>(args.table[b * args.table_stride + run.entry]) : b;
        };
        for (bool more = find_piece(); more; more = next_piece()) {
            Run run;
            bool there = run_of(from, lane, run);
            uint32_t page = there ? page_of(run) : 0;
            for (uint32_t unit = from; unit < to; ++unit) {
                const uint32_t full = smem_u32(barriers + 2 * stage), memory = smem_u32(ring) + stage * stage_bytes;
                Run then;
                const bool then_there = unit + 1 < to && run_of(unit + 1, lane, then);
                const uint32_t then_page = then_there ? page_of(then) : 0;
                if (!mbar_wait(full + 8, parity ^ 1, site, kStallFree, unit)) return;
                uint32_t bytes = 0;
                bool bad = false, single = false;
                for (uint32_t chunk = 32;; chunk += 32) {
                    const bool sound = there && page < args.pages;
                    if (there && !sound) {
                        bad = true;
                        // (Of a page that only fills up 16 tokens beside the gap no row sees anything: it may be gone.)
                        const int32_t begin = static_cast<int32_t>(run.entry * args.page_size + run.inside);
                        const bool seen = begin < args.sinks || begin + static_cast<int32_t>(run.length) > extent.start;
                        if (first_copying && seen) note(status, kBadPage, b, page);
                    }
                    const uint32_t row = (page * args.kv_heads + kv_head) * args.page_size + run.inside;
                    for (uint32_t left = __ballot_sync(0xffffffffu, sound) & own_runs; left; left &= left - 1) {
                        const uint32_t lane_of = __ffs(left) - 1;
                        const uint64_t its_row = __shfl_sync(0xffffffffu, row, lane_of);
                        const uint32_t at = __shfl_sync(0xffffffffu, run.at, lane_of);
                        const uint32_t length = __shfl_sync(0xffffffffu, run.length, lane_of);
                        const uint32_t param_bytes = length * (kGroups * 4);
                        const bool aligned = ((static_cast<uint32_t>(its_row * (kGroups * 4)) | at * (kGroups * 4) | param_bytes) & 15u) == 0;
                        const uint32_t moved = length * (D / 2) + (aligned ? param_bytes : 0);
                        bytes += args.copying > 1 ? moved : 2 * moved;
                        single |= !aligned;
                        if (elect_one()) {
#pragma unroll
                            for (uint32_t which = 0; which < 2; ++which) {
                                if (args.copying > 1 && which != side) continue;
                                bulk_load(memory + which * value_codes + at * (D / 2), args.codes[which] + its_row * (D / 2),
                                          length * (D / 2), full);
                                const uint8_t* const params = args.params[which] + its_row * (kGroups * 4);
                                const uint32_t params_at =
                                    memory + 2 * value_codes + which * warps * Shape::kParamBytes + at * (kGroups * 4);
                                if (aligned) {
                                    bulk_load(params_at, params, param_bytes, full);
                                } else {
#pragma unroll 1
                                    for (uint32_t i = 0; i < param_bytes; i += kGroups * 4)
                                        copy_async<kGroups * 4>(params_at + i, params + i);
                                }
                            }
                        }
                        __syncwarp();
                    }
                    there = run_of(unit, chunk + lane, run);
                    if (!__any_sync(0xffffffffu, there)) break;
                    page = there ? page_of(run) : 0;
                }
                bad = __any_sync(0xffffffffu, bad);
                if (elect_one()) {
                    if (first_copying) bad_pages[stage] = bad;
                    if (single) copy_async_arrive(full);
                    mbar_arrive_expect_tx(full, bytes);
                }
                __syncwarp();
                run = then;
                there = then_there;
                page = then_page;
                next_stage();
            }
        }
        return;
    }

    if constexpr (ALONE) setmaxnreg_inc<Shape::kComputingRegisters>();
    const uint32_t l4 = lane / 4, c4 = lane % 4;
    // Row l4 of tile n, and its largest magnitude (a NaN's aside; 0 if there is an infinity: the row is NaN whatever it is scaled by).
    const auto load_row = [&](uint32_t n, uint4 (&raw)[kKeyWords]) {
        const uint32_t r = first_row + 8 * n + l4, t = args.ratio.quotient(min(r, args.rows - 1));
        const uint8_t* const q = args.q + b * args.q_batch_stride + t * args.q_token_stride +
                                 (kv_head * args.ratio.divisor + (r - t * args.ratio.divisor)) * args.q_head_stride;
        float most = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kKeyWords; ++w) {
            raw[w] = r < args.rows ? reinterpret_cast<const uint4*>(q)[4 * w + c4] : make_uint4(0, 0, 0, 0);
            const uint32_t words[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) most = fmaxf(most, fmaxf(fabsf(E::low(words[i])), fabsf(E::high(words[i]))));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        return most < INFINITY ? most : 0.0f;
    };
    // A piece's queries, on their way to the nearest cache while the piece before is put together.
    const auto fetch_rows = [&]() {
        for (uint32_t r = first_row + warp; r < min(first_row + kRows, args.rows); r += warps) {
            const uint32_t t = args.ratio.quotient(r);
            const uint8_t* const q = args.q + b * args.q_batch_stride + t * args.q_token_stride +
                                     (kv_head * args.ratio.divisor + (r - t * args.ratio.divisor)) * args.q_head_stride;
            if (lane < D / 64) asm volatile("prefetch.global.L1 [%0];" ::"l"(q + lane * 128));
        }
    };
    // The parts of a piece's rows (`parts` of them, `pitch` bytes apart, rows of kPitch floats, then each row's reference and sum)
    // put together: by each block its warps' parts, and by the block that comes last to a segment the blocks'.
    const auto put_together = [&](uint8_t* memory, uint32_t pitch, const Cut& piece, float* part) {
        const uint32_t rows_here = min(kRows, args.rows - piece.first_row);
        for (uint32_t i = threadIdx.x; i < rows_here * (D / 4); i += warps * 32) {
            const uint32_t row = i / (D / 4), d = i % (D / 4) * 4;
            const auto stat_of = [&](uint32_t w) {
                return reinterpret_cast<const float2*>(memory + w * pitch + kRows * kPitch * 4)[row];
            };
            float2 stat = make_float2(-INFINITY, 0.0f);
#pragma unroll 4
            for (uint32_t w = 0; w < warps; ++w) stat.x = fmaxf(stat.x, stat_of(w).x);
            const float minus = stat.x == -INFINITY ? 0.0f : -stat.x;
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (uint32_t w = 0; w < warps; ++w) {
                const float2 its = stat_of(w);
                const float factor = ex2_approx(its.x + minus);
                const float4 z = *reinterpret_cast<const float4*>(memory + w * pitch + (row * kPitch + d) * 4);
                y = make_float4(fmaf(z.x, factor, y.x), fmaf(z.y, factor, y.y), fmaf(z.z, factor, y.z), fmaf(z.w, factor, y.w));
                stat.y = fmaf(its.y, factor, stat.y);
            }
            if (!part) {
                finish_row<D, BF16>(args, piece, row, d, y, stat);
            } else {
                *reinterpret_cast<float4*>(part + row * D + d) = y;
                if (d == 0) *reinterpret_cast<float2*>(part + kMostRows * 128 + 2 * row) = stat;
            }
        }
    };

    bool more = find_piece();
    while (more) {
        // ---- queries as the second operand of the scores' product: lane (l4, c4) holds row l4 of each 8, in the
        // channel order of the key codes. Each row is scaled by a power of two of its own, so that its largest value lies in
        // [2^14, 2^15) whatever the other rows hold. The second register of each pair carries 1/16 for the codes that stay in the
        // upper nibble, so its fp16 form is exact down to 2^-27 of the largest value in bf16 and 2^-24 in fp16, and below that
        // off by 2^-35 of the largest value. q_sum is a group's sum, for the smallest values; to_log2 makes scores of a row's products, in
        // powers of two.
        uint32_t qf[Shape::kSharedQueries ? 1 : D / 16][2];
        float q_sum[Shape::kSharedQueries ? 1 : kGroups][2];
        uint4* const shared_q = reinterpret_cast<uint4*>(shared);
        float* const shared_sums = reinterpret_cast<float*>(shared + kRows * D * 2);
        float* const shared_log2 = shared_sums + kRows * kGroups;
        const auto power_for = [](float most) {
            return most == 0.0f ? 127 : min(268 - static_cast<int32_t>(__float_as_uint(most) >> 23), 254);
        };
        // (With a scale of 0 every finite score is 0, whatever the keys.)
        const auto factor_for = [&](int32_t power) {
            return args.scale == 0.0f ? 0.0f : args.scale < 0.0f ? -power_of_two(power) : power_of_two(power);
        };
        // |scale| log2(e) 2^24 / 2^(power - 127), in two steps that stay inside fp32's range, and kept off its ends: zero or an infinity
        // would make NaN of a hidden token's -inf or of equal scores' difference.
        const auto log2_for = [&](int32_t power) {
            const int32_t exponent = 151 - power, half = exponent / 2;
            const float x = fabsf(args.scale) * 1.4426950408889634f * power_of_two(127 + half) * power_of_two(127 + exponent - half);
            return fminf(fmaxf(x, 1e-37f), 0x1p126f);
        };
        const auto convert_row = [&](const uint4 (&raw)[kKeyWords], float up, uint4 (&f)[kKeyWords], float (&sums)[kGroups]) {
#pragma unroll
            for (uint32_t w = 0; w < kKeyWords; ++w) {
                const uint32_t words[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
                float v[8];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    v[2 * i] = E::low(words[i]) * up;
                    v[2 * i + 1] = E::high(words[i]) * up;
                    sums[w * 32 / G] += v[2 * i] + v[2 * i + 1];
                }
                f[w].x = Element<false>::pack(v[0], v[4]);
                f[w].y = Element<false>::pack(v[1] * 0.0625f, v[5] * 0.0625f);
                f[w].z = Element<false>::pack(v[2], v[6]);
                f[w].w = Element<false>::pack(v[3] * 0.0625f, v[7] * 0.0625f);
            }
#pragma unroll
            for (uint32_t g = 0; g < kGroups; ++g) {
                sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
                sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
                sums[g] *= 0x1p-24f;
            }
        };
        float2 to_log2[NT];
        {
            uint4 raw[kKeyWords], f[kKeyWords];
            if constexpr (Shape::kSharedQueries) {
                for (uint32_t n = warp; n < NT; n += warps) {
                    float sums[kGroups] = {};
                    const int32_t power = power_for(load_row(n, raw));
                    convert_row(raw, factor_for(power), f, sums);
#pragma unroll
                    for (uint32_t w = 0; w < kKeyWords; ++w) shared_q[(n * kKeyWords + w) * 32 + lane] = f[w];
                    if (c4 == 0) {
#pragma unroll
                        for (uint32_t g = 0; g < kGroups; ++g) shared_sums[g * kRows + 8 * n + l4] = sums[g];
                        shared_log2[8 * n + l4] = log2_for(power);
                    }
                }
                sync_computing(warps * 32);
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n) to_log2[n] = *reinterpret_cast<const float2*>(shared_log2 + 8 * n + 2 * c4);
            } else {
                const int32_t power = power_for(load_row(0, raw));
                float sums[kGroups] = {};
                convert_row(raw, factor_for(power), f, sums);
#pragma unroll
                for (uint32_t w = 0; w < kKeyWords; ++w)
                    qf[2 * w][0] = f[w].x, qf[2 * w][1] = f[w].y, qf[2 * w + 1][0] = f[w].z, qf[2 * w + 1][1] = f[w].w;
#pragma unroll
                for (uint32_t g = 0; g < kGroups; ++g)
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) q_sum[g][e] = __shfl_sync(0xffffffffu, sums[g], 8 * c4 + 4 * e);
                const float own = log2_for(power);
                to_log2[0] = make_float2(__shfl_sync(0xffffffffu, own, 8 * c4), __shfl_sync(0xffffffffu, own, 8 * c4 + 4));
            }
        }

        // Pairs are a fragment's two rows. Scores are the products' sums; times to_log2 they are powers of two. minus_peak is the
        // row's reference in powers of two, negated, and ceiling the score 2^kSlack above it: 0 and -inf while nothing is seen.
        float out[kTiles][NT][4] = {};
        float2 lows[kGroups][NT] = {}, ceiling[NT], minus_peak[NT] = {}, sum[NT] = {};
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n) ceiling[n] = make_float2(-INFINITY, -INFINITY);
        float fit[kGroups] = {};  // 0 before the group's first scale

        // Rows of S^T: the tokens of fragment rows 2c and 2c + 1 are 2c and 2c + 1, in this order for c < 2 and in the other
        // for the rest, so that neither the keys' loads (both rows at once) nor the values' (one of each c) crowd the same banks.
        const uint32_t own_token = l4 ^ (l4 >> 2);

#pragma unroll 1
        for (uint32_t unit = from; unit < to; ++unit) {
            const uint32_t full = smem_u32(barriers + 2 * stage);
            if (live) live = mbar_wait(full, parity, site, kStallFull, unit);
            const uint8_t* const keys = ring + stage * stage_bytes + warp * Shape::kCodeBytes;
            const uint8_t* const values = keys + value_codes;
            const uint8_t* const key_params = ring + stage * stage_bytes + 2 * value_codes + warp * Shape::kParamBytes;
            uint8_t* const value_params = const_cast<uint8_t*>(key_params) + warps * Shape::kParamBytes;
            // Whether some row may not see some of the 32 tokens (they rise from place to place), or some are not there.
            const int32_t place = static_cast<int32_t>(unit * unit_tokens + warp * kWarpTokens), here = extent.visible() - place;
            if (here <= 0) {  // nothing of the unit is this warp's
                if (unit + 1 == to) break;
                if (lane == 0) mbar_arrive(full + 8);
                next_stage();
                continue;
            }
            const bool is_masked = here < 32 || bad_pages[stage] || extent.token(place + 31) > extent.first ||
                                   (args.window && extent.token(place + 31) >= args.sinks &&
                                    extent.token(place) <= extent.length - 1 - args.window);

            bool grows = false;
            {
                uint32_t pairs[kGroups];  // lane = token
                load_words(pairs, value_params + lane * (kGroups * 4));
                float least = INFINITY, most = 0.0f;
#pragma unroll
                for (uint32_t g = 0; g < kGroups; ++g) {
                    const float fitted = E::low(pairs[g]) * fit[g];
                    least = fminf(least, fabsf(fitted));
                    most = fmaxf(most, fabsf(fitted));
                }
                grows = least < kLeast || most >= kMost;
            }

            // ---- scores, transposed. A code in the low nibble of a half word IS the fp16 number code * 2^-24 (a
            // subnormal), one in the next nibble code * 2^-20: masks alone unpack them, and products are exact.
            float2 x[2][NT][2];  // [step of 16 tokens][row tile][token of the fragment's upper or lower half] (two rows)
            // Both steps' products, for each load of a query fragment. (With 8 rows, whose fragments stay in registers, it is the
            // two chains that count: 46.4 us for one sequence of 131072 against 48.7 step by step.)
            const auto products = [&](uint32_t g, const uint32_t (&a)[2][2][kKeyWords], float (&part)[2][NT][4]) {
#pragma unroll
                for (uint32_t w = g * (G / 32); w < (g + 1) * (G / 32); ++w)
#pragma unroll
                    for (uint32_t n = 0; n < NT; ++n) {
                        uint32_t f[4];
                        if constexpr (Shape::kSharedQueries)  // each time anew: registers are full
                            ld_shared_v4(smem_u32(shared_q + (n * kKeyWords + w) * 32 + lane), f);
                        else
                            f[0] = qf[2 * w][0], f[1] = qf[2 * w][1], f[2] = qf[2 * w + 1][0], f[3] = qf[2 * w + 1][1];
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            const uint32_t y0 = a[h][0][w] >> 8, y1 = a[h][1][w] >> 8;
                            mma_16x8x16(part[h][n], a[h][0][w] & 0x000f000fu, a[h][1][w] & 0x000f000fu, a[h][0][w] & 0x00f000f0u,
                                        a[h][1][w] & 0x00f000f0u, f[0], f[1]);
                            mma_16x8x16(part[h][n], y0 & 0x000f000fu, y1 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x00f000f0u, f[2],
                                        f[3]);
                        }
                    }
            };
            const auto load_keys = [&](uint32_t h, uint32_t (&a)[2][kKeyWords]) {
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half)
                    load_words(a[half], keys + (16 * h + 8 * half + own_token) * (D / 2) + c4 * (D / 8));
            };
            const auto add_up = [&](uint32_t h, uint32_t g, const uint32_t (&pairs)[2][kGroups], const float (&part)[NT][4]) {
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half) {
                    const float scale = E::low(pairs[half][g]), low = E::high(pairs[half][g]);
#pragma unroll
                    for (uint32_t n = 0; n < NT; ++n) {
                        float2 sums;
                        if constexpr (Shape::kSharedQueries)
                            sums = *reinterpret_cast<const float2*>(shared_sums + g * kRows + 8 * n + 2 * c4);
                        else
                            sums = make_float2(q_sum[g][0], q_sum[g][1]);
                        float2& y = x[h][n][half];
                        y.x = fmaf(scale, part[n][2 * half], g == 0 ? low * sums.x : fmaf(low, sums.x, y.x));
                        y.y = fmaf(scale, part[n][2 * half + 1], g == 0 ? low * sums.y : fmaf(low, sums.y, y.y));
                    }
                }
            };
            uint32_t a[2][2][kKeyWords], pairs[2][2][kGroups];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                load_keys(h, a[h]);
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half)
                    load_words(pairs[h][half], key_params + (16 * h + 8 * half + own_token) * (kGroups * 4));
            }
#pragma unroll
            for (uint32_t g = 0; g < kGroups; ++g) {
                float part[2][NT][4] = {};
                products(g, a, part);
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) add_up(h, g, pairs[h], part[h]);
            }

            // ---- what rarely happens, all in one place: tokens that some row may not see; a score more than kSlack above its
            // row's reference, the score that its exponentials are taken from (so that weights stay under 2^kSlack); a
            // value scale outside its group's window.
            float2 largest[NT];
            const auto look = [&]() {
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n)
                    largest[n] = make_float2(fmaxf(fmaxf(x[0][n][0].x, x[0][n][1].x), fmaxf(x[1][n][0].x, x[1][n][1].x)),
                                             fmaxf(fmaxf(x[0][n][0].y, x[0][n][1].y), fmaxf(x[1][n][0].y, x[1][n][1].y)));
            };
            look();
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) grows |= largest[n].x > ceiling[n].x || largest[n].y > ceiling[n].y;
            if (is_masked || __any_sync(0xffffffffu, grows)) {
                if (is_masked) {
                    const int32_t own = extent.token(place + static_cast<int32_t>(lane));
                    uint32_t real = __ballot_sync(0xffffffffu, static_cast<int32_t>(lane) < here &&
                                                                   (!args.window || own >= extent.start || own < args.sinks));
                    if (bad_pages[stage])
                        real &= __ballot_sync(0xffffffffu, static_cast<int32_t>(lane) < here && page_at(place + lane) < args.pages);
#pragma unroll
                    for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                        for (uint32_t e = 0; e < 2; ++e) {
                            const uint32_t t = args.ratio.quotient(min(first_row + 8 * n + 2 * c4 + e, args.rows - 1));
                            const int32_t i = extent.length - static_cast<int32_t>(args.queries) + static_cast<int32_t>(t);
#pragma unroll
                            for (uint32_t k = 0; k < 4; ++k) {
                                const uint32_t its = 8 * k + own_token;
                                const int32_t j = extent.token(place + static_cast<int32_t>(its));
                                if (!(real >> its & 1u) || j > i || (args.window && j <= i - args.window && j >= args.sinks))
                                    (e ? x[k / 2][n][k % 2].y : x[k / 2][n][k % 2].x) = -INFINITY;
                            }
                        }
                    // Values that are not finite make NaN of the groups of the rows that see them, and of no others: a
                    // weight of zero would make NaN of them too. What no row sees is none at all.
                    uint32_t pairs[kGroups];
                    load_words(pairs, value_params + lane * (kGroups * 4));
                    bool finite = true;
#pragma unroll
                    for (uint32_t g = 0; g < kGroups; ++g) {
                        if (!(real >> lane & 1u)) pairs[g] = 0;
                        finite = finite && usable_params<BF16>(pairs[g]);
                    }
                    if (!__all_sync(0xffffffffu, finite)) {
#pragma unroll
                        for (uint32_t g = 0; g < kGroups; ++g) {
#pragma unroll
                            for (uint32_t k = 0; k < 4; ++k) {
                                const uint32_t its = 8 * k + own_token;
                                const uint32_t pair = reinterpret_cast<const uint32_t*>(value_params)[its * kGroups + g];
                                if ((real >> its & 1u) && !usable_params<BF16>(pair))
#pragma unroll
                                    for (uint32_t n = 0; n < NT; ++n) {
                                        if (x[k / 2][n][k % 2].x != -INFINITY) lows[g][n].x = __uint_as_float(0x7fffffffu);
                                        if (x[k / 2][n][k % 2].y != -INFINITY) lows[g][n].y = __uint_as_float(0x7fffffffu);
                                    }
                            }
                            if (!usable_params<BF16>(pairs[g])) pairs[g] = 0;
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (uint32_t g = 0; g < kGroups; ++g) reinterpret_cast<uint32_t*>(value_params)[lane * kGroups + g] = pairs[g];
                    fence_proxy_async_shared();  // what is copied there next comes by another way than these stores
                    __syncwarp();
                    look();
                }
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n) {
                    float keep[2], m[2] = {largest[n].x, largest[n].y};
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) {
                        m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 4));
                        m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 8));
                        m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 16));
                        // While a row has seen nothing its scores are -inf: so are its exponentials, with nothing taken off.
                        float& minus = e ? minus_peak[n].y : minus_peak[n].x;
                        float& over = e ? ceiling[n].y : ceiling[n].x;
                        const float its_log2 = e ? to_log2[n].y : to_log2[n].x;
                        const float power = m[e] * its_log2, was = over == -INFINITY ? -INFINITY : -minus;
                        keep[e] = 1.0f;
                        if (power > was) {
                            keep[e] = ex2_approx(was - power);
                            minus = -power;
                            over = m[e] + __fdividef(kSlack, its_log2);
                        }
                    }
                    const float2 keep2 = make_float2(keep[0], keep[1]);
                    sum[n] = __fmul2_rn(sum[n], keep2);
#pragma unroll
                    for (uint32_t g = 0; g < kGroups; ++g) lows[g][n] = __fmul2_rn(lows[g][n], keep2);
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
#pragma unroll
                        for (uint32_t j = 0; j < kTiles; ++j) out[j][n][i] *= keep[i % 2];
                    }
                }
                // ---- scales outside their group's window: it is moved if they are many, and what still lies outside is
                // multiplied here, in fp32, by the weights as they are (so that a scale has no say in rows that do not see its token), and
                // counts as zero below.
                uint32_t pairs[kGroups];
                load_words(pairs, value_params + lane * (kGroups * 4));
                bool any_far = false;
#pragma unroll
                for (uint32_t g = 0; g < kGroups; ++g) {
                    constexpr uint32_t kGroupTiles = G / 16;
                    const float size = fabsf(E::low(pairs[g]));
                    const bool counts = size > 0.0f && usable_params<BF16>(pairs[g]);  // (Others that a row sees make NaN of it.)
                    const auto lie_far = [&]() {
                        const float fitted = size * fit[g];
                        return __ballot_sync(0xffffffffu, counts && !(fitted >= kLeast && fitted < kMost));
                    };
                    uint32_t far = lie_far();
                    if (far == 0) continue;
                    const int32_t was = __float_as_int(fit[g]) >> 23;
                    if (was == 0 || __popc(far) >= kManyFar || __any_sync(0xffffffffu, counts && size * fit[g] >= 0x1p87f)) {
                        const uint32_t exponent = counts ? max(__float_as_uint(size) >> 23, 1u) : 0u;
                        const uint32_t together = __reduce_add_sync(0xffffffffu, exponent), all = __popc(__ballot_sync(0xffffffffu, counts));
                        const int32_t middle = max(static_cast<int32_t>((2 * together + all) / (2 * all)),
                                                   static_cast<int32_t>(__reduce_max_sync(0xffffffffu, exponent)) - kFarthest);
                        int32_t power = min(kFitBiased - middle, kMostFit);
                        if (was) {
                            float most = 0.0f;  // of the sums so far, which a window further down would raise: to 2^100 at most
#pragma unroll
                            for (uint32_t j = g * kGroupTiles; j < (g + 1) * kGroupTiles; ++j)
#pragma unroll
                                for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                                    for (uint32_t i = 0; i < 4; ++i) most = fmaxf(most, fabsf(out[j][n][i]));
                            const int32_t room = 227 - static_cast<int32_t>(__reduce_max_sync(0xffffffffu, __float_as_uint(most)) >> 23);
                            power = min(power, was + max(room, 0));
                            const float factor = power_of_two(min(max(127 + power - was, 0), 254));
#pragma unroll
                            for (uint32_t j = g * kGroupTiles; j < (g + 1) * kGroupTiles; ++j)
#pragma unroll
                                for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                                    for (uint32_t i = 0; i < 4; ++i) out[j][n][i] *= factor;
                        }
                        fit[g] = power_of_two(power);
                        far = lie_far();
                    }
#pragma unroll 1
                    for (uint32_t left = far; left; left &= left - 1) {
                        const uint32_t its = __ffs(left) - 1, pair = __shfl_sync(0xffffffffu, pairs[g], its);
                        const uint32_t holder = (its & 7u) ^ ((its & 7u) >> 2);  // its scores lie in lanes (holder, c4)
                        const float low = fmaf(8.0f, E::low(pair), E::high(pair)), fitted = E::low(pair) * fit[g];
                        uint32_t words[kValueWords];
                        load_words(words, values + its * (D / 2) + l4 * (D / 16));
#pragma unroll
                        for (uint32_t n = 0; n < NT; ++n) {
                            const float2 first = its & 8u ? x[0][n][1] : x[0][n][0], last = its & 8u ? x[1][n][1] : x[1][n][0];
                            const float2 power = __ffma2_rn(its & 16u ? last : first, to_log2[n], minus_peak[n]);
                            const float2 p = make_float2(__shfl_sync(0xffffffffu, ex2_approx(power.x), 4 * holder + c4),
                                                         __shfl_sync(0xffffffffu, ex2_approx(power.y), 4 * holder + c4));
                            if (l4 == holder) lows[g][n] = __ffma2_rn(p, make_float2(low, low), lows[g][n]);
                            const float2 weight = __fmul2_rn(p, make_float2(fitted, fitted));
#pragma unroll
                            for (uint32_t j = g * kGroupTiles; j < (g + 1) * kGroupTiles; ++j) {
                                const uint32_t byte = words[j / 4] >> (8 * (j % 4));
                                const float even = static_cast<float>(static_cast<int32_t>(byte & 15u) - 8);
                                const float odd = 16.0f * static_cast<float>(static_cast<int32_t>(byte >> 4 & 15u) - 8);
                                out[j][n][0] = fmaf(even, weight.x, out[j][n][0]);
                                out[j][n][1] = fmaf(even, weight.y, out[j][n][1]);
                                out[j][n][2] = fmaf(odd, weight.x, out[j][n][2]);
                                out[j][n][3] = fmaf(odd, weight.y, out[j][n][3]);
                            }
                        }
                    }
                    if (far >> lane & 1u) reinterpret_cast<uint32_t*>(value_params)[lane * kGroups + g] = 0;
                    any_far |= far != 0;
                }
                if (any_far) {
                    fence_proxy_async_shared();
                    __syncwarp();
                }
            }

#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                // ---- weights, their sums, and weight * scale in fp16, turned to be the values' second operand.
                uint32_t weights[kGroups][NT][2];
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half) {
                    float2 p[NT];
                    uint32_t pairs[kGroups];
                    load_words(pairs, value_params + (16 * h + 8 * half + own_token) * (kGroups * 4));
#pragma unroll
                    for (uint32_t n = 0; n < NT; ++n) {
                        const float2 power = __ffma2_rn(x[h][n][half], to_log2[n], minus_peak[n]);
                        p[n] = make_float2(ex2_approx(power.x), ex2_approx(power.y));
                        sum[n] = __fadd2_rn(sum[n], p[n]);
                    }
#pragma unroll
                    for (uint32_t g = 0; g < kGroups; ++g) {
                        const float scale = E::low(pairs[g]), fitted = scale * fit[g], low = fmaf(8.0f, scale, E::high(pairs[g]));
#pragma unroll
                        for (uint32_t n = 0; n < NT; ++n) {
                            lows[g][n].x = fmaf(p[n].x, low, lows[g][n].x);
                            lows[g][n].y = fmaf(p[n].y, low, lows[g][n].y);
                            weights[g][n][half] = transpose_8x8(Element<false>::pack(p[n].x * fitted, p[n].y * fitted));
                        }
                    }
                }
                // ---- O^T += V^T . (P scale)^T. Two tokens' nibbles of a channel side by side are a pair of the first
                // operand; the odd fragment rows' channels come 16 times too large. Codes are made normal numbers that count
                // from their middle, 8, with 8 * weight in fp32 in `lows`: a token of nearly all the weight and a value near the
                // middle adds nothing to what the product truncates. (A product with a constant 8, to be taken off at the
                // end, saves the additions and up to 3 % of the time, but the truncations of its sum and of the codes' differ by up to 2^-13
                // of a scale, more than everything else there.)
                uint32_t thousands = 0x64006400u;
                asm("" : "+r"(thousands));  // two constants in one instruction: one of them in a register
                uint32_t v[4][kValueWords];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) load_words(v[i], values + (16 * h + 8 * (i / 2) + 2 * c4 + ((i ^ (c4 >> 1)) & 1u)) * (D / 2) + l4 * (D / 16));
#pragma unroll
                for (uint32_t w = 0; w < kValueWords; ++w)
#pragma unroll
                    for (uint32_t half = 0; half < 2; ++half) {
                        uint32_t lo = __byte_perm(v[0][w], v[1][w], half ? 0x7632 : 0x5410);
                        uint32_t hi = __byte_perm(v[2][w], v[3][w], half ? 0x7632 : 0x5410);
#pragma unroll
                        for (uint32_t byte = 0; byte < 2; ++byte) {
                            const uint32_t j = 4 * w + 2 * half + byte, g = 16 * j / G;
                            const uint32_t codes[4] = {
                                add_f16x2(and_or(lo, 0x000f000fu, thousands), 0xe408e408u),  // 1024 + code - 1032
                                add_f16x2(and_or(lo, 0x00f000f0u, thousands), 0xe480e480u),  // 1024 + 16 code - 1152
                                add_f16x2(and_or(hi, 0x000f000fu, thousands), 0xe408e408u),
                                add_f16x2(and_or(hi, 0x00f000f0u, thousands), 0xe480e480u)};
#pragma unroll
                            for (uint32_t n = 0; n < NT; ++n)
                                mma_16x8x16(out[j][n], codes[0], codes[1], codes[2], codes[3], weights[g][n][0], weights[g][n][1]);
                            lo >>= 8;
                            hi >>= 8;
                        }
                    }
            }
            __syncwarp();  // every lane is done with the stage
            if (unit + 1 == to) break;  // the last stage is given back when the merge is done with it
            if (lane == 0) mbar_arrive(full + 8);
            next_stage();
        }

        // ---- the warps' parts of the piece meet in shared memory
        uint8_t* const merge_memory = Shape::kMergeInRing ? ring + stage * stage_bytes : ring + kStages * stage_bytes;
        constexpr uint32_t merge_pitch = Shape::kMergeInRing ? Shape::kStageBytes : Shape::kScratchBytes;
        sync_computing(warps * 32);  // the stage is every warp's
        Cut piece{b, kv_head, first_row, from == 0 && to == units_of(cost) ? 0u : 1u, 0};
        uint32_t which = 0;
        if (piece.parts) {
            const uint32_t first_unit = at - offset + args.segment_cost;
            piece.owner = block_of(first_unit);
            piece.parts = block_of(first_unit + units_of(cost) - 1) - piece.owner + 1;
            which = piece.owner == blockIdx.x;
        }
        {
            float* const merged = reinterpret_cast<float*>(merge_memory + warp * merge_pitch);
            float* const stats = merged + kRows * kPitch;
            float unfit[kGroups];
#pragma unroll
            for (uint32_t g = 0; g < kGroups; ++g) unfit[g] = power_of_two(254 - (__float_as_int(fit[g]) >> 23));
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n)
#pragma unroll
                for (uint32_t e = 0; e < 2; ++e) {
                    float s = e ? sum[n].y : sum[n].x;
                    float low[kGroups];
#pragma unroll
                    for (uint32_t g = 0; g < kGroups; ++g) low[g] = e ? lows[g][n].y : lows[g][n].x;
#pragma unroll
                    for (uint32_t mask = 4; mask < 32; mask *= 2) {
                        s += __shfl_xor_sync(0xffffffffu, s, mask);
#pragma unroll
                        for (uint32_t g = 0; g < kGroups; ++g) low[g] += __shfl_xor_sync(0xffffffffu, low[g], mask);
                    }
                    const uint32_t row = 8 * n + 2 * c4 + e;
#pragma unroll
                    for (uint32_t j = 0; j < kTiles; ++j) {
                        const uint32_t g = 16 * j / G;
                        merged[row * kPitch + 16 * j + l4] = fmaf(out[j][n][e], unfit[g], low[g]);
                        merged[row * kPitch + 16 * j + 8 + l4] = fmaf(out[j][n][2 + e] * 0.0625f, unfit[g], low[g]);
                    }
                    if (l4 == 0) {
                        stats[2 * row] = (e ? ceiling[n].y : ceiling[n].x) == -INFINITY ? -INFINITY : -(e ? minus_peak[n].y : minus_peak[n].x);
                        stats[2 * row + 1] = s;
                    }
                }
        }
        more = next_piece();
        if (more) fetch_rows();
        sync_computing(warps * 32);
        // A part of a segment that is cut over blocks: the block its first unit lies in keeps it in its second place, the others in
        // their first. Parts are handed in together at the end.
        if (piece.parts && threadIdx.x == 0) cuts[which] = piece;
        put_together(merge_memory, merge_pitch, piece,
                     piece.parts ? args.partials + (2 * blockIdx.x + which) * static_cast<size_t>(kPartialFloats) : nullptr);
        // Copies to where the merged rows lay come by another way than these reads.
        fence_proxy_async_shared();
        sync_computing(warps * 32);
        if (lane == 0) mbar_arrive(smem_u32(barriers + 2 * stage + 1));
        next_stage();
    }

    // ---- the parts of segments that are cut over blocks: the block that comes last to one adds them up, always in the same
    // order, and leaves the counter at zero.
    sync_computing(warps * 32);
    if (threadIdx.x == 0) {
        complete[0] = complete[1] = 0;
        if (cuts[0].parts || cuts[1].parts) {
            uint32_t came[2] = {};
#pragma unroll
            for (uint32_t c = 0; c < 2; ++c)
                if (cuts[c].parts) came[c] = arrive(args.arrivals + cuts[c].owner);
#pragma unroll
            for (uint32_t c = 0; c < 2; ++c)
                if (cuts[c].parts && came[c] == cuts[c].parts - 1) {
                    args.arrivals[cuts[c].owner] = 0;
                    complete[c] = 1;
                }
        }
    }
    sync_computing(warps * 32);
    uint8_t* const memory = Shape::kMergeInRing ? ring : ring + kStages * stage_bytes;
    constexpr uint32_t kMergePitch = Shape::kMergeInRing ? Shape::kStageBytes : Shape::kScratchBytes;
    for (uint32_t c = 0; c < 2; ++c) {
        if (!complete[c]) continue;
        const Cut piece = cuts[c];
        const uint32_t rows_here = min(kRows, args.rows - piece.first_row);
        constexpr uint32_t kFew = 4;
        if (piece.parts <= kFew) {  // one thread for four channels, all parts on their way at once
            for (uint32_t i = threadIdx.x; i < rows_here * (D / 4); i += warps * 32) {
                const uint32_t row = i / (D / 4), d = i % (D / 4) * 4;
                float4 z[kFew];
                float2 stat[kFew], all = make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (uint32_t p = 0; p < kFew; ++p) {
                    const float* const its = args.partials + (2 * (piece.owner + min(p, piece.parts - 1)) + (p == 0)) *
                                                                 static_cast<size_t>(kPartialFloats);
                    stat[p] = __ldcg(reinterpret_cast<const float2*>(its + kMostRows * 128 + 2 * row));
                    z[p] = __ldcg(reinterpret_cast<const float4*>(its + row * D + d));
                    if (p >= piece.parts) stat[p] = make_float2(-INFINITY, 0.0f);
                    all.x = fmaxf(all.x, stat[p].x);
                }
                const float minus = all.x == -INFINITY ? 0.0f : -all.x;
                float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (uint32_t p = 0; p < kFew; ++p) {
                    if (p >= piece.parts) continue;
                    const float factor = ex2_approx(stat[p].x + minus);
                    y = make_float4(fmaf(z[p].x, factor, y.x), fmaf(z[p].y, factor, y.y), fmaf(z[p].z, factor, y.z),
                                    fmaf(z[p].w, factor, y.w));
                    all.y = fmaf(stat[p].y, factor, all.y);
                }
                finish_row<D, BF16>(args, piece, row, d, y, all);
            }
            continue;
        }
        // Warp w puts parts w, w + warps, ... together; a lane's loads of a part, eight rows' at most, are all on their way at once.
        float* const merged = reinterpret_cast<float*>(memory + warp * kMergePitch);
        constexpr uint32_t kItems = 8 * D / 128;
#pragma unroll 1
        for (uint32_t first = 0; first < rows_here; first += 8) {
            float4 y[kItems] = {};
            float2 all[kItems];
#pragma unroll
            for (uint32_t k = 0; k < kItems; ++k) all[k] = make_float2(-INFINITY, 0.0f);
#pragma unroll 1
            for (uint32_t p = warp; p < piece.parts; p += warps) {
                const float* const its = args.partials + (2 * (piece.owner + p) + (p == 0)) * static_cast<size_t>(kPartialFloats);
                float4 z[kItems];
                float2 stat[kItems];
#pragma unroll
                for (uint32_t k = 0; k < kItems; ++k) {
                    const uint32_t row = first + (lane + 32 * k) / (D / 4), d = (lane + 32 * k) % (D / 4) * 4;
                    stat[k] = make_float2(-INFINITY, 0.0f);
                    if (row < rows_here) {
                        stat[k] = __ldcg(reinterpret_cast<const float2*>(its + kMostRows * 128 + 2 * row));
                        z[k] = __ldcg(reinterpret_cast<const float4*>(its + row * D + d));
                    }
                }
#pragma unroll
                for (uint32_t k = 0; k < kItems; ++k) {
                    // A part without a visible token. (One whose scores are all NaN has no reference either, but a sum.)
                    if (stat[k].y == 0.0f) continue;
                    const float m = fmaxf(all[k].x, stat[k].x), keep = ex2_approx(all[k].x - m), factor = ex2_approx(stat[k].x - m);
                    y[k] = make_float4(fmaf(z[k].x, factor, y[k].x * keep), fmaf(z[k].y, factor, y[k].y * keep),
                                       fmaf(z[k].z, factor, y[k].z * keep), fmaf(z[k].w, factor, y[k].w * keep));
                    all[k] = make_float2(m, fmaf(stat[k].y, factor, all[k].y * keep));
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < kItems; ++k) {
                const uint32_t row = first + (lane + 32 * k) / (D / 4), d = (lane + 32 * k) % (D / 4) * 4;
                *reinterpret_cast<float4*>(merged + row * kPitch + d) = y[k];
                if (d == 0) *reinterpret_cast<float2*>(merged + kRows * kPitch + 2 * row) = all[k];
            }
        }
        sync_computing(warps * 32);
        put_together(memory, kMergePitch, piece, nullptr);
        sync_computing(warps * 32);
    }
    // After a wait that gave up, copies may still be on their way: give them a while before the block's memory goes.
    if (stop_flag)
        for (uint32_t k = 0; k < 2 * kStages; ++k)
            for (uint32_t i = 0; i < 100 && !mbar_try_wait(smem_u32(barriers + k / 2 * 2), k & 1); ++i) {
            }
}

}  // namespace cache
}  // namespace fk

// ------------------------------------------------------------------ C ABI

using namespace fk;

/// A launch that may be set up while the work before it on the stream still ends; its kernel waits for that work itself, first of
/// all. (Calls in a row, against plain launches: one sequence of 777 tokens 15.0 us from 16.5, 24 with a window of 4096 25.4
/// from 26.8, a write and a read of 8191 tokens 25.9 from 28.7.)
template <typename Arguments>
static cudaError_t launch(void (*kernel)(Arguments, uint32_t*), uint32_t blocks, uint32_t threads, uint32_t shared_bytes, void* stream,
                          const Arguments& args, uint32_t* device_status) {
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared_bytes;
    config.stream = static_cast<cudaStream_t>(stream);
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args, device_status);
}

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

/// A tensor [tokens, heads, dim] of rows of `dim` neighbouring elements; strides in elements.
struct Rows {
    uintptr_t base;
    int64_t token_stride, head_stride;
    uint64_t tokens, heads;
    int64_t dim;

    /// The elements from the first row's begin that the rows lie in: [least, most).
    __int128 least() const { return reach(std::min<int64_t>(token_stride, 0), std::min<int64_t>(head_stride, 0)); }
    __int128 most() const { return reach(std::max<int64_t>(token_stride, 0), std::max<int64_t>(head_stride, 0)) + dim; }
    __int128 reach(int64_t token, int64_t head) const {
        return static_cast<__int128>(token) * (tokens - 1) + static_cast<__int128>(head) * (heads - 1);
    }
    /// Whether two rows `offset` elements and some whole strides apart (but not a row and itself) share an element.
    bool meet(__int128 offset) const {
        const bool by_token = tokens >= heads;  // steps of the other are gone through one by one
        const __int128 a = by_token ? token_stride : head_stride, b = by_token ? head_stride : token_stride;
        const __int128 a_count = by_token ? tokens : heads, b_count = by_token ? heads : tokens;
        for (__int128 j = 1 - b_count; j < b_count; ++j) {
            const __int128 rest = offset + j * b;  // the row nearest to -rest, by whole strides a, and its neighbours
            const __int128 near = a ? -rest / a : 0;
            for (__int128 i : {near - 1, near, near + 1}) {
                if (i <= -a_count || i >= a_count || (offset == 0 && i == 0 && j == 0)) continue;
                const __int128 apart = rest + i * a;
                if (apart < dim && apart > -dim) return true;
            }
        }
        return false;
    }
    bool over_one_another() const {
        const uint64_t token = std::abs(token_stride), head = std::abs(head_stride);
        const unsigned __int128 token_span = static_cast<unsigned __int128>(token) * (tokens - 1) + dim;
        const unsigned __int128 head_span = static_cast<unsigned __int128>(head) * (heads - 1) + dim;
        if ((heads == 1 || head >= static_cast<uint64_t>(dim)) && (tokens == 1 || token >= head_span)) return false;
        if ((tokens == 1 || token >= static_cast<uint64_t>(dim)) && (heads == 1 || head >= token_span)) return false;
        return meet(0);
    }
    /// Whether a row of `other` shares an element with one of these, as far as equal strides or begins tell.
    bool over(const Rows& other) const {
        const __int128 offset = (static_cast<__int128>(other.base) - static_cast<__int128>(base)) / 2;
        if (offset + other.least() >= most() || least() >= offset + other.most()) return false;
        return offset == 0 || (token_stride == other.token_stride && head_stride == other.head_stride && meet(offset));
    }
};

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
    if (!write) {
        const int64_t dim = cache->head_dim;
        const Rows both[2] = {{reinterpret_cast<uintptr_t>(k), k_token_stride, k_head_stride, tokens, cache->kv_heads, dim},
                              {reinterpret_cast<uintptr_t>(v), v_token_stride, v_head_stride, tokens, cache->kv_heads, dim}};
        for (const Rows& rows : both)
            if (rows.over_one_another())
                return fk_fail(FK_ERR_SHAPE, "strides of %lld elements a token and %lld a head lay rows of %u over one another",
                               static_cast<long long>(rows.token_stride), static_cast<long long>(rows.head_stride), cache->head_dim);
        if (both[0].over(both[1])) return fk_fail(FK_ERR_INVALID, "keys and values read would lie over one another");
    } else {
        const uint64_t rows = static_cast<uint64_t>(cache->pages) * cache->page_size * cache->kv_heads;
        const uint64_t codes = rows * (cache->head_dim / 2), params = rows * (cache->head_dim / cache->group) * 4;
        const struct {
            const void* at;
            uint64_t bytes;
        } buffers[4] = {{cache->k_codes, codes}, {cache->v_codes, codes}, {cache->k_params, params}, {cache->v_params, params}};
        for (uint32_t i = 0; i < 4; ++i)
            for (uint32_t j = 0; j < i; ++j) {
                const uintptr_t x = reinterpret_cast<uintptr_t>(buffers[i].at), y = reinterpret_cast<uintptr_t>(buffers[j].at);
                if (x < y + buffers[j].bytes && y < x + buffers[i].bytes)
                    return fk_fail(FK_ERR_INVALID, "the cache's buffers lie over one another");
            }
    }
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
    args.rows = tokens * cache->kv_heads;
    args.capacity = static_cast<uint64_t>(cache->pages) * cache->page_size;
    args.page_size = cache->page_size;
    args.heads = cache::Divider(cache->kv_heads);
    args.page = cache::Divider(cache->page_size);
    args.clear_skipped = clear_skipped != 0;
    return for_cache(cache, [&](auto dim, auto group, auto bf16) {
        const auto move = [&](auto rows_a_thread) {
            const uint32_t rows_a_block = cache::kRowThreads / (dim / 8) * rows_a_thread;
            const uint32_t blocks = (args.rows + rows_a_block - 1) / rows_a_block;
            return write ? launch(cache::write_kernel<dim, group, rows_a_thread, bf16>, blocks, cache::kRowThreads, 0, stream,
                                      args, device_status)
                             : launch(cache::read_kernel<dim, group, rows_a_thread, bf16>, blocks, cache::kRowThreads, 0, stream,
                                      args, device_status);
        };
        // A few rows take one a thread, and so more threads.
        const uint32_t few = static_cast<uint32_t>(facts.sm_count) * 4 * (cache::kRowThreads / (dim / 8));
        FK_CUDA(args.rows <= few ? move(std::integral_constant<int, 1>{}) : move(std::integral_constant<int, 2>{}));
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

// Per resident block a counter and the parts of the two segments that its share may begin and end inside of.
extern "C" uint64_t fk_cache_attention_workspace_bytes(uint32_t sm_count) {
    const uint64_t blocks = static_cast<uint64_t>(sm_count) * cache::kMostBlocksPerSm;
    return (blocks * 4 + 127) / 128 * 128 + blocks * 2 * cache::kPartialFloats * 4;
}

template <int D, int G, int NT, bool BF16>
static int launch_attention(cache::AttentionArguments& args, const DeviceFacts& facts, void* stream, uint32_t* device_status) {
    using Shape = cache::AttentionShape<D, G, NT>;
    args.row_tiles = (args.rows + Shape::kRows - 1) / Shape::kRows;
    const uint64_t segments = static_cast<uint64_t>(args.batch) * args.kv_heads * args.row_tiles;
    // How many warps share a piece. One block an SM, of all the warps it holds, leaves the fewest parts to put together: for
    // segments fewer than the SMs, or than twice the SMs and long. Smaller blocks overlap one's beginnings and ends with others'
    // units: two an SM while each can take a whole segment, three beyond. How long segments are the host does not know, since the
    // lengths live on the device: the table's width stands for it, and a table much wider than its sequences gets the longer ones' plan. (128-wide heads, 8 rows, groups of 64: 256 segments of
    // 15000 tokens, before a lone block's registers were handed over, 135 us against 143 with two blocks; 296 of 2000 27.6 us with two,
    // 34.2 with three, 35.5 with one; 384 of 2000 39.6 with three, 42.0 with two; 1024 of 300 30.3 with three, 35.0 with two, 47.9 with one.)
    const uint64_t sms = static_cast<uint64_t>(facts.sm_count);
    const bool lengthy = static_cast<uint64_t>(args.table_pages) * args.page_size > 8192;
    const uint32_t share = segments <= sms || (lengthy && segments < 2 * sms) ? 1 : segments <= 2 * sms ? 2 : 3;
    // A bulk copy takes its warp some 150 cycles, whatever its size, so four warps copy for a block that is alone on its SM (131072
    // tokens of one sequence in pages of 16, 32, 64: 75, 53 and 48 us; with two 102, 66 and 49). Small blocks spare one (384
    // segments of 2000 tokens in pages of 16 and 32: 54 and 43 us; with two 56 and 49).
    args.copying = share == 1 ? Shape::kCopyingAlone : 1;
    const uint32_t warps = Shape::most_warps(share, args.copying);
    const uint32_t resident = static_cast<uint32_t>(facts.sm_count) * share;
    const uint64_t unit_tokens = warps * cache::kWarpTokens;
    args.unit = cache::Divider(static_cast<uint32_t>(unit_tokens));
    args.tiles = cache::Divider(args.row_tiles);
    args.segment_cost = share == 1 ? 2 : 1;
    const uint64_t most_units = segments * ((static_cast<uint64_t>(args.table_pages) * args.page_size + unit_tokens - 1) / unit_tokens + args.segment_cost);
    if (most_units >= (1ull << 31))
        return fk_fail(FK_ERR_SHAPE, "%u sequences of up to %llu tokens on %u heads are more than a launch counts", args.batch,
                       static_cast<unsigned long long>(args.table_pages) * args.page_size, args.kv_heads);
    const uint32_t grid = most_units < resident ? static_cast<uint32_t>(most_units) : resident;
    const auto kernel = share == 1 ? cache::attention_kernel<D, G, NT, BF16, true> : cache::attention_kernel<D, G, NT, BF16, false>;
    uint32_t limit = 0;
    const int admitted = fk_admit_shared_plan(reinterpret_cast<const void*>(kernel), Shape::shared_bytes(warps), &limit);
    if (admitted != FK_OK) return admitted;
    FK_CUDA(launch(kernel, grid, (warps + args.copying) * 32, Shape::shared_bytes(warps), stream, args, device_status));
    return FK_OK;
}

/// Whether a row of the queries (strides in elements of 2 bytes) lies in part in [begin, end).
static bool queries_meet(const void* q, const int64_t (&strides)[3], uint32_t batch, uint32_t queries, uint32_t heads, uint32_t dim,
                         uintptr_t begin, uintptr_t end) {
    const uint64_t counts[3] = {batch, queries, heads};
    const __int128 base = reinterpret_cast<uintptr_t>(q);
    __int128 least = base, most = base + 2 * dim;
    for (uint32_t i = 0; i < 3; ++i)
        (strides[i] < 0 ? least : most) += static_cast<__int128>(2 * (counts[i] - 1)) * strides[i];
    if (most <= begin || least >= end) return false;
    // Rows with gaps that the other may lie in: one by one, which calls hardly ever come to.
    for (uint32_t b = 0; b < batch; ++b)
        for (uint32_t t = 0; t < queries; ++t)
            for (uint32_t h = 0; h < heads; ++h) {
                const __int128 row = base + 2 * (static_cast<__int128>(strides[0]) * b + static_cast<__int128>(strides[1]) * t +
                                                 static_cast<__int128>(strides[2]) * h);
                if (row < end && row + 2 * dim > begin) return true;
            }
    return false;
}

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
    if (!std::isfinite(scale)) return fk_fail(FK_ERR_INVALID, "the score scale %f is not finite", scale);
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
    if (capacity >= 0x7ffff000ull)
        return fk_fail(FK_ERR_SHAPE, "%u pages of %u tokens are more than 2^31 - 1 tokens a sequence", columns,
                       cache->page_size);
    const uint64_t rows = static_cast<uint64_t>(queries) * (heads / cache->kv_heads);
    const unsigned __int128 all_rows = static_cast<unsigned __int128>(rows) * cache->kv_heads * batch;
    if (rows >= (1ull << 30) || all_rows >= (1ull << 32))
        return fk_fail(FK_ERR_SHAPE, "%u sequences of %u queries of %u heads are more rows than a launch counts", batch, queries, heads);
    const uint64_t asked = static_cast<uint64_t>(all_rows);
    const uintptr_t out_end = reinterpret_cast<uintptr_t>(out) + 2 * asked * cache->head_dim;
    const uintptr_t lse_begin = reinterpret_cast<uintptr_t>(lse), lse_end = lse_begin + 4 * asked;
    if (queries_meet(q, strides, batch, queries, heads, cache->head_dim, reinterpret_cast<uintptr_t>(out), out_end))
        return fk_fail(FK_ERR_INVALID, "the output may not lie over the queries");
    if (lse && lse_begin < out_end && reinterpret_cast<uintptr_t>(out) < lse_end)
        return fk_fail(FK_ERR_INVALID, "lse may not lie over the output");
    if (lse && queries_meet(q, strides, batch, queries, heads, cache->head_dim, lse_begin, lse_end))
        return fk_fail(FK_ERR_INVALID, "lse may not lie over the queries");
    DeviceFacts facts;
    const int known = device_facts(&facts);
    if (known != FK_OK) return known;
    if (workspace_bytes < fk_cache_attention_workspace_bytes(facts.sm_count))
        return fk_fail(FK_ERR_SHAPE, "a workspace of %llu bytes is under the %llu of this device",
                       static_cast<unsigned long long>(workspace_bytes),
                       static_cast<unsigned long long>(fk_cache_attention_workspace_bytes(facts.sm_count)));
    cache::AttentionArguments args;
    args.codes[0] = static_cast<const uint8_t*>(cache->k_codes);
    args.codes[1] = static_cast<const uint8_t*>(cache->v_codes);
    args.params[0] = static_cast<const uint8_t*>(cache->k_params);
    args.params[1] = static_cast<const uint8_t*>(cache->v_params);
    args.q = static_cast<const uint8_t*>(q);
    args.q_batch_stride = 2 * q_batch_stride;
    args.q_token_stride = 2 * q_token_stride;
    args.q_head_stride = 2 * q_head_stride;
    args.out = static_cast<uint16_t*>(out);
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
    args.rows = static_cast<uint32_t>(rows);
    args.scale = scale;
    args.window = static_cast<int32_t>(window < 0x7fffffffu ? window : 0x7fffffffu);
    args.sinks = static_cast<int32_t>(sinks < 0x7fffffffu ? sinks : 0x7fffffffu);
    args.page = cache::Divider(cache->page_size);
    args.ratio = cache::Divider(heads / cache->kv_heads);
    args.arrivals = static_cast<uint32_t*>(workspace);
    const uint64_t counters = (static_cast<uint64_t>(facts.sm_count) * cache::kMostBlocksPerSm * 4 + 127) / 128 * 128;
    args.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + counters);
    return for_cache(cache, [&](auto dim, auto group, auto bf16) {
        if (rows <= 8) return launch_attention<dim, group, 1, bf16>(args, facts, stream, device_status);
        return launch_attention<dim, group, 2, bf16>(args, facts, stream, device_status);
    });
}
