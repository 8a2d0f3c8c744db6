// Device helpers of the 8-bit paged cache: where a block lies, and how e4m3 codes and their scales are made and read.
#pragma once
#include "hstu_fwd_kernel.hip.h"
#include "hstu_paged_fp8.h"

namespace hstu {

// The pages of one sequence, and how many of its rows are live.  Clamped, so that malformed offsets, lengths or page ids never
// become addresses outside the tensors.
struct Fp8Sequence {
    int64_t first;  // of its pages, in page_ids
    int n_pages;
    int len;        // live rows, at most what the pages hold
};

__device__ __forceinline__ Fp8Sequence fp8_pages(const void* offsets, int n_ids, int idx64, int b)
{
    Fp8Sequence s;
    int64_t p0 = load_index_uniform(offsets, b, idx64), p1 = load_index_uniform(offsets, b + 1, idx64);
    p0 = p0 < 0 ? 0 : (p0 > n_ids ? n_ids : p0);
    p1 = p1 < p0 ? p0 : (p1 > n_ids ? n_ids : p1);
    s.first = p0;
    s.n_pages = static_cast<int>(p1 - p0);
    s.len = 0;
    return s;
}

__device__ __forceinline__ int fp8_room(const Fp8Cache& c, int n_pages)
{
    const int64_t room = static_cast<int64_t>(n_pages) * c.blocks_per_page * kFp8Block;
    return static_cast<int>(room < kFp8MostKeys ? room : kFp8MostKeys);
}

__device__ __forceinline__ Fp8Sequence fp8_sequence(const Fp8Cache& c, int b)
{
    Fp8Sequence s = fp8_pages(c.page_offsets, c.n_page_ids, c.idx64, b);
    const int64_t len = load_index_uniform(c.cache_len, b, c.idx64);
    const int room = fp8_room(c, s.n_pages);
    s.len = static_cast<int>(len < 0 ? 0 : (len > room ? room : len));
    return s;
}

// Number of block `blk` of a sequence within the cache tensors, for key head g; -1 where the page id is none.
__device__ __forceinline__ int fp8_block(const Fp8Cache& c, const void* ids, int64_t first, int g, int blk)
{
    const int page = div_small(blk, c.blocks_per_page);
    const int64_t id = load_index(ids, first + page, c.idx64);
    const uint32_t at = (static_cast<uint32_t>(id) * static_cast<uint32_t>(c.n_heads) + static_cast<uint32_t>(g)) * static_cast<uint32_t>(c.blocks_per_page) +
                        static_cast<uint32_t>(blk - page * c.blocks_per_page);
    return static_cast<uint64_t>(id) < static_cast<uint64_t>(c.num_pages) ? static_cast<int>(at) : -1;
}

// This lane's number, worked out where it stands: for what follows a loop, which would else keep a register through it.
__device__ __forceinline__ int lane_here()
{
    uint32_t none = 0;
    asm volatile("" : "+s"(none));
    return static_cast<int>(__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none)));
}

// A value that is the same in all lanes, and what is worked out from it, likewise.
__device__ __forceinline__ int here(int x)
{
    asm volatile("" : "+s"(x));
    return x;
}

// A block's scale from the bits of the largest finite magnitude in it: the smallest power of two, from 2^-126 up, that brings it
// to at most 448 = 1.75 * 2^8; 1 for a block of zeros.  Returned as the exponent field of the scale.
__device__ __forceinline__ uint32_t fp8_scale_field(uint32_t top)
{
    if (top == 0) {
        return 127u;
    }
    const int e = static_cast<int>(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return static_cast<uint32_t>(e < 1 ? 1 : e);
}
__device__ __forceinline__ float fp8_scale_of(uint32_t field) { return __builtin_bit_cast(float, field << 23); }
// 1 / scale, exactly: fields 1 .. 247 have the reciprocals 253 .. 7
__device__ __forceinline__ float fp8_inverse_of(uint32_t field) { return __builtin_bit_cast(float, (254u - field) << 23); }

// Four codes over the largest scale, 2^120: 256 of it is no float any more (a value that is finite rounds to it from 248 on), so 256 becomes 240.
constexpr uint32_t kFp8TopField = 247;
__device__ __forceinline__ uint32_t fp8_below_infinity(uint32_t codes)
{
    const uint32_t other = (codes & 0x7f7f7f7fu) ^ 0x78787878u;  // of a code of +-256: zero
    return codes - ((0x80808080u - other & 0x80808080u) >> 7);
}

// bits of the magnitude of a finite value, 0 of any other
__device__ __forceinline__ uint32_t finite_bits(float x)
{
    const uint32_t m = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
    return m < 0x7f800000u ? m : 0u;
}

// the codes of two values over their scale, in the low or high half of `old`: at most 448 in magnitude or not finite; what is not
// finite becomes NaN (e4m3 has no infinity, and the instruction makes NaN of one)
template <bool HI>
__device__ __forceinline__ uint32_t fp8_codes2(float a, float b, float inverse, uint32_t old)
{
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(a * inverse, b * inverse, static_cast<int>(old), HI));
}

typedef __attribute__((ext_vector_type(2))) short s16x2_t;

// the same of a word of two 16-bit values, in one instruction
template <typename Tag, bool HI>
__device__ __forceinline__ uint32_t fp8_codes2(uint32_t word, float scale, uint32_t old)
{
    const s16x2_t was = __builtin_bit_cast(s16x2_t, old);
    if constexpr (__is_same(Tag, bf16_tag)) {
        typedef __attribute__((ext_vector_type(2))) __bf16 two_t;
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(was, __builtin_bit_cast(two_t, word), scale, HI));
    } else {
        typedef __attribute__((ext_vector_type(2))) _Float16 two_t;
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(was, __builtin_bit_cast(two_t, word), scale, HI));
    }
}

// The largest finite magnitude among 16-bit values, two at a time: magnitudes moved up by as much as makes those that are not finite negative.
template <typename Tag>
struct FiniteTop {
    static constexpr short kUp = __is_same(Tag, bf16_tag) ? 0x80 : 0x400;
    s16x2_t top = {0, 0};
    __device__ __forceinline__ void take(uint32_t word)
    {
        top = __builtin_elementwise_max(top, __builtin_bit_cast(s16x2_t, word & 0x7fff7fffu) + s16x2_t{kUp, kUp});
    }
    __device__ __forceinline__ uint32_t bits() const  // as a float's
    {
        const int a = top[0], b = top[1], most = a > b ? a : b;
        return __builtin_bit_cast(uint32_t, lo_to_float<Tag>(static_cast<uint32_t>(most > kUp ? most - kUp : 0)));
    }
};

typedef __attribute__((ext_vector_type(2))) float f32x2_t;
// two codes of a word (the low or the high ones) as floats
template <bool HI>
__device__ __forceinline__ f32x2_t fp8_values2(uint32_t codes)
{
    return __builtin_bit_cast(f32x2_t, __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes), HI));
}

// the largest of `top` over a workgroup of WAVES wavefronts; `s` has a word per wavefront
template <int WAVES>
__device__ __forceinline__ uint32_t block_top(uint32_t top, uint32_t (&s)[WAVES])
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t other = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, 64));
        top = other > top ? other : top;
    }
    if ((threadIdx.x & 63) == 0) {
        s[threadIdx.x >> 6] = top;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        top = s[w] > top ? s[w] : top;
    }
    return top;
}

}  // namespace hstu
