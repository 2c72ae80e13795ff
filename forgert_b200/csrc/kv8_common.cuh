// kv8_common.cuh - the 8-bit paged KV cache: layout, codes and their scales.
//
// A cached value is code * scale.  Codes are int8 (-127 .. 127) or e4m3
// (largest 448), one byte each; a scale (fp32) belongs to one block of 16
// consecutive rows of a page, one kv head, and K or V:
//   codes   [num_pages][Hkv][page_size][D], any page / head / row strides
//   scales  [num_pages][Hkv][page_size / 16][2]   (K, V)
// Sixteen rows are one m-tile of the decode kernel's products, so a warp
// applies a scale to a whole fragment at once, and re-coding a block whose
// scale has grown touches at most 16 rows of one head.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>

namespace fr {

constexpr int kKv8Block = 16;                   // rows that share a scale

struct Kv8View {
    uint8_t* k;
    uint8_t* v;
    float* scales;
    int num_pages, page_size, Hkv;
    long long page_stride, head_stride, row_stride;   // bytes

    __device__ __forceinline__ size_t row(int page, int head, int r) const {
        return (size_t)page * page_stride + (size_t)head * head_stride + (size_t)r * row_stride;
    }
    // (K, V) scales of the block that holds row r
    __device__ __forceinline__ float2* scale(int page, int head, int r) const {
        return reinterpret_cast<float2*>(scales) +
               ((size_t)page * Hkv + head) * (page_size / kKv8Block) + r / kKv8Block;
    }
};

// Code types.  half2_lo / half2_hi widen the low / high two bytes of a word
// to fp16 exactly (both types' values are fp16 numbers); encode4 rounds four
// values, already divided by their scale, to the nearest codes, ties to even.
struct Int8Code {
    static constexpr float kMax = 127.f;
    static constexpr bool kHasNan = false;
    // With the sign bit flipped a code is u = code + 128 in 0..255, and the
    // fp16 with bits 0x6400 | u is 1024 + u: subtracting 1152 is exact.
    static __device__ __forceinline__ uint32_t prepare(uint32_t w) { return w ^ 0x80808080u; }
    static __device__ __forceinline__ uint32_t widen(uint32_t bits) {
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&bits), bias);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint32_t half2_lo(uint32_t w) {
        return widen(__byte_perm(w, 0x64646464u, 0x4140));
    }
    static __device__ __forceinline__ uint32_t half2_hi(uint32_t w) {
        return widen(__byte_perm(w, 0x64646464u, 0x4342));
    }
    static __device__ __forceinline__ float decode(uint32_t byte) {
        return float(int8_t(byte & 0xff));
    }
    // x + 1.5 * 2^23 is rounded to an integer (ties to even), whose low byte is
    // the code; |x| <= 127.  A block whose scale is not finite has codes 0: the
    // scale carries it.
    static __device__ __forceinline__ uint32_t encode4(const float (&x)[4], bool finite) {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__fadd_rn(x[i], 12582912.f));
        const uint32_t lo = __byte_perm(b[0], b[1], 0x0040), hi = __byte_perm(b[2], b[3], 0x0040);
        return finite ? __byte_perm(lo, hi, 0x5410) : 0u;
    }
};

struct E4m3Code {
    static constexpr float kMax = 448.f;
    static constexpr bool kHasNan = true;       // codes 0x7f and 0xff
    static __device__ __forceinline__ uint32_t prepare(uint32_t w) { return w; }
    static __device__ __forceinline__ uint32_t widen16(uint16_t x) {
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(x));
        return h;
    }
    static __device__ __forceinline__ uint32_t half2_lo(uint32_t w) {
        return widen16(uint16_t(w & 0xffffu));
    }
    static __device__ __forceinline__ uint32_t half2_hi(uint32_t w) {
        return widen16(uint16_t(w >> 16));
    }
    static __device__ __forceinline__ float decode(uint32_t byte) {
        const uint32_t h = widen16(uint16_t(byte & 0xffu));
        return __half2float(__ushort_as_half(uint16_t(h & 0xffffu)));
    }
    static __device__ __forceinline__ uint32_t encode2(float lo, float hi) {
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ uint32_t encode4(const float (&x)[4], bool) {
        return encode2(x[0], x[1]) | (encode2(x[2], x[3]) << 16);
    }
};

}  // namespace fr
