// kv4_common.cuh - the 4-bit paged KV cache: layout, and codes to values.
//
// A row (one token, one kv head) of K or V is coded in groups of 64 dims, each
// with a scale and a bias in fp16; a cached value is code * scale + bias with
// codes 0 .. 15, two to a byte (dim 2i in the low half of byte i):
//   codes   [num_pages][Hkv][page_size][D / 2] bytes, any page / head / row strides
//   scales  [num_pages][Hkv][page_size][2 (K, V)][D / 64][2 (scale, bias)] fp16
// A row stands by itself: writing one changes no other's codes or scales, and
// at D = 128 it takes 64 bytes of K, 64 of V and 16 of scales (4.5 bits a value).
#pragma once
#include <cuda_fp16.h>
#include <cstdint>

namespace fr {

constexpr int kKv4Group = 64;                   // dims that share a scale and a bias
// The largest fp16.  A scale is rounded up, so 15 of them above a bias may stand for
// more than a group's maximum, and for more than this: cut where a value or an
// average of values becomes fp16.  (Nothing lies below -65504: no bias does.)
constexpr float kKv4Top = 65504.f;

struct Kv4View {
    uint8_t* k;
    uint8_t* v;
    __half* scales;
    int num_pages, page_size, Hkv;
    long long page_stride, head_stride, row_stride;   // bytes
    // The same in numbers of 16 bytes, which fit 32 bits: a page, a block of 16
    // rows; a page's scales, a head's part of them.
    uint32_t page16, block16, scales16, head_scales16;

    __device__ __forceinline__ size_t row(int page, int head, int r) const {
        return (size_t)page * page_stride + (size_t)head * head_stride + (size_t)r * row_stride;
    }
    // The row's scales and biases: K's groups, then V's.
    template <int D>
    __device__ __forceinline__ __half2* pairs(int page, int head, int r) const {
        return reinterpret_cast<__half2*>(scales) +
               (((size_t)page * Hkv + head) * page_size + r) * (2 * (D / kKv4Group));
    }
};

}  // namespace fr
