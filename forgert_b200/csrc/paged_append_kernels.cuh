// paged_append_kernels.cuh - decode/prefill prologue of the paged caches whose
// rows stand by themselves, 16-bit pages and 4 bits: q/k/v bias + RoPE (one or
// several position axes) + append through a slot map, in one launch; and the
// read-back of 4-bit slots as fp16.
//
// Mathematics, per token t (all in fp32, one rounding at each output):
//   x = x + bias;  for f < D/2 the pair (x[f], x[f + D/2]) of q and k turns to
//   (a*c - b*s, a*s + b*c) with c, s = tables[positions[axis(f)][t]][f].
// In 4 bits, per group of 64 dims of a row of K or V:
//   bias  = min x rounded down to fp16
//   scale = (max x - bias) / 15 rounded up to fp16
//   code  = round((x - bias) / scale), ties to even (0 where scale is 0)
// so every quotient lies in 0 .. 15 and a value is off by half a scale at most.
// A group with a NaN, an infinity or a minimum below fp16's range gets a NaN
// scale and bias and reads back as NaN.
//
// Layout: LPR = D / 16 lanes share a row, lane l holding the pairs f = 8l ..
// 8l + 7, so that rows move in 16-byte accesses and a lane's codes are two whole
// words.  No row depends on another: CTAs take rows of K, of V, and of q (kQRows
// heads of a token to a lane group, which looks the angles up once).
//
// Bound: bytes and the latency of two rounds of loads (rows, slot and position;
// then the angles).  4800 prompt tokens of 28 / 4 heads of 128 with biases, three
// axes and 16-bit K and V written too, cold: 16-bit pages 19.1 us, 5.3 TB/s, 4 bits
// 19.5.  It took 24.1 with the position looked up after the slot, rows through L1
// (22.2: position early; 21.6: rows past L1) and four heads a lane group (20.4 with
// two; 19.1 at nine CTAs per SM instead of eight, 24 at ten, where it spills; one
// head, 22.5).  A decode step's 64 tokens take 2.2 and 2.6 in a graph.
#pragma once
#include "fr_ptx.cuh"
#include "kv4_common.cuh"
#include <cstdint>

namespace fr {

constexpr int kPagedThreads = 128;
constexpr int kPagedCtas = 9;           // per SM: 56 registers
constexpr int kPagedAxes = 4;
constexpr int kQRows = 2;               // query rows that a lane group has under way

// Page and row of a slot inside the pool (in 32 bits where they do: a 64-bit
// division takes as long as coding a row).
struct SlotPlace {
    int page, row;
    __device__ __forceinline__ SlotPlace(long long slot, int page_size) {
        if (slot >> 32) {
            page = int(slot / page_size);
            row = int(slot - (long long)page * page_size);
        } else {
            page = (uint32_t)slot / (uint32_t)page_size;
            row = (uint32_t)slot - (uint32_t)page * page_size;
        }
    }
};

struct PagedAppendParams {
    const __half* in[3];                // q, k, v
    __half* out[3];                     // k's, v's: nullptr = not written
    long long stride[6];                // halves between tokens: q, k, v, then the outputs
    const __half* bias[3];
    const float* cos_tab;
    const float* sin_tab;
    const int* positions;               // [axes][T]
    const long long* slots;
    __half* pages[2];                   // 16-bit: K's, V's rows [slots][Hkv][D]
    Kv4View cache;                      // 4 bits
    long long pool;                     // slots
    int* err;
    int T, H, Hkv, table_rows;
    int by_eights;                      // every group of eight frequencies has one axis
    int kv_ctas;                        // of K; as many of V
    uint8_t axis[64];                   // axis of frequency f
};

// Sixteen values of a row: its pairs 8l .. 8l + 7 (first halves, second halves).
struct Row16 {
    float lo[8], hi[8];
};

__device__ __forceinline__ void unpack8(uint4 w, float (&x)[8]) {
    const uint32_t h[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// Sixteen bytes of a row, which is read once: past L1, which the angles and biases
// of the next tokens stay in.
__device__ __forceinline__ uint4 load_row(const __half* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]),
                      pack_half2(x[6], x[7]));
}

template <int D>
__device__ __forceinline__ void store_row16(__half* row, int f0, const Row16& r) {
    *reinterpret_cast<uint4*>(row + f0) = pack8(r.lo);
    *reinterpret_cast<uint4*>(row + f0 + D / 2) = pack8(r.hi);
}

// Cosines and sines of token t at the lane's eight frequencies, in two steps: the
// position is on its way with the rows and the slot, ahead of knowing whether the
// token takes part.  A position outside the table is recorded and read as position
// 0.  By eights: each group of eight frequencies turns by one axis, so a lane looks
// up one position.
__device__ __forceinline__ int load_position(const PagedAppendParams& p, int t, int f0) {
    return p.positions[(size_t)p.axis[f0] * p.T + t];
}

template <int D>
__device__ __forceinline__ void load_angles(const PagedAppendParams& p, int t, int f0, int pos,
                                            float (&c)[8], float (&s)[8]) {
    constexpr int kHalf = D / 2;
    auto in_table = [&](int x) {
        if ((unsigned)x < (unsigned)p.table_rows) return x;
        record_error(p.err, kDevBadIndex);
        return 0;
    };
    if (p.by_eights) {
        const size_t e = (size_t)in_table(pos) * kHalf + f0;
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            const float4 cv = *reinterpret_cast<const float4*>(p.cos_tab + e + j);
            const float4 sv = *reinterpret_cast<const float4*>(p.sin_tab + e + j);
            c[j] = cv.x; c[j + 1] = cv.y; c[j + 2] = cv.z; c[j + 3] = cv.w;
            s[j] = sv.x; s[j + 1] = sv.y; s[j + 2] = sv.z; s[j + 3] = sv.w;
        }
        return;
    }
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
        const size_t e = (size_t)in_table(load_position(p, t, f0 + j)) * kHalf + f0 + j;
        const float cj = p.cos_tab[e], sj = p.sin_tab[e];
#pragma unroll
        for (int x = 0; x < 8; ++x)
            if (x == j) { c[x] = cj; s[x] = sj; }
    }
}

// The products are rounded before they are added, as separate operations
// would: which codes a row gets does not hang on contraction.
__device__ __forceinline__ void turn16(Row16& r, const float (&c)[8], const float (&s)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float a = r.lo[j], b = r.hi[j];
        r.lo[j] = __fsub_rn(__fmul_rn(a, c[j]), __fmul_rn(b, s[j]));
        r.hi[j] = __fadd_rn(__fmul_rn(a, s[j]), __fmul_rn(b, c[j]));
    }
}

template <int D>
__device__ __forceinline__ void add_bias16(Row16& r, const __half* bias, int f0) {
    Row16 b;
    unpack8(*reinterpret_cast<const uint4*>(bias + f0), b.lo);
    unpack8(*reinterpret_cast<const uint4*>(bias + f0 + D / 2), b.hi);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        r.lo[j] = __fadd_rn(r.lo[j], b.lo[j]);
        r.hi[j] = __fadd_rn(r.hi[j], b.hi[j]);
    }
}

// ---------------------------------------------------------------- 16-bit pages
struct HalfPages {
    template <int D>
    static __device__ __forceinline__ void put(const PagedAppendParams& p, int which, int h, long long slot,
                                               int f0, const Row16& r, bool real) {
        if (real) store_row16<D>(p.pages[which] + (slot * p.Hkv + h) * D, f0, r);
    }
};

// --------------------------------------------------------------------- 4 bits
struct Kv4Pair {
    float scale, bias, inverse;
    __half2 bits;
};

// Scale and bias of a group whose least and largest values are low and high.
__device__ __forceinline__ Kv4Pair kv4_pair(float low, float high) {
    Kv4Pair r;
    const __half b = __float2half_rd(__fadd_rn(low, 0.f));          // -0 is stored as 0
    r.bias = __half2float(b);
    const __half s = __float2half_ru(__fdiv_rn(__fsub_rn(high, r.bias), 15.f));
    r.scale = __half2float(s);
    r.bits = __halves2half2(s, b);
    // not finite: an exponent of all ones in either
    if (!(fabsf(r.bias) < INFINITY && r.scale < INFINITY)) {
        r.scale = 0.f;
        r.bits = __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff));
    }
    r.inverse = r.scale > 0.f ? __frcp_rn(r.scale) : 0.f;
    return r;
}

// Codes of eight values.  The quotient is rounded as the division itself would:
// q0 = x * (1 / scale), then one correction by the exact remainder (Markstein's
// theorem: correctly rounded when the reciprocal is).  y + 1.5 * 2^23 is rounded
// to a whole number, whose low bits are the code.  The codes of a group that is
// not finite are 0 (inverse 0; NaN and infinity times 0 are not whole numbers).
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], const Kv4Pair& g) {
    uint32_t n[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float d = __fsub_rn(x[j], g.bias);
        const float q0 = __fmul_rn(d, g.inverse);
        const float y = __fmaf_rn(__fmaf_rn(-q0, g.scale, d), g.inverse, q0);
        n[j] = __float_as_uint(__fadd_rn(y, 12582912.f));
    }
    uint32_t two[4];                            // low byte: two codes
#pragma unroll
    for (int j = 0; j < 4; ++j) two[j] = (n[2 * j] & 15u) | (n[2 * j + 1] << 4);
    const uint32_t w = __byte_perm(__byte_perm(two[0], two[1], 0x0040),
                                   __byte_perm(two[2], two[3], 0x0040), 0x5410);
    return g.inverse > 0.f ? w : 0u;
}

struct Kv4Pages {
    // Every lane of the row takes part, also where the row is not cached.
    template <int D>
    static __device__ __forceinline__ void put(const PagedAppendParams& p, int which, int h, long long slot,
                                               int f0, const Row16& r, bool real) {
        constexpr int NG = D / kKv4Group, LPR = D / 16;
        float low[2], high[2];                  // of the first halves, of the second
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const float (&v)[8] = x ? r.hi : r.lo;
            low[x] = high[x] = v[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) {
                low[x] = min_nan(low[x], v[j]);
                high[x] = max_nan(high[x], v[j]);
            }
        }
        if (NG == 1) {
            low[0] = min_nan(low[0], low[1]);
            high[0] = max_nan(high[0], high[1]);
        }
        Kv4Pair g[NG];
#pragma unroll
        for (int x = 0; x < NG; ++x) {
#pragma unroll
            for (int o = 1; o < LPR; o <<= 1) {
                low[x] = min_nan(low[x], __shfl_xor_sync(0xffffffffu, low[x], o));
                high[x] = max_nan(high[x], __shfl_xor_sync(0xffffffffu, high[x], o));
            }
            g[x] = kv4_pair(low[x], high[x]);
        }
        if (!real) return;
        const Kv4View& c = p.cache;
        const SlotPlace at(slot, c.page_size);
        uint8_t* dst = (which ? c.v : c.k) + c.row(at.page, h, at.row) + f0 / 2;
        *reinterpret_cast<uint32_t*>(dst) = kv4_codes(r.lo, g[0]);
        *reinterpret_cast<uint32_t*>(dst + D / 4) = kv4_codes(r.hi, g[NG - 1]);
        __half2* pairs = c.pairs<D>(at.page, h, at.row) + which * NG;
        if (f0 == 0) {
#pragma unroll
            for (int x = 0; x < NG; ++x) pairs[x] = g[x].bits;
        }
    }
};

// CTAs 0 .. kv_ctas - 1: rows of K (a lane group per token and kv head); as
// many: of V; the others: kQRows query heads of a token per lane group.
template <int D, class Pages>
__global__ void __launch_bounds__(kPagedThreads, kPagedCtas)
paged_append_kernel(const __grid_constant__ PagedAppendParams p) {
    constexpr int LPR = D / 16;
    constexpr int ROWS = kPagedThreads / LPR;
    const int f0 = (threadIdx.x % LPR) * 8;
    grid_launch_dependents();
    grid_dependency_wait();
    if (blockIdx.x < 2 * p.kv_ctas) {
        const int which = blockIdx.x >= p.kv_ctas;
        const int i = (blockIdx.x - which * p.kv_ctas) * ROWS + threadIdx.x / LPR;
        const bool there = i < p.T * p.Hkv;
        const int t = there ? i / p.Hkv : 0, h = i - t * p.Hkv;
        long long slot = -1;
        int pos = 0;
        uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (there) {
            const __half* src = p.in[1 + which] + t * p.stride[1 + which] + (size_t)h * D + f0;
            raw[0] = load_row(src);
            raw[1] = load_row(src + D / 2);
            slot = p.slots[t];
            if (!which) pos = load_position(p, t, f0);
        }
        const bool held = slot >= 0 && slot < p.pool;
        Row16 r;
        unpack8(raw[0], r.lo);
        unpack8(raw[1], r.hi);
        if (slot >= 0) {
            if (!held && h == 0 && f0 == 0) record_error(p.err, kDevBadIndex);
            if (p.bias[1 + which]) add_bias16<D>(r, p.bias[1 + which] + (size_t)h * D, f0);
            if (!which) {
                float c[8], s[8];
                load_angles<D>(p, t, f0, pos, c, s);
                turn16(r, c, s);
            }
            if (p.out[1 + which])
                store_row16<D>(p.out[1 + which] + t * p.stride[4 + which] + (size_t)h * D, f0, r);
        }
        Pages::template put<D>(p, which, h, slot, f0, r, held);
        return;
    }
    const int chunks = (p.H + kQRows - 1) / kQRows;
    const long long i = (long long)(blockIdx.x - 2 * p.kv_ctas) * ROWS + threadIdx.x / LPR;
    if (i >= (long long)p.T * chunks) return;
    const int t = int(i / chunks);
    const int h0 = int(i - (long long)t * chunks) * kQRows;
    const __half* src = p.in[0] + t * p.stride[0] + (size_t)h0 * D + f0;
    // The rows are on their way before the slot tells whether the token takes part.
    uint4 raw[kQRows][2];
#pragma unroll
    for (int j = 0; j < kQRows; ++j)
        if (h0 + j < p.H) {
            raw[j][0] = load_row(src + j * D);
            raw[j][1] = load_row(src + j * D + D / 2);
        }
    const long long slot = p.slots[t];
    const int pos = load_position(p, t, f0);
    if (slot < 0) return;
    float c[8], s[8];
    load_angles<D>(p, t, f0, pos, c, s);
    __half* dst = p.out[0] + t * p.stride[3] + (size_t)h0 * D;
#pragma unroll
    for (int j = 0; j < kQRows; ++j)
        if (h0 + j < p.H) {
            Row16 r;
            unpack8(raw[j][0], r.lo);
            unpack8(raw[j][1], r.hi);
            if (p.bias[0]) add_bias16<D>(r, p.bias[0] + (size_t)(h0 + j) * D, f0);
            turn16(r, c, s);
            store_row16<D>(dst + j * D, f0, r);
        }
}

// ---------------------------------------------------------------------------
// Read-back: out[i] = code * scale + bias of slot slots[i], every kv head, rounded
// to fp16 once (65504 at most); a slot outside the pool gives zeros.  D / 16 lanes
// share a row of K and V; lane l widens dims 8l .. 8l + 7 of each half row, so that
// every access of neighbouring lanes is contiguous.
//
// A byte copied to both halves of a word, masked and put under 0x6400, is the fp16
// pair 1024 + n, 1024 + 16 n'; one fused product makes n, n' of it, exactly, and a
// second the value: code * scale is exact, so the sum is rounded once.  (Codes
// through integer conversions and fp32, 16 a lane in two 16-byte pieces: 57 thousand
// rows of 4 x 128, 150 MB, took 33.0 us instead of 26.1, 5.7 TB/s.)
// ---------------------------------------------------------------------------
struct Kv4GatherParams {
    Kv4View cache;
    const long long* slots;
    __half* k_out;
    __half* v_out;
    uint32_t rows;                      // slots x Hkv
};

__device__ __forceinline__ uint4 kv4_widen8(uint32_t w, uint32_t pair) {
    const uint32_t scale = __byte_perm(pair, pair, 0x1010), bias = __byte_perm(pair, pair, 0x3232);
    const __half2 one = __halves2half2(__ushort_as_half(0x3c00), __ushort_as_half(0x2c00));     // 1, 1/16
    const __half2 off = __halves2half2(__ushort_as_half(0xe400), __ushort_as_half(0xd400));     // -1024, -64
    const __half2 top = __float2half2_rn(kKv4Top);
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t both = (__byte_perm(w, w, i * 0x1111) & 0x00f0000fu) | 0x64006400u;
        const __half2 n = __hfma2(*reinterpret_cast<const __half2*>(&both), one, off);
        const __half2 x = __hmin2_nan(__hfma2(n, *reinterpret_cast<const __half2*>(&scale),
                                              *reinterpret_cast<const __half2*>(&bias)), top);
        r[i] = *reinterpret_cast<const uint32_t*>(&x);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

template <int D>
__global__ void __launch_bounds__(256)
kv4_gather_kernel(const Kv4GatherParams p) {
    constexpr int LPR = D / 16;                 // lanes per row
    constexpr int NG = D / kKv4Group;
    grid_launch_dependents();
    grid_dependency_wait();
    const uint32_t row = blockIdx.x * (256u / LPR) + threadIdx.x / LPR;
    if (row >= p.rows) return;
    const Kv4View& c = p.cache;
    const int l = threadIdx.x % LPR;
    const uint32_t i = row / (uint32_t)c.Hkv;
    const int h = row - i * c.Hkv;
    const long long slot = p.slots[i];
    uint32_t w[2][2] = {}, pair[2 * NG] = {};   // K's, V's two words; K's groups, V's groups
    if (slot >= 0 && slot < (long long)c.num_pages * c.page_size) {
        const SlotPlace at(slot, c.page_size);
        const size_t off = c.row(at.page, h, at.row) + 4 * l;
        const __half2* pairs = c.pairs<D>(at.page, h, at.row);
        if constexpr (NG == 2) {
            const uint4 x = *reinterpret_cast<const uint4*>(pairs);
            pair[0] = x.x; pair[1] = x.y; pair[2] = x.z; pair[3] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(pairs);
            pair[0] = x.x; pair[1] = x.y;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (p.k_out) w[0][e] = *reinterpret_cast<const uint32_t*>(c.k + off + e * (D / 4));
            if (p.v_out) w[1][e] = *reinterpret_cast<const uint32_t*>(c.v + off + e * (D / 4));
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const size_t to = (size_t)row * D + e * (D / 2) + 8 * l;
        const int x = NG == 2 ? e : 0;
        if (p.k_out) *reinterpret_cast<uint4*>(p.k_out + to) = kv4_widen8(w[0][e], pair[x]);
        if (p.v_out) *reinterpret_cast<uint4*>(p.v_out + to) = kv4_widen8(w[1][e], pair[NG + x]);
    }
}

}  // namespace fr
