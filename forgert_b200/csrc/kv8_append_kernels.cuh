// kv8_append_kernels.cuh - decode/prefill prologue of the 8-bit paged cache:
// q/k/v bias + RoPE (one or several position axes) + quantised append through
// a slot map, in one launch; and the read-back of slots as fp16.
//
// Mathematics, per token t (all in fp32, one rounding at each output):
//   x = x + bias;  for f < D/2 the pair (x[f], x[f + D/2]) of q and k turns to
//   (a*c - b*s, a*s + b*c) with c, s = tables[positions[axis(f)][t]][f].
// Append: consecutive tokens in consecutive rows of one block of 16 (a "run")
// are coded together,
//   scale = amax / kMax, at least the block's old scale if the run does not
//   start the block;  code = round(x / scale), ties to even.
// If that makes the scale grow, the block's earlier rows are coded anew:
// code' = round(code * old / scale).  All runs of a block are the work of the
// CTA of its first token, in token order (more than one where a token between
// them is left out), so the scale, the old rows and the new ones need no order
// between CTAs.  The maximum is taken over the bit patterns of |x|, where NaN
// is the largest: a block that holds a NaN or an infinity gets such a scale and
// reads back as NaN.
//
// Layout: LPR = D / 8 lanes share a row, lane l holding the pairs f = 4l ..
// 4l + 3: 8-byte loads of both halves, 4-byte code stores, a 16-byte load each
// of cosines and sines.  The four warps of a CTA share a run's 16 rows, which
// stay in registers (two rows' eighths a lane) from the load to the codes.
// (One warp per run, 64 values a lane: 128 registers and straight-line code
// that the instruction cache lost, 60 us for 4800 tokens of 28 / 4 heads.)
//
// Bound: for prompts issue slots (67 % of the cycles) and the loads' latency at
// 27 warps per SM - 4800 tokens of 28 / 4 heads of 128, three axes, biases and
// 16-bit K and V written too, 24 us, 4.0 TB/s; for a decode step latency, four
// dependent rounds of loads (64 tokens 4.5 us in a graph).
#pragma once
#include "fr_ptx.cuh"
#include "decode_kernels.cuh"
#include "kv8_common.cuh"
#include <cstdint>

namespace fr {

constexpr int kAppendThreads = 128;
constexpr int kMaxAxes = 4;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kQHeads = 4;              // query rows that a lane has under way

struct AppendParams {
    const __half* q;
    const __half* k;
    const __half* v;
    __half* q_out;
    __half* k_out;                      // nullptr: not written
    __half* v_out;
    long long stride[6];                // halves between tokens: q, k, v, q_out, k_out, v_out
    const __half* bias[3];
    const float* cos_tab;
    const float* sin_tab;
    const int* positions;               // [axes][T]
    const long long* slots;
    Kv8View cache;
    int* err;
    int T, H, table_rows;
    int window;                         // tokens that a K/V CTA looks through, at most 16
    int q_heads;                        // query heads of a token that one lane group turns
    int by_quads;                       // every group of four frequencies has one axis
    int kv_ctas;
    uint8_t axis[64];                   // axis of frequency f
};

// Eight values of a row: its pairs 4l .. 4l + 3 (first halves, second halves).
struct Row8 {
    float lo[4], hi[4];
};

__device__ __forceinline__ void unpack4(uint2 w, float (&x)[4]) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}

__device__ __forceinline__ uint2 pack4(const float (&x)[4]) {
    return make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
}

template <int D>
__device__ __forceinline__ Row8 load_row(const __half* row, int f0) {
    Row8 r;
    unpack4(*reinterpret_cast<const uint2*>(row + f0), r.lo);
    unpack4(*reinterpret_cast<const uint2*>(row + f0 + D / 2), r.hi);
    return r;
}

template <int D>
__device__ __forceinline__ void store_row(__half* row, int f0, const Row8& r) {
    *reinterpret_cast<uint2*>(row + f0) = pack4(r.lo);
    *reinterpret_cast<uint2*>(row + f0 + D / 2) = pack4(r.hi);
}

// Cosines and sines of token t at the lane's four frequencies.  A position
// outside the table is recorded and read as position 0.  By quads: each group
// of four frequencies turns by one axis, so a lane looks up one position.
template <int D>
__device__ __forceinline__ void load_turn(const AppendParams& p, int t, int f0, float (&c)[4],
                                          float (&s)[4]) {
    constexpr int kHalf = D / 2;
    auto at = [&](int axis) {
        int pos = p.positions[(size_t)axis * p.T + t];
        if ((unsigned)pos >= (unsigned)p.table_rows) {
            record_error(p.err, kDevBadIndex);
            pos = 0;
        }
        return pos;
    };
    if (p.by_quads) {
        const size_t e = (size_t)at(p.axis[f0]) * kHalf + f0;
        const float4 cv = *reinterpret_cast<const float4*>(p.cos_tab + e);
        const float4 sv = *reinterpret_cast<const float4*>(p.sin_tab + e);
        c[0] = cv.x; c[1] = cv.y; c[2] = cv.z; c[3] = cv.w;
        s[0] = sv.x; s[1] = sv.y; s[2] = sv.z; s[3] = sv.w;
        return;
    }
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
        const size_t e = (size_t)at(p.axis[f0 + j]) * kHalf + f0 + j;
        const float cj = p.cos_tab[e], sj = p.sin_tab[e];
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (x == j) { c[x] = cj; s[x] = sj; }
    }
}

// The products are rounded before they are added, as separate operations
// would: which codes a block gets does not hang on contraction.
__device__ __forceinline__ void turn(Row8& r, const float (&c)[4], const float (&s)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = r.lo[j], b = r.hi[j];
        r.lo[j] = __fsub_rn(__fmul_rn(a, c[j]), __fmul_rn(b, s[j]));
        r.hi[j] = __fadd_rn(__fmul_rn(a, s[j]), __fmul_rn(b, c[j]));
    }
}

__device__ __forceinline__ void add_bias(Row8& r, const Row8& b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        r.lo[j] = __fadd_rn(r.lo[j], b.lo[j]);
        r.hi[j] = __fadd_rn(r.hi[j], b.hi[j]);
    }
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

constexpr float kMinScale = 0x1p-100f;  // of a block that is not zeros

// A block's scale with what dividing by it takes.  Quotients are rounded as
// the division itself would: q0 = x / scale by the rounded reciprocal, then
// one correction by the exact remainder (Markstein's theorem: correctly
// rounded when the reciprocal is).  Scale 0 (a block of zeros) gives 0; with a
// scale that is not finite the remainder is NaN and q0 = x * 0 or NaN stands.
struct Divisor {
    float scale, inverse;
    bool finite;
    __device__ __forceinline__ explicit Divisor(float s) {
        scale = s;
        inverse = s == 0.f ? 0.f : __frcp_rn(s);
        finite = abs_bits(s) < 0x7f800000u;
    }
    __device__ __forceinline__ float quotient(float x) const {
        const float q0 = __fmul_rn(x, inverse);
        const float q = __fmaf_rn(__fmaf_rn(-q0, scale, x), inverse, q0);
        return copysignf(finite ? q : q0, x);       // a zero keeps its sign
    }
};

template <class Code>
__device__ __forceinline__ uint32_t code4(const float (&x)[4], const Divisor& d) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = d.quotient(x[j]);
    return Code::encode4(y, d.finite);
}

// K's (which 0) or V's row of token t, with its bias and turned.
template <int D>
__device__ __forceinline__ Row8 finish_row(const AppendParams& p, int which, int t, int f0,
                                           const uint2 (&raw)[2], const uint2 (&bias)[2], bool biased) {
    Row8 r;
    unpack4(raw[0], r.lo);
    unpack4(raw[1], r.hi);
    if (biased) {
        Row8 b;
        unpack4(bias[0], b.lo);
        unpack4(bias[1], b.hi);
        add_bias(r, b);
    }
    if (!which) {
        float c[4], s[4];
        load_turn<D>(p, t, f0, c, s);
        turn(r, c, s);
    }
    return r;
}

// One run: rows t .. t + n - 1 (n <= 16) of K or V head h go to rows row0 ..
// of the block at `slot`.  The whole CTA takes part; tops: one word per warp.
template <int D, class Code>
__device__ __forceinline__ void append_run(const AppendParams& p, int which, int h, int t, int n,
                                           long long slot, const uint2 (&bias)[2], bool biased,
                                           uint32_t* tops) {
    constexpr int LPR = D / 8;
    constexpr int RPW = 32 / LPR;               // rows per warp and pass
    constexpr int PASSES = kKv8Block / (RPW * kAppendWarps);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = warp * RPW + lane / LPR, f0 = (lane % LPR) * 4;
    constexpr int STEP = RPW * kAppendWarps;
    const Kv8View& c = p.cache;
    const int page = int(slot / c.page_size), r0 = int(slot - (long long)page * c.page_size);
    const int first = r0 % kKv8Block;           // rows of the block that are held already
    const __half* x = (which ? p.v : p.k) + (size_t)h * D + f0;
    __half* y = which ? p.v_out : p.k_out;
    const long long xs = p.stride[1 + which], ys = p.stride[4 + which];
    uint8_t* pool = which ? c.v : c.k;
    float* scale_at = reinterpret_cast<float*>(c.scale(page, h, r0)) + which;

    uint2 raw[PASSES][2];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int j = i * STEP + sub;
        if (j < n) {
            const __half* src = x + (t + j) * xs;
            raw[i][0] = *reinterpret_cast<const uint2*>(src);
            raw[i][1] = *reinterpret_cast<const uint2*>(src + D / 2);
        }
    }
    const float old = first ? *scale_at : 0.f;
    Row8 rows[PASSES];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int j = i * STEP + sub;
        if (j < n) {
            Row8& r = rows[i];
            r = finish_row<D>(p, which, t + j, f0, raw[i], bias, biased);
            if (y) store_row<D>(y + (t + j) * ys + (size_t)h * D, f0, r);
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(abs_bits(r.lo[e]), abs_bits(r.hi[e])));
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();                            // every warp has read the old scale, too
#pragma unroll
    for (int w = 0; w < kAppendWarps; ++w) top = max(top, tops[w]);
    float scale = __fdiv_rn(__uint_as_float(top), Code::kMax);
    if (first) scale = __uint_as_float(max(abs_bits(scale), abs_bits(old)));
    // A smaller one's reciprocal and remainders would leave fp32's range.
    if (abs_bits(scale) - 1u < abs_bits(kMinScale) - 1u) scale = kMinScale;
    const Divisor d(scale);
    if (first && abs_bits(scale) > abs_bits(old)) {
#pragma unroll 1
        for (int j = sub; j < first; j += STEP) {
            uint8_t* dst = pool + c.row(page, h, r0 - first + j);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t* w = reinterpret_cast<uint32_t*>(dst + f0 + e * (D / 2));
                const uint32_t codes = *w;
                float z[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) z[b] = __fmul_rn(Code::decode(codes >> (8 * b)), old);
                *w = code4<Code>(z, d);
            }
        }
    }
    uint8_t* dst = pool + c.row(page, h, r0) + f0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int j = i * STEP + sub;
        if (j < n) {
            uint8_t* at = dst + j * c.row_stride;
            *reinterpret_cast<uint32_t*>(at) = code4<Code>(rows[i].lo, d);
            *reinterpret_cast<uint32_t*>(at + D / 2) = code4<Code>(rows[i].hi, d);
        }
    }
    if (threadIdx.x == 0) *scale_at = scale;
    __syncthreads();                            // the next run may be of this block; tops are reused
}

// CTAs 0 .. kv_ctas - 1: (p.window tokens, K or V, kv head), doing the blocks
// that one of these tokens is the first of; the CTAs after them: query rows, a
// lane group per (token, p.q_heads heads).  (Spreading the first among the
// others measured the same or slower.)
template <int D, class Code>
__global__ void __launch_bounds__(kAppendThreads, 8)
kv8_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int LPR = D / 8;
    constexpr int RPW = 32 / LPR;
    __shared__ uint32_t tops[kAppendWarps];
    const int lane = threadIdx.x & 31;
    const int Hkv = p.cache.Hkv;
    const int f0 = (lane % LPR) * 4;
    grid_launch_dependents();
    grid_dependency_wait();
    if (blockIdx.x < p.kv_ctas) {
        const int h = blockIdx.x % Hkv;
        const int which = (blockIdx.x / Hkv) & 1;
        const int t0 = blockIdx.x / (2 * Hkv) * p.window;
        const long long pool = (long long)p.cache.num_pages * p.cache.page_size;
        // The window's rows are on their way to L2 while the slots are read.
        {
            const int tr = t0 + threadIdx.x / (D / 64);             // 128 bytes each
            if (threadIdx.x < p.window * (D / 64) && tr < p.T)
                prefetch_l2((which ? p.v : p.k) + tr * p.stride[1 + which] + (size_t)h * D +
                            threadIdx.x % (D / 64) * 64);
        }
        const __half* b = p.bias[1 + which];
        uint2 bias[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
        if (b) {
            bias[0] = *reinterpret_cast<const uint2*>(b + (size_t)h * D + f0);
            bias[1] = *reinterpret_cast<const uint2*>(b + (size_t)h * D + f0 + D / 2);
        }
        // Lane l holds the slot of token t - 15 + l: the tokens that can share
        // a block with t (lane 31: the last token that can follow t + 15); -1 for
        // a token that is left out, kOutside for a slot past the pool.
        constexpr long long kOutside = -2;
        auto slots_about = [&](int t) {
            const int tl = t - 15 + lane;
            const long long s = tl >= 0 && tl < p.T ? p.slots[tl] : -1;
            if (s >= pool) record_error(p.err, kDevBadIndex);
            return s < 0 ? -1 : s < pool ? s : kOutside;
        };
        const long long near = slots_about(t0);
        const bool mine = lane >= 15 && lane < 15 + p.window;
        // Tokens with a slot past the pool are not cached, but their rows are
        // wanted as the others' are.
        __half* y = which ? p.v_out : p.k_out;
        uint32_t outside = y ? __ballot_sync(0xffffffffu, mine && near == kOutside) : 0u;
#pragma unroll 1
        for (int c = (threadIdx.x >> 5) * RPW + lane / LPR; outside; --c, outside &= outside - 1) {
            if (c % (RPW * kAppendWarps) != 0) continue;            // a lane group per token
            const int t = t0 + __ffs(outside) - 16;
            const __half* src = (which ? p.v : p.k) + t * p.stride[1 + which] + (size_t)h * D + f0;
            const uint2 raw[2] = {*reinterpret_cast<const uint2*>(src),
                                  *reinterpret_cast<const uint2*>(src + D / 2)};
            store_row<D>(y + t * p.stride[4 + which] + (size_t)h * D, f0,
                         finish_row<D>(p, which, t, f0, raw, bias, b != nullptr));
        }
        // The window's tokens (lanes 15 ..) that no earlier token shares a block with
        const uint32_t mates = __match_any_sync(0xffffffffu, near >= 0 ? near / kKv8Block : -1LL);
        uint32_t firsts = __ballot_sync(0xffffffffu, mine && near >= 0 && __ffs(mates) - 1 == lane);
#pragma unroll 1
        while (firsts) {                                            // uniform over the CTA
            const int t = t0 + __ffs(firsts) - 16;
            firsts &= firsts - 1;
            const long long slot = t == t0 ? near : slots_about(t);
            const long long s = __shfl_sync(0xffffffffu, slot, 15);
            const bool same = lane >= 15 && lane < 31 && slot >= 0 && slot / kKv8Block == s / kKv8Block;
            const long long before = __shfl_up_sync(0xffffffffu, slot, 1);
            const uint32_t on = __ballot_sync(0xffffffffu, same && slot == before + 1) >> 15;
            uint32_t left = __ballot_sync(0xffffffffu, same) >> 15; // bit j: token t + j
#pragma unroll 1
            while (left) {
                const int i = __ffs(left) - 1;
                const int n = __ffs(~(on >> (i + 1)));              // 1 + the tokens that go on
                left &= ~(((1u << n) - 1u) << i);
                const long long si = __shfl_sync(0xffffffffu, slot, 15 + i);
                append_run<D, Code>(p, which, h, t + i, n, si, bias, b != nullptr, tops);
            }
        }
        return;
    }
    const int chunks = (p.H + p.q_heads - 1) / p.q_heads;
    const long long item = ((long long)(blockIdx.x - p.kv_ctas) * kAppendWarps + (threadIdx.x >> 5)) * RPW + lane / LPR;
    if (item >= (long long)p.T * chunks) return;
    const int t = int(item / chunks);
    const int h_beg = int(item - (long long)t * chunks) * p.q_heads;
    const int h_end = min(h_beg + p.q_heads, p.H);
    const __half* src = p.q + t * p.stride[0] + f0;
    __half* dst = p.q_out + t * p.stride[3];
    // The first rows and the angles are on their way before the slot tells
    // whether the token takes part.
    const long long slot = p.slots[t];
    uint2 raw[kQHeads][2];
    auto load_heads = [&](int h0) {
#pragma unroll
        for (int j = 0; j < kQHeads; ++j)
            if (h0 + j < h_end) {
                raw[j][0] = *reinterpret_cast<const uint2*>(src + (h0 + j) * D);
                raw[j][1] = *reinterpret_cast<const uint2*>(src + (h0 + j) * D + D / 2);
            }
    };
    load_heads(h_beg);
    if (slot < 0) return;
    float c[4], s[4];
    load_turn<D>(p, t, f0, c, s);
#pragma unroll 1
    for (int h0 = h_beg; h0 < h_end; h0 += kQHeads) {
        if (h0 > h_beg) load_heads(h0);
#pragma unroll
        for (int j = 0; j < kQHeads; ++j)
            if (h0 + j < h_end) {
                Row8 r;
                unpack4(raw[j][0], r.lo);
                unpack4(raw[j][1], r.hi);
                if (p.bias[0]) add_bias(r, load_row<D>(p.bias[0] + (size_t)(h0 + j) * D, f0));
                turn(r, c, s);
                store_row<D>(dst + (size_t)(h0 + j) * D, f0, r);
            }
    }
}

// ---------------------------------------------------------------------------
// Read-back: out[i] = fp16(code * scale) of slot slots[i], every kv head; a
// slot outside the pool gives zeros.  One thread widens 16 codes (a 16-byte
// load) of K and of V; consecutive threads take consecutive pieces of the
// output row, so both sides move whole sectors.  Bound by bytes, two thirds of
// them written: 57 thousand rows of 4 x 128, 118 MB, take 23.4 us, 5.0 TB/s
// (8 codes per thread, two pieces under way, measured the same).
// ---------------------------------------------------------------------------
struct GatherParams {
    Kv8View cache;
    const long long* slots;
    __half* k_out;
    __half* v_out;
    long long pieces;                   // slots x Hkv x D / 16
};

template <class Code>
__device__ __forceinline__ void widen16(uint4 w, float scale, __half* out) {
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = Code::prepare(in[i]);
        const uint32_t pair[2] = {Code::half2_lo(x), Code::half2_hi(x)};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair[e]));
            h[2 * i + e] = pack_half2(f.x * scale, f.y * scale);
        }
    }
    uint4* o = reinterpret_cast<uint4*>(out);
    o[0] = make_uint4(h[0], h[1], h[2], h[3]);
    o[1] = make_uint4(h[4], h[5], h[6], h[7]);
}

template <int D, class Code>
__global__ void __launch_bounds__(256)
kv8_gather_kernel(const GatherParams p) {
    constexpr int PPR = D / 16;                 // pieces per row
    grid_launch_dependents();
    grid_dependency_wait();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.pieces) return;
    const Kv8View& c = p.cache;
    const int e = int(i % PPR) * 16;
    const long long row = i / PPR;
    const int h = int(row % c.Hkv);
    const long long slot = p.slots[row / c.Hkv];
    const bool real = slot >= 0 && slot < (long long)c.num_pages * c.page_size;
    const int page = real ? int(slot / c.page_size) : 0;
    const int r = real ? int(slot - (long long)page * c.page_size) : 0;
    float2 scale = make_float2(0.f, 0.f);
    uint4 kw = make_uint4(0, 0, 0, 0), vw = kw;
    if (real) {
        const size_t at = c.row(page, h, r) + e;
        if (p.k_out) kw = *reinterpret_cast<const uint4*>(c.k + at);
        if (p.v_out) vw = *reinterpret_cast<const uint4*>(c.v + at);
        scale = *c.scale(page, h, r);
    }
    if (p.k_out) widen16<Code>(kw, scale.x, p.k_out + row * D + e);
    if (p.v_out) widen16<Code>(vw, scale.y, p.v_out + row * D + e);
}

}  // namespace fr
