// kv4_decode_kernels.cuh - single-token attention over the 4-bit paged cache.
//
// Mathematics, per (sequence, query head h of kv head j), positions t < len,
// groups g of 64 dims with codes n, K's (a, b) and V's (a', b') as scale, bias:
//   s_t = sum_g a_tg (q_g . n_tg) + b_tg (q_g . 1),  in units of 1 / sqrt(D)
//   p_t = 2^(s_t log2 e - r),  l = sum_t p_t,  mid_tg = b'_tg + 7.5 a'_tg
//   o_g = sum_t (p_t a'_tg) (n'_tg - 7.5) + sum_t p_t mid_tg,  out = o / l
// (zeros for an empty sequence).  Codes enter the products as they are: the
// fp16 with bits n is n 2^-24 exactly, so a mask makes two operands of a word,
// n of the low halves and 16 n of the high ones, and the factors are taken off
// the sums.  15 times the sum of a step's weights comes from a product with a
// constant operand (z), and half of it is taken off o, which so stays small and its
// sums lose little.  Scores, l, o and all other sums are fp32.
//
// A weight p a' enters the product with V as two fp16, itself rounded and what the
// rounding takes off, on a reference of its own group's, 2^8 up, so that one as
// small as 2^-22 of the largest keeps its bits.  (One fp16 alone: 64 sequences of
// 8192 to 32768 tokens in 147 us instead of 171, but the outputs off by 3.0e-4 of
// their 2-norm instead of 2.1e-4, which is what their rounding takes.)  l and the
// middles are on the first group's reference, in fp32 from unrounded p.  What is
// left beside the outputs' rounding are the fp32 sums of the products: 0.3e-4 on
// those sequences, 0.9e-4 over 131072 positions, where the outputs are small beside
// their terms (o centred at every block: 0.65e-4, and 3 % more time).
//
// Bytes: D of codes per position and kv head, D / 8 of scales; 4 * D * G
// operations on them.  Measured in graphs of 20 calls, 28 / 4 heads of 128: 64
// sequences of 8192 to 32768 tokens (1.2 million tokens, 697 MB) 171 us, 4.1 TB/s,
// 0.62 of a copy's rate; of 1024 to 8192 51 us; one sequence of 512 tokens 7.2 (14 /
// 2 heads of 64).  The copies alone take 106 of the 171 and 32 of the 51 us.  No
// pipe is full (issue slots 57 %, integer 43 %, tensor 36 %, fp32 23 %, DRAM 0.55 of
// a copy's rate at 64 x 12288): what bounds it is the latency of a block's chain
// (codes, scores, weights, transposed weights, products) at three warps a scheduler,
// more of which the state leaves no registers for.  At D = 128 a block of 16
// positions and one kv head takes a warp 335 instructions, 127 of them on the
// integer pipe, which takes one in two cycles (80 masks and shifts of codes, 5 for 8
// codes), and 28 products of 8 cycles each; 43 are a half of a step's overhead.  The
// order of the phases changes little (scores of two blocks at once, V loaded early
// or late: within 1 %, with weights in one fp16).
//
// Fragments (mma m16n8k16): of K a lane holds 16 dims of each group in rows 2g and
// 2g + 1 of the block, as they lie in memory; contraction order is free, so q is
// permuted to the order that masks bring K's codes in (Kv4Query).  V comes
// transposed by bytes (ldmatrix m16n16 .trans .b8): four rows' bytes of one pair
// of dims in a word, so that the same masks make (row, row + 2) operands of it.
#pragma once
#include "cached_decode_kernels.cuh"
#include "kv4_common.cuh"
#include <type_traits>

namespace fr {

constexpr float kKv4Shift = 8.f;        // a weight at its reference counts 2^8 ...
constexpr float kKv4Most = 0x1p15f;     // ... and the weights of a lane's rows may sum up to 2^15 before that moves
constexpr float kKv4Least = -24.f;      // a smaller scale's reference is this scale's: p stays below 2^39
constexpr float kKv4Far = 0x1p23f;      // from here on scores are whole numbers
constexpr uint32_t kLowHalves = 0x000f000fu, kHighHalves = 0x00f000f0u;

// A block (16 rows) in shared memory: lines of 128 bytes, of 2 rows (D = 128) or 4,
// as in the cache (copies that scatter a line's 32-byte sectors over lines took
// 170 us where these take 155).  Within a line K's 32-byte half rows and V's
// 16-byte chunks are exchanged by line, so that the loads of K (8 bytes of rows r,
// r + 2, r + 4, r + 6 at a time) and V (16 bytes of 8 rows) hit distinct banks.
template <int D> constexpr int kv4_block_bytes() { return 16 * (D / 2); }
// 16-byte chunk c of row r.
template <int D>
__device__ __forceinline__ uint32_t kv4_k_offset(int r, int c) {
    return D == 128 ? r / 2 * 128 + ((r % 2 * 2 + c / 2) ^ (r / 2 % 4)) * 32 + c % 2 * 16
                    : r / 4 * 128 + (r % 4 ^ (r / 4 % 2)) * 32 + c * 16;
}
template <int D>
__device__ __forceinline__ uint32_t kv4_v_offset(int r, int c) {
    return D == 128 ? r / 2 * 128 + r % 2 * 64 + (c ^ (r / 2 % 4)) * 16
                    : r / 4 * 128 + r % 4 * 32 + (c ^ (r / 4 % 2)) * 16;
}

template <int D, int NT, int MT, int STAGES, int NW>
struct Kv4Smem {
    static constexpr int kStepBytes = MT * kv4_block_bytes<D>();        // K (or V) of one step
    static constexpr int kWarpBytes = 2 * STAGES * kStepBytes;          // a warp's ring
    static constexpr size_t kRingBytes = size_t(NW) * kWarpBytes;
    static constexpr int kXFloats = (D / 16) * 4 + 4;
    static constexpr size_t kXOffset = kRingBytes;
    static constexpr size_t kXBytes = size_t(2) * 32 * kXFloats * sizeof(float);
    static constexpr size_t kScaleOffset = kXOffset + kXBytes;
    static constexpr int kRowScales = 8 * (D / kKv4Group);              // bytes, K and V
    static constexpr int kStepScales = 16 * MT * kRowScales;
    static constexpr size_t kScaleBytes = size_t(NW) * STAGES * kStepScales;
    static constexpr size_t kFlagOffset = kScaleOffset + kScaleBytes;
    static constexpr size_t kMetaOffset = kFlagOffset + 16 * sizeof(int);
    static constexpr size_t kMetaBytes = (2 * kPersistMaxBatch + 1 + 16) * sizeof(int);
    static constexpr size_t kBytes = 1024 + kMetaOffset + kMetaBytes;   // the frame aligns to 1024
    static_assert(kStepBytes % 16 == 0 && kScaleOffset % 16 == 0, "alignment");
    // cached_merge reuses the exchange area: weights [threads] + 2 x heads
    static_assert(kXBytes >= (NW * 32 + 2 * NT * 8) * sizeof(float), "merge area");
};

// q of one item as the B operand, in the order in which masks bring K's codes:
// of each word of eight dims 0, 4 and 2, 6 (low halves), 1, 5 and 3, 7 (high
// ones).  Each head is first scaled by a power of two to 2^10 .. 2^11 at its
// largest element; the low halves' elements then take 16 times as much, so that
// both halves' products sum up in one accumulator without leaving fp16's range
// (what that takes off is below 2^-35 of the largest element).  For the heads
// 2t, 2t + 1: sum of each group's elements, in the same units as the products,
// and unit, which takes a score from these to base 2.
template <int D, int NT>
struct Kv4Query {
    static constexpr int NG = D / kKv4Group;
    uint32_t b[NG][2][2][NT][2];                // group, word, low / high, tile of heads
    float sum[NG][NT][2], unit[NT][2];

    __device__ __forceinline__ void load(const __half* q, int gcount, float sl2, int lane) {
        const int g = lane >> 2, t = lane & 3;
        constexpr uint32_t kOnes = 0x3c003c00u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int hj = nt * 8 + g;
            const __half* row = q + (size_t)hj * D + 16 * t;
            uint4 v[NG][2];
            __half2 top = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
#pragma unroll
            for (int x = 0; x < NG; ++x)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    v[x][w] = make_uint4(0, 0, 0, 0);
                    if (hj < gcount) v[x][w] = *reinterpret_cast<const uint4*>(row + x * kKv4Group + w * 8);
                    const uint32_t e[4] = {v[x][w].x, v[x][w].y, v[x][w].z, v[x][w].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __half2*>(&e[i])));
                }
            const float2 two = __half22float2(top);
            float big = fmaxf(two.x, two.y);
            if (!(two.x < INFINITY && two.y < INFINITY)) big = 1.f;     // stays NaN or infinite
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            // 2^up: big's exponent e (-24 .. 15) becomes 10
            const int up = big > 0.f ? 10 - (int(__float_as_uint(big) >> 23) - 127) : 0;
            const float f = __int_as_float((127 + up) << 23);
#pragma unroll
            for (int x = 0; x < NG; ++x)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    uint32_t e[4] = {v[x][w].x, v[x][w].y, v[x][w].z, v[x][w].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&e[i]));
                        e[i] = pack_half2(z.x * (f * 16.f), z.y * f);   // an even and an odd dim
                    }
                    b[x][w][0][nt][0] = __byte_perm(e[0], e[2], 0x5410);
                    b[x][w][0][nt][1] = __byte_perm(e[1], e[3], 0x5410);
                    b[x][w][1][nt][0] = __byte_perm(e[0], e[2], 0x7632);
                    b[x][w][1][nt][1] = __byte_perm(e[1], e[3], 0x7632);
                }
#pragma unroll
            for (int x = 0; x < NG; ++x) {
                float s[4], s16[4];
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    auto add = [&](float (&acc)[4], int e) {
                        if (w == 0) mma_16816_first(acc, kOnes, kOnes, kOnes, kOnes, b[x][w][e][nt][0], b[x][w][e][nt][1]);
                        else mma_16816(acc, kOnes, kOnes, kOnes, kOnes, b[x][w][e][nt][0], b[x][w][e][nt][1]);
                    };
                    add(s16, 0);
                    add(s, 1);
                }
                sum[x][nt][0] = fmaf(s[0], 16.f, s16[0]) * 0x1p-24f;
                sum[x][nt][1] = fmaf(s[1], 16.f, s16[1]) * 0x1p-24f;
            }
            // products: 2^-24 (codes) * 16 * 2^up
            const float back = sl2 * 0x1p20f * __int_as_float((127 - up) << 23);
            unit[nt][0] = __shfl_sync(0xffffffffu, back, 8 * t);
            unit[nt][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
        }
    }
};

// Running state of a warp over an item, per head column.  r is the reference of
// the first group's weights, in base 2 and a whole number (or a score, where these
// are far from 0), f[x] 2^(r - that of group x).  o: products with V's codes from 7.5 on, in units of 2^-24 (even dims)
// and 2^-28 (odd ones); mid: this lane's rows' part of sum p mid, l that of the row
// sum, both on r.
template <int D, int NT>
struct Kv4State {
    static constexpr int NG = D / kKv4Group;
    float o[D / 16][NT][4];
    float mid[NG][NT][2], l[NT][2];
    float r[NT][2], f[NG][NT][2];               // f[0] is 1
    float m[NT][2];
    bool fresh;                                 // nothing summed yet: no references

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int dm = 0; dm < D / 16; ++dm)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[dm][nt][c] = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int x = 0; x < NG; ++x) {
                    mid[x][nt][j] = 0.f;
                    f[x][nt][j] = 1.f;
                }
                r[nt][j] = l[nt][j] = 0.f;
            }
        }
        fresh = true;
    }
    // Takes 7.5 times the weights' sum off the products with the codes; z is 15
    // times that sum, in units of 2^-24.
    __device__ __forceinline__ void centre(const float (&z)[NG][NT][4]) {
#pragma unroll
        for (int x = 0; x < NG; ++x)
#pragma unroll
            for (int dm = 4 * x; dm < 4 * x + 4; ++dm)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        o[dm][nt][j] = fmaf(-0.5f, z[x][nt][j], o[dm][nt][j]);
                        o[dm][nt][j + 2] = fmaf(-8.f, z[x][nt][j], o[dm][nt][j + 2]);
                    }
    }
    // Sums over the warp's rows, o whole and on r: the (m, l, o) of the merges.
    __device__ __forceinline__ void finish() {
        auto rows = [](float x) {
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            return x + __shfl_xor_sync(0xffffffffu, x, 16);
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                l[nt][j] = rows(l[nt][j]);
                m[nt][j] = fresh ? -INFINITY : r[nt][j];
#pragma unroll
                for (int x = 0; x < NG; ++x) {
                    const float c = rows(mid[x][nt][j]);
                    const float u = x ? 0x1p24f / f[x][nt][j] : 0x1p24f;
#pragma unroll
                    for (int dm = 4 * x; dm < 4 * x + 4; ++dm) {
                        o[dm][nt][j] = fmaf(o[dm][nt][j], u, c);
                        o[dm][nt][j + 2] = fmaf(o[dm][nt][j + 2], 0.0625f * u, c);
                    }
                }
            }
    }
};

// Where a lane's parts of a block lie: K's groups of an even row and of the odd
// one after it, a 16-byte chunk of a row in each group of V, the two rows' scales.
template <int D>
struct Kv4Lane {
    static constexpr int NG = D / kKv4Group;
    uint32_t k[2][NG], v[NG], scales;

    __device__ __forceinline__ Kv4Lane(uint32_t kst, uint32_t vst, uint32_t sc, int lane) {
        const int r = (lane >> 2) * 2;
#pragma unroll
        for (int x = 0; x < NG; ++x) {
#pragma unroll
            for (int i = 0; i < 2; ++i) k[i][x] = kst + kv4_k_offset<D>(r + i, 2 * x) + lane % 4 * 8;
            v[x] = vst + kv4_v_offset<D>(lane % 16, 2 * x + lane / 16);
        }
        scales = sc + r * (8 * NG);
    }
};

// A block of 16 rows on its way through a warp: scores, weights, then the products
// with V.
template <int D, int NT>
struct Kv4Block {
    static constexpr int NG = D / kKv4Group;
    float s[NT][4];                             // scores, in base 2
    float va[2][NG], vm[2][NG];                 // V's scales and middles of the lane's rows
    uint32_t w[NG][NT][2], rest[NG][NT][2];     // weights, and what their rounding took off

    static __device__ __forceinline__ float2 wide(uint32_t h) {
        return __half22float2(*reinterpret_cast<const __half2*>(&h));
    }
    // A sum of weights that does not fit.  NaN counts: an infinite p at a scale of 0
    // gives one, and so does a NaN scale, beside which another group's weights may be
    // infinite.
    static __device__ __forceinline__ bool outgrown(float sum) { return !(sum <= kKv4Most); }

    // TAIL: only the first `valid` (>= 1) rows are positions.
    template <bool TAIL>
    __device__ __forceinline__ void score(const Kv4Lane<D>& at, int block, int valid,
                                          const Kv4Query<D, NT>& q, int lane) {
        uint32_t pair[2][2 * NG];               // of rows 2 g, 2 g + 1: K's groups, V's groups
        {
            const uint4 x = lds128(at.scales + block * (16 * 8 * NG));
            if constexpr (NG == 2) {
                const uint4 y = lds128(at.scales + block * (16 * 8 * NG) + 16);
                pair[0][0] = x.x; pair[0][1] = x.y; pair[0][2] = x.z; pair[0][3] = x.w;
                pair[1][0] = y.x; pair[1][1] = y.y; pair[1][2] = y.z; pair[1][3] = y.w;
            } else {
                pair[0][0] = x.x; pair[0][1] = x.y;
                pair[1][0] = x.z; pair[1][1] = x.w;
            }
        }
        float d[NG][NT][4];
#pragma unroll
        for (int x = 0; x < NG; ++x) {
            const uint2 lo = lds64(at.k[0][x] + block * kv4_block_bytes<D>());
            const uint2 hi = lds64(at.k[1][x] + block * kv4_block_bytes<D>());
            const uint32_t xs[2] = {lo.x, lo.y}, ys[2] = {hi.x, hi.y};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint32_t x8 = xs[w] >> 8, y8 = ys[w] >> 8;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t mask = e ? kHighHalves : kLowHalves;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (w + e == 0)
                            mma_16816_first(d[x][nt], xs[w] & mask, ys[w] & mask, x8 & mask, y8 & mask,
                                            q.b[x][w][e][nt][0], q.b[x][w][e][nt][1]);
                        else
                            mma_16816(d[x][nt], xs[w] & mask, ys[w] & mask, x8 & mask, y8 & mask,
                                      q.b[x][w][e][nt][0], q.b[x][w][e][nt][1]);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float2 k[NG];
#pragma unroll
            for (int x = 0; x < NG; ++x) {
                k[x] = wide(pair[i][x]);
                const float2 a = wide(pair[i][NG + x]);
                va[i][x] = a.x;
                vm[i][x] = fmaf(7.5f, a.x, a.y);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float sum = k[0].y * q.sum[0][nt][j];
#pragma unroll
                    for (int x = 0; x < NG; ++x) {
                        if (x) sum = fmaf(k[x].y, q.sum[x][nt][j], sum);
                        sum = fmaf(k[x].x, d[x][nt][2 * i + j], sum);
                    }
                    s[nt][2 * i + j] = __fmul_rn(sum, q.unit[nt][j]);
                }
            // What rows past the end hold is anything, a NaN included.
            if (TAIL && (lane >> 2) * 2 + i >= valid) {
#pragma unroll
                for (int x = 0; x < NG; ++x) va[i][x] = vm[i][x] = 0.f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][2 * i] = s[nt][2 * i + 1] = -INFINITY;
            }
        }
    }

    // Probabilities, their sums, and the weights P^T a' as two fp16.  Where the weights
    // of a column's rows here sum up to more than 2^15 or to NaN (in fp32, on a pipe
    // with room; with p as weights of the least scale among them), the column's
    // references move, by the scores and finite scales alone: p is finite then.
    // ADDED: z holds what o does since it was last centred, and moves with it.
    template <bool ADDED>
    __device__ __forceinline__ void weigh(Kv4State<D, NT>& st, float (&z)[NG][NT][4], int lane) {
        float p[NT][4], ps[NT][2], all[NT][2];
        bool over = false;
        auto form = [&]() {
            over = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    p[nt][c] = fast_exp2(s[nt][c] - st.r[nt][c & 1]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    ps[nt][j] = p[nt][j] + p[nt][2 + j];
                    all[nt][j] = ps[nt][j] * 0x1p-24f;
                }
#pragma unroll
                for (int x = 0; x < NG; ++x)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float w0 = p[nt][2 * i], w1 = p[nt][2 * i + 1];
                        if (x) {
                            w0 *= st.f[x][nt][0];
                            w1 *= st.f[x][nt][1];
                        }
                        w0 *= va[i][x];
                        w1 *= va[i][x];
                        all[nt][0] += w0;
                        all[nt][1] += w1;
                        const uint32_t h = pack_half2(w0, w1);
                        const float2 r = wide(h);
                        w[x][nt][i] = h;
                        rest[x][nt][i] = pack_half2(w0 - r.x, w1 - r.y);
                    }
                over |= outgrown(max_nan(all[nt][0], all[nt][1]));
            }
        };
        form();
        if (__any_sync(0xffffffffu, over || st.fresh)) {
            // Rescale what is summed so far to the weights' new references.  A column
            // moves for its own weights only: no head's bits depend on another's.
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t column = 0x11111111u << (lane & 3);
                    const bool move = st.fresh || (__ballot_sync(0xffffffffu, outgrown(all[nt][j])) & column);
                    // Scores so large that a step of fp32 is worth a power of two or more: the
                    // first reference is the largest of them, which is exact, no weight is
                    // more than its scale, and the other groups share that reference.
                    const float own = fabsf(fmaxf(s[nt][j], s[nt][2 + j]));
                    const bool far = __ballot_sync(0xffffffffu, own >= kKv4Far && own < INFINITY) & column;
                    const float r0 = st.r[nt][j];
                    float by0 = 0.f;
#pragma unroll
                    for (int x = 0; x < NG; ++x) {
                        float top = -INFINITY;  // log2 of the largest weight as it is
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float at = s[nt][2 * i + j];
                            top = fmaxf(top, far ? at : at - r0 + fmaxf(fast_log2(va[i][x]), kKv4Least));
                        }
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1)
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        const float lead = x ? fast_log2(st.f[x][nt][j]) : 0.f;
                        // up only, but from no reference to any
                        float by = rintf(top + lead - kKv4Shift);
                        if (far) by = x ? by0 + lead : top - r0;
                        const bool up = move && by > (st.fresh ? -INFINITY : 0.f);
                        if (!up) by = 0.f;
                        // without a reference the sums are 0
                        const float u = st.fresh ? 1.f : fast_exp2(-by);
#pragma unroll
                        for (int dm = 4 * x; dm < 4 * x + 4; ++dm) {
                            st.o[dm][nt][j] *= u;
                            st.o[dm][nt][j + 2] *= u;
                        }
                        if constexpr (ADDED) z[x][nt][j] *= u;
                        if (x == 0) {
                            by0 = by;
                            st.r[nt][j] = far && up ? top : r0 + by;
                            st.l[nt][j] *= u;
#pragma unroll
                            for (int y = 0; y < NG; ++y) st.mid[y][nt][j] *= u;
                        } else if (far && up) {
                            st.f[x][nt][j] = 1.f;
                        } else {
                            st.f[x][nt][j] *= fast_exp2(by0 - by);
                        }
                    }
                }
            st.fresh = false;
            form();
        }
        // row sums and middles, of the unrounded p
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 2; ++j) st.l[nt][j] += ps[nt][j];
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int x = 0; x < NG; ++x)
                    st.mid[x][nt][c & 1] = fmaf(p[nt][c], vm[c >> 1][x], st.mid[x][nt][c & 1]);
        }
    }

    // O^T += V^T W^T and z, the weights in the B layout (k = position, n = head).
    // FIRST: z starts here.
    template <bool FIRST>
    __device__ __forceinline__ void apply(const Kv4Lane<D>& at, int block, Kv4State<D, NT>& st,
                                          float (&z)[NG][NT][4]) const {
        constexpr uint32_t kFifteen = 0x000f000fu;
#pragma unroll
        for (int x = 0; x < NG; ++x) {
            uint32_t v[4], wb[NT][2], wr[NT][2];
            ldsm_b8_trans(v, at.v[x] + block * kv4_block_bytes<D>());
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    wb[nt][i] = movmatrix_trans(w[x][nt][i]);
                    wr[nt][i] = movmatrix_trans(rest[x][nt][i]);
                }
            auto product = [&](float (&acc)[NT][4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816(acc[nt], a0, a1, a2, a3, wb[nt][0], wb[nt][1]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816(acc[nt], a0, a1, a2, a3, wr[nt][0], wr[nt][1]);
            };
            if constexpr (FIRST) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma_16816_first(z[x][nt], kFifteen, kFifteen, kFifteen, kFifteen, wb[nt][0], wb[nt][1]);
                    mma_16816(z[x][nt], kFifteen, kFifteen, kFifteen, kFifteen, wr[nt][0], wr[nt][1]);
                }
            } else {
                product(z[x], kFifteen, kFifteen, kFifteen, kFifteen);
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {       // dims 16 y + 2 g, + 1 of the group
                const uint32_t v8 = v[y] >> 8;
                product(st.o[4 * x + y], v[y] & kLowHalves, v[y] & kHighHalves, v8 & kLowHalves,
                        v8 & kHighHalves);
            }
        }
    }
};

// Where a warp's copies are: the tile of its cursor and, looked up already, the
// pages of the warp's MT blocks of it (-1: nothing to copy, zeros are filled in:
// a block without positions or a page id outside the pool).  The page index, the
// block within the page and the positions left go along with the cursor; what
// depends on the sequence and head is formed where these change.
template <int D, int MT, int NW>
struct Kv4Loader {
    static constexpr int kBlock = 16;
    static constexpr int LPB = 32 / MT;         // lanes per block
    static constexpr int CPR = D / 32;          // 16-byte chunks per row
    static constexpr int RPC = LPB / CPR;       // rows of a block per warp-wide copy
    static constexpr int kRowScales = 8 * (D / kKv4Group);
    static constexpr int kTile = kBlock * MT * NW;
    static_assert(32 % MT == 0 && LPB % CPR == 0 && RPC % 2 == 0, "lanes of a block");
    TileCursor cur;
    int idx, sub, left;                         // the lane's block: page index, block within the page, positions from there on
    int page;
    int bpp, step_idx, step_sub;                // blocks per page; NW * MT blocks
    const int* row;                             // the sequence's pages
    uint32_t off, scale_off;                    // the lane's chunk in the kv head's part of page 0, in 16 bytes
    uint32_t k_dst, v_dst, scale_dst;           // ... and in a step in shared memory

    __device__ __forceinline__ void unit(const CachedDecodeParams<Kv4View>& p, const int* lens, int warp,
                                         int lane) {
        const int kvh = p.head_groups == 1 ? cur.j : cur.j / p.head_groups;
        const int blk = (cur.i * NW + warp) * MT + lane / LPB;
        idx = blk / bpp;
        sub = blk - idx * bpp;
        off = (uint32_t)(p.cache.row(0, kvh, lane % LPB / CPR) >> 4) + lane % CPR;
        scale_off = kvh * p.cache.head_scales16 + lane % LPB;
        row = p.block_table + (size_t)cur.b * p.bt_stride;
        left = (cur.b < p.batch ? lens[cur.b] : 0) - blk * kBlock;
    }
    __device__ __forceinline__ void init(const CachedDecodeParams<Kv4View>& p, const TileCursor& start,
                                         const int* lens, int warp, int lane) {
        cur = start;
        bpp = p.cache.page_size / kBlock;
        step_idx = NW * MT / bpp;
        step_sub = NW * MT - step_idx * bpp;
        const int c = lane % CPR, r = lane % LPB / CPR, block = lane / LPB * kv4_block_bytes<D>();
        k_dst = block + kv4_k_offset<D>(r, c);
        v_dst = block + kv4_v_offset<D>(r, c);
        scale_dst = lane / LPB * (kBlock * kRowScales) + lane % LPB * 16;
        unit(p, lens, warp, lane);
        look_up(p, lens, warp);
    }
    __device__ __forceinline__ void look_up(const CachedDecodeParams<Kv4View>& p, const int*, int) {
        page = -1;
        if (left > 0) {
            const int id = row[idx];
            if ((unsigned)id < (unsigned)p.cache.num_pages) page = id;
        }
    }
    // Starts the copies of the step: 16 rows of K and of V and their scales of
    // each block.
    __device__ __forceinline__ void copy(const CachedDecodeParams<Kv4View>& p, uint32_t kst, uint32_t vst,
                                         uint32_t scale_at, int, int lane, uint64_t policy) const {
        // 32-bit numbers of 16 bytes: the host checks that a cache has no more.
        const uint32_t row_stride = p.cache.block16;
        const uint32_t bytes = page >= 0 ? 16u : 0u;
        const uint32_t pg = max(page, 0);
        const size_t at = (size_t)(off + pg * p.cache.page16 + sub * row_stride) * 16;
        const uint8_t* ks = p.cache.k + at;
        const uint8_t* vs = p.cache.v + at;
        auto rows = [&](auto stride) {
#pragma unroll
            for (int i = 0; i < kBlock / RPC; ++i) {
                const int line = i * RPC / (256 / D), turn = line % (D == 128 ? 4 : 2);     // what i * RPC rows add
                cp_async_16(kst + (k_dst ^ (turn * 32)) + line * 128, ks + (size_t)stride * (i * RPC), bytes, policy);
                cp_async_16(vst + (v_dst ^ (turn * 16)) + line * 128, vs + (size_t)stride * (i * RPC), bytes, policy);
            }
        };
        if (row_stride == D / 2) rows(std::integral_constant<uint32_t, D / 2>());
        else rows(row_stride);
        if (kRowScales >= LPB || lane % LPB < kRowScales) {     // 16 rows of kRowScales bytes, 16 at a time
            const uint32_t from = scale_off + pg * p.cache.scales16 + sub * kRowScales;
            const uint8_t* src = reinterpret_cast<const uint8_t*>(p.cache.scales) + (size_t)from * 16;
#pragma unroll
            for (int i = 0; i == 0 || i * LPB < kRowScales; ++i)
                cp_async_16(scale_at + scale_dst + i * LPB * 16, src + i * LPB * 16, bytes, policy);
        }
    }
    __device__ __forceinline__ void advance(const CachedDecodeParams<Kv4View>& p, const int* seq_start,
                                            const int* lens, int B, int upb, int warp, int lane) {
        cur.advance(seq_start, B, upb, 1);
        if (cur.i == 0) {                       // next unit
            unit(p, lens, warp, lane);
        } else {
            left -= kTile;
            idx += step_idx;
            sub += step_sub;
            if (sub >= bpp) { sub -= bpp; ++idx; }
        }
    }
};

// Steps of MT blocks of 16 rows; CTAS per SM.
template <int D, int NT, int MT, int STAGES, int NW, int CTAS>
struct Kv4Format {
    static constexpr int kD = D, kNT = NT, kMT = MT, kStages = STAGES, kNW = NW, kCtas = CTAS, kRun = 1;
    using Params = CachedDecodeParams<Kv4View>;
    using Smem = Kv4Smem<D, NT, MT, STAGES, NW>;
    using Loader = Kv4Loader<D, MT, NW>;
    using Query = Kv4Query<D, NT>;
    using State = Kv4State<D, NT>;

    static __device__ __forceinline__ int dim(int dm, int g) {
        return (dm >> 2) * kKv4Group + 16 * (dm & 3) + 2 * g;
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        return pack_half2(min_nan(lo, kKv4Top), min_nan(hi, kKv4Top));
    }
    static __device__ __forceinline__ void consume(uint32_t kst, uint32_t vst, const unsigned char* sc,
                                                   int valid, const Query& q, State& st, float,
                                                   int lane) {
        const Kv4Lane<D> at(kst, vst, smem_u32(sc), lane);
        float z[D / kKv4Group][NT][4];
        if (valid >= 16 * MT) {
            // The next block's scores beside the products of the one before it.
            Kv4Block<D, NT> b[2];
            b[0].template score<false>(at, 0, 16, q, lane);
            b[0].template weigh<false>(st, z, lane);
#pragma unroll
            for (int i = 1; i < MT; ++i) {
                b[i % 2].template score<false>(at, i, 16, q, lane);
                if (i == 1) b[0].template apply<true>(at, 0, st, z);
                else b[(i - 1) % 2].template apply<false>(at, i - 1, st, z);
                b[i % 2].template weigh<true>(st, z, lane);
            }
            b[(MT - 1) % 2].template apply<MT == 1>(at, MT - 1, st, z);
            st.centre(z);
        } else {
#pragma unroll 1
            for (int i = 0; i * 16 < valid; ++i) {
                Kv4Block<D, NT> b;
                b.template score<true>(at, i, valid - i * 16, q, lane);
                b.template weigh<false>(st, z, lane);
                b.template apply<true>(at, i, st, z);
                st.centre(z);
            }
        }
    }
};

}  // namespace fr
