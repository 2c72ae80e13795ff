// kv8_decode_kernels.cuh - single-token attention over the 8-bit paged cache.
//
// Mathematics, per (sequence, query head h of kv head j), positions t < len
// in blocks of 16:
//   s_t = (q . kc_t) * kscale(block) / sqrt(D)
//   o   = sum_t 2^(s_t log2 e - m) * vscale(block) * vc_t,  l = sum_t 2^(...)
//   out = o / l  (zeros for an empty sequence)
// with kc, vc the 8-bit codes.  Scores, m, l and o are fp32.  Codes widen to
// fp16 exactly; a term 2^s vscale enters the product with V as fp16 on a
// reference of its own (Kv8State), 2^8 up, so that one as small as 2^-22 of the
// largest keeps all its bits.  Long calls take that one fp16 (each term rounded
// by 2^-11 of itself at most, which leaves the outputs 1.2 to 1.3 times as far
// from the exact ones as their own rounding does); in short calls (REST), where
// the outputs average fewer terms (1.5 times) and the warps wait for memory, a
// second product takes the rest of each term: 1 x 512 tokens 8.0 -> 8.1 us, 64
// of 200 to 300 10.0 -> 10.4, 64 of 1024 to 8192 would be 50.1 -> 52.3.  The row
// sum uses the unrounded probabilities.
//
// Bytes: 2 * D of codes per position and kv head, plus 8 of scales per 16
// positions; 4 * D * G operations on them.  Measured, 28 / 4 heads of 128: 64
// sequences of 8192 to 32768 tokens in e4m3 203 us, 6.4 TB/s (0.98 of a copy's
// rate, bound by HBM), in int8 218; of 1024 to 8192 51 to 56 us, 4.9 to 5.3
// TB/s, in int8 61 to 66: issue slots (56 and 61 % of the cycles at 16 warps
// per SM) and latency, about 7 us of them launch, first rows, fold and merge;
// one sequence of 512 tokens 8 (14 / 2 heads of 64).
//
// Decomposition: the frame's (cached_decode_kernels.cuh).  A warp's copies are
// cp.async, so any strides and page size will do.  The page of a step is looked up
// one step before its copies start.
// (Copies by TMA boxes of gcd(page_size, TILE) rows, one producer warp per
// CTA, were measured first: with pages of 16 rows the boxes of 2 KB took 80 ns
// each, 95 us for 304 MB, where pages of 64 rows took 64 us for 272 MB.)
//
// Fragments: each consumer warp takes MT m-tiles of 16 rows.  The codes go
// from shared memory to the operands of mma m16n8k16 without ldmatrix:
// contraction order is free, so k-step w of a row is word w of the 16 bytes
// that a lane loads at once, and for P.V the words of two neighbouring rows
// are interleaved by one byte permutation.  A lane owns D/8 consecutive head
// dims of the output (kv_dim).  All loads are 16 bytes (8 for V at D = 64)
// and free of bank conflicts under the swizzle; at D = 64 (two rows to a
// 128-byte line) that takes rows 2 and 3, 6 and 7 exchanged (pos_of).
#pragma once
#include "cached_decode_kernels.cuh"
#include "kv8_common.cuh"

namespace fr {

constexpr float kShift = 8.f;           // a term at its reference counts 2^8 ...
constexpr float kTop = 15.f;            // ... and may grow to 2^15 before the reference moves (fp16: < 2^16)

template <int D, int NT, int MT, int STAGES, int NW>
struct Kv8Smem {
    static constexpr int kStepBytes = 16 * MT * D;                      // K (or V) of one step
    static constexpr int kWarpBytes = 2 * STAGES * kStepBytes;          // a warp's ring
    static constexpr size_t kRingBytes = size_t(NW) * kWarpBytes;
    static constexpr int kXFloats = (D / 16) * 4 + 4;
    static constexpr size_t kXOffset = kRingBytes;
    static constexpr size_t kXBytes = size_t(2) * 32 * kXFloats * sizeof(float);
    static constexpr size_t kScaleOffset = kXOffset + kXBytes;
    static constexpr int kStepScales = MT * sizeof(float2);
    static constexpr size_t kScaleBytes = size_t(NW) * STAGES * kStepScales;
    static constexpr size_t kFlagOffset = kScaleOffset + kScaleBytes;
    static constexpr size_t kMetaOffset = kFlagOffset + 16 * sizeof(int);
    static constexpr size_t kMetaBytes = (2 * kPersistMaxBatch + 1 + 16) * sizeof(int);
    // +1024: the rings are realigned to 1024 bytes (the swizzle's period).
    static constexpr size_t kBytes = 1024 + kMetaOffset + kMetaBytes;
    static_assert(kStepBytes % 1024 == 0 && kScaleOffset % 8 == 0, "alignment");
    // cached_merge reuses the exchange area: weights [threads] + 2 x heads
    static_assert(kXBytes >= (NW * 32 + 2 * NT * 8) * sizeof(float), "merge area");
};

// Row of a 16-row m-tile that fragment row i stands for.
template <int D>
__device__ __forceinline__ int pos_of(int i) {
    return D == 64 ? i ^ ((i >> 1) & 1) : i;
}

// Byte offset of 16-byte chunk c of row r: chunks are exchanged by row number
// so that eight lanes reading a column of chunks hit distinct banks.
template <int D>
__device__ __forceinline__ uint32_t kv8_offset(int r, int c) {
    return D == 128 ? uint32_t(r * 128 + ((c ^ (r & 7)) << 4))
                    : uint32_t(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// Running state of a warp over an item, per head column.  Scores are in base 2
// (log2 e folded in).  m and mv are references near the running maxima of s
// and of s + log2(vscale): l holds 2^(kShift - m) sum 2^s, o holds
// 2^(kShift - mv) sum 2^s vscale vc.  A reference moves only when a term
// would pass 2^kTop, so most steps need no maximum across lanes and no
// rescaling; with o on its own reference, terms of blocks with small V scales
// keep their bits when they are the ones that count.
template <int D, int NT>
struct Kv8State {
    float o[D / 16][NT][4];
    float m[NT][2], mv[NT][2], l[NT][2];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int dm = 0; dm < D / 16; ++dm)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[dm][nt][c] = 0.f;
            m[nt][0] = m[nt][1] = mv[nt][0] = mv[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }
    }
    // Row sums over the warp, and o on m's reference: the (m, l, o) of the merges.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x = l[nt][j];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                l[nt][j] = x;
                const float f = mv[nt][j] == -INFINITY ? 1.f : fast_exp2(mv[nt][j] - m[nt][j]);
#pragma unroll
                for (int dm = 0; dm < D / 16; ++dm) {
                    o[dm][nt][j] *= f;
                    o[dm][nt][j + 2] *= f;
                }
            }
    }
};

// q of one item as the B operand, in the order that K's words come in: lane
// (g, t) holds dims (D/4) * t .. of head g, as fp16 pairs.  (int8 codes can
// also enter integer products, with q in 16-bit fixed point on its head's
// largest value as two s8 planes: 64 sequences of 8192 to 32768 tokens 209 us
// instead of 220, but a channel far above the others takes their bits.)
template <int D, int NT>
struct Kv8Query {
    uint32_t b[D / 16][NT][2];

    __device__ __forceinline__ void load(const __half* q, int gcount, float, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int hj = nt * 8 + g;
            const __half* row = q + (size_t)hj * D + (D / 4) * t;
#pragma unroll
            for (int w = 0; w < D / 16; w += 2) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (hj < gcount) v = *reinterpret_cast<const uint4*>(row + w * 4);
                b[w][nt][0] = v.x; b[w][nt][1] = v.y;
                b[w + 1][nt][0] = v.z; b[w + 1][nt][1] = v.w;
            }
        }
    }
};

// One step: 16 * MT rows of K at kst and V at vst, of which the first `valid`
// (>= 1) are positions; sc: their blocks' scales.  REST: what rounding a weight
// to fp16 takes off goes into a product of its own.
template <int D, int NT, int MT, bool REST, class Code>
__device__ __forceinline__ void consume_kv8(uint32_t kst, uint32_t vst, const float2* sc, int valid,
                                            const Kv8Query<D, NT>& q,
                                            Kv8State<D, NT>& st, float sl2, int lane) {
    constexpr int KL = D / 64;                  // 16-byte loads per K row and lane
    constexpr int VW = D / 32;                  // words per V row and lane
    const int g = lane >> 2, t = lane & 3;
    const int rg = pos_of<D>(g);                // rows of the A fragments: rg, rg + 8
    const bool tail = valid < 16 * MT;          // uniform over the warp
    float ks[MT], lv[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        // A block without positions has no scales in the stage.  An infinite
        // scale acts as NaN, as the sum of its rows' infinities of both signs
        // would, and not as one infinity of the sum's sign.
        float2 x = mt * 16 < valid ? sc[mt] : make_float2(0.f, 0.f);
        ks[mt] = (x.x + (x.x - x.x)) * sl2;
        lv[mt] = fast_log2(x.y + (x.y - x.y));
    }

    // ---- S^T = K Q^T
    float s[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = mt * 16 + rg;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[mt][nt][c] = 0.f;
#pragma unroll
        for (int j = 0; j < KL; ++j) {
            const int chunk = KL * t + j;
            const uint4 x = lds128(kst + kv8_offset<D>(r, chunk));
            const uint4 y = lds128(kst + kv8_offset<D>(r + 8, chunk));
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int ks0 = j * 4 + w;
                const uint32_t xw = Code::prepare(xs[w]), yw = Code::prepare(ys[w]);
                const uint32_t a0 = Code::half2_lo(xw), a1 = Code::half2_lo(yw);
                const uint32_t a2 = Code::half2_hi(xw), a3 = Code::half2_hi(yw);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_16816(s[mt][nt], a0, a1, a2, a3, q.b[ks0][nt][0], q.b[ks0][nt][1]);
            }
        }
    }

    // ---- exponents of both sums, on the references as they are; a masked
    // position's are -inf whatever its row holds
    float ep[MT][NT][4], ew[MT][NT][4];
    float top = -INFINITY;
    auto exponents = [&]() {
        top = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float mp = st.m[nt][j] == -INFINITY ? -kShift : st.m[nt][j] - kShift;
                const float mw = st.mv[nt][j] == -INFINITY ? -kShift : st.mv[nt][j] - kShift;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int c = j; c < 4; c += 2) {
                        ep[mt][nt][c] = fmaf(s[mt][nt][c], ks[mt], -mp);
                        ew[mt][nt][c] = fmaf(s[mt][nt][c], ks[mt], lv[mt] - mw);
                        if (tail && mt * 16 + rg + (c >> 1) * 8 >= valid)
                            ep[mt][nt][c] = ew[mt][nt][c] = -INFINITY;
                        top = fmaxf(top, fmaxf(ep[mt][nt][c], ew[mt][nt][c]));
                    }
            }
    };
    exponents();
    bool first = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) first |= st.m[nt][0] == -INFINITY || st.m[nt][1] == -INFINITY ||
                                             st.mv[nt][0] == -INFINITY || st.mv[nt][1] == -INFINITY;
    if (__any_sync(0xffffffffu, first || top > kTop)) {
        // move the references to the maxima and rescale what is summed so far
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float xp = -INFINITY, xw = -INFINITY;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int c = j; c < 4; c += 2) {
                        xp = fmaxf(xp, ep[mt][nt][c]);
                        xw = fmaxf(xw, ew[mt][nt][c]);
                    }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    xp = fmaxf(xp, __shfl_xor_sync(0xffffffffu, xp, d));
                    xw = fmaxf(xw, __shfl_xor_sync(0xffffffffu, xw, d));
                }
                // Exponents are relative to the reference (0 while there is none),
                // kShift up.  A column moves for its own terms only: no head's
                // bits depend on another's.
                const float m0 = st.m[nt][j], w0 = st.mv[nt][j];
                const float m1 = m0 == -INFINITY ? xp - kShift : xp > kTop ? m0 - kShift + xp : m0;
                const float w1 = w0 == -INFINITY ? xw - kShift : xw > kTop ? w0 - kShift + xw : w0;
                const float fl = m0 == -INFINITY ? 0.f : fast_exp2(m0 - m1);
                const float fo = w0 == -INFINITY ? 0.f : fast_exp2(w0 - w1);
                st.m[nt][j] = m1;
                st.mv[nt][j] = w1;
                // without a reference the sums are 0, or NaN and stay so
                st.l[nt][j] *= m0 == -INFINITY ? 1.f : fl;
#pragma unroll
                for (int dm = 0; dm < D / 16; ++dm) {
                    st.o[dm][nt][j] *= w0 == -INFINITY ? 1.f : fo;
                    st.o[dm][nt][j + 2] *= w0 == -INFINITY ? 1.f : fo;
                }
            }
        exponents();
    }

    // ---- row sums (unrounded), and W^T = P^T vscale as fp16 in the B layout
    // (k = position, n = head)
    uint32_t wb[MT][NT][2], wr[MT][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                st.l[nt][c & 1] += fast_exp2(ep[mt][nt][c]);
                ew[mt][nt][c] = fast_exp2(ew[mt][nt][c]);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float w0 = ew[mt][nt][2 * e], w1 = ew[mt][nt][2 * e + 1];
                const uint32_t w = pack_half2(w0, w1);
                wb[mt][nt][e] = movmatrix_trans(w);
                if constexpr (REST) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
                    wr[mt][nt][e] = movmatrix_trans(pack_half2(w0 - f.x, w1 - f.y));
                }
            }
        }
    }

    // ---- O^T += V^T W^T
    const int p0 = pos_of<D>(2 * t), p1 = pos_of<D>(2 * t + 1);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = mt * 16;
        uint32_t w[4][VW];                      // rows p0, p1, p0 + 8, p1 + 8
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (i & 1 ? p1 : p0) + (i >> 1) * 8;
            if constexpr (D == 128) {
                const uint4 x = lds128(vst + kv8_offset<D>(r + row, g));
                w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
            } else {
                const uint2 x = lds64(vst + kv8_offset<D>(r + row, g >> 1) + (g & 1) * 8);
                w[i][0] = x.x; w[i][1] = x.y;
            }
            // Rows past the end hold anything, a NaN code included: their
            // weight is 0, and 0 * NaN is not.
            if (Code::kHasNan && tail && mt * 16 + row >= valid) {
#pragma unroll
                for (int x = 0; x < VW; ++x) w[i][x] = 0;
            }
        }
#pragma unroll
        for (int x = 0; x < VW; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e) {       // dims 4x + 2e, 4x + 2e + 1 of the lane's
                const int dm = 2 * x + e;
                const uint32_t lo = Code::prepare(__byte_perm(w[0][x], w[1][x], e ? 0x7362 : 0x5140));
                const uint32_t hi = Code::prepare(__byte_perm(w[2][x], w[3][x], e ? 0x7362 : 0x5140));
                const uint32_t a0 = Code::half2_lo(lo), a1 = Code::half2_hi(lo);
                const uint32_t a2 = Code::half2_lo(hi), a3 = Code::half2_hi(hi);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_16816(st.o[dm][nt], a0, a1, a2, a3, wb[mt][nt][0], wb[mt][nt][1]);
                if constexpr (REST) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_16816(st.o[dm][nt], a0, a1, a2, a3, wr[mt][nt][0], wr[mt][nt][1]);
                }
            }
    }
}

// Where a warp's copies are: the tile of its cursor and, looked up already,
// the pages of the warp's MT blocks of it (-1 where there is no position,
// num_pages for an id outside the pool).  The page index and the block within
// the page go along with the cursor, without divisions.
template <int D, int MT, int NW>
struct Kv8Loader {
    static constexpr int CPR = D / 16;          // 16-byte chunks per row
    static constexpr int RPC = 32 / CPR;        // rows per warp-wide copy
    TileCursor cur;
    int idx, sub;                               // page index and block within it, first block
    int bpp, step_idx, step_sub, idx0, sub0;    // blocks per page; NW * MT blocks; tile 0
    int page[MT];
    long long lane_off;

    __device__ __forceinline__ void init(const CachedDecodeParams<Kv8View>& p, const TileCursor& start,
                                         const int* lens, int warp, int lane) {
        cur = start;
        bpp = p.cache.page_size / kKv8Block;
        step_idx = NW * MT / bpp;
        step_sub = NW * MT - step_idx * bpp;
        idx0 = warp * MT / bpp;
        sub0 = warp * MT - idx0 * bpp;
        const int blk = (cur.i * NW + warp) * MT;
        idx = blk / bpp;
        sub = blk - idx * bpp;
        lane_off = (long long)(lane / CPR) * p.cache.row_stride + (lane % CPR) * 16;
        look_up(p, lens, warp);
    }
    __device__ __forceinline__ void look_up(const CachedDecodeParams<Kv8View>& p, const int* lens, int warp) {
        const int pos = (cur.i * NW + warp) * (16 * MT);
        const int left = cur.b < p.batch ? lens[cur.b] - pos : 0;
        const int* row = p.block_table + (size_t)cur.b * p.bt_stride;
        int at = idx, s = sub;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            page[m] = -1;
            if (16 * m < left) page[m] = min((unsigned)row[at], (unsigned)p.cache.num_pages);
            if (++s == bpp) { s = 0; ++at; }
        }
    }
    // Starts the copies of the step: 16 rows of K and of V and the two scales
    // of each block that holds positions; zeros for a page outside the pool.
    __device__ __forceinline__ void copy(const CachedDecodeParams<Kv8View>& p, uint32_t kst, uint32_t vst,
                                         uint32_t scale_at, int kvh, int lane, uint64_t policy) const {
        const int r0 = lane / CPR, c = lane % CPR;
        int s = sub;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (page[m] >= 0) {                 // uniform over the warp
                const bool real = page[m] < p.cache.num_pages;
                const int pg = real ? page[m] : 0;
                const uint32_t bytes = real ? 16u : 0u;
                const long long off = pg * p.cache.page_stride + kvh * p.cache.head_stride +
                                      s * kKv8Block * p.cache.row_stride + lane_off;
                const uint8_t* ks = p.cache.k + off;
                const uint8_t* vs = p.cache.v + off;
                if (p.cache.row_stride == D) {  // rows one after the other: constant steps
#pragma unroll
                    for (int i = 0; i < 16 / RPC; ++i) {
                        const uint32_t dst = kv8_offset<D>(m * 16 + i * RPC + r0, c);
                        cp_async_16(kst + dst, ks + i * (RPC * D), bytes, policy);
                        cp_async_16(vst + dst, vs + i * (RPC * D), bytes, policy);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16 / RPC; ++i) {
                        const uint32_t dst = kv8_offset<D>(m * 16 + i * RPC + r0, c);
                        cp_async_16(kst + dst, ks, bytes, policy);
                        cp_async_16(vst + dst, vs, bytes, policy);
                        ks += RPC * p.cache.row_stride;
                        vs += RPC * p.cache.row_stride;
                    }
                }
                if (lane == 0)
                    cp_async_8(scale_at + m * 8,
                               reinterpret_cast<const float2*>(p.cache.scales) + ((size_t)pg * p.cache.Hkv + kvh) * bpp + s,
                               real ? 8u : 0u);
            }
            if (++s == bpp) s = 0;
        }
    }
    __device__ __forceinline__ void advance(const CachedDecodeParams<Kv8View>&, const int* seq_start,
                                            const int*, int B, int upb, int, int) {
        cur.advance(seq_start, B, upb, 1);
        if (cur.i == 0) {                       // next unit
            idx = idx0;
            sub = sub0;
        } else {
            idx += step_idx;
            sub += step_sub;
            if (sub >= bpp) { sub -= bpp; ++idx; }
        }
    }
};

// Steps of MT blocks of 16 rows; CTAS per SM; REST as in consume_kv8.
template <int D, int NT, int MT, int STAGES, int NW, int CTAS, bool REST, class Code>
struct Kv8Format {
    static constexpr int kD = D, kNT = NT, kMT = MT, kStages = STAGES, kNW = NW, kCtas = CTAS, kRun = 4;
    using Params = CachedDecodeParams<Kv8View>;
    using Smem = Kv8Smem<D, NT, MT, STAGES, NW>;
    using Loader = Kv8Loader<D, MT, NW>;
    using Query = Kv8Query<D, NT>;
    using State = Kv8State<D, NT>;

    static __device__ __forceinline__ int dim(int dm, int g) { return (D / 8) * g + 2 * dm; }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
    static __device__ __forceinline__ void consume(uint32_t kst, uint32_t vst, const unsigned char* sc,
                                                   int valid, const Query& q, State& st, float sl2,
                                                   int lane) {
        consume_kv8<D, NT, MT, REST, Code>(kst, vst, reinterpret_cast<const float2*>(sc), valid, q,
                                           st, sl2, lane);
    }
};

}  // namespace fr
