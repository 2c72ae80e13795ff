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
// Decomposition: persistent CTAs take equal shares of the batch's work, as in
// batched_kernels.cuh (units, items, pieces merged by the contributor that
// completes a unit), over tiles of TILE = 16 * MT * NW positions.  Inside a
// CTA every warp streams for itself: warp w copies and consumes rows
// 16 * MT * w .. of each tile through a ring of its own (cp.async, STAGES
// steps of MT blocks of K and V and their scales), so a step needs no barrier
// between warps and no producer, and any strides and page size will do.  The
// page of a step is looked up one step before its copies start.
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
#include "batched_kernels.cuh"
#include "kv8_common.cuh"

namespace fr {

struct Kv8DecodeParams {
    Kv8View cache;
    const __half* q;             // [B, H, D], q_stride halves between sequences
    __half* out;                 // [B, H, D]
    const int* kv_lens;          // [B]
    const int* block_table;      // [B, bt_stride]
    float* part_ml;              // two slots per CTA: [GP][2] (m, l), and fragments of acc
    float* part_acc;
    int* counters;               // one per unit, then one per slot; zero between calls
    int max_units;
    long long q_stride;
    int batch, H, G, head_groups;
    int bt_stride;
    int max_len;                 // lengths are cut to this
    int min_tiles_per_cta, min_ctas;
    int item_cost, merge_cost;   // in tile times, see ShareMap
    int whole_tiles;             // at least 1, see ShareMap
    float scale_log2;            // log2(e) / sqrt(D)
};

// Cost-balanced shares in 32-bit arithmetic.  A unit of nb tiles spans xc + nb
// + mc cost points: xc before its first tile (starting an item), mc after its
// last (merging).  Of Ctot points CTA c takes the c-th of C equal shares (the
// first Ctot mod C one point longer) and the tiles whose points lie in it; a
// border that falls into a short unit moves to the unit's nearer end, since
// cutting it costs a merge (some CTAs are then left without tiles).
struct ShareMap {
    const int* seq_start;        // tiles before each sequence, all units
    int B, upb, xc, mc;
    int whole;                   // units of at most this many tiles are not cut
    int C, share, extra;         // Ctot = C * share + extra

    __device__ __forceinline__ void split(int Ctot, int ctas) {
        C = ctas;
        share = Ctot / ctas;
        extra = Ctot - share * ctas;
    }
    __device__ __forceinline__ int cs(int b) const { return seq_start[b] + (xc + mc) * upb * b; }
    __device__ __forceinline__ int beg(int c) const {       // first tile of CTA c
        if (c >= C) return seq_start[B];
        const int v = c * share + min(c, extra);
        int lo = 0, hi = B - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (cs(mid) <= v) lo = mid; else hi = mid - 1;
        }
        const int nb = (seq_start[lo + 1] - seq_start[lo]) / upb;
        const int span = nb + xc + mc;
        const int off = v - cs(lo);
        const int j = min(off / span, upb - 1);
        int i = max(0, min(off - j * span - xc, nb - 1));
        if (nb <= whole) i = 2 * i <= nb ? 0 : nb;      // to the unit's nearer end
        return seq_start[lo] + j * nb + i;
    }
    // CTA that holds tile i of unit j of sequence b: the one with the tile's
    // last cost point
    __device__ __forceinline__ int cta_of(int b, int j, int nb, int i) const {
        const int v = cs(b) + j * (nb + xc + mc) + xc + i + (i == nb - 1 ? mc : 0);
        const int longer = extra * (share + 1);
        return v < longer ? v / (share + 1) : extra + (v - longer) / share;
    }
};

// First of the two dims that lane (g, t) holds in fragment dm.
template <int D>
__device__ __forceinline__ int kv_dim(int dm, int g) { return (D / 8) * g + 2 * dm; }

// 1 / row sum: a sum of NaN stays NaN; an empty unit's gives zeros.
__device__ __forceinline__ float row_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

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
    static constexpr size_t kScaleBytes = size_t(NW) * STAGES * MT * sizeof(float2);
    static constexpr size_t kFlagOffset = kScaleOffset + kScaleBytes;
    static constexpr size_t kMetaOffset = kFlagOffset + 16 * sizeof(int);
    static constexpr size_t kMetaBytes = (2 * kPersistMaxBatch + 1 + 16) * sizeof(int);
    // +1024: the rings are realigned to 1024 bytes (the swizzle's period).
    static constexpr size_t kBytes = 1024 + kMetaOffset + kMetaBytes;
    static_assert(kStepBytes % 1024 == 0 && kScaleOffset % 8 == 0, "alignment");
    // kv8_merge reuses the exchange area: weights [threads] + 2 x heads
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

    __device__ __forceinline__ void load(const __half* q, int gcount, int lane) {
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

    __device__ __forceinline__ void init(const Kv8DecodeParams& p, const TileCursor& start,
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
    __device__ __forceinline__ void look_up(const Kv8DecodeParams& p, const int* lens, int warp) {
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
    __device__ __forceinline__ void copy(const Kv8DecodeParams& p, uint32_t kst, uint32_t vst,
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
    __device__ __forceinline__ void advance(const int* seq_start, int B, int upb) {
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

// Merges `count` pieces of a unit: those of contributors first, first +
// stride, ... (CTA c's slot is 2c, or 2c + 1 for the first one when the unit
// is not its first item).  dst_slot < 0: into the fp16 output of the unit's
// gcount heads; else into that slot, as one piece (it may be a source).
// Pieces lie in the consumers' fragment order, [dm][nt][lane] float4 and
// (m, l) per head, so every thread folds whole 16-byte fragments.  In chunks
// of KW = threads / GP pieces: the first pieces' fragments are requested,
// thread (head, piece) loads (m, l) meanwhile, the KW lanes of a head form the
// maximum and the weights 2^(m_u - m); then FMAs only.  The order of the sums
// is that of the pieces, whoever merges.  All threads take part.
template <int D, int NT, int NW>
__device__ __forceinline__ void kv8_merge(const Kv8DecodeParams& p, float* area, int first,
                                          bool first_tail, int stride, int count, int gcount,
                                          size_t head_base, int dst_slot) {
    constexpr int GP = NT * 8;
    constexpr int NTHR = NW * 32;
    constexpr int KW = NTHR / GP;
    constexpr int NFRAG = (D / 16) * NT * 32;
    constexpr int FPT = NFRAG / NTHR;                     // fragments per thread
    constexpr int UB = 16 / FPT;                          // pieces per load batch
    static_assert(NFRAG % NTHR == 0 && KW <= 32 && 32 % KW == 0, "merge thread layout");
    float* sm_w = area;                                   // [KW][GP] chunk weights
    float* sm_r = sm_w + KW * GP;                         // [GP] rescale of the running state
    float* sm_inv = sm_r + GP;                            // [GP] 1 / row sum
    const int tid = threadIdx.x;
    const int wh = tid / KW, wu = tid - wh * KW;
    float mrun = -INFINITY, lrun = 0.f;
    float4 acc[FPT];
    int ha[FPT];                                          // first head of the fragment
#pragma unroll
    for (int i = 0; i < FPT; ++i) {
        acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int f = tid + i * NTHR;
        ha[i] = ((f >> 5) % NT) * 8 + 2 * (f & 3);
    }
    auto slot_of = [&](int k) { return 2 * (first + k * stride) + (k == 0 && first_tail ? 1 : 0); };
    for (int c0 = 0; c0 < count; c0 += KW) {
        const int kc = min(KW, count - c0);
        float4 v[FPT][UB];
        auto load_batch = [&](int u0) {
#pragma unroll
            for (int i = 0; i < FPT; ++i)
#pragma unroll
                for (int u = 0; u < UB; ++u) {
                    const float4* src = reinterpret_cast<const float4*>(
                        p.part_acc + (size_t)slot_of(c0 + u0 + u) * GP * D) + tid + i * NTHR;
                    v[i][u] = u0 + u < kc ? __ldcg(src) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
        };
        __syncthreads();                                  // the previous chunk's weights are used
        load_batch(0);
        float m = -INFINITY, l = 0.f;
        if (wu < kc) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml) +
                                     (size_t)slot_of(c0 + wu) * GP + wh);
            m = ml.x;
            l = ml.y;
        }
        float mx = m;
#pragma unroll
        for (int o = 1; o < KW; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mnew = fmaxf(mrun, mx);
        const float muse = (mnew == -INFINITY) ? 0.f : mnew;
        const float w = fast_exp2(m - muse);              // 0 for an empty piece (m = -inf)
        const float r = fast_exp2(mrun - muse);
        float ls = l * w;
#pragma unroll
        for (int o = 1; o < KW; o <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, o);
        lrun = fmaf(lrun, r, ls);
        mrun = mnew;
        sm_w[wu * GP + wh] = w;
        if (wu == 0) {
            sm_r[wh] = r;
            sm_inv[wh] = row_inverse(lrun);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < FPT; ++i) {
            const float r0 = sm_r[ha[i]], r1 = sm_r[ha[i] + 1];
            acc[i].x *= r0; acc[i].y *= r1; acc[i].z *= r0; acc[i].w *= r1;
        }
        for (int u0 = 0; u0 < kc; u0 += UB) {
            if (u0 > 0) load_batch(u0);
#pragma unroll
            for (int i = 0; i < FPT; ++i)
#pragma unroll
                for (int u = 0; u < UB; ++u) {
                    if (u0 + u < kc) {
                        const float w0 = sm_w[(u0 + u) * GP + ha[i]];
                        const float w1 = sm_w[(u0 + u) * GP + ha[i] + 1];
                        acc[i].x = fmaf(v[i][u].x, w0, acc[i].x);
                        acc[i].y = fmaf(v[i][u].y, w1, acc[i].y);
                        acc[i].z = fmaf(v[i][u].z, w0, acc[i].z);
                        acc[i].w = fmaf(v[i][u].w, w1, acc[i].w);
                    }
                }
        }
    }
    if (dst_slot >= 0) {
#pragma unroll
        for (int i = 0; i < FPT; ++i)
            reinterpret_cast<float4*>(p.part_acc + (size_t)dst_slot * GP * D)[tid + i * NTHR] = acc[i];
        if (wu == 0)
            reinterpret_cast<float2*>(p.part_ml)[(size_t)dst_slot * GP + wh] = make_float2(mrun, lrun);
        return;
    }
#pragma unroll
    for (int i = 0; i < FPT; ++i) {
        const int f = tid + i * NTHR;
        const int dim = kv_dim<D>(f / (32 * NT), (f & 31) >> 2);
        const int h = ha[i];
        if (h < gcount)
            *reinterpret_cast<uint32_t*>(p.out + (head_base + h) * D + dim) =
                pack_half2(acc[i].x * sm_inv[h], acc[i].z * sm_inv[h]);
        if (h + 1 < gcount)
            *reinterpret_cast<uint32_t*>(p.out + (head_base + h + 1) * D + dim) =
                pack_half2(acc[i].y * sm_inv[h + 1], acc[i].w * sm_inv[h + 1]);
    }
}

// ---------------------------------------------------------------------------
// Persistent kernel: grid = C co-resident CTAs of NW warps; see
// persistent_decode_kernel for units, items, pieces and the merge.
// ---------------------------------------------------------------------------
template <int D, int NT, int MT, int STAGES, int NW, int CTAS, bool REST, class Code>
__global__ void __launch_bounds__(32 * NW, CTAS)
kv8_decode_kernel(const __grid_constant__ Kv8DecodeParams p) {
    constexpr int TILE = 16 * MT * NW;
    using S = Kv8Smem<D, NT, MT, STAGES, NW>;
    constexpr int GP = NT * 8;
    constexpr int DTILES = D / 16;
    constexpr int XF = S::kXFloats;

    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    float* xarea = reinterpret_cast<float*>(smem + S::kXOffset);
    int* xflag = reinterpret_cast<int*>(smem + S::kFlagOffset);
    int* seq_start = reinterpret_cast<int*>(smem + S::kMetaOffset);
    int* lens = seq_start + kPersistMaxBatch + 1;
    int* warp_sums = lens + kPersistMaxBatch;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int B = p.batch;
    const int hg = p.head_groups;
    const int upb = p.cache.Hkv * hg;

    grid_launch_dependents();
    grid_dependency_wait();
    scan_lengths<TILE>(p.kv_lens, B, upb, seq_start, lens, warp_sums, p.max_len);

    const int T = seq_start[B];
    ShareMap sm{seq_start, B, upb, p.item_cost, p.merge_cost, p.whole_tiles, 0, 0, 0};
    const int Ctot = T + B * upb * (sm.xc + sm.mc);
    int C = min((int)gridDim.x, T);
    if (p.min_tiles_per_cta > 0) C = min(C, max(p.min_ctas, T / p.min_tiles_per_cta));
    // No tile of a unit that may be cut spans as many points as a share has, so
    // every CTA from a cut unit's first to its last holds a piece of it.
    sm.split(Ctot, max(1, min(C, Ctot / (max(sm.xc, sm.mc) + 1))));
    if (blockIdx.x >= sm.C) return;
    const int beg = sm.beg(blockIdx.x);
    const int end = sm.beg(blockIdx.x + 1);
    const int n = end - beg;
    if (n == 0) return;                         // its share lies within a unit that another took whole

    TileCursor cur;
    cur.seek(seq_start, B, upb, beg);
    int* xm = xflag + 2;
    if (threadIdx.x == 32 * NW - 1) {
        const TileCursor start = cur;
        TileCursor lc;
        lc.seek(seq_start, B, upb, end - 1);
        const bool one = start.b == lc.b && start.j == lc.j;
        auto note = [&](int r, int bb, int jj, int nbb, bool shared) {
            int* m = xm + 6 * r;
            m[0] = shared ? bb * upb + jj : -1;
            if (!shared) return;
            m[1] = sm.cta_of(bb, jj, nbb, 0);
            m[2] = sm.cta_of(bb, jj, nbb, nbb - 1);
            m[3] = sm.beg(m[1]) < seq_start[bb] + jj * nbb ? 1 : 0;
            m[4] = bb;
            m[5] = jj;
        };
        note(0, start.b, start.j, start.nb,
             one ? !(start.i == 0 && lc.i == lc.nb - 1) : start.i != 0);
        note(1, lc.b, lc.j, lc.nb, !one && lc.i != lc.nb - 1);
    }

    // This warp's ring, and its first STAGES - 1 steps.
    const uint64_t policy = l2_policy_evict_first();
    const uint32_t ring = smem_u32(smem) + warp * S::kWarpBytes;
    float2* scales = reinterpret_cast<float2*>(smem + S::kScaleOffset) + warp * (STAGES * MT);
    const uint32_t scales_s = smem_u32(scales);
    Kv8Loader<D, MT, NW> load;
    load.init(p, cur, lens, warp, lane);
    int ls = 0, lk = 0;                         // stage and step of the next copies
    auto start_step = [&]() {
        if (lk < n) {
            const uint32_t kst = ring + ls * (2 * S::kStepBytes);
            load.copy(p, kst, kst + S::kStepBytes, scales_s + ls * (MT * 8), 
                      hg == 1 ? load.cur.j : load.cur.j / hg, lane, policy);
            load.advance(seq_start, B, upb);
            if (++lk < n) load.look_up(p, lens, warp);
            ls = ls + 1 == STAGES ? 0 : ls + 1;
        }
        cp_async_commit();                      // an empty group past the end: the count goes on
    };
#pragma unroll
    for (int k = 0; k < STAGES - 1; ++k) start_step();

    const int g = lane >> 2;
    const int t = lane & 3;
    const float sl2 = p.scale_log2;
    int k = 0, stage = 0;
    for (int e = 0; k < n; ++e) {
        const int b = cur.b, j = cur.j, nb = cur.nb, i0 = cur.i;
        const int cnt = min(nb - i0, n - k);
        const int kvh = j / hg, hgrp = j - (j / hg) * hg;
        const int h0 = kvh * p.G + hgrp * GP;
        const int gcount = min(GP, p.G - hgrp * GP);
        const int len = lens[b];
        const size_t head_base = (size_t)b * p.H + h0;

        Kv8Query<D, NT> q;
        q.load(p.q + (size_t)b * p.q_stride + (size_t)h0 * D, gcount, lane);
        Kv8State<D, NT> st;
        st.clear();
        for (int tt = 0; tt < cnt; ++tt, ++k) {
            __syncwarp();                       // the stage refilled now is read by every lane
            start_step();
            cp_async_wait<STAGES - 1>();
            __syncwarp();                       // every lane's copies have landed
            const uint32_t kst = ring + stage * (2 * S::kStepBytes);
            const int valid = len - ((i0 + tt) * NW + warp) * (16 * MT);
            if (valid > 0)
                consume_kv8<D, NT, MT, REST, Code>(kst, kst + S::kStepBytes, scales + stage * MT, valid, q,
                                                   st, sl2, lane);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        cur.advance(seq_start, B, upb, cnt);

        st.finish();
        // ---- cross-warp fold: pairs of warps onto warps 0 and 1, then 1 onto 0
        static_assert(NW >= 4 && NW % 2 == 0, "the fold goes by pairs");
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int from = 2; from < NW; from += 2) {
                if (warp >= from && warp < from + 2)
                    x_store<D, NT>(xarea + ((warp - from) * 32 + lane) * XF, st.o, st.m, st.l, nt);
                __syncthreads();
                if (warp < 2) x_fold<D, NT>(xarea + (warp * 32 + lane) * XF, st.o, st.m, st.l, nt);
                __syncthreads();
            }
            if (warp == 1) x_store<D, NT>(xarea + lane * XF, st.o, st.m, st.l, nt);
            __syncthreads();
            if (warp == 0) x_fold<D, NT>(xarea + lane * XF, st.o, st.m, st.l, nt);
            __syncthreads();
        }

        // ---- output of the item
        const bool whole = i0 == 0 && cnt == nb;
        if (whole) {
            if (warp == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) {
                        const int hj = nt * 8 + 2 * t + jj;
                        const float inv = row_inverse(st.l[nt][jj]);
                        if (hj < gcount) {
                            __half* dst = p.out + (head_base + hj) * D + (D / 8) * g;
#pragma unroll
                            for (int dm = 0; dm < DTILES; dm += 4) {
                                uint32_t h[4];
#pragma unroll
                                for (int x = 0; x < 4; ++x)
                                    h[x] = pack_half2(st.o[dm + x][nt][jj] * inv, st.o[dm + x][nt][jj + 2] * inv);
                                *reinterpret_cast<uint4*>(dst + dm * 2) = make_uint4(h[0], h[1], h[2], h[3]);
                            }
                        }
                    }
            }
            continue;
        }
        if (warp == 0) {
            const int slot = 2 * blockIdx.x + (e == 0 ? 0 : 1);
            float4* pa = reinterpret_cast<float4*>(p.part_acc + (size_t)slot * GP * D);
            float* pm = p.part_ml + (size_t)slot * GP * 2;
#pragma unroll
            for (int dm = 0; dm < DTILES; ++dm)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    pa[(dm * NT + nt) * 32 + lane] =
                        make_float4(st.o[dm][nt][0], st.o[dm][nt][1], st.o[dm][nt][2], st.o[dm][nt][3]);
            if (g == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) {
                        const int hj = nt * 8 + 2 * t + jj;
                        pm[hj * 2 + 0] = st.m[nt][jj];
                        pm[hj * 2 + 1] = st.l[nt][jj];
                    }
            }
        }
    }

    // ---- count the pieces and merge what this CTA completes.  A unit of more
    // than TWO pieces is merged in two levels: groups of GROUP contributors
    // into their first one's slot, then the groups (one CTA reading 148 pieces
    // took 12 us of a call of 45).  The last contributor to
    // count does a merge, so no CTA waits; each count releases the pieces
    // before it and the last one acquires them.
    constexpr int GROUP = 16, TWO = 32;
    int* group_counters = p.counters + p.max_units;      // one per slot
    if (warp == 0) {
        __syncwarp();
        if (lane < 2) {
            const int* m = xm + 6 * lane;
            int f = 0;
            if (m[0] >= 0) {
                const int pieces = m[2] - m[1] + 1;
                int* counter = &p.counters[m[0]];
                int need = pieces;
                if (pieces > TWO) {
                    const int lead = ((int)blockIdx.x - m[1]) / GROUP * GROUP;
                    need = min(GROUP, pieces - lead);
                    counter = &group_counters[2 * (m[1] + lead) + (lead == 0 && m[3] ? 1 : 0)];
                }
                f = atom_add_release_gpu(counter, 1) == need - 1;
                if (f) fence_acq_rel_gpu();
            }
            xflag[lane] = f;
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int r = 0; r < 2; ++r) {
        if (!xflag[r]) continue;                          // uniform over the CTA
        const int* m = xm + 6 * r;
        const int cf = m[1], pieces = m[2] - m[1] + 1, bb = m[4], jj = m[5];
        const int kvh = jj / hg, hgrp = jj - (jj / hg) * hg;
        const int gcount = min(GP, p.G - hgrp * GP);
        const size_t head_base = (size_t)bb * p.H + kvh * p.G + hgrp * GP;
        int stride = 1, count = pieces;
        if (pieces > TWO) {
            const int lead = ((int)blockIdx.x - cf) / GROUP * GROUP;
            const bool tail = lead == 0 && m[3] != 0;
            const int slot = 2 * (cf + lead) + (tail ? 1 : 0);
            kv8_merge<D, NT, NW>(p, xarea, cf + lead, tail, 1, min(GROUP, pieces - lead), gcount,
                                 head_base, slot);
            stride = GROUP;
            count = (pieces + GROUP - 1) / GROUP;
            __syncthreads();                              // the group's piece is stored
            if (threadIdx.x == 0) {
                group_counters[slot] = 0;
                const int f = atom_add_release_gpu(&p.counters[m[0]], 1) == count - 1;
                if (f) fence_acq_rel_gpu();
                xflag[r] = f;
            }
            __syncthreads();
            if (!xflag[r]) continue;
        }
        kv8_merge<D, NT, NW>(p, xarea, cf, m[3] != 0, stride, count, gcount, head_base, -1);
        if (threadIdx.x == 0) p.counters[m[0]] = 0;       // every piece was counted: re-arm
    }
}

}  // namespace fr
