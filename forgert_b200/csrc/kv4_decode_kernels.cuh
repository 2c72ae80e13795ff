// kv4_decode_kernels.cuh - single-token attention over the 4-bit paged cache.
//
// Mathematics, per (sequence, query head h of kv head j), positions t < len,
// groups g of 64 dims with codes n, K's (a, b) and V's (a', b') as scale, bias:
//   s_t = sum_g a_tg (q_g . n_tg) + b_tg (q_g . 1),  in units of 1 / sqrt(D)
//   p_t = 2^(s_t log2 e - r),  l = sum_t p_t,  mid_tg = b'_tg + 8 a'_tg
//   o_g = sum_t (p_t a'_tg) (n'_tg - 8) + sum_t p_t mid_tg,  out = o / l
// (zeros for an empty sequence).  Codes enter the products as they are: the
// fp16 with bits n is n 2^-24 exactly, so a mask makes two operands of a word,
// n of the low halves and 16 n of the high ones, and the factors are taken off
// the sums.  8 times the sum of the weights goes into a sum of its own by a
// product with a constant operand (z), so that what rounding a weight to fp16
// takes off counts by the distance from the group's middle, not from its
// bottom (half the error).  Scores, l, o and all other sums are fp32.
//
// A weight p a' enters the product with V as fp16 on a reference of its own
// group's (r_g), 2^8 up, so that one as small as 2^-22 of the largest keeps all
// its bits; REST adds a second product with what the rounding takes off (short
// calls, where the outputs average fewer terms).  l and the middles are on the
// first group's reference, in fp32 from unrounded p.
//
// Bytes: D of codes per position and kv head, D / 8 of scales; 4 * D * G
// operations on them.
//
// Fragments (mma m16n8k16), without ldmatrix: of K a lane holds 16 dims of each
// group in two rows, of V eight dims (one word) of each group in four rows;
// contraction order is free, so q is permuted to the order that masks bring K's
// codes in (Kv4Query), and V's rows are paired by byte permutations.  Row i of a
// block's fragments is row pos_of(i): rows two and four apart then differ mod 4,
// which with the chunks exchanged by row (kv4_offset) keeps all loads from
// shared memory free of bank conflicts.
#pragma once
#include "cached_decode_kernels.cuh"
#include "kv4_common.cuh"

namespace fr {

constexpr float kKv4Shift = 8.f;        // a weight at its reference counts 2^8 ...
constexpr float kKv4Top = 15.f;         // ... and may grow to 2^15 before that moves (fp16: < 2^16)
constexpr float kKv4Least = -24.f;      // a smaller scale's reference is this scale's: p stays below 2^39
constexpr uint32_t kLowHalves = 0x000f000fu, kHighHalves = 0x00f000f0u;

__device__ __forceinline__ int kv4_pos_of(int i) { return i ^ ((i >> 2) & 1); }

// Byte offset of byte b of row r in a step's K or V.
template <int D>
__device__ __forceinline__ uint32_t kv4_offset(int r, int b) {
    return D == 128 ? uint32_t(r * 64 + (b ^ ((r & 2) << 4))) : uint32_t(r * 32 + b);
}

template <int D, int NT, int MT, int STAGES, int NW>
struct Kv4Smem {
    static constexpr int kStepBytes = 16 * MT * (D / 2);                // K (or V) of one step
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
    static_assert(kStepBytes % 128 == 0 && kScaleOffset % 16 == 0, "alignment");
    // cached_merge reuses the exchange area: weights [threads] + 2 x heads
    static_assert(kXBytes >= (NW * 32 + 2 * NT * 8) * sizeof(float), "merge area");
};

// q of one item as the B operand, in the order in which masks bring K's codes:
// of each word of eight dims 0, 4 and 2, 6 (low halves), 1, 5 and 3, 7 (high
// ones).  sum: of each group's elements of the heads 2t, 2t + 1, times 2^-24.
template <int D, int NT>
struct Kv4Query {
    static constexpr int NG = D / kKv4Group;
    uint32_t b[NG][2][2][NT][2];                // group, word, low / high, tile of heads
    float sum[NG][NT][2];

    __device__ __forceinline__ void load(const __half* q, int gcount, int lane) {
        const int g = lane >> 2, t = lane & 3;
        constexpr uint32_t kOnes = 0x3c003c00u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int hj = nt * 8 + g;
            const __half* row = q + (size_t)hj * D + 16 * t;
#pragma unroll
            for (int x = 0; x < NG; ++x) {
                float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (hj < gcount) v = *reinterpret_cast<const uint4*>(row + x * kKv4Group + w * 8);
                    b[x][w][0][nt][0] = __byte_perm(v.x, v.z, 0x5410);
                    b[x][w][0][nt][1] = __byte_perm(v.y, v.w, 0x5410);
                    b[x][w][1][nt][0] = __byte_perm(v.x, v.z, 0x7632);
                    b[x][w][1][nt][1] = __byte_perm(v.y, v.w, 0x7632);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        mma_16816(s, kOnes, kOnes, kOnes, kOnes, b[x][w][e][nt][0], b[x][w][e][nt][1]);
                }
                sum[x][nt][0] = s[0] * 0x1p-24f;
                sum[x][nt][1] = s[1] * 0x1p-24f;
            }
        }
    }
};

// Running state of a warp over an item, per head column.  r[g] is the reference
// of group g's weights, in base 2 and a whole number; f = 2^(r[0] - r[g]).
// o, z: products with V's codes and with 8, in units of 2^-24; mid: this lane's
// rows' part of sum p mid, l that of the row sum, both on r[0].
template <int D, int NT>
struct Kv4State {
    static constexpr int NG = D / kKv4Group;
    float o[D / 16][NT][4], z[NG][NT][4];
    float mid[NG][NT][2], l[NT][2];
    float r[NG][NT][2], f[NG][NT][2];
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
            for (int x = 0; x < NG; ++x) {
#pragma unroll
                for (int c = 0; c < 4; ++c) z[x][nt][c] = 0.f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    mid[x][nt][j] = r[x][nt][j] = 0.f;
                    f[x][nt][j] = 1.f;
                }
            }
            l[nt][0] = l[nt][1] = 0.f;
        }
        fresh = true;
    }
    // Sums over the warp's rows, o whole and on r[0]: the (m, l, o) of the merges.
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
                m[nt][j] = fresh ? -INFINITY : r[0][nt][j];
#pragma unroll
                for (int x = 0; x < NG; ++x) {
                    const float c = rows(mid[x][nt][j]);
                    const float u = 0x1p24f * fast_exp2(r[x][nt][j] - r[0][nt][j]);
#pragma unroll
                    for (int dm = 4 * x; dm < 4 * x + 4; ++dm) {
                        o[dm][nt][j] = fmaf(o[dm][nt][j] - z[x][nt][j], u, c);
                        o[dm][nt][j + 2] = fmaf(fmaf(o[dm][nt][j + 2], 0.0625f, -z[x][nt][j]), u, c);
                    }
                }
            }
    }
};

// One step: 16 * MT rows of K at kst and V at vst, of which the first `valid`
// (>= 1) are positions; sc: their scales.
template <int D, int NT, int MT, bool REST>
__device__ __forceinline__ void consume_kv4(uint32_t kst, uint32_t vst, uint32_t sc, int valid,
                                            const Kv4Query<D, NT>& q, Kv4State<D, NT>& st,
                                            float sl2, int lane) {
    constexpr int NG = D / kKv4Group;
    const int g = lane >> 2, t = lane & 3;
    const int rg = kv4_pos_of(g);               // rows of the A fragments: rg, rg + 8
    const bool tail = valid < 16 * MT;          // uniform over the warp
    const float unit = sl2 * 0x1p24f;

    // ---- scores (times 2^-24), and V's scales and middles of the lane's rows
    float s[MT][NT][4];
    float va[MT][2][NG], vm[MT][2][NG];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float ka[2][NG], kb[2][NG];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = mt * 16 + rg + 8 * i;
            uint32_t w[2 * NG];                 // K's groups, V's groups
            if constexpr (NG == 2) {
                const uint4 x = lds128(sc + row * 16);
                w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            } else {
                const uint2 x = lds64(sc + row * 8);
                w[0] = x.x; w[1] = x.y;
            }
            // What rows past the end hold is anything, a NaN included.
            if (tail && row >= valid) {
#pragma unroll
                for (int x = 0; x < NG; ++x) w[NG + x] = 0u;
            }
#pragma unroll
            for (int x = 0; x < NG; ++x) {
                const float2 kp = __half22float2(*reinterpret_cast<const __half2*>(&w[x]));
                const float2 vp = __half22float2(*reinterpret_cast<const __half2*>(&w[NG + x]));
                ka[i][x] = kp.x;
                kb[i][x] = kp.y;
                va[mt][i][x] = vp.x;
                vm[mt][i][x] = fmaf(8.f, vp.x, vp.y);
            }
        }
        float d[NG][2][NT][4];                  // q . n of the low halves, 16 q . n of the high ones
#pragma unroll
        for (int x = 0; x < NG; ++x) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c) d[x][e][nt][c] = 0.f;
            const int at = x * (kKv4Group / 2) + 8 * t;
            const uint2 lo = lds64(kst + kv4_offset<D>(mt * 16 + rg, at));
            const uint2 hi = lds64(kst + kv4_offset<D>(mt * 16 + rg + 8, at));
            const uint32_t xs[2] = {lo.x, lo.y}, ys[2] = {hi.x, hi.y};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint32_t x8 = xs[w] >> 8, y8 = ys[w] >> 8;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t mask = e ? kHighHalves : kLowHalves;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_16816(d[x][e][nt], xs[w] & mask, ys[w] & mask, x8 & mask, y8 & mask,
                                  q.b[x][w][e][nt][0], q.b[x][w][e][nt][1]);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int i = c >> 1, j = c & 1;
                float sum = 0.f;
#pragma unroll
                for (int x = 0; x < NG; ++x) {
                    sum = fmaf(kb[i][x], q.sum[x][nt][j], sum);
                    sum = fmaf(ka[i][x], fmaf(d[x][1][nt][c], 0.0625f, d[x][0][nt][c]), sum);
                }
                s[mt][nt][c] = sum;
                if (tail && mt * 16 + rg + 8 * i >= valid) s[mt][nt][c] = -INFINITY;
            }
    }

    // ---- probabilities and weights on the references as they are
    float p[MT][NT][4], w[MT][NG][NT][4];
    bool over = false;
    auto weigh = [&]() {
        float top_p = 0.f, top_w = 0.f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float pc = fast_exp2(fmaf(s[mt][nt][c], unit, -st.r[0][nt][c & 1]));
                    p[mt][nt][c] = pc;
                    top_p = fmaxf(top_p, pc);
#pragma unroll
                    for (int x = 0; x < NG; ++x) {
                        const float wc = (x ? pc * st.f[x][nt][c & 1] : pc) * va[mt][c >> 1][x];
                        w[mt][x][nt][c] = wc;
                        top_w = fmaxf(top_w, wc);
                    }
                }
        over = top_w > 0x1p15f || top_p > 0x1p39f;
    };
    weigh();
    if (__any_sync(0xffffffffu, over || st.fresh)) {
        // Move the references that a weight has outgrown to the weights' maxima
        // and rescale what is summed so far.  A column and group moves for its
        // own weights only: no head's bits depend on another's.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int x = 0; x < NG; ++x) {
                    const float r0 = st.r[x][nt][j];
                    float top = -INFINITY;      // log2 of the largest weight on r0
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            top = fmaxf(top, fmaf(s[mt][nt][2 * i + j], unit, -r0) +
                                                 fmaxf(fast_log2(va[mt][i][x]), kKv4Least));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1)
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const bool move = st.fresh ? top > -INFINITY : top > kKv4Top;
                    const float by = move ? rintf(top - kKv4Shift) : 0.f;
                    st.r[x][nt][j] = r0 + by;
                    // without a reference the sums are 0
                    const float u = st.fresh || !move ? 1.f : fast_exp2(-by);
#pragma unroll
                    for (int dm = 4 * x; dm < 4 * x + 4; ++dm) {
                        st.o[dm][nt][j] *= u;
                        st.o[dm][nt][j + 2] *= u;
                    }
                    st.z[x][nt][j] *= u;
                    if (x == 0) {
                        st.l[nt][j] *= u;
#pragma unroll
                        for (int y = 0; y < NG; ++y) st.mid[y][nt][j] *= u;
                    }
                    st.f[x][nt][j] = fast_exp2(st.r[0][nt][j] - st.r[x][nt][j]);
                }
            }
        st.fresh = false;
        weigh();
    }

    // ---- row sums and middles (unrounded p); W^T = P^T a' as fp16 in the B
    // layout (k = position, n = head)
    uint32_t wb[MT][NG][NT][2], wr[MT][NG][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                st.l[nt][c & 1] += p[mt][nt][c];
#pragma unroll
                for (int x = 0; x < NG; ++x)
                    st.mid[x][nt][c & 1] = fmaf(p[mt][nt][c], vm[mt][c >> 1][x], st.mid[x][nt][c & 1]);
            }
#pragma unroll
            for (int x = 0; x < NG; ++x)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float w0 = w[mt][x][nt][2 * e], w1 = w[mt][x][nt][2 * e + 1];
                    const uint32_t h = pack_half2(w0, w1);
                    wb[mt][x][nt][e] = movmatrix_trans(h);
                    if constexpr (REST) {
                        const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&h));
                        wr[mt][x][nt][e] = movmatrix_trans(pack_half2(w0 - r.x, w1 - r.y));
                    }
                }
        }

    // ---- O^T += V^T W^T, and z
    const int p0 = kv4_pos_of(2 * t), p1 = kv4_pos_of(2 * t + 1);
    constexpr uint32_t kEight = 0x00080008u;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int x = 0; x < NG; ++x) {
            const int at = x * (kKv4Group / 2) + 4 * g;
            uint32_t v[4];                      // rows p0, p1, p0 + 8, p1 + 8
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = lds32(vst + kv4_offset<D>(mt * 16 + (i & 1 ? p1 : p0) + (i >> 1) * 8, at));
            auto product = [&](float (&acc)[NT][4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_16816(acc[nt], a0, a1, a2, a3, wb[mt][x][nt][0], wb[mt][x][nt][1]);
                if constexpr (REST) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_16816(acc[nt], a0, a1, a2, a3, wr[mt][x][nt][0], wr[mt][x][nt][1]);
                }
            };
            product(st.z[x], kEight, kEight, kEight, kEight);
#pragma unroll
            for (int e = 0; e < 2; ++e) {       // dims 4e .. 4e + 3 of the lane's eight
                const uint32_t lo = __byte_perm(v[0], v[1], e ? 0x7632 : 0x5410);
                const uint32_t hi = __byte_perm(v[2], v[3], e ? 0x7632 : 0x5410);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint32_t l8 = y ? lo >> 8 : lo, h8 = y ? hi >> 8 : hi;
                    product(st.o[4 * x + 2 * e + y], l8 & kLowHalves, l8 & kHighHalves,
                            h8 & kLowHalves, h8 & kHighHalves);
                }
            }
        }
}

// Where a warp's copies are: the tile of its cursor and, looked up already,
// the pages of the warp's MT blocks of it (-1 where there is no position,
// num_pages for an id outside the pool).  The page index and the block within
// the page go along with the cursor, without divisions.
template <int D, int MT, int NW>
struct Kv4Loader {
    static constexpr int CPR = D / 32;          // 16-byte chunks per row
    static constexpr int RPC = 32 / CPR;        // rows per warp-wide copy
    static constexpr int kBlock = 16;
    static constexpr int kRowScales = 8 * (D / kKv4Group);
    TileCursor cur;
    int idx, sub;                               // page index and block within it, first block
    int bpp, step_idx, step_sub, idx0, sub0;    // blocks per page; NW * MT blocks; tile 0
    int page[MT];
    long long lane_off;

    __device__ __forceinline__ void init(const CachedDecodeParams<Kv4View>& p, const TileCursor& start,
                                         const int* lens, int warp, int lane) {
        cur = start;
        bpp = p.cache.page_size / kBlock;
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
    __device__ __forceinline__ void look_up(const CachedDecodeParams<Kv4View>& p, const int* lens,
                                            int warp) {
        const int pos = (cur.i * NW + warp) * (kBlock * MT);
        const int left = cur.b < p.batch ? lens[cur.b] - pos : 0;
        const int* row = p.block_table + (size_t)cur.b * p.bt_stride;
        int at = idx, s = sub;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            page[m] = -1;
            if (kBlock * m < left) page[m] = min((unsigned)row[at], (unsigned)p.cache.num_pages);
            if (++s == bpp) { s = 0; ++at; }
        }
    }
    // Starts the copies of the step: 16 rows of K and of V and their scales of
    // each block that holds positions; zeros for a page outside the pool.
    __device__ __forceinline__ void copy(const CachedDecodeParams<Kv4View>& p, uint32_t kst, uint32_t vst,
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
                                      s * kBlock * p.cache.row_stride + lane_off;
                const uint8_t* ks = p.cache.k + off;
                const uint8_t* vs = p.cache.v + off;
#pragma unroll
                for (int i = 0; i < kBlock / RPC; ++i) {
                    const uint32_t dst = kv4_offset<D>(m * kBlock + i * RPC + r0, c * 16);
                    cp_async_16(kst + dst, ks, bytes, policy);
                    cp_async_16(vst + dst, vs, bytes, policy);
                    ks += RPC * p.cache.row_stride;
                    vs += RPC * p.cache.row_stride;
                }
                if (lane < kRowScales)          // 16 rows of kRowScales bytes, 16 a lane
                    cp_async_16(scale_at + m * (kBlock * kRowScales) + lane * 16,
                                reinterpret_cast<const char*>(
                                    p.cache.pairs<D>(pg, kvh, s * kBlock)) + lane * 16,
                                bytes, policy);
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

// Steps of MT blocks of 16 rows; CTAS per SM; REST as above.
template <int D, int NT, int MT, int STAGES, int NW, int CTAS, bool REST>
struct Kv4Format {
    static constexpr int kD = D, kNT = NT, kMT = MT, kStages = STAGES, kNW = NW, kCtas = CTAS;
    using Params = CachedDecodeParams<Kv4View>;
    using Smem = Kv4Smem<D, NT, MT, STAGES, NW>;
    using Loader = Kv4Loader<D, MT, NW>;
    using Query = Kv4Query<D, NT>;
    using State = Kv4State<D, NT>;

    static __device__ __forceinline__ int dim(int dm, int g) {
        return (dm >> 2) * kKv4Group + 8 * g + 2 * (dm & 3);
    }
    static __device__ __forceinline__ void consume(uint32_t kst, uint32_t vst, const unsigned char* sc,
                                                   int valid, const Query& q, State& st, float sl2,
                                                   int lane) {
        consume_kv4<D, NT, MT, REST>(kst, vst, smem_u32(sc), valid, q, st, sl2, lane);
    }
};

}  // namespace fr
