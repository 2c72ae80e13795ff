// kv8_decode_kernels.cuh - single-token attention over the 8-bit paged cache.
//
// Mathematics, per (sequence, query head h of kv head j), positions t < len
// in blocks of 16:
//   s_t = (q . kc_t) * kscale(block) / sqrt(D)
//   o   = sum_t 2^(s_t log2 e - m) * vscale(block) * vc_t,  l = sum_t 2^(...)
//   out = o / l  (zeros for an empty sequence)
// with kc, vc the 8-bit codes.  Scores, m, l and o are fp32.  Codes widen to
// fp16 exactly; the probability enters the P.V product as one fp16 (relative
// rounding 2^-12, below the output's own), shifted up by 2^15 so that one as
// small as 2^-29 of the largest keeps all its bits.  The row sum uses the
// unrounded probabilities.
//
// Bound: HBM.  2 * D bytes of codes per position and kv head, plus 8 bytes of
// scales per 16 positions; 4 * D * G operations on them.
//
// Decomposition: the persistent, cost-balanced ranges of batched_kernels.cuh
// (TileCursor, CostMap, pieces merged by the contributor that completes a
// unit), over tiles of TILE positions.  The producer warp is all at work: its
// lanes look up the pages of a tile's boxes (one tile ahead, so that the
// block table's latency is hidden), copy boxes of gcd(page_size, TILE) rows
// with TMA and the blocks' scales with 8-byte cp.async, all counted by the
// stage's full barrier.  Only boxes that hold positions are copied.
//
// Fragments: each consumer warp takes MT m-tiles of 16 rows.  The codes go
// from shared memory to the operands of mma m16n8k16 without ldmatrix:
// contraction order is free, so k-step w of a row is word w of the 16 bytes
// that a lane loads at once, and for P.V the words of two neighbouring rows
// are interleaved by one byte permutation.  A lane owns D/8 consecutive head
// dims of the output (KvDims).  All loads are 16 bytes (8 for V at D = 64)
// and free of bank conflicts under the swizzle; at D = 64 (two rows to a
// 128-byte line) that takes rows 2 and 3, 6 and 7 exchanged (pos_of).
#pragma once
#include "batched_kernels.cuh"
#include "kv8_common.cuh"

namespace fr {

struct Kv8DecodeParams {
    DecodeParams d;              // maps, q, lengths, block table, partials (see there)
    const float* scales;
    int blocks_per_page;
    int max_len;                 // lengths are cut to this
    long long q_stride;          // halves between the sequences' q
};

// Lane (g, t) of fragment dm holds dims (D/8)*g + 2*dm + {0, 1}.
template <int D>
struct KvDims {
    static __device__ __forceinline__ int dim(int dm, int g, int c) { return (D / 8) * g + 2 * dm + (c >> 1); }
    // A row sum of NaN stays NaN; an empty unit's is zero.
    static __device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
};

constexpr float kProbShift = 15.f;      // probabilities are held as 2^15 p

template <int D, int NT, int TILE, int STAGES, int NW>
struct Kv8Smem {
    static constexpr int kTileBytes = TILE * D;
    static constexpr size_t kRingBytes = size_t(2) * STAGES * kTileBytes;
    static constexpr int kXFloats = (D / 16) * 4 + 4;
    static constexpr size_t kXOffset = kRingBytes;
    static constexpr size_t kXBytes = size_t(NW / 2) * 32 * kXFloats * sizeof(float);
    static constexpr size_t kScaleOffset = kXOffset + kXBytes;
    static constexpr size_t kScaleBytes = size_t(STAGES) * (TILE / kKv8Block) * sizeof(float2);
    static constexpr size_t kBarOffset = kScaleOffset + kScaleBytes;
    static constexpr size_t kFlagOffset = kBarOffset + 2 * STAGES * sizeof(uint64_t);
    static constexpr size_t kMetaOffset = kFlagOffset + 16 * sizeof(int);
    static constexpr size_t kMetaBytes = (2 * kPersistMaxBatch + 1 + 16) * sizeof(int);
    static constexpr size_t kBytes = 1024 + kMetaOffset + kMetaBytes;
    static_assert(kTileBytes % 1024 == 0 && kBarOffset % 8 == 0, "alignment");
    // merge_pieces reuses the exchange area: weights [threads] + 2 x heads
    static_assert(kXBytes >= (NW * 32 + 2 * NT * 8) * sizeof(float), "merge area");
};

// Row of a 16-row m-tile that fragment row i stands for.
template <int D>
__device__ __forceinline__ int pos_of(int i) {
    return D == 64 ? i ^ ((i >> 1) & 1) : i;
}

// Byte offset of 16-byte chunk c of row r under the 128- or 64-byte swizzle.
template <int D>
__device__ __forceinline__ uint32_t kv8_offset(int r, int c) {
    return D == 128 ? uint32_t(r * 128 + ((c ^ (r & 7)) << 4))
                    : uint32_t(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// One consumer warp's rows row0 .. row0 + 16 * MT - 1 of a stage, of which
// the first `valid` (>= 1) are positions.  sc: the stage's scales from the
// warp's first block on.
template <int D, int NT, int MT, class Code>
__device__ __forceinline__ void consume_kv8(uint32_t kst, uint32_t vst, const float2* sc, int row0,
                                            int valid, const uint32_t (&qb)[D / 16][NT][2],
                                            float (&o)[D / 16][NT][4], float (&m_run)[NT][2],
                                            float (&l_run)[NT][2], float sl2, int lane) {
    constexpr int KL = D / 64;                  // 16-byte loads per K row and lane
    constexpr int VW = D / 32;                  // words per V row and lane
    const int g = lane >> 2, t = lane & 3;
    const int rg = pos_of<D>(g);                // rows of the A fragments: rg, rg + 8
    float2 scale[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        // a block without positions has no scale in the stage
        scale[mt] = mt * 16 < valid ? sc[mt] : make_float2(0.f, 0.f);
        // An infinite scale acts as NaN, as the sum of its rows' infinities of
        // both signs would, and not as one infinity of the sum's sign.
        scale[mt].x += scale[mt].x - scale[mt].x;
        scale[mt].y += scale[mt].y - scale[mt].y;
    }

    // ---- S^T = K Q^T
    float s[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[mt][nt][c] = 0.f;
        const int r = row0 + mt * 16 + rg;
#pragma unroll
        for (int j = 0; j < KL; ++j) {
            const int chunk = KL * t + j;
            const uint4 x = lds128(kst + kv8_offset<D>(r, chunk));
            const uint4 y = lds128(kst + kv8_offset<D>(r + 8, chunk));
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t xw = Code::prepare(xs[w]), yw = Code::prepare(ys[w]);
                const uint32_t a0 = Code::half2_lo(xw), a1 = Code::half2_lo(yw);
                const uint32_t a2 = Code::half2_hi(xw), a3 = Code::half2_hi(yw);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_16816(s[mt][nt], a0, a1, a2, a3, qb[j * 4 + w][nt][0], qb[j * 4 + w][nt][1]);
            }
        }
    }

    // ---- scale, mask, online softmax per head column (base 2)
    const bool tail = valid < 16 * MT;          // uniform over the warp
    uint32_t pb[MT][NT][2];
    bool grew = false;
    float alpha[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float ks = scale[mt].x * sl2;
#pragma unroll
            for (int c = 0; c < 4; ++c) s[mt][nt][c] *= ks;
            if (tail) {
                if (mt * 16 + rg >= valid) s[mt][nt][0] = s[mt][nt][1] = -INFINITY;
                if (mt * 16 + rg + 8 >= valid) s[mt][nt][2] = s[mt][nt][3] = -INFINITY;
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float mx = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mx = fmaxf(mx, fmaxf(s[mt][nt][j], s[mt][nt][j + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            // the state's maximum is kept kProbShift lower: 2^(s - m) = 2^15 p
            const float m_new = fmaxf(m_run[nt][j], mx - kProbShift);
            const float base = m_new == -INFINITY ? 0.f : m_new;
            grew |= m_new > m_run[nt][j];
            alpha[nt][j] = fast_exp2(m_run[nt][j] - base);
            m_run[nt][j] = m_new;
            float sum = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                s[mt][nt][j] = fast_exp2(s[mt][nt][j] - base);
                s[mt][nt][j + 2] = fast_exp2(s[mt][nt][j + 2] - base);
                sum += s[mt][nt][j] + s[mt][nt][j + 2];
            }
            l_run[nt][j] = fmaf(l_run[nt][j], alpha[nt][j], sum);
        }
        // P^T to the B layout (k = position, n = head)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            pb[mt][nt][0] = movmatrix_trans(pack_half2(s[mt][nt][0], s[mt][nt][1]));
            pb[mt][nt][1] = movmatrix_trans(pack_half2(s[mt][nt][2], s[mt][nt][3]));
        }
    }
    if (__any_sync(0xffffffffu, grew)) {        // the running maximum moved: rescale
#pragma unroll
        for (int dm = 0; dm < D / 16; ++dm)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                o[dm][nt][0] *= alpha[nt][0];
                o[dm][nt][1] *= alpha[nt][1];
                o[dm][nt][2] *= alpha[nt][0];
                o[dm][nt][3] *= alpha[nt][1];
            }
    }

    // ---- O^T += vscale * V^T P^T
    const int p0 = pos_of<D>(2 * t), p1 = pos_of<D>(2 * t + 1);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = row0 + mt * 16;
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
            // probability is 0, and 0 * NaN is not.
            if (Code::kHasNan && tail && mt * 16 + row >= valid) {
#pragma unroll
                for (int x = 0; x < VW; ++x) w[i][x] = 0;
            }
        }
        const float vs = scale[mt].y;
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
                for (int nt = 0; nt < NT; ++nt) {
                    float pv[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_16816(pv, a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[dm][nt][c] = fmaf(pv[c], vs, o[dm][nt][c]);
                }
            }
    }
}

// ---------------------------------------------------------------------------
// Persistent kernel: grid = C co-resident CTAs, block = 32 * (NW + 1); see
// persistent_decode_kernel for the ranges, items, pieces and the merge.
// ---------------------------------------------------------------------------
template <int D, int NT, int MT, int STAGES, int NW, int CTAS, class Code>
__global__ void __launch_bounds__(32 * (NW + 1), CTAS)
kv8_decode_kernel(const __grid_constant__ Kv8DecodeParams kp) {
    constexpr int TILE = 16 * MT * NW;
    using S = Kv8Smem<D, NT, TILE, STAGES, NW>;
    constexpr int GP = NT * 8;
    constexpr int DTILES = D / 16;
    constexpr int XF = S::kXFloats;
    constexpr int BLOCKS = TILE / kKv8Block;
    const DecodeParams& p = kp.d;

    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    unsigned char* kring = smem;
    unsigned char* vring = smem + STAGES * S::kTileBytes;
    float* xarea = reinterpret_cast<float*>(smem + S::kXOffset);
    float2* scales = reinterpret_cast<float2*>(smem + S::kScaleOffset);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBarOffset);
    uint64_t* empty = full + STAGES;
    int* xflag = reinterpret_cast<int*>(smem + S::kFlagOffset);
    int* seq_start = reinterpret_cast<int*>(smem + S::kMetaOffset);
    int* lens = seq_start + kPersistMaxBatch + 1;
    int* warp_sums = lens + kPersistMaxBatch;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int B = p.batch;
    const int hg = p.head_groups;
    const int upb = p.Hkv * hg;

    grid_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1 + 32);        // lane 0's byte count, 32 lanes' cp.async
            mbar_init(&empty[s], NW);
        }
        fence_mbar_init();
    }
    grid_dependency_wait();
    scan_lengths<TILE>(p.kv_lens, B, upb, seq_start, lens, warp_sums, kp.max_len);

    const long long T = seq_start[B];
    CostMap cm{seq_start, B, upb, p.item_cost, p.merge_cost, 0, 0};
    cm.Ctot = T + (long long)B * upb * (cm.xc + cm.mc);
    long long C = min((long long)gridDim.x, T);
    if (p.min_tiles_per_cta > 0)
        C = min(C, max((long long)p.min_ctas, T / p.min_tiles_per_cta));
    C = max(1LL, min(C, cm.Ctot / (cm.xc + cm.mc + 2)));
    cm.C = C;
    if (blockIdx.x >= C) return;
    const int beg = cm.beg(blockIdx.x);
    const int end = cm.beg(blockIdx.x + 1);
    const int n = end - beg;

    TileCursor start;
    start.seek(seq_start, B, upb, beg);

    if (warp == NW) {
        // -------------------------------------------------------- producer
        const uint64_t policy = p.evict_normal ? l2_policy_evict_normal() : l2_policy_evict_first();
        const int box = p.page_box, nbox = TILE / box;
        TileCursor cur = start;
        // Page of box `lane` of the cursor's tile (num_pages, which reads as
        // zeros, for an id outside the pool).
        auto page_of = [&](const TileCursor& c) {
            const int pos = c.i * TILE + lane * box;
            if (c.b >= B || lane >= nbox || pos >= lens[c.b]) return p.num_pages;
            const int id = p.block_table[(size_t)c.b * p.bt_stride + pos / p.page_size];
            return id >= 0 && id < p.num_pages ? id : p.num_pages;
        };
        int page = page_of(cur);
        int issued = 0;
        for (int k = 0; k < n; ++k) {
            const int s = k % STAGES;
            const bool free_slot = k < STAGES || mbar_wait_bounded(&empty[s], ((k / STAGES) - 1) & 1);
            if (!__all_sync(0xffffffffu, free_slot)) {
                record_error(p.err, kDevTimeoutEmpty);
                break;
            }
            const int kvh = cur.j / hg;
            const int pos0 = cur.i * TILE;
            const int left = lens[cur.b] - pos0;        // <= 0: an empty unit's only tile
            const int boxes = left > 0 ? min(nbox, (left + box - 1) / box) : 0;
            if (lane == 0) mbar_arrive_expect_tx(&full[s], uint32_t(2 * boxes * box * D));
            __syncwarp();
            if (lane < boxes) {
                const int row = (pos0 + lane * box) % p.page_size;
                tma_load_4d(kring + s * S::kTileBytes + lane * box * D, &p.kmap, 0, row, kvh, page,
                            &full[s], policy);
                tma_load_4d(vring + s * S::kTileBytes + lane * box * D, &p.vmap, 0, row, kvh, page,
                            &full[s], policy);
            }
            const int id = __shfl_sync(0xffffffffu, page, min(lane * kKv8Block / box, 31));
            if (lane < BLOCKS && lane * kKv8Block < left) {
                const bool real = id < p.num_pages;
                const int blk = (pos0 + lane * kKv8Block) % p.page_size / kKv8Block;
                const float* src = kp.scales;
                if (real) src += (((size_t)id * p.Hkv + kvh) * kp.blocks_per_page + blk) * 2;
                cp_async_8(smem_u32(scales + s * BLOCKS + lane), src, real ? 8u : 0u);
            }
            cp_async_arrive(&full[s]);
            ++issued;
            cur.advance(seq_start, B, upb, 1);
            page = page_of(cur);                        // in flight while the stage is awaited
        }
        // Drain: every copy this CTA issued has landed before it retires.
        for (int i = max(0, issued - STAGES); i < issued; ++i) {
            if (!mbar_wait_bounded(&full[i % STAGES], (i / STAGES) & 1)) {
                record_error(p.err, kDevTimeoutFull);
                break;
            }
        }
        return;
    }

    // ------------------------------------------------------------ consumers
    int* xm = xflag + 2;
    if (threadIdx.x == 0) {
        TileCursor lc;
        lc.seek(seq_start, B, upb, end - 1);
        const bool one = start.b == lc.b && start.j == lc.j;
        auto note = [&](int r, int bb, int jj, int nbb, bool shared) {
            int* m = xm + 6 * r;
            m[0] = shared ? bb * upb + jj : -1;
            if (!shared) return;
            m[1] = cm.cta_of(bb, jj, nbb, 0);
            m[2] = cm.cta_of(bb, jj, nbb, nbb - 1);
            m[3] = cm.beg(m[1]) < seq_start[bb] + jj * nbb ? 1 : 0;
            m[4] = bb;
            m[5] = jj;
        };
        note(0, start.b, start.j, start.nb,
             one ? !(start.i == 0 && lc.i == lc.nb - 1) : start.i != 0);
        note(1, lc.b, lc.j, lc.nb, !one && lc.i != lc.nb - 1);
    }
    const int g = lane >> 2;
    const int t = lane & 3;
    const float sl2 = p.scale_log2;
    const uint32_t kring_s = smem_u32(kring);
    const uint32_t vring_s = smem_u32(vring);
    bool ok = true;
    TileCursor cur = start;
    int k = 0;
    for (int e = 0; k < n; ++e) {
        const int b = cur.b, j = cur.j, nb = cur.nb, i0 = cur.i;
        const int cnt = min(nb - i0, n - k);
        const int kvh = j / hg, hgrp = j - (j / hg) * hg;
        const int h0 = kvh * p.G + hgrp * GP;
        const int gcount = min(GP, p.G - hgrp * GP);
        const int len = lens[b];
        const size_t head_base = (size_t)b * p.H + h0;

        // Q^T as the B operand: lane (g, t) holds dims (D/4)*t .. of head g, in order
        uint32_t qb[DTILES][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int hj = nt * 8 + g;
            const __half* qrow = p.q + (size_t)b * kp.q_stride + (size_t)(h0 + hj) * D + (D / 4) * t;
#pragma unroll
            for (int w = 0; w < DTILES; w += 2) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (hj < gcount) x = *reinterpret_cast<const uint4*>(qrow + w * 4);
                qb[w][nt][0] = x.x; qb[w][nt][1] = x.y;
                qb[w + 1][nt][0] = x.z; qb[w + 1][nt][1] = x.w;
            }
        }
        float o[DTILES][NT][4];
        float m_run[NT][2], l_run[NT][2];
#pragma unroll
        for (int dm = 0; dm < DTILES; ++dm)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[dm][nt][c] = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m_run[nt][0] = m_run[nt][1] = -INFINITY;
            l_run[nt][0] = l_run[nt][1] = 0.f;
        }

        for (int tt = 0; tt < cnt; ++tt, ++k) {
            const int s = k % STAGES;
            if (ok && !mbar_wait_bounded(&full[s], (k / STAGES) & 1)) {
                record_error(p.err, kDevTimeoutFull);
                ok = false;
            }
            const int row0 = warp * 16 * MT;
            const int valid = len - (i0 + tt) * TILE - row0;
            if (ok && valid > 0)
                consume_kv8<D, NT, MT, Code>(kring_s + s * S::kTileBytes, vring_s + s * S::kTileBytes,
                                             scales + s * BLOCKS + warp * MT, row0, valid, qb, o,
                                             m_run, l_run, sl2, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        cur.advance(seq_start, B, upb, cnt);

        // Row sums: each lane summed its own positions; fold the 8 row groups.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
                float l = l_run[nt][jj];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                l_run[nt][jj] = l;
            }

        // ---- cross-warp fold, halving the warps each round
        const int ok_all = consumer_sync_and(ok ? 1 : 0, NW * 32);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int half = NW / 2; half >= 1; half >>= 1) {
                if (warp >= half && warp < 2 * half)
                    x_store<D, NT>(xarea + ((warp - half) * 32 + lane) * XF, o, m_run, l_run, nt);
                consumer_sync(NW * 32);
                if (warp < half) x_fold<D, NT>(xarea + (warp * 32 + lane) * XF, o, m_run, l_run, nt);
                consumer_sync(NW * 32);
            }
        }

        // ---- output of the item
        const bool whole = i0 == 0 && cnt == nb;
        if (whole) {
            if (warp == 0 && ok_all) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) {
                        const int hj = nt * 8 + 2 * t + jj;
                        const float inv = KvDims<D>::inverse(l_run[nt][jj]);
                        if (hj < gcount) {
                            __half* dst = p.out + (head_base + hj) * D + (D / 8) * g;
#pragma unroll
                            for (int dm = 0; dm < DTILES; dm += 4) {
                                uint32_t h[4];
#pragma unroll
                                for (int x = 0; x < 4; ++x)
                                    h[x] = pack_half2(o[dm + x][nt][jj] * inv, o[dm + x][nt][jj + 2] * inv);
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
                        ok_all ? make_float4(o[dm][nt][0], o[dm][nt][1], o[dm][nt][2], o[dm][nt][3])
                               : make_float4(0.f, 0.f, 0.f, 0.f);
            if (g == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) {
                        const int hj = nt * 8 + 2 * t + jj;
                        pm[hj * 2 + 0] = ok_all ? m_run[nt][jj] : -INFINITY;
                        pm[hj * 2 + 1] = ok_all ? l_run[nt][jj] : 0.f;
                    }
            }
        }
    }

    // ---- count the pieces, merge the units whose count this CTA completed
    if (warp == 0) {
        __syncwarp();
        if (lane == 0) {
            int f0 = 0, f1 = 0;
            if (xm[0] >= 0 || xm[6] >= 0) {
                if (xm[0] >= 0) f0 = atom_add_release_gpu(&p.counters[xm[0]], 1) == xm[2] - xm[1];
                if (xm[6] >= 0) f1 = atom_add_release_gpu(&p.counters[xm[6]], 1) == xm[8] - xm[7];
                if (f0 | f1) fence_acq_rel_gpu();
            }
            xflag[0] = f0;
            xflag[1] = f1;
        }
    }
    consumer_sync(NW * 32);
#pragma unroll 1
    for (int r = 0; r < 2; ++r) {
        if (!xflag[r]) continue;
        const int* m = xm + 6 * r;
        const int bb = m[4], jj = m[5];
        const int kvh = jj / hg, hgrp = jj - (jj / hg) * hg;
        const int gcount = min(GP, p.G - hgrp * GP);
        const size_t head_base = (size_t)bb * p.H + kvh * p.G + hgrp * GP;
        merge_pieces<D, NT, NW, KvDims<D>>(p, xarea, m[1], m[2], m[3] != 0, gcount, head_base);
        if (threadIdx.x == 0) p.counters[m[0]] = 0;
    }
}

}  // namespace fr
