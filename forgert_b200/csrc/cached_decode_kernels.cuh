// cached_decode_kernels.cuh - the frame of single-token attention over a coded
// paged cache: shares of a ragged batch, pieces and their merge.  What a step
// copies and how it is consumed is the format's (kv8_decode_kernels.cuh,
// kv4_decode_kernels.cuh).
//
// Persistent CTAs take equal shares of the batch's work, as in
// batched_kernels.cuh (units, items, pieces merged by the contributor that
// completes a unit), over tiles of TILE = 16 * MT * NW positions.  Inside a
// CTA every warp streams for itself: warp w copies and consumes rows
// 16 * MT * w .. of each tile through a ring of its own (STAGES steps of MT
// blocks of 16 rows of K and V and their scales), so a step needs no barrier
// between warps and no producer.
//
// A format F has
//   kD, kNT, kMT, kStages, kNW, kCtas   head dim, tiles of 8 heads, blocks per
//                  step, ring stages, warps, CTAs per SM
//   Params         CachedDecodeParams of its cache
//   Smem           kStepBytes, kWarpBytes, kStepScales and the areas' offsets
//   Loader         init, look_up, copy, advance (cursor and pages of a warp)
//   Query, State   q in registers; the running (m, l, o) of an item
//   consume        one step
//   pack           two outputs as fp16
//   dim(dm, g)     first of the two dims that lane group g holds in fragment
//                  dm of o; kRun (4 or 1) neighbouring dm are consecutive dims
#pragma once
#include "batched_kernels.cuh"

namespace fr {

// View: the cache (num_pages, page_size, Hkv, addresses).
template <class View>
struct CachedDecodeParams {
    View cache;
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

// 1 / row sum: a sum of NaN stays NaN; an empty unit's gives zeros.
__device__ __forceinline__ float row_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

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
template <class F>
__device__ __forceinline__ void cached_merge(const typename F::Params& p, float* area, int first,
                                             bool first_tail, int stride, int count, int gcount,
                                             size_t head_base, int dst_slot) {
    constexpr int D = F::kD, NT = F::kNT, NW = F::kNW;
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
        const int dim = F::dim(f / (32 * NT), (f & 31) >> 2);
        const int h = ha[i];
        if (h < gcount)
            *reinterpret_cast<uint32_t*>(p.out + (head_base + h) * D + dim) =
                F::pack(acc[i].x * sm_inv[h], acc[i].z * sm_inv[h]);
        if (h + 1 < gcount)
            *reinterpret_cast<uint32_t*>(p.out + (head_base + h + 1) * D + dim) =
                F::pack(acc[i].y * sm_inv[h + 1], acc[i].w * sm_inv[h + 1]);
    }
}

// ---------------------------------------------------------------------------
// Persistent kernel: grid = C co-resident CTAs of NW warps; see
// persistent_decode_kernel for units, items, pieces and the merge.
// ---------------------------------------------------------------------------
template <class F>
__global__ void __launch_bounds__(32 * F::kNW, F::kCtas)
cached_decode_kernel(const __grid_constant__ typename F::Params p) {
    constexpr int D = F::kD, NT = F::kNT, MT = F::kMT, NW = F::kNW, STAGES = F::kStages;
    constexpr int TILE = 16 * MT * NW;
    using S = typename F::Smem;
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
    const unsigned char* scales = smem + S::kScaleOffset + warp * (STAGES * S::kStepScales);
    const uint32_t scales_s = smem_u32(scales);
    typename F::Loader load;
    load.init(p, cur, lens, warp, lane);
    int ls = 0, lk = 0;                         // stage and step of the next copies
    auto start_step = [&]() {
        if (lk < n) {
            const uint32_t kst = ring + ls * (2 * S::kStepBytes);
            load.copy(p, kst, kst + S::kStepBytes, scales_s + ls * S::kStepScales,
                      hg == 1 ? load.cur.j : load.cur.j / hg, lane, policy);
            load.advance(p, seq_start, lens, B, upb, warp, lane);
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

        typename F::Query q;
        q.load(p.q + (size_t)b * p.q_stride + (size_t)h0 * D, gcount, sl2, lane);
        typename F::State st;
        st.clear();
        int valid = len - (i0 * NW + warp) * (16 * MT);     // positions from the warp's step on
        const int k_end = k + cnt;
        for (; k < k_end; ++k, valid -= TILE) {
            __syncwarp();                       // the stage refilled now is read by every lane
            start_step();
            cp_async_wait<STAGES - 1>();
            __syncwarp();                       // every lane's copies have landed
            const uint32_t kst = ring + stage * (2 * S::kStepBytes);
            if (valid > 0)
                F::consume(kst, kst + S::kStepBytes, scales + stage * S::kStepScales, valid, q, st, sl2, lane);
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
                            __half* dst = p.out + (head_base + hj) * D;
#pragma unroll
                            for (int dm = 0; dm < DTILES; dm += F::kRun) {
                                uint32_t h[F::kRun];
#pragma unroll
                                for (int x = 0; x < F::kRun; ++x)
                                    h[x] = F::pack(st.o[dm + x][nt][jj] * inv, st.o[dm + x][nt][jj + 2] * inv);
                                if constexpr (F::kRun == 4)
                                    *reinterpret_cast<uint4*>(dst + F::dim(dm, g)) = make_uint4(h[0], h[1], h[2], h[3]);
                                else
                                    *reinterpret_cast<uint32_t*>(dst + F::dim(dm, g)) = h[0];
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
            cached_merge<F>(p, xarea, cf + lead, tail, 1, min(GROUP, pieces - lead), gcount,
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
        cached_merge<F>(p, xarea, cf, m[3] != 0, stride, count, gcount, head_base, -1);
        if (threadIdx.x == 0) p.counters[m[0]] = 0;       // every piece was counted: re-arm
    }
}

}  // namespace fr
