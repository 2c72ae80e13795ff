// paged_step_kernels.cuh - block tables and slot maps of one serving step,
// built on the GPU from the requests' lengths.
//
// Request b holds kv[b] tokens in ceil(kv[b] / P) pages of its block-table
// row and gets new[b] more; new[b] < 0 ends it.  The pages of ended requests
// go on the stack of free pages in (request, block) order, then the pages
// that the others need are popped in (request, block) order: the i-th popped
// page is released page give - 1 - i for i < give and stack entry
// count - 1 - (i - give) after that, so every page, position and slot follows
// from three prefix sums over the requests (new tokens, pages taken, pages
// given) and no output depends on another.
//
// Every CTA forms the three prefix sums in shared memory (the lengths are a
// few KB, read from L2) and takes its share of the tokens and pages; a token
// finds its request by binary search.  kv_lens_out may be kv_lens and
// free_count_out free_count: they are then written by the CTA that is last to
// have read the inputs (one counter, zero between calls), so no CTA waits.
//
// What bounds it: latency (a launch, two dependent rounds of loads, the scan, a
// search per token): 64 requests 3.5 us in a graph, 1024 requests with 122
// thousand new tokens 8.9 (0.2 us of bytes).
#pragma once
#include "fr_ptx.cuh"
#include <cstdint>

namespace fr {

constexpr int kStepThreads = 1024;
constexpr int kStepMaxBatch = 8192;     // requests whose four arrays fit in shared memory

enum StepStatus : int {
    kStepOk = 0,
    kStepNoPages = 1,      // more pages needed than free and released
    kStepBadLength = 2,    // kv_lens < 0, or longer than a block-table row
    kStepTooMany = 3,      // more new tokens than max_tokens
    kStepBadFree = 4,      // free_count outside 0..num_pages, or the stack would overflow
};

struct StepParams {
    const int* kv_lens;
    const int* new_lens;
    int* block_table;
    int* free_pages;
    const int* free_count;
    int* kv_lens_out;
    int* free_count_out;
    int* token_offsets;
    int* positions;
    long long* slots;
    int* status;
    int* ticket;           // nullptr: one CTA, or no output over its input
    int batch, page_size, num_pages, max_blocks, max_tokens;
};

// Sums of numbers up to a cap, at most 2^30, that stop there: a total past its
// limit refuses the call whatever it is.  Two caps make 2^31, past an int.
__device__ __forceinline__ int add_capped(int a, int b, int cap) {
    return (int)min((unsigned)a + (unsigned)b, (unsigned)cap);
}

__device__ __forceinline__ int last_at_most(const int* first, int n, int x) {
    int lo = 0, hi = n - 1;                     // last b with first[b] <= x
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kStepThreads)
paged_step_kernel(const StepParams p) {
    extern __shared__ int step_smem[];
    const int B = p.batch, P = p.page_size;
    int* kv = step_smem;                        // [B]
    int* ftok = kv + B;                         // [B + 1] prefix sums
    int* ftake = ftok + B + 1;
    int* fgive = ftake + B + 1;
    __shared__ int sums[3][32];
    __shared__ int last_cta;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nwarps = blockDim.x >> 5;
    const int cap[3] = {p.max_tokens + 1, p.num_pages + 1, p.num_pages + 1};
    const long long most = (long long)p.max_blocks * P;

    grid_launch_dependents();
    grid_dependency_wait();
    const int count = *p.free_count;
    int carry[3] = {0, 0, 0};
    int bad = 0;
    for (int b0 = 0; b0 < B; b0 += blockDim.x) {
        const int b = b0 + tid;
        int x[3] = {0, 0, 0};
        if (b < B) {
            const int held = p.kv_lens[b], grow = p.new_lens[b];
            const bool fits = held >= 0 && held <= most && held + (long long)max(grow, 0) <= most;
            bad |= fits ? 0 : 1;
            const int h = fits ? held : 0, g = fits ? grow : 0;
            const int pages = (int)(((long long)h + P - 1) / P);
            x[0] = min(max(g, 0), cap[0]);
            x[1] = g > 0 ? min((int)(((long long)h + g + P - 1) / P) - pages, cap[1]) : 0;
            x[2] = g < 0 ? min(pages, cap[2]) : 0;
            kv[b] = h;
        }
        int inc[3];
#pragma unroll
        for (int c = 0; c < 3; ++c) {
            inc[c] = x[c];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, inc[c], o);
                if (lane >= o) inc[c] = add_capped(inc[c], y, cap[c]);
            }
            if (lane == 31) sums[c][warp] = inc[c];
        }
        __syncthreads();
        if (warp < 3) {                         // warp c scans the warps' sums of quantity c
            int s = lane < nwarps ? sums[warp][lane] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s = add_capped(s, y, cap[warp]);
            }
            sums[warp][lane] = s;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 3; ++c) {
            const int before = add_capped(carry[c], warp ? sums[c][warp - 1] : 0, cap[c]);
            const int up = __shfl_up_sync(0xffffffffu, inc[c], 1);
            int* first = c == 0 ? ftok : c == 1 ? ftake : fgive;
            if (b < B) first[b] = add_capped(before, lane ? up : 0, cap[c]);
            carry[c] = add_capped(carry[c], sums[c][31], cap[c]);
        }
        __syncthreads();                        // sums are reused
    }
    if (tid == 0) {
        ftok[B] = carry[0];
        ftake[B] = carry[1];
        fgive[B] = carry[2];
    }
    bad = __syncthreads_or(bad);
    const int toks = carry[0], take = carry[1], give = carry[2];
    int status = kStepOk;
    if (bad) status = kStepBadLength;
    else if (count < 0 || count > p.num_pages || count + give > p.num_pages) status = kStepBadFree;
    else if (toks > p.max_tokens) status = kStepTooMany;
    else if (take > count + give) status = kStepNoPages;

    // This CTA has read every input of the in-place outputs.  The count is only
    // looked at after the tokens, when it has long come back.
    int arrived = 0;
    if (tid == 0 && p.ticket) arrived = atom_add_acq_rel_gpu(p.ticket, 1);
    const int stride = gridDim.x * blockDim.x, at = blockIdx.x * blockDim.x + tid;
    auto released = [&](int i) {                // i-th released page
        const int b = last_at_most(fgive, B, i);
        return p.block_table[(size_t)b * p.max_blocks + (i - fgive[b])];
    };
    auto popped = [&](int i) {
        return i < give ? released(give - 1 - i) : p.free_pages[count - 1 - (i - give)];
    };
    const bool go = status == kStepOk;          // a refused step changes nothing: no token has a place
    auto finish = [&](int first, int step) {    // lengths and the stack's height after the step
        for (int b = first; b < B; b += step) {
            int after = p.kv_lens[b];           // refused: as it was, fitting or not
            if (go) after = p.new_lens[b] < 0 ? 0 : kv[b] + ftok[b + 1] - ftok[b];
            p.kv_lens_out[b] = after;
        }
        if (first == 0) {
            *p.free_count_out = go ? count + give - take : count;
            *p.status = status;
        }
    };
    if (!p.ticket) finish(at, stride);
    for (int b = at; b <= B; b += stride) p.token_offsets[b] = go ? ftok[b] : 0;
    for (int t = at; t < p.max_tokens; t += stride) {
        int pos = 0;
        long long slot = -1;
        if (go && t < toks) {
            const int b = last_at_most(ftok, B, t);
            pos = kv[b] + (t - ftok[b]);
            const int idx = pos / P, have = (kv[b] + P - 1) / P;
            const int page = idx < have ? p.block_table[(size_t)b * p.max_blocks + idx]
                                        : popped(ftake[b] + idx - have);
            if (page >= 0 && page < p.num_pages) slot = (long long)page * P + (pos - idx * P);
        }
        p.positions[t] = pos;
        p.slots[t] = slot;
    }
    if (go) {
        // Entries read (of released rows, of the stack below count) and written
        // (of growing rows, of the stack from count up) are distinct.
        for (int i = at; i < give; i += stride) p.free_pages[count + i] = released(i);
        for (int i = at; i < take; i += stride) {
            const int b = last_at_most(ftake, B, i);
            p.block_table[(size_t)b * p.max_blocks + (kv[b] + P - 1) / P + (i - ftake[b])] = popped(i);
        }
    }
    // In place: the CTA that was last to have read the inputs writes them.
    if (!p.ticket) return;
    if (tid == 0) {
        last_cta = arrived == (int)gridDim.x - 1;
        if (last_cta) *p.ticket = 0;
    }
    __syncthreads();
    if (last_cta) finish(tid, blockDim.x);
}

}  // namespace fr
