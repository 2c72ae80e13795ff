// kv8_api.cuh - entry points of the 8-bit paged cache (included by capi.cu,
// whose device state, workspace and error handling they share).
#pragma once

namespace {

// No exception leaves a C entry (a lock or a map node that cannot be had).
template <class F>
int guarded(F f) noexcept {
    try {
        return f();
    } catch (...) {
        return cuda_fail(cudaErrorMemoryAllocation);
    }
}

int check_kv8(const fr_kv8_cache* c) {
    if (!c || !c->k || !c->v || !c->scales || c->num_pages <= 0 || c->page_size <= 0 ||
        c->page_size % fr::kKv8Block != 0 || c->num_kv_heads <= 0 ||
        (c->dtype != FR_KV8_INT8 && c->dtype != FR_KV8_E4M3))
        return FR_ERR_INVALID_ARG;
    if (c->head_dim != 64 && c->head_dim != 128) return FR_ERR_UNSUPPORTED;
    const long long limit = 1LL << 40;
    for (long long s : {c->page_stride, c->head_stride, c->row_stride})
        if (s < c->head_dim || s >= limit) return FR_ERR_INVALID_ARG;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->scales, 8) ||
        ((c->page_stride | c->head_stride | c->row_stride) & 15))
        return FR_ERR_MISALIGNED;
    return FR_OK;
}

fr::Kv8View kv8_view(const fr_kv8_cache* c) {
    fr::Kv8View v;
    v.k = static_cast<uint8_t*>(c->k);
    v.v = static_cast<uint8_t*>(c->v);
    v.scales = c->scales;
    v.num_pages = c->num_pages;
    v.page_size = c->page_size;
    v.Hkv = c->num_kv_heads;
    v.page_stride = c->page_stride;
    v.head_stride = c->head_stride;
    v.row_stride = c->row_stride;
    return v;
}

// Shapes of the decode kernel: four warps, steps of 16 (D = 128) or 32 (D = 64)
// rows, 4 KB of codes.
//   for long calls, as many warps as an SM holds: up to 8 query heads per kv
//     head four CTAs (128 registers) with two steps under way per warp, more
//     three CTAs (168 registers: the second 8-head tile's state spills at 128)
//     with three;
//   DEEP, for calls of few tiles per SM, where warps are few anyway and wait
//     for memory: fewer CTAs with more steps under way, and weights of 22 bits
//     (REST).
template <int NT, bool DEEP> struct Kv8Shape;
template <> struct Kv8Shape<1, false> { static constexpr int kCtas = 4, kStages = 2; };
template <> struct Kv8Shape<2, false> { static constexpr int kCtas = 3, kStages = 3; };
template <> struct Kv8Shape<1, true> { static constexpr int kCtas = 3, kStages = 4; };
template <> struct Kv8Shape<2, true> { static constexpr int kCtas = 2, kStages = 6; };
constexpr int kKv8Warps = 4;
template <int D> constexpr int kv8_mt() { return 128 / D; }
constexpr int kv8_tile(int head_dim) { return 16 * (128 / head_dim) * kKv8Warps; }

template <int D, int NT, bool DEEP>
using Kv8SmemOf = fr::Kv8Smem<D, NT, kv8_mt<D>(), Kv8Shape<NT, DEEP>::kStages, kKv8Warps>;

template <int D, int NT, bool DEEP, class Code>
auto kv8_ptr() {
    using Shape = Kv8Shape<NT, DEEP>;
    return fr::kv8_decode_kernel<D, NT, kv8_mt<D>(), Shape::kStages, kKv8Warps, Shape::kCtas, DEEP,
                                 Code>;
}

template <int D, int NT, bool DEEP, class Code>
int prepare_kv8(DeviceState* st, int slot) {
    std::lock_guard<std::mutex> lk(g_prep_mu);
    if (st->kv8_occ[slot]) return FR_OK;
    const int bytes = static_cast<int>(Kv8SmemOf<D, NT, DEEP>::kBytes);
    auto fn = kv8_ptr<D, NT, DEEP, Code>();
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return cuda_fail(e);
    int n = 0;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, 32 * kKv8Warps, bytes);
    if (e != cudaSuccess) return cuda_fail(e);
    st->kv8_occ[slot] = std::max(1, n);
    return FR_OK;
}

template <int D, int NT, bool DEEP, class Code>
int launch_kv8(const fr::Kv8DecodeParams& kp, int ctas, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, 1, 1);
    cfg.blockDim = dim3(32 * kKv8Warps, 1, 1);
    cfg.dynamicSmemBytes = Kv8SmemOf<D, NT, DEEP>::kBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kv8_ptr<D, NT, DEEP, Code>(), kp);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? FR_OK : cuda_fail(e);
}

// f(D, NT, Code) for the sizes and type at hand.
template <class F>
int kv8_dispatch(int head_dim, int nt, int dtype, F f) {
    using std::integral_constant;
    auto with_code = [&](auto d, auto n) {
        return dtype == FR_KV8_INT8 ? f(d, n, fr::Int8Code()) : f(d, n, fr::E4m3Code());
    };
    auto with_nt = [&](auto d) {
        return nt == 1 ? with_code(d, integral_constant<int, 1>())
                       : with_code(d, integral_constant<int, 2>());
    };
    return head_dim == 64 ? with_nt(integral_constant<int, 64>())
                          : with_nt(integral_constant<int, 128>());
}

// Counters of a call: one per unit, then one per partial slot.
constexpr int kKv8Units = kMaxUnits / 2;

// Sequences per launch: their lengths' prefix fits shared memory, their units
// the counters, their tiles the kernel's 32-bit tile numbers.  0 = not even one.
int kv8_chunk(int batch, int num_kv_heads, int head_groups, int head_dim, int max_kv_len) {
    const long long upb = (long long)num_kv_heads * head_groups;
    const int tile = kv8_tile(head_dim);
    const long long tiles = std::max(1, (max_kv_len + tile - 1) / tile);
    const long long n = std::min({(long long)fr::kPersistMaxBatch, kKv8Units / upb,
                                  ((1LL << 29) - 1) / (upb * tiles), (long long)batch});
    return (int)n;
}

struct Kv8Plan {
    int nt = 1, head_groups = 1, chunk = 0, ctas = 0;
    bool deep = false;
    size_t ws_bytes = 0;
};

int kv8_plan(DeviceState* st, int batch, int num_heads, int num_kv_heads, int head_dim,
             int max_kv_len, int dtype, Kv8Plan* out) {
    Kv8Plan pl;
    const int group = num_heads / num_kv_heads;
    pl.nt = group <= 8 ? 1 : 2;
    pl.head_groups = (group + 8 * pl.nt - 1) / (8 * pl.nt);
    pl.chunk = kv8_chunk(batch, num_kv_heads, pl.head_groups, head_dim, max_kv_len);
    if (pl.chunk <= 0) return FR_ERR_INVALID_ARG;
    const int tile = kv8_tile(head_dim);
    const long long tiles = (long long)pl.chunk * num_kv_heads * pl.head_groups *
                            std::max(1, (max_kv_len + tile - 1) / tile);
    // The deep shape up to 22 tiles per SM, were every sequence as long as the
    // longest may be (28 / 4 heads of 128, deep / long shape, bursts of calls
    // and one fp16 weight in both: one sequence of 4096 tokens 11.5 / 14.3 us,
    // 64 of up to 300 10.1 / 12.3, 24 of up to 2000 14.0 / 16.4, 48 of up to
    // 1300 19.4 / 18.2, 64 of up to 8192 57.9 / 49.9).
    pl.deep = tiles <= 22LL * st->sm_count;
    const int slot = (head_dim == 64 ? 0 : 8) + (pl.nt - 1) * 4 + (pl.deep ? 2 : 0) + dtype;
    int rc = kv8_dispatch(head_dim, pl.nt, dtype, [&](auto d, auto n, auto code) {
        constexpr int D = decltype(d)::value, NT = decltype(n)::value;
        return pl.deep ? prepare_kv8<D, NT, true, decltype(code)>(st, slot)
                       : prepare_kv8<D, NT, false, decltype(code)>(st, slot);
    });
    if (rc != FR_OK) return rc;
    pl.ctas = (int)std::max<long long>(
        1, std::min<long long>((long long)st->sm_count * st->kv8_occ[slot], tiles));
    pl.ws_bytes = kCounterBytes + (size_t)2 * pl.ctas * 8 * pl.nt * (head_dim + 2) * sizeof(float);
    *out = pl;
    return FR_OK;
}

int run_kv8(const void* q, long long q_stride, const fr_kv8_cache* cache, const int* block_table,
            const int* kv_lens, void* out, int batch, int num_heads, int max_blocks,
            int max_kv_len, cudaStream_t s) {
    DeviceState* st = nullptr;
    int rc = get_state(&st);
    if (rc != FR_OK) return rc;
    const int Hkv = cache->num_kv_heads, D = cache->head_dim;
    const int len = std::max(1, max_kv_len);
    Kv8Plan pl;
    rc = kv8_plan(st, batch, num_heads, Hkv, D, len, cache->dtype, &pl);
    if (rc != FR_OK) return rc;
    rc = ensure_workspace(st, pl.ws_bytes, s);
    if (rc != FR_OK) return rc;
    fr::Kv8DecodeParams p;
    std::memset(&p, 0, sizeof(p));
    p.cache = kv8_view(cache);
    p.q_stride = q_stride;
    p.H = num_heads;
    p.G = num_heads / Hkv;
    p.head_groups = pl.head_groups;
    p.bt_stride = max_blocks;
    p.max_len = max_kv_len;
    p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)D));
    p.counters = static_cast<int*>(st->ws);
    p.max_units = kKv8Units;
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(st->ws) + kCounterBytes);
    p.part_acc = p.part_ml + (size_t)2 * pl.ctas * 8 * pl.nt * 2;
    // At least two tiles per CTA before SMs get more than one.  A unit's start
    // and its merge are charged as one tile each (four each, which suits the
    // 16-bit kernel's longer tiles, left too few CTAs to short calls: one
    // sequence of 2048 tokens 18.6 us instead of 10.6), and units of up to six
    // tiles are not cut: 64 sequences of 200 to 300 tokens 17.4 -> 12.4 us, no
    // call measured slower.
    p.min_tiles_per_cta = 2;
    p.min_ctas = st->sm_count;
    p.item_cost = 1;
    p.merge_cost = 1;
    p.whole_tiles = 6;
    for (int b = 0; b < batch; b += pl.chunk) {
        p.batch = std::min(pl.chunk, batch - b);
        p.q = static_cast<const __half*>(q) + (size_t)b * q_stride;
        p.out = static_cast<__half*>(out) + (size_t)b * num_heads * D;
        p.kv_lens = kv_lens + b;
        p.block_table = block_table + (size_t)b * max_blocks;
        rc = kv8_dispatch(D, pl.nt, cache->dtype, [&](auto d, auto n, auto code) {
            constexpr int kD = decltype(d)::value, NT = decltype(n)::value;
            return pl.deep ? launch_kv8<kD, NT, true, decltype(code)>(p, pl.ctas, s)
                           : launch_kv8<kD, NT, false, decltype(code)>(p, pl.ctas, s);
        });
        if (rc != FR_OK) return rc;
    }
    return FR_OK;
}

// Programmatic dependent launch, on the default stream too: every kernel here
// waits for the grid before it ahead of its first access to memory, so only
// the launch itself overlaps (1.5 to 2 us a call).
template <class... Args>
int launch_plain(void (*fn)(Args...), unsigned grid, unsigned block, size_t smem, cudaStream_t s,
                 Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, fn, args...);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? FR_OK : cuda_fail(e);
}

}  // namespace

extern "C" {

int fr_paged_step(const int* kv_lens, const int* new_lens, int* block_table, int* free_pages,
                  const int* free_count, int* kv_lens_out, int* free_count_out,
                  int* token_offsets, int* positions, long long* slots, int* status, int batch,
                  int page_size, int num_pages, int max_blocks_per_seq, int max_tokens,
                  void* stream) {
    const long long limit = 1LL << 30;
    if (!kv_lens || !new_lens || !block_table || !free_pages || !free_count || !kv_lens_out ||
        !free_count_out || !token_offsets || !positions || !slots || !status || batch <= 0 ||
        batch > fr::kStepMaxBatch || page_size <= 0 || num_pages <= 0 ||
        max_blocks_per_seq <= 0 || max_tokens <= 0 || num_pages >= limit || max_tokens >= limit ||
        (long long)max_blocks_per_seq * page_size >= limit || new_lens == kv_lens_out)
        return FR_ERR_INVALID_ARG;
    for (const void* a : {(const void*)kv_lens, (const void*)new_lens, (const void*)block_table,
                          (const void*)free_pages, (const void*)free_count,
                          (const void*)kv_lens_out, (const void*)free_count_out,
                          (const void*)token_offsets, (const void*)positions,
                          (const void*)status})
        if (!aligned(a, 4)) return FR_ERR_MISALIGNED;
    if (!aligned(slots, 8)) return FR_ERR_MISALIGNED;
    return guarded([&]() -> int {
        DeviceState* st = nullptr;
        int rc = get_state(&st);
        if (rc != FR_OK) return rc;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const size_t smem = (size_t)(4 * batch + 3) * sizeof(int);
        {
            std::lock_guard<std::mutex> lk(g_prep_mu);
            if (!st->step_ready) {
                cudaError_t e = cudaFuncSetAttribute(
                    fr::paged_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                    (int)((4 * fr::kStepMaxBatch + 3) * sizeof(int)));
                if (e != cudaSuccess) return cuda_fail(e);
                st->step_ready = true;
            }
        }
        fr::StepParams p{kv_lens, new_lens, block_table, free_pages, free_count, kv_lens_out,
                         free_count_out, token_offsets, positions, slots, status, nullptr, batch,
                         page_size, num_pages, max_blocks_per_seq, max_tokens};
        // One CTA per 1024 tokens or 256 requests (whose pages change hands),
        // at most one per SM.  Several that update the lengths in place share a
        // counter of the workspace; a capture without a workspace runs with one.
        int ctas = std::min(st->sm_count, std::max((max_tokens + fr::kStepThreads - 1) / fr::kStepThreads,
                                                   (batch + 255) / 256));
        if (ctas > 1 && (kv_lens_out == kv_lens || free_count_out == free_count)) {
            rc = ensure_workspace(st, kCounterBytes, s);
            if (rc == FR_ERR_WORKSPACE) ctas = 1;
            else if (rc != FR_OK) return rc;
            else p.ticket = static_cast<int*>(st->ws);
        }
        const unsigned threads = ctas == 1 && batch <= 256 ? 256 : fr::kStepThreads;
        return launch_plain(fr::paged_step_kernel, (unsigned)ctas, threads, smem, s,
                            static_cast<const fr::StepParams>(p));
    });
}

int fr_qkv_rope_append_kv8(const void* q, const void* k, const void* v, void* q_out, void* k_out,
                           void* v_out, const long long* token_strides, const void* q_bias,
                           const void* k_bias, const void* v_bias, const float* cos_tab,
                           const float* sin_tab, int table_rows, const int* positions,
                           int num_axes, const unsigned char* freq_axis, const long long* slots,
                           const fr_kv8_cache* cache, int num_tokens, int num_heads,
                           void* stream) {
    if (!q || !k || !v || !q_out || !cos_tab || !sin_tab || !positions || !slots ||
        table_rows <= 0 || num_tokens < 0 || num_axes < 1 || num_axes > fr::kMaxAxes ||
        (num_axes > 1 && !freq_axis))
        return FR_ERR_INVALID_ARG;
    int rc = check_kv8(cache);
    if (rc != FR_OK) return rc;
    const int D = cache->head_dim, Hkv = cache->num_kv_heads;
    rc = check_heads(num_heads, Hkv, D);
    if (rc != FR_OK) return rc;
    fr::AppendParams p;
    std::memset(&p, 0, sizeof(p));
    if (num_axes > 1)
        for (int f = 0; f < D / 2; ++f) {
            if (freq_axis[f] >= num_axes) return FR_ERR_INVALID_ARG;
            p.axis[f] = freq_axis[f];
        }
    p.by_quads = 1;
    for (int f = 0; f < D / 2; ++f) p.by_quads &= p.axis[f] == p.axis[f & ~3];
    const long long heads[6] = {num_heads, Hkv, Hkv, num_heads, Hkv, Hkv};
    for (int i = 0; i < 6; ++i) {
        p.stride[i] = token_strides ? token_strides[i] : heads[i] * D;
        const bool used = i < 4 || (i == 4 ? k_out : v_out) != nullptr;
        if (used && p.stride[i] < heads[i] * D) return FR_ERR_INVALID_ARG;
        if (used && (p.stride[i] & 3)) return FR_ERR_MISALIGNED;
    }
    // An output over its input has to lie as the input does.
    if ((q_out == q && p.stride[3] != p.stride[0]) || (k_out == k && p.stride[4] != p.stride[1]) ||
        (v_out == v && p.stride[5] != p.stride[2]))
        return FR_ERR_INVALID_ARG;
    for (const void* a : {q, k, v, (const void*)q_out, (const void*)k_out, (const void*)v_out,
                          q_bias, k_bias, v_bias, (const void*)slots})
        if (!aligned(a, 8)) return FR_ERR_MISALIGNED;
    if (!aligned(cos_tab, 16) || !aligned(sin_tab, 16) || !aligned(positions, 4))
        return FR_ERR_MISALIGNED;
    if (num_tokens == 0) return FR_OK;
    return guarded([&]() -> int {
        DeviceState* st = nullptr;
        int rc = get_state(&st);
        if (rc != FR_OK) return rc;
        p.q = static_cast<const __half*>(q);
        p.k = static_cast<const __half*>(k);
        p.v = static_cast<const __half*>(v);
        p.q_out = static_cast<__half*>(q_out);
        p.k_out = static_cast<__half*>(k_out);
        p.v_out = static_cast<__half*>(v_out);
        p.bias[0] = static_cast<const __half*>(q_bias);
        p.bias[1] = static_cast<const __half*>(k_bias);
        p.bias[2] = static_cast<const __half*>(v_bias);
        p.cos_tab = cos_tab;
        p.sin_tab = sin_tab;
        p.positions = positions;
        p.slots = slots;
        p.cache = kv8_view(cache);
        p.err = st->err;
        p.T = num_tokens;
        p.H = num_heads;
        p.table_rows = table_rows;
        // A CTA per token while the SMs hold them all (a decode step's tokens
        // are blocks of their own, done one after the other in a window);
        // windows of 4 and of 16 tokens for more, where most tokens share the
        // block of one before them and their CTAs would have nothing to do
        // (28 / 4 heads of 128, windows 1 / 4 / 16: 512 decoding sequences 15.4
        // / 12.6 / 36.4 us, 2048 prompt tokens 25.0 / 13.5 / 11.0, 8192 prompt
        // tokens 93 / 49 / 40).
        const long long held = 16LL * st->sm_count, kv = 2LL * num_tokens * Hkv;
        p.window = kv <= held ? 1 : kv <= 8 * held ? 4 : 16;
        const long long kv_ctas = 2LL * ((num_tokens + p.window - 1) / p.window) * Hkv;
        // Query heads of a token in one lane group, which looks its angles up
        // once: four, more when the tokens alone fill the SMs.
        const int rows = 32 / (D / 8) * fr::kAppendWarps;                  // lane groups of a CTA
        const long long fit = std::max(1LL, held * rows / num_tokens);     // lane groups per token
        p.q_heads = (int)std::max<long long>(4, (num_heads + fit - 1) / fit);
        const long long items = (long long)num_tokens * ((num_heads + p.q_heads - 1) / p.q_heads);
        const long long grid = kv_ctas + (items + rows - 1) / rows;
        p.kv_ctas = (int)kv_ctas;
        if (grid >= (1LL << 31)) return FR_ERR_INVALID_ARG;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return kv8_dispatch(D, 1, cache->dtype, [&](auto d, auto, auto code) {
            auto fn = fr::kv8_append_kernel<decltype(d)::value, decltype(code)>;
            return launch_plain(fn, (unsigned)grid, fr::kAppendThreads, 0, s,
                                static_cast<const fr::AppendParams>(p));
        });
    });
}

int fr_kv8_gather(const fr_kv8_cache* cache, const long long* slots, void* k_out, void* v_out,
                  int num_slots, void* stream) {
    if (!slots || (!k_out && !v_out) || num_slots < 0) return FR_ERR_INVALID_ARG;
    int rc = check_kv8(cache);
    if (rc != FR_OK) return rc;
    if (!aligned(slots, 8) || !aligned(k_out, 16) || !aligned(v_out, 16)) return FR_ERR_MISALIGNED;
    if (num_slots == 0) return FR_OK;
    return guarded([&]() -> int {
        fr::GatherParams p;
        p.cache = kv8_view(cache);
        p.slots = slots;
        p.k_out = static_cast<__half*>(k_out);
        p.v_out = static_cast<__half*>(v_out);
        p.pieces = (long long)num_slots * cache->num_kv_heads * (cache->head_dim / 16);
        const long long grid = (p.pieces + 255) / 256;
        if (grid >= (1LL << 31)) return FR_ERR_INVALID_ARG;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return kv8_dispatch(cache->head_dim, 1, cache->dtype, [&](auto d, auto, auto code) {
            return launch_plain(fr::kv8_gather_kernel<decltype(d)::value, decltype(code)>,
                                (unsigned)grid, 256, 0, s,
                                static_cast<const fr::GatherParams>(p));
        });
    });
}

int fr_decode_attn_paged_kv8(const void* q, long long q_stride, const fr_kv8_cache* cache,
                             const int* block_table, const int* kv_lens, void* out, int batch,
                             int num_heads, int max_blocks_per_seq, int max_kv_len,
                             void* stream) {
    if (!q || !block_table || !kv_lens || !out || batch <= 0 || max_blocks_per_seq <= 0 ||
        max_kv_len < 0 || max_kv_len >= (1 << 30))
        return FR_ERR_INVALID_ARG;
    int rc = check_kv8(cache);
    if (rc != FR_OK) return rc;
    if ((long long)max_blocks_per_seq * cache->page_size < max_kv_len) return FR_ERR_INVALID_ARG;
    rc = check_heads(num_heads, cache->num_kv_heads, cache->head_dim);
    if (rc != FR_OK) return rc;
    const long long row = (long long)num_heads * cache->head_dim;
    if (q_stride == 0) q_stride = row;
    if (q_stride < row) return FR_ERR_INVALID_ARG;
    if (!aligned(q, 16) || !aligned(out, 16) || (q_stride & 7) || !aligned(block_table, 4) ||
        !aligned(kv_lens, 4))
        return FR_ERR_MISALIGNED;
    return guarded([&]() -> int {
        return run_kv8(q, q_stride, cache, block_table, kv_lens, out, batch, num_heads,
                       max_blocks_per_seq, max_kv_len, static_cast<cudaStream_t>(stream));
    });
}

size_t fr_kv8_workspace_size(int batch, int num_heads, int num_kv_heads, int head_dim,
                             int max_kv_len) {
    if (batch <= 0 || max_kv_len < 0 || check_heads(num_heads, num_kv_heads, head_dim) != FR_OK)
        return 0;
    size_t bytes = 0;
    guarded([&]() -> int {
        DeviceState* st = nullptr;
        int rc = get_state(&st);
        for (int dtype : {FR_KV8_INT8, FR_KV8_E4M3}) {
            Kv8Plan pl;
            if (rc == FR_OK)
                rc = kv8_plan(st, batch, num_heads, num_kv_heads, head_dim,
                              std::max(1, max_kv_len), dtype, &pl);
            bytes = rc == FR_OK ? std::max(bytes, pl.ws_bytes) : 0;
        }
        return rc;
    });
    return bytes;
}

}  // extern "C"
