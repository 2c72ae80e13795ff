// kv4_api.cuh - entry points of the 4-bit paged cache and of the 16-bit pages'
// append (included by capi.cu after kv8_api.cuh, whose launch and planning
// helpers they share).
#pragma once

namespace {

constexpr int kPageRows = 16;           // pages hold whole blocks of this many rows

int check_kv4(const fr_kv4_cache* c) {
    if (!c || !c->k || !c->v || !c->scales || c->num_pages <= 0 || c->page_size <= 0 ||
        c->page_size % kPageRows != 0 || c->num_kv_heads <= 0)
        return FR_ERR_INVALID_ARG;
    if (c->head_dim != 64 && c->head_dim != 128) return FR_ERR_UNSUPPORTED;
    for (long long s : {c->page_stride, c->head_stride, c->row_stride})
        if (s < c->head_dim / 2) return FR_ERR_INVALID_ARG;
    // The decode kernel counts 16-byte pieces in 32 bits: codes of K (or V) and
    // scales below 64 GB each.
    const long long limit = 1LL << 32, pages = c->num_pages;
    const long long scales = (long long)c->num_kv_heads * c->page_size * (c->head_dim / 8) / 16;
    if (c->page_stride >= limit || c->head_stride > (limit * 16 - 1) / c->num_kv_heads ||
        c->row_stride > (limit * 16 - 1) / c->page_size || scales > (limit - 1) / pages ||
        pages * (c->page_stride / 16) + c->num_kv_heads * (c->head_stride / 16) +
                c->page_size * (c->row_stride / 16) >= limit)
        return FR_ERR_INVALID_ARG;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->scales, 16) ||
        ((c->page_stride | c->head_stride | c->row_stride) & 15))
        return FR_ERR_MISALIGNED;
    return FR_OK;
}

fr::Kv4View kv4_view(const fr_kv4_cache* c) {
    fr::Kv4View v;
    v.k = static_cast<uint8_t*>(c->k);
    v.v = static_cast<uint8_t*>(c->v);
    v.scales = static_cast<__half*>(c->scales);
    v.num_pages = c->num_pages;
    v.page_size = c->page_size;
    v.Hkv = c->num_kv_heads;
    v.page_stride = c->page_stride;
    v.head_stride = c->head_stride;
    v.row_stride = c->row_stride;
    v.page16 = (uint32_t)(c->page_stride / 16);
    v.block16 = (uint32_t)c->row_stride;
    v.head_scales16 = (uint32_t)((long long)c->page_size * (c->head_dim / 8) / 16);
    v.scales16 = c->num_kv_heads * v.head_scales16;
    return v;
}

// Shapes of the decode kernel: four warps, kMT blocks of 16 rows a step (what a
// step costs beside its blocks, about 86 instructions a warp, is a seventh of the
// two blocks' at D = 128; four blocks a step instead of two at D = 64: 32 sequences
// of 8192 to 16384 tokens, 8 heads, 69.4 -> 61.3 us, 64 with 24 / 2 61.6 -> 55.5;
// at D = 128 shared memory holds two with up to 8 heads, and with 16 four are as
// fast: 64 sequences of 8192 to 16384 tokens, 16 / 1 heads, 57.8 and 57.6 us, of
// 1024 to 8192 31.4 and 32.5).
//   for long calls three CTAs per SM with up to 8 heads (168 registers at D = 128,
//     161 at 64; at 128 for four the state spills: 64 sequences of 8192 to 32768
//     tokens 149 -> 246 us, with weights in one fp16), two with 16 (255, of which
//     16 bytes are spilled, and 227);
//   DEEP, for calls of few tiles per SM: up to 8 heads, more steps under way (211
//     registers at D = 128, 155 at 64).
template <int D, int NT, bool DEEP> struct Kv4Shape {
    static constexpr int kMT = 2, kCtas = 2, kStages = 4;
};
template <> struct Kv4Shape<64, 2, false> { static constexpr int kMT = 4, kCtas = 2, kStages = 3; };
template <> struct Kv4Shape<128, 1, false> { static constexpr int kMT = 2, kCtas = 3, kStages = 3; };
template <> struct Kv4Shape<64, 1, false> { static constexpr int kMT = 4, kCtas = 3, kStages = 3; };
template <> struct Kv4Shape<64, 1, true> { static constexpr int kMT = 2, kCtas = 3, kStages = 4; };
constexpr int kKv4Warps = 4;
constexpr int kKv4Tile = 16 * 2 * kKv4Warps;    // the least of any shape: tiles of a call are at most as many

template <int D, int NT, bool DEEP>
using Kv4FormatOf = fr::Kv4Format<D, NT, Kv4Shape<D, NT, DEEP>::kMT, Kv4Shape<D, NT, DEEP>::kStages,
                                  kKv4Warps, Kv4Shape<D, NT, DEEP>::kCtas>;

// f(Format) for the sizes at hand.
template <class F>
int kv4_dispatch(int head_dim, int nt, bool deep, F f) {
    auto with_d = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return deep ? f(Kv4FormatOf<D, 1, true>())
                    : nt == 1 ? f(Kv4FormatOf<D, 1, false>()) : f(Kv4FormatOf<D, 2, false>());
    };
    return head_dim == 64 ? with_d(std::integral_constant<int, 64>())
                          : with_d(std::integral_constant<int, 128>());
}

int kv4_plan(DeviceState* st, int batch, int num_heads, int num_kv_heads, int head_dim,
             int max_kv_len, CachedPlan* out) {
    CachedPlan pl;
    const int group = num_heads / num_kv_heads;
    auto tiles_of = [&](int nt) {
        pl.nt = nt;
        pl.head_groups = (group + 8 * nt - 1) / (8 * nt);
        pl.chunk = cached_chunk(batch, num_kv_heads, pl.head_groups, kKv4Tile, max_kv_len);
        return (long long)pl.chunk * num_kv_heads * pl.head_groups *
               std::max(1, (max_kv_len + kKv4Tile - 1) / kKv4Tile);
    };
    // The deep shape up to 11 tiles per SM, were every sequence as long as the
    // longest may be (28 / 4 heads of 128, deep / long shape: 64 sequences of 200 to
    // 300 tokens 9.9 / 11.4 us, 17 of up to 2999 with 12 / 2 heads 11.6 / 13.2, one of
    // 2048 9.8 / 9.9, 32 of 1000 to 1500 17.9 / 17.9, 64 of 1024 to 8192 52.9 / 50.8;
    // 32 of 8192 to 16384 with 8 heads of 64 69.4 / 61.3).
    long long tiles = tiles_of(group <= 8 ? 1 : 2);
    pl.deep = tiles <= 11LL * st->sm_count;
    // A second tile of 8 heads shares the codes' masks but leaves two CTAs per SM: it
    // pays in long calls (16 / 1 heads of 128, two tiles / each by itself: 64
    // sequences of 8192 to 16384 tokens 57.8 / 61.4 us, one of 2048 14.6 / 9.5).
    if (pl.deep) tiles = tiles_of(1);
    if (pl.chunk <= 0) return FR_ERR_INVALID_ARG;
    int* occ = &st->kv4_occ[(head_dim == 64 ? 0 : 3) + (pl.deep ? 2 : pl.nt - 1)];
    int rc = kv4_dispatch(head_dim, pl.nt, pl.deep,
                          [&](auto format) { return prepare_cached<decltype(format)>(occ); });
    if (rc != FR_OK) return rc;
    pl.ctas = (int)std::max<long long>(1, std::min<long long>((long long)st->sm_count * *occ, tiles));
    pl.ws_bytes = kCounterBytes + (size_t)2 * pl.ctas * 8 * pl.nt * (head_dim + 2) * sizeof(float);
    *out = pl;
    return FR_OK;
}

int run_kv4(const void* q, long long q_stride, const fr_kv4_cache* cache, const int* block_table,
            const int* kv_lens, void* out, int batch, int num_heads, int max_blocks,
            int max_kv_len, cudaStream_t s) {
    DeviceState* st = nullptr;
    int rc = get_state(&st);
    if (rc != FR_OK) return rc;
    const int Hkv = cache->num_kv_heads, D = cache->head_dim;
    CachedPlan pl;
    rc = kv4_plan(st, batch, num_heads, Hkv, D, std::max(1, max_kv_len), &pl);
    if (rc != FR_OK) return rc;
    rc = ensure_workspace(st, pl.ws_bytes, s);
    if (rc != FR_OK) return rc;
    fr::CachedDecodeParams<fr::Kv4View> p;
    std::memset(&p, 0, sizeof(p));
    p.cache = kv4_view(cache);
    p.q_stride = q_stride;
    p.H = num_heads;
    p.G = num_heads / Hkv;
    p.head_groups = pl.head_groups;
    p.bt_stride = max_blocks;
    p.max_len = max_kv_len;
    p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)D));
    p.counters = static_cast<int*>(st->ws);
    p.max_units = kCachedUnits;
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(st->ws) + kCounterBytes);
    p.part_acc = p.part_ml + (size_t)2 * pl.ctas * 8 * pl.nt * 2;
    // The rules below were measured on 64 calls (28 / 4 and 16 / 1 heads of 128, 14 / 2
    // and 8 / 8 of 64; 1 to 128 sequences of up to 8192 tokens).
    // One tile per CTA is enough before SMs get more than one: with two no call is
    // faster, and those of one to two tiles per SM leave half the copies that could
    // be under way (24 sequences of 500 to 2000 tokens, 14 / 2 and 16 / 1 heads, 10.6
    // and 11.9 -> 12.8 and 14.7 us; 64 of up to 1000, 14 / 2, 10.9 -> 13.3).
    // A unit's start and its merge are charged as one tile each: without, one sequence
    // gains (of 900 tokens 9.2 -> 8.5) and ragged batches lose (64 of 1024 to 8192,
    // 28 / 4, 14 / 2 and 16 / 1 heads, 51.2, 20.1 and 31.4 -> 52.9, 21.4 and 33.7); as
    // two, one of 900 takes 9.9 and most batches longer (52.4, 21.4, 30.9).
    // Units of up to four tiles are not cut, since handing a piece over and merging it
    // take a CTA about as long as four tiles do: with two, 64 of 200 to 300 take 15.8
    // us instead of 10.1 and one of 512 (14 / 2) 7.5 instead of 7.1; with six, one of
    // 700 takes 11.3 instead of 9.2 and 9.0 instead of 7.6 (14 / 2).
    p.min_tiles_per_cta = 1;
    p.min_ctas = st->sm_count;
    p.item_cost = 1;
    p.merge_cost = 1;
    p.whole_tiles = 4;
    for (int b = 0; b < batch; b += pl.chunk) {
        p.batch = std::min(pl.chunk, batch - b);
        p.q = static_cast<const __half*>(q) + (size_t)b * q_stride;
        p.out = static_cast<__half*>(out) + (size_t)b * num_heads * D;
        p.kv_lens = kv_lens + b;
        p.block_table = block_table + (size_t)b * max_blocks;
        rc = kv4_dispatch(D, pl.nt, pl.deep,
                          [&](auto format) { return launch_cached<decltype(format)>(p, pl.ctas, s); });
        if (rc != FR_OK) return rc;
    }
    return FR_OK;
}

// Checks and lays out what both appends take; the pages are the caller's.
int fill_append(const void* q, const void* k, const void* v, void* q_out, void* k_out, void* v_out,
                const long long* token_strides, const void* q_bias, const void* k_bias,
                const void* v_bias, const float* cos_tab, const float* sin_tab, int table_rows,
                const int* positions, int num_axes, const unsigned char* freq_axis,
                const long long* slots, int num_tokens, int num_heads, int num_kv_heads,
                int head_dim, fr::PagedAppendParams* out) {
    if (!q || !k || !v || !q_out || !cos_tab || !sin_tab || !positions || !slots ||
        table_rows <= 0 || num_tokens < 0 || num_axes < 1 || num_axes > fr::kPagedAxes ||
        (num_axes > 1 && !freq_axis))
        return FR_ERR_INVALID_ARG;
    int rc = check_heads(num_heads, num_kv_heads, head_dim);
    if (rc != FR_OK) return rc;
    fr::PagedAppendParams p;
    std::memset(&p, 0, sizeof(p));
    if (num_axes > 1)
        for (int f = 0; f < head_dim / 2; ++f) {
            if (freq_axis[f] >= num_axes) return FR_ERR_INVALID_ARG;
            p.axis[f] = freq_axis[f];
        }
    p.by_eights = 1;
    for (int f = 0; f < head_dim / 2; ++f) p.by_eights &= p.axis[f] == p.axis[f & ~7];
    const long long heads[6] = {num_heads, num_kv_heads, num_kv_heads,
                                num_heads, num_kv_heads, num_kv_heads};
    const void* const in[3] = {q, k, v};
    void* const outs[3] = {q_out, k_out, v_out};
    const void* const bias[3] = {q_bias, k_bias, v_bias};
    for (int i = 0; i < 6; ++i) {
        p.stride[i] = token_strides ? token_strides[i] : heads[i] * head_dim;
        const bool used = i < 3 || outs[i - 3];
        if (used && (p.stride[i] < heads[i] * head_dim || p.stride[i] >= (1LL << 32)))
            return FR_ERR_INVALID_ARG;
        if (used && (p.stride[i] & 7)) return FR_ERR_MISALIGNED;
    }
    for (int i = 0; i < 3; ++i) {
        // An output over its input has to lie as the input does.
        if (outs[i] == in[i] && p.stride[3 + i] != p.stride[i]) return FR_ERR_INVALID_ARG;
        if (!aligned(in[i], 16) || !aligned(outs[i], 16) || !aligned(bias[i], 16))
            return FR_ERR_MISALIGNED;
        p.in[i] = static_cast<const __half*>(in[i]);
        p.out[i] = static_cast<__half*>(outs[i]);
        p.bias[i] = static_cast<const __half*>(bias[i]);
    }
    if (!aligned(cos_tab, 16) || !aligned(sin_tab, 16) || !aligned(positions, 4) ||
        !aligned(slots, 8))
        return FR_ERR_MISALIGNED;
    p.cos_tab = cos_tab;
    p.sin_tab = sin_tab;
    p.positions = positions;
    p.slots = slots;
    p.T = num_tokens;
    p.H = num_heads;
    p.Hkv = num_kv_heads;
    p.table_rows = table_rows;
    *out = p;
    return FR_OK;
}

template <class Pages>
int run_append(fr::PagedAppendParams p, int head_dim, cudaStream_t s) {
    DeviceState* st = nullptr;
    int rc = get_state(&st);
    if (rc != FR_OK) return rc;
    p.err = st->err;
    const long long rows = fr::kPagedThreads / (head_dim / 16);             // of a CTA
    const long long kv = (long long)p.T * p.Hkv;
    const long long kv_ctas = (kv + rows - 1) / rows;
    const long long q_rows = (long long)p.T * ((p.H + fr::kQRows - 1) / fr::kQRows);
    const long long grid = 2 * kv_ctas + (q_rows + rows - 1) / rows;
    if (kv + rows >= (1LL << 31) || grid >= (1LL << 31)) return FR_ERR_INVALID_ARG;
    p.kv_ctas = (int)kv_ctas;
    auto fn = head_dim == 64 ? fr::paged_append_kernel<64, Pages> : fr::paged_append_kernel<128, Pages>;
    return launch_plain(fn, (unsigned)grid, fr::kPagedThreads, 0, s,
                        static_cast<const fr::PagedAppendParams>(p));
}

}  // namespace

extern "C" {

int fr_qkv_rope_append_paged(const void* q, const void* k, const void* v, void* q_out, void* k_out,
                             void* v_out, const long long* token_strides, const void* q_bias,
                             const void* k_bias, const void* v_bias, const float* cos_tab,
                             const float* sin_tab, int table_rows, const int* positions,
                             int num_axes, const unsigned char* freq_axis, const long long* slots,
                             void* k_pages, void* v_pages, int page_size, int num_pages,
                             int num_tokens, int num_heads, int num_kv_heads, int head_dim,
                             void* stream) {
    if (!k_pages || !v_pages || page_size <= 0 || page_size % kPageRows != 0 || num_pages <= 0)
        return FR_ERR_INVALID_ARG;
    fr::PagedAppendParams p;
    int rc = fill_append(q, k, v, q_out, k_out, v_out, token_strides, q_bias, k_bias, v_bias, cos_tab,
                         sin_tab, table_rows, positions, num_axes, freq_axis, slots, num_tokens,
                         num_heads, num_kv_heads, head_dim, &p);
    if (rc != FR_OK) return rc;
    if (!aligned(k_pages, 16) || !aligned(v_pages, 16)) return FR_ERR_MISALIGNED;
    if (num_tokens == 0) return FR_OK;
    p.pages[0] = static_cast<__half*>(k_pages);
    p.pages[1] = static_cast<__half*>(v_pages);
    p.pool = (long long)num_pages * page_size;
    return guarded([&]() -> int {
        return run_append<fr::HalfPages>(p, head_dim, static_cast<cudaStream_t>(stream));
    });
}

int fr_qkv_rope_append_kv4(const void* q, const void* k, const void* v, void* q_out, void* k_out,
                           void* v_out, const long long* token_strides, const void* q_bias,
                           const void* k_bias, const void* v_bias, const float* cos_tab,
                           const float* sin_tab, int table_rows, const int* positions,
                           int num_axes, const unsigned char* freq_axis, const long long* slots,
                           const fr_kv4_cache* cache, int num_tokens, int num_heads,
                           void* stream) {
    int rc = check_kv4(cache);
    if (rc != FR_OK) return rc;
    fr::PagedAppendParams p;
    rc = fill_append(q, k, v, q_out, k_out, v_out, token_strides, q_bias, k_bias, v_bias, cos_tab,
                     sin_tab, table_rows, positions, num_axes, freq_axis, slots, num_tokens,
                     num_heads, cache->num_kv_heads, cache->head_dim, &p);
    if (rc != FR_OK) return rc;
    if (num_tokens == 0) return FR_OK;
    p.cache = kv4_view(cache);
    p.pool = (long long)cache->num_pages * cache->page_size;
    return guarded([&]() -> int {
        return run_append<fr::Kv4Pages>(p, cache->head_dim, static_cast<cudaStream_t>(stream));
    });
}

int fr_kv4_gather(const fr_kv4_cache* cache, const long long* slots, void* k_out, void* v_out,
                  int num_slots, void* stream) {
    if (!slots || (!k_out && !v_out) || num_slots < 0) return FR_ERR_INVALID_ARG;
    int rc = check_kv4(cache);
    if (rc != FR_OK) return rc;
    if (!aligned(slots, 8) || !aligned(k_out, 16) || !aligned(v_out, 16)) return FR_ERR_MISALIGNED;
    if (num_slots == 0) return FR_OK;
    return guarded([&]() -> int {
        fr::Kv4GatherParams p;
        p.cache = kv4_view(cache);
        p.slots = slots;
        p.k_out = static_cast<__half*>(k_out);
        p.v_out = static_cast<__half*>(v_out);
        const long long rows = (long long)num_slots * cache->num_kv_heads;
        if (rows >= 1LL << 31) return FR_ERR_INVALID_ARG;
        p.rows = (uint32_t)rows;
        const int per_cta = 256 / (cache->head_dim / 16);
        const long long grid = (rows + per_cta - 1) / per_cta;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        auto fn = cache->head_dim == 64 ? fr::kv4_gather_kernel<64> : fr::kv4_gather_kernel<128>;
        return launch_plain(fn, (unsigned)grid, 256, 0, s, static_cast<const fr::Kv4GatherParams>(p));
    });
}

int fr_decode_attn_paged_kv4(const void* q, long long q_stride, const fr_kv4_cache* cache,
                             const int* block_table, const int* kv_lens, void* out, int batch,
                             int num_heads, int max_blocks_per_seq, int max_kv_len,
                             void* stream) {
    if (!q || !block_table || !kv_lens || !out || batch <= 0 || max_blocks_per_seq <= 0 ||
        max_kv_len < 0 || max_kv_len >= (1 << 30))
        return FR_ERR_INVALID_ARG;
    int rc = check_kv4(cache);
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
        return run_kv4(q, q_stride, cache, block_table, kv_lens, out, batch, num_heads,
                       max_blocks_per_seq, max_kv_len, static_cast<cudaStream_t>(stream));
    });
}

size_t fr_kv4_workspace_size(int batch, int num_heads, int num_kv_heads, int head_dim,
                             int max_kv_len) {
    if (batch <= 0 || max_kv_len < 0 || max_kv_len >= (1 << 30) ||
        check_heads(num_heads, num_kv_heads, head_dim) != FR_OK)
        return 0;
    size_t bytes = 0;
    guarded([&]() -> int {
        DeviceState* st = nullptr;
        CachedPlan pl;
        int rc = get_state(&st);
        if (rc == FR_OK)
            rc = kv4_plan(st, batch, num_heads, num_kv_heads, head_dim, std::max(1, max_kv_len), &pl);
        if (rc == FR_OK) bytes = pl.ws_bytes;
        return rc;
    });
    return bytes;
}

}  // extern "C"
