// Appending new tokens to a paged key/value cache: q and k of every new token are rotated at the token's position in its
// sequence (optionally after a LayerNorm over the head dim), q goes to an output, k and v to their slots of the cache.
//
//   pos = cache_lens[b] + t,  slot = (page_table[b][pos / page_size], pos % page_size)
//   y_c = x_c cos[pos][c] + rot(x)_c sin[pos][c] for c < R and pos < cutoff, x_c elsewhere;  rot(x)_(2i, 2i+1) = (-x_(2i+1), x_2i)
//
// Bound by memory: every new row is read once and written once.  A row of D <= 128 elements belongs to G consecutive lanes, 8
// elements each, so a rotary pair stays inside a lane and the row's mean and variance are sums over G lanes.  The last lane's
// 8 begin at D - 8 where D is no multiple of 8 (where D is even it writes some elements a second time, the same); accesses are 16 bytes at any
// address, which the hardware takes.  Statistics and rotation are fp32, rounded once to the tensor type.
// A lane group takes U = 2 heads of one token: their rows are in flight together, and the token's length, page number, sine
// and cosine, each a round trip behind the other, are read once for both.  U = 1 / 2 / 4 / 8: 8 prompts of 4096 tokens (32 and
// 8 heads, D = 128, bf16, fp32 table) 166 / 144 / 143 / 151 us (839 MB: 5.8 TB/s, a large copy reaches 5.4), one token each
// of 256 sequences 5.1 / 5.2 / 5.8 / 7.4 us.  Streaming loads gain 2 % there and cost 13 % on rows that are still cached.
#include "common.h"

#include <string.h>

namespace {

constexpr int APPEND_HEADS = 2;  // heads of a token that a lane group takes (U above)

struct AppendRows {  // one of q, k, v
    const void* x;
    void* y;             // q: output (batch, head, token); k, v: cache (page, head, slot)
    int64_t sx[3], sy[3];  // (batch, head, token) and (batch or page, head, token or slot)
    uint32_t groups, heads;    // (sequence, token, U heads)
    FastDiv div_b, div_inner;  // by the groups of a sequence and by the inner extent
    int token_inner;
    int cutoff;
};

struct AppendParams {
    AppendRows t[3];
    uint32_t blocks_q, blocks_k;  // row blocks of q, then of k, then of v
    int D, R;
    float inv_d, eps;
    const int32_t* page_table;
    const int32_t* cache_lens;
    const int32_t* new_lens;
    int64_t table_stride;
    int64_t capacity;  // positions a page table row covers
    int num_pages;
    FastDiv div_page;
    const void* pe;
    int64_t pe_ss, pe_sn;
};

typedef u32x4 u32x4_any __attribute__((aligned(2)));

// N elements of a row from `at` on as floats.  WIDE: 16-byte loads at any address; else element by element, those beyond `limit`
// repeat the last.
template <typename T, int N, bool WIDE> __device__ __forceinline__ void load_row(const T* row, int at, int limit, T (&out)[N]) {
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < N * (int)sizeof(T) / 16; ++i) {
            const u32x4 v = reinterpret_cast<const u32x4_any*>(row + at)[i];
            __builtin_memcpy(reinterpret_cast<char*>(out) + 16 * i, &v, 16);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) out[e] = row[min(at + e, limit - 1)];
    }
}

template <typename TP, int N, bool WIDE> __device__ __forceinline__ void load_table(const void* row, int at, int R, float (&out)[N]) {
    TP v[N];
    if (WIDE && at + N <= R) load_row<TP, N, true>(static_cast<const TP*>(row), at, R, v);
    else load_row<TP, N, false>(static_cast<const TP*>(row), at, R, v);  // (the rotary dim ends inside the lane's elements)
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = to_f32(v[e]);
}

// TP: element type of the rotary table.  WIDE: D >= 8 and 8 elements a lane; else 2, element by element.
template <typename T, typename TP, int G, bool WIDE, bool LN>
__global__ __launch_bounds__(256) void cache_append_kernel(const AppendParams p) {
    constexpr int GROUPS = 256 / G, VEC = WIDE ? 8 : 2, U = APPEND_HEADS;
    const int which = blockIdx.x < p.blocks_q ? 0 : (blockIdx.x < p.blocks_q + p.blocks_k ? 1 : 2);
    const AppendRows& a = p.t[which];
    const uint32_t block0 = which == 0 ? 0u : (which == 1 ? p.blocks_q : p.blocks_q + p.blocks_k);
    const uint32_t group = (blockIdx.x - block0) * GROUPS + threadIdx.x / G;
    if (group >= a.groups) return;  // whole lane groups leave: the reductions below stay inside a group
    const int D = p.D;
    const int own = (threadIdx.x % G) * VEC;             // the lane's elements of the row: those from `own` on are no other lane's
    const int first = WIDE ? min(own, D - VEC) : own;    // (WIDE: a lane behind the row's end repeats the last 8)

    const uint32_t b = fast_div(group, a.div_b);
    const uint32_t in_b = group - b * a.div_b.d;
    const uint32_t outer = fast_div(in_b, a.div_inner);
    const uint32_t inner = in_b - outer * a.div_inner.d;
    const uint32_t head0 = (a.token_inner ? outer : inner) * U;
    const uint32_t tok = a.token_inner ? inner : outer;

    // (padding is not read, q's reads the sequence's first row: 8 prompts half of padding 133 -> 110 us, without new_lens 141.5 -> 142.4)
    bool live = !p.new_lens || static_cast<int>(tok) < p.new_lens[b];
    if (!live && which != 0) return;
    const T* from = static_cast<const T*>(a.x) + b * a.sx[0] + (live ? tok : 0u) * a.sx[2];
    T raw[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) load_row<T, VEC, WIDE>(from + min(head0 + u, a.heads - 1) * a.sx[1], first, D, raw[u]);
    const int64_t pos = static_cast<int64_t>(p.cache_lens[b]) + tok;
    live = live && pos >= 0 && pos < p.capacity;
    T* y = static_cast<T*>(a.y);
    const bool turn = which != 2 && live && first < p.R && pos < a.cutoff;
    float sin[VEC], cos[VEC];
    if (turn) {
        const TP* row = static_cast<const TP*>(p.pe) + pos * p.pe_sn;
        load_table<TP, VEC, WIDE>(row, first, p.R, sin);
        load_table<TP, VEC, WIDE>(row + p.pe_ss, first, p.R, cos);
    }
    if (which == 0) {
        y += b * a.sy[0] + tok * a.sy[2];
    } else {
        if (!live) return;
        const uint32_t entry = fast_div(static_cast<uint32_t>(pos), p.div_page);
        const int page = p.page_table[b * p.table_stride + entry];
        if (page < 0 || page >= p.num_pages) return;  // no such page: the token is not stored
        const uint32_t slot = static_cast<uint32_t>(pos) - entry * p.div_page.d;
        y += page * a.sy[0] + slot * a.sy[2];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = to_f32(raw[u][e]);
        if (LN && which != 2) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += first + e >= own && first + e < D ? x[e] : 0.f;
            const float mean = group_reduce<G>(s) * p.inv_d;
            s = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x[e] -= mean;
                s += first + e >= own && first + e < D ? x[e] * x[e] : 0.f;
            }
            const float rstd = rsqrtf(group_reduce<G>(s) * p.inv_d + p.eps);
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] *= rstd;
        }
        if (turn) {
            float out[VEC];
            if (WIDE && (D & 1)) {  // the last lane's elements begin at an odd channel: pairs by the channel's parity
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float even = x[e] * cos[e] - (e + 1 < VEC ? x[e + 1] : 0.f) * sin[e];
                    const float odd = x[e] * cos[e] + (e > 0 ? x[e - 1] : 0.f) * sin[e];
                    out[e] = (first + e) & 1 ? odd : even;
                }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    out[e] = x[e] * cos[e] - x[e + 1] * sin[e];
                    out[e + 1] = x[e + 1] * cos[e + 1] + x[e] * sin[e + 1];
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = first + e < p.R ? out[e] : x[e];
        }
        if (head0 + u < a.heads && own < D) {
            T* to = y + (head0 + u) * a.sy[1] + first;
            T out[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) out[e] = from_f32<T>(live ? x[e] : 0.f);  // (a padded query row is zero)
            if (WIDE && !(first & 1)) {
                u32x4 v;
                __builtin_memcpy(&v, out, VEC * sizeof(T));
                *reinterpret_cast<u32x4_any*>(to) = v;
            } else {  // (from an odd channel on the first element's partner is missing: only the lane's own are written)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (first + e >= own && first + e < D) to[e] = out[e];
            }
        }
    }
}

template <typename T, typename TP, int G, bool WIDE>
int append_launch(AppendParams& p, int64_t B, int64_t tokens, bool ln, hipStream_t s) {
    uint32_t blocks[3];
    for (int i = 0; i < 3; ++i) {
        AppendRows& a = p.t[i];
        const uint32_t chunks = (a.heads + APPEND_HEADS - 1) / APPEND_HEADS;
        a.groups = (uint32_t)(B * tokens * chunks);
        a.div_b = make_fastdiv((uint32_t)(tokens * chunks));
        a.div_inner = make_fastdiv(a.token_inner ? (uint32_t)tokens : chunks);
        blocks[i] = (a.groups + 256 / G - 1) / (256 / G);
    }
    p.blocks_q = blocks[0];
    p.blocks_k = blocks[1];
    const uint64_t all = (uint64_t)blocks[0] + blocks[1] + blocks[2];
    if (all == 0) return RGD_OK;
    RGD_REQUIRE(all < (1u << 24), RGD_ERR_UNSUPPORTED, "rgd_rope_cache_append: more rows than one launch takes");  // 2^32 threads
    const dim3 grid((unsigned)all);
    const hipError_t e = ln ? rgd_launch(cache_append_kernel<T, TP, G, WIDE, true>, grid, dim3(256), 0, s, p)
                            : rgd_launch(cache_append_kernel<T, TP, G, WIDE, false>, grid, dim3(256), 0, s, p);
    return rgd_launch_status("rgd_rope_cache_append", e);
}

template <typename T, typename TP> int append_dispatch(AppendParams& p, int64_t B, int64_t tokens, bool ln, hipStream_t s) {
    if (p.D < 8) return append_launch<T, TP, 4, false>(p, B, tokens, ln, s);
    if (p.D <= 32) return append_launch<T, TP, 4, true>(p, B, tokens, ln, s);
    if (p.D <= 64) return append_launch<T, TP, 8, true>(p, B, tokens, ln, s);
    return append_launch<T, TP, 16, true>(p, B, tokens, ln, s);
}

}  // namespace

extern "C" int rgd_rope_cache_append(const rgd_cache_append_args* args, void* stream) {
    const char* name = "rgd_rope_cache_append";
    RGD_REQUIRE(args, RGD_ERR_INVALID, "%s: null arguments", name);
    const auto& [B, T, Hq, Hkv, D, q, k, v, qo, k_cache, v_cache, num_pages, page_size, page_table, max_pages, table_stride,
                 cache_lens, new_lens, pos_emb, P, R, pe_stride_s, pe_stride_n, q_cutoff, k_cutoff, pe_dtype, layer_norm, dtype,
                 eps] = *args;
    rgd_ensure_init();
    RGD_REQUIRE(dtype == RGD_F16 || dtype == RGD_BF16, RGD_ERR_INVALID, "%s: Only support fp16 and bf16", name);
    RGD_REQUIRE(B >= 0 && T >= 0 && Hq >= 0 && Hkv >= 0 && num_pages >= 0 && max_pages >= 0, RGD_ERR_INVALID,
                "%s: negative shape", name);
    RGD_REQUIRE(D >= 1 && D <= 128, RGD_ERR_INVALID, "%s: Only supports head dimensions up to 128", name);
    RGD_REQUIRE(page_size >= 1, RGD_ERR_INVALID, "%s: page size must be positive", name);
    const int64_t lim = int64_t(1) << 31;
    RGD_REQUIRE(num_pages < lim && page_size < lim && max_pages < lim && max_pages * page_size <= lim - 1024, RGD_ERR_UNSUPPORTED,
                "%s: more than 2^31 positions or pages", name);
    RGD_REQUIRE(B < lim && T < lim && Hq < lim && Hkv < lim, RGD_ERR_UNSUPPORTED, "%s: more than 2^31 rows", name);
    if (B == 0 || T == 0 || Hq + Hkv == 0) return RGD_OK;
    RGD_REQUIRE(B * T < lim && B * T * (Hq > Hkv ? Hq : Hkv) < lim, RGD_ERR_UNSUPPORTED, "%s: more than 2^31 rows", name);
    RGD_REQUIRE(cache_lens && (page_table || max_pages == 0), RGD_ERR_INVALID, "%s: null page table or lengths", name);
    RGD_REQUIRE(R >= 0 && R <= D && R % 2 == 0, RGD_ERR_INVALID, "%s: rotary dim %lld must be even and at most the head dim",
                name, (long long)R);
    RGD_REQUIRE(R == 0 || (pos_emb && rgd_dtype_ok(pe_dtype)), RGD_ERR_INVALID, "%s: bad pos_emb", name);
    RGD_REQUIRE(R == 0 || pe_dtype == dtype || pe_dtype == RGD_F32, RGD_ERR_UNSUPPORTED,
                "%s: pos_emb must have the dtype of the tensors or fp32", name);
    RGD_REQUIRE(R == 0 || P >= max_pages * page_size, RGD_ERR_INVALID,
                "%s: pos_emb must cover every position of the page table", name);

    AppendParams p;
    memset(&p, 0, sizeof(p));  // (heads 0: nothing to do for a tensor)
    const rgd_tensor4* xs[3] = {&q, &k, &v};
    const rgd_tensor4* ys[3] = {&qo, &k_cache, &v_cache};
    for (int i = 0; i < 3; ++i) {
        AppendRows& a = p.t[i];
        const int64_t heads = i == 0 ? Hq : Hkv;
        if (heads == 0 || (i && num_pages == 0)) continue;
        RGD_REQUIRE(xs[i]->ptr && ys[i]->ptr, RGD_ERR_INVALID, "%s: null tensor", name);
        a.x = xs[i]->ptr;
        a.y = ys[i]->ptr;
        a.sx[0] = xs[i]->stride_b, a.sx[1] = xs[i]->stride_h, a.sx[2] = xs[i]->stride_n;
        a.sy[0] = ys[i]->stride_b, a.sy[1] = ys[i]->stride_h, a.sy[2] = ys[i]->stride_n;
        // rows in memory order of the input: the index with the smaller stride is the inner one
        a.token_inner = xs[i]->stride_n <= xs[i]->stride_h;
        a.heads = (uint32_t)heads;
        const int64_t cutoff = i == 0 ? q_cutoff : k_cutoff;
        a.cutoff = (int)(cutoff < 0 ? 0 : (cutoff < lim - 1 ? cutoff : lim - 1));
    }
    p.D = (int)D;
    p.R = (int)R;
    p.inv_d = 1.0f / (float)D;
    p.eps = eps;
    p.page_table = page_table;
    p.cache_lens = cache_lens;
    p.new_lens = new_lens;
    p.table_stride = table_stride;
    p.capacity = max_pages * page_size;
    p.num_pages = (int)num_pages;
    p.div_page = make_fastdiv((uint32_t)page_size);
    p.pe = pos_emb;
    p.pe_ss = pe_stride_s;
    p.pe_sn = pe_stride_n;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool ln = layer_norm != 0, wide = pe_dtype == RGD_F32;
    if (dtype == RGD_F16) return wide ? append_dispatch<f16_t, float>(p, B, T, ln, s) : append_dispatch<f16_t, f16_t>(p, B, T, ln, s);
    return wide ? append_dispatch<bf16_t, float>(p, B, T, ln, s) : append_dispatch<bf16_t, bf16_t>(p, B, T, ln, s);
}
