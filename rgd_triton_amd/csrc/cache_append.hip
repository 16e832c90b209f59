// Appending new tokens to a paged key/value cache: q and k of every new token are rotated at the token's position in its
// sequence (optionally after a LayerNorm over the head dim), q goes to an output, k and v to their slots of the cache.
//
//   pos = cache_lens[b] + t,  slot = (page_table[b][pos / page_size], pos % page_size)
//   y_c = x_c cos[pos][c] + rot(x)_c sin[pos][c] for c < R and pos < cutoff, x_c elsewhere;  rot(x)_(2i, 2i+1) = (-x_(2i+1), x_2i)
//
// Bound by memory: every new row is read once and written once.  A row of D <= 128 elements belongs to G consecutive lanes,
// VEC elements each (16 bytes where pointers and strides allow), so a rotary pair stays inside a lane and the row's mean and
// variance are sums over G lanes.  Statistics and rotation are fp32, rounded once to the tensor type.
#include "common.h"

#include <string.h>

namespace {

struct AppendRows {  // one of q, k, v
    const void* x;
    void* y;             // q: output (batch, head, token); k, v: cache (page, head, slot)
    int64_t sx[3], sy[3];  // (batch, head, token) and (batch or page, head, token or slot)
    uint32_t rows, heads, n_inner;
    FastDiv div_b, div_inner;  // by heads * T and by the inner extent
    int token_inner;
    int cutoff;
};

struct AppendParams {
    AppendRows t[3];
    uint32_t blocks_q, blocks_k;  // row blocks of q, then of k, then of v
    int D, T, R;
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
    int pe_dtype;
};

template <typename T, int G, int VEC, bool VECTOR, bool LN>
__global__ __launch_bounds__(256) void cache_append_kernel(const AppendParams p) {
    constexpr int ROWS = 256 / G;
    const int which = blockIdx.x < p.blocks_q ? 0 : (blockIdx.x < p.blocks_q + p.blocks_k ? 1 : 2);
    const AppendRows& a = p.t[which];
    const uint32_t block0 = which == 0 ? 0u : (which == 1 ? p.blocks_q : p.blocks_q + p.blocks_k);
    const uint32_t row = (blockIdx.x - block0) * ROWS + threadIdx.x / G;
    if (row >= a.rows) return;  // whole lane groups leave: the reductions below stay inside a group
    const int first = (threadIdx.x % G) * VEC;
    const int D = p.D;

    const uint32_t b = fast_div(row, a.div_b);
    const uint32_t in_b = row - b * a.div_b.d;
    const uint32_t outer = fast_div(in_b, a.div_inner);
    const uint32_t inner = in_b - outer * a.div_inner.d;
    const uint32_t head = a.token_inner ? outer : inner;
    const uint32_t tok = a.token_inner ? inner : outer;

    Chunk<T, VEC, VECTOR> c;
    c.load(static_cast<const T*>(a.x) + b * a.sx[0] + head * a.sx[1] + tok * a.sx[2], first, D);
    const int64_t pos = static_cast<int64_t>(p.cache_lens[b]) + tok;
    const bool live = pos >= 0 && pos < p.capacity && (!p.new_lens || static_cast<int>(tok) < p.new_lens[b]);
    T* y = static_cast<T*>(a.y);
    if (which == 0) {
        y += b * a.sy[0] + head * a.sy[1] + tok * a.sy[2];
    } else {
        if (!live) return;
        const uint32_t entry = fast_div(static_cast<uint32_t>(pos), p.div_page);
        const int page = p.page_table[b * p.table_stride + entry];
        if (page < 0 || page >= p.num_pages) return;  // no such page: the token is not stored
        const uint32_t slot = static_cast<uint32_t>(pos) - entry * p.div_page.d;
        y += page * a.sy[0] + head * a.sy[1] + slot * a.sy[2];
    }
    float x[VEC];
    c.decode(first, D, x);
    if (!live) {  // a padded query row
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = 0.f;
        store_chunk<T, VEC, VECTOR>(y, first, D, x);
        return;
    }
    if (which != 2) {
        if constexpr (LN) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += x[e];
            const float mean = group_reduce<G>(s) * p.inv_d;
            s = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x[e] -= mean;
                s += first + e < D ? x[e] * x[e] : 0.f;
            }
            const float rstd = rsqrtf(group_reduce<G>(s) * p.inv_d + p.eps);
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] *= rstd;
        }
        if (first < p.R && pos < a.cutoff) {
            const int ps = p.pe_dtype == RGD_F32 ? 4 : 2;
            const char* sn = static_cast<const char*>(p.pe) + pos * p.pe_sn * ps;
            float sin[VEC], cos[VEC], out[VEC];
            load_chunk_dyn<VEC, VECTOR>(sn, p.pe_dtype, first, p.R, sin);
            load_chunk_dyn<VEC, VECTOR>(sn + p.pe_ss * ps, p.pe_dtype, first, p.R, cos);
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                out[e] = x[e] * cos[e] - x[e + 1] * sin[e];
                out[e + 1] = x[e + 1] * cos[e + 1] + x[e] * sin[e + 1];
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = first + e < p.R ? out[e] : x[e];
        }
    }
    store_chunk<T, VEC, VECTOR>(y, first, D, x);
}

bool vec_ok(const rgd_tensor4* t) {
    return rgd_aligned16(t->ptr) && t->stride_b % 8 == 0 && t->stride_h % 8 == 0 && t->stride_n % 8 == 0;
}

template <typename T, int G, int VEC, bool VECTOR>
int append_launch(AppendParams& p, bool ln, hipStream_t s) {
    const uint32_t rows = 256 / G;
    uint32_t blocks[3];
    for (int i = 0; i < 3; ++i) blocks[i] = (p.t[i].rows + rows - 1) / rows;
    p.blocks_q = blocks[0];
    p.blocks_k = blocks[1];
    const dim3 grid(blocks[0] + blocks[1] + blocks[2]);
    const hipError_t e = ln ? rgd_launch(cache_append_kernel<T, G, VEC, VECTOR, true>, grid, dim3(256), 0, s, p)
                            : rgd_launch(cache_append_kernel<T, G, VEC, VECTOR, false>, grid, dim3(256), 0, s, p);
    return rgd_launch_status("rgd_rope_cache_append", e);
}

template <typename T> int append_dispatch(AppendParams& p, bool vector, bool ln, hipStream_t s) {
    if (!vector) return append_launch<T, 64, 2, false>(p, ln, s);
    if (p.D <= 32) return append_launch<T, 4, 8, true>(p, ln, s);
    if (p.D <= 64) return append_launch<T, 8, 8, true>(p, ln, s);
    return append_launch<T, 16, 8, true>(p, ln, s);
}

}  // namespace

extern "C" int rgd_rope_cache_append(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, const rgd_tensor4* q,
                                     const rgd_tensor4* k, const rgd_tensor4* v, const rgd_tensor4* qo,
                                     const rgd_tensor4* k_cache, const rgd_tensor4* v_cache, int64_t num_pages,
                                     int64_t page_size, const int32_t* page_table, int64_t max_pages, int64_t table_stride,
                                     const int32_t* cache_lens, const int32_t* new_lens, const void* pos_emb, int64_t P,
                                     int64_t R, int64_t pe_stride_s, int64_t pe_stride_n, int pe_dtype, int64_t q_cutoff,
                                     int64_t k_cutoff, int layer_norm, float eps, int dtype, void* stream) {
    const char* name = "rgd_rope_cache_append";
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
    memset(&p, 0, sizeof(p));
    const rgd_tensor4* xs[3] = {q, k, v};
    const rgd_tensor4* ys[3] = {qo, k_cache, v_cache};
    bool vector = D % 8 == 0;
    for (int i = 0; i < 3; ++i) {
        AppendRows& a = p.t[i];
        const int64_t heads = i == 0 ? Hq : Hkv;
        a.div_b = a.div_inner = make_fastdiv(1);
        if (heads == 0 || (i && num_pages == 0)) continue;
        RGD_REQUIRE(xs[i] && xs[i]->ptr && ys[i] && ys[i]->ptr, RGD_ERR_INVALID, "%s: null tensor", name);
        a.x = xs[i]->ptr;
        a.y = ys[i]->ptr;
        a.sx[0] = xs[i]->stride_b, a.sx[1] = xs[i]->stride_h, a.sx[2] = xs[i]->stride_n;
        a.sy[0] = ys[i]->stride_b, a.sy[1] = ys[i]->stride_h, a.sy[2] = ys[i]->stride_n;
        // rows in memory order of the input: the index with the smaller stride is the inner one
        a.token_inner = xs[i]->stride_n <= xs[i]->stride_h;
        a.rows = (uint32_t)(B * heads * T);
        a.heads = (uint32_t)heads;
        a.div_b = make_fastdiv((uint32_t)(heads * T));
        a.div_inner = make_fastdiv((uint32_t)(a.token_inner ? T : heads));
        const int64_t cutoff = i == 0 ? q_cutoff : k_cutoff;
        a.cutoff = (int)(cutoff < 0 ? 0 : (cutoff < lim - 1 ? cutoff : lim - 1));
        vector = vector && vec_ok(xs[i]) && vec_ok(ys[i]);
    }
    if (R > 0) {  // the table is read with the same width as the tensors
        const int64_t ps = rgd_dtype_size(pe_dtype);
        vector = vector && rgd_aligned16(pos_emb) && (pe_stride_s * ps) % 16 == 0 && (pe_stride_n * ps) % 16 == 0 && R % 8 == 0;
    }
    p.D = (int)D;
    p.T = (int)T;
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
    p.pe_dtype = pe_dtype;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == RGD_F16 ? append_dispatch<f16_t>(p, vector, layer_norm != 0, s)
                            : append_dispatch<bf16_t>(p, vector, layer_norm != 0, s);
}
