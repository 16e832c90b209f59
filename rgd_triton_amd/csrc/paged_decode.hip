// Attention of one new token per sequence over a paged key/value cache.
//
//   s_j = softmax_scale q . k_j (+ W[bucket(j - (len - 1))][h]),  o = sum_j softmax(s)_j v_j,  lse = log sum_j exp(s_j)
//
// Simple form: a workgroup per (sequence, query head), a wavefront per key in turn, one pass with a running maximum and sum.
#include "common.h"

#include <string.h>

namespace {

constexpr int MAX_RANGES = 256;

struct DecodeParams {
    const void* q;
    const void* k;
    const void* v;
    void* o;
    float* lse;
    int64_t sq[2], so[2], sk[3], sv[3];  // (batch, head); (page, head, slot)
    const int32_t* page_table;
    const int32_t* seq_lens;
    int64_t table_stride;
    int64_t capacity;
    int B, Hq, group, D, num_pages;
    FastDiv div_page;
    float scale;
    const void* w;  // (buckets, Hq) or null
    int64_t w_stride;
    int w_dtype, n_ranges;
    int start[MAX_RANGES], bucket[MAX_RANGES];
};

__device__ __forceinline__ float load_dyn(const void* p, int dtype, int64_t i) {
    if (dtype == RGD_BF16) return to_f32(static_cast<const bf16_t*>(p)[i]);
    if (dtype == RGD_F16) return to_f32(static_cast<const f16_t*>(p)[i]);
    return static_cast<const float*>(p)[i];
}

template <typename T> __global__ __launch_bounds__(256) void paged_decode_kernel(const DecodeParams p) {
    __shared__ float sm[4], sl[4], so[4][128];
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    const int b = blockIdx.x / p.Hq, h = blockIdx.x % p.Hq;
    const int hk = h / p.group;
    const int D = p.D;
    const int64_t want = p.seq_lens[b];
    const int len = (int)(want < 0 ? 0 : (want < p.capacity ? want : p.capacity));
    const T* q = static_cast<const T*>(p.q) + b * p.sq[0] + h * p.sq[1];
    const int d0 = lane * 2, d1 = lane * 2 + 1;
    const float q0 = d0 < D ? to_f32(q[d0]) : 0.f, q1 = d1 < D ? to_f32(q[d1]) : 0.f;
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int j = wave; j < len; j += 4) {
        const uint32_t entry = fast_div(j, p.div_page);
        const int page = p.page_table[b * p.table_stride + entry];
        if (page < 0 || page >= p.num_pages) continue;  // no such page: the key is absent
        const uint32_t slot = j - entry * p.div_page.d;
        const T* k = static_cast<const T*>(p.k) + page * p.sk[0] + hk * p.sk[1] + slot * p.sk[2];
        const T* v = static_cast<const T*>(p.v) + page * p.sv[0] + hk * p.sv[1] + slot * p.sv[2];
        float s = (d0 < D ? q0 * to_f32(k[d0]) : 0.f) + (d1 < D ? q1 * to_f32(k[d1]) : 0.f);
        s = group_reduce<64>(s) * p.scale;
        if (p.w) {
            const int d = j - (len - 1);
            int r = 0;
            while (r + 1 < p.n_ranges && d >= p.start[r + 1]) ++r;
            s += load_dyn(p.w, p.w_dtype, p.bucket[r] * p.w_stride + h);
        }
        const float nm = fmaxf(m, s);
        const float ref = nm == -INFINITY ? 0.f : nm;
        const float alpha = expf(m - ref), e = expf(s - ref);
        l = l * alpha + e;
        o0 = o0 * alpha + e * (d0 < D ? to_f32(v[d0]) : 0.f);
        o1 = o1 * alpha + e * (d1 < D ? to_f32(v[d1]) : 0.f);
        m = nm;
    }
    sm[wave] = m;
    sl[wave] = l;
    so[wave][d0] = o0;
    so[wave][d1] = o1;
    __syncthreads();
    if (wave == 0) {
        float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
        const float ref = top == -INFINITY ? 0.f : top;
        float total = 0.f, a0 = 0.f, a1 = 0.f;
        for (int w = 0; w < 4; ++w) {
            const float f = expf(sm[w] - ref);
            total += f * sl[w];
            a0 += f * so[w][d0];
            a1 += f * so[w][d1];
        }
        const float inv = total == 0.f ? 0.f : 1.0f / total;
        T* o = static_cast<T*>(p.o) + b * p.so[0] + h * p.so[1];
        if (d0 < D) o[d0] = from_f32<T>(a0 * inv);
        if (d1 < D) o[d1] = from_f32<T>(a1 * inv);
        if (p.lse && lane == 0) p.lse[(int64_t)b * p.Hq + h] = total == 0.f ? -INFINITY : ref + logf(total);
    }
}

}  // namespace

extern "C" {

size_t rgd_paged_decode_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
    (void)B, (void)Hq, (void)Hkv, (void)D;
    return 0;
}

int rgd_paged_decode(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const rgd_tensor4* q, const rgd_tensor4* k_cache,
                     const rgd_tensor4* v_cache, int64_t num_pages, int64_t page_size, const int32_t* page_table,
                     int64_t max_pages, int64_t table_stride, const int32_t* seq_lens, const void* rel_weight, int64_t w_stride,
                     int64_t num_buckets, int w_dtype, int64_t n_ranges, const int32_t* starts, const int32_t* buckets,
                     const rgd_tensor4* o, float* lse, int dtype, float softmax_scale, void* workspace, size_t workspace_bytes,
                     void* stream) {
    const char* name = "rgd_paged_decode";
    rgd_ensure_init();
    RGD_REQUIRE(dtype == RGD_F16 || dtype == RGD_BF16, RGD_ERR_INVALID, "%s: Only support fp16 and bf16", name);
    RGD_REQUIRE(B >= 0 && Hq >= 0 && Hkv >= 0 && num_pages >= 0 && max_pages >= 0, RGD_ERR_INVALID, "%s: negative shape", name);
    RGD_REQUIRE(D >= 1 && D <= 128, RGD_ERR_INVALID, "%s: Only supports head dimensions up to 128", name);
    RGD_REQUIRE(page_size >= 1, RGD_ERR_INVALID, "%s: page size must be positive", name);
    const int64_t lim = int64_t(1) << 31;
    RGD_REQUIRE(num_pages < lim && page_size < lim && max_pages < lim && max_pages * page_size < lim, RGD_ERR_UNSUPPORTED,
                "%s: more than 2^31 positions or pages", name);
    RGD_REQUIRE(B < lim && Hq < lim && B * Hq < lim, RGD_ERR_UNSUPPORTED, "%s: more than 2^31 rows", name);
    if (B == 0 || Hq == 0) return RGD_OK;
    RGD_REQUIRE(Hkv >= 1 && Hq % Hkv == 0, RGD_ERR_INVALID, "%s: query heads must be a multiple of the key heads", name);
    const bool none = num_pages == 0 || max_pages == 0;  // no key can exist
    RGD_REQUIRE(seq_lens && (none || (page_table && k_cache && k_cache->ptr && v_cache && v_cache->ptr)), RGD_ERR_INVALID,
                "%s: null cache, page table or lengths", name);
    RGD_REQUIRE(q && q->ptr && o && o->ptr, RGD_ERR_INVALID, "%s: null tensor", name);
    DecodeParams p;
    memset(&p, 0, sizeof(p));
    if (rel_weight) {
        RGD_REQUIRE(rgd_dtype_ok(w_dtype), RGD_ERR_INVALID, "%s: Only support fp16, bf16, and fp32 bias weights", name);
        RGD_REQUIRE(n_ranges >= 1 && n_ranges <= MAX_RANGES && starts && buckets, RGD_ERR_INVALID, "%s: 1 to %d ranges", name, MAX_RANGES);
        for (int64_t i = 0; i < n_ranges; ++i) {
            RGD_REQUIRE(buckets[i] >= 0 && buckets[i] < num_buckets, RGD_ERR_INVALID, "%s: a bucket outside the weight", name);
            p.start[i] = starts[i];
            p.bucket[i] = buckets[i];
        }
        p.w = rel_weight;
        p.w_stride = w_stride;
        p.w_dtype = w_dtype;
        p.n_ranges = (int)n_ranges;
    }
    p.q = q->ptr;
    p.o = o->ptr;
    p.lse = lse;
    p.sq[0] = q->stride_b, p.sq[1] = q->stride_h;
    p.so[0] = o->stride_b, p.so[1] = o->stride_h;
    if (!none) {
        p.k = k_cache->ptr;
        p.v = v_cache->ptr;
        p.sk[0] = k_cache->stride_b, p.sk[1] = k_cache->stride_h, p.sk[2] = k_cache->stride_n;
        p.sv[0] = v_cache->stride_b, p.sv[1] = v_cache->stride_h, p.sv[2] = v_cache->stride_n;
    }
    p.page_table = page_table;
    p.seq_lens = seq_lens;
    p.table_stride = table_stride;
    p.capacity = none ? 0 : max_pages * page_size;
    p.B = (int)B;
    p.Hq = (int)Hq;
    p.group = (int)(Hq / Hkv);
    p.D = (int)D;
    p.num_pages = (int)num_pages;
    p.div_page = make_fastdiv((uint32_t)page_size);
    p.scale = softmax_scale;
    hipStream_t s = static_cast<hipStream_t>(stream);
    (void)workspace, (void)workspace_bytes;
    const dim3 grid((unsigned)(B * Hq));
    const hipError_t e = dtype == RGD_F16 ? rgd_launch(paged_decode_kernel<f16_t>, grid, dim3(256), 0, s, p)
                                          : rgd_launch(paged_decode_kernel<bf16_t>, grid, dim3(256), 0, s, p);
    return rgd_launch_status(name, e);
}

}  // extern "C"
