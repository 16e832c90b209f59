// Host side of the single-token attention over a paged cache: validation, choice of the kernel variant, entry points.
#include "paged_decode.h"

#include <string.h>

namespace {

int chunks_of(int64_t D) { return (int)((D + 31) / 32); }
// Wavefronts of the decode launch, three per SIMD for head dims up to 64, two above: what the registers of most variants let be
// resident at once (D up to 32, 128 registers, would let four; D = 33 .. 63 with bias, 169, lets two, and a third of the runs waits).
// More wait for their turn and leave more pieces to join, fewer leave loads in flight unused: at 1 / 2 / 3 per SIMD
// (D = 64, 24 heads, 19 lengths to 2000) 44 / 35 / 33 us, (D = 128, 8 key heads, 64 lengths to 4100) 112 / 113 / 117 us,
// (D = 128, 24 heads, 19 lengths to 2000) 58 / 54 / 57 us.
int64_t decode_grid(int64_t D) { return (int64_t)rgd_num_cus() * 4 * (D <= 64 ? 3 : 2); }

template <typename T, int NC, bool SMALL, bool LINES>
int decode_launch(const DecodeParams& p, const DecodeBias* rel, unsigned grid, bool merge, hipStream_t s) {
    const size_t lds = rel ? DEC_NEAR + (rel->half ? 2 * rel->half : 1) * 2 * sizeof(int) + rel->n_ranges * 16 * sizeof(float) : 0;
    const hipError_t e = rel ? rgd_launch(paged_decode_kernel<T, NC, SMALL, LINES, true>, dim3(grid), dim3(64), lds, s, p, *rel)
                             : rgd_launch(paged_decode_kernel<T, NC, SMALL, LINES, false>, dim3(grid), dim3(64), 0, s, p, DecodeNoBias{});
    const int rc = rgd_launch_status("rgd_paged_decode", e);
    if (rc != RGD_OK || !merge) return rc;
    // pieces of a unit, if all units are alike: beyond what the small workgroup keeps in flight at once the large one is faster
    const dim3 heads((unsigned)p.B * (unsigned)p.Hq);
    const bool many = grid / ((int64_t)p.B * p.units << p.bundle_log) > 64;
    return rgd_launch_status("rgd_paged_decode", many ? rgd_launch(paged_decode_merge_kernel<T, NC, SMALL, 1024>, heads, dim3(1024), 0, s, p)
                                                      : rgd_launch(paged_decode_merge_kernel<T, NC, SMALL, 256>, heads, dim3(256), 0, s, p));
}

template <typename T> int decode_dispatch(const DecodeParams& p, const DecodeBias* rel, unsigned grid, bool merge, hipStream_t s) {
    if (p.D < 8) return decode_launch<T, 1, true, false>(p, rel, grid, merge, s);
    if (p.D == 64) return decode_launch<T, 2, false, true>(p, rel, grid, merge, s);
    if (p.D == 128) return decode_launch<T, 4, false, true>(p, rel, grid, merge, s);
    switch (chunks_of(p.D)) {
        case 1: return decode_launch<T, 1, false, false>(p, rel, grid, merge, s);
        case 2: return decode_launch<T, 2, false, false>(p, rel, grid, merge, s);
        case 3: return decode_launch<T, 3, false, false>(p, rel, grid, merge, s);
        default: return decode_launch<T, 4, false, false>(p, rel, grid, merge, s);
    }
}

}  // namespace

extern "C" {

size_t rgd_paged_decode_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || D > 128) return 0;
    const int64_t group = Hq / Hkv, units = Hkv * ((group + 15) / 16), rows = group < 16 ? group : 16;
    const int64_t plan = (B * units * 2 * (int64_t)sizeof(int) + 15) / 16 * 16;
    return (size_t)(plan + 2 * decode_grid(D) * (rows * 32 * chunks_of(D) + 32) * 4);
}

int rgd_paged_decode(const rgd_paged_decode_args* args, void* stream) {
    const char* name = "rgd_paged_decode";
    RGD_REQUIRE(args, RGD_ERR_INVALID, "%s: null arguments", name);
    const auto& [B, Hq, Hkv, D, q, k_cache, v_cache, o, num_pages, page_size, page_table, max_pages, table_stride, seq_lens,
                 rel_weight, w_stride, num_buckets, n_ranges, starts, buckets, lse, workspace, workspace_bytes, w_dtype, dtype,
                 softmax_scale] = *args;
    rgd_ensure_init();
    RGD_REQUIRE(dtype == RGD_F16 || dtype == RGD_BF16, RGD_ERR_INVALID, "%s: Only support fp16 and bf16", name);
    RGD_REQUIRE(B >= 0 && Hq >= 0 && Hkv >= 0 && num_pages >= 0 && max_pages >= 0, RGD_ERR_INVALID, "%s: negative shape", name);
    RGD_REQUIRE(D >= 1 && D <= 128, RGD_ERR_INVALID, "%s: Only supports head dimensions up to 128", name);
    RGD_REQUIRE(page_size >= 1, RGD_ERR_INVALID, "%s: page size must be positive", name);
    const int64_t lim = int64_t(1) << 31;
    RGD_REQUIRE(num_pages < lim && page_size < lim && max_pages < lim && max_pages * page_size <= lim - 1024, RGD_ERR_UNSUPPORTED,
                "%s: more than 2^31 positions or pages", name);
    RGD_REQUIRE(B < lim && Hq < lim && B * Hq < (int64_t(1) << 24), RGD_ERR_UNSUPPORTED, "%s: 2^24 query rows or more", name);
    if (B == 0 || Hq == 0) return RGD_OK;
    RGD_REQUIRE(Hkv >= 1 && Hq % Hkv == 0, RGD_ERR_INVALID, "%s: query heads must be a multiple of the key heads", name);
    const bool none = num_pages == 0 || max_pages == 0;  // no key can exist
    RGD_REQUIRE(seq_lens && (none || (page_table && k_cache.ptr && v_cache.ptr)), RGD_ERR_INVALID,
                "%s: null cache, page table or lengths", name);
    RGD_REQUIRE(q.ptr && o.ptr, RGD_ERR_INVALID, "%s: null tensor", name);
    DecodeParams p;
    memset(&p, 0, sizeof(p));
    DecodeBias rel;
    const DecodeBias* bias = nullptr;
    if (rel_weight) {
        RGD_REQUIRE(rgd_dtype_ok(w_dtype), RGD_ERR_INVALID, "%s: Only support fp16, bf16, and fp32 bias weights", name);
        RGD_REQUIRE(n_ranges >= 1 && n_ranges <= DEC_MAX_RANGES && starts && buckets, RGD_ERR_INVALID, "%s: 1 to %d ranges", name, DEC_MAX_RANGES);
        for (int64_t i = 0; i < n_ranges; ++i) {
            RGD_REQUIRE(buckets[i] >= 0 && buckets[i] < num_buckets, RGD_ERR_INVALID, "%s: a bucket outside the weight", name);
            RGD_REQUIRE(i < 2 || starts[i] > starts[i - 1], RGD_ERR_INVALID, "%s: range starts must ascend", name);
            rel.start[i] = starts[i];
            rel.bucket[i] = buckets[i];
        }
        rel.w = rel_weight;
        rel.w_stride = w_stride;
        rel.w_dtype = w_dtype;
        rel.n_ranges = (int)n_ranges;
        for (rel.half = 0; (rel.half ? 2 * rel.half : 1) < n_ranges;) rel.half = rel.half ? 2 * rel.half : 1;
        uint8_t near[DEC_NEAR];
        for (int n = 0, r = rel.n_ranges - 1; n < DEC_NEAR; ++n) {
            for (; r > 0 && rel.start[r] > -n;) --r;
            near[n] = (uint8_t)r;
        }
        memcpy(rel.near, near, sizeof(near));
        bias = &rel;
    }
    p.q = q.ptr;
    p.o = o.ptr;
    p.lse = lse;
    p.sq[0] = q.stride_b, p.sq[1] = q.stride_h;
    p.so[0] = o.stride_b, p.so[1] = o.stride_h;
    if (!none) {
        p.k = k_cache.ptr;
        p.v = v_cache.ptr;
        p.sk[0] = k_cache.stride_b, p.sk[1] = k_cache.stride_h, p.sk[2] = k_cache.stride_n;
        p.sv[0] = v_cache.stride_b, p.sv[1] = v_cache.stride_h, p.sv[2] = v_cache.stride_n;
    }
    p.page_table = page_table;
    p.seq_lens = seq_lens;
    p.table_stride = table_stride;
    p.capacity = none ? 0 : (int)(max_pages * page_size);
    p.B = (int)B;
    p.Hq = (int)Hq;
    p.group = (int)(Hq / Hkv);
    p.head_tiles = (p.group + 15) / 16;
    p.part_rows = p.group < 16 ? p.group : 16;
    p.D = (int)D;
    p.num_pages = (int)num_pages;
    p.div_page = make_fastdiv((uint32_t)page_size);
    p.scale = softmax_scale;
    hipStream_t s = static_cast<hipStream_t>(stream);
    RGD_REQUIRE(workspace && workspace_bytes >= rgd_paged_decode_workspace(B, Hq, Hkv, D), RGD_ERR_WORKSPACE,
                "%s: workspace of %zu bytes, needs %zu", name, workspace_bytes, rgd_paged_decode_workspace(B, Hq, Hkv, D));
    RGD_REQUIRE(rgd_aligned16(workspace), RGD_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", name);
    p.plan = static_cast<int*>(workspace);
    p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + (B * Hkv * p.head_tiles * 2 * (int64_t)sizeof(int) + 15) / 16 * 16);
    if (none) {
        const dim3 rows((unsigned)(B * Hq));
        return rgd_launch_status(name, dtype == RGD_F16 ? rgd_launch(paged_decode_empty_kernel<f16_t>, rows, dim3(64), 0, s, p)
                                                        : rgd_launch(paged_decode_empty_kernel<bf16_t>, rows, dim3(64), 0, s, p));
    }
    // more wavefronts than there can be tiles have nothing to do; units of one tile are in no two wavefronts
    const int64_t most = p.capacity > DEC_TILE ? (p.capacity + DEC_TILE - 1) / DEC_TILE : 1;
    const int64_t tiles = B * Hkv * p.head_tiles * most;
    const unsigned grid = (unsigned)(tiles < decode_grid(D) ? tiles : decode_grid(D));
    // bundles where rows of neighbouring key heads touch: the fewest heads that end on a line, at most 8 (odd head dims)
    p.bundle_log = 0;
    if (p.sk[1] == D && p.sv[1] == D)
        while (p.bundle_log < 3 && (D * 2 << p.bundle_log) % 128 && Hkv % (2 << p.bundle_log) == 0 && grid % (16 << p.bundle_log) == 0) ++p.bundle_log;
    p.units = (int)(Hkv >> p.bundle_log) * p.head_tiles;
    return dtype == RGD_F16 ? decode_dispatch<f16_t>(p, bias, grid, most > 1, s) : decode_dispatch<bf16_t>(p, bias, grid, most > 1, s);
}

}  // extern "C"
