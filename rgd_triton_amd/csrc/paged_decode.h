// Attention of one new token per sequence over a paged key/value cache.
//
//   s_j = softmax_scale q . k_j (+ W[bucket(j - (len - 1))][h]),  o = sum_j softmax(s)_j v_j,  lse = log sum_j exp(s_j)
//
// Bound by memory: every cached key and value is read once, 4 D bytes per token and key head, for 4 D group operations.
//
// Work.  A unit is (sequence, key head, 16 of the key head's query heads); its keys are cut into tiles of 128.  The tiles of all
// units, in one row, are dealt to the workgroups in equal runs: every workgroup finds its run from the lengths on the GPU, so
// the host need not know them, one long sequence fills the chip like many short ones, and a ragged batch leaves no workgroup
// with more than a tile over the others.  A run that holds a whole unit writes its output; pieces of a unit that several
// workgroups share leave partial results in the workspace (at most two per workgroup: one unit begun earlier, one not ended),
// which the merge launch joins in order.
//
// A step.  Each of the four wavefronts walks every fourth 32 keys on its own, without LDS or barriers, operands straight
// from memory to registers (v_mfma_f32_16x16x32: A lane l holds row l % 16, k = 8 (l / 16) .. + 7; C lane l holds column l % 16,
// rows 4 (l / 16) + 0..3):
//   S^T = K Q^T, two products of 16 keys.  MFMA row i of product a is key 8 (i / 4) + 4 a + i % 4, so that lane group g = l / 16 ends
//   up with the logits of keys 8 g .. 8 g + 7 of query head l % 16: the layout P^T has to have as the second product's B operand.
//   O^T += V^T P^T, one product per element e of a lane's piece of a value row: lane l loads VE = DP / 16 channels from VE (l % 16)
//   on of keys 8 g .. 8 g + 7 (whole rows per load) and pairs them by key with byte permutes; MFMA row m is channel VE m + e.
// So 16 rows of heads are computed whatever the group: at the rate the memory delivers keys the matrix pipe is busy a tenth of
// the time.  P is split into two 16-bit parts (a second product each): rounded to one, its error would be as large as the
// output's own rounding, and the products are free (DEC_HIGH).
// The running maximum is a reference that moves only when a logit exceeds it by LAZY; sums, maxima and outputs are fp32.
#pragma once

#include "attn_common.h"

#include <type_traits>

constexpr int DEC_MAX_RANGES = 256;
constexpr int DEC_TILE = 128;  // keys of a scheduling tile: 4 wavefronts x 32

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
    int32_t capacity;  // positions of a page table row
    int B, Hq, Hkv, group, head_tiles, units;  // units = Hkv * head_tiles, per sequence
    int D, num_pages;
    FastDiv div_page;
    float scale;
    int2* plan;        // per unit of the batch: workgroups its first and last piece are in
    float* part;       // two slots per workgroup: O [rows][DP], then m [16], l [16]
    int part_rows;     // query heads of a slot
};

struct DecodeBias {  // relative bias: weight (buckets, Hq), ranges of the distance and their buckets
    const void* w;
    int64_t w_stride;
    int w_dtype, n_ranges;
    int start[DEC_MAX_RANGES], bucket[DEC_MAX_RANGES];
};
struct DecodeNoBias {};  // (2 KB less to hand over with every launch)

template <typename T> struct Mfma16;
template <> struct Mfma16<bf16_t> {
    static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_v8<bf16_t>(a), as_v8<bf16_t>(b), c, 0, 0, 0);
    }
};
template <> struct Mfma16<f16_t> {
    static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(as_v8<f16_t>(a), as_v8<f16_t>(b), c, 0, 0, 0);
    }
};

// N dwords from an address of any alignment (the hardware takes unaligned vector loads; rows of an odd head dim need them)
template <int N> __device__ __forceinline__ void load_dwords(const char* p, uint32_t (&out)[N]) {
    __builtin_memcpy(out, p, 4 * N);
}

// a value that is the same in all lanes, for the scalar unit
__device__ __forceinline__ int64_t uniform64(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ float xor_lanes(float v, int m) { return __shfl_xor(v, m, 64); }

// log2(e) and how far a logit may exceed the reference before that moves: probabilities stay below e^5.5 = 245
constexpr float DEC_LOG2E = 1.4426950408889634f;
constexpr float DEC_LAZY = 5.5f;
// The high part of a probability is the 16-bit rounding of (1 - 2^-7) p, the low part the rounding of what is left: below p
// by more than half a step of the type (bf16: 2^-8), so the low part is positive wherever p is (down to 2^-18 in fp16, whose
// subnormal numbers end the split), and an infinite value stays infinite instead of meeting a zero or a negative factor.
// What is left is at most (2^-7 + 2^-8) p, its own rounding 2^-14.4 p.
constexpr float DEC_HIGH = 1.0f - 1.0f / 128;

struct DecodePiece {
    int b, unit, len, t0, t1;  // keys [t0, t1)
};

// NC: 32-channel chunks of the head dim (DP = 32 NC).  PAGE8: the page size is a multiple of 8, so the 8 keys of a lane group
// stand in one page (one lookup instead of 8).  SMALL: D < 8, rows are read element by element.
template <typename T, int NC, bool PAGE8, bool SMALL, bool BIAS>
__global__ __launch_bounds__(256) void paged_decode_kernel(const DecodeParams p,
                                                           const std::conditional_t<BIAS, DecodeBias, DecodeNoBias> rel) {
    constexpr int DP = 32 * NC, VE = DP / 16, VW = VE / 2, OSTRIDE = DP + 4;
    __shared__ float s_o[4][16][OSTRIDE];
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ int s_scan[256];
    __shared__ int64_t s_at[4];
    __shared__ int s_start[BIAS ? DEC_MAX_RANGES : 1];
    __shared__ float s_w[BIAS ? DEC_MAX_RANGES : 1][16];

    const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, g = lane >> 4;
    const int D = p.D;
    auto length = [&](int b) {
        const int n = p.seq_lens[b];
        return n < 0 ? 0 : (n < p.capacity ? n : p.capacity);
    };
    auto tiles_of = [](int len) { return len > 0 ? (len + DEC_TILE - 1) / DEC_TILE : 1; };

    // ---- this workgroup's run of tiles
    int64_t total = 0;
    for (int b0 = 0; b0 < p.B; b0 += 256) {
        int n = b0 + tid < p.B ? tiles_of(length(b0 + tid)) : 0;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) n += __shfl_xor(n, m, 64);
        if (lane == 0) s_scan[wave] = n;
        __syncthreads();
        total += uniform64((int64_t)s_scan[0] + s_scan[1] + s_scan[2] + s_scan[3]);
        __syncthreads();
    }
    total *= p.units;
    const int64_t share = (total + gridDim.x - 1) / gridDim.x;
    int64_t x = share * blockIdx.x;
    const int64_t x_end = min(total, x + share);
    if (x >= x_end) return;

    // ---- the sequence, unit and tile it begins with
    int b = 0;
    int64_t base = 0;  // first tile of sequence b
    for (int b0 = 0;; b0 += 256) {
        int n = b0 + tid < p.B ? tiles_of(length(b0 + tid)) : 0;
        int incl = n;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int up = __shfl_up(incl, m, 64);
            if (lane >= m) incl += up;
        }
        if (lane == 63) s_scan[wave] = incl;
        if (tid == 0) s_at[0] = -1;
        __syncthreads();
        int64_t before = 0, all = 0;  // (64 sequences' tiles fit 31 bits, 256 may not)
        for (int w = 0; w < 4; ++w) {
            before += w < wave ? s_scan[w] : 0;
            all += s_scan[w];
        }
        const int64_t end = base + (before + incl) * p.units, begin = end - (int64_t)n * p.units;
        if (x >= begin && x < end) {
            s_at[0] = b0 + tid;
            s_at[1] = begin;
        }
        __syncthreads();
        if (s_at[0] >= 0) {
            b = __builtin_amdgcn_readfirstlane((int)s_at[0]);
            base = uniform64(s_at[1]);
            break;
        }
        base += uniform64(all) * p.units;
        __syncthreads();
    }

    while (x < x_end) {
        const int len = __builtin_amdgcn_readfirstlane(length(b));
        const int ntiles = tiles_of(len);
        const int64_t in_seq = x - base;
        const int unit = (int)(in_seq / ntiles), tile0 = (int)(in_seq - (int64_t)unit * ntiles);
        const int tile1 = (int)min((int64_t)ntiles, tile0 + (x_end - x));
        const int t_end = min(len, tile1 * DEC_TILE);
        const int hk = unit / p.head_tiles, head0 = hk * p.group + (unit - hk * p.head_tiles) * 16;
        const int heads = min(16, (hk + 1) * p.group - head0);

        if constexpr (BIAS) {
            __syncthreads();
            for (int i = tid; i < rel.n_ranges * 16; i += 256) {
                const int r = i >> 4, h = i & 15;
                float wv = 0.f;
                if (h < heads) {
                    const int64_t at = rel.bucket[r] * rel.w_stride + head0 + h;
                    wv = rel.w_dtype == RGD_F32 ? static_cast<const float*>(rel.w)[at]
                         : rel.w_dtype == RGD_F16 ? to_f32(static_cast<const f16_t*>(rel.w)[at]) : to_f32(static_cast<const bf16_t*>(rel.w)[at]);
                }
                s_w[r][h] = wv;
                if (h == 0) s_start[r] = r == 0 ? INT32_MIN : rel.start[r];
            }
            __syncthreads();
        }

        // ---- query operand: B operand of S^T = K Q^T, head n16, channels of chunk 4 c + g
        u32x4 qf[NC];
        u32x4 kmask;  // channels of the last chunk that are not an earlier chunk's (all ones where the row is long enough)
        int kstart[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int ci = (4 * c + g) * 8;
            kstart[c] = SMALL ? 0 : min(ci, D - 8);
            Pack16 raw, keep;
            raw.v = u32x4{0, 0, 0, 0};
            const T* qrow = static_cast<const T*>(p.q) + b * p.sq[0] + (int64_t)(head0 + min(n16, heads - 1)) * p.sq[1];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool mine = SMALL ? ci + e < D : kstart[c] + e >= ci;
                keep.h[e] = mine ? 0xFFFF : 0;
                const int d = SMALL ? min(e, D - 1) : kstart[c] + e;
                const uint16_t qe = reinterpret_cast<const uint16_t*>(qrow)[d];
                raw.h[e] = mine && n16 < heads ? qe : 0;
            }
            qf[c] = raw.v;
            kmask = keep.v;
        }
        const int vstart = SMALL ? n16 * VE : min(n16 * VE, D - VE);

        f32x4 acc[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        float ref = -INFINITY, l = 0.f;

        const T* kbase = static_cast<const T*>(p.k) + hk * p.sk[1];
        const T* vbase = static_cast<const T*>(p.v) + hk * p.sv[1];
        const int32_t* table = p.page_table + b * p.table_stride;
        constexpr int NK = PAGE8 ? 1 : 2, NV = PAGE8 ? 1 : 8;
        int ek[NK], ev[NV];  // page numbers of the next step's keys and values
        u32x4 kf[2][NC];
        uint32_t vr[8][VW];
        bool v_ok[NV], v_ok_next[NV];

        // token a lane's lookup i stands for (clamped to the sequence, so that only its own page numbers are read)
        auto ktok = [&](int t, int i) {
            return PAGE8 ? min(t + 8 * (n16 >> 2), (len - 1) & ~7) : min(t + 8 * (n16 >> 2) + 4 * i + (n16 & 3), len - 1);
        };
        auto vtok = [&](int t, int i) { return PAGE8 ? min(t + 8 * g, (len - 1) & ~7) : min(t + 8 * g + i, len - 1); };
        auto lookup = [&](int t) {
#pragma unroll
            for (int i = 0; i < NK; ++i) ek[i] = table[fast_div(ktok(t, i), p.div_page)];
#pragma unroll
            for (int i = 0; i < NV; ++i) ev[i] = table[fast_div(vtok(t, i), p.div_page)];
        };
        auto load_k = [&](int t) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const int tok = ktok(t, a);
                int slot = tok - (int)(fast_div(tok, p.div_page) * p.div_page.d);
                if (PAGE8) slot += 4 * a + (n16 & 3);
                const int e = ek[PAGE8 ? 0 : a];
                const int page = e >= 0 && e < p.num_pages ? e : 0;
                const T* row = kbase + page * p.sk[0] + slot * p.sk[2];
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    if constexpr (SMALL) {
                        Pack16 r;
#pragma unroll
                        for (int d = 0; d < 8; ++d) r.h[d] = reinterpret_cast<const uint16_t*>(row)[min(d, D - 1)];
                        kf[a][c] = r.v;
                    } else {
                        uint32_t r[4];
                        load_dwords<4>(reinterpret_cast<const char*>(row + kstart[c]), r);
                        kf[a][c] = u32x4{r[0], r[1], r[2], r[3]};
                    }
                }
            }
        };
        auto load_v = [&](int t) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int tok = vtok(t, i);
                int slot = tok - (int)(fast_div(tok, p.div_page) * p.div_page.d);
                if (PAGE8) slot += i;
                const int e = ev[PAGE8 ? 0 : i];
                const bool ok = e >= 0 && e < p.num_pages;
                if (!PAGE8 || i == 0) v_ok_next[PAGE8 ? 0 : i] = ok;
                const int page = ok ? e : 0;
                const T* row = vbase + page * p.sv[0] + slot * p.sv[2];
                if constexpr (SMALL) {
                    const uint16_t* r = reinterpret_cast<const uint16_t*>(row);
                    vr[i][0] = r[min(vstart, D - 1)] | (uint32_t)r[min(vstart + 1, D - 1)] << 16;
                } else {
                    load_dwords<VW>(reinterpret_cast<const char*>(row + vstart), vr[i]);
                }
            }
        };

        auto step = [&](int t, bool prefetch) __attribute__((always_inline)) {
            f32x4 s[2];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                s[a] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    u32x4 kk = kf[a][c];
                    if (c == NC - 1) kk &= kmask;
                    s[a] = Mfma16<T>::run(kk, qf[c], s[a]);
                }
            }
            const bool ok0 = v_ok[0];
            bool ok_all = ok0;
#pragma unroll
            for (int i = 1; i < NV; ++i) ok_all = ok_all && v_ok[i];
            const bool whole = t + 32 <= len && __all(ok_all);
            if (prefetch) load_k(t + DEC_TILE);
            float x8[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x8[i] = s[i >> 2][i & 3] * p.scale;
            if constexpr (BIAS) {
                const int d0 = t + 8 * g - (len - 1);
                if (t + 31 - (len - 1) < s_start[min(1, rel.n_ranges - 1)]) {  // all in the first range
                    const float wv = s_w[0][n16];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x8[i] += wv;
                } else {
                    int lo = 0, hi = rel.n_ranges - 1;  // last range that begins at or before d0
                    while (lo < hi) {
                        const int mid = (lo + hi + 1) >> 1;
                        if (s_start[mid] <= d0) lo = mid;
                        else hi = mid - 1;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        while (lo + 1 < rel.n_ranges && s_start[lo + 1] <= d0 + i) ++lo;
                        x8[i] += s_w[lo][n16];
                    }
                }
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!(t + 8 * g + i < len && v_ok[PAGE8 ? 0 : i])) x8[i] = -INFINITY;
            }
            float top = fmaxf(fmaxf(fmaxf(x8[0], x8[1]), fmaxf(x8[2], x8[3])), fmaxf(fmaxf(x8[4], x8[5]), fmaxf(x8[6], x8[7])));
            if (__any(top > ref + DEC_LAZY)) {
                top = fmaxf(top, xor_lanes(top, 16));
                top = fmaxf(top, xor_lanes(top, 32));
                const float moved = fmaxf(ref, top);
                // (a head that has seen no logit yet has nothing to rescale)
                const float f = ref == -INFINITY ? 0.f : exp2f((ref - moved) * DEC_LOG2E);
                l *= f;
#pragma unroll
                for (int e = 0; e < VE; ++e)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[e][r] *= f;
                ref = moved;
            }
            const float at = ref == -INFINITY ? 0.f : ref;
            float pr[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                pr[i] = __builtin_amdgcn_exp2f((x8[i] - at) * DEC_LOG2E);
                l += pr[i];
            }
            u32x4 hi, lo;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a0 = pr[2 * j] * DEC_HIGH, a1 = pr[2 * j + 1] * DEC_HIGH;
                hi[j] = pack2<T>(a0, a1);
                lo[j] = pack2<T>(pr[2 * j] - to_f32(from_f32<T>(a0)), pr[2 * j + 1] - to_f32(from_f32<T>(a1)));
            }
            if (!whole) {  // what stands in slots of no key may be anything: 0 * NaN is NaN
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool in = t + 8 * g + i < len && v_ok[PAGE8 ? 0 : i];
#pragma unroll
                    for (int w = 0; w < VW; ++w) vr[i][w] = in ? vr[i][w] : 0u;
                }
            }
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                u32x4 vt;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    vt[j] = __builtin_amdgcn_perm(vr[2 * j + 1][e >> 1], vr[2 * j][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
                acc[e] = Mfma16<T>::run(vt, hi, acc[e]);
                acc[e] = Mfma16<T>::run(vt, lo, acc[e]);
            }
        };

        int t = tile0 * DEC_TILE + 32 * wave;
        if (t < t_end) {
            lookup(t);
            load_k(t);
            load_v(t);
            if (t + DEC_TILE < t_end) lookup(t + DEC_TILE);
            for (; t + DEC_TILE < t_end; t += DEC_TILE) {
#pragma unroll
                for (int i = 0; i < NV; ++i) v_ok[i] = v_ok_next[i];
                step(t, true);
                load_v(t + DEC_TILE);
                lookup(t + 2 * DEC_TILE);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) v_ok[i] = v_ok_next[i];
            step(t, false);
        }

        // ---- join the wavefronts
        l += xor_lanes(l, 16);
        l += xor_lanes(l, 32);
        __syncthreads();  // (the buffers' readers of the piece before are done)
        if (g == 0) {
            s_m[wave][n16] = ref;
            s_l[wave][n16] = l;
        }
        if (n16 < heads) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int e = 0; e < VE; ++e) s_o[wave][n16][(4 * g + r) * VE + e] = acc[e][r];
        }
        __syncthreads();
        const bool begins = tile0 == 0, ends = tile1 == ntiles;
        const bool direct = begins && ends;
        if (begins && tid == 0) {
            const int64_t first = base + (int64_t)unit * ntiles;
            p.plan[(int64_t)b * p.units + unit] = make_int2((int)blockIdx.x, (int)((first + ntiles - 1) / share));
        }
        float* slot = p.part + (int64_t)(2 * blockIdx.x + (begins ? 1 : 0)) * ((int64_t)p.part_rows * DP + 32);
        for (int i = tid; i < heads * DP; i += 256) {
            const int h = i / DP, at = i - h * DP;
            const float m0 = s_m[0][h], m1 = s_m[1][h], m2 = s_m[2][h], m3 = s_m[3][h];
            const float top = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
            const float z = top == -INFINITY ? 0.f : top;
            const float f0 = exp2f((m0 - z) * DEC_LOG2E), f1 = exp2f((m1 - z) * DEC_LOG2E), f2 = exp2f((m2 - z) * DEC_LOG2E),
                        f3 = exp2f((m3 - z) * DEC_LOG2E);
            const float sum = f0 * s_l[0][h] + f1 * s_l[1][h] + f2 * s_l[2][h] + f3 * s_l[3][h];
            const float out = f0 * s_o[0][h][at] + f1 * s_o[1][h][at] + f2 * s_o[2][h][at] + f3 * s_o[3][h][at];
            if (direct) {
                const int m = at / VE, ch = (SMALL ? m * VE : min(m * VE, D - VE)) + at % VE;
                if (SMALL ? ch < D : m * VE < D)
                    static_cast<T*>(p.o)[b * p.so[0] + (int64_t)(head0 + h) * p.so[1] + ch] = from_f32<T>(sum == 0.f ? 0.f : out / sum);
                if (p.lse && at == 0) p.lse[(int64_t)b * p.Hq + head0 + h] = sum == 0.f ? -INFINITY : z + logf(sum);
            } else {
                slot[h * DP + at] = out;
                if (at == 0) {
                    slot[p.part_rows * DP + h] = top;
                    slot[p.part_rows * DP + 16 + h] = sum;
                }
            }
        }
        x += tile1 - tile0;
        if (ends && unit + 1 == p.units) {
            base += (int64_t)ntiles * p.units;
            ++b;
        }
    }
}

// One workgroup per (sequence, query head): joins the pieces of its unit, in order.  32 lanes take 4 channels each, 8 groups of
// lanes every eighth piece.
template <typename T, int NC, bool SMALL> __global__ __launch_bounds__(256) void paged_decode_merge_kernel(const DecodeParams p) {
    constexpr int DP = 32 * NC, VE = DP / 16;
    __shared__ float s_o[8][DP];
    __shared__ float s_sum[8], s_top[8];
    const int b = blockIdx.x / p.Hq, h = blockIdx.x % p.Hq;
    const int hk = h / p.group, in_group = h - hk * p.group;
    const int unit = hk * p.head_tiles + (in_group >> 4), row = in_group & 15;
    const int2 span = p.plan[(int64_t)b * p.units + unit];
    if (span.x == span.y) return;  // one piece: written already
    const int64_t slot_size = (int64_t)p.part_rows * DP + 32;
    auto slot = [&](int w) { return p.part + (int64_t)(2 * w + (w == span.x ? 1 : 0)) * slot_size; };
    const int tid = threadIdx.x, grp = tid >> 5, c4 = (tid & 31) * 4;
    float top = -INFINITY;
    for (int w = span.x + tid; w <= span.y; w += 256) top = fmaxf(top, slot(w)[p.part_rows * DP + row]);
    top = group_reduce<64, OpMax>(top);
    if ((tid & 63) == 0) s_top[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    const float z = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int w = span.x + grp; w <= span.y; w += 8) {
        const float* s = slot(w);
        const float f = exp2f((s[p.part_rows * DP + row] - z) * DEC_LOG2E);
        sum += f * s[p.part_rows * DP + 16 + row];
        if (c4 < DP) o += f * *reinterpret_cast<const f32x4*>(s + row * DP + c4);
    }
    if (c4 < DP) *reinterpret_cast<f32x4*>(&s_o[grp][c4]) = o;
    if ((tid & 31) == 0) s_sum[grp] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += s_sum[i];
    if (tid < DP) {
        float out = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) out += s_o[i][tid];
        const int m = tid / VE, ch = (SMALL ? m * VE : min(m * VE, p.D - VE)) + tid % VE;
        if (SMALL ? ch < p.D : m * VE < p.D)
            static_cast<T*>(p.o)[b * p.so[0] + (int64_t)h * p.so[1] + ch] = from_f32<T>(sum == 0.f ? 0.f : out / sum);
        if (p.lse && tid == 0) p.lse[(int64_t)b * p.Hq + h] = sum == 0.f ? -INFINITY : z + logf(sum);
    }
}
