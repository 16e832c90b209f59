// Attention of one new token per sequence over a paged key/value cache.
//
//   s_j = softmax_scale q . k_j (+ W[bucket(j - (len - 1))][h]),  o = sum_j softmax(s)_j v_j,  lse = log sum_j exp(s_j)
//
// Bound by memory: every cached key and value is read once, 4 D bytes per token and key head, for 4 D group operations.
//
// Work.  A unit is (sequence, key head, 16 of the key head's query heads); its keys are cut into tiles of 32.  The tiles of all
// units (of one key head per bundle, see below), in one row, are dealt to the wavefronts in equal runs: every wavefront finds its run from the lengths on the GPU, so
// the host need not know them, one long sequence fills the chip like many short ones, and a ragged batch leaves no wavefront
// with more than a tile over the others.  A run that holds a whole unit writes its output; pieces of a unit that several
// wavefronts share leave partial results in the workspace (at most two per wavefront: one unit begun earlier, one not ended),
// which the merge launch joins in order.
//
// A piece's first loads leave while the piece before ends, so that a wavefront with many short pieces does not wait for each.
//
// A step.  A wavefront (a workgroup of its own) takes 32 keys at a time, without LDS or barriers, operands straight from memory
// to registers (v_mfma_f32_16x16x32: A lane l holds row l % 16, k = 8 (l / 16) .. + 7; C lane l holds column l % 16, rows
// 4 (l / 16) + 0..3):
//   S^T = K Q^T, two products of 16 keys.  MFMA row i of product a is key 8 (i / 4) + 4 a + i % 4, so that lane group g = l / 16 ends
//   up with the logits of keys 8 g .. 8 g + 7 of query head l % 16: the layout P^T has to have as the second product's B operand.
//   O^T += V^T P^T, one product per element e of a lane's piece of a value row: lane l loads VE = DP / 16 channels from VE (l % 16)
//   on of keys 8 g .. 8 g + 7 (whole rows per load) and pairs them by key with byte permutes; MFMA row m is channel VE m + e.
// So 16 rows of heads are computed whatever the group: at the rate the memory delivers keys the matrix pipe is busy a tenth of
// the time.  P is split into two 16-bit parts (a second product each): rounded to one, its error would be as large as the
// output's own rounding, and the products are free (DEC_HIGH).
// The running maximum is a reference that moves only when a logit exceeds it by LAZY (fp16: it stays a headroom below the
// maximum); sums, maxima and outputs are fp32.
//
// Measured (this launch / the merge; a read that streams 512 MB reaches 6.6 TB/s): one sequence of 131000 keys, 32 / 8 heads,
// D = 128: 86 / 7 us, 6.2 TB/s; 64 sequences to 4100 keys, the same heads: 106 / 5 us, 5.5 TB/s; 19 to 2000 keys, 24 heads,
// D = 80, bias, pages of 5: 40 / 5 us; one of 200 keys, 16 heads, D = 64: 5.4 / 3.9 us.  What a launch takes beyond its
// bytes, about 15 us, is the chain of loads in front of the first step (lengths, page numbers, keys), the last steps, in which
// the wavefronts run out one by one, and the merge.
#pragma once

#include "attn_common.h"

#include <type_traits>

constexpr int DEC_MAX_RANGES = 256;
constexpr int DEC_TILE = 32;  // keys of a step
constexpr int DEC_NEAR = 256;  // distances whose range is looked up instead of searched

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
    int B, Hq, group, head_tiles;
    int units;         // of a sequence: key heads / heads of a bundle * head_tiles
    int bundle_log;    // 2^bundle_log key heads in a bundle
    int D, num_pages;
    FastDiv div_page;
    float scale;
    int* plan;         // per unit of the batch: wavefronts its first and last piece are in
    float* part;       // two slots per wavefront: O [rows][DP], then m [16], l [16]
    int part_rows;     // query heads of a slot
};

struct DecodeBias {  // relative bias: weight (buckets, Hq), ranges of the distance and their buckets
    const void* w;
    int64_t w_stride;
    int w_dtype, n_ranges;
    int half;  // largest power of two below n_ranges (0 for one range)
    int start[DEC_MAX_RANGES], bucket[DEC_MAX_RANGES];
    uint32_t near[DEC_NEAR / 4];  // bytes: range of the distance -n, n < DEC_NEAR
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

// N dwords from an address of any alignment (the hardware takes unaligned vector loads; rows of an odd head dim need them); NT:
// streaming
template <int N, bool NT = false> __device__ __forceinline__ void load_dwords(const char* p, uint32_t (&out)[N]) {
    if constexpr (N == 1) {
        typedef uint32_t V __attribute__((aligned(2)));
        const V* from = reinterpret_cast<const V*>(p);
        out[0] = NT ? __builtin_nontemporal_load(from) : *from;
    } else {
        typedef uint32_t V0 __attribute__((ext_vector_type(N)));
        typedef V0 V __attribute__((aligned(2)));
        const V* from = reinterpret_cast<const V*>(p);
        const V0 v = NT ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = v[i];
    }
}

__device__ __forceinline__ float xor_lanes(float v, int m) { return __shfl_xor(v, m, 64); }

// Nothing is scheduled across it.  Waits count loads in order, so the order page numbers, keys, values has to be the same in
// and in front of the loop; and a step's keys, and its values, leave together: with the arithmetic free to move between them
// one sequence of 131000 keys took 100 us instead of 95.
#define DEC_KEEP_LOADS() __builtin_amdgcn_sched_barrier(0)

// log2(e) and how far a logit may exceed the reference and its headroom before that moves: probabilities stay below
// e^(5.5 + headroom)
constexpr float DEC_LOG2E = 1.4426950408889634f;
constexpr float DEC_LAZY = 5.5f;
// The reference is the running maximum less a headroom.  fp16 ends at 65504 above and at 2^-24 below: with 2^8 of headroom (e^5.5
// 2^8 = 62600) a key counts down to 2^-33 of the largest instead of 2^-25 (32768 equal keys 2^-25 below one other, which are 0.1 %
// of the sum, would add nothing to the output).  bf16 ends where fp32 does.
template <typename T> constexpr float DEC_HEADROOM = std::is_same<T, f16_t>::value ? 8.0f * 0.6931471805599453f : 0.0f;
// The high part of a probability is the 16-bit rounding of (1 - 2^-7) p, the low part the rounding of what is left: below p
// by more than half a step of the type (bf16: 2^-8), so the low part is positive wherever p is (in fp16 down to 2^-25 of the
// largest, below which its subnormal numbers end the split), and an infinite value stays infinite instead of meeting a zero or a
// negative factor.  What is left is at most (2^-7 + 2^-8) p, its own rounding 2^-14.4 p (fp16: or 2^-33 of the largest).
constexpr float DEC_HIGH = 1.0f - 1.0f / 128;

// NC: 32-channel chunks of the head dim (DP = 32 NC).  SMALL: D < 8, rows are read element by element.  LINES: D = DP is 64 or 128,
// rows of token-major heads are whole 128-byte lines, which no other wavefront reads: loads stream.
// Else lines are shared by neighbouring heads: loads do not stream, and the key heads that fill lines together are a bundle, whose
// wavefronts take the same tiles of one head each, on one XCD, side by side: the first to come fetches the line for all of
// them.  19 x 24 heads, lengths to 2000, streaming / not / not and in bundles: D = 16: 28 / 27 / 19 us, D = 32: 28 / 28 / 23, D = 40:
// 37 / - / 30, D = 80: 48 / 45 / 40, D = 112: 59 / - / 53; one of 131000 keys, 8 key heads, D = 80: 94 / 82 / 76, D = 128 (no bundles):
// 95 / 104.
// The lanes look up the 32 keys' pages together and pass the row addresses around (20 cross-lane moves a step), whatever the
// page size: a variant for pages of whole groups of 8 keys, in which a lane needs two page numbers and no moves, was no faster
// ((19 x 24 heads, D = 128, lengths to 2000) pages of 16: 54.4 us this way, 54.1 that).
template <typename T, int NC, bool SMALL, bool LINES, bool BIAS>
__global__ __launch_bounds__(64, 2) void paged_decode_kernel(const DecodeParams p,
                                                          const std::conditional_t<BIAS, DecodeBias, DecodeNoBias> rel) {
    constexpr int DP = 32 * NC, VE = DP / 16, VW = VE / 2;
    // BIAS, by the number of ranges (for 256 of them 8 wavefronts fit a compute unit, for 32 all 12 of the small head dims do:
    // D = 64, 24 heads, 19 lengths to 2000 with bias 37 us instead of 42)
    static_assert(DEC_NEAR == 4 * 64, "a dword per lane");
    extern __shared__ uint32_t s_near[];  // then starts, buckets and the weight of 16 heads
    int *s_start = nullptr, *s_bucket = nullptr;
    float (*s_w)[16] = nullptr;

    // run: the wavefront's part of the row of tiles; sub: its key head of a bundle
    const int bl = p.bundle_log, bundle = 1 << bl, runs = gridDim.x >> bl;
    const int sub = blockIdx.x >> 3 & (bundle - 1);
    const int run = (blockIdx.x >> (3 + bl) << 3) + (blockIdx.x & 7);  // (workgroups go round the 8 XCDs)
    const int lane = threadIdx.x;
    const int n16 = lane & 15, g = lane >> 4;
    const int D = LINES ? DP : p.D;
    auto length = [&](int b) {
        const int n = p.seq_lens[b];
        return n < 0 ? 0 : (n < p.capacity ? n : p.capacity);
    };
    auto tiles_of = [](int len) { return len > 0 ? (int)(((uint32_t)len + DEC_TILE - 1) / DEC_TILE) : 1; };

    if constexpr (BIAS) {  // (starts filled up to the next power of two: a search halves it)
        const int fill = max(2 * rel.half, 1);
        s_start = reinterpret_cast<int*>(s_near + DEC_NEAR / 4);
        s_bucket = s_start + fill;
        s_w = reinterpret_cast<float(*)[16]>(s_bucket + fill);
        s_near[lane] = rel.near[lane];
        for (int r = lane; r < fill; r += 64) {
            s_start[r] = r < rel.n_ranges ? (r == 0 ? INT32_MIN : rel.start[r]) : INT32_MAX;
            s_bucket[r] = r < rel.n_ranges ? rel.bucket[r] : 0;
        }
        __syncthreads();  // (one wavefront: orders its LDS accesses)
    }

    // ---- this wavefront's run of tiles [x, x_end) and the sequence it begins in
    auto scan = [&](uint32_t n) {  // inclusive sum over the lanes (64 sequences of at most 2^26 tiles)
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t up = __shfl_up(n, m, 64);
            if (lane >= m) n += up;
        }
        return n;
    };
    auto last_of = [](uint32_t n) { return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)n, 63); };
    uint32_t mine = lane < p.B ? tiles_of(length(lane)) : 0;  // tiles of sequence b0 + lane
    uint32_t incl = scan(mine);
    int64_t total = last_of(incl);
    for (int b0 = 64; b0 < p.B; b0 += 64) total += last_of(scan(b0 + lane < p.B ? tiles_of(length(b0 + lane)) : 0));
    total *= p.units;
    const int64_t even = total <= INT32_MAX ? (int64_t)((uint32_t)total / (uint32_t)runs) : total / runs, rest = total - even * runs;
    int64_t x = even * run + min((int64_t)run, rest);
    const int64_t x_end = x + even + (run < rest ? 1 : 0);
    if (x >= x_end) return;
    int b = 0;
    int64_t base = 0;  // first tile of sequence b
    for (int b0 = 0;;) {
        const uint64_t behind = __ballot(base + (int64_t)incl * p.units > x);
        if (behind) {
            const int at = __builtin_ctzll(behind);
            b = b0 + at;
            base += (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(incl - mine), at) * p.units;
            break;
        }
        base += last_of(incl) * p.units;
        b0 += 64;
        mine = b0 + lane < p.B ? tiles_of(length(b0 + lane)) : 0;
        incl = scan(mine);
    }

    // ---- a piece: tiles tile0 .. tile1 - 1 of one unit
    struct Piece {
        int b, unit, len, ntiles, tile0, tile1, hk, head0, heads;
    };
    auto piece_at = [&]() {
        Piece c;
        c.b = b;
        c.len = __builtin_amdgcn_readfirstlane(length(b));
        c.ntiles = tiles_of(c.len);
        const int64_t in_seq = x - base;
        c.unit = in_seq <= INT32_MAX ? (int)((uint32_t)in_seq / (uint32_t)c.ntiles) : (int)(in_seq / c.ntiles);
        c.tile0 = (int)(in_seq - (int64_t)c.unit * c.ntiles);
        c.tile1 = (int)min((int64_t)c.ntiles, c.tile0 + (x_end - x));
        const int of = c.unit / p.head_tiles;
        c.hk = (of << bl) + sub;
        c.head0 = c.hk * p.group + (c.unit - of * p.head_tiles) * 16;
        c.heads = min(16, (c.hk + 1) * p.group - c.head0);
        return c;
    };

    u32x4 qf[NC];
    u32x4 kmask;  // channels of the last chunk that are not an earlier chunk's (all ones where the row is long enough)
    int kstart[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) kstart[c] = SMALL ? 0 : min((4 * c + g) * 8, D - 8);
    const int vstart = SMALL ? n16 * VE : min(n16 * VE, D - VE);

    // Loads.  Page numbers are looked up two steps ahead and turned into row addresses one step ahead: loads return in order, so
    // a lookup behind a step's loads would hold up the next step's until those are there.  A piece's first loads are
    // on their way while the piece before ends: what follows is aimed at the piece that is loaded, not the one worked on.
    int load_len = 0;
    const T* kbase = nullptr;
    const T* vbase = nullptr;
    const int32_t* table = nullptr;
    u32x4 kf[2][NC];
    uint32_t vr[8][VW];
    int entry = 0;                     // page number of key t + lane % 32
    int64_t koff = 0, voff = 0;        // its row offsets
    uint32_t ok_cur = 0, ok_next = 0;  // bit i: the page of key t + i exists

    auto aim = [&](const Piece& c) __attribute__((always_inline)) {
        load_len = c.len;
        kbase = static_cast<const T*>(p.k) + c.hk * p.sk[1];
        vbase = static_cast<const T*>(p.v) + c.hk * p.sv[1];
        table = p.page_table + c.b * p.table_stride;
    };
    // (only the sequence's own page numbers are read; one without keys reads its first, and what that leads to is not used)
    auto token = [&](int t) { return min(t + (lane & 31), max(load_len - 1, 0)); };
    auto lookup = [&](int t) __attribute__((always_inline)) { entry = table[fast_div(token(t), p.div_page)]; };
    auto locate = [&](int t) __attribute__((always_inline)) {
        const int tok = token(t);
        const int slot = tok - (int)(fast_div(tok, p.div_page) * p.div_page.d);
        const bool ok = entry >= 0 && entry < p.num_pages;
        const int64_t page = ok ? entry : 0;
        ok_next = (uint32_t)__ballot(ok);
        koff = page * p.sk[0] + slot * p.sk[2];
        voff = page * p.sv[0] + slot * p.sv[2];
    };
    auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const T* row = kbase + __shfl(koff, 8 * (n16 >> 2) + 4 * a + (n16 & 3), 64);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if constexpr (SMALL) {
                    Pack16 r;
#pragma unroll
                    for (int d = 0; d < 8; ++d) r.h[d] = reinterpret_cast<const uint16_t*>(row)[min(d, D - 1)];
                    kf[a][c] = r.v;
                } else {
                    uint32_t r[4];
                    load_dwords<4, LINES>(reinterpret_cast<const char*>(row + kstart[c]), r);
                    kf[a][c] = u32x4{r[0], r[1], r[2], r[3]};
                }
            }
        }
    };
    auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const T* row = vbase + __shfl(voff, 8 * g + i, 64);
            if constexpr (SMALL) {
                const uint16_t* r = reinterpret_cast<const uint16_t*>(row);
                vr[i][0] = r[min(vstart, D - 1)] | (uint32_t)r[min(vstart + 1, D - 1)] << 16;
            } else {
                load_dwords<VW, LINES>(reinterpret_cast<const char*>(row + vstart), vr[i]);
            }
        }
    };

    // query: B operand of S^T = K Q^T, head n16, channels of chunk 4 c + g
    auto load_q = [&](const Piece& c) __attribute__((always_inline)) {
        const T* qrow = static_cast<const T*>(p.q) + c.b * p.sq[0] + (int64_t)(c.head0 + min(n16, c.heads - 1)) * p.sq[1];
        const uint32_t head_ok = n16 < c.heads ? ~0u : 0u;  // (as bits: a choice would become a branch around each load)
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            const int ci = (4 * k + g) * 8;
            Pack16 raw, keep;
            if constexpr (SMALL) {
#pragma unroll
                for (int e = 0; e < 8; ++e) raw.h[e] = reinterpret_cast<const uint16_t*>(qrow)[min(e, D - 1)];
            } else {
                load_dwords<4>(reinterpret_cast<const char*>(qrow + kstart[k]), raw.w);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) keep.h[e] = (SMALL ? ci + e < D : kstart[k] + e >= ci) ? 0xFFFF : 0;
            qf[k] = raw.v & keep.v & u32x4{head_ok, head_ok, head_ok, head_ok};
            kmask = keep.v;
        }
    };
    // The piece that is worked on is `cur`; `next` is the one behind it, whose first page numbers are being looked up.
    Piece cur = piece_at(), next = cur;
    bool worked = false;
    aim(next);
    lookup(next.tile0 * DEC_TILE);
    f32x4 acc[VE];
    float ref = -INFINITY, l = 0.f;
    auto finish = [&]() __attribute__((always_inline)) {
        // the piece's result: lane holds channels VE m + e of head n16 for m = 4 g + r
        const int heads = cur.heads, head0 = cur.head0;
        const bool begins = cur.tile0 == 0, ends = cur.tile1 == cur.ntiles;
        l += xor_lanes(l, 16);
        l += xor_lanes(l, 32);
        if (lane == 0) {
            int* plan = &p.plan[2 * ((((int64_t)cur.b * p.units + cur.unit) << bl) + sub)];
            if (begins) plan[0] = run;
            if (ends) plan[1] = run;
        }
        if (n16 < heads) {
            if (begins && ends) {
                const float inv = l == 0.f ? 0.f : 1.0f / l;
                T* orow = static_cast<T*>(p.o) + cur.b * p.so[0] + (int64_t)(head0 + n16) * p.so[1];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int first = (4 * g + r) * VE;
                    T out[VE];
#pragma unroll
                    for (int e = 0; e < VE; ++e) out[e] = from_f32<T>(l == 0.f ? 0.f : acc[e][r] * inv);
                    if constexpr (SMALL) {
#pragma unroll
                        for (int e = 0; e < VE; ++e)
                            if (first + e < D) orow[first + e] = out[e];
                    } else {
                        if (first < D) __builtin_memcpy(orow + min(first, D - VE), out, sizeof(out));
                    }
                }
                if (p.lse && g == 0) p.lse[(int64_t)cur.b * p.Hq + head0 + n16] = l == 0.f ? -INFINITY : (ref == -INFINITY ? 0.f : ref) + logf(l);
            } else {
                float* slot = p.part + (int64_t)(2 * ((run << bl) + sub) + (begins ? 1 : 0)) * ((int64_t)p.part_rows * DP + 32);
                float out[4 * VE];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < VE; ++e) out[r * VE + e] = acc[e][r];
                f32x4* to = reinterpret_cast<f32x4*>(slot + n16 * DP + 4 * g * VE);
#pragma unroll
                for (int i = 0; i < VE; ++i) to[i] = f32x4{out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]};
                if (g == 0) {
                    slot[p.part_rows * DP + n16] = ref;
                    slot[p.part_rows * DP + 16 + n16] = l;
                }
            }
        }
    };
    for (;;) {
        // (one place for these loads: at a second one the registers would differ, and copying them waits)
        load_q(next);
        locate(next.tile0 * DEC_TILE);
        lookup((next.tile0 + 1) * DEC_TILE);
        DEC_KEEP_LOADS();
        load_k();
        DEC_KEEP_LOADS();
        load_v();
        DEC_KEEP_LOADS();
        if (worked) finish();
        cur = next;
        worked = true;
        const int len = cur.len, heads = cur.heads, head0 = cur.head0;
        if constexpr (BIAS) {  // the weight of the unit's heads, by range
            __syncthreads();  // (one wavefront: orders its LDS accesses)
            const int hb = heads > 1 ? 32 - __builtin_clz(heads - 1) : 0;
#pragma unroll 4
            for (int i = lane; i < rel.n_ranges << hb; i += 64) {
                const int r = i >> hb, h = min(i - (r << hb), heads - 1);
                const int64_t at = s_bucket[r] * rel.w_stride + head0 + h;
                s_w[r][h] = rel.w_dtype == RGD_F32 ? static_cast<const float*>(rel.w)[at]
                            : rel.w_dtype == RGD_F16 ? to_f32(static_cast<const f16_t*>(rel.w)[at])
                                                     : to_f32(static_cast<const bf16_t*>(rel.w)[at]);
            }
            __syncthreads();
        }

#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        ref = -INFINITY, l = 0.f;
        const int hrow = min(n16, heads - 1);

        // one step; prefetch: the next one's keys are loaded as soon as this one's are used
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
            const bool whole = t + 32 <= len && ok_cur == ~0u;
            const uint32_t ok8 = ok_cur >> (8 * g);  // of the lane's 8 keys
            if (prefetch) {
                locate(t + DEC_TILE);
                lookup(t + 2 * DEC_TILE);
                DEC_KEEP_LOADS();
                load_k();
            }
            float x8[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x8[i] = s[i >> 2][i & 3] * p.scale;
            if constexpr (BIAS) {
                const int d0 = t + 8 * g - (len - 1);
                if (t + 31 - (len - 1) < s_start[min(1, rel.n_ranges - 1)]) {  // all in the first range
                    const float wv = s_w[0][hrow];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x8[i] += wv;
                } else if (len - t <= DEC_NEAR) {  // (searched, (19 x 24 heads, lengths to 2000) D = 128 takes 58 us instead of 54)
                    const uint8_t* near = reinterpret_cast<const uint8_t*>(s_near);
#pragma unroll
                    for (int i = 0; i < 8; ++i) x8[i] += s_w[near[max(-d0 - i, 0)]][hrow];
                } else {
                    int at[8];  // last range that begins at or before the key's distance, the 8 searches side by side
#pragma unroll
                    for (int i = 0; i < 8; ++i) at[i] = 0;
                    for (int half = rel.half; half > 0; half >>= 1) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) at[i] += s_start[at[i] + half] <= d0 + i ? half : 0;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) x8[i] += s_w[at[i]][hrow];
                }
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!(t + 8 * g + i < len && (ok8 >> i & 1))) x8[i] = -INFINITY;
            }
            float top = fmaxf(fmaxf(fmaxf(x8[0], x8[1]), fmaxf(x8[2], x8[3])), fmaxf(fmaxf(x8[4], x8[5]), fmaxf(x8[6], x8[7])));
            // (the difference, not a sum: of large logits a sum may round up past what fp16 holds)
            if (__any(top - ref > DEC_LAZY + DEC_HEADROOM<T>)) {
                top = fmaxf(top, xor_lanes(top, 16));
                top = fmaxf(top, xor_lanes(top, 32));
                const float moved = fmaxf(ref, top - DEC_HEADROOM<T>);
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
                    const bool in = t + 8 * g + i < len && (ok8 >> i & 1);
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

        const int t_last = (cur.tile1 - 1) * DEC_TILE;
        if (len > 0) {
            for (int t = cur.tile0 * DEC_TILE; t < t_last; t += DEC_TILE) {
                ok_cur = ok_next;
                step(t, true);
                DEC_KEEP_LOADS();
                load_v();
                DEC_KEEP_LOADS();
            }
            ok_cur = ok_next;
        }
        x += cur.tile1 - cur.tile0;
        if (cur.tile1 == cur.ntiles && cur.unit + 1 == p.units) {
            base += (int64_t)cur.ntiles * p.units;
            ++b;
        }
        const bool more = x < x_end;
        if (more) {
            next = piece_at();
            aim(next);
            lookup(next.tile0 * DEC_TILE);
        }
        if (len > 0) step(t_last, false);
        if (!more) break;
    }
    finish();
}

// no page exists: every row is empty
template <typename T> __global__ __launch_bounds__(64) void paged_decode_empty_kernel(const DecodeParams p) {
    const int b = blockIdx.x / p.Hq, h = blockIdx.x % p.Hq;
    for (int d = threadIdx.x; d < p.D; d += 64) static_cast<T*>(p.o)[b * p.so[0] + (int64_t)h * p.so[1] + d] = from_f32<T>(0.f);
    if (p.lse && threadIdx.x == 0) p.lse[(int64_t)b * p.Hq + h] = -INFINITY;
}

// One workgroup of THREADS per (sequence, query head): joins the pieces of its unit, in order.  32 lanes take 4 channels each, G
// groups of lanes every G-th piece, eight at a time in flight.
template <typename T, int NC, bool SMALL, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_decode_merge_kernel(const DecodeParams p) {
    constexpr int DP = 32 * NC, VE = DP / 16, G = THREADS / 32, BATCH = 8 * G;
    __shared__ float s_o[G][DP];
    __shared__ float s_f[BATCH];
    __shared__ float s_red[THREADS / 64];
    const int b = blockIdx.x / p.Hq, h = blockIdx.x % p.Hq;
    const int hk = h / p.group, in_group = h - hk * p.group;
    const int bl = p.bundle_log, sub = hk & ((1 << bl) - 1), unit = (hk >> bl) * p.head_tiles + (in_group >> 4), row = in_group & 15;
    const int* plan = &p.plan[2 * ((((int64_t)b * p.units + unit) << bl) + sub)];
    struct { int x, y; } span = {plan[0], plan[1]};
    if (span.x == span.y) return;  // one piece: written already
    const int64_t slot_size = (int64_t)p.part_rows * DP + 32;
    auto slot = [&](int w) { return p.part + (int64_t)(2 * ((w << bl) + sub) + (w == span.x ? 1 : 0)) * slot_size; };
    const int tid = threadIdx.x, grp = tid >> 5, c4 = (tid & 31) * 4;
    auto over_all = [&](float v, auto op) {  // v over the workgroup, op(a, b)
        __syncthreads();
        if ((tid & 63) == 0) s_red[tid >> 6] = v;
        __syncthreads();
        v = s_red[0];
        for (int i = 1; i < THREADS / 64; ++i) v = op(v, s_red[i]);
        return v;
    };
    float top = -INFINITY;
    for (int w = span.x + tid; w <= span.y; w += THREADS) top = fmaxf(top, slot(w)[p.part_rows * DP + row]);
    top = over_all(group_reduce<64, OpMax>(top), [](float a, float c) { return fmaxf(a, c); });
    const float z = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int w0 = span.x; w0 <= span.y; w0 += BATCH) {
        if (tid < BATCH) {
            float f = 0.f;
            if (w0 + tid <= span.y) {
                const float* s = slot(w0 + tid) + p.part_rows * DP + row;
                f = exp2f((s[0] - z) * DEC_LOG2E);
                sum += f * s[16];
            }
            s_f[tid] = f;
        }
        __syncthreads();
        if (c4 < DP) {
            f32x4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = w0 + i * G + grp <= span.y ? *reinterpret_cast<const f32x4*>(slot(w0 + i * G + grp) + row * DP + c4) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) o += s_f[i * G + grp] * v[i];
        }
        __syncthreads();
    }
    if (c4 < DP) *reinterpret_cast<f32x4*>(&s_o[grp][c4]) = o;
    sum = over_all(group_reduce<64>(sum), [](float a, float c) { return a + c; });
    if (tid < DP) {
        float out = 0.f;
        for (int i = 0; i < G; ++i) out += s_o[i][tid];
        const int m = tid / VE, ch = (SMALL ? m * VE : min(m * VE, p.D - VE)) + tid % VE;
        if (SMALL ? ch < p.D : m * VE < p.D)
            static_cast<T*>(p.o)[b * p.so[0] + (int64_t)h * p.so[1] + ch] = from_f32<T>(sum == 0.f ? 0.f : out / sum);
        if (p.lse && tid == 0) p.lse[(int64_t)b * p.Hq + h] = sum == 0.f ? -INFINITY : z + logf(sum);
    }
}
