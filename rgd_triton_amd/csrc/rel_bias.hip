// Learned relative position bias and the gradient of its weight.
//
//   bias[h][i][j] = W[bucket(j - i - q_offset)][h],   dW[b][h] = sum of dbias[h][i][j] over bucket(j - i - q_offset) = b
//
// A bucket is a range of the relative distance d = j - i - q_offset: the matrix is constant along its diagonals, and the gradient
// is the sum of each diagonal, added up over the diagonals of a bucket.  Bound by memory: the matrix is written (forward) or
// read (backward) once.
//
// Both directions walk the matrix along its diagonals.  A wavefront takes a strip of 512 columns and goes down `chunk` rows, 8 rows
// and 8 columns at a time: lane l holds the 8 x 8 block whose columns begin at strip + 8 l + 8 n in step n, so the 15
// diagonals of a lane's block are the same in every step.
//   forward   the 15 values are looked up once, the 8 rows of the block packed once; each step is eight 16-byte stores
//   backward  15 sums stay in registers; each step is eight 16-byte loads and 64 additions
// Blocks left of the first or right of the last column are skipped, one that the last column cuts goes element by element.
// Rows need no alignment: the hardware takes 16-byte accesses at any address.
#include "common.h"

#include <string.h>

namespace {

constexpr int MAX_RANGES = 256;
constexpr int STRIP = 512;

struct RelRanges {  // range k: start[k] <= d < start[k + 1], ascending, bucket[k]; start[0] covers everything below
    int n;
    int start[MAX_RANGES];
    int bucket[MAX_RANGES];
};

struct RelParams {
    const void* w;      // forward: weight; backward: unused
    void* bias;         // forward: written; backward: dbias, read
    float* part;        // backward: [head][range][task]
    void* dw;
    int64_t w_stride, stride_h, stride_n;
    int w_dtype, H, Tq, Tk, offset;
    int chunk, strips, tasks, num_buckets;
    RelRanges r;
};

struct Split {
    int64_t chunk, chunks, strips, tasks;
};

// Rows of a task.  Long tasks spend less on their beginning and end (looking values up, adding buckets up) and waste fewer lanes at
// the slanted edges, short ones fill the chip: the longest of 16 .. 256 rows that still gives every compute unit 8
// wavefronts.  (24, 4352, 4352) bf16 forward + backward at 256 / 64 rows: MEASURED_LARGE; (8, 128, 128) at 16 / 256: MEASURED_SMALL.
Split split(int64_t H, int64_t Tq, int64_t Tk) {
    Split s;
    for (s.chunk = 256;; s.chunk /= 2) {
        s.chunks = (Tq + s.chunk - 1) / s.chunk;
        s.strips = (Tk + s.chunk - 8 + STRIP - 1) / STRIP;
        s.tasks = s.chunks * s.strips;
        if (s.chunk == 16 || s.tasks * H >= 8 * (int64_t)rgd_num_cus()) return s;
    }
}

template <typename T> struct Block {  // 8 consecutive elements
    static constexpr int NW = 8 * sizeof(T) / 4;
    uint32_t w[NW];
};

// W column of the workgroup's head and the starts of the ranges in LDS
__device__ __forceinline__ void stage_ranges(const RelParams& p, int* s_start) {
    for (int k = threadIdx.x; k < p.r.n; k += 256) s_start[k] = k == 0 ? INT32_MIN : p.r.start[k];
}

__device__ __forceinline__ int find_range(const int* s_start, int n, int d) {  // last range that begins at or before d
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_start[mid] <= d) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename T> __global__ __launch_bounds__(256) void rel_bias_fwd_kernel(const RelParams p) {
    __shared__ int s_start[MAX_RANGES];
    __shared__ float s_w[MAX_RANGES];
    const int h = blockIdx.y;
    stage_ranges(p, s_start);
    for (int k = threadIdx.x; k < p.r.n; k += 256) {
        const int64_t at = p.r.bucket[k] * p.w_stride + h;
        s_w[k] = p.w_dtype == RGD_F32 ? static_cast<const float*>(p.w)[at]
                 : p.w_dtype == RGD_F16 ? to_f32(static_cast<const f16_t*>(p.w)[at]) : to_f32(static_cast<const bf16_t*>(p.w)[at]);
    }
    __syncthreads();
    const int task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (task >= p.tasks) return;
    const int c = task / p.strips, strip = (task - c * p.strips) * STRIP - (p.chunk - 8);
    const int i0 = c * p.chunk, rows = min(p.chunk, p.Tq - i0);
    int col = strip + 8 * lane_id();

    T v[15];
    {
        const int d0 = col - i0 - 7 - p.offset;
        int k = find_range(s_start, p.r.n, d0);
#pragma unroll
        for (int a = 0; a < 15; ++a) {
            while (k + 1 < p.r.n && s_start[k + 1] <= d0 + a) ++k;
            v[a] = from_f32<T>(s_w[k]);
        }
    }
    Block<T> row[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) __builtin_memcpy(&row[r], &v[7 - r], sizeof(row[r]));

    char* out = static_cast<char*>(p.bias) + (h * p.stride_h + i0 * p.stride_n) * (int64_t)sizeof(T) + col * (int64_t)sizeof(T);
    const int64_t step = p.stride_n * (int64_t)sizeof(T);
    for (int n = 0; n < rows; n += 8, col += 8, out += 8 * step + 8 * (int64_t)sizeof(T)) {
        if (col < 0 || col >= p.Tk) continue;
        if (n + 8 <= rows && col + 8 <= p.Tk) {
#pragma unroll
            for (int r = 0; r < 8; ++r) __builtin_memcpy(out + r * step, &row[r], sizeof(row[r]));
        } else {
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (n + r < rows) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (col + e < p.Tk) reinterpret_cast<T*>(out + r * step)[e] = v[e - r + 7];
                }
        }
    }
}

// part[(h * ranges + k) * tasks + task]: what the task adds to range k
template <typename T> __global__ __launch_bounds__(256) void rel_bias_bwd_kernel(const RelParams p) {
    __shared__ int s_start[MAX_RANGES];
    __shared__ float s_sum[4][STRIP + 8];
    const int h = blockIdx.y;
    stage_ranges(p, s_start);
    __syncthreads();
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int task = blockIdx.x * 4 + wave;
    if (task >= p.tasks) return;
    const int c = task / p.strips, strip = (task - c * p.strips) * STRIP - (p.chunk - 8);
    const int i0 = c * p.chunk, rows = min(p.chunk, p.Tq - i0);
    int col = strip + 8 * lane;

    float acc[15];
#pragma unroll
    for (int a = 0; a < 15; ++a) acc[a] = 0.f;
    const char* in = static_cast<const char*>(p.bias) + (h * p.stride_h + i0 * p.stride_n) * (int64_t)sizeof(T) + col * (int64_t)sizeof(T);
    const int64_t step = p.stride_n * (int64_t)sizeof(T);
    for (int n = 0; n < rows; n += 8, col += 8, in += 8 * step + 8 * (int64_t)sizeof(T)) {
        if (col < 0 || col >= p.Tk) continue;
        if (n + 8 <= rows && col + 8 <= p.Tk) {
            T x[8][8];
#pragma unroll
            for (int r = 0; r < 8; ++r) __builtin_memcpy(x[r], in + r * step, sizeof(x[r]));
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e - r + 7] += to_f32(x[r][e]);
        } else {
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n + r < rows && col + e < p.Tk) acc[e - r + 7] += to_f32(reinterpret_cast<const T*>(in + r * step)[e]);
        }
    }

    // diagonal 8 l + a of the strip: the lane's sum and, for a < 7, its left neighbour's a + 8
    float* sum = s_sum[wave];
#pragma unroll
    for (int a = 0; a < 8; ++a) {
        float v = acc[a];
        if (a < 7) {
            const float left = __shfl_up(acc[a + 8], 1, 64);
            v += lane > 0 ? left : 0.f;
        }
        sum[8 * lane + a] = v;
    }
    if (lane == 63) {
#pragma unroll
        for (int a = 8; a < 15; ++a) sum[STRIP + a - 8] = acc[a];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (a wavefront's own LDS rows: its accesses are in order)
    __builtin_amdgcn_wave_barrier();
    const int d0 = strip - i0 - 7 - p.offset;  // d of the first of STRIP + 7 diagonals
    float* out = p.part + (int64_t)h * p.r.n * p.tasks + task;
    for (int k = 0; k < p.r.n; ++k) {
        const int lo = k == 0 ? 0 : max(0, s_start[k] - d0);
        const int hi = k + 1 < p.r.n ? min(STRIP + 7, s_start[k + 1] - d0) : STRIP + 7;
        float s = 0.f;
        if (lo < hi) {
            for (int e = lo + lane; e < hi; e += 64) s += sum[e];
            s = group_reduce<64>(s);
        }
        if (lane == 0) out[(int64_t)k * p.tasks] = s;
    }
}

// one wavefront per (head, bucket): the tasks' sums in a fixed order
__global__ __launch_bounds__(64) void rel_bias_bucket_kernel(const RelParams p) {
    const int b = blockIdx.x, h = blockIdx.y;
    int k = -1;
    for (int i = 0; i < p.r.n; ++i) k = p.r.bucket[i] == b ? i : k;
    float s = 0.f;
    if (k >= 0) {
        const float* row = p.part + ((int64_t)h * p.r.n + k) * p.tasks;
        float s4[4] = {0.f, 0.f, 0.f, 0.f};
        int t = threadIdx.x;
        for (; t + 192 < p.tasks; t += 256) {
#pragma unroll
            for (int u = 0; u < 4; ++u) s4[u] += row[t + 64 * u];
        }
        for (; t < p.tasks; t += 64) s4[0] += row[t];
        s = group_reduce<64>((s4[0] + s4[1]) + (s4[2] + s4[3]));
    }
    if (threadIdx.x == 0) store_dyn(p.dw, p.w_dtype, b * p.w_stride + h, s);
}

int check_shape(const char* name, int64_t H, int64_t Tq, int64_t Tk, int64_t num_buckets, int64_t n_ranges, const int32_t* starts,
                const int32_t* buckets, int64_t offset) {
    RGD_REQUIRE(H >= 0 && Tq >= 0 && Tk >= 0, RGD_ERR_INVALID, "%s: negative shape", name);
    RGD_REQUIRE(H <= 65535, RGD_ERR_UNSUPPORTED, "%s: more than 65535 heads", name);
    const int64_t lim = int64_t(1) << 30;
    RGD_REQUIRE(Tq < lim && Tk < lim && offset > -lim && offset < lim, RGD_ERR_UNSUPPORTED, "%s: positions beyond 2^30", name);
    RGD_REQUIRE(n_ranges >= 1 && n_ranges <= MAX_RANGES && num_buckets >= 1 && num_buckets <= MAX_RANGES && starts && buckets,
                RGD_ERR_INVALID, "%s: 1 to %d ranges and buckets", name, MAX_RANGES);
    bool used[MAX_RANGES] = {};
    for (int64_t k = 0; k < n_ranges; ++k) {
        RGD_REQUIRE(buckets[k] >= 0 && buckets[k] < num_buckets && !used[buckets[k]], RGD_ERR_INVALID,
                    "%s: a bucket outside the weight, or one with two ranges", name);
        used[buckets[k]] = true;
        RGD_REQUIRE(k < 2 || starts[k] > starts[k - 1], RGD_ERR_INVALID, "%s: range starts must ascend", name);
    }
    const Split c = split(H > 0 ? H : 1, Tq, Tk);
    RGD_REQUIRE(c.tasks < (int64_t(1) << 31) - 4, RGD_ERR_UNSUPPORTED, "%s: too many positions", name);
    return RGD_OK;
}

void fill(RelParams* p, int64_t H, int64_t Tq, int64_t Tk, int64_t n_ranges, const int32_t* starts, const int32_t* buckets,
          int64_t offset, const rgd_tensor4* bias) {
    memset(p, 0, sizeof(*p));
    const Split s = split(H, Tq, Tk);
    p->H = (int)H;
    p->Tq = (int)Tq;
    p->Tk = (int)Tk;
    p->offset = (int)offset;
    p->chunk = (int)s.chunk;
    p->strips = (int)s.strips;
    p->tasks = Tq * Tk == 0 ? 0 : (int)s.tasks;
    if (bias) {
        p->bias = bias->ptr;
        p->stride_h = bias->stride_h;
        p->stride_n = bias->stride_n;
    }
    p->r.n = (int)n_ranges;
    memcpy(p->r.start, starts, n_ranges * sizeof(int));
    memcpy(p->r.bucket, buckets, n_ranges * sizeof(int));
}

}  // namespace

extern "C" {

int rgd_rel_bias_fwd(int64_t H, int64_t Tq, int64_t Tk, const void* weight, int64_t w_stride, int64_t num_buckets, int w_dtype,
                     int64_t n_ranges, const int32_t* starts, const int32_t* buckets, int64_t q_offset, const rgd_tensor4* bias,
                     int bias_dtype, void* stream) {
    const char* name = "rgd_rel_bias_fwd";
    rgd_ensure_init();
    RGD_REQUIRE(rgd_dtype_ok(w_dtype) && rgd_dtype_ok(bias_dtype), RGD_ERR_INVALID, "%s: Only support fp16, bf16, and fp32", name);
    const int rc = check_shape(name, H, Tq, Tk, num_buckets, n_ranges, starts, buckets, q_offset);
    if (rc != RGD_OK || H * Tq * Tk == 0) return rc;
    RGD_REQUIRE(weight && bias && bias->ptr, RGD_ERR_INVALID, "%s: null tensor", name);
    RelParams p;
    fill(&p, H, Tq, Tk, n_ranges, starts, buckets, q_offset, bias);
    p.w = weight;
    p.w_stride = w_stride;
    p.w_dtype = w_dtype;
    const dim3 grid((unsigned)((p.tasks + 3) / 4), (unsigned)H);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = bias_dtype == RGD_F16 ? rgd_launch(rel_bias_fwd_kernel<f16_t>, grid, dim3(256), 0, s, p)
                         : bias_dtype == RGD_BF16 ? rgd_launch(rel_bias_fwd_kernel<bf16_t>, grid, dim3(256), 0, s, p)
                                                  : rgd_launch(rel_bias_fwd_kernel<float>, grid, dim3(256), 0, s, p);
    return rgd_launch_status(name, e);
}

size_t rgd_rel_bias_bwd_workspace(int64_t H, int64_t Tq, int64_t Tk, int64_t num_buckets) {
    if (H <= 0 || Tq <= 0 || Tk <= 0 || num_buckets <= 0) return 0;
    return (size_t)(split(H, Tq, Tk).tasks * H * num_buckets) * sizeof(float);
}

int rgd_rel_bias_bwd(int64_t H, int64_t Tq, int64_t Tk, const rgd_tensor4* dbias, int dbias_dtype, int64_t n_ranges,
                     const int32_t* starts, const int32_t* buckets, int64_t q_offset, void* dweight, int64_t dw_stride,
                     int64_t num_buckets, int dw_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const char* name = "rgd_rel_bias_bwd";
    rgd_ensure_init();
    RGD_REQUIRE(rgd_dtype_ok(dw_dtype) && rgd_dtype_ok(dbias_dtype), RGD_ERR_INVALID, "%s: Only support fp16, bf16, and fp32", name);
    const int rc = check_shape(name, H, Tq, Tk, num_buckets, n_ranges, starts, buckets, q_offset);
    if (rc != RGD_OK || H == 0) return rc;
    const bool empty = Tq * Tk == 0;  // the gradient is zero
    RGD_REQUIRE(dweight && (empty || (dbias && dbias->ptr)), RGD_ERR_INVALID, "%s: null tensor", name);
    RGD_REQUIRE(workspace_bytes >= rgd_rel_bias_bwd_workspace(H, Tq, Tk, num_buckets) && (empty || workspace), RGD_ERR_WORKSPACE,
                "%s: workspace of %zu bytes, needs %zu", name, workspace_bytes, rgd_rel_bias_bwd_workspace(H, Tq, Tk, num_buckets));
    RelParams p;
    fill(&p, H, Tq, Tk, n_ranges, starts, buckets, q_offset, dbias);
    p.part = static_cast<float*>(workspace);
    p.dw = dweight;
    p.w_stride = dw_stride;
    p.w_dtype = dw_dtype;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (!empty) {
        const dim3 grid((unsigned)((p.tasks + 3) / 4), (unsigned)H);
        const hipError_t e = dbias_dtype == RGD_F16 ? rgd_launch(rel_bias_bwd_kernel<f16_t>, grid, dim3(256), 0, s, p)
                             : dbias_dtype == RGD_BF16 ? rgd_launch(rel_bias_bwd_kernel<bf16_t>, grid, dim3(256), 0, s, p)
                                                       : rgd_launch(rel_bias_bwd_kernel<float>, grid, dim3(256), 0, s, p);
        const int st = rgd_launch_status(name, e);
        if (st != RGD_OK) return st;
    }
    return rgd_launch_status(name, rgd_launch(rel_bias_bucket_kernel, dim3((unsigned)num_buckets, (unsigned)H), dim3(64), 0, s, p));
}

}  // extern "C"
