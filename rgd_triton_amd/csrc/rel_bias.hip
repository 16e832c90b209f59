// Learned relative position bias and the gradient of its weight.
//
//   bias[h][i][j] = W[bucket(j - i - q_offset)][h],   dW[b][h] = sum of dbias[h][i][j] over bucket(j - i - q_offset) = b
//
// A bucket is a range of the relative distance d = j - i - q_offset, so both directions only ever look at diagonals: the
// matrix is constant along each, and the gradient is the sum of each, added up over the diagonals of a bucket.  Bound by memory:
// the matrix is written (forward) or read (backward) once.
#include "common.h"

#include <string.h>

namespace {

constexpr int MAX_RANGES = 256;
constexpr int ROW_CHUNK = 512;  // rows whose diagonals one partial row of the backward sums

struct RelRanges {  // range k: start[k] <= d < start[k + 1], ascending, bucket[k]; start[0] covers everything below
    int n;
    int start[MAX_RANGES];
    int bucket[MAX_RANGES];
};

struct RelFwdParams {
    const void* w;
    void* bias;
    int64_t w_stride, stride_h, stride_n;
    int w_dtype, bias_dtype, H, Tq, Tk, offset;
    RelRanges r;
};

struct RelBwdParams {
    const void* dbias;
    float* part;
    void* dw;
    int64_t dw_stride, stride_h, stride_n;
    int dw_dtype, dbias_dtype, H, Tq, Tk, offset, width, chunks;
    int lo[MAX_RANGES], hi[MAX_RANGES];  // per bucket: lo <= d < hi
};

__device__ __forceinline__ float load_dyn(const void* p, int dtype, int64_t i) {
    if (dtype == RGD_BF16) return to_f32(static_cast<const bf16_t*>(p)[i]);
    if (dtype == RGD_F16) return to_f32(static_cast<const f16_t*>(p)[i]);
    return static_cast<const float*>(p)[i];
}

__global__ __launch_bounds__(256) void rel_bias_fwd_kernel(const RelFwdParams p) {
    const int h = blockIdx.z;
    for (int i = blockIdx.y; i < p.Tq; i += gridDim.y) {
        const int j = blockIdx.x * 256 + threadIdx.x;
        if (j >= p.Tk) continue;
        const int d = j - i - p.offset;
        int k = 0;
        while (k + 1 < p.r.n && d >= p.r.start[k + 1]) ++k;
        const float v = load_dyn(p.w, p.w_dtype, p.r.bucket[k] * p.w_stride + h);
        store_dyn(p.bias, p.bias_dtype, h * p.stride_h + i * p.stride_n + j, v);
    }
}

// part[(chunk * H + h) * width + e]: sum over the chunk's rows i of dbias[h][i][i - i0 + e - (ROW_CHUNK - 1)]
__global__ __launch_bounds__(256) void rel_bias_diagonal_kernel(const RelBwdParams p) {
    const int e = blockIdx.x * 256 + threadIdx.x;
    if (e >= p.width) return;
    const int h = blockIdx.z;
    const int i0 = blockIdx.y * ROW_CHUNK;
    const int rows = min(ROW_CHUNK, p.Tq - i0);
    float s = 0.f;
    for (int r = 0; r < rows; ++r) {
        const int j = e - (ROW_CHUNK - 1) + r;
        if (j >= 0 && j < p.Tk) s += load_dyn(p.dbias, p.dbias_dtype, h * p.stride_h + (int64_t)(i0 + r) * p.stride_n + j);
    }
    p.part[((int64_t)blockIdx.y * p.H + h) * p.width + e] = s;
}

__global__ __launch_bounds__(256) void rel_bias_bucket_kernel(const RelBwdParams p) {
    __shared__ float sums[4];
    const int b = blockIdx.x, h = blockIdx.y;
    float s = 0.f;
    for (int c = 0; c < p.chunks; ++c) {
        // d = e - (ROW_CHUNK - 1) - i0 - offset
        const int64_t shift = (int64_t)(ROW_CHUNK - 1) + (int64_t)c * ROW_CHUNK + p.offset;
        const int64_t lo = max((int64_t)0, p.lo[b] + shift), hi = min((int64_t)p.width, p.hi[b] + shift);
        const float* row = p.part + ((int64_t)c * p.H + h) * p.width;
        for (int64_t e = lo + threadIdx.x; e < hi; e += 256) s += row[e];
    }
    s = group_reduce<64>(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) store_dyn(p.dw, p.dw_dtype, b * p.dw_stride + h, (sums[0] + sums[1]) + (sums[2] + sums[3]));
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
    return RGD_OK;
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
    RelFwdParams p;
    memset(&p, 0, sizeof(p));
    p.w = weight;
    p.w_stride = w_stride;
    p.w_dtype = w_dtype;
    p.bias = bias->ptr;
    p.stride_h = bias->stride_h;
    p.stride_n = bias->stride_n;
    p.bias_dtype = bias_dtype;
    p.H = (int)H;
    p.Tq = (int)Tq;
    p.Tk = (int)Tk;
    p.offset = (int)q_offset;
    p.r.n = (int)n_ranges;
    memcpy(p.r.start, starts, n_ranges * sizeof(int));
    memcpy(p.r.bucket, buckets, n_ranges * sizeof(int));
    const dim3 grid((unsigned)((Tk + 255) / 256), (unsigned)(Tq < 65535 ? Tq : 65535), (unsigned)H);
    return rgd_launch_status(name, rgd_launch(rel_bias_fwd_kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), p));
}

size_t rgd_rel_bias_bwd_workspace(int64_t H, int64_t Tq, int64_t Tk) {
    if (H <= 0 || Tq <= 0 || Tk <= 0) return 0;
    return (size_t)((Tq + ROW_CHUNK - 1) / ROW_CHUNK) * H * (Tk + ROW_CHUNK - 1) * sizeof(float);
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
    RGD_REQUIRE(workspace_bytes >= rgd_rel_bias_bwd_workspace(H, Tq, Tk) && (empty || workspace), RGD_ERR_WORKSPACE,
                "%s: workspace of %zu bytes, needs %zu", name, workspace_bytes, rgd_rel_bias_bwd_workspace(H, Tq, Tk));
    RelBwdParams p;
    memset(&p, 0, sizeof(p));
    p.part = static_cast<float*>(workspace);
    p.dw = dweight;
    p.dw_stride = dw_stride;
    p.dw_dtype = dw_dtype;
    p.dbias_dtype = dbias_dtype;
    p.H = (int)H;
    p.Tq = (int)Tq;
    p.Tk = (int)Tk;
    p.offset = (int)q_offset;
    p.width = (int)(Tk + ROW_CHUNK - 1);
    p.chunks = empty ? 0 : (int)((Tq + ROW_CHUNK - 1) / ROW_CHUNK);
    for (int64_t k = 0; k < n_ranges; ++k) {
        p.lo[buckets[k]] = k == 0 ? INT32_MIN : starts[k];
        p.hi[buckets[k]] = k + 1 < n_ranges ? starts[k + 1] : INT32_MAX;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (!empty) {
        p.dbias = dbias->ptr;
        p.stride_h = dbias->stride_h;
        p.stride_n = dbias->stride_n;
        RGD_REQUIRE(p.chunks <= 65535, RGD_ERR_UNSUPPORTED, "%s: too many query rows", name);
        const dim3 grid((unsigned)((p.width + 255) / 256), (unsigned)p.chunks, (unsigned)H);
        const int st = rgd_launch_status(name, rgd_launch(rel_bias_diagonal_kernel, grid, dim3(256), 0, s, p));
        if (st != RGD_OK) return st;
    }
    return rgd_launch_status(name, rgd_launch(rel_bias_bucket_kernel, dim3((unsigned)num_buckets, (unsigned)H), dim3(256), 0, s, p));
}

}  // extern "C"
