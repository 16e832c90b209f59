// Learned relative position bias and the gradient of its weight.
//
//   bias[h][i][j] = W[bucket(j - i - q_offset)][h],   dW[b][h] = sum of dbias[h][i][j] over bucket(j - i - q_offset) = b
//
// A bucket is a range of the relative distance d = j - i - q_offset: the matrix is constant along its diagonals, and the gradient
// is the sum of each diagonal, added up over the diagonals of a bucket.  Bound by memory: the matrix is written (forward) or
// read (backward) once.
//
// The backward, and the forward of a matrix of up to 64 MB, walk the matrix along its diagonals.  A wavefront takes a strip of 512
// columns and goes down `chunk` rows, 8 rows and 8 columns at a time: lane l holds the 8 x 8 block whose columns
// begin at strip + 8 l + 8 n in step n, so the 15 diagonals of a lane's block are the same in every step.
//   forward   the 15 values are looked up once, the 8 rows of the block packed once; each step is eight 16-byte stores
//   backward  15 sums stay in registers; each step is eight 16-byte streaming loads and 64 additions
// Blocks left of the first or right of the last column are skipped.
// A matrix beyond 64 MB is written in address order instead: the memory takes 6.9 TB/s from workgroups that write 4 KB side by
// side in the order they are launched, and 4 from the walk, whose workgroups write 8 rows each all over the matrix.  The
// values of a head's diagonals are first laid out in a row of the workspace (read back from the L2), then each thread takes
// 8 columns of two rows (one row: too few bytes in flight for a round trip to the L2, 4.4 TB/s; four rows 5.7, two 6.2).
// bf16, walk / address order: (24, 4352, 4352) 222 / 172 us, (16, 2048, 2048) 33 / 26 us, (16, 1024, 1024) 10.5 / 11 us.  (Between
// 34 and 134 MB, and in fp32, where the walk reaches 3.2 TB/s at 50 MB, the border was not looked for.)
// Rows need no alignment: those written in address order are cut at the 16-byte boundaries of each row, the walk loads and stores
// at any address, which the hardware takes.  A block that the last column cuts is read further left and shifted (element
// by element its wavefront was the last to end: (24, 4352, 4351) bf16 381 us instead of 165).
#include "common.h"

#include <string.h>

namespace {

constexpr int MAX_RANGES = 256;
constexpr int STRIP = 512;
constexpr int64_t ORDERED_BYTES = int64_t(64) << 20;  // larger matrices are written in address order
constexpr int VALUES_BEFORE = 8;                      // values in front of the first row's, for a row that begins off a boundary

struct RelRanges {  // range k: start[k] <= d < start[k + 1], ascending; start[0] covers everything below; the rest INT32_MAX
    int n;
    int half;  // largest power of two below n (0 for one range)
    int start[MAX_RANGES];
    int16_t bucket[MAX_RANGES];  // of a range
    int16_t range[MAX_RANGES];   // of a bucket, -1: none
};

struct RelParams {
    const void* w;  // forward: weight
    void* bias;     // forward: written; backward: dbias, read
    void* part;     // backward: sums [head][range][task]; forward in address order: values of the diagonals [head][width]
    void* dw;
    int64_t w_stride, stride_h, stride_n;
    int w_dtype, H, Tq, Tk, offset;
    int chunk, strips, tasks;
    int width;       // address order: values of a head; value e is that of d = e - VALUES_BEFORE - Tq - offset
    FastDiv blocks;  // address order: 8-column blocks of a row
    RelRanges r;
};

struct Split {
    int64_t chunk, chunks, strips, tasks;
};

// Rows of a task.  Long tasks spend less on their beginning and end (looking values up, adding ranges up) and waste fewer lanes at
// the slanted edges, short ones fill the chip: the longest of 16 .. 256 rows that still gives every compute unit 8
// wavefronts.  Backward with 4 / 8 / 16 / 32 of them, bf16: (24, 4352, 4352) 148 / 148 / 153 / 154 us, (16, 2048, 2048)
// 29 / 28 / 26 / 28 us, (16, 2560, 2560) 37 / 38 / 40 / 42 us.
Split split(int64_t H, int64_t Tq, int64_t Tk) {
    Split s;
    for (s.chunk = 256;; s.chunk /= 2) {
        s.chunks = (Tq + s.chunk - 1) / s.chunk;
        s.strips = (Tk + s.chunk - 8 + STRIP - 1) / STRIP;
        s.tasks = s.chunks * s.strips;
        if (s.chunk == 16 || s.tasks * H >= 8 * (int64_t)rgd_num_cus()) return s;
    }
}

// 8 consecutive elements at any address: 16-byte accesses, unaligned where the row is
typedef u32x4 u32x4_any __attribute__((aligned(2)));
template <typename T> struct Block {
    static constexpr int NV = 8 * sizeof(T) / 16;
    u32x4 v[NV];
    // streaming (a gradient is read once): without it (24, 4352, 4352) bf16 takes 237 us instead of 147
    __device__ __forceinline__ void load(const char* p) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p) + i);
    }
    // element e becomes element e + s, zeros from the end (bit operations: choices by a condition would become branches)
    __device__ __forceinline__ Block down(int s) const {
        constexpr int N = 4 * NV;
        uint32_t w[N];
#pragma unroll
        for (int k = 0; k < N; ++k) w[k] = v[k / 4][k % 4];
        const int bytes = s * (int)sizeof(T);
#pragma unroll
        for (int d = N / 2; d >= 1; d /= 2) {  // by d dwords
            const uint32_t m = 0u - (bytes / (4 * d) & 1);
#pragma unroll
            for (int k = 0; k < N; ++k) w[k] = ((k + d < N ? w[k + d] : 0u) & m) | (w[k] & ~m);
        }
        Block b;
#pragma unroll
        for (int k = 0; k < N; ++k)
            b.v[k / 4][k % 4] = sizeof(T) == 2 ? __builtin_amdgcn_alignbyte(k + 1 < N ? w[k + 1] : 0u, w[k], bytes & 2) : w[k];
        return b;
    }
    __device__ __forceinline__ void fetch(const T* p) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = reinterpret_cast<const u32x4_any*>(p)[i];
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) reinterpret_cast<u32x4_any*>(p)[i] = v[i];
    }
};

__device__ __forceinline__ float load_dyn(const void* p, int dtype, int64_t i) {
    return dtype == RGD_F32 ? static_cast<const float*>(p)[i]
           : dtype == RGD_F16 ? to_f32(static_cast<const f16_t*>(p)[i]) : to_f32(static_cast<const bf16_t*>(p)[i]);
}

// the range starts and the weight of head h by range, for the workgroup
__device__ __forceinline__ void stage_weight(const RelParams& p, int h, int* s_start, float* s_w) {
    const int k = threadIdx.x;  // 256 threads, 256 ranges at most
    s_start[k] = k == 0 ? INT32_MIN : p.r.start[k];
    if (k < p.r.n) s_w[k] = load_dyn(p.w, p.w_dtype, p.r.bucket[k] * p.w_stride + h);
    __syncthreads();
}

// for N distances d, d + 1, ..: the last range that begins at or before each (starts beyond n are INT32_MAX), side by side
template <int N> __device__ __forceinline__ void find_ranges(const int* s_start, int half, int d, int (&at)[N]) {
#pragma unroll
    for (int a = 0; a < N; ++a) at[a] = 0;
    for (; half > 0; half >>= 1) {
#pragma unroll
        for (int a = 0; a < N; ++a) at[a] += s_start[at[a] + half] <= d + a ? half : 0;
    }
}

template <typename T> __global__ __launch_bounds__(256) void rel_bias_fwd_kernel(const RelParams p) {
    __shared__ int s_start[MAX_RANGES];
    __shared__ float s_w[MAX_RANGES];
    const int h = blockIdx.y;
    stage_weight(p, h, s_start, s_w);
    const int task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (task >= p.tasks) return;
    const int c = task / p.strips, strip = (task - c * p.strips) * STRIP - (p.chunk - 8);
    const int i0 = c * p.chunk, rows = min(p.chunk, p.Tq - i0);
    int col = strip + 8 * lane_id();

    T v[15];
    {
        int at[15];
        find_ranges(s_start, p.r.half, col - i0 - 7 - p.offset, at);
#pragma unroll
        for (int a = 0; a < 15; ++a) v[a] = from_f32<T>(s_w[at[a]]);
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
            for (int r = 0; r < 8; ++r) row[r].store(reinterpret_cast<T*>(out + r * step));
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

// the values of a head's diagonals, in the bias type
template <typename T> __global__ __launch_bounds__(256) void rel_bias_values_kernel(const RelParams p) {
    __shared__ int s_start[MAX_RANGES];
    __shared__ float s_w[MAX_RANGES];
    const int h = blockIdx.y, e = blockIdx.x * 256 + threadIdx.x;
    stage_weight(p, h, s_start, s_w);
    if (e >= p.width) return;
    int at[1];
    find_ranges(s_start, p.r.half, e - VALUES_BEFORE - p.Tq - p.offset, at);
    static_cast<T*>(p.part)[(int64_t)h * p.width + e] = from_f32<T>(s_w[at[0]]);
}

// thread: 8 columns of rows 2 rb and 2 rb + 1, in each row from the 16-byte boundary at or before column 8 cb
template <typename T> __global__ __launch_bounds__(256) void rel_bias_ordered_kernel(const RelParams p) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    const uint32_t rb = fast_div(c, p.blocks), cb = c - rb * p.blocks.d;
    const int h = blockIdx.y;
    const T* values = static_cast<const T*>(p.part) + (int64_t)h * p.width;
    Block<T> v[2];
    T* row[2];
    int col[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int i = min(2 * (int)rb + r, p.Tq - 1);
        row[r] = static_cast<T*>(p.bias) + h * p.stride_h + i * p.stride_n;
        col[r] = 8 * (int)cb - (int)(reinterpret_cast<uintptr_t>(row[r]) % 16 / sizeof(T));
        v[r].fetch(values + (col[r] - i + p.Tq + VALUES_BEFORE));
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if (2 * (int)rb + r >= p.Tq) break;
        if (col[r] >= 0 && col[r] + 8 <= p.Tk) {
            v[r].store(row[r] + col[r]);
        } else {
            T one[8];
            __builtin_memcpy(one, &v[r], sizeof(one));
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col[r] + e >= 0 && col[r] + e < p.Tk) row[r][col[r] + e] = one[e];
        }
    }
}

// part[(h * ranges + k) * tasks + task]: what the task adds to range k
template <typename T> __global__ __launch_bounds__(256) void rel_bias_bwd_kernel(const RelParams p) {
    __shared__ double s_sum[4][STRIP + 8];
    __shared__ alignas(8) uint8_t s_begin[4][STRIP + 8];  // a range begins at this diagonal
    const int h = blockIdx.y;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int task = blockIdx.x * 4 + wave;
    if (task >= p.tasks) return;
    const int c = task / p.strips, strip = (task - c * p.strips) * STRIP - (p.chunk - 8);
    const int i0 = c * p.chunk, rows = min(p.chunk, p.Tq - i0);
    int col = strip + 8 * lane;

    float acc[15];
#pragma unroll
    for (int a = 0; a < 15; ++a) acc[a] = 0.f;
    const int64_t step = p.stride_n * (int64_t)sizeof(T);
    const char* in = static_cast<const char*>(p.bias) + (h * p.stride_h + i0 * p.stride_n) * (int64_t)sizeof(T) + col * (int64_t)sizeof(T);
    const int over = (8 - p.Tk % 8) % 8;  // columns that a block cut by the last column lacks: it is read that much further left
    if (p.Tk >= 8) {
        for (int n = 0; n < rows; n += 8, col += 8, in += 8 * step + 8 * (int64_t)sizeof(T)) {
            if (col < 0 || col >= p.Tk) continue;
            const bool cut = col + 8 > p.Tk;
            const char* from = in - (cut ? over * (int)sizeof(T) : 0);
            const int left = rows - n;
            Block<T> x[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r].load(from + min(r, left - 1) * step);
            if (__any(cut)) {
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const Block<T> y = x[r].down(over);
#pragma unroll
                    for (int i = 0; i < Block<T>::NV; ++i) x[r].v[i] = cut ? y.v[i] : x[r].v[i];
                }
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (r < left) {
                    T row[8];
                    __builtin_memcpy(row, &x[r], sizeof(row));
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[e - r + 7] += to_f32(row[e]);
                }
            }
        }
    } else {  // rows shorter than a block: element by element
        for (int n = 0; n < rows; n += 8, col += 8, in += 8 * step + 8 * (int64_t)sizeof(T)) {
            if (col < 0 || col >= p.Tk) continue;
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n + r < rows && col + e < p.Tk) acc[e - r + 7] += to_f32(reinterpret_cast<const T*>(in + r * step)[e]);
        }
    }

    // Diagonal 8 l + a of the strip is the lane's sum and, for a < 7, its left neighbour's a + 8; the last lane's a + 8 are the
    // last seven.
    float line[8];
#pragma unroll
    for (int a = 0; a < 8; ++a) {
        line[a] = acc[a];
        if (a < 7) {
            const float left = __shfl_up(acc[a + 8], 1, 64);
            line[a] += lane > 0 ? left : 0.f;
        }
    }
    // A running sum of the diagonals, in 64 bits, that starts anew where a range begins: a range's sum is what stands at its last
    // diagonal, and no range sees another's infinities or large numbers, as it would in differences of one running sum (those are
    // 0.3 us shorter: (8, 128, 128) 7.0 / 7.3 us, (16, 2048, 2048) 28.4 / 28.8 us, (16, 1024, 1024) with 256 buckets 16.5 / 18.0 us).
    double* sum = s_sum[wave];
    uint8_t* begin = s_begin[wave];
    const int d0 = strip - i0 - 7 - p.offset;  // d of the first of STRIP + 7 diagonals
    auto first_of = [&](int k) { return (int)min((int64_t)STRIP + 7, max((int64_t)0, (int64_t)p.r.start[k] - d0)); };
    auto ordered = [] {  // (a wavefront's own LDS rows: its accesses are in order)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    reinterpret_cast<uint64_t*>(begin)[lane] = 0;
    if (lane == 0) reinterpret_cast<uint64_t*>(begin)[64] = 0;
    ordered();
    for (int k = lane; k < p.r.n; k += 64)
        if (k > 0) begin[first_of(k)] = 1;  // (range 0 has no beginning; STRIP + 7 is no diagonal)
    ordered();
    const uint64_t mine = reinterpret_cast<const uint64_t*>(begin)[lane], rest = reinterpret_cast<const uint64_t*>(begin)[64];
    auto begins = [&](int a) { return ((a < 8 ? mine : rest) >> (8 * (a & 7)) & 1) != 0; };
    double total = 0.;  // of the lane's diagonals from its last beginning on
#pragma unroll
    for (int a = 0; a < 8; ++a) total = (begins(a) ? 0. : total) + line[a];
    int any = mine != 0;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const double up = __shfl_up(total, m, 64);
        const int up_any = __shfl_up(any, m, 64);
        if (lane >= m) {
            total = any ? total : up + total;
            any |= up_any;
        }
    }
    const double before = __shfl_up(total, 1, 64);
    double run = lane > 0 ? before : 0.;
#pragma unroll
    for (int a = 0; a < 15; ++a) {
        if (a >= 8 && lane < 63) break;
        run = (begins(a) ? 0. : run) + (a < 8 ? line[a & 7] : acc[a]);
        sum[8 * lane + a] = run;
    }
    ordered();
    float* out = static_cast<float*>(p.part) + (int64_t)h * p.r.n * p.tasks + task;
    for (int k = lane; k < p.r.n; k += 64) {
        const int lo = k == 0 ? 0 : first_of(k), hi = k + 1 < p.r.n ? first_of(k + 1) : STRIP + 7;
        out[(int64_t)k * p.tasks] = hi > lo ? (float)sum[hi - 1] : 0.f;
    }
}

// one wavefront per (head, bucket): the tasks' sums in a fixed order
__global__ __launch_bounds__(64) void rel_bias_bucket_kernel(const RelParams p) {
    const int b = blockIdx.x, h = blockIdx.y;
    const int k = p.r.range[b];
    float s = 0.f;
    if (k >= 0) {
        const float* row = static_cast<const float*>(p.part) + ((int64_t)h * p.r.n + k) * p.tasks;
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
    RGD_REQUIRE(Tq + Tk + (offset < 0 ? -offset : offset) <= 2 * lim - 2048, RGD_ERR_UNSUPPORTED, "%s: distances beyond 2^31", name);
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
    for (p->r.half = 0; (p->r.half ? 2 * p->r.half : 1) < n_ranges;) p->r.half = p->r.half ? 2 * p->r.half : 1;
    for (int k = 0; k < MAX_RANGES; ++k) {
        p->r.start[k] = k < n_ranges ? starts[k] : INT32_MAX;
        p->r.range[k] = -1;
    }
    for (int k = 0; k < n_ranges; ++k) {
        p->r.bucket[k] = (int16_t)buckets[k];
        p->r.range[buckets[k]] = (int16_t)k;
    }
}

// values of a head's diagonals: VALUES_BEFORE, then d = -Tq - offset .. Tk - 1 - offset, then what the last block holds beyond: it
// begins at column Tk + 6 at most, value VALUES_BEFORE + Tq + Tk + 6 in the first row
int64_t values_of(int64_t Tq, int64_t Tk) { return (VALUES_BEFORE + Tq + Tk + 6 + 8 + 7) / 8 * 8; }

template <typename T> int ordered(const char* name, RelParams& p, hipStream_t s) {
    const int64_t es = sizeof(T);
    const bool aligned = rgd_aligned16(p.bias) && p.stride_n * es % 16 == 0 && p.stride_h * es % 16 == 0;
    p.blocks = make_fastdiv((uint32_t)((p.Tk + (aligned ? 7 : 14)) / 8));  // (one more where rows begin off a boundary)
    const dim3 values((unsigned)((p.width + 255) / 256), (unsigned)p.H);
    const int rc = rgd_launch_status(name, rgd_launch(rel_bias_values_kernel<T>, values, dim3(256), 0, s, p));
    if (rc != RGD_OK) return rc;
    const int64_t blocks = (int64_t)((p.Tq + 1) / 2) * p.blocks.d;
    const dim3 grid((unsigned)((blocks + 255) / 256), (unsigned)p.H);
    return rgd_launch_status(name, rgd_launch(rel_bias_ordered_kernel<T>, grid, dim3(256), 0, s, p));
}

}  // namespace

extern "C" {

size_t rgd_rel_bias_fwd_workspace(int64_t H, int64_t Tq, int64_t Tk, int bias_dtype) {
    const int64_t lim = int64_t(1) << 30;
    if (H <= 0 || Tq <= 0 || Tk <= 0 || Tq >= lim || Tk >= lim || !rgd_dtype_ok(bias_dtype)) return 0;
    const int64_t es = rgd_dtype_size(bias_dtype);
    if (H * ((double)Tq * Tk * es) <= (double)ORDERED_BYTES || ((Tq + 1) / 2) * ((Tk + 14) / 8) >= (int64_t(1) << 31) - 256) return 0;
    return (size_t)(H * values_of(Tq, Tk) * es);
}

int rgd_rel_bias_fwd(int64_t H, int64_t Tq, int64_t Tk, const void* weight, int64_t w_stride, int64_t num_buckets, int w_dtype,
                     int64_t n_ranges, const int32_t* starts, const int32_t* buckets, int64_t q_offset, const rgd_tensor4* bias,
                     int bias_dtype, void* workspace, size_t workspace_bytes, void* stream) {
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
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (workspace && workspace_bytes > 0 && workspace_bytes >= rgd_rel_bias_fwd_workspace(H, Tq, Tk, bias_dtype) &&
        rgd_rel_bias_fwd_workspace(H, Tq, Tk, bias_dtype) > 0) {
        RGD_REQUIRE(rgd_aligned16(workspace), RGD_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", name);
        p.part = workspace;
        p.width = (int)values_of(Tq, Tk);
        return bias_dtype == RGD_F16 ? ordered<f16_t>(name, p, s) : bias_dtype == RGD_BF16 ? ordered<bf16_t>(name, p, s) : ordered<float>(name, p, s);
    }
    const dim3 grid((unsigned)((p.tasks + 3) / 4), (unsigned)H);
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
    RGD_REQUIRE(empty || rgd_aligned16(workspace), RGD_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", name);
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
