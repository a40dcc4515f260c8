// Layer norm over the rows of the atomic networks, forward and backward, and the pieces that the kernels of activation
// checkpoints share with it (ani_checkpoint.cuh).
//
// Rows are atoms in element order (start[t] .. start[t + 1] of element t), every element has its own gain and bias:
//   mean = sum x / w,  rstd = 1 / sqrt(sum (x - mean)^2 / w + eps),  xhat = (x - mean) rstd,  y = gain xhat + bias;
//   g = gain dy:  dx = rstd (g - sum g / w - xhat sum(g xhat) / w),  dgain = sum over rows dy xhat,  dbias = sum over rows dy.
//
// A row belongs to a TEAM of threads (8, 16 or 32 lanes of a warp, or 2, 4 or 8 warps), which keeps it in registers: thread l
// holds the NV groups of four consecutive columns 4 (l + k TEAM), so that the row is read once and the variance is the
// two-pass one (a mean far from zero costs the rounding of the mean itself, not that of its square).  Columns are four to a thread whether or not the rows are 16-byte
// aligned; only the load instruction differs.  All sums are held in the type of the rows: 32 bits for float.
//
// Sums over rows: a CTA takes a contiguous range of rows of ONE element, its teams add up in registers, the CTA adds its
// teams in order through shared memory and writes one partial row; a second launch adds the partial rows in order.  No
// atomics: results do not change from run to run.  An element with one range is written by the first launch, and when that
// holds for all of them there is no second one.
//
// Bound by memory: 110,000 x 384 forward 55 us (6.1 TB/s), 110,000 x 512 backward 108 us (6.2 TB/s, a copy runs at 6.5); rows of
// a training batch (13,750 x 128 backward, 3 us of traffic) by the length of a team's chain of rows, 7 us, and the second launch.
#pragma once

#include "ani_common.cuh"
#include "ani_launch.cuh"

namespace ani {

constexpr int kNormThreads = 256;
constexpr int kNormMaxWidth = 4096;

struct RowGroups {
    long long start[kTypes + 1];   // rows of element t: start[t] .. start[t + 1]
};
// Ranges of rows, one per CTA, each of one element.
struct RowRanges {
    RowGroups groups;
    long long rows;                // rows per range
    int range_start[kTypes + 1];   // prefix of ceil(rows of the element / rows)
};

__device__ __forceinline__ int element_of_row(const RowGroups& g, long long row)
{
    return (row >= g.start[1] ? 1 : 0) + (row >= g.start[2] ? 1 : 0) + (row >= g.start[3] ? 1 : 0);
}
struct RowRange {
    int element;
    long long first, end;
};
__device__ __forceinline__ RowRange range_of_cta(const RowRanges& r, int cta)
{
    RowRange out;
    out.element = 0;
#pragma unroll
    for (int t = 1; t < kTypes; t++) out.element += cta >= r.range_start[t] ? 1 : 0;
    out.first = r.groups.start[out.element] + (long long)(cta - r.range_start[out.element]) * r.rows;
    out.end = min(out.first + r.rows, r.groups.start[out.element + 1]);
    return out;
}

// Four consecutive columns of a row; columns >= w read as zero and are not written.  VEC: w is a multiple of four and the
// columns are one 16-byte access (two in double).
template <bool VEC, typename T> __device__ __forceinline__ void load_columns(const T* row, int col, int w, T* v)
{
    if (VEC) {
        if (col < w) {
            load4(row + col, v);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = T(0);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = col + i < w ? row[col + i] : T(0);
    }
}
// Whether column i of the four is inside the row (with VEC all are, or none).
template <bool VEC> __device__ __forceinline__ bool column_in(int col, int i, int w) { return VEC ? col < w : col + i < w; }
__device__ __forceinline__ void store4(float* p, const float* v) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(double* p, const double* v)
{
    *reinterpret_cast<double2*>(p) = make_double2(v[0], v[1]);
    *reinterpret_cast<double2*>(p + 2) = make_double2(v[2], v[3]);
}
template <bool VEC, typename T> __device__ __forceinline__ void store_columns(T* row, int col, int w, const T* v)
{
    if (VEC) {
        if (col < w) store4(row + col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (col + i < w) row[col + i] = v[i];
    }
}

// Barrier of the threads of a team of several warps.  (With the number in a register the compiler sets all sixteen barriers
// of a CTA aside.)
template <int TEAM> __device__ __forceinline__ void team_sync()
{
    if (TEAM == kNormThreads) {
        __syncthreads();
    } else {
        const int team = threadIdx.x / TEAM;
        if (team == 0) asm volatile("bar.sync 1, %0;" ::"n"(TEAM) : "memory");
        else if (team == 1) asm volatile("bar.sync 2, %0;" ::"n"(TEAM) : "memory");
        else if (team == 2) asm volatile("bar.sync 3, %0;" ::"n"(TEAM) : "memory");
        else asm volatile("bar.sync 4, %0;" ::"n"(TEAM) : "memory");
    }
}
static_assert(kNormThreads / 64 == 4, "teams of two warps or more: four at most");
// Where the warps of a team meet; two places in turn, so that a sum needs one barrier.
template <typename T> struct TeamScratch {
    T* values;      // [2][2 * warps of the CTA]
    int which;
    __device__ __forceinline__ T* next()
    {
        which ^= 1;
        return values + which * (2 * kNormThreads / kWarp);
    }
};
// Sums over a team, the same value in all of its threads; N <= 2.  Every thread of the CTA takes part.
template <int TEAM, int N, typename T> __device__ __forceinline__ void team_sum(T* v, TeamScratch<T>& scratch)
{
#pragma unroll
    for (int o = (TEAM < kWarp ? TEAM : kWarp) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(kFull, v[i], o);
    if (TEAM > kWarp) {
        T* place = scratch.next() + threadIdx.x / TEAM * (TEAM / kWarp) * N;
        if (lane_id() == 0)
#pragma unroll
            for (int i = 0; i < N; i++) place[warp_id() % (TEAM / kWarp) * N + i] = v[i];
        team_sync<TEAM>();
#pragma unroll
        for (int i = 0; i < N; i++) {
            T s = T(0);
#pragma unroll
            for (int k = 0; k < TEAM / kWarp; k++) s += place[k * N + i];
            v[i] = s;
        }
    }
}

__device__ __forceinline__ float rsqrt_full(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double rsqrt_full(double v) { return 1.0 / sqrt(v); }

// mean and 1 / sqrt(variance + eps) of the row that the team holds in x.
template <int TEAM, int NV, bool VEC, typename T>
__device__ __forceinline__ void row_statistics(const T (*x)[4], int lane, int w, T inv_w, T eps, TeamScratch<T>& scratch,
                                               T* mean, T* rstd)
{
    T s = T(0);
#pragma unroll
    for (int k = 0; k < NV; k++) s += (x[k][0] + x[k][1]) + (x[k][2] + x[k][3]);
    team_sum<TEAM, 1>(&s, scratch);
    const T m = s * inv_w;
    T q = T(0);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int col = 4 * (lane + k * TEAM);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const T d = column_in<VEC>(col, i, w) ? x[k][i] - m : T(0);
            q += d * d;
        }
    }
    team_sum<TEAM, 1>(&q, scratch);
    *mean = m;
    *rstd = rsqrt_full(q * inv_w + eps);
}

// The sums over the rows of a CTA's range, from the sums of its teams: added in the order of the teams and written to
// out[0 .. w).  Every thread of the CTA takes part.
template <int TEAM, int NV, typename T>
__device__ __forceinline__ void store_column_sums(const T (*v)[4], T* tile, T* out, int w)
{
    constexpr int teams = kNormThreads / TEAM;
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    if (TEAM == kNormThreads) {
#pragma unroll
        for (int k = 0; k < NV; k++) store_columns<false>(out, 4 * (lane + k * TEAM), w, v[k]);
        return;
    }
    __syncthreads();      // the tile of the sums before has been read
#pragma unroll
    for (int k = 0; k < NV; k++) store4(tile + (size_t)team * (TEAM * NV * 4) + 4 * (lane + k * TEAM), v[k]);
    __syncthreads();
    for (int c = threadIdx.x; c < w; c += kNormThreads) {
        T s = T(0);
#pragma unroll
        for (int t = 0; t < teams; t++) s += tile[t * (TEAM * NV * 4) + c];
        out[c] = s;
    }
}

// What the launches with sums over rows write: Q sums per element, each [width].
template <typename T, int Q> struct ColumnSums {
    T* out[Q][kTypes];     // null: not wanted
    T* partial;            // [ranges][Q][width]
};
template <typename T, int Q>
__device__ __forceinline__ T* column_sums_place(const ColumnSums<T, Q>& s, const RowRanges& r, int element, int cta, int q, int w)
{
    return r.range_start[element + 1] - r.range_start[element] == 1 ? s.out[q][element] : s.partial + ((size_t)cta * Q + q) * w;
}
// Sums of an element without rows are zero: written by the first CTA of the first launch.
template <typename T, int Q>
__device__ __forceinline__ void zero_sums_without_rows(const ColumnSums<T, Q>& s, const RowRanges& r, int w)
{
    if (blockIdx.x) return;
#pragma unroll
    for (int t = 0; t < kTypes; t++)
        if (r.range_start[t] == r.range_start[t + 1])
#pragma unroll
            for (int q = 0; q < Q; q++)
                if (s.out[q][t])
                    for (int c = threadIdx.x; c < w; c += kNormThreads) s.out[q][t][c] = T(0);
}

// A thread has a column and every 16th range: the launch is as long as a thread's chain of loads.
constexpr int kSumColumns = 32, kSumParts = 16;
template <typename T, int Q>
__global__ void __launch_bounds__(kSumColumns* kSumParts)
    column_sums_kernel(const __grid_constant__ ColumnSums<T, Q> s, const __grid_constant__ RowRanges r, int w)
{
    __shared__ T part[kSumParts][kSumColumns];
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.y / Q, q = blockIdx.y % Q, c = blockIdx.x * kSumColumns + threadIdx.x;
    const int first = r.range_start[t], n = r.range_start[t + 1] - first;
    if (n <= 1 || !s.out[q][t]) return;      // written by the first launch, or not wanted
    T sum = T(0);
    if (c < w) {
#pragma unroll 8
        for (int k = threadIdx.y; k < n; k += kSumParts) sum += s.partial[((size_t)(first + k) * Q + q) * w + c];
    }
    part[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y == 0 && c < w) {
        sum = part[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < kSumParts; k++) sum += part[k][threadIdx.x];
        s.out[q][t][c] = sum;
    }
}

// ------------------------------------------------------------------ layer norm
template <typename T> struct LayerNormParams {
    const T* x;
    long long x_stride;
    const T* gain[kTypes];
    const T* bias[kTypes];
    T *y, *mean, *rstd;
    RowGroups groups;
    int width;
    T inv_w, eps;
};

template <typename T, int TEAM, int NV, bool VEC>
__global__ void __launch_bounds__(kNormThreads) layer_norm_kernel(const __grid_constant__ LayerNormParams<T> p)
{
    __shared__ T scratch_sh[4 * kNormThreads / kWarp];
    TeamScratch<T> scratch = {scratch_sh, 0};
    constexpr int teams = kNormThreads / TEAM;
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const long long n = p.groups.start[kTypes];
    pdl_wait();
    pdl_trigger();
    for (long long base = (long long)blockIdx.x * teams; base < n; base += (long long)gridDim.x * teams) {
        const long long row = base + team;
        const bool live = row < n;
        T x[NV][4];
#pragma unroll
        for (int k = 0; k < NV; k++)
            load_columns<VEC>(p.x + (live ? row : 0) * p.x_stride, 4 * (lane + k * TEAM), live ? p.width : 0, x[k]);
        // asked for before the sums, whose chain is as long as a load from the second-level cache
        const int e = element_of_row(p.groups, live ? row : 0);
        T gain[NV][4], bias[NV][4];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            load_columns<VEC>(p.gain[e], 4 * (lane + k * TEAM), p.width, gain[k]);
            load_columns<VEC>(p.bias[e], 4 * (lane + k * TEAM), p.width, bias[k]);
        }
        T mean, rstd;
        row_statistics<TEAM, NV, VEC>(x, lane, p.width, p.inv_w, p.eps, scratch, &mean, &rstd);
        if (!live) continue;      // the teams of a CTA of 256 are one, and live
        T* y = p.y + row * p.width;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            if (col >= p.width) break;
#pragma unroll
            for (int i = 0; i < 4; i++) x[k][i] = (x[k][i] - mean) * rstd * gain[k][i] + bias[k][i];
            store_columns<VEC>(y, col, p.width, x[k]);
        }
        if (lane == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
    }
}

template <typename T> struct LayerNormGradParams {
    const T* grad_y;
    long long grad_stride;
    const T* x;
    long long x_stride;
    const T* gain[kTypes];
    const T *mean, *rstd;
    T* grad_x;
    ColumnSums<T, 2> sums;      // gain, bias
    RowRanges ranges;
    int width;
    T inv_w;
};

template <typename T, int TEAM, int NV, bool VEC>
__global__ void __launch_bounds__(kNormThreads) layer_norm_grad_kernel(const __grid_constant__ LayerNormGradParams<T> p)
{
    __shared__ T scratch_sh[4 * kNormThreads / kWarp];
    TeamScratch<T> scratch = {scratch_sh, 0};
    __shared__ alignas(16) T tile[TEAM == kNormThreads ? 4 : kNormThreads * NV * 4];
    constexpr int teams = kNormThreads / TEAM;
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM, w = p.width;
    pdl_wait();
    pdl_trigger();
    zero_sums_without_rows(p.sums, p.ranges, w);
    if ((int)blockIdx.x >= p.ranges.range_start[kTypes]) return;      // no rows at all: one CTA, for the zeros
    const RowRange range = range_of_cta(p.ranges, blockIdx.x);
    T gain[NV][4], dgain[NV][4], dbias[NV][4];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        load_columns<VEC>(p.gain[range.element], 4 * (lane + k * TEAM), w, gain[k]);
#pragma unroll
        for (int i = 0; i < 4; i++) dgain[k][i] = dbias[k][i] = T(0);
    }
    // with few columns to a thread a row is loaded one turn ahead (at 128 columns a range is four rows to a team)
    constexpr bool kAhead = NV == 1;
    T x_next[NV][4], up_next[NV][4], mean_next = T(0), rstd_next = T(0);
    auto load = [&](long long base) {
        const bool live = base + team < range.end;
        const long long row = live ? base + team : range.first;
        mean_next = p.mean[row];
        rstd_next = p.rstd[row];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            load_columns<VEC>(p.x + row * p.x_stride, col, live ? w : 0, x_next[k]);
            load_columns<VEC>(p.grad_y + row * p.grad_stride, col, live ? w : 0, up_next[k]);
        }
    };
    if (kAhead) load(range.first);
    for (long long base = range.first; base < range.end; base += teams) {
        const bool live = base + team < range.end;
        const long long row = base + team;
        if (!kAhead) load(base);
        T xhat[NV][4], up[NV][4];
        const T mean = mean_next, rstd = rstd_next;
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                xhat[k][i] = x_next[k][i];
                up[k][i] = up_next[k][i];
            }
        if (kAhead && base + teams < range.end) load(base + teams);
        T sum[2] = {T(0), T(0)};
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                xhat[k][i] = live && column_in<VEC>(col, i, w) ? (xhat[k][i] - mean) * rstd : T(0);
                dgain[k][i] += up[k][i] * xhat[k][i];
                dbias[k][i] += up[k][i];
                up[k][i] *= gain[k][i];
                sum[0] += up[k][i];
                sum[1] += up[k][i] * xhat[k][i];
            }
        }
        team_sum<TEAM, 2>(sum, scratch);
        if (!live) continue;
        sum[0] *= p.inv_w;
        sum[1] *= p.inv_w;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            if (col >= w) break;
#pragma unroll
            for (int i = 0; i < 4; i++) up[k][i] = rstd * (up[k][i] - sum[0] - xhat[k][i] * sum[1]);
            store_columns<VEC>(p.grad_x + row * w, col, w, up[k]);
        }
    }
    store_column_sums<TEAM, NV>(dgain, tile, column_sums_place(p.sums, p.ranges, range.element, blockIdx.x, 0, w), w);
    store_column_sums<TEAM, NV>(dbias, tile, column_sums_place(p.sums, p.ranges, range.element, blockIdx.x, 1, w), w);
}

}  // namespace ani
