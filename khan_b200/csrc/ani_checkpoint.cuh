// Activations of a layer whose input is kept in 8 bits for the backward pass.
//
// Forward, row by row (z: what the dense layer left; with a gain, u = gain (z - mean) rstd + bias, else u = z):
//   a = act(u);  codes: of every block of 128 columns  base = min z, step = (max z - min z) / 255,
//   code = rint((z - base) / step) in 0 .. 255, one byte;  mean and rstd are those of z itself.
// Backward, from codes alone:  z~ = base + code step (|z~ - z| <= step / 2),  u~ from z~ as u from z,
//   du = da act'(u~);  without gain dz = du, with it dz as in the layer norm's backward pass with xhat~ = (z~ - mean) rstd;
//   column sums of dz (the gradient of the dense layer's bias) and with a gain of du xhat~ and du.
// The codes are defined by float32 operations, each rounded once, so that they do not depend on who computes them:
//   step = (max - min) * (1 / 255),  code = rint((z - base) * (1 / step)),
// a block whose step is below 1e-30 is its base (step 0).  Counting from the minimum, not from the middle or from zero,
// keeps z - base exact where it matters: a block far from zero still has all of its 256 steps.  A block that holds something
// that is not finite, or that spans more than the largest float, has base NaN: its gradients are NaN and not wrong.
//
// One byte a value and 8 bytes a block (6 %) instead of the 8 bytes a value that z and a, or a and its derivative, take.
//
// 9.06 bytes a value either way.  110,000 x 512 with a norm, one call behind the other: forward 87 us with celu, 91 with softplus
// (78 us of traffic; bound by instructions, 40 for 32 values, 70 % of the issue slots), backward with its sums 96 and 100 us (bound
// by the latency of its loads: a row's sums, xhat and gradients are 126 registers, which leaves 16 warps an SM).
#pragma once

#include "ani_mlp.cuh"
#include "ani_norm.cuh"

namespace ani {

constexpr int kCheckpointBlock = 128;
__host__ __device__ __forceinline__ int checkpoint_row_bytes(int width) { return (width + 15) & ~15; }
__host__ __device__ __forceinline__ int checkpoint_blocks(int width) { return (width + kCheckpointBlock - 1) / kCheckpointBlock; }

// Smaller / larger of two values, NaN if one of them is.
__device__ __forceinline__ float min_nan(float a, float b)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The activation functions on the special function unit's exponential (2^-22 of its value; the argument's rounding adds
// |x| 2^-24): a few 1e-7 of max(1, |a|), in a quarter of the instructions of expf and log1pf, and without a branch: celu as
// "u or 0.1 (exp(10 u) - 1)" was compiled to one, and 32 values of a thread took 5000 clocks instead of 700.
constexpr float kLog2E = 1.4426950408889634f;
__device__ __forceinline__ float fast_exp2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float fast_reciprocal(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Two values at a time: the kernels here are bound by instructions issued, and a packed one does two operations.
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 fast_exp2(float2 x) { return make_float2(fast_exp2(x.x), fast_exp2(x.y)); }
__device__ __forceinline__ float2 fast_reciprocal(float2 x) { return make_float2(fast_reciprocal(x.x), fast_reciprocal(x.y)); }
__device__ __forceinline__ float2 negative_part(float2 x) { return make_float2(min_nan(x.x, 0.0f), min_nan(x.y, 0.0f)); }
__device__ __forceinline__ float2 positive_part(float2 x) { return make_float2(fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f)); }

// log(1 + e) for e in [0, 1] = 2 artanh(s), s = e / (2 + e) <= 1/3, by its series: what is cut off is below 2e-8 of it.
__device__ __forceinline__ float2 log1p_unit(float2 e)
{
    const float2 s = __fmul2_rn(e, fast_reciprocal(__fadd2_rn(e, both(2.0f)))), t = __fmul2_rn(s, s);
    float2 p = both(2.0f / 13.0f);
    p = __ffma2_rn(p, t, both(2.0f / 11.0f));
    p = __ffma2_rn(p, t, both(2.0f / 9.0f));
    p = __ffma2_rn(p, t, both(2.0f / 7.0f));
    p = __ffma2_rn(p, t, both(2.0f / 5.0f));
    p = __ffma2_rn(p, t, both(2.0f / 3.0f));
    p = __ffma2_rn(p, t, both(2.0f));
    return __fmul2_rn(p, s);
}
template <int ACT> __device__ __forceinline__ float2 act_value(float2 u)
{
    if (ACT == kActCelu) {
        const float2 e = fast_exp2(negative_part(__fmul2_rn(u, both(10.0f * kLog2E))));
        return __fadd2_rn(positive_part(u), __ffma2_rn(e, both(0.1f), both(-0.1f)));
    }
    if (ACT == kActGaussian) return fast_exp2(__fmul2_rn(__fmul2_rn(u, u), both(-kLog2E)));
    if (ACT == kActNormal) return fast_exp2(__fmul2_rn(__fmul2_rn(u, u), both(-0.5f * kLog2E)));
    const float2 l = log1p_unit(fast_exp2(__fmul2_rn(make_float2(fabsf(u.x), fabsf(u.y)), both(-kLog2E))));
    return __fadd2_rn(__fadd2_rn(positive_part(u), both(-0.69314718056f)), l);
}
template <int ACT> __device__ __forceinline__ float2 act_derivative(float2 u)
{
    if (ACT == kActCelu) return fast_exp2(negative_part(__fmul2_rn(u, both(10.0f * kLog2E))));
    if (ACT == kActGaussian)
        return __fmul2_rn(__fmul2_rn(u, both(-2.0f)), fast_exp2(__fmul2_rn(__fmul2_rn(u, u), both(-kLog2E))));
    if (ACT == kActNormal)
        return __fmul2_rn(make_float2(-u.x, -u.y), fast_exp2(__fmul2_rn(__fmul2_rn(u, u), both(-0.5f * kLog2E))));
    return fast_reciprocal(__fadd2_rn(fast_exp2(__fmul2_rn(u, both(-kLog2E))), both(1.0f)));
}
// All of a thread's values, the choice of the function outside the loop.
template <int ACT, int NV> __device__ __forceinline__ void act_values_of(float2 (*u)[2])
{
#pragma unroll
    for (int k = 0; k < NV; k++) {
        u[k][0] = act_value<ACT>(u[k][0]);
        u[k][1] = act_value<ACT>(u[k][1]);
    }
}
template <int NV> __device__ __forceinline__ void act_values(int act, float2 (*u)[2])
{
    if (act == kActCelu) act_values_of<kActCelu, NV>(u);
    else if (act == kActGaussian) act_values_of<kActGaussian, NV>(u);
    else if (act == kActNormal) act_values_of<kActNormal, NV>(u);
    else act_values_of<kActSoftplus, NV>(u);
}
template <int ACT> __device__ __forceinline__ void act_derivatives_of(float2* u)
{
    u[0] = act_derivative<ACT>(u[0]);
    u[1] = act_derivative<ACT>(u[1]);
}
__device__ __forceinline__ void act_derivatives(int act, float2* u)
{
    if (act == kActCelu) act_derivatives_of<kActCelu>(u);
    else if (act == kActGaussian) act_derivatives_of<kActGaussian>(u);
    else if (act == kActNormal) act_derivatives_of<kActNormal>(u);
    else act_derivatives_of<kActSoftplus>(u);
}
__device__ __forceinline__ float2 first2(const float* v) { return make_float2(v[0], v[1]); }
__device__ __forceinline__ float2 last2(const float* v) { return make_float2(v[2], v[3]); }

// Smallest and largest value of a block: over the lanes that share it, NaN if one of them has one.  All lanes of the warp
// take part (volatile: not to be moved to where the result is used, which is not in all of them).
template <int TEAM> __device__ __forceinline__ void block_extremes(float* low, float* high)
{
    if (TEAM >= kWarp) {
        float l, h;
        asm volatile("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;" : "=f"(l) : "f"(*low));
        asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(h) : "f"(*high));
        *low = l;
        *high = h;
    } else {
#pragma unroll
        for (int o = TEAM / 2; o > 0; o >>= 1) {
            *low = min_nan(*low, __shfl_xor_sync(kFull, *low, o));
            *high = max_nan(*high, __shfl_xor_sync(kFull, *high, o));
        }
    }
}

struct CheckpointParams {
    const float* z;
    long long z_stride;
    const float* gain[kTypes];
    const float* bias[kTypes];
    float* a;
    unsigned char* codes;      // [n][checkpoint_row_bytes]
    float2* blocks;            // [n][checkpoint_blocks]: base, step
    float *mean, *rstd;
    RowGroups groups;
    int width, act;
    float inv_w, eps;
};

template <int TEAM, int NV, bool NORM, bool VEC>
__global__ void __launch_bounds__(kNormThreads) checkpoint_activation_kernel(const __grid_constant__ CheckpointParams p)
{
    __shared__ float scratch_sh[4 * kNormThreads / kWarp];
    TeamScratch<float> scratch = {scratch_sh, 0};
    constexpr int teams = kNormThreads / TEAM;
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM, w = p.width;
    const int row_bytes = checkpoint_row_bytes(w), row_blocks = checkpoint_blocks(w);
    const long long n = p.groups.start[kTypes];
    pdl_wait();
    pdl_trigger();
    for (long long first = (long long)blockIdx.x * teams; first < n; first += (long long)gridDim.x * teams) {
        const bool live = first + team < n;
        const long long row = live ? first + team : first;
        float z[NV][4];
#pragma unroll
        for (int k = 0; k < NV; k++)
            load_columns<VEC>(p.z + row * p.z_stride, 4 * (lane + k * TEAM), w, z[k]);
        float mean = 0.0f, rstd = 1.0f;
        if (NORM) row_statistics<TEAM, NV, VEC>(z, lane, w, p.inv_w, p.eps, scratch, &mean, &rstd);
        // The extremes of the thread's blocks; what follows from them (a correctly rounded reciprocal among it) is formed for all
        // of them at once, block k by the lanes k, k + 4, ..: 93 us at 110,000 x 512, 101 with all lanes forming all of them.
        float low[NV], high[NV];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            low[k] = __int_as_float(0x7f800000);
            high[k] = -low[k];
            if (VEC && col < w) {
                low[k] = min_nan(min_nan(z[k][0], z[k][1]), min_nan(z[k][2], z[k][3]));
                high[k] = max_nan(max_nan(z[k][0], z[k][1]), max_nan(z[k][2], z[k][3]));
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (col + i < w) {
                        low[k] = min_nan(low[k], z[k][i]);
                        high[k] = max_nan(high[k], z[k][i]);
                    }
            }
            block_extremes<TEAM>(&low[k], &high[k]);
        }
        const int mine = NV == 1 ? 0 : min(lane_id() & 3, NV - 1);
        float my_low = low[0], my_high = high[0];
#pragma unroll
        for (int k = 1; k < NV; k++) {
            my_low = mine == k ? low[k] : my_low;
            my_high = mine == k ? high[k] : my_high;
        }
        const float spread = __fsub_rn(my_high, my_low), step = __fmul_rn(spread, 1.0f / 255.0f);
        const bool finite = spread < __int_as_float(0x7f800000), some = finite && step >= 1e-30f;
        const float my_inv = some ? __frcp_rn(step) : 0.0f;
        const int my_col = 4 * (lane % TEAM - lane % (TEAM < kWarp ? TEAM : kWarp) + mine * TEAM);      // the block's first column
        if (live && my_col < w && (NV == 1 ? lane % (TEAM < kWarp ? TEAM : kWarp) == 0 : lane_id() < NV))
            p.blocks[row * row_blocks + my_col / kCheckpointBlock] = make_float2(finite ? my_low : __int_as_float(0x7fffffff), some ? step : 0.0f);
        const int e = element_of_row(p.groups, row);
        float2 u[NV][2];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            const float inv = NV == 1 ? my_inv : __shfl_sync(kFull, my_inv, k);
            u[k][0] = u[k][1] = both(0.0f);
            if (!live || col >= w) continue;
            // rint of 0 .. 255 in one addition: 2^23 + q has its last place at 1, and q in the low bits.  Nothing is above
            // 255: (max - base) (1 / step) is 255 but for four roundings.
            // (The product by itself: the packed one may be fused with the sum behind it, which rounds once instead of twice.)
            const float2 d[2] = {__fadd2_rn(first2(z[k]), both(-low[k])), __fadd2_rn(last2(z[k]), both(-low[k]))};
            unsigned q[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                q[i] = __float_as_uint(__fadd_rn(__fmul_rn(i % 2 ? d[i / 2].y : d[i / 2].x, inv), 8388608.0f));
            const unsigned code = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
            *reinterpret_cast<unsigned*>(p.codes + row * row_bytes + col) = code;
            u[k][0] = first2(z[k]);
            u[k][1] = last2(z[k]);
            if (NORM) {
                float g[4], h[4];
                load_columns<VEC>(p.gain[e], col, w, g);
                load_columns<VEC>(p.bias[e], col, w, h);
                u[k][0] = __ffma2_rn(__fmul2_rn(__fadd2_rn(u[k][0], both(-mean)), both(rstd)), first2(g), first2(h));
                u[k][1] = __ffma2_rn(__fmul2_rn(__fadd2_rn(u[k][1], both(-mean)), both(rstd)), last2(g), last2(h));
            }
        }
        act_values<NV>(p.act, u);
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            const float a[4] = {u[k][0].x, u[k][0].y, u[k][1].x, u[k][1].y};
            if (col < w) store_columns<VEC>(p.a + row * w, col, w, a);
        }
        if (NORM && lane == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
    }
}

struct CheckpointGradParams {
    const unsigned char* codes;
    const float2* blocks;
    const float *mean, *rstd;
    const float* grad_a;
    long long grad_stride;
    const float* gain[kTypes];
    const float* bias[kTypes];
    float* grad_z;
    ColumnSums<float, 3> sums;      // of dz, and with a gain of its gradient and the bias'
    RowRanges ranges;
    int width, act;
    float inv_w;
};

// Two CTAs an SM where a thread has twelve or sixteen columns, as many as the ranges are made for: with three there are 80
// registers a thread, and twelve columns do not fit them (110,000 x 384 with a norm: 126 us, 82 with two).
template <int TEAM, int NV, bool NORM, bool VEC>
__global__ void __launch_bounds__(kNormThreads, NV >= 3 ? 2 : 3) checkpoint_activation_grad_kernel(const __grid_constant__ CheckpointGradParams p)
{
    constexpr int Q = NORM ? 3 : 1;
    __shared__ float scratch_sh[4 * kNormThreads / kWarp];
    TeamScratch<float> scratch = {scratch_sh, 0};
    __shared__ alignas(16) float tile[TEAM == kNormThreads ? 4 : kNormThreads * NV * 4];
    constexpr int teams = kNormThreads / TEAM;
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM, w = p.width;
    const int row_bytes = checkpoint_row_bytes(w), row_blocks = checkpoint_blocks(w);
    pdl_wait();
    pdl_trigger();
    zero_sums_without_rows(p.sums, p.ranges, w);
    if ((int)blockIdx.x >= p.ranges.range_start[kTypes]) return;      // no rows at all: one CTA, for the zeros
    const RowRange range = range_of_cta(p.ranges, blockIdx.x);
    // gain and bias in shared memory: in registers they would cost half of the resident warps at 512 columns
    __shared__ alignas(16) float gain_sh[NORM ? TEAM * NV * 4 : 4], bias_sh[NORM ? TEAM * NV * 4 : 4];
    if (NORM) {
        for (int c = threadIdx.x; c < TEAM * NV * 4; c += kNormThreads) {
            gain_sh[c] = c < w ? p.gain[range.element][c] : 0.0f;
            bias_sh[c] = c < w ? p.bias[range.element][c] : 0.0f;
        }
        __syncthreads();
    }
    float2 sums[Q][NV][2];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int q = 0; q < Q; q++) sums[q][k][0] = sums[q][k][1] = both(0.0f);
    // Everything a row needs is asked for before any of it is used, and with few columns to a thread a turn ahead.
    constexpr bool kAhead = NV == 1;
    float up_next[NV][4], mean_next = 0.0f, rstd_next = 0.0f;
    unsigned code_next[NV];
    float2 block_next[NV];
    auto load = [&](long long first) {
        const bool live = first + team < range.end;
        const long long row = live ? first + team : range.first;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            const bool in = live && col < w;
            code_next[k] = in ? *reinterpret_cast<const unsigned*>(p.codes + row * row_bytes + col) : 0u;
            block_next[k] = in ? p.blocks[row * row_blocks + col / kCheckpointBlock] : make_float2(0.0f, 0.0f);
            load_columns<VEC>(p.grad_a + row * p.grad_stride, col, live ? w : 0, up_next[k]);
        }
        if (NORM) {
            mean_next = p.mean[row];
            rstd_next = p.rstd[row];
        }
    };
    if (kAhead) load(range.first);
    for (long long first = range.first; first < range.end; first += teams) {
        const bool live = first + team < range.end;
        const long long row = first + team;
        if (!kAhead) load(first);
        float up[NV][4];
        unsigned code[NV];
        float2 block[NV];
        const float mean = mean_next, rstd = rstd_next;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            code[k] = code_next[k];
            block[k] = block_next[k];
#pragma unroll
            for (int i = 0; i < 4; i++) up[k][i] = up_next[k][i];
        }
        if (kAhead && first + teams < range.end) load(first + teams);
        // pairs of columns: what the codes stand for, xhat of that
        float2 xhat[NV][2], g2[NV][2];
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float2 c = make_float2((float)((code[k] >> (16 * i)) & 255u), (float)((code[k] >> (16 * i + 8)) & 255u));
                xhat[k][i] = __ffma2_rn(c, both(block[k].y), both(block[k].x));
                g2[k][i] = make_float2(up[k][2 * i], up[k][2 * i + 1]);
            }
        if constexpr (NORM) {
            float2 sum_du = both(0.0f), sum_dx = both(0.0f);
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int col = 4 * (lane + k * TEAM);
                float g[4], h[4];
                load4(gain_sh + col, g);
                load4(bias_sh + col, h);
                // Columns behind the row, and rows behind the range, have a gradient of zero and an xhat of zero: nothing of them
                // is in a sum.  (With the row's rstd their xhat may be infinite, and zero times that is not zero.)
                const float scale = live && col < w ? rstd : 0.0f;
                float2 d[2];
#pragma unroll
                for (int i = 0; i < 2; i++) xhat[k][i] = __fmul2_rn(__fadd2_rn(xhat[k][i], both(-mean)), both(scale));
                if (!VEC && col < w && col + 4 > w) {      // one thread's columns of a row (a choice for every value: 16 % at 497 columns)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        if (col + 2 * i >= w) xhat[k][i].x = 0.0f;
                        if (col + 2 * i + 1 >= w) xhat[k][i].y = 0.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; i++)
                    d[i] = __ffma2_rn(xhat[k][i], make_float2(g[2 * i], g[2 * i + 1]), make_float2(h[2 * i], h[2 * i + 1]));
                act_derivatives(p.act, d);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float2 du = __fmul2_rn(g2[k][i], d[i]);
                    sums[Q - 2][k][i] = __ffma2_rn(du, xhat[k][i], sums[Q - 2][k][i]);
                    sums[Q - 1][k][i] = __fadd2_rn(sums[Q - 1][k][i], du);
                    g2[k][i] = __fmul2_rn(du, make_float2(g[2 * i], g[2 * i + 1]));
                    sum_du = __fadd2_rn(sum_du, g2[k][i]);
                    sum_dx = __ffma2_rn(g2[k][i], xhat[k][i], sum_dx);
                }
            }
            float sum[2] = {sum_du.x + sum_du.y, sum_dx.x + sum_dx.y};
            team_sum<TEAM, 2>(sum, scratch);
            const float2 c1 = both(-sum[0] * p.inv_w), c2 = both(-sum[1] * p.inv_w);
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    g2[k][i] = __fmul2_rn(__ffma2_rn(xhat[k][i], c2, __fadd2_rn(g2[k][i], c1)), both(rstd));
        } else {
#pragma unroll
            for (int k = 0; k < NV; k++) {
                act_derivatives(p.act, xhat[k]);
#pragma unroll
                for (int i = 0; i < 2; i++) g2[k][i] = __fmul2_rn(g2[k][i], xhat[k][i]);
            }
        }
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            if (col >= w) break;
#pragma unroll
            for (int i = 0; i < 2; i++) sums[0][k][i] = __fadd2_rn(sums[0][k][i], g2[k][i]);
            const float dz[4] = {g2[k][0].x, g2[k][0].y, g2[k][1].x, g2[k][1].y};
            store_columns<VEC>(p.grad_z + row * w, col, w, dz);
        }
    }
#pragma unroll
    for (int q = 0; q < Q; q++) {
        float v[NV][4];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            v[k][0] = sums[q][k][0].x; v[k][1] = sums[q][k][0].y; v[k][2] = sums[q][k][1].x; v[k][3] = sums[q][k][1].y;
        }
        store_column_sums<TEAM, NV>(v, tile, column_sums_place(p.sums, p.ranges, range.element, blockIdx.x, q, w), w);
    }
}

}  // namespace ani
