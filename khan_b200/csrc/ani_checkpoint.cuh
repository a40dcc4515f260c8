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
// log(1 + e) for e in [0, 1] = 2 artanh(s), s = e / (2 + e) <= 1/3, by its series: what is cut off is below 2e-8 of it.
__device__ __forceinline__ float log1p_unit(float e)
{
    const float s = e * fast_reciprocal(2.0f + e), t = s * s;
    float p = 1.0f / 13.0f;
    p = fmaf(p, t, 1.0f / 11.0f);
    p = fmaf(p, t, 1.0f / 9.0f);
    p = fmaf(p, t, 1.0f / 7.0f);
    p = fmaf(p, t, 0.2f);
    p = fmaf(p, t, 1.0f / 3.0f);
    return 2.0f * fmaf(p * t, s, s);
}
template <int ACT> __device__ __forceinline__ float act_value(float u)
{
    if (ACT == kActCelu) return fmaxf(u, 0.0f) + fmaf(0.1f, fast_exp2(min_nan(10.0f * kLog2E * u, 0.0f)), -0.1f);
    if (ACT == kActGaussian) return fast_exp2(-kLog2E * u * u);
    if (ACT == kActNormal) return fast_exp2(-0.5f * kLog2E * u * u);
    return fmaxf(u, 0.0f) + log1p_unit(fast_exp2(-kLog2E * fabsf(u))) - 0.69314718056f;
}
template <int ACT> __device__ __forceinline__ float act_derivative(float u)
{
    if (ACT == kActCelu) return fast_exp2(min_nan(10.0f * kLog2E * u, 0.0f));
    if (ACT == kActGaussian) return -2.0f * u * fast_exp2(-kLog2E * u * u);
    if (ACT == kActNormal) return -u * fast_exp2(-0.5f * kLog2E * u * u);
    return fast_reciprocal(1.0f + fast_exp2(-kLog2E * u));
}
// All of a thread's values, the choice of the function outside the loop.
template <int ACT, int NV> __device__ __forceinline__ void act_values_of(float (*u)[4])
{
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) u[k][i] = act_value<ACT>(u[k][i]);
}
template <int NV> __device__ __forceinline__ void act_values(int act, float (*u)[4])
{
    if (act == kActCelu) act_values_of<kActCelu, NV>(u);
    else if (act == kActGaussian) act_values_of<kActGaussian, NV>(u);
    else if (act == kActNormal) act_values_of<kActNormal, NV>(u);
    else act_values_of<kActSoftplus, NV>(u);
}
template <int ACT, int NV> __device__ __forceinline__ void act_derivatives_of(float (*u)[4])
{
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) u[k][i] = act_derivative<ACT>(u[k][i]);
}
template <int NV> __device__ __forceinline__ void act_derivatives(int act, float (*u)[4])
{
    if (act == kActCelu) act_derivatives_of<kActCelu, NV>(u);
    else if (act == kActGaussian) act_derivatives_of<kActGaussian, NV>(u);
    else if (act == kActNormal) act_derivatives_of<kActNormal, NV>(u);
    else act_derivatives_of<kActSoftplus, NV>(u);
}

// Smallest and largest value of a block: over the lanes that share it, NaN if one of them has one.
template <int TEAM> __device__ __forceinline__ void block_extremes(float* low, float* high)
{
    if (TEAM >= kWarp) {
        float l, h;
        asm("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;" : "=f"(l) : "f"(*low));
        asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(h) : "f"(*high));
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
        const int e = element_of_row(p.groups, row);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            float low = __int_as_float(0x7f800000), high = -low;
            if (VEC && col < w) {
                low = min_nan(min_nan(z[k][0], z[k][1]), min_nan(z[k][2], z[k][3]));
                high = max_nan(max_nan(z[k][0], z[k][1]), max_nan(z[k][2], z[k][3]));
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (col + i < w) {
                        low = min_nan(low, z[k][i]);
                        high = max_nan(high, z[k][i]);
                    }
            }
            block_extremes<TEAM>(&low, &high);
            if (!live || col >= w) continue;
            const float spread = __fsub_rn(high, low);
            float step = __fmul_rn(spread, 1.0f / 255.0f);
            const bool finite = spread < __int_as_float(0x7f800000), some = finite && step >= 1e-30f;
            const float inv = some ? __frcp_rn(step) : 0.0f;
            step = some ? step : 0.0f;
            // rint of 0 .. 255 in one addition: 2^23 + q has its last place at 1, and q in the low bits.  Nothing is above
            // 255: (max - base) (1 / step) is 255 but for four roundings.
            unsigned q[4];
#pragma unroll
            for (int i = 0; i < 4; i++) q[i] = __float_as_uint(__fadd_rn(__fmul_rn(__fsub_rn(z[k][i], low), inv), 8388608.0f));
            const unsigned code = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
            *reinterpret_cast<unsigned*>(p.codes + row * row_bytes + col) = code;
            if (col % kCheckpointBlock == 0)
                p.blocks[row * row_blocks + col / kCheckpointBlock] = make_float2(finite ? low : __int_as_float(0x7fffffff), step);
            if (NORM) {
                float g[4], h[4];
                load_columns<VEC>(p.gain[e], col, w, g);
                load_columns<VEC>(p.bias[e], col, w, h);
#pragma unroll
                for (int i = 0; i < 4; i++) z[k][i] = (z[k][i] - mean) * rstd * g[i] + h[i];
            }
        }
        act_values<NV>(p.act, z);
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            if (col < w) store_columns<VEC>(p.a + row * w, col, w, z[k]);
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

template <int TEAM, int NV, bool NORM, bool VEC>
__global__ void __launch_bounds__(kNormThreads, NV == 4 ? 2 : 3) checkpoint_activation_grad_kernel(const __grid_constant__ CheckpointGradParams p)
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
    float sums[Q][NV][4];
#pragma unroll
    for (int k = 0; k < NV; k++) {
#pragma unroll
        for (int q = 0; q < Q; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) sums[q][k][i] = 0.0f;
    }
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
        float kept[NV][4], up[NV][4];
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
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) kept[k][i] = fmaf((float)((code[k] >> (8 * i)) & 255u), block[k].y, block[k].x);
        if constexpr (NORM) {
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int col = 4 * (lane + k * TEAM);
                float g[4], h[4], d[1][4];
                load4(gain_sh + col, g);
                load4(bias_sh + col, h);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    kept[k][i] = live && column_in<VEC>(col, i, w) ? (kept[k][i] - mean) * rstd : 0.0f;
                    d[0][i] = kept[k][i] * g[i] + h[i];
                }
                act_derivatives<1>(p.act, d);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float du = up[k][i] * d[0][i];      // up is zero where there is no value
                    sums[Q - 2][k][i] += du * kept[k][i];
                    sums[Q - 1][k][i] += du;
                    up[k][i] = du * g[i];
                    sum[0] += up[k][i];
                    sum[1] += up[k][i] * kept[k][i];
                }
            }
            team_sum<TEAM, 2>(sum, scratch);
            sum[0] *= p.inv_w;
            sum[1] *= p.inv_w;
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) up[k][i] = rstd * (up[k][i] - sum[0] - kept[k][i] * sum[1]);
        } else {
            act_derivatives<NV>(p.act, kept);
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) up[k][i] *= kept[k][i];
        }
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int col = 4 * (lane + k * TEAM);
            if (col >= w) break;
#pragma unroll
            for (int i = 0; i < 4; i++) sums[0][k][i] += up[k][i];
            store_columns<VEC>(p.grad_z + row * w, col, w, up[k]);
        }
    }
#pragma unroll
    for (int q = 0; q < Q; q++)
        store_column_sums<TEAM, NV>(sums[q], tile, column_sums_place(p.sums, p.ranges, range.element, blockIdx.x, q, w), w);
}

}  // namespace ani
