// Weight gradient of the dense layer behind a checkpointed activation (ani_checkpoint.cuh):
//   dW = sum over the rows of an element  act(u~)^T dz   [width, out],  u~ from the codes as in the backward pass.
// The activations are never in memory: a row's bytes become activations on their way into the product.
//
// K, the long axis, is the atom; a CTA takes a range of rows of one element and one tile of the output, and where an
// element has several ranges they write partial products that a second launch adds in order.
#pragma once

#include "ani_checkpoint.cuh"

namespace ani {

struct CheckpointWgradParams {
    const unsigned char* codes;
    const float2* blocks;
    const float *mean, *rstd;
    const float* gain[kTypes];
    const float* bias[kTypes];
    const float* grad_z;
    long long grad_stride;
    float* grad_w[kTypes];      // [width][out]
    float* partial;             // [ranges][width][out]
    RowRanges ranges;
    int width, out, act, norm;
};

constexpr int kCwTile = 64, kCwK = 16;

__global__ void __launch_bounds__(256) checkpoint_wgrad_kernel(const __grid_constant__ CheckpointWgradParams p)
{
    __shared__ alignas(16) float a[kCwK][kCwTile], b[kCwK][kCwTile];
    pdl_wait();
    pdl_trigger();
    const RowRange range = range_of_cta(p.ranges, blockIdx.x);
    const int row_bytes = checkpoint_row_bytes(p.width), row_blocks = checkpoint_blocks(p.width);
    const int m0 = blockIdx.y * kCwTile, n0 = blockIdx.z * kCwTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int col = threadIdx.x % kCwTile, k_in = threadIdx.x / kCwTile;
    const int m = m0 + col, n = n0 + col;
    const float gain = p.norm && m < p.width ? p.gain[range.element][m] : 1.0f;
    const float bias = p.norm && m < p.width ? p.bias[range.element][m] : 0.0f;
    float acc[4][4] = {};
    for (long long r0 = range.first; r0 < range.end; r0 += kCwK) {
#pragma unroll
        for (int k = k_in; k < kCwK; k += 4) {
            const long long row = r0 + k;
            float va = 0.0f, vb = 0.0f;
            if (row < range.end) {
                if (m < p.width) {
                    const float2 block = p.blocks[row * row_blocks + m / kCheckpointBlock];
                    float u = fmaf((float)p.codes[row * row_bytes + m], block.y, block.x);
                    if (p.norm) u = (u - p.mean[row]) * p.rstd[row] * gain + bias;
                    va = act_value(p.act, u);
                }
                if (n < p.out) vb = p.grad_z[row * p.grad_stride + n];
            }
            a[k][col] = va;
            b[k][col] = vb;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kCwK; k++) {
            const float4 x = *reinterpret_cast<const float4*>(&a[k][4 * ty]), y = *reinterpret_cast<const float4*>(&b[k][4 * tx]);
            const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(xs[i], ys[j], acc[i][j]);
        }
        __syncthreads();
    }
    const bool single = p.ranges.range_start[range.element + 1] - p.ranges.range_start[range.element] == 1;
    float* out = single ? p.grad_w[range.element] : p.partial + (size_t)blockIdx.x * p.width * p.out;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int row = m0 + 4 * ty + i, c = n0 + 4 * tx + j;
            if (row < p.width && c < p.out) out[(size_t)row * p.out + c] = acc[i][j];
        }
}

// The partial products of an element's ranges, added in order; zeros for an element without rows.
__global__ void __launch_bounds__(256) checkpoint_wgrad_sum_kernel(const __grid_constant__ CheckpointWgradParams p)
{
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.y, first = p.ranges.range_start[t], n = p.ranges.range_start[t + 1] - first;
    if (n == 1 || !p.grad_w[t]) return;      // written already, or an element without rows and without a place
    const size_t size = (size_t)p.width * p.out;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < size; i += (size_t)gridDim.x * blockDim.x) {
        float s = 0.0f;
        for (int k = 0; k < n; k++) s += p.partial[(size_t)(first + k) * size + i];
        p.grad_w[t][i] = s;
    }
}

}  // namespace ani
