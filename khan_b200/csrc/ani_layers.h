// Entry points of the normalised layers and of activation checkpoints: argument checks, launch plans.  Included by
// ani_b200.cu behind its helpers.
#pragma once

#include "ani_checkpoint.cuh"
#include "ani_checkpoint_wgrad.cuh"
#include "ani_norm.cuh"

#include <math.h>

#include <type_traits>

namespace {

bool aligned16(std::initializer_list<const void*> ptrs)
{
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    return true;
}

RowGroups row_groups(const int* acs)
{
    RowGroups g;
    g.start[0] = 0;
    for (int t = 0; t < kTypes; t++) g.start[t + 1] = g.start[t] + acs[t];
    return g;
}

// Ranges of a multiple of `step` rows, about `target` of them, none shorter than `least` but for an element's last.
RowRanges row_ranges(const int* acs, long long target, long long step, long long least)
{
    RowRanges r;
    r.groups = row_groups(acs);
    const long long n = r.groups.start[kTypes];
    const long long rows = std::max(least, (n + target - 1) / target);
    r.rows = (rows + step - 1) / step * step;
    r.range_start[0] = 0;
    for (int t = 0; t < kTypes; t++) r.range_start[t + 1] = r.range_start[t] + (int)((acs[t] + r.rows - 1) / r.rows);
    return r;
}
bool one_range_each(const RowRanges& r)
{
    for (int t = 0; t < kTypes; t++)
        if (r.range_start[t + 1] - r.range_start[t] > 1) return false;
    return true;
}

// The team and the columns per thread for a row of `width` values.  Sixteen columns to a thread once a row is wider than a warp
// has at four: the fewer threads a row has, the fewer instructions and meetings it costs (backward pass of the activations,
// 110,000 rows of 512: 101 us with a warp of 16 columns to a thread, 117 with two of 8, 132 with four of 4; 50,000 rows of 1024:
// 102 us with 64 threads, 110 with 128, 116 with 256).  In double precision 16 columns are too many registers (HEAVY; gradient
// at 512 columns: 171 us with 64 threads, 187 with 32).
template <bool HEAVY, typename F> cudaError_t with_team(int width, bool vec, F f)
{
#define ANI_TEAM(TEAM, NV)                                                                                            \
    (vec ? f(std::integral_constant<int, TEAM>(), std::integral_constant<int, NV>(), std::true_type())               \
         : f(std::integral_constant<int, TEAM>(), std::integral_constant<int, NV>(), std::false_type()))
    const int quads = (width + 3) / 4;
    if (quads <= 8) return ANI_TEAM(8, 1);
    if (quads <= 16) return ANI_TEAM(16, 1);
    if (quads <= 32) return ANI_TEAM(32, 1);
    if (quads <= 64) return ANI_TEAM(32, 2);
    if constexpr (HEAVY) {
        if (quads <= 128) return ANI_TEAM(64, 2);
        if (quads <= 256) return ANI_TEAM(128, 2);
        if (quads <= 512) return ANI_TEAM(256, 2);
    } else {
        if (quads <= 96) return ANI_TEAM(32, 3);      // the 384 features
        if (quads <= 128) return ANI_TEAM(32, 4);
        if (quads <= 256) return ANI_TEAM(64, 4);
        if (quads <= 512) return ANI_TEAM(128, 4);
    }
    return ANI_TEAM(256, 4);
#undef ANI_TEAM
}
template <bool HEAVY> int rows_at_once(int width)
{
    int rows = 1;
    with_team<HEAVY>(width, true, [&](auto team, auto, auto) {
        rows = kNormThreads / team();
        return cudaSuccess;
    });
    return rows;
}

// Ranges of the launches with sums over rows: as many CTAs as are resident at once (by their registers, 48 to 254 a thread;
// one more or less costs 10 to 30 %).
RowRanges sum_ranges(const int* acs, int width, int sums, size_t size)
{
    const int quads = (width + 3) / 4;
    const bool heavy = size > 4;
    const int rows = heavy ? rows_at_once<true>(width) : rows_at_once<false>(width);
    const int per_sm = quads <= 32 ? (heavy || sums > 2 ? 3 : 4)
                       : quads <= 64 ? (heavy ? 2 : sums > 2 ? 3 : 4)
                                     : (heavy && quads > 512 ? 1 : 2);
    // up to sixteen rows to a team an element is one range, which saves the second launch (2.1 us of the host, 3 of the device)
    return row_ranges(acs, per_sm * kSms, rows, *std::max_element(acs, acs + kTypes) <= 16 * rows ? 16 * rows : 4 * rows);
}
size_t sums_workspace(const RowRanges& r, int sums, int width, size_t size)
{
    return one_range_each(r) ? 0 : (size_t)r.range_start[kTypes] * sums * width * size;
}

int check_layer(const int* acs, int width, long long* n)
{
    if (int rc = check_acs(acs, n)) return rc;
    return width < 1 || width > kNormMaxWidth ? ANI_ERR_BAD_SIZE : ANI_OK;
}
// Per-element pointers: present where the element has rows.
template <typename T, typename P>
int take_pointers(T* const* from_host, const int* acs, P* to, bool* vec = nullptr)
{
    for (int t = 0; t < kTypes; t++) {
        to[t] = from_host ? from_host[t] : nullptr;
        if (acs[t] == 0) continue;
        if (!to[t]) return ANI_ERR_NULL_POINTER;
        if (vec) *vec = *vec && aligned16({to[t]});
    }
    return ANI_OK;
}
int rows_grid(long long n, int at_once)
{
    return (int)std::min<long long>((n + at_once - 1) / at_once, 0x7fffffff);
}

template <typename T, int Q>
int column_sums_launch(const ColumnSums<T, Q>& s, const RowRanges& r, int width, cudaStream_t st)
{
    if (one_range_each(r)) return ANI_OK;
    const dim3 grid((width + kSumColumns - 1) / kSumColumns, kTypes * Q);
    ANI_CUDA(launch_chain(column_sums_kernel<T, Q>, grid, dim3(kSumColumns, kSumParts), 0, st, 1, s, r, width));
    return ANI_OK;
}

template <typename T>
int layer_norm(const T* x, long long x_stride, const T* const* gain, const T* const* bias, int width, double eps,
               const int* acs, T* y, T* mean, T* rstd, void* stream)
{
    long long n = 0;
    if (int rc = check_layer(acs, width, &n)) return rc;
    if (x_stride < width || !(eps >= 0.0) || !(eps < HUGE_VAL)) return ANI_ERR_BAD_SIZE;
    if (n == 0) return ANI_OK;
    if (!x || !gain || !bias || !y || !mean || !rstd) return ANI_ERR_NULL_POINTER;
    LayerNormParams<T> p;
    bool vec = aligned16({x, y}) && width % 4 == 0 && x_stride % 4 == 0;
    if (int rc = take_pointers(gain, acs, p.gain, &vec)) return rc;
    if (int rc = take_pointers(bias, acs, p.bias, &vec)) return rc;
    p.x = x; p.x_stride = x_stride; p.y = y; p.mean = mean; p.rstd = rstd;
    p.groups = row_groups(acs);
    p.width = width; p.inv_w = T(1) / T(width); p.eps = T(eps);
    constexpr bool heavy = sizeof(T) > 4;
    const int grid = rows_grid(n, rows_at_once<heavy>(width));
    ANI_CUDA(with_team<heavy>(width, vec, [&](auto team, auto nv, auto aligned) {
        return launch_chain(layer_norm_kernel<T, team(), nv(), aligned()>, grid, kNormThreads, 0, (cudaStream_t)stream, 1, p);
    }));
    return ANI_OK;
}

template <typename T>
int layer_norm_grad(const T* grad_y, long long grad_stride, const T* x, long long x_stride, const T* const* gain, const T* mean,
                    const T* rstd, int width, const int* acs, T* grad_x, T* const* grad_gain, T* const* grad_bias,
                    void* workspace, void* stream)
{
    long long n = 0;
    if (int rc = check_layer(acs, width, &n)) return rc;
    if (x_stride < width || grad_stride < width) return ANI_ERR_BAD_SIZE;
    if (n > 0 && (!grad_y || !x || !gain || !mean || !rstd || !grad_x)) return ANI_ERR_NULL_POINTER;
    LayerNormGradParams<T> p;
    bool vec = aligned16({grad_y, x, grad_x}) && width % 4 == 0 && x_stride % 4 == 0 && grad_stride % 4 == 0;
    if (int rc = take_pointers(gain, acs, p.gain, &vec)) return rc;
    if (int rc = take_pointers(grad_gain, acs, p.sums.out[0])) return rc;
    if (int rc = take_pointers(grad_bias, acs, p.sums.out[1])) return rc;
    p.ranges = sum_ranges(acs, width, 2, sizeof(T));
    if (sums_workspace(p.ranges, 2, width, sizeof(T)) && !workspace) return ANI_ERR_NULL_POINTER;
    if (!aligned16({workspace})) return ANI_ERR_MISALIGNED;
    p.sums.partial = static_cast<T*>(workspace);
    p.grad_y = grad_y; p.grad_stride = grad_stride; p.x = x; p.x_stride = x_stride; p.mean = mean; p.rstd = rstd;
    p.grad_x = grad_x; p.width = width; p.inv_w = T(1) / T(width);
    const int grid = std::max(1, p.ranges.range_start[kTypes]);
    ANI_CUDA(with_team<(sizeof(T) > 4)>(width, vec, [&](auto team, auto nv, auto aligned) {
        return launch_chain(layer_norm_grad_kernel<T, team(), nv(), aligned()>, grid, kNormThreads, 0, (cudaStream_t)stream, 1, p);
    }));
    return column_sums_launch(p.sums, p.ranges, width, (cudaStream_t)stream);
}

bool known_activation(int act) { return act >= kActCelu && act <= kActSoftplus; }

// Ranges of the weight gradient: a CTA holds an SM, so the ranges of all tiles are to fill whole waves of SMs.  Of one to
// four waves the one that takes least is chosen, counted in rows of a CTA (33 ns each): setting up a CTA and writing its tile
// are 192, the second launch 128, and what it reads and writes of partial products 8e-5 a value (37 ranges of 512 x 512 took
// 25 us more than 9).
RowRanges wgrad_ranges(const int* acs, int width, int out)
{
    const long long tiles = (long long)((width + kCwTile - 1) / kCwTile) * ((out + kCwTile - 1) / kCwTile);
    int elements = 0;
    long long most = 0;
    for (int t = 0; t < kTypes; t++) {
        elements += acs[t] > 0;
        most = std::max<long long>(most, acs[t]);
    }
    long long best_rows = (most + kCwK - 1) / kCwK * kCwK;      // a range per element
    long long best = ((elements * tiles + kSms - 1) / kSms) * (best_rows + 192);
    for (int waves = 1; waves <= 4; waves++) {
        const long long budget = (long long)waves * kSms / tiles;      // ranges
        if (budget < elements) continue;
        long long low = 1, high = std::max<long long>(1, (most + kCwK - 1) / kCwK);      // chunks per range
        while (low < high) {
            const long long mid = (low + high) / 2;
            long long count = 0;
            for (int t = 0; t < kTypes; t++) count += (acs[t] + mid * kCwK - 1) / (mid * kCwK);
            if (count <= budget) high = mid;
            else low = mid + 1;
        }
        long long count = 0;
        for (int t = 0; t < kTypes; t++) count += (acs[t] + low * kCwK - 1) / (low * kCwK);
        const long long joined = count > elements ? 128 + count * width * out / 12500 : 0;
        const long long work = waves * (low * kCwK + 192) + joined;
        if (work < best) {
            best = work;
            best_rows = low * kCwK;
        }
    }
    return row_ranges(acs, 0x7fffffff, kCwK, std::max<long long>(kCwK, best_rows));
}

}  // namespace

extern "C" {

int ani_layer_norm_f32(const float* x, long long x_stride, const float* const* gain_host, const float* const* bias_host,
                       int width, double eps, const int* acs_host, float* y, float* mean, float* rstd, void* stream)
{
    return layer_norm(x, x_stride, gain_host, bias_host, width, eps, acs_host, y, mean, rstd, stream);
}
int ani_layer_norm_f64(const double* x, long long x_stride, const double* const* gain_host,
                       const double* const* bias_host, int width, double eps, const int* acs_host, double* y, double* mean,
                       double* rstd, void* stream)
{
    return layer_norm(x, x_stride, gain_host, bias_host, width, eps, acs_host, y, mean, rstd, stream);
}

int ani_layer_norm_grad_f32(const float* grad_y, long long grad_stride, const float* x, long long x_stride,
                            const float* const* gain_host, const float* mean, const float* rstd, int width,
                            const int* acs_host, float* grad_x, float* const* grad_gain_host, float* const* grad_bias_host,
                            void* workspace, void* stream)
{
    return layer_norm_grad(grad_y, grad_stride, x, x_stride, gain_host, mean, rstd, width, acs_host, grad_x, grad_gain_host,
                           grad_bias_host, workspace, stream);
}
int ani_layer_norm_grad_f64(const double* grad_y, long long grad_stride, const double* x, long long x_stride,
                            const double* const* gain_host, const double* mean, const double* rstd, int width,
                            const int* acs_host, double* grad_x, double* const* grad_gain_host,
                            double* const* grad_bias_host, void* workspace, void* stream)
{
    return layer_norm_grad(grad_y, grad_stride, x, x_stride, gain_host, mean, rstd, width, acs_host, grad_x, grad_gain_host,
                           grad_bias_host, workspace, stream);
}
size_t ani_layer_sums_workspace_bytes(int width, const int* acs_host, int sums, int value_bytes)
{
    long long n = 0;
    if (check_layer(acs_host, width, &n) || sums < 0 || value_bytes < 0) return 0;
    return sums_workspace(sum_ranges(acs_host, width, sums, (size_t)value_bytes), sums, width, (size_t)value_bytes);
}

int ani_checkpoint_row_bytes(int width) { return width < 1 || width > kNormMaxWidth ? ANI_ERR_BAD_SIZE : checkpoint_row_bytes(width); }
int ani_checkpoint_blocks(int width) { return width < 1 || width > kNormMaxWidth ? ANI_ERR_BAD_SIZE : checkpoint_blocks(width); }

int ani_checkpoint_activation_f32(const float* z, long long z_stride, const float* const* gain_host,
                                  const float* const* bias_host, int width, double eps, int activation, const int* acs_host,
                                  float* a, unsigned char* codes, float* blocks, float* mean, float* rstd, void* stream)
{
    long long n = 0;
    if (int rc = check_layer(acs_host, width, &n)) return rc;
    if (z_stride < width || !known_activation(activation)) return ANI_ERR_BAD_SIZE;
    if (gain_host && (!(eps >= 0.0) || !(eps < HUGE_VAL))) return ANI_ERR_BAD_SIZE;
    if (n == 0) return ANI_OK;
    if (!z || !a || !codes || !blocks || !gain_host != !bias_host || (gain_host && (!mean || !rstd))) return ANI_ERR_NULL_POINTER;
    CheckpointParams p = {};
    bool vec = aligned16({z, a}) && width % 4 == 0 && z_stride % 4 == 0;
    if (gain_host) {
        if (int rc = take_pointers(gain_host, acs_host, p.gain, &vec)) return rc;
        if (int rc = take_pointers(bias_host, acs_host, p.bias, &vec)) return rc;
    }
    if (!aligned16({codes}) || (reinterpret_cast<uintptr_t>(blocks) & 7)) return ANI_ERR_MISALIGNED;
    p.z = z; p.z_stride = z_stride; p.a = a; p.codes = codes; p.blocks = reinterpret_cast<float2*>(blocks);
    p.mean = mean; p.rstd = rstd; p.groups = row_groups(acs_host);
    p.width = width; p.act = activation; p.inv_w = 1.0f / (float)width; p.eps = (float)eps;
    const int grid = rows_grid(n, rows_at_once<false>(width));
    ANI_CUDA(with_team<false>(width, vec, [&](auto team, auto nv, auto aligned) {
        return gain_host ? launch_chain(checkpoint_activation_kernel<team(), nv(), true, aligned()>, grid, kNormThreads, 0, (cudaStream_t)stream, 1, p)
                         : launch_chain(checkpoint_activation_kernel<team(), nv(), false, aligned()>, grid, kNormThreads, 0, (cudaStream_t)stream, 1, p);
    }));
    return ANI_OK;
}

int ani_checkpoint_activation_grad_f32(const unsigned char* codes, const float* blocks, const float* mean, const float* rstd,
                                       const float* grad_a, long long grad_stride, const float* const* gain_host,
                                       const float* const* bias_host, int width, int activation, const int* acs_host,
                                       float* grad_z, float* const* grad_sum_host, float* const* grad_gain_host,
                                       float* const* grad_bias_host, void* workspace, void* stream)
{
    long long n = 0;
    if (int rc = check_layer(acs_host, width, &n)) return rc;
    if (grad_stride < width || !known_activation(activation)) return ANI_ERR_BAD_SIZE;
    if (!gain_host != !bias_host) return ANI_ERR_NULL_POINTER;
    if (n > 0 && (!codes || !blocks || !grad_a || !grad_z || (gain_host && (!mean || !rstd)))) return ANI_ERR_NULL_POINTER;
    CheckpointGradParams p = {};
    bool vec = aligned16({grad_a, grad_z}) && width % 4 == 0 && grad_stride % 4 == 0;
    if (int rc = take_pointers(grad_sum_host, acs_host, p.sums.out[0])) return rc;
    if (gain_host) {
        if (int rc = take_pointers(gain_host, acs_host, p.gain, &vec)) return rc;
        if (int rc = take_pointers(bias_host, acs_host, p.bias, &vec)) return rc;
        if (int rc = take_pointers(grad_gain_host, acs_host, p.sums.out[1])) return rc;
        if (int rc = take_pointers(grad_bias_host, acs_host, p.sums.out[2])) return rc;
    }
    if (!aligned16({codes}) || (reinterpret_cast<uintptr_t>(blocks) & 7)) return ANI_ERR_MISALIGNED;
    p.ranges = sum_ranges(acs_host, width, 3, sizeof(float));
    if (sums_workspace(p.ranges, 3, width, sizeof(float)) && !workspace) return ANI_ERR_NULL_POINTER;
    if (!aligned16({workspace})) return ANI_ERR_MISALIGNED;
    p.sums.partial = static_cast<float*>(workspace);
    p.codes = codes; p.blocks = reinterpret_cast<const float2*>(blocks); p.mean = mean; p.rstd = rstd;
    p.grad_a = grad_a; p.grad_stride = grad_stride; p.grad_z = grad_z;
    p.width = width; p.act = activation; p.inv_w = 1.0f / (float)width;
    const int grid = std::max(1, p.ranges.range_start[kTypes]);
    ANI_CUDA(with_team<false>(width, vec, [&](auto team, auto nv, auto aligned) {
        return gain_host ? launch_chain(checkpoint_activation_grad_kernel<team(), nv(), true, aligned()>, grid, kNormThreads, 0, (cudaStream_t)stream, 1, p)
                         : launch_chain(checkpoint_activation_grad_kernel<team(), nv(), false, aligned()>, grid, kNormThreads, 0, (cudaStream_t)stream, 1, p);
    }));
    return column_sums_launch(p.sums, p.ranges, width, (cudaStream_t)stream);
}

int ani_checkpoint_weight_grad_f32(const unsigned char* codes, const float* blocks, const float* mean, const float* rstd,
                                   const float* const* gain_host, const float* const* bias_host, int width, int activation,
                                   const float* grad_z, long long grad_stride, int out_width, const int* acs_host,
                                   float* const* grad_w_host, void* workspace, void* stream)
{
    long long n = 0;
    if (int rc = check_layer(acs_host, width, &n)) return rc;
    if (out_width < 1 || out_width > kNormMaxWidth || grad_stride < out_width || !known_activation(activation))
        return ANI_ERR_BAD_SIZE;
    if (!gain_host != !bias_host || !grad_w_host) return ANI_ERR_NULL_POINTER;
    if (n > 0 && (!codes || !blocks || !grad_z || (gain_host && (!mean || !rstd)))) return ANI_ERR_NULL_POINTER;
    CheckpointWgradParams p = {};
    if (gain_host) {
        if (int rc = take_pointers(gain_host, acs_host, p.gain)) return rc;
        if (int rc = take_pointers(bias_host, acs_host, p.bias)) return rc;
    }
    if (int rc = take_pointers(grad_w_host, acs_host, p.grad_w)) return rc;
    if (!aligned16({codes}) || (reinterpret_cast<uintptr_t>(blocks) & 7)) return ANI_ERR_MISALIGNED;
    p.ranges = wgrad_ranges(acs_host, width, out_width);
    if (!one_range_each(p.ranges) && !workspace) return ANI_ERR_NULL_POINTER;
    if (!aligned16({workspace})) return ANI_ERR_MISALIGNED;
    p.codes = codes; p.blocks = reinterpret_cast<const float2*>(blocks); p.mean = mean; p.rstd = rstd;
    p.grad_z = grad_z; p.grad_stride = grad_stride; p.partial = static_cast<float*>(workspace);
    p.width = width; p.out = out_width; p.norm = gain_host != nullptr;
    p.whole = aligned16({grad_z}) && grad_stride % 4 == 0 && out_width % 4 == 0;
    if (n > 0) {
        const dim3 grid(p.ranges.range_start[kTypes], (width + kCwTile - 1) / kCwTile, (out_width + kCwTile - 1) / kCwTile);
        auto kernel = activation == kActCelu       ? checkpoint_wgrad_kernel<kActCelu>
                      : activation == kActGaussian ? checkpoint_wgrad_kernel<kActGaussian>
                      : activation == kActNormal   ? checkpoint_wgrad_kernel<kActNormal>
                                                   : checkpoint_wgrad_kernel<kActSoftplus>;
        if (int rc = set_smem(kernel, sizeof(CwShared))) return rc;
        ANI_CUDA(launch_chain(kernel, grid, kMlpAllThreads, sizeof(CwShared), (cudaStream_t)stream, 1, p));
    }
    bool all_written = true;      // by that launch
    for (int t = 0; t < kTypes; t++) all_written = all_written && (acs_host[t] == 0 ? !p.grad_w[t] : p.ranges.range_start[t + 1] - p.ranges.range_start[t] == 1);
    if (all_written) return ANI_OK;
    // about eight ranges to a thread
    int most = 1, parts = 1;
    for (int t = 0; t < kTypes; t++) most = std::max(most, p.ranges.range_start[t + 1] - p.ranges.range_start[t]);
    while (parts < kCwSumParts && 8 * parts < most) parts *= 2;
    const dim3 sum_grid(32 / kCwSumColumns * cw_blocks(width) * cw_blocks(out_width), kTypes);
    ANI_CUDA(launch_chain(checkpoint_wgrad_sum_kernel, sum_grid, dim3(kCwSumLanes, parts), 0, (cudaStream_t)stream, 1, p));
    return ANI_OK;
}
size_t ani_checkpoint_weight_grad_workspace_bytes(int width, int out_width, const int* acs_host)
{
    long long n = 0;
    if (check_layer(acs_host, width, &n) || out_width < 1 || out_width > kNormMaxWidth) return 0;
    const RowRanges r = wgrad_ranges(acs_host, width, out_width);
    return one_range_each(r) ? 0 : (size_t)r.range_start[kTypes] * cw_blocks(width) * cw_blocks(out_width) * 1024 * sizeof(float);
}

}  // extern "C"
