// Weight gradient of the dense layer behind a checkpointed activation (ani_checkpoint.cuh), on the tensor cores:
//   dW = sum over the rows of an element  act(u~)^T dz   [width, out],  u~ from the codes as in the backward pass.
// The activations are never in memory: a row's bytes become activations on their way into the product.
//
// K, the long axis, is the atom.  A CTA takes a range of rows of one element and a tile of 128 x 128 of the output, and
// where an element has several ranges they write partial products that a second launch adds in order (no atomics).
// Chunks of 32 rows are staged by four groups of 128 threads in turn.  A chunk's bytes and its part of dz come to shared
// memory by asynchronous copies of 16 bytes (4 where rows of dz are not aligned), asked for when the group has read the
// chunk before.  (Bulk copies of a row each, 64 a chunk, took the issuing warp 5000 clocks and everybody's shared-memory
// reads with it.)  Then a thread has one column of A (a byte per row: with the row's base, step, mean and rstd, two numbers
// a row, and its column's gain and bias the activation is two FMAs and the function) and one column of B.  A goes to tensor
// memory, B to shared memory, both as tf32 high and low parts; hi hi, hi lo and lo hi are three instructions per eight rows.
//
// The tensor core cuts a sum off at the accumulator's last place, always towards zero, so a long chain of additions drifts:
// 1e-6 of the value per 32 additions.  So hi hi goes to two accumulators in turn, 128 rows to each, and while one is filled
// the other is added to float32 sums; the small products (2^-11 of the large ones) have one accumulator for the whole range.
// Error against float64 in the 2-norm 3e-7 to 4e-7 where layers are wide (plain float32 products 5e-7 to 9e-7), 2e-7 to 3e-7 for
// one column of 13,750 rows (plain float32 2e-7); with all products in the large accumulators 1.0e-6, and no faster.  Low times low is left out, 2^-22
// of a product.  There is no variant in single tf32 products.  Activations and gradients are finite: an infinite one has parts
// that are not, and its products come out as NaN.
//
// 512 x 512 of 110,000 rows: 397 us, 145 TFLOP/s of float32 products (three times that in tf32, 53 % of its rate).  A chunk and
// tile takes 1,900 clocks, of which the tensor core is busy 775; 56 % of the issue slots are used, by four staging warps a
// scheduler whose chains of shared-memory loads, exponentials and tensor-memory stores the rest waits for.
#pragma once

#include "ani_checkpoint.cuh"
#include "ani_mlp_wgrad.cuh"

namespace ani {

__host__ __device__ __forceinline__ int cw_blocks(int size) { return (size + 31) / 32; }

struct CheckpointWgradParams {
    const unsigned char* codes;
    const float2* blocks;
    const float *mean, *rstd;
    const float* gain[kTypes];
    const float* bias[kTypes];
    const float* grad_z;
    long long grad_stride;
    float* grad_w[kTypes];      // [width][out]
    float* partial;             // [ranges][row blocks][column blocks][32 columns][32 rows], blocks of 32 x 32 of the product
    RowRanges ranges;
    int width, out, norm;
    int whole;                  // rows of grad_z are whole 16-byte pieces
};

constexpr int kCwTile = 128, kCwK = kPipeK;       // output tile, rows of a chunk
static_assert(kCwTile == kCheckpointBlock, "the columns of a tile share their rows' base and step");
constexpr int kCwRound = kChainGroups;            // chunks per accumulator: one of every group
constexpr unsigned kCwMain = 0, kCwSmall = 256, kCwA = 384;      // tensor memory columns: two of 128, 128, two stages of 64

// 16 or 4 bytes to shared memory; the last `size` .. BYTES of them are zeros, and with size 0 nothing is read.
template <int BYTES> __device__ __forceinline__ void copy_async(void* dst_smem, const void* src, int size)
{
    if (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst_smem)), "l"(src), "r"(size) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst_smem)), "l"(src), "r"(size) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

struct CwShared {
    alignas(1024) unsigned char b[kChainGroups][2 * kPipeOperandBytes];
    alignas(16) unsigned char codes[kChainGroups][kCwK][kCwTile];      // a chunk's rows as they are
    alignas(16) float dz[kChainGroups][kCwK][kCwTile];
    alignas(16) float row[kMlpThreads / kWarp][2 * kCwK];   // per warp and two rows: step rstd of both, (base - mean) rstd of both
    alignas(8) unsigned long long full[kChainGroups], empty[kChainGroups], done[2], drained[2], end;
    unsigned tmem_base;
    int failed;
};

template <int ACT>
__global__ void __launch_bounds__(kMlpAllThreads, 1) checkpoint_wgrad_kernel(const __grid_constant__ CheckpointWgradParams p)
{
    extern __shared__ __align__(1024) unsigned char cw_smem_raw[];
    CwShared& sh = *reinterpret_cast<CwShared*>(cw_smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const RowRange range = range_of_cta(p.ranges, blockIdx.x);
    const int n_here = (int)(range.end - range.first);
    const int m0 = blockIdx.y * kCwTile, n0 = blockIdx.z * kCwTile;
    const int nchunks = (n_here + kCwK - 1) / kCwK, rounds = (nchunks + kCwRound - 1) / kCwRound;
    const int n_columns = min(kCwTile, (p.out - n0 + 15) & ~15);      // of the instruction

    if (warp == kMlpThreads / 32) tmem_alloc(&sh.tmem_base, 512);
    if (tid == 0) {
        for (int g = 0; g < kChainGroups; g++) {
            mbar_init(&sh.full[g], kMlpThreads / kChainGroups);
            mbar_init(&sh.empty[g], 1);
        }
        for (int k = 0; k < 2; k++) {
            mbar_init(&sh.done[k], 1);
            mbar_init(&sh.drained[k], kMlpThreads);
        }
        mbar_init(&sh.end, 1);
        sh.failed = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();
    pdl_trigger();
    const unsigned tmem = sh.tmem_base;

    if (warp == kMlpThreads / 32) {
        // ---- the products: one thread.  An instruction is issued when the tensor core is about to take it, so what this thread
        // waits for elsewhere (300 clocks a barrier) is lost there: the barriers of the next chunk are looked at in between. ----
        if (lane == 0) {
            bool ok = true;
            unsigned full_seen = 0, drained_seen = 0;
            const unsigned idesc = instr_desc(kCwTile, n_columns);
            for (int c = 0; c < nchunks && ok; c++) {
                const int g = c % kChainGroups, r = c / kCwRound;
                if (c % kCwRound == 0 && r >= 2 && !drained_seen) ok = mbar_wait(&sh.drained[r & 1], (unsigned)(r / 2 - 1) & 1u);
                if (!full_seen) ok = ok && mbar_wait(&sh.full[g], (unsigned)(c / kChainGroups) & 1u);
                if (!ok) break;
                tc_fence_after();
                const unsigned b_hi = smem_u32(sh.b[g]), b_lo = b_hi + kPipeOperandBytes;
                const unsigned a_hi = tmem + kCwA + (c & 1) * 2 * kPipeK, a_lo = a_hi + kPipeK;
                const unsigned acc = tmem + kCwMain + (r & 1) * 128;
                full_seen = drained_seen = 0;
#pragma unroll
                for (int ks = 0; ks < kPipeK / 8; ks++) {
                    const unsigned step = ks * 2 * kMlpLbo, col = ks * 8;
                    mma_tf32_ts(acc, a_hi + col, pipe_desc(b_hi + step), idesc, !(c % kCwRound == 0 && ks == 0));
                    mma_tf32_ts(tmem + kCwSmall, a_hi + col, pipe_desc(b_lo + step), idesc, !(c == 0 && ks == 0));
                    mma_tf32_ts(tmem + kCwSmall, a_lo + col, pipe_desc(b_hi + step), idesc, true);
                    if (ks == 2 && c + 1 < nchunks) {
                        const int next = c + 1, next_round = next / kCwRound;
                        full_seen = mbar_test(&sh.full[next % kChainGroups], (unsigned)(next / kChainGroups) & 1u);
                        if (next % kCwRound == 0 && next_round >= 2)
                            drained_seen = mbar_test(&sh.drained[next_round & 1], (unsigned)(next_round / 2 - 1) & 1u);
                    }
                }
                mma_commit(&sh.empty[g]);
                if (c % kCwRound == kCwRound - 1 || c == nchunks - 1) mma_commit(&sh.done[r & 1]);
            }
            if (ok) mma_commit(&sh.end);
            else sh.failed = 1;
        }
    } else {
        // ---- staging: group g of 128 threads takes chunks g, g + 4, ...; every warp has 32 x 32 of the sums ----
        const int g = warp >> 2, me = tid & 127;
        const unsigned lanes = tmem + ((unsigned)((warp & 3) * 32) << 16);
        const int row_bytes = checkpoint_row_bytes(p.width), row_blocks = checkpoint_blocks(p.width);
        const bool a_in = m0 + me < p.width;
        const unsigned char* a_src = p.codes + range.first * row_bytes + m0;
        const float* b_src = p.grad_z + range.first * p.grad_stride + n0;
        const int a_bytes = min(kCwTile, row_bytes - m0), b_columns = min(kCwTile, p.out - n0);
        const float2* blocks = p.blocks + range.first * row_blocks + blockIdx.y;
        const int b_shift = 32 - __clz(b_columns - 1);      // 2^b_shift >= b_columns
        // the copies of a chunk, by the group; rows of dz behind the range are zeros, bytes there are left as they are
        constexpr int kAPieces = kCwTile / 16, kBPieces = kCwTile / 4;      // of 16 bytes in a row
        const int a_row = me / kAPieces, a_at = 16 * (me % kAPieces), b_row = me / kBPieces, b_at = 4 * (me % kBPieces);
        auto fetch = [&](int c) {
            const int k0 = c * kCwK, valid = min(kCwK, n_here - k0);
            const unsigned char* a_from = a_src + (size_t)(k0 + a_row) * row_bytes + a_at;
#pragma unroll
            for (int i = 0; i < kCwK * kAPieces / 128; i++)
                if (a_row + i * (128 / kAPieces) < valid && a_at < a_bytes)
                    copy_async<16>(&sh.codes[g][a_row + i * (128 / kAPieces)][a_at], a_from + i * (128 / kAPieces) * row_bytes, 16);
            if (p.whole) {
                const float* b_from = b_src + (size_t)(k0 + b_row) * p.grad_stride + b_at;
                if (valid == kCwK && b_at < b_columns) {
                    const long long step = (128 / kBPieces) * p.grad_stride;
#pragma unroll
                    for (int i = 0; i < kCwK * kBPieces / 128; i++, b_from += step)
                        copy_async<16>(&sh.dz[g][b_row + i * (128 / kBPieces)][b_at], b_from, 16);
                } else if (b_at < b_columns) {
                    for (int i = 0; i < kCwK * kBPieces / 128; i++) {
                        const int row = b_row + i * (128 / kBPieces);
                        copy_async<16>(&sh.dz[g][row][b_at], row < valid ? b_from + (size_t)i * (128 / kBPieces) * p.grad_stride : b_src,
                                       row < valid ? 16 : 0);
                    }
                }
            } else {
                // single values; a row of few columns is shared out among fewer threads (by one thread 32 copies take 4,400 clocks)
                const int column = me & ((1 << b_shift) - 1);
                if (column < b_columns)
#pragma unroll 4
                    for (int row = me >> b_shift; row < kCwK; row += 128 >> b_shift)
                        copy_async<4>(&sh.dz[g][row][column], b_src + (row < valid ? (size_t)(k0 + row) * p.grad_stride + column : 0), row < valid ? 4 : 0);
            }
        };
        auto group_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(2 + g) : "memory"); };
        const float gain = p.norm && a_in ? p.gain[range.element][m0 + me] : 1.0f;
        const float bias = p.norm && a_in ? p.bias[range.element][m0 + me] : 0.0f;
        bool timed_out = false;
        float sum[32];
#pragma unroll
        for (int i = 0; i < 32; i++) sum[i] = 0.0f;
        auto drain = [&](int r) {
            if (!timed_out) {
                timed_out = !mbar_wait(&sh.done[r & 1], (unsigned)(r / 2) & 1u);
                if (timed_out) sh.failed = 1;
            }
            __syncwarp();
            tc_fence_after();
            if (g * 32 < n_columns) {
                float v[32];
                tmem_load32(lanes + kCwMain + (r & 1) * 128 + g * 32, v);
#pragma unroll
                for (int i = 0; i < 32; i++) sum[i] += v[i];
            }
            tc_fence_before();
            mbar_arrive(&sh.drained[r & 1]);
        };
        // step rstd and (base - mean) rstd of the chunk's row `lane`, read a turn ahead
        float2 block = make_float2(0.0f, 0.0f);
        float mean = 0.0f, rstd = 1.0f;
        auto read_row = [&](int c) {
            const int k = c * kCwK + lane;
            const bool live = k < n_here;
            block = live ? blocks[(size_t)k * row_blocks] : make_float2(0.0f, 0.0f);
            mean = live && p.norm ? p.mean[range.first + k] : 0.0f;
            rstd = live && p.norm ? p.rstd[range.first + k] : 1.0f;
        };
        // Turn -1 asks for the first chunks, turn `rounds` only drains.  Every part stands once.
#pragma unroll 1
        for (int r = -1; r <= rounds; r++) {
            const int c = r * kCwRound + g;
            const bool staged = r >= 0 && c < nchunks;
            if (staged) {
                sh.row[warp][(lane & ~1) * 2 + (lane & 1)] = block.y * rstd;
                sh.row[warp][(lane & ~1) * 2 + (lane & 1) + 2] = (block.x - mean) * rstd;
                copies_wait();
                group_sync();      // everybody's copies
                // the products of the group's chunk before read this stage of shared memory
                if (r > 0 && !timed_out) timed_out = !mbar_wait(&sh.empty[g], (unsigned)(r - 1) & 1u);
                // columns behind the width of dz: columns of the product that are not stored
                if (me < n_columns) {
#pragma unroll
                    for (int k0 = 0; k0 < kCwK; k0 += 16) {
                        float v[16];
#pragma unroll
                        for (int k = 0; k < 16; k++) v[k] = sh.dz[g][k0 + k][me];
#pragma unroll
                        for (int k = 0; k < 16; k += 4)
                            pipe_store4<true>(sh.b[g], sh.b[g] + kPipeOperandBytes, pipe_offset(me, k0 + k),
                                              make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]));
                    }
                }
                fence_async_smem();
                // rows behind the range: their bytes are old ones, times a step of zero; the zeros of B take them out.
                // Columns behind the width: rows of the product that are not stored.
                // Half of A is formed before the wait for the stage of tensor memory (all of it would not fit the registers).
                const unsigned stage = lanes + kCwA + (c & 1) * 2 * kPipeK;
#pragma unroll
                for (int half = 0; half < kCwK; half += kCwK / 2) {
                    float2 a[kCwK / 4];
#pragma unroll
                    for (int k0 = 0; k0 < kCwK / 2; k0 += 8) {
                        // eight at a time, all loads first: one behind the other a value took 100 clocks.  A byte becomes a float
                        // by an OR and a subtraction: conversions share the unit of the exponentials.
                        float4 s[4];
                        unsigned code[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) code[k] = sh.codes[g][half + k0 + k][me];
#pragma unroll
                        for (int k = 0; k < 4; k++) s[k] = *reinterpret_cast<const float4*>(&sh.row[warp][2 * (half + k0) + 4 * k]);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            float2 q = __fadd2_rn(make_float2(__uint_as_float(code[2 * k] | 0x4b000000u), __uint_as_float(code[2 * k + 1] | 0x4b000000u)),
                                                  both(-8388608.0f));
                            q = __ffma2_rn(q, make_float2(s[k].x, s[k].y), make_float2(s[k].z, s[k].w));
                            a[k0 / 2 + k] = act_value<ACT>(__ffma2_rn(q, both(gain), both(bias)));
                        }
                    }
                    if (half == 0) {      // the products of chunk c - 2 read this stage of tensor memory
                        if (c >= 2 && !timed_out)
                            timed_out = !mbar_wait(&sh.empty[(c - 2) % kChainGroups], (unsigned)((c - 2) / kChainGroups) & 1u);
                        if (timed_out) sh.failed = 1;
                        __syncwarp();
                        tc_fence_after();
                    }
#pragma unroll
                    for (int k0 = 0; k0 < kCwK / 2; k0 += 8) {
                        float part[8];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            part[2 * k] = tf32_round(a[k0 / 2 + k].x);
                            part[2 * k + 1] = tf32_round(a[k0 / 2 + k].y);
                            a[k0 / 2 + k] = __fadd2_rn(a[k0 / 2 + k], make_float2(-part[2 * k], -part[2 * k + 1]));
                        }
                        tmem_store8(stage + half + k0, part);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            part[2 * k] = a[k0 / 2 + k].x;
                            part[2 * k + 1] = a[k0 / 2 + k].y;
                        }
                        tmem_store8(stage + kPipeK + half + k0, part);
                    }
                }
                tmem_store_wait();
                tc_fence_before();
                mbar_arrive(&sh.full[g]);
            }
            if (c + kChainGroups < nchunks) {
                if (staged) group_sync();      // the group has read the chunk's rows
                fetch(c + kChainGroups);
                read_row(c + kChainGroups);
            }
            if (r > 0) drain(r - 1);
        }
        bool ok = !timed_out;
        if (ok && !mbar_wait(&sh.end, 0u)) {
            ok = false;
            sh.failed = 1;
        }
        __syncwarp();
        tc_fence_after();
        float small[32];
        tmem_load32(lanes + kCwSmall + g * 32, small);
#pragma unroll
        for (int i = 0; i < 32; i++) sum[i] += small[i];
        producer_sync();      // the operand stages become transposition scratch; everybody knows of a failure
        if (ok && !sh.failed) {
            const int row_block = m0 / 32 + (warp & 3), column_block = n0 / 32 + g;
            if (p.ranges.range_start[range.element + 1] - p.ranges.range_start[range.element] != 1) {
                // as it is held, a column of 32 rows behind the other (rows through the scratch were 2 us)
                if (row_block < cw_blocks(p.width) && column_block < cw_blocks(p.out)) {
                    float* to = p.partial + (((size_t)blockIdx.x * cw_blocks(p.width) + row_block) * cw_blocks(p.out) + column_block) * 1024 + lane;
#pragma unroll
                    for (int i = 0; i < 32; i++) to[32 * i] = sum[i];
                }
            } else {
                float* scratch = reinterpret_cast<float*>(sh.b[0]) + warp * (32 * kMlpScratchStride);
#pragma unroll
                for (int i = 0; i < 32; i++) scratch[lane * kMlpScratchStride + i] = sum[i];
                __syncwarp();
                const int column = column_block * 32 + lane, first = row_block * 32;
                float* to = p.grad_w[range.element] + (size_t)first * p.out + column;
                if (column < p.out)
#pragma unroll 4
                    for (int i = 0; i < 32; i++, to += p.out)
                        if (first + i < p.width) *to = scratch[i * kMlpScratchStride + lane];
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && sh.failed) report(ANI_ERR_TIMEOUT);
    tc_fence_after();
    if (warp == kMlpThreads / 32) tmem_dealloc(tmem, 512);
}

// The partial products of an element's ranges, added in order.  A CTA has a quarter of a block, 8 columns of 32 rows; blockDim.y
// threads have a part of the ranges each, four rows at a time, and their sums are added in order too.  Zeros for an element
// without rows.
constexpr int kCwSumColumns = 8, kCwSumLanes = kCwSumColumns * 8, kCwSumParts = 8;
__global__ void __launch_bounds__(kCwSumLanes* kCwSumParts) checkpoint_wgrad_sum_kernel(const __grid_constant__ CheckpointWgradParams p)
{
    __shared__ alignas(16) float part[kCwSumParts][kCwSumColumns * 32];
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.y, first = p.ranges.range_start[t], n = p.ranges.range_start[t + 1] - first;
    if (n == 1 || !p.grad_w[t]) return;      // written already, or an element without rows and without a place
    constexpr int pieces = 32 / kCwSumColumns;
    const int parts = blockDim.y, blocks = cw_blocks(p.width) * cw_blocks(p.out), block = blockIdx.x / pieces, piece = blockIdx.x % pieces;
    const float* from = p.partial + ((size_t)first * blocks + block) * 1024 + piece * (kCwSumColumns * 32) + 4 * threadIdx.x;
    const int each = (n + parts - 1) / parts, begin = threadIdx.y * each, end = min(n, begin + each);
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int k = begin; k < end; k++) {
        float v[4];
        load4(from + (size_t)k * blocks * 1024, v);
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] += v[i];
    }
    store4(&part[threadIdx.y][4 * threadIdx.x], s);
    __syncthreads();
    // a thread has a place of the piece: 8 columns next to each other in memory
    const int column0 = block % cw_blocks(p.out) * 32 + piece * kCwSumColumns, row0 = block / cw_blocks(p.out) * 32;
    for (int i = threadIdx.y * kCwSumLanes + threadIdx.x; i < kCwSumColumns * 32; i += parts * kCwSumLanes) {
        const int c = i % kCwSumColumns, r = i / kCwSumColumns;
        if (column0 + c >= p.out || row0 + r >= p.width) continue;
        float total = part[0][c * 32 + r];
        for (int k = 1; k < parts; k++) total += part[k][c * 32 + r];
        p.grad_w[t][(size_t)(row0 + r) * p.out + column0 + c] = total;
    }
}

}  // namespace ani
