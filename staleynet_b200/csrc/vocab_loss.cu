// vocab_loss.cu — softmax cross entropy over a large vocabulary, with its gradients, without keeping the logits.
//
//   z = H W^T,  lse_i = log sum_v exp(z_iv),  loss_i = lse_i - z_it,  P = softmax(z) - onehot(t)
//   dH = c P W,  dW = c P^T H
//
// Pass 1 computes z tile by tile on the tensor cores and reduces each tile in its epilogue to one (maximum, sum) pair
// for each row and 128 classes (lse_tile in gemm_tc.cuh); combine_kernel joins the pairs of a row in a fixed order. Pass
// 2, for gradients, takes the vocabulary in pieces: each piece's tiles of z are computed again, turned into P in the
// epilogue (softmax_grad_tile), and the piece of P is the operand of two ordinary products. No logits are kept: the
// piece of P is bounded by kPieceBytes, and the pairs of pass 1 take one byte for each 16 logits.
//
// What bounds it: the products, 2 rows x width x classes operations for the loss and 8 for loss and gradients (6 and
// the second computation of z), except for a few rows, where it is the one (loss) or three (gradients) passes over the
// weight.
//
// f32 operands: x = hi + lo with hi its nearest value of 11 significant bits and lo the rest's, and
// x y = lo hi' + hi lo' + hi hi' up to 2^-22 of |x y|: three TF32 products with f32 sums. The logits take them as one
// product over three times the width (H packed as lo|hi|hi, W as hi|lo|hi), so that the epilogue sees whole logits; the
// tensor core cuts off what a sum's last bit cannot hold at every instruction, so the small products come first, where
// that costs little. A gradient product takes its three in one launch, each unit of work the small ones and then at most
// kSumLength of the large one, added into f32 outputs; or, in the deterministic order, one after the other.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "internal.h"

namespace snb {
namespace {

constexpr uint32_t kEmptyToken = 0xFFFFFFFFu;      // EMPTY_TOKEN (kernels/mod.rs:46)
constexpr uint64_t kPieceBytes = 768ull << 20;     // bound of a piece of P
constexpr uint64_t kWeightBytes = 256ull << 20;    // bound of a packed piece of the weight
// Longest sum of f32 products on the tensor core, which cuts off the accumulator's lost bits at each instruction (8
// products) instead of rounding: 2^-24 of the sum each time on average, always towards zero. Measured as the relative
// error of a weight gradient over 1,021 rows: 2.5e-6 in one sum, 0.7e-6 in sums of 256 (0.6e-6 with f32 arithmetic).
constexpr uint64_t kSumLength = 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint64_t kHalfTile = 128;                // classes that one (maximum, sum) pair covers

__device__ __forceinline__ uint16_t bf16_bits(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return static_cast<uint16_t>((u >> 16) | 0x40u);  // NaN stays NaN
    return static_cast<uint16_t>((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

// A packed copy of a row-major matrix: dst[i, j] = src[i, j] (rows src_ld and dst_ld elements apart), zero outside
// [rows, cols] up to [dst_rows, dst_cols] and in the rows that have no target (`targets`, may be null): their hidden
// vectors may hold anything, and 0 * NaN must not reach the weight's gradient. bf16 stays bf16; f32 becomes three
// planes of TF32 values, plane k at dst + plane[k], holding the leading part (low bit k of `low` clear) or the rest.
struct PackParams {
    const void* src;
    int64_t src_ld, rows, cols;
    void* dst;
    int64_t dst_ld, dst_rows, dst_cols;
    const uint32_t* targets;
    int64_t plane[3];
    int32_t low;
    uint4* zero[2];         // f32: arrays that become zeros on the way, of zero_count 16-byte pieces
    int64_t zero_count[2];
};

// Small kernels start while the kernel before them drains (programmatic launch) and wait for it here.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ bool has_target(const uint32_t* targets, int64_t row) {
    return targets == nullptr || __ldg(targets + row) != kEmptyToken;
}

// The three elementwise kernels (the two that pack, and store_kernel) take 4 columns (16 bytes of f32) a thread: blockDim.x
// threads along a row, blockDim.y rows a block, rows in steps of the grid. `vec`: the side that is not in the workspace
// allows 4-element accesses. Memory bounds them; at the sizes where they are needed, a launch's few microseconds do: packing
// 8,192 x 768 bf16 takes 9 us (25 MB, 2.8 TB/s), splitting 10,007 x 256 f32 9 us (41 MB, 4.6 TB/s), storing 8,192 x 768
// f32 sums as bf16 10.6 us (38 MB, 3.6 TB/s).
//
// The pack kernels wait for the kernel before them only at their end: a packed weight may be written while the hidden rows
// are still being packed, and whoever waits for the weight then waits for both.
__global__ void __launch_bounds__(256) pack_bf16_kernel(const PackParams p, int vec) {
    allow_next_kernel();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; i < p.dst_rows;
         i += static_cast<int64_t>(gridDim.x) * blockDim.y) {
        const bool live = i < p.rows && has_target(p.targets, i);
        const uint16_t* src = static_cast<const uint16_t*>(p.src) + i * p.src_ld;
        uint16_t* dst = static_cast<uint16_t*>(p.dst) + i * p.dst_ld;
        for (int64_t j = 4 * threadIdx.x; j < p.dst_cols; j += 4 * blockDim.x) {
            uint2 q = make_uint2(0, 0);
            if (live && vec && j + 4 <= p.cols) {
                q = __ldg(reinterpret_cast<const uint2*>(src + j));
            } else if (live) {
                uint32_t h[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) h[k] = j + k < p.cols ? src[j + k] : 0;
                q = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
            }
            *reinterpret_cast<uint2*>(dst + j) = q;
        }
    }
    wait_for_previous_kernel();
}

// The nearest value of 11 significant bits; a finite value that would round past the largest float is cut off instead.
__device__ __forceinline__ float tf32_nearest(float x) {
    const uint32_t u = __float_as_uint(x);
    const uint32_t r = (u + 0x0FFFu + ((u >> 13) & 1u)) & 0xFFFFE000u;
    return __uint_as_float((r & 0x7F800000u) == 0x7F800000u ? u & 0xFFFFE000u : r);
}

__global__ void __launch_bounds__(256) pack_split_kernel(const PackParams p, int vec) {
    allow_next_kernel();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; i < p.dst_rows;
         i += static_cast<int64_t>(gridDim.x) * blockDim.y) {
        const bool live = i < p.rows && has_target(p.targets, i);
        const float* src = static_cast<const float*>(p.src) + i * p.src_ld;
        float* dst = static_cast<float*>(p.dst) + i * p.dst_ld;
        for (int64_t j = 4 * threadIdx.x; j < p.dst_cols; j += 4 * blockDim.x) {
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, hi[4], lo[4];
            if (live && vec && j + 4 <= p.cols) {
                const float4 q = __ldg(reinterpret_cast<const float4*>(src + j));
                x[0] = q.x; x[1] = q.y; x[2] = q.z; x[3] = q.w;
            } else if (live) {
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = j + k < p.cols ? src[j + k] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // An infinity or NaN stays whole in the leading part (inf - inf would make the rest NaN).
                const bool finite = (__float_as_uint(x[k]) & 0x7F800000u) != 0x7F800000u;
                hi[k] = finite ? tf32_nearest(x[k]) : x[k];
                lo[k] = finite ? tf32_nearest(x[k] - hi[k]) : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 3; ++k)
                *reinterpret_cast<float4*>(dst + p.plane[k] + j) =
                    (p.low >> k) & 1 ? make_float4(lo[0], lo[1], lo[2], lo[3]) : make_float4(hi[0], hi[1], hi[2], hi[3]);
        }
    }
    const int64_t thread = threadIdx.y * blockDim.x + threadIdx.x, block = blockDim.x * blockDim.y;
#pragma unroll
    for (int z = 0; z < 2; ++z)
        for (int64_t i = blockIdx.x * block + thread; i < p.zero_count[z]; i += gridDim.x * block)
            p.zero[z][i] = make_uint4(0, 0, 0, 0);
    wait_for_previous_kernel();
}

// out[i, j] (+)= ws[i, j] for i < rows, j < cols; the workspace's rows are multiples of 4 elements.
__global__ void __launch_bounds__(256) store_kernel(const float* ws, int64_t ws_ld, void* out, int out_bf16,
                                                    int64_t out_ld, int64_t rows, int64_t cols, int accumulate, int vec) {
    allow_next_kernel();
    wait_for_previous_kernel();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; i < rows;
         i += static_cast<int64_t>(gridDim.x) * blockDim.y) {
        const float* src = ws + i * ws_ld;
        for (int64_t j = 4 * threadIdx.x; j < cols; j += 4 * blockDim.x) {
            const float4 q = *reinterpret_cast<const float4*>(src + j);
            const float v[4] = {q.x, q.y, q.z, q.w};
            const int n = static_cast<int>(min(static_cast<int64_t>(4), cols - j));
            if (out_bf16) {
                uint16_t* dst = static_cast<uint16_t*>(out) + i * out_ld + j;
                if (vec && n == 4)
                    *reinterpret_cast<uint2*>(dst) = make_uint2(bf16_bits(v[0]) | static_cast<uint32_t>(bf16_bits(v[1])) << 16,
                                                                bf16_bits(v[2]) | static_cast<uint32_t>(bf16_bits(v[3])) << 16);
                else
                    for (int k = 0; k < n; ++k) dst[k] = bf16_bits(v[k]);
            } else {
                float* dst = static_cast<float*>(out) + i * out_ld + j;
                if (vec && n == 4 && !accumulate)
                    *reinterpret_cast<float4*>(dst) = q;
                else
                    for (int k = 0; k < n; ++k) dst[k] = accumulate ? dst[k] + v[k] : v[k];
            }
        }
    }
}

constexpr int kCombineRows = 32, kCombineLanes = 32;

// Joins a (maximum, sum) pair into another.
__device__ __forceinline__ void join(float2& a, float2 b) {
    const float inf = __int_as_float(0x7f800000);
    const float next = fmaxf(a.x, b.x);
    const float base = next == -inf ? 0.0f : __fmul_rn(next, kLog2e);
    a.y = a.y * exp2f(__fmul_rn(a.x, kLog2e) - base) + b.y * exp2f(__fmul_rn(b.x, kLog2e) - base);
    a.x = next;
}

// Joins the (maximum, sum) pairs of each row: the block's 32 rows lie along the threads of a warp (coalesced reads), its
// 32 warps take every 32nd pair; then a warp for each row joins the 32 results in a fixed tree, so the result does not
// depend on scheduling. Writes the row's loss and, for pass 2, (log2 e maximum, log2 sum), with a maximum of +inf in a row
// without a target (every exponential is then 0) and NaN for a target that is no class. A grid of one block also writes
// the sum of the losses. (Having the block that finishes last write it for larger grids, by a ticket, measured no faster
// than loss_sum_kernel, whose launch hides behind this kernel: 189.8 against 189.1 us for 4,096 x 512 x 50,021 bf16.)
//   Bound by the latency of the chain read, join, tree: 6.5 us for one row of 32,000 classes, 9 us for 8,192 rows of
// 32,768 (17 MB).
__global__ void __launch_bounds__(kCombineRows * kCombineLanes)
    combine_kernel(const float2* partials, int64_t pairs, int64_t rows, const uint32_t* targets, uint64_t classes,
                   const float* target_logit, const float* exact_logit, float* losses, float2* row_stats, float* loss_sum) {
    __shared__ float2 part[kCombineLanes][kCombineRows + 1];
    __shared__ float row_loss[kCombineRows];
    allow_next_kernel();
    wait_for_previous_kernel();
    const int r = threadIdx.x & 31, w = threadIdx.x >> 5;
    const float inf = __int_as_float(0x7f800000);
    float2 v = make_float2(-inf, 0.0f);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kCombineRows + w;
    uint32_t t = kEmptyToken;
    float z = 0.0f, exact = 0.0f;
    if (r == 0 && row < rows) {  // (read early: the tree below waits for the pairs anyway)
        t = targets[row];
        z = target_logit[row];
        exact = exact_logit != nullptr ? exact_logit[row] : z;
    }
    const int64_t read_row = static_cast<int64_t>(blockIdx.x) * kCombineRows + r;
    if (read_row < rows) {
        // Several pairs at a time: their reads overlap, and all but one factor of their sums are independent of each other.
        constexpr int kBatch = 8;
        for (int64_t k = w; k < pairs; k += kBatch * kCombineLanes) {
            float2 in[kBatch];
            float next = v.x;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int64_t pair = k + i * kCombineLanes;
                in[i] = pair < pairs ? partials[pair * rows + read_row] : make_float2(-inf, 0.0f);
                next = fmaxf(next, in[i].x);
            }
            const float base = next == -inf ? 0.0f : __fmul_rn(next, kLog2e);
            v.y *= exp2f(__fmul_rn(v.x, kLog2e) - base);
#pragma unroll
            for (int i = 0; i < kBatch; ++i) v.y += in[i].y * exp2f(__fmul_rn(in[i].x, kLog2e) - base);
            v.x = next;
        }
    }
    part[w][r] = v;
    __syncthreads();
    v = part[r][w];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, v.x, d), __shfl_xor_sync(0xffffffffu, v.y, d));
        join(v, other);
    }
    float loss = 0.0f;
    if (r == 0 && row < rows) {
        const float nan = __int_as_float(0x7fc00000);
        // The sum is one of exponentials above the rounded product `base`, so lse = ln 2 (base + log2 sum): taken against the
        // maximum itself, each loss would be off by base's rounding (up to 1e-5 for logits of 200). The fused difference of
        // base and k z rounds once more, after the two have cancelled.
        const float base = __fmul_rn(v.x, kLog2e);
        if (t != kEmptyToken) loss = t < classes ? kLn2 * (fmaf(-z, kLog2e, base) + log2f(v.y)) : nan;
        // The exact logit z + d in the place of z, in the target's term of the sum as well: with p its share exp(-loss),
        // lse grows by log(1 + p (e^d - 1)). (Not where z or the loss is no number or infinite.)
        const float d = exact - z;
        if (t < classes && fabsf(d) < 1.0f && loss < inf) loss += log1pf(expf(-loss) * expm1f(d)) - d;
        if (loss < 0.0f) loss = 0.0f;  // what is left of the roundings of a loss of 0
        losses[row] = loss;
        if (row_stats != nullptr)
            row_stats[row] = t == kEmptyToken ? make_float2(inf, 0.0f)
                                              : make_float2(t < classes ? __fmul_rn(v.x, kLog2e) : nan, log2f(v.y));
    }
    if (loss_sum == nullptr || gridDim.x > 1) return;
    if (r == 0) row_loss[w] = loss;
    __syncthreads();
    if (w != 0) return;
    loss = row_loss[r];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, d);
    if (r == 0) *loss_sum = loss;
}

// The loss alone of a few rows where the tensor cores could not read the weight as it lies (see few_rows): up to four rows
// in one pass over the weight, which is what bounds it, on the CUDA cores. Logits are f32 sums; each thread block leaves one
// (maximum, sum) pair for each row.
constexpr int kFewThreads = 256;
constexpr uint64_t kFewWidth = 4096;  // longest hidden row: four as f32 take 64 KB of shared memory

struct FewParams {
    const void* hidden;
    int64_t hidden_ld;
    const void* weight;
    int64_t weight_ld;
    int32_t rows, all_rows, width;  // of this launch (1 to 4) and of the call
    int64_t classes;
    const uint32_t* targets;
    float2* partials;               // [blocks, all_rows], from this launch's first row on
    float* target_logit;
    int32_t vec;  // f32: 16-byte accesses to the weight's rows (bf16 rows that allow them are the tensor cores')
};

__device__ __forceinline__ float element_of(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float element_of(const uint16_t* p, int64_t i) {
    return __uint_as_float(static_cast<uint32_t>(p[i]) << 16);
}

// The hidden rows as f32 in shared memory, [R, ld], zero past the call's rows.
template <int R, typename E>
__device__ __forceinline__ void stage_hidden(const FewParams& p, float* h, int ld) {
    for (int k = threadIdx.x; k < p.width; k += kFewThreads) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            h[r * ld + k] = r < p.rows ? element_of(static_cast<const E*>(p.hidden), r * p.hidden_ld + k) : 0.0f;
    }
    __syncthreads();
}

// Takes the logits z[0 .. n) of the classes from v on into a row's statistics.
template <int N>
__device__ __forceinline__ void take_logits(const FewParams& p, int r, int64_t v, const float (&z)[N], int n, float2& stats) {
    const float inf = __int_as_float(0x7f800000);
    float next = stats.x;
#pragma unroll
    for (int c = 0; c < N; ++c) next = c < n ? fmaxf(next, z[c]) : next;
    const float base = next == -inf ? 0.0f : __fmul_rn(next, kLog2e);
    float sum = stats.y * exp2f(__fmul_rn(stats.x, kLog2e) - base);
#pragma unroll
    for (int c = 0; c < N; ++c) sum += c < n ? exp2f(fmaf(z[c], kLog2e, -base)) : 0.0f;
    stats = make_float2(next, sum);
    const int64_t t = r < p.rows ? static_cast<int64_t>(__ldg(p.targets + r)) - v : -1;
    if (t >= 0 && t < n) {
#pragma unroll
        for (int c = 0; c < N; ++c)
            if (t == c) p.target_logit[r] = z[c];
    }
}

// Leaves the block's pair of each row, joined from its warps' in a fixed order; every lane of a warp holds the warp's.
template <int R>
__device__ __forceinline__ void leave_pairs(const FewParams& p, const float2 (&stats)[R]) {
    __shared__ float2 part[R][kFewThreads / 32];
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) part[r][threadIdx.x >> 5] = stats[r];
    __syncthreads();
    if (threadIdx.x < R && static_cast<int>(threadIdx.x) < p.rows) {
        float2 v = part[threadIdx.x][0];
        for (int w = 1; w < kFewThreads / 32; ++w) join(v, part[threadIdx.x][w]);
        p.partials[static_cast<int64_t>(blockIdx.x) * p.all_rows + threadIdx.x] = v;
    }
}

// Weight [classes, width]: a warp takes four classes at a time, its lanes 16 bytes of each f32 row in turn, or an element.
template <int R, typename E>
__global__ void __launch_bounds__(kFewThreads) few_rows_kernel(const FewParams p) {
    extern __shared__ __align__(16) float h[];
    allow_next_kernel();
    const int ld = (p.width + 3) & ~3;
    stage_hidden<R, E>(p, h, ld);
    const int lane = threadIdx.x & 31;
    const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kFewThreads / 32) + (threadIdx.x >> 5);
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (kFewThreads / 32);
    const E* weight = static_cast<const E*>(p.weight);
    float2 stats[R];
#pragma unroll
    for (int r = 0; r < R; ++r) stats[r] = make_float2(-__int_as_float(0x7f800000), 0.0f);
    for (int64_t v0 = 4 * warp; v0 < p.classes; v0 += 4 * warps) {
        const int n = static_cast<int>(min(static_cast<int64_t>(4), p.classes - v0));
        float z[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r) z[r][0] = z[r][1] = z[r][2] = z[r][3] = 0.0f;
        const E* rows = weight + v0 * p.weight_ld;
        bool done = false;
        if constexpr (sizeof(E) == 4) {
            if (p.vec) {
                done = true;
#pragma unroll 3
                for (int k = lane * 4; k < p.width; k += 32 * 4) {
                    float4 q[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        q[c] = c < n ? __ldg(reinterpret_cast<const float4*>(rows + c * p.weight_ld + k)) : make_float4(0, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float4 x = *reinterpret_cast<const float4*>(h + r * ld + k);
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            z[r][c] = fmaf(q[c].w, x.w, fmaf(q[c].z, x.z, fmaf(q[c].y, x.y, fmaf(q[c].x, x.x, z[r][c]))));
                    }
                }
            }
        }
        if (!done) {
            for (int k = lane; k < p.width; k += 32)
                for (int c = 0; c < n; ++c) {
                    const float w = element_of(rows, c * p.weight_ld + k);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float sum = fmaf(w, h[r * ld + k], c == 0 ? z[r][0] : c == 1 ? z[r][1] : c == 2 ? z[r][2] : z[r][3]);
                        if (c == 0) z[r][0] = sum;
                        else if (c == 1) z[r][1] = sum;
                        else if (c == 2) z[r][2] = sum;
                        else z[r][3] = sum;
                    }
                }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1)
#pragma unroll
                for (int c = 0; c < 4; ++c) z[r][c] += __shfl_xor_sync(0xffffffffu, z[r][c], d);
            take_logits(p, r, v0, z[r], n, stats[r]);
        }
    }
    leave_pairs<R>(p, stats);
}

// Weight [width, classes]: a block takes 32 PER classes, a lane PER of them, its warps an eighth of the width each; their
// sums meet in shared memory.
template <int R, typename E>
__global__ void __launch_bounds__(kFewThreads) few_rows_across_kernel(const FewParams p) {
    extern __shared__ __align__(16) float h[];  // [R, width], then [8 warps, R, 32 PER] sums
    allow_next_kernel();
    stage_hidden<R, E>(p, h, p.width);
    constexpr int PER = 16 / sizeof(E);
    constexpr int WARPS = kFewThreads / 32;
    float* sums = h + (R * p.width + 3) / 4 * 4;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t v0 = static_cast<int64_t>(blockIdx.x) * 32 * PER;
    const int64_t v = v0 + lane * PER;
    const E* weight = static_cast<const E*>(p.weight);
    float z[R][PER];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < PER; ++e) z[r][e] = 0.0f;
    const int each = (p.width + WARPS - 1) / WARPS;
    const int end = min(p.width, (w + 1) * each);
    const bool whole = sizeof(E) == 4 && p.vec && v + PER <= p.classes;
#pragma unroll 8
    for (int k = w * each; k < end; ++k) {
        const E* row = weight + static_cast<int64_t>(k) * p.weight_ld + v;
        float x[PER];
        if (whole) {
            if constexpr (sizeof(E) == 4) {
                const float4 q = __ldg(reinterpret_cast<const float4*>(row));
                x[0] = q.x; x[1] = q.y; x[2] = q.z; x[3] = q.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < PER; ++e) x[e] = v + e < p.classes ? element_of(row, e) : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < PER; ++e) z[r][e] = fmaf(x[e], h[r * p.width + k], z[r][e]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < PER; ++e) sums[(w * R + r) * 32 * PER + lane * PER + e] = z[r][e];
    __syncthreads();
    float2 stats[R];
#pragma unroll
    for (int r = 0; r < R; ++r) stats[r] = make_float2(-__int_as_float(0x7f800000), 0.0f);
    for (int c = threadIdx.x; c < 32 * PER; c += kFewThreads) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < WARPS; ++k) sum += sums[(k * R + r) * 32 * PER + c];
            const float z1[1] = {sum};
            if (v0 + c < p.classes) take_logits(p, r, v0 + c, z1, 1, stats[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int d = 16; d > 0; d >>= 1)
            join(stats[r], make_float2(__shfl_xor_sync(0xffffffffu, stats[r].x, d), __shfl_xor_sync(0xffffffffu, stats[r].y, d)));
    leave_pairs<R>(p, stats);
}

// The sum of the losses of more than 32 rows: one block, each thread every 1024th row, then a tree.
__global__ void __launch_bounds__(1024) loss_sum_kernel(const float* losses, int64_t rows, float* loss_sum) {
    __shared__ double part[32];
    allow_next_kernel();
    wait_for_previous_kernel();
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += 1024) s += static_cast<double>(losses[i]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = part[threadIdx.x];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (threadIdx.x == 0) *loss_sum = static_cast<float>(s);
    }
}

uint64_t round_up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// The shapes and the workspace of one call. Offsets are from a 256-byte aligned base.
struct Layout {
    bool f32, gradients, few, pack_hidden, pack_weight;
    uint64_t few_blocks;    // thread blocks of the few rows' kernels
    uint64_t elem;          // bytes of an operand element
    uint64_t seg;           // width rounded up to 16 bytes: a packed row, or one of the three planes of an f32 row
    uint64_t k_logits;      // length of the logits' sums
    uint64_t piece, pieces; // classes of a piece (the last one may have fewer) and pieces
    uint64_t hidden_ld, weight_ld;   // of the operands that the products read
    uint64_t grad_ld;       // of a piece of P
    uint64_t wgrad_ld, wgrad_rows;   // f32 weight gradient of a piece before it is stored
    bool hidden_grad_direct;         // dH is summed where the caller wants it
    bool weight_grad_direct;         // so is dW [classes, width]
    bool exact;                      // the targets' logits are computed once more (target_logits)
    uint64_t hidden_at, weight_at, partials_at, target_at, exact_at, stats_at, p_at, dh_at, dw_at, bytes;
};

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Whether the few rows' kernels take a call: the loss alone of hidden rows that fit into shared memory as f32 (64 KB for
// four), where the tensor cores would need a packed copy of the weight first. Measured over 100,000 x 1,024 f32 (63 us at
// the copy rate): 1 row 90 us, 4 rows 100 us, 16 rows 388 us (weight [classes, width]) or 578 us, by way of the split copy 5
// to 17 rows 592 to 634 us, so f32 goes up to 16 rows, four a
// pass; over 512 x 50,021 bf16, whose rows lie off every boundary: 1 row 48 us, 4 rows 53 us, packed 62 us. A bf16 weight
// that TMA can read stays with the tensor cores (32,000 x 768: 1 row 23 us here, 19 us there).
bool few_rows(const snb_vocabulary_loss_args& a) {
    const uint64_t per16 = a.type == SNB_TYPE_BF16 ? 8 : 4;
    const bool readable = a.type == SNB_TYPE_BF16 && aligned16(a.weight) && a.weight_stride % per16 == 0;
    return a.hidden_grad == nullptr && a.weight_grad == nullptr && !readable &&
           a.rows <= (a.type == SNB_TYPE_BF16 ? 4 : 16) && a.width <= kFewWidth;
}

Layout layout_of(const snb_vocabulary_loss_args& a, int sms) {
    Layout l{};
    l.f32 = a.type == SNB_TYPE_F32;
    l.gradients = a.hidden_grad != nullptr || a.weight_grad != nullptr;
    l.elem = l.f32 ? 4 : 2;
    const uint64_t per16 = 16 / l.elem;
    l.seg = round_up(a.width, per16);
    l.few = few_rows(a);
    l.few_blocks = a.weight_transposed ? std::min<uint64_t>((a.classes + 31) / 32, 4ull * sms)
                                       : (a.classes + 32 * per16 - 1) / (32 * per16);
    l.k_logits = l.f32 ? 3 * l.seg : a.width;
    // Gradients need the hidden rows without a target to be zero: both their logits and the weight's gradient read them.
    l.pack_hidden = !l.few && (l.f32 || l.gradients || !aligned16(a.hidden) || a.hidden_stride % per16 != 0);
    // (The hidden gradient's product has `seg` columns: those past the width must be zeros of a packed weight.)
    l.pack_weight = !l.few && (l.f32 || !aligned16(a.weight) || a.weight_stride % per16 != 0 ||
                               (a.hidden_grad != nullptr && a.width != l.seg));
    // (Fitted to the whole device, whatever the budget of SMs, so that the workspace does not depend on that.)
    // A piece is as long as the bounds allow for P [rows, piece] and for the packed weight, in whole tiles: long pieces
    // make long sums for the hidden gradient and few additions into it. Between half that length and all of it, the one is
    // taken whose weight gradient fills the last round of CTA pairs best (measured at 16,384 x 768 x 131,072: pieces of
    // 8,192 classes, 96 tiles on 74 pairs, 12.3 ms; of 12,544, 147 tiles, 10.7 ms; of 16,384, 192 tiles, 10.5 ms).
    uint64_t tiles = (a.classes + 255) / 256;
    auto bound = [&](uint64_t bytes, uint64_t bytes_a_class) {
        tiles = std::min(tiles, std::max<uint64_t>(1, bytes / std::max<uint64_t>(1, bytes_a_class) / 256));
    };
    if (l.gradients) bound(kPieceBytes, a.rows * (l.f32 ? 8 : 2));
    if (l.pack_weight) bound(kWeightBytes, l.f32 ? 12 * l.seg : 2 * l.seg);
    if (tiles * 256 < a.classes && a.weight_grad != nullptr) {
        const uint64_t across = (a.width + 255) / 256, pairs = static_cast<uint64_t>(std::max(1, sms / 2));
        uint64_t best = tiles;
        double best_fill = 0.0;
        for (uint64_t t = tiles; t >= std::max<uint64_t>(1, tiles / 2) && t > 0; --t) {
            const double fill = static_cast<double>(t * across) / static_cast<double>(round_up(t * across, pairs));
            if (fill > best_fill + 1e-9) {
                best = t;
                best_fill = fill;
            }
        }
        tiles = best;
    }
    l.piece = std::min(tiles * 256, a.classes);
    l.pieces = (a.classes + l.piece - 1) / l.piece;
    const uint64_t piece_ld = round_up(l.piece, 8);
    l.hidden_ld = l.pack_hidden ? (l.f32 ? 3 * l.seg : l.seg) : a.hidden_stride;
    l.weight_ld = !l.pack_weight ? a.weight_stride
                                 : a.weight_transposed ? (l.f32 ? 3 * l.seg : l.seg) : piece_ld;
    l.grad_ld = piece_ld;
    l.wgrad_rows = a.weight_transposed ? l.piece : l.seg;
    l.wgrad_ld = a.weight_transposed ? l.seg : piece_ld;
    l.hidden_grad_direct = a.hidden_grad_type == SNB_TYPE_F32 && aligned16(a.hidden_grad) && a.width % 4 == 0;
    l.weight_grad_direct = a.weight_transposed != 0 && a.weight_grad_type == SNB_TYPE_F32 && aligned16(a.weight_grad) &&
                           a.width % 4 == 0;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    l.hidden_at = take(l.pack_hidden ? a.rows * l.hidden_ld * l.elem : 0);
    l.weight_at = take(l.pack_weight ? (a.weight_transposed ? l.piece * l.weight_ld
                                                            : (l.f32 ? 3 : 1) * l.seg * l.weight_ld) * l.elem : 0);
    l.partials_at = take((l.few ? l.few_blocks : (a.classes + kHalfTile - 1) / kHalfTile) * a.rows * sizeof(float2));
    // (The tensor cores wait for the epilogue warps meanwhile, and their waits are bounded: this keeps it to milliseconds.)
    // Not for many rows of bf16 over a weight [width, classes], whose columns are gathered element by element (8,192 x 768 x
    // 32,768: 33 us of 1,416) for losses that are 4e-7 off without.
    l.exact = !l.few && a.rows * a.width <= (1ull << 31) &&
              (l.f32 || a.weight_transposed != 0 || a.rows <= 16 * static_cast<uint64_t>(sms));
    l.target_at = take(a.rows * 4);
    l.exact_at = take(l.exact ? a.rows * 4 : 0);
    l.stats_at = take(a.rows * sizeof(float2));
    l.p_at = take(l.gradients ? a.rows * l.grad_ld * (l.f32 ? 8 : 2) : 0);
    l.dh_at = take(a.hidden_grad != nullptr && !l.hidden_grad_direct ? a.rows * l.seg * 4 : 0);
    l.dw_at = take(a.weight_grad != nullptr ? l.wgrad_rows * l.wgrad_ld * 4 : 0);
    l.bytes = a.rows == 0 ? 0 : at + 256;
    return l;
}

// Launches a kernel that waits for the one before it by itself.
template <typename... KArgs, typename... Args>
void launch_early(void (*kernel)(KArgs...), unsigned grid, dim3 threads, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = threads;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

int launched(const char* what, std::string* err) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return SNB_OK;
    *err = cuda_message(what, e);
    return SNB_ERR_CUDA;
}

// Threads and blocks of the elementwise kernels for rows x cols: as many threads along a row as have 4 columns, a power of
// two, and enough blocks to fill the device eight times over at most.
dim3 row_threads(uint64_t cols) {
    unsigned x = 1;
    while (x < 256 && 4ull * x < cols) x *= 2;
    return dim3(x, 256 / x);
}
unsigned row_blocks(uint64_t rows, dim3 threads, int sms) {
    return static_cast<unsigned>(std::max<uint64_t>(1, std::min<uint64_t>((rows + threads.y - 1) / threads.y, 8ull * sms)));
}

// One call's stream, arguments and choices, and the products it issues.
struct Call {
    cudaStream_t stream;
    const snb_vocabulary_loss_args& a;
    const Layout l;
    bool deterministic;
    int sm_budget, sms;
    uint8_t* base;
    std::string* err;

    void* at(uint64_t offset) const { return base + offset; }

    // An operand of a gradient product; for f32 its leading parts, with the rest at `low` in the same layout.
    struct Part {
        const void* lead;
        const void* low;
    };

    int pack(const void* src, uint64_t src_ld, uint64_t rows, uint64_t cols, void* dst, uint64_t dst_ld,
             uint64_t dst_rows, uint64_t dst_cols, const uint32_t* targets, uint64_t plane, int low, bool early,
             bool zeros = false) const {
        PackParams p{};
        if (zeros && zero_hidden_grad()) {
            p.zero[0] = static_cast<uint4*>(hidden_sums());
            p.zero_count[0] = static_cast<int64_t>(a.rows * (l.hidden_grad_direct ? a.width : l.seg) / 4);
        }
        if (zeros && zero_weight_grad()) {
            p.zero[1] = static_cast<uint4*>(a.weight_grad);
            p.zero_count[1] = static_cast<int64_t>(a.classes * a.width / 4);
        }
        p.src = src;
        p.src_ld = static_cast<int64_t>(src_ld);
        p.rows = static_cast<int64_t>(rows);
        p.cols = static_cast<int64_t>(cols);
        p.dst = dst;
        p.dst_ld = static_cast<int64_t>(dst_ld);
        p.dst_rows = static_cast<int64_t>(dst_rows);
        p.dst_cols = static_cast<int64_t>(dst_cols);
        p.targets = targets;
        for (int k = 0; k < 3; ++k) p.plane[k] = static_cast<int64_t>(k * plane);
        p.low = low;
        const dim3 threads = row_threads(dst_cols);
        const unsigned grid = row_blocks(dst_rows, threads, sms);
        const int vec = reinterpret_cast<uintptr_t>(src) % (4 * l.elem) == 0 && src_ld % 4 == 0;
        const auto kernel = l.f32 ? pack_split_kernel : pack_bf16_kernel;
        if (early) launch_early(kernel, grid, threads, stream, p, vec);
        else kernel<<<grid, threads, 0, stream>>>(p, vec);
        return launched("vocabulary loss pack kernel launch", err);
    }

    // f32 gradients whose sums are split have to start from zeros, which the hidden rows' packing writes: a memset before
    // each product takes 2.5 us and keeps the product's set-up from overlapping the kernel before it (1,021 x 256 x 10,007:
    // 168 us, 163 us this way). Not over hidden rows that the gradient is to replace: they are still being read.
    bool zero_hidden_grad() const {
        const auto h = reinterpret_cast<uintptr_t>(a.hidden), g = reinterpret_cast<uintptr_t>(a.hidden_grad);
        const uint64_t h_bytes = ((a.rows - 1) * a.hidden_stride + a.width) * l.elem, g_bytes = a.rows * a.width * 4;
        return l.f32 && !deterministic && a.hidden_grad != nullptr && l.piece > kSumLength &&
               (!l.hidden_grad_direct || g + g_bytes <= h || h + h_bytes <= g);
    }
    bool zero_weight_grad() const {
        return l.f32 && !deterministic && a.weight_grad != nullptr && a.accumulate == 0 && l.weight_grad_direct &&
               a.rows > kSumLength;
    }

    void* hidden_sums() const { return l.hidden_grad_direct ? a.hidden_grad : at(l.dh_at); }

    float* exact_logit() const { return l.exact ? static_cast<float*>(at(l.exact_at)) : nullptr; }

    const void* hidden() const { return l.pack_hidden ? at(l.hidden_at) : a.hidden; }

    Part hidden_part() const {
        const float* h = static_cast<const float*>(at(l.hidden_at));
        return l.f32 ? Part{h + l.seg, h} : Part{hidden(), nullptr};
    }

    Part weight_part(const void* w) const {
        const uint64_t plane = a.weight_transposed ? l.seg : l.seg * l.weight_ld;
        return l.f32 ? Part{w, static_cast<const float*>(w) + plane} : Part{w, nullptr};
    }

    Part grad_part() const {
        const void* p = at(l.p_at);
        return l.f32 ? Part{p, static_cast<const float*>(p) + a.rows * l.grad_ld} : Part{p, nullptr};
    }

    // The weight of the classes from v0 on, packed into the workspace where the products cannot read it in place. early:
    // the kernel before it on the stream packs the hidden rows.
    int weight(uint64_t v0, uint64_t n, const void** w, bool early = false) const {
        const uint64_t offset = (a.weight_transposed ? v0 * a.weight_stride : v0) * l.elem;
        const void* src = static_cast<const uint8_t*>(a.weight) + offset;
        *w = src;
        if (!l.pack_weight) return SNB_OK;
        *w = at(l.weight_at);
        constexpr int kHiLoHi = 2;
        if (a.weight_transposed)
            return pack(src, a.weight_stride, n, a.width, at(l.weight_at), l.weight_ld, n, l.seg, nullptr, l.seg, kHiLoHi,
                        early);
        return pack(src, a.weight_stride, a.width, n, at(l.weight_at), l.weight_ld, l.seg, round_up(n, 8), nullptr,
                    l.seg * l.weight_ld, kHiLoHi, early);
    }

    VocabProduct logits(uint64_t v0, uint64_t n, const void* w) const {
        VocabProduct v{};
        v.type = a.type;
        v.rows = a.rows;
        v.classes = n;
        v.inner = l.k_logits;
        v.A = hidden();
        v.a_ld = l.hidden_ld;
        v.B = w;
        v.b_ld = l.weight_ld;
        v.b_mn_major = a.weight_transposed == 0;
        v.targets = a.targets;
        v.class_begin = static_cast<int64_t>(v0);
        v.partials = static_cast<float2*>(at(l.partials_at)) + v0 / kHalfTile * a.rows;
        v.target_logit = static_cast<float*>(at(l.target_at));
        v.exact_logit = v0 == 0 ? exact_logit() : nullptr;
        v.vocabulary = a.classes;
        v.hidden = a.hidden;
        v.weight = a.weight;
        v.hidden_row = a.hidden_stride;
        v.weight_class = a.weight_transposed ? a.weight_stride : 1;
        v.weight_inner = a.weight_transposed ? 1 : a.weight_stride;
        v.width = a.width;
        v.row_stats = static_cast<const float2*>(at(l.stats_at));
        v.sm_budget = sm_budget;
        return v;
    }

    // C [rows, cols] (dense) (+)= grad_scale * A B; for f32 the three products of the split operands. c_ld: rows of C that
    // far apart, on the tensor cores or (`tensor_only` false) not at all.
    int product(uint64_t rows, uint64_t cols, uint64_t inner, Part A, snb_operand left, Part B, snb_operand right,
                void* C, int c_type, bool accumulate, uint64_t c_ld = 0, bool* tensor_only = nullptr) const {
        GemmRequest r{};
        r.p.rows = rows;
        r.p.cols = cols;
        r.p.inner = inner;
        r.p.left = left;
        r.p.right = right;
        r.p.scale = a.grad_scale;
        r.p.accumulate = accumulate ? 1 : 0;
        r.count = 1;
        r.a_type = r.b_type = a.type;
        r.c_type = c_type;
        r.precision = l.f32 ? SNB_PRECISION_TF32 : SNB_PRECISION_BF16;
        r.C = C;
        r.aux_type = c_type;
        r.deterministic = deterministic;
        r.sm_budget = sm_budget;
        r.c_ld = c_ld;
        auto issue = [&]() {
            bool tensor = false;
            int path = 0;
            int rc = tc_gemm_try(stream, r, &tensor, &path, err);
            if (tensor_only != nullptr) *tensor_only = tensor;
            else if (rc == SNB_OK && !tensor) rc = simt_gemm(stream, r, err);
            r.p.accumulate = 1;
            return rc;
        };
        r.A = A.lead;
        r.B = B.lead;
        if (!l.f32) return issue();
        if (!deterministic) {
            // All three products in one launch, where the small ones share the splits of the large one.
            auto lower = [](const Part& x) { return x.low < x.lead ? x.low : x.lead; };
            auto apart = [](const Part& x) {
                const auto lead = static_cast<const float*>(x.lead), low = static_cast<const float*>(x.low);
                return static_cast<uint64_t>(lead < low ? low - lead : lead - low);
            };
            r.A = lower(A);
            r.B = lower(B);
            r.split_inner = kSumLength;
            r.a_plane_stride = apart(A);
            r.b_plane_stride = apart(B);
            r.a_low = A.low < A.lead ? 0 : 1;
            r.b_low = B.low < B.lead ? 0 : 1;
            bool tensor = false;
            int path = 0;
            const int rc = tc_gemm_try(stream, r, &tensor, &path, err);
            if (rc != SNB_OK || tensor) return rc;
            r.split_inner = 0;
        }
        // One product after the other, the one of the leading parts in pieces of K: the deterministic order, and the way for
        // layouts that the tensor cores cannot read.
        r.A = A.low;
        r.B = B.lead;
        int rc = issue();
        r.A = A.lead;
        r.B = B.low;
        if (rc == SNB_OK) rc = issue();
        for (uint64_t k = 0; k < inner && rc == SNB_OK; k += kSumLength) {
            r.p.inner = std::min(kSumLength, inner - k);
            r.A = static_cast<const float*>(A.lead) + k * left.col_stride;
            r.B = static_cast<const float*>(B.lead) + k * right.row_stride;
            rc = issue();
        }
        return rc;
    }

    int store(const void* ws, uint64_t ws_ld, void* out, int out_type, uint64_t out_ld, uint64_t rows, uint64_t cols,
              bool accumulate) const {
        const dim3 threads = row_threads(cols);
        const int vec = reinterpret_cast<uintptr_t>(out) % (out_type == SNB_TYPE_BF16 ? 8 : 16) == 0 && out_ld % 4 == 0;
        launch_early(store_kernel, row_blocks(rows, threads, sms), threads, stream, static_cast<const float*>(ws), ws_ld, out,
                     out_type == SNB_TYPE_BF16, out_ld, rows, cols, accumulate, vec);
        return launched("vocabulary loss store kernel launch", err);
    }

    // dH (+)= P W of one piece, in f32: in the caller's gradient, or in the workspace with rows of `seg` columns. (The first,
    // and packing both operands side by side, took a call of 1,021 x 256 x 10,007 f32 from 174 to 169 us.)
    int hidden_grad(uint64_t v0, uint64_t n, const void* w) const {
        const snb_operand left{l.grad_ld, 1, 0};
        const snb_operand right = a.weight_transposed ? snb_operand{l.weight_ld, 1, 0} : snb_operand{1, l.weight_ld, 0};
        return product(a.rows, l.hidden_grad_direct ? a.width : l.seg, n, grad_part(), left, weight_part(w), right,
                       hidden_sums(), SNB_TYPE_F32, v0 > 0 || zero_hidden_grad());
    }

    // Whether an output's tiles, unsplit, keep three fifths of the CTA pairs' rounds busy.
    bool fills(uint64_t rows, uint64_t cols) const {
        const uint64_t tiles = (rows + 255) / 256 * ((cols + 255) / 256), pairs = static_cast<uint64_t>(std::max(1, sms / 2));
        return tiles * 10 >= round_up(tiles, pairs) * 6;
    }

    // dW (+)= P^T H of one piece (or its transpose, for a [width, classes] weight).
    int weight_grad(uint64_t v0, uint64_t n) const {
        const uint64_t es = a.weight_grad_type == SNB_TYPE_BF16 ? 2 : 4;
        const snb_operand p_t{1, l.grad_ld, 0}, h{l.hidden_ld, 1, 0}, h_t{1, l.hidden_ld, 0}, p_n{l.grad_ld, 1, 0};
        uint8_t* out = static_cast<uint8_t*>(a.weight_grad) + (a.weight_transposed ? v0 * a.width : v0) * es;
        int rc;
        if (a.weight_transposed) {
            // The rows of the piece are contiguous in the gradient: written there unless a row is no multiple of 16
            // bytes, or a bf16 gradient has so few tiles that its sums are better split (which needs f32).
            const bool dense = a.width * es % 16 == 0 && aligned16(out);
            if (l.weight_grad_direct || (dense && a.weight_grad_type == SNB_TYPE_BF16 && fills(n, a.width)))
                return product(n, a.width, a.rows, grad_part(), p_t, hidden_part(), h, out, a.weight_grad_type,
                               a.accumulate != 0 || zero_weight_grad());
            rc = product(n, l.seg, a.rows, grad_part(), p_t, hidden_part(), h, at(l.dw_at), SNB_TYPE_F32, false);
            return rc != SNB_OK ? rc : store(at(l.dw_at), l.wgrad_ld, out, a.weight_grad_type, a.width, n, a.width,
                                             a.accumulate != 0);
        }
        // The gradient's rows are strided here: written there under the same conditions, if no sums are split.
        if (a.classes * es % 16 == 0 && aligned16(out) && !l.f32 && a.accumulate == 0 && fills(a.width, n)) {
            bool tensor = false;
            rc = product(a.width, n, a.rows, hidden_part(), h_t, grad_part(), p_n, out, a.weight_grad_type, false, a.classes,
                         &tensor);
            if (rc != SNB_OK || tensor) return rc;
        }
        // Rows of round_up(n, 8) columns: those past n come from P's padding, are never stored, and touch no others.
        const uint64_t cols = round_up(n, 8);
        rc = product(l.seg, cols, a.rows, hidden_part(), h_t, grad_part(), p_n, at(l.dw_at), SNB_TYPE_F32, false);
        return rc != SNB_OK ? rc : store(at(l.dw_at), cols, out, a.weight_grad_type, a.classes, a.width, n,
                                         a.accumulate != 0);
    }

    template <int R, typename E>
    int few_typed(const FewParams& p) const {
        const auto shared = [&](int64_t width) -> int64_t {
            if (a.weight_transposed) return 4ll * R * ((width + 3) & ~3ll);
            return (4ll * R * width + 15) / 16 * 16 + 4ll * kFewThreads * R * (16 / static_cast<int>(sizeof(E)));
        };
        const int64_t smem = shared(p.width), most = shared(kFewWidth);
        const auto kernel = a.weight_transposed ? few_rows_kernel<R, E> : few_rows_across_kernel<R, E>;
        // What the kernel may use is a setting of the kernel, not of the launch: always the same one, or a call of another
        // thread could lower it between this call's setting and its launch.
        if (most > (44 << 10)) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
            if (e != cudaSuccess) {
                *err = cuda_message("cudaFuncSetAttribute(few_rows_kernel)", e);
                return SNB_ERR_CUDA;
            }
        }
        kernel<<<static_cast<unsigned>(l.few_blocks), kFewThreads, static_cast<size_t>(smem), stream>>>(p);
        return launched("few_rows_kernel launch", err);
    }

    int few() const {
        FewParams p{};
        p.hidden = a.hidden;
        p.hidden_ld = static_cast<int64_t>(a.hidden_stride);
        p.weight = a.weight;
        p.weight_ld = static_cast<int64_t>(a.weight_stride);
        p.all_rows = static_cast<int32_t>(a.rows);
        p.width = static_cast<int32_t>(a.width);
        p.classes = static_cast<int64_t>(a.classes);
        p.targets = a.targets;
        p.partials = static_cast<float2*>(at(l.partials_at));
        p.target_logit = static_cast<float*>(at(l.target_at));
        p.vec = l.f32 && aligned16(a.weight) && a.weight_stride % 4 == 0 && (!a.weight_transposed || a.width % 4 == 0);
        for (uint64_t row = 0; row < a.rows; row += 4) {
            p.rows = static_cast<int32_t>(std::min<uint64_t>(4, a.rows - row));
            int rc;
            if (l.f32) rc = p.rows == 1 ? few_typed<1, float>(p) : p.rows == 2 ? few_typed<2, float>(p) : few_typed<4, float>(p);
            else rc = p.rows == 1 ? few_typed<1, uint16_t>(p) : p.rows == 2 ? few_typed<2, uint16_t>(p) : few_typed<4, uint16_t>(p);
            if (rc != SNB_OK) return rc;
            p.hidden = static_cast<const uint8_t*>(p.hidden) + 4 * a.hidden_stride * l.elem;
            p.targets += 4;
            p.partials += 4;
            p.target_logit += 4;
        }
        return SNB_OK;
    }

    int run() const {
        int rc = SNB_OK;
        constexpr int kLoHiHi = 1;
        if (l.pack_hidden) {
            rc = pack(a.hidden, a.hidden_stride, a.rows, a.width, at(l.hidden_at), l.hidden_ld, a.rows, l.seg,
                      l.gradients ? a.targets : nullptr, l.seg, kLoHiHi, false, true);
            if (rc != SNB_OK) return rc;
        }
        // Pass 1: a weight that is read in place needs no pieces here.
        const uint64_t step = l.pack_weight ? l.piece : a.classes;
        const void* w = nullptr;
        if (l.few && (rc = few()) != SNB_OK) return rc;
        for (uint64_t v0 = 0; v0 < a.classes && !l.few; v0 += step) {
            const uint64_t n = std::min(step, a.classes - v0);
            if ((rc = weight(v0, n, &w, l.pack_hidden && v0 == 0)) != SNB_OK) return rc;
            if ((rc = tc_vocab_product(stream, logits(v0, n, w), err)) != SNB_OK) return rc;
        }
        const uint64_t blocks = (a.rows + kCombineRows - 1) / kCombineRows;
        launch_early(combine_kernel, static_cast<unsigned>(blocks), kCombineRows * kCombineLanes, stream,
                     static_cast<const float2*>(at(l.partials_at)), l.few ? l.few_blocks : (a.classes + kHalfTile - 1) / kHalfTile, a.rows, a.targets,
                     a.classes, static_cast<const float*>(at(l.target_at)), exact_logit(), a.losses,
                     l.gradients ? static_cast<float2*>(at(l.stats_at)) : nullptr, a.loss_sum);
        if ((rc = launched("combine_kernel launch", err)) != SNB_OK) return rc;
        if (a.loss_sum != nullptr && blocks > 1) {
            launch_early(loss_sum_kernel, 1, 1024, stream, a.losses, a.rows, a.loss_sum);
            if ((rc = launched("loss_sum_kernel launch", err)) != SNB_OK) return rc;
        }
        if (!l.gradients) return SNB_OK;
        // Pass 2. With one piece the packed weight is still there.
        for (uint64_t v0 = 0; v0 < a.classes; v0 += l.piece) {
            const uint64_t n = std::min(l.piece, a.classes - v0);
            if ((l.pieces > 1 || !l.pack_weight) && (rc = weight(v0, n, &w)) != SNB_OK) return rc;
            VocabProduct v = logits(v0, n, w);
            v.grad = at(l.p_at);
            v.grad_low = const_cast<void*>(grad_part().low);
            v.grad_ld = l.grad_ld;
            if ((rc = tc_vocab_product(stream, v, err)) != SNB_OK) return rc;
            if (a.weight_grad != nullptr && (rc = weight_grad(v0, n)) != SNB_OK) return rc;
            if (a.hidden_grad != nullptr && (rc = hidden_grad(v0, n, w)) != SNB_OK) return rc;
        }
        if (a.hidden_grad == nullptr || l.hidden_grad_direct) return SNB_OK;
        return store(at(l.dh_at), l.seg, a.hidden_grad, a.hidden_grad_type, a.width, a.rows, a.width, false);
    }
};

}  // namespace

bool vocab_loss_few_rows(const snb_vocabulary_loss_args& a) { return few_rows(a); }

int vocab_loss_workspace(const snb_vocabulary_loss_args& a, uint64_t* bytes, std::string* err) {
    DeviceInfo dev{};
    const int rc = a.rows == 0 ? SNB_OK : current_device_info(&dev, err);
    if (rc == SNB_OK) *bytes = layout_of(a, dev.sm_count).bytes;
    return rc;
}

int vocab_loss_launch(cudaStream_t stream, const snb_vocabulary_loss_args& a, bool deterministic, int sm_budget,
                      std::string* err) {
    if (a.rows == 0) {
        // No row: the sum and an overwritten weight gradient are zero.
        cudaError_t e = a.loss_sum != nullptr ? cudaMemsetAsync(a.loss_sum, 0, sizeof(float), stream) : cudaSuccess;
        if (e == cudaSuccess && a.weight_grad != nullptr && a.accumulate == 0)
            e = cudaMemsetAsync(a.weight_grad, 0, a.classes * a.width * (a.weight_grad_type == SNB_TYPE_BF16 ? 2 : 4),
                                stream);
        if (e == cudaSuccess) return SNB_OK;
        *err = cuda_message("cudaMemsetAsync(vocabulary loss of no rows)", e);
        return SNB_ERR_CUDA;
    }
    DeviceInfo dev;
    const int rc = current_device_info(&dev, err);
    if (rc != SNB_OK) return rc;
    const uintptr_t base = (reinterpret_cast<uintptr_t>(a.workspace) + 255) & ~uintptr_t(255);
    return Call{stream, a, layout_of(a, dev.sm_count), deterministic, sm_budget, dev.sm_count, reinterpret_cast<uint8_t*>(base), err}.run();
}

}  // namespace snb
