// layer_norm.cu — layer norm's forward and backward pass, with the reduction of the gain's and bias's gradients.
//
//   mu = mean(x),  s = 1 / sqrt(mean((x - mu)^2) + epsilon),  y = (x - mu) s g + b                       (each row)
//   n = (x - mu) s,  d = dy g:  dx = s (d - mean(d) - n mean(d n));  dg = sum_rows dy n,  db = sum_rows dy
//
// Both passes are bound by memory (x and y once; x, dy and dx once), so a row is read once and held in registers: by a
// warp up to 1,024 columns, else by a block (Shape below). The variance is taken from the deviations, not from the
// squares, whose difference would lose what a mean far from zero leaves. The backward pass runs a fixed grid whose warps
// or blocks walk over the rows; each thread always has the same columns, so it keeps their dg and db sums in registers, and a second kernel adds the grid's sums in a fixed order (no
// atomics: gradients are the same from run to run). Rows too long for that are read again instead (the wide kernels).
// All sums are f32.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "internal.h"

namespace snb {
namespace {

constexpr int kWarpsPerBlock = 8;

// One thread's 8 elements of a row: as they lie in memory (VEC: 16 bytes of bf16 or 32 of f32), or read one by one.
struct Raw {
    uint32_t w[8];
};

// Column of element e of piece v of thread t. VEC: 8 consecutive columns a thread (one or two 16-byte accesses); else
// neighbouring threads take neighbouring columns, which coalesces single elements of rows that start anywhere.
template <int T, bool VEC>
__device__ __forceinline__ int64_t column(int t, int v, int e) {
    return VEC ? static_cast<int64_t>(v * T + t) * 8 + e : static_cast<int64_t>(v * 8 + e) * T + t;
}

template <int T, bool VEC, bool BF16>
__device__ __forceinline__ Raw load_piece(const void* row, int t, int v, int64_t cols) {
    Raw r;
    if constexpr (VEC) {
        const int64_t c = column<T, true>(t, v, 0);
        if (c < cols) {
            if constexpr (BF16) {
                const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + c);
                r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
            } else {
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const float*>(row) + c);
                const uint4 a = src[0], b = src[1];
                r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
                r.w[4] = b.x; r.w[5] = b.y; r.w[6] = b.z; r.w[7] = b.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < (BF16 ? 4 : 8); ++e) r.w[e] = 0;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int64_t c = column<T, false>(t, v, e);
            if (BF16) r.w[e] = c < cols ? static_cast<uint32_t>(static_cast<const uint16_t*>(row)[c]) << 16 : 0;
            else r.w[e] = c < cols ? static_cast<const uint32_t*>(row)[c] : 0;
        }
    }
    return r;
}

template <bool VEC, bool BF16>
__device__ __forceinline__ float value(const Raw& r, int e) {
    if constexpr (VEC && BF16)
        return __uint_as_float(e & 1 ? r.w[e >> 1] & 0xFFFF0000u : r.w[e >> 1] << 16);
    else
        return __uint_as_float(r.w[e]);
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int T, bool VEC>
__device__ __forceinline__ void store_piece(void* row, bool bf16, int t, int v, int64_t cols, const float (&y)[8]) {
    if constexpr (VEC) {
        const int64_t c = column<T, true>(t, v, 0);
        if (c >= cols) return;
        if (bf16) {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(row) + c) = make_uint4(
                bf16_pair(y[0], y[1]), bf16_pair(y[2], y[3]), bf16_pair(y[4], y[5]), bf16_pair(y[6], y[7]));
        } else {
            float4* dst = reinterpret_cast<float4*>(static_cast<float*>(row) + c);
            dst[0] = make_float4(y[0], y[1], y[2], y[3]);
            dst[1] = make_float4(y[4], y[5], y[6], y[7]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int64_t c = column<T, false>(t, v, e);
            if (c >= cols) continue;
            if (bf16) static_cast<uint16_t*>(row)[c] = static_cast<uint16_t>(bf16_pair(y[e], 0.0f));
            else static_cast<float*>(row)[c] = y[e];
        }
    }
}

template <int T, bool VEC>
__device__ __forceinline__ void load_params(const float* p, int t, int v, int64_t cols, float (&out)[8]) {
    const Raw r = load_piece<T, VEC, false>(p, t, v, cols);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = __uint_as_float(r.w[e]);
}

__device__ __forceinline__ float2 warp_sum2(float2 v) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, s);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, s);
    }
    return v;
}

// The sums of two values over the T threads of a row. `part` holds two sets of one pair for each warp, used in turn, so
// that one barrier a sum is enough: a set is written again only after the other set's barrier.
template <int T>
__device__ __forceinline__ float2 row_sum2(float2 v, float2 (*part)[32], int& turn) {
    v = warp_sum2(v);
    if constexpr (T > 32) {
        const int w = threadIdx.x >> 5;
        float2* set = part[turn];
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) set[w] = v;
        __syncthreads();
        v = (threadIdx.x & 31) < T / 32 ? set[threadIdx.x & 31] : make_float2(0.0f, 0.0f);
        v = warp_sum2(v);
    }
    return v;
}

__device__ __forceinline__ const void* row_of(const void* base, int64_t row, int64_t stride, bool bf16) {
    return static_cast<const uint8_t*>(base) + row * stride * (bf16 ? 2 : 4);
}
__device__ __forceinline__ void* row_of(void* base, int64_t row, int64_t stride, bool bf16) {
    return static_cast<uint8_t*>(base) + row * stride * (bf16 ? 2 : 4);
}

struct NormParams {
    int64_t rows, cols;
    const void* x;
    const void* dy;
    void* y;            // forward: the output; backward: the input gradient
    int64_t x_stride, dy_stride, y_stride;
    int32_t x_bf16, dy_bf16, y_bf16;
    const float* gain;
    const float* bias;  // or null
    float epsilon;
    float* mean;
    float* inv_std;
    float* sums;        // backward: [2, grid, cols] partial dg and db
};

// T threads a row, NV pieces of 8 elements a thread.
template <int T, int NV, bool VEC, bool XB>
__global__ void __launch_bounds__(T == 32 ? 32 * kWarpsPerBlock : T) layer_norm_kernel(const NormParams p) {
    __shared__ float2 part[2][32];
    int turn = 0;
    const int t = T == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = T == 32 ? static_cast<int64_t>(blockIdx.x) * kWarpsPerBlock + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= p.rows) return;
    const void* x = row_of(p.x, row, p.x_stride, XB);
    Raw r[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) r[v] = load_piece<T, VEC, XB>(x, t, v, p.cols);
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += value<VEC, XB>(r[v], e);
    const float mean = row_sum2<T>(make_float2(sum, 0.0f), part, turn).x / static_cast<float>(p.cols);
    float squares = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = value<VEC, XB>(r[v], e) - mean;
            squares += column<T, VEC>(t, v, e) < p.cols ? d * d : 0.0f;
        }
    const float variance = row_sum2<T>(make_float2(squares, 0.0f), part, turn).x / static_cast<float>(p.cols);
    const float inv = 1.0f / sqrtf(variance + p.epsilon);
    if (t == 0) {
        p.mean[row] = mean;
        p.inv_std[row] = inv;
    }
    void* y = row_of(p.y, row, p.y_stride, p.y_bf16);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        float g[8], b[8], out[8];
        load_params<T, VEC>(p.gain, t, v, p.cols, g);
        if (p.bias != nullptr) {
            load_params<T, VEC>(p.bias, t, v, p.cols, b);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) b[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = fmaf((value<VEC, XB>(r[v], e) - mean) * inv, g[e], b[e]);
        store_piece<T, VEC>(y, p.y_bf16, t, v, p.cols, out);
    }
}

// The backward pass on a fixed grid (see the top): block b's rows, or warps', are b, b + grid, ... . Elements past the
// row's end are zeros in x and dy, so they add nothing to any sum.
template <int T, int NV, bool VEC, bool XB, bool DB>
__global__ void __launch_bounds__(T == 32 ? 32 * kWarpsPerBlock : T, T == 32 ? 2 : 1)
    layer_norm_backward_kernel(const NormParams p) {
    extern __shared__ float column_sums[];  // T == 32: [2, cols], the block's sums
    __shared__ float2 part[2][32];
    int turn = 0;
    const int t = T == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t first = T == 32 ? static_cast<int64_t>(blockIdx.x) * kWarpsPerBlock + (threadIdx.x >> 5) : blockIdx.x;
    const int64_t step = T == 32 ? static_cast<int64_t>(gridDim.x) * kWarpsPerBlock : gridDim.x;
    const float per_column = 1.0f / static_cast<float>(p.cols);
    float dg[NV][8], db[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) dg[v][e] = db[v][e] = 0.0f;
    Raw x[NV], dy[NV];
    float mean = 0.0f, inv = 0.0f;
    auto request = [&](int64_t row) {
        const void* xr = row_of(p.x, row, p.x_stride, XB);
        const void* dr = row_of(p.dy, row, p.dy_stride, DB);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            x[v] = load_piece<T, VEC, XB>(xr, t, v, p.cols);
            dy[v] = load_piece<T, VEC, DB>(dr, t, v, p.cols);
        }
        mean = __ldg(p.mean + row);
        inv = __ldg(p.inv_std + row);
    };
    for (int64_t row = first; row < p.rows; row += step) {
        request(row);
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float g[8];
            load_params<T, VEC>(p.gain, t, v, p.cols, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float n = (value<VEC, XB>(x[v], e) - mean) * inv;
                const float o = value<VEC, DB>(dy[v], e);
                s.x += o * g[e];
                s.y += o * g[e] * n;
                db[v][e] += o;
                dg[v][e] += o * n;
            }
        }
        s = row_sum2<T>(s, part, turn);
        const float mean_d = s.x * per_column, mean_dn = s.y * per_column;
        void* out = row_of(p.y, row, p.y_stride, XB);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float g[8], dx[8];
            load_params<T, VEC>(p.gain, t, v, p.cols, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float n = (value<VEC, XB>(x[v], e) - mean) * inv;
                dx[e] = inv * (value<VEC, DB>(dy[v], e) * g[e] - mean_d - n * mean_dn);
            }
            store_piece<T, VEC>(out, XB, t, v, p.cols, dx);
        }
    }
    float* out_g = p.sums + static_cast<int64_t>(blockIdx.x) * p.cols;
    float* out_b = out_g + static_cast<int64_t>(gridDim.x) * p.cols;
    if constexpr (T == 32) {
        // The block's warps add their sums one after the other.
        for (int w = 0; w < kWarpsPerBlock; ++w) {
            if (static_cast<int>(threadIdx.x >> 5) == w) {
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int64_t c = column<T, VEC>(t, v, e);
                        if (c < p.cols) {
                            column_sums[c] = (w > 0 ? column_sums[c] : 0.0f) + dg[v][e];
                            column_sums[p.cols + c] = (w > 0 ? column_sums[p.cols + c] : 0.0f) + db[v][e];
                        }
                    }
            }
            __syncthreads();
        }
        for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
            out_g[c] = column_sums[c];
            out_b[c] = column_sums[p.cols + c];
        }
    } else {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int64_t c = column<T, VEC>(t, v, e);
                if (c < p.cols) {
                    out_g[c] = dg[v][e];
                    out_b[c] = db[v][e];
                }
            }
    }
}

// out[c] (+)= the sum of sums[0 .. parts, c], in a fixed order: a block's 32 warps take every 32nd part of 32 columns.
// blockIdx.y: 0 the gain's gradient, 1 the bias's.
__global__ void __launch_bounds__(1024) layer_norm_columns_kernel(const float* sums, int64_t parts, int64_t cols,
                                                                  float* gain_grad, float* bias_grad, int accumulate) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float* out = blockIdx.y == 0 ? gain_grad : bias_grad;
    if (out == nullptr) return;
    const float* src = sums + static_cast<int64_t>(blockIdx.y) * parts * cols;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 4
        for (int64_t k = w; k < parts; k += 32) s += __ldg(src + k * cols + c);
    }
    part[w][lane] = s;
    __syncthreads();
    if (w != 0 || c >= cols) return;
    s = 0.0f;
    for (int k = 0; k < 32; ++k) s += part[k][lane];
    out[c] = accumulate ? out[c] + s : s;
}

// Rows of any length, a block each, read three times (forward) or twice (backward).
constexpr int kWideThreads = 512;

__device__ __forceinline__ float element(const void* row, int64_t c, bool bf16) {
    return bf16 ? __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[c]) << 16)
                : static_cast<const float*>(row)[c];
}

__device__ __forceinline__ void put(void* row, int64_t c, bool bf16, float v) {
    if (bf16) static_cast<uint16_t*>(row)[c] = static_cast<uint16_t>(bf16_pair(v, 0.0f));
    else static_cast<float*>(row)[c] = v;
}

__global__ void __launch_bounds__(kWideThreads) layer_norm_wide_kernel(const NormParams p) {
    __shared__ float2 part[2][32];
    int turn = 0;
    const int64_t row = blockIdx.x;
    const void* x = row_of(p.x, row, p.x_stride, p.x_bf16);
    float sum = 0.0f;
    for (int64_t c = threadIdx.x; c < p.cols; c += kWideThreads) sum += element(x, c, p.x_bf16);
    const float mean = row_sum2<kWideThreads>(make_float2(sum, 0.0f), part, turn).x / static_cast<float>(p.cols);
    float squares = 0.0f;
    for (int64_t c = threadIdx.x; c < p.cols; c += kWideThreads) {
        const float d = element(x, c, p.x_bf16) - mean;
        squares += d * d;
    }
    const float variance = row_sum2<kWideThreads>(make_float2(squares, 0.0f), part, turn).x / static_cast<float>(p.cols);
    const float inv = 1.0f / sqrtf(variance + p.epsilon);
    if (threadIdx.x == 0) {
        p.mean[row] = mean;
        p.inv_std[row] = inv;
    }
    void* y = row_of(p.y, row, p.y_stride, p.y_bf16);
    for (int64_t c = threadIdx.x; c < p.cols; c += kWideThreads)
        put(y, c, p.y_bf16, fmaf((element(x, c, p.x_bf16) - mean) * inv, __ldg(p.gain + c),
                                 p.bias != nullptr ? __ldg(p.bias + c) : 0.0f));
}

__global__ void __launch_bounds__(kWideThreads) layer_norm_backward_wide_kernel(const NormParams p) {
    __shared__ float2 part[2][32];
    int turn = 0;
    const int64_t row = blockIdx.x;
    const void* x = row_of(p.x, row, p.x_stride, p.x_bf16);
    const void* dy = row_of(p.dy, row, p.dy_stride, p.dy_bf16);
    const float mean = __ldg(p.mean + row), inv = __ldg(p.inv_std + row);
    float2 s = make_float2(0.0f, 0.0f);
    for (int64_t c = threadIdx.x; c < p.cols; c += kWideThreads) {
        const float d = element(dy, c, p.dy_bf16) * __ldg(p.gain + c);
        s.x += d;
        s.y += d * (element(x, c, p.x_bf16) - mean) * inv;
    }
    s = row_sum2<kWideThreads>(s, part, turn);
    const float mean_d = s.x / static_cast<float>(p.cols), mean_dn = s.y / static_cast<float>(p.cols);
    void* out = row_of(p.y, row, p.y_stride, p.x_bf16);
    for (int64_t c = threadIdx.x; c < p.cols; c += kWideThreads) {
        const float n = (element(x, c, p.x_bf16) - mean) * inv;
        put(out, c, p.x_bf16, inv * (element(dy, c, p.dy_bf16) * __ldg(p.gain + c) - mean_d - n * mean_dn));
    }
}

// Their column sums: block (b, k) takes 256 columns of the rows k, k + parts, ... .
__global__ void __launch_bounds__(256) layer_norm_wide_columns_kernel(const NormParams p) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= p.cols) return;
    float dg = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const float o = element(row_of(p.dy, row, p.dy_stride, p.dy_bf16), c, p.dy_bf16);
        const float x = element(row_of(p.x, row, p.x_stride, p.x_bf16), c, p.x_bf16);
        db += o;
        dg += o * (x - __ldg(p.mean + row)) * __ldg(p.inv_std + row);
    }
    p.sums[static_cast<int64_t>(blockIdx.y) * p.cols + c] = dg;
    p.sums[static_cast<int64_t>(gridDim.y + blockIdx.y) * p.cols + c] = db;
}

// How a row is held: T threads with NV pieces of 8 elements. T = 0: not at all (the wide kernels). A warp alone needs no
// barrier, but past 1,024 columns its registers run out; blocks are as narrow as holds the row in few pieces, since
// barriers cost more the more warps meet.
struct Shape {
    int threads, pieces;
};

Shape shape_of(uint64_t cols, bool backward) {
    if (cols <= 1024) return {32, static_cast<int>((cols + 255) / 256)};
    if (cols <= 2048) return {256, 1};
    if (cols <= 4096) return {512, 1};
    if (cols <= 8192) return {512, 2};
    // The backward pass holds four values for each column of a thread's.
    if (!backward && cols <= 16384) return {1024, 2};
    if (!backward && cols <= 32768) return {1024, 4};
    return {0, 0};
}

// Blocks of the backward pass, which is also how many partial sums there are.
uint64_t backward_grid(uint64_t rows, uint64_t cols, int sms) {
    const Shape s = shape_of(cols, true);
    if (s.threads == 0) return std::min<uint64_t>(rows, 64);
    if (s.threads == 32) return std::min<uint64_t>((rows + kWarpsPerBlock - 1) / kWarpsPerBlock, 2ull * sms);
    return std::min<uint64_t>(rows, (s.threads == 256 ? 3ull : s.pieces == 1 ? 2ull : 1ull) * sms);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int launched(const char* what, std::string* err) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return SNB_OK;
    *err = cuda_message(what, e);
    return SNB_ERR_CUDA;
}

template <int T, int NV, bool VEC>
void forward_typed(const NormParams& p, unsigned grid, cudaStream_t s) {
    const int threads = T == 32 ? 32 * kWarpsPerBlock : T;
    if (p.x_bf16) layer_norm_kernel<T, NV, VEC, true><<<grid, threads, 0, s>>>(p);
    else layer_norm_kernel<T, NV, VEC, false><<<grid, threads, 0, s>>>(p);
}

template <int T, int NV>
void forward_shaped(const NormParams& p, bool vec, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>(T == 32 ? (p.rows + kWarpsPerBlock - 1) / kWarpsPerBlock : p.rows);
    if (vec) forward_typed<T, NV, true>(p, grid, s);
    else forward_typed<T, NV, false>(p, grid, s);
}

template <int T, int NV, bool VEC>
void backward_typed(const NormParams& p, unsigned grid, cudaStream_t s) {
    const int threads = T == 32 ? 32 * kWarpsPerBlock : T;
    const size_t smem = T == 32 ? 2 * p.cols * sizeof(float) : 0;
    if (p.x_bf16 && p.dy_bf16) layer_norm_backward_kernel<T, NV, VEC, true, true><<<grid, threads, smem, s>>>(p);
    else if (p.x_bf16) layer_norm_backward_kernel<T, NV, VEC, true, false><<<grid, threads, smem, s>>>(p);
    else if (p.dy_bf16) layer_norm_backward_kernel<T, NV, VEC, false, true><<<grid, threads, smem, s>>>(p);
    else layer_norm_backward_kernel<T, NV, VEC, false, false><<<grid, threads, smem, s>>>(p);
}

template <int T, int NV>
void backward_shaped(const NormParams& p, bool vec, unsigned grid, cudaStream_t s) {
    if (vec) backward_typed<T, NV, true>(p, grid, s);
    else backward_typed<T, NV, false>(p, grid, s);
}

NormParams params_of(const snb_layer_norm_args& a) {
    NormParams p{};
    p.rows = static_cast<int64_t>(a.rows);
    p.cols = static_cast<int64_t>(a.cols);
    p.x = a.input;
    p.x_stride = static_cast<int64_t>(a.input_stride);
    p.x_bf16 = a.input_type == SNB_TYPE_BF16;
    p.gain = a.gain;
    p.bias = a.bias;
    p.epsilon = a.epsilon;
    p.mean = a.mean;
    p.inv_std = a.inv_std;
    return p;
}

// Whether a tensor's rows can be read 8 elements at a time.
bool vectors(const void* base, uint64_t stride, uint64_t cols, int type) {
    return aligned16(base) && cols % 8 == 0 && stride * (type == SNB_TYPE_BF16 ? 2 : 4) % 16 == 0;
}

}  // namespace

int layer_norm_workspace(uint64_t rows, uint64_t cols, uint64_t* bytes, std::string* err) {
    DeviceInfo dev;
    const int rc = current_device_info(&dev, err);
    if (rc != SNB_OK) return rc;
    *bytes = 2 * backward_grid(rows, cols, dev.sm_count) * cols * sizeof(float);
    return SNB_OK;
}

int layer_norm_forward_launch(cudaStream_t s, const snb_layer_norm_args& a, std::string* err) {
    if (a.rows == 0) return SNB_OK;
    NormParams p = params_of(a);
    p.y = a.output;
    p.y_stride = static_cast<int64_t>(a.output_stride);
    p.y_bf16 = a.output_type == SNB_TYPE_BF16;
    const bool vec = vectors(a.input, a.input_stride, a.cols, a.input_type) &&
                     vectors(a.output, a.output_stride, a.cols, a.output_type) && aligned16(a.gain) && aligned16(a.bias);
    const Shape shape = shape_of(a.cols, false);
    switch (shape.threads * 8 + shape.pieces) {
        case 32 * 8 + 1: forward_shaped<32, 1>(p, vec, s); break;
        case 32 * 8 + 2: forward_shaped<32, 2>(p, vec, s); break;
        case 32 * 8 + 3: forward_shaped<32, 3>(p, vec, s); break;
        case 32 * 8 + 4: forward_shaped<32, 4>(p, vec, s); break;
        case 256 * 8 + 1: forward_shaped<256, 1>(p, vec, s); break;
        case 512 * 8 + 1: forward_shaped<512, 1>(p, vec, s); break;
        case 512 * 8 + 2: forward_shaped<512, 2>(p, vec, s); break;
        case 1024 * 8 + 2: forward_shaped<1024, 2>(p, vec, s); break;
        case 1024 * 8 + 4: forward_shaped<1024, 4>(p, vec, s); break;
        default: layer_norm_wide_kernel<<<static_cast<unsigned>(a.rows), kWideThreads, 0, s>>>(p); break;
    }
    return launched("layer_norm_kernel launch", err);
}

int layer_norm_backward_launch(cudaStream_t s, const snb_layer_norm_args& a, std::string* err) {
    if (a.rows == 0) {
        if (a.accumulate) return SNB_OK;
        cudaError_t e = cudaMemsetAsync(a.gain_grad, 0, a.cols * sizeof(float), s);
        if (e == cudaSuccess && a.bias_grad != nullptr) e = cudaMemsetAsync(a.bias_grad, 0, a.cols * sizeof(float), s);
        if (e == cudaSuccess) return SNB_OK;
        *err = cuda_message("cudaMemsetAsync(layer norm gradients of no rows)", e);
        return SNB_ERR_CUDA;
    }
    DeviceInfo dev;
    int rc = current_device_info(&dev, err);
    if (rc != SNB_OK) return rc;
    NormParams p = params_of(a);
    p.dy = a.output_grad;
    p.dy_stride = static_cast<int64_t>(a.output_grad_stride);
    p.dy_bf16 = a.output_grad_type == SNB_TYPE_BF16;
    p.y = a.input_grad;
    p.y_stride = static_cast<int64_t>(a.input_grad_stride);
    p.y_bf16 = p.x_bf16;
    p.sums = static_cast<float*>(a.workspace);
    const bool vec = vectors(a.input, a.input_stride, a.cols, a.input_type) &&
                     vectors(a.output_grad, a.output_grad_stride, a.cols, a.output_grad_type) &&
                     vectors(a.input_grad, a.input_grad_stride, a.cols, a.input_type) && aligned16(a.gain);
    const unsigned grid = static_cast<unsigned>(backward_grid(a.rows, a.cols, dev.sm_count));
    const Shape shape = shape_of(a.cols, true);
    switch (shape.threads * 8 + shape.pieces) {
        case 32 * 8 + 1: backward_shaped<32, 1>(p, vec, grid, s); break;
        case 32 * 8 + 2: backward_shaped<32, 2>(p, vec, grid, s); break;
        case 32 * 8 + 3: backward_shaped<32, 3>(p, vec, grid, s); break;
        case 32 * 8 + 4: backward_shaped<32, 4>(p, vec, grid, s); break;
        case 256 * 8 + 1: backward_shaped<256, 1>(p, vec, grid, s); break;
        case 512 * 8 + 1: backward_shaped<512, 1>(p, vec, grid, s); break;
        case 512 * 8 + 2: backward_shaped<512, 2>(p, vec, grid, s); break;
        default:
            // The columns first: the input gradient may overwrite the output gradient.
            layer_norm_wide_columns_kernel<<<dim3(static_cast<unsigned>((a.cols + 255) / 256), grid), 256, 0, s>>>(p);
            if ((rc = launched("layer_norm_wide_columns_kernel launch", err)) != SNB_OK) return rc;
            layer_norm_backward_wide_kernel<<<static_cast<unsigned>(a.rows), kWideThreads, 0, s>>>(p);
            break;
    }
    if ((rc = launched("layer_norm_backward_kernel launch", err)) != SNB_OK) return rc;
    layer_norm_columns_kernel<<<dim3(static_cast<unsigned>((a.cols + 31) / 32), 2), 1024, 0, s>>>(
        p.sums, grid, p.cols, a.gain_grad, a.bias_grad, a.accumulate != 0);
    return launched("layer_norm_columns_kernel launch", err);
}

}  // namespace snb
