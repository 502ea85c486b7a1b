// layer_norm.cu — layer norm's forward and backward pass, with the reduction of the gain's and bias's gradients.
//
//   mu = mean(x),  s = 1 / sqrt(mean((x - mu)^2) + epsilon),  y = (x - mu) s g + b                       (each row)
//   n = (x - mu) s,  d = dy g:  dx = s (d - mean(d) - n mean(d n));  dg = sum_rows dy n,  db = sum_rows dy
//
// Both passes are bound by memory (x and y once; x, dy and dx once), so a row is read once, asynchronously into shared
// memory, several rows ahead of the one at hand, and held in registers by a warp or, if long, by a block (Shape below). A
// fixed grid walks over the rows: the gain and bias stay in registers, and in the backward pass so do each thread's sums
// of dg and db, since it always has the same columns. A second kernel adds the grid's sums in a fixed order (no atomics:
// gradients are the same from run to run). The variance is taken from the deviations, not from the squares, whose
// difference would lose what a mean far from zero leaves. Rows too long for registers are read again instead (the wide
// kernels). All sums are f32.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>

#include "internal.h"

namespace snb {
namespace {

constexpr int kWarpsPerBlock = 8;

// Copies from global to shared memory that run on while their thread computes. A thread waits for its own copies only;
// what other threads copied it sees after a barrier.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// The next kernel of the stream may be scheduled from here on / waits here for this one (programmatic launch).
__device__ __forceinline__ void allow_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float bf16_value(uint32_t h) { return __uint_as_float(h << 16); }

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Which columns a thread has. G = 8 or 4: groups of G consecutive ones, 16 bytes of the widest type of the call, so that
// every access of a warp is contiguous; G = 1: single ones, for rows that start anywhere.
template <int T, int G>
__device__ __forceinline__ int column(int t, int e) {
    return (e / G * T + t) * G + e % G;
}

// Elements are kept in pairs (2k, 2k + 1) for the packed f32x2 arithmetic, which halves the instructions that would
// otherwise bind these kernels before memory does.
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 minus(float2 a, float b) { return __fadd2_rn(a, both(-b)); }

__device__ __forceinline__ const uint8_t* row_of(const void* base, int64_t row, int64_t stride, bool bf16) {
    return static_cast<const uint8_t*>(base) + row * stride * (bf16 ? 2 : 4);
}
__device__ __forceinline__ uint8_t* row_of(void* base, int64_t row, int64_t stride, bool bf16) {
    return static_cast<uint8_t*>(base) + row * stride * (bf16 ? 2 : 4);
}

// Bytes of a row in shared memory. G = 1 has room for every element of its threads, so that reading one needs no test for
// the row's end, and keeps the row's position within 16 bytes, hence 16 bytes more.
__host__ __device__ constexpr int64_t slot_bytes(int64_t elements, bool bf16, bool groups) {
    return elements * (bf16 ? 2 : 4) + (groups ? 0 : 16);
}

// Where a row starts within 16 bytes, in global and in shared memory.
__device__ __forceinline__ int phase_of(const uint8_t* row) { return static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15); }

// The T threads that share a row copy it to `slot`. Groups: each thread its own, which it alone will read. Singles: the
// 16-byte pieces that lie in the row, one after the other; the up to 15 bytes before and after them go through a register
// of the first threads (`edge`, put in place by place_edge) so that nothing outside the row is read.
template <int T, int NE, int G, bool BF16>
__device__ __forceinline__ void request_row(const uint8_t* row, uint8_t* to, int t, int cols, uint32_t& edge) {
    constexpr int ES = BF16 ? 2 : 4;
    const uint32_t slot = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    if constexpr (G > 1) {
#pragma unroll
        for (int e = 0; e < NE; e += G) {
            const int c = column<T, G>(t, e);
            if (c < cols) copy_async<G * ES == 8 ? 8 : 16>(slot + c * ES, row + c * ES);
            if (G * ES == 32 && c < cols) copy_async<16>(slot + c * ES + 16, row + c * ES + 16);
        }
    } else {
        const int phase = phase_of(row);
        const int bytes = cols * ES;
        const int head = min((16 - phase) & 15, bytes);
        const int pieces = (bytes - head) / 16;
#pragma unroll
        for (int i = 0; i < (NE * ES + 15) / 16; ++i) {
            const int k = t + i * T;
            if (k < pieces) copy_async<16>(slot + phase + head + 16 * k, row + head + 16 * k);
        }
        // Element t of the edges: `head` bytes in front, then what follows the pieces.
        if (t * ES < 32) {
            const int at = t * ES < head ? t * ES : t * ES + 16 * pieces;
            if (at < bytes)
                edge = BF16 ? *reinterpret_cast<const uint16_t*>(row + at) : *reinterpret_cast<const uint32_t*>(row + at);
        }
    }
}

// Also clears what is read of the 16 bytes past the row's end, which hold what an earlier row at another position left.
template <int ELEMENTS, bool BF16>
__device__ __forceinline__ void place_edge(int phase, uint8_t* slot, int t, int cols, uint32_t edge) {
    constexpr int ES = BF16 ? 2 : 4;
    if (t * ES >= 48) return;
    const int bytes = cols * ES;
    const int head = min((16 - phase) & 15, bytes);
    const int at = t * ES < head ? t * ES : t * ES + (bytes - head) / 16 * 16;
    if (at >= min(bytes + 16, ELEMENTS * ES)) return;
    const uint32_t v = at < bytes ? edge : 0;
    if (BF16) *reinterpret_cast<uint16_t*>(slot + phase + at) = static_cast<uint16_t>(v);
    else *reinterpret_cast<uint32_t*>(slot + phase + at) = v;
}

// Fills a ring with zeros, which is what stays past the rows' ends.
__device__ __forceinline__ void clear(uint8_t* ring, int bytes) {
    for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<uint4*>(ring + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
}

// A thread's elements of a row from shared memory. (Groups: volatile reads, each behind its test, so that the compiler
// does not move all of them up and spill what they would hold: 94 us against 55 us for the backward pass of 65,536 x 768.)
template <int T, int NE, int G, bool BF16>
__device__ __forceinline__ void read_row(int phase, const uint8_t* slot, int t, int cols, float2 (&v)[NE / 2]) {
    constexpr int ES = BF16 ? 2 : 4;
    if constexpr (G > 1) {
        constexpr int PER = G * ES == 8 ? 4 : 16 / ES;  // elements of one access
        const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(slot)) + t * G * ES;
#pragma unroll
        for (int e = 0; e < NE; e += PER) {
            const uint32_t at = mine + (e / G * T * G + e % G) * ES;
            uint32_t w[4] = {0, 0, 0, 0};
            if (column<T, G>(t, e) < cols) {
                if constexpr (G * ES == 8)
                    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
                else
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
            }
#pragma unroll
            for (int k = 0; k < PER / 2; ++k)
                v[e / 2 + k] = BF16 ? make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xFFFF0000u))
                                    : make_float2(__uint_as_float(w[(2 * k) & 3]), __uint_as_float(w[(2 * k + 1) & 3]));
        }
    } else {
        const uint8_t* mine = slot + phase + t * ES;
        float one[NE];
#pragma unroll
        for (int e = 0; e < NE; ++e)
            one[e] = BF16 ? bf16_value(*reinterpret_cast<const uint16_t*>(mine + e * T * ES))
                          : *reinterpret_cast<const float*>(mine + e * T * ES);
#pragma unroll
        for (int k = 0; k < NE / 2; ++k) v[k] = make_float2(one[2 * k], one[2 * k + 1]);
    }
}

template <int T, int NE, int G>
__device__ __forceinline__ void load_params(const float* p, int t, int cols, float2 (&v)[NE / 2]) {
#pragma unroll
    for (int e = 0; e < NE; e += G == 1 ? 2 : 4) {
        const int c = column<T, G>(t, e);
        if constexpr (G == 1) {
            const int next = column<T, 1>(t, e + 1);
            v[e / 2] = make_float2(c < cols ? __ldg(p + c) : 0.0f, next < cols ? __ldg(p + next) : 0.0f);
        } else {
            const float4 q = c < cols ? __ldg(reinterpret_cast<const float4*>(p + c)) : make_float4(0, 0, 0, 0);
            v[e / 2] = make_float2(q.x, q.y);
            v[e / 2 + 1] = make_float2(q.z, q.w);
        }
    }
}

template <int T, int NE, int G>
__device__ __forceinline__ void store_row(uint8_t* row, bool bf16, int t, int cols, const float2 (&y)[NE / 2]) {
    if constexpr (G == 1) {
        const int left = cols - t;
        if (bf16) {
            uint16_t* mine = reinterpret_cast<uint16_t*>(row) + t;
#pragma unroll
            for (int e = 0; e < NE; ++e)
                if (e * T < left) mine[e * T] = static_cast<uint16_t>(bf16_pair(e & 1 ? y[e / 2].y : y[e / 2].x, 0.0f));
        } else {
            float* mine = reinterpret_cast<float*>(row) + t;
#pragma unroll
            for (int e = 0; e < NE; ++e)
                if (e * T < left) mine[e * T] = e & 1 ? y[e / 2].y : y[e / 2].x;
        }
    } else {
#pragma unroll
        for (int e = 0; e < NE; e += G) {
            const int c = column<T, G>(t, e);
            if (c >= cols) continue;
            const float2* q = y + e / 2;
            if (!bf16) {
#pragma unroll
                for (int k = 0; k < G; k += 4)
                    *reinterpret_cast<float4*>(row + (c + k) * 4) =
                        make_float4(q[k / 2].x, q[k / 2].y, q[k / 2 + 1].x, q[k / 2 + 1].y);
            } else if constexpr (G == 8) {
                *reinterpret_cast<uint4*>(row + c * 2) = make_uint4(bf16_pair(q[0].x, q[0].y), bf16_pair(q[1].x, q[1].y),
                                                                    bf16_pair(q[2].x, q[2].y), bf16_pair(q[3].x, q[3].y));
            } else {
                *reinterpret_cast<uint2*>(row + c * 2) = make_uint2(bf16_pair(q[0].x, q[0].y), bf16_pair(q[1].x, q[1].y));
            }
        }
    }
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

// The same of one value in both halves (their sum over the threads).
template <int T>
__device__ __forceinline__ float row_sum(float2 v, float2 (*part)[32], int& turn) {
    float one = v.x + v.y;
    if constexpr (T == 32) {
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) one += __shfl_xor_sync(0xffffffffu, one, s);
        return one;
    } else {
        return row_sum2<T>(make_float2(one, 0.0f), part, turn).x;
    }
}

template <int T>
__device__ __forceinline__ void row_barrier() {
    if constexpr (T == 32) __syncwarp();
    else __syncthreads();
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
    int32_t depth;      // rows in flight
};

// Both kernels: T threads a row, NE elements a thread, `depth` rows in flight in shared memory (a ring for each warp when
// T is 32, else one of the block), rows first, first + step, ... . kMaxDepth bounds the waits' immediate operands.
//
// Measured. Forward, 65,536 x 768 bf16 (202 MB, 31 us at the copy rate): 33 us; f32 (403 MB, 62 us): 73 us a call, backward
// 105 us (605 MB, 94 us); one row of 768 f32: 2.4 us, a launch.
// Backward, 65,536 x 768 bf16 (302 MB, 47 us at the copy rate): 51 us; 4,096 x 256 f32: 4.1 us; 3,001 x 5,003 bf16, whose
// rows start off every boundary (90 MB, 14 us): 29 us, bound by the chain of each row, which two barriers interrupt, and by
// its single-element reads from shared memory.
constexpr int kMaxDepth = 4;

__device__ __forceinline__ void wait_for_row(int depth) {
    // All but the newest depth - 1 groups of copies have arrived.
    if (depth >= 4) copies_wait<3>();
    else if (depth == 3) copies_wait<2>();
    else if (depth == 2) copies_wait<1>();
    else copies_wait<0>();
}

template <int T, int NE, int G, bool XB>
__global__ void __launch_bounds__(T == 32 ? 32 * kWarpsPerBlock : T, T == 32 ? 2 : 1) layer_norm_kernel(const NormParams p) {
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float2 part[2][32];
    int turn = 0;
    const int t = T == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int warp = threadIdx.x >> 5;
    const int64_t first = T == 32 ? static_cast<int64_t>(blockIdx.x) * kWarpsPerBlock + warp : blockIdx.x;
    const int64_t step = T == 32 ? static_cast<int64_t>(gridDim.x) * kWarpsPerBlock : gridDim.x;
    const int cols = static_cast<int>(p.cols);
    constexpr int slot = static_cast<int>(slot_bytes(T * NE, XB, G > 1));
    if constexpr (G == 1) clear(ring, slot * p.depth * (T == 32 ? kWarpsPerBlock : 1));
    uint8_t* base = ring + (T == 32 ? warp * p.depth * slot : 0);
    uint32_t edge = 0;
    int phase = 0;  // of the row asked for last
    int64_t ahead = first;
    const int64_t x_step = step * p.x_stride * (XB ? 2 : 4), y_step = step * p.y_stride * (p.y_bf16 ? 2 : 4);
    const uint8_t* x = row_of(p.x, first, p.x_stride, XB);
    uint8_t* y = row_of(p.y, first, p.y_stride, p.y_bf16);
    int in = 0, out = 0;
    auto request = [&]() {
        if (ahead < p.rows) {
            request_row<T, NE, G, XB>(x, base + in * slot, t, cols, edge);
            if (G == 1) phase = phase_of(x);
        }
        copies_commit();
        ahead += step;
        x += x_step;
        if (++in == p.depth) in = 0;
    };
    // Singles' edges pass through one register: their rows are requested one ahead only.
    for (int k = 0; k < (G > 1 ? p.depth - 1 : 1); ++k) request();
    float2 gain[NE / 2], bias[NE / 2];
    load_params<T, NE, G>(p.gain, t, cols, gain);
    if (p.bias != nullptr) {
        load_params<T, NE, G>(p.bias, t, cols, bias);
    } else {
#pragma unroll
        for (int k = 0; k < NE / 2; ++k) bias[k] = both(0.0f);
    }
    const float columns = static_cast<float>(cols);
    for (int64_t row = first; row < p.rows; row += step) {
        const int here = phase;
        if constexpr (G > 1) {
            request();
            wait_for_row(p.depth);
        } else {
            copies_wait<0>();
            place_edge<T * NE, XB>(here, base + out * slot, t, cols, edge);
            row_barrier<T>();
            request();
        }
        float2 v[NE / 2];
        read_row<T, NE, G, XB>(here, base + out * slot, t, cols, v);
        if (++out == p.depth) out = 0;
        float2 sum = both(0.0f);
#pragma unroll
        for (int k = 0; k < NE / 2; ++k) sum = __fadd2_rn(sum, v[k]);
        const float mean = row_sum<T>(sum, part, turn) / columns;
        float2 squares = both(0.0f);
#pragma unroll
        for (int k = 0; k < NE / 2; ++k) {
            v[k] = minus(v[k], mean);
            // (Groups lie in the row or past it as a whole; singles each by themselves.)
            const bool in_row = column<T, G>(t, 2 * k) < cols;
            const bool next_in_row = G > 1 ? in_row : column<T, G>(t, 2 * k + 1) < cols;
            const float2 live = make_float2(in_row ? v[k].x : 0.0f, next_in_row ? v[k].y : 0.0f);
            squares = __ffma2_rn(live, live, squares);
        }
        const float variance = row_sum<T>(squares, part, turn) / columns;
        const float inv = 1.0f / sqrtf(variance + p.epsilon);
        if (t == 0) {
            p.mean[row] = mean;
            p.inv_std[row] = inv;
        }
#pragma unroll
        for (int k = 0; k < NE / 2; ++k) v[k] = __ffma2_rn(__fmul2_rn(v[k], both(inv)), gain[k], bias[k]);
        store_row<T, NE, G>(y, p.y_bf16, t, cols, v);
        y += y_step;
    }
}

// With 24 elements a thread the gain's registers would be the ones too many in the backward pass: the threads read it from
// shared memory, a copy in their order.
template <int NE>
constexpr bool kSharedGain = NE >= 24;

constexpr int64_t kPartBytes = 2 * 32 * sizeof(float2);  // of row_sum2

// Elements past the row's end are zeros in dy and the gain, so they add nothing to any sum.
template <int T, int NE, int G, bool XB, bool DB>
__global__ void __launch_bounds__(T == 32 ? 32 * kWarpsPerBlock : T, T <= 256 ? 2 : 1)
    layer_norm_backward_kernel(const NormParams p) {
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float2 part[2][32];
    allow_next_kernel();
    int turn = 0;
    const int t = T == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int warp = threadIdx.x >> 5;
    const int64_t first = T == 32 ? static_cast<int64_t>(blockIdx.x) * kWarpsPerBlock + warp : blockIdx.x;
    const int64_t step = T == 32 ? static_cast<int64_t>(gridDim.x) * kWarpsPerBlock : gridDim.x;
    const int cols = static_cast<int>(p.cols);
    constexpr int x_slot = static_cast<int>(slot_bytes(T * NE, XB, G > 1));
    constexpr int slot = x_slot + static_cast<int>(slot_bytes(T * NE, DB, G > 1));
    if constexpr (G == 1) clear(ring, slot * p.depth * (T == 32 ? kWarpsPerBlock : 1));
    uint8_t* base = ring + (T == 32 ? warp * p.depth * slot : 0);
    uint32_t x_edge = 0, dy_edge = 0;
    int x_phase = 0, dy_phase = 0;              // of the row asked for last
    float mean_ahead = 0.0f, inv_ahead = 0.0f;  // of the next row
    int64_t ahead = first;
    const int64_t x_step = step * p.x_stride * (XB ? 2 : 4), dy_step = step * p.dy_stride * (DB ? 2 : 4);
    const int64_t dx_step = step * p.y_stride * (XB ? 2 : 4);
    const uint8_t* x = row_of(p.x, first, p.x_stride, XB);
    const uint8_t* dy = row_of(p.dy, first, p.dy_stride, DB);
    uint8_t* dx = row_of(p.y, first, p.y_stride, XB);
    int in = 0, out = 0;
    auto request = [&]() {
        if (ahead < p.rows) {
            request_row<T, NE, G, XB>(x, base + in * slot, t, cols, x_edge);
            request_row<T, NE, G, DB>(dy, base + in * slot + x_slot, t, cols, dy_edge);
            if (G == 1) {
                x_phase = phase_of(x);
                dy_phase = phase_of(dy);
            }
        }
        copies_commit();
        ahead += step;
        x += x_step;
        dy += dy_step;
        if (++in == p.depth) in = 0;
    };
    auto statistics = [&](int64_t row) {
        if (row < p.rows) {
            mean_ahead = __ldg(p.mean + row);
            inv_ahead = __ldg(p.inv_std + row);
        }
    };
    for (int k = 0; k < (G > 1 ? p.depth - 1 : 1); ++k) request();
    statistics(first);
    __shared__ float4 shared_gain[kSharedGain<NE> ? NE / 4 : 1][T];
    float2 gain[NE / 2], dg[NE / 2], db[NE / 2];
    if constexpr (kSharedGain<NE>) {
        load_params<T, NE, G>(p.gain, t, cols, gain);
        if (T > 32 || warp == 0) {
#pragma unroll
            for (int k = 0; k < NE / 4; ++k)
                shared_gain[k][t] = make_float4(gain[2 * k].x, gain[2 * k].y, gain[2 * k + 1].x, gain[2 * k + 1].y);
        }
        __syncthreads();
    } else {
        load_params<T, NE, G>(p.gain, t, cols, gain);
    }
#pragma unroll
    for (int k = 0; k < NE / 2; ++k) dg[k] = db[k] = both(0.0f);
    const float per_column = 1.0f / static_cast<float>(cols);
    for (int64_t row = first; row < p.rows; row += step) {
        const int x_here = x_phase, dy_here = dy_phase;
        uint8_t* here = base + out * slot;
        const float mean = mean_ahead, inv = inv_ahead;
        if constexpr (G > 1) {
            request();
            statistics(row + step);
            wait_for_row(p.depth);
        } else {
            // (A slot is asked for again two rows later at the earliest, behind the barrier of the row in between.)
            copies_wait<0>();
            place_edge<T * NE, XB>(x_here, here, t, cols, x_edge);
            place_edge<T * NE, DB>(dy_here, here + x_slot, t, cols, dy_edge);
            row_barrier<T>();
            request();
            statistics(row + step);
        }
        if (++out == p.depth) out = 0;
        // d = dy g of one pair of elements.
        auto gained = [&](float2 o, int k) {
            if constexpr (kSharedGain<NE>) {
                const float4 g = shared_gain[k / 2][t];
                return __fmul2_rn(o, k & 1 ? make_float2(g.z, g.w) : make_float2(g.x, g.y));
            } else {
                return __fmul2_rn(o, gain[k]);
            }
        };
        float2 sum = both(0.0f), product = both(0.0f);
        float2 n[NE / 2], d[NE / 2];
        read_row<T, NE, G, XB>(x_here, here, t, cols, n);
        read_row<T, NE, G, DB>(dy_here, here + x_slot, t, cols, d);
#pragma unroll
        for (int k = 0; k < NE / 2; ++k) {
            n[k] = __fmul2_rn(minus(n[k], mean), both(inv));
            db[k] = __fadd2_rn(db[k], d[k]);
            dg[k] = __ffma2_rn(d[k], n[k], dg[k]);
            d[k] = gained(d[k], k);
            sum = __fadd2_rn(sum, d[k]);
            product = __ffma2_rn(d[k], n[k], product);
        }
        const float2 s = row_sum2<T>(make_float2(sum.x + sum.y, product.x + product.y), part, turn);
        const float mean_d = s.x * per_column, mean_dn = s.y * per_column;
        if constexpr (kSharedGain<NE>) {
            // Held until here the row would not fit beside the column sums: it is read from shared memory again.
            read_row<T, NE, G, XB>(x_here, here, t, cols, n);
            read_row<T, NE, G, DB>(dy_here, here + x_slot, t, cols, d);
#pragma unroll
            for (int k = 0; k < NE / 2; ++k) {
                n[k] = __fmul2_rn(minus(n[k], mean), both(inv));
                d[k] = gained(d[k], k);
            }
        }
#pragma unroll
        for (int k = 0; k < NE / 2; ++k)
            d[k] = __fmul2_rn(both(inv), __ffma2_rn(n[k], both(-mean_dn), minus(d[k], mean_d)));
        store_row<T, NE, G>(dx, XB, t, cols, d);
        dx += dx_step;
    }
    float* out_g = p.sums + static_cast<int64_t>(blockIdx.x) * p.cols;
    float* out_b = out_g + static_cast<int64_t>(gridDim.x) * p.cols;
    if constexpr (T == 32) {
        // The block's warps leave their sums in the ring's memory, where they are added up in warp order.
        copies_wait<0>();
        __syncthreads();
        float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int c = column<T, G>(t, e);
            if (c < cols) {
                sums[(2 * warp) * cols + c] = e & 1 ? dg[e / 2].y : dg[e / 2].x;
                sums[(2 * warp + 1) * cols + c] = e & 1 ? db[e / 2].y : db[e / 2].x;
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * cols; c += blockDim.x) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarpsPerBlock; ++w) sum += sums[2 * w * cols + c];
            (c < cols ? out_g + c : out_b + c - cols)[0] = sum;
        }
    } else {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int c = column<T, G>(t, e);
            if (c < cols) {
                out_g[c] = e & 1 ? dg[e / 2].y : dg[e / 2].x;
                out_b[c] = e & 1 ? db[e / 2].y : db[e / 2].x;
            }
        }
    }
}

// out[c] (+)= the sum of sums[0 .. parts, c], in a fixed order: a block's 32 warps take every 32nd part of 32 columns.
// blockIdx.y: 0 the gain's gradient, 1 the bias's. Bound by the latency of its few reads: 5 to 6 us for 768 columns of 296
// parts, 8.5 us for 5,003 (12 MB). Ten reads at a time or half the warps moved the whole pass by less than 2 % either way.
__global__ void __launch_bounds__(1024) layer_norm_columns_kernel(const float* sums, int64_t parts, int64_t cols,
                                                                  float* gain_grad, float* bias_grad, int accumulate) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float* out = blockIdx.y == 0 ? gain_grad : bias_grad;
    wait_for_previous_kernel();
    if (out == nullptr) return;
    const float* src = sums + static_cast<int64_t>(blockIdx.y) * parts * cols;
    float s = 0.0f;
    if (c < cols) {
        // (Ordinary loads: the sums are still being written when this kernel starts, which rules out the read-only path.)
#pragma unroll 4
        for (int64_t k = w; k < parts; k += 32) s += src[k * cols + c];
    }
    part[w][lane] = s;
    __syncthreads();
    if (w != 0 || c >= cols) return;
    s = 0.0f;
    for (int k = 0; k < 32; ++k) s += part[k][lane];
    out[c] = accumulate ? out[c] + s : s;
}

// Rows of any length, a block each, read three times (forward) or twice (backward). What binds them is those passes, which
// mostly hit L1 and L2, element by element; they stand for rows that the shapes below have no registers for. Backward pass of
// 4,096 x 9,001 bf16: 224 us (221 MB, 34 us at the copy rate); of 4,096 x 12,288: 309 us (302 MB, 47 us).
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

// How a row is held: T threads with up to `elements` each. T = 0: not at all (the wide kernels). A warp alone needs no
// barrier, but past 1,024 columns (768 in the backward pass, which holds five values for each) its registers run out.
// Blocks are as narrow as can hold the row: what binds them is the chain of barriers and reads of a row, so two blocks of
// 256 threads on an SM, with a row each, beat one of 512 (backward pass of 3,001 x 5,003 bf16: 30 us, with 512 threads
// 46 us, with 1,024 50 us). A thread has the fewest elements that hold the row, in fours: 12 against 16 for 5,001 rows of 2,999
// columns, 41.2 against 45.3 us bf16 and 50.1 against 51.0 f32, 36.1 against 44.3 for 2,816 columns f32; 20 against 24, which
// read the row twice, for 3,401 of 4,403, 37.2 against 40.8 bf16 and 46.6 against 58.7 f32 (whole calls). Eights of bf16 round
// up to 16 and 24. Past 6,144 columns the five values a column (8,192), or the forward pass's three (16,384), are too many.
struct Shape {
    int threads, elements;
};

Shape shape_of(uint64_t cols, bool backward) {
    if (cols <= (backward ? 768 : 1024)) return {32, static_cast<int>((cols + 255) / 256) * 8};
    if (cols <= 1024) return {128, 8};
    if (cols <= 2048) return {256, 8};
    if (backward && cols <= 6144) return {256, static_cast<int>((cols + 1023) / 1024) * 4};
    if (cols <= 4096) return {512, 8};
    if (cols <= 6144) return {512, 12};
    if (cols <= 8192) return {512, 16};
    if (!backward && cols <= 16384) return {1024, 16};
    return {0, 0};
}

constexpr int64_t kRingBytes = 96 << 10;  // of a wide thread block, so that two fit on an SM

// Rows in flight: as many as kMaxDepth and the ring allow, at least two.
int depth_of(const Shape& s, int64_t row_bytes) {
    const int64_t rings = s.threads == 32 ? kWarpsPerBlock : 1;
    const int64_t bytes = s.threads == 128 ? kRingBytes / 3 : kRingBytes - (24 << 10);  // (a gain's copy takes 24 KB)
    return static_cast<int>(std::max<int64_t>(2, std::min<int64_t>(kMaxDepth, bytes / (rings * row_bytes))));
}

// Blocks of the backward pass, which is also how many partial sums there are.
uint64_t backward_grid(uint64_t rows, uint64_t cols, int sms) {
    const Shape s = shape_of(cols, true);
    if (s.threads == 0) return std::min<uint64_t>(rows, 64);
    if (s.threads == 32) return std::min<uint64_t>((rows + kWarpsPerBlock - 1) / kWarpsPerBlock, 2ull * sms);
    return std::min<uint64_t>(rows, (s.threads == 128 ? 4ull : s.threads == 256 ? 2ull : 1ull) * sms);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int launched(const char* what, std::string* err) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return SNB_OK;
    *err = cuda_message(what, e);
    return SNB_ERR_CUDA;
}

// Launches `kernel` with a ring of shared memory, always of the same size. Above 48 KB together with the kernel's `fixed`
// bytes that has to be allowed first, once on each device.
template <auto kernel>
void launch_ring(unsigned grid, int threads, int64_t smem, int64_t fixed, cudaStream_t s, const NormParams& p) {
    static std::atomic<int> allowed{-1};  // the device of the last call
    if (smem + fixed > (48 << 10)) {
        int dev = 0;
        cudaGetDevice(&dev);
        if (allowed.load(std::memory_order_relaxed) != dev &&
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) == cudaSuccess)
            allowed.store(dev, std::memory_order_relaxed);
    }
    kernel<<<grid, threads, static_cast<size_t>(smem), s>>>(p);
}

template <int T, int NE, int G>
void forward_typed(NormParams p, int sms, cudaStream_t s) {
    constexpr int threads = T == 32 ? 32 * kWarpsPerBlock : T;
    const int64_t slot = slot_bytes(T * NE, p.x_bf16 != 0, G > 1);
    p.depth = depth_of({T, NE}, slot);
    const int64_t smem = p.depth * slot * (T == 32 ? kWarpsPerBlock : 1);
    const int64_t blocks = T == 32 ? (p.rows + kWarpsPerBlock - 1) / kWarpsPerBlock : p.rows;
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(blocks, (T == 1024 ? 1ll : T == 256 ? 4ll : 2ll) * sms));
    if (p.x_bf16) {
        launch_ring<layer_norm_kernel<T, NE, G, true>>(grid, threads, smem, kPartBytes, s, p);
    } else {
        if constexpr (G != 8) launch_ring<layer_norm_kernel<T, NE, G, false>>(grid, threads, smem, kPartBytes, s, p);
    }
}

// group: the columns of 16 bytes of the call's widest type, or 1 where its rows do not allow 16-byte accesses.
template <int T, int NE>
void forward_shaped(const NormParams& p, int group, int sms, cudaStream_t s) {
    if (group == 8) forward_typed<T, (NE + 7) / 8 * 8, 8>(p, sms, s);
    else if (group == 4) forward_typed<T, NE, 4>(p, sms, s);
    else forward_typed<T, NE, 1>(p, sms, s);
}

template <int T, int NE, int G>
void backward_typed(NormParams p, unsigned grid, cudaStream_t s) {
    constexpr int threads = T == 32 ? 32 * kWarpsPerBlock : T;
    const int64_t slot = slot_bytes(T * NE, p.x_bf16 != 0, G > 1) + slot_bytes(T * NE, p.dy_bf16 != 0, G > 1);
    p.depth = depth_of({T, NE}, slot);
    // (Two rows of at least 4 bytes a column for each warp: room for the warps' column sums at the end.)
    const int64_t smem = p.depth * slot * (T == 32 ? kWarpsPerBlock : 1);
    constexpr int64_t fixed = kPartBytes + (kSharedGain<NE> ? 4 * T * NE : 16 * T);
    if (p.x_bf16 && p.dy_bf16) {
        launch_ring<layer_norm_backward_kernel<T, NE, G, true, true>>(grid, threads, smem, fixed, s, p);
    } else if constexpr (G != 8) {
        if (p.x_bf16) launch_ring<layer_norm_backward_kernel<T, NE, G, true, false>>(grid, threads, smem, fixed, s, p);
        else if (p.dy_bf16) launch_ring<layer_norm_backward_kernel<T, NE, G, false, true>>(grid, threads, smem, fixed, s, p);
        else launch_ring<layer_norm_backward_kernel<T, NE, G, false, false>>(grid, threads, smem, fixed, s, p);
    }
}

template <int T, int NE>
void backward_shaped(const NormParams& p, int group, unsigned grid, cudaStream_t s) {
    if (group == 8) backward_typed<T, (NE + 7) / 8 * 8, 8>(p, grid, s);
    else if (group == 4) backward_typed<T, NE, 4>(p, grid, s);
    else backward_typed<T, NE, 1>(p, grid, s);
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

// Whether every row of a tensor can be taken in whole 16-byte pieces.
bool pieces16(const void* base, uint64_t stride, uint64_t cols, int type) {
    const uint64_t es = type == SNB_TYPE_BF16 ? 2 : 4;
    return aligned16(base) && cols * es % 16 == 0 && stride * es % 16 == 0;
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
    DeviceInfo dev;
    const int rc = current_device_info(&dev, err);
    if (rc != SNB_OK) return rc;
    const bool whole = pieces16(a.input, a.input_stride, a.cols, a.input_type) &&
                       pieces16(a.output, a.output_stride, a.cols, a.output_type) && aligned16(a.gain) &&
                       aligned16(a.bias);
    // (An f32 output of a bf16 input keeps groups of 8: two stores of 16 bytes.)
    const int group = !whole ? 1 : p.x_bf16 ? 8 : 4;
    const Shape shape = shape_of(a.cols, false);
    switch (shape.threads * 64 + shape.elements) {
        case 32 * 64 + 8: forward_shaped<32, 8>(p, group, dev.sm_count, s); break;
        case 32 * 64 + 16: forward_shaped<32, 16>(p, group, dev.sm_count, s); break;
        case 32 * 64 + 24: forward_shaped<32, 24>(p, group, dev.sm_count, s); break;
        case 32 * 64 + 32: forward_shaped<32, 32>(p, group, dev.sm_count, s); break;
        case 256 * 64 + 8: forward_shaped<256, 8>(p, group, dev.sm_count, s); break;
        case 512 * 64 + 8: forward_shaped<512, 8>(p, group, dev.sm_count, s); break;
        case 512 * 64 + 12: forward_shaped<512, 12>(p, group, dev.sm_count, s); break;
        case 512 * 64 + 16: forward_shaped<512, 16>(p, group, dev.sm_count, s); break;
        case 1024 * 64 + 16: forward_shaped<1024, 16>(p, group, dev.sm_count, s); break;
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
    const bool whole = pieces16(a.input, a.input_stride, a.cols, a.input_type) &&
                       pieces16(a.output_grad, a.output_grad_stride, a.cols, a.output_grad_type) &&
                       pieces16(a.input_grad, a.input_grad_stride, a.cols, a.input_type) && aligned16(a.gain);
    const int group = !whole ? 1 : p.x_bf16 && p.dy_bf16 ? 8 : 4;
    const unsigned grid = static_cast<unsigned>(backward_grid(a.rows, a.cols, dev.sm_count));
    const Shape shape = shape_of(a.cols, true);
    switch (shape.threads * 64 + shape.elements) {
        case 32 * 64 + 8: backward_shaped<32, 8>(p, group, grid, s); break;
        case 32 * 64 + 16: backward_shaped<32, 16>(p, group, grid, s); break;
        case 32 * 64 + 24: backward_shaped<32, 24>(p, group, grid, s); break;
        case 128 * 64 + 8: backward_shaped<128, 8>(p, group, grid, s); break;
        case 256 * 64 + 8: backward_shaped<256, 8>(p, group, grid, s); break;
        case 256 * 64 + 12: backward_shaped<256, 12>(p, group, grid, s); break;
        case 256 * 64 + 16: backward_shaped<256, 16>(p, group, grid, s); break;
        case 256 * 64 + 20: backward_shaped<256, 20>(p, group, grid, s); break;
        case 256 * 64 + 24: backward_shaped<256, 24>(p, group, grid, s); break;
        case 512 * 64 + 16: backward_shaped<512, 16>(p, group, grid, s); break;
        default:
            // The columns first: the input gradient may overwrite the output gradient.
            layer_norm_wide_columns_kernel<<<dim3(static_cast<unsigned>((a.cols + 255) / 256), grid), 256, 0, s>>>(p);
            if ((rc = launched("layer_norm_wide_columns_kernel launch", err)) != SNB_OK) return rc;
            layer_norm_backward_wide_kernel<<<static_cast<unsigned>(a.rows), kWideThreads, 0, s>>>(p);
            break;
    }
    if ((rc = launched("layer_norm_backward_kernel launch", err)) != SNB_OK) return rc;
    // Scheduled while the grid above drains; it waits for that grid before it reads.
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((a.cols + 31) / 32), 2);
    cfg.blockDim = dim3(1024);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, layer_norm_columns_kernel, static_cast<const float*>(p.sums), static_cast<int64_t>(grid),
                       p.cols, a.gain_grad, a.bias_grad, a.accumulate != 0 ? 1 : 0);
    return launched("layer_norm_columns_kernel launch", err);
}

}  // namespace snb
