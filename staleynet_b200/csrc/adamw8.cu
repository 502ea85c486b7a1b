// adamw8.cu — an AdamW step over many tensors with both moments held in 8 bits.
//
// Moments. A block of 256 consecutive elements of a tensor shares an f32 scale S for each moment, the largest magnitude
// in the block, and each element an 8-bit code: m = sign(q) (q / 127)^2 S with q in -127 .. 127, v = (q / 255)^4 S with q
// in 0 .. 255. The levels are powers because a block's gradients differ by orders of magnitude: equal steps would leave
// nothing of the small ones, while here the steps near a value x of the block shrink like sqrt(x) and x^(3/4).
//   A value between two levels goes to the upper one with the probability that keeps its expectation, drawn from a
// caller's seed. Rounding to nearest instead would freeze v: with beta2 = 0.999 a step moves it by a thousandth, and
// neighbouring levels are 1.6 % apart or more. A v above 0 keeps at least code 1: a v of 0 next to an m that is not
// would divide that m by epsilon.
//   The random bits of elements 2i and 2i + 1 of a tensor are the halves of output first_draw + i + 1 of the reference's
// SplitMix64 (Random::new(seed), crates/staleynet-model/src/random.rs:27-50): 16 bits for each moment.
//   Everything that decides a code is made of f32 operations that are rounded one by one, so codes do not depend on the
// compiler. (It contracts packed products and sums to multiply-adds, even where both ask for their own rounding: sums of
// products are therefore scalar additions, sum_of.)
//
// Step. As the reference's (kernels/optimizer.rs:57-70) on g = gradient times the clip factor max_norm / norm; the norm is
// that of all tensors together, its squares summed in f64 in a fixed order, so steps are the same from run to run.
//
// What bounds it: memory, an element's parameter (4 bytes read, 4 written, and 2 for its bf16 copy), gradient (2 or 4,
// twice: once for the norm) and two codes (2 read, 2 written); and in the step nearly as much the issue of its
// instructions, about a hundred for an element, most of them for the two roundings.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "internal.h"

namespace snb {
namespace {

constexpr int kBlock = 256;             // elements that share a scale
constexpr int kWarps = 8;               // warps of a thread block
constexpr int kPart = kWarps * kBlock;  // elements that a thread block takes at once
constexpr int kStepBlocks = 3;          // thread blocks of the step that are resident on an SM (80 registers a thread)
constexpr int kMaxTensors = 256;        // of one launch (its table is a kernel parameter)
constexpr int kSumBlocks = 888;         // thread blocks of the norm's sum, and partial sums of one launch: six an SM (97.6
                                        // million f32 gradients: 77 us; 80 us on three an SM, 78 on eight)
constexpr uint64_t kGolden = 0x9E3779B97F4A7C15ull;

// How a launch's grid shares the parts of its tensors: a contiguous run each, `longer` blocks one part more than the rest.
// The tensor in which each run begins comes from the host, since a search through the table in every block would wait for
// one uncached constant after the other. (Blocks that took every gridDim.x-th piece of 8,192 elements, with that search at
// each, were slower: 434 us for a step on 97.6 million elements that takes 418 us here.)
constexpr int kMaxGrid = 2048;
struct Shares {
    int64_t each, longer;
    uint8_t first_tensor[kMaxGrid];
};

struct Table {
    int32_t n;
    Shares shares;
    snb_adamw8_tensor t[kMaxTensors];
    int64_t part_start[kMaxTensors + 1];
};
static_assert(sizeof(Table) < 32000, "kernel parameters");

// A thread block's share, through which it walks tensor by tensor.
struct Share {
    int64_t part, end;  // the run's next part and its end
    int tensor;         // that holds `part`
};

template <typename T>
__device__ __forceinline__ Share share_of(const T& m) {
    const int64_t b = blockIdx.x, part = b * m.shares.each + min(b, m.shares.longer);
    return {part, part + m.shares.each + (b < m.shares.longer ? 1 : 0), m.shares.first_tensor[b]};
}

// The end of the run within its current tensor, in elements.
template <typename T>
__device__ __forceinline__ int64_t end_of(const T& m, const Share& s) {
    return min((s.end - m.part_start[s.tensor]) * kPart, static_cast<int64_t>(m.t[s.tensor].count));
}

template <typename T>
__device__ __forceinline__ void next_tensor(const T& m, Share& s) {
    s.part = m.part_start[++s.tensor];
    while (s.part < s.end && m.part_start[s.tensor + 1] == s.part) ++s.tensor;
}

__device__ __forceinline__ float bf16_value(uint16_t h) { return __uint_as_float(static_cast<uint32_t>(h) << 16); }

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ bool multiple(const void* p, uint32_t n) {
    return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

// The arithmetic goes on pairs of elements with packed f32x2 instructions: a step costs about as many instructions as its
// memory traffic leaves time for. Their constants come as pairs from the kernel's parameters, where an instruction can
// take them from; pairs of literals would be assembled in registers at each use.
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ float2 sum_of(float2 a, float2 b) { return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)); }

struct Constants {
    float2 first, second;       // 1 / 127^2, 1 / 255^2
    float2 integer, code, one;  // -2^23, -2^23 - 128, 1
    float2 round;               // 2^23
    float2 guess1, guess2;      // 127 and 255, less 2^-20 of them
    float2 unit, unit_shift;    // 2^-16, 2^-17 - 128
};

// The share of its block's scale that a magnitude code stands for.
__device__ __forceinline__ float2 first_level(float2 q, const Constants& k) {
    return __fmul2_rn(__fmul2_rn(q, q), k.first);
}
__device__ __forceinline__ float2 second_level(float2 q, const Constants& k) {
    const float2 s = __fmul2_rn(__fmul2_rn(q, q), k.second);
    return __fmul2_rn(s, s);
}

__device__ __forceinline__ float sqrt_fast(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The larger of two magnitudes, NaN if either is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(fabsf(b)));
    return y;
}

// Floats 2^23 + n are integers n in their low bits: codes go in and out of f32 by additions, not conversions.
constexpr float kInteger = 8388608.0f;

// (b + 0.5) / 65536 for the 16 random bits b of one half of each word: 2^23 + b, scaled and shifted in one exact operation.
template <int HALF>
__device__ __forceinline__ float2 random_units(uint32_t bits0, uint32_t bits1, const Constants& k) {
    const float2 b = make_float2(__uint_as_float(__byte_perm(bits0, 0x4B000000u, HALF == 0 ? 0x7410 : 0x7432)),
                                 __uint_as_float(__byte_perm(bits1, 0x4B000000u, HALF == 0 ? 0x7410 : 0x7432)));
    return __ffma2_rn(b, k.unit, k.unit_shift);
}

// The codes of a pair of shares (magnitudes over their block's scale), in the low bits of the results. q is the last
// level up to a share, at most one below the highest; its upper neighbour is taken if the random threshold between the two
// lies below the share. `guess` is q before it is rounded down, from approximate roots (2^-22) made smaller by 2^-20: it
// gives q or, for shares that close above a level, q - 1, which the comparison with the upper level shows. Shares of
// 0.9999 and more belong to the last step whatever it says.
template <typename Level>
__device__ __forceinline__ uint2 encode(float2 share, float2 guess, float2 u, const Constants& k, Level level) {
    float2 r = __fadd2_rd(guess, k.round);
    float2 q = __fadd2_rn(r, k.integer);
    float2 low = level(q), high = level(__fadd2_rn(q, k.one));
    const bool more_x = high.x <= fminf(share.x, 0.9999f), more_y = high.y <= fminf(share.y, 0.9999f);
    if (more_x || more_y) {
        r = __fadd2_rn(r, make_float2(more_x ? 1.0f : 0.0f, more_y ? 1.0f : 0.0f));
        q = __fadd2_rn(r, k.integer);
        low = level(q);
        high = level(__fadd2_rn(q, k.one));
    }
    const float2 step = sum_of(high, make_float2(-low.x, -low.y));  // (levels are products)
    const float2 threshold = sum_of(low, __fmul2_rn(u, step));
    return make_uint2(__float_as_uint(r.x) + (threshold.x < share.x ? 1u : 0u),
                      __float_as_uint(r.y) + (threshold.y < share.y ? 1u : 0u));
}

// Byte k of a word of codes as a float: as it is, or of a word whose sign bits were flipped, as a signed value.
__device__ __forceinline__ float code_value(uint32_t word, int k) {
    return __uint_as_float(__byte_perm(word, 0x4B000000u, 0x7540 + k));
}

// (scale, 1 / scale) of a block whose largest magnitude has these bits (as integers magnitudes order like floats, with
// infinity and NaN above all others). A block that holds one of those gets NaN, so that all of it decodes to NaN, whatever
// its codes. Subnormal scales count as 0.
__device__ __forceinline__ float2 scale_of(uint32_t bits) {
    if (bits >= 0x7F800000u) return make_float2(__uint_as_float(0x7FFFFFFFu), 0.0f);
    if (bits < 0x00800000u) return make_float2(0.0f, 0.0f);
    return make_float2(__uint_as_float(bits), __frcp_rn(__uint_as_float(bits)));
}

__device__ __forceinline__ float reciprocal_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// SplitMix64's output for a state.
__device__ __forceinline__ uint64_t mix(uint64_t z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

// A lane's elements of a block: 4 from 4 * lane and 4 from 128 + 4 * lane, so that every access of a warp is contiguous.
__device__ __forceinline__ int element_of(int lane, int j) { return (j >> 2) * 128 + 4 * lane + (j & 3); }

// The f64 sum of v over the thread block, in every thread, in a fixed order.
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[kWarps];
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    double sum = 0.0;
    for (int w = 0; w < kWarps; ++w) sum += part[w];
    return sum;
}

// The sum of the squares of all gradients, a partial sum for each thread block. Bound by memory: 97.6 million f32 gradients
// (391 MB, 60 us at the copy rate) take 77 us, bf16 ones (195 MB, 30 us) 42 us; 4.8 million bf16 ones, a latency, 6.3 us.
__global__ void __launch_bounds__(32 * kWarps) adamw8_norm_kernel(const __grid_constant__ Table m, double* partials) {
    double sum = 0.0;
    for (Share s = share_of(m); s.part < s.end; next_tensor(m, s)) {
        const snb_adamw8_tensor& x = m.t[s.tensor];
        const int64_t begin = (s.part - m.part_start[s.tensor]) * kPart;
        const int64_t n = end_of(m, s) - begin;
        const bool bf16 = x.gradient_type == SNB_TYPE_BF16;
        int64_t scalar_begin = 0;
        if (bf16 && multiple(x.gradient, 16)) {
            const uint4* g = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x.gradient) + begin);
            for (int64_t i = threadIdx.x; i < n / 8; i += 32 * kWarps) {
                const uint4 q = __ldg(g + i);
                for (uint32_t w : {q.x, q.y, q.z, q.w}) {
                    const double lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xFFFF0000u);
                    sum += lo * lo;
                    sum += hi * hi;
                }
            }
            scalar_begin = n / 8 * 8;
        } else if (!bf16 && multiple(x.gradient, 16)) {
            const float4* g = reinterpret_cast<const float4*>(static_cast<const float*>(x.gradient) + begin);
#pragma unroll 8
            for (int64_t i = threadIdx.x; i < n / 4; i += 32 * kWarps) {
                const float4 q = __ldg(g + i);
                for (double v : {static_cast<double>(q.x), static_cast<double>(q.y), static_cast<double>(q.z),
                                 static_cast<double>(q.w)})
                    sum += v * v;
            }
            scalar_begin = n / 4 * 4;
        }
        for (int64_t i = scalar_begin + threadIdx.x; i < n; i += 32 * kWarps) {
            const double v = bf16 ? bf16_value(static_cast<const uint16_t*>(x.gradient)[begin + i])
                                  : static_cast<const float*>(x.gradient)[begin + i];
            sum += v * v;
        }
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

struct StepParams {
    float2 minus_learning_rate, beta1, beta2, one_minus_beta1, one_minus_beta2, epsilon;
    float2 first_correction, second_correction;  // 1 / (1 - beta^step)
    Constants k;
    float max_norm;
    uint64_t seed;
    const double* partials;
    int32_t partial_count;
    double* square_sum;
};

// The step. A warp takes the 256 elements that share a scale, eight a lane, and holds them in registers from the read to the
// code, since the new scale is known only when the last of them is. 97.6 million elements with f32 gradients and bf16 copies
// (1.76 GB, 272 us at the copy rate) take 407 to 418 us, with the arithmetic and the memory traffic (348 us alone) overlapping
// for the most part, and with bf16 gradients (1.56 GB, 242 us) 409 us; three resident blocks an SM at 80 registers, against 469 us for two. 4.8 million elements with bf16
// gradients (76 MB): 28 us, bound by the latency of five passes of a warp.
__global__ void __launch_bounds__(32 * kWarps, kStepBlocks) adamw8_step_kernel(const __grid_constant__ Table m, const StepParams a) {
    // Every thread block adds the norm's partial sums in the same order.
    double sum = 0.0;
    for (int i = threadIdx.x; i < a.partial_count; i += 32 * kWarps) sum += a.partials[i];
    sum = block_sum(sum);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.square_sum = sum;
    const float norm = static_cast<float>(sqrt(sum));
    const float clip = norm > a.max_norm ? __fdiv_rn(a.max_norm, norm) : 1.0f;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (Share s = share_of(m); s.part < s.end; next_tensor(m, s)) {
        const snb_adamw8_tensor& x = m.t[s.tensor];
        const int64_t begin = (s.part - m.part_start[s.tensor]) * kPart, end = end_of(m, s);
        const int64_t count = static_cast<int64_t>(x.count);
        const bool grad_bf16 = x.gradient_type == SNB_TYPE_BF16;
        const bool aligned = multiple(x.parameter, 16) && multiple(x.gradient, grad_bf16 ? 8 : 16) &&
                             multiple(x.first, 4) && multiple(x.second, 4) && multiple(x.shadow, 8);
        for (int64_t at = begin + warp * kBlock; at < end; at += kPart) {
            const bool whole = aligned && at + kBlock <= count;
            float w[8], g[8];
            uint32_t c1[2] = {0, 0}, c2[2] = {0, 0};
            if (whole) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int64_t e = at + element_of(lane, 4 * h);
                    const float4 wv = *reinterpret_cast<const float4*>(x.parameter + e);
                    w[4 * h] = wv.x; w[4 * h + 1] = wv.y; w[4 * h + 2] = wv.z; w[4 * h + 3] = wv.w;
                    if (grad_bf16) {
                        const uint2 q = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(x.gradient) + e));
                        g[4 * h] = __uint_as_float(q.x << 16); g[4 * h + 1] = __uint_as_float(q.x & 0xFFFF0000u);
                        g[4 * h + 2] = __uint_as_float(q.y << 16); g[4 * h + 3] = __uint_as_float(q.y & 0xFFFF0000u);
                    } else {
                        const float4 q = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(x.gradient) + e));
                        g[4 * h] = q.x; g[4 * h + 1] = q.y; g[4 * h + 2] = q.z; g[4 * h + 3] = q.w;
                    }
                    c1[h] = *reinterpret_cast<const uint32_t*>(x.first + e);
                    c2[h] = *reinterpret_cast<const uint32_t*>(x.second + e);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int64_t e = at + element_of(lane, j);
                    const bool live = e < count;
                    w[j] = live ? x.parameter[e] : 0.0f;
                    g[j] = !live ? 0.0f
                                 : grad_bf16 ? bf16_value(static_cast<const uint16_t*>(x.gradient)[e])
                                             : static_cast<const float*>(x.gradient)[e];
                    const uint32_t b1 = live ? static_cast<uint8_t>(x.first[e]) : 0, b2 = live ? x.second[e] : 0;
                    c1[j >> 2] |= b1 << (8 * (j & 3));
                    c2[j >> 2] |= b2 << (8 * (j & 3));
                }
            }
            const float s1 = x.first_scale[at / kBlock], s2 = x.second_scale[at / kBlock];
            float2 mean[4], variance[4];
            float top1 = 0.0f, top2 = 0.0f;
            c1[0] ^= 0x80808080u;
            c1[1] ^= 0x80808080u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // elements 2j and 2j + 1
                const int b = 2 * j & 3;
                const float2 q1 = __fadd2_rn(make_float2(code_value(c1[j >> 1], b), code_value(c1[j >> 1], b + 1)), a.k.code);
                const float2 q2 = __fadd2_rn(make_float2(code_value(c2[j >> 1], b), code_value(c2[j >> 1], b + 1)), a.k.integer);
                const float2 gj = __fmul2_rn(make_float2(g[2 * j], g[2 * j + 1]), both(clip));
                const float2 signed_square = make_float2(__fmul_rn(q1.x, fabsf(q1.x)), __fmul_rn(q1.y, fabsf(q1.y)));
                const float2 old1 = __fmul2_rn(__fmul2_rn(signed_square, a.k.first), both(s1));
                const float2 old2 = __fmul2_rn(second_level(q2, a.k), both(s2));
                mean[j] = sum_of(__fmul2_rn(old1, a.beta1), __fmul2_rn(gj, a.one_minus_beta1));
                variance[j] = sum_of(__fmul2_rn(old2, a.beta2), __fmul2_rn(__fmul2_rn(gj, a.one_minus_beta2), gj));
                top1 = max_or_nan(max_or_nan(top1, mean[j].x), mean[j].y);
                top2 = max_or_nan(max_or_nan(top2, variance[j].x), variance[j].y);
                // The update itself decides no code: approximate root and reciprocal (2^-22) far below its own step.
                const float2 vh = __fmul2_rn(variance[j], a.second_correction);
                const float2 root = __fadd2_rn(make_float2(sqrt_fast(vh.x), sqrt_fast(vh.y)), a.epsilon);
                const float2 mh = __fmul2_rn(mean[j], a.first_correction);
                const float2 old = make_float2(w[2 * j], w[2 * j + 1]);
                const float2 rate = __fmul2_rn(mh, make_float2(reciprocal_fast(root.x), reciprocal_fast(root.y)));
                const float2 next = __ffma2_rn(a.minus_learning_rate, __ffma2_rn(both(x.weight_decay), old, rate), old);
                w[2 * j] = next.x;
                w[2 * j + 1] = next.y;
            }
            // The parameter leaves now, so that its registers serve the encoding.
            if (whole) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int64_t e = at + element_of(lane, 4 * h);
                    *reinterpret_cast<float4*>(x.parameter + e) = make_float4(w[4 * h], w[4 * h + 1], w[4 * h + 2],
                                                                              w[4 * h + 3]);
                    if (x.shadow != nullptr)
                        *reinterpret_cast<uint2*>(x.shadow + e) = make_uint2(bf16_pair(w[4 * h], w[4 * h + 1]),
                                                                             bf16_pair(w[4 * h + 2], w[4 * h + 3]));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int64_t e = at + element_of(lane, j);
                    if (e >= count) continue;
                    x.parameter[e] = w[j];
                    if (x.shadow != nullptr) x.shadow[e] = static_cast<uint16_t>(bf16_pair(w[j], 0.0f));
                }
            }
            const float2 n1 = scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(top1) & 0x7FFFFFFFu));
            const float2 n2 = scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(top2) & 0x7FFFFFFFu));
            // States of the lane's draws: elements 2j and 2j + 1 share one; pairs 0 and 1 are 64 draws before 2 and 3.
            const uint64_t state = a.seed + (x.first_draw + static_cast<uint64_t>(at / 2 + 2 * lane) + 1) * kGolden;
            uint32_t code1[8], code2[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint64_t bits = mix(state + ((j & 1) + (j >> 1) * 64) * kGolden);
                const uint32_t b0 = static_cast<uint32_t>(bits), b1 = static_cast<uint32_t>(bits >> 32);
                const float2 share1 = __fmul2_rn(make_float2(fabsf(mean[j].x), fabsf(mean[j].y)), both(n1.y));
                const float2 share2 = __fmul2_rn(variance[j], both(n2.y));
                const float2 guess1 = __fmul2_rn(make_float2(sqrt_fast(share1.x), sqrt_fast(share1.y)), a.k.guess1);
                const float2 guess2 = __fmul2_rn(
                    make_float2(sqrt_fast(sqrt_fast(share2.x)), sqrt_fast(sqrt_fast(share2.y))), a.k.guess2);
                const uint2 e1 = encode(share1, guess1, random_units<0>(b0, b1, a.k), a.k,
                                        [&](float2 q) { return first_level(q, a.k); });
                const uint2 e2 = encode(share2, guess2, random_units<1>(b0, b1, a.k), a.k,
                                        [&](float2 q) { return second_level(q, a.k); });
                // m's sign; v's lowest code above 0.
                const uint32_t m0 = static_cast<uint32_t>(static_cast<int32_t>(__float_as_uint(mean[j].x)) >> 31);
                const uint32_t m1 = static_cast<uint32_t>(static_cast<int32_t>(__float_as_uint(mean[j].y)) >> 31);
                code1[2 * j] = (e1.x ^ m0) - m0;
                code1[2 * j + 1] = (e1.y ^ m1) - m1;
                code2[2 * j] = max(e2.x, variance[j].x > 0.0f ? 0x4B000001u : 0x4B000000u);
                code2[2 * j + 1] = max(e2.y, variance[j].y > 0.0f ? 0x4B000001u : 0x4B000000u);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                c1[h] = __byte_perm(__byte_perm(code1[4 * h], code1[4 * h + 1], 0x0040),
                                    __byte_perm(code1[4 * h + 2], code1[4 * h + 3], 0x0040), 0x5410);
                c2[h] = __byte_perm(__byte_perm(code2[4 * h], code2[4 * h + 1], 0x0040),
                                    __byte_perm(code2[4 * h + 2], code2[4 * h + 3], 0x0040), 0x5410);
            }
            if (lane == 0) {
                x.first_scale[at / kBlock] = n1.x;
                x.second_scale[at / kBlock] = n2.x;
            }
            if (whole) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int64_t e = at + element_of(lane, 4 * h);
                    *reinterpret_cast<uint32_t*>(x.first + e) = c1[h];
                    *reinterpret_cast<uint32_t*>(x.second + e) = c2[h];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int64_t e = at + element_of(lane, j);
                    if (e >= count) continue;
                    x.first[e] = static_cast<int8_t>(c1[j >> 2] >> (8 * (j & 3)));
                    x.second[e] = static_cast<uint8_t>(c2[j >> 2] >> (8 * (j & 3)));
                }
            }
        }
    }
}

// The moments' values in f32, for checkpoints and inspection. Bound by memory, most of it the 8 bytes written for an element:
// 97.6 million elements (976 MB, 151 us at the copy rate) take 164 us on three blocks an SM; four, whose writes go to more
// places at once, take 174 us and eight 178 us. Where L2 holds the values more blocks do no harm and hide more latency:
// 4.8 million elements take 10.4 us on eight, 12.1 us on three.
constexpr int64_t kCachedBytes = 96 << 20;

struct MomentTable {
    int32_t n;
    Shares shares;
    snb_adamw8_moments_out t[kMaxTensors];
    int64_t part_start[kMaxTensors + 1];
};
static_assert(sizeof(MomentTable) < 32000, "kernel parameters");

__global__ void __launch_bounds__(32 * kWarps) adamw8_moments_kernel(const __grid_constant__ MomentTable m) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (Share s = share_of(m); s.part < s.end; next_tensor(m, s)) {
        const snb_adamw8_moments_out& x = m.t[s.tensor];
        const int64_t begin = (s.part - m.part_start[s.tensor]) * kPart, end = end_of(m, s);
        const int64_t count = static_cast<int64_t>(x.count);
        const bool aligned = multiple(x.first, 4) && multiple(x.second, 4) && multiple(x.first_out, 16) &&
                             multiple(x.second_out, 16);
        for (int64_t at = begin + warp * kBlock; at < end; at += kPart) {
            const float s1 = x.first_scale[at / kBlock], s2 = x.second_scale[at / kBlock];
            auto value1 = [&](int8_t c) {
                const float q = static_cast<float>(c);
                return __fmul_rn(__fmul_rn(__fmul_rn(q, fabsf(q)), 1.0f / 16129.0f), s1);
            };
            auto value2 = [&](uint32_t c) {
                const float q = static_cast<float>(c), root = __fmul_rn(__fmul_rn(q, q), 1.0f / 65025.0f);
                return __fmul_rn(__fmul_rn(root, root), s2);
            };
            if (aligned && at + kBlock <= count) {
                uint32_t c1[2], c2[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int64_t e = at + element_of(lane, 4 * h);
                    c1[h] = *reinterpret_cast<const uint32_t*>(x.first + e);
                    c2[h] = *reinterpret_cast<const uint32_t*>(x.second + e);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int64_t e = at + element_of(lane, 4 * h);
                    *reinterpret_cast<float4*>(x.first_out + e) =
                        make_float4(value1(static_cast<int8_t>(c1[h])), value1(static_cast<int8_t>(c1[h] >> 8)),
                                    value1(static_cast<int8_t>(c1[h] >> 16)), value1(static_cast<int8_t>(c1[h] >> 24)));
                    *reinterpret_cast<float4*>(x.second_out + e) =
                        make_float4(value2(c2[h] & 0xFFu), value2((c2[h] >> 8) & 0xFFu), value2((c2[h] >> 16) & 0xFFu),
                                    value2(c2[h] >> 24));
                }
            } else {
                for (int j = 0; j < 8; ++j) {
                    const int64_t e = at + element_of(lane, j);
                    if (e >= count) continue;
                    x.first_out[e] = value1(x.first[e]);
                    x.second_out[e] = value2(x.second[e]);
                }
            }
        }
    }
}

int launched(const char* what, std::string* err) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return SNB_OK;
    *err = cuda_message(what, e);
    return SNB_ERR_CUDA;
}

// The table of tensors [first, first + up to kMaxTensors); returns how many it holds.
template <typename T, typename Source>
uint64_t fill(T* table, const Source* tensors, uint64_t first, uint64_t n) {
    const uint64_t take = std::min<uint64_t>(n - first, kMaxTensors);
    int64_t parts = 0;
    for (uint64_t i = 0; i < take; ++i) {
        table->t[i] = tensors[first + i];
        table->part_start[i] = parts;
        parts += static_cast<int64_t>((tensors[first + i].count + kPart - 1) / kPart);
    }
    table->part_start[take] = parts;
    table->n = static_cast<int32_t>(take);
    return take;
}

// Shares a table's parts between at most `most` blocks; returns how many.
template <typename T>
unsigned share(T* table, int64_t most) {
    const int64_t parts = table->part_start[table->n];
    const int64_t blocks = std::min<int64_t>(parts, std::min<int64_t>(most, kMaxGrid));
    table->shares.each = parts / blocks;
    table->shares.longer = parts % blocks;
    int tensor = 0;
    for (int64_t b = 0, part = 0; b < blocks; ++b) {
        while (table->part_start[tensor + 1] <= part) ++tensor;
        table->shares.first_tensor[b] = static_cast<uint8_t>(tensor);
        part += table->shares.each + (b < table->shares.longer ? 1 : 0);
    }
    return static_cast<unsigned>(blocks);
}

}  // namespace

uint64_t adamw8_workspace(uint64_t tensor_count) {
    const uint64_t launches = (tensor_count + kMaxTensors - 1) / kMaxTensors;
    return std::max<uint64_t>(1, launches) * kSumBlocks * sizeof(double);
}

int adamw8_step_launch(cudaStream_t s, const snb_adamw8_tensor* tensors, uint64_t n, const snb_adamw_hyper& h,
                       float max_gradient_norm, uint64_t seed, double* square_sum, double* partials, std::string* err) {
    DeviceInfo dev;
    int rc = current_device_info(&dev, err);
    if (rc != SNB_OK) return rc;
    Table table{};
    int32_t sums = 0;
    for (uint64_t i = 0; i < n; i += kMaxTensors) {
        fill(&table, tensors, i, n);
        if (table.part_start[table.n] == 0) continue;
        const unsigned blocks = share(&table, kSumBlocks);
        adamw8_norm_kernel<<<blocks, 32 * kWarps, 0, s>>>(table, partials + sums);
        if ((rc = launched("adamw8_norm_kernel launch", err)) != SNB_OK) return rc;
        sums += blocks;
    }
    if (sums == 0) {
        const cudaError_t e = cudaMemsetAsync(square_sum, 0, sizeof(double), s);
        if (e == cudaSuccess) return SNB_OK;
        *err = cuda_message("cudaMemsetAsync(gradient square sum)", e);
        return SNB_ERR_CUDA;
    }
    StepParams a{};
    auto pair = [](double v) { return make_float2(static_cast<float>(v), static_cast<float>(v)); };
    a.minus_learning_rate = pair(-h.learning_rate);
    a.beta1 = pair(h.beta1);
    a.beta2 = pair(h.beta2);
    a.one_minus_beta1 = pair(1.0f - h.beta1);
    a.one_minus_beta2 = pair(1.0f - h.beta2);
    a.epsilon = pair(h.epsilon);
    a.first_correction = pair(1.0 / (1.0 - std::pow(static_cast<double>(h.beta1), h.step)));
    a.second_correction = pair(1.0 / (1.0 - std::pow(static_cast<double>(h.beta2), h.step)));
    a.k.first = pair(1.0f / 16129.0f);
    a.k.second = pair(1.0f / 65025.0f);
    a.k.round = pair(kInteger);
    a.k.integer = pair(-kInteger);
    a.k.code = pair(-kInteger - 128.0f);
    a.k.one = pair(1.0);
    a.k.guess1 = pair(127.0 * (1.0 - 0x1p-20));
    a.k.guess2 = pair(255.0 * (1.0 - 0x1p-20));
    a.k.unit = pair(0x1p-16);
    a.k.unit_shift = pair(0x1p-17 - 128.0);
    a.max_norm = max_gradient_norm;
    a.seed = seed;
    a.partials = partials;
    a.partial_count = sums;
    a.square_sum = square_sum;
    for (uint64_t i = 0; i < n; i += kMaxTensors) {
        if (n > kMaxTensors) fill(&table, tensors, i, n);
        if (table.part_start[table.n] == 0) continue;
        const unsigned blocks = share(&table, kStepBlocks * dev.sm_count);
        adamw8_step_kernel<<<blocks, 32 * kWarps, 0, s>>>(table, a);
        if ((rc = launched("adamw8_step_kernel launch", err)) != SNB_OK) return rc;
    }
    return SNB_OK;
}

int adamw8_moments_launch(cudaStream_t s, const snb_adamw8_moments_out* tensors, uint64_t n, std::string* err) {
    DeviceInfo dev;
    int rc = current_device_info(&dev, err);
    if (rc != SNB_OK) return rc;
    MomentTable table{};
    for (uint64_t i = 0; i < n; i += kMaxTensors) {
        fill(&table, tensors, i, n);
        if (table.part_start[table.n] == 0) continue;
        const bool cached = table.part_start[table.n] * kPart * 8 <= kCachedBytes;
        const unsigned blocks = share(&table, (cached ? 8 : 3) * dev.sm_count);
        adamw8_moments_kernel<<<blocks, 32 * kWarps, 0, s>>>(table);
        if ((rc = launched("adamw8_moments_kernel launch", err)) != SNB_OK) return rc;
    }
    return SNB_OK;
}

}  // namespace snb
