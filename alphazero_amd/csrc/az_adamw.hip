// az_adamw.hip -- the AdamW step over all tensors of a network in one launch, moments in 32 or in 8 bits (the
// reference trains with SGD: alphazero/training.py:27-29; az_sgd_momentum in az_train.hip).
//
//   t = t + 1
//   m = (b1 * m) + ((1 - b1) * g)          v = (b2 * v) + ((1 - b2) * (g * g))
//   p = p * (1 - lr * wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)        (0 / 0, where eps is 0, taken as 0)
//
// The tensors lie behind each other in flat buffers, each from a multiple of 256 elements on (the gaps are zero and stay
// zero); tensors with the same settings form a run.  The step count lives in device memory, so that a launch recorded
// in a HIP graph counts on: one counter for each workgroup, which reads it first and writes it back one higher.
//
// Moments in 8 bits, for each block of 256 elements: `top` = the 11 leading bits of a float (exponent, 3 bits of
// mantissa) of the block's largest magnitude, rounded up, and per element how many such steps below the top it is:
//   m: a sign and 7 bits k, 0 = zero, else leading bits top - 127 + k (16 octaves);   v: 8 bits k, top - 255 + k (32 octaves).
// Rounding to leading bits is an integer addition below them and a shift.  It is done at random, up with the probability
// that leaves the expectation unchanged: with b2 = 0.999 a step moves v by a thousandth of itself, far less than the
// half step of 6 % that rounding to the nearest would swallow, and v would never follow its gradients.  A v > 0 below the
// lowest code is kept AT the lowest, so that no denominator collapses to eps; an m there becomes zero or the
// lowest at random.  The random bits are splitmix64's output (Steele, Lea, Flood 2014) of a counter made from (seed, t,
// element), 16 for each value.  A NaN makes its block's top 0x7FF, whose code 127 / 255 is a NaN again; beside it, as
// beside an infinity, the block's other values are lost.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/azhip.h"
#include "az_host.h"

#define ADAMW_BLOCK AZ_ADAMW_BLOCK   // elements: four of each lane of a wave
static_assert(ADAMW_BLOCK == 4 * 64, "a wave takes a block");
// A wave takes a block, four neighbouring elements to a lane, so that every load and store of a wave is one piece of memory.
// Bound by memory in 32 bits (28 bytes an element): 46 M parameters 223 us = 5.8 TB/s, where a copy of as much has 4.7 to
// 5.2.  In 8 bits (16 bytes) by memory and instructions alike: 138 us = 5.4 TB/s, and 77 vector instructions an element
// keep the SIMDs busy for 69 % of it, the random numbers about a sixth of them.  Workgroups of 512 threads whose waves take
// one block and end, or, beyond 33.5 M elements (AZ_ADAMW_STEPS workgroups), walk in steps of the whole grid: their traffic
// moves along memory as one front.  2048 workgroups that walk took 238 to 250 us beside 222, and 137 to 146 beside 129.
#define ADAMW_THREADS 512
#define ADAMW_GOLDEN 0x9E3779B97F4A7C15ull

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

struct AdamwRun { long first_block; double lr, beta1, beta2, log1, log2, eps, weight_decay; int half, lr_index; };
struct AdamwRuns { AdamwRun r[AZ_ADAMW_MAX_RUNS]; int n; };
struct AdamwScalars { float keep, step, root, b1, c1, b2, c2, eps; int half, fast; };

__device__ __forceinline__ uint64_t adamw_mix(uint64_t z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

// largest value of the 64 lanes, in a scalar register: within rows of 16, then across them, into lane 63
__device__ __forceinline__ uint32_t adamw_wave_max(uint32_t v) {
#define ADAMW_DPP_MAX(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false))
    ADAMW_DPP_MAX(0x111, 0xf);        // row_shr 1, 2, 4, 8
    ADAMW_DPP_MAX(0x112, 0xf);
    ADAMW_DPP_MAX(0x114, 0xf);
    ADAMW_DPP_MAX(0x118, 0xf);
    ADAMW_DPP_MAX(0x142, 0xa);        // lane 15 of each row to the next row, lane 31 to the upper half
    ADAMW_DPP_MAX(0x143, 0xc);
#undef ADAMW_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ uint32_t adamw_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// leading bits of the largest magnitude of a block, rounded up
__device__ __forceinline__ int adamw_top(const f32x4& x) {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) a = max(a, adamw_bits(x[i]));
    const uint32_t most = adamw_wave_max(a);
    return most > 0x7F800000u ? 0x7FF : (int)((most + 0xFFFFFu) >> 20);
}

// The codes of a lane's four values; random: 16 bits for each.  `top` is the same in all lanes.  The first loop is right
// for blocks without a NaN whose values reach the codes or are zero; the second, which most waves skip, for the others.
__device__ __forceinline__ uint32_t adamw_codes_m(const f32x4& x, uint64_t random, int top) {
    const int base = top - 127, lowest = max(top - 126, 1);
    uint32_t out = 0;
    bool below = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = adamw_bits(x[i]), r = (uint32_t)(random >> (16 * i)) & 0xFFFFu;
        const int q = (int)((a + (r << 4)) >> 20), k = q - base;
        below |= q < lowest && a;
        out |= (q >= lowest ? (uint32_t)k | ((__float_as_uint(x[i]) >> 24) & 0x80u) : 0u) << (8 * i);
    }
    if (top == 0x7FF || __any(below)) {
        out = 0;
        const float vmin = __uint_as_float((uint32_t)lowest << 20);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a = adamw_bits(x[i]), r = (uint32_t)(random >> (16 * i)) & 0xFFFFu;
            const int q = a > 0x7F800000u ? 0x7FF : (int)((a + (r << 4)) >> 20);
            // (2^17 |x| and (2 r + 1) vmin are exact)
            const int k = q >= lowest ? q - base : __uint_as_float(a) * 131072.0f > (float)(2 * r + 1) * vmin ? lowest - base : 0;
            out |= (k ? (uint32_t)k | ((__float_as_uint(x[i]) >> 24) & 0x80u) : 0u) << (8 * i);
        }
    }
    return out;
}

__device__ __forceinline__ uint32_t adamw_codes_v(const f32x4& x, uint64_t random, int top) {
    const int base = top - 255, lowest = max(top - 254, 1);
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = adamw_bits(x[i]), r = (uint32_t)(random >> (16 * i)) & 0xFFFFu;
        int q = (int)((a + (r << 4)) >> 20);
        if (top == 0x7FF && a > 0x7F800000u) q = 0x7FF;
        out |= (a ? (uint32_t)(max(q, lowest) - base) : 0u) << (8 * i);
    }
    return out;
}

// (base: top - 127 or top - 255, as leading bits)
__device__ __forceinline__ float adamw_value(uint32_t k, int base) { return k ? __uint_as_float((k << 20) + ((uint32_t)base << 20)) : 0.0f; }

__device__ __forceinline__ f32x4 adamw_values_m(uint32_t codes, int top) {
    f32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x[i] = __uint_as_float(__float_as_uint(adamw_value((codes >> (8 * i)) & 127u, top - 127)) | ((codes << (24 - 8 * i)) & 0x80000000u));
    return x;
}

__device__ __forceinline__ f32x4 adamw_values_v(uint32_t codes, int top) {
    f32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = adamw_value((codes >> (8 * i)) & 255u, top - 255);
    return x;
}

// Moments, gradients and codes are read and written once a step: their lines are marked as not worth keeping, which
// leaves the caches to the parameters that the next forward pass reads (46 M parameters, 32 bits: 270 -> 250 us).
template <typename T> __device__ __forceinline__ T adamw_load(const void* p) { return __builtin_nontemporal_load(reinterpret_cast<const T*>(p)); }
template <typename T> __device__ __forceinline__ void adamw_store(void* p, const T& v) { __builtin_nontemporal_store(v, reinterpret_cast<T*>(p)); }

// what a lane reads of a block
template <int BITS> struct AdamwIn {
    f32x4 p, g, m, v;
    bf16x4 h, p16;                    // bfloat16 runs: gradient and parameter
    uint32_t m8, v8, top;
};

template <int BITS>
__device__ __forceinline__ void adamw_read(const az_adamw_buffers& q, long blk, int lane, int half, AdamwIn<BITS>& in) {
    const long at = blk * ADAMW_BLOCK + lane * 4;
    in.p = *reinterpret_cast<const f32x4*>(q.p + at);
    if (half) {
        in.h = adamw_load<bf16x4>(q.g16 + at);
        in.p16 = *reinterpret_cast<const bf16x4*>(q.p16 + at);
    } else in.g = adamw_load<f32x4>(q.g + at);
    if constexpr (BITS == 32) {
        in.m = adamw_load<f32x4>(q.m + at);
        in.v = adamw_load<f32x4>(q.v + at);
    } else {
        in.m8 = adamw_load<uint32_t>(q.m8 + at);
        in.v8 = adamw_load<uint32_t>(q.v8 + at);
        in.top = *reinterpret_cast<const uint32_t*>(q.top + 2 * blk);
    }
}

template <int BITS>
__global__ void __launch_bounds__(ADAMW_THREADS)
k_adamw(az_adamw_buffers q, long blocks, AdamwRuns runs, const double* __restrict__ lr_dev, uint64_t seed,
        const float* __restrict__ guard, float limit, int* __restrict__ withheld) {
    if (guard && !(guard[0] < limit)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) withheld[0] += 1;
        return;
    }
    __shared__ AdamwScalars sc[AZ_ADAMW_MAX_RUNS];
    const int tid = threadIdx.x, lane = tid & 63;
    const long stride = (long)gridDim.x * (ADAMW_THREADS / 64);
    long blk = (long)blockIdx.x * (ADAMW_THREADS / 64) + __builtin_amdgcn_readfirstlane(tid >> 6);
    int run = 0;
    // the first block is on its way while the scalars are made (two functions in 64 bits; 1.2 M parameters in 32 bits:
    // 7.9 -> 6.7 us)
    AdamwIn<BITS> in;
    const int64_t t = q.step[blockIdx.x] + 1;
    if (blk < blocks) {
        while (run + 1 < runs.n && blk >= runs.r[run + 1].first_block) ++run;
        adamw_read<BITS>(q, blk, lane, runs.r[run].half, in);
    }
    if (tid < runs.n) {
        const AdamwRun& r = runs.r[tid];
        const double lr = lr_dev ? lr_dev[r.lr_index] : r.lr;
        AdamwScalars s;
        s.keep = (float)(1.0 - lr * r.weight_decay);
        s.step = (float)(lr / -expm1((double)t * r.log1));
        s.root = (float)(1.0 / sqrt(-expm1((double)t * r.log2)));
        s.b1 = (float)r.beta1; s.c1 = (float)(1.0 - r.beta1);
        s.b2 = (float)r.beta2; s.c2 = (float)(1.0 - r.beta2);
        s.eps = (float)r.eps; s.half = r.half;
        // The hardware's square root and reciprocal are good to 2^-23, but the root takes a subnormal number for zero: up to
        // 2^-63, which is root times that in the denominator, half a step of eps or less where eps is 2^-39 root and more (with
        // the customary betas and an eps of 1e-8 at every step; an eps of 1e-12 never, whose steps take IEEE's functions:
        // 46 M parameters in 8 bits 143 us for 131, in 32 bits the same).
        s.fast = s.eps >= s.root * 0x1p-39f;
        sc[tid] = s;
    }
    __syncthreads();
    if (tid == 0) q.step[blockIdx.x] = t;                                 // (behind the barrier: every thread has read it)
    const uint64_t key = adamw_mix(seed + ADAMW_GOLDEN * (uint64_t)t);
    while (blk < blocks) {
        const AdamwScalars s = sc[run];
        const long at = blk * ADAMW_BLOCK + lane * 4;
        f32x4 p = in.p, g, m, v;
        if (s.half) {
            g = __builtin_convertvector(in.h, f32x4);
            // a parameter that is not its master's rounding was written by somebody else (a checkpoint loaded): it counts
            const u16x4 have = __builtin_bit_cast(u16x4, in.p16), mine = __builtin_bit_cast(u16x4, __builtin_convertvector(p, bf16x4));
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = have[i] != mine[i] ? (float)in.p16[i] : p[i];
        } else g = in.g;
        if constexpr (BITS == 32) { m = in.m; v = in.v; }
        else {
            m = adamw_values_m(in.m8, in.top & 0xFFFFu);
            v = adamw_values_v(in.v8, in.top >> 16);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = m[i] * s.b1 + g[i] * s.c1;
            v[i] = v[i] * s.b2 + (g[i] * g[i]) * s.c2;
        }
        if (s.fast) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                p[i] = p[i] * s.keep - s.step * m[i] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[i]) * s.root + s.eps);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // (0 / 0 without an eps: no update, in the gaps and where every gradient was zero)
                const float den = sqrtf(v[i]) * s.root + s.eps;
                p[i] = p[i] * s.keep - (den == 0.0f && m[i] == 0.0f ? 0.0f : s.step * m[i] / den);
            }
        }
        *reinterpret_cast<f32x4*>(q.p + at) = p;
        if (s.half) *reinterpret_cast<bf16x4*>(q.p16 + at) = __builtin_convertvector(p, bf16x4);
        if constexpr (BITS == 32) {
            adamw_store(q.m + at, m);
            adamw_store(q.v + at, v);
        } else {
            const int tm = adamw_top(m), tv = adamw_top(v);
            const uint64_t counter = key + ADAMW_GOLDEN * ((uint64_t)at / 2);       // two numbers for every four elements
            adamw_store(q.m8 + at, adamw_codes_m(m, adamw_mix(counter), tm));
            adamw_store(q.v8 + at, adamw_codes_v(v, adamw_mix(counter + ADAMW_GOLDEN), tv));
            if (lane == 0) *reinterpret_cast<uint32_t*>(q.top + 2 * blk) = (uint32_t)tm | ((uint32_t)tv << 16);
        }
        blk += stride;
        if (blk < blocks) {
            while (run + 1 < runs.n && blk >= runs.r[run + 1].first_block) ++run;
            adamw_read<BITS>(q, blk, lane, runs.r[run].half, in);
        }
    }
}

__global__ void __launch_bounds__(ADAMW_THREADS)
k_adamw_decode(const uint8_t* __restrict__ m8, const uint8_t* __restrict__ v8, const uint16_t* __restrict__ top, long blocks,
               float* __restrict__ m, float* __restrict__ v) {
    const int lane = threadIdx.x & 63;
    for (long blk = (long)blockIdx.x * (ADAMW_THREADS / 64) + (threadIdx.x >> 6); blk < blocks; blk += (long)gridDim.x * (ADAMW_THREADS / 64)) {
        const long at = blk * ADAMW_BLOCK + lane * 4;
        *reinterpret_cast<f32x4*>(m + at) = adamw_values_m(*reinterpret_cast<const uint32_t*>(m8 + at), top[2 * blk]);
        *reinterpret_cast<f32x4*>(v + at) = adamw_values_v(*reinterpret_cast<const uint32_t*>(v8 + at), top[2 * blk + 1]);
    }
}

// (values that are no codes' -- moments that were kept in 32 bits -- are rounded to the nearest leading bits)
__global__ void __launch_bounds__(ADAMW_THREADS)
k_adamw_encode(const float* __restrict__ m, const float* __restrict__ v, long blocks, uint8_t* __restrict__ m8,
               uint8_t* __restrict__ v8, uint16_t* __restrict__ top) {
    const int lane = threadIdx.x & 63;
    const uint64_t half = 0x8000800080008000ull;
    for (long blk = (long)blockIdx.x * (ADAMW_THREADS / 64) + (threadIdx.x >> 6); blk < blocks; blk += (long)gridDim.x * (ADAMW_THREADS / 64)) {
        const long at = blk * ADAMW_BLOCK + lane * 4;
        const f32x4 a = *reinterpret_cast<const f32x4*>(m + at), b = *reinterpret_cast<const f32x4*>(v + at);
        const int tm = adamw_top(a), tv = adamw_top(b);
        *reinterpret_cast<uint32_t*>(m8 + at) = adamw_codes_m(a, half, tm);
        *reinterpret_cast<uint32_t*>(v8 + at) = adamw_codes_v(b, half, tv);
        if (lane == 0) *reinterpret_cast<uint32_t*>(top + 2 * blk) = (uint32_t)tm | ((uint32_t)tv << 16);
    }
}

static unsigned adamw_grid(long blocks) {
    const long need = (blocks + ADAMW_THREADS / 64 - 1) / (ADAMW_THREADS / 64);
    return (unsigned)(need < AZ_ADAMW_STEPS ? need : AZ_ADAMW_STEPS);
}

extern "C" {

int az_adamw_step(const az_adamw_buffers* b, int64_t blocks, const az_adamw_run* runs, int32_t num_runs, int32_t state_bits,
                  const double* lr_dev, uint64_t seed, const float* guard_dev, float guard_limit, int32_t* withheld_dev,
                  void* stream) {
    if (!b || !runs || blocks < 0) return az_fail("az_adamw_step: null pointer");
    if (num_runs < 1 || num_runs > AZ_ADAMW_MAX_RUNS) return az_fail("az_adamw_step: 1 to 32 runs");
    if (state_bits != 8 && state_bits != 32) return az_fail("az_adamw_step: moments in 8 or in 32 bits");
    if (!b->p || !b->step || (state_bits == 32 ? !b->m || !b->v : !b->m8 || !b->v8 || !b->top) || (guard_dev && !withheld_dev))
        return az_fail("az_adamw_step: null pointer");
    AdamwRuns r = {};
    r.n = num_runs;
    for (int i = 0; i < num_runs; ++i) {
        r.r[i] = {(long)runs[i].first_block, runs[i].lr, runs[i].beta1, runs[i].beta2, log(runs[i].beta1), log(runs[i].beta2), runs[i].eps,
                  runs[i].weight_decay, runs[i].half, runs[i].lr_index};
        if (runs[i].first_block < (i ? runs[i - 1].first_block : 0) || (i == 0 && runs[i].first_block != 0) || runs[i].first_block > blocks)
            return az_fail("az_adamw_step: runs begin at block 0 and follow each other");
        if (!(runs[i].beta1 >= 0.0 && runs[i].beta1 < 1.0 && runs[i].beta2 >= 0.0 && runs[i].beta2 < 1.0 && runs[i].eps >= 0.0))
            return az_fail("az_adamw_step: 0 <= beta < 1, eps >= 0");
        if (runs[i].half ? !b->p16 || !b->g16 : !b->g) return az_fail("az_adamw_step: null pointer");
        if (lr_dev && (runs[i].lr_index < 0 || runs[i].lr_index >= AZ_ADAMW_MAX_RUNS)) return az_fail("az_adamw_step: lr_index is 0 to 31");
    }
    const void* all[] = {b->p, b->g, b->p16, b->g16, b->m, b->v, b->m8, b->v8, b->top};
    for (const void* p : all)
        if ((uintptr_t)p % 16) return az_fail("az_adamw_step: buffers are aligned to 16 bytes");
    if (blocks == 0) return 0;
    if (state_bits == 32)
        hipLaunchKernelGGL((k_adamw<32>), dim3(adamw_grid(blocks)), dim3(ADAMW_THREADS), 0, (hipStream_t)stream, *b, (long)blocks, r,
                           lr_dev, seed, guard_dev, guard_limit, withheld_dev);
    else
        hipLaunchKernelGGL((k_adamw<8>), dim3(adamw_grid(blocks)), dim3(ADAMW_THREADS), 0, (hipStream_t)stream, *b, (long)blocks, r,
                           lr_dev, seed, guard_dev, guard_limit, withheld_dev);
    AZ_LAUNCH_CHECK("k_adamw");
    return 0;
}

int az_adamw_decode8(const uint8_t* m8, const uint8_t* v8, const uint16_t* top, int64_t blocks, float* m, float* v, void* stream) {
    if (blocks < 0 || !m8 || !v8 || !top || !m || !v) return az_fail("az_adamw_decode8: null pointer");
    if (((uintptr_t)m8 | (uintptr_t)v8 | (uintptr_t)top | (uintptr_t)m | (uintptr_t)v) % 16)
        return az_fail("az_adamw_decode8: buffers are aligned to 16 bytes");
    if (blocks == 0) return 0;
    hipLaunchKernelGGL(k_adamw_decode, dim3(adamw_grid(blocks)), dim3(ADAMW_THREADS), 0, (hipStream_t)stream, m8, v8, top, (long)blocks, m, v);
    AZ_LAUNCH_CHECK("k_adamw_decode");
    return 0;
}

int az_adamw_encode8(const float* m, const float* v, int64_t blocks, uint8_t* m8, uint8_t* v8, uint16_t* top, void* stream) {
    if (blocks < 0 || !m8 || !v8 || !top || !m || !v) return az_fail("az_adamw_encode8: null pointer");
    if (((uintptr_t)m8 | (uintptr_t)v8 | (uintptr_t)top | (uintptr_t)m | (uintptr_t)v) % 16)
        return az_fail("az_adamw_encode8: buffers are aligned to 16 bytes");
    if (blocks == 0) return 0;
    hipLaunchKernelGGL(k_adamw_encode, dim3(adamw_grid(blocks)), dim3(ADAMW_THREADS), 0, (hipStream_t)stream, m, v, (long)blocks, m8, v8, top);
    AZ_LAUNCH_CHECK("k_adamw_encode");
    return 0;
}

}  // extern "C"
