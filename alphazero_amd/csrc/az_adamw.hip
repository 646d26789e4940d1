// az_adamw.hip -- the AdamW step over all tensors of a network in one launch, moments in 32 or in 8 bits (the
// reference trains with SGD: alphazero/training.py:27-29; az_sgd_momentum in az_train.hip).
//
//   t = t + 1
//   m = (b1 * m) + ((1 - b1) * g)          v = (b2 * v) + ((1 - b2) * (g * g))
//   p = p * (1 - lr * wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The tensors lie behind each other in flat buffers, each from a multiple of 256 elements on (the gaps are zero and stay
// zero); tensors with the same settings form a run.  The step count lives in device memory, so that a launch recorded
// in a HIP graph counts on: every workgroup reads it first, the last one to finish writes it.
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

#define ADAMW_BLOCK 256          // elements: four of each lane of a wave
#define ADAMW_THREADS 256
#define ADAMW_GOLDEN 0x9E3779B97F4A7C15ull

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

struct AdamwRuns { az_adamw_run r[AZ_ADAMW_MAX_RUNS]; int n; };
struct AdamwScalars { float keep, step, root, b1, c1, b2, c2, eps; int half; };

__device__ __forceinline__ uint64_t adamw_mix(uint64_t z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

__device__ __forceinline__ uint32_t adamw_wave_max(uint32_t v) {
#pragma unroll
    for (int bit = 1; bit < 64; bit <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, bit, 64));
    return v;
}

// leading bits of the largest magnitude of a block, rounded up
__device__ __forceinline__ int adamw_top(uint32_t most) { return most > 0x7F800000u ? 0x7FF : (int)((most + 0xFFFFFu) >> 20); }

__device__ __forceinline__ uint32_t adamw_code_m(float x, uint32_t r, int top) {
    const uint32_t a = __float_as_uint(x) & 0x7FFFFFFFu;
    const int q = a > 0x7F800000u ? 0x7FF : (int)((a + (r << 4)) >> 20), lowest = max(top - 126, 1);
    const int up = __uint_as_float(a) * 131072.0f > (float)(2 * r + 1) * __uint_as_float((uint32_t)lowest << 20) ? lowest - (top - 127) : 0;
    const int k = q >= lowest ? q - (top - 127) : up;
    return (uint32_t)k | (k ? (__float_as_uint(x) >> 24) & 0x80u : 0u);
}

__device__ __forceinline__ uint32_t adamw_code_v(float x, uint32_t r, int top) {
    const uint32_t a = __float_as_uint(x) & 0x7FFFFFFFu;
    const int q = a > 0x7F800000u ? 0x7FF : (int)((a + (r << 4)) >> 20);
    return a ? (uint32_t)(max(q, max(top - 254, 1)) - (top - 255)) : 0u;
}

__device__ __forceinline__ float adamw_value(uint32_t k, int top, int codes) {
    return k ? __uint_as_float((uint32_t)((int)k + top - codes) << 20) : 0.0f;
}

__device__ __forceinline__ float adamw_value_m(uint32_t c, int top) {
    return __uint_as_float(__float_as_uint(adamw_value(c & 127u, top, 127)) | ((c & 0x80u) << 24));
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
    const int64_t t = q.step[0] + 1;
    if (tid < runs.n) {
        const az_adamw_run& r = runs.r[tid];
        const double lr = lr_dev ? lr_dev[r.lr_index] : r.lr;
        AdamwScalars s;
        s.keep = (float)(1.0 - lr * r.weight_decay);
        s.step = (float)(lr / -expm1((double)t * log(r.beta1)));
        s.root = (float)(1.0 / sqrt(-expm1((double)t * log(r.beta2))));
        s.b1 = (float)r.beta1; s.c1 = (float)(1.0 - r.beta1);
        s.b2 = (float)r.beta2; s.c2 = (float)(1.0 - r.beta2);
        s.eps = (float)r.eps; s.half = r.half;
        sc[tid] = s;
    }
    __syncthreads();
    const uint64_t key = adamw_mix(seed + ADAMW_GOLDEN * (uint64_t)t);
    int run = 0;
    for (long blk = (long)blockIdx.x * (ADAMW_THREADS / 64) + (tid >> 6); blk < blocks; blk += (long)gridDim.x * (ADAMW_THREADS / 64)) {
        while (run + 1 < runs.n && blk >= runs.r[run + 1].first_block) ++run;
        const AdamwScalars s = sc[run];
        const long at = blk * ADAMW_BLOCK + lane * 4;
        f32x4 p = *reinterpret_cast<const f32x4*>(q.p + at), g, m, v;
        if (s.half) {
            const bf16x4 h = *reinterpret_cast<const bf16x4*>(reinterpret_cast<const __bf16*>(q.g16) + at);
            g = __builtin_convertvector(h, f32x4);
            // a parameter that is not its master's rounding was written by somebody else (a checkpoint loaded): it counts
            const bf16x4 cur = *reinterpret_cast<const bf16x4*>(reinterpret_cast<const __bf16*>(q.p16) + at);
            const u16x4 have = __builtin_bit_cast(u16x4, cur), mine = __builtin_bit_cast(u16x4, __builtin_convertvector(p, bf16x4));
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = have[i] != mine[i] ? (float)cur[i] : p[i];
        } else g = *reinterpret_cast<const f32x4*>(q.g + at);
        if constexpr (BITS == 32) {
            m = *reinterpret_cast<const f32x4*>(q.m + at);
            v = *reinterpret_cast<const f32x4*>(q.v + at);
        } else {
            const uint32_t cm = *reinterpret_cast<const uint32_t*>(q.m8 + at), cv = *reinterpret_cast<const uint32_t*>(q.v8 + at);
            const int tm = q.top[2 * blk], tv = q.top[2 * blk + 1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                m[i] = adamw_value_m((cm >> (8 * i)) & 255u, tm);
                v[i] = adamw_value((cv >> (8 * i)) & 255u, tv, 255);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = m[i] * s.b1 + g[i] * s.c1;
            v[i] = v[i] * s.b2 + (g[i] * g[i]) * s.c2;
            p[i] = p[i] * s.keep - s.step * m[i] / (sqrtf(v[i]) * s.root + s.eps);
        }
        *reinterpret_cast<f32x4*>(q.p + at) = p;
        if (s.half) *reinterpret_cast<bf16x4*>(reinterpret_cast<__bf16*>(q.p16) + at) = __builtin_convertvector(p, bf16x4);
        if constexpr (BITS == 32) {
            *reinterpret_cast<f32x4*>(q.m + at) = m;
            *reinterpret_cast<f32x4*>(q.v + at) = v;
        } else {
            uint32_t am = 0, av = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                am = max(am, __float_as_uint(m[i]) & 0x7FFFFFFFu);
                av = max(av, __float_as_uint(v[i]) & 0x7FFFFFFFu);
            }
            const int tm = adamw_top(adamw_wave_max(am)), tv = adamw_top(adamw_wave_max(av));
            const uint64_t counter = (uint64_t)at / 2;                    // two numbers for every four elements
            const uint64_t rm = adamw_mix(counter * ADAMW_GOLDEN + key), rv = adamw_mix((counter + 1) * ADAMW_GOLDEN + key);
            uint32_t cm = 0, cv = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                cm |= adamw_code_m(m[i], (uint32_t)(rm >> (16 * i)) & 0xFFFFu, tm) << (8 * i);
                cv |= adamw_code_v(v[i], (uint32_t)(rv >> (16 * i)) & 0xFFFFu, tv) << (8 * i);
            }
            *reinterpret_cast<uint32_t*>(q.m8 + at) = cm;
            *reinterpret_cast<uint32_t*>(q.v8 + at) = cv;
            if (lane == 0) { q.top[2 * blk] = (uint16_t)tm; q.top[2 * blk + 1] = (uint16_t)tv; }
        }
    }
    // the last workgroup to come here has seen every other one read the step count
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        if (atomicAdd(q.arrived, 1) == (int)gridDim.x - 1) { q.arrived[0] = 0; q.step[0] = t; }
    }
}

__global__ void __launch_bounds__(ADAMW_THREADS)
k_adamw_decode(const uint8_t* __restrict__ m8, const uint8_t* __restrict__ v8, const uint16_t* __restrict__ top, long blocks,
               float* __restrict__ m, float* __restrict__ v) {
    const int lane = threadIdx.x & 63;
    for (long blk = (long)blockIdx.x * 4 + (threadIdx.x >> 6); blk < blocks; blk += (long)gridDim.x * 4) {
        const long at = blk * ADAMW_BLOCK + lane * 4;
        const uint32_t cm = *reinterpret_cast<const uint32_t*>(m8 + at), cv = *reinterpret_cast<const uint32_t*>(v8 + at);
        const int tm = top[2 * blk], tv = top[2 * blk + 1];
        f32x4 a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = adamw_value_m((cm >> (8 * i)) & 255u, tm);
            b[i] = adamw_value((cv >> (8 * i)) & 255u, tv, 255);
        }
        *reinterpret_cast<f32x4*>(m + at) = a;
        *reinterpret_cast<f32x4*>(v + at) = b;
    }
}

// (values that are no codes' -- moments that were kept in 32 bits -- are rounded to the nearest leading bits)
__global__ void __launch_bounds__(ADAMW_THREADS)
k_adamw_encode(const float* __restrict__ m, const float* __restrict__ v, long blocks, uint8_t* __restrict__ m8,
               uint8_t* __restrict__ v8, uint16_t* __restrict__ top) {
    const int lane = threadIdx.x & 63;
    for (long blk = (long)blockIdx.x * 4 + (threadIdx.x >> 6); blk < blocks; blk += (long)gridDim.x * 4) {
        const long at = blk * ADAMW_BLOCK + lane * 4;
        const f32x4 a = *reinterpret_cast<const f32x4*>(m + at), b = *reinterpret_cast<const f32x4*>(v + at);
        uint32_t am = 0, av = 0, cm = 0, cv = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            am = max(am, __float_as_uint(a[i]) & 0x7FFFFFFFu);
            av = max(av, __float_as_uint(b[i]) & 0x7FFFFFFFu);
        }
        const int tm = adamw_top(adamw_wave_max(am)), tv = adamw_top(adamw_wave_max(av));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cm |= adamw_code_m(a[i], 0x8000u, tm) << (8 * i);
            cv |= adamw_code_v(b[i], 0x8000u, tv) << (8 * i);
        }
        *reinterpret_cast<uint32_t*>(m8 + at) = cm;
        *reinterpret_cast<uint32_t*>(v8 + at) = cv;
        if (lane == 0) { top[2 * blk] = (uint16_t)tm; top[2 * blk + 1] = (uint16_t)tv; }
    }
}

static unsigned adamw_grid(long blocks) {
    const long need = (blocks + 3) / 4;
    return (unsigned)(need < 2048 ? need : 2048);
}

extern "C" {

int az_adamw_step(const az_adamw_buffers* b, int64_t blocks, const az_adamw_run* runs, int32_t num_runs, int32_t state_bits,
                  const double* lr_dev, uint64_t seed, const float* guard_dev, float guard_limit, int32_t* withheld_dev,
                  void* stream) {
    if (!b || !runs || blocks < 0) return az_fail("az_adamw_step: null pointer");
    if (num_runs < 1 || num_runs > AZ_ADAMW_MAX_RUNS) return az_fail("az_adamw_step: 1 to 32 runs");
    if (state_bits != 8 && state_bits != 32) return az_fail("az_adamw_step: moments in 8 or in 32 bits");
    if (!b->p || !b->step || !b->arrived || (state_bits == 32 ? !b->m || !b->v : !b->m8 || !b->v8 || !b->top) || (guard_dev && !withheld_dev))
        return az_fail("az_adamw_step: null pointer");
    AdamwRuns r = {};
    r.n = num_runs;
    for (int i = 0; i < num_runs; ++i) {
        r.r[i] = runs[i];
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
