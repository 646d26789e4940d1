// az_norm.hip -- group norm with an activation and a residual sum, channels last: the normalisation of the residual
// tower's blocks for networks without batch statistics (models.AlphaZero(norm='group'); the reference's blocks use
// batch-norm: alphazero/models.py:6-28).
//
//   x [N][HW][C], G groups of Cg = C / G channels, n = HW * Cg values per (sample, group):
//     mean = sum(x) / n    var = sum(x^2) / n - mean^2    rstd = 1 / sqrt(var + eps)
//     z = (x - mean) * rstd * w[c] + b[c] (+ res)         y = act(z)
//   backward, dz = dy * act'(z), a = dz * w[c], xhat = (x - mean) * rstd:
//     db = sum dz    dw = sum dz * xhat    dres = dz    dx = rstd * (a - sum_g(a) / n - xhat * sum_g(a * xhat) / n)
//
// Statistics are summed and kept in 64 bits, of x less the first value x0 of its group: with d = x - x0 one pass over x gives
// the mean x0 + E[d] and the variance E[d^2] - E[d]^2 without the cancellation that E[x^2] - mean^2 has where the mean is
// large against the spread (d is of the spread's size unless x0 lies far out, by at most sqrt(n) spreads).  The sign of z --
// the border at which relu cuts the gradient -- can be decided exactly: z is formed in 32 bits, and where it lies closer to
// zero than its rounding errors it is formed again in 64.  Sums of the backward pass: of a thread in 32 bits, with up to 48
// terms for a group of a sample held in registers (8 in the two passes) and GN_CHAIN for a channel; of chunks, and of
// workgroups' parts, in 64.
//
// Bound by memory where there is much of it (one MI355X; a copy reaches 4.7 TB/s, 6.9 where the caches hold it):
//   8192 x 42 cells x 128 channels, float32, forward with residual and relu     97 us for 528 MB    5.4 TB/s
//   4096 x 42 x 128, bfloat16, with residual and relu     forward 29 us for 132 MB, backward 46 + 4 us for 220 MB    4.5, 4.4 TB/s
//   128 x 42 x 256, float32, as in a training step of the shipped batch         forward 6, backward 8 + 3 us
//   1 x 42 x 256, float32, one position                                         3.8 us, a launch that does nothing 2.8
//   61 x 361 x 192, float16, silu     forward 10.6, backward 15 + 4 us: one workgroup of 1024 a compute unit loads, waits,
//     computes and stores in turn (0.5 us of the forward pass are the subtraction of x0)
//   3 x 4096 x 320, bfloat16, silu    5.7 + 7.5 us: two launches, x from the caches the second time
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/azhip.h"
#include "az_host.h"

#define GN_THREADS 256
#define GN_CHAIN 2048         // rows that a thread adds up in 32 bits for dweight and dbias, at most; all sums of such sums in 64

struct GnArgs {
    const void* x; const void* dy; const void* res; const void* w; const void* b;
    void* y; void* dx; void* dres;
    double* stats;                    // [N][G][2] mean, rstd
    double* part;                     // [N][G][pieces * chunks][2] partial sums
    float* dpart;                     // [N * chunks][2][C] partial sums of dz and dz * xhat
    long N;
    int HW, C, G, Cg, cpg;            // cpg: vectors per group
    int cb, gb, rb, sb, tb;           // held samples: bits of column, group, row, sample in a team's thread; of the team
    int gs, cw, rstep, share;         // others: groups of a slice, vectors of a group (or piece of one), rows of a workgroup
    int slices, pieces, chunks, rows; // rows per chunk
    int together;                     // slices share lines of memory
    int walkers;                      // teams that share a slice's samples in the backward pass
    int wtype, wide;                  // wide: weight and bias may be read 16 bytes at a time
    float low, near;                  // relu: 0, 2^-20 (below); none: NaN, 0 -- no value is at or below a NaN
    double eps, count, inv;           // count: values of a group, and 1 / count
};

template <typename T, int VW> struct GnVec { typedef T type __attribute__((ext_vector_type(VW))); };
template <typename T> struct GnVec<T, 1> { typedef T type; };

template <typename T, int VW>
__device__ __forceinline__ void gn_load(const void* base, long at, float (&out)[VW]) {
    typedef typename GnVec<T, VW>::type V;
    const V v = *reinterpret_cast<const V*>(reinterpret_cast<const T*>(base) + at);
    if constexpr (VW == 1) out[0] = (float)v;
    else {
#pragma unroll
        for (int i = 0; i < VW; ++i) out[i] = (float)v[i];
    }
}

// (one rounding, to the nearest, from 32 bits to the tensor's type)
template <typename T, int VW>
__device__ __forceinline__ void gn_store(void* base, long at, const float (&in)[VW]) {
    typedef typename GnVec<T, VW>::type V;
    V v;
    if constexpr (VW == 1) v = (T)in[0];
    else {
#pragma unroll
        for (int i = 0; i < VW; ++i) v[i] = (T)in[i];
    }
    *reinterpret_cast<V*>(reinterpret_cast<T*>(base) + at) = v;
}

// VW neighbouring entries of weight or bias; `otherwise` where there is none
template <int VW, typename P>
__device__ __forceinline__ void gn_param_of(const void* p, int at, bool wide, float (&out)[VW]) {
    if constexpr (VW > 1) {
        if (wide) {                                                   // 16-byte aligned
            if constexpr (sizeof(P) == 4 && VW == 8) {
                float lo[4], hi[4];
                gn_load<P, 4>(p, at, lo);
                gn_load<P, 4>(p, at + 4, hi);
#pragma unroll
                for (int i = 0; i < 4; ++i) { out[i] = lo[i]; out[4 + i] = hi[i]; }
            } else gn_load<P, VW>(p, at, out);
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < VW; ++i) out[i] = (float)reinterpret_cast<const P*>(p)[at + i];
}
template <int VW>
__device__ __forceinline__ void gn_param(const void* p, int type, bool wide, int at, float otherwise, float (&out)[VW]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < VW; ++i) out[i] = otherwise;
    } else if (type == AZ_F32) gn_param_of<VW, float>(p, at, wide, out);
    else if (type == AZ_BF16) gn_param_of<VW, __bf16>(p, at, wide, out);
    else gn_param_of<VW, _Float16>(p, at, wide, out);
}

// x of the lane whose index differs in one bit.  (row_ror:4 is that for bit 4 once the sums over bit 8 are made.)
template <int CTRL> __device__ __forceinline__ uint32_t gn_dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false);
}
template <int CTRL> __device__ __forceinline__ float gn_dpp(float x) { return __uint_as_float(gn_dpp<CTRL>(__float_as_uint(x))); }
template <int CTRL> __device__ __forceinline__ double gn_dpp(double x) {
    return __hiloint2double((int)gn_dpp<CTRL>((uint32_t)__double2hiint(x)), (int)gn_dpp<CTRL>((uint32_t)__double2loint(x)));
}
__device__ __forceinline__ float gn_swizzle4(float x) { return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(x), (4 << 10) | 0x1f)); }
__device__ __forceinline__ double gn_swizzle4(double x) {
    return __hiloint2double(__builtin_amdgcn_ds_swizzle(__double2hiint(x), (4 << 10) | 0x1f),
                            __builtin_amdgcn_ds_swizzle(__double2loint(x), (4 << 10) | 0x1f));
}
// sums over lane bit 16 / 32: a register's odd rows of 16 (upper half) change places with a copy's even rows (lower half)
__device__ __forceinline__ float gn_add16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float gn_add32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ double gn_add16(double x) {
    const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)__double2hiint(x), (uint32_t)__double2hiint(x), false, false);
    const auto l = __builtin_amdgcn_permlane16_swap((uint32_t)__double2loint(x), (uint32_t)__double2loint(x), false, false);
    return __hiloint2double((int)h[0], (int)l[0]) + __hiloint2double((int)h[1], (int)l[1]);
}
__device__ __forceinline__ double gn_add32(double x) {
    const auto h = __builtin_amdgcn_permlane32_swap((uint32_t)__double2hiint(x), (uint32_t)__double2hiint(x), false, false);
    const auto l = __builtin_amdgcn_permlane32_swap((uint32_t)__double2loint(x), (uint32_t)__double2loint(x), false, false);
    return __hiloint2double((int)h[0], (int)l[0]) + __hiloint2double((int)h[1], (int)l[1]);
}

// sums of (s, q) over the lanes of a wave whose index differs in the bits of `mask` only; all of them get the same bits
template <typename F>
__device__ __forceinline__ void gn_wave_sum(F& s, F& q, int mask) {
    if (mask & 32) { s = gn_add32(s); q = gn_add32(q); }
    if (mask & 16) { s = gn_add16(s); q = gn_add16(q); }
    if (mask & 8) { s += gn_dpp<0x128>(s); q += gn_dpp<0x128>(q); }                          // row_ror:8
    if (mask & 4) {
        if (mask & 8) { s += gn_dpp<0x124>(s); q += gn_dpp<0x124>(q); }                      // row_ror:4
        else { s += gn_swizzle4(s); q += gn_swizzle4(q); }
    }
    if (mask & 2) { s += gn_dpp<0x4E>(s); q += gn_dpp<0x4E>(q); }                            // quad_perm 2 3 0 1
    if (mask & 1) { s += gn_dpp<0xB1>(s); q += gn_dpp<0xB1>(q); }                            // quad_perm 1 0 3 2
}

// the same over a workgroup whose threads are one team (bits 6 and up of `mask`: waves); every thread comes here
template <typename F>
__device__ __forceinline__ void gn_team_sum(F& s, F& q, int mask, F (*lds)[2]) {
    gn_wave_sum(s, q, mask);
    if (mask >> 6) {
        const int tid = threadIdx.x, waves = blockDim.x >> 6;
        __syncthreads();
        lds[tid][0] = s; lds[tid][1] = q;
        __syncthreads();
        s = q = (F)0;
        for (int w = 0; w < waves; ++w)
            if ((((w ^ (tid >> 6)) << 6) & ~mask) == 0) { s += lds[(w << 6) + (tid & 63)][0]; q += lds[(w << 6) + (tid & 63)][1]; }
    }
}

// mean and 1 / sqrt(var + eps) of a group's values from sums s and q of x - x0 and its square
__device__ __forceinline__ void gn_moments(double s, double q, double x0, const GnArgs& a, double& mean, double& rstd) {
    // (the product is corrected to the quotient)
    double m = s * a.inv;
    m = fma(fma(-m, a.count, s), a.inv, m);
    mean = x0 + m;
    const double v = fmax(fma(q, a.inv, -m * m), 0.0) + a.eps;
    // the instruction is good to some 2^-23; each step doubles the digits
    double y = __builtin_amdgcn_rsq(v);
    y *= fma(-0.5 * v * y, y, 1.5);
    rstd = y * fma(-0.5 * v * y, y, 1.5);
}

// (addresses: a scalar base, the same for a wave, and 32 bits of a lane's own; two registers an address and vector otherwise)
template <typename T, int VW> __device__ __forceinline__ typename GnVec<T, VW>::type gn_raw(const void* base, long at, uint32_t lane) {
    return *reinterpret_cast<const typename GnVec<T, VW>::type*>(reinterpret_cast<const char*>(base) + at + lane);
}
template <typename T, int VW> __device__ __forceinline__ float gn_at(const typename GnVec<T, VW>::type& v, int i) {
    if constexpr (VW == 1) return (float)v;
    else return (float)v[i];
}
template <typename T, int VW> __device__ __forceinline__ void gn_get(const void* base, long at, uint32_t lane, float (&out)[VW]) {
    gn_load<T, VW>(reinterpret_cast<const char*>(base) + at + lane, 0, out);
}
template <typename T, int VW> __device__ __forceinline__ void gn_put(void* base, long at, uint32_t lane, const float (&in)[VW]) {
    gn_store<T, VW>(reinterpret_cast<char*>(base) + at + lane, 0, in);
}

// ---- samples too large for registers: two passes over chunks of their rows -------------------------------------------
// A workgroup has a slice (gs groups; or a piece of one that is wider than 256 vectors) of a chunk of a sample's rows, its
// threads side by side along memory: thread = row * gs * cw + group * cw + column.  First pass: sums; second: the rest,
// whose every workgroup adds the parts of its groups up again.
// Workgroups go to the card's 8 dies in turn; where the slices of a sample share lines of memory, neighbours in this
// numbering are on one die, whose L2 then fetches a line once.
__device__ __forceinline__ unsigned gn_block(const GnArgs& a) {
    const unsigned b = blockIdx.x, die = b & 7, per = gridDim.x >> 3, more = gridDim.x & 7;
    return a.together ? die * per + min(die, more) + (b >> 3) : b;
}

struct GnPlace {
    long n; int g, gl, col, row, chunk, piece, width, rows; bool on;
    long base;                        // bytes to the chunk: the same for the workgroup
    uint32_t lane, step;              // bytes on to this thread's first row, and to its next
};

__device__ __forceinline__ GnPlace gn_place(const GnArgs& a, int VW, int size) {
    GnPlace p;
    unsigned u = gn_block(a);
    const int slice = u % a.slices, t = threadIdx.x; u /= a.slices;
    p.piece = u % a.pieces; u /= a.pieces;
    p.chunk = u % a.chunks;
    p.n = u / a.chunks;
    p.width = a.gs * a.cw;
    p.row = t / p.width;
    p.gl = t % p.width / a.cw;
    p.col = t % a.cw + p.piece * a.cw;
    p.g = slice * a.gs + p.gl;
    p.on = p.row < a.rstep && p.col < a.cpg && p.g < a.G;
    p.rows = min(a.rows, a.HW - p.chunk * a.rows);
    p.base = (p.n * a.HW + (long)p.chunk * a.rows) * a.C * size;
    p.lane = ((uint32_t)p.row * a.C + p.g * a.Cg + p.col * VW) * size;
    p.step = (uint32_t)a.rstep * a.C * size;
    return p;
}

// (s, q) over the threads of each group -> the workgroup's entry of that group's parts; a.share neighbouring threads add
// for a group
__device__ __forceinline__ void gn_put_parts(const GnArgs& a, const GnPlace& p, double s, double q, double (*lds)[2]) {
    const int t = threadIdx.x, gl = t / a.share, g = p.g - p.gl + gl;
    lds[t][0] = s; lds[t][1] = q;
    __syncthreads();
    s = q = 0.0;
    if (gl < a.gs)
        for (int k = t % a.share; k < a.rstep * a.cw; k += a.share) {
            const int from = k / a.cw * p.width + gl * a.cw + k % a.cw;
            s += lds[from][0]; q += lds[from][1];
        }
    gn_wave_sum(s, q, a.share - 1);
    if (gl < a.gs && g < a.G && t % a.share == 0) {
        double* out = a.part + ((p.n * a.G + g) * (a.pieces * a.chunks) + p.piece * a.chunks + p.chunk) * 2;
        out[0] = s; out[1] = q;
    }
}

// the sums of the parts of this thread's group, in order
__device__ __forceinline__ void gn_get_parts(const GnArgs& a, const GnPlace& p, double& s, double& q, double (*lds)[2]) {
    const int t = threadIdx.x, parts = a.pieces * a.chunks, gl = t / a.share, g = p.g - p.gl + gl;
    s = q = 0.0;
    if (gl < a.gs && g < a.G) {
        const double* in = a.part + (p.n * a.G + g) * parts * 2;
        for (int k = t % a.share; k < parts; k += a.share) { s += in[2 * k]; q += in[2 * k + 1]; }
    }
    gn_wave_sum(s, q, a.share - 1);
    if (t % a.share == 0) { lds[gl][0] = s; lds[gl][1] = q; }
    __syncthreads();
    s = lds[p.gl][0]; q = lds[p.gl][1];
}

// the first value of this thread's group in its sample
template <typename T> __device__ __forceinline__ T gn_first(const GnArgs& a, const GnPlace& p) {
    return gn_raw<T, 1>(a.x, p.base - (long)p.chunk * a.rows * a.C * (long)sizeof(T), p.on ? (uint32_t)(p.g * a.Cg) * (uint32_t)sizeof(T) : 0);
}
template <typename T> __device__ __forceinline__ double gn_here(T x) {
    // (x as something that is not known before now: its conversion is not made, and the load of x not waited for, further up;
    // 3 x 4096 cells x 320 channels, bfloat16: 5.6 against 6.0 us)
    if constexpr (sizeof(T) == 4) {
        asm volatile("" : "+v"(x));
        return x;
    } else {
        uint16_t bits = __builtin_bit_cast(uint16_t, x);
        asm volatile("" : "+v"(bits));
        return (float)__builtin_bit_cast(T, bits);
    }
}

template <typename T, int VW>
__global__ void __launch_bounds__(GN_THREADS)
k_gn_stats(GnArgs a) {
    __shared__ double lds[GN_THREADS][2];
    const GnPlace p = gn_place(a, VW, sizeof(T));
    double s = 0.0, q = 0.0;
    const T x0 = gn_first<T>(a, p);
    if (p.on) {
        typedef typename GnVec<T, VW>::type V;
        const auto add = [&](const V& x, double o) {
#pragma unroll
            for (int i = 0; i < VW; ++i) { const double d = gn_at<T, VW>(x, i) - o; s += d; q = fma(d, d, q); }
        };
        constexpr int U = 4;                                              // rows whose loads are on their way together
        uint32_t at = p.lane;
        int r = p.row;
        for (; r + (U - 1) * a.rstep < p.rows; r += U * a.rstep, at += U * p.step) {
            V x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = gn_raw<T, VW>(a.x, p.base, at + u * p.step);
            const double o = gn_here<T>(x0);
#pragma unroll
            for (int u = 0; u < U; ++u) add(x[u], o);
        }
        for (; r < p.rows; r += a.rstep, at += p.step) {
            const V x = gn_raw<T, VW>(a.x, p.base, at);
            add(x, gn_here<T>(x0));
        }
    }
    gn_put_parts(a, p, s, q, lds);
}

// 1 / (1 + exp(-z)) by the hardware's 2^x and reciprocal, each good to 2^-23: with log2(e) and its product rounded to 24 bits
// (1.22 * 2^-24 together) off by at most (0.61 |z| + 2.5) 2^-23 of itself, down to z = -87; what is below 2^-126 may be 0
__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z)); }
__device__ __forceinline__ float gn_silu(float z) { return z * gn_sigmoid(z); }

template <bool SILU> __device__ __forceinline__ float gn_act(float z, float low) {
    if constexpr (SILU) return gn_silu(z);
    else return z <= low ? 0.0f : z;                                  // (a NaN stays one)
}

// x - mean keeps its precision where the mean is large against the spread, with the mean as two floats mh + ml:
// xhat = (x - mh) * rs - ml * rs
struct GnNorm { double mean, rstd; float mh, rs, off, slack; };

__device__ __forceinline__ GnNorm gn_norm(double mean, double rstd) {
    GnNorm k;
    k.mean = mean; k.rstd = rstd;
    k.mh = (float)mean; k.rs = (float)rstd;
    k.off = -(float)(mean - (double)k.mh) * k.rs;
    k.slack = 0.0f;
    return k;
}
__device__ __forceinline__ float gn_xhat(const GnNorm& k, float x) { return fmaf(x - k.mh, k.rs, k.off); }

template <int VW>
__device__ __forceinline__ void gn_affine(const GnNorm& k, float (&w)[VW], float (&b)[VW]) {       // z = (x - mh) * w + b
#pragma unroll
    for (int i = 0; i < VW; ++i) { b[i] = fmaf(k.off, w[i], b[i]); w[i] *= k.rs; }
}

// (wmax: the largest |weight| of the thread's channels)
__device__ __forceinline__ GnNorm gn_saved(const GnArgs& a, long n, int g, float wmax) {
    GnNorm k = gn_norm(a.stats[(n * a.G + g) * 2], a.stats[(n * a.G + g) * 2 + 1]);
    k.slack = fabsf(k.off) * wmax * a.near;
    return k;
}
template <int VW> __device__ __forceinline__ float gn_largest(const float (&w)[VW]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < VW; ++i) m = fmaxf(m, fabsf(w[i]));
    return m;
}

#define GN_ROWS(VW) ((VW) == 8 ? 2 : 4)          // rows whose loads are on their way together

template <typename T, int VW, bool SILU>
__global__ void __launch_bounds__(GN_THREADS)
k_gn_apply(GnArgs a) {
    __shared__ double lds[GN_THREADS][2];
    const GnPlace p = gn_place(a, VW, sizeof(T));
    double s, q, mean, rstd;
    const float x0 = (float)gn_first<T>(a, p);
    gn_get_parts(a, p, s, q, lds);
    if (!p.on) return;
    gn_moments(s, q, x0, a, mean, rstd);
    if (a.stats && p.chunk == 0 && p.col == 0 && p.row == 0) {
        a.stats[(p.n * a.G + p.g) * 2] = mean;
        a.stats[(p.n * a.G + p.g) * 2 + 1] = rstd;
    }
    const GnNorm k = gn_norm(mean, rstd);
    float w[VW], b[VW];
    gn_param<VW>(a.w, a.wtype, a.wide, p.g * a.Cg + p.col * VW, 1.0f, w);
    gn_param<VW>(a.b, a.wtype, a.wide, p.g * a.Cg + p.col * VW, 0.0f, b);
    gn_affine<VW>(k, w, b);
    constexpr int U = GN_ROWS(VW);
    uint32_t at = p.lane;
    for (int r0 = p.row; r0 < p.rows; r0 += U * a.rstep, at += U * p.step) {
        float x[U][VW], z[U][VW] = {};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (r0 + u * a.rstep < p.rows) {
                gn_get<T, VW>(a.x, p.base, at + u * p.step, x[u]);
                if (a.res) gn_get<T, VW>(a.res, p.base, at + u * p.step, z[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (r0 + u * a.rstep < p.rows) {
#pragma unroll
                for (int i = 0; i < VW; ++i) z[u][i] = gn_act<SILU>(fmaf(x[u][i] - k.mh, w[i], b[i]) + z[u][i], a.low);
                gn_put<T, VW>(a.y, p.base, at + u * p.step, z[u]);
            }
        }
    }
}

// dz of one value.  relu: z in 32 bits is off by less than 8 * 2^-24 * (|xhat w| + |b| + |off w|) (three roundings of xhat
// and of its part off, one each of the product and the two sums, and |res| <= |xhat w| + |b| where z is small); closer to
// zero than twice that `near` is set, and gn_relu_exact says.
template <bool SILU>
__device__ __forceinline__ float gn_dz(const GnArgs& a, const GnNorm& k, float x, float w, float b, float res, float dy, bool& near) {
    const float t = gn_xhat(k, x) * w, z = t + b + res;
    if constexpr (SILU) {
        const float sig = gn_sigmoid(z);
        return dy * (sig * fmaf(z, 1.0f - sig, 1.0f));
    }
    near |= fabsf(z) < fmaf(fabsf(t) + fabsf(b), a.near, k.slack);
    return z <= a.low ? 0.0f : dy;
}

// (Opaque copies: otherwise w and b in 64 bits are made ahead of the loop and kept, four registers a channel, and all
// channels' values are formed side by side.)
__device__ __forceinline__ float gn_relu_exact(const GnNorm& k, float x, float w, float b, float res, float dy) {
    asm volatile("" : "+v"(w), "+v"(b));
    float dz = ((double)x - k.mean) * k.rstd * (double)w + (double)b + (double)res <= 0.0 ? 0.0f : dy;
    asm volatile("" : "+v"(dz));
    return dz;
}

template <int VW, bool SILU>
__device__ __forceinline__ void gn_dz_row(const GnArgs& a, const GnNorm& k, const float (&x)[VW], const float (&w)[VW], const float (&b)[VW],
                                          const float (&res)[VW], float (&dy)[VW]) {
    bool near = false;
    float dz[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) dz[i] = gn_dz<SILU>(a, k, x[i], w[i], b[i], res[i], dy[i], near);
    if (!SILU && near) {
#pragma unroll
        for (int i = 0; i < VW; ++i) dz[i] = gn_relu_exact(k, x[i], w[i], b[i], res[i], dy[i]);
    }
#pragma unroll
    for (int i = 0; i < VW; ++i) dy[i] = dz[i];
}

// sums over a chunk of rows: of a and a * xhat per group, of dz and dz * xhat per channel; writes the residual's gradient
template <typename T, int VW, bool SILU>
__global__ void __launch_bounds__(GN_THREADS)
k_gn_bwd_sums(GnArgs a) {
    __shared__ double lds[GN_THREADS][2];
    __shared__ float sums[2 * VW][GN_THREADS];
    const GnPlace p = gn_place(a, VW, sizeof(T));
    double sa = 0.0, sx = 0.0;
    float dw[VW] = {}, db[VW] = {};
    if (p.on) {
        float w[VW], b[VW];
        gn_param<VW>(a.w, a.wtype, a.wide, p.g * a.Cg + p.col * VW, 1.0f, w);
        gn_param<VW>(a.b, a.wtype, a.wide, p.g * a.Cg + p.col * VW, 0.0f, b);
        const GnNorm k = gn_saved(a, p.n, p.g, gn_largest<VW>(w));
        constexpr int U = GN_ROWS(VW);
        uint32_t at = p.lane;
        for (int r0 = p.row; r0 < p.rows; r0 += U * a.rstep, at += U * p.step) {
            float x[U][VW], dy[U][VW], res[U][VW] = {};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r0 + u * a.rstep < p.rows) {
                    gn_get<T, VW>(a.x, p.base, at + u * p.step, x[u]);
                    gn_get<T, VW>(a.dy, p.base, at + u * p.step, dy[u]);
                    if (a.res) gn_get<T, VW>(a.res, p.base, at + u * p.step, res[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r0 + u * a.rstep < p.rows) {
                    gn_dz_row<VW, SILU>(a, k, x[u], w, b, res[u], dy[u]);
                    float fa = 0.0f, fx = 0.0f;
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
                        const float xhat = gn_xhat(k, x[u][i]), f = dy[u][i] * w[i];
                        db[i] += dy[u][i];
                        dw[i] = fmaf(dy[u][i], xhat, dw[i]);
                        fa += f;
                        fx = fmaf(f, xhat, fx);
                    }
                    sa += fa; sx += fx;
                    if (a.dres) gn_put<T, VW>(a.dres, p.base, at + u * p.step, dy[u]);
                }
            }
        }
    }
    if (a.dpart) {
#pragma unroll
        for (int i = 0; i < VW; ++i) { sums[2 * i][threadIdx.x] = db[i]; sums[2 * i + 1][threadIdx.x] = dw[i]; }
    }
    if (a.part) gn_put_parts(a, p, sa, sx, lds);
    if (!a.dpart) return;
    __syncthreads();
    for (int o = threadIdx.x; o < 2 * VW * p.width; o += GN_THREADS) {
        const int t = o % p.width, v = o / p.width, col = t % a.cw + p.piece * a.cw, g = p.g - p.gl + t / a.cw;
        double total = 0.0;
        for (int r = 0; r < a.rstep; ++r) total += sums[v][r * p.width + t];
        if (col < a.cpg && g < a.G) a.dpart[((p.n * a.chunks + p.chunk) * 2 + (v & 1)) * a.C + g * a.Cg + col * VW + (v >> 1)] = (float)total;
    }
}

template <typename T, int VW, bool SILU>
__global__ void __launch_bounds__(GN_THREADS)
k_gn_bwd_apply(GnArgs a) {
    __shared__ double lds[GN_THREADS][2];
    const GnPlace p = gn_place(a, VW, sizeof(T));
    double sa, sx;
    gn_get_parts(a, p, sa, sx, lds);
    if (!p.on) return;
    const float ma = (float)(sa * a.inv), mx = (float)(sx * a.inv);
    float w[VW], b[VW];
    gn_param<VW>(a.w, a.wtype, a.wide, p.g * a.Cg + p.col * VW, 1.0f, w);
    gn_param<VW>(a.b, a.wtype, a.wide, p.g * a.Cg + p.col * VW, 0.0f, b);
    const GnNorm k = gn_saved(a, p.n, p.g, gn_largest<VW>(w));
    // what the first pass wrote as the residual's gradient is dz, except where silu's was rounded to 16 bits
    const bool have = a.dres && (!SILU || sizeof(T) == 4);
    constexpr int U = GN_ROWS(VW);
    uint32_t at = p.lane;
    for (int r0 = p.row; r0 < p.rows; r0 += U * a.rstep, at += U * p.step) {
        float x[U][VW], dy[U][VW], res[U][VW] = {};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (r0 + u * a.rstep < p.rows) {
                gn_get<T, VW>(a.x, p.base, at + u * p.step, x[u]);
                gn_get<T, VW>(have ? a.dres : a.dy, p.base, at + u * p.step, dy[u]);
                if (a.res && !have) gn_get<T, VW>(a.res, p.base, at + u * p.step, res[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (r0 + u * a.rstep < p.rows) {
                if (!have) gn_dz_row<VW, SILU>(a, k, x[u], w, b, res[u], dy[u]);
#pragma unroll
                for (int i = 0; i < VW; ++i) dy[u][i] = (fmaf(dy[u][i], w[i], -ma) - gn_xhat(k, x[u][i]) * mx) * k.rs;
                gn_put<T, VW>(a.dx, p.base, at + u * p.step, dy[u]);
            }
        }
    }
}

// dw, db: the partial sums of `parts` workgroups, added in a fixed order in 64 bits.  One workgroup: 16 of the 2 C columns.
// (2 to 4 us.  In the launch before it, whose last workgroup would add the rows up, a counter would be needed that some
// earlier launch clears: not tried.)
__global__ void __launch_bounds__(1024)
k_gn_dparams(const float* __restrict__ dpart, long parts, int first, int C, int wtype, void* dw, void* db) {
    __shared__ double lds[64][17];
    const int col = first + blockIdx.x * 16 + (threadIdx.x & 15), r0 = threadIdx.x >> 4;
    double s = 0.0;
    if (col < 2 * C)
#pragma unroll 8
        for (long r = r0; r < parts; r += 64) s += (double)dpart[r * 2 * C + col];
    lds[r0][threadIdx.x & 15] = s;
    for (int half = 32; half > 0; half >>= 1) {
        __syncthreads();
        if (r0 < half) lds[r0][threadIdx.x & 15] += lds[r0 + half][threadIdx.x & 15];
    }
    if (r0 == 0 && col < 2 * C) {
        const float v = (float)lds[0][threadIdx.x & 15];
        void* out = col < C ? db : dw;
        const int at = col < C ? col : col - C;
        if (!out) return;
        if (wtype == AZ_F32) reinterpret_cast<float*>(out)[at] = v;
        else if (wtype == AZ_BF16) reinterpret_cast<__bf16*>(out)[at] = (__bf16)v;
        else reinterpret_cast<_Float16*>(out)[at] = (_Float16)v;
    }
}

// ---- samples held in registers -----------------------------------------------------------------------------------
// One pass over x (and dy, res): a team -- a wave, or a workgroup where a wave's registers do not hold a sample's slice --
// loads its slice (some groups of a sample, 256 bytes of each row where it can, or of several small samples), K vectors to a
// thread, and has everything else in registers: in float32, without a residual, 8 bytes of traffic a value instead of the
// two passes' 12, and backward 12 instead of 20.
// A thread holds VW neighbouring channels of one group in each of its rows.  The bits of its index in the team are, from
// the lowest: column within the group (cb), group within the slice (gb), row (rb), sample (sb).  Sums over a group are
// butterflies over the column and row bits, so a wave's loads run along memory whatever the group's width.
struct GnSeat { int col, gl, row, sample; };

__device__ __forceinline__ GnSeat gn_seat(const GnArgs& a, int t) {
    GnSeat p;
    p.col = t & ((1 << a.cb) - 1);
    p.gl = (t >> a.cb) & ((1 << a.gb) - 1);
    p.row = (t >> (a.cb + a.gb)) & ((1 << a.rb) - 1);
    p.sample = t >> (a.cb + a.gb + a.rb);
    return p;
}

template <typename T, int VW, int K, int THREADS, bool SILU>
__global__ void __launch_bounds__(THREADS)
k_gn_held(GnArgs a) {
    typedef typename GnVec<T, VW>::type V;
    __shared__ double lds[THREADS][2];
    const bool alone = a.tb == 6;                                     // a wave is a team
    const unsigned block = gn_block(a);
    const unsigned unit = alone ? block * (THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : block;
    const int slice = (int)(unit % (unsigned)a.slices);
    const long batch = unit / (unsigned)a.slices;
    if ((batch << a.sb) >= a.N) return;                               // (whole waves, or nobody)
    const GnSeat p = gn_seat(a, threadIdx.x & ((1 << a.tb) - 1));
    const long n0 = batch << a.sb, n = n0 + p.sample;
    const int g = (slice << a.gb) + p.gl, c = g * a.Cg + p.col * VW;
    const bool on = p.col < a.cpg && g < a.G && n < a.N;
    const long base = n0 * a.HW * a.C * (long)sizeof(T), step = ((long)a.C << a.rb) * (long)sizeof(T);
    const uint32_t lane = (uint32_t)(((p.sample * a.HW + p.row) * a.C + c) * (int)sizeof(T));
    V x[K], r[K] = {};
    // (the first value of this thread's group)
    const float x0 = (float)gn_raw<T, 1>(a.x, base, on ? lane - (uint32_t)((p.row * a.C + p.col * VW) * (int)sizeof(T)) : 0);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int row = p.row + (k << a.rb);
        x[k] = on && row < a.HW ? gn_raw<T, VW>(a.x, base + k * step, lane) : V{};
    }
    if (a.res) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int row = p.row + (k << a.rb);
            r[k] = on && row < a.HW ? gn_raw<T, VW>(a.res, base + k * step, lane) : V{};
        }
    }
    float w[VW], b[VW];
    gn_param<VW>(a.w, a.wtype, a.wide, on ? c : 0, 1.0f, w);
    gn_param<VW>(a.b, a.wtype, a.wide, on ? c : 0, 0.0f, b);
    double s = 0.0, q = 0.0, mean, rstd;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const double o = on && p.row + (k << a.rb) < a.HW ? x0 : 0.0f;    // (no value: zero, less zero)
#pragma unroll
        for (int i = 0; i < VW; ++i) { const double d = gn_at<T, VW>(x[k], i) - o; s += d; q = fma(d, d, q); }
    }
    const int groups = ((1 << a.gb) - 1) << a.cb, inside = (1 << (a.cb + a.gb + a.rb)) - 1;
    gn_team_sum(s, q, inside & ~groups, lds);
    gn_moments(s, q, x0, a, mean, rstd);
    if (a.stats && on && p.row == 0 && p.col == 0) {
        a.stats[(n * a.G + g) * 2] = mean;
        a.stats[(n * a.G + g) * 2 + 1] = rstd;
    }
    const GnNorm m = gn_norm(mean, rstd);
    gn_affine<VW>(m, w, b);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float z[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i)
            z[i] = gn_act<SILU>(fmaf(gn_at<T, VW>(x[k], i) - m.mh, w[i], b[i]) + gn_at<T, VW>(r[k], i), a.low);
        const int row = p.row + (k << a.rb);
        if (on && row < a.HW) gn_put<T, VW>(a.y, base + k * step, lane, z);
    }
}

// a workgroup's sum for one channel: v = 2 * (channel of the vector) + (0: db, 1: dw)
template <int VW>
__device__ __forceinline__ void gn_put_param(const GnArgs& a, int slice, int walker, int t, int v, double total) {
    const int col = t & ((1 << a.cb) - 1), g = (slice << a.gb) + (t >> a.cb);
    if (col < a.cpg && g < a.G) a.dpart[((long)walker * 2 + (v & 1)) * a.C + g * a.Cg + col * VW + (v >> 1)] = (float)total;
}

// A team walks over the samples of its slice, so that dw and db stay in its registers; the teams of a workgroup have the
// same slice and add theirs up at the end: one row of partial sums a workgroup.
// SILU: dz is kept in 32 bits; the other activations' dz is dy or zero and takes dy's place, in half the registers for a
// 16-bit type.
template <typename T, int VW, int K, int THREADS, bool SILU>
__global__ void __launch_bounds__(THREADS)
k_gn_bwd_held(GnArgs a) {
    typedef typename GnVec<T, VW>::type V;
    __shared__ float lds[THREADS][2];
    __shared__ alignas(8) float sums[2 * VW][THREADS];
    const bool alone = a.tb == 6;
    const unsigned block = gn_block(a);
    const int slice = block % a.slices, walker0 = block / a.slices;
    const int walker = alone ? walker0 * (THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : walker0;
    const long batches = (a.N + (1 << a.sb) - 1) >> a.sb;
    const GnSeat p = gn_seat(a, threadIdx.x & ((1 << a.tb) - 1));
    const int g = (slice << a.gb) + p.gl, c = g * a.Cg + p.col * VW;
    const bool seated = p.col < a.cpg && g < a.G;
    const int groups = ((1 << a.gb) - 1) << a.cb, inside = (1 << (a.cb + a.gb + a.rb)) - 1;
    const float inv = (float)a.inv;
    float w[VW], b[VW], dw[VW], db[VW];
    gn_param<VW>(a.w, a.wtype, a.wide, seated ? c : 0, 1.0f, w);
    gn_param<VW>(a.b, a.wtype, a.wide, seated ? c : 0, 0.0f, b);
#pragma unroll
    for (int i = 0; i < VW; ++i) dw[i] = db[i] = 0.0f;
    const float wmax = gn_largest<VW>(w);
    const long step = ((long)a.C << a.rb) * (long)sizeof(T);
    const uint32_t lane = (uint32_t)(((p.sample * a.HW + p.row) * a.C + c) * (int)sizeof(T));
    for (long batch = walker; batch < batches; batch += a.walkers) {
        const long n = (batch << a.sb) + p.sample;
        const bool on = seated && n < a.N;
        const long base = (batch << a.sb) * a.HW * a.C * (long)sizeof(T);
        V x[K], d[K], r[K] = {};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int row = p.row + (k << a.rb);
            const bool in = on && row < a.HW;
            x[k] = in ? gn_raw<T, VW>(a.x, base + k * step, lane) : V{};
            d[k] = in ? gn_raw<T, VW>(a.dy, base + k * step, lane) : V{};
            if (a.res) r[k] = in ? gn_raw<T, VW>(a.res, base + k * step, lane) : V{};
        }
        GnNorm s = {};
        if (on) s = gn_saved(a, n, g, wmax);
        float dz[SILU ? K : 1][VW], fa = 0.0f, fx = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int row = p.row + (k << a.rb);
            float z[VW];
#pragma unroll
            for (int i = 0; i < VW; ++i) z[i] = 0.0f;
            if (on && row < a.HW) {
                bool near = false;
#pragma unroll
                for (int i = 0; i < VW; ++i)
                    z[i] = gn_dz<SILU>(a, s, gn_at<T, VW>(x[k], i), w[i], b[i], gn_at<T, VW>(r[k], i), gn_at<T, VW>(d[k], i), near);
                if (!SILU && near) {
#pragma unroll
                    for (int i = 0; i < VW; ++i)
                        z[i] = gn_relu_exact(s, gn_at<T, VW>(x[k], i), w[i], b[i], gn_at<T, VW>(r[k], i), gn_at<T, VW>(d[k], i));
                }
                if (a.dres) gn_put<T, VW>(a.dres, base + k * step, lane, z);
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    const float xhat = gn_xhat(s, gn_at<T, VW>(x[k], i)), f = z[i] * w[i];
                    db[i] += z[i];
                    dw[i] = fmaf(z[i], xhat, dw[i]);
                    fa += f;
                    fx = fmaf(f, xhat, fx);
                }
            }
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                if constexpr (SILU) dz[k][i] = z[i];
                else if constexpr (VW == 1) d[k] = (T)z[i];
                else d[k][i] = (T)z[i];
            }
        }
        if (a.dx) {
            gn_team_sum(fa, fx, inside & ~groups, lds);
            const float ma = fa * inv, mx = fx * inv;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float dx[VW];
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    float z;
                    if constexpr (SILU) z = dz[k][i];
                    else z = gn_at<T, VW>(d[k], i);
                    dx[i] = (fmaf(z, w[i], -ma) - gn_xhat(s, gn_at<T, VW>(x[k], i)) * mx) * s.rs;
                }
                const int row = p.row + (k << a.rb);
                if (on && row < a.HW) gn_put<T, VW>(a.dx, base + k * step, lane, dx);
            }
        }
    }
    if (!a.dpart) return;
    // over the rows, samples and waves of the workgroup, in order: up to 16 threads for a sum, then one
    const int bits = a.cb + a.gb, keep = (1 << bits) - 1, outs = 2 * VW << bits;
#pragma unroll
    for (int i = 0; i < VW; ++i) { sums[2 * i][threadIdx.x] = db[i]; sums[2 * i + 1][threadIdx.x] = dw[i]; }
    __syncthreads();
    const int share = outs >= THREADS ? 1 : min(16, THREADS / outs);
    double total = 0.0;
    for (int o = threadIdx.x; o < outs * share; o += THREADS) {
        const int t = o & keep, v = (o >> bits) % (2 * VW), part = o / outs;
        total = 0.0;
        for (int r = t + (part << bits); r < THREADS; r += share << bits) total += sums[v][r];
        if (share == 1) gn_put_param<VW>(a, slice, walker0, t, v, total);
    }
    if (share == 1) return;
    __syncthreads();
    double* flat = reinterpret_cast<double*>(&sums[0][0]);            // (outs * share <= THREADS of them)
    if (threadIdx.x < outs * share) flat[threadIdx.x] = total;
    __syncthreads();
    if (threadIdx.x < outs) {
        total = 0.0;
        for (int part = 0; part < share; ++part) total += flat[part * outs + threadIdx.x];
        gn_put_param<VW>(a, slice, walker0, threadIdx.x & keep, (int)threadIdx.x >> bits, total);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------
static int gn_log2_ceil(long v) { int b = 0; while ((1l << b) < v) ++b; return b; }

static int gn_check(const az_group_norm* g, const char* who) {
    static thread_local char text[160];
    const char* why = nullptr;
    if (!g) why = "null descriptor";
    else if (g->batch < 0 || g->cells <= 0 || g->channels <= 0 || g->groups <= 0) why = "batch >= 0, cells, channels and groups > 0";
    else if (g->channels % g->groups) why = "channels must divide by groups";
    else if (g->act < 0 || g->act > 2) why = "act is AZ_ACT_NONE, AZ_ACT_RELU or AZ_ACT_SILU";
    else if (g->dtype < 0 || g->dtype > 2 || g->param_dtype < 0 || g->param_dtype > 2) why = "dtype is AZ_F32, AZ_BF16 or AZ_F16";
    else if (!(g->eps >= 0.0)) why = "eps >= 0";
    else if ((int64_t)g->cells * g->channels > INT32_MAX) why = "a sample has at most 2^31 - 1 values";
    else if (g->channels > (1 << 28)) why = "at most 2^28 channels";
    else if ((int64_t)g->batch * ((int64_t)g->cells * g->channels / 32 + g->groups + 1) > (1ll << 40)) why = "tensor too large";
    if (!why) return 0;
    snprintf(text, sizeof text, "%s: %s", who, why);
    return az_fail(text);
}

static int gn_size(int dtype) { return dtype == AZ_F32 ? 4 : 2; }

static int gn_width(const az_group_norm* g, const void* const* tensors, int count) {
    const int most = 16 / gn_size(g->dtype), Cg = g->channels / g->groups;
    for (int w = most; w >= 2; w >>= 1) {
        if (Cg % w) continue;
        bool ok = true;
        for (int i = 0; i < count; ++i) ok = ok && ((uintptr_t)tensors[i] % (w * gn_size(g->dtype)) == 0);
        if (ok) return w;
    }
    return 1;
}

static GnArgs gn_base(const az_group_norm* g, int VW) {
    GnArgs a = {};
    a.N = g->batch; a.HW = g->cells; a.C = g->channels; a.G = g->groups;
    a.Cg = a.C / a.G; a.cpg = a.Cg / VW;
    a.wtype = g->param_dtype; a.eps = g->eps;
    a.low = g->act == AZ_ACT_RELU ? 0.0f : NAN; a.near = g->act == AZ_ACT_RELU ? 0x1p-20f : 0.0f;
    a.count = (double)a.HW * a.Cg; a.inv = 1.0 / a.count;
    a.pieces = 1;
    return a;
}

// for the kernels that take two passes
static void gn_plan_split(GnArgs& a, int VW, int dtype) {
    a.cw = a.cpg < GN_THREADS ? a.cpg : GN_THREADS;
    a.pieces = (a.cpg + a.cw - 1) / a.cw;
    a.gs = 1;
    if (a.pieces == 1) {
        // groups side by side: 64 bytes of a row at least, then the fewest idle threads
        const int line = 64 / (VW * gn_size(dtype)), most = a.G < GN_THREADS / a.cw ? a.G : GN_THREADS / a.cw;
        int low = (line + a.cw - 1) / a.cw;
        if (low > most) low = most;
        long best = -1;
        for (int gs = low; gs <= most; ++gs) {
            const int width = gs * a.cw, rows = a.HW < GN_THREADS / width ? a.HW : GN_THREADS / width;
            const long busy = (long)width * rows * 1000 / (((a.G + gs - 1) / gs) * gs);
            if (busy > best) { best = busy; a.gs = gs; }
        }
    }
    a.rstep = GN_THREADS / (a.gs * a.cw);
    for (a.share = 16; a.share * a.gs > GN_THREADS; a.share >>= 1) {}
    a.slices = (a.G + a.gs - 1) / a.gs;
    a.together = (int64_t)a.gs * a.Cg * gn_size(dtype) % 128 != 0;
    // Rows in chunks while there are too few workgroups to fill the card, four rows of a thread at least; every chunk of the
    // second pass reads the parts of all, so not too many (3 x 4096 cells x 320 channels, bfloat16, forward: 13.4 us with up
    // to 32, 15.2 with up to 128)
    const long units = a.N * a.slices * a.pieces;
    long chunks = units ? (1024 + units - 1) / units : 1;
    const long most = ((long)a.HW + 4 * a.rstep - 1) / (4 * a.rstep);
    if (chunks > most) chunks = most;
    if (chunks > 32) chunks = 32;
    long least = ((long)a.HW * a.C * gn_size(dtype) >> 31) + 1;               // (a chunk's offsets in 32 bits)
    if (least * a.rstep * GN_CHAIN < a.HW) least = ((long)a.HW + a.rstep * GN_CHAIN - 1) / (a.rstep * GN_CHAIN);
    if (chunks < least) chunks = least;
    a.rows = (int)((a.HW + chunks - 1) / chunks);
    a.chunks = (int)(((long)a.HW + a.rows - 1) / a.rows);                     // (HW + rows passes 2^31 in long samples)
}

// For the kernels that hold a sample's slice in registers: the team and K; false where no team can.
//   Slices take 256 bytes of a row, less only where no team holds that: 42 cells x 128 channels, backward, 4096 boards in
// bfloat16: 54 us at 256 bytes (a workgroup, K = 3), 61 at 128 (a wave, K = 6), 67 at 64.  Slices of 64 bytes share lines;
// with neighbours on one die they still beat the two passes (64 x 1024 cells x 128 channels, forward: 12.5 against 16.9 us).
//   Workgroups of 1024 do not go deeper than this table: 3 x 4096 cells x 320 channels, bfloat16, forward, takes 24 us held
// 32 vectors of 4 bytes deep and 12.4 in two passes; 64 x 1024 cells, 16 deep, 66 and 53.
//   A wave is taken before a workgroup: it needs no barrier (hw 1, 8192 x 512 channels: 7 against 14 us forward).
static bool gn_plan_held(GnArgs& a, int VW, int dtype, bool silu, bool backward, int& K, int& threads) {
    // vectors of a thread that its registers hold, in a team of a wave, 256 and 1024 threads: forward, backward, with silu
    static const int narrow[3][3] = {{8, 16, 8}, {8, 8, 4}, {8, 8, 4}}, wide[3][3] = {{8, 12, 4}, {6, 6, 0}, {4, 4, 2}};
    const int* most = (VW == 8 ? wide : narrow)[!backward ? 0 : silu ? 2 : 1];
    if ((int64_t)a.HW * a.C * gn_size(dtype) >= (1ll << 25)) return false;        // (64 samples' offsets in 31 bits)
    const int cb = gn_log2_ceil(a.cpg);
    for (int bytes = 256; bytes >= 64; bytes >>= 1) {
        const int line = gn_log2_ceil(bytes / (VW * gn_size(dtype)));           // lanes that cover so many bytes of a row
        for (int kind = 0; kind < 3; ++kind) {
            const int tb = kind == 0 ? 6 : kind == 1 ? 8 : 10;
            if (cb > tb) continue;
            int gb = line > cb ? line - cb : 0;
            const int spare = tb - cb - gn_log2_ceil(a.HW);
            if (spare > gb) gb = spare;
            if (gb > tb - cb) gb = tb - cb;
            if (gb > gn_log2_ceil(a.G)) gb = gn_log2_ceil(a.G);
            const int slices = (a.G + (1 << gb) - 1) >> gb;
            int rb = tb - cb - gb;
            const long rows = (a.HW + (1 << rb) - 1) >> rb;
            if (rows > most[kind]) continue;
            // a wave's lanes beyond a sample's rows take further samples, as many as leave the fewest lanes idle -- unless
            // the batch is small, where every wave that there can be is wanted
            if (kind == 0 && a.N * slices >= 4096) {
                int best = rb;
                for (int r = rb; r >= 0; --r) {
                    const int k = (a.HW + (1 << r) - 1) >> r, kb = (a.HW + (1 << best) - 1) >> best;
                    if (k <= most[0] && ((long)k << r) <= ((long)kb << best)) best = r;
                }
                rb = best;
            }
            a.tb = tb; a.cb = cb; a.gb = gb; a.rb = rb; a.slices = slices;
            a.sb = kind == 0 ? tb - cb - gb - rb : 0;
            a.together = ((int64_t)a.Cg << gb) * gn_size(dtype) % 128 != 0 && slices > 1;
            K = (a.HW + (1 << rb) - 1) >> rb;
            threads = kind == 2 ? 1024 : 256;
            if (backward) {
                const long batches = (a.N + (1 << a.sb) - 1) >> a.sb, teams = kind == 0 ? 4 : 1;
                // Workgroups to each compute unit: enough for 64 KiB on their way (8192 boards x 128 channels, float32: 512
                // take 171 us, 1024 178; at 30 channels in 5 groups, half the lanes idle, 512 take 19.8 and 1024 17.0);
                // two of 256 threads, one of which works while the other's loads are on their way (81 cells x 128
                // channels, 4096 boards, bfloat16: 144 us with one, 106 with two, 118 with three); one of 1024, which
                // fills the registers (61 x 361 cells x 192 channels, float16, silu: 18.7 us with two, 16.7 with one).
                // But no more than a sixteenth of the traffic in partial sums (8192 x 512 channels of one cell: 512 take
                // 14.4 us, 2048 24.5).
                const long lanes = (long)threads * a.cpg / (1 << cb) * (a.G < (1 << gb) ? a.G : 1 << gb) / (1 << gb);
                const long flight = 3 * lanes * K * VW * gn_size(dtype);
                long per = 65536 / (flight > 0 ? flight : 1) + 1;
                if (threads == 1024) per = 1;
                else if (per < 2) per = 2;
                long blocks = 256 * per / slices;
                const long most_rows = a.N * a.HW * gn_size(dtype) * 3 / 128;
                if (blocks > 1536 / slices) blocks = 1536 / slices;
                if (blocks > most_rows) blocks = most_rows;
                const long least = (batches * K + teams * GN_CHAIN - 1) / (teams * GN_CHAIN);
                if (blocks < least) blocks = least;
                if (blocks > (batches + teams - 1) / teams) blocks = (batches + teams - 1) / teams;
                if (blocks < 1) blocks = 1;
                a.walkers = (int)(blocks * teams);
                a.chunks = (int)blocks;                                         // rows of partial sums
            }
            return true;
        }
    }
    return false;
}

template <typename T, int VW, int K, int THREADS, bool SILU>
static void gn_held_forward(const GnArgs& a, hipStream_t st) {
    const long units = ((a.N + (1 << a.sb) - 1) >> a.sb) * a.slices;
    const long blocks = a.tb == 6 ? (units + THREADS / 64 - 1) / (THREADS / 64) : units;
    hipLaunchKernelGGL((k_gn_held<T, VW, K, THREADS, SILU>), dim3((unsigned)blocks), dim3(THREADS), 0, st, a);
}

template <typename T, int VW, int K, int THREADS, bool SILU>
static void gn_held_backward(const GnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((k_gn_bwd_held<T, VW, K, THREADS, SILU>), dim3((unsigned)(a.chunks * a.slices)), dim3(THREADS), 0, st, a);
}

// (K rounded up to a size that is compiled: gn_plan_held gives none beyond them)
template <typename T, int VW, bool SILU>
static void gn_held_k(const GnArgs& a, bool backward, int K, int threads, hipStream_t st) {
    if (!backward) {
        if (threads == 1024) {
            if (VW == 8 || K <= 4) gn_held_forward<T, VW, 4, 1024, SILU>(a, st);
            else if constexpr (VW < 8) gn_held_forward<T, VW, 8, 1024, SILU>(a, st);
        } else if (K <= 1) gn_held_forward<T, VW, 1, 256, SILU>(a, st);
        else if (K <= 2) gn_held_forward<T, VW, 2, 256, SILU>(a, st);
        else if (K <= 3) gn_held_forward<T, VW, 3, 256, SILU>(a, st);
        else if (K <= 4) gn_held_forward<T, VW, 4, 256, SILU>(a, st);
        else if (K <= 6) gn_held_forward<T, VW, 6, 256, SILU>(a, st);
        else if (K <= 8) gn_held_forward<T, VW, 8, 256, SILU>(a, st);
        else if (VW == 8 || K <= 12) gn_held_forward<T, VW, 12, 256, SILU>(a, st);
        else if constexpr (VW < 8) gn_held_forward<T, VW, 16, 256, SILU>(a, st);
    } else {
        if (threads == 1024) {
            if constexpr (SILU || VW < 8) gn_held_backward<T, VW, VW == 8 ? 2 : 4, 1024, SILU>(a, st);
        } else if (K <= 1) gn_held_backward<T, VW, 1, 256, SILU>(a, st);
        else if (K <= 2) gn_held_backward<T, VW, 2, 256, SILU>(a, st);
        else if (K <= 3) gn_held_backward<T, VW, 3, 256, SILU>(a, st);
        else if ((SILU && VW == 8) || K <= 4) gn_held_backward<T, VW, 4, 256, SILU>(a, st);
        else if constexpr (!(SILU && VW == 8)) {
            if (VW == 8 || K <= 6) gn_held_backward<T, VW, 6, 256, SILU>(a, st);
            else if constexpr (VW < 8) gn_held_backward<T, VW, 8, 256, SILU>(a, st);
        }
    }
}

template <typename T, bool SILU>
static void gn_held_w(const GnArgs& a, int VW, bool backward, int K, int threads, hipStream_t st) {
    if (VW == 1) gn_held_k<T, 1, SILU>(a, backward, K, threads, st);
    else if (VW == 2) gn_held_k<T, 2, SILU>(a, backward, K, threads, st);
    else if (VW == 4) gn_held_k<T, 4, SILU>(a, backward, K, threads, st);
    else if constexpr (sizeof(T) == 2) gn_held_k<T, 8, SILU>(a, backward, K, threads, st);
}

template <bool SILU>
static void gn_held_t(const GnArgs& a, int VW, int dtype, bool backward, int K, int threads, hipStream_t st) {
    if (dtype == AZ_F32) gn_held_w<float, SILU>(a, VW, backward, K, threads, st);
    else if (dtype == AZ_BF16) gn_held_w<__bf16, SILU>(a, VW, backward, K, threads, st);
    else gn_held_w<_Float16, SILU>(a, VW, backward, K, threads, st);
}

// HIP takes fewer than 2^32 work-items in a launch
static bool gn_fits(long blocks, int threads) { return blocks > 0 && blocks * threads < (1l << 32); }
static const char gn_too_many[] = "az_group_norm_act: the tensor takes 2^32 work-items or more, which is more than a launch";

static int gn_held(const GnArgs& a, int VW, const az_group_norm* g, bool backward, int K, int threads, hipStream_t st) {
    const long units = ((a.N + (1 << a.sb) - 1) >> a.sb) * a.slices, teams = a.tb == 6 ? threads / 64 : 1;
    if (!gn_fits(backward ? (long)a.chunks * a.slices : (units + teams - 1) / teams, threads)) return az_fail(gn_too_many);
    if (g->act == AZ_ACT_SILU) gn_held_t<true>(a, VW, g->dtype, backward, K, threads, st);
    else gn_held_t<false>(a, VW, g->dtype, backward, K, threads, st);
    AZ_LAUNCH_CHECK("a group norm kernel");
    return 0;
}

static size_t gn_part_bytes(const GnArgs& a) { return (size_t)a.N * a.G * a.pieces * a.chunks * 16; }
static size_t gn_dpart_bytes(const GnArgs& a) { return (size_t)a.N * a.chunks * 2 * a.C * 4; }

template <int STEP, typename T, bool SILU>
static void gn_go_w(const GnArgs& a, int VW, dim3 grid, hipStream_t st) {
#define GN_GO(W)                                                                                                                  \
    do {                                                                                                                          \
        if (STEP == 0) hipLaunchKernelGGL((k_gn_stats<T, W>), grid, dim3(GN_THREADS), 0, st, a);                                  \
        if (STEP == 1) hipLaunchKernelGGL((k_gn_apply<T, W, SILU>), grid, dim3(GN_THREADS), 0, st, a);                            \
        if (STEP == 2) hipLaunchKernelGGL((k_gn_bwd_sums<T, W, SILU>), grid, dim3(GN_THREADS), 0, st, a);                         \
        if (STEP == 3) hipLaunchKernelGGL((k_gn_bwd_apply<T, W, SILU>), grid, dim3(GN_THREADS), 0, st, a);                        \
    } while (0)
    if (VW == 1) GN_GO(1);
    else if (VW == 2) GN_GO(2);
    else if (VW == 4) GN_GO(4);
    else if constexpr (sizeof(T) == 2) GN_GO(8);
#undef GN_GO
}

template <int STEP, bool SILU>
static void gn_go_t(const GnArgs& a, int VW, int dtype, dim3 grid, hipStream_t st) {
    if (dtype == AZ_F32) gn_go_w<STEP, float, SILU>(a, VW, grid, st);
    else if (dtype == AZ_BF16) gn_go_w<STEP, __bf16, SILU>(a, VW, grid, st);
    else gn_go_w<STEP, _Float16, SILU>(a, VW, grid, st);
}

template <int STEP>
static int gn_go(const GnArgs& a, int VW, const az_group_norm* g, hipStream_t st) {
    const long blocks = a.N * a.slices * a.pieces * a.chunks;
    if (!gn_fits(blocks, GN_THREADS)) return az_fail(gn_too_many);                  // (both steps of a call have this grid)
    if (STEP > 0 && g->act == AZ_ACT_SILU) gn_go_t<STEP, true>(a, VW, g->dtype, dim3((unsigned)blocks), st);
    else gn_go_t<STEP, false>(a, VW, g->dtype, dim3((unsigned)blocks), st);
    AZ_LAUNCH_CHECK("a group norm kernel");
    return 0;
}

extern "C" {

int64_t az_group_norm_workspace_bytes(const az_group_norm* g, int32_t backward) {
    if (gn_check(g, "az_group_norm_workspace_bytes")) return -1;
    size_t most = 0;
    for (int VW = 1; VW <= 8; VW <<= 1) {                  // (the width depends on the pointers: room for any)
        if ((g->channels / g->groups) % VW) continue;
        GnArgs a = gn_base(g, VW);
        int K, threads;
        const bool held = gn_plan_held(a, VW, g->dtype, g->act == AZ_ACT_SILU, backward, K, threads);
        if (!held) gn_plan_split(a, VW, g->dtype);
        const size_t n = held ? (backward ? (size_t)a.chunks * 2 * a.C * 4 : 0) : gn_part_bytes(a) + (backward ? gn_dpart_bytes(a) : 0);
        if (n > most) most = n;
    }
    return (int64_t)most;
}

int az_group_norm_act(const az_group_norm* g, const void* x, const void* weight, const void* bias, const void* residual,
                      void* y, double* stats, void* workspace, int64_t workspace_bytes, void* stream) {
    if (gn_check(g, "az_group_norm_act")) return -1;
    if (g->batch == 0) return 0;
    if (!x || !y) return az_fail("az_group_norm_act: null pointer");
    const int64_t need = az_group_norm_workspace_bytes(g, 0);
    if (workspace_bytes < need || (need && !workspace)) return az_fail("az_group_norm_act: workspace too small");
    if ((uintptr_t)workspace % 16) return az_fail("az_group_norm_act: workspace is aligned to 16 bytes");
    const void* all[] = {x, y, residual};
    const int VW = gn_width(g, all, 3);
    GnArgs a = gn_base(g, VW);
    a.x = x; a.w = weight; a.b = bias; a.res = residual; a.y = y; a.stats = stats;
    a.wide = ((uintptr_t)weight | (uintptr_t)bias) % 16 == 0;
    int K, threads;
    if (gn_plan_held(a, VW, g->dtype, g->act == AZ_ACT_SILU, false, K, threads)) return gn_held(a, VW, g, false, K, threads, (hipStream_t)stream);
    gn_plan_split(a, VW, g->dtype);
    a.part = (double*)workspace;
    if (int rc = gn_go<0>(a, VW, g, (hipStream_t)stream)) return rc;
    return gn_go<1>(a, VW, g, (hipStream_t)stream);
}

int az_group_norm_act_backward(const az_group_norm* g, const void* dy, const void* x, const void* weight, const void* bias,
                               const void* residual, const double* stats, void* dx, void* dweight, void* dbias,
                               void* dresidual, void* workspace, int64_t workspace_bytes, void* stream) {
    if (gn_check(g, "az_group_norm_act_backward")) return -1;
    hipStream_t st = (hipStream_t)stream;
    if (g->batch && (!dy || !x || !stats)) return az_fail("az_group_norm_act_backward: null pointer");
    if (dresidual && !residual) return az_fail("az_group_norm_act_backward: a residual's gradient without a residual");
    const int64_t need = az_group_norm_workspace_bytes(g, 1);
    if (workspace_bytes < need || (need && !workspace))
        return az_fail("az_group_norm_act_backward: workspace too small");
    if ((uintptr_t)workspace % 16) return az_fail("az_group_norm_act_backward: workspace is aligned to 16 bytes");
    const void* all[] = {dy, x, residual, dx, dresidual};
    const int VW = gn_width(g, all, 5);
    GnArgs a = gn_base(g, VW);
    a.dy = dy; a.x = x; a.w = weight; a.b = bias; a.res = residual; a.stats = const_cast<double*>(stats);
    a.dx = dx; a.dres = dresidual;
    a.wide = ((uintptr_t)weight | (uintptr_t)bias) % 16 == 0;
    const bool params = dweight || dbias;
    int K, threads;
    long parts;                                            // rows of partial sums
    if (gn_plan_held(a, VW, g->dtype, g->act == AZ_ACT_SILU, true, K, threads)) {
        a.dpart = params ? (float*)workspace : nullptr;
        parts = g->batch ? a.chunks : 0;
        if (g->batch)
            if (int rc = gn_held(a, VW, g, true, K, threads, st)) return rc;
    } else {
        gn_plan_split(a, VW, g->dtype);
        a.part = dx ? (double*)workspace : nullptr;
        a.dpart = params ? (float*)((char*)workspace + gn_part_bytes(a)) : nullptr;
        parts = a.N * a.chunks;
        if (g->batch) {
            if (int rc = gn_go<2>(a, VW, g, st)) return rc;
            if (dx) { if (int rc = gn_go<3>(a, VW, g, st)) return rc; }
        }
    }
    if (params) {
        for (int first = 0, most = 16 << 20; first < 2 * a.C; first += most) {       // (2^30 work-items at a time)
            const int cols = 2 * a.C - first < most ? 2 * a.C - first : most;
            hipLaunchKernelGGL(k_gn_dparams, dim3((unsigned)((cols + 15) / 16)), dim3(1024), 0, st, a.dpart, parts, first, a.C, a.wtype, dweight, dbias);
            AZ_LAUNCH_CHECK("k_gn_dparams");
        }
    }
    return 0;
}

}  // extern "C"
