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
// Statistics are summed and kept in 64 bits.  With them one pass over x gives mean and variance without the
// cancellation that E[x^2] - mean^2 has in 32 bits, and the sign of z -- the border at which relu cuts the gradient --
// can be decided exactly: z is formed in 32 bits, and where it lies closer to zero than its rounding errors it is
// formed again in 64.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/azhip.h"
#include "az_host.h"

#define GN_THREADS 256
#define GN_ACT_NONE 0
#define GN_ACT_RELU 1
#define GN_ACT_SILU 2

// A thread holds VW neighbouring channels of one group; the bits of its index in the team are, from the lowest:
// column within the group (cb), group within the slice (gb), row (rb).  Sums over a group are butterflies over the
// column and row bits, so a wave's loads run along memory whatever the group's width.
struct GnArgs {
    const void* x; const void* dy; const void* res; const void* w; const void* b;
    void* y; void* dx; void* dres;
    double* stats;                    // [N][G][2] mean, rstd
    double* part;                     // [N][G][pieces * chunks][2] partial sums
    float* dpart;                     // [N * chunks][2][C] partial sums of dz and dz * xhat
    long N;
    int HW, C, G, Cg, cpg;            // cpg: vectors per group
    int cb, gb, rb;
    int slices, pieces, chunks, rows; // rows per chunk
    int act, wtype;
    double eps;
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

__device__ __forceinline__ float gn_param(const void* p, int type, int at, float otherwise) {
    if (!p) return otherwise;
    if (type == AZ_F32) return reinterpret_cast<const float*>(p)[at];
    if (type == AZ_BF16) return (float)reinterpret_cast<const __bf16*>(p)[at];
    return (float)reinterpret_cast<const _Float16*>(p)[at];
}

__device__ __forceinline__ double gn_xor(double v, int mask) { return __shfl_xor(v, mask, 64); }

// sums of (s, q) over the threads of a workgroup whose index differs in the bits of `mask` only; every thread of a
// group gets the same bits
__device__ __forceinline__ void gn_team_sum(double& s, double& q, int mask, double (*lds)[2]) {
    const int tid = threadIdx.x, waves = blockDim.x >> 6;
    for (int bit = 1; bit < 64; bit <<= 1)
        if (mask & bit) { s += gn_xor(s, bit); q += gn_xor(q, bit); }
    if (mask >> 6) {
        __syncthreads();
        lds[tid][0] = s; lds[tid][1] = q;
        __syncthreads();
        s = q = 0.0;
        for (int w = 0; w < waves; ++w)
            if ((((w ^ (tid >> 6)) << 6) & ~mask) == 0) { s += lds[(w << 6) + (tid & 63)][0]; q += lds[(w << 6) + (tid & 63)][1]; }
    }
}

// mean and 1 / sqrt(var + eps) of n values with sum s and sum of squares q
__device__ __forceinline__ void gn_moments(double s, double q, double n, double eps, double& mean, double& rstd) {
    mean = s / n;                     // (a division: a group of equal values has exactly their value as its mean)
    const double var = fmax(q / n - mean * mean, 0.0);
    rstd = 1.0 / sqrt(var + eps);
}

struct GnPlace {                      // where a thread of the workgroup stands
    long n; int g, col, row, chunk, piece, slice; bool on;
    long base;                        // element of its first channel in row 0
};

__device__ __forceinline__ GnPlace gn_place(const GnArgs& a, int VW) {
    GnPlace p;
    long u = blockIdx.x;
    p.chunk = (int)(u % a.chunks); u /= a.chunks;
    p.piece = (int)(u % a.pieces); u /= a.pieces;
    p.slice = (int)(u % a.slices);
    p.n = u / a.slices;
    const int t = threadIdx.x;
    p.col = (t & ((1 << a.cb) - 1)) + (p.piece << a.cb);
    p.g = (p.slice << a.gb) + ((t >> a.cb) & ((1 << a.gb) - 1));
    p.row = t >> (a.cb + a.gb);
    p.on = p.col < a.cpg && p.g < a.G;
    p.base = p.n * a.HW * a.C + (long)p.g * a.Cg + (long)p.col * VW;
    return p;
}

template <typename T, int VW>
__global__ void __launch_bounds__(GN_THREADS)
k_gn_stats(GnArgs a) {
    __shared__ double lds[GN_THREADS][2];
    const GnPlace p = gn_place(a, VW);
    double s = 0.0, q = 0.0;
    const int r1 = min(a.HW, (p.chunk + 1) * a.rows);
    if (p.on)
        for (int r = p.chunk * a.rows + p.row; r < r1; r += 1 << a.rb) {
            float x[VW];
            gn_load<T, VW>(a.x, p.base + (long)r * a.C, x);
#pragma unroll
            for (int i = 0; i < VW; ++i) { const double d = x[i]; s += d; q = fma(d, d, q); }
        }
    gn_team_sum(s, q, (GN_THREADS - 1) & ~(((1 << a.gb) - 1) << a.cb), lds);
    if (p.on && p.row == 0 && (threadIdx.x & ((1 << a.cb) - 1)) == 0) {
        double* out = a.part + ((p.n * a.G + p.g) * (a.pieces * a.chunks) + p.piece * a.chunks + p.chunk) * 2;
        out[0] = s; out[1] = q;
    }
}

// the sums of a group's parts, in order
__device__ __forceinline__ void gn_parts(const GnArgs& a, const GnPlace& p, double& s, double& q) {
    const double* in = a.part + (p.n * a.G + p.g) * (a.pieces * a.chunks) * 2;
    s = q = 0.0;
    for (int k = 0; k < a.pieces * a.chunks; ++k) { s += in[2 * k]; q += in[2 * k + 1]; }
}

__device__ __forceinline__ float gn_silu(float z) { return z / (1.0f + expf(-z)); }

__device__ __forceinline__ float gn_act(float z, int act) {
    if (act == GN_ACT_RELU) return z <= 0.0f ? 0.0f : z;      // (a NaN stays one)
    if (act == GN_ACT_SILU) return gn_silu(z);
    return z;
}

template <typename T, int VW>
__global__ void __launch_bounds__(GN_THREADS)
k_gn_apply(GnArgs a) {
    const GnPlace p = gn_place(a, VW);
    if (!p.on) return;
    double s, q, mean, rstd;
    gn_parts(a, p, s, q);
    gn_moments(s, q, (double)a.HW * a.Cg, a.eps, mean, rstd);
    if (a.stats && p.chunk == 0 && p.col == 0 && p.row == 0) {
        a.stats[(p.n * a.G + p.g) * 2] = mean;
        a.stats[(p.n * a.G + p.g) * 2 + 1] = rstd;
    }
    // the mean as two floats: x - mean keeps its precision where the mean is large against the spread
    const float mh = (float)mean, ml = (float)(mean - (double)mh), rs = (float)rstd;
    float w[VW], b[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) {
        w[i] = gn_param(a.w, a.wtype, p.g * a.Cg + p.col * VW + i, 1.0f);
        b[i] = gn_param(a.b, a.wtype, p.g * a.Cg + p.col * VW + i, 0.0f);
    }
    const int r1 = min(a.HW, (p.chunk + 1) * a.rows);
    for (int r = p.chunk * a.rows + p.row; r < r1; r += 1 << a.rb) {
        const long at = p.base + (long)r * a.C;
        float x[VW], z[VW];
        gn_load<T, VW>(a.x, at, x);
        if (a.res) gn_load<T, VW>(a.res, at, z);
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const float t = fmaf(((x[i] - mh) - ml) * rs, w[i], b[i]);
            z[i] = gn_act(a.res ? t + z[i] : t, a.act);
        }
        gn_store<T, VW>(a.y, at, z);
    }
}

struct GnNorm { double mean, rstd; float mh, ml, rs; };

__device__ __forceinline__ GnNorm gn_saved(const GnArgs& a, long n, int g) {
    GnNorm k;
    k.mean = a.stats[(n * a.G + g) * 2];
    k.rstd = a.stats[(n * a.G + g) * 2 + 1];
    k.mh = (float)k.mean; k.ml = (float)(k.mean - (double)k.mh); k.rs = (float)k.rstd;
    return k;
}

// dz of one value, and its xhat.  relu: z in 32 bits is off by less than 8 * 2^-24 * (|xhat w| + |b|) (three roundings
// of x - mean and rstd, one each of the product and the two sums, and |res| <= |xhat w| + |b| where z is small);
// closer to zero than twice that its sign is taken from 64 bits.
__device__ __forceinline__ float gn_dz(const GnNorm& k, int act, float x, float w, float b, bool has_res, float res, float dy, float& xhat) {
    xhat = ((x - k.mh) - k.ml) * k.rs;
    if (act == GN_ACT_NONE) return dy;
    const float t = xhat * w;
    float z = t + b;
    if (has_res) z += res;
    if (act == GN_ACT_RELU) {
        if (fabsf(z) < (fabsf(t) + fabsf(b)) * 0x1p-20f) {
            double d = ((double)x - k.mean) * k.rstd * (double)w + (double)b;
            if (has_res) d += (double)res;
            return d <= 0.0 ? 0.0f : dy;
        }
        return z <= 0.0f ? 0.0f : dy;
    }
    const float sig = 1.0f / (1.0f + expf(-z));
    return dy * (sig * fmaf(z, 1.0f - sig, 1.0f));
}

// sums over a chunk of rows: of a and a * xhat per group, of dz and dz * xhat per channel; writes the residual's gradient
template <typename T, int VW>
__global__ void __launch_bounds__(GN_THREADS)
k_gn_bwd_sums(GnArgs a) {
    __shared__ double lds[GN_THREADS][2];
    const GnPlace p = gn_place(a, VW);
    double sa = 0.0, sx = 0.0;
    float dw[VW], db[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) dw[i] = db[i] = 0.0f;
    if (p.on) {
        const GnNorm k = gn_saved(a, p.n, p.g);
        float w[VW], b[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            w[i] = gn_param(a.w, a.wtype, p.g * a.Cg + p.col * VW + i, 1.0f);
            b[i] = gn_param(a.b, a.wtype, p.g * a.Cg + p.col * VW + i, 0.0f);
        }
        const int r1 = min(a.HW, (p.chunk + 1) * a.rows);
        for (int r = p.chunk * a.rows + p.row; r < r1; r += 1 << a.rb) {
            const long at = p.base + (long)r * a.C;
            float x[VW], dy[VW], res[VW];
            gn_load<T, VW>(a.x, at, x);
            gn_load<T, VW>(a.dy, at, dy);
            if (a.res) gn_load<T, VW>(a.res, at, res);
            float fa = 0.0f, fx = 0.0f;
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                float xhat;
                const float dz = gn_dz(k, a.act, x[i], w[i], b[i], a.res != nullptr, a.res ? res[i] : 0.0f, dy[i], xhat);
                db[i] += dz;
                dw[i] = fmaf(dz, xhat, dw[i]);
                fa = fmaf(dz, w[i], fa);
                fx = fmaf(dz * w[i], xhat, fx);
                dy[i] = dz;
            }
            sa += fa; sx += fx;
            if (a.dres) gn_store<T, VW>(a.dres, at, dy);
        }
    }
    const int all = GN_THREADS - 1, cols = (1 << a.cb) - 1, groups = ((1 << a.gb) - 1) << a.cb;
    if (a.part) {
        gn_team_sum(sa, sx, all & ~groups, lds);
        if (p.on && p.row == 0 && (threadIdx.x & cols) == 0) {
            double* out = a.part + ((p.n * a.G + p.g) * (a.pieces * a.chunks) + p.piece * a.chunks + p.chunk) * 2;
            out[0] = sa; out[1] = sx;
        }
    }
    if (a.dpart) {
        for (int i = 0; i < VW; ++i) {
            double u = db[i], v = dw[i];
            gn_team_sum(u, v, all & ~(groups | cols), lds);
            if (p.on && p.row == 0) {
                float* out = a.dpart + (p.n * a.chunks + p.chunk) * 2 * a.C + p.g * a.Cg + p.col * VW + i;
                out[0] = (float)u; out[a.C] = (float)v;
            }
        }
    }
}

template <typename T, int VW>
__global__ void __launch_bounds__(GN_THREADS)
k_gn_bwd_apply(GnArgs a) {
    const GnPlace p = gn_place(a, VW);
    if (!p.on) return;
    double sa, sx;
    gn_parts(a, p, sa, sx);
    const double n = (double)a.HW * a.Cg;
    const float ma = (float)(sa / n), mx = (float)(sx / n);
    const GnNorm k = gn_saved(a, p.n, p.g);
    float w[VW], b[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) {
        w[i] = gn_param(a.w, a.wtype, p.g * a.Cg + p.col * VW + i, 1.0f);
        b[i] = gn_param(a.b, a.wtype, p.g * a.Cg + p.col * VW + i, 0.0f);
    }
    const int r1 = min(a.HW, (p.chunk + 1) * a.rows);
    for (int r = p.chunk * a.rows + p.row; r < r1; r += 1 << a.rb) {
        const long at = p.base + (long)r * a.C;
        float x[VW], dy[VW], res[VW];
        gn_load<T, VW>(a.x, at, x);
        gn_load<T, VW>(a.dy, at, dy);
        if (a.res) gn_load<T, VW>(a.res, at, res);
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            float xhat;
            const float dz = gn_dz(k, a.act, x[i], w[i], b[i], a.res != nullptr, a.res ? res[i] : 0.0f, dy[i], xhat);
            dy[i] = (fmaf(dz, w[i], -ma) - xhat * mx) * k.rs;
        }
        gn_store<T, VW>(a.dx, at, dy);
    }
}

// dw, db: the partial sums of `parts` workgroups, added in a fixed order in 64 bits.  One workgroup: 16 of the 2 C columns.
__global__ void __launch_bounds__(1024)
k_gn_dparams(const float* __restrict__ dpart, long parts, int C, int wtype, void* dw, void* db) {
    __shared__ double lds[64][17];
    const int col = blockIdx.x * 16 + (threadIdx.x & 15), r0 = threadIdx.x >> 4;
    double s = 0.0;
    if (col < 2 * C)
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
    else if ((int64_t)g->batch * ((int64_t)g->cells * g->channels / 32 + g->groups + 1) > (1ll << 40)) why = "tensor too large";
    if (!why) return 0;
    snprintf(text, sizeof text, "%s: %s", who, why);
    return az_fail(text);
}

static int gn_size(int dtype) { return dtype == AZ_F32 ? 4 : 2; }

static int gn_width(const az_group_norm* g, const void* const* tensors, int count) {
    const int most = 16 / gn_size(g->dtype), Cg = g->channels / g->groups;
    for (int w = most; w >= 4; w >>= 1) {
        if (Cg % w) continue;
        bool ok = true;
        for (int i = 0; i < count; ++i) ok = ok && ((uintptr_t)tensors[i] % (w * gn_size(g->dtype)) == 0);
        if (ok) return w;
    }
    return 1;
}

static GnArgs gn_plan(const az_group_norm* g, int VW) {
    GnArgs a = {};
    a.N = g->batch; a.HW = g->cells; a.C = g->channels; a.G = g->groups;
    a.Cg = a.C / a.G; a.cpg = a.Cg / VW;
    a.act = g->act; a.wtype = g->param_dtype; a.eps = g->eps;
    a.pieces = 1;
    if (a.cpg > GN_THREADS) { a.cb = 8; a.pieces = (a.cpg + GN_THREADS - 1) / GN_THREADS; }
    else {
        a.cb = gn_log2_ceil(a.cpg);
        const int line = gn_log2_ceil(128 / (VW * gn_size(g->dtype)));      // lanes that cover 128 bytes of a row
        int gb = line > a.cb ? line - a.cb : 0;
        const int spare = 8 - a.cb - gn_log2_ceil(a.HW);
        if (spare > gb) gb = spare;
        if (gb > 8 - a.cb) gb = 8 - a.cb;
        if (gb > gn_log2_ceil(a.G)) gb = gn_log2_ceil(a.G);
        a.gb = gb;
    }
    a.rb = 8 - a.cb - a.gb;
    a.slices = (a.G + (1 << a.gb) - 1) >> a.gb;
    // rows in chunks while there are too few workgroups to fill the card, four rows of a thread at least
    const long units = a.N * a.slices * a.pieces;
    long chunks = units ? (1024 + units - 1) / units : 1;
    const long most = (a.HW + (4 << a.rb) - 1) / (4 << a.rb);
    if (chunks > most) chunks = most;
    if (chunks > 64) chunks = 64;
    if (chunks < 1) chunks = 1;
    a.rows = (int)((a.HW + chunks - 1) / chunks);
    a.chunks = (a.HW + a.rows - 1) / a.rows;
    return a;
}

static size_t gn_part_bytes(const GnArgs& a) { return (size_t)a.N * a.G * a.pieces * a.chunks * 16; }
static size_t gn_dpart_bytes(const GnArgs& a) { return (size_t)a.N * a.chunks * 2 * a.C * 4; }

template <int STEP, typename T>
static void gn_go_w(const GnArgs& a, int VW, dim3 grid, hipStream_t st) {
#define GN_GO(W)                                                                                                                  \
    do {                                                                                                                          \
        if (STEP == 0) hipLaunchKernelGGL((k_gn_stats<T, W>), grid, dim3(GN_THREADS), 0, st, a);                                  \
        if (STEP == 1) hipLaunchKernelGGL((k_gn_apply<T, W>), grid, dim3(GN_THREADS), 0, st, a);                                  \
        if (STEP == 2) hipLaunchKernelGGL((k_gn_bwd_sums<T, W>), grid, dim3(GN_THREADS), 0, st, a);                               \
        if (STEP == 3) hipLaunchKernelGGL((k_gn_bwd_apply<T, W>), grid, dim3(GN_THREADS), 0, st, a);                              \
    } while (0)
    if (VW == 1) GN_GO(1);
    else if (VW == 4) GN_GO(4);
    else if constexpr (sizeof(T) == 2) GN_GO(8);
#undef GN_GO
}

template <int STEP>
static int gn_go(const GnArgs& a, int VW, int dtype, hipStream_t st) {
    const long blocks = a.N * a.slices * a.pieces * a.chunks;
    if (blocks > INT32_MAX) return az_fail("az_group_norm_act: more workgroups than a launch takes");
    const dim3 grid((unsigned)blocks);
    if (dtype == AZ_F32) gn_go_w<STEP, float>(a, VW, grid, st);
    else if (dtype == AZ_BF16) gn_go_w<STEP, __bf16>(a, VW, grid, st);
    else gn_go_w<STEP, _Float16>(a, VW, grid, st);
    AZ_LAUNCH_CHECK("a group norm kernel");
    return 0;
}

extern "C" {

int64_t az_group_norm_workspace_bytes(const az_group_norm* g, int32_t backward) {
    if (gn_check(g, "az_group_norm_workspace_bytes")) return -1;
    size_t most = 0;
    for (int VW = 1; VW <= 8; VW <<= 1) {                  // (the width depends on the pointers: room for any)
        if ((g->channels / g->groups) % VW) continue;
        const GnArgs a = gn_plan(g, VW);
        const size_t n = gn_part_bytes(a) + (backward ? gn_dpart_bytes(a) : 0);
        if (n > most) most = n;
    }
    return (int64_t)most;
}

int az_group_norm_act(const az_group_norm* g, const void* x, const void* weight, const void* bias, const void* residual,
                      void* y, double* stats, void* workspace, int64_t workspace_bytes, void* stream) {
    if (gn_check(g, "az_group_norm_act")) return -1;
    if (g->batch == 0) return 0;
    if (!x || !y) return az_fail("az_group_norm_act: null pointer");
    if (workspace_bytes < az_group_norm_workspace_bytes(g, 0) || !workspace) return az_fail("az_group_norm_act: workspace too small");
    const void* all[] = {x, y, residual};
    const int VW = gn_width(g, all, 3);
    GnArgs a = gn_plan(g, VW);
    a.x = x; a.w = weight; a.b = bias; a.res = residual; a.y = y; a.stats = stats; a.part = (double*)workspace;
    if (int rc = gn_go<0>(a, VW, g->dtype, (hipStream_t)stream)) return rc;
    return gn_go<1>(a, VW, g->dtype, (hipStream_t)stream);
}

int az_group_norm_act_backward(const az_group_norm* g, const void* dy, const void* x, const void* weight, const void* bias,
                               const void* residual, const double* stats, void* dx, void* dweight, void* dbias,
                               void* dresidual, void* workspace, int64_t workspace_bytes, void* stream) {
    if (gn_check(g, "az_group_norm_act_backward")) return -1;
    hipStream_t st = (hipStream_t)stream;
    if (g->batch && (!dy || !x || !stats)) return az_fail("az_group_norm_act_backward: null pointer");
    if (dresidual && !residual) return az_fail("az_group_norm_act_backward: a residual's gradient without a residual");
    if (workspace_bytes < az_group_norm_workspace_bytes(g, 1) || (g->batch && !workspace))
        return az_fail("az_group_norm_act_backward: workspace too small");
    const void* all[] = {dy, x, residual, dx, dresidual};
    const int VW = gn_width(g, all, 5);
    GnArgs a = gn_plan(g, VW);
    a.dy = dy; a.x = x; a.w = weight; a.b = bias; a.res = residual; a.stats = const_cast<double*>(stats);
    a.dx = dx; a.dres = dresidual;
    a.part = dx ? (double*)workspace : nullptr;
    const bool params = dweight || dbias;
    a.dpart = params ? (float*)((char*)workspace + gn_part_bytes(a)) : nullptr;
    if (g->batch) {
        if (int rc = gn_go<2>(a, VW, g->dtype, st)) return rc;
        if (dx) { if (int rc = gn_go<3>(a, VW, g->dtype, st)) return rc; }
    }
    if (params) {
        hipLaunchKernelGGL(k_gn_dparams, dim3((unsigned)((2 * a.C + 15) / 16)), dim3(1024), 0, st, a.dpart, a.N * a.chunks, a.C,
                           a.wtype, dweight, dbias);
        AZ_LAUNCH_CHECK("k_gn_dparams");
    }
    return 0;
}

}  // extern "C"
