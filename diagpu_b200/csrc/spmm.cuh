/*
 * spmm.cuh -- what the translation units of the block-vector product share
 * (spmm.cu: plan, choice of form and C entry points; spmm_f32, spmm_f16,
 * spmm_bf16.cu: CUDA-core kernels of a type; spmm_tc.cu: tcgen05 kernels): the
 * plan, argument blocks, activations, expert lookup.
 */
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <string.h>

#include <atomic>
#include <type_traits>
#include <vector>

#include "../../include/diagpu_b200.h"

namespace dia {

/* Up to four diagonals whose offsets share a multiple of four: slot s holds
 * the storage index of offset base + s, or -1.  col: where input i0 + base of
 * a window lies (Windows). */
struct __align__(32) Quad {
    int base;
    int k[4];
    int col;
    int pad[2];
};

/* The inputs that a tile of outputs i0 .. i0+F-1 reads through diagonals
 * [k0, k1) of the sorted list, side by side in shared memory: spans [k0, k1)
 * of the span table, `cols` columns in all.  A span holds inputs i0 + from ..
 * i0 + from + len - 1 from column `at` on; from, len and at are multiples of
 * eight, and at least eight columns follow the last input that is read. */
struct __align__(16) InputSpan {
    int from, len, at, pad;
};
struct __align__(16) GradWindow {
    int k0, k1, s0, s1;
    int cols, pad[3];
};

/* A tile of 128 outputs from i0 reads, for diagonal d, inputs i0+d ..
 * i0+d+127.  Boxes are the 64-wide pieces of input, disjoint and in ascending
 * order, that cover all of these: inputs i0+col .. i0+col+63, col a multiple
 * of 8 (16 bytes: where a TMA copy may start).  Diagonals [k0, k1) of the
 * sorted list meet it. */
struct __align__(16) Box {
    int col;
    int k0, k1;
    int pad;
};

constexpr int kTileWarps = 8;                   /* of spmm_tile_kernel and spmm_grad_kernel */
constexpr int kGradDiags = 8;                   /* most diagonals of a warp of the latter */
constexpr int kTileF[3] = {256, 512, 1024};   /* feature tiles of spmm_tile_kernel */

struct SpmmDir {
    const Box* boxes;    /* device */
    const int2* offs;    /* device: (offset, storage index), ascending */
    int nboxes;
    /* CUDA-core form: per feature tile one window over all diagonals, its
     * spans, and the column of each diagonal and of each quad */
    const Quad* quads[3];
    const InputSpan* spans[3];
    const int* cols[3];
    int nquads, nspans[3], width[3];
    /* gradient of the diagonals, 128 features: windows over groups of diagonals */
    const GradWindow* wins;
    const InputSpan* wspans;
    const InputSpan* tile_span;   /* the tile's own 128 features */
    const int* wcols;
    int nwins, wwidth, wdiags;
};

}  // namespace dia

struct DiaSpmmPlan {
    int n_rows, n_cols, K;
    int device;
    void* blob;          /* device: every table of the plan */
    dia::SpmmDir fwd, trn;
};

namespace dia {

/* rows [r0, r1) of expert e; e < 0: nothing to do */
struct RowGroup {
    int e;
    int r0, r1;
    int hi;              /* end of the expert's rows */
    int part, nparts;    /* of the expert's parts */
    int slot;            /* index of its first part among experts of several parts */
};

/* seg is the caller's device memory: entries are clamped to [0, M] and a
 * decreasing pair is an empty expert, so no value of it leads out of the
 * block (rows that two experts claim are computed by both). */
__device__ __forceinline__ void expert_rows(const long long* seg, int e, int M, int& lo, int& hi)
{
    const long long a = seg[e], b = seg[e + 1];
    lo = (int)(a < 0 ? 0 : (a > M ? M : a));
    hi = (int)(b < 0 ? 0 : (b > M ? M : b));
    if (hi < lo) hi = lo;
}

/* The g-th group of at most `per` consecutive rows of one expert, experts in
 * order; an expert without rows has one empty group where `empties` is set,
 * else none.  All 32 lanes call it and get the same answer.  Without seg the
 * block is one expert. */
__device__ __forceinline__ RowGroup row_group(const long long* seg, int E, int M, int per,
                                              long long g, bool empties)
{
    RowGroup r;
    if (!seg) {
        const int cnt = max((M + per - 1) / per, empties ? 1 : 0);
        r.e = g < cnt ? 0 : -1;
        r.r0 = (int)min((long long)M, g * per);
        r.r1 = (int)min((long long)M, (g + 1) * per);
        r.hi = M;
        r.part = (int)g;
        r.nparts = cnt;
        r.slot = 0;
        return r;
    }
    const int lane = threadIdx.x & 31;
    int slot0 = 0, nlo = 0, nhi = 0;
    if (lane < E) expert_rows(seg, lane, M, nlo, nhi);
    for (int e0 = 0; e0 < E; e0 += 32) {
        const int e = e0 + lane;
        int lo = nlo, hi = nhi, cnt = 0;
        /* the next experts' rows are on their way while these are counted */
        if (e + 32 < E) expert_rows(seg, e + 32, M, nlo, nhi);
        if (e < E) cnt = max((hi - lo + per - 1) / per, empties ? 1 : 0);
        int inc = cnt, sl = cnt > 1 ? cnt : 0;
        int sinc = sl;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, d);
            const int v = __shfl_up_sync(0xffffffffu, sinc, d);
            if (lane >= d) {
                inc += u;
                sinc += v;
            }
        }
        const int total = __shfl_sync(0xffffffffu, inc, 31);
        if (g < total) {
            const unsigned hit = __ballot_sync(0xffffffffu, g < inc);
            const int src = __ffs(hit) - 1;
            const int part = (int)g - __shfl_sync(0xffffffffu, inc - cnt, src);
            lo = __shfl_sync(0xffffffffu, lo, src);
            hi = __shfl_sync(0xffffffffu, hi, src);
            r.e = e0 + src;
            r.r0 = (int)min((long long)hi, lo + (long long)part * per);
            r.r1 = (int)min((long long)hi, (long long)r.r0 + per);
            r.hi = hi;
            r.part = part;
            r.nparts = __shfl_sync(0xffffffffu, cnt, src);
            r.slot = slot0 + __shfl_sync(0xffffffffu, sinc - sl, src);
            return r;
        }
        g -= total;
        slot0 += __shfl_sync(0xffffffffu, sinc, 31);
    }
    r.e = -1;
    r.r0 = r.r1 = r.hi = r.part = r.nparts = r.slot = 0;
    return r;
}

/* how many such groups there are (whole warp) */
__device__ __forceinline__ long long row_groups(const long long* seg, int E, int M, int per)
{
    if (!seg) return (M + per - 1) / per;
    long long n = 0;
    for (int e = threadIdx.x & 31; e < E; e += 32) {
        int lo, hi;
        expert_rows(seg, e, M, lo, hi);
        n += (hi - lo + per - 1) / per;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
    return n;
}

/* ------------------------------------------------------------ activations */

/* fp32 blocks: CUDA's functions, in forms without a difference of nearly equal
 * numbers, so that a small result (a negative z) is as exact as a large one:
 * z Phi(z) by erfc, tanh by the logistic function. */
template <int ACT>
__device__ __forceinline__ float act_of(float z)
{
    if (ACT == DIA_ACT_RELU) return z < 0.0f ? 0.0f : z;          /* NaN stays NaN */
    if (ACT == DIA_ACT_SILU) return z / (1.0f + expf(-z));
    if (ACT == DIA_ACT_GELU) return 0.5f * z * erfcf(z * -0.70710678f);
    if (ACT == DIA_ACT_GELU_TANH)
        return z / (1.0f + expf(-2.0f * 0.79788456f * z * fmaf(0.044715f * z, z, 1.0f)));
    return z;
}

/* beyond +-16 the tanh form's derivative is 0 or 1, while its z^2 may overflow
 * (NaN stays NaN) */
__device__ __forceinline__ float within16(float z)
{
    return z > 16.0f ? 16.0f : (z < -16.0f ? -16.0f : z);
}

template <int ACT>
__device__ __forceinline__ float dact_of(float z)
{
    if (ACT == DIA_ACT_RELU) return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
    if (ACT == DIA_ACT_SILU) {
        const float s = 1.0f / (1.0f + expf(-z));
        return s * fmaf(z, 1.0f - s, 1.0f);
    }
    if (ACT == DIA_ACT_GELU)
        return 0.5f * erfcf(z * -0.70710678f) + z * 0.39894228f * expf(-0.5f * z * z);
    if (ACT == DIA_ACT_GELU_TANH) {
        z = within16(z);
        const float s =
            1.0f / (1.0f + expf(-2.0f * 0.79788456f * z * fmaf(0.044715f * z, z, 1.0f)));
        return s + 2.0f * 0.79788456f * z * fmaf(0.134145f * z, z, 1.0f) * s * (1.0f - s);
    }
    return 1.0f;
}

__device__ __forceinline__ float act_any(int act, float z)
{
    switch (act) {
        case DIA_ACT_RELU: return act_of<DIA_ACT_RELU>(z);
        case DIA_ACT_SILU: return act_of<DIA_ACT_SILU>(z);
        case DIA_ACT_GELU: return act_of<DIA_ACT_GELU>(z);
        case DIA_ACT_GELU_TANH: return act_of<DIA_ACT_GELU_TANH>(z);
        default: return z;
    }
}

/* one copy of the functions for every row of a tile: inlined 32 times they
 * did not fit the instruction cache, inlined eight times eight rows of 4096
 * under 33 diagonals, without an activation, took 6.45 us in place of 5.2 */
static __device__ __noinline__ float act1(int act, float z) { return act_any(act, z); }
static __device__ __noinline__ float4 act4(int act, float4 z)
{
    return make_float4(act_any(act, z.x), act_any(act, z.y), act_any(act, z.z), act_any(act, z.w));
}

/* 16-bit blocks: two elements at a time, with the two-element fp32
 * instructions and the hardware's approximations of 2^x and 1/x (relative
 * errors of a few 2^-23).
 *   Phi(-x) = (a1 t + .. + a6 t^6) exp(-x^2 / 2), t = 1 / (1 + p x), x >= 0: the
 *     form of Abramowitz and Stegun's 7.1.26, p and a fitted here to the least
 *     relative error up to x = 13.5 (iterated reweighted least squares, Lawson
 *     1961): 3.7e-6, and 1e-5 with the rounding of x^2.  Theirs bounds the
 *     absolute error, which passes half a step of the result below z = -4.
 *   tanh u = 2 s - 1 with the logistic function s of 2 u.
 * So values are within 2^-16 of themselves, a 32nd of half a step of fp16 or
 * less; z Phi(z) underflows from z = -13 on. */
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 exp2_2(float2 z)
{
    float2 d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d.x) : "f"(z.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d.y) : "f"(z.y));
    return d;
}
__device__ __forceinline__ float2 rcp2(float2 z)
{
    float2 d;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d.x) : "f"(z.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d.y) : "f"(z.y));
    return d;
}

/* 1 / (1 + 2^(c z)) for c = -log2 e times a factor */
__device__ __forceinline__ float2 logistic2(float2 z, float c)
{
    return rcp2(add2(exp2_2(mul2(z, both(c))), both(1.0f)));
}

/* Phi(z), and e = exp(-z^2 / 2) */
__device__ __forceinline__ float2 normal_cdf2(float2 z, float2& e)
{
    const float2 x = make_float2(fabsf(z.x), fabsf(z.y));
    const float2 t = rcp2(fma2(x, both(0.3076393f), both(1.0f)));
    e = exp2_2(mul2(mul2(z, z), both(-0.72134752f)));
    float2 p = fma2(t, both(-0.07581779f), both(0.19163735f));
    p = fma2(p, t, both(0.00532099f));
    p = fma2(p, t, both(0.13731957f));
    p = fma2(p, t, both(0.11854316f));
    p = fma2(p, t, both(0.12299492f));
    p = mul2(p, mul2(t, e));
    const float2 q = fma2(p, both(-1.0f), both(1.0f));
    return make_float2(z.x < 0.0f ? p.x : q.x, z.y < 0.0f ? p.y : q.y);
}

template <int ACT>
__device__ __forceinline__ float2 act2(float2 z)
{
    if (ACT == DIA_ACT_RELU)
        return make_float2(z.x < 0.0f ? 0.0f : z.x, z.y < 0.0f ? 0.0f : z.y);
    if (ACT == DIA_ACT_SILU) return mul2(z, logistic2(z, -1.44269504f));
    if (ACT == DIA_ACT_GELU) {
        float2 e;
        return mul2(z, normal_cdf2(z, e));
    }
    if (ACT == DIA_ACT_GELU_TANH) {
        const float2 u = mul2(z, fma2(mul2(z, both(0.044715f)), z, both(1.0f)));
        return mul2(z, logistic2(u, -2.0f * 0.79788456f * 1.44269504f));
    }
    return z;
}

template <int ACT>
__device__ __forceinline__ float2 dact2(float2 z)
{
    if (ACT == DIA_ACT_RELU) return make_float2(dact_of<ACT>(z.x), dact_of<ACT>(z.y));
    if (ACT == DIA_ACT_SILU) {
        const float2 s = logistic2(z, -1.44269504f);
        return mul2(s, fma2(z, fma2(s, both(-1.0f), both(1.0f)), both(1.0f)));
    }
    if (ACT == DIA_ACT_GELU) {
        float2 e;
        const float2 c = normal_cdf2(z, e);
        return fma2(mul2(z, both(0.39894228f)), e, c);
    }
    if (ACT == DIA_ACT_GELU_TANH) {
        z = make_float2(within16(z.x), within16(z.y));
        const float2 w = mul2(z, both(0.044715f));
        const float2 u = mul2(z, fma2(w, z, both(1.0f)));
        const float2 s = logistic2(u, -2.0f * 0.79788456f * 1.44269504f);
        /* s + 2 z s (1 - s) u', u' = sqrt(2 / pi) (1 + 3 * 0.044715 z^2) */
        const float2 du = fma2(mul2(w, both(3.0f)), z, both(1.0f));
        const float2 k = mul2(mul2(mul2(z, both(2.0f * 0.79788456f)), du),
                              fma2(s, both(-1.0f), both(1.0f)));
        return fma2(k, s, s);
    }
    return both(1.0f);
}

/* --------------------------------------------------------------- elements */

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}

/* pairs of elements in a word */
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u)
{
    return __half22float2(*(const __half2*)&u);
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u)
{
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
/* an infinity, or what would round to one, is the type's largest number (NaN
 * stays NaN) */
template <typename T>
__device__ __forceinline__ uint32_t pack2_finite(float a, float b)
{
    uint32_t d;
    if (std::is_same<T, __half>::value)
        asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    else
        asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
}

/* four consecutive elements, p aligned to four elements (global or shared) */
template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p)
{
    return *(const float4*)p;
}
template <>
__device__ __forceinline__ float4 load4<__half>(const __half* p)
{
    const uint2 u = *(const uint2*)p;
    const float2 a = __half22float2(*(const __half2*)&u.x);
    const float2 b = __half22float2(*(const __half2*)&u.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p)
{
    const uint2 u = *(const uint2*)p;
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                       __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}

__device__ __forceinline__ void store4(float* p, float4 v) { *(float4*)p = v; }
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v)
{
    const T h[4] = {from_f<T>(v.x), from_f<T>(v.y), from_f<T>(v.z), from_f<T>(v.w)};
    uint2 u;
    memcpy(&u, h, 8);
    *(uint2*)p = u;
}

/* ------------------------------------------------------------- arguments */

/* out = act(in * A + bias) + res of one direction, z kept where given */
struct ProdArgs {
    const void* in;
    const void* lo;       /* tensor-core form of dx: the rest of dz (kDzPair), or null */
    bool in32;            /* CUDA-core form of dx: dz is fp32 */
    const void* vals;
    const void* bias;
    const void* res;
    void* z;
    void* out;
    void* pack;           /* tensor-core form: spmm_tc_pack_bytes, 256-byte aligned */
    const long long* seg;
    long long ldi, ldr, ldz, ldo, stride, estride;
    int M, E, n_in, n_out, K;
    int act;
    SpmmDir dir;
    bool trans;
    int groups;           /* set by the tensor-core launch, */
    bool build;           /* and this */
    bool dependent;       /* tensor-core form: a launch of the same call is before it */
    bool early;           /* tensor-core form: inputs are complete when the kernel may begin */
};

/* dvals[k, i] = sum_t dz[t, i] x[t, i + off_k], dbias[i] = sum_t dz[t, i] */
struct GradArgs {
    const void* dz;       /* act other than none: the workspace's */
    const void* lo;       /* tensor-core form: the rest of dz (kDzPair), or null */
    bool dz32;            /* CUDA-core form: dz is fp32 */
    const void* dy;
    const void* z;
    const void* x;
    void* dvals;          /* may be null */
    void* dbias;          /* may be null */
    float* part;          /* [slots][K + 1][stride] sums of experts with several parts */
    const long long* seg;
    long long lddz, lddy, ldz, ldx, stride, estride;
    int M, E, n_rows, n_cols, K, act;
    int per;              /* rows a part */
    long long slots;      /* parts that `part` holds */
    SpmmDir dir;          /* forward */
};

/* ------------------------------------------------------- dependent launches
 *
 * The launches of one call overlap (programmatic dependent launch): a kernel
 * may begin once every CTA of the one before has said dependents_begin() or
 * ended, and dependency_wait() returns when that one has completed.  The
 * first launch of a call is an ordinary one: it begins when all that was on
 * the stream has completed, so arguments in device memory may be read before
 * any wait.  Every later one waits before it ends, so that its own completion
 * means that of all before. */
__device__ __forceinline__ void dependency_wait()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ void dependents_begin()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

/* Allows a kernel `smem` bytes of dynamic shared memory (always the same) on
 * the current device; asks the driver once (`most`: the kernel's own record,
 * one place a device). */
struct SmemRecord {
    std::atomic<int> bytes[64];
};

template <typename K>
static cudaError_t allow_smem(K kernel, int smem, SmemRecord& most)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::atomic<int>* rec = dev >= 0 && dev < 64 ? &most.bytes[dev] : nullptr;
    if (rec && rec->load(std::memory_order_relaxed) >= smem) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && rec) rec->store(smem, std::memory_order_relaxed);
    return e;
}

/* dependent: the launch may overlap the one before, which is of the same call */
template <typename... P, typename... A>
static cudaError_t launch(bool dependent, void (*kernel)(P...), int grid, int block, int smem,
                          cudaStream_t stream, A... args)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = dependent ? 1 : 0;
    cfg.attrs = &at;
    cfg.numAttrs = dependent ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

/* How dz = dy * act'(z) is kept for the gradients that read it.  Rounded to 16
 * bits it would double the variance of their error (0.0024 of a bf16 gradient's
 * size in place of 0.0017), so blocks of 16-bit types keep 32 bits: an fp32
 * for the CUDA cores; for the tensor cores, whose operands are of the block's
 * type, dz rounded to a finite number and, in a second array, the rest of it
 * rounded (2^-18 of dz for bf16; infinite where dz is).  Where there is no
 * activation dz is dy, and kDzSame a copy of a block whose rows TMA does not
 * take. */
enum DzForm { kDzSame, kDzF32, kDzPair };

/* CUDA-core forms (spmm_cores.cuh); join: sums of experts with several parts,
 * for either form of the gradient */
template <typename T>
struct Cores {
    static int product(const ProdArgs& a, cudaStream_t stream);
    static int dz(DzForm form, int act, const void* dy, long long lddy, const void* z,
                  long long ldz, void* dz, void* lo, long long lddz, int M, int n, bool dependent,
                  cudaStream_t stream);
    static int gradient(const GradArgs& a, cudaStream_t stream);
    static int join(const GradArgs& a, cudaStream_t stream);
};

/* Tensor-core forms for 16-bit blocks (spmm_tc.cu).  spmm_tc_block: address
 * and row stride are ones TMA takes. */
bool spmm_tc_block(const void* p, long long ld);
/* 0 where the product makes the operator's boxes itself; spmm_tc_pack then
 * launches nothing */
long long spmm_tc_pack_bytes(const SpmmDir& d, int K, int n_out, long long M, int E);
int spmm_tc_pack(const ProdArgs& a, bool dependent, cudaStream_t stream);
int spmm_tc_product(const ProdArgs& a, int dtype, cudaStream_t stream);
/* make: dz (kDzPair) is made there from dy and z (spmm_tc_makes_dz says whether
 * it can be) */
bool spmm_tc_makes_dz(const GradArgs& a);
int spmm_tc_gradient(const GradArgs& a, int dtype, bool make, bool dependent, cudaStream_t stream);
cudaError_t spmm_tc_status(unsigned int* flags, bool clear);
cudaError_t spmm_tc_test_wait(unsigned long long wait_ns, int withhold);

}  // namespace dia
