/*
 * spmm_tc.cu -- tcgen05 forms of the block-vector product and of the gradient
 * of its diagonals, for fp16 and bf16 blocks.
 *
 * A tile of 128 features meets its inputs through boxes of 64 inputs (Box).
 * Within a box the operator is a dense 128 x 64 matrix of which the diagonals
 * are the entries, so the product over a box is an MMA with 64 * 128
 * multiplications a vector for at most 64 * (diagonals of the box) useful
 * ones.  The tensor cores do twenty times the CUDA cores' rate in 16 bits, and
 * a box that a few diagonals cross is already cheaper there; a band fills its
 * boxes by half or more.
 *
 * spmm_tc_kernel: the operator's boxes of a feature tile are laid out once in
 * shared memory (K-major, 128-byte swizzle) by four warps and kept while the
 * CTA walks along the rows of the block, whose boxes arrive by TMA; one thread
 * issues the MMAs (D = 128 rows x 128 features, fp32, tensor memory, four
 * accumulators), eight warps run the epilogue of one tile under the MMAs of
 * the next.  An operator of more boxes than shared memory holds is laid out
 * again for every four tiles.
 *
 * Zeros of a box meet inputs that no diagonal joins to its features; where
 * such an input is infinite or undefined, so is the sum.  A sum that is not
 * finite is therefore computed again from its terms alone (finite ones had no
 * such input), so results do not depend on the form chosen.
 *
 * Every wait is bounded; when one runs out the kernel records DIA_TC_TIMEOUT
 * (dia_device_status), stops, lets its copies and MMAs land and returns.
 */
#include <algorithm>
#include <climits>

#include "dia_core.cuh"
#include "spmm.cuh"
#include "tcgen05.cuh"

namespace dia {

static __device__ unsigned int g_mm_status;
constexpr unsigned long long kMmWaitNs = 2000000000ull;

constexpr int kTM = 128;             /* rows of a tile */
constexpr int kTN = 128;             /* features of a tile */
constexpr int kBoxCols = 64;         /* one 128-byte swizzle row */
constexpr int kBoxBytes = 128 * kBoxCols * 2;
constexpr int kWSlots = 6;           /* operator boxes in shared memory */
constexpr int kXStages = 6;          /* block boxes in flight */
constexpr int kAccs = 4;             /* accumulators of 128 columns */
constexpr int kBuildWarp0 = 2, kEpiWarp0t = 6, kTcWarps = 14;
constexpr int kEpiThreads = 256;
constexpr int kTcSmem = (kWSlots + kXStages) * kBoxBytes + 1024;

struct MmBars {
    unsigned long long xfull[kXStages], xempty[kXStages];
    unsigned long long wfull[kWSlots], wempty[kWSlots];
    unsigned long long afull[kAccs], aempty[kAccs];
    unsigned long long drain;
};

__device__ __forceinline__ void mbar_init(unsigned long long& b, int count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&b)), "r"(count));
}

/* waits for the phase of `bar` with parity `parity`; false when the kernel
 * gives up (another role did, or this wait ran past its limit) */
__device__ __noinline__ bool mm_wait_long(uint32_t bar, uint32_t parity, volatile int* abort_flag)
{
    const unsigned long long t0 = global_ns();
    for (;;) {
        if (mbar_try(bar, parity)) return true;
        if (*abort_flag) return false;
        if (global_ns() - t0 > kMmWaitNs) {
            *abort_flag = 1;
            atomicOr(&g_mm_status, (unsigned)DIA_TC_TIMEOUT);
            return false;
        }
    }
}

__device__ __forceinline__ bool mm_wait(unsigned long long& b, uint32_t parity,
                                        volatile int* abort_flag)
{
    const uint32_t bar = smem_u32(&b);
    for (int it = 0; it < 64; ++it)
        if (mbar_try(bar, parity)) return true;
    return mm_wait_long(bar, parity, abort_flag);
}

/* without regard to the abort flag: copies and MMAs already issued land */
__device__ void mm_drain(unsigned long long& b, uint32_t parity)
{
    const uint32_t bar = smem_u32(&b);
    const unsigned long long t0 = global_ns();
    while (!mbar_try(bar, parity))
        if (global_ns() - t0 > kMmWaitNs) {
            atomicOr(&g_mm_status, (unsigned)DIA_TC_TIMEOUT);
            return;
        }
}

__device__ __forceinline__ void mm_commit(unsigned long long& b)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 ::"r"(smem_u32(&b)) : "memory");
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc,
                                        bool accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate ? 1u : 0u) : "memory");
}

/* Operand cells are written by these: only the tensor cores read them, so the
 * compiler sees no reader and may drop plain stores. */
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t v)
{
    asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void sts16(uint32_t addr, uint16_t v)
{
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(addr), "h"(v) : "memory");
}

/* copy of a box whose barrier already expects its bytes */
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int y,
                                        uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"((unsigned long long)map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

/* 16 columns of the warp's 32 accumulator rows; the load has completed */
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
          "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
          "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(addr)
        : "memory");
}

/* one column of them */
__device__ __forceinline__ float tmem_ld1(uint32_t addr)
{
    float v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=f"(v) : "r"(addr) : "memory");
    return v;
}

/* ------------------------------------------------- 16 elements of a row */

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

/* `wide`: p is 32-byte aligned and all 16 elements exist (one full sector a
 * lane); else the first n elements one by one */
template <typename T>
__device__ __forceinline__ void store16(T* p, const float (&v)[16], bool wide, int n)
{
    if (wide) {
        uint32_t u[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) u[c] = pack2<T>(v[2 * c], v[2 * c + 1]);
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                     ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]),
                       "r"(u[6]), "r"(u[7]) : "memory");
    } else {
#pragma unroll
        for (int c = 0; c < 16; ++c)
            if (c < n) p[c] = from_f<T>(v[c]);
    }
}

template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&v)[16], bool wide, int n)
{
    if (wide) {
        uint32_t u[8];
        asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]),
                       "=r"(u[6]), "=r"(u[7])
                     : "l"(p));
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float2 f = unpack2<T>(u[c]);
            v[2 * c] = f.x;
            v[2 * c + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = c < n ? to_f(p[c]) : 0.0f;
    }
}

/* the sum of one output's own terms, in ascending order of the offsets */
template <typename T, bool TRANS>
__device__ __noinline__ float product_terms(const ProdArgs& a, int K, int e, long long row, int i)
{
    const T* in = (const T*)a.in + row * a.ldi;
    const T* vals = (const T*)a.vals + e * a.estride;
    float s = 0.0f;
    for (int k = 0; k < K; ++k) {
        const int2 ok = a.dir.offs[k];
        const int j = i + ok.x;
        if ((unsigned)j < (unsigned)a.n_in)
            s = fmaf(to_f(vals[ok.y * a.stride + (TRANS ? j : i)]), to_f(in[j]), s);
    }
    return s;
}

/* A run of tiles of one feature block and one expert. */
struct Run {
    int fb, e, r0, hi, ntiles;
};

__device__ __forceinline__ bool next_run(const ProdArgs& a, long long nt, long long& w,
                                         long long w1, Run& r)
{
    if (w >= w1) return false;
    r.fb = (int)(w / nt);
    const RowGroup g = row_group(a.seg, a.E, a.M, kTM, w % nt, false);
    r.e = g.e;
    r.r0 = g.r0;
    r.hi = g.hi;
    r.ntiles = (int)min((long long)(g.nparts - g.part), w1 - w);
    w += r.ntiles;
    return g.e >= 0;
}

/* boxes of a feature block that hold inputs; one is kept where none does,
 * so that every accumulator is written */
__device__ __forceinline__ bool box_used(const Box& b, int i0, int n_in)
{
    return i0 + b.col < n_in && i0 + b.col + kBoxCols > 0;
}

__device__ __forceinline__ int used_boxes(const SpmmDir& d, int i0, int n_in)
{
    int n = 0;
    for (int b = 0; b < d.nboxes; ++b) n += box_used(d.boxes[b], i0, n_in);
    return n;
}

template <typename T, bool TRANS, int ACT>
__global__ void __launch_bounds__(kTcWarps * 32, 1)
spmm_tc_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ ProdArgs a, int K)
{
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    __shared__ __align__(8) MmBars bars;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ float s_bias[kTN];
    volatile int* abort_flag = &s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned char* wslot = smem;
    unsigned char* xstage = smem + kWSlots * kBoxBytes;

    if (tid == 0) {
        s_abort = 0;
        for (int s = 0; s < kXStages; ++s) {
            mbar_init(bars.xfull[s], 1);
            mbar_init(bars.xempty[s], 1);
        }
        for (int s = 0; s < kWSlots; ++s) {
            mbar_init(bars.wfull[s], 4);
            mbar_init(bars.wempty[s], 1);
        }
        for (int s = 0; s < kAccs; ++s) {
            mbar_init(bars.afull[s], 1);
            mbar_init(bars.aempty[s], 8);
        }
        mbar_init(bars.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&s_tmem)), "r"(kAccs * kTN));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;

    /* this CTA's share of the tiles: feature blocks outer, rows inner, so a
     * block's operator is laid out once for a long stretch of rows */
    const long long nt = row_groups(a.seg, a.E, a.M, kTM);
    const long long items = nt * ((a.n_out + kTN - 1) / kTN);
    long long w = items * blockIdx.x / gridDim.x;
    const long long w1 = items * (blockIdx.x + 1) / gridDim.x;
    const int NB = a.dir.nboxes;
    Run r;

    if (warp == 0) {
        /* ---------------- TMA: the block's boxes */
        int g = 0;
        bool ok = true;
        while (ok && next_run(a, nt, w, w1, r)) {
            const int i0 = r.fb * kTN;
            const int used = used_boxes(a.dir, i0, a.n_in);
            const int group = used <= kWSlots ? 1 : kAccs;
            if (lane == 0) {
                for (int j0 = 0; j0 < r.ntiles && ok; j0 += group)
                    for (int b = 0; b < NB && ok; ++b) {
                        const Box bx = a.dir.boxes[b];
                        if (!(box_used(bx, i0, a.n_in) || (used == 0 && b == 0))) continue;
                        for (int j = j0; j < min(j0 + group, r.ntiles); ++j, ++g) {
                            const int s = g % kXStages;
                            ok = mm_wait(bars.xempty[s], ((g / kXStages) & 1) ^ 1, abort_flag);
                            if (!ok) break;
                            tma_load_2d(smem_u32(xstage + s * kBoxBytes), &tmX, i0 + bx.col,
                                        r.r0 + j * kTM, smem_u32(&bars.xfull[s]), kBoxBytes);
                        }
                    }
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0);
        }
        /* no copy may still be landing when the CTA exits */
        if (lane == 0)
            for (int i = max(0, g - kXStages); i < g; ++i)
                mm_drain(bars.xfull[i % kXStages], (i / kXStages) & 1);
    } else if (warp == 1) {
        /* ---------------- MMA issue */
        const uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) |
                               ((uint32_t)(kTN >> 3) << 17) | ((uint32_t)(kTM >> 4) << 24);
        int g = 0, q = 0, tc = 0;
        bool ok = true;
        while (ok && next_run(a, nt, w, w1, r)) {
            const int i0 = r.fb * kTN;
            const int used = max(1, used_boxes(a.dir, i0, a.n_in));
            const bool keep = used <= kWSlots;
            const int group = keep ? 1 : kAccs;
            if (lane == 0) {
                for (int j0 = 0; j0 < r.ntiles && ok; j0 += group) {
                    const int j1 = min(j0 + group, r.ntiles);
                    const bool last_use = !keep || j1 == r.ntiles;
                    for (int u = 0; u < used && ok; ++u) {
                        const int qs = q + u, slot = qs % kWSlots;
                        if (!keep || j0 == 0)
                            ok = mm_wait(bars.wfull[slot], (qs / kWSlots) & 1, abort_flag);
                        const uint32_t wb = smem_u32(wslot + slot * kBoxBytes);
                        for (int j = j0; j < j1 && ok; ++j, ++g) {
                            const int t = tc + j - j0, acc = t % kAccs;
                            if (u == 0)
                                ok = mm_wait(bars.aempty[acc], ((t / kAccs) & 1) ^ 1, abort_flag);
                            const int s = g % kXStages;
                            ok = ok && mm_wait(bars.xfull[s], (g / kXStages) & 1, abort_flag);
                            if (!ok) break;
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            const uint32_t xb = smem_u32(xstage + s * kBoxBytes);
#pragma unroll
                            for (int kk = 0; kk < kBoxCols / 16; ++kk)
                                mma_f16(tmem + (uint32_t)(acc * kTN), smem_desc(xb + 32u * kk),
                                        smem_desc(wb + 32u * kk), idesc, u > 0 || kk > 0);
                            mm_commit(bars.xempty[s]);
                            if (u == used - 1) mm_commit(bars.afull[acc]);
                        }
                        if (ok && last_use) mm_commit(bars.wempty[slot]);
                    }
                    tc += j1 - j0;
                    if (!keep) q += used;
                }
                if (keep) q += used;
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0);
        }
        if (lane == 0) {
            /* every MMA issued has completed before tensor memory is freed */
            mm_commit(bars.drain);
            mm_drain(bars.drain, 0);
        }
    } else if (warp < kEpiWarp0t) {
        /* ---------------- operator boxes: one feature a thread */
        const int f = (warp - kBuildWarp0) * 32 + lane;
        const uint16_t* vals0 = (const uint16_t*)a.vals;
        int q = 0;
        bool ok = true;
        while (ok && next_run(a, nt, w, w1, r)) {
            const int i0 = r.fb * kTN, i = i0 + f;
            const int used = used_boxes(a.dir, i0, a.n_in);
            const int reps = used <= kWSlots ? 1 : (r.ntiles + kAccs - 1) / kAccs;
            const uint16_t* vals = vals0 + r.e * a.estride;
            for (int rep = 0; rep < reps && ok; ++rep)
                for (int b = 0; b < NB && ok; ++b) {
                    const Box bx = a.dir.boxes[b];
                    if (!(box_used(bx, i0, a.n_in) || (used == 0 && b == 0))) continue;
                    const int slot = q % kWSlots;
                    ok = mm_wait(bars.wempty[slot], ((q / kWSlots) & 1) ^ 1, abort_flag);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const uint32_t row = smem_u32(wslot + slot * kBoxBytes) + f * 128;
#pragma unroll
                    for (int c = 0; c < 8; ++c) sts128(row + ((c ^ (f & 7)) << 4), 0);
                    for (int k0 = bx.k0; k0 < bx.k1; k0 += 8) {
                        uint16_t v[8];
                        int col[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            col[u] = -1;
                            if (k0 + u < bx.k1) {
                                const int2 ok2 = __ldg(&a.dir.offs[k0 + u]);
                                const int c = ok2.x + f - bx.col, j = i + ok2.x;
                                if ((unsigned)c < (unsigned)kBoxCols && i < a.n_out &&
                                    (unsigned)j < (unsigned)a.n_in) {
                                    col[u] = c;
                                    v[u] = __ldg(vals + ok2.y * a.stride + (TRANS ? j : i));
                                }
                            }
                        }
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            if (col[u] >= 0)
                                sts16(row + (((col[u] >> 3) ^ (f & 7)) << 4) + (col[u] & 7) * 2,
                                      v[u]);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&bars.wfull[slot]));
                    ++q;
                }
        }
    } else {
        /* ---------------- epilogue: a lane is a row, a warp 64 features */
        const int half = (warp - kEpiWarp0t) >> 2;
        const uint32_t tq = (uint32_t)(warp & 3);
        const bool al = ((uintptr_t)a.out % 32 == 0) && (a.ldo % 16 == 0);
        const bool alz = ((uintptr_t)a.z % 32 == 0) && (a.ldz % 16 == 0);
        const bool alr = ((uintptr_t)a.res % 32 == 0) && (a.ldr % 16 == 0);
        int tc = 0;
        bool ok = true;
        while (ok && next_run(a, nt, w, w1, r)) {
            const int i0 = r.fb * kTN;
            if (!TRANS) {
                asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory");
                const int f = tid - kEpiWarp0t * 32;
                if (f < kTN)
                    s_bias[f] = a.bias && i0 + f < a.n_out
                                    ? to_f(((const T*)a.bias)[(long long)r.e * a.n_out + i0 + f])
                                    : 0.0f;
                asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory");
            }
            for (int j = 0; j < r.ntiles && ok; ++j, ++tc) {
                const int acc = tc % kAccs;
                ok = mm_wait(bars.afull[acc], (tc / kAccs) & 1, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const long long row = (long long)r.r0 + j * kTM + 32 * (int)tq + lane;
                const bool live = row < r.hi;
                const uint32_t ta = tmem + ((tq * 32) << 16) + (uint32_t)(acc * kTN + 64 * half);
#pragma unroll
                for (int cc = 0; cc < 4; ++cc) {
                    float v[16];
                    tmem_ld16(ta + 16u * cc, v);
                    if (cc == 3) {
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&bars.aempty[acc]));
                    }
                    const int fo = 64 * half + 16 * cc, i = i0 + fo;
                    const int n = a.n_out - i;
                    if (live && n > 0) {
                        float chk = 0.0f;
    #pragma unroll
                        for (int c = 0; c < 16; ++c) chk = fmaf(v[c], 0.0f, chk);
                        if (chk != 0.0f) {   /* some sum is not finite */
    #pragma unroll
                            for (int c = 0; c < 16; ++c)
                                if (c < n && !isfinite(v[c]))
                                    v[c] = product_terms<T, TRANS>(a, K, r.e, row, i + c);
                        }
                        if (!TRANS) {
    #pragma unroll
                            for (int c = 0; c < 16; ++c) v[c] += s_bias[fo + c];
                            if (a.z)
                                store16<T>((T*)a.z + row * a.ldz + i, v, alz && n >= 16, n);
                            if (ACT != DIA_ACT_NONE) {
    #pragma unroll
                                for (int c = 0; c < 16; ++c) v[c] = act_of<ACT>(v[c]);
                            }
                            if (a.res) {
                                float u[16];
                                load16<T>((const T*)a.res + row * a.ldr + i, u, alr && n >= 16, n);
    #pragma unroll
                                for (int c = 0; c < 16; ++c) v[c] += u[c];
                            }
                        }
                        store16<T>((T*)a.out + row * a.ldo + i, v, al && n >= 16, n);
                    }
                    __syncwarp();
                }
            }
        }
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                     ::"r"(tmem), "r"(kAccs * kTN));
}

/* ----------------------------------------------------------- diagonals' gradient
 *
 * sum_t dz[t, i] x[t, i + d] of 128 features and up to four boxes of inputs:
 * D = dz^T x is a 128 x 256 product over the rows of one part of an expert,
 * both operands as TMA leaves them (rows of features: MN-major).  Of D the
 * diagonals are the result; it is copied to shared memory, where a diagonal
 * is a run of consecutive features.  A box of ones beside x makes dbias.
 * Rows of the last stage that are not the part's are cleared in both operands
 * before the MMAs read them. */
constexpr int kGRows = 64;                     /* rows of a stage */
constexpr int kGBoxBytes = kGRows * 128;
constexpr int kGBoxes = 4;                     /* boxes of inputs of a CTA */
constexpr int kGStageBytes = (2 + kGBoxes) * kGBoxBytes;
constexpr int kGStages = 4;
constexpr int kGOnesBytes = 16 * 128;
constexpr int kGSmem = kGStages * kGStageBytes + kGOnesBytes + 1024;
constexpr int kGWarps = 10;                    /* TMA, MMA, eight for the results */
constexpr int kGPitch = kGBoxes * kBoxCols + 1;

/* MN-major operand with the 128-byte swizzle: groups of 64 elements kGBoxBytes
 * apart, eight rows of K 1024 bytes apart */
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr)
{
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3FFF);
    d |= (uint64_t)((kGBoxBytes >> 4) & 0x3FFF) << 16;
    d |= (uint64_t)((1024u >> 4) & 0x3FFF) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

template <typename T>
__device__ __noinline__ float gradient_terms(const GradArgs& a, int r0, int r1, int i, int j)
{
    float s = 0.0f;
    for (int t = r0; t < r1; ++t)
        s = fmaf(to_f(((const T*)a.dz)[t * a.lddz + i]), to_f(((const T*)a.x)[t * a.ldx + j]), s);
    return s;
}

template <typename T>
__global__ void __launch_bounds__(kGWarps * 32, 1)
spmm_grad_tc_kernel(const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmX,
                    const __grid_constant__ GradArgs a, int nfb, int nch)
{
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    __shared__ __align__(8) unsigned long long xfull[kGStages], xempty[kGStages], done;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    volatile int* abort_flag = &s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long b = blockIdx.x;
    const int fb = (int)(b % nfb), ch = (int)(b / nfb % nch);
    const RowGroup rg = row_group(a.seg, a.E, a.M, a.per, b / nfb / nch, true);
    if (rg.e < 0 || (rg.nparts > 1 && rg.slot + rg.part >= a.slots)) return;   /* whole CTA */
    const int i0 = fb * 128;
    /* boxes in nch nearly equal shares */
    const int b0 = (int)((long long)a.dir.nboxes * ch / nch);
    const int nb = (int)((long long)a.dir.nboxes * (ch + 1) / nch) - b0;
    const bool bias = a.dbias && ch == 0;
    const int nst = i0 < a.n_rows ? (rg.r1 - rg.r0 + kGRows - 1) / kGRows : 0;
    unsigned char* ones = smem + kGStages * kGStageBytes;

    if (tid == 0) {
        s_abort = 0;
        for (int s = 0; s < kGStages; ++s) {
            mbar_init(xfull[s], 1);
            mbar_init(xempty[s], 1);
        }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    {
        const uint32_t one = pack2<T>(1.0f, 1.0f);
        for (int o = tid; o < kGOnesBytes / 16; o += kGWarps * 32)
            sts128(smem_u32(ones) + 16 * o, one);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&s_tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            int g = 0;
            for (; g < nst; ++g) {
                const int s = g % kGStages, r = rg.r0 + g * kGRows;
                ok = mm_wait(xempty[s], ((g / kGStages) & 1) ^ 1, abort_flag);
                if (!ok) break;
                const uint32_t st = smem_u32(smem + s * kGStageBytes), bar = smem_u32(&xfull[s]);
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                             ::"r"(bar), "r"((2 + nb) * kGBoxBytes) : "memory");
                tma_box(st, &tmD, i0, r, bar);
                tma_box(st + kGBoxBytes, &tmD, i0 + 64, r, bar);
                for (int c = 0; c < nb; ++c)
                    tma_box(st + (2 + c) * kGBoxBytes, &tmX, i0 + a.dir.boxes[b0 + c].col, r, bar);
            }
            for (int i = max(0, g - kGStages); i < g; ++i)
                mm_drain(xfull[i % kGStages], (i / kGStages) & 1);
        }
    } else if (warp == 1) {
        const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        const uint32_t id0 = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (1u << 16) |
                             ((uint32_t)(128 >> 4) << 24);
        const uint32_t idx = id0 | ((uint32_t)(nb * kBoxCols >> 3) << 17);
        const uint32_t ido = id0 | ((uint32_t)(kBoxCols >> 3) << 17);
        for (int g = 0; g < nst; ++g) {
            const int s = g % kGStages, left = rg.r1 - rg.r0 - g * kGRows;
            ok = mm_wait(xfull[s], (g / kGStages) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            unsigned char* st = smem + s * kGStageBytes;
            if (left < kGRows) {
                /* rows past the part: another expert's, or nobody's */
                const int per = (kGRows - left) * 8;
                for (int o = lane; o < per * (2 + nb); o += 32)
                    sts128(smem_u32(st) + o / per * kGBoxBytes + left * 128 + o % per * 16, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            if (lane == 0) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t sa = smem_u32(st), so = smem_u32(ones);
#pragma unroll
                for (int kk = 0; kk < kGRows / 16; ++kk) {
                    const uint64_t ad = mn_desc(sa + 2048u * kk);
                    if (nb > 0)
                        mma_f16(tmem, ad, mn_desc(sa + 2 * kGBoxBytes + 2048u * kk), idx,
                                g > 0 || kk > 0);
                }
                /* a loop of its own: alternating the two accumulators' MMAs in
                 * one unrolled loop gave undefined sums in the second (nvcc 12.9) */
                if (bias) {
#pragma unroll
                    for (int kk = 0; kk < kGRows / 16; ++kk)
                        mma_f16(tmem + 256, mn_desc(sa + 2048u * kk), mn_desc(so), ido,
                                g > 0 || kk > 0);
                }
                mm_commit(xempty[s]);
            }
            __syncwarp();
        }
        if (lane == 0) {
            mm_commit(done);
            mm_drain(done, 0);
        }
    }
    /* the results: every MMA has completed (the stages are free) */
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    ok = !__syncthreads_or(!ok);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    float* tile = (float*)smem;
    if (ok && warp >= 2 && nst > 0) {
        const uint32_t tq = (uint32_t)(warp & 3);
        const int half = (warp - 2) >> 2, f = 32 * (int)tq + lane;
        for (int c0 = half * 16; c0 < nb * kBoxCols; c0 += 32) {
            float v[16];
            tmem_ld16(tmem + ((tq * 32) << 16) + (uint32_t)c0, v);
#pragma unroll
            for (int c = 0; c < 16; ++c) tile[f * kGPitch + c0 + c] = v[c];
        }
        if (bias && half == 0) {
            const float v = tmem_ld1(tmem + ((tq * 32) << 16) + 256u);
            const int i = i0 + f;
            if (i < a.n_rows) {
                if (rg.nparts > 1)
                    a.part[((long long)(rg.slot + rg.part) * (a.K + 1) + a.K) * a.stride + i] = v;
                else
                    ((T*)a.dbias)[(long long)rg.e * a.n_rows + i] = from_f<T>(v);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    if (!ok) return;
    if (nst == 0 && bias && tid < 128 && i0 + tid < a.n_rows) {
        if (rg.nparts > 1)
            a.part[((long long)(rg.slot + rg.part) * (a.K + 1) + a.K) * a.stride + i0 + tid] = 0.0f;
        else
            ((T*)a.dbias)[(long long)rg.e * a.n_rows + i0 + tid] = from_f<T>(0.0f);
    }
    if (!a.dvals) return;
    for (int c = 0; c < nb; ++c) {
        const Box bx = a.dir.boxes[b0 + c];
        for (int k = bx.k0 + warp; k < bx.k1; k += kGWarps) {
            const int2 ok2 = a.dir.offs[k];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int f = 32 * s + lane, i = i0 + f, p = ok2.x + f - bx.col;
                if ((unsigned)p >= (unsigned)kBoxCols || i >= a.stride) continue;
                const int j = i + ok2.x;
                float v = 0.0f;
                /* an entry outside the matrix, or in the padding, has no gradient */
                if (nst > 0 && i < a.n_rows && (unsigned)j < (unsigned)a.n_cols) {
                    v = tile[f * kGPitch + c * kBoxCols + p];
                    if (!isfinite(v)) v = gradient_terms<T>(a, rg.r0, rg.r1, i, j);
                }
                if (rg.nparts > 1)
                    a.part[((long long)(rg.slot + rg.part) * (a.K + 1) + ok2.y) * a.stride + i] = v;
                else
                    ((T*)a.dvals)[rg.e * a.estride + ok2.y * a.stride + i] = from_f<T>(v);
            }
        }
    }
}

/* ---------------------------------------------------------------- host */

bool spmm_tc_block(const void* p, long long ld)
{
    return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && encode_tiled();
}

/* rows x width block of 16-bit elements; box of 64 columns x box_rows */
static bool block_map(CUtensorMap* map, const void* base, int dtype, int width, int rows,
                      long long ld, int box_rows)
{
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {kBoxCols, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map,
              dtype == DIA_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
              2, (void*)base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool TRANS, int ACT>
static int launch_tc(const CUtensorMap& map, const ProdArgs& a, int K, cudaStream_t stream)
{
    const long long tiles = a.seg ? a.M / kTM + std::min(a.E, a.M) : (a.M + kTM - 1) / kTM;
    const long long items = tiles * ((a.n_out + kTN - 1) / kTN);
    const int grid = (int)std::min<long long>(items, num_sms());
    DIA_TRY_CUDA(cudaFuncSetAttribute(spmm_tc_kernel<T, TRANS, ACT>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmem));
    spmm_tc_kernel<T, TRANS, ACT><<<grid, kTcWarps * 32, kTcSmem, stream>>>(map, a, K);
    DIA_TRY_CUDA(cudaGetLastError());
    return DIA_OK;
}

template <typename T>
static int launch_tc_type(const CUtensorMap& map, const ProdArgs& a, int K, cudaStream_t stream)
{
    if (a.trans) return launch_tc<T, true, DIA_ACT_NONE>(map, a, K, stream);
    switch (a.act) {
        case DIA_ACT_RELU: return launch_tc<T, false, DIA_ACT_RELU>(map, a, K, stream);
        case DIA_ACT_SILU: return launch_tc<T, false, DIA_ACT_SILU>(map, a, K, stream);
        case DIA_ACT_GELU: return launch_tc<T, false, DIA_ACT_GELU>(map, a, K, stream);
        case DIA_ACT_GELU_TANH: return launch_tc<T, false, DIA_ACT_GELU_TANH>(map, a, K, stream);
        default: return launch_tc<T, false, DIA_ACT_NONE>(map, a, K, stream);
    }
}

int spmm_tc_product(const ProdArgs& a, int dtype, cudaStream_t stream)
{
    CUtensorMap map;
    if (!block_map(&map, a.in, dtype, a.n_in, a.M, a.ldi, kTM))
        return fail(DIA_ERR_CUDA, "dia_spmm: cuTensorMapEncodeTiled failed");
    return dtype == DIA_F16 ? launch_tc_type<__half>(map, a, a.K, stream)
                            : launch_tc_type<__nv_bfloat16>(map, a, a.K, stream);
}

template <typename T>
static int launch_grad_tc(const CUtensorMap& md, const CUtensorMap& mx, const GradArgs& a,
                          cudaStream_t stream)
{
    const int nfb = (int)((a.stride + 127) / 128);
    const int nch = std::max(1, (a.dir.nboxes + kGBoxes - 1) / kGBoxes);
    const long long parts = a.seg ? a.M / a.per + a.E : std::max(1, (a.M + a.per - 1) / a.per);
    const long long grid = parts * nfb * nch;
    if (grid > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm_backward: block too large");
    DIA_TRY_CUDA(cudaFuncSetAttribute(spmm_grad_tc_kernel<T>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, kGSmem));
    spmm_grad_tc_kernel<T><<<(unsigned)grid, kGWarps * 32, kGSmem, stream>>>(md, mx, a, nfb, nch);
    DIA_TRY_CUDA(cudaGetLastError());
    return DIA_OK;
}

int spmm_tc_gradient(const GradArgs& a, int dtype, cudaStream_t stream)
{
    CUtensorMap md, mx;
    if (!block_map(&md, a.dz, dtype, a.n_rows, a.M, a.lddz, kGRows) ||
        !block_map(&mx, a.x, dtype, a.n_cols, a.M, a.ldx, kGRows))
        return fail(DIA_ERR_CUDA, "dia_spmm_backward: cuTensorMapEncodeTiled failed");
    return dtype == DIA_F16 ? launch_grad_tc<__half>(md, mx, a, stream)
                            : launch_grad_tc<__nv_bfloat16>(md, mx, a, stream);
}

cudaError_t spmm_tc_status(unsigned int* flags, bool clear)
{
    cudaError_t e = cudaMemcpyFromSymbol(flags, g_mm_status, sizeof(unsigned int));
    if (e == cudaSuccess && clear) {
        const unsigned int z = 0;
        e = cudaMemcpyToSymbol(g_mm_status, &z, sizeof(unsigned int));
    }
    return e;
}

}  // namespace dia
