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
 * spmm_pack_kernel writes the boxes of the operator as the tensor cores read
 * them.  spmm_tc_kernel keeps a feature tile's boxes in shared memory while
 * the CTA walks along the rows of the block, whose boxes arrive by TMA; one
 * thread issues the MMAs (D = 128 rows x 128 features, fp32, tensor memory,
 * four accumulators), twelve warps run the epilogue of one tile under the MMAs
 * of the next.  An operator of more boxes than shared memory holds is read
 * again for every four tiles.
 *
 * 4096 rows of 4096 under 129 diagonals, bf16, bias, GELU, residual, z kept:
 * 40 us (135 MB: 3.4 TB/s; 21 us at the memory's rate).  The epilogue's
 * instructions and the first tile's latency make it up: a CTA has eight tiles,
 * DRAM is 26 % busy, the tensor cores 11 %, instructions issue in 43 % of the
 * cycles.
 *
 * Zeros of a box meet inputs that no diagonal joins to its features; where
 * such an input is infinite or undefined, so is the sum.  Sums that are not
 * finite, and those beside them in the row, are therefore computed again from
 * their terms alone (rows_again), so an infinity reaches the same outputs in
 * either form.
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
/* limit of every wait, and a test switch: CTA 0 withholds its first copy of
 * the block, so that the MMA issuer's wait runs out (dia_test_tc_wait) */
static __device__ unsigned long long g_mm_wait_ns = kMmWaitNs;
static __device__ int g_mm_withhold;

constexpr int kTM = 128;             /* rows of a tile */
constexpr int kTN = 128;             /* features of a tile */
constexpr int kBoxCols = 64;         /* one 128-byte swizzle row */
constexpr int kBoxBytes = 128 * kBoxCols * 2;
constexpr int kWSlots = 6;           /* operator boxes in shared memory */
constexpr int kXStages = 5;          /* block boxes in flight */
constexpr int kAccs = 4;             /* accumulators of 128 columns */
constexpr int kGroup = kAccs;        /* tiles that share a reading of a large operator */
constexpr int kSharedBoxes = 64;     /* boxes whose places are kept in shared memory */
constexpr int kEpiWarp0t = 4, kEpiQuad = 3, kEpiWarpsT = 4 * kEpiQuad, kTcWarps = kEpiWarp0t + kEpiWarpsT;
constexpr int kOffs = 512;           /* offsets kept in shared memory */
constexpr int kEpiThreads = kEpiWarpsT * 32;
constexpr int kEpiBuf = 32 * 64;     /* a warp's 32 rows of 32 features */
constexpr int kTcSmem = (kWSlots + kXStages) * kBoxBytes + 2 * kEpiWarpsT * kEpiBuf + 1024;

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
 * gives up (another role did, or this wait ran past its limit).  state[0]: it
 * gives up; state[1] counts the steps of rows_again, which takes its time: the
 * limit runs from the last of them. */
__device__ __noinline__ bool mm_wait_long(uint32_t bar, uint32_t parity, volatile int* state)
{
    unsigned long long t0 = global_ns();
    int step = state[1];
    for (;;) {
        if (mbar_try(bar, parity)) return true;
        if (state[0]) return false;
        if (state[1] != step) {
            step = state[1];
            t0 = global_ns();
        }
        if (global_ns() - t0 > g_mm_wait_ns) {
            state[0] = 1;
            atomicOr(&g_mm_status, (unsigned)DIA_TC_TIMEOUT);
            return false;
        }
    }
}

__device__ __forceinline__ bool mm_wait(uint32_t bar, uint32_t parity, volatile int* state)
{
    return mbar_try(bar, parity) || mm_wait_long(bar, parity, state);
}

/* without regard to the state: copies and MMAs already issued land */
__device__ void mm_drain(uint32_t bar, uint32_t parity)
{
    const unsigned long long t0 = global_ns();
    while (!mbar_try(bar, parity))
        if (global_ns() - t0 > g_mm_wait_ns) {
            atomicOr(&g_mm_status, (unsigned)DIA_TC_TIMEOUT);
            return;
        }
}

__device__ __forceinline__ void mm_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 ::"r"(bar) : "memory");
}

/* the same one lane of the warp wherever it is asked; unlike lane == 0 it
 * leaves the warp's control flow uniform */
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

/* a ring of N stages: the stage and the parity of its current round */
template <int N>
struct Ring {
    uint32_t s = 0, round = 0;
    __device__ __forceinline__ void next()
    {
        if (++s == N) {
            s = 0;
            round ^= 1;
        }
    }
    /* address of the stage's barrier in an array of them */
    __device__ __forceinline__ uint32_t bar(uint32_t base) const { return base + 8 * s; }
};

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
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w)
{
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};"
                 ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&v)[4])
{
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
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

/* 32 columns */
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
          "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
          "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
          "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]),
          "=f"(v[31])
        : "r"(addr)
        : "memory");
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, int bytes, uint32_t bar)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                 ::"r"(bar), "r"(bytes) : "memory");
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

/* The operator as the tensor cores read it: for every expert, feature tile and
 * box a dense 128 x 64 matrix, K-major with the 128-byte swizzle.  One CTA
 * makes one box.  It copies the pieces of the diagonals that cross the box to
 * shared memory (each 128 consecutive features, all copies in flight at
 * once), then a thread gathers eight columns of a feature at a time: their
 * offsets are consecutive, a table gives their rows. */
constexpr int kPackRows = 191;                      /* offsets that can cross a box */
constexpr int kPackPitch = 136;                     /* 128 features, up to 7 before them */
constexpr int kPackSmem = kBoxBytes + kPackRows * kPackPitch * 2;

template <bool TRANS>
__global__ void __launch_bounds__(256) spmm_pack_kernel(const __grid_constant__ ProdArgs a)
{
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ int16_t s_row[kPackRows + 1];
    __shared__ int2 s_off[kPackRows + 1];
    dependents_begin();
    const int tid = threadIdx.x;
    unsigned char* box = smem_raw;
    uint16_t* slab = (uint16_t*)(smem_raw + kBoxBytes);
    const int nb = a.dir.nboxes, nfb = (a.n_out + kTN - 1) / kTN;
    const int b = blockIdx.x % nb, fb = blockIdx.x / nb % nfb, e = blockIdx.x / nb / nfb;
    if (a.seg) {
        int lo, hi;
        expert_rows(a.seg, e, a.M, lo, hi);
        if (lo == hi) {   /* nobody reads them */
            dependency_wait();
            return;
        }
    }
    const Box bx = a.dir.boxes[b];
    const int nk = bx.k1 - bx.k0, i0 = fb * kTN;
    for (int d = tid; d < kPackRows; d += 256) s_row[d] = -1;
    if (tid < nk) s_off[tid] = a.dir.offs[bx.k0 + tid];
    __syncthreads();
    if (tid < nk) s_row[s_off[tid].x - (bx.col - 127)] = (int16_t)tid;
    const uint16_t* vals = (const uint16_t*)a.vals + e * a.estride;
    /* rows of 17 pieces of eight elements, from the aligned element at or
     * before the first; elements outside [0, stride) are not read */
    for (int o = tid; o < nk * 17; o += 256) {
        const int k = o / 17, c = o - k * 17;
        const int first = (TRANS ? i0 + s_off[k].x : i0) & ~7;
        const int x = first + c * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (x >= 0 && x < a.stride) v = __ldg((const uint4*)(vals + s_off[k].y * a.stride + x));
        *(uint4*)(slab + k * kPackPitch + c * 8) = v;
    }
    __syncthreads();
    /* element (f, c) is offset col + c - f; lanes take consecutive features */
    const int f = tid & 127, i = i0 + f;
#pragma unroll
    for (int q = tid >> 7; q < 8; q += 2) {
        uint32_t u[4] = {0, 0, 0, 0};
        if (i < a.n_out) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const int t = 8 * q + c - f + 127;            /* index into s_row */
                const int d = t + bx.col - 127;
                const int k = s_row[t];
                if (k >= 0 && (unsigned)(i + d) < (unsigned)a.n_in) {
                    const int shift = TRANS ? (i0 + d) & 7 : 0;
                    const uint32_t v = slab[k * kPackPitch + f + shift];
                    u[c >> 1] |= c & 1 ? v << 16 : v;
                }
            }
        }
        *(uint4*)(box + f * 128 + ((q ^ (f & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
    }
    __syncthreads();
    uint4* dst = (uint4*)((char*)a.pack + (long long)blockIdx.x * kBoxBytes);
#pragma unroll
    for (int o = 0; o < kBoxBytes / 16; o += 256) dst[o + tid] = ((const uint4*)box)[o + tid];
    dependency_wait();
}

/* The same by the epilogue's warps of spmm_tc_kernel, straight into its
 * operator slots: for a CTA that keeps one feature tile and expert this takes
 * less than a launch.  Boxes [b0, b1) of tile i0 go to slots 0, 1, ..; mem:
 * the epilogue's buffers, not in use yet. */
constexpr int kInlineDiags = 160;
constexpr int kInlineOffs = kWSlots * 192 * 2;                 /* after the tables of rows */
constexpr int kInlineSlab = kInlineOffs + kInlineDiags * 8;    /* after the offsets */
static_assert(kInlineSlab % 16 == 0 &&
              kInlineSlab + kInlineDiags * kPackPitch * 2 <= 2 * kEpiWarpsT * kEpiBuf, "slab");

template <bool TRANS>
__device__ __forceinline__ void build_operator(const ProdArgs& a, int K, int e, unsigned char* mem,
                                               uint32_t slots, int i0, int b0, int b1, const int* cols,
                                               int t)
{
    int16_t* s_row = (int16_t*)mem;
    int2* s_off = (int2*)(mem + kInlineOffs);
    uint16_t* slab = (uint16_t*)(mem + kInlineSlab);
    for (int c = t; c < (b1 - b0) * 192; c += kEpiThreads) s_row[c] = -1;
    if (t < K) s_off[t] = a.dir.offs[t];
    asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory");
    for (int b = b0; b < b1; ++b) {
        const Box bx = a.dir.boxes[b];
        const int k = bx.k0 + t;
        if (k < bx.k1) s_row[(b - b0) * 192 + s_off[k].x - (bx.col - 127)] = (int16_t)k;
    }
    const uint16_t* vals = (const uint16_t*)a.vals + e * a.estride;
    /* four pieces a thread on their way at a time */
    for (int o0 = t; o0 < K * 17; o0 += 4 * kEpiThreads) {
        uint4 v[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int o = min(o0 + h * kEpiThreads, K * 17 - 1), k = o / 17;
            const int2 of = s_off[k];
            const int x = ((TRANS ? i0 + of.x : i0) & ~7) + (o - k * 17) * 8;
            v[h] = make_uint4(0, 0, 0, 0);
            if (x >= 0 && x < a.stride) v[h] = __ldg((const uint4*)(vals + of.y * a.stride + x));
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int o = o0 + h * kEpiThreads, k = o / 17;
            if (o < K * 17) *(uint4*)(slab + k * kPackPitch + (o - k * 17) * 8) = v[h];
        }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory");
    /* eight columns of a feature at a time; consecutive threads, consecutive
     * features.  Consecutive offsets need no table, and entries of an inner
     * tile no check. */
    const int d0 = s_off[0].x, d1 = s_off[K - 1].x;
    const bool band = d1 - d0 == K - 1;
    const bool inner = i0 + 128 <= a.n_out && i0 + d0 >= 0 && i0 + 127 + d1 < a.n_in;
    for (int c = t; c < (b1 - b0) * 1024; c += kEpiThreads) {
        const int b = c >> 10, q = (c >> 7) & 7, f = c & 127, i = i0 + f;
        const int d = cols[b0 + b] + 8 * q - f;      /* offset of the first column */
        uint32_t u[4] = {0, 0, 0, 0};
        if (band && inner) {
            const uint16_t* p = slab + (d - d0) * kPackPitch + f;
#pragma unroll
            for (int h = 0; h < 8; ++h)
                if ((unsigned)(d - d0 + h) < (unsigned)K) {
                    const uint32_t v = p[h * kPackPitch + (TRANS ? (i0 + d + h) & 7 : 0)];
                    u[h >> 1] |= h & 1 ? v << 16 : v;
                }
        } else if (i < a.n_out) {
            const int16_t* rows = s_row + b * 192 + 8 * q - f + 127;
#pragma unroll
            for (int h = 0; h < 8; ++h) {
                const int k = rows[h];
                if (k >= 0 && (unsigned)(i + d + h) < (unsigned)a.n_in) {
                    const uint32_t v = slab[k * kPackPitch + f + (TRANS ? (i0 + d + h) & 7 : 0)];
                    u[h >> 1] |= h & 1 ? v << 16 : v;
                }
            }
        }
        sts128(slots + b * kBoxBytes + f * 128 + ((q ^ (f & 7)) << 4), u[0], u[1], u[2], u[3]);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory");
}

/* Rows of a 32 x 32 block with sums that are not finite (bits of `rows`, from
 * row0 on), computed from their own terms in ascending order of the offsets
 * and stored.  Lanes are features, so that values and inputs are read side by
 * side, and a value serves kAgainRows rows (eight would leave the caller too
 * few registers: 41 -> 43 us for blocks that never come here).  4096 rows of
 * 4096, 129 diagonals, fp16, no input finite: 3.7 ms, a tenth of what a lane
 * for each row took and ten times the CUDA-core form; one infinity: 0.11 ms. */
constexpr int kAgainRows = 4;

template <typename T, bool TRANS, int ACT>
__device__ __noinline__ void rows_again(const ProdArgs& a, int K, int e, int row0, int i,
                                        uint32_t rows, volatile int* state)
{
    const bool on = i < a.n_out;
    const T* vals = (const T*)a.vals + e * a.estride;
    const float bias =
        !TRANS && a.bias && on ? to_f(((const T*)a.bias)[(long long)e * a.n_out + i]) : 0.0f;
    while (rows) {
        int r[kAgainRows];
        float sum[kAgainRows];
        const T* in[kAgainRows];
        const int n = min(kAgainRows, __popc(rows));
        const long long rest = TRANS && a.lo ? (const T*)a.lo - (const T*)a.in : 0;
#pragma unroll
        for (int u = 0; u < kAgainRows; ++u) {   /* a row twice where there are fewer */
            r[u] = row0 + (u < n ? __ffs(rows) - 1 : r[0] - row0);
            rows &= rows - 1;
            in[u] = (const T*)a.in + (long long)r[u] * a.ldi;
            sum[u] = 0.0f;
        }
#pragma unroll 4
        for (int k = 0; k < K; ++k) {
            const int2 ok = __ldg(&a.dir.offs[k]);
            const int j = i + ok.x;
            if (on && (unsigned)j < (unsigned)a.n_in) {
                const float w = to_f(vals[ok.y * a.stride + (TRANS ? j : i)]);
#pragma unroll
                for (int u = 0; u < kAgainRows; ++u) {
                    float x = to_f(in[u][j]);
                    if (TRANS && rest) x += to_f(in[u][j + rest]);
                    sum[u] = fmaf(w, x, sum[u]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kAgainRows; ++u) {
            if (!on || u >= n) continue;
            float y = sum[u] + bias;
            if (!TRANS) {
                if (a.z) ((T*)a.z)[r[u] * a.ldz + i] = from_f<T>(y);
                y = act2<ACT>(both(y)).x;
                if (a.res) y += to_f(((const T*)a.res)[r[u] * a.ldr + i]);
            }
            ((T*)a.out)[r[u] * a.ldo + i] = from_f<T>(y);
        }
        if ((threadIdx.x & 31) == 0) atomicAdd((int*)&state[1], 1);   /* waits wait on */
    }
}

/* A run of tiles of one feature block and one expert. */
struct Run {
    int fb, e, r0, hi, ntiles;
};

/* A CTA's share of the tiles: w, w + step, .. below w1 of the list that has
 * feature blocks outside and the nt tiles of rows inside. */
struct Share {
    long long w, w1, nt;
    int step, fb0;
};

__device__ __forceinline__ bool next_run(const ProdArgs& a, Share& s, Run& r)
{
    if (s.w >= s.w1) return false;
    r.fb = s.fb0;
    long long tile = s.w - s.fb0 * s.nt;
    if (tile >= s.nt) {   /* only where a share crosses feature blocks */
        r.fb = (int)(s.w / s.nt);
        tile = s.w - r.fb * s.nt;
        s.fb0 = r.fb;
    }
    const RowGroup g = row_group(a.seg, a.E, a.M, kTM, tile, false);
    r.e = g.e;
    r.r0 = g.r0;
    r.hi = g.hi;
    r.ntiles = (int)((min((long long)(g.nparts - g.part), s.w1 - s.w) + s.step - 1) / s.step);
    s.w += (long long)r.ntiles * s.step;
    return g.e >= 0;
}

/* boxes [b0, b1) of a feature block hold inputs (boxes ascend); one is kept
 * where none does, so that every accumulator is written */
__device__ __forceinline__ void used_boxes(const int* cols, const SpmmDir& d, int i0, int n_in,
                                           int& b0, int& b1)
{
    auto col = [&](int b) { return b < kSharedBoxes ? cols[b] : d.boxes[b].col; };
    b0 = 0;
    b1 = d.nboxes;
    while (b1 > 1 && i0 + col(b1 - 1) >= n_in) --b1;
    while (b0 < b1 - 1 && i0 + col(b0) + kBoxCols <= 0) ++b0;
}

template <typename T, bool TRANS, int ACT>
__global__ void __launch_bounds__(kTcWarps * 32, 1)
spmm_tc_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmL,
               const __grid_constant__ ProdArgs a, int K)
{
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    __shared__ __align__(8) MmBars bars;
    __shared__ uint32_t s_tmem;
    __shared__ int s_state[2];   /* mm_wait_long */
    __shared__ int s_cols[kSharedBoxes];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t wst = smem_u32(smem), xst = wst + kWSlots * kBoxBytes;

    for (int b = tid; b < min(a.dir.nboxes, kSharedBoxes); b += kTcWarps * 32)
        s_cols[b] = a.dir.boxes[b].col;
    if (tid == 0) {
        s_state[0] = s_state[1] = 0;
        for (int s = 0; s < kXStages; ++s) {
            mbar_init(bars.xfull[s], 1);
            mbar_init(bars.xempty[s], 1);
        }
        for (int s = 0; s < kWSlots; ++s) {
            mbar_init(bars.wfull[s], 1);
            mbar_init(bars.wempty[s], 1);
        }
        for (int s = 0; s < kAccs; ++s) {
            mbar_init(bars.afull[s], 1);
            mbar_init(bars.aempty[s], 16);   /* blocks of 32 x 32 */
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

    /* Either (a.groups > 0) the CTA stays with one feature block and takes
     * every groups-th tile of rows: all feature blocks of a few tiles of rows
     * are worked on at the same time, whole rows of the block's memory.  Or it
     * takes a stretch of the list. */
    Share sh;
    sh.nt = row_groups(a.seg, a.E, a.M, kTM);
    const int nfb = (a.n_out + kTN - 1) / kTN;
    if (a.groups > 0) {
        const int fb = blockIdx.x % nfb;
        sh.w = fb * sh.nt + blockIdx.x / nfb;
        sh.w1 = (fb + 1) * sh.nt;
        sh.step = a.groups;
        sh.fb0 = fb;
    } else {
        sh.w = sh.nt * nfb * blockIdx.x / gridDim.x;
        sh.w1 = sh.nt * nfb * (blockIdx.x + 1) / gridDim.x;
        sh.step = 1;
        sh.fb0 = sh.nt > 0 ? (int)(sh.w / sh.nt) : 0;
    }
    const int row_step = sh.step * kTM;
    const int NB = a.dir.nboxes;
    const int halves = TRANS && a.lo ? 2 : 1;   /* of dz: each box of it, then of the rest */
    Run r;

    const uint32_t xfull = smem_u32(bars.xfull), xempty = smem_u32(bars.xempty);
    const uint32_t wfull = smem_u32(bars.wfull), wempty = smem_u32(bars.wempty);
    const uint32_t afull = smem_u32(bars.afull), aempty = smem_u32(bars.aempty);
    if (warp == 0) {
        /* ---------------- TMA: the block's boxes */
        /* dx: the block is dz, which the launch before may still be making */
        if (TRANS && !a.early) dependency_wait();
        Ring<kXStages> x;
        int issued = 0;
        bool ok = true;
        const bool leader = elect_one();
        while (ok && next_run(a, sh, r)) {
            const int i0 = r.fb * kTN;
            int b0, b1;
            used_boxes(s_cols, a.dir, i0, a.n_in, b0, b1);
            const int used = b1 - b0;
            const int group = used <= kWSlots ? 1 : kGroup;
            for (int j0 = 0; j0 < r.ntiles && ok; j0 += group)
                for (int b = b0; b < b1 && ok; ++b) {
                    const int x0 = i0 + (b < kSharedBoxes ? s_cols[b] : a.dir.boxes[b].col);
                    const int n = min(group, r.ntiles - j0) * halves;
                    for (int j = 0; j < n; ++j) {
                        ok = mm_wait(x.bar(xempty), x.round ^ 1, s_state);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        const bool rest = TRANS && halves == 2 && (j & 1);
                        const int tile = j0 + (TRANS && halves == 2 ? j >> 1 : j);
                        if (leader && !(g_mm_withhold && blockIdx.x == 0 && issued == 0))
                            tma_load_2d(xst + x.s * kBoxBytes, rest ? &tmL : &tmX, x0,
                                        r.r0 + tile * row_step, x.bar(xfull), kBoxBytes);
                        x.next();
                        ++issued;
                    }
                }
        }
        /* no copy may still be landing when the CTA exits: each stage's last */
        for (int n = min(issued, kXStages); n < kXStages; ++n) x.next();
        for (int n = 0; n < min(issued, kXStages); ++n, x.next())
            mm_drain(x.bar(xfull), x.round ^ 1);
    } else if (warp == 1) {
        /* ---------------- MMA issue */
        const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) |
                               ((uint32_t)(kTN >> 3) << 17) | ((uint32_t)(kTM >> 4) << 24);
        const bool leader = elect_one();
        const uint64_t xdesc = smem_desc(xst), wdesc = smem_desc(wst);
        if (!a.early) dependency_wait();   /* no wait below lasts as long as that launch */
        Ring<kXStages> x;
        Ring<kWSlots> wq;
        Ring<kAccs> ac;
        bool ok = true;
        /* one box of one tile; the stage goes back to the TMA */
        auto box = [&](uint32_t wslot, uint32_t acc, bool first) {
            ok = mm_wait(x.bar(xfull), x.round, s_state);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (leader) {
                const uint64_t xd = xdesc + x.s * (kBoxBytes >> 4);
                const uint64_t wd = wdesc + wslot * (kBoxBytes >> 4);
                const uint32_t d = tmem + acc * kTN;
#pragma unroll
                for (int kk = 0; kk < kBoxCols / 16; ++kk)
                    mma_f16(d, xd + 2 * kk, wd + 2 * kk, idesc, !first || kk > 0);
                mm_commit(x.bar(xempty));
            }
            x.next();
        };
        auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = mm_wait(bar, parity, s_state);
            ok = __all_sync(0xffffffffu, ok);
            return ok;
        };
        while (ok && next_run(a, sh, r)) {
            int b0, b1;
            used_boxes(s_cols, a.dir, r.fb * kTN, a.n_in, b0, b1);
            const int used = b1 - b0;
            if (used <= kWSlots) {
                /* the boxes stay for the whole run */
                for (int j = 0; j < r.ntiles && ok; ++j) {
                    if (!wait(ac.bar(aempty), ac.round ^ 1)) break;
                    Ring<kWSlots> q = wq;
                    for (int u = 0; u < used && ok; ++u, q.next()) {
                        if (j == 0 && !wait(q.bar(wfull), q.round)) break;
                        box(q.s, ac.s, u == 0);
                        if (TRANS && halves == 2 && ok) box(q.s, ac.s, false);
                        if (ok && j == r.ntiles - 1 && leader) mm_commit(q.bar(wempty));
                    }
                    if (ok && leader) mm_commit(ac.bar(afull));
                    ac.next();
                    if (j == r.ntiles - 1) wq = q;
                }
            } else {
                for (int j0 = 0; j0 < r.ntiles && ok; j0 += kGroup) {
                    const int n = min(kGroup, r.ntiles - j0);
                    Ring<kAccs> t = ac;
                    for (int j = 0; j < n && ok; ++j, t.next()) wait(t.bar(aempty), t.round ^ 1);
                    for (int u = 0; u < used && ok; ++u, wq.next()) {
                        if (!wait(wq.bar(wfull), wq.round)) break;
                        t = ac;
                        for (int j = 0; j < n && ok; ++j, t.next()) {
                            box(wq.s, t.s, u == 0);
                            if (TRANS && halves == 2 && ok) box(wq.s, t.s, false);
                            if (ok && u == used - 1 && leader) mm_commit(t.bar(afull));
                        }
                        if (ok && leader) mm_commit(wq.bar(wempty));
                    }
                    ac = t;
                }
            }
        }
        /* every MMA issued has completed before tensor memory is freed */
        if (leader) mm_commit(smem_u32(&bars.drain));
        mm_drain(smem_u32(&bars.drain), 0);
    } else if (warp == 2) {
        /* ---------------- the operator's boxes, as spmm_pack_kernel left them */
        if (!a.early) dependency_wait();
        Ring<kWSlots> q;
        int issued = 0;
        bool ok = true;
        const bool leader = elect_one();
        while (ok && !a.build && next_run(a, sh, r)) {
            int b0, b1;
            used_boxes(s_cols, a.dir, r.fb * kTN, a.n_in, b0, b1);
            const int used = b1 - b0;
            const int reps = used <= kWSlots ? 1 : (r.ntiles + kGroup - 1) / kGroup;
            const char* src = (const char*)a.pack +
                              ((long long)r.e * ((a.n_out + kTN - 1) / kTN) + r.fb) * NB * kBoxBytes;
            for (int rep = 0; rep < reps && ok; ++rep)
                for (int b = b0; b < b1; ++b) {
                    ok = mm_wait(q.bar(wempty), q.round ^ 1, s_state);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (leader)
                        bulk_load(wst + q.s * kBoxBytes, src + (long long)b * kBoxBytes, kBoxBytes,
                                  q.bar(wfull));
                    q.next();
                    ++issued;
                }
        }
        for (int n = min(issued, kWSlots); n < kWSlots; ++n) q.next();
        for (int n = 0; n < min(issued, kWSlots); ++n, q.next())
            mm_drain(q.bar(wfull), q.round ^ 1);
        if (a.early) dependency_wait();
    } else if (warp >= kEpiWarp0t) {
        /* ---------------- epilogue, in blocks of 32 rows x 32 features.  A
         * warp can read a quarter of the accumulator's rows, and the kEpiQuad
         * warps of a quarter take its blocks in turn (three: as many as leave
         * each 128 registers).  The
         * accumulators come a row a lane; memory is read and written eight
         * rows of 64 bytes at a time, by way of the warp's own shared memory
         * (a lane that wrote its own row's 32-byte sectors to memory kept the
         * L1 busy four times as long).  A block's residual is copied
         * there while the block before is worked on: two buffers a warp. */
        const int ew = warp - kEpiWarp0t;
        const int turn = ew >> 2;
        const uint32_t tq = (uint32_t)(warp & 3);
        const bool has_res = !TRANS && a.res, has_z = !TRANS && a.z;
        const bool al = ((uintptr_t)a.out % 16 == 0) && (a.ldo % 8 == 0);
        const bool alz = ((uintptr_t)a.z % 16 == 0) && (a.ldz % 8 == 0);
        const bool alr = ((uintptr_t)a.res % 16 == 0) && (a.ldr % 8 == 0);
        const uint32_t buf0 = smem_u32(smem) + (kWSlots + kXStages) * kBoxBytes + 2 * ew * kEpiBuf;
        /* a row's four 16-byte pieces are spread over the banks: this lane's
         * own row, and its piece of rows lane / 4, + 8, + 16, + 24 */
        const uint32_t own = lane * 64, spread = (lane >> 1) & 3;
        const int crow = lane >> 2;
        const uint32_t mine = crow * 64 + (((lane & 3) ^ ((crow >> 1) & 3)) << 4);
        const int cfeat = 8 * (lane & 3);
        uint32_t flip = 0;                        /* the buffer in use, 0 or kEpiBuf */

        /* the rows of a 32 x 32 block (a bit each) out of the buffer */
        auto copy_out = [&](T* p, long long ld, int i, int row0, uint32_t rows, bool vec) {
            __syncwarp();
            const uint32_t src = buf0 + flip + mine;
            const int nc = a.n_out - i;           /* of this lane's eight features */
            T* q = p + (row0 + crow) * ld + i;
#pragma unroll
            for (int it = 0; it < 4; ++it, q += 8 * ld) {
                uint32_t x[4];
                asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                             : "r"(src + it * 512));
                if (rows >> (crow + 8 * it) & 1) {
                    if (vec && nc >= 8)
                        *(uint4*)q = make_uint4(x[0], x[1], x[2], x[3]);
                    else
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            if (c < nc) ((uint16_t*)q)[c] = (uint16_t)(x[c >> 1] >> (16 * (c & 1)));
                }
            }
            __syncwarp();
        };
        /* a block's residual into a buffer */
        auto fetch = [&](int i, int row0, int left, uint32_t to) {
            const int nc = a.n_out - i;
            const T* q = (const T*)a.res + (row0 + crow) * a.ldr + i;
#pragma unroll
            for (int it = 0; it < 4; ++it, q += 8 * a.ldr) {
                if (crow + 8 * it < left) {
                    if (alr && nc >= 8)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                     ::"r"(buf0 + to + mine + it * 512), "l"(q) : "memory");
                    else
                        for (int c = 0; c < nc && c < 8; ++c)
                            sts16(buf0 + to + mine + it * 512 + 2 * c, ((const uint16_t*)q)[c]);
                }
            }
        };
        Ring<kAccs> ac;
        bool ok = true;
        /* the block whose residual is fetched next, one ahead of the work */
        Share psh = sh;
        Run pr;
        int pleft = 0, prow = 0, pi = 0, phi = 0;   /* tiles left of its run, row, feature, end */
        int pcb = turn;                             /* its place in the tile */
        auto next_fetch = [&](uint32_t to) {
            if (pcb >= 4) {
                pcb -= 4;
                --pleft;
                prow += row_step;
            }
            if (pleft == 0 && next_run(a, psh, pr)) {
                pleft = pr.ntiles;
                prow = pr.r0 + 32 * (int)tq;
                pi = pr.fb * kTN + cfeat;
                phi = pr.hi;
            }
            if (pleft > 0) fetch(pi + 32 * pcb, prow, phi - prow, to);
            pcb += kEpiQuad;
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        if (a.build && sh.w < sh.w1) {
            Share first = sh;
            next_run(a, first, r);
            int b0, b1;
            used_boxes(s_cols, a.dir, r.fb * kTN, a.n_in, b0, b1);
            build_operator<TRANS>(a, K, r.e, smem + (kWSlots + kXStages) * kBoxBytes, wst,
                                  r.fb * kTN, b0, b1, s_cols, tid - kEpiWarp0t * 32);
            if (tid < kEpiWarp0t * 32 + b1 - b0)
                mbar_arrive(wfull + 8 * (tid - kEpiWarp0t * 32));
        }
        if (!a.early) dependency_wait();
        if (has_res) next_fetch(0);
        int cb = turn;
        while (ok && next_run(a, sh, r)) {
            const int i0 = r.fb * kTN, hi = r.hi, e = r.e;
            /* a lane keeps the bias of four features, the others ask it */
            const bool has_bias = !TRANS && a.bias;
            uint32_t mybias[2] = {0, 0};
            if (has_bias) {
                const int n = a.n_out - i0 - 4 * lane;
                const uint16_t* p =
                    (const uint16_t*)a.bias + (long long)e * a.n_out + i0 + 4 * lane;
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    if (h < n) mybias[h >> 1] |= (uint32_t)__ldg(p + h) << (16 * (h & 1));
            }
            int row0 = r.r0 + 32 * (int)tq;
            for (int j = r.ntiles; j > 0 && ok; --j, row0 += row_step, ac.next()) {
                const int left = hi - row0;
                ok = mm_wait(ac.bar(afull), ac.round, s_state);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                for (; cb < 4; cb += kEpiQuad) {
                const int fw = 32 * cb;
                if (has_res) next_fetch(flip ^ kEpiBuf);
                float v[32];
                tmem_ld32(tmem + ((tq * 32) << 16) + (uint32_t)(ac.s * kTN + fw), v);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(ac.bar(aempty));
                float2 chk = both(0.0f);
#pragma unroll
                for (int c = 0; c < 32; c += 2)
                    chk = fma2(make_float2(v[c], v[c + 1]), both(0.0f), chk);
                /* rows of the expert; those with a sum that is not finite are
                 * stored by rows_again (a result may lie over its residual) */
                const uint32_t rows = left >= 32 ? ~0u : (1u << max(left, 0)) - 1;
                const uint32_t again = rows & __ballot_sync(0xffffffffu, chk.x + chk.y != 0.0f);
                if (has_res) {
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    __syncwarp();
                }
                const uint32_t row = buf0 + flip + own;
                uint32_t y[16];
#pragma unroll
                for (int c = 0; c < 4; ++c) {   /* eight features */
                    const uint32_t at = row + ((c ^ spread) << 4);
                    uint32_t res[4];
                    if (has_res)
                        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(res[0]), "=r"(res[1]), "=r"(res[2]), "=r"(res[3])
                                     : "r"(at));
                    float2 u[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) u[h] = make_float2(v[8 * c + 2 * h], v[8 * c + 2 * h + 1]);
                    if (!TRANS) {
                        if (has_bias)
#pragma unroll
                            for (int h = 0; h < 4; ++h)
                                u[h] = add2(u[h], unpack2<T>(__shfl_sync(
                                                      0xffffffffu, mybias[h & 1],
                                                      8 * cb + 2 * c + (h >> 1))));
                        /* the row's residual makes room for its z */
                        if (has_z)
                            sts128(at, pack2<T>(u[0].x, u[0].y), pack2<T>(u[1].x, u[1].y),
                                   pack2<T>(u[2].x, u[2].y), pack2<T>(u[3].x, u[3].y));
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            u[h] = act2<ACT>(u[h]);
                            if (has_res) u[h] = add2(u[h], unpack2<T>(res[h]));
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 4; ++h) y[4 * c + h] = pack2<T>(u[h].x, u[h].y);
                }
                if (has_z) copy_out((T*)a.z, a.ldz, i0 + cfeat + fw, row0, rows & ~again, alz);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    sts128(row + ((c ^ spread) << 4), y[4 * c], y[4 * c + 1], y[4 * c + 2],
                           y[4 * c + 3]);
                copy_out((T*)a.out, a.ldo, i0 + cfeat + fw, row0, rows & ~again, al);
                if (again)
                    rows_again<T, TRANS, ACT>(a, K, e, row0, i0 + fw + lane, again, s_state);
                if (has_res) flip ^= kEpiBuf;
                }
                cb -= 4;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
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
 * is a run of consecutive features.  dy, z and x are read once.  4096 rows of
 * 4096, 129 diagonals, bf16, GELU: 41 us for 168 MB with both halves of dz
 * written (4.1 TB/s; DRAM 45 % busy, tensor cores 27 %).  One CTA an SM does not overlap its start, the making of
 * dz and the diagonals' way out with its neighbour's stream.
 * Rows of the last stage that are not the part's are cleared in both operands
 * before the MMAs read them, so that an entry of D sums its own terms alone:
 * infinities and NaN reach the entries that they belong to and no others. */
constexpr int kGRows = 64;                     /* rows of a stage */
constexpr int kGBoxBytes = kGRows * 128;
constexpr int kGBoxes = 4;                     /* boxes of inputs of a CTA */
constexpr int kGDz = kGBoxes * kGBoxBytes;     /* in a stage: x, then dz (or dy), then its
                                                * rest (or z) */
constexpr int kGSmem = 192 * 1024 + 1024;
constexpr int kGWarps = 18;                    /* TMA, MMA, sixteen for the results */
constexpr int kGConv = (kGWarps - 2) * 32;     /* threads that look at every stage */
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

/* PAIR: dz comes as a rounded part and the rest of it (kDzPair), and the sum
 * over both is two MMAs.  ACT other than none: the pair is made here, from dy
 * and z, by the warps that wait for the results otherwise: into the stage, for
 * the MMAs, and to a.dz and a.lo, for the product that follows. */
template <typename T, int ACT, bool PAIR>
__global__ void __launch_bounds__(kGWarps * 32, 1)
spmm_grad_tc_kernel(const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmZ,
                    const __grid_constant__ CUtensorMap tmX, const __grid_constant__ GradArgs a,
                    int nfb, int nch)
{
    constexpr bool MAKE = ACT != DIA_ACT_NONE;
    static_assert(PAIR || !MAKE, "made in pairs");
    constexpr int ROWS = PAIR ? 4 : 2;             /* boxes of dz, or of dy and z */
    constexpr int STAGES = PAIR ? 3 : 4;
    constexpr int STAGE = (kGBoxes + ROWS) * kGBoxBytes;
    static_assert(STAGES * STAGE + 1024 <= kGSmem, "stages");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    __shared__ __align__(8) unsigned long long xfull[STAGES], xempty[STAGES], xready[STAGES], done;
    __shared__ uint32_t s_tmem;
    __shared__ int s_state[2];   /* mm_wait_long */
    __shared__ Box s_box[kGBoxes];
    __shared__ int2 s_offs[kOffs];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long b = blockIdx.x;
    const int fb = (int)(b % nfb), ch = (int)(b / nfb % nch);
    const RowGroup rg = row_group(a.seg, a.E, a.M, a.per, b / nfb / nch, true);
    if (rg.e < 0 || (rg.nparts > 1 && rg.slot + rg.part >= a.slots)) {
        dependency_wait();
        return;   /* whole CTA */
    }
    const int i0 = fb * 128;
    /* boxes in nch nearly equal shares */
    const int b0 = (int)((long long)a.dir.nboxes * ch / nch);
    const int nb = (int)((long long)a.dir.nboxes * (ch + 1) / nch) - b0;
    const bool bias = a.dbias && ch == 0;
    const bool conv = MAKE || bias;   /* the result warps look at every stage */
    const int nst = i0 < a.n_rows ? (rg.r1 - rg.r0 + kGRows - 1) / kGRows : 0;

    for (int k = tid; k < min(a.K, kOffs); k += kGWarps * 32) s_offs[k] = a.dir.offs[k];
    if (tid < nb) s_box[tid] = a.dir.boxes[b0 + tid];
    if (tid == 0) {
        s_state[0] = s_state[1] = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(xfull[s], 1);
            mbar_init(xempty[s], 1);
            mbar_init(xready[s], kGConv / 32);
        }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&s_tmem)), "r"(256));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    bool ok = true;
    /* dz may be the launch before this one's */
    dependency_wait();
    dependents_begin();

    const uint32_t st0 = smem_u32(smem), full0 = smem_u32(xfull), empty0 = smem_u32(xempty);
    const uint32_t ready0 = smem_u32(xready);
    float sums[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (warp == 0) {
        const bool leader = elect_one();
        Ring<STAGES> x;
        int g = 0;
        for (; g < nst; ++g, x.next()) {
            ok = mm_wait(x.bar(empty0), x.round ^ 1, s_state);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (leader && !(g_mm_withhold && blockIdx.x == 0 && g == 0)) {
                const int r = rg.r0 + g * kGRows;
                const uint32_t st = st0 + x.s * STAGE, bar = x.bar(full0);
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                             ::"r"(bar), "r"((ROWS + nb) * kGBoxBytes) : "memory");
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tma_box(st + kGDz + h * kGBoxBytes, &tmD, i0 + 64 * h, r, bar);
                    if (PAIR)
                        tma_box(st + kGDz + (2 + h) * kGBoxBytes, &tmZ, i0 + 64 * h, r, bar);
                }
                for (int c = 0; c < nb; ++c)
                    tma_box(st + c * kGBoxBytes, &tmX, i0 + s_box[c].col, r, bar);
            }
        }
        for (int n = min(g, STAGES); n < STAGES; ++n) x.next();
        for (int n = 0; n < min(g, STAGES); ++n, x.next())
            mm_drain(x.bar(full0), x.round ^ 1);
    } else if (warp == 1) {
        const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (1u << 16) |
                               ((uint32_t)(128 >> 4) << 24) |
                               ((uint32_t)(nb * kBoxCols >> 3) << 17);
        const bool leader = elect_one();
        const uint64_t desc0 = mn_desc(st0);
        Ring<STAGES> x;
        for (int g = 0; g < nst; ++g, x.next()) {
            const int left = rg.r1 - rg.r0 - g * kGRows;
            ok = mm_wait(x.bar(full0), x.round, s_state) &&
                 (!conv || mm_wait(x.bar(ready0), x.round, s_state));
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (left < kGRows) {
                /* rows past the part: another expert's, or nobody's */
                const uint32_t st = st0 + x.s * STAGE;
                const int per = (kGRows - left) * 8;
                for (int o = lane; o < per * (kGBoxes + ROWS); o += 32)
                    sts128(st + o / per * kGBoxBytes + left * 128 + o % per * 16, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (leader) {
                const uint64_t bd = desc0 + x.s * (STAGE >> 4);
                const uint64_t ad = bd + (kGDz >> 4);
                if (nb > 0) {
#pragma unroll
                    for (int kk = 0; kk < kGRows / 16; ++kk) {
                        mma_f16(tmem, ad + 128 * kk, bd + 128 * kk, idesc, g > 0 || kk > 0);
                        if (PAIR)
                            mma_f16(tmem, ad + (2 * kGBoxBytes >> 4) + 128 * kk, bd + 128 * kk,
                                    idesc, true);
                    }
                }
                mm_commit(x.bar(empty0));
            }
        }
        if (leader) mm_commit(smem_u32(&done));
        mm_drain(smem_u32(&done), 0);
    } else if (conv) {
        /* a thread looks at eight features of two rows of every stage.  Every
         * warp takes part in every stage, so that it has seen every phase of a
         * barrier before the next can end.  (Halves of the warps in turn did not:
         * with three stages a half came back to one whose round before it had
         * not waited for, and the parity of the round before that let it pass:
         * stale rows, or a wait that ran out.) */
        const int c = tid & 15, r0 = (tid - 64) >> 4, i = i0 + 8 * c;
        Ring<STAGES> x;
        for (int g = 0; g < nst; ++g, x.next()) {
            ok = mm_wait(x.bar(full0), x.round, s_state);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int left = rg.r1 - rg.r0 - g * kGRows;
            const uint32_t at = st0 + x.s * STAGE + kGDz + (c >> 3) * kGBoxBytes + r0 * 128 +
                                (((c ^ r0) & 7) << 4);
            uint32_t d[2][4], z[2][4];   /* z, then the rest of dz */
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                lds128(at + h * 32 * 128, d[h]);
                if (PAIR) lds128(at + h * 32 * 128 + 2 * kGBoxBytes, z[h]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float2 v = unpack2<T>(d[h][q]);
                    if (MAKE) {
                        v = mul2(v, dact2<ACT>(unpack2<T>(z[h][q])));
                        d[h][q] = pack2_finite<T>(v.x, v.y);
                        const float2 w = fma2(unpack2<T>(d[h][q]), both(-1.0f), v);
                        z[h][q] = pack2<T>(w.x, w.y);
                    } else if (PAIR) {
                        v = add2(v, unpack2<T>(z[h][q]));
                    }
                    if (bias && r0 + 32 * h < left) {
                        sums[2 * q] += v.x;
                        sums[2 * q + 1] += v.y;
                    }
                }
                if (MAKE) {
                    const uint32_t to = at + h * 32 * 128;
                    sts128(to, d[h][0], d[h][1], d[h][2], d[h][3]);
                    sts128(to + 2 * kGBoxBytes, z[h][0], z[h][1], z[h][2], z[h][3]);
                }
            }
            if (MAKE) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(x.bar(ready0));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = r0 + 32 * h;
                if (!MAKE || r >= left || i >= a.n_rows) continue;
                const long long to = (long long)(rg.r0 + g * kGRows + r) * a.lddz + i;
                *(uint4*)((T*)a.dz + to) = make_uint4(d[h][0], d[h][1], d[h][2], d[h][3]);
                *(uint4*)((T*)a.lo + to) = make_uint4(z[h][0], z[h][1], z[h][2], z[h][3]);
            }
        }
    }
    /* the results: every MMA has completed (the stages are free) */
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    ok = !__syncthreads_or(!ok);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    float* tile = (float*)smem;
    float* colsum = tile + 128 * kGPitch;   /* [32 rows][128] */
    if (ok && warp >= 2 && nst > 0) {
        const uint32_t tq = (uint32_t)(warp & 3);
        const int grp = (warp - 2) >> 2, f = 32 * (int)tq + lane;
        for (int c0 = grp * 16; c0 < nb * kBoxCols; c0 += 64) {
            float v[16];
            tmem_ld16(tmem + ((tq * 32) << 16) + (uint32_t)c0, v);
#pragma unroll
            for (int c = 0; c < 16; ++c) tile[f * kGPitch + c0 + c] = v[c];
        }
    }
    if (bias && warp >= 2)
#pragma unroll
        for (int q = 0; q < 8; ++q) colsum[((tid - 64) >> 4) * 128 + (tid & 15) * 8 + q] = sums[q];
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256));
    if (!ok) return;
    if (bias && tid < 128 && i0 + tid < a.n_rows) {
        float v = 0.0f;
        for (int r = 0; r < 32; ++r) v += colsum[r * 128 + tid];
        if (rg.nparts > 1)
            a.part[((long long)(rg.slot + rg.part) * (a.K + 1) + a.K) * a.stride + i0 + tid] = v;
        else
            ((T*)a.dbias)[(long long)rg.e * a.n_rows + i0 + tid] = from_f<T>(v);
    }
    if (!a.dvals) return;
    /* a diagonal's 128 entries: consecutive features, consecutive columns of
     * one box or more; what lies in other CTAs' boxes is theirs */
    const int k_lo = nb > 0 ? s_box[0].k0 : 0, k_hi = nb > 0 ? s_box[nb - 1].k1 : 0;
    int col[kGBoxes];
#pragma unroll
    for (int c = 0; c < kGBoxes; ++c) col[c] = c < nb ? s_box[c].col : INT_MAX / 2;
    const bool adjoin = nb > 0 && s_box[nb - 1].col == col[0] + kBoxCols * (nb - 1);
    const bool parts = rg.nparts > 1;
    const int f_end = (int)min(128ll, a.stride - i0);
    float* part0 = a.part + (long long)(rg.slot + rg.part) * (a.K + 1) * a.stride + i0 + lane;
    T* out0 = (T*)a.dvals + rg.e * a.estride + i0 + lane;
    const float* row = tile + lane * kGPitch;
    const int k_first = k_lo + warp;
    /* the usual tile: every entry of every diagonal in the matrix and here */
    if (nch == 1 && adjoin && nst > 0 && a.K <= kOffs && i0 + 128 <= a.n_rows &&
        i0 + s_offs[0].x >= 0 && i0 + 127 + s_offs[a.K - 1].x < a.n_cols) {
        const float* src = row - col[0] + lane;
#pragma unroll 2
        for (int k = k_first; k < k_hi; k += kGWarps) {
            const int2 o = s_offs[k];
            const long long at = (long long)o.y * a.stride;
            float v[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) v[s] = src[32 * s * (kGPitch + 1) + o.x];
            if (parts) {
#pragma unroll
                for (int s = 0; s < 4; ++s) part0[at + 32 * s] = v[s];
            } else {
#pragma unroll
                for (int s = 0; s < 4; ++s) out0[at + 32 * s] = from_f<T>(v[s]);
            }
        }
        return;
    }
    for (int k = k_first; k < k_hi; k += kGWarps) {
        const int2 o = a.K <= kOffs ? s_offs[k] : a.dir.offs[k];
        /* features whose entry lies in the matrix; outside, and in the
         * padding, there is no gradient */
        const int in_lo = max(0, -(i0 + o.x));
        const int in_hi = nst > 0 ? min(a.n_rows - i0, a.n_cols - i0 - o.x) : 0;
        float v[4];
        bool on[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int f = 32 * s + lane, p = o.x + f;
            int at = p - col[0];
            if (adjoin) {   /* the boxes are one wide one */
                if (at >= kBoxCols * nb) at = -1;
            } else {
                at = -1;
#pragma unroll
                for (int c = 0; c < kGBoxes; ++c)
                    if ((unsigned)(p - col[c]) < (unsigned)kBoxCols) at = c * kBoxCols + p - col[c];
            }
            on[s] = at >= 0 && f < f_end;
            v[s] = on[s] && f >= in_lo && f < in_hi ? row[32 * s * kGPitch + at] : 0.0f;
        }
        const long long at = (long long)o.y * a.stride;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (!on[s]) continue;
            if (parts)
                part0[at + 32 * s] = v[s];
            else
                out0[at + 32 * s] = from_f<T>(v[s]);
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

/* CTAs a feature tile, each with every so-manieth tile of rows; 0: stretches
 * of the list of tiles instead, where that would leave a quarter of the SMs
 * idle (4096 x 4096 band, 2048 rows: 28.1 us against 30.6 by stretches) */
static int row_groups_of(int n_out, long long M, int E, bool seg)
{
    const int nfb = (n_out + kTN - 1) / kTN;
    const long long tiles = seg ? M / kTM + std::min<long long>(E, M) : (M + kTM - 1) / kTM;
    const long long groups = std::min<long long>(num_sms() / nfb, tiles);
    return groups * nfb < std::min<long long>(tiles * nfb, num_sms() * 3 / 4) ? 0 : (int)groups;
}

/* the product makes the operator's boxes itself */
static bool builds(const SpmmDir& d, int K, int n_out, long long M, int E)
{
    return E == 1 && K <= kInlineDiags && d.nboxes <= kWSlots &&
           row_groups_of(n_out, M, 1, false) > 0 && row_groups_of(n_out, M, 1, true) > 0;
}

long long spmm_tc_pack_bytes(const SpmmDir& d, int K, int n_out, long long M, int E)
{
    if (builds(d, K, n_out, M, E)) return 0;
    return (long long)E * ((n_out + kTN - 1) / kTN) * d.nboxes * kBoxBytes;
}

template <typename T, bool TRANS, int ACT>
static int launch_tc(const CUtensorMap (&map)[2], const ProdArgs& a_, int K, cudaStream_t stream)
{
    const long long tiles = a_.seg ? a_.M / kTM + std::min(a_.E, a_.M) : (a_.M + kTM - 1) / kTM;
    const int nfb = (a_.n_out + kTN - 1) / kTN;
    ProdArgs a = a_;
    a.groups = row_groups_of(a.n_out, a.M, a.E, a.seg != nullptr);
    a.build = builds(a.dir, K, a.n_out, a.M, a.E);
    const int grid = a.groups > 0 ? a.groups * nfb
                                  : (int)std::min<long long>(tiles * nfb, num_sms());
    static SmemRecord most;
    DIA_TRY_CUDA(allow_smem(spmm_tc_kernel<T, TRANS, ACT>, kTcSmem, most));
    DIA_TRY_CUDA(launch(a.dependent, spmm_tc_kernel<T, TRANS, ACT>, grid, kTcWarps * 32, kTcSmem, stream,
                        map[0], map[1], a, K));
    return DIA_OK;
}

template <typename T>
static int launch_tc_type(const CUtensorMap (&map)[2], const ProdArgs& a, int K,
                          cudaStream_t stream)
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

int spmm_tc_pack(const ProdArgs& a, bool dependent, cudaStream_t stream)
{
    const long long boxes = spmm_tc_pack_bytes(a.dir, a.K, a.n_out, a.M, a.E) / kBoxBytes;
    if (boxes == 0) return DIA_OK;
    if (boxes > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm: operator too large");
    const auto pack = a.trans ? spmm_pack_kernel<true> : spmm_pack_kernel<false>;
    static SmemRecord most[2];
    DIA_TRY_CUDA(allow_smem(pack, kPackSmem, most[a.trans]));
    DIA_TRY_CUDA(launch(dependent, pack, (int)boxes, 256, kPackSmem, stream, a));
    return DIA_OK;
}

int spmm_tc_product(const ProdArgs& a, int dtype, cudaStream_t stream)
{
    CUtensorMap map[2];
    if (!block_map(&map[0], a.in, dtype, a.n_in, a.M, a.ldi, kTM) ||
        !block_map(&map[1], a.lo ? a.lo : a.in, dtype, a.n_in, a.M, a.ldi, kTM))
        return fail(DIA_ERR_CUDA, "dia_spmm: cuTensorMapEncodeTiled failed");
    return dtype == DIA_F16 ? launch_tc_type<__half>(map, a, a.K, stream)
                            : launch_tc_type<__nv_bfloat16>(map, a, a.K, stream);
}

bool spmm_tc_makes_dz(const GradArgs& a)
{
    /* an operator of several shares of boxes would make dz as many times */
    return a.act != DIA_ACT_NONE && a.dir.nboxes <= kGBoxes && spmm_tc_block(a.dy, a.lddy) &&
           spmm_tc_block(a.z, a.ldz);
}

template <typename T, int ACT, bool PAIR>
static int launch_grad_tc(const GradArgs& a, int dtype, bool dependent, cudaStream_t stream)
{
    CUtensorMap md, mz, mx;
    const bool make = ACT != DIA_ACT_NONE;
    const void* second = make ? a.z : (PAIR ? a.lo : a.dz);
    if (!block_map(&md, make ? a.dy : a.dz, dtype, a.n_rows, a.M, make ? a.lddy : a.lddz, kGRows) ||
        !block_map(&mx, a.x, dtype, a.n_cols, a.M, a.ldx, kGRows) ||
        !block_map(&mz, second, dtype, a.n_rows, a.M, make ? a.ldz : a.lddz, kGRows))
        return fail(DIA_ERR_CUDA, "dia_spmm_backward: cuTensorMapEncodeTiled failed");
    const int nfb = (int)((a.stride + 127) / 128);
    const int nch = std::max(1, (a.dir.nboxes + kGBoxes - 1) / kGBoxes);
    const long long parts = a.seg ? a.M / a.per + a.E : std::max(1, (a.M + a.per - 1) / a.per);
    const long long grid = parts * nfb * nch;
    if (grid > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm_backward: block too large");
    const auto kernel = spmm_grad_tc_kernel<T, ACT, PAIR>;
    static SmemRecord most;
    DIA_TRY_CUDA(allow_smem(kernel, kGSmem, most));
    DIA_TRY_CUDA(launch(dependent, kernel, (int)grid, kGWarps * 32, kGSmem, stream, md, mz, mx, a,
                        nfb, nch));
    return DIA_OK;
}

template <typename T>
static int launch_grad_act(const GradArgs& a, int dtype, bool make, bool dependent,
                           cudaStream_t stream)
{
    switch (make ? a.act : DIA_ACT_NONE) {
        case DIA_ACT_RELU: return launch_grad_tc<T, DIA_ACT_RELU, true>(a, dtype, dependent, stream);
        case DIA_ACT_SILU: return launch_grad_tc<T, DIA_ACT_SILU, true>(a, dtype, dependent, stream);
        case DIA_ACT_GELU: return launch_grad_tc<T, DIA_ACT_GELU, true>(a, dtype, dependent, stream);
        case DIA_ACT_GELU_TANH:
            return launch_grad_tc<T, DIA_ACT_GELU_TANH, true>(a, dtype, dependent, stream);
        default:
            return a.lo ? launch_grad_tc<T, DIA_ACT_NONE, true>(a, dtype, dependent, stream)
                        : launch_grad_tc<T, DIA_ACT_NONE, false>(a, dtype, dependent, stream);
    }
}

int spmm_tc_gradient(const GradArgs& a, int dtype, bool make, bool dependent, cudaStream_t stream)
{
    return dtype == DIA_F16 ? launch_grad_act<__half>(a, dtype, make, dependent, stream)
                            : launch_grad_act<__nv_bfloat16>(a, dtype, make, dependent, stream);
}

cudaError_t spmm_tc_test_wait(unsigned long long wait_ns, int withhold)
{
    if (wait_ns == 0) wait_ns = kMmWaitNs;
    const cudaError_t e = cudaMemcpyToSymbol(g_mm_wait_ns, &wait_ns, sizeof(wait_ns));
    return e != cudaSuccess ? e : cudaMemcpyToSymbol(g_mm_withhold, &withhold, sizeof(withhold));
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
