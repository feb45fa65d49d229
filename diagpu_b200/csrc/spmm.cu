/*
 * spmm.cu -- a DIA operator times a block of vectors, with an epilogue, its
 * gradients, and the same product grouped by expert.
 *
 *     z[t, i]    = bias[i] + sum_k vals[k, i] * x[t, i + d_k]
 *     y[t, i]    = act(z[t, i]) + residual[t, i]
 *     dz         = dy * act'(z)
 *     dx[t, j]   = sum_k vals[k, j - d_k] * dz[t, j - d_k]
 *     dvals[k,i] = sum_t dz[t, i] * x[t, i + d_k]
 *     dbias[i]   = sum_t dz[t, i]
 *
 * The block holds one vector per row, so neighbouring lanes read neighbouring
 * features and every diagonal value is read once for several vectors instead
 * of once per vector, which is what a loop of SpMVs would do.  All sums are
 * held in fp32, in ascending order of the offsets, and rounded once to the
 * block's type.  Grouped: the rows are sorted by expert, rows [seg[e],
 * seg[e+1]) use the diagonals vals[e].
 */
#include <algorithm>
#include <atomic>
#include <climits>
#include <cstring>
#include <new>
#include <numeric>
#include <vector>

#include "dia_core.cuh"
#include "spmm.cuh"

namespace dia {

/* ------------------------------------------------- few rows, or any at all
 *
 * A lane is a feature; a diagonal value is read once for TT rows, an input
 * straight from memory.  With few rows a call is as long as its chain of
 * memory latencies, so the CTA's warps split the diagonals `ks` ways (four at
 * a time in flight each) and add up in shared memory in a fixed order, and
 * what the epilogue reads is fetched first.  The other 16 / ks warps take
 * other features. */
constexpr int kFewWarps = 16;
constexpr int kFewOffs = 512;   /* offsets staged at once */

template <typename T, bool TRANS, int TT>
__global__ void __launch_bounds__(kFewWarps * 32)
spmm_few_kernel(const __grid_constant__ ProdArgs a, int ks, int ftiles, long long ngroups,
                bool rows_first)
{
    __shared__ int2 s_off[kFewOffs];
    __shared__ float s_sum[kFewWarps][TT][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int part = warp % ks, sub = warp / ks, fper = kFewWarps / ks;
    const int fblocks = (ftiles + fper - 1) / fper;
    const long long b = blockIdx.x;
    const long long g = rows_first ? b % ngroups : b / fblocks;
    const int fb = (int)(rows_first ? b / ngroups : b % fblocks);
    for (int k = tid; k < min(a.K, kFewOffs); k += kFewWarps * 32) s_off[k] = a.dir.offs[k];
    const RowGroup rg = row_group(a.seg, a.E, a.M, TT, g, false);
    if (rg.e < 0) return;   /* whole CTA */
    const int i = (fb * fper + sub) * 32 + lane;
    const bool on = i < a.n_out;
    const int nt = rg.r1 - rg.r0;
    const T* vals = (const T*)a.vals + rg.e * a.estride;
    const T* in = (const T*)a.in + rg.r0 * a.ldi;
    float bias = 0.0f, res[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) res[t] = 0.0f;
    if (!TRANS && part == 0 && on) {
        if (a.bias) bias = to_f(((const T*)a.bias)[(long long)rg.e * a.n_out + i]);
        if (a.res)
#pragma unroll
            for (int t = 0; t < TT; ++t)
                if (t < nt) res[t] = to_f(((const T*)a.res)[(rg.r0 + t) * a.ldr + i]);
    }
    float acc[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = 0.0f;
    for (int base = 0; base < a.K; base += kFewOffs) {
        const int n = min(a.K - base, kFewOffs);
        if (base > 0) {
            __syncthreads();
            for (int k = tid; k < n; k += kFewWarps * 32) s_off[k] = a.dir.offs[base + k];
        }
        __syncthreads();
        const int k0 = n * part / ks, k1 = n * (part + 1) / ks;
        constexpr int U = TT == 1 ? 8 : 4;
        for (int k = k0; k < k1; k += U) {
            float w[U], x[U][TT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int2 o = s_off[min(k + u, k1 - 1)];
                const int j = i + o.x;
                const bool ok = k + u < k1 && on && (unsigned)j < (unsigned)a.n_in;
                w[u] = ok ? to_f(vals[o.y * a.stride + (TRANS ? j : i)]) : 0.0f;
#pragma unroll
                for (int t = 0; t < TT; ++t)
                    x[u][t] = ok && t < nt ? to_f(in[t * a.ldi + j]) : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < TT; ++t) acc[t] = fmaf(w[u], x[u][t], acc[t]);
        }
    }
    if (ks > 1) {
#pragma unroll
        for (int t = 0; t < TT; ++t) s_sum[warp][t][lane] = acc[t];
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int t = 0; t < TT; ++t)
            for (int p = 1; p < ks; ++p) acc[t] += s_sum[warp + p][t][lane];
    }
    if (!on) return;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        if (t >= nt) break;
        const long long row = rg.r0 + t;
        const float z = acc[t] + bias;
        if (!TRANS && a.z) ((T*)a.z)[row * a.ldz + i] = from_f<T>(z);
        ((T*)a.out)[row * a.ldo + i] = from_f<T>(TRANS ? z : act_any(a.act, z) + res[t]);
    }
}

/* ----------------------------------------------------------- many rows
 *
 * A CTA takes a tile of features and copies the inputs it reads to
 * shared memory; a warp takes 128 features of eight rows.  QUADS: a lane owns
 * four consecutive features, and the up to four diagonals of a quad read
 * seven consecutive inputs as two 16-byte pieces, of which the second is the
 * next quad's first: for runs of consecutive offsets shared memory gives a
 * piece per sixteen products.  Otherwise (fewer than three diagonals a quad)
 * a lane owns features 32 apart and reads an input per product, without bank
 * conflicts at any offset.  Shared memory's bandwidth bounds both. */
constexpr int kTileWarps = 8;
constexpr int kTileRows = 8;    /* rows of a warp */
constexpr int kTileSmem = 112 * 1024;   /* two CTAs an SM */

/* `rows` rows of the spans' inputs to shared memory, zero outside the block
 * and for rows from nt on; pitch in elements; a warp takes a row */
template <typename T, bool VEC>
__device__ __forceinline__ void stage_spans(T* dst, int pitch, const InputSpan* spans, int s0,
                                            int s1, const T* in, long long ld, int i0, int n_in,
                                            int rows, int nt)
{
    constexpr int V = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
    for (int s = s0; s < s1; ++s) {
        const int4 sp = __ldg((const int4*)(spans + s));   /* from, len, at */
        const int j0 = i0 + sp.x;
        for (int t = threadIdx.x >> 5; t < rows; t += kTileWarps) {
            T* d = dst + t * pitch + sp.z;
            const T* p = in + t * ld + j0;
            const int n = t < nt ? n_in : INT_MIN;     /* no input of the row is read */
#pragma unroll 4
            for (int c = lane * V; c < sp.y; c += 32 * V) {
                if (VEC && j0 + c >= 0 && j0 + c + V <= n) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                 ::"r"((uint32_t)__cvta_generic_to_shared(d + c)), "l"(p + c)
                                 : "memory");
                } else {
                    T v[V];
#pragma unroll
                    for (int u = 0; u < V; ++u)
                        v[u] = j0 + c + u >= 0 && j0 + c + u < n ? p[c + u] : from_f<T>(0.0f);
#pragma unroll
                    for (int u = 0; u < V; ++u) d[c + u] = v[u];
                }
            }
        }
    }
}

template <typename T, bool TRANS, bool VEC, bool QUADS>
__global__ void __launch_bounds__(kTileWarps * 32)
spmm_tile_kernel(const __grid_constant__ ProdArgs a, int shape, int ftiles, long long ngroups,
                 bool rows_first)
{
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T* xs = (T*)smem_raw;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int F = kTileF[0] << shape, wf = F / 128;   /* warps side by side */
    const int rows = kTileWarps / wf * kTileRows;
    const long long b = blockIdx.x;
    const long long g = rows_first ? b % ngroups : b / ftiles;
    const int i0 = (int)(rows_first ? b / ngroups : b % ftiles) * F;
    const RowGroup rg = row_group(a.seg, a.E, a.M, rows, g, false);
    if (rg.e < 0) return;   /* whole CTA */
    const int nt = rg.r1 - rg.r0, pitch = a.dir.width[shape];
    stage_spans<T, VEC>(xs, pitch, a.dir.spans[shape], 0, a.dir.nspans[shape],
                        (const T*)a.in + rg.r0 * a.ldi, a.ldi, i0, a.n_in, rows, nt);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    const int t0 = warp / wf * kTileRows, f0 = warp % wf * 128;
    if (t0 >= nt || i0 + f0 >= a.n_out) return;
    const int live = min(nt - t0, kTileRows);
    const T* vals = (const T*)a.vals + rg.e * a.estride;
    const T* xw = xs + t0 * pitch;
    float acc[kTileRows][4];
#pragma unroll
    for (int t = 0; t < kTileRows; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][r] = 0.0f;

    constexpr int STEP = QUADS ? 1 : 32;             /* between a lane's features */
    const int f = f0 + (QUADS ? 4 * lane : lane), i = i0 + f;
    if (QUADS) {
        const Quad* quads = a.dir.quads[shape];
        float carry[kTileRows][4];
        int next = INT_MIN;   /* base of the quad whose first piece `carry` holds */
        for (int q = 0; q < a.dir.nquads; ++q) {
            const int4 h = __ldg((const int4*)&quads[q]);
            const int2 h2 = __ldg((const int2*)&quads[q].k[3]);
            const int kk[4] = {h.y, h.z, h.w, h2.x};
            const int c = i + h.x;
            float w[4][4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (kk[s] < 0) continue;
                const T* vp = vals + (long long)kk[s] * a.stride;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = c + s + r;
                    w[s][r] = i + r < a.n_out && (unsigned)j < (unsigned)a.n_in
                                  ? to_f(vp[TRANS ? j : i + r]) : 0.0f;
                }
            }
            const T* p = xw + h2.y + f;
            if (h.x != next) {
#pragma unroll
                for (int t = 0; t < kTileRows; ++t) *(float4*)carry[t] = load4<T>(p + t * pitch);
            }
            next = h.x + 4;
#pragma unroll
            for (int t = 0; t < kTileRows; ++t) {
                float x[8];
                *(float4*)x = *(float4*)carry[t];
                *(float4*)(x + 4) = load4<T>(p + t * pitch + 4);
                *(float4*)carry[t] = *(float4*)(x + 4);
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    if (kk[s] >= 0)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            acc[t][r] = fmaf(w[s][r], x[s + r], acc[t][r]);
            }
        }
    } else {
        const int* cols = a.dir.cols[shape];
        /* the next diagonal's values are on their way while one is worked on */
        auto fetch = [&](int k, float (&w)[4], int& col) {
            const int2 o = __ldg(&a.dir.offs[k]);
            col = __ldg(cols + k);
            const T* vp = vals + (long long)o.y * a.stride;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int ir = i + 32 * r, j = ir + o.x;
                w[r] = ir < a.n_out && (unsigned)j < (unsigned)a.n_in
                           ? to_f(__ldg(vp + (TRANS ? j : ir))) : 0.0f;
            }
        };
        float w[4], wn[4];
        int col = 0, cn = 0;
        if (a.K > 0) fetch(0, w, col);
#pragma unroll 2
        for (int k = 0; k < a.K; ++k) {
            if (k + 1 < a.K) fetch(k + 1, wn, cn);
            const T* p = xw + col + f;
#pragma unroll
            for (int t = 0; t < kTileRows; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    acc[t][r] = fmaf(w[r], to_f(p[t * pitch + 32 * r]), acc[t][r]);
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = wn[r];
            col = cn;
        }
    }
    float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!TRANS && a.bias)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (i + STEP * r < a.n_out)
                bias[r] = to_f(((const T*)a.bias)[(long long)rg.e * a.n_out + i + STEP * r]);
#pragma unroll
    for (int t = 0; t < kTileRows; ++t) {
        if (t >= live) break;
        const long long row = (long long)rg.r0 + t0 + t;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int ir = i + STEP * r;
            if (ir >= a.n_out) continue;
            const float z = acc[t][r] + bias[r];
            float y = z;
            if (!TRANS) {
                if (a.z) ((T*)a.z)[row * a.ldz + ir] = from_f<T>(z);
                y = act_any(a.act, z);
                if (a.res) y += to_f(((const T*)a.res)[row * a.ldr + ir]);
            }
            ((T*)a.out)[row * a.ldo + ir] = from_f<T>(y);
        }
    }
}

/* ------------------------------------------------- gradient of the diagonals
 *
 * A CTA takes 128 features, one window of diagonals (at most 64) and one part
 * of an expert's rows, `rows` of them at a time by way of shared memory, the
 * next ones on their way meanwhile; a warp keeps the sums of its eight
 * diagonals at its lanes' four features.  Sums of an expert with one part go
 * out at once, others to `part`. */
constexpr int kGradDiags = 8;             /* diagonals of a warp */
constexpr int kGradSmem = 160 * 1024;     /* two buffers of at least eight rows */

template <typename T, bool VEC, int ND>
__global__ void __launch_bounds__(kTileWarps * 32)
spmm_grad_kernel(const __grid_constant__ GradArgs a, int ftiles, int nwins, int rows)
{
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long b = blockIdx.x;
    const int f0 = (int)(b % ftiles) * 128, wi = (int)(b / ftiles % nwins);
    const RowGroup rg = row_group(a.seg, a.E, a.M, a.per, b / ftiles / nwins, true);
    if (rg.e < 0 || (rg.nparts > 1 && rg.slot + rg.part >= a.slots)) return;
    const bool diags = a.dvals && a.dir.nwins > 0;
    GradWindow win{};
    if (diags) win = a.dir.wins[wi];
    const int pitch = diags ? a.dir.wwidth : 0;
    const int buf = rows * (pitch + 128);            /* x, then dz [row][128] */
    const int per = (win.k1 - win.k0 + kTileWarps - 1) / kTileWarps;
    const int k0 = win.k0 + warp * per, nk = max(0, min(per, win.k1 - k0));
    /* a warp with fewer than ND repeats its last (or column 0) and drops it */
    int col[ND];
#pragma unroll
    for (int u = 0; u < ND; ++u)
        col[u] = (nk > 0 ? a.dir.wcols[k0 + min(u, nk - 1)] : 0) + lane;
    const bool bias = a.dbias && wi == 0 && warp == 0;
    float acc[ND][4], sb[4] = {0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < ND; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[u][r] = 0.0f;
    if (f0 < a.n_rows) {
        auto fetch = [&](int t0, int which) {
            const int nt = min(rg.r1 - t0, rows);
            T* xs = (T*)smem_raw + which * buf;
            if (nt > 0) {
                if (diags)
                    stage_spans<T, VEC>(xs, pitch, a.dir.wspans, win.s0, win.s1,
                                        (const T*)a.x + t0 * a.ldx, a.ldx, f0, a.n_cols, nt, nt);
                stage_spans<T, VEC>(xs + rows * pitch, 128, a.dir.tile_span, 0, 1,
                                    (const T*)a.dz + t0 * a.lddz, a.lddz, f0, a.n_rows, nt, nt);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int which = 0;
        fetch(rg.r0, 0);
        for (int t0 = rg.r0; t0 < rg.r1; t0 += rows, which ^= 1) {
            const int nt = min(rg.r1 - t0, rows);
            fetch(t0 + rows, which ^ 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();
            const T* xs = (const T*)smem_raw + which * buf;
            const T* ds = xs + rows * pitch;
            if (nk > 0 || bias) {
#pragma unroll 4
                for (int t = 0; t < nt; ++t) {
                    float d[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) d[r] = to_f(ds[t * 128 + lane + 32 * r]);
#pragma unroll
                    for (int u = 0; u < ND; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            acc[u][r] = fmaf(d[r], to_f(xs[t * pitch + col[u] + 32 * r]), acc[u][r]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) sb[r] += d[r];
                }
            }
            __syncthreads();   /* the buffer is filled again */
        }
    }
    const bool parts = rg.nparts > 1;
    float* part = a.part + (long long)(rg.slot + rg.part) * (a.K + 1) * a.stride;
#pragma unroll
    for (int u = 0; u < ND; ++u) {
        if (u >= nk) break;
        const int2 o = a.dir.offs[k0 + u];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = f0 + lane + 32 * r;
            if (i >= a.stride) continue;
            /* an entry outside the matrix, or in the padding, has no gradient */
            const bool in = i < a.n_rows && (unsigned)(i + o.x) < (unsigned)a.n_cols;
            const float v = in ? acc[u][r] : 0.0f;
            if (parts)
                part[o.y * a.stride + i] = v;
            else
                ((T*)a.dvals)[rg.e * a.estride + o.y * a.stride + i] = from_f<T>(v);
        }
    }
    if (bias)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = f0 + lane + 32 * r;
            if (i >= a.n_rows) continue;
            if (parts)
                part[a.K * a.stride + i] = sb[r];
            else
                ((T*)a.dbias)[(long long)rg.e * a.n_rows + i] = from_f<T>(sb[r]);
        }
}

/* Sums the parts of experts that have several, in the parts' order; four
 * columns a thread. */
template <typename T>
__global__ void __launch_bounds__(128) spmm_join_kernel(GradArgs a, int cblocks)
{
    const int k = (int)(blockIdx.x / cblocks) % (a.K + 1);
    const int e = (int)(blockIdx.x / cblocks / (a.K + 1));
    const int col = ((int)(blockIdx.x % cblocks) * 128 + threadIdx.x) * 4;
    int nparts, slot = 0;
    if (a.seg) {
        int mine = 0;
        for (int j = threadIdx.x & 31; j <= e; j += 32) {
            int lo, hi;
            expert_rows(a.seg, j, a.M, lo, hi);
            const int c = (hi - lo + a.per - 1) / a.per;
            if (j < e) slot += c > 1 ? c : 0;
            if (j == e) mine = c;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            slot += __shfl_xor_sync(0xffffffffu, slot, d);
            mine += __shfl_xor_sync(0xffffffffu, mine, d);
        }
        nparts = mine;
    } else {
        nparts = (a.M + a.per - 1) / a.per;
    }
    dependency_wait();
    if (nparts <= 1 || col >= a.stride || slot + nparts > a.slots) return;
    if (k == a.K ? !a.dbias : !a.dvals) return;
    const float* p = a.part + ((long long)slot * (a.K + 1) + k) * a.stride + col;
    const long long step = (long long)(a.K + 1) * a.stride;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int s = 0; s < nparts; ++s) {
        const float4 u = *(const float4*)(p + s * step);
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
    }
    const float o[4] = {v.x, v.y, v.z, v.w};
    T* dst = k == a.K ? (T*)a.dbias + (long long)e * a.n_rows + col
                      : (T*)a.dvals + e * a.estride + (long long)k * a.stride + col;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (k < a.K || col + c < a.n_rows) dst[c] = from_f<T>(o[c]);
}

/* eight elements, p aligned to 16 bytes */
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8])
{
    if (sizeof(T) == 4) {
        *(float4*)v = __ldg((const float4*)p);
        *(float4*)(v + 4) = __ldg((const float4*)p + 1);
    } else {
        __align__(16) T h[8];
        *(uint4*)h = __ldg((const uint4*)p);
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = to_f(h[c]);
    }
}

/* dz = dy * act'(z), rounded to the block's type: both gradients read it as
 * a matrix operand of that type, and one rounding of half a step is no more
 * than the ones dy and z already carry.  Eight elements a thread at a time,
 * two of them in flight. */
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256)
spmm_dz_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ z, long long ldz,
               T* __restrict__ dz, long long lddz, int M, int n)
{
    dependents_begin();
    const int per = (n + 7) / 8;
    const long long total = (long long)per * M, step = gridDim.x * 256ll;
    for (long long p0 = blockIdx.x * 256ll + threadIdx.x; p0 < total; p0 += 2 * step) {
        float a[2][8], b[2][8];
        long long at[2];
        bool wide[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long p = p0 + h * step;
            const long long t = p < total ? p / per : 0;
            const int i = (int)(p - t * per) * 8;
            at[h] = p < total ? t * lddz + i : -1;
            wide[h] = VEC && i + 8 <= n;
            if (at[h] < 0) continue;
            if (wide[h]) {
                load8<T>(dy + t * lddy + i, a[h]);
                load8<T>(z + t * ldz + i, b[h]);
            } else {
                for (int c = 0; c < 8 && i + c < n; ++c)
                    dz[at[h] + c] = from_f<T>(to_f(dy[t * lddy + i + c]) *
                                              dact_of<ACT>(to_f(z[t * ldz + i + c])));
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (at[h] < 0 || !wide[h]) continue;
            __align__(16) T r[8];
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
                const float2 d = sizeof(T) == 2
                                     ? dact2<ACT>(make_float2(b[h][c], b[h][c + 1]))
                                     : make_float2(dact_of<ACT>(b[h][c]), dact_of<ACT>(b[h][c + 1]));
                r[c] = from_f<T>(a[h][c] * d.x);
                r[c + 1] = from_f<T>(a[h][c + 1] * d.y);
            }
#pragma unroll
            for (int c = 0; c < (int)(8 * sizeof(T)); c += 16)
                *(uint4*)((char*)(dz + at[h]) + c) = *(const uint4*)((const char*)r + c);
        }
    }
    dependency_wait();
}

/* ---------------------------------------------------------------- host */

/* test hook (dia_test_spmm_form): 0 the rule, 1 CUDA cores, 2 tensor cores
 * wherever they can run */
static std::atomic<int> g_form{0};

static bool tensor_form(int dtype, long long M, int E, const SpmmDir& d)
{
    const int form = g_form.load(std::memory_order_relaxed);
    if (dtype == DIA_F32 || d.nboxes == 0 || form == 1) return false;
    if (form == 2) return true;
    return M / std::max(E, 1) >= 64;
}

static size_t elem_size(int dtype) { return dtype == DIA_F32 ? 4 : 2; }

static bool vec16(const void* p, long long ld, int dtype)
{
    return (uintptr_t)p % 16 == 0 && ld * (long long)elem_size(dtype) % 16 == 0;
}

template <typename T, bool TRANS, int TT>
static int launch_few(const ProdArgs& a, cudaStream_t stream)
{
    const int ftiles = (a.n_out + 31) / 32;
    const long long ngroups = a.seg ? a.M / TT + std::min(a.E, a.M) : (a.M + TT - 1) / TT;
    /* warps that share a tile: until every SM has 32, or a warp four diagonals */
    int ks = 1;
    while (ks < kFewWarps && (long long)ftiles * ngroups * ks < 32ll * num_sms() && a.K > 4 * ks)
        ks *= 2;
    const int fper = kFewWarps / ks;
    const long long grid = ngroups * ((ftiles + fper - 1) / fper);
    if (grid > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm: block too large");
    /* the larger of block and operator is streamed once, the other stays in L2 */
    const bool rows_first = (long long)a.M * a.n_in < a.stride * a.K;
    spmm_few_kernel<T, TRANS, TT><<<(unsigned)grid, kFewWarps * 32, 0, stream>>>(
        a, ks, ftiles, ngroups, rows_first);
    DIA_TRY_CUDA(cudaGetLastError());
    return DIA_OK;
}

template <typename T, bool TRANS, bool VEC, bool QUADS>
static int launch_tile_as(const ProdArgs& a, int shape, int smem, cudaStream_t stream)
{
    const int F = kTileF[shape], rows = kTileWarps * kTileRows * 128 / F;
    const int ftiles = (a.n_out + F - 1) / F;
    const long long ngroups = a.seg ? a.M / rows + std::min(a.E, a.M) : (a.M + rows - 1) / rows;
    if (ngroups * ftiles > INT_MAX)
        return fail(DIA_ERR_UNSUPPORTED, "dia_spmm: block too large");
    const bool rows_first = (long long)a.M * a.n_in < a.stride * a.K;
    const auto kernel = spmm_tile_kernel<T, TRANS, VEC, QUADS>;
    static SmemRecord most;
    DIA_TRY_CUDA(allow_smem(kernel, kTileSmem, most));
    kernel<<<(unsigned)(ngroups * ftiles), kTileWarps * 32, smem, stream>>>(a, shape, ftiles,
                                                                            ngroups, rows_first);
    DIA_TRY_CUDA(cudaGetLastError());
    return DIA_OK;
}

static int tile_smem(const SpmmDir& d, int shape, size_t elem)
{
    return (int)std::min<long long>(INT_MAX, (long long)kTileWarps * kTileRows * 128 /
                                                 kTileF[shape] * d.width[shape] * (long long)elem);
}

template <typename T, bool TRANS>
static int launch_cores(const ProdArgs& a, int dtype, cudaStream_t stream)
{
    const int per = a.M / std::max(a.E, 1);   /* rows of a usual expert */
    if (per >= 8 && a.K > 0) {
        /* the widest tile (an input is read again by fewer tiles) whose inputs
         * fit and that leaves a CTA for every SM */
        for (int shape = 2; shape >= 0; --shape) {
            const int smem = tile_smem(a.dir, shape, sizeof(T));
            const int rows = kTileWarps * kTileRows * 128 / kTileF[shape];
            const long long ctas = (long long)((a.n_out + kTileF[shape] - 1) / kTileF[shape]) *
                                   ((a.M + rows - 1) / rows);
            if (smem > kTileSmem || (shape > 0 && ctas < num_sms())) continue;
            const bool vec = vec16(a.in, a.ldi, dtype), quads = 3 * a.dir.nquads <= a.K;
            if (vec)
                return quads ? launch_tile_as<T, TRANS, true, true>(a, shape, smem, stream)
                             : launch_tile_as<T, TRANS, true, false>(a, shape, smem, stream);
            return quads ? launch_tile_as<T, TRANS, false, true>(a, shape, smem, stream)
                         : launch_tile_as<T, TRANS, false, false>(a, shape, smem, stream);
        }
    }
    if (per >= 5) return launch_few<T, TRANS, 8>(a, stream);
    return per >= 2 ? launch_few<T, TRANS, 4>(a, stream) : launch_few<T, TRANS, 1>(a, stream);
}

/* the tensor-core form it is (its operator has to be packed first) */
static bool product_on_tc(const ProdArgs& a, int dtype)
{
    return a.M > 0 && a.n_out > 0 && a.n_in > 0 && tensor_form(dtype, a.M, a.E, a.dir) &&
           spmm_tc_block(a.in, a.ldi);
}

template <typename T>
static int launch_product(const ProdArgs& a, int dtype, cudaStream_t stream)
{
    if (a.M == 0 || a.n_out == 0) return DIA_OK;
    if (product_on_tc(a, dtype)) return spmm_tc_product(a, dtype, stream);
    return a.trans ? launch_cores<T, true>(a, dtype, stream)
                   : launch_cores<T, false>(a, dtype, stream);
}

template <typename T, int ACT>
static cudaError_t launch_dz_act(const void* dy, long long lddy, const void* z, long long ldz,
                                 void* dz, long long lddz, int M, int n, bool dependent,
                                 cudaStream_t stream)
{
    const long long work = (long long)M * ((n + 7) / 8);
    const int grid = (int)std::min<long long>((work + 511) / 512, 8ll * num_sms());
    const int dtype = sizeof(T) == 4 ? DIA_F32 : DIA_F16;
    const auto kernel = vec16(dy, lddy, dtype) && vec16(z, ldz, dtype)
                            ? spmm_dz_kernel<T, ACT, true>
                            : spmm_dz_kernel<T, ACT, false>;
    if (dependent)
        return launch_dependent(kernel, grid, 256, 0, stream, (const T*)dy, lddy, (const T*)z, ldz,
                                (T*)dz, lddz, M, n);
    kernel<<<grid, 256, 0, stream>>>((const T*)dy, lddy, (const T*)z, ldz, (T*)dz, lddz, M, n);
    return cudaGetLastError();
}

template <typename T>
static int launch_dz(int act, const void* dy, long long lddy, const void* z, long long ldz,
                     void* dz, long long lddz, int M, int n, bool dependent, cudaStream_t stream)
{
    if (M == 0 || n == 0) return DIA_OK;
    const auto launch = act == DIA_ACT_RELU   ? launch_dz_act<T, DIA_ACT_RELU>
                        : act == DIA_ACT_SILU ? launch_dz_act<T, DIA_ACT_SILU>
                        : act == DIA_ACT_GELU ? launch_dz_act<T, DIA_ACT_GELU>
                                              : launch_dz_act<T, DIA_ACT_GELU_TANH>;
    DIA_TRY_CUDA(launch(dy, lddy, z, ldz, dz, lddz, M, n, dependent, stream));
    return DIA_OK;
}

/* rows of a part of the gradient's sum: enough parts to fill the GPU, none
 * so short that writing and joining its sums costs more than it saves */
static int grad_part_rows(const DiaSpmmPlan* p, int dtype, long long M, int E, long long stride)
{
    if (tensor_form(dtype, M, E, p->fwd)) {
        /* one CTA an SM, of which every expert takes one a tile */
        const long long tiles = std::max<long long>(1, (stride + 127) / 128) *
                                ((p->fwd.nboxes + 3) / 4);
        const long long want = std::max<long long>(1, num_sms() / tiles - (E - 1));
        const long long per = std::max<long long>(256, (M + want - 1) / want);
        return (int)((per + 63) / 64 * 64);
    }
    /* a few CTAs an SM */
    const long long tiles = std::max<long long>(1, (stride + 127) / 128) * std::max(1, p->fwd.nwins);
    const long long want = std::max<long long>(1, 4ll * num_sms() / tiles - (E - 1));
    const long long per = std::max<long long>(32, (M + want - 1) / want);
    return (int)((per + 7) / 8 * 8);
}

/* parts of experts that have several: at most two a `per` rows */
static long long grad_slots(long long M, long long per) { return M > per ? 2 * (M / per) + 1 : 0; }

static bool grad_on_tc(const GradArgs& a, int dtype)
{
    return tensor_form(dtype, a.M, a.E, a.dir) && a.M > 0 && a.n_cols > 0 && a.n_rows > 0 &&
           a.dvals && spmm_tc_block(a.dz, a.lddz) && spmm_tc_block(a.x, a.ldx);
}

template <typename T>
static int launch_grad(const GradArgs& a, int dtype, cudaStream_t stream)
{
    if (grad_on_tc(a, dtype)) return spmm_tc_gradient(a, dtype, stream);
    const int ftiles = (int)((a.stride + 127) / 128);
    const int nwins = a.dvals ? std::max(a.dir.nwins, 1) : 1;
    const long long parts = a.seg ? a.M / a.per + a.E : std::max(1, (a.M + a.per - 1) / a.per);
    const long long grid = parts * ftiles * nwins;
    if (grid > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm_backward: block too large");
    /* rows a stage: two CTAs an SM where that leaves eight or more */
    const int row_bytes = 2 * ((a.dvals ? a.dir.wwidth : 0) + 128) * (int)sizeof(T);
    const int rows = std::min(32, std::max(8, 100 * 1024 / row_bytes / 8 * 8));
    const int smem = rows * row_bytes;
    const bool vec = vec16(a.dz, a.lddz, dtype) && vec16(a.x, a.ldx, dtype);
    const int nd = a.dvals ? (a.dir.wdiags + kTileWarps - 1) / kTileWarps : 1;
    const int pick = nd <= 1 ? 0 : nd <= 2 ? 1 : nd <= 3 ? 2 : nd <= 5 ? 3 : 4;
    using Kernel = void (*)(GradArgs, int, int, int);
    static const Kernel kernels[2][5] = {
        {spmm_grad_kernel<T, false, 1>, spmm_grad_kernel<T, false, 2>,
         spmm_grad_kernel<T, false, 3>, spmm_grad_kernel<T, false, 5>,
         spmm_grad_kernel<T, false, 8>},
        {spmm_grad_kernel<T, true, 1>, spmm_grad_kernel<T, true, 2>, spmm_grad_kernel<T, true, 3>,
         spmm_grad_kernel<T, true, 5>, spmm_grad_kernel<T, true, 8>}};
    const Kernel kernel = kernels[vec][pick];
    static SmemRecord most[2][5];
    DIA_TRY_CUDA(allow_smem(kernel, kGradSmem, most[vec][pick]));
    kernel<<<(unsigned)grid, kTileWarps * 32, smem, stream>>>(a, ftiles, nwins, rows);
    DIA_TRY_CUDA(cudaGetLastError());
    return DIA_OK;
}

template <typename T>
static int launch_join(const GradArgs& a, cudaStream_t stream)
{
    if (a.M <= a.per) return DIA_OK;   /* no expert has several parts */
    const int cblocks = (int)((a.stride + 511) / 512);
    const long long grid = (long long)a.E * (a.K + 1) * cblocks;
    if (grid > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm_backward: block too large");
    DIA_TRY_CUDA(launch_dependent(spmm_join_kernel<T>, (int)grid, 128, 0, stream, a, cblocks));
    return DIA_OK;
}

/* (offset, storage index) in ascending order */
static std::vector<int2> sorted_offsets(const std::vector<int>& off)
{
    std::vector<int2> s(off.size());
    for (size_t k = 0; k < off.size(); ++k) s[k] = make_int2(off[k], (int)k);
    std::sort(s.begin(), s.end(), [](int2 a, int2 b) { return a.x < b.x; });
    return s;
}

static std::vector<Box> build_boxes(const std::vector<int2>& s)
{
    std::vector<Box> boxes;
    int end = INT_MIN;   /* inputs below this are covered */
    for (const int2& o : s)
        for (end = std::max(end, o.x & ~7); end < o.x + 128; end += 64) {
            Box b{end, 0, 0, 0};
            auto first = [&](int d) {
                return (int)(std::lower_bound(s.begin(), s.end(), d,
                                              [](int2 a, int v) { return a.x < v; }) - s.begin());
            };
            b.k0 = first(end - 127);
            b.k1 = first(end + 64);
            boxes.push_back(b);
        }
    return boxes;
}

/* Windows of F features: spans for the sorted offsets [k0, k1), neighbouring
 * ones in one span where the gap is below 32 inputs; the columns they take.
 * cols[k - k0] becomes the column that input i0 + offset of diagonal k has. */
static int build_spans(const std::vector<int2>& s, size_t k0, size_t k1, int F,
                       std::vector<InputSpan>& spans, std::vector<int>& cols)
{
    const size_t first = spans.size();
    long long at = 0;
    for (size_t k = k0; k < k1; ++k) {
        const int d = s[k].x, end = d + F;
        if (spans.size() == first || d > spans.back().from + spans.back().len + 24) {
            InputSpan sp{d & ~7, 0, 0, 0};
            spans.push_back(sp);
        }
        spans.back().len = (end - spans.back().from + 15) / 8 * 8;   /* eight to spare */
    }
    for (size_t i = first; i < spans.size(); ++i) {
        spans[i].at = (int)std::min<long long>(at, INT_MAX / 2);
        at += spans[i].len;
    }
    size_t i = first;
    for (size_t k = k0; k < k1; ++k) {
        while (s[k].x >= spans[i].from + spans[i].len) ++i;
        cols.push_back(spans[i].at + s[k].x - spans[i].from);
    }
    return (int)std::min<long long>(at, INT_MAX / 2);
}

static std::vector<Quad> build_quads(const std::vector<int2>& s, const std::vector<int>& cols)
{
    std::vector<Quad> quads;
    for (size_t k = 0; k < s.size(); ++k) {
        const int base = s[k].x & ~3;   /* floor to a multiple of four */
        if (quads.empty() || quads.back().base != base) {
            Quad q;
            std::memset(&q, 0, sizeof(q));
            q.base = base;
            q.k[0] = q.k[1] = q.k[2] = q.k[3] = -1;
            q.col = cols[k] - (s[k].x - base);   /* spans begin at multiples of eight */
            quads.push_back(q);
        }
        quads.back().k[s[k].x - base] = s[k].y;
    }
    return quads;
}

/* One direction's tables appended to `blob`: `dir` with offsets into it in
 * place of pointers, which dir_on_device makes pointers. */
template <typename T>
static const T* append(std::vector<char>& blob, const std::vector<T>& v)
{
    const size_t at = (blob.size() + 31) / 32 * 32;
    blob.resize(at + v.size() * sizeof(T));
    if (!v.empty()) std::memcpy(blob.data() + at, v.data(), v.size() * sizeof(T));
    return (const T*)at;
}

constexpr int kWinCols = 2304;   /* columns of a gradient window: 72 KB of eight fp32 rows */

static SpmmDir append_dir(std::vector<char>& blob, const std::vector<int>& off)
{
    const std::vector<int2> s = sorted_offsets(off);
    const std::vector<Box> b = build_boxes(s);
    SpmmDir d{};
    d.nboxes = (int)b.size();
    d.boxes = append(blob, b);
    d.offs = append(blob, s);
    for (int shape = 0; shape < 3; ++shape) {
        std::vector<InputSpan> spans;
        std::vector<int> cols;
        d.width[shape] = build_spans(s, 0, s.size(), kTileF[shape], spans, cols);
        const std::vector<Quad> q = build_quads(s, cols);
        d.nquads = (int)q.size();
        d.nspans[shape] = (int)spans.size();
        d.quads[shape] = append(blob, q);
        d.spans[shape] = append(blob, spans);
        d.cols[shape] = append(blob, cols);
    }
    /* up to 64 diagonals a window, fewer where they lie apart (two always fit) */
    std::vector<GradWindow> wins;
    std::vector<InputSpan> wspans;
    std::vector<int> wcols;
    for (size_t k0 = 0; k0 < s.size();) {
        size_t k1 = std::min(s.size(), k0 + kTileWarps * kGradDiags);
        std::vector<InputSpan> spans;
        std::vector<int> cols;
        int width = build_spans(s, k0, k1, 128, spans, cols);
        while (width > kWinCols) {
            k1 = k0 + (k1 - k0 + 1) / 2;
            spans.clear();
            cols.clear();
            width = build_spans(s, k0, k1, 128, spans, cols);
        }
        GradWindow w{};
        w.k0 = (int)k0;
        w.k1 = (int)k1;
        w.s0 = (int)wspans.size();
        w.s1 = w.s0 + (int)spans.size();
        w.cols = width;
        wins.push_back(w);
        wspans.insert(wspans.end(), spans.begin(), spans.end());
        wcols.insert(wcols.end(), cols.begin(), cols.end());
        d.wwidth = std::max(d.wwidth, width);
        d.wdiags = std::max(d.wdiags, (int)(k1 - k0));
        k0 = k1;
    }
    d.nwins = (int)wins.size();
    d.tile_span = append(blob, std::vector<InputSpan>{InputSpan{0, 128, 0, 0}});
    d.wins = append(blob, wins);
    d.wspans = append(blob, wspans);
    d.wcols = append(blob, wcols);
    return d;
}

template <typename T>
static void place(const T*& p, const void* blob)
{
    p = (const T*)((const char*)blob + (size_t)p);
}

static SpmmDir dir_on_device(const void* blob, SpmmDir d)
{
    place(d.boxes, blob);
    place(d.offs, blob);
    for (int shape = 0; shape < 3; ++shape) {
        place(d.quads[shape], blob);
        place(d.spans[shape], blob);
        place(d.cols[shape], blob);
    }
    place(d.tile_span, blob);
    place(d.wins, blob);
    place(d.wspans, blob);
    place(d.wcols, blob);
    return d;
}

/* arguments both directions share; DIA_OK or the error */
static int check_common(const char* who, const DiaSpmmPlan* p, int dtype, int64_t M, int E,
                        const int64_t* seg, int act, int64_t stride, const void* vals)
{
    const std::string w = std::string(who) + ": ";
    if (dtype != DIA_F32 && dtype != DIA_F16 && dtype != DIA_BF16)
        return fail(DIA_ERR_INVALID, w + "unknown dtype");
    if (act < DIA_ACT_NONE || act > DIA_ACT_GELU_TANH)
        return fail(DIA_ERR_INVALID, w + "unknown activation");
    if (M < 0 || M > INT_MAX / 2) return fail(DIA_ERR_INVALID, w + "bad number of rows");
    if (E < 1 || E > (1 << 20)) return fail(DIA_ERR_INVALID, w + "bad number of experts");
    if (E > 1 && !seg) return fail(DIA_ERR_INVALID, w + "experts without seg");
    if (!p) return fail(DIA_ERR_INVALID, w + "null plan");
    int dev = -1;
    DIA_TRY_CUDA(cudaGetDevice(&dev));
    if (dev != p->device)
        return fail(DIA_ERR_INVALID, w + "the plan belongs to another device");
    if (stride < p->n_rows || stride % 32 != 0)
        return fail(DIA_ERR_INVALID, w + "stride must be a multiple of 32, at least n_rows");
    if (stride > INT_MAX / 2) return fail(DIA_ERR_UNSUPPORTED, w + "stride too large");
    if (p->K > 0 && p->n_rows > 0 && !vals) return fail(DIA_ERR_INVALID, w + "null values");
    if ((uintptr_t)vals % 16) return fail(DIA_ERR_INVALID, w + "values must be 16-byte aligned");
    return DIA_OK;
}

/* a block of M rows of n elements: pointer, row stride and element alignment */
static int check_block(const char* who, const char* name, const void* ptr, int64_t ld, int64_t M,
                       int n, int dtype)
{
    const std::string w = std::string(who) + ": " + name;
    if (M == 0 || n == 0) return DIA_OK;
    if (!ptr) return fail(DIA_ERR_INVALID, w + " is null");
    if (M > 1 && ld < n) return fail(DIA_ERR_INVALID, w + " has rows shorter than its width");
    if ((uintptr_t)ptr % elem_size(dtype)) return fail(DIA_ERR_INVALID, w + " is misaligned");
    return DIA_OK;
}

template <typename F>
static int by_type(int dtype, F f)
{
    if (dtype == DIA_F32) return f((float*)nullptr);
    if (dtype == DIA_F16) return f((__half*)nullptr);
    return f((__nv_bfloat16*)nullptr);
}

static long long align256(long long b) { return (b + 255) / 256 * 256; }

/* the operator in tensor-core form */
static long long pack_bytes(const SpmmDir& d, int dtype, int64_t M, int E, int n_out)
{
    return M > 0 && tensor_form(dtype, M, E, d) ? spmm_tc_pack_bytes(n_out, d.nboxes, E) : 0;
}

/* the gradient's workspace: dz (where the activation makes one), then sums
 * of parts (where there are several), then the operator's boxes */
struct GradPlan {
    int per;
    long long lddz, dz_bytes, part_bytes, pack_bytes;
    long long bytes() const { return dz_bytes + part_bytes + pack_bytes; }
};

static GradPlan grad_plan(const DiaSpmmPlan* p, int dtype, int64_t M, int E, int64_t stride,
                          int act)
{
    GradPlan g;
    g.per = grad_part_rows(p, dtype, M, E, stride);
    g.lddz = (p->n_rows + 7) / 8 * 8;
    g.dz_bytes = act == DIA_ACT_NONE ? 0 : align256(M * g.lddz * (long long)elem_size(dtype));
    g.part_bytes = align256(grad_slots(M, g.per) * (p->K + 1) * stride * 4);
    g.pack_bytes = pack_bytes(p->trn, dtype, M, E, p->n_cols);
    return g;
}

}  // namespace dia

using namespace dia;

extern "C" int dia_spmm_plan_create(int64_t n_rows, int64_t n_cols, int num_diags,
                                    const int* h_offsets, DiaSpmmPlan** plan)
{
    if (!plan) return fail(DIA_ERR_INVALID, "dia_spmm_plan_create: null plan");
    *plan = nullptr;
    if (n_rows < 0 || n_cols < 0 || num_diags < 0)
        return fail(DIA_ERR_INVALID, "dia_spmm_plan_create: negative size");
    if (num_diags > 0 && !h_offsets)
        return fail(DIA_ERR_INVALID, "dia_spmm_plan_create: null offsets");
    /* every i + d of a stored entry, and a tile beyond, stays a 32-bit int */
    if (n_rows + n_cols > INT_MAX / 2 || num_diags > (1 << 20))
        return fail(DIA_ERR_UNSUPPORTED, "dia_spmm_plan_create: operator too large");
    try {
        std::vector<int> fwd(h_offsets, h_offsets + num_diags);
        std::vector<int> sorted = fwd;
        std::sort(sorted.begin(), sorted.end());
        if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end())
            return fail(DIA_ERR_INVALID, "dia_spmm_plan_create: an offset occurs twice");
        /* a diagonal outside the matrix has no entries: its place in the
         * tables is any offset out of reach, one for each */
        int out = (int)n_cols;
        for (int& d : fwd)
            if (d <= -n_rows || d >= n_cols) d = out++;
        std::vector<int> trn(fwd.size());
        for (size_t k = 0; k < fwd.size(); ++k) trn[k] = -fwd[k];
        std::vector<char> blob;
        const SpmmDir tf = append_dir(blob, fwd), tt = append_dir(blob, trn);
        DiaSpmmPlan* p = new DiaSpmmPlan();
        p->n_rows = (int)n_rows;
        p->n_cols = (int)n_cols;
        p->K = num_diags;
        cudaError_t e = cudaGetDevice(&p->device);
        if (e == cudaSuccess && !blob.empty()) e = cudaMalloc(&p->blob, blob.size());
        if (e == cudaSuccess && !blob.empty())
            e = cudaMemcpy(p->blob, blob.data(), blob.size(), cudaMemcpyHostToDevice);
        if (e != cudaSuccess) {
            if (p->blob) cudaFree(p->blob);
            delete p;
            return cuda_fail(e, "dia_spmm_plan_create");
        }
        p->fwd = dir_on_device(p->blob, tf);
        p->trn = dir_on_device(p->blob, tt);
        *plan = p;
        return DIA_OK;
    } catch (const std::bad_alloc&) {
        return fail(DIA_ERR_CAPACITY, "dia_spmm_plan_create: out of host memory");
    }
}

extern "C" int dia_spmm_plan_destroy(DiaSpmmPlan* plan)
{
    if (!plan) return DIA_OK;
    if (plan->blob) cudaFree(plan->blob);
    delete plan;
    return DIA_OK;
}

extern "C" int dia_spmm(const DiaSpmmPlan* plan, int dtype, int64_t M, int num_experts,
                        const int64_t* d_seg, const void* d_x, int64_t ldx, const void* d_vals,
                        int64_t stride, const void* d_bias, int act, const void* d_res,
                        int64_t ldr, void* d_z, int64_t ldz, void* d_y, int64_t ldy,
                        void* d_work, int64_t work_bytes, cudaStream_t stream)
{
    const char* who = "dia_spmm";
    int rc = check_common(who, plan, dtype, M, num_experts, d_seg, act, stride, d_vals);
    if (rc == DIA_OK && plan->K > 0)
        rc = check_block(who, "x", d_x, ldx, M, plan->n_cols, dtype);
    if (rc == DIA_OK) rc = check_block(who, "y", d_y, ldy, M, plan->n_rows, dtype);
    if (rc == DIA_OK && d_res) rc = check_block(who, "residual", d_res, ldr, M, plan->n_rows, dtype);
    if (rc == DIA_OK && d_z) rc = check_block(who, "z", d_z, ldz, M, plan->n_rows, dtype);
    if (rc != DIA_OK) return rc;
    const long long need = pack_bytes(plan->fwd, dtype, M, num_experts, plan->n_rows);
    if (need > work_bytes) return fail(DIA_ERR_CAPACITY, "dia_spmm: workspace too small");
    if (need > 0 && (!d_work || (uintptr_t)d_work % 256))
        return fail(DIA_ERR_INVALID, "dia_spmm: workspace must be 256-byte aligned");
    ProdArgs a{};
    a.pack = d_work;
    a.in = d_x;
    a.vals = d_vals;
    a.bias = d_bias;
    a.res = d_res;
    a.z = d_z;
    a.out = d_y;
    a.seg = (const long long*)d_seg;
    a.ldi = ldx;
    a.ldr = ldr;
    a.ldz = ldz;
    a.ldo = ldy;
    a.stride = stride;
    a.estride = stride * plan->K;
    a.M = (int)M;
    a.E = num_experts;
    a.n_in = plan->n_cols;
    a.n_out = plan->n_rows;
    a.K = plan->K;
    a.act = act;
    a.dir = plan->fwd;
    a.trans = false;
    if (product_on_tc(a, dtype)) {
        rc = spmm_tc_pack(a, stream);
        if (rc != DIA_OK) return rc;
    }
    return by_type(dtype, [&](auto* t) {
        return launch_product<std::remove_pointer_t<decltype(t)>>(a, dtype, stream);
    });
}

extern "C" int64_t dia_spmm_workspace(const DiaSpmmPlan* plan, int dtype, int64_t M,
                                      int num_experts)
{
    if (!plan || M < 0 || M > INT_MAX / 2 || num_experts < 1) return -1;
    return pack_bytes(plan->fwd, dtype, M, num_experts, plan->n_rows);
}

extern "C" int64_t dia_spmm_backward_workspace(const DiaSpmmPlan* plan, int dtype, int64_t M,
                                               int num_experts, int64_t stride, int act)
{
    if (!plan || M < 0 || M > INT_MAX / 2 || stride < 0 || num_experts < 1) return -1;
    const GradPlan g = grad_plan(plan, dtype, M, num_experts, stride, act);
    return g.bytes();
}

extern "C" int dia_spmm_backward(const DiaSpmmPlan* plan, int dtype, int64_t M, int num_experts,
                                 const int64_t* d_seg, const void* d_x, int64_t ldx,
                                 const void* d_vals, int64_t stride, const void* d_dy,
                                 int64_t lddy, int act, const void* d_z, int64_t ldz, void* d_dx,
                                 int64_t lddx, void* d_dvals, void* d_dbias, void* d_work,
                                 int64_t work_bytes, cudaStream_t stream)
{
    const char* who = "dia_spmm_backward";
    int rc = check_common(who, plan, dtype, M, num_experts, d_seg, act, stride,
                          d_dx ? d_vals : (const void*)16);
    if (rc == DIA_OK && d_dvals && plan->K > 0)
        rc = check_block(who, "x", d_x, ldx, M, plan->n_cols, dtype);
    if (rc == DIA_OK) rc = check_block(who, "dy", d_dy, lddy, M, plan->n_rows, dtype);
    if (rc == DIA_OK && act != DIA_ACT_NONE)
        rc = check_block(who, "z", d_z, ldz, M, plan->n_rows, dtype);
    if (rc == DIA_OK && d_dx) rc = check_block(who, "dx", d_dx, lddx, M, plan->n_cols, dtype);
    if (rc != DIA_OK) return rc;
    const GradPlan g = grad_plan(plan, dtype, M, num_experts, stride, act);
    if (g.bytes() > work_bytes)
        return fail(DIA_ERR_CAPACITY, "dia_spmm_backward: workspace too small");
    if (g.bytes() > 0 && (!d_work || (uintptr_t)d_work % 256))
        return fail(DIA_ERR_INVALID, "dia_spmm_backward: workspace must be 256-byte aligned");

    return by_type(dtype, [&](auto* t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        const bool made = act != DIA_ACT_NONE;
        ProdArgs p{};
        p.in = made ? d_work : d_dy;
        p.vals = d_vals;
        p.out = d_dx;
        p.pack = (char*)d_work + g.dz_bytes + g.part_bytes;
        p.seg = (const long long*)d_seg;
        p.ldi = made ? g.lddz : lddy;
        p.ldo = lddx;
        p.stride = stride;
        p.estride = stride * plan->K;
        p.M = (int)M;
        p.E = num_experts;
        p.n_in = plan->n_rows;
        p.n_out = plan->n_cols;
        p.K = plan->K;
        p.dir = plan->trn;
        p.trans = true;
        GradArgs a{};
        a.dz = p.in;
        a.x = d_x;
        a.dvals = plan->K > 0 ? d_dvals : nullptr;
        a.dbias = d_dbias;
        a.part = (float*)((char*)d_work + g.dz_bytes);
        a.seg = p.seg;
        a.lddz = p.ldi;
        a.ldx = ldx;
        a.stride = stride;
        a.estride = p.estride;
        a.M = p.M;
        a.E = num_experts;
        a.n_rows = plan->n_rows;
        a.n_cols = plan->n_cols;
        a.K = plan->K;
        a.per = g.per;
        a.slots = grad_slots(M, g.per);
        a.dir = plan->fwd;
        const bool grad = (a.dvals || a.dbias) && stride > 0;
        /* launches overlap where each is of the tensor-core form: operator
         * packed, dz, gradient of the diagonals, dx, parts joined */
        const bool tc = d_dx && product_on_tc(p, dtype);
        int r = DIA_OK;
        if (tc) r = spmm_tc_pack(p, stream);
        if (r == DIA_OK && made)
            r = launch_dz<T>(act, d_dy, lddy, d_z, ldz, d_work, p.ldi, p.M, p.n_in, tc, stream);
        if (r == DIA_OK && grad) {
            const bool overlap = tc && grad_on_tc(a, dtype);
            r = launch_grad<T>(a, dtype, stream);
            p.early = overlap;
        }
        if (r == DIA_OK && d_dx) r = launch_product<T>(p, dtype, stream);
        if (r == DIA_OK && grad) r = launch_join<T>(a, stream);
        return r;
    });
}

extern "C" int dia_test_spmm_form(int form)
{
    if (form < 0 || form > 2) return fail(DIA_ERR_INVALID, "dia_test_spmm_form: 0, 1 or 2");
    g_form.store(form);
    return DIA_OK;
}
