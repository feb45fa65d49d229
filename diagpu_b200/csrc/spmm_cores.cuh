/*
 * spmm_cores.cuh -- CUDA-core kernels of the block-vector product and its
 * gradients for one element type, and their launches (Cores<T>); one
 * translation unit a type includes it.
 */
#pragma once

#include <algorithm>
#include <climits>

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
 * other features.  One row of 4096 under 129 diagonals, bf16: 5.5 us; eight
 * rows under 33, fp32: 5.2 us; 64 rows of 64 experts (1024, 33 diagonals,
 * fp16): 10.1 us, all a launch and three or four dependent reads (their bytes
 * take 0.1 to 0.7 us). */
constexpr int kFewWarps = 16;
constexpr int kFewOffs = 512;   /* offsets staged at once */

template <typename T, typename IN, bool TRANS, int TT>
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
    const IN* in = (const IN*)a.in + rg.r0 * a.ldi;
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
        float y = acc[t] + bias;
        if (!TRANS) {
            if (a.z) ((T*)a.z)[row * a.ldz + i] = from_f<T>(y);
            if (a.act != DIA_ACT_NONE) y = act1(a.act, y);
            y += res[t];
        }
        ((T*)a.out)[row * a.ldo + i] = from_f<T>(y);
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
 * conflicts at any offset.  Shared memory's bandwidth bounds both: 64 rows of
 * 262144 under a 27-point stencil, fp32, 115 us (3.9 products a picosecond,
 * load and store unit two thirds busy; the 163 MB that memory has to give
 * would take 25).  Twice the warps with half the features each took 128, two
 * rows a packed multiplication changed nothing. */
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

template <typename T, typename IN, bool TRANS, bool VEC, bool QUADS>
__global__ void __launch_bounds__(kTileWarps * 32)
spmm_tile_kernel(const __grid_constant__ ProdArgs a, int shape, int ftiles, long long ngroups,
                 bool rows_first)
{
    extern __shared__ __align__(16) unsigned char smem_raw[];
    IN* xs = (IN*)smem_raw;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int F = kTileF[0] << shape, wf = F / 128;   /* warps side by side */
    const int rows = kTileWarps / wf * kTileRows;
    const long long b = blockIdx.x;
    const long long g = rows_first ? b % ngroups : b / ftiles;
    const int i0 = (int)(rows_first ? b / ngroups : b % ftiles) * F;
    const RowGroup rg = row_group(a.seg, a.E, a.M, rows, g, false);
    if (rg.e < 0) return;   /* whole CTA */
    const int nt = rg.r1 - rg.r0, pitch = a.dir.width[shape];
    stage_spans<IN, VEC>(xs, pitch, a.dir.spans[shape], 0, a.dir.nspans[shape],
                         (const IN*)a.in + rg.r0 * a.ldi, a.ldi, i0, a.n_in, rows, nt);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    const int t0 = warp / wf * kTileRows, f0 = warp % wf * 128;
    if (t0 >= nt || i0 + f0 >= a.n_out) return;
    const int live = min(nt - t0, kTileRows);
    const T* vals = (const T*)a.vals + rg.e * a.estride;
    const IN* xw = xs + t0 * pitch;
    float acc[kTileRows][4];
#pragma unroll
    for (int t = 0; t < kTileRows; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][r] = 0.0f;

    constexpr int STEP = QUADS ? 1 : 32;             /* between a lane's features */
    const int f = f0 + (QUADS ? 4 * lane : lane), i = i0 + f;
    if (QUADS) {
        const Quad* quads = a.dir.quads[shape];
        /* a quad's values are read while the one before is worked on */
        struct Weights {
            float w[4][4];
            int base, col, on;   /* on: bit s where slot s has a diagonal */
        };
        auto fetch = [&](int q, Weights& v) {
            const int4 h = __ldg((const int4*)&quads[q]);
            const int2 h2 = __ldg((const int2*)&quads[q].k[3]);
            const int kk[4] = {h.y, h.z, h.w, h2.x};
            v.base = h.x;
            v.col = h2.y;
            v.on = 0;
            const int c = i + h.x;
            const bool inside = c >= 0 && c + 7 <= a.n_in && i + 4 <= a.n_out;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (kk[s] < 0) continue;
                v.on |= 1 << s;
                const T* vp = vals + (long long)kk[s] * a.stride + (TRANS ? c + s : i);
                if (!TRANS && inside) {
                    *(float4*)v.w[s] = load4<T>(vp);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        v.w[s][r] = i + r < a.n_out && (unsigned)(c + s + r) < (unsigned)a.n_in
                                        ? to_f(vp[r]) : 0.0f;
                }
            }
        };
        float carry[kTileRows][4];
        int next = INT_MIN;   /* base of the quad whose first piece `carry` holds */
        auto work = [&](const Weights& v) {
            const IN* p = xw + v.col + f;
            if (v.base != next) {
#pragma unroll
                for (int t = 0; t < kTileRows; ++t) *(float4*)carry[t] = load4<IN>(p + t * pitch);
            }
            next = v.base + 4;
#pragma unroll
            for (int t = 0; t < kTileRows; ++t) {
                float x[8];
                *(float4*)x = *(float4*)carry[t];
                *(float4*)(x + 4) = load4<IN>(p + t * pitch + 4);
                *(float4*)carry[t] = *(float4*)(x + 4);
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    if (v.on >> s & 1)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            acc[t][r] = fmaf(v.w[s][r], x[s + r], acc[t][r]);
            }
        };
        Weights u, v;
        fetch(0, u);
        for (int q = 0; q < a.dir.nquads; q += 2) {
            if (q + 1 < a.dir.nquads) fetch(q + 1, v);
            work(u);
            if (q + 1 >= a.dir.nquads) break;
            if (q + 2 < a.dir.nquads) fetch(q + 2, u);
            work(v);
        }
    } else {
        const int* cols = a.dir.cols[shape];
        /* diagonals in fours; the next four's values are read while these are
         * worked on */
        constexpr int U = 4;
        /* every entry of the warp's features is in the matrix */
        const bool inside = i0 + f0 + 128 <= a.n_out && i0 + f0 + __ldg(&a.dir.offs[0].x) >= 0 &&
                            i0 + f0 + 127 + __ldg(&a.dir.offs[a.K - 1].x) < a.n_in;
        auto fetch = [&](int k0, float (&w)[U][4], int (&col)[U]) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool on = k0 + u < a.K;
                const int k = on ? k0 + u : 0;
                const int2 o = __ldg(&a.dir.offs[k]);
                col[u] = __ldg(cols + k);
                const T* vp = vals + (long long)o.y * a.stride + (TRANS ? o.x : 0) + i;
                if (inside) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) w[u][r] = to_f(__ldg(vp + 32 * r));
                    continue;
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int ir = i + 32 * r;
                    w[u][r] = on && ir < a.n_out && (unsigned)(ir + o.x) < (unsigned)a.n_in
                                  ? to_f(vp[32 * r]) : 0.0f;
                }
            }
        };
        auto work = [&](const float (&w)[U][4], const int (&col)[U], int n) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u >= n) break;
                const IN* p = xw + col[u] + f;
#pragma unroll
                for (int t = 0; t < kTileRows; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[t][r] = fmaf(w[u][r], to_f(p[t * pitch + 32 * r]), acc[t][r]);
            }
        };
        float w[U][4], wn[U][4];
        int col[U], cn[U];
        fetch(0, w, col);
        for (int k = 0; k < a.K; k += 2 * U) {
            fetch(k + U, wn, cn);
            work(w, col, a.K - k);
            if (k + U >= a.K) break;
            fetch(k + 2 * U, w, col);
            work(wn, cn, a.K - k - U);
        }
    }
    float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!TRANS && a.bias)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (i + STEP * r < a.n_out)
                bias[r] = to_f(((const T*)a.bias)[(long long)rg.e * a.n_out + i + STEP * r]);
    /* a lane's four features in one access, where they are adjacent and aligned */
    auto quad = [&](const void* p, long long ld) {
        return QUADS && i + 4 <= a.n_out && (uintptr_t)p % (4 * sizeof(T)) == 0 && ld % 4 == 0;
    };
    const bool vo = quad(a.out, a.ldo), vz = quad(a.z, a.ldz), vr = quad(a.res, a.ldr);
    auto store = [&](void* base, long long at, float4 v, bool vec) {
        T* p = (T*)base + at;
        if (vec) {
            store4(p, v);
            return;
        }
        if (i < a.n_out) p[0] = from_f<T>(v.x);
        if (i + STEP < a.n_out) p[STEP] = from_f<T>(v.y);
        if (i + 2 * STEP < a.n_out) p[2 * STEP] = from_f<T>(v.z);
        if (i + 3 * STEP < a.n_out) p[3 * STEP] = from_f<T>(v.w);
    };
#pragma unroll
    for (int t = 0; t < kTileRows; ++t) {
        if (t >= live) break;
        const long long row = (long long)rg.r0 + t0 + t;
        float4 y = make_float4(acc[t][0] + bias[0], acc[t][1] + bias[1], acc[t][2] + bias[2],
                               acc[t][3] + bias[3]);
        if (!TRANS) {
            if (a.z) store(a.z, row * a.ldz + i, y, vz);
            if (a.act != DIA_ACT_NONE) y = act4(a.act, y);
            if (a.res) {
                const T* p = (const T*)a.res + row * a.ldr + i;
                float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (vr) {
                    r = load4<T>(p);
                } else {
                    if (i < a.n_out) r.x = to_f(p[0]);
                    if (i + STEP < a.n_out) r.y = to_f(p[STEP]);
                    if (i + 2 * STEP < a.n_out) r.z = to_f(p[2 * STEP]);
                    if (i + 3 * STEP < a.n_out) r.w = to_f(p[3 * STEP]);
                }
                y.x += r.x;
                y.y += r.y;
                y.z += r.z;
                y.w += r.w;
            }
        }
        store(a.out, row * a.ldo + i, y, vo);
    }
}

/* ------------------------------------------------- gradient of the diagonals
 *
 * A CTA takes 128 features, one window of diagonals (at most 64) and one part
 * of an expert's rows, `rows` of them at a time by way of shared memory, the
 * next ones on their way meanwhile; a warp keeps the sums of its eight
 * diagonals at its lanes' four features.  Sums of an expert with one part go
 * out at once, others to `part`.  A product costs a read of shared memory, which
 * bounds it (load and store unit 58 % busy, instructions issued in 51 % of the
 * cycles): 511 rows of 4096 under 33 diagonals, fp32, 30 us. */
constexpr int kGradSmem = 160 * 1024;     /* two buffers of at least eight rows */

template <typename T, typename DZ, bool VEC, int ND>
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
    /* a buffer: x, then dz [row][128] */
    const int xbytes = rows * pitch * (int)sizeof(T), buf = xbytes + rows * 128 * (int)sizeof(DZ);
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
            unsigned char* xs = smem_raw + which * buf;
            if (nt > 0) {
                if (diags)
                    stage_spans<T, VEC>((T*)xs, pitch, a.dir.wspans, win.s0, win.s1,
                                        (const T*)a.x + t0 * a.ldx, a.ldx, f0, a.n_cols, nt, nt);
                stage_spans<DZ, VEC>((DZ*)(xs + xbytes), 128, a.dir.tile_span, 0, 1,
                                     (const DZ*)a.dz + t0 * a.lddz, a.lddz, f0, a.n_rows, nt, nt);
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
            const T* xs = (const T*)(smem_raw + which * buf);
            const DZ* ds = (const DZ*)(smem_raw + which * buf + xbytes);
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

/* Sums the parts of experts that have several, in the parts' order, so that
 * the bits do not depend on which CTA was first; four columns a thread (129
 * diagonals of 4096, four parts: 8.5 MB in 4 to 7 us). */
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

/* eight elements, p aligned to 16 bytes */
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8])
{
    __align__(16) T r[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) r[c] = from_f<T>(v[c]);
#pragma unroll
    for (int c = 0; c < (int)(8 * sizeof(T)); c += 16)
        *(uint4*)((char*)p + c) = *(const uint4*)((const char*)r + c);
}

/* dz = dy * act'(z) in one of its forms (DzForm).  Eight elements a thread at a
 * time, two of them in flight; rows of dz are padded to eight. */
template <typename T, int ACT, DzForm FORM, bool VEC>
__global__ void __launch_bounds__(256)
spmm_dz_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ z, long long ldz,
               void* __restrict__ dz, void* __restrict__ lo, long long lddz, int M, int n)
{
    dependents_begin();
    const int per = (n + 7) / 8;
    const long long total = (long long)per * M, step = gridDim.x * 256ll;
    for (long long p0 = blockIdx.x * 256ll + threadIdx.x; p0 < total; p0 += 2 * step) {
        float a[2][8], b[2][8];
        long long at[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long p = p0 + h * step;
            const long long t = p < total ? p / per : 0;
            const int i = (int)(p - t * per) * 8;
            at[h] = p < total ? t * lddz + i : -1;
            if (at[h] < 0) continue;
            if (VEC && i + 8 <= n) {
                load8<T>(dy + t * lddy + i, a[h]);
                if (ACT != DIA_ACT_NONE) load8<T>(z + t * ldz + i, b[h]);
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    a[h][c] = i + c < n ? to_f(dy[t * lddy + i + c]) : 0.0f;
                    if (ACT != DIA_ACT_NONE)
                        b[h][c] = i + c < n ? to_f(z[t * ldz + i + c]) : 0.0f;
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (at[h] < 0) continue;
            float v[8];
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
                float2 d = make_float2(1.0f, 1.0f);
                if (ACT != DIA_ACT_NONE)
                    d = sizeof(T) == 2
                            ? dact2<ACT>(make_float2(b[h][c], b[h][c + 1]))
                            : make_float2(dact_of<ACT>(b[h][c]), dact_of<ACT>(b[h][c + 1]));
                v[c] = a[h][c] * d.x;
                v[c + 1] = a[h][c + 1] * d.y;
            }
            if constexpr (FORM == kDzF32) {
                store8<float>((float*)dz + at[h], v);
            } else if constexpr (FORM == kDzSame) {
                store8<T>((T*)dz + at[h], v);
            } else {
                uint32_t hi[4], rest[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    hi[c] = pack2_finite<T>(v[2 * c], v[2 * c + 1]);
                    const float2 w = unpack2<T>(hi[c]);
                    rest[c] = pack2<T>(v[2 * c] - w.x, v[2 * c + 1] - w.y);
                }
                *(uint4*)((T*)dz + at[h]) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *(uint4*)((T*)lo + at[h]) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
            }
        }
    }
    dependency_wait();
}

/* ---------------------------------------------------------------- host */

template <typename T>
static bool vec16(const void* p, long long ld)
{
    return (uintptr_t)p % 16 == 0 && ld * (long long)sizeof(T) % 16 == 0;
}

template <typename T, typename IN, bool TRANS, int TT>
static int launch_few(const ProdArgs& a, cudaStream_t stream)
{
    const int ftiles = (a.n_out + 31) / 32;
    const long long ngroups = a.seg ? a.M / TT + std::min(a.E, a.M) : (a.M + TT - 1) / TT;
    /* warps that share a tile: until every SM has a CTA (two where a warp has
     * one row), or a warp four diagonals (32 rows of 4096 under 129 diagonals,
     * bf16: 28 us; with twice the CTAs 38; the rule gives that call to the
     * tensor cores, 11 us) */
    const long long warps = TT == 1 ? 2 * kFewWarps : kFewWarps;
    int ks = 1;
    while (ks < kFewWarps && ftiles * ngroups * ks < warps * num_sms() && a.K > 4 * ks) ks *= 2;
    const int fper = kFewWarps / ks;
    const long long grid = ngroups * ((ftiles + fper - 1) / fper);
    if (grid > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm: block too large");
    /* the larger of block and operator is streamed once, the other stays in L2 */
    const bool rows_first = (long long)a.M * a.n_in < a.stride * a.K;
    DIA_TRY_CUDA(launch(false, spmm_few_kernel<T, IN, TRANS, TT>, (int)grid, kFewWarps * 32, 0, stream,
                        a, ks, ftiles, ngroups, rows_first));
    return DIA_OK;
}

template <typename T, typename IN, bool TRANS, bool VEC, bool QUADS>
static int launch_tile_as(const ProdArgs& a, int shape, int smem, cudaStream_t stream)
{
    const int F = kTileF[shape], rows = kTileWarps * kTileRows * 128 / F;
    const int ftiles = (a.n_out + F - 1) / F;
    const long long ngroups = a.seg ? a.M / rows + std::min(a.E, a.M) : (a.M + rows - 1) / rows;
    if (ngroups * ftiles > INT_MAX)
        return fail(DIA_ERR_UNSUPPORTED, "dia_spmm: block too large");
    const bool rows_first = (long long)a.M * a.n_in < a.stride * a.K;
    const auto kernel = spmm_tile_kernel<T, IN, TRANS, VEC, QUADS>;
    static SmemRecord most;
    DIA_TRY_CUDA(allow_smem(kernel, kTileSmem, most));
    DIA_TRY_CUDA(launch(false, kernel, (int)(ngroups * ftiles), kTileWarps * 32, smem, stream, a,
                        shape, ftiles, ngroups, rows_first));
    return DIA_OK;
}

static int tile_smem(const SpmmDir& d, int shape, size_t elem)
{
    return (int)std::min<long long>(INT_MAX, (long long)kTileWarps * kTileRows * 128 /
                                                 kTileF[shape] * d.width[shape] * (long long)elem);
}

template <typename T, typename IN, bool TRANS>
static int launch_cores(const ProdArgs& a, cudaStream_t stream)
{
    const int per = a.M / std::max(a.E, 1);   /* rows of a usual expert */
    /* below this there are too few warps of 128 features x 8 rows to hide the
     * latency of the diagonals one after the other (4096 x 4096, 129 diagonals,
     * bf16 in this form: 57 us from 64 rows to 256; by few rows 28 at 32 rows, in
     * proportion beyond).  Operators whose inputs fit no tile have no other
     * kernel than the few rows' (fp32 27-point stencil, 64 rows: 0.25 us a
     * million products on 64^3 and 76^3, 0.77 on 80^3 to 128^3) */
    if (per >= 8 && a.K > 0 && (long long)a.M * a.n_out >= 196608) {
        /* the widest tile (an input is read again by fewer tiles) whose inputs
         * fit and that leaves a CTA for every SM; else the narrowest that fits */
        int shape = 2;
        auto fits = [&](int s) { return tile_smem(a.dir, s, sizeof(IN)) <= kTileSmem; };
        auto ctas = [&](int s) {
            const int rows = kTileWarps * kTileRows * 128 / kTileF[s];
            return (long long)((a.n_out + kTileF[s] - 1) / kTileF[s]) * ((a.M + rows - 1) / rows);
        };
        while (shape >= 0 && !(fits(shape) && ctas(shape) >= num_sms())) --shape;
        if (shape < 0)
            for (shape = 0; shape < 3 && !fits(shape);) ++shape;
        if (shape < 3) {
            const int smem = tile_smem(a.dir, shape, sizeof(IN));
            const bool vec = vec16<IN>(a.in, a.ldi), quads = 3 * a.dir.nquads <= a.K;
            if (vec)
                return quads ? launch_tile_as<T, IN, TRANS, true, true>(a, shape, smem, stream)
                             : launch_tile_as<T, IN, TRANS, true, false>(a, shape, smem, stream);
            return quads ? launch_tile_as<T, IN, TRANS, false, true>(a, shape, smem, stream)
                         : launch_tile_as<T, IN, TRANS, false, false>(a, shape, smem, stream);
        }
    }
    if (per >= 5) return launch_few<T, IN, TRANS, 8>(a, stream);
    return per >= 2 ? launch_few<T, IN, TRANS, 4>(a, stream)
                    : launch_few<T, IN, TRANS, 1>(a, stream);
}

template <typename T>
int Cores<T>::product(const ProdArgs& a, cudaStream_t stream)
{
    if (!a.trans) return launch_cores<T, T, false>(a, stream);
    return a.in32 ? launch_cores<T, float, true>(a, stream) : launch_cores<T, T, true>(a, stream);
}

template <typename T, int ACT, DzForm FORM>
static cudaError_t launch_dz_act(const void* dy, long long lddy, const void* z, long long ldz,
                                 void* dz, void* lo, long long lddz, int M, int n, bool dependent,
                                 cudaStream_t stream)
{
    const long long work = (long long)M * ((n + 7) / 8);
    const int grid = (int)std::min<long long>((work + 511) / 512, 8ll * num_sms());
    const auto kernel = vec16<T>(dy, lddy) && vec16<T>(z, ldz)
                            ? spmm_dz_kernel<T, ACT, FORM, true>
                            : spmm_dz_kernel<T, ACT, FORM, false>;
    return launch(dependent, kernel, grid, 256, 0, stream, (const T*)dy, lddy, (const T*)z, ldz,
                  dz, lo, lddz, M, n);
}

template <typename T>
int Cores<T>::dz(DzForm form, int act, const void* dy, long long lddy, const void* z,
                 long long ldz, void* dz, void* lo, long long lddz, int M, int n, bool dependent,
                 cudaStream_t stream)
{
    if (M == 0 || n == 0) return DIA_OK;
    constexpr DzForm F32 = kDzF32, PAIR = sizeof(T) == 2 ? kDzPair : kDzF32;
    const bool pair = form == kDzPair;
    const auto run =
        act == DIA_ACT_NONE   ? launch_dz_act<T, DIA_ACT_NONE, kDzSame>
        : act == DIA_ACT_RELU ? (pair ? launch_dz_act<T, DIA_ACT_RELU, PAIR>
                                      : launch_dz_act<T, DIA_ACT_RELU, F32>)
        : act == DIA_ACT_SILU ? (pair ? launch_dz_act<T, DIA_ACT_SILU, PAIR>
                                      : launch_dz_act<T, DIA_ACT_SILU, F32>)
        : act == DIA_ACT_GELU ? (pair ? launch_dz_act<T, DIA_ACT_GELU, PAIR>
                                      : launch_dz_act<T, DIA_ACT_GELU, F32>)
                              : (pair ? launch_dz_act<T, DIA_ACT_GELU_TANH, PAIR>
                                      : launch_dz_act<T, DIA_ACT_GELU_TANH, F32>);
    DIA_TRY_CUDA(run(dy, lddy, z, ldz, dz, lo, lddz, M, n, dependent, stream));
    return DIA_OK;
}

template <typename T, typename DZ>
static int launch_gradient(const GradArgs& a, cudaStream_t stream)
{
    const int ftiles = (int)((a.stride + 127) / 128);
    const int nwins = a.dvals ? std::max(a.dir.nwins, 1) : 1;
    const long long parts = a.seg ? a.M / a.per + a.E : std::max(1, (a.M + a.per - 1) / a.per);
    const long long grid = parts * ftiles * nwins;
    if (grid > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm_backward: block too large");
    /* rows a stage: two CTAs an SM where that leaves eight or more */
    const int row_bytes =
        2 * ((a.dvals ? a.dir.wwidth : 0) * (int)sizeof(T) + 128 * (int)sizeof(DZ));
    const int rows = std::min(32, std::max(8, 100 * 1024 / row_bytes / 8 * 8));
    const int smem = rows * row_bytes;
    const bool vec = vec16<DZ>(a.dz, a.lddz) && vec16<T>(a.x, a.ldx);
    const int nd = a.dvals ? (a.dir.wdiags + kTileWarps - 1) / kTileWarps : 1;
    const int pick = nd <= 1 ? 0 : nd <= 2 ? 1 : nd <= 3 ? 2 : nd <= 5 ? 3 : 4;
    using Kernel = void (*)(GradArgs, int, int, int);
    static const Kernel kernels[2][5] = {
        {spmm_grad_kernel<T, DZ, false, 1>, spmm_grad_kernel<T, DZ, false, 2>,
         spmm_grad_kernel<T, DZ, false, 3>, spmm_grad_kernel<T, DZ, false, 5>,
         spmm_grad_kernel<T, DZ, false, 8>},
        {spmm_grad_kernel<T, DZ, true, 1>, spmm_grad_kernel<T, DZ, true, 2>,
         spmm_grad_kernel<T, DZ, true, 3>, spmm_grad_kernel<T, DZ, true, 5>,
         spmm_grad_kernel<T, DZ, true, 8>}};
    const Kernel kernel = kernels[vec][pick];
    static SmemRecord most[2][5];
    DIA_TRY_CUDA(allow_smem(kernel, kGradSmem, most[vec][pick]));
    DIA_TRY_CUDA(launch(false, kernel, (int)grid, kTileWarps * 32, smem, stream, a, ftiles, nwins,
                        rows));
    return DIA_OK;
}

template <typename T>
int Cores<T>::gradient(const GradArgs& a, cudaStream_t stream)
{
    return a.dz32 ? launch_gradient<T, float>(a, stream) : launch_gradient<T, T>(a, stream);
}

template <typename T>
int Cores<T>::join(const GradArgs& a, cudaStream_t stream)
{
    if (a.M <= a.per) return DIA_OK;   /* no expert has several parts */
    const int cblocks = (int)((a.stride + 511) / 512);
    const long long grid = (long long)a.E * (a.K + 1) * cblocks;
    if (grid > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm_backward: block too large");
    DIA_TRY_CUDA(launch(true, spmm_join_kernel<T>, (int)grid, 128, 0, stream, a, cblocks));
    return DIA_OK;
}

}  // namespace dia
