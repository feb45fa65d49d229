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

constexpr int kMmWarps = 8;
constexpr int kMmThreads = kMmWarps * 32;
constexpr int kMmFeat = 128;   /* features of a warp: four per lane */

/* elements c .. c+3 of a row of n elements, zero outside */
template <typename T, bool VEC>
__device__ __forceinline__ float4 row4(const T* row, int c, int n)
{
    if (VEC && c >= 0 && c + 4 <= n) return load4<T>(row + c);
    float4 v;
    v.x = (unsigned)c < (unsigned)n ? to_f(row[c]) : 0.0f;
    v.y = (unsigned)(c + 1) < (unsigned)n ? to_f(row[c + 1]) : 0.0f;
    v.z = (unsigned)(c + 2) < (unsigned)n ? to_f(row[c + 2]) : 0.0f;
    v.w = (unsigned)(c + 3) < (unsigned)n ? to_f(row[c + 3]) : 0.0f;
    return v;
}

/* One warp: 128 features (four consecutive ones a lane), TT rows.  A quad's
 * up to four diagonals read the window of seven inputs from two aligned
 * chunks of four, so a run of consecutive offsets costs one chunk per four
 * diagonals; a weight is read once for TT rows.  The CTA's warps split the
 * quads `ks` ways (few rows: there are too few warps otherwise) and add up
 * in shared memory in a fixed order; the other 8 / ks take other features. */
template <typename T, bool TRANS, int TT, bool VEC>
__global__ void __launch_bounds__(kMmThreads)
spmm_kernel(ProdArgs a, int ks, int ftiles, long long ngroups, bool rows_first)
{
    __shared__ float s_sum[kMmWarps][TT * 4][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = warp % ks, sub = warp / ks, fper = kMmWarps / ks;
    const int fblocks = (ftiles + fper - 1) / fper;
    const long long b = blockIdx.x;
    const long long g = rows_first ? b % ngroups : b / fblocks;
    const int fb = (int)(rows_first ? b / ngroups : b % fblocks);
    const RowGroup rg = row_group(a.seg, a.E, a.M, TT, g, false);
    const int i = (fb * fper + sub) * kMmFeat + lane * 4;

    float acc[TT][4];
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][r] = 0.0f;

    if (rg.e >= 0 && i < a.n_out) {
        const T* vals = (const T*)a.vals + rg.e * a.estride;
        const T* in = (const T*)a.in + (long long)rg.r0 * a.ldi;
        const int nt = rg.r1 - rg.r0;
        const int q0 = (int)((long long)a.dir.nquads * part / ks);
        const int q1 = (int)((long long)a.dir.nquads * (part + 1) / ks);
        for (int q = q0; q < q1; ++q) {
            const int4 h = __ldg((const int4*)&a.dir.quads[q]);
            const int k3 = __ldg(&a.dir.quads[q].k[3]);
            const int kk[4] = {h.y, h.z, h.w, k3};
            const int c = i + h.x;
            if (c + 7 <= 0 || c >= a.n_in) continue;
            float w[4][4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (kk[s] < 0) continue;
                const T* vp = vals + (long long)kk[s] * a.stride;
                if (TRANS) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = c + s + r;
                        w[s][r] = ((unsigned)j < (unsigned)a.n_in && i + r < a.n_out)
                                      ? to_f(vp[j]) : 0.0f;
                    }
                } else {
                    const float4 v = load4<T>(vp + i);
                    w[s][0] = v.x;
                    w[s][1] = v.y;
                    w[s][2] = v.z;
                    w[s][3] = v.w;
                    if (c < 0 || c + 7 > a.n_in) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if ((unsigned)(c + s + r) >= (unsigned)a.n_in) w[s][r] = 0.0f;
                    }
                }
            }
            float xs[TT][8];
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                if (t < nt) {
                    const T* row = in + t * a.ldi;
                    const float4 u = row4<T, VEC>(row, c, a.n_in);
                    const float4 v = row4<T, VEC>(row, c + 4, a.n_in);
                    xs[t][0] = u.x; xs[t][1] = u.y; xs[t][2] = u.z; xs[t][3] = u.w;
                    xs[t][4] = v.x; xs[t][5] = v.y; xs[t][6] = v.z; xs[t][7] = v.w;
                } else {
#pragma unroll
                    for (int r = 0; r < 8; ++r) xs[t][r] = 0.0f;
                }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (kk[s] < 0) continue;
#pragma unroll
                for (int t = 0; t < TT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[t][r] = fmaf(w[s][r], xs[t][s + r], acc[t][r]);
            }
        }
    }
    if (ks > 1) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s_sum[warp][t * 4 + r][lane] = acc[t][r];
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v = acc[t][r];
                for (int p = 1; p < ks; ++p) v += s_sum[warp + p][t * 4 + r][lane];
                acc[t][r] = v;
            }
    }
    if (rg.e < 0 || i >= a.n_out) return;
    const T* bias = a.bias ? (const T*)a.bias + (long long)rg.e * a.n_out : nullptr;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        const long long row = (long long)rg.r0 + t;
        if (row >= rg.r1) break;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (i + r >= a.n_out) break;
            float z = acc[t][r];
            if (bias) z += to_f(bias[i + r]);
            if (a.z) ((T*)a.z)[row * a.ldz + i + r] = from_f<T>(z);
            float y = act_any(a.act, z);
            if (a.res) y += to_f(((const T*)a.res)[row * a.ldr + i + r]);
            ((T*)a.out)[row * a.ldo + i + r] = from_f<T>(y);
        }
    }
}

/* One CTA: 128 features, one quad, one part of an expert's rows; its warps
 * take every eighth row and add up in shared memory in a fixed order.  Sums
 * of an expert with one part go out at once, others to `part`. */
template <typename T, bool VEC>
__global__ void __launch_bounds__(kMmThreads)
spmm_grad_kernel(GradArgs a, int ftiles)
{
    __shared__ float s_sum[kMmWarps][20][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nq = max(a.dir.nquads, 1);
    const long long b = blockIdx.x;
    const int f = (int)(b % ftiles), q = (int)((b / ftiles) % nq);
    const RowGroup rg = row_group(a.seg, a.E, a.M, a.per, b / ftiles / nq, true);
    if (rg.e < 0 || (rg.nparts > 1 && rg.slot + rg.part >= a.slots)) return;
    const int i = f * kMmFeat + lane * 4;
    const bool on = i < a.n_rows;
    int kk[4] = {-1, -1, -1, -1}, base = 0;
    if (q < a.dir.nquads && a.dvals) {
        base = a.dir.quads[q].base;
#pragma unroll
        for (int s = 0; s < 4; ++s) kk[s] = a.dir.quads[q].k[s];
    }
    const int c = i + base;
    float acc[4][4], sb[4] = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[s][r] = 0.0f;
    if (on) {
        for (int t = rg.r0 + warp; t < rg.r1; t += kMmWarps) {
            const float4 d = row4<T, VEC>((const T*)a.dz + t * a.lddz, i, a.n_rows);
            const T* row = (const T*)a.x + t * a.ldx;
            const float4 u = row4<T, VEC>(row, c, a.n_cols);
            const float4 v = row4<T, VEC>(row, c + 4, a.n_cols);
            const float dd[4] = {d.x, d.y, d.z, d.w};
            const float xs[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
            for (int s = 0; s < 4; ++s)
                if (kk[s] >= 0)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[s][r] = fmaf(dd[r], xs[s + r], acc[s][r]);
#pragma unroll
            for (int r = 0; r < 4; ++r) sb[r] += dd[r];
        }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_sum[warp][s * 4 + r][lane] = acc[s][r];
#pragma unroll
    for (int r = 0; r < 4; ++r) s_sum[warp][16 + r][lane] = sb[r];
    __syncthreads();
    /* output s * 128 + f: slot s (4: dbias) of feature f */
    for (int o = threadIdx.x; o < 5 * kMmFeat; o += kMmThreads) {
        const int s = o / kMmFeat, fi = o % kMmFeat, col = f * kMmFeat + fi;
        if (col >= a.stride) continue;
        float v = 0.0f;
        for (int w = 0; w < kMmWarps; ++w) v += s_sum[w][s * 4 + (fi & 3)][fi >> 2];
        if (s == 4) {
            if (q != 0 || !a.dbias || col >= a.n_rows) continue;
            if (rg.nparts > 1)
                a.part[((long long)(rg.slot + rg.part) * (a.K + 1) + a.K) * a.stride + col] = v;
            else
                ((T*)a.dbias)[(long long)rg.e * a.n_rows + col] = from_f<T>(v);
        } else if (kk[s] >= 0) {
            /* an entry outside the matrix has no gradient */
            if (col >= a.n_rows || (unsigned)(col + base + s) >= (unsigned)a.n_cols) v = 0.0f;
            if (rg.nparts > 1)
                a.part[((long long)(rg.slot + rg.part) * (a.K + 1) + kk[s]) * a.stride + col] = v;
            else
                ((T*)a.dvals)[rg.e * a.estride + (long long)kk[s] * a.stride + col] = from_f<T>(v);
        }
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

static bool vec4(const void* p, long long ld, int dtype)
{
    return (uintptr_t)p % (4 * elem_size(dtype)) == 0 && ld % 4 == 0;
}

template <typename T, bool TRANS, int TT>
static int launch_product_tt(const ProdArgs& a, int dtype, cudaStream_t stream)
{
    const int ftiles = (a.n_out + kMmFeat - 1) / kMmFeat;
    const long long ngroups =
        a.seg ? a.M / TT + std::min(a.E, a.M) : (a.M + TT - 1) / TT;
    /* warps that share a tile: enough to give every SM a few */
    int ks = 1;
    while (ks < kMmWarps && (long long)ftiles * ngroups * ks < 8ll * num_sms() &&
           a.dir.nquads > 2 * ks)
        ks *= 2;
    const int fper = kMmWarps / ks;
    const long long grid = ngroups * ((ftiles + fper - 1) / fper);
    if (grid > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm: block too large");
    /* the larger of block and operator is streamed once, the other stays in L2 */
    const bool rows_first = (long long)a.M * a.n_in < a.stride * 4 * a.dir.nquads;
    if (vec4(a.in, a.ldi, dtype))
        spmm_kernel<T, TRANS, TT, true>
            <<<(unsigned)grid, kMmThreads, 0, stream>>>(a, ks, ftiles, ngroups, rows_first);
    else
        spmm_kernel<T, TRANS, TT, false>
            <<<(unsigned)grid, kMmThreads, 0, stream>>>(a, ks, ftiles, ngroups, rows_first);
    DIA_TRY_CUDA(cudaGetLastError());
    return DIA_OK;
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
    const int per = a.M / std::max(a.E, 1);   /* rows of a usual expert */
    if (a.trans)
        return per >= 4 ? launch_product_tt<T, true, 4>(a, dtype, stream)
                        : launch_product_tt<T, true, 1>(a, dtype, stream);
    return per >= 4 ? launch_product_tt<T, false, 4>(a, dtype, stream)
                    : launch_product_tt<T, false, 1>(a, dtype, stream);
}

static bool vec16(const void* p, long long ld, int dtype)
{
    return (uintptr_t)p % 16 == 0 && ld * (long long)elem_size(dtype) % 16 == 0;
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
    const long long tiles = std::max<long long>(1, (stride + kMmFeat - 1) / kMmFeat) *
                            std::max(1, p->fwd.nquads);
    const long long want = std::max<long long>(1, 4ll * num_sms() / tiles);
    const long long per = std::max<long long>(256, (M + want - 1) / want);
    return (int)std::min<long long>(per, INT_MAX / 2);
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
    const int ftiles = (int)((a.stride + kMmFeat - 1) / kMmFeat);
    const long long parts = a.seg ? a.M / a.per + a.E : std::max(1, (a.M + a.per - 1) / a.per);
    const long long grid = parts * ftiles * std::max(a.dir.nquads, 1);
    if (grid > INT_MAX) return fail(DIA_ERR_UNSUPPORTED, "dia_spmm_backward: block too large");
    if (vec4(a.dz, a.lddz, dtype) && vec4(a.x, a.ldx, dtype))
        spmm_grad_kernel<T, true><<<(unsigned)grid, kMmThreads, 0, stream>>>(a, ftiles);
    else
        spmm_grad_kernel<T, false><<<(unsigned)grid, kMmThreads, 0, stream>>>(a, ftiles);
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

static std::vector<Quad> build_quads(const std::vector<int2>& s)
{
    std::vector<Quad> quads;
    for (const int2& o : s) {
        const int base = o.x & ~3;   /* floor to a multiple of four */
        if (quads.empty() || quads.back().base != base) {
            Quad q;
            std::memset(&q, 0, sizeof(q));
            q.base = base;
            q.k[0] = q.k[1] = q.k[2] = q.k[3] = -1;
            quads.push_back(q);
        }
        quads.back().k[o.x - base] = o.y;
    }
    return quads;
}

/* One direction's tables appended to `blob`; offsets into it, made pointers
 * once the blob is on the device. */
struct DirTables {
    size_t quads, boxes, offs;
    int nquads, nboxes;
};

template <typename T>
static size_t append(std::vector<char>& blob, const std::vector<T>& v)
{
    const size_t at = (blob.size() + 31) / 32 * 32;
    blob.resize(at + v.size() * sizeof(T));
    if (!v.empty()) std::memcpy(blob.data() + at, v.data(), v.size() * sizeof(T));
    return at;
}

static DirTables append_dir(std::vector<char>& blob, const std::vector<int>& off)
{
    const std::vector<int2> s = sorted_offsets(off);
    const std::vector<Quad> q = build_quads(s);
    const std::vector<Box> b = build_boxes(s);
    DirTables t;
    t.nquads = (int)q.size();
    t.nboxes = (int)b.size();
    t.quads = append(blob, q);
    t.boxes = append(blob, b);
    t.offs = append(blob, s);
    return t;
}

static SpmmDir dir_on_device(const void* blob, const DirTables& t)
{
    const char* p = (const char*)blob;
    return SpmmDir{(const Quad*)(p + t.quads), (const Box*)(p + t.boxes),
                   (const int2*)(p + t.offs), t.nquads, t.nboxes};
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
        const DirTables tf = append_dir(blob, fwd), tt = append_dir(blob, trn);
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
        if (!a.dvals) {   /* dbias alone: x is not looked at */
            a.dir.nquads = 0;
            a.n_cols = 0;
        }
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
