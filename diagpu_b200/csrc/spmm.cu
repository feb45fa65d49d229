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
 * held in fp32, in an order that the sizes and the form fix (the same bits on
 * every run), and rounded once to the block's type; dz is held in 32 bits.
 * Grouped: the rows are sorted by expert, rows [seg[e],
 * seg[e+1]) use the diagonals vals[e].
 */
#include <algorithm>
#include <atomic>
#include <climits>
#include <cstring>
#include <new>
#include <vector>

#include "dia_core.cuh"
#include "spmm.cuh"

namespace dia {

/* test hook (dia_test_spmm_form): 0 the rule, 1 CUDA cores, 2 tensor cores
 * wherever they can run */
static std::atomic<int> g_form{0};

/* Which form a call takes: the one whose time, by the measured costs of both,
 * is shorter (16-bit types, one B200; over 174 calls of 8 to 4096 rows, 3 to
 * 129 diagonals, 1 to 64 experts the form taken is 1.4 % slower than the better
 * one on average, 43 % at worst).
 *
 * CUDA cores, us.  Few rows: 6, and 4 for every million (row, feature, group of
 * four offsets).  Many: a wave of CTAs takes 10 + 0.4 K, then every million
 * features 4.5 + 0.2 K.
 * Tensor cores: the operator's boxes are packed and read (4 ns each, 10 where
 * they no longer fit L2) and every tile has a way through the kernel; a packing
 * launch of its own 2.5 us, one that makes dz 8.
 * 4096 x 129 diagonals: cores 57 us, tensor cores 12 at 64 rows; 27-point
 * stencil on 262144: 26 and 324 at 8 rows, 306 and 374 at 128.  The ratio of the
 * gradients is near that of the products (65536, 33 scattered diagonals, 128
 * rows: 97 and 107, gradients 179 and 237). */
static bool tensor_form(const DiaSpmmPlan* p, int dtype, long long M, int E, bool backward)
{
    const int form = g_form.load(std::memory_order_relaxed);
    const SpmmDir& d = p->fwd;
    if (dtype == DIA_F32 || d.nboxes == 0 || p->n_rows == 0 || p->n_cols == 0 || form == 1)
        return false;
    if (form == 2) return true;
    if (M < 8) return false;   /* the cores' time does not grow up to there */
    /* The packed operator takes 16 KB a box, for a few scattered diagonals up to
     * fifty times the diagonals themselves (27-point stencil on 128^3: 5.6 GB),
     * and a caller may lack the room: it takes no more than the block and its
     * result do, or 2 GB. */
    const double block = 2.0 * M * ((double)p->n_rows + p->n_cols);
    const long long pack = backward ? spmm_tc_pack_bytes(p->trn, p->K, p->n_cols, M, E)
                                    : spmm_tc_pack_bytes(d, p->K, p->n_rows, M, E);
    if ((double)pack > std::max(block, 2147483648.0)) return false;
    const double nfb = (p->n_rows + 127) / 128, boxes = nfb * E * d.nboxes;
    const double tiles = nfb * (M / 128.0 + (E > 1 ? (double)std::min<long long>(E, M) : 1.0));
    const double mega = (double)M * p->n_rows * 1e-6;
    const double cores = mega < 0.2 ? 6 + 4 * mega * d.nquads
                                    : std::max(10 + 0.4 * p->K, (4.5 + 0.2 * p->K) * mega);
    const double tensor = 8 + (E > 1 || d.nboxes > 6 ? 2.5 : 0.0) + 0.004 * boxes +
                          0.006 * std::max(0.0, boxes - 2500) + 0.02 * tiles +
                          (backward && d.nboxes > 4 ? 8.0 : 0.0);
    return (backward ? 1.1 : 1.0) * cores > tensor;
}

static size_t elem_size(int dtype) { return dtype == DIA_F32 ? 4 : 2; }

/* the tensor-core form it is (its operator has to be packed first) */
static bool product_on_tc(const ProdArgs& a, bool tensor)
{
    return a.M > 0 && a.n_out > 0 && a.n_in > 0 && tensor && spmm_tc_block(a.in, a.ldi);
}

template <typename T>
static int launch_product(const ProdArgs& a, int dtype, bool tensor, cudaStream_t stream)
{
    if (a.M == 0 || a.n_out == 0) return DIA_OK;
    if (product_on_tc(a, tensor)) return spmm_tc_product(a, dtype, stream);
    return Cores<T>::product(a, stream);
}

/* rows of a part of the gradient's sum: enough parts to fill the GPU, none
 * so short that writing and joining its sums costs more than it saves */
static int grad_part_rows(const DiaSpmmPlan* p, bool tensor, long long M, int E, long long stride)
{
    if (tensor) {
        /* one CTA an SM; an expert's last part is half full on average (8
         * experts, 4096 rows, 2048 features: 56 us at 704 rows a part, 61 at
         * 384, 74 at 2048) */
        const long long tiles = std::max<long long>(1, (stride + 127) / 128) *
                                ((p->fwd.nboxes + 3) / 4);
        const long long want = std::max<long long>(1, num_sms() / tiles - (E - 1) / 2);
        const long long per = std::max<long long>(256, (M + want - 1) / want);
        return (int)((per + 63) / 64 * 64);
    }
    /* two CTAs an SM, all at once (511 rows of 4096, 33 scattered diagonals,
     * fp32: 53 us against 56 with four); uneven experts want four to share out
     * (16 experts, 4096 rows: 80 against 90) */
    const long long tiles = std::max<long long>(1, (stride + 127) / 128) * std::max(1, p->fwd.nwins);
    const long long want =
        std::max<long long>(1, (E > 1 ? 4ll : 2ll) * num_sms() / tiles - (E - 1));
    const long long per = std::max<long long>(32, (M + want - 1) / want);
    return (int)((per + 7) / 8 * 8);
}

/* parts of experts that have several: at most two a `per` rows */
static long long grad_slots(long long M, long long per) { return M > per ? 2 * (M / per) + 1 : 0; }

static bool grad_on_tc(const GradArgs& a, bool tensor)
{
    return tensor && a.M > 0 && a.n_cols > 0 && a.n_rows > 0 &&
           a.dvals && spmm_tc_block(a.dz, a.lddz) && spmm_tc_block(a.x, a.ldx);
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

/* Plans come and go while other work is captured into a graph (a collected
 * plan of an earlier layer, say); their memory is no part of it.  Without this
 * the runtime refuses cudaMalloc and cudaFree then, and the capture is lost. */
struct BesideCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    BesideCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~BesideCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

/* A device copy of the tables that any stream may read once this returns: a
 * plain cudaMemcpy from pageable memory may return before the copy has reached
 * the device, and streams that do not wait for the default one would read the
 * tables half written. */
static cudaError_t upload(void** dst, const std::vector<char>& blob)
{
    if (blob.empty()) return cudaSuccess;
    BesideCapture beside;
    cudaStream_t s = nullptr;
    cudaError_t e = cudaMalloc(dst, blob.size());
    if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking);
    if (e == cudaSuccess)
        e = cudaMemcpyAsync(*dst, blob.data(), blob.size(), cudaMemcpyHostToDevice, s);
    if (s) {
        const cudaError_t done = cudaStreamSynchronize(s);
        if (e == cudaSuccess) e = done;
        cudaStreamDestroy(s);
    }
    return e;
}

static void release(DiaSpmmPlan* p)
{
    BesideCapture beside;
    if (p->blob && cudaFree(p->blob) != cudaSuccess) cudaGetLastError();
    delete p;
}

/* arguments both directions share; DIA_OK or the error */
static int check_common(const char* who, const DiaSpmmPlan* p, int dtype, int64_t M, int E,
                        const int64_t* seg, int act, int64_t stride, const void* vals)
{
    auto bad = [&](const char* what) {
        return fail(DIA_ERR_INVALID, std::string(who) + ": " + what);
    };
    if (dtype != DIA_F32 && dtype != DIA_F16 && dtype != DIA_BF16) return bad("unknown dtype");
    if (act < DIA_ACT_NONE || act > DIA_ACT_GELU_TANH) return bad("unknown activation");
    if (M < 0 || M > INT_MAX / 2) return bad("bad number of rows");
    if (E < 1 || E > (1 << 20)) return bad("bad number of experts");
    if (E > 1 && !seg) return bad("experts without seg");
    if ((uintptr_t)seg % sizeof(int64_t)) return bad("seg is misaligned");
    if (!p) return bad("null plan");
    int dev = -1;
    DIA_TRY_CUDA(cudaGetDevice(&dev));
    if (dev != p->device) return bad("the plan belongs to another device");
    if (stride < p->n_rows || stride % 32 != 0)
        return bad("stride must be a multiple of 32, at least n_rows");
    if (stride > INT_MAX / 2) return bad("stride too large");
    if (p->K > 0 && p->n_rows > 0 && !vals) return bad("null values");
    if ((uintptr_t)vals % 16) return bad("values must be 16-byte aligned");
    return DIA_OK;
}

/* a block of M rows of n elements: pointer, row stride and element alignment */
static int check_block(const char* who, const char* name, const void* ptr, int64_t ld, int64_t M,
                       int n, int dtype)
{
    auto bad = [&](const char* what) {
        return fail(DIA_ERR_INVALID, std::string(who) + ": " + name + what);
    };
    if (M == 0 || n == 0) return DIA_OK;
    if (!ptr) return bad(" is null");
    if (M > 1 && ld < n) return bad(" has rows shorter than its width");
    if ((uintptr_t)ptr % elem_size(dtype)) return bad(" is misaligned");
    return DIA_OK;
}

/* a vector for each expert, or NULL */
static int check_vector(const char* who, const char* name, const void* ptr, int dtype)
{
    if ((uintptr_t)ptr % elem_size(dtype) == 0) return DIA_OK;
    return fail(DIA_ERR_INVALID, std::string(who) + ": " + name + " is misaligned");
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
static long long pack_bytes(const SpmmDir& d, int K, bool tensor, int64_t M, int E, int n_out)
{
    return M > 0 && n_out > 0 && tensor
               ? align256(spmm_tc_pack_bytes(d, K, n_out, M, E)) : 0;
}

/* a copy of a block whose rows are not multiples of 16 bytes apart, which the
 * tensor-core form reads instead */
static long long copy_bytes(bool tensor, int64_t M, int n, int64_t ld)
{
    return M > 0 && ld % 8 != 0 && tensor ? align256(M * ((n + 7) / 8 * 8) * 2ll) : 0;
}

/* the gradient's workspace: dz (32 bits, where there is an activation, or a
 * copy of dy), sums of parts (where there are several), the operator's boxes, a
 * copy of x */
struct GradPlan {
    int per;
    bool tensor, made;
    long long lddz, dz_bytes, part_bytes, pack_bytes, x_bytes;
    long long bytes() const { return dz_bytes + part_bytes + pack_bytes + x_bytes; }
};

static GradPlan grad_plan(const DiaSpmmPlan* p, int dtype, int64_t M, int E, int64_t ldx,
                          int64_t stride, int64_t lddy, int act)
{
    GradPlan g;
    g.tensor = tensor_form(p, dtype, M, E, true);
    g.per = grad_part_rows(p, g.tensor, M, E, stride);
    g.lddz = (p->n_rows + 7) / 8 * 8;
    g.made = act != DIA_ACT_NONE || copy_bytes(g.tensor, M, p->n_rows, lddy) > 0;
    g.dz_bytes = !g.made ? 0 : align256(M * g.lddz * (act != DIA_ACT_NONE ? 4ll : 2ll));
    g.part_bytes = align256(grad_slots(M, g.per) * (p->K + 1) * stride * 4);
    g.pack_bytes = pack_bytes(p->trn, p->K, g.tensor, M, E, p->n_cols);
    g.x_bytes = copy_bytes(g.tensor, M, p->n_cols, ldx);
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
    if (n_rows > INT_MAX / 2 || n_cols > INT_MAX / 2 - n_rows || num_diags > (1 << 20))
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
        if (e == cudaSuccess) e = upload(&p->blob, blob);
        if (e != cudaSuccess) {
            release(p);
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
    if (plan) release(plan);
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
    if (rc == DIA_OK) rc = check_vector(who, "bias", d_bias, dtype);
    if (rc != DIA_OK) return rc;
    const bool tensor = tensor_form(plan, dtype, M, num_experts, false);
    const long long pack = pack_bytes(plan->fwd, plan->K, tensor, M, num_experts, plan->n_rows);
    const long long copy = copy_bytes(tensor, M, plan->n_cols, ldx);
    const long long need = pack + copy;
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
    return by_type(dtype, [&](auto* t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        int r = DIA_OK;
        if (copy > 0) {
            a.in = (char*)d_work + pack;
            a.ldi = (plan->n_cols + 7) / 8 * 8;
            r = Cores<T>::dz(kDzSame, DIA_ACT_NONE, d_x, ldx, nullptr, 0, (char*)d_work + pack,
                             nullptr, a.ldi, a.M, a.n_in, false, stream);
        }
        if (r == DIA_OK && product_on_tc(a, tensor)) {
            r = spmm_tc_pack(a, false, stream);
            a.dependent = pack > 0;
        }
        return r == DIA_OK ? launch_product<T>(a, dtype, tensor, stream) : r;
    });
}

extern "C" int64_t dia_spmm_workspace(const DiaSpmmPlan* plan, int dtype, int64_t M,
                                      int num_experts, int64_t ldx)
{
    if (!plan || M < 0 || M > INT_MAX / 2 || num_experts < 1) return -1;
    const bool tensor = tensor_form(plan, dtype, M, num_experts, false);
    return pack_bytes(plan->fwd, plan->K, tensor, M, num_experts, plan->n_rows) +
           copy_bytes(tensor, M, plan->n_cols, ldx);
}

extern "C" int64_t dia_spmm_backward_workspace(const DiaSpmmPlan* plan, int dtype, int64_t M,
                                               int num_experts, int64_t ldx, int64_t stride,
                                               int64_t lddy, int act)
{
    if (!plan || M < 0 || M > INT_MAX / 2 || stride < 0 || num_experts < 1) return -1;
    const GradPlan g = grad_plan(plan, dtype, M, num_experts, ldx, stride, lddy, act);
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
    if (rc == DIA_OK) rc = check_vector(who, "dbias", d_dbias, dtype);
    if (rc == DIA_OK && (uintptr_t)d_dvals % 16)
        rc = fail(DIA_ERR_INVALID, "dia_spmm_backward: dvals must be 16-byte aligned");
    if (rc != DIA_OK) return rc;
    const GradPlan g = grad_plan(plan, dtype, M, num_experts, ldx, stride, lddy, act);
    if (g.bytes() > work_bytes)
        return fail(DIA_ERR_CAPACITY, "dia_spmm_backward: workspace too small");
    if (g.bytes() > 0 && (!d_work || (uintptr_t)d_work % 256))
        return fail(DIA_ERR_INVALID, "dia_spmm_backward: workspace must be 256-byte aligned");

    return by_type(dtype, [&](auto* t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        const bool made = g.made;
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
        a.dy = d_dy;
        a.z = d_z;
        a.lddy = lddy;
        a.ldz = ldz;
        a.act = act;
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
        int r = DIA_OK;
        if (g.x_bytes > 0 && a.dvals) {
            a.x = (char*)d_work + g.dz_bytes + g.part_bytes + g.pack_bytes;
            a.ldx = (plan->n_cols + 7) / 8 * 8;
            r = Cores<T>::dz(kDzSame, DIA_ACT_NONE, d_x, ldx, nullptr, 0, (void*)a.x, nullptr, a.ldx,
                             a.M, a.n_cols, false, stream);
        }
        /* Who reads dz on the CUDA cores has it in fp32, who does on the tensor
         * cores as a pair.  Where the tensor cores take dx alone, the diagonals'
         * or the bias's gradient goes first and dz is made twice. */
        const bool tc = d_dx && product_on_tc(p, g.tensor);
        const bool gtc = grad && grad_on_tc(a, g.tensor);
        const bool acts = act != DIA_ACT_NONE;
        const bool twice = acts && tc && grad && !gtc;
        const bool makes = gtc && acts && spmm_tc_makes_dz(a);
        const bool pair = acts && (tc || gtc);
        char* const rest = (char*)d_work + (long long)p.M * p.ldi * 2;
        auto make_dz = [&](DzForm form, bool dependent) {
            return Cores<T>::dz(form, act, d_dy, lddy, d_z, ldz, d_work, rest, p.ldi, p.M, p.n_in,
                                dependent, stream);
        };
        p.lo = pair && tc ? rest : nullptr;
        a.lo = pair && gtc ? rest : nullptr;
        p.in32 = acts && !tc;
        a.dz32 = acts && !gtc;
        if (r == DIA_OK && twice) {
            r = make_dz(kDzF32, false);
            if (r == DIA_OK) r = Cores<T>::gradient(a, stream);
        }
        /* Launches of the tensor-core form overlap.  Where the diagonals'
         * gradient makes dz itself it goes first, the operator is packed on
         * the SMs that it leaves free; else the operator is packed under dz. */
        if (r != DIA_OK) return r;
        if (makes) {
            r = spmm_tc_gradient(a, dtype, true, false, stream);
            if (r == DIA_OK && tc) r = spmm_tc_pack(p, true, stream);
            p.dependent = true;
        } else {
            const bool packed = tc && g.pack_bytes > 0;
            if (packed) r = spmm_tc_pack(p, false, stream);
            if (r == DIA_OK && made)
                r = make_dz(!acts ? kDzSame : pair ? kDzPair : kDzF32, packed);
            if (r == DIA_OK && grad && !twice)
                r = gtc ? spmm_tc_gradient(a, dtype, false, packed || made, stream)
                        : Cores<T>::gradient(a, stream);
            p.early = tc && gtc;   /* what it reads is older than the gradient */
            p.dependent = packed || made || grad;
        }
        if (r == DIA_OK && d_dx) r = launch_product<T>(p, dtype, g.tensor, stream);
        if (r == DIA_OK && grad) r = Cores<T>::join(a, stream);
        return r;
    });
}

extern "C" int dia_test_spmm_form(int form)
{
    if (form < 0 || form > 2) return fail(DIA_ERR_INVALID, "dia_test_spmm_form: 0, 1 or 2");
    g_form.store(form);
    return DIA_OK;
}
