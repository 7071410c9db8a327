// lcrc_api_ops.cpp -- the operators on matrices in device memory behind the C ABI (include/lcrc_pipeline.h: lcrc_score,
// lcrc_fp8_pack / _unpack / _linear): checks of arguments, the device of the call, launches.  No context, no allocation, no
// wait; the kernels are in score_kernels.hip, fp8_kernels.hip and softmax_kernels.hip, an object that the first call loads.
#include "lcrc_ctx.h"

#include <dlfcn.h>

#include "ops_dev.h"

using namespace lcrc_impl;

namespace {

// The device of a call becomes the thread's current one for its launches and is put back afterwards.
struct DeviceScope {
    int before = -1;
    ~DeviceScope() { if (before >= 0) (void)hipSetDevice(before); }
    int enter(int device_id)
    {
        static const int n_devices = [] { int n = 0; return hipGetDeviceCount(&n) == hipSuccess ? n : 0; }();
        if (n_devices <= 0) return fail(nullptr, LCRC_E_DEVICE, "no HIP device available (this library has no CPU path)");
        if (device_id < 0 || device_id >= n_devices) return fail(nullptr, LCRC_E_DEVICE, "device_id out of range");
        int now = 0;
        HIP_TRY(nullptr, hipGetDevice(&now));
        if (now != device_id) {
            HIP_TRY(nullptr, hipSetDevice(device_id));
            before = now;
        }
        return LCRC_OK;
    }
};

// The kernels' object (ops_dev.h); NULL and a text where it cannot be had.  Loaded once, by the first call that launches something,
// and never unloaded.  It lies beside this library: the library's own search path is its folder, as it was when it was loaded.
const OpsTable *ops(std::string *why)
{
    struct Loaded {
        const OpsTable *table = nullptr;
        std::string error;
        Loaded()
        {
            void *const object = dlopen("libphnrec_lcrc_ops.so", RTLD_NOW | RTLD_LOCAL);
            const auto table_of = object ? reinterpret_cast<const OpsTable *(*)()>(dlsym(object, "lcrc_ops_table")) : nullptr;
            if (!table_of) { const char *e = dlerror(); error = e ? e : "libphnrec_lcrc_ops.so"; return; }
            if (table_of()->version == kOpsVersion) table = table_of();
            else error = "libphnrec_lcrc_ops.so is of another build";
        }
    };
    static const Loaded loaded;
    *why = loaded.error;
    return loaded.table;
}
// ... for a call, with its error
int kernels(lcrc_ctx *c, const OpsTable **table)
{
    std::string why;
    *table = ops(&why);
    return *table ? LCRC_OK : fail(c, LCRC_E_DEVICE, "cannot load the operators' kernels: " + why);
}

int element_bytes(int type) { return type == LCRC_T_F32 ? 4 : type == LCRC_T_E4M3 ? 1 : 2; }
bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int bad(const char *call, const char *what) { return fail(nullptr, LCRC_E_ARG, std::string(call) + ": " + what); }

int launched(const char *call, hipError_t e)
{
    if (e == hipSuccess) return LCRC_OK;
    (void)hipGetLastError();
    return fail(nullptr, LCRC_E_DEVICE, std::string(call) + ": " + hipGetErrorString(e));
}

// rows in one of the plain types: pointer, row distance
int check_rows(const char *call, const void *p, int type, int cols, long long ld)
{
    if (!p) return bad(call, "NULL matrix");
    if (!aligned(p, element_bytes(type))) return bad(call, "a matrix must be aligned to its elements");
    if (ld < cols) return bad(call, "the distance of rows is smaller than their length");
    if (ld > (1ll << 40)) return bad(call, "the distance of rows is too large");
    return LCRC_OK;
}

// a matrix in the 8-bit form: the launches over its tiles stay within a grid
int check_held(const char *call, const void *p, int rows, int cols)
{
    if (!p || !aligned(p, 16)) return bad(call, "an 8-bit matrix must be aligned to 16 bytes");
    const Q8Shape s(rows, cols);
    if (s.rt * s.kb >= kQMaxTiles) return bad(call, "an 8-bit matrix of 2^26 tiles of 16 x 128 or more");
    return LCRC_OK;
}

}  // namespace

namespace lcrc_impl {

// ---- the merger of an unfused system with 8-bit operands (lcrc_set_merger_fp8) ----
// inputs -> normalised, in 8 bits -> hidden layer (FEXP sigmoid), in 8 bits -> outputs in f32 -> softmax and output transform
size_t merger_fp8_bytes(const lcrc_ctx *c, size_t n_rows)
{
    const NetDev &net = c->nets[2];
    return (size_t)Q8Shape((int)n_rows, net.n_inp).bytes() + (size_t)Q8Shape((int)n_rows, net.n_hid).bytes() + n_rows * net.n_out * sizeof(float);
}
int merger_fp8(lcrc_ctx *c, const float *d_in, int n_rows, const MlpParams &m, hipStream_t s)
{
    const NetDev &net = c->nets[2];
    const size_t x_bytes = (size_t)Q8Shape(n_rows, net.n_inp).bytes(), h_bytes = (size_t)Q8Shape(n_rows, net.n_hid).bytes();
    unsigned char *x = c->d_fp8, *h = x + x_bytes;
    float *y = reinterpret_cast<float *>(h + h_bytes);
    const OpsTable *k;
    if (const int rc = kernels(c, &k)) return rc;
    Fp8PackParams pack = {d_in, nullptr, LCRC_T_F32, n_rows, net.n_inp, net.n_inp, x, net.mean, net.dev};
    HIP_TRY(c, k->fp8_pack(pack, s));
    HIP_TRY(c, k->fp8_product({x, c->fp8_w1, net.b1, n_rows, net.n_inp, net.n_hid, LCRC_ACT_FSIGMOID, LCRC_T_E4M3, h, 0}, s));
    HIP_TRY(c, k->fp8_product({h, c->fp8_w2, net.b2, n_rows, net.n_hid, net.n_out, LCRC_ACT_NONE, LCRC_T_F32, y, net.n_out}, s));
    SoftmaxRowsParams o;
    memset(&o, 0, sizeof o);
    o.in = y; o.out = m.out; o.out_ld = m.out_ld; o.n_rows = n_rows; o.n = net.n_out;
    memcpy(o.out_func, m.out_func, sizeof o.out_func);
    memcpy(o.out_c, m.out_c, sizeof o.out_c);
    memcpy(o.out_l, m.out_l, sizeof o.out_l);
    o.out_be = m.out_be;
    HIP_TRY(c, k->softmax_rows(o, s));
    return LCRC_OK;
}

// ---- scores behind the posteriors (lcrc_posteriors_scored) ----
namespace {
// one block: [labels][ln p of them][entropy][best classes][their ln p] (labels and scores: also in pinned memory), scratch
struct ScoreLayout {
    size_t labels, logp, entropy, index, top, host_end, end;
    ScoreLayout(const lcrc_ctx *c, const HostScores &w, size_t n)
    {
        size_t at = 0;
        const auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
        labels = take(n * w.n_labels * sizeof(int));
        logp = take(n * w.n_labels * sizeof(float));
        entropy = take(n * sizeof(float));
        index = take(n * w.k * sizeof(int));
        top = take(n * w.k * sizeof(float));
        host_end = at;
        end = at + score_workspace_bytes((int)n, c->nets[2].n_out, w.k);
    }
};
}  // namespace

int scores_after(lcrc_ctx *c, const HostScores &w, int n_rows, const float *d_post)
{
    const OpsTable *kernel;
    if (const int rc = kernels(c, &kernel)) return rc;
    const ScoreLayout l(c, w, n_rows);
    if (l.end > c->cap_scores) {
        if (c->d_scores) (void)hipFree(c->d_scores);
        if (c->h_scores) (void)pinned_free(c->h_scores);
        c->d_scores = c->h_scores = nullptr;
        c->cap_scores = 0;
        const size_t cap = l.end + l.end / 4;
        if (dev_alloc((void **)&c->d_scores, cap) != hipSuccess || pinned_alloc((void **)&c->h_scores, cap) != hipSuccess) {
            if (c->d_scores) (void)hipFree(c->d_scores);
            c->d_scores = c->h_scores = nullptr;
            (void)hipGetLastError();
            return fail(c, LCRC_E_NOMEM, "cannot allocate the scores of " + std::to_string(n_rows) + " frames");
        }
        c->cap_scores = cap;
    }
    char *d = c->d_scores, *h = c->h_scores;
    if (w.n_labels > 0) {
        const size_t bytes = (size_t)n_rows * w.n_labels * sizeof(int);
        memcpy(h + l.labels, w.labels, bytes);
        HIP_TRY(c, hipMemcpyAsync(d + l.labels, h + l.labels, bytes, hipMemcpyHostToDevice, c->stream));
    }
    lcrc_score_args a;
    memset(&a, 0, sizeof a);
    a.x = d_post; a.type = LCRC_T_F32; a.form = LCRC_SCORE_PROBS;
    a.rows = n_rows; a.cols = c->nets[2].n_out; a.ld = a.cols;
    a.labels = (const int *)(d + l.labels); a.n_labels = w.n_labels; a.k = w.k;
    a.logp = w.n_labels > 0 ? (float *)(d + l.logp) : nullptr;
    a.entropy = (float *)(d + l.entropy);
    a.top_index = w.k > 0 ? (int *)(d + l.index) : nullptr;
    a.top_logp = w.k > 0 ? (float *)(d + l.top) : nullptr;
    a.workspace = d + l.host_end; a.workspace_bytes = l.end - l.host_end;
    HIP_TRY(c, kernel->score(a, c->stream));
    HIP_TRY(c, hipMemcpyAsync(h + l.logp, d + l.logp, l.host_end - l.logp, hipMemcpyDeviceToHost, c->stream));
    return LCRC_OK;
}

void fetch_scores(lcrc_ctx *c, const HostScores &w, int n_rows)
{
    const ScoreLayout l(c, w, n_rows);
    const size_t n = n_rows;
    const char *h = c->h_scores;
    if (w.logp) memcpy(w.logp, h + l.logp, n * w.n_labels * sizeof(float));
    if (w.entropy) memcpy(w.entropy, h + l.entropy, n * sizeof(float));
    if (w.top_index) memcpy(w.top_index, h + l.index, n * w.k * sizeof(int));
    if (w.top_logp) memcpy(w.top_logp, h + l.top, n * w.k * sizeof(float));
}

}  // namespace lcrc_impl

extern "C" {

int lcrc_set_merger_fp8(lcrc_ctx *c, int enabled)
{
    if (!c) return LCRC_E_ARG;
    if (!enabled) { c->fp8_merger = false; return LCRC_OK; }
    if (c->system == SYS_LCRC)
        return fail(c, LCRC_E_UNSUPPORTED, "lcrc_set_merger_fp8: the fused LCRC kernels hold their operands in f32 or split f16");
    HIP_TRY(c, hipSetDevice(c->device));
    const OpsTable *k;
    if (const int rc = kernels(c, &k)) return rc;
    if (!c->fp8_w1) {
        const HostNet &net = c->model->host[2];
        for (const std::vector<float> *w : {&net.w1, &net.w2})
            for (float v : *w)
                if (!std::isfinite(v)) return fail(c, LCRC_E_UNSUPPORTED, "lcrc_set_merger_fp8: non-finite weights have no 8-bit form");
        const size_t bytes1 = lcrc_fp8_bytes(net.n_hid, net.n_inp), bytes2 = lcrc_fp8_bytes(net.n_out, net.n_hid);
        void *w1 = nullptr, *w2 = nullptr, *rows = nullptr;
        const auto pack = [&](const std::vector<float> &w, int n_out, int n_in, void *dst) {
            if (const hipError_t e = hipMemcpy(rows, w.data(), w.size() * sizeof(float), hipMemcpyHostToDevice); e != hipSuccess) return e;
            if (const hipError_t e = k->fp8_pack({rows, nullptr, LCRC_T_F32, n_out, n_in, n_in, (unsigned char *)dst, nullptr, nullptr}, c->stream);
                e != hipSuccess) return e;
            return hipStreamSynchronize(c->stream);
        };
        hipError_t e = dev_alloc(&w1, bytes1);
        if (e == hipSuccess) e = dev_alloc(&w2, bytes2);
        if (e == hipSuccess) e = dev_alloc(&rows, std::max(net.w1.size(), net.w2.size()) * sizeof(float));
        const bool room = e == hipSuccess;
        if (e == hipSuccess) e = pack(net.w1, net.n_hid, net.n_inp, w1);
        if (e == hipSuccess) e = pack(net.w2, net.n_out, net.n_hid, w2);
        if (rows) (void)hipFree(rows);
        if (e != hipSuccess) {
            if (w1) (void)hipFree(w1);
            if (w2) (void)hipFree(w2);
            (void)hipGetLastError();
            return fail(c, room ? LCRC_E_DEVICE : LCRC_E_NOMEM, std::string("lcrc_set_merger_fp8: ") + hipGetErrorString(e));
        }
        c->allocs.push_back(w1);
        c->allocs.push_back(w2);
        c->fp8_w1 = (unsigned char *)w1;
        c->fp8_w2 = (unsigned char *)w2;
    }
    c->fp8_merger = true;
    return LCRC_OK;
}

int lcrc_posteriors_scored(lcrc_ctx *c, const float *mel, const int *off, int n_utts, float *post, const int *labels, int n_labels,
                           int k, float *logp, float *entropy, int *top_index, float *top_logp)
{
    const auto bad_arg = [&](const char *what) { return fail(c, LCRC_E_ARG, std::string("lcrc_posteriors_scored: ") + what); };
    if (!c) return LCRC_E_ARG;
    if (n_utts < 0 || (n_utts > 0 && !off)) return bad_arg("bad argument");
    if (n_labels < 0 || n_labels > kScoreMaxLabels) return bad_arg("n_labels: 0 .. 64");
    if (k < 0 || k > kScoreMaxTop || k > c->nets[2].n_out) return bad_arg("k: 0 .. 64, at most the model's outputs");
    if (n_utts == 0) return LCRC_OK;
    if (off[0] != 0) return bad_arg("off[0] must be 0");
    for (int u = 0; u < n_utts; u++)
        if (off[u + 1] < off[u]) return bad_arg("offsets must be non-decreasing");
    const int n = off[n_utts];
    if (n == 0) return LCRC_OK;
    if (!mel || (n_labels > 0 && !labels)) return bad_arg("NULL buffer");
    if (c->soft[0].func != LCRC_SOFT_NONE || c->soft[1].func != LCRC_SOFT_NONE || c->out_be)
        return bad_arg("scores are taken of plain posteriors (lcrc_output_configure without stages, in host byte order)");
    HIP_TRY(c, hipSetDevice(c->device));
    const HostScores want = {labels, n_labels, k, logp, entropy, top_index, top_logp};
    return run_host(c, mel, off, n_utts, n, post, nullptr, false, &want);
}

size_t lcrc_score_workspace(int rows, int cols, int k)
{
    if (rows <= 0 || cols <= 0 || cols > kScoreMaxCols || k < 0 || k > kScoreMaxTop) return 0;
    return score_workspace_bytes(rows, cols, k);
}

int lcrc_score(int device_id, const lcrc_score_args *a, void *hip_stream)
{
    const char *call = "lcrc_score";
    if (!a) return bad(call, "NULL argument");
    if (a->type != LCRC_T_F32 && a->type != LCRC_T_F16 && a->type != LCRC_T_BF16) return bad(call, "type: LCRC_T_F32, LCRC_T_F16 or LCRC_T_BF16");
    if (a->form != LCRC_SCORE_LOGITS && a->form != LCRC_SCORE_PROBS) return bad(call, "form: LCRC_SCORE_LOGITS or LCRC_SCORE_PROBS");
    if (a->rows < 0) return bad(call, "negative size");
    if (a->cols < 1 || a->cols > kScoreMaxCols) return bad(call, "cols: 1 .. 2^30");
    if (a->k < 0 || a->k > kScoreMaxTop || a->k > a->cols) return bad(call, "k: 0 .. 64, at most cols");
    if (a->n_labels < 0 || a->n_labels > kScoreMaxLabels) return bad(call, "n_labels: 0 .. 64");
    if (a->rows == 0) return LCRC_OK;
    if (const int rc = check_rows(call, a->x, a->type, a->cols, a->ld)) return rc;
    if (a->n_labels > 0 && a->logp && !a->labels) return bad(call, "NULL labels");
    if (!aligned(a->labels, 4) || !aligned(a->logp, 4) || !aligned(a->entropy, 4) || !aligned(a->top_index, 4) || !aligned(a->top_logp, 4))
        return bad(call, "labels and outputs must be aligned to 4 bytes");
    const size_t need = score_workspace_bytes(a->rows, a->cols, a->k);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16)))
        return bad(call, "workspace missing, smaller than lcrc_score_workspace says or not aligned to 16 bytes");
    DeviceScope device;
    if (const int rc = device.enter(device_id)) return rc;
    const OpsTable *k;
    if (const int rc = kernels(nullptr, &k)) return rc;
    return launched(call, k->score(*a, static_cast<hipStream_t>(hip_stream)));
}

size_t lcrc_fp8_bytes(int rows, int cols)
{
    return rows <= 0 || cols <= 0 ? 0 : (size_t)Q8Shape(rows, cols).bytes();
}

int lcrc_fp8_pack(int device_id, const void *src, int type, int rows, int cols, long long ld, const unsigned char *scales,
                  void *dst, void *hip_stream)
{
    const char *call = "lcrc_fp8_pack";
    if (type < LCRC_T_F32 || type > LCRC_T_E4M3) return bad(call, "unknown type");
    if (rows < 0 || cols < 1) return bad(call, "sizes: rows >= 0, cols >= 1");
    if ((type == LCRC_T_E4M3) != (scales != nullptr) && rows > 0) return bad(call, "scales belong to LCRC_T_E4M3 and to no other type");
    if (rows == 0) return LCRC_OK;
    if (const int rc = check_rows(call, src, type, cols, ld)) return rc;
    if (const int rc = check_held(call, dst, rows, cols)) return rc;
    DeviceScope device;
    if (const int rc = device.enter(device_id)) return rc;
    const OpsTable *k;
    if (const int rc = kernels(nullptr, &k)) return rc;
    const Fp8PackParams p = {src, scales, type, rows, cols, ld, static_cast<unsigned char *>(dst), nullptr, nullptr};
    return launched(call, k->fp8_pack(p, static_cast<hipStream_t>(hip_stream)));
}

int lcrc_fp8_unpack(int device_id, const void *src, int rows, int cols, void *dst, int type, long long ld, void *hip_stream)
{
    const char *call = "lcrc_fp8_unpack";
    if (type < LCRC_T_F32 || type > LCRC_T_BF16) return bad(call, "type: LCRC_T_F32, LCRC_T_F16 or LCRC_T_BF16");
    if (rows < 0 || cols < 1) return bad(call, "sizes: rows >= 0, cols >= 1");
    if (rows == 0) return LCRC_OK;
    if (const int rc = check_rows(call, dst, type, cols, ld)) return rc;
    if (const int rc = check_held(call, src, rows, cols)) return rc;
    DeviceScope device;
    if (const int rc = device.enter(device_id)) return rc;
    const OpsTable *k;
    if (const int rc = kernels(nullptr, &k)) return rc;
    const Fp8UnpackParams p = {static_cast<const unsigned char *>(src), type, rows, cols, ld, dst};
    return launched(call, k->fp8_unpack(p, static_cast<hipStream_t>(hip_stream)));
}

size_t lcrc_fp8_linear_workspace(int rows, int n_in, int x_type)
{
    return x_type == LCRC_T_E4M3 ? 0 : lcrc_fp8_bytes(rows, n_in);
}

int lcrc_fp8_linear(int device_id, const lcrc_fp8_linear_args *a, void *hip_stream)
{
    const char *call = "lcrc_fp8_linear";
    if (!a) return bad(call, "NULL argument");
    if (a->x_type < LCRC_T_F32 || a->x_type > LCRC_T_E4M3 || a->y_type < LCRC_T_F32 || a->y_type > LCRC_T_E4M3) return bad(call, "unknown type");
    if (a->act < LCRC_ACT_NONE || a->act > LCRC_ACT_FSIGMOID) return bad(call, "unknown activation");
    if (a->rows < 0 || a->n_in < 1 || a->n_in > kQMaxIn || a->n_out < 1) return bad(call, "sizes: rows >= 0, n_in 1 .. 2^23, n_out >= 1");
    if (a->rows == 0) return LCRC_OK;
    if (a->x_type == LCRC_T_E4M3) {
        if (const int rc = check_held(call, a->x, a->rows, a->n_in)) return rc;
    } else if (const int rc = check_rows(call, a->x, a->x_type, a->n_in, a->ldx)) return rc;
    if (a->y_type == LCRC_T_E4M3) {
        if (const int rc = check_held(call, a->y, a->rows, a->n_out)) return rc;
    } else if (const int rc = check_rows(call, a->y, a->y_type, a->n_out, a->ldy)) return rc;
    if (const int rc = check_held(call, a->w, a->n_out, a->n_in)) return rc;
    const Q8Shape sx(a->rows, a->n_in), sy(a->rows, a->n_out);
    if (sx.rt * sx.kb >= kQMaxTiles || sy.rt * sy.kb >= kQMaxTiles) return bad(call, "x or y of 2^26 tiles of 16 x 128 or more");
    // (a last tile of outputs or rows counts as a whole one)
    const Fp8Route route = fp8_route(a->rows, a->n_in, a->n_out, a->y_type);
    if (route != kFp8SharedSums &&
        fp8_tiles(a->rows, a->n_out, route == kFp8Tiles256x128 ? 256 : 128, route == kFp8Tiles128x64 ? 64 : 128) + 7 >= (1ll << 32) / 256)
        return bad(call, "more rows and outputs than a grid has threads for");
    if (!aligned(a->bias, 4)) return bad(call, "bias must be aligned to 4 bytes");
    const size_t need = lcrc_fp8_linear_workspace(a->rows, a->n_in, a->x_type);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16)))
        return bad(call, "workspace missing, smaller than lcrc_fp8_linear_workspace says or not aligned to 16 bytes");
    DeviceScope device;
    if (const int rc = device.enter(device_id)) return rc;
    const OpsTable *k;
    if (const int rc = kernels(nullptr, &k)) return rc;
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const unsigned char *x = a->x_type == LCRC_T_E4M3 ? static_cast<const unsigned char *>(a->x) : nullptr;
    Fp8ProductParams p = {x, static_cast<const unsigned char *>(a->w), a->bias, a->rows, a->n_in, a->n_out, a->act, a->y_type, a->y, a->ldy};
    if (a->x_type != LCRC_T_E4M3) {
        if (a->rows <= kQRows && a->n_out <= kQFewOut) return launched(call, k->fp8_few_rows(p, a->x, a->x_type, a->ldx, s));
        const Fp8PackParams pack = {a->x, nullptr, a->x_type, a->rows, a->n_in, a->ldx, static_cast<unsigned char *>(a->workspace), nullptr, nullptr};
        if (const int rc = launched(call, k->fp8_pack(pack, s))) return rc;
        p.x = pack.dst;
    }
    return launched(call, k->fp8_product(p, s));
}

int lcrc_debug_score_blocks(int most)
{
    const OpsTable *k;
    if (most < 1 || most > 1 << 22) return fail(nullptr, LCRC_E_ARG, "lcrc_debug_score_blocks: 1 .. 2^22");
    if (const int rc = kernels(nullptr, &k)) return rc;
    return k->score_most_blocks(most);
}

int lcrc_debug_fp8_route(int rows, int n_in, int n_out, int y_type)
{
    return fp8_route(rows, n_in, n_out, y_type) + (fp8_sums_in_32_bits(y_type) ? 4 : 0);
}

}  // extern "C"
