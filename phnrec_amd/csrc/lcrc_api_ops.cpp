// lcrc_api_ops.cpp -- the operators on matrices in device memory behind the C ABI (include/lcrc_pipeline.h: lcrc_score,
// lcrc_fp8_pack / _unpack / _linear): checks of arguments, the device of the call, launches.  No context, no allocation, no
// wait; the kernels are in score_kernels.hip and fp8_kernels.hip.
#include "lcrc_ctx.h"
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
    if (s.rt * s.kb > kQMaxTiles) return bad(call, "an 8-bit matrix of more than 2^26 tiles of 16 x 128");
    return LCRC_OK;
}

}  // namespace

extern "C" {

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
    return launched(call, score_launch(*a, static_cast<hipStream_t>(hip_stream)));
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
    const Fp8PackParams p = {src, scales, type, rows, cols, ld, static_cast<unsigned char *>(dst)};
    return launched(call, fp8_pack_launch(p, static_cast<hipStream_t>(hip_stream)));
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
    const Fp8UnpackParams p = {static_cast<const unsigned char *>(src), type, rows, cols, ld, dst};
    return launched(call, fp8_unpack_launch(p, static_cast<hipStream_t>(hip_stream)));
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
    if (sx.rt * sx.kb > kQMaxTiles || sy.rt * sy.kb > kQMaxTiles) return bad(call, "x or y of more than 2^26 tiles of 16 x 128");
    if (!aligned(a->bias, 4)) return bad(call, "bias must be aligned to 4 bytes");
    const size_t need = lcrc_fp8_linear_workspace(a->rows, a->n_in, a->x_type);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16)))
        return bad(call, "workspace missing, smaller than lcrc_fp8_linear_workspace says or not aligned to 16 bytes");
    DeviceScope device;
    if (const int rc = device.enter(device_id)) return rc;
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const unsigned char *x = a->x_type == LCRC_T_E4M3 ? static_cast<const unsigned char *>(a->x) : nullptr;
    Fp8ProductParams p = {x, static_cast<const unsigned char *>(a->w), a->bias, a->rows, a->n_in, a->n_out, a->act, a->y_type, a->y, a->ldy};
    if (a->x_type != LCRC_T_E4M3) {
        if (a->rows <= kQRows && a->n_out <= kQFewOut) return launched(call, fp8_few_rows_launch(p, a->x, a->x_type, a->ldx, s));
        const Fp8PackParams pack = {a->x, nullptr, a->x_type, a->rows, a->n_in, a->ldx, static_cast<unsigned char *>(a->workspace)};
        if (const int rc = launched(call, fp8_pack_launch(pack, s))) return rc;
        p.x = pack.dst;
    }
    return launched(call, fp8_product_launch(p, s));
}

}  // extern "C"
