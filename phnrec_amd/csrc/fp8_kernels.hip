// fp8_kernels.hip -- matrices held in e4m3 with a power-of-two scale for each block of 128 columns (ops_dev.h: the form), and
// their products on the block-scaled matrix instructions (include/lcrc_pipeline.h: lcrc_fp8_pack / _unpack / _linear).
#include <cmath>

#include "ops_dev.h"

namespace phnrec {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

// the column a lane's byte j stands for, within its block of 128 (ops_dev.h)
__device__ __forceinline__ int column_of(int g, int j) { return 16 * (j >> 2) + 4 * g + (j & 3); }

// The smallest e >= -127 with most <= 448 * 2^e; 0 for 0.  From the bits of most = 1.f * 2^E: 448 = 1.75 * 2^8, so e = E - 8,
// and one more where 1.f exceeds 1.75 (subnormals: E = -127 and the bound holds).
__device__ __forceinline__ int block_exponent(float most)
{
    const int b = __float_as_int(most);
    const int e = (b >> 23) - 127 - 8 + ((b & 0x7fffff) > 0x600000 ? 1 : 0);
    return b == 0 ? 0 : max(e, -127);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127

// four values, already divided by their block's scale, as four e4m3 bytes: round to nearest even in hardware (OCP on gfx950)
__device__ __forceinline__ int to_e4m3(float a, float b, float c, float d)
{
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// A lane's 32 values of one (row, block): scale over the row's four lanes, bytes, exponent.
__device__ __forceinline__ i8 quantise(const float (&v)[32], int *exponent)
{
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; j++) {
        const float t = fabsf(v[j]);
        most = fmaxf(most, t < INFINITY ? t : 0.0f);          // (NaN and infinities do not count)
    }
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    const int e = block_exponent(most);
    const float inv = pow2(-e);
    i8 q;
#pragma unroll
    for (int t = 0; t < 8; t++) {
        float s[4];
#pragma unroll
        for (int r = 0; r < 4; r++) s[r] = fabsf(v[4 * t + r]) < INFINITY ? v[4 * t + r] * inv : NAN;
        q[t] = to_e4m3(s[0], s[1], s[2], s[3]);
    }
    *exponent = e;
    return q;
}

__device__ __forceinline__ void store_tile(unsigned char *tile, int lane, const i8 &q)
{
    reinterpret_cast<i4 *>(tile)[lane] = i4{q[0], q[1], q[2], q[3]};
    reinterpret_cast<i4 *>(tile)[64 + lane] = i4{q[4], q[5], q[6], q[7]};
}

__device__ __forceinline__ i8 load_tile(const unsigned char *tile, int lane)
{
    const i4 a = reinterpret_cast<const i4 *>(tile)[lane], b = reinterpret_cast<const i4 *>(tile)[64 + lane];
    return i8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// One wave per tile of 16 rows x 128 columns.
template <typename X>
__global__ __launch_bounds__(256) void fp8_pack_kernel(const Fp8PackParams p)
{
    const Q8Shape s(p.rows, p.cols);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= s.rt * s.kb) return;
    const long long t = tile / s.kb, kb = tile % s.kb;
    const long long row = 16 * t + c;
    const bool live = row < p.rows;
    i8 q;
    int e = 0;
    if constexpr (sizeof(X) == 1) {
        const unsigned char *src = static_cast<const unsigned char *>(p.src) + (live ? row : 0) * p.ld;
#pragma unroll
        for (int w = 0; w < 8; w++) {
            unsigned v = 0;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const long long k = kb * 128 + column_of(g, 4 * w + r);
                if (live && k < p.cols) v |= (unsigned)src[k] << (8 * r);
            }
            q[w] = (int)v;
        }
        if (live) e = (int)p.scales[row * s.kb + kb] - 127;
    } else {
        const X *src = static_cast<const X *>(p.src) + (live ? row : 0) * p.ld;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; j++) {
            const long long k = kb * 128 + column_of(g, j);
            v[j] = live && k < p.cols ? to_f32(src[k]) : 0.0f;
        }
        q = quantise(v, &e);
    }
    store_tile(p.dst + tile * kQTileBytes, lane, q);
    unsigned char *scales = p.dst + s.scales_at() + ((t * s.kb4 + kb / 4) * 16 + c) * 4;
    if (g == 0) scales[kb & 3] = (unsigned char)(e + 127);
    if (kb == s.kb - 1 && g > (kb & 3)) scales[g] = 127;               // the blocks that fill the last group up
}

template <typename Y>
__global__ __launch_bounds__(256) void fp8_unpack_kernel(const Fp8UnpackParams p)
{
    const Q8Shape s(p.rows, p.cols);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= s.rt * s.kb) return;
    const long long t = tile / s.kb, kb = tile % s.kb, row = 16 * t + c;
    if (row >= p.rows) return;
    const i8 q = load_tile(p.src + tile * kQTileBytes, lane);
    const int e = (int)p.src[s.scales_at() + ((t * s.kb4 + kb / 4) * 16 + c) * 4 + (kb & 3)] - 127;
    Y *dst = static_cast<Y *>(p.dst) + row * p.ld;
#pragma unroll
    for (int w = 0; w < 8; w++) {
        const float v[4] = {__builtin_amdgcn_cvt_f32_fp8(q[w], 0), __builtin_amdgcn_cvt_f32_fp8(q[w], 1),
                            __builtin_amdgcn_cvt_f32_fp8(q[w], 2), __builtin_amdgcn_cvt_f32_fp8(q[w], 3)};
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const long long k = kb * 128 + column_of(g, 4 * w + r);
            // (ldexpf: 2^-127 and 2^128 are no normal f32 factors; byte 255 is no number)
            if (k < p.cols) dst[k] = (Y)(e == 128 ? NAN : ldexpf(v[r], e));
        }
    }
}

template <int ACT>
__device__ __forceinline__ float activate(float v)
{
    if constexpr (ACT == LCRC_ACT_SIGMOID) return 1.0f / (1.0f + expf(-v));
    if constexpr (ACT == LCRC_ACT_FSIGMOID) {
        // FEXP (fexp.h:14-21): the exponent's bits of a double from one truncated product; out of range as x86 converts it
        const float y = -v;
        int i = __double2int_rz(1048576.0 / 0.69314718055994530942 * (double)y);
        if (!(y < 0x1.62e43p+10f)) i = (int)0x80000000u;
        return 1.0f / (1.0f + (float)__hiloint2double((int)((unsigned)i + 1072632447u), 0));
    }
    return v;
}

// ---- the sums ----
// The 8-bit matrix instructions multiply exactly, but inside a group of eight products (eight bytes of a lane that follow one
// another) they cut every product off 13 bits below the group's largest one before they add (measured, for the scaled and the
// plain form alike: 2^16 + 3 * 2^3 comes out whole, of 2^16 + 3 * 7 the sevens are gone); the groups' sums are added in 32
// bits.  That is up to 7 * 2^-13 of the products' absolute sum, 1.4e-5 relative on normal values: nothing beside a result
// that is rounded to 16 or 8 bits (2^-8 .. 2^-11, 2^-4), too much for one in 32 bits.  So products with an f32 result turn
// their operands into bf16 -- exact: 4 significant bits, the block's scale goes into bf16's exponent (v_cvt_scalef32_pk_bf16_fp8;
// below 2^-126 it loses bits) -- and use the bf16 instruction, whose sums are f32 throughout: half the rate.
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

// bytes 8 s .. 8 s + 7 of a lane, times the block's scale
__device__ __forceinline__ b8 to_bf16(const i8 &q, int s, float scale)
{
    b2 v[4];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        v[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * s + h], scale, false);
        v[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * s + h], scale, true);
    }
    return b8{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
}

// acc += A B over one block of 128 columns; as / bs: the block's scale byte of the lane's row, in the low byte
template <bool EXACT>
__device__ __forceinline__ f4 block_product(const i8 &a, const i8 &b, f4 acc, int as, int bs)
{
    if constexpr (!EXACT) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 0, as, 0, bs);
    const float sa = __int_as_float((as & 255) << 23), sb = __int_as_float((bs & 255) << 23);
#pragma unroll
    for (int s = 0; s < 4; s++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(a, s, sa), to_bf16(b, s, sb), acc, 0, 0, 0);
    return acc;
}

// D = W X^T per tile of 16 x 16: lane (c, g) holds features 4 g + r (register r) of x row c.
// One wave per 16 rows x 128 outputs, operands straight from memory.
template <int ACT, typename Y>
__global__ __launch_bounds__(256) void fp8_product_kernel(const Fp8ProductParams p)
{
    const Q8Shape sx(p.rows, p.n_in), sw(p.n_out, p.n_in), sy(p.rows, p.n_out);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= sx.rt * sy.kb) return;
    const long long t = id / sy.kb, ob = id % sy.kb;                   // row tile, block of 128 outputs
    const unsigned char *x = p.x + t * sx.kb * kQTileBytes;
    const int *xs = reinterpret_cast<const int *>(p.x + sx.scales_at()) + t * sx.kb4 * 16 + c;
    const unsigned char *w[8];
    const int *ws[8];
#pragma unroll
    for (int n = 0; n < 8; n++) {
        const long long wt = min(8 * ob + n, sw.rt - 1);
        w[n] = p.w + wt * sw.kb * kQTileBytes;
        ws[n] = reinterpret_cast<const int *>(p.w + sw.scales_at()) + wt * sw.kb4 * 16 + c;
    }
    f4 acc[8];
#pragma unroll
    for (int n = 0; n < 8; n++) acc[n] = f4{0.f, 0.f, 0.f, 0.f};
    for (long long kb = 0; kb < sx.kb; kb++) {
        const i8 b = load_tile(x + kb * kQTileBytes, lane);
        const int shift = 8 * (int)(kb & 3);
        const int bs = xs[(kb >> 2) * 16] >> shift;
#pragma unroll
        for (int n = 0; n < 8; n++) {
            const i8 a = load_tile(w[n] + kb * kQTileBytes, lane);
            const int as = ws[n][(kb >> 2) * 16] >> shift;
            acc[n] = block_product<sizeof(Y) == 4>(a, b, acc[n], as, bs);
        }
    }
    const long long row = 16 * t + c;
    float v[32];
#pragma unroll
    for (int n = 0; n < 8; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const long long o = 128 * ob + 16 * n + 4 * g + r;
            const bool live = row < p.rows && o < p.n_out;
            v[4 * n + r] = live ? activate<ACT>(acc[n][r] + (p.bias ? p.bias[o] : 0.0f)) : 0.0f;
        }
    if constexpr (sizeof(Y) == 1) {
        unsigned char *y = static_cast<unsigned char *>(p.y);
        int e;
        const i8 q = quantise(v, &e);
        store_tile(y + (t * sy.kb + ob) * kQTileBytes, lane, q);
        unsigned char *scales = y + sy.scales_at() + ((t * sy.kb4 + ob / 4) * 16 + c) * 4;
        if (g == 0) scales[ob & 3] = (unsigned char)(e + 127);
        if (ob == sy.kb - 1 && g > (ob & 3)) scales[g] = 127;
    } else {
        Y *y = static_cast<Y *>(p.y) + row * p.ldy;
#pragma unroll
        for (int n = 0; n < 8; n++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const long long o = 128 * ob + 16 * n + 4 * g + r;
                if (row < p.rows && o < p.n_out) y[o] = (Y)v[4 * n + r];
            }
    }
}

template <int ACT>
void product_by_type(const Fp8ProductParams &p, unsigned blocks, hipStream_t stream)
{
    switch (p.y_type) {
    case LCRC_T_F32: fp8_product_kernel<ACT, float><<<blocks, 256, 0, stream>>>(p); break;
    case LCRC_T_F16: fp8_product_kernel<ACT, _Float16><<<blocks, 256, 0, stream>>>(p); break;
    case LCRC_T_BF16: fp8_product_kernel<ACT, __bf16><<<blocks, 256, 0, stream>>>(p); break;
    default: fp8_product_kernel<ACT, unsigned char><<<blocks, 256, 0, stream>>>(p); break;
    }
}

}  // namespace

hipError_t fp8_pack_launch(const Fp8PackParams &p, hipStream_t stream)
{
    const Q8Shape s(p.rows, p.cols);
    const unsigned blocks = (unsigned)((s.rt * s.kb + 3) / 4);
    switch (p.type) {
    case LCRC_T_F32: fp8_pack_kernel<float><<<blocks, 256, 0, stream>>>(p); break;
    case LCRC_T_F16: fp8_pack_kernel<_Float16><<<blocks, 256, 0, stream>>>(p); break;
    case LCRC_T_BF16: fp8_pack_kernel<__bf16><<<blocks, 256, 0, stream>>>(p); break;
    default: fp8_pack_kernel<unsigned char><<<blocks, 256, 0, stream>>>(p); break;
    }
    return hipGetLastError();
}

hipError_t fp8_unpack_launch(const Fp8UnpackParams &p, hipStream_t stream)
{
    const Q8Shape s(p.rows, p.cols);
    const unsigned blocks = (unsigned)((s.rt * s.kb + 3) / 4);
    switch (p.type) {
    case LCRC_T_F32: fp8_unpack_kernel<float><<<blocks, 256, 0, stream>>>(p); break;
    case LCRC_T_F16: fp8_unpack_kernel<_Float16><<<blocks, 256, 0, stream>>>(p); break;
    default: fp8_unpack_kernel<__bf16><<<blocks, 256, 0, stream>>>(p); break;
    }
    return hipGetLastError();
}

hipError_t fp8_product_launch(const Fp8ProductParams &p, hipStream_t stream)
{
    const Q8Shape sx(p.rows, p.n_in), sy(p.rows, p.n_out);
    const unsigned blocks = (unsigned)((sx.rt * sy.kb + 3) / 4);
    switch (p.act) {
    case LCRC_ACT_NONE: product_by_type<LCRC_ACT_NONE>(p, blocks, stream); break;
    case LCRC_ACT_SIGMOID: product_by_type<LCRC_ACT_SIGMOID>(p, blocks, stream); break;
    default: product_by_type<LCRC_ACT_FSIGMOID>(p, blocks, stream); break;
    }
    return hipGetLastError();
}

}  // namespace phnrec
