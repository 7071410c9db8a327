// fp8_kernels.hip -- matrices held in e4m3 with a power-of-two scale for each block of 128 columns (ops_dev.h: the form), and
// their products on the block-scaled matrix instructions (include/lcrc_pipeline.h: lcrc_fp8_pack / _unpack / _linear).
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

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

// A lane's 32 values of one (row, block): scale over the row's four lanes, bytes, exponent.  A maximum skips NaN, and the
// conversion keeps it; infinities, which do not count for the scale and become NaN, take a way of their own.
__device__ __forceinline__ i8 quantise(float (&v)[32], int *exponent)
{
    const auto largest = [&] {
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < 32; j++) most = fmaxf(most, fabsf(v[j]));
        most = fmaxf(most, __shfl_xor(most, 16));
        return fmaxf(most, __shfl_xor(most, 32));
    };
    float most = largest();
    if (__any(most == INFINITY)) {
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] = fabsf(v[j]) < INFINITY ? v[j] : NAN;
        most = largest();
    }
    const int e = block_exponent(most);
    const float inv = pow2(-e);
    i8 q;
#pragma unroll
    for (int t = 0; t < 8; t++) q[t] = to_e4m3(v[4 * t] * inv, v[4 * t + 1] * inv, v[4 * t + 2] * inv, v[4 * t + 3] * inv);
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

// A lane's 32 values of block kb of a row, four at a time.  In a block that the row's end cuts off, a group of four that would
// pass the end is read so that it ends there and moved into place afterwards.
template <typename X>
struct RawBlock {
    struct Four { X v[4]; } f[8];
    static __device__ __forceinline__ int moved(int w, int g, int left) { return max(16 * w + 4 * g + 4 - left, 0); }
    __device__ __forceinline__ void load(const X *row, long long kb, int cols, int g)
    {
        const X *x = row + kb * 128;
        const int left = (int)min((long long)cols - kb * 128, 128ll);
        if (cols >= 4) {
#pragma unroll
            for (int w = 0; w < 8; w++) __builtin_memcpy(&f[w], x + (16 * w + 4 * g - moved(w, g, left)), sizeof(Four));
        } else {
#pragma unroll
            for (int w = 0; w < 8; w++)
#pragma unroll
                for (int r = 0; r < 4; r++) f[w].v[r] = w == 0 ? x[min(r, cols - 1)] : X(0);
        }
    }
    // live: the row exists
    __device__ __forceinline__ void values(float (&out)[32], bool live, long long kb, int cols, int g) const
    {
        const int left = (int)min((long long)cols - kb * 128, 128ll);
#pragma unroll
        for (int w = 0; w < 8; w++) {
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = live ? to_f32(f[w].v[r]) : 0.0f;
            if (left < 128) {
                const int by = cols >= 4 ? moved(w, g, left) : 0;
                if (by & 1) v[0] = v[1], v[1] = v[2], v[2] = v[3];
                if (by & 2) v[0] = v[2], v[1] = v[3];
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (16 * w + 4 * g + r >= left) v[r] = 0.0f;
            }
#pragma unroll
            for (int r = 0; r < 4; r++) out[4 * w + r] = v[r];
        }
    }
};

// One wave per tile of 16 rows x 128 columns: 8192 x 8192 bf16 in 41 us, 4.9 TB/s.  NORM: the values are normalised first, (v - mean[column]) * dev[column]
// (Normalize, nn.cpp:702-716).
template <typename X, bool NORM = false>
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
        RawBlock<X> raw;
        raw.load(src, kb, p.cols, g);
        raw.values(v, live, kb, p.cols, g);
        if constexpr (NORM) {
#pragma unroll
            for (int j = 0; j < 32; j++) {
                const long long k = kb * 128 + column_of(g, j);
                if (live && k < p.cols) v[j] = (v[j] - p.mean[k]) * p.dev[k];
            }
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

// LCRC_ACT_SIGMOID on the hardware's 2^x and reciprocal (1 ulp each)
__device__ __forceinline__ float sigmoid(float v)
{
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
}
// LCRC_ACT_FSIGMOID.  FEXP (fexp.h:14-21): the exponent's bits of a double from one truncated product; out of range as x86
// converts it
__device__ __forceinline__ float fsigmoid(float v)
{
    const float y = -v;
    int i = __double2int_rz(1048576.0 / 0.69314718055994530942 * (double)y);
    if (!(y < 0x1.62e43p+10f)) i = (int)0x80000000u;
    return 1.0f / (1.0f + (float)__hiloint2double((int)((unsigned)i + 1072632447u), 0));
}
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act)
{
    if (act == LCRC_ACT_SIGMOID) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = sigmoid(v[i]);
    } else if (act == LCRC_ACT_FSIGMOID) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = fsigmoid(v[i]);
    }
}

// ---- the sums ----
// The 8-bit matrix instructions multiply exactly, but inside a group of eight products (eight bytes of a lane that follow one
// another) they cut every product off 13 bits below the group's largest one before they add (measured, for the scaled and the
// plain form alike: 2^16 + 3 * 2^3 comes out whole, of 2^16 + 3 * 7 the sevens are gone); the groups' sums are added in 32
// bits.  That is up to 7 * 2^-13 = 0.22 * 2^-8 of the products' absolute sum, 1.4e-5 of it on normal values: beside the rounding
// of a result to bf16, 2^-8, it changes the neighbour that 4 (276 inputs) to 16 (8192) of 1000 results are rounded to and not
// their distance from the definition (rms 1.6597e-3 of them, with sums in 32 bits 1.6595e-3).  It is more than f16's rounding,
// 2^-11; too much for a result in 32 bits; and for one in 8, whose rounding turns 1.4e-5 into a whole step, 2^-3, wherever it
// lies that near to a border: a net with hidden values in 8 bits was off by 5.5e-4 of its results where sums in 32 bits leave
// 2.1e-4.  So products with results in anything but bf16 turn their operands into bf16 --
// exact: 4 significant bits, the block's scale goes into bf16's exponent (v_cvt_scalef32_pk_bf16_fp8; below 2^-126 it loses
// bits) -- and use the bf16 instruction, whose sums are f32 throughout: half the rate.
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

// a block's scale from its byte; 255 is no number
__device__ __forceinline__ float block_scale(int byte) { return byte == 255 ? NAN : __int_as_float(byte << 23); }

// acc += A B over one block of 128 columns with sums in 32 bits; as / bs: the block's scale byte of the lane's row, in the low byte
__device__ __forceinline__ f4 exact_product(const i8 &a, const i8 &b, f4 acc, int as, int bs)
{
    const float sa = block_scale(as & 255), sb = block_scale(bs & 255);
#pragma unroll
    for (int s = 0; s < 4; s++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(a, s, sa), to_bf16(b, s, sb), acc, 0, 0, 0);
    return acc;
}

// D = W X^T per tile of 16 x 16: lane (c, g) holds outputs 4 g + r (register r) of x row c.

// four outputs o .. o + 3 of a row, as they lie in a lane; o is a multiple of 4
template <typename Y>
__device__ __forceinline__ void store_four(Y *row, long long o, int n_out, const float *v)
{
    if (o + 4 <= n_out) {
        struct Four { Y v[4]; } f = {{(Y)v[0], (Y)v[1], (Y)v[2], (Y)v[3]}};
        __builtin_memcpy(row + o, &f, sizeof(f));
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (o + r < n_out) row[o + r] = (Y)v[r];
    }
}
__device__ __forceinline__ void store_rows(const Fp8ProductParams &p, long long row, long long o, const float *v)
{
    if (row >= p.rows) return;
    if (p.y_type == LCRC_T_F32) store_four(static_cast<float *>(p.y) + row * p.ldy, o, p.n_out, v);
    else if (p.y_type == LCRC_T_F16) store_four(static_cast<_Float16 *>(p.y) + row * p.ldy, o, p.n_out, v);
    else store_four(static_cast<__bf16 *>(p.y) + row * p.ldy, o, p.n_out, v);
}
// A lane's 32 outputs o .. o + 127 of rows row0 .. row0 + 15, turned in LDS (`turn`, this wave's own) so that 16 lanes write
// 256 consecutive bytes of a row: written as they lie in the registers, 32 bytes of a row at a time, they cost 2 to 3 times
// as long.  (Rows of 288 bytes in LDS: eight lanes' writes of 8 bytes meet no bank twice.)
constexpr int kTurnRow = 256 + 32, kTurn = 16 * kTurnRow;
template <typename Y>
__device__ __forceinline__ void store_block(const Fp8ProductParams &p, long long row0, long long o, int lane, const float (&v)[32], unsigned char *turn)
{
    constexpr int kOutputs = 256 / sizeof(Y), E = 16 / sizeof(Y);
    struct Four { Y v[4]; };
    struct Chunk { Y v[E]; };
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int half = 0; half < 128 / kOutputs; half++) {
#pragma unroll
        for (int n = 0; n < kOutputs / 16; n++) {
            const float *f = v + 4 * (half * (kOutputs / 16) + n);
            const Four q = {{(Y)f[0], (Y)f[1], (Y)f[2], (Y)f[3]}};
            __builtin_memcpy(__builtin_assume_aligned(turn + c * kTurnRow + (16 * n + 4 * g) * (int)sizeof(Y), 8), &q, sizeof(q));
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const long long at = o + half * kOutputs + c * E;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 4 * i + g;
            Chunk q;
            __builtin_memcpy(&q, __builtin_assume_aligned(turn + r * kTurnRow + c * 16, 16), 16);
            if (row0 + r >= p.rows) continue;
            Y *y = static_cast<Y *>(p.y) + (row0 + r) * p.ldy + at;
            if (at + E <= p.n_out) __builtin_memcpy(y, &q, 16);
            else
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (at + e < p.n_out) y[e] = q.v[e];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}
// the bias of outputs o .. o + 3 (0 without one; what lies behind the last output is not used)
__device__ __forceinline__ f4 bias_of(const Fp8ProductParams &p, long long o)
{
    f4 b = {0.f, 0.f, 0.f, 0.f};
    if (!p.bias) return b;
    if (o + 4 <= p.n_out) __builtin_memcpy(&b, p.bias + o, sizeof(b));
    else
#pragma unroll
        for (int r = 0; r < 4; r++) b[r] = p.bias[min(o + r, (long long)p.n_out - 1)];
    return b;
}
// a lane's 32 outputs of row 16 t + c, block ob of 128, as the tile (t, ob) of the 8-bit form; what fills it up is 0
__device__ __forceinline__ void store_held(const Fp8ProductParams &p, const Q8Shape &sy, long long t, long long ob, int lane, float (&v)[32])
{
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < 32; j++)
        if (16 * t + c >= p.rows || 128 * ob + column_of(g, j) >= p.n_out) v[j] = 0.0f;
    unsigned char *y = static_cast<unsigned char *>(p.y);
    int e;
    const i8 q = quantise(v, &e);
    store_tile(y + (t * sy.kb + ob) * kQTileBytes, lane, q);
    unsigned char *scales = y + sy.scales_at() + ((t * sy.kb4 + ob / 4) * 16 + c) * 4;
    if (g == 0) scales[ob & 3] = (unsigned char)(e + 127);
    if (ob == sy.kb - 1 && g > (ob & 3)) scales[g] = 127;
}

typedef unsigned char __attribute__((address_space(3))) *lds_bytes;

// N bytes for each lane from base + lane_offset + offset to the LDS, lane by lane, past the registers.  (As a buffer load: with
// one on its way, a wait for LDS reads that were asked for before it need not become a wait for all of them.)
template <int N>
__device__ __forceinline__ void copy_to_lds(const unsigned char *base, unsigned lane_offset, int offset, unsigned char *to)
{
#ifdef __HIP_DEVICE_COMPILE__               // (the host has no such type)
    const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(base), 0, -1, 0x00027000);
    if constexpr (N == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (lds_bytes)to, 16, lane_offset, offset, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (lds_bytes)to, 4, lane_offset, offset, 0, 0);
#endif
}

// block J of a group of four, scale bytes J of the groups' dwords
template <bool EXACT, int J>
__device__ __forceinline__ f4 scaled_product(const i8 &a, const i8 &b, f4 acc, int as, int bs)
{
    if constexpr (EXACT) return exact_product(a, b, acc, as >> (8 * J), bs >> (8 * J));
    else return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, J, as, J, bs);
}

template <typename F, int... M>
__device__ __forceinline__ void for_each(const F &f, std::integer_sequence<int, M...>)
{
    (f(std::integral_constant<int, M>()), ...);
}

// A workgroup of WW x WX waves makes 16 FW WW outputs of 16 FX WX rows, each wave FW x FX tiles in its registers.
// 256 x 128, two workgroups to a CU so that one copies and reads while the other multiplies: 8192^3 to bf16 in 431 - 475 us,
// 2.3 - 2.55 PFLOP/s (first version, operands straight from memory, 1630; 256 x 256 with a wave to a SIMD 535 - 570, nothing
// runs beside its epilogue).  With bf16 operands (EXACT, 128 x 128): 8192^3 to f16 901 us, 4096 x 2048 x 8192 140 - 150.  Small
// tiles are chains of sixteen blocks: 777 x 1999 x 2309 to bf16 14.6 us, to f16 19.5; a third stage of LDS changes nothing there.
template <bool EXACT, int FW, int FX, int WW, int WX, int STAGES = 1>
__global__ __launch_bounds__(64 * WW * WX, 2) void fp8_tile_kernel(const Fp8ProductParams p, int across, int down)
{
    constexpr int kWaves = WW * WX, TW = FW * WW, TX = FX * WX, PW = 2 * TW / kWaves, PX = 2 * TX / kWaves, kPiece = kQTileBytes / 2;
    static_assert(FW == 8 && PW * kWaves == 2 * TW && PX * kWaves == 2 * TX, "whole blocks of outputs; the copies are shared out evenly");
    constexpr int kStage = (TW + TX) * kQTileBytes;
    __shared__ __attribute__((aligned(16))) unsigned char stages[STAGES * kStage];
    __shared__ __attribute__((aligned(16))) unsigned char scale_stages[2 * (TW + TX) * 64];
    const Q8Shape sx(p.rows, p.n_in), sw(p.n_out, p.n_in), sy(p.rows, p.n_out);
    const int lane = threadIdx.x & 63, c = lane & 15, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ww = wave % WW, wx = wave / WW;
    // Workgroup i runs on XCD i mod 8, each with an L2 of its own: an XCD takes a run of neighbouring tiles, eight rows of
    // tiles by columns, so that what runs together shares its operands.
    const long long all = (long long)across * down, per = (all + 7) / 8;
    const long long id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || id >= all) return;
    const long long band = id / (8ll * across), in_band = id - band * 8 * across, high = min(8ll, down - band * 8);
    const long long tx = band * 8 + in_band % high, tw = in_band / high;

    // the copies of a wave: pieces of 1 KB, half a tile, from where they lie behind the workgroup's first tile (n_in <= 2^23:
    // within 32 bits)
    const unsigned char *const w0 = p.w + tw * TW * sw.kb * kQTileBytes, *const x0 = p.x + tx * TX * sx.kb * kQTileBytes;
    const int w_left = (int)min(sw.rt - tw * TW, (long long)TW) - 1, x_left = (int)min(sx.rt - tx * TX, (long long)TX) - 1;
    const unsigned tile_stride = (unsigned)sx.kb * kQTileBytes, scale_stride = (unsigned)sx.kb4 * 64;
    unsigned wp[PW], xp[PX];
#pragma unroll
    for (int q = 0; q < PW; q++) wp[q] = min((wave * PW + q) >> 1, w_left) * tile_stride + (q & 1) * kPiece + lane * 16;
#pragma unroll
    for (int q = 0; q < PX; q++) xp[q] = min((wave * PX + q) >> 1, x_left) * tile_stride + (q & 1) * kPiece + lane * 16;
    const auto fetch = [&](int kb, int to) {                // block kb of the operands into a stage, past the registers
        unsigned char *const stage = stages + to * kStage;
#pragma unroll
        for (int q = 0; q < PW; q++) copy_to_lds<16>(w0, wp[q], kb * kQTileBytes, stage + (wave * PW + q) * kPiece);
#pragma unroll
        for (int q = 0; q < PX; q++) copy_to_lds<16>(x0, xp[q], kb * kQTileBytes, stage + (2 * TW + wave * PX + q) * kPiece);
    };
    const unsigned char *const ws = p.w + sw.scales_at() + tw * TW * sw.kb4 * 64, *const xs = p.x + sx.scales_at() + tx * TX * sx.kb4 * 64;
    const auto fetch_scales = [&](int kb4) {                // of four blocks: a dword for each row, four tiles to a copy
#pragma unroll
        for (int q = 0; q < (TW + TX) / 4; q++) {
            const int tile = 4 * q + (lane >> 4);
            if (q % kWaves != wave) continue;
            const unsigned at = (4 * q < TW ? min(tile, w_left) : min(tile - TW, x_left)) * scale_stride + c * 4;
            copy_to_lds<4>(4 * q < TW ? ws : xs, at, kb4 * 64, scale_stages + (kb4 & 1) * (TW + TX) * 64 + q * 256);
        }
    };
    int s[FW + FX];

    f4 acc[FW][FX];
#pragma unroll
    for (int n = 0; n < FW; n++)
#pragma unroll
        for (int m = 0; m < FX; m++) acc[n][m] = f4{0.f, 0.f, 0.f, 0.f};
    const int blocks = (int)sx.kb;
    const auto step = [&](int kb, auto j) {
        constexpr int J = decltype(j)::value;
        // this wave's copies of the block have arrived (a barrier alone does not wait for them), its reads of the one before are done
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                       // ... and everyone's
        asm volatile("" ::: "memory");
        const unsigned char *const stage = stages + (kb % STAGES) * kStage;
        if constexpr (J == 0) {
            const int *const rows = reinterpret_cast<const int *>(scale_stages + (kb >> 2 & 1) * (TW + TX) * 64) + c;
#pragma unroll
            for (int n = 0; n < FW; n++) s[n] = rows[16 * (ww * FW + n)];
#pragma unroll
            for (int m = 0; m < FX; m++) s[FW + m] = rows[16 * (TW + wx * FX + m)];
        }
        i8 a[FW], b[FX];
        a[0] = load_tile(stage + ww * FW * kQTileBytes, lane);
#pragma unroll
        for (int m = 0; m < FX; m++) b[m] = load_tile(stage + (TW + wx * FX + m) * kQTileBytes, lane);
#pragma unroll
        for (int n = 1; n < FW; n++) a[n] = load_tile(stage + (ww * FW + n) * kQTileBytes, lane);
        if constexpr (STAGES == 1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();                   // ... and read by all
        }
        __builtin_amdgcn_sched_barrier(0);
        // on its way while the products run (behind the last block: that one again, without a branch around the copies)
        fetch(min(kb + 1, blocks - 1), (kb + 1) % STAGES);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < FW; n++)
#pragma unroll
            for (int m = 0; m < FX; m++) acc[n][m] = scaled_product<EXACT, J>(a[n], b[m], acc[n][m], s[n], s[FW + m]);
    };
    fetch_scales(0);
    fetch(0, 0);
    for (int kb = 0; kb < blocks; kb += 4) {
        step(kb, std::integral_constant<int, 0>());
        if (kb + 4 < blocks) fetch_scales(kb / 4 + 1);
        if (kb + 1 < blocks) step(kb + 1, std::integral_constant<int, 1>());
        if (kb + 2 < blocks) step(kb + 2, std::integral_constant<int, 2>());
        if (kb + 3 < blocks) step(kb + 3, std::integral_constant<int, 3>());
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // (no copy outlives the workgroup's LDS)

    const long long ob = tw * WW + ww;                      // the wave's block of 128 outputs
    f4 bias[FW];
#pragma unroll
    for (int n = 0; n < FW; n++) bias[n] = bias_of(p, 128 * ob + 16 * n + 4 * (lane >> 4));
    const auto finish = [&](auto which) {
        constexpr int m = decltype(which)::value;
        const long long t = tx * TX + wx * FX + m;
        float v[32];
#pragma unroll
        for (int n = 0; n < FW; n++)
#pragma unroll
            for (int r = 0; r < 4; r++) v[4 * n + r] = acc[n][m][r] + bias[n][r];
        activate(v, p.act);
        if (p.y_type == LCRC_T_E4M3) {
            if (t < sy.rt && ob < sy.kb) store_held(p, sy, t, ob, lane, v);
        } else if (p.y_type == LCRC_T_F32) store_block<float>(p, 16 * t, 128 * ob, lane, v, stages + wave * kTurn);
        else if (p.y_type == LCRC_T_F16) store_block<_Float16>(p, 16 * t, 128 * ob, lane, v, stages + wave * kTurn);
        else store_block<__bf16>(p, 16 * t, 128 * ob, lane, v, stages + wave * kTurn);
    };
    static_assert(kWaves * kTurn <= STAGES * kStage, "the stages hold the turned results");
    __syncthreads();                                        // the stages are read
    // (spelled out: an accumulator with an index that is not known when compiling would leave the registers)
    for_each(finish, std::make_integer_sequence<int, FX>());
}

// (5 x 8192 x 8192, bf16 to f32: 19 us, 3.5 TB/s of weights, first version 229 in two launches; 1 x 276 x 1500: 4 us.)
// Few rows, or few results for a long sum: the waves of a workgroup share out the blocks of the sum, each for all of the
// workgroup's 16 FW outputs x 16 FX rows, and the partial results are added up in LDS, in the waves' order.  Operands come
// straight from memory.  X: rows of that type, which every wave converts for its own blocks (FX = 1), or unsigned char: rows
// in the 8-bit form.
template <bool EXACT, typename X, int FW, int FX, int NW>
__global__ __launch_bounds__(64 * NW) void fp8_split_kernel(const Fp8ProductParams p, const void *x_rows, long long ldx)
{
    constexpr bool kRaw = sizeof(X) > 1;
    static_assert(!kRaw || FX == 1, "one tile of rows is converted");
    constexpr int U = FW <= 2 && sizeof(X) < 4 ? 2 : 1;     // blocks on their way at once (what the registers hold)
    extern __shared__ __attribute__((aligned(16))) f4 parts[];           // [NW][FW * FX][64]
    const Q8Shape sx(p.rows, p.n_in), sw(p.n_out, p.n_in), sy(p.rows, p.n_out);
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long w0 = (long long)blockIdx.x * FW, t0 = (long long)blockIdx.y * FX;
    const X *row = kRaw ? static_cast<const X *>(x_rows) + (c < p.rows ? c : 0) * ldx : nullptr;
    f4 acc[FW][FX];
#pragma unroll
    for (int n = 0; n < FW; n++)
#pragma unroll
        for (int m = 0; m < FX; m++) acc[n][m] = f4{0.f, 0.f, 0.f, 0.f};
    for (long long k0 = wave; k0 < sx.kb; k0 += U * NW) {
        i8 a[U][FW], b[U][FX];
        int as[U][FW], bs[U][FX];
        RawBlock<X> raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long kb = min(k0 + u * NW, sx.kb - 1);
#pragma unroll
            for (int n = 0; n < FW; n++) {
                const long long t = min(w0 + n, sw.rt - 1);
                a[u][n] = load_tile(p.w + (t * sw.kb + kb) * kQTileBytes, lane);
                as[u][n] = p.w[sw.scales_at() + ((t * sw.kb4 + (kb >> 2)) * 16 + c) * 4 + (kb & 3)];
            }
            if constexpr (kRaw) raw[u].load(row, kb, p.n_in, g);
            else
#pragma unroll
                for (int m = 0; m < FX; m++) {
                    const long long t = min(t0 + m, sx.rt - 1);
                    b[u][m] = load_tile(p.x + (t * sx.kb + kb) * kQTileBytes, lane);
                    bs[u][m] = p.x[sx.scales_at() + ((t * sx.kb4 + (kb >> 2)) * 16 + c) * 4 + (kb & 3)];
                }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long kb = k0 + u * NW;
            if (kb >= sx.kb) break;
            if constexpr (kRaw) {
                float v[32];
                int e;
                raw[u].values(v, c < p.rows, kb, p.n_in, g);
                b[u][0] = quantise(v, &e);
                bs[u][0] = e + 127;
            }
#pragma unroll
            for (int n = 0; n < FW; n++)
#pragma unroll
                for (int m = 0; m < FX; m++) acc[n][m] = scaled_product<EXACT, 0>(a[u][n], b[u][m], acc[n][m], as[u][n], bs[u][m]);
        }
    }
#pragma unroll
    for (int n = 0; n < FW; n++)
#pragma unroll
        for (int m = 0; m < FX; m++) parts[(wave * FW * FX + m * FW + n) * 64 + lane] = acc[n][m];
    __syncthreads();
    const auto total = [&](int tile) {
        f4 v = parts[tile * 64 + lane];
        for (int w = 1; w < NW; w++) v += parts[(w * FW * FX + tile) * 64 + lane];
        return v;
    };
    if constexpr (FW == 8) {                                // whole blocks of outputs: the 8-bit form
        if (wave >= FX) return;
        float v[32];
#pragma unroll
        for (int n = 0; n < 8; n++) {
            const f4 sum = total(wave * 8 + n) + bias_of(p, 16 * (w0 + n) + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; r++) v[4 * n + r] = sum[r];
        }
        activate(v, p.act);
        if (t0 + wave < sy.rt) store_held(p, sy, t0 + wave, blockIdx.x, lane, v);
    } else {
        for (int tile = wave; tile < FW * FX; tile += NW) {
            const long long o = 16 * (w0 + tile % FW) + 4 * g;
            const f4 sum = total(tile) + bias_of(p, o);
            float v[4] = {sum[0], sum[1], sum[2], sum[3]};
            activate(v, p.act);
            store_rows(p, 16 * (t0 + tile / FW) + c, o, v);
        }
    }
}

template <bool EXACT, typename X, int FW, int FX, int NW>
void split_launch(const Fp8ProductParams &p, const void *x, long long ldx, hipStream_t stream)
{
    const dim3 grid((unsigned)(((long long)p.n_out + 16 * FW - 1) / (16 * FW)), (unsigned)(((long long)p.rows + 16 * FX - 1) / (16 * FX)));
    fp8_split_kernel<EXACT, X, FW, FX, NW><<<grid, 64 * NW, NW * FW * FX * 1024, stream>>>(p, x, ldx);
}
template <bool EXACT, typename X>
void split_launch(const Fp8ProductParams &p, const void *x, long long ldx, hipStream_t stream)
{
    const bool deep = p.n_in > 128 * 4;
    if (p.y_type == LCRC_T_E4M3) {
        if constexpr (EXACT) {
            if (deep) split_launch<EXACT, X, 8, 1, 8>(p, x, ldx, stream);
            else split_launch<EXACT, X, 8, 1, 4>(p, x, ldx, stream);
        }
        return;
    }
    if constexpr (sizeof(X) == 1) {
        if (p.rows > 32) {
            if (deep) split_launch<EXACT, X, 1, 4, 16>(p, x, ldx, stream);
            else split_launch<EXACT, X, 1, 4, 4>(p, x, ldx, stream);
            return;
        }
        if (p.rows > 16) {
            if (deep) split_launch<EXACT, X, 1, 2, 16>(p, x, ldx, stream);
            else split_launch<EXACT, X, 1, 2, 4>(p, x, ldx, stream);
            return;
        }
    }
    if (!deep) split_launch<EXACT, X, 1, 1, 4>(p, x, ldx, stream);
    else if (p.n_out >= 16 * 512) split_launch<EXACT, X, 2, 1, 16>(p, x, ldx, stream);
    else split_launch<EXACT, X, 1, 1, 16>(p, x, ldx, stream);
}
template <typename X>
hipError_t split_by_sums(const Fp8ProductParams &p, const void *x, long long ldx, hipStream_t stream)
{
    if (fp8_sums_in_32_bits(p.y_type)) split_launch<true, X>(p, x, ldx, stream);
    else split_launch<false, X>(p, x, ldx, stream);
    return hipGetLastError();
}

template <bool EXACT, int FW, int FX, int WW, int WX, int STAGES = 1>
void tile_launch(const Fp8ProductParams &p, hipStream_t stream)
{
    const long long across = ((long long)p.n_out + 16 * FW * WW - 1) / (16 * FW * WW), down = ((long long)p.rows + 16 * FX * WX - 1) / (16 * FX * WX);
    const long long blocks = (across * down + 7) / 8 * 8;
    static_assert(WW * WX == 4, "fp8_route's tiles are 256 threads each");
    fp8_tile_kernel<EXACT, FW, FX, WW, WX, STAGES><<<(unsigned)blocks, 64 * WW * WX, 0, stream>>>(p, (int)across, (int)down);
}

}  // namespace

hipError_t fp8_pack_launch(const Fp8PackParams &p, hipStream_t stream)
{
    const Q8Shape s(p.rows, p.cols);
    const unsigned blocks = (unsigned)((s.rt * s.kb + 3) / 4);
    if (p.mean) {
        fp8_pack_kernel<float, true><<<blocks, 256, 0, stream>>>(p);
        return hipGetLastError();
    }
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
    const bool exact = fp8_sums_in_32_bits(p.y_type);
    switch (fp8_route(p.rows, p.n_in, p.n_out, p.y_type)) {
    case kFp8SharedSums: return split_by_sums<unsigned char>(p, nullptr, 0, stream);
    case kFp8Tiles256x128: tile_launch<false, 8, 4, 2, 2>(p, stream); break;          // (not with sums in 32 bits)
    case kFp8Tiles128x128:
        if (exact) tile_launch<true, 8, 2, 1, 4>(p, stream);
        else tile_launch<false, 8, 2, 1, 4>(p, stream);
        break;
    case kFp8Tiles128x64:
        if (exact) tile_launch<true, 8, 1, 1, 4, 2>(p, stream);
        else tile_launch<false, 8, 1, 1, 4, 2>(p, stream);
        break;
    }
    return hipGetLastError();
}

hipError_t fp8_few_rows_launch(const Fp8ProductParams &p, const void *x, int x_type, long long ldx, hipStream_t stream)
{
    if (x_type == LCRC_T_F32) return split_by_sums<float>(p, x, ldx, stream);
    if (x_type == LCRC_T_F16) return split_by_sums<_Float16>(p, x, ldx, stream);
    return split_by_sums<__bf16>(p, x, ldx, stream);
}

}  // namespace phnrec
