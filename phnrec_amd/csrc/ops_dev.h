// ops_dev.h -- what the operators on matrices in device memory (include/lcrc_pipeline.h: lcrc_score, lcrc_fp8_*) share between
// their C entries (lcrc_api_ops.cpp) and their kernels (score_kernels.hip, fp8_kernels.hip).
#ifndef PHNREC_OPS_DEV_H
#define PHNREC_OPS_DEV_H

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/lcrc_pipeline.h"

namespace phnrec {

// ---- lcrc_score -----------------------------------------------------------------------------------------------------
constexpr int kScoreMaxTop = 64, kScoreMaxLabels = 64;
constexpr int kScoreMaxCols = 1 << 30;

size_t score_workspace_bytes(int rows, int cols, int k);
hipError_t score_launch(const lcrc_score_args &a, hipStream_t stream);

// ---- the 8-bit matrix form ------------------------------------------------------------------------------------------
// A matrix [rows][cols] in e4m3, rows in tiles of 16, columns in blocks of 128, in the order in which a lane of
// v_mfma_scale_f32_16x16x128_f8f6f4 takes its operand.  Tile (t, kb) is 2048 bytes at (t * KB + kb) * 2048: 16 bytes of lane
// l at l * 16, its other 16 at 1024 + l * 16.  Lane l = c + 16 g holds row 16 t + c; its byte j (0..31) is column
//     128 kb + 16 (j >> 2) + 4 g + (j & 3).
// The product does not care which columns a lane holds as long as both operands agree; this order is the one in which the
// instruction's own result lies (column 4 g + r of sixteen in register r), so a product's epilogue writes its result as the
// next product's operand without moving a value between lanes.
// Behind the tiles: one byte per (row, block), the block's power of two biased by 127 (E8M0), [t][kb / 4][16 rows][kb & 3]:
// a lane's load of one dword brings the scales of four blocks.  Rows and columns that only fill a tile up hold zeros, 2^0.
constexpr int kQRows = 16, kQCols = 128, kQTileBytes = kQRows * kQCols;

struct Q8Shape {
    long long rt, kb, kb4;      // row tiles, column blocks, groups of four blocks
    __host__ __device__ Q8Shape(int rows, int cols)
        : rt(((long long)rows + kQRows - 1) / kQRows), kb(((long long)cols + kQCols - 1) / kQCols), kb4((kb + 3) / 4) {}
    __host__ __device__ long long scales_at() const { return rt * kb * kQTileBytes; }
    __host__ __device__ long long bytes() const { return scales_at() + rt * kb4 * (kQRows * 4); }
};

struct Fp8PackParams {
    const void *src;
    const unsigned char *scales;   // type e4m3: [rows][ceil(cols / 128)], biased by 127
    int type, rows, cols;
    long long ld;
    unsigned char *dst;
    const float *mean, *dev;       // type f32: [cols], or NULL: the values are normalised before they are rounded
};
struct Fp8UnpackParams {
    const unsigned char *src;
    int type, rows, cols;
    long long ld;
    void *dst;
};
struct Fp8ProductParams {
    const unsigned char *x, *w;    // [rows][n_in], [n_out][n_in] in the 8-bit form
    const float *bias;
    int rows, n_in, n_out, act, y_type;
    void *y;
    long long ldy;
};
hipError_t fp8_pack_launch(const Fp8PackParams &p, hipStream_t stream);
hipError_t fp8_unpack_launch(const Fp8UnpackParams &p, hipStream_t stream);
hipError_t fp8_product_launch(const Fp8ProductParams &p, hipStream_t stream);
// up to kQRows rows of f32, f16 or bf16: converted by the product itself (p.x is not read)
hipError_t fp8_few_rows_launch(const Fp8ProductParams &p, const void *x, int x_type, long long ldx, hipStream_t stream);
constexpr int kQFewOut = 1 << 25;     // ... and up to this many outputs
constexpr long long kQMaxTiles = 1ll << 26;      // of a matrix in the 8-bit form, of x and of y (a grid holds 2^32 threads)
constexpr int kQMaxIn = 1 << 23;      // columns of the operands of a product: their tiles' offsets stay within 32 bits

}  // namespace phnrec
#endif
