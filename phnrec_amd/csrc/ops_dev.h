// ops_dev.h -- what the operators on matrices in device memory (include/lcrc_pipeline.h: lcrc_score, lcrc_fp8_*) share between
// their C entries (lcrc_api_ops.cpp) and their kernels (score_kernels.hip, fp8_kernels.hip, softmax_kernels.hip).  The kernels
// are a shared object of their own, libphnrec_lcrc_ops.so, which the first call that needs one of them loads: a process
// that uses none of them -- the `phnrec` command line -- registers none with the HIP runtime.
#ifndef PHNREC_OPS_DEV_H
#define PHNREC_OPS_DEV_H

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "../../include/lcrc_pipeline.h"
#include "lcrc_dev.h"

namespace phnrec {

// ---- lcrc_score -----------------------------------------------------------------------------------------------------
constexpr int kScoreMaxTop = 64, kScoreMaxLabels = 64;
constexpr int kScoreMaxCols = 1 << 30;

// Rows of up to this many chunks of 16 bytes lie in a wave's registers, a chunk to a lane; up to so many a wave streams its
// row, beyond it a workgroup.  (30000 x 3000 f16, k = 16: streamed by a wave 77 us, 8 chunks to a lane in registers 578, the
// register file full of keys; 60000 x 1000 f32, k = 5: 68 and 101.  20000 x 4096 f32, k = 8: by a wave 65 us, by a workgroup 109;
// 12000 x 8192: 79 and 88.)
constexpr int kScoreThreads = 256, kScoreHeldChunks = 64, kScoreWaveChunks = 32 * 64;

// a row's cut into parts of so many chunks of 16 bytes, a workgroup to each
struct ScoreParts {
    int parts, chunks;
};
inline ScoreParts score_parts(int rows, int cols, int type)
{
    const int w = type == LCRC_T_F32 ? 4 : 8, n_chunks = (cols - 1) / w + 1;
    // enough workgroups for every CU to have eight, but no part below 2 chunks a thread (300 x 50001 bf16: 32 us as with
    // fewer, larger parts; 600 x 100000 f32: 54 us, with 512 workgroups 69)
    const long long most = std::min<long long>(kScoreThreads, (n_chunks + 2 * kScoreThreads - 1) / (2 * kScoreThreads));
    const long long want = rows >= 2048 ? 1 : (2048 + rows - 1) / rows;
    const int parts = (int)std::max<long long>(1, std::min(most, want)), chunks = (n_chunks - 1) / parts + 1;
    return {(n_chunks - 1) / chunks + 1, chunks};
}
// the parts' statistics (16 bytes) and lists of k keys, of either width of type: the size function does not take the type
inline size_t score_workspace_bytes(int rows, int cols, int k)
{
    size_t most = 0;
    for (const int type : {(int)LCRC_T_F32, (int)LCRC_T_BF16}) {
        const int w = type == LCRC_T_F32 ? 4 : 8;
        if ((cols - 1) / w + 1 <= kScoreWaveChunks) continue;
        const ScoreParts p = score_parts(rows, cols, type);
        if (p.parts > 1) most = std::max(most, (size_t)rows * p.parts * (16 + (size_t)k * 8));
    }
    return most;
}

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

// Which kernel makes a product (measured, us): large tiles of outputs x rows read least per product, but need two workgroups for
// every CU:
//   4096 x 8192 x 2048 bf16   256 x 128 (256 tiles) 86, 128 x 128 (512) 73, 128 x 64 100
//   777 x 1999 x 2309 bf16    128 x 128 16.4, 128 x 64 (247) 12.6, shared-out sums 27;  300 x 4000 x 1000 (40): 18, sums 11
// In short sums nothing is read often enough to count, and small tiles fill the card better:
//   8192 x 372 x 1500 in 8 bits  128 x 128 26.5, 128 x 64 25.3
enum Fp8Route { kFp8SharedSums = 0, kFp8Tiles128x64 = 1, kFp8Tiles128x128 = 2, kFp8Tiles256x128 = 3 };
inline long long fp8_tiles(int rows, int n_out, int tile_outputs, int tile_rows)
{
    return (((long long)n_out + tile_outputs - 1) / tile_outputs) * (((long long)rows + tile_rows - 1) / tile_rows);
}
// (fp8_kernels.hip: what the 8-bit matrix instructions cut off is little beside the rounding of a result in bf16, and of no other)
inline bool fp8_sums_in_32_bits(int y_type) { return y_type != LCRC_T_BF16; }
inline Fp8Route fp8_route(int rows, int n_in, int n_out, int y_type)
{
    if (fp8_tiles(rows, n_out, 128, 64) <= 128) return kFp8SharedSums;
    if (n_in <= 512) return kFp8Tiles128x64;
    if (!fp8_sums_in_32_bits(y_type) && fp8_tiles(rows, n_out, 256, 128) >= 512) return kFp8Tiles256x128;
    return fp8_tiles(rows, n_out, 128, 128) >= 512 ? kFp8Tiles128x128 : kFp8Tiles128x64;
}

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
constexpr int kQFewOut = 1 << 25;     // outputs of a product that converts its rows itself
constexpr long long kQMaxTiles = 1ll << 26;      // a matrix in the 8-bit form, x and y have fewer: 64 threads each, and a grid has fewer than 2^32
constexpr int kQMaxIn = 1 << 23;      // columns of the operands of a product: their tiles' offsets stay within 32 bits

// ---- the kernels' object ----------------------------------------------------------------------------------------------
// Its one exported symbol, lcrc_ops_table, gives the launches.  The version goes up with every change of the table or of the
// structures it hands over.
constexpr int kOpsVersion = 2;
struct OpsTable {
    int version;
    hipError_t (*score)(const lcrc_score_args &a, hipStream_t stream);
    hipError_t (*fp8_pack)(const Fp8PackParams &p, hipStream_t stream);
    hipError_t (*fp8_unpack)(const Fp8UnpackParams &p, hipStream_t stream);
    hipError_t (*fp8_product)(const Fp8ProductParams &p, hipStream_t stream);
    // up to kQRows rows of f32, f16 or bf16: converted by the product itself (p.x is not read)
    hipError_t (*fp8_few_rows)(const Fp8ProductParams &p, const void *x, int x_type, long long ldx, hipStream_t stream);
    hipError_t (*softmax_rows)(const SoftmaxRowsParams &p, hipStream_t stream);
    int (*score_most_blocks)(int most);          // of a launch from now on -> what it was
};
int score_most_blocks(int most);
hipError_t score_launch(const lcrc_score_args &a, hipStream_t stream);
hipError_t fp8_pack_launch(const Fp8PackParams &p, hipStream_t stream);
hipError_t fp8_unpack_launch(const Fp8UnpackParams &p, hipStream_t stream);
hipError_t fp8_product_launch(const Fp8ProductParams &p, hipStream_t stream);
hipError_t fp8_few_rows_launch(const Fp8ProductParams &p, const void *x, int x_type, long long ldx, hipStream_t stream);

}  // namespace phnrec
#endif
