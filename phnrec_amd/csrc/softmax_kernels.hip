// softmax_kernels.hip -- softmax, softening functions and byte order over rows of a net's outputs in memory: the merger whose
// products ran in 8 bits (include/lcrc_pipeline.h: lcrc_set_merger_fp8).  8192 x 138: 4.5 MB read and written once, a few us.
#include <hip/hip_runtime.h>

#include "lcrc_dev.h"
#include "mlp_dev.h"
#include "ops_dev.h"

namespace phnrec {

// One wave per row, four rows per workgroup; a row's outputs in registers: up to 256 (a merger has at most 208, mlp_supports).
constexpr int J = 4;
__global__ __launch_bounds__(256) void softmax_rows_kernel(const SoftmaxRowsParams p)
{
    const int lane = threadIdx.x & 63;
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.n_rows) return;
    const float *in = p.in + row * p.n;
    float v[J], m = -3.40282346638528859812e38f, sum = 0.0f;
#pragma unroll
    for (int j = 0; j < J; j++) {
        v[j] = in[min(64 * j + lane, p.n - 1)];
        m = fmaxf(m, v[j]);
    }
    for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
#pragma unroll
    for (int j = 0; j < J; j++) {
        v[j] = 64 * j + lane < p.n ? fexp_nonpos_f(v[j] - m) : 0.0f;
        sum += v[j];
    }
    for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
#pragma unroll
    for (int j = 0; j < J; j++) {
        float q = v[j] / sum;
        q = soften(p.out_func[0], p.out_c[0], p.out_l[0], q);
        q = soften(p.out_func[1], p.out_c[1], p.out_l[1], q);
        if (p.out_be) q = __builtin_bit_cast(float, __builtin_bswap32(__builtin_bit_cast(unsigned, q)));
        if (64 * j + lane < p.n) p.out[row * p.out_ld + 64 * j + lane] = q;
    }
}

hipError_t softmax_rows_launch(const SoftmaxRowsParams &p, hipStream_t stream)
{
    const int blocks = (p.n_rows + 3) / 4;
    if (p.n > 64 * J) return hipErrorInvalidValue;
    softmax_rows_kernel<<<blocks, 256, 0, stream>>>(p);
    return hipGetLastError();
}

}  // namespace phnrec

// the launches of this object (ops_dev.h)
extern "C" __attribute__((visibility("default"))) const phnrec::OpsTable *lcrc_ops_table()
{
    static const phnrec::OpsTable table = {phnrec::kOpsVersion, phnrec::score_launch, phnrec::fp8_pack_launch, phnrec::fp8_unpack_launch, phnrec::fp8_product_launch,
                                           phnrec::fp8_few_rows_launch, phnrec::softmax_rows_launch, phnrec::score_most_blocks};
    return &table;
}
