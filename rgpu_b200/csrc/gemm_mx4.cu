// Product of two microscaled 4-bit matrices, C[m,n] = A[m,k] B[n,k]^T.
#include "mx4.cuh"

namespace rt {
namespace {

using namespace mx4;

// 64 x 64 outputs by 256 threads, 4 x 4 each; one block of 32 of k at a time,
// decoded into shared memory.
template <typename T>
__global__ void __launch_bounds__(256) product_kernel(rt_mx4 a, rt_mx4 b, T* __restrict__ c, int64_t ldc,
                                                      const float* __restrict__ bias, int relu) {
    __shared__ float sa[32][65], sb[32][65];
    const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t blocks = a.blocks(), groups = a.groups();
    float acc[4][4] = {};
    for (int64_t kb = 0; kb < blocks; ++kb) {
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int r = i >> 4, p = i & 15;
            uint32_t ca = 0, cb = 0;
            float va = 0.0f, vb = 0.0f;
            if (m0 + r < a.rows) {
                ca = a.codes[((m0 + r) * blocks + kb) * 16 + p];
                va = scale_value(a.scales[scale_offset(m0 + r, kb, groups)]);
            }
            if (n0 + r < b.rows) {
                cb = b.codes[((n0 + r) * blocks + kb) * 16 + p];
                vb = scale_value(b.scales[scale_offset(n0 + r, kb, groups)]);
            }
            sa[2 * p][r] = decode(ca & 15u) * va;
            sa[2 * p + 1][r] = decode(ca >> 4) * va;
            sb[2 * p][r] = decode(cb & 15u) * vb;
            sb[2 * p + 1][r] = decode(cb >> 4) * vb;
        }
        __syncthreads();
        for (int kk = 0; kk < 32; ++kk)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[kk][ty * 4 + i], sb[kk][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t row = m0 + ty * 4 + i, col = n0 + tx * 4 + j;
            if (row >= a.rows || col >= b.rows) continue;
            float v = acc[i][j] + (bias ? bias[col] : 0.0f);
            if (relu) v = v < 0.0f ? 0.0f : v;
            if constexpr (sizeof(T) == 2)
                c[row * ldc + col] = __float2bfloat16_rn(v);
            else
                c[row * ldc + col] = v;
        }
}

}  // namespace

int launch_gemm_mx4(rt_ctx* ctx, const rt_mx4& a, const rt_mx4& b, const rt_tensor& c, const float* bias, bool relu,
                    cudaStream_t stream) {
    const dim3 grid((unsigned)((b.rows + 63) / 64), (unsigned)((a.rows + 63) / 64));
    if (c.dtype == RT_BF16)
        product_kernel<<<grid, 256, 0, stream>>>(a, b, static_cast<__nv_bfloat16*>(c.ptr), c.ld, bias, (int)relu);
    else
        product_kernel<<<grid, 256, 0, stream>>>(a, b, static_cast<float*>(c.ptr), c.ld, bias, (int)relu);
    RT_CUDA(cudaGetLastError());
    count_launch(ctx);
    return RT_OK;
}

}  // namespace rt
