// Product of 8-bit integer matrices with a scale per row and per column.
#include "int8.cuh"

namespace chebykan {
namespace int8 {
namespace {

constexpr int T = 64, KT = 64;

// 64 x 64 outputs per block, 4 x 4 per thread, four products per instruction
template <typename OUT>
__global__ void __launch_bounds__(256) dot_kernel(const Product p) {
    __shared__ int sq[KT / 4][T + 1], sw[KT / 4][T + 1];
    const int64_t m0 = blockIdx.x * (int64_t)T, n0 = blockIdx.y * (int64_t)T;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int64_t k0 = 0; k0 < p.K; k0 += KT) {
        for (int e = threadIdx.x; e < T * KT / 4; e += 256) {
            const int k = e % (KT / 4), r = e / (KT / 4);
            uint32_t a = 0, b = 0;
            for (int j = 0; j < 4; ++j) {
                const int64_t kk = k0 + 4 * k + j;
                if (kk >= p.K) break;
                if (m0 + r < p.M) a |= (uint32_t)(uint8_t)p.q[(m0 + r) * p.ldq + kk] << (8 * j);
                if (n0 + r < p.N) b |= (uint32_t)(uint8_t)p.wq[(n0 + r) * p.ldw + kk] << (8 * j);
            }
            sq[k][r] = (int)a;
            sw[k][r] = (int)b;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KT / 4; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sq[k][ty * 4 + i], sw[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    OUT* y = reinterpret_cast<OUT*>(p.y);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m < p.M && n < p.N)
                y[m * p.N + n] = to_type<OUT>(fmaf((float)acc[i][j] * p.q_scale[m], p.w_scale[n], p.bias ? p.bias[n] : 0.f));
        }
}

template <typename OUT>
int launch_typed(const Product& p, cudaStream_t s) {
    const dim3 grid((unsigned)ceil_div(p.M, T), (unsigned)ceil_div(p.N, T));
    dot_kernel<OUT><<<grid, 256, 0, s>>>(p);
    return check_cuda(cudaGetLastError());
}
}  // namespace

int64_t matmul_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

int launch_matmul(const Product& p, void*, int32_t*, cudaStream_t s) {
    if (p.dtype == CHEBYKAN_DTYPE_FP32) return launch_typed<float>(p, s);
    if (p.dtype == CHEBYKAN_DTYPE_BF16) return launch_typed<__nv_bfloat16>(p, s);
    return launch_typed<__half>(p, s);
}

}  // namespace int8
}  // namespace chebykan
