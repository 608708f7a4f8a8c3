// 8-bit forward: what the quantising kernels and the integer product share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace chebykan {
namespace int8 {

// |q| <= 128 on both sides and an int32 sum: 131071 * 2^14 < 2^31
constexpr int64_t MAX_K = 131071;

inline int64_t in_pad(int64_t in) { return round_up(in, 16); }

// Few rows on the CUDA cores: every row adds to row_kernel's time, while a tile of up to 128 costs the same; four rows as
// long as 48 KB of shared memory hold.  Measured (us, row_kernel / split_kernel): 8192 -> 1024 with 2 rows 3.4 / 13, 4 rows 5.2 / 13.5,
// 8 rows 23 / 13.5; 2048 -> 8192 with 4 rows 7.9 / 10.5, 8 rows 15 / 11; 512 -> 2048 with 8 rows 5.3 / 5.3; 16000 -> 1024 with 4 rows
// 25 / 17.
inline bool few_rows(int64_t M, int64_t K) { return M <= 2 || (M <= 4 && M * K <= 48 * 1024) || (M <= 8 && K <= 512); }

struct Product {
    const int8_t* q;          // [M][K], rows ldq bytes apart
    const float* q_scale;     // [M]
    const int8_t* wq;         // [N][K], rows ldw bytes apart
    const float* w_scale;     // [N]
    const float* bias;        // [N] or null
    void* y;                  // [M][N]
    int dtype;
    int64_t M, N, K, ldq, ldw;
};

template <typename T> __device__ __forceinline__ T to_type(float v);
template <> __device__ __forceinline__ float to_type<float>(float v) { return v; }
template <> __device__ __forceinline__ __half to_type<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 to_type<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// bytes of scratch the product needs, and the product itself
int64_t matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t ldq, int64_t ldw);
// `after`: the kernel before it in the stream writes q and lets it start early (launch_after)
int launch_matmul(const Product& p, void* ws, int32_t* status, cudaStream_t s, bool after);

}  // namespace int8
}  // namespace chebykan
