// Newton-Schulz orthogonalisation: the data layout shared by the packing kernels and the products.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace chebykan {
namespace ns {

// A matrix is worked on with its shorter side as rows: X[s][l], s <= l.  Operands are fp16 planes: the value times a
// power of two, rounded (plane 0), and in FP32X3 mode also the remainder, rounded (plane 1): 11 or 22 significant
// bits.  Plane p of matrix b is slab b*planes + p of [rows][pitch], pitches rounded up to 8 elements (16 bytes).
//
// Powers of two.  The entries of X_k (k >= 1), A and P are bounded by the singular values (|x| <= 1.21, |A| <= 1.45,
// |P| <= 10 under the usual coefficients; up to 7, 49 and 4000 under others that are accepted), while typical
// entries are 1/sqrt(l).  So X and A carry 2^10 and P 2^4: the largest accepted stay below fp16's 65504, and the
// remainders of typical entries stay above its smallest numbers.  X_0 is stored as G * 2^k with its Frobenius norm in
// [2^14, 2^15): exact in the exponent, so that 16-bit gradients are not rounded a second time.  The factors that turn
// stored numbers into values are kept per matrix: alpha[0][b] = 1 / (max(|G|, eps) 2^k) for X_0 and alpha[1][b], a power
// of two, for the later X: 2^-X_EXP, and less where |G| is so far below eps that the steps cannot bring X back to 1.
constexpr int X_EXP = 10, A_EXP = 10, P_EXP = 4;

struct Shape {
    int batch, s, l;      // matrices, rows (shorter side), columns
    int ss, ls;           // pitches of A / P and of X
    int planes;           // 2 in FP32X3 mode, 1 in TF32 mode
    __host__ __device__ int64_t x_slab() const { return (int64_t)s * ls; }
    __host__ __device__ int64_t a_slab() const { return (int64_t)s * ss; }
};

struct Workspace {        // byte offsets of the buffers
    int64_t x0, x1, a, p, o, partial, alpha, total;
};

// per-matrix partial sums of squares written by the norm kernels
constexpr int NORM_BLOCKS = 64;

__device__ __forceinline__ void split_half(float v, __half& hi, __half& lo) {
    hi = __float2half_rn(v);
    lo = __float2half_rn(v - __half2float(hi));
}

// A = X X^T with X = alpha[b] * stored
int launch_gram(const __half* x, __half* a, const float* alpha, const Shape& sh, int32_t* status, cudaStream_t s);
// P = ca I + cb A + cc A A
int launch_poly(const __half* a, __half* p, float ca, float cb, float cc, const Shape& sh, int32_t* status, cudaStream_t s);
// X' = P X as planes (x_next, stored over alpha_next[b]), or as fp32 [batch][s][l] (o) where x_next is null
int launch_apply(const __half* p, const __half* x, __half* x_next, float* o, const float* alpha, const float* alpha_next,
                 const Shape& sh, int32_t* status, cudaStream_t s);

}  // namespace ns
}  // namespace chebykan
