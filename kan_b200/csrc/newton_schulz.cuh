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
    int64_t x0, x1, a, p, u, partial, alpha, total;
};

// per-matrix partial sums of squares written by the norm kernels
constexpr int NORM_BLOCKS = 148 * 6;

__device__ __forceinline__ uint32_t half2_bits(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Heads and tails of eight values as packed fp16.  The head is the value rounded to 11 bits by the splitting of Veltkamp and
// Dekker (c = 8193 v, head = c - (c - v)), which stays in fp32 and leaves two values per conversion instruction; a
// conversion each way per value is what an epilogue would otherwise spend most of its time on.  Below fp16's normal range
// the head is rounded once more, by at most 2^-25, as the tail is.
template <int PLANES>
__device__ __forceinline__ void split8(const float (&x)[8], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    if (PLANES == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) hi[e] = half2_bits(x[2 * e], x[2 * e + 1]);
        return;
    }
    const f32x2 k = pair_of(8193.f, 8193.f), minus = pair_of(-1.f, -1.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const f32x2 v = pair_of(x[2 * e], x[2 * e + 1]), c = mul2(v, k);
        const f32x2 h = fma2(fma2(v, minus, c), minus, c), t = fma2(h, minus, v);      // c - (c - v), v - h
        float a, b;
        halves(h, a, b);
        hi[e] = half2_bits(a, b);
        halves(t, a, b);
        lo[e] = half2_bits(a, b);
    }
}
// values of eight packed heads (and tails)
template <int PLANES>
__device__ __forceinline__ void join8(const uint32_t (&hi)[4], const uint32_t (&lo)[4], float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
        if (PLANES == 2) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&lo[e]));
            v.x += t.x; v.y += t.y;
        }
        x[2 * e] = v.x; x[2 * e + 1] = v.y;
    }
}

// power of two that puts the norm into [2^14, 2^15), the factor that is left of 1 / max(norm, eps), and the scale of the
// later X: growth bounds log2 of what the steps multiply a small X by, and below eps 2^-growth that leaves X under 1,
// which its scale then makes up for.  A norm that is not finite makes the whole matrix NaN.
__device__ __forceinline__ void scales_of(double norm, float eps, int growth, double* pow2, float* alpha, float* later) {
    *pow2 = 1.; *alpha = 1.f; *later = exp2f(-(float)X_EXP);
    if (!(norm <= 1.7e308)) { *alpha = __int_as_float(0x7fc00000); return; }
    if (norm == 0.) return;
    int e;
    frexp(norm, &e);                       // norm = f 2^e, f in [1/2, 1)
    *pow2 = ldexp(1., 15 - e);
    *alpha = (float)(1. / (fmax(norm, (double)eps) * *pow2));
    if (norm < eps) {
        int r;
        frexp(norm / eps, &r);             // |X_0| < 2^r
        const int up = -r - growth;
        if (up > 0) *later = (float)ldexp(1., -X_EXP - (up < 110 ? up : 110));
    }
}

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A = X X^T with X = alpha[b] * stored
int launch_gram(const __half* x, __half* a, const float* alpha, const Shape& sh, int32_t* status, cudaStream_t s);
// P = ca I + cb A + cc A A
int launch_poly(const __half* a, __half* p, float ca, float cb, float cc, const Shape& sh, int32_t* status, cudaStream_t s);
// X' = P X as planes, stored over alpha_next[b]
int launch_apply(const __half* p, const __half* x, __half* x_next, const float* alpha, const float* alpha_next, const Shape& sh,
                 int32_t* status, cudaStream_t s);
// the last step: P X, transposed back if the matrix is tall, to o [batch][m][n] of `dtype`
int launch_apply_last(const __half* p, const __half* x, void* o, int dtype, bool tall, const float* alpha, const Shape& sh,
                      int32_t* status, cudaStream_t s);

// ---- whole calls for small matrices in one launch (ns_small.cu) ----
struct Steps {
    int n;
    float a, b, c, eps;
    int growth;
};
bool small_supported(const Shape& sh);
// out may be g's own memory; after: see launch_after
int launch_small(const void* g, int dtype, int64_t sb, int64_t sr, int64_t sc, void* out, int64_t m, int64_t n, const Shape& sh,
                 const Steps& st, int32_t* status, cudaStream_t s, bool after);

}  // namespace ns
}  // namespace chebykan
