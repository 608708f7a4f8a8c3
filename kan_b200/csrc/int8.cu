// 8-bit forward of a Chebyshev layer: packing of the coefficients, quantised basis rows, entry points.
//
//   T_d = T_d(tanh x), d = 1..deg;  scale = max |T| / 127 over the row;  q = round(T / scale)
//
// Degree 0 is the constant 1 and lives in the bias.  A row with any input near zero has |T_2| close to 1, so from
// degree 2 on the scale is all but 1/127; it is taken from the row all the same, because a row of small inputs into
// a layer of degree 1 would lose most of its 8 bits to a fixed one.
#include "int8.cuh"

namespace chebykan {
namespace int8 {
namespace {

// tanh: a series below 0.3 (relative error below 1e-7), above it the exponential form, whose error is absolute: a row of
// small inputs would show that, scaled up to 127 steps
__device__ __forceinline__ float tanh_of(float x) {
    if (fabsf(x) < 0.3f) {
        const float z = x * x;
        float p = -0.0088632355f;                 // -1382/155925
        p = fmaf(p, z, 0.021869488f);             // 62/2835
        p = fmaf(p, z, -0.053968254f);            // -17/315
        p = fmaf(p, z, 0.13333333f);              // 2/15
        p = fmaf(p, z, -0.33333333f);
        return fmaf(x * z, p, x);
    }
    return tanh_fast(x);
}

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// eight values from p (values past `left` are zero): 16-byte loads where the rows allow
template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, bool vec, float (&v)[8]) {
    if (vec && left >= 8) {
        alignas(16) T t[8];
        *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(p);
        if (sizeof(T) == 4) *reinterpret_cast<uint4*>(t + 8 - 16 / sizeof(T)) = *reinterpret_cast<const uint4*>(p + 8 - 16 / sizeof(T));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = load1(t + e);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? load1(p + e) : 0.f;
    }
}

// round(v * inv) for four values with |v * inv| < 128, as bytes: adding 1.5 * 2^23 leaves the rounded integer (ties to
// even) in the low bits of the sum, whose lowest bytes a byte permutation collects.  A conversion instruction per value
// has a quarter of the throughput.
__device__ __forceinline__ uint32_t quantise4(const float (&v)[8], int at, float inv) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(fmaf(v[at + e], inv, 12582912.f));
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// A row per group of G threads, eight neighbouring inputs per thread and chunk.  The first pass finds the row's largest
// |T_d|, the second evaluates the recurrence again and writes it; tanh, by far the dearer part, is kept in registers in
// between (CHUNKS per thread; 0: rows longer than that evaluate it twice).
// Bound by issue slots and memory alike: 32768 x 2048, degree 4 moves 268 MB in and 268 MB out.
template <typename T, int G, int CHUNKS>
__global__ void __launch_bounds__(256)
basis_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale, int64_t B, int in, int pad, int deg, int vec) {
    constexpr int ROWS = 256 / G, KEEP = CHUNKS ? CHUNKS : 1;
    __shared__ float red[8];
    const int lane = threadIdx.x % G;
    const int64_t row = blockIdx.x * (int64_t)ROWS + threadIdx.x / G;
    const bool live = row < B;
    const T* src = x + row * in;
    let_next_start();
    const int chunks = CHUNKS ? CHUNKS : (pad + 8 * G - 1) / (8 * G);
    float t[KEEP][8];
    float top = 0.f;
    bool nan = false;
#pragma unroll
    for (int c = 0; c < chunks; ++c) {
        float (&tc)[8] = t[CHUNKS ? c : 0];
        const int i0 = (c * G + lane) * 8;
        if (live && i0 < in) {
            load8(src + i0, in - i0, vec, tc);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                tc[e] = tanh_of(tc[e]);
                nan = nan || tc[e] != tc[e];
            }
            // from degree 2 on inputs past the row's end would count as T_2(0) = -1
            const int n = in - i0 < 8 ? in - i0 : 8;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n) {
                    float a = tc[e], b = 1.f;
                    const float tt = 2.f * a;
                    top = fmaxf(top, fabsf(a));
                    for (int d = 2; d <= deg; ++d) {
                        const float next = fmaf(tt, a, -b);
                        b = a; a = next;
                        top = fmaxf(top, fabsf(a));
                    }
                }
        }
    }
    if (nan) top = __int_as_float(0x7f800000);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (G > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
        __syncthreads();
        const int w0 = threadIdx.x / G * (G / 32);
#pragma unroll
        for (int w = 0; w < G / 32; ++w) top = fmaxf(top, red[w0 + w]);
    }
    if (!live) return;
    const bool bad = top > 3.f;                    // |T_d| <= 1 up to rounding
    const float s = bad ? __int_as_float(0x7fc00000) : __fdiv_rn(top, 127.f);
    const float inv = (bad || s == 0.f) ? 0.f : __fdiv_rn(1.f, s);
    if (lane == 0) scale[row] = s;
    int8_t* dst = q + row * (int64_t)deg * pad;
#pragma unroll
    for (int c = 0; c < chunks; ++c) {
        float (&tc)[8] = t[CHUNKS ? c : 0];
        const int i0 = (c * G + lane) * 8;
        if (i0 >= pad) continue;
        const int n = in - i0;                     // inputs of the chunk; the rest of the padded row is zero
        if (CHUNKS == 0 && n > 0) {
            load8(src + i0, n, vec, tc);
#pragma unroll
            for (int e = 0; e < 8; ++e) tc[e] = tanh_of(tc[e]);
        }
        float a[8], b[8];
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
        if (bad) keep0 = keep1 = 0;
        else if (n < 8) {
            keep0 = n <= 0 ? 0 : (n >= 4 ? keep0 : (1u << (8 * n)) - 1u);
            keep1 = n <= 4 ? 0 : (1u << (8 * (n - 4))) - 1u;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            a[e] = tc[e]; b[e] = 1.f;
            tc[e] *= 2.f;
        }
        for (int d = 1; d <= deg; ++d) {
            *reinterpret_cast<uint2*>(dst + (int64_t)(d - 1) * pad + i0) = make_uint2(quantise4(a, 0, inv) & keep0, quantise4(a, 4, inv) & keep1);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float next = fmaf(tc[e], a[e], -b[e]);
                b[e] = a[e]; a[e] = next;
            }
        }
    }
}

// one block per output: its scale, its 8-bit coefficients [deg][pad] and its bias
__global__ void __launch_bounds__(256)
pack_kernel(const float* __restrict__ c, int8_t* __restrict__ wq, float* __restrict__ w_scale, float* __restrict__ bias, int in,
            int out, int deg, int pad) {
    __shared__ float redm[8];
    __shared__ double reds[8];
    const int o = blockIdx.x, dp1 = deg + 1, warp = threadIdx.x >> 5;
    float top = 0.f;
    double sum = 0.;
    bool bad = false;
    for (int i = threadIdx.x; i < in; i += 256) {
        const float* p = c + ((int64_t)i * out + o) * dp1;
        sum += p[0];
        for (int d = 1; d <= deg; ++d) {
            bad = bad || !(fabsf(p[d]) <= 3.4e38f);
            top = fmaxf(top, fabsf(p[d]));
        }
    }
    if (bad) top = __int_as_float(0x7f800000);
#pragma unroll
    for (int k = 16; k; k >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        sum += __shfl_xor_sync(0xffffffffu, sum, k);
    }
    if ((threadIdx.x & 31) == 0) { redm[warp] = top; reds[warp] = sum; }
    __syncthreads();
    sum = 0.;
    for (int w = 0; w < 8; ++w) { top = fmaxf(top, redm[w]); sum += reds[w]; }
    bad = top > 3.4e38f;
    const float s = bad ? __int_as_float(0x7fc00000) : __fdiv_rn(top, 127.f);
    if (threadIdx.x == 0) { w_scale[o] = s; bias[o] = (float)sum; }
    for (int i = threadIdx.x; i < pad; i += 256)
        for (int d = 1; d <= deg; ++d) {
            int v = 0;
            if (i < in && !bad && s > 0.f) {
                v = __float2int_rn(__fdiv_rn(c[((int64_t)i * out + o) * dp1 + d], s));
                v = v > 127 ? 127 : (v < -127 ? -127 : v);
            }
            wq[((int64_t)o * deg + d - 1) * pad + i] = (int8_t)v;
        }
}

template <typename T, int G, int CHUNKS>
int launch_basis_one(const T* x, int8_t* q, float* scale, int64_t B, int64_t in, int64_t deg, cudaStream_t s) {
    const int vec = (in * sizeof(T)) % 16 == 0;
    basis_kernel<T, G, CHUNKS><<<(unsigned)ceil_div(B, 256 / G), 256, 0, s>>>(x, q, scale, B, (int)in, (int)in_pad(in), (int)deg, vec);
    return check_cuda(cudaGetLastError());
}
// the narrowest group that needs at most two chunks per thread: more rows per block, fewer idle threads at a row's end
template <typename T>
int launch_basis_typed(const void* x, int8_t* q, float* scale, int64_t B, int64_t in, int64_t deg, cudaStream_t s) {
    const T* xt = reinterpret_cast<const T*>(x);
    const int64_t pad = in_pad(in);
    if (pad <= 256) return launch_basis_one<T, 32, 1>(xt, q, scale, B, in, deg, s);
    if (pad <= 512) return launch_basis_one<T, 32, 2>(xt, q, scale, B, in, deg, s);
    if (pad <= 1024) return launch_basis_one<T, 64, 2>(xt, q, scale, B, in, deg, s);
    if (pad <= 2048) return launch_basis_one<T, 256, 1>(xt, q, scale, B, in, deg, s);
    if (pad <= 4096) return launch_basis_one<T, 256, 2>(xt, q, scale, B, in, deg, s);
    return launch_basis_one<T, 256, 0>(xt, q, scale, B, in, deg, s);
}

int launch_basis(const void* x, int dtype, int8_t* q, float* scale, int64_t B, int64_t in, int64_t deg, cudaStream_t s) {
    if (dtype == CHEBYKAN_DTYPE_FP32) return launch_basis_typed<float>(x, q, scale, B, in, deg, s);
    if (dtype == CHEBYKAN_DTYPE_BF16) return launch_basis_typed<__nv_bfloat16>(x, q, scale, B, in, deg, s);
    return launch_basis_typed<__half>(x, q, scale, B, in, deg, s);
}

bool dtype_ok(int dtype) { return dtype >= CHEBYKAN_DTYPE_FP32 && dtype <= CHEBYKAN_DTYPE_FP16; }
// row numbers are 32-bit inside the kernels, and a tile may reach past the last row
constexpr int64_t MAX_ROWS = 0x7fffffff - 4096;
// B rows of in values: the layer limits of the other entry points and an exact integer sum
bool layer_ok(int64_t B, int64_t in, int64_t out, int64_t deg) {
    return B >= 0 && B <= MAX_ROWS && in >= 1 && in <= (1 << 20) && out >= 1 && out <= (1 << 20) && deg >= 1 && deg <= 127 &&
           in_pad(in) * deg <= MAX_K;
}
bool product_ok(int64_t M, int64_t N, int64_t K, int64_t ldq, int64_t ldw) {
    return M >= 0 && M <= MAX_ROWS && N >= 1 && N <= (1 << 20) && K >= 0 && K <= MAX_K && ldq >= K && ldw >= K &&
           ldq <= ((int64_t)1 << 32) && ldw <= ((int64_t)1 << 32);
}
int64_t a256(int64_t b) { return round_up(b, 256); }

}  // namespace
}  // namespace int8
}  // namespace chebykan

using namespace chebykan;
using namespace chebykan::int8;

extern "C" {

int chebykan_int8_pack_coeffs(const float* coeffs, int8_t* wq, float* w_scale, float* bias, int64_t in, int64_t out,
                              int64_t deg, void* stream) {
    if (!layer_ok(0, in, out, deg) || !coeffs || !wq || !w_scale || !bias) return CHEBYKAN_EINVAL;
    if (!aligned16(coeffs) || !aligned16(wq) || !aligned16(w_scale) || !aligned16(bias)) return CHEBYKAN_EALIGN;
    int rc = check_device();
    if (rc) return rc;
    int8::pack_kernel<<<(unsigned)out, 256, 0, (cudaStream_t)stream>>>(coeffs, wq, w_scale, bias, (int)in, (int)out, (int)deg,
                                                                       (int)in_pad(in));
    return check_cuda(cudaGetLastError());
}

int chebykan_int8_basis(const void* x, int dtype, int8_t* q, float* scale, int64_t B, int64_t in, int64_t deg, void* stream) {
    if (!layer_ok(B, in, 1, deg) || !dtype_ok(dtype)) return CHEBYKAN_EINVAL;
    if (B == 0) return CHEBYKAN_OK;
    if (!x || !q || !scale) return CHEBYKAN_EINVAL;
    if (!aligned16(x) || !aligned16(q) || !aligned16(scale)) return CHEBYKAN_EALIGN;
    int rc = check_device();
    if (rc) return rc;
    return launch_basis(x, dtype, q, scale, B, in, deg, (cudaStream_t)stream);
}

int64_t chebykan_int8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t ldq, int64_t ldw) {
    if (!product_ok(M, N, K, ldq, ldw)) return CHEBYKAN_EINVAL;
    return matmul_workspace_bytes(M, N, K, ldq, ldw);
}

int chebykan_int8_matmul(const int8_t* q, int64_t ldq, const float* q_scale, const int8_t* wq, int64_t ldw,
                         const float* w_scale, const float* bias, void* y, int dtype, void* workspace, int64_t workspace_bytes,
                         int64_t M, int64_t N, int64_t K, int32_t* status, void* stream) {
    if (!product_ok(M, N, K, ldq, ldw) || !dtype_ok(dtype)) return CHEBYKAN_EINVAL;
    if (M == 0) return CHEBYKAN_OK;
    if ((K > 0 && (!q || !wq)) || !q_scale || !w_scale || !y || !status) return CHEBYKAN_EINVAL;
    if (!aligned16(q) || !aligned16(wq) || !aligned16(y) || !aligned16(workspace)) return CHEBYKAN_EALIGN;
    const int64_t need = matmul_workspace_bytes(M, N, K, ldq, ldw);
    if (workspace_bytes < need || (need > 0 && !workspace)) return CHEBYKAN_EWORKSPACE;
    int rc = check_device();
    if (rc) return rc;
    return launch_matmul({q, q_scale, wq, w_scale, bias, y, dtype, M, N, K, ldq, ldw}, workspace, status, (cudaStream_t)stream, false);
}

int64_t chebykan_int8_fwd_workspace_bytes(int64_t B, int64_t in, int64_t out, int64_t deg) {
    if (!layer_ok(B, in, out, deg)) return CHEBYKAN_EINVAL;
    const int64_t K = in_pad(in) * deg;
    return a256(B * K) + a256(B * 4) + a256(matmul_workspace_bytes(B, out, K, K, K));
}

int chebykan_int8_fwd(const void* x, int x_dtype, const int8_t* wq, const float* w_scale, const float* bias, void* y, int y_dtype,
                      void* workspace, int64_t workspace_bytes, int64_t B, int64_t in, int64_t out, int64_t deg, int32_t* status,
                      void* stream) {
    const int64_t need = chebykan_int8_fwd_workspace_bytes(B, in, out, deg);
    if (need < 0) return (int)need;
    if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype)) return CHEBYKAN_EINVAL;
    if (B == 0) return CHEBYKAN_OK;
    if (!x || !wq || !w_scale || !y || !workspace || !status) return CHEBYKAN_EINVAL;
    if (!aligned16(x) || !aligned16(wq) || !aligned16(y) || !aligned16(workspace)) return CHEBYKAN_EALIGN;
    if (workspace_bytes < need) return CHEBYKAN_EWORKSPACE;
    int rc = check_device();
    if (rc) return rc;
    const int64_t K = in_pad(in) * deg;
    char* ws = reinterpret_cast<char*>(workspace);
    int8_t* q = reinterpret_cast<int8_t*>(ws);
    float* scale = reinterpret_cast<float*>(ws + a256(B * K));
    if ((rc = launch_basis(x, x_dtype, q, scale, B, in, deg, (cudaStream_t)stream))) return rc;
    return launch_matmul({q, scale, wq, w_scale, bias, y, y_dtype, B, out, K, K, K}, ws + a256(B * K) + a256(B * 4), status,
                         (cudaStream_t)stream, true);
}

}  // extern "C"
