// Muon update and Newton-Schulz orthogonalisation: norms, packing of the operands, the weights' update, entry points.
//
//   X_0 = G / max(|G|_F, eps),  A = X X^T,  P = a I + b A + c A^2,  X <- P X   (steps times, shorter side as rows)
//
// The steps are products (ns_gemm.cu); the kernels here read the gradient twice (its norm is needed before the first
// operand can be scaled) and the result once.
#include <math.h>
#include "newton_schulz.cuh"

namespace chebykan {
namespace ns {
namespace {

// sum over the block in a fixed order; the total is returned to thread 0
__device__ __forceinline__ double block_sum(double v, double* smem) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_down_sync(0xffffffffu, v, d);
    if (lane == 0) smem[warp] = v;
    __syncthreads();
    double t = 0.;
    if (threadIdx.x == 0)
        for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += smem[w];
    __syncthreads();
    return t;
}

// partial[b][block] = sum of squares (in double: no gradient's square over- or underflows, and the sum over millions of
// elements keeps its digits)
template <typename T>
__global__ void __launch_bounds__(256) norm_kernel(StridedSource<T> src, int64_t m, int64_t n, double* partial) {
    __shared__ double smem[8];
    double v = 0.;
    for (int64_t e = blockIdx.x * 256 + threadIdx.x; e < m * n; e += (int64_t)gridDim.x * 256) {
        const double g = src.load(blockIdx.y, e / n, e % n);
        v += g * g;
    }
    v = block_sum(v, smem);
    if (threadIdx.x == 0) partial[blockIdx.y * NORM_BLOCKS + blockIdx.x] = v;
}

// momentum update of the whole tensor and, per degree, the partial sums of squares of the update u.  The active threads
// are a multiple of deg+1, so a thread stays on one degree as the block strides along the contiguous tensor.
__global__ void __launch_bounds__(256)
momentum_kernel(const float* __restrict__ grad, float* __restrict__ buf, int64_t n, int dp1, float momentum, int nesterov,
                float gs, double* __restrict__ partial) {
    __shared__ double smem[256];
    const int active = 256 / dp1 * dp1;
    double v = 0.;
    if ((int)threadIdx.x < active)
        for (int64_t e = blockIdx.x * (int64_t)active + threadIdx.x; e < n; e += (int64_t)gridDim.x * active) {
            const float g = grad[e] * gs;
            const float m = fmaf(1.f - momentum, g - buf[e], buf[e]);
            buf[e] = m;
            const double u = nesterov ? fmaf(momentum, m - g, g) : m;
            v += u * u;
        }
    smem[threadIdx.x] = v;
    __syncthreads();
    if ((int)threadIdx.x < dp1) {
        double t = 0.;
        for (int k = threadIdx.x; k < active; k += dp1) t += smem[k];
        partial[(int64_t)threadIdx.x * NORM_BLOCKS + blockIdx.x] = t;
    }
}

// X_0 planes of one matrix tile: 32 x 32 elements, transposed on the way where the matrix is tall
template <typename Src>
__global__ void __launch_bounds__(256)
pack_kernel(Src src, int64_t m, int64_t n, __half* __restrict__ x, float* __restrict__ alpha, const double* __restrict__ partial,
            float eps, int growth, Shape sh) {
    __shared__ float tile[32][33];
    __shared__ double pow2;
    const int64_t b = blockIdx.z, r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;
    if (threadIdx.x == 0) {
        float al, later;
        double t = 0.;
        for (int k = 0; k < NORM_BLOCKS; ++k) t += partial[b * NORM_BLOCKS + k];
        scales_of(sqrt(t), eps, growth, &pow2, &al, &later);
        if (blockIdx.x == 0 && blockIdx.y == 0) { alpha[b] = al; alpha[sh.batch + b] = later; }
    }
    __syncthreads();
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int k = ty; k < 32; k += 8)
        if (r0 + k < m && c0 + tx < n) tile[k][tx] = (float)((double)src.load(b, r0 + k, c0 + tx) * pow2);
    __syncthreads();
    const bool tall = m > n;
    const int64_t y0 = tall ? c0 : r0, x0 = tall ? r0 : c0;
    __half* dst = x + b * sh.planes * sh.x_slab();
    for (int k = ty; k < 32; k += 8)
        if (y0 + k < sh.s && x0 + tx < sh.l) {
            __half hi, lo;
            split_half(tall ? tile[tx][k] : tile[k][tx], hi, lo);
            const int64_t at = (y0 + k) * sh.ls + x0 + tx;
            dst[at] = hi;
            if (sh.planes == 2) dst[at + sh.x_slab()] = lo;
        }
}

// out[b][m][n] from o[b][s][l]
template <typename T>
__global__ void __launch_bounds__(256) unpack_kernel(const float* __restrict__ o, T* __restrict__ out, int64_t m, int64_t n, int64_t total) {
    for (int64_t e = blockIdx.x * (int64_t)256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        const int64_t b = e / (m * n), w = e % (m * n), r = w / n, c = w % n;
        out[e] = from_float<T>(m > n ? o[b * m * n + c * m + r] : o[e]);
    }
}

// param = keep * param - step * O
__global__ void __launch_bounds__(256)
update_kernel(float* __restrict__ param, const float* __restrict__ o, int64_t in, int64_t out, int dp1, float keep, float step) {
    const int64_t total = in * out * dp1;
    for (int64_t e = blockIdx.x * (int64_t)256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        const int64_t d = e % dp1, w = e / dp1, i = w / out, c = w % out;
        const float v = o[d * in * out + (in > out ? c * in + i : w)];
        param[e] = fmaf(-step, v, keep * param[e]);
    }
}

unsigned blocks_for(int64_t n) {
    int64_t b = ceil_div(n, 256);
    return (unsigned)(b < 1 ? 1 : (b > 148 * 16 ? 148 * 16 : b));
}

int64_t a256(int64_t b) { return round_up(b, 256); }

Shape shape_of(int64_t batch, int64_t m, int64_t n, int mode) {
    Shape sh;
    sh.batch = (int)batch;
    sh.s = (int)(m < n ? m : n);
    sh.l = (int)(m < n ? n : m);
    sh.ss = (int)round_up(sh.s, 8);
    sh.ls = (int)round_up(sh.l, 8);
    sh.planes = mode == CHEBYKAN_MODE_FP32X3 ? 2 : 1;
    return sh;
}

Workspace layout_of(const Shape& sh) {
    Workspace w{};
    if (small_supported(sh)) return w;           // one launch that keeps everything on chip
    const int64_t xb = a256(2 * sh.x_slab() * sh.planes * sh.batch), ab = a256(2 * sh.a_slab() * sh.planes * sh.batch);
    int64_t at = 0;
    w.x0 = at; at += xb;
    w.x1 = at; at += xb;
    w.a = at; at += ab;
    w.p = at; at += ab;
    w.o = at; at += a256(4 * (int64_t)sh.batch * sh.s * sh.l);
    w.partial = at; at += a256(8 * (int64_t)NORM_BLOCKS * sh.batch);
    w.alpha = at; at += a256(8 * (int64_t)sh.batch);
    w.total = at;
    return w;
}

bool shape_fits(int64_t batch, int64_t m, int64_t n) {
    return batch >= 0 && batch <= 65535 && m >= 0 && n >= 0 && m <= 65536 && n <= 65536;
}

// Whether the operands' ranges hold: follows the largest singular value that the steps can reach from 1 (X_0 has a norm of
// at most 1) and the largest |P|.  *growth = log2 of the product of the latter, rounded up.
bool coefficients_ok(int64_t steps, float a, float b, float c, int* growth) {
    double top = 1., log_growth = 0.;
    for (int64_t k = 0; k < steps; ++k) {
        double next = 0., pmax = 0.;
        for (int i = 0; i <= 512; ++i) {
            const double x = top * i / 512., p = a + x * x * (b + c * x * x);
            if (!(fabs(p * x) <= 7.) || !(fabs(p) <= 4000.)) return false;      // NaN included
            next = fmax(next, fabs(p * x));
            pmax = fmax(pmax, fabs(p));
        }
        log_growth += log2(fmax(pmax, 1.));
        if (next > top) top = next;
    }
    *growth = (int)ceil(log_growth);
    return true;
}

// steps on packed operands; leaves O in o [batch][s][l]
int run_steps(char* ws, const Workspace& w, const Shape& sh, int64_t steps, float a, float b, float c, int32_t* status,
              cudaStream_t s) {
    __half* x[2] = {reinterpret_cast<__half*>(ws + w.x0), reinterpret_cast<__half*>(ws + w.x1)};
    __half* A = reinterpret_cast<__half*>(ws + w.a);
    __half* P = reinterpret_cast<__half*>(ws + w.p);
    float* o = reinterpret_cast<float*>(ws + w.o);
    const float* alpha = reinterpret_cast<const float*>(ws + w.alpha);
    for (int64_t k = 0; k < steps; ++k) {
        const float *later = alpha + sh.batch, *al = k == 0 ? alpha : later;
        int rc;
        if ((rc = launch_gram(x[k & 1], A, al, sh, status, s))) return rc;
        if ((rc = launch_poly(A, P, a, b, c, sh, status, s))) return rc;
        if ((rc = launch_apply(P, x[k & 1], k + 1 < steps ? x[(k + 1) & 1] : nullptr, o, al, later, sh, status, s))) return rc;
    }
    return CHEBYKAN_OK;
}

template <typename Src>
int launch_pack_planes(const Src& src, int64_t m, int64_t n, char* ws, const Workspace& w, const Shape& sh, float eps, int growth,
                       cudaStream_t s) {
    const dim3 grid((unsigned)ceil_div(n, 32), (unsigned)ceil_div(m, 32), (unsigned)sh.batch);
    pack_kernel<<<grid, 256, 0, s>>>(src, m, n, reinterpret_cast<__half*>(ws + w.x0), reinterpret_cast<float*>(ws + w.alpha),
                                     reinterpret_cast<const double*>(ws + w.partial), eps, growth, sh);
    return check_cuda(cudaGetLastError());
}

template <typename T>
int orthogonalize_typed(const void* g, int64_t sb, int64_t sr, int64_t sc, void* out, char* ws, const Workspace& w, const Shape& sh,
                        int64_t m, int64_t n, int64_t steps, float a, float b, float c, float eps, int growth, int32_t* status, cudaStream_t s) {
    const StridedSource<T> src{reinterpret_cast<const T*>(g), sb, sr, sc};
    norm_kernel<T><<<dim3(NORM_BLOCKS, (unsigned)sh.batch), 256, 0, s>>>(src, m, n, reinterpret_cast<double*>(ws + w.partial));
    int rc = check_cuda(cudaGetLastError());
    if (rc) return rc;
    if ((rc = launch_pack_planes(src, m, n, ws, w, sh, eps, growth, s))) return rc;
    if ((rc = run_steps(ws, w, sh, steps, a, b, c, status, s))) return rc;
    const int64_t total = sh.batch * m * n;
    unpack_kernel<T><<<blocks_for(total), 256, 0, s>>>(reinterpret_cast<const float*>(ws + w.o), reinterpret_cast<T*>(out), m, n, total);
    return check_cuda(cudaGetLastError());
}

bool ns_mode(int mode) { return mode == CHEBYKAN_MODE_FP32X3 || mode == CHEBYKAN_MODE_TF32; }
bool known_mode(int mode) { return ns_mode(mode) || mode == CHEBYKAN_MODE_FP32 || mode == CHEBYKAN_MODE_BF16; }

}  // namespace
}  // namespace ns
}  // namespace chebykan

using namespace chebykan;
using namespace chebykan::ns;

extern "C" {

int64_t chebykan_orthogonalize_workspace_bytes(int64_t batch, int64_t m, int64_t n, int mode) {
    if (!shape_fits(batch, m, n) || !known_mode(mode)) return CHEBYKAN_EINVAL;
    if (!ns_mode(mode)) return CHEBYKAN_EUNSUPPORTED;
    return layout_of(shape_of(batch, m, n, mode)).total;
}

int chebykan_orthogonalize(const void* g, int64_t stride_batch, int64_t stride_row, int64_t stride_col, int dtype, void* out,
                           void* workspace, int64_t workspace_bytes, int64_t batch, int64_t m, int64_t n, int64_t steps,
                           float a, float b, float c, float eps, int mode, int32_t* status, void* stream) {
    const int64_t need = chebykan_orthogonalize_workspace_bytes(batch, m, n, mode);
    if (need < 0) return (int)need;
    int growth = 0;
    if (stride_batch < 0 || stride_row < 0 || stride_col < 0 || dtype < CHEBYKAN_DTYPE_FP32 || dtype > CHEBYKAN_DTYPE_FP16 ||
        steps < 1 || steps > 32 || !(eps > 0.f) || !coefficients_ok(steps, a, b, c, &growth))
        return CHEBYKAN_EINVAL;
    if (batch == 0 || m == 0 || n == 0) return CHEBYKAN_OK;
    if (!g || !out || !status) return CHEBYKAN_EINVAL;
    if (!aligned16(out) || !aligned16(workspace)) return CHEBYKAN_EALIGN;
    if (workspace_bytes < need || (need > 0 && !workspace)) return CHEBYKAN_EWORKSPACE;
    int rc = check_device();
    if (rc) return rc;
    const Shape sh = shape_of(batch, m, n, mode);
    cudaStream_t s = (cudaStream_t)stream;
    if (small_supported(sh))
        return launch_small_orthogonalize(g, dtype, stride_batch, stride_row, stride_col, out, m, n, sh,
                                          {(int)steps, a, b, c, eps, growth}, status, s);
    const Workspace w = layout_of(sh);
    char* ws = reinterpret_cast<char*>(workspace);
    if (dtype == CHEBYKAN_DTYPE_FP32)
        return orthogonalize_typed<float>(g, stride_batch, stride_row, stride_col, out, ws, w, sh, m, n, steps, a, b, c, eps, growth, status, s);
    if (dtype == CHEBYKAN_DTYPE_BF16)
        return orthogonalize_typed<__nv_bfloat16>(g, stride_batch, stride_row, stride_col, out, ws, w, sh, m, n, steps, a, b, c, eps, growth, status, s);
    return orthogonalize_typed<__half>(g, stride_batch, stride_row, stride_col, out, ws, w, sh, m, n, steps, a, b, c, eps, growth, status, s);
}

int64_t chebykan_muon_workspace_bytes(int64_t in, int64_t out, int64_t deg, int mode) {
    if (in < 1 || out < 1 || deg < 0 || deg > 127 || !known_mode(mode) || !shape_fits(deg + 1, in, out)) return CHEBYKAN_EINVAL;
    if (!ns_mode(mode)) return CHEBYKAN_EUNSUPPORTED;
    return layout_of(shape_of(deg + 1, in, out, mode)).total;
}

int chebykan_muon_step(float* param, const float* grad, float* buf, void* workspace, int64_t workspace_bytes, int64_t in,
                       int64_t out, int64_t deg, float lr, float weight_decay, float momentum, int nesterov, float update_scale,
                       int64_t steps, float a, float b, float c, float eps, float grad_scale, int mode, int32_t* status,
                       void* stream) {
    const int64_t need = chebykan_muon_workspace_bytes(in, out, deg, mode);
    if (need < 0) return (int)need;
    int growth = 0;
    if (!param || !grad || !buf || !status || steps < 1 || steps > 32 || !(eps > 0.f) ||
        !(momentum >= 0.f && momentum < 1.f) || !coefficients_ok(steps, a, b, c, &growth))
        return CHEBYKAN_EINVAL;
    if (!aligned16(param) || !aligned16(grad) || !aligned16(buf) || !aligned16(workspace)) return CHEBYKAN_EALIGN;
    if (workspace_bytes < need || (need > 0 && !workspace)) return CHEBYKAN_EWORKSPACE;
    int rc = check_device();
    if (rc) return rc;
    const int dp1 = (int)deg + 1;
    const Shape sh = shape_of(dp1, in, out, mode);
    cudaStream_t s = (cudaStream_t)stream;
    if (small_supported(sh))
        return launch_small_muon(param, grad, buf, in, out, dp1, 1.f - lr * weight_decay, lr * update_scale, momentum, nesterov,
                                 grad_scale, sh, {(int)steps, a, b, c, eps, growth}, status, s);
    const Workspace w = layout_of(sh);
    char* ws = reinterpret_cast<char*>(workspace);
    momentum_kernel<<<NORM_BLOCKS, 256, 0, s>>>(grad, buf, in * out * dp1, dp1, momentum, nesterov, grad_scale,
                                                reinterpret_cast<double*>(ws + w.partial));
    if ((rc = check_cuda(cudaGetLastError()))) return rc;
    const MomentumSource src{grad, buf, out, dp1, momentum, grad_scale, nesterov};
    if ((rc = launch_pack_planes(src, in, out, ws, w, sh, eps, growth, s))) return rc;
    if ((rc = run_steps(ws, w, sh, steps, a, b, c, status, s))) return rc;
    update_kernel<<<blocks_for(in * out * dp1), 256, 0, s>>>(param, reinterpret_cast<const float*>(ws + w.o), in, out, dp1,
                                                             1.f - lr * weight_decay, lr * update_scale);
    return check_cuda(cudaGetLastError());
}

}  // extern "C"
