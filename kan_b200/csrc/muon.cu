// Muon update and Newton-Schulz orthogonalisation: norms, packing of the operands, the weights' update, entry points.
//
//   X_0 = G / max(|G|_F, eps),  A = X X^T,  P = a I + b A + c A^2,  X <- P X   (steps times, shorter side as rows)
//
// The steps are products (ns_gemm.cu; ns_small.cu for small matrices); the kernels here read the gradient twice (its norm is
// needed before the first operand can be scaled) and the result once.  They are bound by memory: on 1024 x 1024 x 9 the momentum
// (151 MB) takes 32 us, packing (75 MB, half of it from L2) 14 us, the update (113 MB) 31 us.
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

// A matrix as rows that lie closest together in memory: element (r, c) at r*pitch + c*step, step <= pitch.
struct Plane {
    int64_t rows, cols, pitch, step, batch;       // batch: distance of matrices
};

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// eight neighbours from p: one or two 16-byte loads where p allows (the address is the same modulo 16 for a whole matrix,
// or the branch is a coin that all threads throw alike), else eight loads; values past `left` are zero
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t step, int64_t left, float (&v)[8]) {
    if (step == 1 && left >= 8 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        alignas(16) T t[8];
        *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(p);
        if (sizeof(T) == 4) *reinterpret_cast<uint4*>(t + 8 - 16 / sizeof(T)) = *reinterpret_cast<const uint4*>(p + 8 - 16 / sizeof(T));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = load1(t + e);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? load1(p + e * step) : 0.f;
    }
}

// partial[b][block] = sum of squares (in double: no gradient's square over- or underflows, and the sum over millions of
// elements keeps its digits).  Two groups of eight elements per thread in flight.
template <typename T>
__global__ void __launch_bounds__(256) norm_kernel(const T* __restrict__ g, const Plane pl, double* __restrict__ partial) {
    __shared__ double smem[8];
    let_next_start();
    const T* src = g + blockIdx.y * pl.batch;
    const int64_t groups = (pl.cols + 7) / 8, total = pl.rows * groups, stride = (int64_t)gridDim.x * 256;
    double v = 0.;
    for (int64_t e = blockIdx.x * 256 + threadIdx.x; e < total; e += 2 * stride) {
        float x[2][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t w = e + u * stride, r = w / groups, c = (w - r * groups) * 8;
            if (w < total) load8(src + r * pl.pitch + c * pl.step, pl.step, pl.cols - c, x[u]);
            else
#pragma unroll
                for (int k = 0; k < 8; ++k) x[u][k] = 0.f;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < 8; ++k) v = fma((double)x[u][k], (double)x[u][k], v);
    }
    v = block_sum(v, smem);
    if (threadIdx.x == 0) partial[blockIdx.y * NORM_BLOCKS + blockIdx.x] = v;
}

// Momentum of the whole tensor, and the update u turned from [in*out][deg+1] to a plane per degree, through a tile in shared
// memory (deg+1 made odd, so that a column of it meets every bank): both sides are contiguous.  With `partial` also the
// sums of squares of each degree's u.
// `width` elements of every degree: as many as 24 KB hold (so that several blocks share an SM), fewer where the tensor would
// not give every SM two tiles
int tile_width(int64_t pairs, int dp1) {
    int width = 256;
    while (width > 32 && ((dp1 | 1) * width * 4 > 24 * 1024 || ceil_div(pairs, width) < 2 * 148)) width /= 2;
    return width;
}
// quotient by dp1 of numbers below 2^16 without a division
__device__ __forceinline__ uint32_t divide(uint32_t e, uint32_t magic) { return __umulhi(e, magic); }
uint32_t magic_of(int dp1) { return dp1 == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + dp1 - 1) / dp1); }

__global__ void __launch_bounds__(256)
momentum_kernel(const float* __restrict__ grad, float* __restrict__ buf, float* __restrict__ u, int64_t pairs, int dp1, int width,
                uint32_t magic, float momentum, int nesterov, float gs, double* __restrict__ partial) {
    extern __shared__ float tile[];
    __shared__ double sums[128];
    let_next_start();
    const int odd = dp1 | 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int d = threadIdx.x; d < dp1; d += 256) sums[d] = 0.;
    const int64_t tiles = (pairs + width - 1) / width;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t p0 = t * width;
        const int count = (int)((pairs - p0 < width ? pairs - p0 : width) * dp1);
        __syncthreads();                           // the tile is free
        const float* gt = grad + p0 * dp1;
        float* bt = buf + p0 * dp1;
        auto one = [&](int e, float g, float m) {
            g *= gs;
            m = fmaf(1.f - momentum, g - m, m);
            const int w = magic ? (int)divide((uint32_t)e, magic) : e;
            tile[w * odd + e - w * dp1] = nesterov ? fmaf(momentum, m - g, g) : m;
            return m;
        };
        // tiles start on multiples of 32 elements, so on 16 bytes; three vectors of both arrays in flight per thread
        for (int e0 = threadIdx.x * 4; e0 < (count & ~3); e0 += 3 * 1024) {
            float4 g[3], m[3];
#pragma unroll
            for (int k = 0; k < 3; ++k)
                if (e0 + k * 1024 < (count & ~3)) {
                    g[k] = *reinterpret_cast<const float4*>(gt + e0 + k * 1024);
                    m[k] = *reinterpret_cast<const float4*>(bt + e0 + k * 1024);
                }
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const int e = e0 + k * 1024;
                if (e < (count & ~3))
                    *reinterpret_cast<float4*>(bt + e) = make_float4(one(e, g[k].x, m[k].x), one(e + 1, g[k].y, m[k].y),
                                                                     one(e + 2, g[k].z, m[k].z), one(e + 3, g[k].w, m[k].w));
            }
        }
        if ((int)threadIdx.x < (count & 3)) {
            const int e = (count & ~3) + threadIdx.x;
            bt[e] = one(e, gt[e], bt[e]);
        }
        __syncthreads();
        const int n = count / dp1;
        for (int d = warp; d < dp1; d += 8) {
            double v = 0.;
            for (int w = lane; w < n; w += 32) {
                const float x = tile[w * odd + d];
                u[d * pairs + p0 + w] = x;
                v = fma((double)x, (double)x, v);
            }
            if (partial != nullptr) {
#pragma unroll
                for (int k = 16; k; k >>= 1) v += __shfl_down_sync(0xffffffffu, v, k);
                if (lane == 0) sums[d] += v;       // only this warp touches degree d
            }
        }
    }
    __syncthreads();
    if (partial != nullptr)
        for (int d = threadIdx.x; d < dp1; d += 256) partial[(int64_t)d * NORM_BLOCKS + blockIdx.x] = sums[d];
}

// param = keep * param - step * O, O one plane per degree: the same tile the other way
__global__ void __launch_bounds__(256)
update_kernel(float* param, const float* o, int64_t pairs, int dp1, int width, uint32_t magic, float keep, float step) {
    extern __shared__ float tile[];
    wait_for_previous();
    const int odd = dp1 | 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t tiles = (pairs + width - 1) / width;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t p0 = t * width;
        const int n = (int)(pairs - p0 < width ? pairs - p0 : width), count = n * dp1;
        __syncthreads();
        for (int d = warp; d < dp1; d += 8) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (lane + k * 32 < n) x[k] = __ldcg(o + d * pairs + p0 + lane + k * 32);     // see launch_after
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (lane + k * 32 < n) tile[(lane + k * 32) * odd + d] = x[k];
        }
        __syncthreads();
        float* pt = param + p0 * dp1;
        auto one = [&](int e, float p) {
            const int w = magic ? (int)divide((uint32_t)e, magic) : e;
            return fmaf(-step, tile[w * odd + e - w * dp1], keep * p);
        };
        for (int e0 = threadIdx.x * 4; e0 < (count & ~3); e0 += 3 * 1024) {
            float4 p[3];
#pragma unroll
            for (int k = 0; k < 3; ++k)
                if (e0 + k * 1024 < (count & ~3)) p[k] = *reinterpret_cast<const float4*>(pt + e0 + k * 1024);
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const int e = e0 + k * 1024;
                if (e < (count & ~3))
                    *reinterpret_cast<float4*>(pt + e) = make_float4(one(e, p[k].x), one(e + 1, p[k].y), one(e + 2, p[k].z), one(e + 3, p[k].w));
            }
        }
        if ((int)threadIdx.x < (count & 3)) {
            const int e = (count & ~3) + threadIdx.x;
            pt[e] = one(e, pt[e]);
        }
    }
}

// the scales of a matrix from its partial sums, by the block (thread 0 writes them; a barrier follows in the caller)
__device__ __forceinline__ void block_scales(const double* partial, float eps, int growth, double* pow2, float* alpha, float* later) {
    __shared__ double smem[8];
    double t = 0.;
    for (int k = threadIdx.x; k < NORM_BLOCKS; k += 256) t += __ldcg(partial + k);
    t = block_sum(t, smem);
    if (threadIdx.x == 0) scales_of(sqrt(t), eps, growth, pow2, alpha, later);
}

// X_0 planes where X's rows are the rows of the source: eight columns per thread
template <typename T, int PLANES>
__global__ void __launch_bounds__(256)
pack_rows_kernel(const T* g, const Plane pl, __half* x, float* alpha, const double* partial,
                 float eps, int growth, Shape sh) {
    __shared__ double pow2;
    __shared__ float scales[2];
    const int64_t b = blockIdx.y;
    let_next_start();
    wait_for_previous();
    block_scales(partial + b * NORM_BLOCKS, eps, growth, &pow2, &scales[0], &scales[1]);
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) { alpha[b] = scales[0]; alpha[sh.batch + b] = scales[1]; }
    const int64_t groups = sh.ls / 8, total = sh.s * groups;
    __half* dst = x + b * PLANES * sh.x_slab();
    for (int64_t w = blockIdx.x * (int64_t)256 + threadIdx.x; w < total; w += (int64_t)gridDim.x * 256) {
        const int64_t r = w / groups, c = (w - r * groups) * 8;
        float v[8];
        load8(g + b * pl.batch + r * pl.pitch + c * pl.step, pl.step, pl.cols - c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)((double)v[e] * pow2);
        uint32_t hi[4], lo[4];
        split8<PLANES>(v, hi, lo);
        *reinterpret_cast<uint4*>(dst + w * 8) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (PLANES == 2) *reinterpret_cast<uint4*>(dst + w * 8 + sh.x_slab()) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}

// X_0 planes where X's rows are the source's columns: tiles of 32 source rows x 64 source columns turned in shared memory
template <typename T, int PLANES>
__global__ void __launch_bounds__(256)
pack_turned_kernel(const T* g, const Plane pl, __half* x, float* alpha, const double* partial,
                   float eps, int growth, Shape sh) {
    __shared__ float tile[64][33];                 // [source column = X row][source row = X column]
    __shared__ double pow2;
    __shared__ float scales[2];
    const int64_t b = blockIdx.z, r0 = blockIdx.y * 32, c0 = blockIdx.x * 64;
    let_next_start();
    wait_for_previous();
    block_scales(partial + b * NORM_BLOCKS, eps, growth, &pow2, &scales[0], &scales[1]);
    __syncthreads();
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) { alpha[b] = scales[0]; alpha[sh.batch + b] = scales[1]; }
    {
        const int c = (threadIdx.x & 7) * 8, r = threadIdx.x >> 3;
        float v[8];
        if (r0 + r < pl.rows && c0 + c < pl.cols) load8(g + b * pl.batch + (r0 + r) * pl.pitch + (c0 + c) * pl.step, pl.step, pl.cols - c0 - c, v);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) tile[c + e][r] = (float)((double)v[e] * pow2);
    }
    __syncthreads();
    const int row = threadIdx.x >> 2, col = (threadIdx.x & 3) * 8;          // 64 rows of X x 4 groups of 8 columns
    if (c0 + row >= sh.s || r0 + col >= sh.ls) return;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[row][col + e];
    uint32_t hi[4], lo[4];
    split8<PLANES>(v, hi, lo);
    __half* dst = x + b * PLANES * sh.x_slab() + (c0 + row) * sh.ls + r0 + col;
    *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (PLANES == 2) *reinterpret_cast<uint4*>(dst + sh.x_slab()) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
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

// `update`: the Muon step's, which also holds u, one fp32 plane per degree (and later O in its place)
Workspace layout_of(const Shape& sh, bool update) {
    Workspace w{};
    const int64_t ub = update ? a256(4 * (int64_t)sh.batch * sh.s * sh.l) : 0;
    if (small_supported(sh)) { w.total = ub; return w; }           // one launch that keeps everything else on chip
    const int64_t xb = a256(2 * sh.x_slab() * sh.planes * sh.batch), ab = a256(2 * sh.a_slab() * sh.planes * sh.batch);
    int64_t at = 0;
    w.x0 = at; at += xb;
    w.x1 = at; at += xb;
    w.a = at; at += ab;
    w.p = at; at += ab;
    w.u = at; at += ub;
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
        // P = a + b y + c y^2 and the new value x P over y = x^2 in [0, top^2]: the ends, P's vertex, and where
        // d(x P)/dx = a + 3 b y + 5 c y^2 vanishes
        const double A = a, B = b, C = c, Y = top * top;
        double at[5] = {0., Y, -1., -1., -1.};
        if (C != 0.) {
            at[2] = -B / (2 * C);
            const double disc = 9 * B * B - 20 * A * C;
            if (disc >= 0.) {
                at[3] = (-3 * B + sqrt(disc)) / (10 * C);
                at[4] = (-3 * B - sqrt(disc)) / (10 * C);
            }
        } else if (B != 0.) {
            at[3] = -A / (3 * B);
        }
        double next = 0., pmax = 0.;
        for (double y : at) {
            if (!(y >= 0. && y <= Y)) continue;
            const double p = A + y * (B + C * y), v = fabs(p) * sqrt(y);
            if (!(v <= 7.) || !(fabs(p) <= 4000.)) return false;      // NaN included
            next = fmax(next, v);
            pmax = fmax(pmax, fabs(p));
        }
        log_growth += log2(fmax(pmax, 1.));
        if (next > top) top = next;
    }
    *growth = (int)ceil(log_growth);
    return true;
}

// steps on packed operands; leaves the result in o [batch][m][n]
int run_steps(char* ws, const Workspace& w, const Shape& sh, const Steps& st, void* o, int dtype, bool tall, int32_t* status, cudaStream_t s) {
    __half* x[2] = {reinterpret_cast<__half*>(ws + w.x0), reinterpret_cast<__half*>(ws + w.x1)};
    __half* A = reinterpret_cast<__half*>(ws + w.a);
    __half* P = reinterpret_cast<__half*>(ws + w.p);
    const float* alpha = reinterpret_cast<const float*>(ws + w.alpha);
    for (int k = 0; k < st.n; ++k) {
        const float *later = alpha + sh.batch, *al = k == 0 ? alpha : later;
        int rc;
        if ((rc = launch_gram(x[k & 1], A, al, sh, status, s))) return rc;
        if ((rc = launch_poly(A, P, st.a, st.b, st.c, sh, status, s))) return rc;
        if (k + 1 < st.n) rc = launch_apply(P, x[k & 1], x[(k + 1) & 1], al, later, sh, status, s);
        else rc = launch_apply_last(P, x[k & 1], o, dtype, tall, al, sh, status, s);
        if (rc) return rc;
    }
    return CHEBYKAN_OK;
}

// [batch][m][n] with the given strides, with the closer one inside
Plane plane_of(int64_t m, int64_t n, int64_t sb, int64_t sr, int64_t sc, bool* swapped) {
    *swapped = sr < sc;
    return *swapped ? Plane{n, m, sc, sr, sb} : Plane{m, n, sr, sc, sb};
}

template <typename T, int PLANES>
int pack_planes(const T* g, const Plane& pl, bool turned, char* ws, const Workspace& w, const Shape& sh, const Steps& st, cudaStream_t s) {
    __half* x = reinterpret_cast<__half*>(ws + w.x0);
    float* alpha = reinterpret_cast<float*>(ws + w.alpha);
    const double* partial = reinterpret_cast<const double*>(ws + w.partial);
    if (turned) {
        const dim3 grid((unsigned)ceil_div(pl.cols, 64), (unsigned)ceil_div(pl.rows, 32), (unsigned)sh.batch);
        return check_cuda(launch_after(true, pack_turned_kernel<T, PLANES>, grid, dim3(256), 0, s, 0, g, pl, x, alpha, partial, st.eps, st.growth, sh));
    } else {
        // about four groups per thread, so that the norm's partial sums are not added up by too many blocks
        int64_t blocks = ceil_div((int64_t)sh.s * sh.ls / 8, 4 * 256);
        return check_cuda(launch_after(true, pack_rows_kernel<T, PLANES>, dim3((unsigned)blocks, (unsigned)sh.batch), dim3(256), 0, s, 0, g, pl, x, alpha,
                                       partial, st.eps, st.growth, sh));
    }
}
template <typename T>
int pack(const T* g, const Plane& pl, bool turned, char* ws, const Workspace& w, const Shape& sh, const Steps& st, cudaStream_t s) {
    return sh.planes == 2 ? pack_planes<T, 2>(g, pl, turned, ws, w, sh, st, s) : pack_planes<T, 1>(g, pl, turned, ws, w, sh, st, s);
}

template <typename T>
int orthogonalize_typed(const void* g, int dtype, int64_t sb, int64_t sr, int64_t sc, void* out, char* ws, const Workspace& w,
                        const Shape& sh, int64_t m, int64_t n, const Steps& st, int32_t* status, cudaStream_t s) {
    bool swapped;
    const Plane pl = plane_of(m, n, sb, sr, sc, &swapped);
    const T* src = reinterpret_cast<const T*>(g);
    norm_kernel<T><<<dim3(NORM_BLOCKS, (unsigned)sh.batch), 256, 0, s>>>(src, pl, reinterpret_cast<double*>(ws + w.partial));
    int rc = check_cuda(cudaGetLastError());
    if (rc) return rc;
    if ((rc = pack(src, pl, swapped != (m > n), ws, w, sh, st, s))) return rc;
    return run_steps(ws, w, sh, st, out, dtype, m > n, status, s);
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
    return layout_of(shape_of(batch, m, n, mode), false).total;
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
    const int64_t size = dtype == CHEBYKAN_DTYPE_FP32 ? 4 : 2;
    // CTAs write one matrix while others still read the next
    if (overlap(out, size * batch * m * n, g, size * ((batch - 1) * stride_batch + (m - 1) * stride_row + (n - 1) * stride_col + 1)))
        return CHEBYKAN_EOVERLAP;
    int rc = check_device();
    if (rc) return rc;
    const Shape sh = shape_of(batch, m, n, mode);
    const Steps st{(int)steps, a, b, c, eps, growth};
    cudaStream_t s = (cudaStream_t)stream;
    if (small_supported(sh))
        return launch_small(g, dtype, stride_batch, stride_row, stride_col, out, m, n, sh, st, status, s, false);
    const Workspace w = layout_of(sh, false);
    char* ws = reinterpret_cast<char*>(workspace);
    if (dtype == CHEBYKAN_DTYPE_FP32)
        return orthogonalize_typed<float>(g, dtype, stride_batch, stride_row, stride_col, out, ws, w, sh, m, n, st, status, s);
    if (dtype == CHEBYKAN_DTYPE_BF16)
        return orthogonalize_typed<__nv_bfloat16>(g, dtype, stride_batch, stride_row, stride_col, out, ws, w, sh, m, n, st, status, s);
    return orthogonalize_typed<__half>(g, dtype, stride_batch, stride_row, stride_col, out, ws, w, sh, m, n, st, status, s);
}

int64_t chebykan_muon_workspace_bytes(int64_t in, int64_t out, int64_t deg, int mode) {
    if (in < 1 || out < 1 || deg < 0 || deg > 127 || !known_mode(mode) || !shape_fits(deg + 1, in, out)) return CHEBYKAN_EINVAL;
    if (!ns_mode(mode)) return CHEBYKAN_EUNSUPPORTED;
    return layout_of(shape_of(deg + 1, in, out, mode), true).total;
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
    const int64_t bytes = 4 * in * out * (deg + 1);
    if (overlap(param, bytes, grad, bytes) || overlap(param, bytes, buf, bytes) || overlap(buf, bytes, grad, bytes)) return CHEBYKAN_EOVERLAP;
    int rc = check_device();
    if (rc) return rc;
    const int dp1 = (int)deg + 1;
    const Shape sh = shape_of(dp1, in, out, mode);
    const Steps st{(int)steps, a, b, c, eps, growth};
    const Workspace w = layout_of(sh, true);
    char* ws = reinterpret_cast<char*>(workspace);
    float* u = reinterpret_cast<float*>(ws + w.u);
    cudaStream_t s = (cudaStream_t)stream;
    const bool small = small_supported(sh);
    const int64_t pairs = in * out;
    const int width = tile_width(pairs, dp1), smem = (dp1 | 1) * width * 4;
    const int64_t tiles = ceil_div(pairs, width);
    const uint32_t magic = magic_of(dp1);
    // a block of the norm's partial sums each, also where it has no tile
    const unsigned blocks = (unsigned)(small && tiles < NORM_BLOCKS ? tiles : NORM_BLOCKS);
    momentum_kernel<<<blocks, 256, smem, s>>>(grad, buf, u, pairs, dp1, width, magic, momentum, nesterov, grad_scale,
                                              small ? nullptr : reinterpret_cast<double*>(ws + w.partial));
    if ((rc = check_cuda(cudaGetLastError()))) return rc;
    const float keep = 1.f - lr * weight_decay, step = lr * update_scale;
    // O takes u's place
    if (small) {
        rc = launch_small(u, CHEBYKAN_DTYPE_FP32, pairs, out, 1, u, in, out, sh, st, status, s, true);
    } else {
        if ((rc = pack(u, Plane{in, out, out, 1, pairs}, in > out, ws, w, sh, st, s))) return rc;
        rc = run_steps(ws, w, sh, st, u, CHEBYKAN_DTYPE_FP32, in > out, status, s);
    }
    if (rc) return rc;
    return check_cuda(launch_after(true, update_kernel, dim3((unsigned)(tiles < 148 * 8 ? tiles : 148 * 8)), dim3(256), smem, s, 0, param, u, pairs, dp1,
                                   width, magic, keep, step));
}

}  // extern "C"
