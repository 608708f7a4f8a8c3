// The three products of a Newton-Schulz step (see newton_schulz.cuh for the operands' layout).
#include "newton_schulz.cuh"

namespace chebykan {
namespace ns {
namespace {

enum { GRAM = 0, POLY = 1, APPLY = 2 };
constexpr int T = 64, KT = 16;

struct Args {
    const __half* left;       // [M][K] planes
    const __half* right;      // GRAM, POLY: [N][K] planes; APPLY: [K][N] planes
    __half* out;              // planes [M][N], or null
    float* out32;             // fp32 [M][N] (APPLY's last step)
    const float *alpha, *alpha_next;
    int M, N, K, pitch_l, pitch_r, pitch_o, planes;
    int64_t slab_l, slab_r, slab_o;
    float ca, cb, cc;
};

__device__ __forceinline__ float value(const __half* p, int64_t slab, int planes) {
    float v = __half2float(p[0]);
    if (planes == 2) v += __half2float(p[slab]);
    return v;
}

// 64 x 64 outputs per block, 4 x 4 per thread, fp32 on the CUDA cores
template <int KIND>
__global__ void __launch_bounds__(256) product_kernel(const Args p) {
    __shared__ float sl[KT][T + 1], sr[KT][T + 1];
    const int b = blockIdx.z, m0 = blockIdx.y * T, n0 = blockIdx.x * T;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const __half* left = p.left + (int64_t)b * p.planes * p.slab_l;
    const __half* right = p.right + (int64_t)b * p.planes * p.slab_r;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += KT) {
        for (int e = threadIdx.x; e < T * KT; e += 256) {
            const int k = e % KT, r = e / KT;
            const bool okk = k0 + k < p.K;
            sl[k][r] = (okk && m0 + r < p.M) ? value(left + (int64_t)(m0 + r) * p.pitch_l + k0 + k, p.slab_l, p.planes) : 0.f;
            if (KIND != APPLY)
                sr[k][r] = (okk && n0 + r < p.N) ? value(right + (int64_t)(n0 + r) * p.pitch_r + k0 + k, p.slab_r, p.planes) : 0.f;
        }
        if (KIND == APPLY)
            for (int e = threadIdx.x; e < T * KT; e += 256) {
                const int r = e % T, k = e / T;
                sr[k][r] = (k0 + k < p.K && n0 + r < p.N)
                               ? value(right + (int64_t)(k0 + k) * p.pitch_r + n0 + r, p.slab_r, p.planes) : 0.f;
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sl[k][ty * 4 + i], sr[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    const float al = p.alpha ? p.alpha[b] : 1.f;
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m >= p.M || n >= p.N) continue;
            const int64_t at = (int64_t)b * p.planes * p.slab_o + (int64_t)m * p.pitch_o + n;
            float v;
            if (KIND == GRAM) v = acc[i][j] * al * al * exp2f((float)A_EXP);
            else if (KIND == POLY) {
                const float av = value(p.left + (int64_t)b * p.planes * p.slab_l + (int64_t)m * p.pitch_l + n, p.slab_l, p.planes) * exp2f(-(float)A_EXP);
                v = fmaf(p.cc, acc[i][j] * exp2f(-2.f * A_EXP), p.cb * av);
                if (m == n) v += p.ca;
                v *= exp2f((float)P_EXP);
            } else v = acc[i][j] * exp2f(-(float)P_EXP) * al;
            if (KIND == APPLY && p.out == nullptr) {
                p.out32[((int64_t)b * p.M + m) * p.N + n] = v;
                continue;
            }
            if (KIND == APPLY) v /= p.alpha_next[b];
            __half hi, lo;
            split_half(v, hi, lo);
            p.out[at] = hi;
            if (p.planes == 2) p.out[at + p.slab_o] = lo;
        }
}

template <int KIND>
int launch(const Args& p, int batch, cudaStream_t s) {
    const dim3 grid((unsigned)ceil_div(p.N, T), (unsigned)ceil_div(p.M, T), (unsigned)batch);
    product_kernel<KIND><<<grid, 256, 0, s>>>(p);
    return check_cuda(cudaGetLastError());
}
}  // namespace

int launch_gram(const __half* x, __half* a, const float* alpha, const Shape& sh, int32_t*, cudaStream_t s) {
    Args p{x, x, a, nullptr, alpha, nullptr, sh.s, sh.s, sh.l, sh.ls, sh.ls, sh.ss, sh.planes, sh.x_slab(), sh.x_slab(), sh.a_slab(), 0, 0, 0};
    return launch<GRAM>(p, sh.batch, s);
}
int launch_poly(const __half* a, __half* q, float ca, float cb, float cc, const Shape& sh, int32_t*, cudaStream_t s) {
    Args p{a, a, q, nullptr, nullptr, nullptr, sh.s, sh.s, sh.s, sh.ss, sh.ss, sh.ss, sh.planes, sh.a_slab(), sh.a_slab(), sh.a_slab(), ca, cb, cc};
    return launch<POLY>(p, sh.batch, s);
}
int launch_apply(const __half* q, const __half* x, __half* x_next, float* o, const float* alpha,
                 const float* alpha_next, const Shape& sh, int32_t*,
                 cudaStream_t s) {
    Args p{q, x, x_next, o, alpha, alpha_next, sh.s, sh.l, sh.s, sh.ss, sh.ls, sh.ls, sh.planes, sh.a_slab(), sh.x_slab(), sh.x_slab(), 0, 0, 0};
    return launch<APPLY>(p, sh.batch, s);
}

}  // namespace ns
}  // namespace chebykan
