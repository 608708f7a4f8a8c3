// 8-bit forward of a Chebyshev layer: packing of the coefficients, quantised basis rows, entry points.
//
//   T_d = T_d(tanh x), d = 1..deg;  scale = max |T| / 127 over the row;  q = round(T / scale)
//
// Degree 0 is the constant 1 and lives in the bias.  A row with any input near zero has |T_2| close to 1, so from
// degree 2 on the scale is all but 1/127; it is taken from the row all the same, because a row of small inputs into
// a layer of degree 1 would lose most of its 8 bits to a fixed one.
#include <float.h>
#include "int8.cuh"

namespace chebykan {
namespace int8 {
namespace {

// tanh of two values, 1 - 2 / (1 + 2^(2x log2 e)) as tanh_fast: about 2e-7 absolute.  SMALL adds an odd series below 0.3,
// relative to 1e-7: a layer of degree 1 may see rows of small inputs only, which their scale blows up to 127 steps; from
// degree 2 on every row's largest |T_d| is of the order of 1.
template <bool SMALL>
__device__ __forceinline__ f32x2 tanh2(f32x2 x) {
    float z0, z1, e0, e1;
    halves(mul2(x, pair_of(2.885390081777927f, 2.885390081777927f)), z0, z1);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(z0));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(z1));
    halves(add2(pair_of(e0, e1), pair_of(1.f, 1.f)), z0, z1);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(z0));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(z1));
    const f32x2 t = fma2(pair_of(-2.f, -2.f), pair_of(e0, e1), pair_of(1.f, 1.f));
    if (!SMALL) return t;
    const f32x2 z = mul2(x, x);
    f32x2 p = pair_of(-0.0088632355f, -0.0088632355f);           // -1382/155925
    p = fma2(p, z, pair_of(0.021869488f, 0.021869488f));         // 62/2835
    p = fma2(p, z, pair_of(-0.053968254f, -0.053968254f));       // -17/315
    p = fma2(p, z, pair_of(0.13333333f, 0.13333333f));           // 2/15
    p = fma2(p, z, pair_of(-0.33333333f, -0.33333333f));
    float x0, x1, t0, t1, s0, s1;
    halves(x, x0, x1);
    halves(t, t0, t1);
    halves(fma2(mul2(x, z), p, x), s0, s1);
    return pair_of(fabsf(x0) < 0.3f ? s0 : t0, fabsf(x1) < 0.3f ? s1 : t1);
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
__device__ __forceinline__ uint32_t quantise4(f32x2 v0, f32x2 v1, f32x2 inv) {
    const f32x2 magic = pair_of(12582912.f, 12582912.f);
    float b0, b1, b2, b3;
    halves(fma2(v0, inv, magic), b0, b1);
    halves(fma2(v1, inv, magic), b2, b3);
    return __byte_perm(__byte_perm(__float_as_uint(b0), __float_as_uint(b1), 0x0040),
                       __byte_perm(__float_as_uint(b2), __float_as_uint(b3), 0x0040), 0x5410);
}

// The recurrence as N_{d+1} = +-2t N_d + N_{d-1}: N_d = T_d up to a sign that goes + + - - with d, and no operand has to be
// negated.  Steps to even degrees take -2t, to odd ones 2t.
struct Recurrence {
    f32x2 tt[4], ntt[4], a[4], b[4];
    __device__ __forceinline__ void start(const f32x2 (&t)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            tt[e] = add2(t[e], t[e]);
            ntt[e] = mul2(t[e], pair_of(-2.f, -2.f));
            a[e] = t[e]; b[e] = pair_of(1.f, 1.f);
        }
    }
    __device__ __forceinline__ void even() {
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = fma2(ntt[e], a[e], b[e]);
    }
    __device__ __forceinline__ void odd() {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = fma2(tt[e], b[e], a[e]);
    }
};

// One row by a group of G threads (lane: the thread's number in it), eight neighbouring inputs per thread and chunk.  The first
// pass finds the row's largest |T_d|, the second evaluates the recurrence again and writes dst[deg][pad]; tanh, by far the
// dearer part, is kept in registers in between (CHUNKS per thread; 0: rows longer than that evaluate it twice).  Every thread
// of the block comes here, live or not; red: a float per warp.
template <typename T, int G, int CHUNKS, bool SMALL>
__device__ __forceinline__ void quantise_row(const T* __restrict__ src, bool live, int lane, int in, int pad, int deg, int vec, float* red,
                                             int8_t* dst, float* scale) {
    constexpr int KEEP = CHUNKS ? CHUNKS : 1;
    const int chunks = CHUNKS ? CHUNKS : (pad + 8 * G - 1) / (8 * G);
    f32x2 t[KEEP][4];
    auto load = [&](int i0, f32x2 (&tc)[4]) {
        float v[8];
        load8(src + i0, in - i0, vec, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) tc[e] = tanh2<SMALL>(pair_of(v[2 * e], v[2 * e + 1]));
    };
    float top = 0.f;
    f32x2 nan = pair_of(0.f, 0.f);                    // 0, or NaN once an input was one
#pragma unroll
    for (int c = 0; c < chunks; ++c) {
        f32x2 (&tc)[4] = t[CHUNKS ? c : 0];
        const int i0 = (c * G + lane) * 8;
        if (live && i0 < in) {
            load(i0, tc);
            Recurrence r;
            r.start(tc);
            float big[8];
            auto look = [&](const f32x2 (&v)[4], bool first) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v0, v1;
                    halves(v[e], v0, v1);
                    big[2 * e] = first ? fabsf(v0) : fmaxf(big[2 * e], fabsf(v0));
                    big[2 * e + 1] = first ? fabsf(v1) : fmaxf(big[2 * e + 1], fabsf(v1));
                }
            };
            look(r.a, true);
            for (int d = 2; d <= deg; d += 2) {
                r.even();
                look(r.b, false);
                if (d < deg) { r.odd(); look(r.a, false); }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) nan = fma2(tc[e], pair_of(0.f, 0.f), nan);
            const int n = in - i0;
            if (n >= 8) {
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, big[e]);
            } else {                               // not the zeros past the row's end: T_2(0) = -1
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < n) top = fmaxf(top, big[e]);
            }
        }
    }
    float n0, n1;
    halves(nan, n0, n1);
    if (n0 != 0.f || n1 != 0.f || n0 != n0 || n1 != n1) top = __int_as_float(0x7f800000);
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
    // A degree-1 row may be so small that 1 / s overflows (from degree 2 on top is of the order of 1).  Its values and scale are
    // lifted by 2^100, which is exact; a subnormal scale has few bits, so that values may lie beyond 127 of it and are clamped
    const bool tiny = SMALL && top < 1e-30f;
    const float lift = tiny ? 1.2676506e30f : 1.f;
    const float inv = (bad || s == 0.f) ? 0.f : __fdiv_rn(1.f, s * lift);
    if (lane == 0) *scale = s;
    const f32x2 plus = pair_of(inv, inv), minus = pair_of(-inv, -inv);
#pragma unroll
    for (int c = 0; c < chunks; ++c) {
        f32x2 (&tc)[4] = t[CHUNKS ? c : 0];
        const int i0 = (c * G + lane) * 8;
        if (i0 >= pad) continue;
        const int n = in - i0;                     // inputs of the chunk; the rest of the padded row is zero
        if (CHUNKS == 0 && chunks > 1 && n > 0) load(i0, tc);
        if (tiny) {
            const float most = inv > 0.f ? 127.f * (s * lift) : 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v0, v1;
                halves(tc[e], v0, v1);
                tc[e] = pair_of(fminf(fmaxf(v0 * lift, -most), most), fminf(fmaxf(v1 * lift, -most), most));
            }
        }
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
        if (bad) keep0 = keep1 = 0;
        else if (n < 8) {
            keep0 = n <= 0 ? 0 : (n >= 4 ? keep0 : (1u << (8 * n)) - 1u);
            keep1 = n <= 4 ? 0 : (1u << (8 * (n - 4))) - 1u;
        }
        Recurrence r;
        r.start(tc);
        int8_t* to = dst + i0;
        auto put = [&](const f32x2 (&v)[4], f32x2 by) {
            *reinterpret_cast<uint2*>(to) = make_uint2(quantise4(v[0], v[1], by) & keep0, quantise4(v[2], v[3], by) & keep1);
            to += pad;
        };
        // signs + + - - from degree 0 on
        put(r.a, plus);
        for (int d = 2; d <= deg; d += 2) {
            const f32x2 by = d & 2 ? minus : plus;
            r.even();
            put(r.b, by);
            if (d < deg) { r.odd(); put(r.a, by); }
        }
    }
}

// 256 / G rows per block.  32768 x 2048, degree 4: 138 us, 3.9 TB/s; groups of 128 or 64 threads with two or four chunks each
// took 146 and 181 us, five blocks per SM (by spilling) 181 us.
template <typename T, int G, int CHUNKS, bool SMALL>
__global__ void __launch_bounds__(256)
basis_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale, int64_t B, int in, int pad, int deg, int vec) {
    __shared__ float red[8];
    const int64_t row = blockIdx.x * (int64_t)(256 / G) + threadIdx.x / G;
    let_next_start();
    quantise_row<T, G, CHUNKS, SMALL>(x + row * in, row < B, threadIdx.x % G, in, pad, deg, vec, red, q + row * (int64_t)deg * pad, scale + row);
}

// The whole forward of a few rows in one launch: every block quantises the rows for itself, into shared memory, while the first
// of its weights are on their way, and then takes columns as row_kernel does.  The same arithmetic, so the same bits, as the two
// kernels, without the launch, the workspace and the wait between them.  Bound by latency: the rows' quantisation, 2 us, then one
// trip to memory for the weights after the first.  In a graph (us, in brackets as two kernels that overlap) 1 x 2048 -> 2048 of
// degree 4 takes 4.8 (8.0), 2 x 1024 -> 1000 4.0 (5.1), 4 x 784 -> 64 of degree 8 7.9 (9.3), 8 x 128 -> 4096 9.0 (13.0).  The 256 threads
// share out the rows, so a row of several has 64 or 128 of them, and beyond 1024 inputs they fall behind: 2 x 1040 -> 1000 5.8
// (4.7), 2 x 2048 -> 2048 7.4 (5.8), 4 x 1040 -> 1000 8.2 (7.4), 4 x 2048 -> 2048 11.8 (9.6), 4 x 11000 -> 2048 of degree 1 32 (15).
// There in_one_launch() takes the two kernels, although a call from Python, which is bound by the host, then costs 14.6 instead of 11.
template <typename OUT, typename T, int ROWS, bool SMALL>
__global__ void __launch_bounds__(256)
few_rows_kernel(const T* __restrict__ x, const int8_t* __restrict__ wq, const float* __restrict__ w_scale, const float* __restrict__ bias,
                OUT* __restrict__ y, int B, int N, int in, int pad, int deg, int vec) {
    extern __shared__ int4 rows[];                     // [B][K / 16]
    __shared__ float red[8], scale[ROWS];
    const int lane = threadIdx.x & 31, step = (int)gridDim.x * 8, whole = deg * pad / 16;
    constexpr int U = ROWS == 1 ? 16 : 8;
    int4 wv[U];
    auto weights = [&](int o, int c0) {
        const int4* w = reinterpret_cast<const int4*>(wq) + (int64_t)o * whole;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            wv[u] = make_int4(0, 0, 0, 0);
            if (c0 + u * 32 < whole) wv[u] = __ldg(w + c0 + u * 32);
        }
    };
    int o = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (o < N) weights(o, lane);
    constexpr int G = 256 / ROWS;                      // all rows at once
    const int row = threadIdx.x / G;
    quantise_row<T, G, 0, SMALL>(x + (int64_t)row * in, row < B, threadIdx.x % G, in, pad, deg, vec, red,
                                 reinterpret_cast<int8_t*>(rows + row * whole), scale + row);
    __syncthreads();
    for (; o < N; o += step) {
        int acc[ROWS] = {};
        for (int c0 = lane; c0 < whole;) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                if (r < B)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (c0 + u * 32 < whole) {
                            const int4 v = rows[r * whole + c0 + u * 32];
                            acc[r] = __dp4a(v.x, wv[u].x, __dp4a(v.y, wv[u].y, __dp4a(v.z, wv[u].z, __dp4a(v.w, wv[u].w, acc[r]))));
                        }
            c0 += U * 32;
            if (c0 < whole) weights(o, c0);
        }
        if (o + step < N) weights(o + step, lane);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
#pragma unroll
            for (int d = 16; d; d >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], d);
            if (lane == r && r < B)
                y[(int64_t)r * N + o] = to_type<OUT>(fmaf((float)acc[r] * scale[r], __ldg(w_scale + o), bias ? __ldg(bias + o) : 0.f));
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
            bad = bad || !(fabsf(p[d]) <= FLT_MAX);
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
    bad = top > FLT_MAX;
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
    auto kernel = deg == 1 ? basis_kernel<T, G, CHUNKS, true> : basis_kernel<T, G, CHUNKS, false>;
    kernel<<<(unsigned)ceil_div(B, 256 / G), 256, 0, s>>>(x, q, scale, B, (int)in, (int)in_pad(in), (int)deg, vec);
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

template <typename OUT, typename T>
int launch_few_rows(const void* x, const int8_t* wq, const float* w_scale, const float* bias, void* y, int64_t B, int64_t N, int64_t in,
                    int64_t deg, cudaStream_t s) {
    const int pad = (int)in_pad(in), vec = (in * sizeof(T)) % 16 == 0;
    auto kernel = B == 1 ? (deg == 1 ? few_rows_kernel<OUT, T, 1, true> : few_rows_kernel<OUT, T, 1, false>)
                : B == 2 ? (deg == 1 ? few_rows_kernel<OUT, T, 2, true> : few_rows_kernel<OUT, T, 2, false>)
                : B <= 4 ? (deg == 1 ? few_rows_kernel<OUT, T, 4, true> : few_rows_kernel<OUT, T, 4, false>)
                         : (deg == 1 ? few_rows_kernel<OUT, T, 8, true> : few_rows_kernel<OUT, T, 8, false>);
    const int64_t blocks = ceil_div(N, 8);
    kernel<<<(unsigned)(blocks < 2 * 148 ? blocks : 2 * 148), 256, (size_t)(B * deg * pad), s>>>(
        reinterpret_cast<const T*>(x), wq, w_scale, bias, reinterpret_cast<OUT*>(y), (int)B, (int)N, (int)in, pad, (int)deg, vec);
    return check_cuda(cudaGetLastError());
}
template <typename OUT>
int launch_few_rows_to(const void* x, int x_dtype, const int8_t* wq, const float* w_scale, const float* bias, void* y, int64_t B, int64_t N,
                       int64_t in, int64_t deg, cudaStream_t s) {
    if (x_dtype == CHEBYKAN_DTYPE_FP32) return launch_few_rows<OUT, float>(x, wq, w_scale, bias, y, B, N, in, deg, s);
    if (x_dtype == CHEBYKAN_DTYPE_BF16) return launch_few_rows<OUT, __nv_bfloat16>(x, wq, w_scale, bias, y, B, N, in, deg, s);
    return launch_few_rows<OUT, __half>(x, wq, w_scale, bias, y, B, N, in, deg, s);
}

bool dtype_ok(int dtype) { return dtype >= CHEBYKAN_DTYPE_FP32 && dtype <= CHEBYKAN_DTYPE_FP16; }
int64_t dtype_size(int dtype) { return dtype == CHEBYKAN_DTYPE_FP32 ? 4 : 2; }
// whether what is written covers part of the columns' scales or biases
bool over_vectors(const void* y, int64_t bytes, const float* w_scale, const float* bias, int64_t n) {
    return overlap(y, bytes, w_scale, 4 * n) || overlap(y, bytes, bias, 4 * n);
}
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
// A few rows go through one launch while they fit 48 KB of shared memory; several only up to 1024 inputs, because the threads of
// a block then share out the rows and evaluate the basis of longer ones in turn, in every block (see few_rows_kernel)
bool in_one_launch(int64_t B, int64_t in, int64_t deg) {
    const int64_t pad = in_pad(in), K = pad * deg;
    return few_rows(B, K) && B * K <= 46 * 1024 && (B == 1 || pad <= 1024);
}
// rows worked on at a time: 1 GiB of quantised rows at most (8192 of the longest, MAX_K bytes)
int64_t chunk_rows(int64_t B, int64_t K) {
    const int64_t rows = ((int64_t)1 << 30) / K / 256 * 256;
    return B < rows ? B : rows;
}

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
    const int64_t read = 4 * in * out * (deg + 1);
    if (overlap(wq, out * in_pad(in) * deg, coeffs, read) || overlap(w_scale, 4 * out, coeffs, read) || overlap(bias, 4 * out, coeffs, read))
        return CHEBYKAN_EOVERLAP;
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
    const int64_t read = B * in * dtype_size(dtype);
    if (overlap(q, B * in_pad(in) * deg, x, read) || overlap(scale, 4 * B, x, read)) return CHEBYKAN_EOVERLAP;
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
    const int64_t written = M * N * dtype_size(dtype);
    if (overlap(y, written, q, (M - 1) * ldq + K) || overlap(y, written, wq, (N - 1) * ldw + K) || over_vectors(y, written, w_scale, bias, N) ||
        overlap(y, written, q_scale, 4 * M))
        return CHEBYKAN_EOVERLAP;
    int rc = check_device();
    if (rc) return rc;
    return launch_matmul({q, q_scale, wq, w_scale, bias, y, dtype, M, N, K, ldq, ldw}, workspace, status, (cudaStream_t)stream, false);
}

int64_t chebykan_int8_fwd_workspace_bytes(int64_t B, int64_t in, int64_t out, int64_t deg) {
    if (!layer_ok(B, in, out, deg)) return CHEBYKAN_EINVAL;
    const int64_t K = in_pad(in) * deg, rows = chunk_rows(B, K);
    if (in_one_launch(B, in, deg)) return 0;
    return a256(rows * K) + a256(rows * 4);
}

int chebykan_int8_fwd(const void* x, int x_dtype, const int8_t* wq, const float* w_scale, const float* bias, void* y, int y_dtype,
                      void* workspace, int64_t workspace_bytes, int64_t B, int64_t in, int64_t out, int64_t deg, int32_t* status,
                      void* stream) {
    const int64_t need = chebykan_int8_fwd_workspace_bytes(B, in, out, deg);
    if (need < 0) return (int)need;
    if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype)) return CHEBYKAN_EINVAL;
    if (B == 0) return CHEBYKAN_OK;
    if (!x || !wq || !w_scale || !y || !status) return CHEBYKAN_EINVAL;
    if (!aligned16(x) || !aligned16(wq) || !aligned16(y) || !aligned16(workspace)) return CHEBYKAN_EALIGN;
    if (workspace_bytes < need || (need > 0 && !workspace)) return CHEBYKAN_EWORKSPACE;
    const int64_t K = in_pad(in) * deg, rows = chunk_rows(B, K), x_size = dtype_size(x_dtype), y_size = dtype_size(y_dtype);
    const int64_t written = B * out * y_size;
    if (overlap(y, written, x, B * in * x_size) || overlap(y, written, wq, out * K) || over_vectors(y, written, w_scale, bias, out))
        return CHEBYKAN_EOVERLAP;
    int rc = check_device();
    if (rc) return rc;
    if (need == 0) {
        cudaStream_t s = (cudaStream_t)stream;
        if (y_dtype == CHEBYKAN_DTYPE_FP32) return launch_few_rows_to<float>(x, x_dtype, wq, w_scale, bias, y, B, out, in, deg, s);
        if (y_dtype == CHEBYKAN_DTYPE_BF16) return launch_few_rows_to<__nv_bfloat16>(x, x_dtype, wq, w_scale, bias, y, B, out, in, deg, s);
        return launch_few_rows_to<__half>(x, x_dtype, wq, w_scale, bias, y, B, out, in, deg, s);
    }
    char* ws = reinterpret_cast<char*>(workspace);
    int8_t* q = reinterpret_cast<int8_t*>(ws);
    float* scale = reinterpret_cast<float*>(ws + a256(rows * K));
    for (int64_t r = 0; r < B; r += rows) {        // rows is a multiple of 256 where there is more than one turn: pointers stay aligned
        const int64_t n = B - r < rows ? B - r : rows;
        const char* xr = reinterpret_cast<const char*>(x) + r * in * x_size;
        char* yr = reinterpret_cast<char*>(y) + r * out * y_size;
        if ((rc = launch_basis(xr, x_dtype, q, scale, n, in, deg, (cudaStream_t)stream))) return rc;
        // rows of q and wq are K bytes apart, a multiple of 16: the product needs no scratch
        if ((rc = launch_matmul({q, scale, wq, w_scale, bias, yr, y_dtype, n, out, K, K, K}, nullptr, status, (cudaStream_t)stream, true))) return rc;
    }
    return CHEBYKAN_OK;
}

}  // extern "C"
