// Product of 8-bit integer matrices with a scale per row and per column:
//   y[r][o] = (sum_k q[r][k] wq[o][k]) * q_scale[r] * w_scale[o] + bias[o]
// The sum is exact in int32 whatever its order, so the kernels below give the same bits.  1 x 8192 -> 1024 5 us, 256 x 3136 -> 64
// 8 us, 65536 x 8192 -> 1024 340 us.
//
//   few rows         row_kernel: bound by reading wq once; CUDA cores, four products per instruction
//   few tiles        tcgen05 kind::i8, one tile per cluster, K split over its CTAs (gemm_tc.cuh)
//   else             tcgen05 kind::i8, persistent pairs on 256 x 256 tiles (256 x 128 or x 64 for fewer columns)
#include "gemm_tc.cuh"
#include "int8.cuh"

namespace chebykan {
namespace int8 {
namespace {
using gemm::Tiles;

struct EpiArgs {
    const float *q_scale, *w_scale, *bias;
    void* y;
    int vec, vec_scales;      // whether y's rows, and the columns' scales, allow 16-byte accesses
};

template <typename OUT>
struct Epilogue {
    using Args = EpiArgs;
    static constexpr bool BULK = false;
    struct Fetched {};
    static __device__ __forceinline__ void fetch(const Args&, const Tiles&, int, int, int, Fetched&) {}

    // the scales and biases of NC columns: every load first; one after the other, each waited for, they would take longer than
    // the tile's MMAs
    template <int NC>
    static __device__ __forceinline__ void columns(const Args& p, const Tiles& g, int col0, float (&ws)[NC], float (&bs)[NC]) {
        if (col0 + NC <= g.N && p.vec_scales) {
#pragma unroll
            for (int c = 0; c < NC; c += 4) *reinterpret_cast<float4*>(ws + c) = __ldg(reinterpret_cast<const float4*>(p.w_scale + col0 + c));
#pragma unroll
            for (int c = 0; c < NC; c += 4)
                *reinterpret_cast<float4*>(bs + c) = p.bias ? __ldg(reinterpret_cast<const float4*>(p.bias + col0 + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
#pragma unroll
            for (int e = 0; e < NC; ++e) {
                const int col = col0 + e < g.N ? col0 + e : g.N - 1;
                ws[e] = __ldg(p.w_scale + col);
                bs[e] = p.bias ? __ldg(p.bias + col) : 0.f;
            }
        }
    }
    static __device__ __forceinline__ void emit(const Args& p, const Tiles& g, int, int row0, int col0, uint32_t (&r)[32], const Fetched&, uint32_t buf) {
        const int row = row0 + (threadIdx.x & 31);
        alignas(16) float ws[32], bs[32];
        columns(p, g, col0, ws, bs);
        const float qs = row < g.M ? __ldcg(p.q_scale + row) : 0.f;       // see launch_after
        alignas(16) OUT out[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) out[e] = to_type<OUT>(fmaf((float)(int)r[e] * qs, ws[e], bs[e]));
        gemm::store_rows(buf, out, reinterpret_cast<OUT*>(p.y) + (int64_t)row0 * g.N + col0, g.N, g.M - row0, g.N - col0, p.vec);
    }
    // 8 columns of one row, from the kernel that splits K
    static __device__ __forceinline__ void emit8(const Args& p, const Tiles& g, int row, int col0, const uint32_t (&r)[8]) {
        alignas(16) float ws[8], bs[8];
        columns(p, g, col0, ws, bs);
        const float qs = __ldcg(p.q_scale + row);
        OUT* dst = reinterpret_cast<OUT*>(p.y) + (int64_t)row * g.N + col0;
        alignas(16) OUT out[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = to_type<OUT>(fmaf((float)(int)r[e] * qs, ws[e], bs[e]));
        if (p.vec && col0 + 8 <= g.N) {
#pragma unroll
            for (int c = 0; c < 8; c += 16 / (int)sizeof(OUT))
                *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(out + c);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col0 + e < g.N) dst[e] = out[e];
        }
    }
};

// ---- few rows -----------------------------------------------------------------------------------------------------
// A warp per output column: lanes take 16 bytes of the column's weights each, U loads in flight, against the same bytes of
// every row (from the caches).  The first weights are asked for before the rows' producer is waited for.
// STAGED: the block copies the rows into shared memory first, all at once: with four rows of 8192 the reads row after row took
// 13.3 us (1024 outputs), staged 5.2; rows of 2048 (8192 outputs) 8.8 and 7.9.  Two rows (2.9 / 3.3) and eight short ones (512 ->
// 2048 5.1 / 6.3) are faster from the caches.
template <typename OUT, int ROWS, bool STAGED>
__global__ void __launch_bounds__(256) row_kernel(const Product p) {
    extern __shared__ int4 staged[];                   // [M][K / 16]
    const int lane = threadIdx.x & 31;
    const int64_t o = blockIdx.x * (int64_t)8 + (threadIdx.x >> 5);
    if (!STAGED && o >= p.N) return;
    const bool mine = o < p.N;
    const int8_t* w = p.wq + o * p.ldw;
    const int whole = (int)(p.K / 16);                 // 16-byte pieces; the rest is one lane's, byte by byte
    int acc[ROWS] = {};
    constexpr int U = ROWS <= 2 ? 16 : 8;
    int4 wv[U];
    auto weights = [&](int c0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            wv[u] = make_int4(0, 0, 0, 0);
            if (c0 + u * 32 < whole) wv[u] = __ldg(reinterpret_cast<const int4*>(w) + c0 + u * 32);
        }
    };
    if (mine) weights(lane);
    const float ws = mine ? __ldg(p.w_scale + o) : 0.f, bias = mine && p.bias ? __ldg(p.bias + o) : 0.f;
    wait_for_previous();
    if (STAGED) {
        for (int r = 0; r < ROWS; ++r)
            if (r < p.M)
#pragma unroll 4
                for (int c = threadIdx.x; c < whole; c += 256) staged[r * whole + c] = reinterpret_cast<const int4*>(p.q + r * p.ldq)[c];
        __syncthreads();
        if (!mine) return;
    }
    for (int c0 = lane; c0 < whole;) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            if (r < p.M) {
                const int4* q = STAGED ? staged + r * whole : reinterpret_cast<const int4*>(p.q + r * p.ldq);
                int4 v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    v[u] = make_int4(0, 0, 0, 0);
                    if (c0 + u * 32 < whole) v[u] = q[c0 + u * 32];
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    acc[r] = __dp4a(v[u].x, wv[u].x, __dp4a(v[u].y, wv[u].y, __dp4a(v[u].z, wv[u].z, __dp4a(v[u].w, wv[u].w, acc[r]))));
            }
        c0 += U * 32;
        if (c0 < whole) weights(c0);
    }
    if (lane == 0)
        for (int64_t k = (int64_t)whole * 16; k < p.K; ++k)
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                if (r < p.M) acc[r] += (int)p.q[r * p.ldq + k] * (int)w[k];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int d = 16; d; d >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], d);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if (lane == r && r < p.M) reinterpret_cast<OUT*>(p.y)[r * p.N + o] = to_type<OUT>(fmaf((float)acc[r] * __ldcg(p.q_scale + r), ws, bias));
}

// no columns at all: the sums are zero
template <typename OUT>
__global__ void __launch_bounds__(256) empty_kernel(const Product p) {
    for (int64_t e = blockIdx.x * (int64_t)256 + threadIdx.x; e < p.M * p.N; e += (int64_t)gridDim.x * 256)
        reinterpret_cast<OUT*>(p.y)[e] = to_type<OUT>(fmaf(0.f * p.q_scale[e / p.N], p.w_scale[e % p.N], p.bias ? p.bias[e % p.N] : 0.f));
}

// rows of any byte pitch -> rows of a pitch that is a multiple of 16, 16 bytes per thread: the five aligned words around a
// piece, shifted into place; words that reach out of the matrix are read byte by byte.  One launch for both matrices
// (blockIdx.y): 64 x 1001 -> 700 7.9 us, one after the other 9.2
struct Padding {
    const int8_t* src;
    int8_t* dst;
    int64_t ld, rows;
};
__global__ void __launch_bounds__(256) pad_kernel(const Padding first, const Padding second, int64_t pitch, int64_t K) {
    const Padding m = blockIdx.y ? second : first;
    const int8_t* __restrict__ src = m.src;
    int8_t* __restrict__ dst = m.dst;
    const int64_t ld = m.ld, rows = m.rows;
    const int64_t pieces = pitch / 16, last = (rows - 1) * ld + K;      // bytes from src to the matrix's end
    for (int64_t e = blockIdx.x * (int64_t)256 + threadIdx.x; e < rows * pieces; e += (int64_t)gridDim.x * 256) {
        const int64_t r = e / pieces, k = (e - r * pieces) * 16, from = r * ld + k, aligned = from & ~(int64_t)3;
        const uint32_t shift = (uint32_t)(from & 3) * 8;
        uint32_t w[5];
#pragma unroll
        for (int j = 0; j < 5; ++j) {
            const int64_t at = aligned + 4 * j;
            w[j] = 0;
            if (at + 4 <= last) w[j] = *reinterpret_cast<const uint32_t*>(src + at);
            else
                for (int i = 0; i < 4 && at + i < last; ++i) w[j] |= (uint32_t)(uint8_t)src[at + i] << (8 * i);
        }
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j] = __funnelshift_r(w[j], w[j + 1], shift);
            const int64_t left = K - k - 4 * j;                         // the next row's bytes are not this one's padding
            if (left < 4) o[j] &= left <= 0 ? 0u : (1u << (8 * left)) - 1u;
        }
        *reinterpret_cast<uint4*>(dst + r * pitch + k) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

template <typename OUT>
int launch_rows(const Product& p, cudaStream_t s, bool after) {
    const int64_t bytes = p.M * (p.K / 16) * 16;
    const bool staged = p.M > 2 && p.M <= 4;           // few_rows: they fit
    auto kernel = p.M == 1 ? row_kernel<OUT, 1, false>
                : p.M == 2 ? row_kernel<OUT, 2, false>
                : staged ? row_kernel<OUT, 4, true>
                         : row_kernel<OUT, 8, false>;
    return check_cuda(launch_after(after, kernel, dim3((unsigned)ceil_div(p.N, 8)), dim3(256), staged ? (size_t)bytes : 0, s, 0, p));
}

template <class C>
int maps_of(const Product& p, CUtensorMap* mq, CUtensorMap* mw) {
    const int rc = gemm::make_map(mq, gemm::I8, p.q, p.K, p.M, 1, p.ldq, p.ldq, C::KE, 128);      // one slab: its distance is not used
    return rc ? rc : gemm::make_map(mw, gemm::I8, p.wq, p.K, p.N, 1, p.ldw, p.ldw, C::KE, C::BN / C::CG);
}

template <class C, typename OUT>
int run_split(const Product& p, const Tiles& g, const EpiArgs& args, int32_t* status, cudaStream_t s, bool after) {
    CUtensorMap mq, mw;
    const int rc = maps_of<C>(p, &mq, &mw);
    if (rc) return rc;
    return gemm::launch_split<C, Epilogue<OUT>>(mq, mw, g, args, gemm::split_of(g), status, s, after);
}
template <class C, typename OUT>
int run_persistent(const Product& p, const EpiArgs& args, int32_t* status, cudaStream_t s, bool after) {
    CUtensorMap mq, mw;
    const int rc = maps_of<C>(p, &mq, &mw);
    if (rc) return rc;
    return gemm::launch<C, Epilogue<OUT>>(mq, mw, gemm::tiles_of<C>((int)p.M, (int)p.N, (int)p.K, 1, false), args, status, s, after);
}

template <typename OUT>
int launch_typed(const Product& p, int32_t* status, cudaStream_t s, bool after) {
    if (p.K == 0) {
        empty_kernel<OUT><<<(unsigned)(ceil_div(p.M * p.N, 256) < 148 * 8 ? ceil_div(p.M * p.N, 256) : 148 * 8), 256, 0, s>>>(p);
        return check_cuda(cudaGetLastError());
    }
    if (few_rows(p.M, p.K)) return launch_rows<OUT>(p, s, after);
    const EpiArgs args{p.q_scale, p.w_scale, p.bias, p.y, p.N % (16 / (int64_t)sizeof(OUT)) == 0,
                       aligned16(p.w_scale) && aligned16(p.bias)};
    using Pair = gemm::Config<gemm::I8, 1, 2, 256, false>;
    using Pair128 = gemm::Config<gemm::I8, 1, 2, 128, false>;
    using Pair64 = gemm::Config<gemm::I8, 1, 2, 64, false>;
    using Narrow = gemm::Config<gemm::I8, 1, 1, 64, false>;
    using Wide = gemm::Config<gemm::I8, 1, 1, 128, false>;
    // tiles of 128 x 64 as long as that leaves SMs idle, of 128 x 128 up to one each; beyond, pairs on 256 rows and as many
    // columns as there are, up to 256
    const int M = (int)p.M, N = (int)p.N, K = (int)p.K;
    const Tiles narrow = gemm::tiles_of<Narrow>(M, N, K, 1, false), wide = gemm::tiles_of<Wide>(M, N, K, 1, false);
    if (narrow.total <= 148) return run_split<Narrow, OUT>(p, narrow, args, status, s, after);
    if (wide.total <= 148) return run_split<Wide, OUT>(p, wide, args, status, s, after);
    if (N <= 64) return run_persistent<Pair64, OUT>(p, args, status, s, after);
    if (N <= 128) return run_persistent<Pair128, OUT>(p, args, status, s, after);
    return run_persistent<Pair, OUT>(p, args, status, s, after);
}

int64_t a256(int64_t b) { return round_up(b, 256); }
}  // namespace

int64_t matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t ldq, int64_t ldw) {
    const int64_t pitch = round_up(K, 16);
    return (ldq % 16 ? a256(M * pitch) : 0) + (ldw % 16 ? a256(N * pitch) : 0);
}

int launch_matmul(const Product& given, void* ws, int32_t* status, cudaStream_t s, bool after) {
    Product p = given;
    const int64_t pitch = round_up(p.K, 16);
    int8_t* at = reinterpret_cast<int8_t*>(ws);
    Padding job[2];
    int jobs = 0;
    int64_t most = 0;
    auto pad = [&](const int8_t*& m, int64_t& ld, int64_t rows) {
        if (ld % 16 == 0 || p.K == 0) return;
        job[jobs++] = {m, at, ld, rows};
        if (rows > most) most = rows;
        m = at; ld = pitch; at += a256(rows * pitch);
    };
    pad(p.q, p.ldq, p.M);
    pad(p.wq, p.ldw, p.N);
    if (jobs > 0) {
        const int64_t blocks = ceil_div(most * pitch / 16, 256);
        pad_kernel<<<dim3((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), (unsigned)jobs), 256, 0, s>>>(job[0], job[jobs - 1], pitch, p.K);
        const int rc = check_cuda(cudaGetLastError());
        if (rc) return rc;
    }
    if (p.dtype == CHEBYKAN_DTYPE_FP32) return launch_typed<float>(p, status, s, after);
    if (p.dtype == CHEBYKAN_DTYPE_BF16) return launch_typed<__nv_bfloat16>(p, status, s, after);
    return launch_typed<__half>(p, status, s, after);
}

}  // namespace int8
}  // namespace chebykan
