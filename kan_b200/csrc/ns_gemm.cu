// The three products of a Newton-Schulz step on tcgen05 (gemm_tc.cuh; see newton_schulz.cuh for the operands' layout):
//   A = X X^T            both operands are X's rows; symmetric
//   P = a I + b A + c A A      both operands are A's rows (A is symmetric); symmetric
//   X' = P X             P's rows against X as it lies, [K][N]: no transposed copy of X exists
// Of the symmetric two only the 256 x 256 blocks on and above the diagonal are computed and stored; the products that read
// them take a block below the diagonal from its mirror image.
#include <type_traits>
#include "gemm_tc.cuh"
#include "newton_schulz.cuh"

namespace chebykan {
namespace ns {
namespace {
using gemm::Tiles;

enum { GRAM = 0, POLY = 1, APPLY = 2, LAST = 3 };       // LAST: the final APPLY, to the caller's layout and type

struct alignas(64) EpiArgs {
    CUtensorMap map;          // planes of the result: boxes of 32 x 32
    const __half* a;          // POLY: A's planes
    void* o;                  // LAST: [batch][m][n]
    int tall;                 // LAST: o is the transposed result
    const float *alpha, *alpha_next;
    int pitch;                // of a
    int64_t slab;
    float ca, cb, cc;
};

template <int KIND, int PLANES, typename OUT = float>
struct Epilogue {
    using Args = EpiArgs;
    static constexpr bool BULK = KIND != LAST;
    struct Ahead { uint4 hi[4], lo[PLANES == 2 ? 4 : 1]; };       // 32 columns of A's row
    struct Nothing {};
    using Fetched = typename std::conditional<KIND == POLY, Ahead, Nothing>::type;

    static __device__ __forceinline__ void fetch(const Args& p, const Tiles& g, int b, int row, int col0, Fetched& f) {
        if constexpr (KIND == POLY) {
            if (row >= g.M) return;
            const __half* a = p.a + (int64_t)b * PLANES * p.slab + (int64_t)row * p.pitch + col0;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (col0 + c * 8 < g.N) {
                    f.hi[c] = *reinterpret_cast<const uint4*>(a + c * 8);
                    if (PLANES == 2) f.lo[c] = *reinterpret_cast<const uint4*>(a + c * 8 + p.slab);
                }
        }
    }

    // what the accumulator is multiplied with
    static __device__ __forceinline__ float scale(const Args& p, int b) {
        if (KIND == GRAM) { const float al = p.alpha[b]; return al * al * exp2f((float)A_EXP); }
        if (KIND == POLY) return p.cc * exp2f(-2.f * A_EXP + P_EXP);
        if (KIND == APPLY) return exp2f(-(float)P_EXP) * p.alpha[b] / p.alpha_next[b];
        return exp2f(-(float)P_EXP) * p.alpha[b];
    }
    // POLY: what the product is added to, ca I + cb A, for eight columns
    static __device__ __forceinline__ void addend(const Args& p, int row, int col0, const uint32_t (&ah)[4], const uint32_t (&al)[4], float (&v)[8]) {
        float a[8];
        join8<PLANES>(ah, al, a);
        const float by = p.cb * exp2f((float)(P_EXP - A_EXP));
#pragma unroll
        for (int e = 0; e < 8; e += 2) halves(mul2(pair_of(a[e], a[e + 1]), pair_of(by, by)), v[e], v[e + 1]);
        if (row >= col0 && row < col0 + 8) {                // the diagonal passes through
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col0 + e == row) v[e] += p.ca * exp2f((float)P_EXP);
        }
    }
    static constexpr bool INIT = KIND == POLY;
    // A's 32 x NC block: lanes read along rows (a row per lane would touch 32 lines per load) and meet their rows in buf
    template <int NC>
    static __device__ __forceinline__ void init(const Args& p, const Tiles& g, int b, int row0, int col0, float (&v)[NC], uint32_t buf) {
        const int lane = threadIdx.x & 31, ch = lane & 3;
        const __half* a = p.a + (int64_t)b * PLANES * p.slab + (int64_t)row0 * p.pitch + col0;
        auto place = [&](int plane, int r, int c) { return buf + (uint32_t)(plane * 2048 + r * 64 + ((c ^ ((r >> 1) & 3)) << 4)); };
        uint4 x[NC / 32][4 * PLANES];           // the whole block in flight: v takes its registers block by block
#pragma unroll
        for (int c = 0; c < NC; c += 32)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + (lane >> 2);
                const bool in = row0 + r < g.M && col0 + c + ch * 8 < g.N;
#pragma unroll
                for (int q = 0; q < PLANES; ++q)
                    x[c / 32][i * PLANES + q] = in ? *reinterpret_cast<const uint4*>(a + (int64_t)r * p.pitch + c + ch * 8 + q * p.slab) : make_uint4(0, 0, 0, 0);
            }
        if (lane == 0) gemm::bulk_wait_read();
        __syncwarp();
#pragma unroll
        for (int c = 0; c < NC; c += 32) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int q = 0; q < PLANES; ++q) {
                    const uint4 w = x[c / 32][i * PLANES + q];
                    gemm::st_shared_v4(place(q, i * 8 + (lane >> 2), ch), w.x, w.y, w.z, w.w);
                }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t ah[4], al[4] = {};
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(ah[0]), "=r"(ah[1]), "=r"(ah[2]), "=r"(ah[3]) : "r"(place(0, lane, k)));
                if (PLANES == 2)
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(al[0]), "=r"(al[1]), "=r"(al[2]), "=r"(al[3]) : "r"(place(1, lane, k)));
                float y[8];
                addend(p, row0 + lane, col0 + c + k * 8, ah, al, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c + k * 8 + e] = y[e];
            }
            __syncwarp();
        }
    }

    // 32 columns from col0 of the rows from row0, one per lane; buf: the warp's 4 KB
    static __device__ __forceinline__ void put(const Args& p, const Tiles& g, int b, int row0, int col0, const float (&x)[32], uint32_t buf) {
        const int lane = threadIdx.x & 31, row = row0 + lane;
        if constexpr (KIND == LAST) {
            OUT* o = reinterpret_cast<OUT*>(p.o) + (int64_t)b * g.M * g.N;
            if (p.tall) {                       // the warp's lanes hold consecutive rows, which are o's columns
                if (row < g.M)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (col0 + e < g.N) o[(int64_t)(col0 + e) * g.M + row] = from_float<OUT>(x[e]);
                return;
            }
            alignas(16) OUT v[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = from_float<OUT>(x[e]);
            gemm::store_rows(buf, v, o + (int64_t)row0 * g.N + col0, g.N, g.M - row0, g.N - col0, g.N % (16 / (int)sizeof(OUT)) == 0);
        } else {
            // both planes of 32 x 32 into shared memory, 64-byte rows with the 16-byte chunks permuted as the map's swizzle has
            // it (chunk ^ bits 1-2 of the row), and from there by TMA, which clips what lies outside the matrix
            if (lane == 0) gemm::bulk_wait_read();
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float v[8] = {x[c * 8], x[c * 8 + 1], x[c * 8 + 2], x[c * 8 + 3], x[c * 8 + 4], x[c * 8 + 5], x[c * 8 + 6], x[c * 8 + 7]};
                uint32_t hi[4], lo[4];
                split8<PLANES>(v, hi, lo);
                const uint32_t at = buf + (uint32_t)(lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4));
                gemm::st_shared_v4(at, hi[0], hi[1], hi[2], hi[3]);
                if (PLANES == 2) gemm::st_shared_v4(at + 2048, lo[0], lo[1], lo[2], lo[3]);
            }
            gemm::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                gemm::store_3d(&p.map, buf, col0, row0, b * PLANES);
                if (PLANES == 2) gemm::store_3d(&p.map, buf + 2048, col0, row0, b * PLANES + 1);
                gemm::bulk_commit();
            }
        }
    }
    static __device__ __forceinline__ void emit(const Args& p, const Tiles& g, int b, int row0, int col0, uint32_t (&r)[32], const Fetched& f,
                                                uint32_t buf) {
        const float factor = scale(p, b);
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = __uint_as_float(r[e]) * factor;
        if constexpr (KIND == POLY) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t ah[4] = {f.hi[c].x, f.hi[c].y, f.hi[c].z, f.hi[c].w};
                uint32_t al[4] = {};
                if (PLANES == 2) { al[0] = f.lo[c].x; al[1] = f.lo[c].y; al[2] = f.lo[c].z; al[3] = f.lo[c].w; }
                float v[8];
                addend(p, row0 + (threadIdx.x & 31), col0 + c * 8, ah, al, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[c * 8 + e] += v[e];
            }
        }
        put(p, g, b, row0, col0, x, buf);
    }
};

struct Operands {
    const __half *left, *right;
    int M, N, K, pitch_l, pitch_r;
    int64_t slab_l, slab_r;
    int batch;
};

// pairs: tiles of 256 x 256; single CTAs: 128 x 128
template <int KIND, int PP, int CG>
using TileShape = gemm::Config<gemm::F16, PP, CG, CG == 2 ? 256 : 128, KIND == APPLY || KIND == LAST, KIND != GRAM, KIND == POLY>;

template <int KIND, int PP, int CG, typename OUT>
int run(const Operands& o, __half* out, int64_t out_pitch, int64_t out_slab, EpiArgs& args, int32_t* status, cudaStream_t s) {
    using C = TileShape<KIND, PP, CG>;
    CUtensorMap ml, mr;
    const int64_t slabs = (int64_t)o.batch * C::PLANES;
    int rc = gemm::make_map(&ml, gemm::F16, o.left, o.K, o.M, slabs, 2 * o.pitch_l, 2 * o.slab_l, 64, C::LSYM ? 64 : 128);
    if (rc) return rc;
    if (C::RMN) rc = gemm::make_map(&mr, gemm::F16, o.right, o.N, o.K, slabs, 2 * o.pitch_r, 2 * o.slab_r, 64, 64);
    else rc = gemm::make_map(&mr, gemm::F16, o.right, o.K, o.N, slabs, 2 * o.pitch_r, 2 * o.slab_r, 64, 64);
    if (rc) return rc;
    if (KIND != LAST) {
        rc = gemm::make_map(&args.map, gemm::F16, out, o.N, o.M, slabs, 2 * out_pitch, 2 * out_slab, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
        if (rc) return rc;
    }
    return gemm::launch<C, Epilogue<KIND, C::PLANES, OUT>>(ml, mr, gemm::tiles_of<C>(o.M, o.N, o.K, o.batch, KIND == GRAM || KIND == POLY), args,
                                                          status, s, true);
}

// Pairs or single CTAs, by the cycles that the waves of their tiles take per K block: a pair's 256 x 256 tile 512 (PP = 3:
// 1536), which is the tensor pipe's; a CTA's 128 x 128 tile 512 (1250), which is shared memory's.  Pairs are the better the
// more tiles there are; 16 + 16 rows of tiles of 777 x 1000 on 148 SMs run in one wave of pairs or two of single CTAs.
template <int KIND, int PP, typename OUT>
int choose(const Operands& o, __half* out, int64_t out_pitch, int64_t out_slab, EpiArgs& args, int32_t* status, cudaStream_t s) {
    constexpr bool SYM = KIND == GRAM || KIND == POLY;
    const int64_t pairs = gemm::tiles_of<TileShape<KIND, PP, 2>>(o.M, o.N, o.K, o.batch, SYM).total;
    const int64_t singles = gemm::tiles_of<TileShape<KIND, PP, 1>>(o.M, o.N, o.K, o.batch, SYM).total;
    const int64_t rest = pairs % 74;
    // half tiles in the last wave (see Tiles) count as 0.6
    const double pair_waves = pairs / 74 + (rest == 0 ? 0. : (pairs > 74 && 2 * rest <= 74 ? 0.6 : 1.));
    const double pair_time = pair_waves * (PP == 3 ? 1536 : 512), single_time = (double)ceil_div(singles, 148) * (PP == 3 ? 1250 : 512);
    return pair_time < single_time ? run<KIND, PP, 2, OUT>(o, out, out_pitch, out_slab, args, status, s)
                                   : run<KIND, PP, 1, OUT>(o, out, out_pitch, out_slab, args, status, s);
}
template <int KIND, typename OUT = float>
int product(const Shape& sh, const Operands& o, __half* out, int64_t out_pitch, int64_t out_slab, EpiArgs& args, int32_t* status, cudaStream_t s) {
    return sh.planes == 2 ? choose<KIND, 3, OUT>(o, out, out_pitch, out_slab, args, status, s)
                          : choose<KIND, 1, OUT>(o, out, out_pitch, out_slab, args, status, s);
}
}  // namespace

int launch_gram(const __half* x, __half* a, const float* alpha, const Shape& sh, int32_t* status, cudaStream_t s) {
    EpiArgs args{};
    args.alpha = alpha;
    return product<GRAM>(sh, {x, x, sh.s, sh.s, sh.l, sh.ls, sh.ls, sh.x_slab(), sh.x_slab(), sh.batch}, a, sh.ss, sh.a_slab(), args, status, s);
}
int launch_poly(const __half* a, __half* q, float ca, float cb, float cc, const Shape& sh, int32_t* status, cudaStream_t s) {
    EpiArgs args{};
    args.a = a; args.pitch = sh.ss; args.slab = sh.a_slab();
    args.ca = ca; args.cb = cb; args.cc = cc;
    return product<POLY>(sh, {a, a, sh.s, sh.s, sh.s, sh.ss, sh.ss, sh.a_slab(), sh.a_slab(), sh.batch}, q, sh.ss, sh.a_slab(), args, status, s);
}
int launch_apply(const __half* q, const __half* x, __half* x_next, const float* alpha, const float* alpha_next, const Shape& sh,
                 int32_t* status, cudaStream_t s) {
    EpiArgs args{};
    args.alpha = alpha; args.alpha_next = alpha_next;
    return product<APPLY>(sh, {q, x, sh.s, sh.l, sh.s, sh.ss, sh.ls, sh.a_slab(), sh.x_slab(), sh.batch}, x_next, sh.ls, sh.x_slab(), args, status, s);
}
int launch_apply_last(const __half* q, const __half* x, void* o, int dtype, bool tall, const float* alpha, const Shape& sh,
                      int32_t* status, cudaStream_t s) {
    EpiArgs args{};
    args.o = o; args.tall = tall; args.alpha = alpha;
    const Operands p{q, x, sh.s, sh.l, sh.s, sh.ss, sh.ls, sh.a_slab(), sh.x_slab(), sh.batch};
    if (dtype == CHEBYKAN_DTYPE_FP32) return product<LAST, float>(sh, p, nullptr, 0, 0, args, status, s);
    if (dtype == CHEBYKAN_DTYPE_BF16) return product<LAST, __nv_bfloat16>(sh, p, nullptr, 0, 0, args, status, s);
    return product<LAST, __half>(sh, p, nullptr, 0, 0, args, status, s);
}

}  // namespace ns
}  // namespace chebykan
