// The three products of a Newton-Schulz step on tcgen05 (gemm_tc.cuh; see newton_schulz.cuh for the operands' layout):
//   A = X X^T            both operands are X's rows; symmetric
//   P = a I + b A + c A A      both operands are A's rows (A is symmetric); symmetric
//   X' = P X             P's rows against X as it lies, [K][N]: no transposed copy of X exists
// The symmetric two compute the tiles on and above the diagonal and write each block to both places.
#include <type_traits>
#include "gemm_tc.cuh"
#include "newton_schulz.cuh"

namespace chebykan {
namespace ns {
namespace {
using gemm::Tiles;

enum { GRAM = 0, POLY = 1, APPLY = 2, LAST = 3 };       // LAST: the final APPLY, to the caller's layout and type

struct EpiArgs {
    const __half* a;          // POLY: A's planes
    __half* out;              // planes
    void* o;                  // LAST: [batch][m][n]
    int tall;                 // LAST: o is the transposed result
    const float *alpha, *alpha_next;
    int pitch;                // of out (and of a)
    int64_t slab;
    float ca, cb, cc;
};

// 8 columns of A's row, fetched ahead of the accumulator's
template <int NC, int PLANES>
struct Ahead {
    uint4 hi[NC / 8], lo[PLANES == 2 ? NC / 8 : 1];
};
struct Nothing {};

template <int KIND, int PLANES, typename OUT = float>
struct Epilogue {
    using Args = EpiArgs;
    template <int NC>
    using Fetched = typename std::conditional<KIND == POLY, Ahead<NC, PLANES>, Nothing>::type;

    // what emit() reads from memory, for the caller to ask for early
    template <int NC>
    static __device__ __forceinline__ void fetch(const Args& p, const Tiles& g, int b, int row, int col0, Fetched<NC>& f) {
        if constexpr (KIND == POLY) {
            if (row >= g.M) return;
            const __half* a = p.a + (int64_t)b * PLANES * p.slab + (int64_t)row * p.pitch + col0;
#pragma unroll
            for (int c = 0; c < NC / 8; ++c)
                if (col0 + c * 8 < g.N) {
                    f.hi[c] = *reinterpret_cast<const uint4*>(a + c * 8);
                    if (PLANES == 2) f.lo[c] = *reinterpret_cast<const uint4*>(a + c * 8 + p.slab);
                }
        }
    }

    // NC consecutive columns of one row
    template <int NC>
    static __device__ __forceinline__ void emit(const Args& p, const Tiles& g, int b, int row, int col0, uint32_t (&r)[NC], bool mirror,
                                                const Fetched<NC>& f) {
        float factor;
        if (KIND == GRAM) { const float al = p.alpha[b]; factor = al * al * exp2f((float)A_EXP); }
        else if (KIND == POLY) factor = p.cc * exp2f(-2.f * A_EXP + P_EXP);
        else if (KIND == APPLY) factor = exp2f(-(float)P_EXP) * p.alpha[b] / p.alpha_next[b];
        else factor = exp2f(-(float)P_EXP) * p.alpha[b];
        if (row >= g.M) return;
        if constexpr (KIND == LAST) {
            OUT* o = reinterpret_cast<OUT*>(p.o) + (int64_t)b * g.M * g.N;
            if (p.tall) {                       // the warp's lanes hold consecutive rows, which are o's columns
#pragma unroll
                for (int e = 0; e < NC; ++e)
                    if (col0 + e < g.N) o[(int64_t)(col0 + e) * g.M + row] = from_float<OUT>(__uint_as_float(r[e]) * factor);
                return;
            }
            OUT* dst = o + (int64_t)row * g.N + col0;
            constexpr int V = 16 / (int)sizeof(OUT);
            const bool vec = g.N % V == 0;
#pragma unroll
            for (int c = 0; c < NC; c += V) {
                alignas(16) OUT v[V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = from_float<OUT>(__uint_as_float(r[c + e]) * factor);
                if (vec) {
                    if (col0 + c < g.N) *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(v);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (col0 + c + e < g.N) dst[c + e] = v[e];
                }
            }
            return;
        } else {
            const int64_t slab0 = (int64_t)b * PLANES * p.slab, at = slab0 + (int64_t)row * p.pitch + col0;
            // eight columns (16 bytes of a plane) at a time; a row's last group may run into its padding, which nothing reads
#pragma unroll
            for (int c = 0; c < NC; c += 8) {
                if (col0 + c >= g.N) break;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r[c + e]) * factor;
                if constexpr (KIND == POLY) {
                    float a[8];
                    const uint32_t ah[4] = {f.hi[c / 8].x, f.hi[c / 8].y, f.hi[c / 8].z, f.hi[c / 8].w};
                    uint32_t al[4] = {};
                    if (PLANES == 2) { al[0] = f.lo[c / 8].x; al[1] = f.lo[c / 8].y; al[2] = f.lo[c / 8].z; al[3] = f.lo[c / 8].w; }
                    join8<PLANES>(ah, al, a);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[e] = fmaf(p.cb * exp2f((float)(P_EXP - A_EXP)), a[e], v[e]);
                        if (col0 + c + e == row) v[e] += p.ca * exp2f((float)P_EXP);
                    }
                }
                uint32_t hi[4], lo[4];
                split8<PLANES>(v, hi, lo);
                *reinterpret_cast<uint4*>(p.out + at + c) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if (PLANES == 2) *reinterpret_cast<uint4*>(p.out + at + c + p.slab) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                if (KIND != APPLY && mirror) {
                    // the warp's lanes hold consecutive rows: 64 bytes of one row of the transposed block
                    unsigned short* to = reinterpret_cast<unsigned short*>(p.out) + slab0 + (int64_t)(col0 + c) * p.pitch + row;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (col0 + c + e < g.N) {
                            to[(int64_t)e * p.pitch] = (unsigned short)(hi[e >> 1] >> (16 * (e & 1)));
                            if (PLANES == 2) to[(int64_t)e * p.pitch + p.slab] = (unsigned short)(lo[e >> 1] >> (16 * (e & 1)));
                        }
                }
            }
        }
    }
};

struct Operands {
    const __half *left, *right;
    int M, N, K, pitch_l, pitch_r;
    int64_t slab_l, slab_r;
    int batch;
};

template <int KIND, int PP, int CG, typename OUT>
int run(const Operands& o, const EpiArgs& args, int32_t* status, cudaStream_t s) {
    constexpr bool MN = KIND == APPLY || KIND == LAST;
    using C = gemm::Config<gemm::F16, PP, CG, PP == 3 ? 128 : 256, MN>;
    CUtensorMap ml, mr;
    const int64_t slabs = (int64_t)o.batch * C::PLANES;
    int rc = gemm::make_map(&ml, gemm::F16, o.left, o.K, o.M, slabs, 2 * o.pitch_l, 2 * o.slab_l, C::KE, 128);
    if (rc) return rc;
    if (MN) rc = gemm::make_map(&mr, gemm::F16, o.right, o.N, o.K, slabs, 2 * o.pitch_r, 2 * o.slab_r, 64, 64);
    else rc = gemm::make_map(&mr, gemm::F16, o.right, o.K, o.N, slabs, 2 * o.pitch_r, 2 * o.slab_r, C::KE, C::BN / CG);
    if (rc) return rc;
    return gemm::launch<C, Epilogue<KIND, C::PLANES, OUT>>(ml, mr, gemm::tiles_of<C>(o.M, o.N, o.K, o.batch, !MN), args, status, s);
}

// CTA pairs (tiles of 256 rows) where there are enough of them to occupy every SM; single CTAs otherwise
template <int KIND, int PP, typename OUT>
int choose(const Operands& o, const EpiArgs& args, int32_t* status, cudaStream_t s) {
    constexpr bool MN = KIND == APPLY || KIND == LAST;
    using Pair = gemm::Config<gemm::F16, PP, 2, PP == 3 ? 128 : 256, MN>;
    if (gemm::tiles_of<Pair>(o.M, o.N, o.K, o.batch, !MN).total >= 74) return run<KIND, PP, 2, OUT>(o, args, status, s);
    return run<KIND, PP, 1, OUT>(o, args, status, s);
}
template <int KIND, typename OUT = float>
int product(const Shape& sh, const Operands& o, const EpiArgs& args, int32_t* status, cudaStream_t s) {
    return sh.planes == 2 ? choose<KIND, 3, OUT>(o, args, status, s) : choose<KIND, 1, OUT>(o, args, status, s);
}
}  // namespace

int launch_gram(const __half* x, __half* a, const float* alpha, const Shape& sh, int32_t* status, cudaStream_t s) {
    const EpiArgs args{nullptr, a, nullptr, 0, alpha, nullptr, sh.ss, sh.a_slab(), 0, 0, 0};
    return product<GRAM>(sh, {x, x, sh.s, sh.s, sh.l, sh.ls, sh.ls, sh.x_slab(), sh.x_slab(), sh.batch}, args, status, s);
}
int launch_poly(const __half* a, __half* q, float ca, float cb, float cc, const Shape& sh, int32_t* status, cudaStream_t s) {
    const EpiArgs args{a, q, nullptr, 0, nullptr, nullptr, sh.ss, sh.a_slab(), ca, cb, cc};
    return product<POLY>(sh, {a, a, sh.s, sh.s, sh.s, sh.ss, sh.ss, sh.a_slab(), sh.a_slab(), sh.batch}, args, status, s);
}
int launch_apply(const __half* q, const __half* x, __half* x_next, const float* alpha, const float* alpha_next, const Shape& sh,
                 int32_t* status, cudaStream_t s) {
    const EpiArgs args{nullptr, x_next, nullptr, 0, alpha, alpha_next, sh.ls, sh.x_slab(), 0, 0, 0};
    return product<APPLY>(sh, {q, x, sh.s, sh.l, sh.s, sh.ss, sh.ls, sh.a_slab(), sh.x_slab(), sh.batch}, args, status, s);
}
int launch_apply_last(const __half* q, const __half* x, void* o, int dtype, bool tall, const float* alpha, const Shape& sh,
                      int32_t* status, cudaStream_t s) {
    const EpiArgs args{nullptr, nullptr, o, tall, alpha, nullptr, sh.ls, sh.x_slab(), 0, 0, 0};
    const Operands p{q, x, sh.s, sh.l, sh.s, sh.ss, sh.ls, sh.a_slab(), sh.x_slab(), sh.batch};
    if (dtype == CHEBYKAN_DTYPE_FP32) return product<LAST, float>(sh, p, args, status, s);
    if (dtype == CHEBYKAN_DTYPE_BF16) return product<LAST, __nv_bfloat16>(sh, p, args, status, s);
    return product<LAST, __half>(sh, p, args, status, s);
}

}  // namespace ns
}  // namespace chebykan
