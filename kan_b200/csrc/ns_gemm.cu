// The three products of a Newton-Schulz step on tcgen05 (gemm_tc.cuh; see newton_schulz.cuh for the operands' layout):
//   A = X X^T            both operands are X's rows; symmetric
//   P = a I + b A + c A A      both operands are A's rows (A is symmetric); symmetric
//   X' = P X             P's rows against X as it lies, [K][N]: no transposed copy of X exists
// The symmetric two compute the tiles on and above the diagonal and write each block to both places.
#include "gemm_tc.cuh"
#include "newton_schulz.cuh"

namespace chebykan {
namespace ns {
namespace {
using gemm::Tiles;

enum { GRAM = 0, POLY = 1, APPLY = 2 };

struct EpiArgs {
    const __half* a;          // POLY: A's planes
    __half* out;              // planes, or null (APPLY's last step)
    float* out32;             // [batch][M][N]
    const float *alpha, *alpha_next;
    int pitch;                // of out (and of a)
    int64_t slab;
    float ca, cb, cc;
};

__device__ __forceinline__ uint32_t pack2(__half x, __half y) {
    return (uint32_t)__half_as_ushort(x) | ((uint32_t)__half_as_ushort(y) << 16);
}

template <int KIND, int PLANES>
struct Epilogue {
    using Args = EpiArgs;
    // NC consecutive columns of one row
    template <int NC>
    static __device__ __forceinline__ void emit(const Args& p, const Tiles& g, int b, int row, int col0, uint32_t (&r)[NC], bool mirror) {
        const int64_t slab0 = (int64_t)b * PLANES * p.slab;
        float factor;
        if (KIND == GRAM) { const float al = p.alpha[b]; factor = al * al * exp2f((float)A_EXP); }
        else if (KIND == POLY) factor = p.cc * exp2f(-2.f * A_EXP + P_EXP);
        else factor = exp2f(-(float)P_EXP) * p.alpha[b] / (p.out ? p.alpha_next[b] : 1.f);
        if (row >= g.M) return;
        if (KIND == APPLY && p.out == nullptr) {
            float* dst = p.out32 + ((int64_t)b * g.M + row) * g.N + col0;
            if ((g.N & 3) == 0) {
#pragma unroll
                for (int e = 0; e < NC; e += 4)
                    if (col0 + e < g.N)
                        *reinterpret_cast<float4*>(dst + e) = make_float4(__uint_as_float(r[e]) * factor, __uint_as_float(r[e + 1]) * factor,
                                                                          __uint_as_float(r[e + 2]) * factor, __uint_as_float(r[e + 3]) * factor);
            } else {
#pragma unroll
                for (int e = 0; e < NC; ++e)
                    if (col0 + e < g.N) dst[e] = __uint_as_float(r[e]) * factor;
            }
            return;
        }
        const int64_t at = slab0 + (int64_t)row * p.pitch + col0;
        // eight columns (16 bytes of a plane) at a time; a row's last group may run into its padding, which nothing reads
#pragma unroll
        for (int c = 0; c < NC; c += 8) {
            if (col0 + c >= g.N) break;
            __half hi[8], lo[8];
            uint4 ah, al;
            if (KIND == POLY) {
                ah = *reinterpret_cast<const uint4*>(p.a + at + c);
                if (PLANES == 2) al = *reinterpret_cast<const uint4*>(p.a + at + c + p.slab);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float v = __uint_as_float(r[c + e]) * factor;
                if (KIND == POLY) {
                    float a = __half2float(reinterpret_cast<const __half*>(&ah)[e]);
                    if (PLANES == 2) a += __half2float(reinterpret_cast<const __half*>(&al)[e]);
                    v = fmaf(p.cb * exp2f((float)(P_EXP - A_EXP)), a, v);
                    if (col0 + c + e == row) v += p.ca * exp2f((float)P_EXP);
                }
                split_half(v, hi[e], lo[e]);
            }
            *reinterpret_cast<uint4*>(p.out + at + c) = make_uint4(pack2(hi[0], hi[1]), pack2(hi[2], hi[3]), pack2(hi[4], hi[5]), pack2(hi[6], hi[7]));
            if (PLANES == 2)
                *reinterpret_cast<uint4*>(p.out + at + c + p.slab) = make_uint4(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]), pack2(lo[4], lo[5]), pack2(lo[6], lo[7]));
            if (KIND != APPLY && mirror) {
                // the warp's lanes hold consecutive rows: 64 bytes of one row of the transposed block
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col0 + c + e < g.N) {
                        const int64_t to = slab0 + (int64_t)(col0 + c + e) * p.pitch + row;
                        p.out[to] = hi[e];
                        if (PLANES == 2) p.out[to + p.slab] = lo[e];
                    }
            }
        }
    }
};

template <int KIND, int PP, int CG>
int run(const __half* left, const __half* right, int M, int N, int K, int pitch_l, int pitch_r, int64_t slab_l, int64_t slab_r, int batch,
        const EpiArgs& args, int32_t* status, cudaStream_t s) {
    using C = gemm::Config<gemm::F16, PP, CG, PP == 3 ? 128 : 256, KIND == APPLY>;
    CUtensorMap ml, mr;
    int rc = gemm::make_map(&ml, gemm::F16, left, K, M, (int64_t)batch * C::PLANES, 2 * pitch_l, 2 * slab_l, C::KE, 128);
    if (rc) return rc;
    if (KIND == APPLY) rc = gemm::make_map(&mr, gemm::F16, right, N, K, (int64_t)batch * C::PLANES, 2 * pitch_r, 2 * slab_r, 64, 64);
    else rc = gemm::make_map(&mr, gemm::F16, right, K, N, (int64_t)batch * C::PLANES, 2 * pitch_r, 2 * slab_r, C::KE, C::BN / C::CG);
    if (rc) return rc;
    return gemm::launch<C, Epilogue<KIND, C::PLANES>>(ml, mr, gemm::tiles_of<C>(M, N, K, batch, KIND != APPLY), args, status, s);
}

// CTA pairs (tiles of 256 rows) where there are enough of them to occupy every SM; single CTAs otherwise
template <int KIND, int PP>
int choose(const __half* left, const __half* right, int M, int N, int K, int pitch_l, int pitch_r, int64_t slab_l, int64_t slab_r, int batch,
           const EpiArgs& args, int32_t* status, cudaStream_t s) {
    using Pair = gemm::Config<gemm::F16, PP, 2, PP == 3 ? 128 : 256, KIND == APPLY>;
    if (gemm::tiles_of<Pair>(M, N, K, batch, KIND != APPLY).total >= 74)
        return run<KIND, PP, 2>(left, right, M, N, K, pitch_l, pitch_r, slab_l, slab_r, batch, args, status, s);
    return run<KIND, PP, 1>(left, right, M, N, K, pitch_l, pitch_r, slab_l, slab_r, batch, args, status, s);
}
template <int KIND>
int product(const Shape& sh, const __half* left, const __half* right, int N, int K, int pitch_l, int pitch_r, int64_t slab_l, int64_t slab_r,
            const EpiArgs& args, int32_t* status, cudaStream_t s) {
    if (sh.planes == 2)
        return choose<KIND, 3>(left, right, sh.s, N, K, pitch_l, pitch_r, slab_l, slab_r, sh.batch, args, status, s);
    return choose<KIND, 1>(left, right, sh.s, N, K, pitch_l, pitch_r, slab_l, slab_r, sh.batch, args, status, s);
}
}  // namespace

int launch_gram(const __half* x, __half* a, const float* alpha, const Shape& sh, int32_t* status, cudaStream_t s) {
    const EpiArgs args{nullptr, a, nullptr, alpha, nullptr, sh.ss, sh.a_slab(), 0, 0, 0};
    return product<GRAM>(sh, x, x, sh.s, sh.l, sh.ls, sh.ls, sh.x_slab(), sh.x_slab(), args, status, s);
}
int launch_poly(const __half* a, __half* q, float ca, float cb, float cc, const Shape& sh, int32_t* status, cudaStream_t s) {
    const EpiArgs args{a, q, nullptr, nullptr, nullptr, sh.ss, sh.a_slab(), ca, cb, cc};
    return product<POLY>(sh, a, a, sh.s, sh.s, sh.ss, sh.ss, sh.a_slab(), sh.a_slab(), args, status, s);
}
int launch_apply(const __half* q, const __half* x, __half* x_next, float* o, const float* alpha, const float* alpha_next, const Shape& sh,
                 int32_t* status, cudaStream_t s) {
    const EpiArgs args{nullptr, x_next, o, alpha, alpha_next, sh.ls, sh.x_slab(), 0, 0, 0};
    return product<APPLY>(sh, q, x, sh.l, sh.s, sh.ss, sh.ls, sh.a_slab(), sh.x_slab(), args, status, s);
}

}  // namespace ns
}  // namespace chebykan
