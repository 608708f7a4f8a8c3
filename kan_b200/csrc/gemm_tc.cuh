// D[M][N] = L[M][K] R on tcgen05, for 16-bit floating and 8-bit integer operands: the pipeline shared by the products of
// the Newton-Schulz steps and of the 8-bit forward.  What happens to the accumulator is the epilogue's, a template argument:
// emit() takes 32 columns of a row per lane, fetch() asks one step earlier for what emit() will read from memory.  (PP = 3
// sums in registers anyway: there the sums start from init() and take the accumulators times scale(), and put() writes.)
//
//   warp 0     TMA: one stage = 128 bytes of K of the tile's L rows (128 per CTA) and of R, 128-byte swizzle, no multicast.
//              R is either [N][K] (K-major) or [K][N] (boxes of 64 K rows x 64 columns, read through an MN-major descriptor)
//   warp 1     MMA: one elected lane issues tcgen05.mma and the commits that free stages and publish accumulators
//   warps 2-9  epilogue: tcgen05.ld, then emit(); two warps share a quarter of tensor memory's lanes, half of the columns each
//
// CG = 2: a pair of CTAs works on 256 rows with cta_group::2, each staging its own 128 rows of L and half of R's columns,
// which halves R's traffic out of L2 and the shared-memory reads per MMA.  The even CTA's thread issues the MMAs.
// PP = 3: both operands come as two fp16 planes (head and tail) and three products are summed.  The tensor pipe's fp32 sums
// truncate, by about 2^-26 of the accumulator per MMA, so the accumulator of head x head takes one K block (4 MMAs) at a
// time and the epilogue warps add the blocks up in registers, rounding to nearest (580 cycles), while the MMAs of
// head x tail and tail x head run (1024); those are 2^11 times smaller and stay in an accumulator of their own for the
// whole of K.  Two K blocks at a time were no faster and lost half a digit.
// BN = 256 with pairs: per K block of 64 an SM's shared memory then takes 64 KB and gives 96 KB in the 1536 cycles of 12 MMAs
// (104 of its 128 bytes per cycle); with BN = 128 it would be 160 bytes per cycle, which held the products at 3/4 of the
// pipe's rate.
// PP = 1: two accumulators alternate, so a tile's epilogue overlaps the next tile's MMAs.
// Symmetric operands (LSYM, RSYM) are stored only in the 256 x 256 blocks on and above the diagonal: a block below it is
// loaded from its mirror image and read through the other major-ness, which is a bit of the instruction descriptor.
// Measured: 65536 x 8192 -> 1024 in int8 340 us alone (3.2 POP/s; the tensor pipe's 512 cycles per K block, plus a tail of one
// epilogue); 4 x 2048 x 2048 bf16 P X 54 to 57 us from its start to the next kernel's (1.2 to
// 1.28 PFLOP/s); 9 x 1024 x 1024 in two planes 127 us for a step's A, P and X' (71 at the
// pipe's rate): an epilogue of some 7000 cycles (twice that for P, which also reads A) holds up the 24600 cycles of a tile's MMAs.
// Every wait is bounded (see tc_common.cuh).
#pragma once
#include "tc_common.cuh"

namespace chebykan {
namespace gemm {
using namespace tc;

enum Kind { F16 = 0, I8 = 1 };

template <Kind KIND_, int PP_, int CG_, int BN_, bool RMN_, bool LSYM_ = false, bool RSYM_ = false>
struct Config {
    static constexpr Kind KIND = KIND_;
    static constexpr int PP = PP_, CG = CG_, BN = BN_;
    static constexpr bool RMN = RMN_, LSYM = LSYM_, RSYM = RSYM_;
    static constexpr int PLANES = PP == 3 ? 2 : 1;
    static constexpr bool HALVES = KIND == F16 && CG == 2;     // the last tiles may be cut in two (see Tiles)
    static constexpr int BM = 128 * CG;                        // rows of a tile
    static constexpr int KE = KIND == I8 ? 128 : 64;           // K elements per stage (128 bytes)
    static constexpr int L_PANEL = 128 * 128, R_PANEL = BN / CG * 128;
    static constexpr int STAGE = PLANES * (L_PANEL + R_PANEL);
    static constexpr int STAGES = (192 * 1024) / STAGE > 8 ? 8 : (192 * 1024) / STAGE;
    static constexpr int TMEM_COLS = 2 * BN;                   // two accumulators; PP = 3: heads, cross products
    static constexpr int BARS = 2 * STAGES + 5;
    static constexpr int OUT_OFFSET = STAGES * STAGE;          // 4 KB per epilogue warp
    static constexpr int BAR_OFFSET = OUT_OFFSET + 8 * 4096;
    static constexpr int SMEM = BAR_OFFSET + BARS * 8 + 16 + 1024;
    static constexpr uint32_t IDESC = KIND == I8
        ? (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24)
        : (1u << 4) | ((RMN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
    static_assert(TMEM_COLS <= 512 && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "accumulators must fit tensor memory");
    static_assert(KIND == F16 || (PP == 1 && !RMN && !LSYM && !RSYM), "integer products have one plane and K-major operands");
    static_assert(!(RMN && RSYM), "a symmetric right operand is K-major");
};
constexpr int THREADS = 320, EPI_THREADS = 256;
enum { ST_LOAD = 21, ST_MMA = 22, ST_MMA_ACC = 23, ST_EPILOGUE = 24 };

struct Tiles {
    int M, N;
    int nkb;              // K blocks of a tile
    int ntm, ntn;         // tile rows and columns
    int per_batch;        // tiles of one matrix
    int sym;              // only the 256 x 256 blocks on and above the diagonal
    // Tiles from `whole` on are cut into two of half the width: what is left after the last full wave, where the halves fit
    // into one.  90 tiles on 74 pairs then take about 1.6 tiles' time instead of 2.  total counts the halves.
    int64_t whole, total;
};

// whether element (i, j) of a symmetric matrix is stored
__host__ __device__ __forceinline__ bool stored(int i, int j) { return j / 256 >= i / 256; }

// position of tile t: matrix b, first row, first column; true for half a tile
template <int BM, int BN>
__device__ __forceinline__ bool decode(const Tiles& g, int64_t t, int& b, int& m0, int& n0) {
    const bool half = t >= g.whole;
    const int second = half ? (int)(t - g.whole) & 1 : 0;
    if (half) t = g.whole + ((t - g.whole) >> 1);
    b = (int)(t / g.per_batch);
    int r = (int)(t - (int64_t)b * g.per_batch);
    if (!g.sym) {
        m0 = r / g.ntn * BM;
        n0 = r % g.ntn * BN;
    } else {
        int tm = 0;
        for (;; ++tm) {
            const int first = tm * BM / 256 * (256 / BN), count = g.ntn - first;
            if (r < count) { m0 = tm * BM; n0 = (first + r) * BN; break; }
            r -= count;
        }
    }
    n0 += second * (BN / 2);
    return half;
}
inline int sym_tiles(int ntm, int ntn, int bm, int bn) {
    int n = 0;
    for (int tm = 0; tm < ntm; ++tm) n += ntn - tm * bm / 256 * (256 / bn);
    return n;
}

template <Kind KIND, int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (KIND == F16) {
        if constexpr (CG == 2) umma2<CHEBYKAN_MODE_BF16>(d, a, b, idesc, accumulate);
        else umma<CHEBYKAN_MODE_BF16>(d, a, b, idesc, accumulate);
    } else if constexpr (CG == 2) {
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    } else {
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    }
}
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
__device__ __forceinline__ void load_3d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
// v[0..BN) (+)= scale * columns of an accumulator; the next 16 are on their way while 16 are added
template <int BN, bool SET>
__device__ __forceinline__ void add_columns(uint32_t taddr, float scale, float (&v)[BN]) {
    uint32_t r[2][16];
    tmem_ld16(taddr, r[0]);
#pragma unroll
    for (int c = 0; c < BN / 16; ++c) {
        tmem_ld_wait();
        if (c + 1 < BN / 16) tmem_ld16(taddr + (c + 1) * 16, r[(c + 1) & 1]);
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const f32x2 x = pair_of(__uint_as_float(r[c & 1][e]), __uint_as_float(r[c & 1][e + 1]));
            const int i = c * 16 + e;
            halves(SET ? mul2(x, pair_of(scale, scale)) : fma2(x, pair_of(scale, scale), pair_of(v[i], v[i + 1])), v[i], v[i + 1]);
        }
    }
}
// ---- writing a warp's 32 rows x 32 columns, through its 4 KB of shared memory so that lanes write along rows ----
__device__ __forceinline__ void st_shared_v4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// each lane holds a row's 32 values; rows are `pitch` elements apart from dst on, `rows` x `cols` of them exist.  vec: the
// row's start and pitch are multiples of 16 bytes
template <typename OUT>
__device__ __forceinline__ void store_rows(uint32_t buf, const OUT (&v)[32], OUT* dst, int64_t pitch, int rows, int cols, bool vec) {
    constexpr int ROW = 32 * (int)sizeof(OUT), CHUNKS = ROW / 16, V = 16 / (int)sizeof(OUT);
    const int lane = threadIdx.x & 31;
    // 16-byte chunks are permuted within a row so that neither side's eight lanes meet in a bank
    auto place = [&](int r, int c) { return buf + (uint32_t)(r * ROW + ((CHUNKS == 8 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4)); };
    const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) st_shared_v4(place(lane, c), w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
    __syncwarp();
    if (vec && cols >= 32) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const int r = (i * 32 + lane) / CHUNKS, c = (i * 32 + lane) % CHUNKS;
            uint32_t x[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(place(r, c)));
            if (r < rows) *reinterpret_cast<uint4*>(dst + r * pitch + c * V) = make_uint4(x[0], x[1], x[2], x[3]);
        }
    } else {
        // ragged right edge, or rows that are not 16 bytes apart: a column per lane, row after row
        const uint32_t in = (uint32_t)(lane % V * (int)sizeof(OUT));
        OUT* to = dst + lane;
#pragma unroll 8
        for (int r = 0; r < 32; ++r) {
            const uint32_t at = place(r, lane / V) + in;
            if constexpr (sizeof(OUT) == 4) {
                uint32_t x;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at));
                if (r < rows && lane < cols) *reinterpret_cast<uint32_t*>(to + r * pitch) = x;
            } else {
                unsigned short x;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at));
                if (r < rows && lane < cols) *reinterpret_cast<unsigned short*>(to + r * pitch) = x;
            }
        }
    }
    __syncwarp();
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                 ::"l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(src) : "memory");
}

template <class C, class Epi>
__global__ void __launch_bounds__(THREADS, 1)
gemm_kernel(const __grid_constant__ CUtensorMap map_l, const __grid_constant__ CUtensorMap map_r, const Tiles g,
             const __grid_constant__ typename Epi::Args args, int32_t* status) {
    constexpr int CG = C::CG, BN = C::BN, S = C::STAGES, PLANES = C::PLANES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + C::BAR_OFFSET;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (S + s); };
    auto acc_full = [&](int a) { return bars + 8u * (2 * S + a); };
    auto acc_empty = [&](int a) { return bars + 8u * (2 * S + 2 + a); };
    const uint32_t drain = bars + 8u * (2 * S + 4);
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + C::BAR_OFFSET + C::BARS * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + C::BAR_OFFSET + C::BARS * 8 + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
    const int64_t unit = blockIdx.x / CG, units = gridDim.x / CG;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(acc_full(a), 1); mbar_init(acc_empty(a), EPI_THREADS * CG); }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                         ::"r"(smem_u32((const void*)tmem_slot)), "r"((uint32_t)C::TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                         ::"r"(smem_u32((const void*)tmem_slot)), "r"((uint32_t)C::TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();      // the peer's barriers exist before anything arrives on them
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    let_next_start();
    wait_for_previous();

    if (warp == 0) {
        if (lane == 0) {
            int s = 0; uint32_t ph = 0;
            bool alive = true;
            for (int64_t t = unit; t < g.total && alive; t += units) {
                int b, m0, n0;
                const bool half = decode<C::BM, BN>(g, t, b, m0, n0);
                const int width = (half ? BN / 2 : BN) / CG;             // this CTA's share of R's columns
                const int row = m0 + (int)rank * 128, col = n0 + (int)rank * width;
                const uint32_t bytes = (uint32_t)(PLANES * CG * (C::L_PANEL + width * 128));
                for (int kb = 0; kb < g.nkb; ++kb) {
                    if (!mbar_wait(empty(s), ph ^ 1u, abort_flag, status, ST_LOAD)) { alive = false; break; }
                    const uint32_t dst = base + s * C::STAGE;
                    uint32_t bar = full(s);
                    if (rank == 0) mbar_arrive_expect_tx(bar, bytes);
                    if (CG == 2) bar = mapa_cluster(bar, 0);
                    auto load = [&](uint32_t to, const CUtensorMap* map, int c0, int c1, int z) {
                        if (CG == 2) load_3d_pair(to, map, c0, c1, z, bar);
                        else load_3d(to, map, c0, c1, z, bar);
                    };
                    const int k0 = kb * C::KE;
                    // 128 (or 64) rows from r0 of a symmetric matrix against its columns from k0: two boxes, or their mirror images
                    auto load_sym = [&](uint32_t to, const CUtensorMap* map, int r0, int rows, int z) {
                        const bool direct = stored(r0, k0);
                        for (int q = 0; q < rows; q += 64) load(to + q * 128, map, direct ? k0 : r0 + q, direct ? r0 + q : k0, z);
                    };
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) {
                        const int z = b * PLANES + p;
                        if (C::LSYM) load_sym(dst + p * C::L_PANEL, &map_l, row, 128, z);
                        else load(dst + p * C::L_PANEL, &map_l, k0, row, z);
                        const uint32_t rd = dst + PLANES * C::L_PANEL + p * C::R_PANEL;
                        if (C::RMN) {
                            for (int q = 0; q < width; q += 64) load(rd + q * 128, &map_r, col + q, k0, z);
                        } else if (C::RSYM) {
                            load_sym(rd, &map_r, col, width, z);
                        } else if (C::KIND == F16) {
                            for (int q = 0; q < width; q += 64) load(rd + q * 128, &map_r, k0, col + q, z);
                        } else {
                            load(rd, &map_r, k0, col, z);
                        }
                    }
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
            }
            if (!alive) {
                // let the copies already issued land before the CTA gives up its shared memory
                const uint64_t t0 = globaltimer_ns();
                while (globaltimer_ns() - t0 < 200000ull) { }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const bool elected = elect_one_sync();
            int s = 0; uint32_t ph = 0;
            int acc = 0; uint32_t acc_ph = 0, cross_ph = 0;
            bool alive = true;
            // descriptors of the first stage; only low words move.  K-major: a step of 16 (32) columns is 32 bytes; MN-major: 16
            // rows of 128 bytes, and the next 64 columns a box further (bits 16-29)
            const uint64_t l_desc = make_smem_desc(base), r_desc = make_smem_desc(base + PLANES * C::L_PANEL);
            const uint32_t l_hi = (uint32_t)(l_desc >> 32), r_hi = (uint32_t)(r_desc >> 32);
            constexpr uint32_t L_TAIL = C::L_PANEL >> 4, R_TAIL = C::R_PANEL >> 4;
            constexpr uint32_t KSTEP = 32 >> 4, MNSTEP = 2048 >> 4, MNBOX = (8192u >> 4) << 16, LBO = 0x3fffu << 16;
            const uint32_t l_k = (uint32_t)l_desc, l_mn = ((uint32_t)l_desc & ~LBO) | MNBOX;
            const uint32_t r_k = (uint32_t)r_desc, r_mn = ((uint32_t)r_desc & ~LBO) | MNBOX;
            auto wait_all = [&](uint32_t bar, uint32_t parity, int code) {
                if (!__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code))) alive = false;
                tc_fence_after();
                return alive;
            };
            auto commit = [&](uint32_t bar) {
                if (elected) { if (CG == 2) umma2_commit_both(bar); else umma_commit(bar); }
                __syncwarp();
            };
            for (int64_t t = unit; t < g.total && alive; t += units) {
                int b, m0 = 0, n0 = 0;
                const bool half = decode<C::BM, BN>(g, t, b, m0, n0);
                const uint32_t idesc0 = half ? C::IDESC - ((uint32_t)(BN >> 4) << 17) : C::IDESC;       // N halved
                if (C::PP == 1 && !wait_all(acc_empty(acc), acc_ph ^ 1u, ST_MMA_ACC)) break;
                const uint32_t d = C::PP == 1 ? tmem + (uint32_t)(acc * BN) : tmem, cross = tmem + BN;
                // one stage's operands: low words and steps of the descriptors, and the instruction's
                struct Operand { uint32_t l, r, lstep, rstep, idesc; };
                auto operands = [&](int kb) {
                    const uint32_t off = (uint32_t)((s * C::STAGE) >> 4);
                    const bool lmn = C::LSYM && !stored(m0, kb * C::KE);
                    const bool rmn = C::RMN || (C::RSYM && !stored(n0, kb * C::KE));
                    return Operand{(lmn ? l_mn : l_k) + off, (rmn ? r_mn : r_k) + off, lmn ? MNSTEP : KSTEP, rmn ? MNSTEP : KSTEP,
                                   idesc0 | (lmn ? 1u << 15 : 0u) | (rmn ? 1u << 16 : 0u)};
                };
                // operands are formed by the whole warp, in uniform registers, and only the MMA itself is one lane's
                auto issue = [&](uint32_t dst, uint32_t l, uint32_t r, uint32_t id, uint32_t accumulate) {
                    const uint64_t ld = desc_from_words(l, l_hi), rd = desc_from_words(r, r_hi);
                    if (elected) mma<C::KIND, CG>(dst, ld, rd, id, accumulate);
                };
                auto heads = [&](const Operand& o, bool start) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) issue(d, o.l + o.lstep * k, o.r + o.rstep * k, o.idesc, k ? 1u : (uint32_t)!start);
                };
                auto next_stage = [&]() { if (++s == S) { s = 0; ph ^= 1u; } };
                if constexpr (C::PP == 1) {
                    for (int kb = 0; kb < g.nkb; ++kb) {
                        if (!wait_all(full(s), ph, ST_MMA)) break;
                        heads(operands(kb), kb == 0);
                        commit(empty(s));
                        next_stage();
                    }
                } else {
                    auto tails = [&](const Operand& o, bool start) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t la = o.l + o.lstep * k, ra = o.r + o.rstep * k;
                            issue(cross, la, ra + R_TAIL, o.idesc, k ? 1u : (uint32_t)!start);
                            issue(cross, la + L_TAIL, ra, o.idesc, 1u);
                        }
                    };
                    for (int kb = 0; kb < g.nkb; ++kb) {
                        if (!wait_all(acc_empty(0), acc_ph ^ 1u, ST_MMA_ACC)) break;
                        if (!wait_all(full(s), ph, ST_MMA)) break;
                        const Operand o = operands(kb);
                        heads(o, true);
                        commit(acc_full(0));                       // added up while the cross products run
                        acc_ph ^= 1u;
                        if (kb == 0) {
                            if (!wait_all(acc_empty(1), cross_ph ^ 1u, ST_MMA_ACC)) break;
                            cross_ph ^= 1u;
                        }
                        tails(o, kb == 0);
                        commit(empty(s));
                        next_stage();
                    }
                }
                if (!alive) break;
                if (C::PP == 3) {
                    commit(acc_full(1));
                } else {
                    commit(acc_full(acc));
                    acc ^= 1;
                    if (acc == 0) acc_ph ^= 1u;
                }
            }
            if (!alive && elected) {
                // wait (bounded) until the MMAs already issued have retired
                if (CG == 2) umma2_commit(drain); else umma_commit(drain);
                const uint64_t t0 = globaltimer_ns();
                while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < 10000000ull) { }
            }
            __syncwarp();
        }
    } else {
        const int q = warp & 3;               // quarter of the tensor memory's lanes that this warp may read
        const uint32_t buf = base + C::OUT_OFFSET + (uint32_t)((warp - 2) * 4096);
        int acc = 0; uint32_t acc_ph = 0, cross_ph = 0;
        bool alive = true;
        auto wait_all = [&](uint32_t bar, uint32_t parity) {
            if (!__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, ST_EPILOGUE))) alive = false;
            tc_fence_after();
            return alive;
        };
        auto release = [&](int a) {
            tc_fence_before();
            if (CG == 2 && rank != 0) mbar_arrive_cluster(mapa_cluster(acc_empty(a), 0));
            else mbar_arrive(acc_empty(a));
        };
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        constexpr int EB = BN / 2;            // columns of this warp (half of them mean nothing in half a tile)
        for (int64_t t = unit; t < g.total && alive; t += units) {
            int b, m0, n0;
            const int width = decode<C::BM, BN>(g, t, b, m0, n0) ? EB / 2 : EB;
            const int half0 = (warp - 2) / 4 * width;
            n0 += half0;
            const int row0 = m0 + (int)rank * 128 + q * 32;
            int ncols = g.N - n0;
            if (ncols > width) ncols = width;
            const int nch = ncols > 0 && row0 < g.M ? (ncols + 31) >> 5 : 0;
            if constexpr (C::PP == 3) {
                const float scale = Epi::scale(args, b);
                float v[EB];
                if (Epi::INIT) Epi::init(args, g, b, row0, n0, v, buf);      // while the first MMAs run
                for (int kb = 0; kb < g.nkb; ++kb) {
                    if (!wait_all(acc_full(0), acc_ph)) break;
                    acc_ph ^= 1u;
                    if (!Epi::INIT && kb == 0) add_columns<EB, true>(tmem + lanes + (uint32_t)half0, scale, v);
                    else add_columns<EB, false>(tmem + lanes + (uint32_t)half0, scale, v);
                    release(0);
                }
                if (!alive) break;
                if (!wait_all(acc_full(1), cross_ph)) break;
                cross_ph ^= 1u;
                add_columns<EB, false>(tmem + lanes + (uint32_t)(BN + half0), scale, v);
                release(1);
#pragma unroll
                for (int c = 0; c < EB / 32; ++c)
                    if (c < nch) {
                        float x[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] = v[c * 32 + e];
                        Epi::put(args, g, b, row0, n0 + c * 32, x, buf);
                    }
            } else {
                typename Epi::Fetched fa, fb;
                Epi::fetch(args, g, b, row0 + lane, n0, fa);
                if (!wait_all(acc_full(acc), acc_ph)) break;
                const uint32_t ta = tmem + lanes + (uint32_t)(acc * BN + half0);
                // two register buffers: the load of the next 32 columns is in flight while these are written
                uint32_t ra[32], rb[32];
                if (nch > 0) tmem_ld32(ta, ra);
                else release(acc);
#pragma unroll 1
                for (int c = 0; c < nch; c += 2) {
                    tmem_ld_wait();
                    if (c + 1 < nch) {
                        tmem_ld32(ta + (c + 1) * 32, rb);
                        Epi::fetch(args, g, b, row0 + lane, n0 + (c + 1) * 32, fb);
                    } else {
                        release(acc);
                    }
                    Epi::emit(args, g, b, row0, n0 + c * 32, ra, fa, buf);
                    if (c + 1 < nch) {
                        tmem_ld_wait();
                        if (c + 2 < nch) {
                            tmem_ld32(ta + (c + 2) * 32, ra);
                            Epi::fetch(args, g, b, row0 + lane, n0 + (c + 2) * 32, fa);
                        } else {
                            release(acc);
                        }
                        Epi::emit(args, g, b, row0, n0 + (c + 1) * 32, rb, fb, buf);
                    }
                }
                acc ^= 1;
                if (acc == 0) acc_ph ^= 1u;
            }
        }
        if (Epi::BULK && lane == 0) bulk_wait_all();
    }

    tc_fence_before();
    __syncthreads();
    // neither CTA of a pair leaves (or frees tensor memory) while the other may still arrive on its barriers
    if (CG == 2) cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        if (CG == 2)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::TMEM_COLS) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::TMEM_COLS) : "memory");
    }
}

// ---- few tiles: the K range of a tile split over the CTAs of a cluster ------------------------------------------------
// Integer products.  One tile of 128 x BN per cluster of SPLIT CTAs (SPLIT a run-time power of two up to 8).  Every CTA sums its share of the
// K blocks in tensor memory, leaves the partial tile in its shared memory, and after a cluster barrier adds up 128 / SPLIT
// rows of all partials through distributed shared memory, in rank order, and writes them: one launch, no scratch, no
// atomics, the same result every time.
__device__ __forceinline__ void ld_cluster_v4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <class C>
struct SplitSmem {
    static constexpr int PITCH = (C::BN + 4) * 4;                   // bytes of a partial row: 16-byte stores of 8 rows meet no bank twice
    static constexpr int PARTIAL = 128 * PITCH;
    static constexpr int RING = C::STAGES * C::STAGE > PARTIAL ? C::STAGES * C::STAGE : PARTIAL;
    static constexpr int BARS = 2 * C::STAGES + 2;
    static constexpr int TOTAL = RING + BARS * 8 + 16 + 1024;
};

template <class C, class Epi>
__global__ void __launch_bounds__(THREADS, 1)
split_kernel(const __grid_constant__ CUtensorMap map_l, const __grid_constant__ CUtensorMap map_r, const Tiles g,
             const __grid_constant__ typename Epi::Args args, int split, int32_t* status) {
    static_assert(C::KIND == I8 && C::CG == 1, "integer sums, one CTA per accumulator");
    using L = SplitSmem<C>;
    constexpr int BN = C::BN, S = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + L::RING;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (S + s); };
    const uint32_t done = bars + 8u * (2 * S), drain = done + 8u;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + L::RING + L::BARS * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + L::RING + L::BARS * 8 + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        mbar_init(done, 1);
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void*)tmem_slot)), "r"((uint32_t)C::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    let_next_start();
    wait_for_previous();

    int b, m0, n0;
    decode<C::BM, BN>(g, blockIdx.x / split, b, m0, n0);
    // this CTA's K blocks (every CTA has at least one: the launch sees to it)
    const int k_first = (int)((int64_t)g.nkb * rank / split), k_last = (int)((int64_t)g.nkb * (rank + 1) / split);

    if (warp == 0) {
        if (lane == 0) {
            int s = 0; uint32_t ph = 0;
            bool alive = true;
            for (int kb = k_first; kb < k_last; ++kb) {
                if (!mbar_wait(empty(s), ph ^ 1u, abort_flag, status, ST_LOAD)) { alive = false; break; }
                const uint32_t dst = base + s * C::STAGE;
                mbar_arrive_expect_tx(full(s), (uint32_t)C::STAGE);
                load_3d(dst, &map_l, kb * C::KE, m0, 0, full(s));
                load_3d(dst + C::L_PANEL, &map_r, kb * C::KE, n0, 0, full(s));
                if (++s == S) { s = 0; ph ^= 1u; }
            }
            if (!alive) {
                const uint64_t t0 = globaltimer_ns();
                while (globaltimer_ns() - t0 < 200000ull) { }
            }
        }
    } else if (warp == 1) {
        const bool elected = elect_one_sync();
        int s = 0; uint32_t ph = 0;
        bool alive = true;
        const uint64_t l_desc = make_smem_desc(base), r_desc = make_smem_desc(base + C::L_PANEL);
        const uint32_t l_hi = (uint32_t)(l_desc >> 32), r_hi = (uint32_t)(r_desc >> 32);
        for (int kb = k_first; kb < k_last; ++kb) {
            if (!__all_sync(0xffffffffu, mbar_wait(full(s), ph, abort_flag, status, ST_MMA))) { alive = false; break; }
            tc_fence_after();
            const uint32_t off = (uint32_t)((s * C::STAGE) >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint64_t ld = desc_from_words((uint32_t)l_desc + off + 2u * k, l_hi), rd = desc_from_words((uint32_t)r_desc + off + 2u * k, r_hi);
                if (elected) mma<C::KIND, 1>(tmem, ld, rd, C::IDESC, k ? 1u : (uint32_t)(kb != k_first));
            }
            if (elected) umma_commit(empty(s));
            __syncwarp();
            if (++s == S) { s = 0; ph ^= 1u; }
        }
        if (alive && elected) umma_commit(done);
        __syncwarp();
        if (!alive && elected) {
            umma_commit(drain);
            const uint64_t t0 = globaltimer_ns();
            while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < 10000000ull) { }
        }
        __syncwarp();
    } else {
        const int q = warp & 3;
        constexpr int EB = BN / 2;
        const int half0 = (warp - 2) / 4 * EB;
        if (__all_sync(0xffffffffu, mbar_wait(done, 0, abort_flag, status, ST_EPILOGUE))) {
            tc_fence_after();
            // the accumulator is complete, so every MMA has read its stages and the ring is free for the partial tile
            const uint32_t dst = base + (uint32_t)((q * 32 + lane) * L::PITCH + half0 * 4);
#pragma unroll
            for (int c = 0; c < EB / 32; ++c) {
                uint32_t v[32];
                tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half0 + c * 32), v);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; e += 4) st_shared_v4(dst + (c * 32 + e) * 4, v[e], v[e + 1], v[e + 2], v[e + 3]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                    // every CTA's partial tile is in place
    {
        const int rows = 128 / split;
        for (int w = threadIdx.x; w < rows * (BN / 8); w += THREADS) {
            const int r_in = w / (BN / 8), col = w % (BN / 8) * 8;
            const int lrow = rank * rows + r_in;
            if (m0 + lrow >= g.M || n0 + col >= g.N) continue;
            uint32_t sum[8];
            const uint32_t at = base + (uint32_t)(lrow * L::PITCH + col * 4);
            for (int k = 0; k < split; ++k) {
                uint32_t r0[4], r1[4];
                const uint32_t from = mapa_cluster(at, (uint32_t)k);
                ld_cluster_v4(from, r0);
                ld_cluster_v4(from + 16, r1);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sum[e] = k ? sum[e] + r0[e] : r0[e];
                    sum[4 + e] = k ? sum[4 + e] + r1[e] : r1[e];
                }
            }
            Epi::emit8(args, g, m0 + lrow, n0 + col, sum);
        }
    }
    __syncthreads();
    cluster_sync_all();                    // nobody leaves while its shared memory is still read
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::TMEM_COLS) : "memory");
    }
}

// how many CTAs share a tile: as many as keep two K blocks each and the SMs no more than full
inline int split_of(const Tiles& g, int sms = 148) {
    int split = 1;
    while (split < 8 && g.total * split * 2 <= sms && g.nkb >= 4 * split) split *= 2;
    return split;
}

template <class C, class Epi>
int launch_split(const CUtensorMap& map_l, const CUtensorMap& map_r, const Tiles& g, const typename Epi::Args& args, int split,
                 int32_t* status, cudaStream_t s, bool after) {
    static bool ready[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return CHEBYKAN_EINVAL;
    auto kernel = split_kernel<C, Epi>;
    if (!ready[dev]) {
        const int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SplitSmem<C>::TOTAL));
        if (rc) return rc;
        ready[dev] = true;
    }
    return check_cuda(launch_after(after, kernel, dim3((unsigned)(g.total * split)), dim3(THREADS), SplitSmem<C>::TOTAL, s, split, map_l, map_r, g,
                                   args, split, status));
}

// map of `slabs` row-major matrices [rows][cols], rows pitch_bytes and matrices slab_bytes apart, read in boxes of
// box_cols x box_rows (stores: written, clipped to the matrix); what lies outside a matrix reads as zero
inline int make_map(CUtensorMap* map, Kind kind, const void* base, int64_t cols, int64_t rows, int64_t slabs, int64_t pitch_bytes,
                    int64_t slab_bytes, int box_cols, int box_rows, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    EncodeTiledFn encode = get_encode_fn();
    if (!encode) return CHEBYKAN_ECUDA;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)slabs};
    const cuuint64_t strides[2] = {(cuuint64_t)pitch_bytes, (cuuint64_t)slab_bytes};
    const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
    const cuuint32_t one[3] = {1, 1, 1};
    const CUresult r = encode(map, kind == I8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                              const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_last_cuda_error((int)r); return CHEBYKAN_ECUDA; }
    return CHEBYKAN_OK;
}

template <class C>
Tiles tiles_of(int M, int N, int K, int batch, bool sym) {
    Tiles g;
    g.M = M; g.N = N;
    g.nkb = (int)ceil_div(K, C::KE);
    g.ntm = (int)ceil_div(M, C::BM);
    g.ntn = (int)ceil_div(N, C::BN);
    g.sym = sym;
    g.per_batch = sym ? sym_tiles(g.ntm, g.ntn, C::BM, C::BN) : g.ntm * g.ntn;
    g.whole = g.total = (int64_t)g.per_batch * batch;
    return g;
}

// persistent launch, one CTA (or pair) per SM (or two); after: see launch_after
template <class C, class Epi>
int launch(const CUtensorMap& map_l, const CUtensorMap& map_r, const Tiles& g, const typename Epi::Args& args, int32_t* status,
           cudaStream_t s, bool after) {
    static int max_units[64] = {0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return CHEBYKAN_EINVAL;
    auto kernel = gemm_kernel<C, Epi>;
    if (max_units[dev] == 0) {
        int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        if (rc) return rc;
        int sms = 148, n = 0;
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        n = sms / C::CG;
        if (C::CG == 2) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)(sms & ~1)); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = C::SMEM;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = C::CG; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr; cfg.numAttrs = 1;
            int clusters = 0;
            if ((rc = check_cuda(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg)))) return rc;
            if (clusters < 1) return CHEBYKAN_ECUDA;
            if (clusters < n) n = clusters;
        }
        max_units[dev] = n;
    }
    Tiles h = g;
    const int64_t left = g.total % max_units[dev];
    if (C::HALVES && left > 0 && 2 * left <= max_units[dev]) {
        h.whole = g.total - left;
        h.total = h.whole + 2 * left;
    }
    const int64_t units = h.total < max_units[dev] ? h.total : max_units[dev];
    return check_cuda(launch_after(after, kernel, dim3((unsigned)(units * C::CG)), dim3(THREADS), C::SMEM, s, C::CG, map_l, map_r, h, args, status));
}

}  // namespace gemm
}  // namespace chebykan
