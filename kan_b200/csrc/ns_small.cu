// Newton-Schulz orthogonalisation of small matrices (shorter side up to 128, longer up to 2048) in one launch.
//
// A matrix of this size is a few microseconds of reading and no arithmetic to speak of, but 3 * steps products that wait
// for one another: as launches of their own each costs a launch, a pipeline's start and its drain (about 9 us; 150 us for
// five steps on 33 matrices of 64 x 64).  Here a cluster of up to 8 CTAs keeps the matrix in shared memory throughout.  Every
// CTA holds a slice of up to 256 columns of X, rows padded to 128, as fp16 planes in 64-column panels of 128-byte swizzled
// rows, which serve as they lie as both operands of A = X X^T (K-major) and as the right operand of P X (MN-major).  A and P
// share one buffer: a row of P is formed from the same row of A by the thread that then overwrites it.
//   A  = X X^T   each CTA over its columns; with several CTAs the fp32 partial results of a row go to the CTA
//                that owns its band, which adds them in rank order and sends the finished row to all
//   P  = a I + b A + c A A    every CTA for itself
//   X' = P X     on the CTA's own columns
// With at most 64 rows (NARROW) the tail plane lies in the panels' second 64 rows.  Then M = 64, which halves what an MMA reads
// of its left operand (a product of this size is bound by that: some 80 cycles per MMA of M = 128, whatever N), and one MMA
// multiplies head x head and head x tail side by side, as N = 128.
// Products are tcgen05.mma (cta_group::1) issued by one elected lane; between two of them all sixteen warps turn the
// accumulator into the next operand.  Heads are summed over at most 128 columns of K in an
// accumulator: the tensor pipe's sums truncate (see gemm_tc.cuh).
// Measured: 33 matrices of 64 x 64 24 us, five of 784 x 64 47 us, one of 64 x 10 17 us.  A product takes about 2200 cycles: 650 to
// issue, 170 to finish, 230 for the barriers and the rest to form the next operand.
#include <math.h>
#include "newton_schulz.cuh"
#include "tc_common.cuh"

namespace chebykan {
namespace ns {
namespace {
using namespace tc;

constexpr int THREADS = 512, GROUPS = THREADS / 128;       // GROUPS warps per 32 lanes of tensor memory share the columns
constexpr int PANEL = 128 * 128;                 // 128 rows of 64 fp16 columns
constexpr int MAX_CLUSTER = 8, MAX_SLICE = 256;
enum { ST_GRAM = 31, ST_POLY = 32, ST_APPLY = 33 };

constexpr int MOST_SMEM = 224 * 1024;            // of operands and inbox; a little more for barriers and alignment

struct Geometry {
    int s, l;
    int cluster, slice;      // CTAs per matrix, columns per CTA (a multiple of 16)
    int s16, acc;            // rows rounded up to 16; columns of one accumulator
    int planes, tall;
    int band;                // rows of A that a CTA of a cluster sums
    int x_bytes, a_bytes;    // shared memory: X planes, and A / P with the inbox of partial sums
    int inbox;               // its offset in the latter: behind A, or on A where there is no room for both
};

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster_v4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}
// 16 bytes (8 columns from col) of a row of panels
__device__ __forceinline__ uint32_t chunk_at(int row, int col) {
    return (uint32_t)((col >> 6) * PANEL + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4));
}
template <typename T>
struct Io {
    const T* g;                   // element (b, r, c) at b*sb + r*sr + c*sc
    int64_t sb, sr, sc;
    T* out;                       // [batch][m][n]; may be g's own memory: a CTA has read its columns before it writes them
    int64_t m, n;
};
template <typename T, int PLANES, bool NARROW>
__global__ void __launch_bounds__(THREADS, 1) small_kernel(const Io<T> io, const Geometry g, const Steps st, int32_t* status) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    uint8_t* tail = gen + g.x_bytes + g.a_bytes;
    double* red = reinterpret_cast<double*>(tail);                               // a sum per warp, and the CTA's in [16]
    float* scales = reinterpret_cast<float*>(tail + 144);                         // alpha of X_0 and of the later X
    double* pow2 = reinterpret_cast<double*>(tail + 152);
    const uint32_t bar = base + (uint32_t)(g.x_bytes + g.a_bytes) + 160;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(tail + 168);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 172);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    const int64_t b = blockIdx.x / g.cluster;
    const int col0 = rank * g.slice;
    const int cols = g.l - col0 < g.slice ? g.l - col0 : g.slice;               // at least 1
    const uint32_t xs = base, as = base + (uint32_t)g.x_bytes;
    constexpr bool STACK = NARROW && PLANES == 2;
    const int x_plane = NARROW ? PANEL / 2 : g.x_bytes / PLANES, a_plane = NARROW ? PANEL / 2 : (g.s16 + 63) / 64 * PANEL;
    const uint32_t tmem_cols = PLANES == 2 ? 512u : (uint32_t)g.acc;

    if (threadIdx.x == 0) {
        mbar_init(bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void*)tmem_slot)), "r"(tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    let_next_start();
    wait_for_previous();

    // ---- norm, then X_0 ----
    // elements in the order of the matrix's own columns, so that reads are coalesced whichever side is the shorter
    const int count = g.s * cols;
    auto place = [&](int e, int& r, int& c) {
        if (g.tall) { c = e / g.s; r = e - c * g.s; } else { r = e / cols; c = e - r * cols; }
    };
    constexpr int U = 8;
    // this thread's next U elements from the e0-th on: their places in the slice and values, all loads in flight
    struct Batch { int r[U], c[U]; float v[U]; };
    auto fetch = [&](int e0, Batch& t) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (e0 + u * THREADS < count) {
                place(e0 + u * THREADS, t.r[u], t.c[u]);
                t.v[u] = (float)io.g[b * io.sb + (g.tall ? (col0 + t.c[u]) * io.sr + t.r[u] * io.sc : t.r[u] * io.sr + (col0 + t.c[u]) * io.sc)];
            }
    };
    double sum = 0.;
    Batch batch;                                        // the first, kept for X_0: it is all there is of a matrix of 4096 elements
    for (int e0 = threadIdx.x; e0 < count; e0 += U * THREADS) {
        Batch t;
        fetch(e0, t);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (e0 + u * THREADS < count) sum = fma((double)t.v[u], (double)t.v[u], sum);
        if (e0 == (int)threadIdx.x) batch = t;
    }
    for (uint32_t at = threadIdx.x * 16; at < (uint32_t)(g.x_bytes + g.a_bytes); at += THREADS * 16)
        *reinterpret_cast<uint4*>(gen + at) = make_uint4(0, 0, 0, 0);           // rows and columns of padding
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.;
        for (int w = 0; w < THREADS / 32; ++w) t += red[w];
        red[16] = t;
    }
    __syncthreads();
    if (g.cluster > 1) cluster_sync_all();
    if (threadIdx.x == 0) {
        double t = red[16];
        if (g.cluster > 1) {
            t = 0.;
            for (int k = 0; k < g.cluster; ++k) t += ld_cluster_f64(mapa_cluster(base + (uint32_t)(g.x_bytes + g.a_bytes) + 128, (uint32_t)k));
        }
        scales_of(sqrt(t), st.eps, st.growth, pow2, &scales[0], &scales[1]);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    {
        const double p2 = *pow2;
        for (int e0 = threadIdx.x; e0 < count; e0 += U * THREADS) {
            if (e0 != (int)threadIdx.x) fetch(e0, batch);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (e0 + u * THREADS < count) {
                    const float v = (float)((double)batch.v[u] * p2);
                    const __half hi = __float2half_rn(v);
                    uint8_t* at = gen + chunk_at(batch.r[u], batch.c[u]) + 2 * (batch.c[u] & 7);
                    *reinterpret_cast<__half*>(at) = hi;
                    if (PLANES == 2) *reinterpret_cast<__half*>(at + x_plane) = __float2half_rn(v - __half2float(hi));
                }
        }
    }

    // ---- one product: operands in shared memory, rows of 128; returns with the accumulator readable by every thread ----
    const bool elected = warp == 0 && elect_one_sync();
    uint32_t phase = 0;
    // left: K-major panels from `left`; right: the same, or X as [K][N].  ksteps of 16, n columns.  PLANES = 2: heads in one
    // accumulator or, to keep sums short (they truncate), the first and the second half of K in two; cross products in another
    uint32_t second = 0;                                // its column for the product at hand; 0: there is none
    constexpr uint32_t CROSS = STACK ? 64 : 256;        // from a head column to its cross product's
    auto product = [&](uint32_t left, int left_plane, uint32_t right, int right_plane, bool mn, int ksteps, int n, int code) {
        if (PLANES == 2) second = ksteps > 4 && (STACK || n <= 128) ? (STACK ? 256u : 128u) : 0u;
        fence_proxy_async_smem();
        tc_fence_before();
        __syncthreads();
        if (warp == 0) {
            tc_fence_after();
            // the whole warp runs the loop and one lane issues (see elect_one_sync); only the low words of descriptors move
            auto idesc_of = [&](int cols) {
                return (1u << 4) | ((mn ? 1u : 0u) << 16) | ((uint32_t)(cols >> 3) << 17) | ((NARROW ? 64u : 128u) >> 4 << 24);
            };
            const uint64_t ld = make_smem_desc(left), rd = make_smem_desc(right);
            const uint32_t l_hi = (uint32_t)(ld >> 32), l_lo = (uint32_t)ld, l_tail = (uint32_t)(left_plane >> 4);
            // MN-major: columns 64 apart are a panel apart; stacked, a panel's tails follow its heads half a panel on
            const uint32_t r_hi = (uint32_t)(rd >> 32), r_tail = (uint32_t)(right_plane >> 4);
            const uint32_t box = (uint32_t)((STACK ? PANEL / 2 : PANEL) >> 4) << 16;
            const uint32_t r_lo = mn ? ((uint32_t)rd & 0xffffu) | box : (uint32_t)rd;
            const int turn = second ? (ksteps + 1) / 2 : ksteps;
            const int panels = STACK && mn ? (n + 63) / 64 : 1;
            const uint32_t idesc = idesc_of(n), idesc64 = idesc_of(64), idesc128 = idesc_of(128), idesc256 = idesc_of(256);
#pragma unroll 4
            for (int k = 0; k < ksteps; ++k) {
                const uint32_t kmaj = (uint32_t)((k >> 2) * (PANEL >> 4) + (k & 3) * 2), kr = mn ? (uint32_t)(k * 128) : kmaj;
                const uint32_t go = (uint32_t)(k != 0 && k != turn), d = tmem + (k < turn ? 0u : second);
                // operands are formed by the whole warp, in uniform registers, and only the MMA itself is one lane's
                auto issue = [&](uint32_t dst, uint32_t l, uint32_t r, uint32_t id, uint32_t accumulate) {
                    const uint64_t ldesc = desc_from_words(l, l_hi), rdesc = desc_from_words(r, r_hi);
                    if (elected) umma<CHEBYKAN_MODE_BF16>(dst, ldesc, rdesc, id, accumulate);
                };
                const uint32_t l0 = l_lo + kmaj, r0 = r_lo + kr;
                if (STACK) {
                    // [heads | cross] in 64 columns each, panel by panel
                    for (int p = 0; p < panels; p += 2) {
                        const uint32_t at = r0 + (uint32_t)(p * (PANEL >> 4)), dp = d + (uint32_t)(p * 128);
                        issue(dp, l0, at, p + 1 < panels ? idesc256 : idesc128, go);
                        issue(dp + 64, l0 + l_tail, at, idesc64, 1u);
                        if (p + 1 < panels) issue(dp + 192, l0 + l_tail, at + (uint32_t)(PANEL >> 4), idesc64, 1u);
                    }
                } else {
                    issue(d, l0, r0, idesc, go);
                    if (PLANES == 2) {
                        issue(tmem + CROSS, l0, r0 + r_tail, idesc, k > 0);
                        issue(tmem + CROSS, l0 + l_tail, r0, idesc, 1u);
                    }
                }
            }
            if (elected) umma_commit(bar);
            __syncwarp();
        }
        mbar_wait(bar, phase, abort_flag, status, code);
        phase ^= 1u;
        __syncwarp();
        tc_fence_after();
    };
    const int q = warp & 3, group = warp >> 2;         // lanes of tensor memory, and which of the interleaved column groups
    // M = 64 fills 16 lanes of each quarter
    const int row = NARROW ? (lane < 16 ? q * 16 + lane : 1 << 20) : q * 32 + lane;
    // visits the accumulator's columns 16 at a time: f(first column, values)
    auto columns = [&](int n, auto f) {
        for (int c = group * 16; c < n; c += GROUPS * 16) {
            __syncwarp();                               // the loads are warp-collective
            uint32_t v[16], w[16];
            const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(STACK ? (c >> 6) * 128 + (c & 63) : c);
            tmem_ld16(at, v);
            if (PLANES == 2) tmem_ld16(at + CROSS, w);
            tmem_ld_wait();
            float x[16];
            auto plus = [&](const uint32_t (&y)[16]) {
#pragma unroll
                for (int e = 0; e < 16; e += 2)
                    halves(add2(pair_of(x[e], x[e + 1]), pair_of(__uint_as_float(y[e]), __uint_as_float(y[e + 1]))), x[e], x[e + 1]);
            };
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(v[e]);
            if (PLANES == 2) plus(w);
            if (PLANES == 2 && second) {
                tmem_ld16(at + second, v);
                if (STACK) tmem_ld16(at + second + CROSS, w);
                tmem_ld_wait();
                plus(v);
                if (STACK) plus(w);
            }
            f(c, x);
        }
    };
    auto put = [&](uint32_t dst, int plane, int r, int c, const float (&x)[8]) {       // 8 columns of a row, both planes
        uint32_t hi[4], lo[4];
        split8<PLANES>(x, hi, lo);
        const uint32_t at = dst + chunk_at(r, c);
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
        if (PLANES == 2)
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at + (uint32_t)plane), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]) : "memory");
    };

    auto times = [&](const float (&x)[16], int j, float by, float (&y)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) halves(mul2(pair_of(x[j + e], x[j + e + 1]), pair_of(by, by)), y[e], y[e + 1]);
    };
    // P's coefficients in the units of the stored numbers
    const float pa = st.a * exp2f((float)P_EXP), pb = st.b * exp2f((float)(P_EXP - A_EXP)), pc = st.c * exp2f((float)(P_EXP - 2 * A_EXP));

    const int cols16 = (cols + 15) & ~15;
    if (g.cluster > 1) { __syncwarp(); cluster_arrive(); }      // every wait below has its arrival a phase earlier
    for (int k = 0; k < st.n; ++k) {
        const float al = scales[k ? 1 : 0];
        // A = X X^T
        product(xs, x_plane, xs, x_plane, false, cols16 / 16, g.s16, ST_GRAM);
        const float fa = al * al * exp2f((float)A_EXP);
        if (g.cluster == 1) {
            columns(g.s16, [&](int c, const float (&x)[16]) {
                if (row >= g.s) return;
#pragma unroll
                for (int j = 0; j < 16; j += 8) {
                    float y[8];
                    times(x, j, fa, y);
                    put(as, a_plane, row, c + j, y);
                }
            });
        } else {
            // Each CTA sums a band of rows: the partial sums of a row go straight to the CTA that owns it, which adds them in
            // rank order and sends the finished row to every CTA.  Remote stores need no answer, so an exchange costs its two
            // barriers and little else; fetching from the others instead cost four times as much.
            const int pitch = (g.s16 + 4) * 4;          // 16-byte accesses of 8 rows meet no bank twice
            const uint32_t inbox = as + (uint32_t)g.inbox;
            cluster_wait();                             // everybody's P (which an inbox may lie on) has been used
            columns(g.s16, [&](int c, const float (&x)[16]) {
                if (row >= g.s) return;
                const int owner = row / g.band;
                const uint32_t to = mapa_cluster(inbox + (uint32_t)((rank * g.band + row - owner * g.band) * pitch + c * 4), (uint32_t)owner);
#pragma unroll
                for (int j = 0; j < 16; j += 4) st_cluster_v4(to + j * 4, __float_as_uint(x[j]), __float_as_uint(x[j + 1]), __float_as_uint(x[j + 2]), __float_as_uint(x[j + 3]));
            });
            tc_fence_before();
            __syncwarp();
            cluster_sync_all();
            // 8 columns per thread; a band of at most 64 rows x 16 groups is 2 per thread.  Rows from s to s16 become zero:
            // the next product reads them.
            constexpr int W = 1024 / THREADS;
            const int r0 = rank * g.band, groups = g.s16 / 8;
            const int nrow = g.s16 - r0 < g.band ? (g.s16 - r0 > 0 ? g.s16 - r0 : 0) : g.band, todo = nrow * groups;
            float y[W][8];
#pragma unroll
            for (int u = 0; u < W; ++u) {
                const int w = threadIdx.x + u * THREADS;
#pragma unroll
                for (int e = 0; e < 8; ++e) y[u][e] = 0.f;
                if (w < todo && r0 + w / groups < g.s)
                    for (int p = 0; p < g.cluster; ++p) {
                        const float* from = reinterpret_cast<const float*>(gen + g.x_bytes + g.inbox + (p * g.band + w / groups) * pitch + w % groups * 32);
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[u][e] += from[e];
                    }
#pragma unroll
                for (int e = 0; e < 8; ++e) y[u][e] *= fa;
            }
            if (g.inbox == 0) cluster_sync_all();       // every inbox is read: the buffer becomes A
#pragma unroll
            for (int u = 0; u < W; ++u) {
                const int w = threadIdx.x + u * THREADS;
                if (w < todo) {
                    uint32_t hi[4], lo[4];
                    split8<PLANES>(y[u], hi, lo);
                    const uint32_t at = as + chunk_at(r0 + w / groups, w % groups * 8);
                    for (int p = 0; p < g.cluster; ++p) {
                        const uint32_t to = mapa_cluster(at, (uint32_t)p);
                        st_cluster_v4(to, hi[0], hi[1], hi[2], hi[3]);
                        if (PLANES == 2) st_cluster_v4(to + (uint32_t)a_plane, lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            }
            asm volatile("fence.proxy.async;" ::: "memory");
            __syncwarp();
            cluster_sync_all();
        }
        // P = a I + b A + c A A
        product(as, a_plane, as, a_plane, false, g.s16 / 16, g.s16, ST_POLY);
        columns(g.s16, [&](int c, const float (&x)[16]) {
            if (row >= g.s) return;
#pragma unroll
            for (int j = 0; j < 16; j += 8) {
                const uint32_t at = as + chunk_at(row, c + j);
                uint32_t h[4], t[4];
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(at));
                if (PLANES == 2)
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(t[0]), "=r"(t[1]), "=r"(t[2]), "=r"(t[3]) : "r"(at + (uint32_t)a_plane));
                float a[8], y[8];
                join8<PLANES>(h, t, a);
                times(x, j, pc, y);
#pragma unroll
                for (int e = 0; e < 8; e += 2) halves(fma2(pair_of(a[e], a[e + 1]), pair_of(pb, pb), pair_of(y[e], y[e + 1])), y[e], y[e + 1]);
                if (row >= c + j && row < c + j + 8) {          // the diagonal passes through
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (c + j + e == row) y[e] += pa;
                }
                put(as, a_plane, row, c + j, y);
            }
        });
        // X' = P X
        product(as, a_plane, xs, x_plane, true, g.s16 / 16, cols16, ST_APPLY);
        if (g.cluster > 1) cluster_arrive();            // P has been used
        const bool last = k + 1 == st.n;
        const float fx = exp2f(-(float)P_EXP) * al / (last ? 1.f : scales[1]);
        columns(cols16, [&](int c, const float (&x)[16]) {
            if (row >= g.s) return;
            if (last) {
                // tall: lanes (rows) are neighbours in memory, else the 16 columns are
                T* to = io.out + b * io.m * io.n + (g.tall ? (int64_t)(col0 + c) * io.n + row : (int64_t)row * io.n + col0 + c);
                const int64_t pitch = g.tall ? io.n : 1;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (c + e < cols) to[e * pitch] = from_float<T>(x[e] * fx);
            } else {
#pragma unroll
                for (int j = 0; j < 16; j += 8) {
                    float y[8];
                    times(x, j, fx, y);
                    put(xs, x_plane, row, c + j, y);
                }
            }
        });
    }

    tc_fence_before();
    __syncthreads();
    if (g.cluster > 1) cluster_wait();                  // the last arrival's
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
    }
}

Geometry geometry(const Shape& sh, bool tall) {
    Geometry g;
    g.s = sh.s; g.l = sh.l; g.planes = sh.planes; g.tall = tall;
    // slices of 128 columns while that leaves SMs idle (a thread's share of the reading is what they divide), else as few
    // CTAs as hold the matrix
    g.cluster = (int)ceil_div(sh.l, MAX_SLICE / 2);
    if (g.cluster > MAX_CLUSTER || (int64_t)g.cluster * sh.batch > 148) g.cluster = (int)ceil_div(sh.l, MAX_SLICE);
    g.slice = (int)round_up(ceil_div(sh.l, g.cluster), 16);
    g.cluster = (int)ceil_div(sh.l, g.slice);                                    // rounding may leave the last one nothing
    g.s16 = (int)round_up(sh.s, 16);
    g.acc = 32;
    while (g.acc < g.s16 || g.acc < g.slice) g.acc *= 2;
    const int layers = g.s16 <= 64 ? 1 : sh.planes;            // panels per 64 columns (see NARROW)
    g.x_bytes = layers * (int)ceil_div(g.slice, 64) * PANEL;
    const int operand = layers * (int)ceil_div(g.s16, 64) * PANEL;
    g.a_bytes = operand;
    g.inbox = 0;
    g.band = (int)ceil_div(g.s16, g.cluster);
    if (g.cluster > 1) {
        const int box = (int)round_up((int64_t)g.cluster * g.band * (g.s16 + 4) * 4, 1024);
        if (g.x_bytes + operand + box <= MOST_SMEM) {
            g.inbox = operand;
            g.a_bytes = operand + box;
        } else if (box > operand) {
            g.a_bytes = box;
        }
    }
    return g;
}

template <typename T, int PLANES, bool NARROW>
int launch(const Io<T>& io, const Geometry& g, int64_t batch, const Steps& st, int32_t* status, cudaStream_t s, bool after) {
    constexpr int MOST = MOST_SMEM + 2048;
    static bool ready[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return CHEBYKAN_EINVAL;
    auto kernel = small_kernel<T, PLANES, NARROW>;
    if (!ready[dev]) {
        const int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST));
        if (rc) return rc;
        ready[dev] = true;
    }
    // A CTA that waits for tensor memory may not hold up a cluster whose other CTAs are waited for: kernels with clusters
    // take more than half of an SM's shared memory, so that no two of them share one.
    size_t smem = (size_t)(g.x_bytes + g.a_bytes + 256 + 1024);
    if (g.cluster > 1 && smem < 116 * 1024) smem = 116 * 1024;
    return check_cuda(launch_after(after, kernel, dim3((unsigned)(batch * g.cluster)), dim3(THREADS), smem, s, g.cluster, io, g, st, status));
}
template <typename T>
int launch_typed(const void* g, int64_t sb, int64_t sr, int64_t sc, void* out, int64_t m, int64_t n, const Shape& sh, const Steps& st,
                 int32_t* status, cudaStream_t s, bool after) {
    const Io<T> io{reinterpret_cast<const T*>(g), sb, sr, sc, reinterpret_cast<T*>(out), m, n};
    const Geometry geo = geometry(sh, m > n);
    if (geo.s16 <= 64)
        return sh.planes == 2 ? launch<T, 2, true>(io, geo, sh.batch, st, status, s, after) : launch<T, 1, true>(io, geo, sh.batch, st, status, s, after);
    return sh.planes == 2 ? launch<T, 2, false>(io, geo, sh.batch, st, status, s, after) : launch<T, 1, false>(io, geo, sh.batch, st, status, s, after);
}
}  // namespace

bool small_supported(const Shape& sh) { return sh.s <= 128 && sh.l <= MAX_CLUSTER * MAX_SLICE; }

int launch_small(const void* g, int dtype, int64_t sb, int64_t sr, int64_t sc, void* out, int64_t m, int64_t n, const Shape& sh,
                 const Steps& st, int32_t* status, cudaStream_t s, bool after) {
    if (dtype == CHEBYKAN_DTYPE_FP32) return launch_typed<float>(g, sb, sr, sc, out, m, n, sh, st, status, s, after);
    if (dtype == CHEBYKAN_DTYPE_BF16) return launch_typed<__nv_bfloat16>(g, sb, sr, sc, out, m, n, sh, st, status, s, after);
    return launch_typed<__half>(g, sb, sr, sc, out, m, n, sh, st, status, s, after);
}

}  // namespace ns
}  // namespace chebykan
