// Products on the tensor cores: D[i][j] = sum_k A[i][k] B[j][k], f32 sums, for
// bf16 or f16 operands in either order (k contiguous, or i / j contiguous).
//
// One persistent block per SM walks 128 x BN tiles of D. Warp 0 brings 64-deep
// stages of both operands by TMA into 128-byte-swizzled shared memory, warp 1
// issues tcgen05.mma into one of two accumulators in Tensor Memory, and eight
// more warps empty the other one through the epilogue, so that the tensor cores
// wait neither for memory nor for the epilogue. The lanes of an epilogue warp
// are neighbours in i: the caller makes i the contiguous side of D.
//
// PL > 1: each operand is PL 16-bit planes whose sum is the value, and D is the
// sum of the plane products that matter: two planes hi hi + (hi lo + lo hi);
// three planes the six products down to 2^-16 of the first. The small ones go
// to an accumulator of their own: the tensor cores cut each addition off at the
// accumulator's last bit, and the main sum should not pay for that two to five
// times more often.
#pragma once

#include "pz_nn.cuh"
#include "pz_tma.cuh"
#include "pz_tma.h"

#include <atomic>

namespace pz {

constexpr int GEMM_BM = 128, GEMM_BK = 64;
constexpr int GEMM_EPI_WARPS = 8;
constexpr int GEMM_THREADS = 32 * (2 + GEMM_EPI_WARPS);
constexpr int GEMM_SMS = 148;

template <int BN, int PL>
struct GemmShape {
    static constexpr int A_BYTES = GEMM_BM * GEMM_BK * 2, B_BYTES = BN * GEMM_BK * 2;
    static constexpr int STAGE = PL * (A_BYTES + B_BYTES);
    static constexpr int FIT = (200 * 1024) / STAGE;
    static constexpr int STAGES = FIT > 6 ? 6 : FIT;
    static constexpr int ACCS = PL > 1 ? 2 : 1;      // main, small terms
    static constexpr int COLS = 2 * ACCS * BN;       // two tiles in flight
    static constexpr int BYTES = STAGES * STAGE + 1024 + 256;
    static_assert(COLS <= 512 && STAGES >= 2);
};

// An operand: R rows (i or j) by K, z matrices zs apart.
struct GemmSide {
    CUtensorMap map[3];
    int mn;  // rows contiguous instead of k
};

struct GemmArgs {
    GemmSide a, b;
    int m, n;             // rows of A, rows of B
    int ti, tj;           // tiles of 128 and of BN
    int kblocks;          // of 64 in all
    int splits;           // ranges of k; a unit is (tile, split, batch)
    int per;              // k blocks of a split
    int units;
    int symmetric;        // D = D^T: tiles wholly above the diagonal blocks are left out
    uint32_t idesc;       // instruction descriptor (types, orders, shape)
};

__device__ __forceinline__ void tmem_alloc(uint32_t* slot, int cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, int cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// the barrier gets one arrival when every mma issued so far has finished
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void mma_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mma_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_load(uint32_t addr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory descriptor of a 128-byte-swizzled operand stage. k contiguous:
// rows of 128 bytes, groups of eight 1024 bytes apart. Rows contiguous: blocks
// of 64 rows (64 k lines of 128 bytes) 8192 bytes apart, eight k lines 1024.
__device__ __forceinline__ uint64_t gemm_desc(uint32_t addr, int mn) {
    const uint64_t lead = mn ? 8192 >> 4 : 1;
    return (uint64_t)((addr >> 4) & 0x3fff) | lead << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

struct GemmUnit {
    int i, j, k0, k1, split, z;
};
template <int BN>
__device__ __forceinline__ GemmUnit gemm_unit(const GemmArgs& g, int u) {
    GemmUnit q;
    constexpr int W = GEMM_BM / BN > 0 ? GEMM_BM / BN : 1;  // tiles across a diagonal block
    const int tiles = g.symmetric ? W * g.ti * (g.ti + 1) / 2 : g.ti * g.tj;
    const int t = u % tiles, r = u / tiles;
    if (g.symmetric) {  // row i has W (i + 1) tiles
        int i = (int)((sqrtf(8.0f * (t / W) + 1.0f) - 1.0f) * 0.5f);
        while (W * (i + 1) * (i + 2) / 2 <= t) i++;
        while (W * i * (i + 1) / 2 > t) i--;
        q.i = i;
        q.j = t - W * i * (i + 1) / 2;
    } else {
        // the side with fewer tiles first: the other operand's tile is then read by
        // neighbours at the same time, and comes from memory once
        const bool i_first = g.ti <= g.tj;
        q.i = i_first ? t % g.ti : t / g.tj;
        q.j = i_first ? t / g.ti : t % g.tj;
    }
    q.split = r % g.splits;
    q.z = r / g.splits;
    q.k0 = q.split * g.per;
    q.k1 = q.k0 + g.per < g.kblocks ? q.k0 + g.per : g.kblocks;
    return q;
}

// wait that also ends when another role of the block has given up
__device__ __forceinline__ bool gemm_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* gave_up) {
    for (int i = 0; i < WAIT_TRIES; i++) {
        if (mbar_try(bar, parity)) return true;
        if (*gave_up) return false;
    }
    *gave_up = 1;
    return false;
}

// Epi: void operator()(const GemmUnit&, long long i, int j0, int cols, const float* sum) const for 32 columns
// from j0 (cols of them inside D) of row i, called by whole warps (rows past m too).
template <int BN, int PL, class Epi>
__global__ void __launch_bounds__(GEMM_THREADS, 1) gemm_kernel(const __grid_constant__ GemmArgs g,
                                                               const __grid_constant__ Epi epi, unsigned int* fault) {
    using S = GemmShape<BN, PL>;
    extern __shared__ unsigned char raw[];
    // 128-byte swizzle repeats every 1024 bytes
    unsigned char* const sm = raw + (1024 - (smem_addr(raw) & 1023)) % 1024;
    uint64_t* const full = reinterpret_cast<uint64_t*>(sm + S::STAGES * S::STAGE);
    uint64_t* const empty = full + S::STAGES;
    uint64_t* const acc_full = empty + S::STAGES;
    uint64_t* const acc_empty = acc_full + 2;
    uint64_t* const done = acc_empty + 2;
    uint32_t* const slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile uint32_t* const gave_up = slot + 1;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        for (int k = 0; k < S::STAGES; k++) {
            mbar_init(&full[k], 1);
            mbar_init(&empty[k], 1);
        }
        for (int k = 0; k < 2; k++) {
            mbar_init(&acc_full[k], 1);
            mbar_init(&acc_empty[k], GEMM_EPI_WARPS);
        }
        mbar_init(done, 1);
        *gave_up = 0;
        mbar_init_fence();
        for (int k = 0; k < PL; k++) {
            tma_prefetch(&g.a.map[k]);
            tma_prefetch(&g.b.map[k]);
        }
    }
    if (warp == 1) tmem_alloc(slot, S::COLS);
    mma_fence_before();
    __syncthreads();
    mma_fence_after();
    const uint32_t tmem = *slot;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0, phase = 0, asked = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < g.units && ok; u += gridDim.x) {
                const GemmUnit q = gemm_unit<BN>(g, u);
                for (int k = q.k0; k < q.k1; k++) {
                    ok = gemm_wait(&empty[stage], phase ^ 1, gave_up);
                    if (!ok) break;
                    mbar_expect(&full[stage], S::STAGE);
                    unsigned char* const at = sm + stage * S::STAGE;
#pragma unroll
                    for (int p = 0; p < PL; p++) {
                        unsigned char* const pa = at + p * S::A_BYTES;
                        unsigned char* const pb = at + PL * S::A_BYTES + p * S::B_BYTES;
                        if (g.a.mn)
                            for (int h = 0; h < GEMM_BM / 64; h++)
                                tma_load(pa + h * 8192, &g.a.map[p], &full[stage], q.i * GEMM_BM + h * 64, k * GEMM_BK,
                                         q.z);
                        else
                            tma_load(pa, &g.a.map[p], &full[stage], k * GEMM_BK, q.i * GEMM_BM, q.z);
                        if (g.b.mn)
                            for (int h = 0; h < BN / 64; h++)
                                tma_load(pb + h * 8192, &g.b.map[p], &full[stage], q.j * BN + h * 64, k * GEMM_BK, q.z);
                        else
                            tma_load(pb, &g.b.map[p], &full[stage], k * GEMM_BK, q.j * BN, q.z);
                    }
                    asked++;
                    if (++stage == S::STAGES) stage = 0, phase ^= 1;
                }
            }
            if (!ok)  // not before the copies asked for have come
                for (int r = asked > S::STAGES ? asked - S::STAGES : 0; r < asked; r++)
                    mbar_wait(&full[r % S::STAGES], (r / S::STAGES) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0, phase = 0, acc = 0, aphase = 0;
            bool ok = true;
            const int ka = g.a.mn ? 2048 >> 4 : 32 >> 4, kb = g.b.mn ? 2048 >> 4 : 32 >> 4;  // 16 k further
            for (int u = blockIdx.x; u < g.units && ok; u += gridDim.x) {
                const GemmUnit q = gemm_unit<BN>(g, u);
                ok = gemm_wait(&acc_empty[acc], aphase ^ 1, gave_up);
                if (!ok) break;
                mma_fence_after();
                const uint32_t d = tmem + acc * S::ACCS * BN;
                for (int k = q.k0; k < q.k1; k++) {
                    ok = gemm_wait(&full[stage], phase, gave_up);
                    if (!ok) break;
                    mma_fence_after();
                    const uint32_t at = smem_addr(sm) + stage * S::STAGE;
#pragma unroll
                    for (int pa = 0; pa < PL; pa++)
#pragma unroll
                        for (int pb = 0; pb + pa < PL; pb++) {
                            const uint64_t da = gemm_desc(at + pa * S::A_BYTES, g.a.mn);
                            const uint64_t db = gemm_desc(at + PL * S::A_BYTES + pb * S::B_BYTES, g.b.mn);
                            const bool small = pa + pb > 0;
                            // the first product into an accumulator starts it: (0, 0), and (0, 1) of the small ones
                            const bool starts = k == q.k0 && (!small || (pa == 0 && pb == 1));
#pragma unroll
                            for (int s = 0; s < GEMM_BK / 16; s++)
                                mma_f16(d + (small ? BN : 0), da + s * ka, db + s * kb, g.idesc, !(starts && s == 0));
                        }
                    mma_commit(&empty[stage]);
                    if (++stage == S::STAGES) stage = 0, phase ^= 1;
                }
                if (ok) mma_commit(&acc_full[acc]);
                if (++acc == 2) acc = 0, aphase ^= 1;
            }
            if (!ok) {  // not before what was issued has finished
                mma_commit(done);
                mbar_wait(done, 0);
            }
        }
    } else {
        // lanes 32 (warp % 4) .. of the accumulator are this warp's to read
        const int quarter = warp % 4, half = (warp - 2) / 4;
        int acc = 0, aphase = 0;
        for (int u = blockIdx.x; u < g.units; u += gridDim.x) {
            const GemmUnit q = gemm_unit<BN>(g, u);
            if (!__all_sync(0xffffffffu, gemm_wait(&acc_full[acc], aphase, gave_up))) break;
            mma_fence_after();
            const uint32_t d = tmem + acc * S::ACCS * BN + ((uint32_t)quarter * 32 << 16);
            const long long i = (long long)q.i * GEMM_BM + quarter * 32 + lane;
            const bool any = q.k0 < q.k1;
            for (int c = half * 32; c < BN; c += 64) {
                const int j = q.j * BN + c, cols = g.n - j < 32 ? g.n - j : 32;
                if (cols <= 0) break;
                float v[32];
                tmem_load(d + c, v);
                if (PL > 1) {
                    float w[32];
                    tmem_load(d + BN + c, w);
                    tmem_load_wait();
#pragma unroll
                    for (int e = 0; e < 32; e++) v[e] += w[e];
                } else {
                    tmem_load_wait();
                }
                if (!any) {
#pragma unroll
                    for (int e = 0; e < 32; e++) v[e] = 0.0f;
                }
                epi(q, i, j, cols, v);
            }
            mma_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);
            if (++acc == 2) acc = 0, aphase ^= 1;
        }
    }
    __syncwarp();
    mma_fence_before();
    __syncthreads();
    mma_fence_after();
    if (warp == 1) tmem_free(tmem, S::COLS);
    if (threadIdx.x == 0 && *gave_up) atomicAdd(fault, 1u);
}

// ── host side ─────────────────────────────────────────────────────────────

// A matrix of 16-bit values that TMA can address: rows x k.
struct GemmMat {
    const void* p = nullptr;
    long long rs = 0, ks = 0, zs = 0;  // strides of a row, of k, of a batch
};

// Whether its rows are the contiguous side.
inline bool gemm_mn(const GemmMat& m, long long k) { return m.rs == 1 && (m.ks != 1 || k == 1); }

inline bool gemm_tma_ok(const GemmMat& m, long long rows, long long k, long long batch) {
    auto stride_ok = [](long long s) { return s > 0 && s % 8 == 0 && s < ((long long)1 << 39); };
    if ((uintptr_t)m.p % 16 || (batch > 1 && !stride_ok(m.zs))) return false;
    if (gemm_mn(m, k)) return k == 1 || stride_ok(m.ks);
    return m.ks == 1 && (rows == 1 || stride_ok(m.rs));
}

inline bool gemm_map(GemmSide* s, int plane, const GemmMat& m, long long rows, long long k, long long batch, int tile,
                     bool bf16) {
    s->mn = gemm_mn(m, k);
    const cuuint64_t zs = batch > 1 ? (cuuint64_t)m.zs * 2 : 16;
    const CUtensorMapDataType t = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const long long in = s->mn ? rows : k, out = s->mn ? k : rows, os = s->mn ? m.ks : m.rs;
    const cuuint64_t size[3] = {(cuuint64_t)in, (cuuint64_t)out, (cuuint64_t)batch};
    const cuuint64_t stride[2] = {out > 1 ? (cuuint64_t)os * 2 : 16, zs};
    const cuuint32_t box[3] = {64, (cuuint32_t)(s->mn ? GEMM_BK : tile), 1};
    return encode_tiled(&s->map[plane], t, 3, const_cast<void*>(m.p), size, stride, box, CU_TENSOR_MAP_SWIZZLE_128B) ==
           CUDA_SUCCESS;
}

// A kernel's shared memory, set once per device (two threads that both do so
// set the same).
struct GemmOnce {
    std::atomic<bool> ready[64];
    template <class F>
    cudaError_t smem(F* kernel, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess || (dev < 64 && ready[dev].load(std::memory_order_acquire))) return e;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess && dev < 64) ready[dev].store(true, std::memory_order_release);
        return e;
    }
};

// Splits of k that make `units` up to about two per SM, each of 8 blocks at least.
inline int gemm_splits(long long tiles, long long kblocks) {
    if (tiles >= GEMM_SMS / 2) return 1;
    long long n = 2 * GEMM_SMS / tiles;
    if (n > kblocks / 8) n = kblocks / 8;
    if (n < 2) return 1;
    const long long per = (kblocks + n - 1) / n;
    return (int)((kblocks + per - 1) / per);
}

// D = A B^T (rows ma of A, nb of B). a, b: PL planes each. splits > 1: the
// epilogue gets each split's part.
template <int BN, int PL, class Epi>
cudaError_t gemm_launch(const GemmMat* a, const GemmMat* b, long long ma, long long nb, long long k, int batch,
                        int splits, bool symmetric, bool bf16, const Epi& epi, unsigned int* fault, cudaStream_t st) {
    using S = GemmShape<BN, PL>;
    GemmArgs g{};
    for (int p = 0; p < PL; p++) {
        if (!gemm_map(&g.a, p, a[p], ma, k, batch, GEMM_BM, bf16)) return cudaErrorInvalidValue;
        if (!gemm_map(&g.b, p, b[p], nb, k, batch, BN, bf16)) return cudaErrorInvalidValue;
    }
    g.m = (int)ma;
    g.n = (int)nb;
    g.ti = (int)((ma + GEMM_BM - 1) / GEMM_BM);
    g.tj = (int)((nb + BN - 1) / BN);
    g.kblocks = (int)((k + GEMM_BK - 1) / GEMM_BK);
    g.splits = splits;
    g.per = (g.kblocks + splits - 1) / splits;
    g.symmetric = symmetric;
    const long long tiles =
        symmetric ? (long long)(GEMM_BM / BN) * g.ti * (g.ti + 1) / 2 : (long long)g.ti * g.tj;
    if (tiles * splits * batch >= 1 << 30) return cudaErrorInvalidValue;
    g.units = (int)(tiles * splits * batch);
    g.idesc = 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (uint32_t)g.a.mn << 15 |
              (uint32_t)g.b.mn << 16 | (uint32_t)(BN >> 3) << 17 | (uint32_t)(GEMM_BM >> 4) << 24;
    auto kernel = gemm_kernel<BN, PL, Epi>;
    static GemmOnce once;
    const cudaError_t e = once.smem(kernel, S::BYTES);
    if (e != cudaSuccess) return e;
    kernel<<<g.units < GEMM_SMS ? g.units : GEMM_SMS, GEMM_THREADS, S::BYTES, st>>>(g, epi, fault);
    return cudaGetLastError();
}

}  // namespace pz
