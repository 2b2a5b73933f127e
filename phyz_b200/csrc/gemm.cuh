// Products on the tensor cores: D[i][j] = sum_k A[i][k] B[j][k], f32 sums, for
// bf16 or f16 operands in either order (k contiguous, or i / j contiguous).
//
// One persistent block per SM walks tiles of D. Warp 0 brings 64-deep stages of
// both operands by TMA into 128-byte-swizzled shared memory, warp 1 issues
// tcgen05.mma into one of two accumulators in Tensor Memory, and eight or sixteen
// more warps empty the other one through the epilogue, so that the tensor cores
// wait neither for memory nor for the epilogue. In the epilogue a lane has 32
// neighbours in j and a warp 32 in i: a chunk. Where TMA can address them, what
// the epilogue reads comes into the warp's own slots of shared memory a chunk
// ahead, and what it writes leaves from there.
//
// CTAS = 2: the two blocks of a cluster (the SMs of a pair) make one tile of 256 x
// BN: each brings its 128 rows of A and half of B's, one mma reads both shared
// memories, and each gets its rows' sums. A tile of 128 x 256 alone takes 96 bytes
// a clock from L2 for every SM, more than it gives (13.8 TB/s were measured, about
// 50); the pair's takes 64. Measured without an epilogue, 262144 x 1024 x 1024
// bf16: pairs of 256 columns 390 us (1.41 PFLOP/s), of 128 637, lone blocks of 128
// 620.
//
// PL > 1: each operand is PL 16-bit planes whose sum is the value, and D is the
// sum of the plane products that matter: two planes hi hi + (hi lo + lo hi);
// three planes the six products down to 2^-16 of the first. The small ones go
// to an accumulator of their own: the tensor cores cut each addition off at the
// accumulator's last bit, and the main sum should not pay for that two to five
// times more often. With Epi::FLUSH the accumulators are emptied every so many k
// blocks into f32 registers of the epilogue's warps, whose additions round: the
// cut ends, all towards zero, then stay few.
#pragma once

#include "pz_nn.cuh"
#include "pz_tma.cuh"
#include "pz_tma.h"

namespace pz {

constexpr int GEMM_BM = 128, GEMM_BK = 64;
constexpr int GEMM_SMS = 148;

// A chunk's slot: 32 rows of 32 16-bit values, one or two planes.
constexpr int GEMM_PLANE = 32 * 64;

template <int BN, int PL, int CTAS, class Epi>
struct GemmShape {
    static constexpr int ROWS = GEMM_BM * CTAS;      // of a tile
    static constexpr int BR = BN / CTAS;             // rows of B that a block brings
    static constexpr int A_BYTES = GEMM_BM * GEMM_BK * 2, B_BYTES = BR * GEMM_BK * 2;
    static constexpr int STAGE = PL * (A_BYTES + B_BYTES);
    static constexpr int WARP_SLOTS = Epi::PLANES * Epi::SLOTS * GEMM_PLANE;
    static constexpr int THREADS = 32 * (2 + Epi::WARPS);
    static constexpr int SLOTS = Epi::WARPS * WARP_SLOTS;
    static constexpr int FIT = (224 * 1024 - SLOTS) / STAGE;
    static constexpr int STAGES = FIT > 6 ? 6 : FIT;
    static constexpr int ACCS = PL > 1 ? 2 : 1;      // main, small terms
    static constexpr int FLUSH = PL > 1 ? Epi::FLUSH : 0;
    static constexpr int EVERY = Epi::WARPS * 8;  // columns from one of a warp's chunks to the next
    static constexpr int CHUNKS = (BN + EVERY - 1) / EVERY;   // of a warp in a tile, at most
    static constexpr int BUFS = 2 * ACCS * BN <= 512 ? 2 : 1;  // tiles in Tensor Memory
    static constexpr int COLS = BUFS * ACCS * BN;
    static constexpr int BYTES = STAGES * STAGE + SLOTS + 1024 + 512;
    static_assert(BYTES <= 227 * 1024);
    static_assert(COLS <= 512 && STAGES >= 2 && BR >= 64 && (!FLUSH || BN <= 128));
};

// An operand: R rows (i or j) by K, z matrices zs apart.
struct GemmSide {
    CUtensorMap map[3];
    int mn;  // rows contiguous instead of k
};

// What the epilogue reads and writes through slots: planes of arrays [batch][i][j]
// (j contiguous) as tensor maps, in boxes of 32 x 32.
struct GemmIo {
    CUtensorMap in[2], out[2];
    int reads, writes;  // whether through slots
};

struct GemmArgs {
    GemmSide a, b;
    GemmIo io;
    int m, n;             // rows of A, rows of B
    int ti, tj;           // tiles of ROWS and of BN
    int kblocks;          // of 64 in all
    int splits;           // ranges of k; a unit is (tile, split, batch)
    int per;              // k blocks of a split, one at least
    int units;
    int symmetric;        // D = D^T: tiles wholly above the diagonal blocks are left out
    uint32_t idesc;       // instruction descriptor (types, orders, shape)
};

template <int CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, int cols) {
    if constexpr (CTAS == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t addr, int cols) {
    if constexpr (CTAS == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
template <int CTAS>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    if constexpr (CTAS == 2)
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
            : "memory");
}
// the barrier (with two blocks, each one's) gets one arrival when every mma
// issued so far has finished
template <int CTAS>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    if constexpr (CTAS == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_addr(bar)),
            "h"((uint16_t)3)
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                     : "memory");
}
// The same place in the first block's shared memory.
__device__ __forceinline__ uint32_t lead_addr(const void* p) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(p)));
    return a;
}
// Relaxed: what it reports is Tensor Memory that has been read (and waited for);
// a release would wait for the epilogue's stores to global memory.
__device__ __forceinline__ void mbar_arrive_at(uint32_t addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// A box into this block's shared memory; its bytes complete on the first block's
// barrier (address in the cluster).
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
template <int CTAS>
__device__ __forceinline__ void block_sync() {  // of the tile's blocks
    if constexpr (CTAS == 2) {
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
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
// of 64 rows (k lines of 128 bytes) `block` bytes apart, eight k lines 1024.
__device__ __forceinline__ uint64_t gemm_desc(uint32_t addr, int mn, int block = 8192) {
    const uint64_t lead = mn ? block >> 4 : 1;
    return (uint64_t)((addr >> 4) & 0x3fff) | lead << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

struct GemmUnit {
    int row0, j, k0, k1, split, z;  // row0: the tile's first row
    int i;
};
template <int BN, int ROWS>
__device__ __forceinline__ GemmUnit gemm_unit(const GemmArgs& g, int u) {
    GemmUnit q;
    constexpr int W = ROWS / BN;  // tiles across a diagonal block
    const int tiles = g.symmetric ? W * g.ti * (g.ti + 1) / 2 : g.ti * g.tj;
    const int r = u < tiles ? 0 : u / tiles, t = u - r * tiles;
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
        const int fast = i_first ? g.ti : g.tj, slow = t / fast;
        q.i = i_first ? t - slow * fast : slow;
        q.j = i_first ? slow : t - slow * fast;
    }
    q.row0 = q.i * ROWS;
    q.z = r < g.splits ? 0 : r / g.splits;
    q.split = r - q.z * g.splits;
    q.k0 = q.split * g.per;
    q.k1 = q.k0 + g.per < g.kblocks ? q.k0 + g.per : g.kblocks;
    return q;
}

// wait that also ends when another role of the block has given up
__device__ __forceinline__ bool gemm_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* gave_up) {
    if (mbar_try(bar, parity)) return true;
    const long long begin = clock64();
    while (!mbar_try(bar, parity)) {
        if (*gave_up) return false;
        if (clock64() - begin > WAIT_CLOCKS) {
            *gave_up = 1;
            return false;
        }
    }
    return true;
}

// Where 16 bytes (8 values, the c-th) of a row of a slot's plane are (64-byte
// swizzle).
__device__ __forceinline__ int slot_at(int row, int c) { return row * 64 + ((c ^ (row >> 1 & 3)) << 4); }
// A lane's 32 values.
__device__ __forceinline__ void slot_load(const unsigned char* plane, uint32_t* w) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint4 q = *reinterpret_cast<const uint4*>(plane + slot_at(threadIdx.x % 32, c));
        w[4 * c] = q.x, w[4 * c + 1] = q.y, w[4 * c + 2] = q.z, w[4 * c + 3] = q.w;
    }
}
__device__ __forceinline__ void slot_store(unsigned char* plane, const uint32_t* w) {
#pragma unroll
    for (int c = 0; c < 4; c++)
        *reinterpret_cast<uint4*>(plane + slot_at(threadIdx.x % 32, c)) =
            make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
}

// Epi: void operator()(const GemmUnit&, long long i, int j0, int cols, float* sum,
// const unsigned char* in, unsigned char* out) const for 32 columns from j0 (cols
// of them inside D) of row i, called by whole warps (rows past m too). in, out:
// the chunk's slot where GemmIo says so (the same one), else null. PLANES of a
// slot, SLOTS of a warp, 8 or 16 WARPS. MIRROR: where mirrored(unit, j0) says so,
// the chunk's mirror image is written as well, by turn(sum, slot). FLUSH: k blocks
// to a sum of the tensor cores, where a product has planes (0: all).
template <int BN, int PL, int CTAS, class Epi>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__((GemmShape<BN, PL, CTAS, Epi>::THREADS), 1)
    gemm_kernel(const __grid_constant__ GemmArgs g, const __grid_constant__ Epi epi, unsigned int* fault) {
    using S = GemmShape<BN, PL, CTAS, Epi>;
    extern __shared__ unsigned char raw[];
    // 128-byte swizzle repeats every 1024 bytes
    unsigned char* const sm = raw + (1024 - (smem_addr(raw) & 1023)) % 1024;
    unsigned char* const slots = sm + S::STAGES * S::STAGE;
    uint64_t* const full = reinterpret_cast<uint64_t*>(slots + S::SLOTS);
    uint64_t* const empty = full + S::STAGES;
    uint64_t* const acc_full = empty + S::STAGES;
    uint64_t* const acc_empty = acc_full + 2;
    uint64_t* const done = acc_empty + 2;
    uint64_t* const slot_full = done + 1;
    uint32_t* const slot = reinterpret_cast<uint32_t*>(slot_full + Epi::WARPS * Epi::SLOTS);
    volatile uint32_t* const gave_up = slot + 1;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = CTAS == 2 ? blockIdx.x % 2 : 0;  // in the cluster; the first one leads
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int k = 0; k < S::STAGES; k++) {
            mbar_init(&full[k], 1);
            mbar_init(&empty[k], 1);
        }
        for (int k = 0; k < 2; k++) {
            mbar_init(&acc_full[k], 1);
            mbar_init(&acc_empty[k], CTAS * Epi::WARPS);
        }
        mbar_init(done, 1);
        for (int k = 0; k < Epi::WARPS * Epi::SLOTS; k++) mbar_init(&slot_full[k], 1);
        *gave_up = 0;
        mbar_init_fence();
        for (int k = 0; k < PL; k++) {
            tma_prefetch(&g.a.map[k]);
            tma_prefetch(&g.b.map[k]);
        }
    }
    __syncthreads();
    if (warp == 1) tmem_alloc<CTAS>(slot, S::COLS);
    mma_fence_before();
    block_sync<CTAS>();
    mma_fence_after();
    const uint32_t tmem = *slot;
    // launched ahead of the end of the kernel before it (gemm_launch_as): what that
    // one wrote is there from here on
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0, phase = 0, asked = 0;
            bool ok = true;
            for (int u = first; u < g.units && ok; u += step) {
                const GemmUnit q = gemm_unit<BN, S::ROWS>(g, u);
                const int ra = q.row0 + rank * GEMM_BM, rb = q.j * BN + rank * S::BR;
                for (int k = q.k0; k < q.k1; k++) {
                    ok = gemm_wait(&empty[stage], phase ^ 1, gave_up);
                    if (!ok) break;
                    const uint32_t bar = CTAS == 2 ? lead_addr(&full[stage]) : 0;
                    // (the other block's boxes of this round may complete before this: it asks for
                    // them when the stage is empty, so the last round is over)
                    if (rank == 0) mbar_expect(&full[stage], CTAS * S::STAGE);
                    auto load = [&](unsigned char* at, const CUtensorMap* map, int x, int y) {
                        if constexpr (CTAS == 2)
                            tma_load_pair(at, map, bar, x, y, q.z);
                        else
                            tma_load(at, map, &full[stage], x, y, q.z);
                    };
                    unsigned char* const at = sm + stage * S::STAGE;
#pragma unroll
                    for (int p = 0; p < PL; p++) {
                        unsigned char* const pa = at + p * S::A_BYTES;
                        unsigned char* const pb = at + PL * S::A_BYTES + p * S::B_BYTES;
                        if (g.a.mn)
                            for (int h = 0; h < GEMM_BM / 64; h++)
                                load(pa + h * 8192, &g.a.map[p], ra + h * 64, k * GEMM_BK);
                        else
                            load(pa, &g.a.map[p], k * GEMM_BK, ra);
                        if (g.b.mn)
                            for (int h = 0; h < S::BR / 64; h++)
                                load(pb + h * 8192, &g.b.map[p], rb + h * 64, k * GEMM_BK);
                        else
                            load(pb, &g.b.map[p], k * GEMM_BK, rb);
                    }
                    asked++;
                    if (++stage == S::STAGES) stage = 0, phase ^= 1;
                }
            }
            if (!ok && rank == 0)  // not before the copies asked for have come
                for (int r = asked > S::STAGES ? asked - S::STAGES : 0; r < asked; r++)
                    mbar_wait(&full[r % S::STAGES], (r / S::STAGES) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int stage = 0, phase = 0, acc = 0, aphase = 0;
            bool ok = true;
            const int ka = g.a.mn ? 2048 >> 4 : 32 >> 4, kb = g.b.mn ? 2048 >> 4 : 32 >> 4;  // 16 k further
            for (int u = first; u < g.units && ok; u += step) {
                const GemmUnit q = gemm_unit<BN, S::ROWS>(g, u);
                uint32_t d = 0;
                int begin = q.k0;  // of what the accumulator holds
                auto next = [&]() {
                    ok = gemm_wait(&acc_empty[acc], aphase ^ 1, gave_up);
                    mma_fence_after();
                    d = tmem + acc * S::ACCS * BN;
                };
                auto hand_over = [&]() {
                    mma_commit<CTAS>(&acc_full[acc]);
                    if (++acc == S::BUFS) acc = 0, aphase ^= 1;
                };
                next();
                if (!ok) break;
                for (int k = q.k0; k < q.k1; k++) {
                    if (S::FLUSH && k - begin == S::FLUSH) {
                        hand_over();
                        begin = k;
                        next();
                        if (!ok) break;
                    }
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
                            const bool starts = k == begin && (!small || (pa == 0 && pb == 1));
#pragma unroll
                            for (int s = 0; s < GEMM_BK / 16; s++)
                                mma_f16<CTAS>(d + (small ? BN : 0), da + s * ka, db + s * kb, g.idesc, !(starts && s == 0));
                        }
                    mma_commit<CTAS>(&empty[stage]);
                    if (++stage == S::STAGES) stage = 0, phase ^= 1;
                }
                if (ok) hand_over();
            }
            if (!ok) {  // not before what was issued has finished
                mma_commit<CTAS>(done);
                mbar_wait(done, 0);
            }
        }
    } else {
        // lanes 32 (warp % 4) .. of the accumulator are this warp's to read
        const int quarter = warp % 4, from = (warp - 2) / 4 * 32, own = rank * GEMM_BM + quarter * 32;
        constexpr int EVERY = S::EVERY;
        constexpr int NS = Epi::SLOTS, MOD = NS > 0 ? NS : 1;
        unsigned char* const mine = slots + (warp - 2) * S::WARP_SLOTS;
        uint64_t* const bars = slot_full + (warp - 2) * NS;
        // lane 0's place in the sequence of chunks, ahead of the warp's
        int au = first, ac = from, asked = 0;
        GemmUnit aq{};
        if (au < g.units) aq = gemm_unit<BN, S::ROWS>(g, au);
        auto request = [&]() {
            while (au < g.units) {
                const bool there = ac < BN && aq.row0 + own < g.m && aq.j * BN + ac < g.n;
                if (there) {
                    unsigned char* const at = mine + asked % MOD * Epi::PLANES * GEMM_PLANE;
                    mbar_expect(&bars[asked % MOD], Epi::PLANES * GEMM_PLANE);
#pragma unroll
                    for (int p = 0; p < Epi::PLANES; p++)
                        tma_load(at + p * GEMM_PLANE, &g.io.in[p], &bars[asked % MOD], aq.j * BN + ac, aq.row0 + own, aq.z);
                    asked++;
                    ac += EVERY;
                    return;
                }
                ac = from;
                au += step;
                if (au < g.units) aq = gemm_unit<BN, S::ROWS>(g, au);
            }
        };
        const bool reads = Epi::PLANES && g.io.reads, writes = Epi::PLANES && g.io.writes;
        // (a chunk's slot is asked for again two chunks after its results left, one where there are two slots)
        if (reads && lane == 0)
            for (int k = 0; k < (NS > 2 ? NS - 2 : 1); k++) request();
        int acc = 0, aphase = 0, n = 0;
        bool ok = true;
        for (int u = first; u < g.units && ok; u += step) {
            const GemmUnit q = gemm_unit<BN, S::ROWS>(g, u);
            uint32_t d = 0;
            auto take = [&]() {
                ok = __all_sync(0xffffffffu, gemm_wait(&acc_full[acc], aphase, gave_up));
                mma_fence_after();
                d = tmem + acc * S::ACCS * BN + ((uint32_t)quarter * 32 << 16);
            };
            auto give_back = [&]() {
                mma_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CTAS == 2)
                        mbar_arrive_at(lead_addr(&acc_empty[acc]));
                    else
                        mbar_arrive(&acc_empty[acc]);
                }
                if (++acc == S::BUFS) acc = 0, aphase ^= 1;
            };
            // 32 columns from c of the accumulator, small terms and all
            auto sum_of = [&](int c, float* v) {
                tmem_load(d + c, v);
                if constexpr (PL > 1) {
                    float w[32];
                    tmem_load(d + BN + c, w);
                    tmem_load_wait();
#pragma unroll
                    for (int e = 0; e < 32; e++) v[e] += w[e];
                } else {
                    tmem_load_wait();
                }
            };
            const long long i = q.row0 + own + lane;
            float held[S::FLUSH ? S::CHUNKS : 1][32];  // FLUSH: the sums so far
            if constexpr (S::FLUSH > 0) {
#pragma unroll
                for (int m = 0; m < S::CHUNKS; m++)
#pragma unroll
                    for (int e = 0; e < 32; e++) held[m][e] = 0.0f;
                for (int k = q.k0; k < q.k1 && ok; k += S::FLUSH) {
                    take();
                    if (!ok) break;
#pragma unroll
                    for (int m = 0; m < S::CHUNKS; m++) {
                        if (from + m * EVERY >= BN) break;
                        float v[32];
                        sum_of(from + m * EVERY, v);
#pragma unroll
                        for (int e = 0; e < 32; e++) held[m][e] += v[e];
                    }
                    give_back();
                }
            } else {
                take();
            }
            if (!ok) break;
#pragma unroll
            for (int m = 0; m < S::CHUNKS; m++) {
                const int c = from + m * EVERY, j = q.j * BN + c;
                if (c >= BN || j >= g.n || q.row0 + own >= g.m) break;
                unsigned char* const at = mine + n % MOD * Epi::PLANES * GEMM_PLANE;
                if constexpr (NS > 0) {
                    if (writes || reads) {
                        // the slot of a chunk ahead, or this one's, is empty again
                        if (lane == 0) {
                            if (reads && NS > 1) {
                                tma_store_wait_read<(NS > 2 ? 1 : 0)>();
                                request();
                            } else {
                                tma_store_wait_read<NS - 1>();
                            }
                        }
                        __syncwarp();
                    }
                    if (reads) {
                        ok = __all_sync(0xffffffffu, gemm_wait(&bars[n % MOD], (n / MOD) & 1, gave_up));
                        if (!ok) break;
                    }
                }
                const int cols = g.n - j < 32 ? g.n - j : 32;
                float v[32];
                if constexpr (S::FLUSH > 0) {
#pragma unroll
                    for (int e = 0; e < 32; e++) v[e] = held[m][e];
                } else {
                    sum_of(c, v);
                }
                epi(q, i, j, cols, v, reads ? at : nullptr, writes ? at : nullptr);
                if constexpr (NS > 0) {
                    if (writes) {
                        fence_async();
                        __syncwarp();
                        if (lane == 0) {  // (past m and n nothing is written)
#pragma unroll
                            for (int p = 0; p < Epi::PLANES; p++)
                                tma_store(&g.io.out[p], at + p * GEMM_PLANE, j, q.row0 + own, q.z);
                            tma_store_commit();
                        }
                        if constexpr (Epi::MIRROR) {
                            if (epi.mirrored(q, j)) {
                                if (lane == 0) tma_store_wait_read<0>();
                                __syncwarp();
                                epi.turn(v, at);
                                fence_async();
                                __syncwarp();
                                if (lane == 0) {
#pragma unroll
                                    for (int p = 0; p < Epi::PLANES; p++)
                                        tma_store(&g.io.out[p], at + p * GEMM_PLANE, q.row0 + own, j, q.z);
                                    tma_store_commit();
                                }
                            }
                        }
                    } else {
                        __syncwarp();
                    }
                    if (NS == 1 && reads && lane == 0) {
                        tma_store_wait_read<0>();
                        request();
                    }
                }
                n++;
            }
            if (!S::FLUSH) give_back();
        }
        if constexpr (NS > 0) {
            if (lane == 0) {
                if (!ok)  // not before the boxes asked for have come
                    for (int r = asked > NS ? asked - NS : 0; r < asked; r++) mbar_wait(&bars[r % NS], (r / NS) & 1);
                tma_store_wait_read<0>();
            }
        }
    }
    __syncwarp();
    mma_fence_before();
    block_sync<CTAS>();
    mma_fence_after();
    if (warp == 1) tmem_free<CTAS>(tmem, S::COLS);
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

// The tensor map of a plane that an epilogue reads or writes: [batch][rows][cols],
// cols contiguous. False where TMA cannot address it.
inline bool gemm_io_map(CUtensorMap* m, const void* p, long long rs, long long cs, long long zs, long long rows,
                        long long cols, long long batch, bool bf16) {
    if (cs != 1 || !gemm_tma_ok({p, rs, 1, zs}, rows, cols, batch)) return false;
    const cuuint64_t size[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
    const cuuint64_t stride[2] = {rows > 1 ? (cuuint64_t)rs * 2 : 16, batch > 1 ? (cuuint64_t)zs * 2 : 16};
    const cuuint32_t box[3] = {32, 32, 1};
    return encode_tiled(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<void*>(p), size, stride, box, CU_TENSOR_MAP_SWIZZLE_64B) == CUDA_SUCCESS;
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

// How a product is cut.
struct GemmCut {
    int ctas, bn, splits;
};

// The shape that takes least by a rough count of clocks: rounds of tiles over the
// SMs (pairs for two blocks), each its k blocks' mma time (a lone block's are held
// up by L2) and 1500 to fill and empty. `planes`: products per product. splits: k
// is cut too where that fills SMs that the tiles leave empty (parts of 8 k blocks
// at least; joining them costs about 3000 more).
inline GemmCut gemm_cut(long long rows, long long cols, long long k, long long batch, int products, bool symmetric,
                        bool may_split, bool flush) {
    const struct {
        int ctas, bn;
        double clocks;  // of a k block
    } shapes[] = {{2, 256, 540}, {2, 128, 300}, {1, 128, 340}, {1, 64, 230}};
    const long long kb = (k + GEMM_BK - 1) / GEMM_BK;
    GemmCut best{};
    double least = 0;
    for (const auto& s : shapes) {
        if (flush && s.bn == 256) continue;  // (its sums do not fit the epilogue's registers)
        const long long r = GEMM_BM * s.ctas, ti = (rows + r - 1) / r, tj = (cols + s.bn - 1) / s.bn;
        const long long tiles = (symmetric ? r / s.bn * ti * (ti + 1) / 2 : ti * tj) * batch;
        const long long slots = GEMM_SMS / s.ctas;
        long long most = may_split && tiles < slots ? kb / 8 : 1;
        if (most > 64) most = 64;
        for (long long n = 1; n == 1 || n <= most; n++) {
            const long long per = (kb + n - 1) / n;
            if (n > 1 && (kb + per - 1) / per != n) continue;
            const double c = (double)((tiles * n + slots - 1) / slots) * (per * s.clocks * products + 1500) +
                             (n > 1 ? 3000 + n * 100.0 : 0);
            if (!best.ctas || c < least) {
                best = {s.ctas, s.bn, (int)n};
                least = c;
            }
            if (tiles * n > 2 * slots) break;
        }
    }
    return best;
}

// D = A B^T (rows ma of A, nb of B). a, b: PL planes each. splits > 1: the
// epilogue gets each split's part.
template <int BN, int PL, int CTAS, class Epi>
cudaError_t gemm_launch_as(const GemmMat* a, const GemmMat* b, long long ma, long long nb, long long k, int batch,
                           int splits, bool symmetric, bool bf16, const GemmIo& io, const Epi& epi, unsigned int* fault,
                           cudaStream_t st) {
    using S = GemmShape<BN, PL, CTAS, Epi>;
    GemmArgs g{};
    g.io = io;
    for (int p = 0; p < PL; p++) {
        if (!gemm_map(&g.a, p, a[p], ma, k, batch, GEMM_BM, bf16)) return cudaErrorInvalidValue;
        if (!gemm_map(&g.b, p, b[p], nb, k, batch, S::BR, bf16)) return cudaErrorInvalidValue;
    }
    g.m = (int)ma;
    g.n = (int)nb;
    g.ti = (int)((ma + S::ROWS - 1) / S::ROWS);
    g.tj = (int)((nb + BN - 1) / BN);
    g.kblocks = (int)((k + GEMM_BK - 1) / GEMM_BK);
    g.splits = splits;
    g.per = (g.kblocks + splits - 1) / splits;
    if ((splits - 1) * g.per >= g.kblocks) return cudaErrorInvalidValue;  // (the kernel waits for sums of every split)
    g.symmetric = symmetric;
    const long long tiles = symmetric ? (long long)(S::ROWS / BN) * g.ti * (g.ti + 1) / 2 : (long long)g.ti * g.tj;
    if (tiles * splits * batch >= 1 << 30) return cudaErrorInvalidValue;
    g.units = (int)(tiles * splits * batch);
    g.idesc = 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (uint32_t)g.a.mn << 15 |
              (uint32_t)g.b.mn << 16 | (uint32_t)(BN >> 3) << 17 | (uint32_t)(S::ROWS >> 4) << 24;
    auto kernel = gemm_kernel<BN, PL, CTAS, Epi>;
    static SmemOnce once;
    const cudaError_t e = once.smem(kernel, S::BYTES);
    if (e != cudaSuccess) return e;
    const int slots = GEMM_SMS / CTAS;
    // The next product's launch, barriers and Tensor Memory overlap this one's end.
    cudaLaunchAttribute ahead{};
    ahead.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    ahead.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)((g.units < slots ? g.units : slots) * CTAS));
    c.blockDim = dim3(S::THREADS);
    c.dynamicSmemBytes = S::BYTES;
    c.stream = st;
    c.attrs = &ahead;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, g, epi, fault);
}

template <int PL, class Epi>
cudaError_t gemm_launch(const GemmMat* a, const GemmMat* b, long long ma, long long nb, long long k, int batch,
                        const GemmCut& c, bool symmetric, bool bf16, const GemmIo& io, const Epi& epi,
                        unsigned int* fault, cudaStream_t st) {
    if constexpr (PL == 1 || Epi::FLUSH == 0)
        if (c.ctas == 2 && c.bn == 256)
            return gemm_launch_as<256, PL, 2>(a, b, ma, nb, k, batch, c.splits, symmetric, bf16, io, epi, fault, st);
    if (c.ctas == 2) return gemm_launch_as<128, PL, 2>(a, b, ma, nb, k, batch, c.splits, symmetric, bf16, io, epi, fault, st);
    if (c.bn == 128) return gemm_launch_as<128, PL, 1>(a, b, ma, nb, k, batch, c.splits, symmetric, bf16, io, epi, fault, st);
    return gemm_launch_as<64, PL, 1>(a, b, ma, nb, k, batch, c.splits, symmetric, bf16, io, epi, fault, st);
}

}  // namespace pz
