// Products on the FMA units: D[i][j] = sum_k A[i][k] B[j][k] in f32, for
// operands of any type and strides, with the sum handed to an epilogue.
#pragma once

#include "pz_nn.cuh"

namespace pz {

// Element (i, k) at p[i * is + k * ks], batch z at p + z * zs.
struct GemmOperand {
    const void* p = nullptr;
    long long is = 0, ks = 0, zs = 0;
};

// 256 threads compute a 128 x 64 tile, 8 x 4 values each (two groups of four
// rows 64 apart, four columns), from stages of 16 k in shared memory; the next
// stage is loaded into registers while the current one is multiplied.
// blockIdx = (tiles of i, tiles of j, batch or split). With `splits` > 1, z is
// a split of the k range instead of a batch.
template <class TA, class TB, class Epi>
__global__ void __launch_bounds__(256) simt_gemm_kernel(GemmOperand A, GemmOperand B, long long M, long long N,
                                                        long long K, int splits, Epi epi) {
    constexpr int TM = 128, TN = 64, TK = 16;
    __shared__ __align__(16) float As[TK][TM + 4];
    __shared__ __align__(16) float Bs[TK][TN + 4];
    const long long i0 = (long long)blockIdx.x * TM, j0 = (long long)blockIdx.y * TN;
    const long long z = blockIdx.z;
    const TA* a = (const TA*)A.p + (splits > 1 ? 0 : z * A.zs);
    const TB* b = (const TB*)B.p + (splits > 1 ? 0 : z * B.zs);
    long long k0 = 0, k1 = K;
    if (splits > 1) {
        const long long per = (K + splits - 1) / splits;
        k0 = z * per;
        k1 = k0 + per < K ? k0 + per : K;
    }
    const int t = threadIdx.x, tj = t % 16, ti = t / 16;
    // consecutive threads walk the operand's unit stride
    const bool ak = A.ks == 1, bk = B.ks == 1;
    float acc[8][4] = {};
    float ra[8], rb[4];
    auto load = [&](long long k) {
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int e = t + u * 256, ii = ak ? e / TK : e % TM, kk = ak ? e % TK : e / TM;
            ra[u] = i0 + ii < M && k + kk < k1 ? to_f32(a[(i0 + ii) * A.is + (k + kk) * A.ks]) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int e = t + u * 256, jj = bk ? e / TK : e % TN, kk = bk ? e % TK : e / TN;
            rb[u] = j0 + jj < N && k + kk < k1 ? to_f32(b[(j0 + jj) * B.is + (k + kk) * B.ks]) : 0.0f;
        }
    };
    if (k0 < k1) load(k0);
    for (long long k = k0; k < k1; k += TK) {
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int e = t + u * 256;
            As[ak ? e % TK : e / TM][ak ? e / TK : e % TM] = ra[u];
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int e = t + u * 256;
            Bs[bk ? e % TK : e / TN][bk ? e / TK : e % TN] = rb[u];
        }
        __syncthreads();
        if (k + TK < k1) load(k + TK);
#pragma unroll
        for (int kk = 0; kk < TK; kk++) {
            float av[8], bv[4];
            *(float4*)&av[0] = *(const float4*)&As[kk][ti * 4];
            *(float4*)&av[4] = *(const float4*)&As[kk][64 + ti * 4];
            *(float4*)&bv[0] = *(const float4*)&Bs[kk][tj * 4];
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const long long ii = i0 + (i / 4) * 64 + ti * 4 + i % 4;
        if (ii >= M) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long long jj = j0 + tj * 4 + j;
            if (jj < N) epi(z, ii, jj, acc[i][j]);
        }
    }
}

template <class TA, class TB, class Epi>
cudaError_t simt_gemm(const GemmOperand& A, const GemmOperand& B, long long M, long long N, long long K, int batch,
                      int splits, const Epi& epi, cudaStream_t s) {
    const dim3 grid((unsigned)((M + 127) / 128), (unsigned)((N + 63) / 64), (unsigned)(splits > 1 ? splits : batch));
    simt_gemm_kernel<TA, TB><<<grid, 256, 0, s>>>(A, B, M, N, K, splits, epi);
    return cudaGetLastError();
}

}  // namespace pz
