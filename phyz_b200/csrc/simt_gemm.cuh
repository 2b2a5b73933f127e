// Products on the FMA units, for f32 layers too small for the tensor cores'
// plane products: D[i][j] = sum_k A[i][k] B[j][k], operands of any strides.
#pragma once

#include "pz_nn.cuh"

namespace pz {

// Element (i, k) at p[i * is + k * ks].
struct SimtOperand {
    const float* p = nullptr;
    long long is = 0, ks = 0;
};

// 256 threads compute a 128 x 64 tile, 8 x 4 values each (two groups of four
// rows 64 apart, four columns), from stages of 16 k in shared memory; the next
// stage is loaded into registers while the current one is multiplied. blockIdx
// = (tiles of i, tiles of j, split of the k range). ALONG_I: D is contiguous in
// i; lanes then run along i, and the epilogue gets four values along it.
// Epi: void four(int split, long long i, long long j, const float* v, int n, bool along_i)
template <bool ALONG_I, class Epi>
__global__ void __launch_bounds__(256) simt_gemm_kernel(SimtOperand A, SimtOperand B, long long M, long long N,
                                                        long long K, long long per, Epi epi) {
    constexpr int TM = 128, TN = 64, TK = 16;
    __shared__ __align__(16) float As[TK][TM + 4];
    __shared__ __align__(16) float Bs[TK][TN + 4];
    const long long i0 = (long long)blockIdx.x * TM, j0 = (long long)blockIdx.y * TN;
    const long long k0 = blockIdx.z * per, k1 = k0 + per < K ? k0 + per : K;
    const int t = threadIdx.x, tj = ALONG_I ? t / 16 : t % 16, ti = ALONG_I ? t % 16 : t / 16;
    // consecutive threads walk the operand's unit stride
    const bool ak = A.ks == 1, bk = B.ks == 1;
    float acc[8][4] = {};
    float ra[8], rb[4];
    auto load = [&](long long k) {
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int e = t + u * 256, ii = ak ? e / TK : e % TM, kk = ak ? e % TK : e / TM;
            ra[u] = i0 + ii < M && k + kk < k1 ? A.p[(i0 + ii) * A.is + (k + kk) * A.ks] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int e = t + u * 256, jj = bk ? e / TK : e % TN, kk = bk ? e % TK : e / TN;
            rb[u] = j0 + jj < N && k + kk < k1 ? B.p[(j0 + jj) * B.is + (k + kk) * B.ks] : 0.0f;
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
    auto left = [](long long n) { return n < 4 ? (int)n : 4; };
    const long long jj = j0 + tj * 4;
    if (ALONG_I) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const long long ii = i0 + h * 64 + ti * 4;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float v[4] = {acc[h * 4][j], acc[h * 4 + 1][j], acc[h * 4 + 2][j], acc[h * 4 + 3][j]};
                if (ii < M && jj + j < N) epi.four(blockIdx.z, ii, jj + j, v, left(M - ii), true);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const long long ii = i0 + (i / 4) * 64 + ti * 4 + i % 4;
            if (ii < M && jj < N) epi.four(blockIdx.z, ii, jj, acc[i], left(N - jj), false);
        }
    }
}

template <class Epi>
cudaError_t simt_gemm(const SimtOperand& A, const SimtOperand& B, long long M, long long N, long long K, int splits,
                      bool along_i, const Epi& epi, cudaStream_t s) {
    const dim3 grid((unsigned)((M + 127) / 128), (unsigned)((N + 63) / 64), (unsigned)splits);
    const long long per = (K + splits - 1) / splits;
    if (along_i)
        simt_gemm_kernel<true><<<grid, 256, 0, s>>>(A, B, M, N, K, per, epi);
    else
        simt_gemm_kernel<false><<<grid, 256, 0, s>>>(A, B, M, N, K, per, epi);
    return cudaGetLastError();
}

}  // namespace pz
