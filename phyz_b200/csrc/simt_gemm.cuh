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
// = (tiles of i, tiles of j, split of the k range), or with wide (tiles of j, of i,
// split): a grid's second side ends at 65535. Bound by instructions: 65536 x
// 30 x 64 with bias, tanh and pre-activations, 41 MB, 20.2 us. ALONG_I: D is contiguous in
// i; lanes then run along i, and the epilogue gets four values along it.
// Epi: each(f) calls f(kind) once, and f void four(kind, int split, long long i, long long j, const float* v, int n,
// bool along_i)
template <bool ALONG_I, class Epi>
__global__ void __launch_bounds__(256) simt_gemm_kernel(SimtOperand A, SimtOperand B, long long M, long long N,
                                                        long long K, long long per, bool wide, Epi epi) {
    constexpr int TM = 128, TN = 64, TK = 16;
    __shared__ __align__(16) float As[TK][TM + 4];
    __shared__ __align__(16) float Bs[TK][TN + 4];
    const long long i0 = (long long)(wide ? blockIdx.y : blockIdx.x) * TM;
    const long long j0 = (long long)(wide ? blockIdx.x : blockIdx.y) * TN;
    const long long k0 = blockIdx.z * per, k1 = k0 + per < K ? k0 + per : K;
    const int t = threadIdx.x, tj = ALONG_I ? t / 16 : t % 16, ti = ALONG_I ? t % 16 : t / 16;
    // consecutive threads walk the operand's unit stride: a thread's elements of a
    // stage are one column (or row) apart by a fixed step
    const bool ak = A.ks == 1, bk = B.ks == 1;
    float acc[8][4] = {};
    float ra[8], rb[4];
    const int ai = ak ? t / TK : t % TM, akk = ak ? t % TK : t / TM;
    const int bj = bk ? t / TK : t % TN, bkk = bk ? t % TK : t / TN;
    const float* pa = A.p + (i0 + ai) * A.is + (k0 + akk) * A.ks;
    const float* pb = B.p + (j0 + bj) * B.is + (k0 + bkk) * B.ks;
    const long long sa = ak ? 16 * A.is : 2 * A.ks, sb = bk ? 16 * B.is : 4 * B.ks;
    const int mleft = M - i0 < TM ? (int)(M - i0) : TM, nleft = N - j0 < TN ? (int)(N - j0) : TN;
    auto load = [&](long long k) {
        const int kleft = k1 - k < TK ? (int)(k1 - k) : TK;
        const float* p = pa;
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const bool on = ak ? akk < kleft && ai + 16 * u < mleft : ai < mleft && akk + 2 * u < kleft;
            ra[u] = on ? *p : 0.0f;
            p += sa;
        }
        p = pb;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const bool on = bk ? bkk < kleft && bj + 16 * u < nleft : bj < nleft && bkk + 4 * u < kleft;
            rb[u] = on ? *p : 0.0f;
            p += sb;
        }
        pa += TK * A.ks;
        pb += TK * B.ks;
    };
    if (k0 < k1) load(k0);
    for (long long k = k0; k < k1; k += TK) {
#pragma unroll
        for (int u = 0; u < 8; u++) As[ak ? akk : akk + 2 * u][ak ? ai + 16 * u : ai] = ra[u];
#pragma unroll
        for (int u = 0; u < 4; u++) Bs[bk ? bkk : bkk + 4 * u][bk ? bj + 16 * u : bj] = rb[u];
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
    auto left = [](int n) { return n < 4 ? n : 4; };
    const int jj = tj * 4;
    epi.each([&](auto kind) {
        if (ALONG_I) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int ii = h * 64 + ti * 4;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float v[4] = {acc[h * 4][j], acc[h * 4 + 1][j], acc[h * 4 + 2][j], acc[h * 4 + 3][j]};
                    if (ii < mleft && jj + j < nleft)
                        epi.four(kind, blockIdx.z, i0 + ii, j0 + jj + j, v, left(mleft - ii), true);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int ii = (i / 4) * 64 + ti * 4 + i % 4;
                if (ii < mleft && jj < nleft) epi.four(kind, blockIdx.z, i0 + ii, j0 + jj, acc[i], left(nleft - jj), false);
            }
        }
    });
}

template <class Epi>
cudaError_t simt_gemm(const SimtOperand& A, const SimtOperand& B, long long M, long long N, long long K, int splits,
                      bool along_i, const Epi& epi, cudaStream_t s) {
    const unsigned ti = (unsigned)((M + 127) / 128), tj = (unsigned)((N + 63) / 64);
    const bool wide = tj > 65535;
    const dim3 grid(wide ? tj : ti, wide ? ti : tj, (unsigned)splits);
    const long long per = (K + splits - 1) / splits;
    if (along_i)
        simt_gemm_kernel<true><<<grid, 256, 0, s>>>(A, B, M, N, K, per, wide, epi);
    else
        simt_gemm_kernel<false><<<grid, 256, 0, s>>>(A, B, M, N, K, per, wide, epi);
    return cudaGetLastError();
}

}  // namespace pz
