// The linear layer y = act(x w^T + b) + r and its gradients.
#include "simt_gemm.cuh"

namespace pz {

namespace {

template <class T>
struct LinearEpi {
    const float* bias;
    NnMat res, y, pre;
    int act;
    __device__ void operator()(long long, long long i, long long j, float z) const {
        if (bias) z += bias[j];
        if (pre.p) ((T*)pre.p)[i * pre.rs + j * pre.cs] = from_f32<T>(z);
        float v = act_f32(z, act);
        if (res.p) v += to_f32(((const T*)res.p)[i * res.rs + j * res.cs]);
        ((T*)y.p)[i * y.rs + j * y.cs] = from_f32<T>(v);
    }
};

template <class T>
struct StoreEpi {
    NnMat out;
    __device__ void operator()(long long, long long i, long long j, float v) const {
        ((T*)out.p)[i * out.rs + j * out.cs] = from_f32<T>(v);
    }
};

// Partial sums of a split product, [split][M][N] f32.
struct PartEpi {
    float* part;
    long long M, N;
    __device__ void operator()(long long z, long long i, long long j, float v) const {
        part[(z * M + i) * N + j] = v;
    }
};

template <class T>
__global__ void join_kernel(const float* part, int splits, long long M, long long N, NnMat out) {
    const long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= M * N) return;
    float v = 0.0f;
    for (int s = 0; s < splits; s++) v += part[s * M * N + e];
    ((T*)out.p)[e / N * out.rs + e % N * out.cs] = from_f32<T>(v);
}

constexpr int DZ_ROWS = 256;  // rows per block of dz_kernel

// dz = dy act'(pre) into [m][n], and each block's column sums of the unrounded
// dz into part [row block][n].
template <class T>
__global__ void __launch_bounds__(128) dz_kernel(const phyzb_linear_grad_args a, T* dz, float* part) {
    const long long j = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (j >= a.n) return;
    const long long i0 = (long long)blockIdx.y * DZ_ROWS, i1 = i0 + DZ_ROWS < a.m ? i0 + DZ_ROWS : a.m;
    float sum = 0.0f;
    for (long long i = i0; i < i1; i++) {
        float v = to_f32(((const T*)a.dy)[i * a.dy_stride[0] + j * a.dy_stride[1]]);
        if (a.activation != PHYZB_ACT_NONE)
            v *= act_grad_f32(to_f32(((const T*)a.pre)[i * a.pre_stride[0] + j * a.pre_stride[1]]), a.activation);
        sum += v;
        dz[i * a.n + j] = from_f32<T>(v);
    }
    part[blockIdx.y * a.n + j] = sum;
}

__global__ void column_sum_kernel(const float* part, long long rows, long long n, float* out) {
    const long long j = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (j >= n) return;
    float v = 0.0f;
    for (long long r = 0; r < rows; r++) v += part[r * n + j];
    out[j] = v;
}

long long up(long long v) { return (v + 255) / 256 * 256; }
long long esize(int dtype) { return dtype == PHYZB_DT_F32 ? 4 : 2; }

// Splits of dw's sum over the rows: enough that its tiles fill the SMs, at
// least 512 rows each.
int dw_splits(const phyzb_linear_grad_args& a) {
    const long long tiles = ((a.n + 127) / 128) * ((a.k + 63) / 64);
    long long s = 444 / tiles, most = a.m / 512;
    s = s < most ? s : most;
    return (int)(s < 1 ? 1 : s > 128 ? 128 : s);
}

struct GradWs {
    long long dz, part, dw, total;
};
GradWs grad_ws(const phyzb_linear_grad_args& a) {
    GradWs w{};
    long long at = 0;
    w.dz = at;
    at += up(a.m * a.n * esize(a.dtype));
    w.part = at;
    at += up((a.m + DZ_ROWS - 1) / DZ_ROWS * a.n * 4);
    w.dw = at;
    const int s = dw_splits(a);
    if (s > 1) at += up((long long)s * a.n * a.k * 4);
    w.total = at;
    return w;
}

template <class T>
cudaError_t backward(const phyzb_linear_grad_args& a, char* ws, cudaStream_t s) {
    const GradWs w = grad_ws(a);
    T* dz = (T*)(ws + w.dz);
    float* part = (float*)(ws + w.part);
    const unsigned nb = (unsigned)((a.n + 127) / 128);
    const long long rb = (a.m + DZ_ROWS - 1) / DZ_ROWS;
    if (a.m) dz_kernel<T><<<dim3(nb, (unsigned)rb), 128, 0, s>>>(a, dz, part);
    if (a.dbias) column_sum_kernel<<<nb, 128, 0, s>>>(part, rb, a.n, a.dbias);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && a.dx && a.m)
        e = simt_gemm<T, T>({dz, a.n, 1, 0}, {a.w, a.w_stride[1], a.w_stride[0], 0}, a.m, a.k, a.n, 1, 1,
                            StoreEpi<T>{{a.dx, a.dx_stride[0], a.dx_stride[1]}}, s);
    if (e == cudaSuccess && a.dw) {
        const GemmOperand A{dz, 1, a.n, 0}, B{a.x, a.x_stride[1], a.x_stride[0], 0};
        const NnMat dw{a.dw, a.dw_stride[0], a.dw_stride[1]};
        const int splits = dw_splits(a);
        if (splits == 1) return simt_gemm<T, T>(A, B, a.n, a.k, a.m, 1, 1, StoreEpi<T>{dw}, s);
        float* p = (float*)(ws + w.dw);
        e = simt_gemm<T, T>(A, B, a.n, a.k, a.m, 1, splits, PartEpi{p, a.n, a.k}, s);
        if (e != cudaSuccess) return e;
        join_kernel<T><<<(unsigned)((a.n * a.k + 255) / 256), 256, 0, s>>>(p, splits, a.n, a.k, dw);
        e = cudaGetLastError();
    }
    return e;
}

template <class T>
cudaError_t forward(const phyzb_linear_args& a, cudaStream_t s) {
    const LinearEpi<T> epi{a.bias,
                           {(void*)a.residual, a.residual_stride[0], a.residual_stride[1]},
                           {a.y, a.y_stride[0], a.y_stride[1]},
                           {a.pre, a.pre_stride[0], a.pre_stride[1]},
                           a.activation};
    return simt_gemm<T, T>({a.x, a.x_stride[0], a.x_stride[1], 0}, {a.w, a.w_stride[0], a.w_stride[1], 0}, a.m, a.n,
                           a.k, 1, 1, epi, s);
}

}  // namespace

long long linear_workspace(const phyzb_linear_args&) { return 0; }
long long linear_grad_workspace(const phyzb_linear_grad_args& a) { return grad_ws(a).total; }

cudaError_t linear_forward(const phyzb_linear_args& a, void*, cudaStream_t s) {
    if (a.dtype == PHYZB_DT_F32) return forward<float>(a, s);
    if (a.dtype == PHYZB_DT_BF16) return forward<__nv_bfloat16>(a, s);
    return forward<__half>(a, s);
}

cudaError_t linear_backward(const phyzb_linear_grad_args& a, void* ws, cudaStream_t s) {
    if (a.dtype == PHYZB_DT_F32) return backward<float>(a, (char*)ws, s);
    if (a.dtype == PHYZB_DT_BF16) return backward<__nv_bfloat16>(a, (char*)ws, s);
    return backward<__half>(a, (char*)ws, s);
}

}  // namespace pz
