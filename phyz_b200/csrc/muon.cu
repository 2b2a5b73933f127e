// The Muon update: momentum, orthogonalisation by Newton-Schulz products,
// weight update.
#include "simt_gemm.cuh"

namespace pz {

namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f, NS_EPS = 1e-7f;
constexpr int NORM_BLOCKS = 64;

// A [batch][rows][cols] view in its short-side-first orientation is
// [batch][s][l]: element (z, i, j) at p[z * zs + i * is + j * js].
struct View {
    void* p = nullptr;
    long long zs = 0, is = 0, js = 0;
};

struct Problem {
    int batch, s, l, steps;
    View g, m, w, copy, out;
    int dtype, copy_dtype, out_dtype;
    bool nesterov;
    float mu, decay, lr;  // decay = 1 - lr * weight_decay, lr already scaled
};

__device__ __forceinline__ float load_as(const void* p, long long e, int dtype) {
    return dtype == PHYZB_DT_F32    ? ((const float*)p)[e]
           : dtype == PHYZB_DT_BF16 ? __bfloat162float(((const __nv_bfloat16*)p)[e])
                                    : __half2float(((const __half*)p)[e]);
}
__device__ __forceinline__ void store_as(void* p, long long e, int dtype, float v) {
    if (dtype == PHYZB_DT_F32)
        ((float*)p)[e] = v;
    else if (dtype == PHYZB_DT_BF16)
        ((__nv_bfloat16*)p)[e] = __float2bfloat16_rn(v);
    else
        ((__half*)p)[e] = __float2half_rn(v);
}

// u = the direction, momentum advanced; each block's sum of u^2.
__global__ void __launch_bounds__(256) direction_kernel(Problem q, float* u, float* part) {
    const long long n = (long long)q.s * q.l, z = blockIdx.y;
    float sum = 0.0f;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
        const long long i = e / q.l, j = e % q.l;
        float v = load_as(q.g.p, z * q.g.zs + i * q.g.is + j * q.g.js, q.dtype);
        if (q.m.p) {
            float* m = (float*)q.m.p + z * q.m.zs + i * q.m.is + j * q.m.js;
            const float mn = fmaf(q.mu, *m, v);
            *m = mn;
            v = q.nesterov ? fmaf(q.mu, mn, v) : mn;
        }
        u[z * n + e] = v;
        sum = fmaf(v, v, sum);
    }
    __shared__ float sm[256];
    sm[threadIdx.x] = sum;
    __syncthreads();
    for (int h = 128; h; h /= 2) {
        if (threadIdx.x < h) sm[threadIdx.x] += sm[threadIdx.x + h];
        __syncthreads();
    }
    if (threadIdx.x == 0) part[z * NORM_BLOCKS + blockIdx.x] = sm[0];
}

__global__ void __launch_bounds__(256) normalize_kernel(float* u, const float* part, long long n) {
    float sum = 0.0f;
    for (int k = 0; k < NORM_BLOCKS; k++) sum += part[blockIdx.y * NORM_BLOCKS + k];
    const float r = 1.0f / (sqrtf(sum) + NS_EPS);
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256)
        u[blockIdx.y * n + e] *= r;
}

// out = alpha * C + beta * sum
struct AxpbyEpi {
    const float* c;
    float* out;
    float alpha, beta;
    long long zs, ld;
    __device__ void operator()(long long z, long long i, long long j, float v) const {
        const long long e = z * zs + i * ld + j;
        out[e] = (c ? alpha * c[e] : 0.0f) + beta * v;
    }
};

__global__ void apply_kernel(Problem q, const float* x) {
    const long long n = (long long)q.s * q.l, z = blockIdx.y;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
        const long long i = e / q.l, j = e % q.l;
        const float v = x[z * n + e];
        if (q.out.p) store_as(q.out.p, z * q.out.zs + i * q.out.is + j * q.out.js, q.out_dtype, v);
        if (q.w.p) {
            float* w = (float*)q.w.p + z * q.w.zs + i * q.w.is + j * q.w.js;
            *w = fmaf(-q.lr, v, q.decay * *w);
            if (q.copy.p) store_as(q.copy.p, z * q.copy.zs + i * q.copy.is + j * q.copy.js, q.copy_dtype, *w);
        }
    }
}

struct Ws {
    long long x, y, g, p, part, total;
};
Ws layout(long long batch, long long s, long long l) {
    Ws w{};
    long long at = 0;
    auto take = [&](long long n) {
        const long long o = at;
        at += (n * 4 + 255) / 256 * 256;
        return o;
    };
    w.x = take(batch * s * l);
    w.y = take(batch * s * l);
    w.g = take(batch * s * s);
    w.p = take(batch * s * s);
    w.part = take(batch * NORM_BLOCKS);
    w.total = at;
    return w;
}

cudaError_t solve(const Problem& q, char* ws, cudaStream_t st) {
    const Ws o = layout(q.batch, q.s, q.l);
    float *x = (float*)(ws + o.x), *y = (float*)(ws + o.y), *g = (float*)(ws + o.g), *p = (float*)(ws + o.p);
    float* part = (float*)(ws + o.part);
    const dim3 grid(NORM_BLOCKS, (unsigned)q.batch);
    const long long n = (long long)q.s * q.l, ss = (long long)q.s * q.s, s = q.s, l = q.l;
    direction_kernel<<<grid, 256, 0, st>>>(q, x, part);
    normalize_kernel<<<grid, 256, 0, st>>>(x, part, n);
    cudaError_t e = cudaGetLastError();
    for (int k = 0; k < q.steps && e == cudaSuccess; k++) {
        e = simt_gemm<float, float>({x, l, 1, n}, {x, l, 1, n}, s, s, l, q.batch, 1,
                                    AxpbyEpi{nullptr, g, 0.0f, 1.0f, ss, s}, st);
        if (e == cudaSuccess)
            e = simt_gemm<float, float>({g, s, 1, ss}, {g, s, 1, ss}, s, s, s, q.batch, 1,
                                        AxpbyEpi{g, p, NS_B, NS_C, ss, s}, st);
        if (e == cudaSuccess)
            e = simt_gemm<float, float>({p, s, 1, ss}, {x, 1, l, n}, s, l, s, q.batch, 1,
                                        AxpbyEpi{x, y, NS_A, 1.0f, n, l}, st);
        float* t = x;
        x = y;
        y = t;
    }
    if (e != cudaSuccess) return e;
    apply_kernel<<<grid, 256, 0, st>>>(q, x);
    return cudaGetLastError();
}

View view(const void* p, const int64_t* st, bool tall) {
    return {(void*)p, st[0], tall ? st[2] : st[1], tall ? st[1] : st[2]};
}

Problem sides(long long batch, long long rows, long long cols, int steps) {
    Problem q{};
    q.batch = (int)batch;
    q.s = (int)(rows < cols ? rows : cols);
    q.l = (int)(rows < cols ? cols : rows);
    q.steps = steps;
    return q;
}

}  // namespace

long long muon_workspace(const phyzb_muon_args& a) {
    const Problem q = sides(a.batch, a.rows, a.cols, a.steps);
    return layout(q.batch, q.s, q.l).total;
}

cudaError_t muon_update(const phyzb_muon_args& a, void* ws, cudaStream_t s) {
    Problem q = sides(a.batch, a.rows, a.cols, a.steps);
    const bool tall = a.rows > a.cols;
    q.g = view(a.grad, a.grad_stride, tall);
    q.m = view(a.momentum, a.momentum_stride, tall);
    q.w = view(a.weight, a.weight_stride, tall);
    q.copy = view(a.copy, a.copy_stride, tall);
    q.dtype = a.dtype;
    q.copy_dtype = a.copy_dtype;
    q.nesterov = a.nesterov != 0;
    q.mu = (float)a.mu;
    q.decay = (float)(1.0 - a.lr * a.weight_decay);
    q.lr = (float)(a.lr * a.scale);
    return solve(q, (char*)ws, s);
}

long long orthogonalize_workspace(const phyzb_orthogonalize_args& a) {
    const Problem q = sides(a.batch, a.rows, a.cols, a.steps);
    return layout(q.batch, q.s, q.l).total;
}

cudaError_t orthogonalize(const phyzb_orthogonalize_args& a, void* ws, cudaStream_t s) {
    Problem q = sides(a.batch, a.rows, a.cols, a.steps);
    const bool tall = a.rows > a.cols;
    q.g = view(a.x, a.x_stride, tall);
    q.out = view(a.out, a.out_stride, tall);
    q.dtype = q.out_dtype = a.dtype;
    return solve(q, (char*)ws, s);
}

}  // namespace pz
