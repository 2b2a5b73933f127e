// The Muon update: momentum, orthogonalisation of the direction by
// Newton-Schulz products, weight update.
//
//   X = u / |u|_F;  5 times: G = X X^T, X <- a X + (b G + c G G) X
//
// (from the right where the matrix is tall: G is on the short side s, and X
// stays in the order of the caller's matrix). The polynomial's slope is up to
// 3.4445 an iteration, 485 over five, so a product's error grows: in bf16 the
// result is 2 % off, in bf16 pairs 4e-5, in f16 pairs 1e-6 to 1e-5, which is
// where f32 products are. So values are kept as f16 pairs hi + lo, at a fixed
// scale of 2^12: |X| <= 1.3, |G| <= 1.7 and |b G + c G G| <= 2.8 then stay under
// 11500 (f16 ends at 65504), and what is lost below lo is 2^-25 2^-12 of one.
// Three products of the tensor cores to a product (gemm.cuh), f32 sums; G and
// b G + c G G are symmetric and only half their tiles are computed.
#include "gemm.cuh"

namespace pz {

namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f, NS_EPS = 1e-7f;
constexpr float SCALE = 4096.0f;
constexpr int NORM_BLOCKS = 64;  // partial sums of a matrix's |u|^2

__device__ unsigned int g_muon_fault;  // waits that ran out (pz_tma.cuh)

unsigned int* fault_word() {
    static std::atomic<unsigned int*> at[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return nullptr;
    unsigned int* p = at[dev].load(std::memory_order_acquire);
    if (!p) {
        void* q = nullptr;
        if (cudaGetSymbolAddress(&q, g_muon_fault) != cudaSuccess) return nullptr;
        at[dev].store(p = (unsigned int*)q, std::memory_order_release);
    }
    return p;
}

// A stack of matrices: element (z, r, c) at p[z * zs + r * rs + c * cs].
struct View {
    void* p = nullptr;
    long long zs = 0, rs = 0, cs = 0;
};

struct Problem {
    int batch, rows, cols, steps;
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

// f16 pairs of a stack of matrices [batch][rows][pitch], at SCALE.
struct Pair {
    __half* p = nullptr;
    long long lo = 0, zs = 0, pitch = 0;  // offset of the low plane; strides
    __device__ __forceinline__ float get(long long e) const {
        return __half2float(p[e]) + __half2float(p[e + lo]);
    }
    __device__ __forceinline__ void put(long long e, float v) const {
        const __half h = __float2half_rn(v);
        p[e] = h;
        p[e + lo] = __float2half_rn(v - __half2float(h));
    }
};

// The direction at (z, r, c) from the advanced momentum.
__device__ __forceinline__ float direction(const Problem& q, int z, long long r, long long c) {
    const float g = load_as(q.g.p, z * q.g.zs + r * q.g.rs + c * q.g.cs, q.dtype);
    if (!q.m.p) return g;
    const float m = ((const float*)q.m.p)[z * q.m.zs + r * q.m.rs + c * q.m.cs];
    return q.nesterov ? fmaf(q.mu, m, g) : m;
}

// Momentum advanced, and each block's sum of u^2 (rows r = block, block + 64, ..).
__global__ void __launch_bounds__(256) momentum_kernel(const __grid_constant__ Problem q, float* part) {
    const int z = blockIdx.y;
    float sum = 0.0f;
    const long long n = (long long)q.rows * q.cols, per = (n + NORM_BLOCKS - 1) / NORM_BLOCKS;
    const long long e0 = blockIdx.x * per, e1 = e0 + per < n ? e0 + per : n;
    for (long long e = e0 + threadIdx.x; e < e1; e += 256) {
        const int r = (int)e / q.cols, c = (int)e - r * q.cols;  // (at most 2^28 elements)
        if (q.m.p) {
            float* m = (float*)q.m.p + z * q.m.zs + r * q.m.rs + c * q.m.cs;
            *m = fmaf(q.mu, *m, load_as(q.g.p, z * q.g.zs + r * q.g.rs + c * q.g.cs, q.dtype));
        }
        const float u = direction(q, z, r, c);
        sum = fmaf(u, u, sum);
    }
    __shared__ float sm[8];
#pragma unroll
    for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; w++) s += sm[w];
        part[z * NORM_BLOCKS + blockIdx.x] = s;
    }
}

// 1 / (|u| + eps) from the blocks' sums, the same in every thread of a warp.
__device__ __forceinline__ float inverse_norm(const float* part, int z) {
    const int lane = threadIdx.x % 32;
    float s = part[z * NORM_BLOCKS + lane] + part[z * NORM_BLOCKS + 32 + lane];
#pragma unroll
    for (int o = 16; o; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    return 1.0f / (sqrtf(s) + NS_EPS);
}

__global__ void __launch_bounds__(256) normalize_kernel(const __grid_constant__ Problem q, const float* part, Pair x) {
    const int z = blockIdx.y;
    const float k = inverse_norm(part, z) * SCALE;
    const long long n = (long long)q.rows * q.cols;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
        const int r = (int)e / q.cols, c = (int)e - r * q.cols;
        x.put(z * x.zs + r * x.pitch + c, direction(q, z, r, c) * k);
    }
}

// ── epilogues: D is at SCALE^2 ────────────────────────────────────────────

// G = sum, or b G + c sum, and its mirror image: D[i][j] = D[j][i].
struct SquareEpi {
    Pair out, g;
    float b, c;  // c / SCALE
    int s;
    __device__ __forceinline__ void operator()(const GemmUnit& q, long long i, int j0, int cols, const float* sum) const {
        if (i >= s) return;
        const long long z = q.z * out.zs;
        // the tile's mirror image, unless it is inside a diagonal block
        const bool mirror = j0 < q.i * GEMM_BM;
        float v[32];
        if (g.p) {
#pragma unroll
            for (int k = 0; k < 32; k++) v[k] = k < cols ? g.get(z + (j0 + k) * g.pitch + i) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 32; k++) {
            v[k] = g.p ? fmaf(b, v[k], c * sum[k]) : c * sum[k];
            if (k < cols) out.put(z + (j0 + k) * out.pitch + i, v[k]);
        }
        if (mirror) {
#pragma unroll
            for (int k = 0; k < 32; k++)
                if (k < cols) out.put(z + i * out.pitch + j0 + k, v[k]);
        }
    }
};

// a X + sum; i along the columns of X, j along its rows.
struct StepEpi {
    Pair x, out;
    int cols_;
    __device__ __forceinline__ void operator()(const GemmUnit& q, long long i, int j0, int cols, const float* sum) const {
        if (i >= cols_) return;
        const long long e = q.z * x.zs + j0 * x.pitch + i;
        float v[32];
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] = k < cols ? x.get(e + k * x.pitch) : 0.0f;
#pragma unroll
        for (int k = 0; k < 32; k++)
            if (k < cols) out.put(e + k * x.pitch, fmaf(NS_A, v[k], sum[k] * (1.0f / SCALE)));
    }
};

// The last a X + sum, into the weights or the result.
struct LastEpi {
    Pair x;
    Problem q;
    __device__ __forceinline__ void operator()(const GemmUnit& u, long long i, int j0, int cols, const float* sum) const {
        if (i >= q.cols) return;
        const long long z = u.z, e = z * x.zs + j0 * x.pitch + i;
        float v[32];
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] = k < cols ? x.get(e + k * x.pitch) : 0.0f;
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] = fmaf(NS_A, v[k], sum[k] * (1.0f / SCALE)) * (1.0f / SCALE);
        if (q.out.p) {
#pragma unroll
            for (int k = 0; k < 32; k++)
                if (k < cols) store_as(q.out.p, z * q.out.zs + (j0 + k) * q.out.rs + i * q.out.cs, q.out_dtype, v[k]);
            return;
        }
        float* w = (float*)q.w.p + z * q.w.zs + j0 * q.w.rs + i * q.w.cs;
        float old[32];
#pragma unroll
        for (int k = 0; k < 32; k++) old[k] = k < cols ? w[k * q.w.rs] : 0.0f;
#pragma unroll
        for (int k = 0; k < 32; k++) {
            if (k >= cols) break;
            const float t = fmaf(-q.lr, v[k], q.decay * old[k]);
            w[k * q.w.rs] = t;
            if (q.copy.p)
                store_as(q.copy.p, z * q.copy.zs + (j0 + k) * q.copy.rs + i * q.copy.cs, q.copy_dtype, t);
        }
    }
};

// ── host side ─────────────────────────────────────────────────────────────

long long up(long long v, long long to) { return (v + to - 1) / to * to; }

struct Ws {
    Pair x, y, g, p;
    long long x_at, y_at, g_at, p_at, part_at, total;
};
Ws layout(long long batch, long long rows, long long cols) {
    Ws w{};
    const long long s = rows < cols ? rows : cols;
    long long at = 0;
    auto take = [&](Pair& p, long long r, long long c) {
        p.pitch = up(c, 8);
        p.zs = r * p.pitch;
        p.lo = up(batch * p.zs, 128);
        const long long o = at;
        at += 2 * p.lo * 2;
        return o;
    };
    w.x_at = take(w.x, rows, cols);
    w.y_at = take(w.y, rows, cols);
    w.g_at = take(w.g, s, s);
    w.p_at = take(w.p, s, s);
    w.part_at = at;
    w.total = at + up(batch * NORM_BLOCKS * 4, 256);
    return w;
}

// D = A B^T on pairs. BN = 128 does twice the work of 64 per byte of shared
// memory; 64 where 128 leaves SMs idle in the only round.
template <class Epi>
cudaError_t multiply(const Pair& a, bool a_mn, const Pair& b, bool b_mn, long long rows, long long cols, long long k,
                     int batch, bool symmetric, const Epi& epi, unsigned int* fault, cudaStream_t st) {
    GemmMat ma[2], mb[2];
    for (int h = 0; h < 2; h++) {
        ma[h] = {a.p + h * a.lo, a_mn ? 1 : a.pitch, a_mn ? a.pitch : 1, a.zs};
        mb[h] = {b.p + h * b.lo, b_mn ? 1 : b.pitch, b_mn ? b.pitch : 1, b.zs};
    }
    const long long ti = (rows + 127) / 128, tj = (cols + 127) / 128;
    const long long units = (symmetric ? ti * (ti + 1) / 2 : ti * tj) * batch;
    if (units * 2 <= GEMM_SMS)
        return gemm_launch<64, 2>(ma, mb, rows, cols, k, batch, 1, symmetric, false, epi, fault, st);
    return gemm_launch<128, 2>(ma, mb, rows, cols, k, batch, 1, symmetric, false, epi, fault, st);
}

cudaError_t solve(const Problem& q, char* ws, cudaStream_t st) {
    unsigned int* fault = fault_word();
    if (!fault) return cudaErrorInvalidSymbol;
    Ws o = layout(q.batch, q.rows, q.cols);
    o.x.p = (__half*)(ws + o.x_at);
    o.y.p = (__half*)(ws + o.y_at);
    o.g.p = (__half*)(ws + o.g_at);
    o.p.p = (__half*)(ws + o.p_at);
    float* part = (float*)(ws + o.part_at);
    const bool tall = q.rows > q.cols;
    const int s = tall ? q.cols : q.rows, l = tall ? q.rows : q.cols;
    const long long n = (long long)q.rows * q.cols;
    momentum_kernel<<<dim3(NORM_BLOCKS, (unsigned)q.batch), 256, 0, st>>>(q, part);
    const long long blocks = (n + 1023) / 1024;
    normalize_kernel<<<dim3((unsigned)(blocks < 1024 ? blocks : 1024), (unsigned)q.batch), 256, 0, st>>>(q, part, o.x);
    cudaError_t e = cudaGetLastError();
    Pair x = o.x, y = o.y;
    for (int k = 0; k < q.steps && e == cudaSuccess; k++) {
        // G: the short side's products along the long one
        e = multiply(x, tall, x, tall, s, s, l, q.batch, true, SquareEpi{o.g, Pair{}, 0.0f, 1.0f / SCALE, s}, fault, st);
        if (e != cudaSuccess) break;
        e = multiply(o.g, false, o.g, false, s, s, s, q.batch, true, SquareEpi{o.p, o.g, NS_B, NS_C / SCALE, s}, fault, st);
        if (e != cudaSuccess) break;
        // i = columns of X. Wide: X^T's rows by P's; tall: P's rows by X's
        const Pair &a = tall ? o.p : x, &b = tall ? x : o.p;
        if (k + 1 < q.steps)
            e = multiply(a, !tall, b, false, q.cols, q.rows, s, q.batch, false, StepEpi{x, y, q.cols}, fault, st);
        else
            e = multiply(a, !tall, b, false, q.cols, q.rows, s, q.batch, false, LastEpi{x, q}, fault, st);
        const Pair t = x;
        x = y;
        y = t;
    }
    return e;
}

View view(const void* p, const int64_t* st) { return {(void*)p, st[0], st[1], st[2]}; }

}  // namespace

long long muon_workspace(const phyzb_muon_args& a) { return layout(a.batch, a.rows, a.cols).total; }

cudaError_t muon_update(const phyzb_muon_args& a, void* ws, cudaStream_t s) {
    Problem q{};
    q.batch = (int)a.batch;
    q.rows = (int)a.rows;
    q.cols = (int)a.cols;
    q.steps = a.steps;
    q.g = view(a.grad, a.grad_stride);
    q.m = view(a.momentum, a.momentum_stride);
    q.w = view(a.weight, a.weight_stride);
    q.copy = view(a.copy, a.copy_stride);
    q.dtype = a.dtype;
    q.copy_dtype = a.copy_dtype;
    q.nesterov = a.nesterov != 0;
    q.mu = (float)a.mu;
    q.decay = (float)(1.0 - a.lr * a.weight_decay);
    q.lr = (float)(a.lr * a.scale);
    return solve(q, (char*)ws, s);
}

long long orthogonalize_workspace(const phyzb_orthogonalize_args& a) { return layout(a.batch, a.rows, a.cols).total; }

cudaError_t orthogonalize(const phyzb_orthogonalize_args& a, void* ws, cudaStream_t s) {
    Problem q{};
    q.batch = (int)a.batch;
    q.rows = (int)a.rows;
    q.cols = (int)a.cols;
    q.steps = a.steps;
    q.g = view(a.x, a.x_stride);
    q.out = view(a.out, a.out_stride);
    q.dtype = q.out_dtype = a.dtype;
    return solve(q, (char*)ws, s);
}

cudaError_t muon_faults(unsigned int* n) { return cudaMemcpyFromSymbol(n, g_muon_fault, sizeof(*n)); }

}  // namespace pz
