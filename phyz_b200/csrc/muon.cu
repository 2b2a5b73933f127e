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
//
// The tensor cores cut their sums' additions off towards zero, and five
// iterations make 1.3e-5 of it at 515 x 1030 (f32 products: 2.9e-6). That is far
// below what an update by lr X shows, so the update takes it. orthogonalize,
// whose result is X itself, has the sums flushed every 128 of k (FLUSH = 2):
// 3.3e-6, for 4 % more time.
#include "gemm.cuh"

namespace pz {

namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f, NS_EPS = 1e-7f;
constexpr float SCALE = 4096.0f;
constexpr int NORM_BLOCKS = 512;  // partial sums of a matrix's |u|^2, at most

__device__ unsigned int g_muon_fault;  // waits that ran out (pz_tma.cuh)

unsigned int* fault_word() {
    static FaultWord word;
    return word.get(g_muon_fault);
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
// f16 pairs of a stack of matrices [batch][rows][pitch], at SCALE.
struct Pair {
    __half* p = nullptr;
    long long lo = 0, zs = 0, pitch = 0;  // offset of the low plane; strides
};

// V neighbours of row r from column c: momentum advanced (ADVANCE) or as it is,
// and the direction u from it.
template <int V, bool ADVANCE>
__device__ __forceinline__ void direction(const Problem& q, int z, int r, int c, float* u) {
    const long long eg = z * q.g.zs + r * q.g.rs + c * q.g.cs;
    if constexpr (V == 4) {
        if (q.dtype == PHYZB_DT_F32) {
            *(float4*)u = *(const float4*)((const float*)q.g.p + eg);
        } else {
            const uint2 w = *(const uint2*)((const uint16_t*)q.g.p + eg);
            const uint16_t h[4] = {(uint16_t)w.x, (uint16_t)(w.x >> 16), (uint16_t)w.y, (uint16_t)(w.y >> 16)};
#pragma unroll
            for (int v = 0; v < 4; v++)
                u[v] = q.dtype == PHYZB_DT_BF16 ? __bfloat162float(*(const __nv_bfloat16*)&h[v])
                                                : __half2float(*(const __half*)&h[v]);
        }
    } else {
        u[0] = load_as(q.g.p, eg, q.dtype);
    }
    if (!q.m.p) return;
    float* pm = (float*)q.m.p + z * q.m.zs + r * q.m.rs + c * q.m.cs;
    float m[V];
    if constexpr (V == 4)
        *(float4*)m = *(const float4*)pm;
    else
        m[0] = *pm;
#pragma unroll
    for (int v = 0; v < V; v++) {
        if (ADVANCE) m[v] = fmaf(q.mu, m[v], u[v]);
        u[v] = q.nesterov ? fmaf(q.mu, m[v], u[v]) : m[v];
    }
    if (!ADVANCE) return;
    if constexpr (V == 4)
        *(float4*)pm = *(const float4*)m;
    else
        *pm = m[0];
}

// Stretches of 256 V columns of a row, one to a block at a time: f(row, column).
template <int V, class F>
__device__ __forceinline__ void each_stretch(const Problem& q, F f) {
    const int per = (q.cols + 256 * V - 1) / (256 * V), n = per * q.rows;
#pragma unroll 2
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int r = i / per, c = (i - r * per) * 256 * V + threadIdx.x * V;
        if (c < q.cols) f(r, c);
    }
}

// Momentum advanced, and each block's sum of u^2.
template <int V>
__global__ void __launch_bounds__(256) momentum_kernel(const __grid_constant__ Problem q, float* part) {
    const int z = blockIdx.y;
    float sum = 0.0f;
    each_stretch<V>(q, [&](int r, int c) {
        float u[V];
        direction<V, true>(q, z, r, c, u);
#pragma unroll
        for (int v = 0; v < V; v++) sum = fmaf(u[v], u[v], sum);
    });
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

// 1 / (|u| + eps) from `blocks` sums, the same in every thread of a warp.
__device__ __forceinline__ float inverse_norm(const float* part, int z, int blocks) {
    float s = 0.0f;
#pragma unroll 4
    for (int k = threadIdx.x % 32; k < blocks; k += 32) s += part[z * NORM_BLOCKS + k];
#pragma unroll
    for (int o = 16; o; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    return 1.0f / (sqrtf(s) + NS_EPS);
}

template <int V>
__global__ void __launch_bounds__(256) normalize_kernel(const __grid_constant__ Problem q, const float* part, Pair x) {
    const int z = blockIdx.y;
    const float k = inverse_norm(part, z, gridDim.x) * SCALE;
    each_stretch<V>(q, [&](int r, int c) {
        float u[V];
        direction<V, false>(q, z, r, c, u);
        __half h[V], l[V];
#pragma unroll
        for (int v = 0; v < V; v++) {
            h[v] = __float2half_rn(u[v] * k);
            l[v] = __float2half_rn(u[v] * k - __half2float(h[v]));
        }
        __half* p = x.p + z * x.zs + r * x.pitch + c;
        if constexpr (V == 4) {
            *(uint2*)p = *(const uint2*)h;
            *(uint2*)(p + x.lo) = *(const uint2*)l;
        } else {
            p[0] = h[0];
            p[x.lo] = l[0];
        }
    });
}

// ── epilogues: D is at SCALE^2 ────────────────────────────────────────────

// a lane's 32 values of a slot's pair
__device__ __forceinline__ void pair_load(const unsigned char* in, float* v) {
    uint32_t w[16];
    float l[32];
    slot_load(in, w);
    unpack32(w, v, __half());
    slot_load(in + GEMM_PLANE, w);
    unpack32(w, l, __half());
#pragma unroll
    for (int k = 0; k < 32; k++) v[k] += l[k];
}
__device__ __forceinline__ void split(const float* v, __half* h, __half* l) {
#pragma unroll
    for (int k = 0; k < 32; k++) {
        h[k] = __float2half_rn(v[k]);
        l[k] = __float2half_rn(v[k] - __half2float(h[k]));
    }
}

// G = sum, or b G + c sum, and its mirror image: D[i][j] = D[j][i]. (The pairs are
// in the workspace: all of this goes through slots.)
template <int F>  // k blocks to a sum of the tensor cores (0: all)
struct SquareEpi {
    static constexpr int PLANES = 2, SLOTS = 1, WARPS = 8, FLUSH = F;
    static constexpr bool MIRROR = true;
    float b, c;  // c / SCALE
    // the tile's mirror image is another one, unless it is inside a diagonal block
    __device__ __forceinline__ bool mirrored(const GemmUnit& q, int j0) const { return j0 < q.row0; }
    __device__ __forceinline__ void operator()(const GemmUnit& q, long long i, int j0, int cols, float* sum,
                                               const unsigned char* in, unsigned char* out) const {
        float v[32];
        if (in) pair_load(in, v);
#pragma unroll
        for (int k = 0; k < 32; k++) sum[k] = in ? fmaf(b, v[k], c * sum[k]) : c * sum[k];
        __half h[32], l[32];
        split(sum, h, l);
        slot_store(out, reinterpret_cast<const uint32_t*>(h));
        slot_store(out + GEMM_PLANE, reinterpret_cast<const uint32_t*>(l));
    }
    __device__ __forceinline__ void turn(const float* v, unsigned char* out) const {
        __half h[32], l[32];
        split(v, h, l);
        const int lane = threadIdx.x % 32;
#pragma unroll
        for (int k = 0; k < 32; k++) {
            const int at = slot_at(k, lane >> 3) + (lane & 7) * 2;
            *reinterpret_cast<__half*>(out + at) = h[k];
            *reinterpret_cast<__half*>(out + GEMM_PLANE + at) = l[k];
        }
    }
};

// a X + sum; i along the rows of X, j along its columns.
template <int F>
struct StepEpi {
    static constexpr int PLANES = 2, SLOTS = 1, WARPS = 8, FLUSH = F;
    static constexpr bool MIRROR = false;
    __device__ __forceinline__ void operator()(const GemmUnit&, long long, int, int, const float* sum,
                                               const unsigned char* in, unsigned char* out) const {
        float v[32];
        pair_load(in, v);
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] = fmaf(NS_A, v[k], sum[k] * (1.0f / SCALE));
        __half h[32], l[32];
        split(v, h, l);
        slot_store(out, reinterpret_cast<const uint32_t*>(h));
        slot_store(out + GEMM_PLANE, reinterpret_cast<const uint32_t*>(l));
    }
};

// The last a X + sum, into the weights or the result.
template <int F>
struct LastEpi {
    static constexpr int PLANES = 2, SLOTS = 1, WARPS = 8, FLUSH = F;
    static constexpr bool MIRROR = false;
    Problem q;
    template <class T>
    __device__ __forceinline__ static void write(const View& o, long long at, long long stride, int n, const float* v) {
        T t[32];
#pragma unroll
        for (int k = 0; k < 32; k++) t[k] = from_f32<T>(v[k]);
        store32((T*)o.p + at, stride, n, t);
    }
    __device__ __forceinline__ static void write(const View& o, int dtype, long long at, long long stride, int n,
                                                 const float* v) {
        if (dtype == PHYZB_DT_F32) return write<float>(o, at, stride, n, v);
        if (dtype == PHYZB_DT_BF16) return write<__nv_bfloat16>(o, at, stride, n, v);
        return write<__half>(o, at, stride, n, v);
    }
    // n values (at SCALE) of matrix z from (r, c) along c, or down r
    __device__ __forceinline__ void finish(long long z, long long r, long long c, bool down, int n, float* v) const {
        auto at = [&](const View& o) { return z * o.zs + r * o.rs + c * o.cs; };
        auto stride = [&](const View& o) { return down ? o.rs : o.cs; };
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] *= 1.0f / SCALE;
        if (q.out.p) return write(q.out, q.out_dtype, at(q.out), stride(q.out), n, v);
        float old[32];
        float* w = (float*)q.w.p + at(q.w);
        load32(w, stride(q.w), n, old);
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] = fmaf(-q.lr, v[k], q.decay * old[k]);
        store32(w, stride(q.w), n, v);
        if (q.copy.p) write(q.copy, q.copy_dtype, at(q.copy), stride(q.copy), n, v);
    }
    __device__ __forceinline__ void operator()(const GemmUnit& u, long long i, int j0, int cols, float* sum,
                                               const unsigned char* in, unsigned char*) const {
        if (i >= q.rows) return;
        float v[32];
        pair_load(in, v);
#pragma unroll
        for (int k = 0; k < 32; k++) v[k] = fmaf(NS_A, v[k], sum[k] * (1.0f / SCALE));
        finish(u.z, i, j0, false, cols, v);
    }
};

// ── small matrices: all of it in one block ───────────────────────────────

// s <= 128 and l <= LB: X, G and P stay in shared memory as f16 pairs, the
// accumulators in Tensor Memory, and one launch does the whole update. X is
// [128 rows][l] in blocks of 64 columns, 128-byte swizzled: as it lies it is the
// operand with k along l (X X^T) and the one with k along its rows (P X). What is
// left of five iterations is latency: three products and epilogues of a microsecond
// and more each. 8 matrices of 128 x 128: 43 us; as 17 launches 104.
constexpr int SMALL_THREADS = 512;
constexpr int SMALL_BLOCK = 128 * 128;  // bytes of 128 rows of 64 values

template <int LB>
struct Small {
    static constexpr int X = LB / 64 * SMALL_BLOCK, G = 2 * SMALL_BLOCK;  // bytes of a plane
    static constexpr int BYTES = 2 * X + 2 * G + 1024 + 128;
};

// bytes of value (row, col) in a plane
__device__ __forceinline__ int small_at(int row, int col) {
    return (col >> 6) * SMALL_BLOCK + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
}
// 32 columns from c (a multiple of 32) of a lane's row
__device__ __forceinline__ void small_load(const unsigned char* hi, int lo, int row, int c, float* v) {
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            __half t[8];
            *(uint4*)t = *(const uint4*)(hi + p * lo + small_at(row, c + q * 8));
#pragma unroll
            for (int e = 0; e < 8; e++) v[q * 8 + e] = p ? v[q * 8 + e] + __half2float(t[e]) : __half2float(t[e]);
        }
}
__device__ __forceinline__ void small_store(unsigned char* hi, int lo, int row, int c, const float* v) {
    __half h[32], l[32];
    split(v, h, l);
#pragma unroll
    for (int q = 0; q < 4; q++) {
        *(uint4*)(hi + small_at(row, c + q * 8)) = *(const uint4*)(h + q * 8);
        *(uint4*)(hi + lo + small_at(row, c + q * 8)) = *(const uint4*)(l + q * 8);
    }
}
// the sum of an accumulator and its small terms
__device__ __forceinline__ void small_sum(uint32_t main, uint32_t small, float* v) {
    float w[32];
    tmem_load(main, v);
    tmem_load(small, w);
    tmem_load_wait();
#pragma unroll
    for (int e = 0; e < 32; e++) v[e] += w[e];
}

template <int LB, int V>
__global__ void __launch_bounds__(SMALL_THREADS, 1) small_kernel(const __grid_constant__ Problem q, unsigned int* fault) {
    using C = Small<LB>;
    extern __shared__ unsigned char raw[];
    __shared__ float sums[SMALL_THREADS / 32];
    unsigned char* const X = raw + (1024 - (smem_addr(raw) & 1023)) % 1024;
    unsigned char* const G = X + 2 * C::X;
    uint64_t* const bar = reinterpret_cast<uint64_t*>(G + 2 * C::G);
    uint32_t* const slot = reinterpret_cast<uint32_t*>(bar + 1);
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, z = blockIdx.x;
    const bool tall = q.rows > q.cols;
    const int s = tall ? q.cols : q.rows, l = tall ? q.rows : q.cols;
    if (tid == 0) {
        mbar_init(bar, 1);
        mbar_init_fence();
    }
    if (warp == 0) tmem_alloc<1>(slot, 512);
    // momentum and |u|^2, then X = u / |u| as pairs, zeros around it
    const int per = q.cols / V, n = per * q.rows;
    float sum = 0.0f;
#pragma unroll 4
    for (int e = tid; e < n; e += SMALL_THREADS) {
        const int r = e / per, c = (e - r * per) * V;
        float u[V];
        direction<V, true>(q, z, r, c, u);
#pragma unroll
        for (int v = 0; v < V; v++) sum = fmaf(u[v], u[v], sum);
    }
    for (int e = tid; e < 2 * C::X / 16; e += SMALL_THREADS) reinterpret_cast<uint4*>(X)[e] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[warp] = sum;
    mma_fence_before();
    __syncthreads();
    mma_fence_after();
    const uint32_t tmem = *slot;
    float norm = 0.0f;
#pragma unroll
    for (int w = 0; w < SMALL_THREADS / 32; w++) norm += sums[w];
    const float scale = SCALE / (sqrtf(norm) + NS_EPS);
#pragma unroll 4
    for (int e = tid; e < n; e += SMALL_THREADS) {
        const int r = e / per, c = (e - r * per) * V;
        float u[V];
        direction<V, false>(q, z, r, c, u);
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float x = u[v] * scale;
            const __half h = __float2half_rn(x);
            unsigned char* const at = X + (tall ? small_at(c + v, r) : small_at(r, c + v));
            *(__half*)at = h;
            *(__half*)(at + C::X) = __float2half_rn(x - __half2float(h));
        }
    }
    const int quarter = warp % 4, from = warp / 4 * 32, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)quarter * 32 << 16);
    const int ns = (s + 15) / 16 * 16, nl = (l + 15) / 16 * 16;
    constexpr uint32_t GS = 128, P = 256, PS = 384, XS = 256;  // columns: G at 0, its small terms, P's, X's small terms
    int phase = 0;
    bool ok = true;
    // D (main, small) = A B^T on pairs, K in steps of 16; then every thread waits
    auto product = [&](uint32_t main, uint32_t small, const unsigned char* A, int a_lo, const unsigned char* B, int b_lo,
                       bool b_mn, int cols, int ksteps) {
        fence_async();
        mma_fence_before();
        ok = __syncthreads_and(ok);
        mma_fence_after();
        if (!ok) return;
        if (tid == 0) {
            const uint32_t idesc = 1u << 4 | (uint32_t)b_mn << 16 | (uint32_t)(cols >> 3) << 17 | (128u >> 4) << 24;
            for (int k = 0; k < ksteps; k++)
#pragma unroll
                for (int p = 0; p < 3; p++) {  // hi hi; hi lo, lo hi
                    const uint32_t a = smem_addr(A) + (p == 2 ? a_lo : 0) + (k >> 2) * SMALL_BLOCK + (k & 3) * 32;
                    const uint32_t b = smem_addr(B) + (p == 1 ? b_lo : 0) +
                                       (b_mn ? k * 2048 : (k >> 2) * SMALL_BLOCK + (k & 3) * 32);
                    mma_f16<1>(tmem + (p ? small : main), gemm_desc(a, 0), gemm_desc(b, b_mn, SMALL_BLOCK), idesc,
                               k > 0 || p == 2);
                }
            mma_commit<1>(bar);
        }
        ok = mbar_wait(bar, phase);
        phase ^= 1;
        mma_fence_after();
    };
    for (int k = 0; k < q.steps; k++) {
        float v[32], g[32];
        product(0, GS, X, C::X, X, C::X, false, ns, (l + 15) / 16);
        if (from < ns) {
            small_sum(lanes + from, lanes + GS + from, v);
#pragma unroll
            for (int e = 0; e < 32; e++) v[e] *= 1.0f / SCALE;
            small_store(G, C::G, row, from, v);
        }
        product(P, PS, G, C::G, G, C::G, false, ns, ns / 16);
        if (from < ns) {
            small_sum(lanes + from, lanes + GS + from, g);
            small_sum(lanes + P + from, lanes + PS + from, v);
#pragma unroll
            for (int e = 0; e < 32; e++) v[e] = fmaf(NS_B / SCALE, g[e], NS_C / SCALE * v[e]);
            small_store(G, C::G, row, from, v);
        }
        product(0, XS, G, C::G, X, C::X, true, nl, ns / 16);
        for (int c = from; c < nl; c += 128) {
            small_sum(lanes + c, lanes + XS + c, v);
            small_load(X, C::X, row, c, g);
#pragma unroll
            for (int e = 0; e < 32; e++) v[e] = fmaf(NS_A, g[e], v[e] * (1.0f / SCALE));
            if (k + 1 < q.steps)
                small_store(X, C::X, row, c, v);
            else if (ok && row < s && c < l)
                LastEpi<0>{q}.finish(z, tall ? c : row, tall ? row : c, tall, l - c < 32 ? l - c : 32, v);
        }
    }
    mma_fence_before();
    __syncthreads();
    mma_fence_after();
    if (warp == 0) tmem_free<1>(tmem, 512);
    if (!ok && tid == 0) atomicAdd(fault, 1u);
}

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
        p.pitch = up(c, 16);
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

bool is_small(long long rows, long long cols) {
    const long long s = rows < cols ? rows : cols, l = rows < cols ? cols : rows;
    return s <= 128 && l <= 256;
}

template <int LB, int V>
cudaError_t run_small(const Problem& q, unsigned int* fault, cudaStream_t st) {
    auto kernel = small_kernel<LB, V>;
    static SmemOnce once;
    const cudaError_t e = once.smem(kernel, Small<LB>::BYTES);
    if (e != cudaSuccess) return e;
    kernel<<<q.batch, SMALL_THREADS, Small<LB>::BYTES, st>>>(q, fault);
    return cudaGetLastError();
}

// D = A B^T on pairs; the epilogue reads `in` and writes `out` (either may be
// absent), pairs of D's shape.
template <class Epi>
cudaError_t multiply(const Pair& a, bool a_mn, const Pair& b, bool b_mn, long long rows, long long cols, long long k,
                     int batch, bool symmetric, const Pair& in, const Pair& out, const Epi& epi, unsigned int* fault,
                     cudaStream_t st) {
    GemmMat ma[2], mb[2];
    GemmIo io{};
    for (int h = 0; h < 2; h++) {
        ma[h] = {a.p + h * a.lo, a_mn ? 1 : a.pitch, a_mn ? a.pitch : 1, a.zs};
        mb[h] = {b.p + h * b.lo, b_mn ? 1 : b.pitch, b_mn ? b.pitch : 1, b.zs};
        if (in.p && !gemm_io_map(&io.in[h], in.p + h * in.lo, in.pitch, 1, in.zs, rows, cols, batch, false))
            return cudaErrorInvalidValue;
        if (out.p && !gemm_io_map(&io.out[h], out.p + h * out.lo, out.pitch, 1, out.zs, rows, cols, batch, false))
            return cudaErrorInvalidValue;
    }
    io.reads = in.p != nullptr;
    io.writes = out.p != nullptr;
    const GemmCut cut = gemm_cut(rows, cols, k, batch, 3, symmetric, false, Epi::FLUSH > 0);
    return gemm_launch<2>(ma, mb, rows, cols, k, batch, cut, symmetric, false, io, epi, fault, st);
}

template <int F>
cudaError_t solve(const Problem& q, char* ws, cudaStream_t st) {
    unsigned int* fault = fault_word();
    if (!fault) return cudaErrorInvalidSymbol;
    auto wide = [&](const View& v, int e) {
        return !v.p || ((uintptr_t)v.p % (4 * e) == 0 && v.cs == 1 && v.rs % 4 == 0 && (q.batch == 1 || v.zs % 4 == 0));
    };
    const bool by4 = q.cols % 4 == 0 && wide(q.g, q.dtype == PHYZB_DT_F32 ? 4 : 2) && wide(q.m, 4);
    if (is_small(q.rows, q.cols)) {
        const bool narrow = q.rows <= 128 && q.cols <= 128;
        if (by4) return narrow ? run_small<128, 4>(q, fault, st) : run_small<256, 4>(q, fault, st);
        return narrow ? run_small<128, 1>(q, fault, st) : run_small<256, 1>(q, fault, st);
    }
    Ws o = layout(q.batch, q.rows, q.cols);
    o.x.p = (__half*)(ws + o.x_at);
    o.y.p = (__half*)(ws + o.y_at);
    o.g.p = (__half*)(ws + o.g_at);
    o.p.p = (__half*)(ws + o.p_at);
    float* part = (float*)(ws + o.part_at);
    const bool tall = q.rows > q.cols;
    const int s = tall ? q.cols : q.rows, l = tall ? q.rows : q.cols;
    // blocks of a few stretches, at most NORM_BLOCKS
    const long long stretches = q.rows * ((q.cols + (by4 ? 1023 : 255)) / (by4 ? 1024 : 256));
    const dim3 grid((unsigned)(stretches < NORM_BLOCKS ? stretches : NORM_BLOCKS), (unsigned)q.batch);
    if (by4) {
        momentum_kernel<4><<<grid, 256, 0, st>>>(q, part);
        normalize_kernel<4><<<grid, 256, 0, st>>>(q, part, o.x);
    } else {
        momentum_kernel<1><<<grid, 256, 0, st>>>(q, part);
        normalize_kernel<1><<<grid, 256, 0, st>>>(q, part, o.x);
    }
    cudaError_t e = cudaGetLastError();
    Pair x = o.x, y = o.y;
    for (int k = 0; k < q.steps && e == cudaSuccess; k++) {
        // G: the short side's products along the long one
        e = multiply(x, tall, x, tall, s, s, l, q.batch, true, Pair{}, o.g, SquareEpi<F>{0.0f, 1.0f / SCALE}, fault, st);
        if (e != cudaSuccess) break;
        e = multiply(o.g, false, o.g, false, s, s, s, q.batch, true, o.g, o.p, SquareEpi<F>{NS_B, NS_C / SCALE}, fault, st);
        if (e != cudaSuccess) break;
        // i = rows of X, j = columns. Wide: P's rows by X^T's; tall: X's rows by P's
        const Pair &a = tall ? x : o.p, &b = tall ? o.p : x;
        if (k + 1 < q.steps)
            e = multiply(a, false, b, !tall, q.rows, q.cols, s, q.batch, false, x, y, StepEpi<F>{}, fault, st);
        else
            e = multiply(a, false, b, !tall, q.rows, q.cols, s, q.batch, false, x, Pair{}, LastEpi<F>{q}, fault, st);
        const Pair t = x;
        x = y;
        y = t;
    }
    return e;
}

View view(const void* p, const int64_t* st) { return {(void*)p, st[0], st[1], st[2]}; }

}  // namespace

long long muon_workspace(const phyzb_muon_args& a) {
    return is_small(a.rows, a.cols) ? 0 : layout(a.batch, a.rows, a.cols).total;
}

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
    return solve<0>(q, (char*)ws, s);
}

long long orthogonalize_workspace(const phyzb_orthogonalize_args& a) {
    return is_small(a.rows, a.cols) ? 0 : layout(a.batch, a.rows, a.cols).total;
}

cudaError_t orthogonalize(const phyzb_orthogonalize_args& a, void* ws, cudaStream_t s) {
    Problem q{};
    q.batch = (int)a.batch;
    q.rows = (int)a.rows;
    q.cols = (int)a.cols;
    q.steps = a.steps;
    q.g = view(a.x, a.x_stride);
    q.out = view(a.out, a.out_stride);
    q.dtype = q.out_dtype = a.dtype;
    return solve<2>(q, (char*)ws, s);
}

cudaError_t muon_faults(unsigned int* n) { return cudaMemcpyFromSymbol(n, g_muon_fault, sizeof(*n)); }

}  // namespace pz
