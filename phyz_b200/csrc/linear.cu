// The linear layer y = act(x w^T + b) + r and its gradients.
//
// Forward: one product with everything else in its epilogue. Backward: dz =
// dy act'(z) and its column sums (db) in one pass, then dx = dz w and dw =
// dz^T x, the long sum of dw over the rows cut into splits that fill the GPU.
// In the epilogue of a product D[i][j] a lane has 32 neighbours in j, a warp 32 in
// i: j is the contiguous side of the result where a lane can take its neighbours
// by 16 or 32 bytes, else i is.
//
// Three ways to multiply:
//   rows_kernel       a few rows (serving): the weights go by once, on the FMA
//                     units, a warp to a feature.
//   gemm.cuh          tensor cores, bf16 and f16 as they are, f32 as three bf16
//                     planes.
//   simt_gemm.cuh     f32 on the FMA units, where the layer is small.
// Operands that TMA cannot address (odd strides, odd bases) and f32 planes are
// written to the workspace first, in the order in which they are.
#include <type_traits>

#include "gemm.cuh"
#include "simt_gemm.cuh"

namespace pz {

namespace {

__device__ unsigned int g_linear_fault;  // waits that ran out (pz_tma.cuh)

unsigned int* fault_word() {
    static FaultWord word;
    return word.get(g_linear_fault);
}

long long up(long long v, long long to = 256) { return (v + to - 1) / to * to; }
long long esize(int dtype) { return dtype == PHYZB_DT_F32 ? 4 : 2; }

// ── epilogues ─────────────────────────────────────────────────────────────

// An array seen from D: element (i, j) at p[i * is + j * js].
template <class T>
struct Out {
    T* p = nullptr;
    long long is = 0, js = 0;
};

// four neighbours along the contiguous side, in one access where they are
// aligned
template <class T>
__device__ __forceinline__ bool whole4(const T* p, long long stride, int n) {
    return n == 4 && stride == 1 && ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0;
}
__device__ __forceinline__ void load4(const float* p, long long stride, int n, float* v) {
    if (whole4(p, stride, n)) {
        *(float4*)v = *(const float4*)p;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = e < n ? p[e * stride] : 0.0f;
    }
}
__device__ __forceinline__ void store4(float* p, long long stride, int n, const float* v) {
    if (whole4(p, stride, n)) {
        *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < n) p[e * stride] = v[e];
    }
}

// 16-bit results go through slots where TMA can address them; f32 ones are few
// beside their six products, and go straight.
template <class T>
struct Slotted {
    static constexpr int PLANES = sizeof(T) == 2 ? 1 : 0, SLOTS = sizeof(T) == 2 ? 2 : 0;
    static constexpr int WARPS = sizeof(T) == 2 ? 16 : 8, FLUSH = 4;
    static constexpr bool MIRROR = false;
};

template <class T>
struct LinearEpi : Slotted<T> {
    const float* bias;
    int by_i;  // bias along i
    int act;
    Out<const T> res;
    Out<T> y, pre;
    long long m;  // rows of D

    __device__ __forceinline__ void one(long long i, long long j, float z) const {
        if (bias) z += bias[by_i ? i : j];
        if (pre.p) pre.p[i * pre.is + j * pre.js] = from_f32<T>(z);
        float v = z, unused = 0.0f;
        with_act(act, [&](auto kind) { act_pair<decltype(kind)::value>(v, unused); });
        if (res.p) v += to_f32(res.p[i * res.is + j * res.js]);
        y.p[i * y.is + j * y.js] = from_f32<T>(v);
    }
    // f once with the activation as a constant
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        with_act(act, f);
    }
    template <class K>
    __device__ __forceinline__ void four(K, int, long long i, long long j, const float* sum, int n, bool along_i) const {
        if constexpr (sizeof(T) == 4) {
            float z[4], r[4] = {};
            if (bias) {
                const bool runs = (by_i != 0) == along_i;  // along with the four values
                const float* p = bias + (by_i ? i : j);
#pragma unroll
                for (int e = 0; e < 4; e++) z[e] = sum[e] + (e < n ? p[runs ? e : 0] : 0.0f);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) z[e] = sum[e];
            }
            if (pre.p) store4(pre.p + i * pre.is + j * pre.js, along_i ? pre.is : pre.js, n, z);
            if (res.p) load4(res.p + i * res.is + j * res.js, along_i ? res.is : res.js, n, r);
#pragma unroll
            for (int e = 0; e < 4; e += 2) act_pair<K::value>(z[e], z[e + 1]);
#pragma unroll
            for (int e = 0; e < 4; e++) z[e] += r[e];
            store4(y.p + i * y.is + j * y.js, along_i ? y.is : y.js, n, z);
        }
    }
    __device__ __forceinline__ void operator()(const GemmUnit&, long long i, int j0, int cols, float* z,
                                               const unsigned char* in, unsigned char* out) const {
        if (i >= m) return;
        uint32_t w[8 * sizeof(T)];  // 32 values
        if (bias) {
            if (by_i) {
                const float b = bias[i];
#pragma unroll
                for (int c = 0; c < 32; c++) z[c] += b;
            } else {
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    float b[8];
                    load8(bias + j0 + c, cols - c, b);
#pragma unroll
                    for (int e = 0; e < 8; e++) z[c + e] += b[e];
                }
            }
        }
        if (pre.p) {
            pack32(z, w, T());
            store32(pre.p + i * pre.is + j0 * pre.js, pre.js, cols, reinterpret_cast<const T*>(w));
        }
        with_act(act, [&](auto kind) {
#pragma unroll
            for (int c = 0; c < 32; c += 2) act_pair<decltype(kind)::value>(z[c], z[c + 1]);
        });
        if (res.p) {  // (the residual may be y itself: a lane's are read before they are written)
            if (in)
                slot_load(in, w);
            else
                load32(res.p + i * res.is + j0 * res.js, res.js, cols, reinterpret_cast<T*>(w));
            add32(w, z, T());
        }
        pack32(z, w, T());
        if (out)
            slot_store(out, w);
        else
            store32(y.p + i * y.is + j0 * y.js, y.js, cols, reinterpret_cast<const T*>(w));
    }
};

template <class T>
struct StoreEpi : Slotted<T> {
    Out<T> out;
    long long m;
    __device__ __forceinline__ void one(long long i, long long j, float v) const {
        out.p[i * out.is + j * out.js] = from_f32<T>(v);
    }
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        f(0);
    }
    __device__ __forceinline__ void four(int, int, long long i, long long j, const float* v, int n, bool along_i) const {
        if constexpr (sizeof(T) == 4) store4(out.p + i * out.is + j * out.js, along_i ? out.is : out.js, n, v);
    }
    __device__ __forceinline__ void operator()(const GemmUnit&, long long i, int j0, int cols, const float* v,
                                               const unsigned char*, unsigned char* slot) const {
        if (i >= m) return;
        uint32_t w[8 * sizeof(T)];
        pack32(v, w, T());
        if (slot)
            slot_store(slot, w);
        else
            store32(out.p + i * out.is + j0 * out.js, out.js, cols, reinterpret_cast<const T*>(w));
    }
};

template <class T>
StoreEpi<T> store_epi(const Out<T>& out, long long m) {
    StoreEpi<T> e;
    e.out = out;
    e.m = m;
    return e;
}

// The slots' side of an epilogue for D [rows][cols].
template <class T>
GemmIo io_of(const LinearEpi<T>& e, long long rows, long long cols) {
    GemmIo io{};
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    if constexpr (sizeof(T) == 2) {
        io.writes = gemm_io_map(&io.out[0], e.y.p, e.y.is, e.y.js, 0, rows, cols, 1, bf16);
        io.reads = e.res.p && gemm_io_map(&io.in[0], e.res.p, e.res.is, e.res.js, 0, rows, cols, 1, bf16);
    }
    return io;
}
template <class T>
GemmIo io_of(const StoreEpi<T>& e, long long rows, long long cols) {
    GemmIo io{};
    if constexpr (sizeof(T) == 2)
        io.writes = gemm_io_map(&io.out[0], e.out.p, e.out.is, e.out.js, 0, rows, cols, 1, !std::is_same<T, __half>::value);
    return io;
}

// A split's part, [split][m][n] f32.
struct PartEpi : Slotted<float> {
    float* part;
    long long m, n;
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        f(0);
    }
    __device__ __forceinline__ void four(int, int split, long long i, long long j, const float* v, int k, bool along_i) const {
        store4(part + (split * m + i) * n + j, along_i ? n : 1, k, v);
    }
    __device__ __forceinline__ void operator()(const GemmUnit& q, long long i, int j0, int cols, const float* v,
                                               const unsigned char*, unsigned char*) const {
        if (i < m) store32(part + (q.split * m + i) * n + j0, 1, cols, v);
    }
};

inline GemmIo io_of(const PartEpi&, long long, long long) { return {}; }

// The parts in order, through the epilogue; threads along D's contiguous side.
template <class Epi>
__global__ void __launch_bounds__(256) join_kernel(const float* part, int splits, long long m, long long n, Epi epi) {
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    if (e >= m * n) return;
    float v = 0.0f;
#pragma unroll 8
    for (int s = 0; s < splits; s++) v += part[s * m * n + e];
    epi.one(e / n, e % n, v);
}

// ── operands ──────────────────────────────────────────────────────────────

// x as three bf16 terms that sum to it to 2^-24 (each the nearest to what is
// left). What is past bf16's range towards infinity is cut, not rounded up; an
// infinity or a NaN is in the first term alone.
__device__ __forceinline__ void planes_of(float x, __nv_bfloat16* p) {
    float left = x;
#pragma unroll
    for (int k = 0; k < 3; k++) {
        p[k] = __float2bfloat16_rn(left);
        if (isinf(__bfloat162float(p[k])) && !isinf(left)) p[k] = __float2bfloat16_rz(left);
        left = isfinite(left) ? left - __bfloat162float(p[k]) : 0.0f;
    }
}

// rows x k values into 16-bit planes [outer][pitch], in the order of src: inner is
// the side that is contiguous there. A thread takes two neighbours, the threads go
// through all pairs (I: an index type that holds their number). 120613 x 248 f32,
// 300 MB, 69 us (4.4 TB/s).
template <class T, class I>
__global__ void __launch_bounds__(256) pack_kernel(const T* src, long long os, long long is, I outer, I inner, I pitch,
                                                   uint32_t* dst, long long plane) {
    const I pairs = pitch / 2, n = outer * pairs, step = (I)gridDim.x * 256;
#pragma unroll 4
    for (I e = (I)blockIdx.x * 256 + threadIdx.x; e < n; e += step) {
        const I o = e / pairs, i = (e - o * pairs) * 2;
        const T* p = src + o * os + i * is;
        T v[2] = {from_f32<T>(0.0f), from_f32<T>(0.0f)};
        if (i < inner) v[0] = p[0];
        if (i + 1 < inner) v[1] = p[is];
        if constexpr (sizeof(T) == 2) {
            dst[e] = *reinterpret_cast<const uint32_t*>(v);
        } else {
            __nv_bfloat16 x[3], y[3];
            planes_of(v[0], x);
            planes_of(v[1], y);
#pragma unroll
            for (int k = 0; k < 3; k++) {
                const __nv_bfloat162 w = __halves2bfloat162(x[k], y[k]);
                dst[k * (plane / 2) + e] = *reinterpret_cast<const uint32_t*>(&w);
            }
        }
    }
}

// An operand of a tensor-core product: where it is, and whether it has to be
// packed first (f32 always).
struct Operand {
    GemmMat mat;  // as given; element strides
    long long rows, k;
    int dtype;
    bool pack;
    long long pitch, plane, bytes;

    Operand(const void* p, long long rs, long long ks, long long rows, long long k, int dtype)
        : mat{p, rs, ks, 0}, rows(rows), k(k), dtype(dtype) {
        pack = dtype == PHYZB_DT_F32 || !gemm_tma_ok(mat, rows, k, 1);
        const bool mn = gemm_mn(mat, k);
        pitch = up(mn ? rows : k, 8);
        plane = up(pitch * (mn ? k : rows), 128);
        bytes = pack ? plane * 2 * (dtype == PHYZB_DT_F32 ? 3 : 1) : 0;
    }
    // the planes, packed into ws where need be
    cudaError_t ready(char* ws, GemmMat* out, cudaStream_t st) const {
        if (!pack) {
            out[0] = mat;
            return cudaSuccess;
        }
        const bool mn = gemm_mn(mat, k);
        const long long outer = mn ? k : rows, inner = mn ? rows : k, os = mn ? mat.ks : mat.rs, is = mn ? 1 : mat.ks;
        const long long n = outer * (pitch / 2), blocks = (n + 1023) / 1024;
        const unsigned grid = (unsigned)(blocks < 16 * GEMM_SMS ? blocks : 16 * GEMM_SMS);
        auto run = [&](auto* src) {
            using T = std::remove_const_t<std::remove_pointer_t<decltype(src)>>;
            if (n < 1ll << 31)
                pack_kernel<T, uint32_t><<<grid, 256, 0, st>>>(src, os, is, (uint32_t)outer, (uint32_t)inner,
                                                               (uint32_t)pitch, (uint32_t*)ws, plane);
            else
                pack_kernel<T, long long><<<grid, 256, 0, st>>>(src, os, is, outer, inner, pitch, (uint32_t*)ws, plane);
        };
        if (dtype == PHYZB_DT_F32)
            run((const float*)mat.p);
        else
            run((const __half*)mat.p);
        for (int p = 0; p < (dtype == PHYZB_DT_F32 ? 3 : 1); p++)
            out[p] = {ws + p * plane * 2, mn ? 1 : pitch, mn ? pitch : 1, 0};
        return cudaGetLastError();
    }
};

// ── tensor-core products ──────────────────────────────────────────────────

using Cut = GemmCut;
Cut cut_of(long long rows, long long cols, long long k, bool f32) {
    return gemm_cut(rows, cols, k, 1, f32 ? 6 : 1, false, true, f32);
}

long long part_bytes(const Cut& c, long long rows, long long cols) {
    return c.splits > 1 ? up(c.splits * rows * cols * 4) : 0;
}

// T's planes: three for f32, else the values themselves.
template <class T, class Epi>
cudaError_t multiply_cut(const GemmMat* a, const GemmMat* b, long long rows, long long cols, long long k, const Cut& c,
                         const Epi& epi, cudaStream_t st) {
    unsigned int* fault = fault_word();
    if (!fault) return cudaErrorInvalidSymbol;
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    constexpr int PL = sizeof(T) == 4 ? 3 : 1;
    return gemm_launch<PL>(a, b, rows, cols, k, 1, c, false, bf16, io_of(epi, rows, cols), epi, fault, st);
}

// D = A B^T through `epi`; part: room for the splits' parts.
template <class T, class Epi>
cudaError_t multiply(const GemmMat* a, const GemmMat* b, long long rows, long long cols, long long k, const Cut& c,
                     char* part, const Epi& epi, cudaStream_t st) {
    if (c.splits == 1) return multiply_cut<T>(a, b, rows, cols, k, c, epi, st);
    const cudaError_t e = multiply_cut<T>(a, b, rows, cols, k, c, PartEpi{{}, (float*)part, rows, cols}, st);
    if (e != cudaSuccess) return e;
    join_kernel<<<(unsigned)((rows * cols + 255) / 256), 256, 0, st>>>((const float*)part, c.splits, rows, cols, epi);
    return cudaGetLastError();
}

// ── f32 on the FMA units ──────────────────────────────────────────────────

// Rough times of both ways in microseconds: the FMA units at 25 TFLOP/s; the
// tensor cores at 200 (six products) behind two packing launches that move ten
// bytes a value at 4 TB/s.
bool simt_is_faster(double rows, double cols, double k) {
    const double flop = 2e-6 * rows * cols * k;
    return flop / 25.0 < flop / 200.0 + 10e-6 * (rows + cols) * k / 4.0 + 12.0;
}

// Splits of k so that the 128 x 64 tiles are two to an SM, each of 256 at least.
int simt_splits(long long rows, long long cols, long long k) {
    const long long tiles = ((rows + 127) / 128) * ((cols + 63) / 64);
    if (tiles >= GEMM_SMS / 2) return 1;
    long long s = 2 * GEMM_SMS / tiles;
    if (s > k / 256) s = k / 256;
    return s < 2 ? 1 : (int)s;
}

// Whether a result [i][j] is contiguous in i: lanes then run along i, else along j.
bool along_i_of(const int64_t* stride) { return stride[1] != 1 && stride[0] == 1; }

template <class Epi>
cudaError_t simt_multiply(const SimtOperand& a, const SimtOperand& b, long long rows, long long cols, long long k,
                          int splits, bool along_i, char* part, const Epi& epi, cudaStream_t st) {
    if (splits == 1) return simt_gemm(a, b, rows, cols, k, 1, along_i, epi, st);
    const cudaError_t e = simt_gemm(a, b, rows, cols, k, splits, false, PartEpi{{}, (float*)part, rows, cols}, st);
    if (e != cudaSuccess) return e;
    join_kernel<<<(unsigned)((rows * cols + 255) / 256), 256, 0, st>>>((const float*)part, splits, rows, cols, epi);
    return cudaGetLastError();
}

// ── a few rows ────────────────────────────────────────────────────────────

constexpr int FEW = 8;

// Bound by the weights' bytes, or by latency: one row of 512 to 1024 features, 1 MB
// of bf16 weights, 2.7 us. A warp takes a feature: its weights once, 16 bytes a lane
// where V > 1, against M rows of x (which stay in the caches), sums in f32, joined
// by shuffles; lane r finishes row r.
template <class T, int M, int V>
__global__ void __launch_bounds__(128) rows_kernel(const __grid_constant__ phyzb_linear_args a, LinearEpi<T> epi) {
    const int lane = threadIdx.x % 32;
    const long long n = (long long)blockIdx.x * 4 + threadIdx.x / 32;
    if (n >= a.n) return;
    const T* w = (const T*)a.w + n * a.w_stride[0];
    const T* x = (const T*)a.x;
    float sum[M] = {};
#pragma unroll 4
    for (long long k = lane * V; k < a.k; k += 32 * V) {
        T wv[V];
        if constexpr (V > 1) {
            *reinterpret_cast<uint4*>(wv) = *reinterpret_cast<const uint4*>(w + k);
        } else {
            wv[0] = w[k * a.w_stride[1]];
        }
#pragma unroll
        for (int r = 0; r < M; r++) {
            if (r >= a.m) break;
            T xv[V];
            if constexpr (V > 1) {
                *reinterpret_cast<uint4*>(xv) = *reinterpret_cast<const uint4*>(x + r * a.x_stride[0] + k);
            } else {
                xv[0] = x[r * a.x_stride[0] + k * a.x_stride[1]];
            }
#pragma unroll
            for (int v = 0; v < V; v++) sum[r] = fmaf(to_f32(wv[v]), to_f32(xv[v]), sum[r]);
        }
    }
    float mine = 0.0f;
#pragma unroll
    for (int r = 0; r < M; r++) {
#pragma unroll
        for (int o = 16; o; o /= 2) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], o);
        if (lane == r) mine = sum[r];
    }
    if (lane < a.m) epi.one(n, lane, mine);
}

template <class T>
bool rows_wide(const phyzb_linear_args& a) {
    const int v = 16 / (int)sizeof(T);
    return a.k % v == 0 && a.w_stride[1] == 1 && a.x_stride[1] == 1 && (uintptr_t)a.w % 16 == 0 &&
           (uintptr_t)a.x % 16 == 0 && (a.n == 1 || a.w_stride[0] % v == 0) && (a.m == 1 || a.x_stride[0] % v == 0);
}

// ── forward ───────────────────────────────────────────────────────────────

enum Way { ROWS, SIMT, TENSOR };

Way way_of(const phyzb_linear_args& a) {
    // (a warp's lanes walk k: weights with n contiguous would be read a sector a value)
    if (a.m <= FEW && (a.w_stride[1] == 1 || a.k == 1)) return ROWS;
    return a.dtype == PHYZB_DT_F32 && simt_is_faster((double)a.m, (double)a.n, (double)a.k) ? SIMT : TENSOR;
}

// Whether D's i should be the first index of a result [r][c] (see above).
bool first_is_i(const void* p, const int64_t* stride, int e) {
    auto wide = [&](int64_t other) { return (uintptr_t)p % 16 == 0 && other * e % 16 == 0; };
    if (stride[1] == 1) return wide(stride[0]);
    if (stride[0] == 1) return !wide(stride[1]);
    return true;
}

// A tile is 128 along i: up to 64 rows are left to j, whose tiles can be 64.
bool rows_are_i(long long m, const void* p, const int64_t* stride, int dtype) {
    return m > 64 && first_is_i(p, stride, (int)esize(dtype));
}

struct Forward {
    bool rows_first;  // i = rows of x
    long long di, dj;
    Operand x, w;
    Cut cut;
    long long ws_x, ws_w, ws_part, total;
    explicit Forward(const phyzb_linear_args& a)
        : rows_first(rows_are_i(a.m, a.y, a.y_stride, a.dtype)),
          di(rows_first ? a.m : a.n),
          dj(rows_first ? a.n : a.m),
          x(a.x, a.x_stride[0], a.x_stride[1], a.m, a.k, a.dtype),
          w(a.w, a.w_stride[0], a.w_stride[1], a.n, a.k, a.dtype),
          cut(cut_of(di, dj, a.k, a.dtype == PHYZB_DT_F32)) {
        ws_x = 0;
        ws_w = up(x.bytes);
        ws_part = ws_w + up(w.bytes);
        total = ws_part + part_bytes(cut, di, dj);
    }
};

template <class T>
LinearEpi<T> epilogue(const phyzb_linear_args& a, bool rows_first) {
    auto turn = [&](auto* p, const int64_t* s) {
        return Out<std::remove_pointer_t<decltype(p)>>{p, rows_first ? s[0] : s[1], rows_first ? s[1] : s[0]};
    };
    return {{}, a.bias, !rows_first, a.activation, turn((const T*)a.residual, a.residual_stride), turn((T*)a.y, a.y_stride),
            turn((T*)a.pre, a.pre_stride), rows_first ? a.m : a.n};
}

template <class T>
cudaError_t forward(const phyzb_linear_args& a, char* ws, cudaStream_t st) {
    const Way way = way_of(a);
    if (way == ROWS) {
        const LinearEpi<T> epi = epilogue<T>(a, false);
        const unsigned grid = (unsigned)((a.n + 3) / 4);
        constexpr int V = 16 / sizeof(T);
        const bool wide = rows_wide<T>(a);
        auto run = [&](auto m) {
            constexpr int M = decltype(m)::value;
            if (wide)
                rows_kernel<T, M, V><<<grid, 128, 0, st>>>(a, epi);
            else
                rows_kernel<T, M, 1><<<grid, 128, 0, st>>>(a, epi);
            return cudaGetLastError();
        };
        if (a.m == 1) return run(std::integral_constant<int, 1>());
        if (a.m <= 4) return run(std::integral_constant<int, 4>());
        return run(std::integral_constant<int, FEW>());
    }
    if constexpr (sizeof(T) == 4) {
        if (way == SIMT) {
            // (i = rows here; the epilogue takes either order)
            return simt_multiply({(const float*)a.x, a.x_stride[0], a.x_stride[1]},
                                 {(const float*)a.w, a.w_stride[0], a.w_stride[1]}, a.m, a.n, a.k,
                                 simt_splits(a.m, a.n, a.k), along_i_of(a.y_stride), ws, epilogue<T>(a, true), st);
        }
    }
    const Forward f(a);
    GemmMat x[3], w[3];
    cudaError_t e = f.x.ready(ws + f.ws_x, x, st);
    if (e == cudaSuccess) e = f.w.ready(ws + f.ws_w, w, st);
    if (e != cudaSuccess) return e;
    return multiply<T>(f.rows_first ? x : w, f.rows_first ? w : x, f.di, f.dj, a.k, f.cut, ws + f.ws_part,
                    epilogue<T>(a, f.rows_first), st);
}

// ── backward ──────────────────────────────────────────────────────────────

// dz = dy act'(pre) in dy's order (inner: its contiguous side; the rows, where pre
// has another order than dy), and the sums of
// the unrounded dz over the rows: each block's part to part[block][n]. dz
// [outer][pitch]: T, or three bf16 planes. dz or part may be null.
//
// A 16-bit layer's dz is rounded to its type, as the tensor cores take it: dy, which it
// is made of, has no more bits, and a second plane would double both products. It is
// most of what a gradient is off by beyond its own rounding (bf16 65536 x 1024 x 1024:
// 2.3e-3 to 64 bits, 1.7e-3 with an unrounded dz; f16 2.9e-4, 2.1e-4). In f16 a dz
// under 2^-25 is lost, which is the half of dy's own last place.
struct DzArgs {
    const void *dy, *pre;
    long long dy_o, dy_i, pre_o, pre_i;  // strides along outer and inner
    long long outer, inner, pitch, plane;
    void* dz;
    float* part;
    int act, planes;
    int lines;  // outer lines of a block
};
constexpr int DZ_OUTER = 128;   // outer lines of a block, at most
constexpr int DZ_TURNED = 512;  // the same, where one operand is turned
constexpr int DZ_INNER = 2048;  // inner values of a block, where it sums along them

// (at: o * pitch + i)
template <class T>
__device__ __forceinline__ void dz_store(const DzArgs& a, long long at, float v) {
    if (!a.dz) return;
    if (sizeof(T) == 4 && a.planes == 3) {
        __nv_bfloat16 p[3];
        planes_of(v, p);
#pragma unroll
        for (int k = 0; k < 3; k++) ((__nv_bfloat16*)a.dz)[k * a.plane + at] = p[k];
    } else {
        ((T*)a.dz)[at] = from_f32<T>(v);
    }
}

// inner = features. V neighbours per thread, 256 threads = 32 along the features
// x 8 rows. Bound by memory, and by the slope's instructions: 65536 x 1024 bf16
// with gelu, 403 MB, 90 us (4.5 TB/s; tanh and silu 15 less).
template <class T, int V>
__global__ void __launch_bounds__(256, 4) dz_rows_kernel(const __grid_constant__ DzArgs a) {
    __shared__ float sums[8][32 * V];
    const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    const long long i0 = ((long long)blockIdx.x * 32 + tx) * V;
    const long long o0 = blockIdx.y * (long long)a.lines, o1 = o0 + a.lines < a.outer ? o0 + a.lines : a.outer;
    float sum[V] = {};
    with_act(a.act, [&](auto kind) {
        if (i0 >= a.inner) return;
        constexpr int ACT = decltype(kind)::value;
#pragma unroll 2
        for (long long o = o0 + ty; o < o1; o += 8) {
            T d[V], z[V], out[V];
            const T *pd = (const T*)a.dy + o * a.dy_o + i0 * a.dy_i, *pz = (const T*)a.pre + o * a.pre_o + i0 * a.pre_i;
            if constexpr (V > 1) {
                *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(pd);
                if (ACT != PHYZB_ACT_NONE) *reinterpret_cast<uint4*>(z) = *reinterpret_cast<const uint4*>(pz);
            } else {
                d[0] = *pd;
                if (ACT != PHYZB_ACT_NONE) z[0] = *pz;
            }
            float v[V];
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const int f = V > 1 ? e + 1 : 0;
                v[e] = to_f32(d[e]);
                v[f] = to_f32(d[f]);
                if (ACT != PHYZB_ACT_NONE) {
                    float p = to_f32(z[e]), q = to_f32(z[f]);
                    act_grad_pair<ACT>(p, q);
                    v[e] *= p;
                    if (V > 1) v[f] *= q;
                }
            }
#pragma unroll
            for (int e = 0; e < V; e++) {
                sum[e] += v[e];
                out[e] = from_f32<T>(v[e]);
            }
            if (!a.dz) continue;
            if (sizeof(T) == 4 && a.planes == 3) {
#pragma unroll
                for (int e = 0; e < V; e++) dz_store<T>(a, o * a.pitch + i0 + e, v[e]);
            } else if constexpr (V > 1) {
                *reinterpret_cast<uint4*>((T*)a.dz + o * a.pitch + i0) = *reinterpret_cast<const uint4*>(out);
            } else {
                ((T*)a.dz)[o * a.pitch + i0] = out[0];
            }
        }
    });
    if (!a.part) return;
#pragma unroll
    for (int e = 0; e < V; e++) sums[ty][tx * V + e] = sum[e];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * V; c += 256) {
        float s = 0.0f;
#pragma unroll
        for (int r = 0; r < 8; r++) s += sums[r][c];
        const long long i = (long long)blockIdx.x * 32 * V + c;
        if (i < a.inner) a.part[blockIdx.y * a.inner + i] = s;
    }
}

// inner = rows: a block takes DZ_INNER of one feature's, V neighbours a thread. The
// same 403 MB as above in this order: 100 us (4.0 TB/s), 110 with the column sums; one
// value at a time 259.
template <class T, int V>
__global__ void __launch_bounds__(256, 4) dz_features_kernel(const __grid_constant__ DzArgs a) {
    __shared__ float sums[8];
    constexpr int GROUPS = DZ_INNER / 256 / V;
    const long long i0 = (long long)blockIdx.x * DZ_INNER + threadIdx.x * V, left = a.inner - i0;
    const int mine = (int)(left < DZ_INNER ? left : DZ_INNER);  // values from this thread's first on
    for (long long o = blockIdx.y; o < a.outer; o += gridDim.y) {
        float sum = 0.0f;
        // (contiguous: that is what makes it the inner side)
        const T *pd = (const T*)a.dy + o * a.dy_o + i0, *pz = (const T*)a.pre + o * a.pre_o + i0 * a.pre_i;
        const long long at = o * a.pitch + i0;
        with_act(a.act, [&](auto kind) {
            constexpr int ACT = decltype(kind)::value;
            T d[DZ_INNER / 256], z[DZ_INNER / 256];
#pragma unroll
            for (int g = 0; g < GROUPS; g++) {
                const int i = g * 256 * V;
                if (i >= mine) continue;  // (leaving the loop here: f32 tanh 210 us instead of 193)
                if constexpr (V > 1) {
                    *reinterpret_cast<uint4*>(d + g * V) = *reinterpret_cast<const uint4*>(pd + i);
                    if (ACT != PHYZB_ACT_NONE) *reinterpret_cast<uint4*>(z + g * V) = *reinterpret_cast<const uint4*>(pz + i);
                } else {
                    d[g] = pd[i];
                    if (ACT != PHYZB_ACT_NONE) z[g] = pz[i * a.pre_i];
                }
            }
#pragma unroll
            for (int g = 0; g < GROUPS; g++) {
                if (g * 256 * V >= mine) continue;
                float v[V];
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const int f = V > 1 ? e + 1 : 0;
                    v[e] = to_f32(d[g * V + e]);
                    v[f] = to_f32(d[g * V + f]);
                    if (ACT == PHYZB_ACT_NONE) continue;
                    float p = to_f32(z[g * V + e]), q = to_f32(z[g * V + f]);
                    act_grad_pair<ACT>(p, q);
                    v[e] *= p;
                    if (V > 1) v[f] *= q;
                }
#pragma unroll
                for (int e = 0; e < V; e++) sum += v[e];
                if (!a.dz) continue;
                if constexpr (V == 1) {
                    dz_store<T>(a, at + g * 256, v[0]);
                } else if (sizeof(T) == 4 && a.planes == 3) {
                    __nv_bfloat16 p[V][3], w[V];
#pragma unroll
                    for (int e = 0; e < V; e++) planes_of(v[e], p[e]);
#pragma unroll
                    for (int k = 0; k < 3; k++) {
#pragma unroll
                        for (int e = 0; e < V; e++) w[e] = p[e][k];
                        *reinterpret_cast<uint2*>((__nv_bfloat16*)a.dz + k * a.plane + at + g * 256 * V) =
                            *reinterpret_cast<const uint2*>(w);
                    }
                } else {
                    T out[V];
#pragma unroll
                    for (int e = 0; e < V; e++) out[e] = from_f32<T>(v[e]);
                    *reinterpret_cast<uint4*>((T*)a.dz + at + g * 256 * V) = *reinterpret_cast<const uint4*>(out);
                }
            }
        });
        if (!a.part) continue;
#pragma unroll
        for (int s = 16; s; s /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; w++) s += sums[w];
            a.part[blockIdx.x * a.outer + o] = s;
        }
        __syncthreads();
    }
}

// dy and pre in different orders: inner = rows, a block takes DZ_TURNED rows of 32
// features in tiles of 32 x 64. The operand whose features are contiguous (TDY: dy,
// else pre) is read along them and turned in shared memory; the other is read, and
// dz written, along the rows: 1320 x 34390 f16 with gelu, 272 MB, 100 us with the column
// sums (2.7 TB/s, bound by instructions and the turn); 233 where one of the two was read
// against its order. A row-major dy comes to a feature-major layer where the loss takes
// its difference from row-major targets.
template <class T, bool TDY>
__global__ void __launch_bounds__(256) dz_mixed_kernel(const __grid_constant__ DzArgs a) {
    constexpr int PITCH = 64 + 4 / sizeof(T);  // a tile's column goes to 32 different banks
    __shared__ T tile[32 * PITCH];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const long long i0 = (long long)blockIdx.x * DZ_TURNED, i1 = i0 + DZ_TURNED < a.inner ? i0 + DZ_TURNED : a.inner;
    const long long ti = TDY ? a.dy_i : a.pre_i, so = TDY ? a.pre_o : a.dy_o;
    for (long long o0 = blockIdx.y * 32ll; o0 < a.outer; o0 += gridDim.y * 32ll) {
        const int no = (int)(a.outer - o0 < 32 ? a.outer - o0 : 32);
        const T* turned = (const T*)(TDY ? a.dy : a.pre) + o0 + lane + (i0 + warp) * ti;
        const T* direct = (const T*)(TDY ? a.pre : a.dy) + (o0 + warp * 4) * so + i0 + lane;
        long long at = (o0 + warp * 4) * a.pitch + i0 + lane;
        float sum[4] = {};
        for (long long ib = i0; ib < i1; ib += 64, turned += 64 * ti, direct += 64, at += 64) {
            const int ni = (int)(i1 - ib < 64 ? i1 - ib : 64);
            T t[8], d[8];
#pragma unroll
            for (int u = 0; u < 8; u++)  // rows ib + 8 u + warp, features o0 + lane
                t[u] = u * 8 + warp < ni && lane < no ? turned[u * 8 * ti] : from_f32<T>(0.0f);
#pragma unroll
            for (int u = 0; u < 8; u++)  // features o0 + 4 warp + u / 2, rows ib + 32 (u % 2) + lane
                d[u] = u % 2 * 32 + lane < ni && warp * 4 + u / 2 < no ? direct[u / 2 * so + u % 2 * 32]
                                                                       : from_f32<T>(0.0f);
            __syncthreads();  // the last tile has been read
#pragma unroll
            for (int u = 0; u < 8; u++) tile[lane * PITCH + u * 8 + warp] = t[u];
            __syncthreads();
            float v[8], z[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const float f = to_f32(tile[(warp * 4 + u / 2) * PITCH + u % 2 * 32 + lane]), g = to_f32(d[u]);
                v[u] = TDY ? f : g;
                z[u] = TDY ? g : f;
            }
            with_act(a.act, [&](auto kind) {
#pragma unroll
                for (int u = 0; u < 8; u += 2) act_grad_pair<decltype(kind)::value>(z[u], z[u + 1]);
            });
#pragma unroll
            for (int u = 0; u < 8; u++) {
                if (u % 2 * 32 + lane >= ni || warp * 4 + u / 2 >= no) continue;
                v[u] *= z[u];
                dz_store<T>(a, at + u / 2 * a.pitch + u % 2 * 32, v[u]);
                sum[u / 2] += v[u];
            }
        }
        if (!a.part) continue;
#pragma unroll
        for (int f = 0; f < 4; f++) {
#pragma unroll
            for (int s = 16; s; s /= 2) sum[f] += __shfl_xor_sync(0xffffffffu, sum[f], s);
            const long long o = o0 + warp * 4 + f;
            if (lane == 0 && o < a.outer) a.part[blockIdx.x * a.outer + o] = sum[f];
        }
    }
}

// out[j] = sum over the blocks of part[block][j]: 32 warps take every 32nd block.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* part, long long blocks, long long n, float* out) {
    __shared__ float sums[32][33];
    const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    const long long j = (long long)blockIdx.x * 32 + tx;
    float v = 0.0f;
    if (j < n) {
#pragma unroll 8
        for (long long r = ty; r < blocks; r += 32) v += part[r * n + j];
    }
    sums[ty][tx] = v;
    __syncthreads();
    v = sums[tx][ty];  // warp ty finishes column ty
#pragma unroll
    for (int o = 16; o; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (tx == 0 && (long long)blockIdx.x * 32 + ty < n) out[(long long)blockIdx.x * 32 + ty] = v;
}

struct Backward {
    bool features;            // dy has its rows contiguous: dz is [n][m padded]
    bool simt_dx, simt_dw;    // f32 on the FMA units
    bool mixed, turn_dy;      // dy and pre in different orders; dy is the one by rows
    bool own_dz;              // dz is written (else dy is used as it is)
    int planes;               // of dz: 0 = T
    int lines;                // of a dz_rows_kernel block
    long long outer, inner, pitch, plane, blocks;
    bool dx_rows_first;       // dx: i = rows
    bool dw_n_first;          // dw: i = n
    Cut cut_dx, cut_dw;
    int split_dx, split_dw;   // of the FMA products
    long long ws_dz, ws_part, ws_w, ws_x, ws_sum, total;

    static Operand w_of(const phyzb_linear_grad_args& a) {
        return Operand(a.w, a.w_stride[1], a.w_stride[0], a.k, a.n, a.dtype);
    }
    static Operand x_of(const phyzb_linear_grad_args& a) {
        return Operand(a.x, a.x_stride[1], a.x_stride[0], a.k, a.m, a.dtype);
    }
    explicit Backward(const phyzb_linear_grad_args& a) {
        const bool f32 = a.dtype == PHYZB_DT_F32;
        const auto by_features = [&](const int64_t (&s)[2]) { return s[0] == 1 && s[1] != 1; };
        const auto by_rows = [&](const int64_t (&s)[2]) { return s[1] == 1 && s[0] != 1; };
        features = by_features(a.dy_stride) && a.m > 1;
        mixed = a.activation != PHYZB_ACT_NONE && a.m >= 32 && a.n >= 32;  // (a tile; fewer take one of the plain ways)
        turn_dy = by_rows(a.dy_stride);
        mixed = mixed && (turn_dy ? by_features(a.pre_stride) : features && by_rows(a.pre_stride));
        features = features || mixed;
        outer = features ? a.n : a.m;
        inner = features ? a.m : a.n;
        pitch = up(inner, 8);
        plane = up(pitch * outer, 128);
        // fewer lines to a block while blocks are fewer than four per SM
        lines = DZ_OUTER;
        while (outer / lines >= 65535) lines *= 2;
        while (lines > 16 && (outer + lines - 1) / lines * ((inner + 255) / 256) < 4 * GEMM_SMS) lines /= 2;
        const int along = mixed ? DZ_TURNED : DZ_INNER;
        blocks = features ? (inner + along - 1) / along : (outer + lines - 1) / lines;
        // (both products of a layer have the same size: one way serves both)
        simt_dx = simt_dw = f32 && simt_is_faster((double)a.m, (double)a.n, (double)a.k);
        planes = f32 && !simt_dx ? 3 : 0;
        const GemmMat dy{a.dy, a.dy_stride[0], a.dy_stride[1], 0}, dyt{a.dy, a.dy_stride[1], a.dy_stride[0], 0};
        own_dz = a.activation != PHYZB_ACT_NONE || planes ||
                 (!f32 && !(gemm_tma_ok(dy, a.m, a.n, 1) && gemm_tma_ok(dyt, a.n, a.m, 1)));
        dx_rows_first = rows_are_i(a.m, a.dx, a.dx_stride, a.dtype);
        dw_n_first = first_is_i(a.dw, a.dw_stride, (int)esize(a.dtype));
        cut_dx = dx_rows_first ? cut_of(a.m, a.k, a.n, f32) : cut_of(a.k, a.m, a.n, f32);
        cut_dw = dw_n_first ? cut_of(a.n, a.k, a.m, f32) : cut_of(a.k, a.n, a.m, f32);
        split_dx = simt_splits(a.m, a.k, a.n);
        split_dw = simt_splits(a.n, a.k, a.m);
        long long at = 0;
        auto take = [&](long long bytes) {
            const long long o = at;
            at += up(bytes);
            return o;
        };
        ws_dz = take(own_dz ? (planes ? 3 * plane * 2 : pitch * outer * esize(a.dtype)) : 0);
        ws_part = take(a.dbias ? blocks * a.n * 4 : 0);
        ws_w = take(a.dx && !simt_dx ? w_of(a).bytes : 0);
        ws_x = take(a.dw && !simt_dw ? x_of(a).bytes : 0);
        long long dxs = 0, dws = 0;
        if (a.dx) dxs = simt_dx ? (split_dx > 1 ? split_dx * a.m * a.k * 4 : 0) : part_bytes(cut_dx, a.m, a.k);
        if (a.dw) dws = simt_dw ? (split_dw > 1 ? split_dw * a.n * a.k * 4 : 0) : part_bytes(cut_dw, a.n, a.k);
        ws_sum = take(dxs > dws ? dxs : dws);  // the products run one after the other
        total = at;
    }
};

template <class T>
cudaError_t backward(const phyzb_linear_grad_args& a, char* ws, cudaStream_t st) {
    const Out<T> dw{(T*)a.dw, a.dw_stride[0], a.dw_stride[1]};  // i = n
    if (a.m == 0) {  // no rows: sums of nothing
        if (a.dw) join_kernel<<<(unsigned)((a.n * a.k + 255) / 256), 256, 0, st>>>(nullptr, 0, a.n, a.k, store_epi<T>(dw, a.n));
        if (a.dbias) column_sum_kernel<<<(unsigned)((a.n + 31) / 32), 1024, 0, st>>>(nullptr, 0, a.n, a.dbias);
        return cudaGetLastError();
    }
    const Backward p(a);
    cudaError_t e = cudaSuccess;
    if (p.own_dz || a.dbias) {
        DzArgs d{};
        d.dy = a.dy;
        d.pre = a.pre;
        d.dy_o = a.dy_stride[p.features ? 1 : 0];
        d.dy_i = a.dy_stride[p.features ? 0 : 1];
        d.pre_o = a.pre_stride[p.features ? 1 : 0];
        d.pre_i = a.pre_stride[p.features ? 0 : 1];
        d.outer = p.outer;
        d.inner = p.inner;
        d.pitch = p.pitch;
        d.plane = p.plane;
        d.dz = p.own_dz ? ws + p.ws_dz : nullptr;
        d.part = a.dbias ? (float*)(ws + p.ws_part) : nullptr;
        d.act = a.activation;
        d.planes = p.planes;
        d.lines = p.lines;
        constexpr int V = 16 / sizeof(T);
        auto wide = [&](const void* q, long long os, long long is) {
            return (uintptr_t)q % 16 == 0 && is == 1 && (p.outer == 1 || os % V == 0);
        };
        const bool neighbours = p.inner % V == 0 && wide(d.dy, d.dy_o, d.dy_i) &&
                                (a.activation == PHYZB_ACT_NONE || wide(d.pre, d.pre_o, d.pre_i));
        if (p.mixed) {
            const long long tiles = (p.outer + 31) / 32;
            const dim3 grid((unsigned)p.blocks, (unsigned)(tiles < 65535 ? tiles : 65535));
            if (p.turn_dy)
                dz_mixed_kernel<T, true><<<grid, 256, 0, st>>>(d);
            else
                dz_mixed_kernel<T, false><<<grid, 256, 0, st>>>(d);
        } else if (p.features) {
            const dim3 grid((unsigned)p.blocks, (unsigned)(p.outer < 65535 ? p.outer : 65535));
            if (neighbours)
                dz_features_kernel<T, V><<<grid, 256, 0, st>>>(d);
            else
                dz_features_kernel<T, 1><<<grid, 256, 0, st>>>(d);
        } else if (neighbours) {
            dz_rows_kernel<T, V><<<dim3((unsigned)((p.inner + 32 * V - 1) / (32 * V)), (unsigned)p.blocks), 256, 0, st>>>(d);
        } else {
            dz_rows_kernel<T, 1><<<dim3((unsigned)((p.inner + 31) / 32), (unsigned)p.blocks), 256, 0, st>>>(d);
        }
        if (a.dbias)
            column_sum_kernel<<<(unsigned)((a.n + 31) / 32), 1024, 0, st>>>(d.part, p.blocks, a.n, a.dbias);
        e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    // dz as rows x n
    const long long zr = p.own_dz ? (p.features ? 1 : p.pitch) : a.dy_stride[0];
    const long long zn = p.own_dz ? (p.features ? p.pitch : 1) : a.dy_stride[1];
    const char* zp = p.own_dz ? ws + p.ws_dz : (const char*)a.dy;
    GemmMat dz[3], dzt[3];
    for (int k = 0; k < 3; k++) {
        dz[k] = {zp + k * p.plane * 2, zr, zn, 0};
        dzt[k] = {zp + k * p.plane * 2, zn, zr, 0};
    }
    char* const part = ws + p.ws_sum;
    if (a.dx) {
        const bool rf = p.dx_rows_first;
        if constexpr (sizeof(T) == 4) {
            if (p.simt_dx) {
                e = simt_multiply({(const float*)zp, zr, zn}, {(const float*)a.w, a.w_stride[1], a.w_stride[0]}, a.m, a.k,
                                  a.n, p.split_dx, along_i_of(a.dx_stride), part,
                                  store_epi<T>({(T*)a.dx, a.dx_stride[0], a.dx_stride[1]}, a.m), st);
            }
        }
        if (!p.simt_dx) {
            GemmMat w[3];
            e = Backward::w_of(a).ready(ws + p.ws_w, w, st);
            if (e != cudaSuccess) return e;
            const StoreEpi<T> epi =
                store_epi<T>({(T*)a.dx, a.dx_stride[rf ? 0 : 1], a.dx_stride[rf ? 1 : 0]}, rf ? a.m : a.k);
            e = multiply<T>(rf ? dz : w, rf ? w : dz, rf ? a.m : a.k, rf ? a.k : a.m, a.n, p.cut_dx, part, epi, st);
        }
        if (e != cudaSuccess) return e;
    }
    if (a.dw) {
        if constexpr (sizeof(T) == 4) {
            if (p.simt_dw)
                return simt_multiply({(const float*)zp, zn, zr}, {(const float*)a.x, a.x_stride[1], a.x_stride[0]}, a.n,
                                     a.k, a.m, p.split_dw, along_i_of(a.dw_stride), part,
                                     store_epi<T>(dw, a.n), st);
        }
        GemmMat x[3];
        e = Backward::x_of(a).ready(ws + p.ws_x, x, st);
        if (e != cudaSuccess) return e;
        if (p.dw_n_first)
            e = multiply<T>(dzt, x, a.n, a.k, a.m, p.cut_dw, part, store_epi<T>(dw, a.n), st);
        else
            e = multiply<T>(x, dzt, a.k, a.n, a.m, p.cut_dw, part, store_epi<T>({dw.p, dw.js, dw.is}, a.k), st);
    }
    return e;
}

}  // namespace

long long linear_workspace(const phyzb_linear_args& a) {
    const Way way = way_of(a);
    if (way == ROWS) return 0;
    if (way == SIMT) {
        const int s = simt_splits(a.m, a.n, a.k);
        return s > 1 ? s * a.m * a.n * 4 : 0;
    }
    return Forward(a).total;
}
long long linear_grad_workspace(const phyzb_linear_grad_args& a) { return a.m ? Backward(a).total : 0; }

cudaError_t linear_forward(const phyzb_linear_args& a, void* ws, cudaStream_t s) {
    if (a.dtype == PHYZB_DT_F32) return forward<float>(a, (char*)ws, s);
    if (a.dtype == PHYZB_DT_BF16) return forward<__nv_bfloat16>(a, (char*)ws, s);
    return forward<__half>(a, (char*)ws, s);
}

cudaError_t linear_backward(const phyzb_linear_grad_args& a, void* ws, cudaStream_t s) {
    if (a.dtype == PHYZB_DT_F32) return backward<float>(a, (char*)ws, s);
    if (a.dtype == PHYZB_DT_BF16) return backward<__nv_bfloat16>(a, (char*)ws, s);
    return backward<__half>(a, (char*)ws, s);
}

cudaError_t linear_faults(unsigned int* n) { return cudaMemcpyFromSymbol(n, g_linear_fault, sizeof(*n)); }

}  // namespace pz
