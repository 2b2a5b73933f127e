// Gated linear recurrence along t of [b][t][c] arrays,
//   h_t = a_t h_{t-1} + (1 - a_t) x_t,  a = sigmoid(gate),
// and its gradients. One thread walks one chain (b, c).
//
// A stretch of steps maps the state before it to the state after it as
// h -> A h + B, and two in a row compose to (A2 A1, A2 B1 + B2). So where the
// chains are too few threads, the time axis is cut: a first launch takes each
// split's (A, B), the second one starts each split from the given state through
// the splits before it, in their order (no result depends on timing). A reset
// makes a stretch forget what came before: it is marked by A = -1 (A is a
// product of sigmoids otherwise, >= 0 or NaN), and the state before is then not
// used at all, so that a NaN or an infinity in it does not pass.
//
// The bound is memory: x and gate read once, h written once (backward: dh, x,
// gate, h in, dx, dgate out; a cut reads gate and x, or dh, twice), with 13 to
// 25 instructions a value. What it takes is bytes in flight:
//   step_kernel   one step (serving): neighbouring chains by 16-byte loads.
//   lane_kernel   TMA tiles of steps x chains run through a ring in shared
//                 memory ahead of the arithmetic, and results leave through it.
//   loose_kernel  any strides and alignment, by plain loads some steps ahead.
#include "pz_nn.cuh"
#include "pz_tma.cuh"
#include "pz_tma.h"

#include <type_traits>

namespace pz {

namespace {

constexpr float DROP = -1.0f;  // A of a stretch that begins anew within itself

// one more step (a, b) behind the stretch (A, B); drop: the state before the
// step is not used
__device__ __forceinline__ void append(float& A, float& B, float a, float b, bool drop) {
    B = drop ? b : fmaf(a, B, b);
    A = drop || A < 0.0f ? DROP : A * a;
}

__device__ unsigned int g_scan_fault;  // waits that ran out (pz_tma.cuh)

// ── one step ──────────────────────────────────────────────────────────────

struct alignas(16) Bytes16 {
    uint32_t w[4];
};

// V = 1: any strides. V = 16 bytes of values: channels contiguous and aligned.
// Bound by memory and by a launch's own two microseconds: 4096 x 256 f32, 21 MB,
// 5.5 us.
template <class T, int V>
__global__ void __launch_bounds__(256) step_kernel(const __grid_constant__ phyzb_scan_args a) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long per_row = a.c / V;
    if (i >= a.b * per_row) return;
    const long long b = a.b * per_row < 0x7fffffff ? (int)i / (int)per_row : i / per_row;
    const long long c = (i - b * per_row) * V;
    const T* xp = (const T*)a.x + b * a.x_stride[0] + c * a.x_stride[2];
    const T* gp = (const T*)a.gate + b * a.gate_stride[0] + c * a.gate_stride[2];
    const float* hp = a.h0 ? a.h0 + b * a.h0_stride[0] + c * a.h0_stride[1] : nullptr;
    const uint8_t* rp = a.reset ? a.reset + b * a.reset_stride[0] + c * a.reset_stride[2] : nullptr;
    T x[V], g[V], y[V];
    float h[V];
    if constexpr (V > 1) {
        *reinterpret_cast<Bytes16*>(x) = *reinterpret_cast<const Bytes16*>(xp);
        *reinterpret_cast<Bytes16*>(g) = *reinterpret_cast<const Bytes16*>(gp);
    } else {
        x[0] = *xp;
        g[0] = *gp;
    }
#pragma unroll
    for (int v = 0; v < V; v++) h[v] = hp ? hp[v * a.h0_stride[1]] : 0.0f;
#pragma unroll
    for (int v = 0; v < V; v++) {
        float s, shut;
        gate_f32(to_f32(g[v]), s, shut);
        const float u = shut * to_f32(x[v]);
        h[v] = rp && rp[v * a.reset_stride[2]] ? u : fmaf(s, h[v], u);
        y[v] = from_f32<T>(h[v]);
    }
    T* yp = (T*)a.h + b * a.h_stride[0] + c * a.h_stride[2];
    if constexpr (V > 1)
        *reinterpret_cast<Bytes16*>(yp) = *reinterpret_cast<const Bytes16*>(y);
    else
        *yp = y[0];
    if (a.h_last) {
#pragma unroll
        for (int v = 0; v < V; v++) a.h_last[b * a.c + c + v] = h[v];
    }
}

// ── sequences ─────────────────────────────────────────────────────────────

// The arrays of either direction. Forward: in = {gate, x}, out = {h}. Backward:
// in = {gate, dh, x, h}, out = {dx, dgate}. The time axis is cut into `splits`
// ranges of `per` steps; backward they, and the steps in them, are walked from
// the last one.
struct Side {
    const void* in[4];
    long long in_b[4], in_t[4], in_c[4];
    void* out[2];
    long long out_b[2], out_t[2], out_c[2];
    const uint8_t* reset;
    long long reset_b, reset_t, reset_c;
    const float* start;  // h0, or dh_last
    long long start_b, start_c;
    const float* h0;  // backward: h before the first step
    long long h0_b, h0_c;
    float* end;  // h_last, or dh0, [b][c]
    long long b, t, c, per;
    int splits;
    float* agg;  // [split][2][b * c]: (A, B) of each split but the last, in walking order
};

// The state of chain (b, c) before split sp: the given one through the splits
// before. OUT = false: nothing is known of it.
template <bool OUT>
__device__ __forceinline__ float start_of(const Side& s, long long b, long long c, int sp) {
    if (!OUT) return 0.0f;
    float h = s.start ? s.start[b * s.start_b + c * s.start_c] : 0.0f;
    const long long n = s.b * s.c;
    const float* p = s.agg + b * s.c + c;
#pragma unroll 16
    for (int k = 0; k < sp; k++) {
        const float A = p[0], B = p[n];
        h = A < 0.0f ? B : fmaf(A, h, B);
        p += 2 * n;
    }
    return h;
}

template <bool OUT>
__device__ __forceinline__ void finish(const Side& s, long long b, long long c, int sp, float A, float h) {
    const long long i = b * s.c + c, n = s.b * s.c;
    if (!OUT) {
        s.agg[2 * sp * n + i] = A;
        s.agg[(2 * sp + 1) * n + i] = h;
    } else if (s.end && sp == s.splits - 1) {
        s.end[i] = h;
    }
}

constexpr int NT = 128;  // threads of a block; its chains in lane_kernel: cw along c x NT / cw rows of b

// Boxes of 4 KB, two stages ahead and two behind: 24 KB a block forward, 48
// backward (six and four blocks to an SM). Measured: 64 x 64 x 16384 f32 in the
// history's order with resets 132 us, 6.2 TB/s or 94 % of a plain copy; backward 64 x
// 1024 x 1024 bf16 138 us, 5.9 TB/s; 2 x 32769 x 512 bf16, cut in 108, 65 us with
// its first launch's 27. Longer boxes or a third stage leave room for fewer
// blocks: 188 us instead of 149 backward. Blocks of 64 threads: the same. Eight
// warps to 32 chains, each with a run of the steps and a join a tile, took 32
// instructions a value and 86 us where this takes 65.
template <class T, bool BWD, bool OUT>
struct Lane {
    static constexpr int S = 32 / (int)sizeof(T);  // steps of a tile
    static constexpr int NIN = BWD && OUT ? 4 : 2, NOUT = !OUT ? 0 : BWD ? 2 : 1;
    static constexpr int BOX = S * NT * (int)sizeof(T);
    static constexpr int STAGES = 2;
    static constexpr int BYTES = (STAGES * NIN + 2 * NOUT) * BOX + 64;
    static constexpr int BLOCKS = BWD && OUT ? 4 : 6;  // per SM
};

struct LaneArgs {
    CUtensorMap in[4], out[2];  // (c, b, t): a box is [step][row of b][chain], NT values to a step
    Side s;
    int cw, cbits;  // chains of a tile along c (a power of two), its exponent
    int ctiles;     // tiles in a row of c
    int btiles;     // and along b
    int units;      // tiles x splits walked
};

// Unit u of a block's sequence: chains from (b, x) in split sp, n tiles of steps.
struct Unit {
    int b = 0, x = 0, sp = 0, t0 = 0, n = 0;
    template <class C, bool BWD>
    __device__ __forceinline__ void set(const LaneArgs& a, int u) {
        const int tiles = a.ctiles * a.btiles;
        sp = a.s.splits > 1 ? u / tiles : 0;
        u -= sp * tiles;
        b = u / a.ctiles;
        x = (u - b * a.ctiles) << a.cbits;
        b *= NT >> a.cbits;
        const int per = (int)a.s.per;
        t0 = (BWD ? a.s.splits - 1 - sp : sp) * per;
        const int len = (int)a.s.t - t0 < per ? (int)a.s.t - t0 : per;
        n = (len + C::S - 1) / C::S;
    }
    // first step of its k-th tile
    template <class C, bool BWD>
    __device__ __forceinline__ int tile(int k) const {
        return t0 + (BWD ? n - 1 - k : k) * C::S;
    }
};

template <class T, bool RESET, bool BWD, bool OUT>
__global__ void __launch_bounds__(NT, (Lane<T, BWD, OUT>::BLOCKS)) lane_kernel(const __grid_constant__ LaneArgs a) {
    using C = Lane<T, BWD, OUT>;
    constexpr int S = C::S, NIN = C::NIN, NOUT = C::NOUT, NST = C::STAGES, BOX = S * NT;
    extern __shared__ __align__(128) unsigned char sm[];
    T* const ring = reinterpret_cast<T*>(sm);  // [stage][input][step][chain]
    T* const outs = ring + NST * NIN * BOX;    // [2][output][step][chain]
    uint64_t* const full = reinterpret_cast<uint64_t*>(outs + 2 * NOUT * BOX);
    const Side& s = a.s;
    const bool lead = threadIdx.x == 0;
    if (lead) {
        for (int k = 0; k < NST; k++) mbar_init(&full[k], 1);
        mbar_init_fence();
        for (int k = 0; k < NIN; k++) tma_prefetch(&a.in[k]);
    }
    __syncthreads();
    // the lead's place in the sequence of tiles, ahead of the block's
    Unit ahead;
    int au = blockIdx.x, ak = 0, asked = 0;
    ahead.set<C, BWD>(a, au);
    auto request = [&](int stage) {
        if (au >= a.units) return;
        const int t = ahead.tile<C, BWD>(ak);
        mbar_expect(&full[stage], NIN * C::BOX);
#pragma unroll
        for (int k = 0; k < NIN; k++)  // h is read one step back (at t = 0 the box's first step is zeros)
            tma_load(ring + (stage * NIN + k) * BOX, &a.in[k], &full[stage], ahead.x, ahead.b, BWD && k == 3 ? t - 1 : t);
        asked++;
        if (++ak == ahead.n) {
            ak = 0;
            au += gridDim.x;
            if (au < a.units) ahead.set<C, BWD>(a, au);
        }
    };
    if (lead)
        for (int k = 0; k < NST; k++) request(k);
    bool failed = false;
    int stage = 0, phase = 0, buf = 0;
    for (int u = blockIdx.x; u < a.units && !failed; u += gridDim.x) {
        Unit q;
        q.set<C, BWD>(a, u);
        const int b = q.b + (threadIdx.x >> a.cbits), c = q.x + (threadIdx.x & (a.cw - 1));
        const bool on = b < s.b && c < s.c;
        // Resets of a tile's steps, loaded a tile ahead. Where all chains share a
        // step's flag, a lane reads one step's (a warp has one b); else each thread
        // reads its own, left in registers as they come.
        const bool shared = s.reset_c == 0;
        uint8_t next[RESET ? S : 1];
        const uint8_t* flag = RESET ? s.reset + b * s.reset_b + c * s.reset_c : nullptr;
        auto resets = [&](int k) {
            if (!RESET || k == q.n) return;
            const int t = q.tile<C, BWD>(k);
            if (shared) {
                const int v = threadIdx.x % 32, at = BWD ? t + S - 1 - v : t + v;
                next[0] = 0;
                if (v < S && at < s.t && b < s.b) next[0] = flag[at * s.reset_t];
                return;
            }
            const uint8_t* p = flag + (BWD ? t + S - 1 : t) * s.reset_t;
#pragma unroll
            for (int v = 0; v < S; v++) {
                next[RESET ? v : 0] = 0;
                if (on && (BWD ? t + S - 1 - v : t + v) < s.t) next[RESET ? v : 0] = *p;
                p += BWD ? -s.reset_t : s.reset_t;
            }
        };
        resets(0);
        float A = 1.0f, h = on ? start_of<OUT>(s, b, c, q.sp) : 0.0f;
        const float h0 = BWD && OUT && on && s.h0 ? s.h0[b * s.h0_b + c * s.h0_c] : 0.0f;
        for (int k = 0; k < q.n; k++) {
            const int t = q.tile<C, BWD>(k);
            const bool came = mbar_wait(&full[stage], phase);
            const T* const in = ring + stage * NIN * BOX + threadIdx.x;
            T* const out = outs + buf * NOUT * BOX + threadIdx.x;
            uint8_t drops[RESET ? S : 1];
            bool some = RESET;
            if (RESET && shared) {
                const uint32_t bits = __ballot_sync(0xffffffffu, next[0] != 0);
                some = bits != 0;
#pragma unroll
                for (int v = 0; v < S; v++) drops[RESET ? v : 0] = bits >> v & 1;
            } else if (RESET) {
#pragma unroll
                for (int v = 0; v < S; v++) drops[RESET ? v : 0] = next[RESET ? v : 0];
            }
            // the results of two tiles ago have left their buffer
            if (OUT && lead) tma_store_wait_read<1>();
            if (__syncthreads_or(!came)) {
                failed = true;
                break;
            }
            resets(k + 1);
            const int n = s.t - t < S ? (int)s.t - t : S;  // steps here
            auto walk = [&](auto whole, auto marked) {
                // values first, then the recurrence: a store between two loads
                // would keep the second one waiting
                float g[S], x[S];
                [[maybe_unused]] float shut[NIN == 4 ? S : 1], slope[NIN == 4 ? S : 1];  // of dgate over dx
#pragma unroll
                for (int v = 0; v < S; v++) {
                    const int e = (BWD ? S - 1 - v : v) * NT;
                    float q;
                    gate_f32(to_f32(in[e]), g[v], q);
                    x[v] = to_f32(in[BOX + e]);
                    if (!BWD) x[v] *= q;
                    if constexpr (NIN == 4) {
                        float before = to_f32(in[3 * BOX + e]);
                        if (v == S - 1 && t == 0) before = h0;
                        if (decltype(marked)::value && drops[RESET ? v : 0]) before = 0.0f;
                        shut[v] = q;
                        slope[v] = g[v] * (before - to_f32(in[2 * BOX + e]));
                    }
                }
#pragma unroll
                for (int v = 0; v < S; v++) {
                    const int row = BWD ? S - 1 - v : v;
                    if (!decltype(whole)::value && row >= n) continue;
                    const bool drop = decltype(marked)::value && drops[RESET ? v : 0];
                    if constexpr (!OUT) {
                        // backward, a reset passes nothing to the step before it
                        if (BWD)
                            append(A, h, drop ? 0.0f : g[v], drop ? 0.0f : g[v] * x[v], drop);
                        else
                            append(A, h, g[v], x[v], drop);
                    } else if constexpr (!BWD) {
                        h = drop ? x[v] : fmaf(g[v], h, x[v]);
                        out[row * NT] = from_f32<T>(h);
                    } else {
                        const float d = h + x[v], dx = shut[v] * d;
                        out[row * NT] = from_f32<T>(dx);
                        out[BOX + row * NT] = from_f32<T>(dx * slope[v]);
                        h = drop ? 0.0f : g[v] * d;
                    }
                }
            };
            if (n == S && !some)
                walk(std::true_type(), std::false_type());
            else if (n == S)
                walk(std::true_type(), std::true_type());
            else
                walk(std::false_type(), std::bool_constant<RESET>());
            if (OUT) fence_async();
            __syncthreads();
            if (lead) {  // steps past t, rows past b and chains past c are not written
                request(stage);
                T* const o = outs + buf * NOUT * BOX;
#pragma unroll
                for (int j = 0; j < NOUT; j++) tma_store(&a.out[j], o + j * BOX, q.x, q.b, t);
                if (OUT) tma_store_commit();
            }
            buf ^= 1;
            if (++stage == NST) stage = 0, phase ^= 1;
        }
        if (!failed && on) finish<OUT>(s, b, c, q.sp, A, h);
    }
    if (failed && lead) {  // leave the rest, but not before the boxes asked for
        atomicAdd(&g_scan_fault, 1u);
        for (int q = asked > NST ? asked - NST : 0; q < asked; q++) mbar_wait(&full[q % NST], (q / NST) & 1);
    }
    if (OUT && lead) tma_store_wait<0>();
}

// One chain per thread along the flattened (b, c); the values of the next L
// steps are loaded while the present ones are worked on.
template <bool BWD, bool OUT>
constexpr int loose_steps = BWD && OUT ? 4 : 8;

template <class T, bool RESET, bool BWD, bool OUT>
__global__ void __launch_bounds__(NT) loose_kernel(const __grid_constant__ Side s) {
    constexpr int L = loose_steps<BWD, OUT>, NIN = BWD && OUT ? 4 : 2;
    const int sp = blockIdx.y;
    const long long i = (long long)blockIdx.x * NT + threadIdx.x;
    if (i >= s.b * s.c) return;
    const long long b = s.b * s.c < 0x7fffffff ? (int)i / (int)s.c : i / s.c, c = i - b * s.c;
    const long long t0 = (BWD ? s.splits - 1 - sp : sp) * s.per, t1 = t0 + s.per < s.t ? t0 + s.per : s.t, n = t1 - t0;
    // step p of the walk is t = t0 + p, or t1 - 1 - p
    const long long first = BWD ? t1 - 1 : t0;
    const T* in[NIN];
    long long step[NIN];
#pragma unroll
    for (int k = 0; k < NIN; k++) {
        in[k] = (const T*)s.in[k] + b * s.in_b[k] + c * s.in_c[k] + first * s.in_t[k];
        step[k] = BWD ? -s.in_t[k] : s.in_t[k];
        if (k == 3) in[k] += step[k];  // h is read one step back
    }
    const uint8_t* flag = RESET ? s.reset + b * s.reset_b + c * s.reset_c + first * s.reset_t : nullptr;
    const long long fstep = BWD ? -s.reset_t : s.reset_t;
    T* out[2];
    long long ostep[2];
#pragma unroll
    for (int k = 0; k < (BWD ? 2 : 1); k++) {
        out[k] = (T*)s.out[k] + b * s.out_b[k] + c * s.out_c[k] + first * s.out_t[k];
        ostep[k] = BWD ? -s.out_t[k] : s.out_t[k];
    }
    T raw[NIN][L];
    uint8_t drops[L];
    auto load = [&](long long p) {
#pragma unroll
        for (int k = 0; k < NIN; k++) {
            const long long stop = k == 3 && t0 == 0 ? n - 1 : n;  // (before the first step h is h0)
#pragma unroll
            for (int u = 0; u < L; u++) {
                if (p + u < stop) raw[k][u] = *in[k];
                in[k] += step[k];
            }
        }
        if (RESET) {
#pragma unroll
            for (int u = 0; u < L; u++) {
                drops[u] = 0;
                if (p + u < n) drops[u] = *flag;
                flag += fstep;
            }
        }
    };
    load(0);
    const float h0 = BWD && OUT && s.h0 ? s.h0[b * s.h0_b + c * s.h0_c] : 0.0f;
    float A = 1.0f, h = start_of<OUT>(s, b, c, sp);
    for (long long p = 0; p < n; p += L) {
        float g[L], x[L], shut[L], slope[NIN == 4 ? L : 1];  // of dgate over dx
        bool drop[L];
#pragma unroll
        for (int u = 0; u < L; u++) {
            gate_f32(to_f32(raw[0][u]), g[u], shut[u]);
            x[u] = to_f32(raw[1][u]);
            if (!BWD) x[u] *= shut[u];
            drop[u] = RESET && drops[u];
            if constexpr (NIN == 4) {
                const float before = drop[u] ? 0.0f : t0 == 0 && p + u == n - 1 ? h0 : to_f32(raw[3][u]);
                slope[u] = g[u] * (before - to_f32(raw[2][u]));
            }
        }
        load(p + L);
#pragma unroll
        for (int u = 0; u < L; u++) {
            if (p + u >= n) break;
            if constexpr (!OUT) {
                if (BWD)
                    append(A, h, drop[u] ? 0.0f : g[u], drop[u] ? 0.0f : g[u] * x[u], drop[u]);
                else
                    append(A, h, g[u], x[u], drop[u]);
            } else if constexpr (!BWD) {
                h = drop[u] ? x[u] : fmaf(g[u], h, x[u]);
                *out[0] = from_f32<T>(h);
                out[0] += ostep[0];
            } else {
                const float d = h + x[u], dx = shut[u] * d;
                *out[0] = from_f32<T>(dx);
                *out[1] = from_f32<T>(dx * slope[u]);
                out[0] += ostep[0];
                out[1] += ostep[1];
                h = drop[u] ? 0.0f : g[u] * d;
            }
        }
    }
    finish<OUT>(s, b, c, sp, A, h);
}

// ── the choice between them ───────────────────────────────────────────────

constexpr int SMS = 148;

enum Kind { STEP, LANE, LOOSE };

struct Plan {
    Kind kind;
    int v;  // STEP: 1, or 16 bytes of values; LANE: chains of a tile along c
    int splits;
    long long per;
};

int esize(int dtype) { return dtype == PHYZB_DT_F32 ? 4 : 2; }

// Cuts the time axis where there is less than one block per SM, so that six per
// SM are there, each of four stretches of `steps` at least.
Plan cut(Kind kind, int v, long long blocks, long long t, int steps) {
    Plan p{kind, v, 1, t};
    if (blocks >= SMS) return p;
    long long n = 6 * SMS / blocks;
    if (n > t / (4 * steps)) n = t / (4 * steps);
    if (n < 2) return p;
    p.per = ((t + n - 1) / n + steps - 1) / steps * steps;
    p.splits = (int)((t + p.per - 1) / p.per);
    return p;
}

// Whether TMA can address [b][t][c] tiles of an array: channels contiguous,
// rows on 16-byte boundaries, sides and strides in the descriptor's ranges.
bool tma_ok(const void* p, const int64_t* stride, const int64_t* n, int dtype) {
    const int e = esize(dtype);
    if ((uintptr_t)p % 16 || (n[2] > 1 && stride[2] != 1)) return false;
    for (int k = 0; k < 2; k++)
        if (n[k] > 1 && (stride[k] * e % 16 || stride[k] <= 0 || stride[k] * e >= ((int64_t)1 << 40))) return false;
    return true;
}

// The width of a lane_kernel tile along c: the one of 128, 64, 32 that leaves the
// fewest of its chains empty, the widest of equals.
int lane_width(long long c) {
    int best = NT;
    for (int w = NT / 2; w >= 32; w /= 2)
        if ((c + w - 1) / w * w < (c + best - 1) / best * best) best = w;
    return best;
}

// Tiles take rows of c that fill most of a width, and more than a few steps.
Plan plan_of(const int64_t* n, int dtype, bool bwd, bool tma) {
    const long long b = n[0], t = n[1], c = n[2];
    if (tma && c >= 24 && t >= 8 && b * ((c + 31) / 32) < 1 << 20) {
        const int w = lane_width(c);
        return cut(LANE, w, (b + NT / w - 1) / (NT / w) * ((c + w - 1) / w), t, 32 / esize(dtype));
    }
    return cut(LOOSE, 1, (b * c + NT - 1) / NT, t, bwd ? loose_steps<true, true> : loose_steps<false, true>);
}

// The tensor map of an array as (c, b, t), in boxes of `rows` rows of cw chains
// at `steps` steps.
template <class T>
bool encode(CUtensorMap* m, const Side& s, const void* p, long long sb, long long st, int cw, int rows, int steps) {
    const cuuint64_t size[3] = {(cuuint64_t)s.c, (cuuint64_t)s.b, (cuuint64_t)s.t};
    const cuuint64_t e = sizeof(T), bytes[2] = {s.b > 1 ? sb * e : 16, s.t > 1 ? st * e : 16};
    const cuuint32_t box[3] = {(cuuint32_t)cw, (cuuint32_t)rows, (cuuint32_t)steps};
    // (16-bit values are moved, not computed on)
    const CUtensorMapDataType type = e == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    return encode_tiled(m, type, 3, const_cast<void*>(p), size, bytes, box, CU_TENSOR_MAP_SWIZZLE_NONE) == CUDA_SUCCESS;
}

template <class T, bool RESET, bool BWD, bool OUT>
cudaError_t run_lanes(LaneArgs& a, cudaStream_t st) {
    using C = Lane<T, BWD, OUT>;
    auto kernel = lane_kernel<T, RESET, BWD, OUT>;
    static SmemOnce once;
    const cudaError_t e = once.smem(kernel, C::BYTES);
    if (e != cudaSuccess) return e;
    a.units = a.ctiles * a.btiles * (OUT ? a.s.splits : a.s.splits - 1);
    const int slots = SMS * C::BLOCKS;
    kernel<<<a.units < slots ? a.units : slots, NT, C::BYTES, st>>>(a);
    return cudaGetLastError();
}

template <class T, bool RESET, bool BWD>
cudaError_t launch(const Side& s, const Plan& p, cudaStream_t st) {
    if (p.kind == LANE) {
        using C = Lane<T, BWD, true>;
        const int cw = p.v, rows = NT / cw;
        LaneArgs a;
        a.s = s;
        a.cw = cw;
        a.cbits = cw == 128 ? 7 : cw == 64 ? 6 : 5;
        a.ctiles = (int)((s.c + cw - 1) / cw);
        a.btiles = (int)((s.b + rows - 1) / rows);
        for (int k = 0; k < C::NIN; k++)
            if (!encode<T>(&a.in[k], s, s.in[k], s.in_b[k], s.in_t[k], cw, rows, C::S)) return cudaErrorInvalidValue;
        for (int k = 0; k < C::NOUT; k++)
            if (!encode<T>(&a.out[k], s, s.out[k], s.out_b[k], s.out_t[k], cw, rows, C::S)) return cudaErrorInvalidValue;
        if (s.splits > 1) {
            const cudaError_t e = run_lanes<T, RESET, BWD, false>(a, st);
            if (e != cudaSuccess) return e;
        }
        return run_lanes<T, RESET, BWD, true>(a, st);
    }
    const unsigned blocks = (unsigned)((s.b * s.c + NT - 1) / NT);
    if (s.splits > 1) {
        loose_kernel<T, RESET, BWD, false><<<dim3(blocks, (unsigned)s.splits - 1), NT, 0, st>>>(s);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    loose_kernel<T, RESET, BWD, true><<<dim3(blocks, (unsigned)s.splits), NT, 0, st>>>(s);
    return cudaGetLastError();
}

template <bool BWD>
cudaError_t launch(Side& s, const Plan& p, int dtype, void* ws, cudaStream_t st) {
    s.splits = p.splits;
    s.per = p.per;
    s.agg = (float*)ws;
    if (dtype == PHYZB_DT_F32) return s.reset ? launch<float, true, BWD>(s, p, st) : launch<float, false, BWD>(s, p, st);
    if (dtype == PHYZB_DT_BF16)
        return s.reset ? launch<__nv_bfloat16, true, BWD>(s, p, st) : launch<__nv_bfloat16, false, BWD>(s, p, st);
    return s.reset ? launch<__half, true, BWD>(s, p, st) : launch<__half, false, BWD>(s, p, st);
}

// Whether a step's chains can be taken 16 bytes at a time.
bool wide_ok(const void* p, const int64_t* stride, const int64_t* n, int e) {
    return (uintptr_t)p % 16 == 0 && stride[2] == 1 && n[2] % (16 / e) == 0 && (n[0] == 1 || stride[0] * e % 16 == 0);
}

Plan plan(const phyzb_scan_args& a) {
    const int64_t n[] = {a.b, a.t, a.c};
    if (a.t == 1) {
        const int e = esize(a.dtype);
        const bool wide = wide_ok(a.x, a.x_stride, n, e) && wide_ok(a.gate, a.gate_stride, n, e) &&
                          wide_ok(a.h, a.h_stride, n, e);
        return {STEP, wide ? 16 / e : 1, 1, 1};
    }
    const bool tma = a.t > 0 && tma_ok(a.x, a.x_stride, n, a.dtype) && tma_ok(a.gate, a.gate_stride, n, a.dtype) &&
                     tma_ok(a.h, a.h_stride, n, a.dtype);
    return plan_of(n, a.dtype, false, tma);
}

Plan plan(const phyzb_scan_grad_args& a) {
    const int64_t n[] = {a.b, a.t, a.c};
    const bool tma = a.t > 0 && tma_ok(a.x, a.x_stride, n, a.dtype) && tma_ok(a.gate, a.gate_stride, n, a.dtype) &&
                     tma_ok(a.h, a.h_stride, n, a.dtype) && tma_ok(a.dh, a.dh_stride, n, a.dtype) &&
                     tma_ok(a.dx, a.dx_stride, n, a.dtype) && tma_ok(a.dgate, a.dgate_stride, n, a.dtype);
    return plan_of(n, a.dtype, true, tma);
}

long long agg_bytes(const Plan& p, long long chains) { return (p.splits - 1) * 2 * chains * 4; }

template <class T>
cudaError_t step(const phyzb_scan_args& a, int v, cudaStream_t st) {
    const unsigned grid = (unsigned)((a.b * (a.c / v) + 255) / 256);
    if (v > 1)
        step_kernel<T, 16 / sizeof(T)><<<grid, 256, 0, st>>>(a);
    else
        step_kernel<T, 1><<<grid, 256, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace

long long scan_workspace(const phyzb_scan_args& a) { return agg_bytes(plan(a), a.b * a.c); }
long long scan_grad_workspace(const phyzb_scan_grad_args& a) { return agg_bytes(plan(a), a.b * a.c); }

cudaError_t scan_forward(const phyzb_scan_args& a, void* ws, cudaStream_t st) {
    const Plan p = plan(a);
    if (p.kind == STEP) {
        if (a.dtype == PHYZB_DT_F32) return step<float>(a, p.v, st);
        if (a.dtype == PHYZB_DT_BF16) return step<__nv_bfloat16>(a, p.v, st);
        return step<__half>(a, p.v, st);
    }
    Side s{};
    auto in = [&](int k, const void* x, const int64_t* st3) {
        s.in[k] = x;
        s.in_b[k] = st3[0];
        s.in_t[k] = st3[1];
        s.in_c[k] = st3[2];
    };
    in(0, a.gate, a.gate_stride);
    in(1, a.x, a.x_stride);
    s.out[0] = a.h;
    s.out_b[0] = a.h_stride[0];
    s.out_t[0] = a.h_stride[1];
    s.out_c[0] = a.h_stride[2];
    s.reset = a.reset;
    s.reset_b = a.reset_stride[0];
    s.reset_t = a.reset_stride[1];
    s.reset_c = a.reset_stride[2];
    s.start = a.h0;
    s.start_b = a.h0_stride[0];
    s.start_c = a.h0_stride[1];
    s.end = a.h_last;
    s.b = a.b;
    s.t = a.t;
    s.c = a.c;
    return launch<false>(s, p, a.dtype, ws, st);
}

cudaError_t scan_backward(const phyzb_scan_grad_args& a, void* ws, cudaStream_t st) {
    Side s{};
    auto in = [&](int k, const void* x, const int64_t* st3) {
        s.in[k] = x;
        s.in_b[k] = st3[0];
        s.in_t[k] = st3[1];
        s.in_c[k] = st3[2];
    };
    auto out = [&](int k, void* x, const int64_t* st3) {
        s.out[k] = x;
        s.out_b[k] = st3[0];
        s.out_t[k] = st3[1];
        s.out_c[k] = st3[2];
    };
    in(0, a.gate, a.gate_stride);
    in(1, a.dh, a.dh_stride);
    in(2, a.x, a.x_stride);
    in(3, a.h, a.h_stride);
    out(0, a.dx, a.dx_stride);
    out(1, a.dgate, a.dgate_stride);
    s.reset = a.reset;
    s.reset_b = a.reset_stride[0];
    s.reset_t = a.reset_stride[1];
    s.reset_c = a.reset_stride[2];
    s.start = a.dh_last;
    s.start_b = a.dh_last_stride[0];
    s.start_c = a.dh_last_stride[1];
    s.h0 = a.h0;
    s.h0_b = a.h0_stride[0];
    s.h0_c = a.h0_stride[1];
    s.end = a.dh0;
    s.b = a.b;
    s.t = a.t;
    s.c = a.c;
    return launch<true>(s, plan(a), a.dtype, ws, st);
}

cudaError_t scan_faults(unsigned int* n) { return cudaMemcpyFromSymbol(n, g_scan_fault, sizeof(*n)); }

}  // namespace pz
