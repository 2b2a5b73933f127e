// Gated linear recurrence h_t = a_t h_{t-1} + (1 - a_t) x_t, a = sigmoid(gate),
// and its gradients: one thread per chain (b, c), stepping along t.
#include "pz_nn.cuh"

namespace pz {

namespace {

template <class T>
__global__ void __launch_bounds__(128) scan_kernel(const phyzb_scan_args a) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.b * a.c) return;
    const long long b = i / a.c, c = i % a.c;
    const T* x = (const T*)a.x + b * a.x_stride[0] + c * a.x_stride[2];
    const T* g = (const T*)a.gate + b * a.gate_stride[0] + c * a.gate_stride[2];
    T* y = (T*)a.h + b * a.h_stride[0] + c * a.h_stride[2];
    const uint8_t* r = a.reset ? a.reset + b * a.reset_stride[0] + c * a.reset_stride[2] : nullptr;
    float h = a.h0 ? a.h0[b * a.h0_stride[0] + c * a.h0_stride[1]] : 0.0f;
    for (long long t = 0; t < a.t; t++) {
        const float s = sigmoid_f32(to_f32(g[t * a.gate_stride[1]]));
        if (r && r[t * a.reset_stride[1]]) h = 0.0f;
        h = fmaf(s, h, (1.0f - s) * to_f32(x[t * a.x_stride[1]]));
        y[t * a.h_stride[1]] = from_f32<T>(h);
    }
    if (a.h_last) a.h_last[i] = h;
}

template <class T>
__global__ void __launch_bounds__(128) scan_grad_kernel(const phyzb_scan_grad_args a) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.b * a.c) return;
    const long long b = i / a.c, c = i % a.c;
    const T* dh = (const T*)a.dh + b * a.dh_stride[0] + c * a.dh_stride[2];
    const T* x = (const T*)a.x + b * a.x_stride[0] + c * a.x_stride[2];
    const T* g = (const T*)a.gate + b * a.gate_stride[0] + c * a.gate_stride[2];
    const T* h = (const T*)a.h + b * a.h_stride[0] + c * a.h_stride[2];
    T* dx = (T*)a.dx + b * a.dx_stride[0] + c * a.dx_stride[2];
    T* dg = (T*)a.dgate + b * a.dgate_stride[0] + c * a.dgate_stride[2];
    const uint8_t* r = a.reset ? a.reset + b * a.reset_stride[0] + c * a.reset_stride[2] : nullptr;
    const float h0 = a.h0 ? a.h0[b * a.h0_stride[0] + c * a.h0_stride[1]] : 0.0f;
    float carry = a.dh_last ? a.dh_last[b * a.dh_last_stride[0] + c * a.dh_last_stride[1]] : 0.0f;
    for (long long t = a.t - 1; t >= 0; t--) {
        const float s = sigmoid_f32(to_f32(g[t * a.gate_stride[1]]));
        const bool reset = r && r[t * a.reset_stride[1]];
        const float prev = reset ? 0.0f : t ? to_f32(h[(t - 1) * a.h_stride[1]]) : h0;
        const float d = to_f32(dh[t * a.dh_stride[1]]) + carry;
        const float u = (1.0f - s) * d;
        dx[t * a.dx_stride[1]] = from_f32<T>(u);
        dg[t * a.dgate_stride[1]] = from_f32<T>(u * s * (prev - to_f32(x[t * a.x_stride[1]])));
        carry = reset ? 0.0f : s * d;
    }
    if (a.dh0) a.dh0[i] = carry;
}

unsigned blocks_of(long long n) { return (unsigned)((n + 127) / 128); }

}  // namespace

long long scan_workspace(const phyzb_scan_args&) { return 0; }
long long scan_grad_workspace(const phyzb_scan_grad_args&) { return 0; }

cudaError_t scan_forward(const phyzb_scan_args& a, void*, cudaStream_t s) {
    const unsigned n = blocks_of(a.b * a.c);
    if (a.dtype == PHYZB_DT_F32) scan_kernel<float><<<n, 128, 0, s>>>(a);
    if (a.dtype == PHYZB_DT_BF16) scan_kernel<__nv_bfloat16><<<n, 128, 0, s>>>(a);
    if (a.dtype == PHYZB_DT_F16) scan_kernel<__half><<<n, 128, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t scan_backward(const phyzb_scan_grad_args& a, void*, cudaStream_t s) {
    const unsigned n = blocks_of(a.b * a.c);
    if (a.dtype == PHYZB_DT_F32) scan_grad_kernel<float><<<n, 128, 0, s>>>(a);
    if (a.dtype == PHYZB_DT_BF16) scan_grad_kernel<__nv_bfloat16><<<n, 128, 0, s>>>(a);
    if (a.dtype == PHYZB_DT_F16) scan_grad_kernel<__half><<<n, 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace pz
