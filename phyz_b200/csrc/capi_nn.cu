// C ABI of the recurrent-block operators (include/phyzb.h): the checks of
// their arguments, then linear.cu, scan.cu and muon.cu. Nothing here allocates
// device memory or waits for the device.
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <exception>
#include <string>

#include "capi_internal.h"
#include "pz_nn.h"

using namespace pzc;

namespace {

// No exception crosses the C boundary.
template <class F>
int guarded(F f) {
    try {
        return f();
    } catch (const std::exception& e) {
        return fail(PHYZB_ERR_INVALID, e.what());
    } catch (...) {
        return fail(PHYZB_ERR_INVALID, "unknown exception");
    }
}

int bad(const std::string& msg) { return fail(PHYZB_ERR_INVALID, msg); }

constexpr int64_t MAX_SIDE = ((int64_t)1 << 31) - 1024;  // one side of an array (32-bit tile coordinates)
constexpr int64_t MAX_SPAN = (int64_t)1 << 46;   // elements that an array spans

int check_dtype(int dtype, const char* what) {
    if (dtype < PHYZB_DT_F32 || dtype > PHYZB_DT_F16)
        return bad(std::string(what) + " " + std::to_string(dtype) + " is none of PHYZB_DT_F32, _BF16, _F16");
    return PHYZB_OK;
}

// `n` sides each in lo..2^31
int check_sides(const int64_t* v, const char* const* names, int n, int64_t lo) {
    for (int i = 0; i < n; i++)
        if (v[i] < lo || v[i] >= MAX_SIDE)
            return bad(std::string(names[i]) + " = " + std::to_string(v[i]) + " not in " + std::to_string(lo) +
                       ".." + std::to_string(MAX_SIDE - 1));
    return PHYZB_OK;
}

// An array's pointer and strides; `out`: written, so that no two elements may
// share an address (a stride of 0 on an axis longer than 1).
int check_array(const void* p, const int64_t* stride, const int64_t* size, int n, int esize, bool out,
                const char* name) {
    if (!p) return bad(std::string(name) + " is null");
    if ((uintptr_t)p % (uintptr_t)esize) return bad(std::string(name) + " is not aligned to its element size");
    int64_t span = 0;
    for (int i = 0; i < n; i++) {
        if (stride[i] < 0) return bad(std::string(name) + " has a negative stride");
        if (out && stride[i] == 0 && size[i] > 1) return bad(std::string(name) + " is written and has a stride of 0");
        if (size[i] > 1) {
            if (stride[i] > MAX_SPAN / size[i]) return bad(std::string(name) + " spans more than 2^46 elements");
            span += stride[i] * (size[i] - 1);
        }
    }
    if (span > MAX_SPAN) return bad(std::string(name) + " spans more than 2^46 elements");
    return PHYZB_OK;
}

int esize(int dtype) { return dtype == PHYZB_DT_F32 ? 4 : 2; }

int check_device(int device) {
    static std::atomic<int> count{0};  // devices do not come and go in a process
    int ndev = count.load(std::memory_order_relaxed);
    if (ndev < 1) {
        if (cudaGetDeviceCount(&ndev) != cudaSuccess || ndev < 1) {
            cudaGetLastError();
            return fail(PHYZB_ERR_NO_DEVICE, "no CUDA device");
        }
        count.store(ndev, std::memory_order_relaxed);
    }
    if (device < 0 || device >= ndev) return bad("device " + std::to_string(device) + " out of range");
    return PHYZB_OK;
}

int check_workspace(const void* ws, int64_t given, long long need) {
    if (need <= 0) return PHYZB_OK;
    if (given < need)
        return bad("workspace of " + std::to_string(given) + " bytes is smaller than the " + std::to_string(need) +
                   " that this call needs");
    if (!ws) return bad("workspace is null");
    if ((uintptr_t)ws % 256) return bad("workspace is not 256-byte aligned");
    return PHYZB_OK;
}

int check(const phyzb_linear_args* a) {
    if (!a) return bad("args is null");
    PZ_TRY(check_dtype(a->dtype, "dtype"));
    if (a->activation < PHYZB_ACT_NONE || a->activation > PHYZB_ACT_GELU)
        return bad("activation " + std::to_string(a->activation) + " unknown");
    const char* names[] = {"k", "n"};
    const int64_t kn[] = {a->k, a->n}, xs[] = {a->m, a->k}, wsz[] = {a->n, a->k}, ys[] = {a->m, a->n};
    PZ_TRY(check_sides(kn, names, 2, 1));
    const char* mname[] = {"m"};
    PZ_TRY(check_sides(&a->m, mname, 1, 0));
    const int e = esize(a->dtype);
    PZ_TRY(check_array(a->w, a->w_stride, wsz, 2, e, false, "w"));
    if (a->bias && (uintptr_t)a->bias % 4) return bad("bias is not aligned to its element size");
    if (a->m == 0) return PHYZB_OK;
    PZ_TRY(check_array(a->x, a->x_stride, xs, 2, e, false, "x"));
    PZ_TRY(check_array(a->y, a->y_stride, ys, 2, e, true, "y"));
    if (a->residual) PZ_TRY(check_array(a->residual, a->residual_stride, ys, 2, e, false, "residual"));
    if (a->pre) PZ_TRY(check_array(a->pre, a->pre_stride, ys, 2, e, true, "pre"));
    return PHYZB_OK;
}

int check(const phyzb_linear_grad_args* a) {
    if (!a) return bad("args is null");
    PZ_TRY(check_dtype(a->dtype, "dtype"));
    if (a->activation < PHYZB_ACT_NONE || a->activation > PHYZB_ACT_GELU)
        return bad("activation " + std::to_string(a->activation) + " unknown");
    const char* names[] = {"k", "n"};
    const int64_t kn[] = {a->k, a->n}, xs[] = {a->m, a->k}, wsz[] = {a->n, a->k}, ys[] = {a->m, a->n};
    PZ_TRY(check_sides(kn, names, 2, 1));
    const char* mname[] = {"m"};
    PZ_TRY(check_sides(&a->m, mname, 1, 0));
    const int e = esize(a->dtype);
    if (a->dw) PZ_TRY(check_array(a->dw, a->dw_stride, wsz, 2, e, true, "dw"));
    if (a->dbias && (uintptr_t)a->dbias % 4) return bad("dbias is not aligned to its element size");
    if (a->dx) PZ_TRY(check_array(a->w, a->w_stride, wsz, 2, e, false, "w"));
    if (a->m == 0) return PHYZB_OK;
    PZ_TRY(check_array(a->dy, a->dy_stride, ys, 2, e, false, "dy"));
    if (a->activation != PHYZB_ACT_NONE) PZ_TRY(check_array(a->pre, a->pre_stride, ys, 2, e, false, "pre"));
    if (a->dw) PZ_TRY(check_array(a->x, a->x_stride, xs, 2, e, false, "x"));
    if (a->dx) PZ_TRY(check_array(a->dx, a->dx_stride, xs, 2, e, true, "dx"));
    return PHYZB_OK;
}

int check(const phyzb_scan_args* a) {
    if (!a) return bad("args is null");
    PZ_TRY(check_dtype(a->dtype, "dtype"));
    const int64_t n[] = {a->b, a->t, a->c}, bc[] = {a->b, a->c};
    const char* names[] = {"b", "t", "c"};
    PZ_TRY(check_sides(n, names, 3, 0));
    if (a->c && a->b > ((int64_t)1 << 37) / a->c) return bad("b * c exceeds 2^37 chains");
    if (a->b == 0 || a->c == 0) return PHYZB_OK;
    const int e = esize(a->dtype);
    if (a->h0) PZ_TRY(check_array(a->h0, a->h0_stride, bc, 2, 4, false, "h0"));
    if (a->h_last && (uintptr_t)a->h_last % 4) return bad("h_last is not aligned to its element size");
    if (a->t == 0) return PHYZB_OK;
    PZ_TRY(check_array(a->x, a->x_stride, n, 3, e, false, "x"));
    PZ_TRY(check_array(a->gate, a->gate_stride, n, 3, e, false, "gate"));
    if (a->reset) PZ_TRY(check_array(a->reset, a->reset_stride, n, 3, 1, false, "reset"));
    return check_array(a->h, a->h_stride, n, 3, e, true, "h");
}

int check(const phyzb_scan_grad_args* a) {
    if (!a) return bad("args is null");
    PZ_TRY(check_dtype(a->dtype, "dtype"));
    const int64_t n[] = {a->b, a->t, a->c}, bc[] = {a->b, a->c};
    const char* names[] = {"b", "t", "c"};
    PZ_TRY(check_sides(n, names, 3, 0));
    if (a->c && a->b > ((int64_t)1 << 37) / a->c) return bad("b * c exceeds 2^37 chains");
    if (a->b == 0 || a->c == 0) return PHYZB_OK;
    const int e = esize(a->dtype);
    if (a->h0) PZ_TRY(check_array(a->h0, a->h0_stride, bc, 2, 4, false, "h0"));
    if (a->dh_last) PZ_TRY(check_array(a->dh_last, a->dh_last_stride, bc, 2, 4, false, "dh_last"));
    if (a->dh0 && (uintptr_t)a->dh0 % 4) return bad("dh0 is not aligned to its element size");
    if (a->t == 0) return PHYZB_OK;
    PZ_TRY(check_array(a->dh, a->dh_stride, n, 3, e, false, "dh"));
    PZ_TRY(check_array(a->x, a->x_stride, n, 3, e, false, "x"));
    PZ_TRY(check_array(a->gate, a->gate_stride, n, 3, e, false, "gate"));
    PZ_TRY(check_array(a->h, a->h_stride, n, 3, e, false, "h"));
    if (a->reset) PZ_TRY(check_array(a->reset, a->reset_stride, n, 3, 1, false, "reset"));
    PZ_TRY(check_array(a->dx, a->dx_stride, n, 3, e, true, "dx"));
    return check_array(a->dgate, a->dgate_stride, n, 3, e, true, "dgate");
}

int check_matrices(int64_t batch, int64_t rows, int64_t cols, int steps) {
    if (batch < 0 || batch > 65535) return bad("batch = " + std::to_string(batch) + " not in 0..65535");
    if (rows < 1 || cols < 1) return bad("rows and cols must be >= 1");
    if (rows > PHYZB_MUON_MAX_SIDE || cols > PHYZB_MUON_MAX_SIDE)
        return fail(PHYZB_ERR_TOO_LARGE, "a side of " + std::to_string(rows > cols ? rows : cols) + " exceeds " +
                                             std::to_string(PHYZB_MUON_MAX_SIDE));
    if (steps < 1 || steps > 16) return bad("steps = " + std::to_string(steps) + " not in 1..16");
    return PHYZB_OK;
}

int check(const phyzb_muon_args* a) {
    if (!a) return bad("args is null");
    PZ_TRY(check_dtype(a->dtype, "dtype"));
    PZ_TRY(check_matrices(a->batch, a->rows, a->cols, a->steps));
    if (!std::isfinite(a->lr) || !std::isfinite(a->mu) || !std::isfinite(a->weight_decay) || !std::isfinite(a->scale))
        return bad("lr, mu, weight_decay or scale is not finite");
    if (a->batch == 0) return PHYZB_OK;
    const int64_t n[] = {a->batch, a->rows, a->cols};
    PZ_TRY(check_array(a->grad, a->grad_stride, n, 3, esize(a->dtype), false, "grad"));
    PZ_TRY(check_array(a->momentum, a->momentum_stride, n, 3, 4, true, "momentum"));
    PZ_TRY(check_array(a->weight, a->weight_stride, n, 3, 4, true, "weight"));
    if (a->copy) {
        if (a->copy_dtype != PHYZB_DT_BF16 && a->copy_dtype != PHYZB_DT_F16)
            return bad("copy_dtype must be PHYZB_DT_BF16 or PHYZB_DT_F16");
        PZ_TRY(check_array(a->copy, a->copy_stride, n, 3, 2, true, "copy"));
    }
    return PHYZB_OK;
}

int check(const phyzb_orthogonalize_args* a) {
    if (!a) return bad("args is null");
    PZ_TRY(check_dtype(a->dtype, "dtype"));
    PZ_TRY(check_matrices(a->batch, a->rows, a->cols, a->steps));
    if (a->batch == 0) return PHYZB_OK;
    const int64_t n[] = {a->batch, a->rows, a->cols};
    PZ_TRY(check_array(a->x, a->x_stride, n, 3, esize(a->dtype), false, "x"));
    return check_array(a->out, a->out_stride, n, 3, esize(a->dtype), true, "out");
}

// Whether a call has nothing to write.
bool empty(const phyzb_linear_args& a) { return a.m == 0; }
bool empty(const phyzb_linear_grad_args&) { return false; }
bool empty(const phyzb_scan_args& a) { return a.b == 0 || a.c == 0; }
bool empty(const phyzb_scan_grad_args& a) { return a.b == 0 || a.c == 0; }
bool empty(const phyzb_muon_args& a) { return a.batch == 0; }
bool empty(const phyzb_orthogonalize_args& a) { return a.batch == 0; }

template <class Args, class Size>
int workspace_of(const Args* a, int64_t* bytes, Size size) {
    return guarded([&] {
        if (!bytes) return bad("bytes is null");
        PZ_TRY(check(a));
        *bytes = empty(*a) ? 0 : size(*a);
        return (int)PHYZB_OK;
    });
}

template <class Args, class Size, class Run>
int call(const Args* a, void* ws, int64_t ws_bytes, void* stream, Size size, Run run) {
    return guarded([&] {
        PZ_TRY(check(a));
        if (!empty(*a)) PZ_TRY(check_workspace(ws, ws_bytes, size(*a)));
        PZ_TRY(check_device(a->device));
        if (empty(*a)) return (int)PHYZB_OK;
        DeviceGuard g(a->device);
        PZ_CUDA(run(*a, ws, (cudaStream_t)stream));
        return (int)PHYZB_OK;
    });
}

}  // namespace

extern "C" {

int phyzb_linear_workspace(const phyzb_linear_args* a, int64_t* bytes) {
    return workspace_of(a, bytes, pz::linear_workspace);
}
int phyzb_linear(const phyzb_linear_args* a, void* ws, int64_t ws_bytes, void* stream) {
    return call(a, ws, ws_bytes, stream, pz::linear_workspace, pz::linear_forward);
}

int phyzb_linear_grad_workspace(const phyzb_linear_grad_args* a, int64_t* bytes) {
    return workspace_of(a, bytes, pz::linear_grad_workspace);
}
int phyzb_linear_grad(const phyzb_linear_grad_args* a, void* ws, int64_t ws_bytes, void* stream) {
    return call(a, ws, ws_bytes, stream, pz::linear_grad_workspace, pz::linear_backward);
}

int phyzb_gated_scan_workspace(const phyzb_scan_args* a, int64_t* bytes) {
    return workspace_of(a, bytes, pz::scan_workspace);
}
int phyzb_gated_scan(const phyzb_scan_args* a, void* ws, int64_t ws_bytes, void* stream) {
    return call(a, ws, ws_bytes, stream, pz::scan_workspace, pz::scan_forward);
}

int phyzb_gated_scan_grad_workspace(const phyzb_scan_grad_args* a, int64_t* bytes) {
    return workspace_of(a, bytes, pz::scan_grad_workspace);
}
int phyzb_gated_scan_grad(const phyzb_scan_grad_args* a, void* ws, int64_t ws_bytes, void* stream) {
    return call(a, ws, ws_bytes, stream, pz::scan_grad_workspace, pz::scan_backward);
}

int phyzb_muon_workspace(const phyzb_muon_args* a, int64_t* bytes) {
    return workspace_of(a, bytes, pz::muon_workspace);
}
int phyzb_muon_update(const phyzb_muon_args* a, void* ws, int64_t ws_bytes, void* stream) {
    return call(a, ws, ws_bytes, stream, pz::muon_workspace, pz::muon_update);
}

int phyzb_orthogonalize_workspace(const phyzb_orthogonalize_args* a, int64_t* bytes) {
    return workspace_of(a, bytes, pz::orthogonalize_workspace);
}
int phyzb_orthogonalize(const phyzb_orthogonalize_args* a, void* ws, int64_t ws_bytes, void* stream) {
    return call(a, ws, ws_bytes, stream, pz::orthogonalize_workspace, pz::orthogonalize);
}

int phyzb_nn_status(int32_t device) {
    return guarded([&] {
        PZ_TRY(check_device(device));
        DeviceGuard g(device);
        unsigned int linear = 0, scan = 0, muon = 0;
        // (the copies below are ordered after the default stream's work, not after a non-blocking stream's)
        PZ_CUDA(cudaDeviceSynchronize());
        PZ_CUDA(pz::linear_faults(&linear));
        PZ_CUDA(pz::scan_faults(&scan));
        PZ_CUDA(pz::muon_faults(&muon));
        if (linear + scan + muon)
            return fail(PHYZB_ERR_CUDA, "waits that ran out: linear " + std::to_string(linear) + ", scan " +
                                            std::to_string(scan) + ", muon " + std::to_string(muon));
        return (int)PHYZB_OK;
    });
}

}  // extern "C"
