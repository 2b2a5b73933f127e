// The recurrent-block operators (linear layer, gated scan, Muon update):
// host-side launch interface, used by capi_nn.cu. Every argument is checked
// there; strides count elements.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/phyzb.h"

namespace pz {

// linear.cu. Workspace sizes are exact for the same arguments.
long long linear_workspace(const phyzb_linear_args& a);
cudaError_t linear_forward(const phyzb_linear_args& a, void* ws, cudaStream_t s);
long long linear_grad_workspace(const phyzb_linear_grad_args& a);
cudaError_t linear_backward(const phyzb_linear_grad_args& a, void* ws, cudaStream_t s);

// scan.cu
long long scan_workspace(const phyzb_scan_args& a);
cudaError_t scan_forward(const phyzb_scan_args& a, void* ws, cudaStream_t s);
long long scan_grad_workspace(const phyzb_scan_grad_args& a);
cudaError_t scan_backward(const phyzb_scan_grad_args& a, void* ws, cudaStream_t s);

// muon.cu
long long muon_workspace(const phyzb_muon_args& a);
cudaError_t muon_update(const phyzb_muon_args& a, void* ws, cudaStream_t s);
long long orthogonalize_workspace(const phyzb_orthogonalize_args& a);
cudaError_t orthogonalize(const phyzb_orthogonalize_args& a, void* ws, cudaStream_t s);

// Waits of each file's kernels on the current device that ran out.
cudaError_t linear_faults(unsigned int* n);
cudaError_t scan_faults(unsigned int* n);
cudaError_t muon_faults(unsigned int* n);

}  // namespace pz
