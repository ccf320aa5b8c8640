// What the native host side's source files share (one module, `_host_calls`).
#pragma once

#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>

namespace ascendflow_host {

// The block that reports of launches on `stream` go to (see host_calls.cpp); `kept` holds its memory until the launch is enqueued.
cudaError_t status_block(const c10::cuda::CUDAStream& stream, at::Tensor* kept, void** block);

// The functions of the operators around dense latent attention (latent_calls.cpp).
extern PyMethodDef latent_methods[];

}  // namespace ascendflow_host
