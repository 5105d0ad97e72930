// What the operator sources of libmdl_torch.so share (defined in torch_ops.cpp).
#pragma once

#include <ATen/ATen.h>

namespace mdl_torch {

// Raises with mdl_last_error() unless rc is MDL_OK.
void check(int rc, const char* what);
// The current HIP stream of a device.
void* stream_of(const at::Device& d);
// MDL_F32 / MDL_BF16; a TypeError for any other type.
int dtype_code(at::ScalarType t);
void require_device(const at::Tensor& t, const char* what);

}  // namespace mdl_torch
