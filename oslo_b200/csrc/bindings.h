// What the files of bindings share (defined in bindings.cpp).
#pragma once
#include <cuda_runtime.h>
#include <torch/torch.h>

namespace oslo_bind {
int dt_code(const at::Tensor& t);                       // OSLO_DT_*
void check_rc(int rc, const char* what);                // an exception for what a launcher returned
cudaStream_t cur_stream(int kernels = 1);               // the current stream; counts the kernels about to be enqueued
int* error_word(int device);
int sms(int device);
}  // namespace oslo_bind
