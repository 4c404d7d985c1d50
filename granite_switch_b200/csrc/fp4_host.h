// Host-side pieces of the MXFP4 ops that the quantisers and the GEMM share (quant_fp4.cu).
#pragma once

#include <ATen/ATen.h>
#include <cuda_runtime.h>

namespace gsb {
namespace f4 {

inline bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// bf16 [M, K] on `dev`, K a multiple of 32, rows 16-byte aligned.
void check_rows(const char* op, const char* what, const at::Tensor& x, const at::Device& dev);

// New code and scale buffers of an [M, K] matrix in place of undefined ones.
void make_codes(int64_t M, int64_t K, const at::Device& dev, at::Tensor& x4, at::Tensor& sf);

// Quantises M > 0 rows on the current device. The kernel lets a programmatic dependent
// start only once everything before it in the stream is done.
void quantize_launch(const void* x, int64_t ldx, int64_t M, int64_t K, uint8_t* x4, int64_t ld4, uint8_t* sf,
                     cudaStream_t st);

}  // namespace f4
}  // namespace gsb
