// Host-side pieces of the MXFP4 ops that the quantisers and the GEMM share (quant_fp4.cu).
#pragma once

#include "tma_util.h"

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <cuda_runtime.h>

#include <utility>

namespace gsb {
namespace f4 {

// An uninitialised tensor on `dev`, without the dispatcher (these ops' host time is their
// smallest calls' time).
inline at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(sizes, type, dev, c10::nullopt);
}

inline bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// Bytes that a matrix (or a contiguous tensor, as one row) takes: rows of `width` bytes, `stride` apart.
struct Span {
  uintptr_t at;
  int64_t rows, width, stride;
};
inline Span span(const at::Tensor& t) {
  const int64_t item = (int64_t)t.element_size();
  const bool matrix = t.dim() == 2 && t.size(0) > 1 && t.stride(0) != 0;
  const int64_t width = (t.dim() == 2 ? t.size(1) : t.numel()) * item;
  return {reinterpret_cast<uintptr_t>(t.data_ptr()), t.numel() == 0 ? 0 : (matrix ? t.size(0) : 1), width,
          matrix ? t.stride(0) * item : 0};
}
// Whether two spans share a byte; columns of one buffer do not. (Rows at different strides whose ranges meet: yes.)
inline bool overlap(const Span& a, const Span& b) {
  if (a.rows == 0 || b.rows == 0) return false;
  if (a.at + (a.rows - 1) * a.stride + a.width <= b.at || b.at + (b.rows - 1) * b.stride + b.width <= a.at) return false;
  const int64_t stride = a.rows > 1 ? a.stride : b.stride;
  if ((a.rows == 1 && b.rows == 1) || (a.rows > 1 && b.rows > 1 && a.stride != b.stride)) return true;
  const int64_t d = ((int64_t)(b.at - a.at) % stride + stride) % stride;
  return d < a.width || d + b.width > stride;
}
// Refuses an output that shares bytes with another operand: its CTAs would read what others have written.
inline void check_apart(const char* op, const char* what, const at::Tensor& out, const char* other, const at::Tensor& t) {
  GSB_CHECK(!overlap(span(out), span(t)), op, ": ", what, " must not overlap ", other);
}
// The same, but the output may be the operand itself.
inline void check_same_or_apart(const char* op, const char* what, const at::Tensor& out, const char* other,
                                const at::Tensor& t) {
  if (out.data_ptr() == t.data_ptr() && (out.size(0) <= 1 || out.stride(0) == t.stride(0))) return;
  check_apart(op, what, out, other, t);
}

// Launches an MXFP4 kernel with `cluster` CTAs a cluster (1: none, or compiled in), unless set_pdl(0) turned
// that off as a programmatic dependent of the kernel before it in the stream: before they wait for that one
// (griddep_wait), these kernels touch their own shared and tensor memory only and prefetch
// weights into L2, which reads nothing that could be stale. It saves 1 to 2 us a launch.
template <typename... KArgs, typename... Args>
inline void launch(void (*kernel)(KArgs...), dim3 grid, int threads, int smem, int cluster, cudaStream_t st,
                   Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_allowed() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  count_launch();
  GSB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
}

// bf16 [M, K] on `dev`, K a multiple of 32, rows 16-byte aligned.
void check_rows(const char* op, const char* what, const at::Tensor& x, const at::Device& dev);

// New code and scale buffers of an [M, K] matrix in place of undefined ones (two new ones share a storage).
void make_codes(int64_t M, int64_t K, const at::Device& dev, at::Tensor& x4, at::Tensor& sf);

// Quantises M > 0 rows on the current device.
void quantize_launch(const void* x, int64_t ldx, int64_t M, int64_t K, uint8_t* x4, int64_t ld4, uint8_t* sf,
                     cudaStream_t st);

}  // namespace f4
}  // namespace gsb
