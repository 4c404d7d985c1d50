// MXFP4 quantisation of bf16 rows, the same fused behind RMSNorm, and the way back
// (format: fp4.cuh). All three stream their rows once and are bound by memory.
//
//   quantize_mxfp4: a warp takes 256 neighbours of a row, eight per lane (one 16-byte
//     load), so a block of 32 is four lanes and its maximum two shuffles; several such
//     units are in flight per warp.
//   rmsnorm_mxfp4: one CTA per row, the row in registers (as in elementwise.cu's
//     RMSNorm). y = x w / sqrt(mean(x^2) + eps) in fp32 (the product x w is exact), then
//     one rounding, to 4 bits; with `out` the row also leaves as bf16, rounded exactly
//     as the RMSNorm kernel does, for the LoRA shrink.
//   dequantize_mxfp4: codes times scale, exact in bf16.
#include "common.cuh"
#include "fp4.cuh"
#include "tma_util.h"

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>

namespace gsb {
namespace f4 {

constexpr int kQuantThreads = 256;
constexpr int kUnits = 4;  // 256-value units in flight per warp

__device__ __forceinline__ void unpack8(const uint4& q, float (&v)[8]) {
  const uint32_t p[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = unpack_bf16x2(p[j]);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

__global__ void __launch_bounds__(kQuantThreads)
    quantize_mxfp4_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int64_t K, int64_t k2s, int64_t units,
                          uint8_t* __restrict__ x4, int64_t ld4, uint8_t* __restrict__ sf) {
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  const int64_t first = warp * kUnits;
  uint4 q[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t unit = first + u;
    q[u] = make_uint4(0u, 0u, 0u, 0u);
    const int64_t row = unit / k2s, k = (unit % k2s) * 256 + lane * 8;
    if (unit < units && k < K) q[u] = *reinterpret_cast<const uint4*>(x + row * ldx + k);
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t unit = first + u;
    if (unit >= units) break;  // the whole warp
    const int64_t row = unit / k2s, k2 = unit % k2s, k = k2 * 256 + lane * 8;
    float v[8];
    unpack8(q[u], v);
    store_warp256(v, lane, k < K, x4 + row * ld4 + k / 2, sf, row, k2, 2 * k2s);
  }
}

template <int VPT>
__global__ void __launch_bounds__(256)
    rmsnorm_mxfp4_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ w, int H,
                         float eps, uint8_t* __restrict__ x4, int64_t ld4, uint8_t* __restrict__ sf,
                         __nv_bfloat16* __restrict__ out, int64_t ldo) {
  griddep_launch();
  griddep_wait();
  const int r = blockIdx.x;
  const uint4* xv = reinterpret_cast<const uint4*>(x + (int64_t)r * ldx);
  const uint4* wv = reinterpret_cast<const uint4*>(w);
  const int nvec = H / 8, nvec_pad = (int)k_tiles(H) * 16;
  uint4 buf[VPT];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * 256;
    buf[i] = make_uint4(0u, 0u, 0u, 0u);
    if (v < nvec) {
      buf[i] = xv[v];
      float f[8];
      unpack8(buf[i], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) ss += f[2 * j] * f[2 * j] + f[2 * j + 1] * f[2 * j + 1];
    }
  }
  __shared__ float red[32];
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  if (threadIdx.x < 32) {
    float t = threadIdx.x < 8 ? red[threadIdx.x] : 0.f;
    t = warp_sum(t);
    if (threadIdx.x == 0) red[0] = t;
  }
  __syncthreads();
  const float inv = rsqrtf(red[0] / (float)H + eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * 256;
    if (v >= nvec_pad) break;  // the whole warp: nvec_pad is a multiple of 32
    const bool inside = v < nvec;
    float f[8], g[8], y[8];
    unpack8(buf[i], f);
    unpack8(inside ? wv[v] : make_uint4(0u, 0u, 0u, 0u), g);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (f[j] * g[j]) * inv;
    if (!inside) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = 0.f;  // a row that is not finite has inv = NaN
    }
    store_warp256(y, threadIdx.x & 31, inside, x4 + (int64_t)r * ld4 + v * 4, sf, r, v / 32, k_tiles(H));
    if (out != nullptr && inside) {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = pack_bf16x2(__bfloat162float(__float2bfloat16_rn(f[2 * j] * inv)) * g[2 * j],
                           __bfloat162float(__float2bfloat16_rn(f[2 * j + 1] * inv)) * g[2 * j + 1]);
      reinterpret_cast<uint4*>(out + (int64_t)r * ldo)[v] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

__global__ void __launch_bounds__(kQuantThreads)
    dequantize_mxfp4_kernel(const uint8_t* __restrict__ x4, int64_t ld4, const uint8_t* __restrict__ sf, int64_t K,
                            int64_t k2s, int64_t units, __nv_bfloat16* __restrict__ out, int64_t ldo) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  uint32_t c[kUnits], b[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t unit = warp * kUnits + u, row = unit / k2s, k2 = unit % k2s, k = k2 * 256 + lane * 8;
    c[u] = b[u] = 0u;
    if (unit < units && k < K) {
      c[u] = *reinterpret_cast<const uint32_t*>(x4 + row * ld4 + k / 2);
      b[u] = sf[sf_word(row, 2 * k2 + (lane >> 4), 2 * k2s) + ((lane >> 2) & 3)];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t unit = warp * kUnits + u, row = unit / k2s, k = (unit % k2s) * 256 + lane * 8;
    if (unit >= units || k >= K) continue;
    const float s = scale_value(b[u]);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(c[u] >> (8 * j)), __NV_E2M1);
      const float2 f = __half22float2(__half2(h));
      o[j] = pack_bf16x2(f.x * s, f.y * s);
    }
    *reinterpret_cast<uint4*>(out + row * ldo + k) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

static bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// Codes [M, K / 2] and scale atoms of an [M, K] matrix.
static void check_codes(const char* op, const at::Tensor& x4, const at::Tensor& sf, int64_t M, int64_t K,
                        const at::Device& dev) {
  GSB_CHECK(x4.device() == dev && sf.device() == dev, op, ": every tensor must be on one device");
  GSB_CHECK(x4.scalar_type() == at::kByte && x4.dim() == 2 && x4.size(0) == M && x4.size(1) * 2 == K &&
                x4.stride(1) == 1 && x4.stride(0) % 16 == 0 && aligned16(x4),
            op, ": codes must be uint8 [M, K / 2] with 16-byte aligned rows");
  GSB_CHECK(sf.scalar_type() == at::kByte && sf.is_contiguous() && aligned16(sf) &&
                sf.numel() == (M + 127) / 128 * k_tiles(K) * 512,
            op, ": scales must be uint8 atoms [ceil(M / 128), 2 ceil(K / 256), 512]");
}

static void check_rows(const char* op, const char* what, const at::Tensor& x, const at::Device& dev) {
  GSB_CHECK(x.is_cuda() && x.device() == dev && x.scalar_type() == at::kBFloat16 && x.dim() == 2 &&
                (x.size(1) == 1 || x.stride(1) == 1) && (x.size(0) <= 1 || x.stride(0) % 8 == 0) && aligned16(x),
            op, ": ", what, " must be bf16 [M, K] on one CUDA device with 16-byte aligned rows");
  GSB_CHECK(x.size(1) >= kBlock && x.size(1) % kBlock == 0 && x.size(1) < (int64_t(1) << 31) &&
                x.size(0) < (int64_t(1) << 31),
            op, ": K must be a positive multiple of 32");
}

static unsigned unit_grid(const char* op, int64_t units) {
  const int64_t per = (int64_t)(kQuantThreads / 32) * kUnits, n = (units + per - 1) / per;
  GSB_CHECK(n < (int64_t(1) << 31), op, ": too many rows");
  return (unsigned)n;
}

}  // namespace f4
}  // namespace gsb

using namespace gsb;

// x [M, K] bf16 -> x4 [M, K / 2] codes, sf [ceil(M / 128), 2 ceil(K / 256), 512] scale atoms.
void gsb_quantize_mxfp4(const at::Tensor& x, const at::Tensor& x4, const at::Tensor& sf) {
  f4::check_rows("quantize_mxfp4", "x", x, x.device());
  const int64_t M = x.size(0), K = x.size(1), k2s = f4::k_tiles(K) / 2;
  f4::check_codes("quantize_mxfp4", x4, sf, M, K, x.device());
  if (M == 0) return;
  c10::cuda::CUDAGuard g(x.device());
  auto st = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  launch_dependent(f4::quantize_mxfp4_kernel, dim3(f4::unit_grid("quantize_mxfp4", M * k2s)), dim3(f4::kQuantThreads),
                   0, st, reinterpret_cast<const __nv_bfloat16*>(x.data_ptr()), x.stride(0), K, k2s, M * k2s,
                   x4.data_ptr<uint8_t>(), x4.stride(0), sf.data_ptr<uint8_t>());
}

// RMSNorm of x [M, H] and its quantisation; `out` (optional) also receives the bf16 rows.
void gsb_rmsnorm_mxfp4(const at::Tensor& x, const at::Tensor& w, double eps, const at::Tensor& x4,
                       const at::Tensor& sf, const c10::optional<at::Tensor>& out) {
  f4::check_rows("rmsnorm_mxfp4", "x", x, x.device());
  const int64_t M = x.size(0), H = x.size(1);
  GSB_CHECK(H <= 16384, "rmsnorm_mxfp4: at most 16384 columns");
  GSB_CHECK(w.device() == x.device() && w.scalar_type() == at::kBFloat16 && w.is_contiguous() && w.numel() == H &&
                f4::aligned16(w),
            "rmsnorm_mxfp4: the weight must be bf16 [H], contiguous and 16-byte aligned");
  f4::check_codes("rmsnorm_mxfp4", x4, sf, M, H, x.device());
  __nv_bfloat16* op = nullptr;
  int64_t ldo = 0;
  if (out.has_value()) {
    f4::check_rows("rmsnorm_mxfp4", "out", *out, x.device());
    GSB_CHECK(out->size(0) == M && out->size(1) == H, "rmsnorm_mxfp4: out must be [M, H]");
    op = reinterpret_cast<__nv_bfloat16*>(out->data_ptr());
    ldo = out->stride(0);
  }
  if (M == 0) return;
  c10::cuda::CUDAGuard g(x.device());
  auto st = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  auto* xp = reinterpret_cast<const __nv_bfloat16*>(x.data_ptr());
  auto* wp = reinterpret_cast<const __nv_bfloat16*>(w.data_ptr());
  const int vpt = (int)((f4::k_tiles(H) * 16 + 255) / 256);
  auto go = [&](auto kernel) {
    launch_dependent(kernel, dim3((unsigned)M), dim3(256), 0, st, xp, x.stride(0), wp, (int)H, (float)eps,
                     x4.data_ptr<uint8_t>(), x4.stride(0), sf.data_ptr<uint8_t>(), op, ldo);
  };
  if (vpt <= 1) go(f4::rmsnorm_mxfp4_kernel<1>);
  else if (vpt <= 2) go(f4::rmsnorm_mxfp4_kernel<2>);
  else if (vpt <= 4) go(f4::rmsnorm_mxfp4_kernel<4>);
  else go(f4::rmsnorm_mxfp4_kernel<8>);
}

// out [M, K] bf16 <- codes x4 and scale atoms sf.
void gsb_dequantize_mxfp4(const at::Tensor& x4, const at::Tensor& sf, const at::Tensor& out) {
  f4::check_rows("dequantize_mxfp4", "out", out, out.device());
  const int64_t M = out.size(0), K = out.size(1), k2s = f4::k_tiles(K) / 2;
  f4::check_codes("dequantize_mxfp4", x4, sf, M, K, out.device());
  if (M == 0) return;
  c10::cuda::CUDAGuard g(out.device());
  auto st = c10::cuda::getCurrentCUDAStream(out.device().index()).stream();
  f4::dequantize_mxfp4_kernel<<<(::gsb::count_launch(), f4::unit_grid("dequantize_mxfp4", M * k2s)), f4::kQuantThreads,
                                0, st>>>(x4.data_ptr<uint8_t>(), x4.stride(0), sf.data_ptr<uint8_t>(), K, k2s,
                                         M * k2s, reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), out.stride(0));
  GSB_CUDA_CHECK(cudaGetLastError());
}
