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
#include "fp4_host.h"
#include "tma_util.h"

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <tuple>

namespace gsb {
namespace f4 {

constexpr int kQuantThreads = 256;
constexpr int kUnits = 4;  // 256-value units of one row in flight per warp

// Warp `blockIdx.x * 8 + ..` takes `kUnits` units of one row; `per_row` warps make a row.
__global__ void __launch_bounds__(kQuantThreads)
    quantize_mxfp4_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int K, int k2s, uint32_t per_row,
                          uint32_t warps, uint8_t* __restrict__ x4, int64_t ld4, uint8_t* __restrict__ sf) {
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t warp = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  if (warp >= warps) return;
  const uint32_t row = warp / per_row;
  const int first = (int)(warp - row * per_row) * kUnits;
  const __nv_bfloat16* xr = x + row * ldx + lane * 8;
  uint4 q[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int k = (first + u) * 256;
    q[u] = make_uint4(0u, 0u, 0u, 0u);
    if (k + lane * 8 < K) q[u] = *reinterpret_cast<const uint4*>(xr + k);
  }
  uint8_t* xo = x4 + row * ld4 + lane * 4;
  uint8_t* so = sf + sf_word(row, 2 * first, 2 * k2s);
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int k2 = first + u, k = k2 * 256 + lane * 8;
    if (k2 >= k2s) break;  // the whole warp
    uint32_t codes;
    const uint32_t byte = quantise8(q[u], codes);
    if (k < K) *reinterpret_cast<uint32_t*>(xo + k2 * 128) = codes;
    store_scales256(byte, lane, so + u * 1024);
  }
}

__device__ __forceinline__ float max_abs3(float a, float b, float c) {  // NaN if any is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}

// Eight normalised values -> codes, scales and (optionally) their part of the bf16 row. The
// products x w are exact, and one multiplication by inv (times the block's power of two,
// exact too) rounds each value; the maximum may be taken before it, since rounding keeps order.
__device__ __forceinline__ void norm_store8(const uint4& xq, const uint4& wq, float inv, bool inside, int lane,
                                            uint8_t* codes_out, uint8_t* sf, uint4* out) {
  float f[8], g[8], y[8];
  unpack8(xq, f);
  unpack8(wq, g);
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = f[j] * g[j];
  const float top = max_abs3(max_abs3(y[0], y[1], y[2]), max_abs3(y[3], y[4], y[5]), max_abs3(y[6], y[7], y[7]));
  uint32_t byte = scale_byte(quad_max(__float_as_uint(top * inv) & 0x7fffffffu));
  byte = inside ? byte : 0u;  // past the row (whole blocks): inv is NaN in a row that is not finite
  float s = inv_scale(byte);
  if (byte < 32u) {  // inv * 2^-e may overflow
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] *= inv;
  } else {
    s *= inv;
  }
  const uint32_t codes = pack8(y, s);
  if (inside) {
    *reinterpret_cast<uint32_t*>(codes_out) = byte == 255u ? 0u : codes;
    if (out != nullptr) {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = pack_bf16x2(__bfloat162float(__float2bfloat16_rn(f[2 * j] * inv)) * g[2 * j],
                           __bfloat162float(__float2bfloat16_rn(f[2 * j + 1] * inv)) * g[2 * j + 1]);
      *out = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
  store_scales256(byte, lane, sf);
}

// One CTA per row; the sum of squares in the RMSNorm kernel's order.
template <int VPT>
__global__ void __launch_bounds__(256)
    rmsnorm_mxfp4_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ w, int H,
                         float eps, uint8_t* __restrict__ x4, int64_t ld4, uint8_t* __restrict__ sf,
                         __nv_bfloat16* __restrict__ out, int64_t ldo) {
  griddep_launch();
  griddep_wait();
  const int64_t r = blockIdx.x;
  const uint4* xv = reinterpret_cast<const uint4*>(x + r * ldx);
  const uint4* wv = reinterpret_cast<const uint4*>(w);
  const int nvec = H / 8, nvec_pad = (int)k_tiles(H) * 16;
  uint4 buf[VPT];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * 256;
    buf[i] = v < nvec ? xv[v] : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const uint32_t p[4] = {buf[i].x, buf[i].y, buf[i].z, buf[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack_bf16x2(p[j]);
      ss += f.x * f.x + f.y * f.y;
    }
  }
  __shared__ float red[8], s_inv;
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  if (threadIdx.x < 32) {
    float t = threadIdx.x < 8 ? red[threadIdx.x] : 0.f;
    t = warp_sum(t);
    if (threadIdx.x == 0) s_inv = rsqrtf(t / (float)H + eps);
  }
  __syncthreads();
  const float inv = s_inv;
  const int lane = threadIdx.x & 31;
  uint8_t* codes = x4 + r * ld4 + threadIdx.x * 4;
  uint8_t* scales = sf + sf_word(r, 2 * (threadIdx.x >> 5), k_tiles(H));
  uint4* ov = out ? reinterpret_cast<uint4*>(out + r * ldo) + threadIdx.x : nullptr;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * 256;
    if (v >= nvec_pad) break;  // the whole warp: nvec_pad is a multiple of 32
    const bool inside = v < nvec;
    norm_store8(buf[i], inside ? wv[v] : make_uint4(0u, 0u, 0u, 0u), inv, inside, lane, codes + i * 1024,
                scales + i * 8 * 1024, ov ? ov + i * 256 : nullptr);
  }
}

__global__ void __launch_bounds__(kQuantThreads)
    dequantize_mxfp4_kernel(const uint8_t* __restrict__ x4, int64_t ld4, const uint8_t* __restrict__ sf, int K,
                            int k2s, uint32_t per_row, uint32_t warps, __nv_bfloat16* __restrict__ out, int64_t ldo) {
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t warp = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  if (warp >= warps) return;
  const uint32_t row = warp / per_row;
  const int first = (int)(warp - row * per_row) * kUnits;
  const uint8_t* xi = x4 + row * ld4 + lane * 4;
  uint32_t c[kUnits], b[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int k2 = first + u;
    c[u] = b[u] = 0u;
    if (k2 * 256 + lane * 8 < K) {
      c[u] = *reinterpret_cast<const uint32_t*>(xi + k2 * 128);
      b[u] = sf[sf_word(row, 2 * k2 + (lane >> 4), 2 * k2s) + ((lane >> 2) & 3)];
    }
  }
  __nv_bfloat16* oo = out + row * ldo + lane * 8;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int k = (first + u) * 256;
    if (k + lane * 8 >= K) continue;
    const float s = scale_value(b[u]);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(c[u] >> (8 * j)), __NV_E2M1);
      const float2 f = __half22float2(__half2(h));
      o[j] = pack_bf16x2(f.x * s, f.y * s);
    }
    *reinterpret_cast<uint4*>(oo + k) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

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

void check_rows(const char* op, const char* what, const at::Tensor& x, const at::Device& dev) {
  GSB_CHECK(x.is_cuda() && x.device() == dev && x.scalar_type() == at::kBFloat16 && x.dim() == 2 &&
                (x.size(1) == 1 || x.stride(1) == 1) && (x.size(0) <= 1 || x.stride(0) % 8 == 0) && aligned16(x),
            op, ": ", what, " must be bf16 [M, K] on one CUDA device with 16-byte aligned rows");
  GSB_CHECK(x.size(1) >= kBlock && x.size(1) % kBlock == 0 && x.size(1) < (int64_t(1) << 31) &&
                x.size(0) < (int64_t(1) << 31),
            op, ": K must be a positive multiple of 32");
}

// Warps per row and in all, and the grid, of the streaming kernels.
struct StreamGrid {
  uint32_t per_row, warps;
  dim3 grid;
};
static StreamGrid stream_grid(const char* op, int64_t M, int64_t K) {
  const int64_t per_row = (k_tiles(K) / 2 + kUnits - 1) / kUnits, warps = M * per_row;
  GSB_CHECK(warps < (int64_t(1) << 32) - 64, op, ": too many rows");
  return {(uint32_t)per_row, (uint32_t)warps, dim3((unsigned)((warps + kQuantThreads / 32 - 1) / (kQuantThreads / 32)))};
}

void make_codes(int64_t M, int64_t K, const at::Device& dev, at::Tensor& x4, at::Tensor& sf) {
  const auto opt = at::TensorOptions().dtype(at::kByte).device(dev);
  if (!x4.defined()) x4 = at::empty({M, K / 2}, opt);
  if (!sf.defined()) sf = at::empty({(M + 127) / 128, k_tiles(K), 512}, opt);
}

void quantize_launch(const void* x, int64_t ldx, int64_t M, int64_t K, uint8_t* x4, int64_t ld4, uint8_t* sf,
                     cudaStream_t st) {
  const StreamGrid g = stream_grid("quantize_mxfp4", M, K);
  launch(quantize_mxfp4_kernel, g.grid, kQuantThreads, 0, 1, st, reinterpret_cast<const __nv_bfloat16*>(x), ldx,
         (int)K, (int)(k_tiles(K) / 2), g.per_row, g.warps, x4, ld4, sf);
}

}  // namespace f4
}  // namespace gsb

using namespace gsb;

// x [M, K] bf16 -> (x4 [M, K / 2] codes, sf [ceil(M / 128), 2 ceil(K / 256), 512] scale atoms).
std::tuple<at::Tensor, at::Tensor> gsb_quantize_mxfp4(const at::Tensor& x, const c10::optional<at::Tensor>& x4_,
                                                      const c10::optional<at::Tensor>& sf_) {
  f4::check_rows("quantize_mxfp4", "x", x, x.device());
  const int64_t M = x.size(0), K = x.size(1);
  c10::cuda::CUDAGuard g(x.device());
  at::Tensor x4 = x4_.value_or(at::Tensor()), sf = sf_.value_or(at::Tensor());
  f4::make_codes(M, K, x.device(), x4, sf);
  f4::check_codes("quantize_mxfp4", x4, sf, M, K, x.device());
  if (M > 0)
    f4::quantize_launch(x.data_ptr(), x.stride(0), M, K, x4.data_ptr<uint8_t>(), x4.stride(0), sf.data_ptr<uint8_t>(),
                        c10::cuda::getCurrentCUDAStream(x.device().index()).stream());
  return {x4, sf};
}

// RMSNorm of x [M, H] and its quantisation; `out` (optional) also receives the bf16 rows.
std::tuple<at::Tensor, at::Tensor> gsb_rmsnorm_mxfp4(const at::Tensor& x, const at::Tensor& w, double eps,
                                                     const c10::optional<at::Tensor>& x4_,
                                                     const c10::optional<at::Tensor>& sf_,
                                                     const c10::optional<at::Tensor>& out) {
  f4::check_rows("rmsnorm_mxfp4", "x", x, x.device());
  const int64_t M = x.size(0), H = x.size(1);
  GSB_CHECK(H <= 16384, "rmsnorm_mxfp4: at most 16384 columns");
  GSB_CHECK(w.device() == x.device() && w.scalar_type() == at::kBFloat16 && w.is_contiguous() && w.numel() == H &&
                f4::aligned16(w),
            "rmsnorm_mxfp4: the weight must be bf16 [H], contiguous and 16-byte aligned");
  c10::cuda::CUDAGuard g(x.device());
  at::Tensor x4 = x4_.value_or(at::Tensor()), sf = sf_.value_or(at::Tensor());
  f4::make_codes(M, H, x.device(), x4, sf);
  f4::check_codes("rmsnorm_mxfp4", x4, sf, M, H, x.device());
  __nv_bfloat16* op = nullptr;
  int64_t ldo = 0;
  if (out.has_value()) {
    f4::check_rows("rmsnorm_mxfp4", "out", *out, x.device());
    GSB_CHECK(out->size(0) == M && out->size(1) == H, "rmsnorm_mxfp4: out must be [M, H]");
    op = reinterpret_cast<__nv_bfloat16*>(out->data_ptr());
    ldo = out->stride(0);
  }
  if (M == 0) return {x4, sf};
  auto st = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  auto* xp = reinterpret_cast<const __nv_bfloat16*>(x.data_ptr());
  auto* wp = reinterpret_cast<const __nv_bfloat16*>(w.data_ptr());
  const int vpt = (int)((f4::k_tiles(H) * 16 + 255) / 256);
  auto go = [&](auto kernel) {
    f4::launch(kernel, dim3((unsigned)M), 256, 0, 1, st, xp, x.stride(0), wp, (int)H, (float)eps,
               x4.data_ptr<uint8_t>(), x4.stride(0), sf.data_ptr<uint8_t>(), op, ldo);
  };
  if (vpt <= 1) go(f4::rmsnorm_mxfp4_kernel<1>);
  else if (vpt <= 2) go(f4::rmsnorm_mxfp4_kernel<2>);
  else if (vpt <= 4) go(f4::rmsnorm_mxfp4_kernel<4>);
  else go(f4::rmsnorm_mxfp4_kernel<8>);
  return {x4, sf};
}

// out [M, K] bf16 <- codes x4 and scale atoms sf.
at::Tensor gsb_dequantize_mxfp4(const at::Tensor& x4, const at::Tensor& sf, const c10::optional<at::Tensor>& out_) {
  GSB_CHECK(x4.is_cuda() && x4.dim() == 2, "dequantize_mxfp4: codes must be a CUDA matrix");
  const int64_t M = x4.size(0), K = x4.size(1) * 2;
  c10::cuda::CUDAGuard g(x4.device());
  at::Tensor out = out_.has_value() ? *out_
                                    : at::empty({M, K}, at::TensorOptions().dtype(at::kBFloat16).device(x4.device()));
  f4::check_rows("dequantize_mxfp4", "out", out, x4.device());
  GSB_CHECK(out.size(0) == M && out.size(1) == K, "dequantize_mxfp4: out must be [M, K]");
  f4::check_codes("dequantize_mxfp4", x4, sf, M, K, x4.device());
  if (M == 0) return out;
  const f4::StreamGrid s = f4::stream_grid("dequantize_mxfp4", M, K);
  f4::launch(f4::dequantize_mxfp4_kernel, s.grid, f4::kQuantThreads, 0, 1,
             c10::cuda::getCurrentCUDAStream(x4.device().index()).stream(), x4.data_ptr<uint8_t>(), x4.stride(0),
             sf.data_ptr<uint8_t>(), (int)K, (int)(f4::k_tiles(K) / 2), s.per_row, s.warps,
             reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), out.stride(0));
  return out;
}
