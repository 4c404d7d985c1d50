// MXFP4 quantisation of bf16 rows, the same fused behind RMSNorm, and the way back
// (format: fp4.cuh). All three stream their rows once.
//
//   quantize_mxfp4: a warp takes 256 neighbours of a row, eight per lane (one 16-byte
//     load), so a block of 32 is four lanes and its maximum two shuffles; one, two or four such
//     units are in flight per warp. 8192 x 12800 rows: 45 us, 5.9 TB/s, 0.91 of the measured copy.
//   rmsnorm_mxfp4: the row in registers between the sum of squares and the conversion.
//     y = x w / sqrt(mean(x^2) + eps) in fp32 (the product x w is exact), then one rounding, to
//     4 bits; with `out` the row also leaves as bf16, rounded exactly as the RMSNorm kernel does,
//     for the LoRA shrink. 8192 x 4096 rows: 19.1 us, 4.4 TB/s, bound by instruction issue (2.75 of
//     4 a cycle: unpacking, squares, products, maxima and conversions of every value); with `out`
//     29.1 us, 5.2 TB/s.
//   dequantize_mxfp4: codes times scale, exact in bf16. 8192 x 12800 rows: 42 us, 6.4 TB/s.
#include "common.cuh"
#include "fp4.cuh"
#include "fp4_host.h"
#include "tma_util.h"

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <tuple>
#include <utility>

namespace gsb {
namespace f4 {

constexpr int kSms = 148;
constexpr int kQuantThreads = 256;

// Warp `blockIdx.x * 8 + ..` takes UNITS units of one row; `per_row` warps make a row.
template <int UNITS>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_mxfp4_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int K, int k2s, uint32_t per_row,
                          uint32_t warps, uint8_t* __restrict__ x4, int64_t ld4, uint8_t* __restrict__ sf) {
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t warp = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  if (warp >= warps) return;
  const uint32_t row = warp / per_row;
  const int first = (int)(warp - row * per_row) * UNITS;
  const __nv_bfloat16* xr = x + row * ldx + lane * 8;
  uint4 q[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int k = (first + u) * 256;
    q[u] = make_uint4(0u, 0u, 0u, 0u);
    if (k + lane * 8 < K) q[u] = *reinterpret_cast<const uint4*>(xr + k);
  }
  uint8_t* xo = x4 + row * ld4 + lane * 4;
  uint8_t* so = sf + sf_word(row, 2 * first, 2 * k2s);
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
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

// The norm kernel's NT threads hold VPT 16-byte vectors of a row each. Up to 4096 columns 128 threads
// share a row's fixed instructions among more values than 256 would (8192 x 4096 19.4 against 21.2 us,
// 8192 x 2048 12.2 against 14.5, 16 x 4096 1.70 against 1.65). Rows in flight per CTA, and resident
// CTAs per SM (what the registers allow without spills):
__host__ __device__ constexpr int norm_stages(int vpt) { return vpt <= 4 ? 4 : 2; }
__host__ __device__ constexpr int norm_ctas(int vpt, int nt) { return nt == 256 ? 2 : (vpt <= 2 ? 8 : 5); }

// Persistent: a CTA walks rows, each thread copying its own vectors of the next rows into shared
// memory (cp.async; a thread reads only what it copied, so that needs no barrier) and keeping
// the weight in registers; one barrier a row, for the sum of squares, which is added in the order
// of the RMSNorm kernel.
//
// A block's maximum is taken of the exact products x w, before the sum is known: rounding keeps
// order, so it is the normalised block's after one multiplication. inv and the block's power of
// two then make one factor, and each value is rounded once, by that product's conversion.
template <int NT, int VPT, bool OUT>
__global__ void __launch_bounds__(NT, norm_ctas(VPT, NT))
    rmsnorm_mxfp4_kernel(const __nv_bfloat16* __restrict__ x, int ldx, const __nv_bfloat16* __restrict__ w, int M, int H,
                         float eps, uint8_t* __restrict__ x4, int ld4, uint8_t* __restrict__ sf,
                         __nv_bfloat16* __restrict__ out, int ldo) {
  constexpr int STAGES = norm_stages(VPT);
  constexpr int GROUPS = 256 / NT;  // threads of the RMSNorm kernel that one thread stands for
  extern __shared__ uint4 ring[];  // [STAGES][VPT][NT]
  __shared__ float4 red[2][2];
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x, lane = tid & 31;
  const int nvec = H / 8, units = (int)k_tiles(H) / 2;
  const uint4* xv = reinterpret_cast<const uint4*>(x) + tid;
  uint4* slots = ring + tid;
  constexpr bool KEEP = VPT <= 4;  // fp32 weights and products stay in registers, or are formed again
  uint4 wq[KEEP ? 1 : VPT];
  uint64_t wf[KEEP ? VPT : 1][4];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * NT;
    const uint4 q = v < nvec ? reinterpret_cast<const uint4*>(w)[v] : make_uint4(0u, 0u, 0u, 0u);
    if constexpr (KEEP) unpack_pairs(q, wf[i]);
    else wq[i] = q;
    if (v >= nvec)  // past the row: zeros for good
      for (int s = 0; s < STAGES; ++s) slots[(s * VPT + i) * NT] = make_uint4(0u, 0u, 0u, 0u);
  }
  auto fetch = [&](int r, int s) {
    if (r < M) {
      const uint4* src = xv + (int64_t)r * (ldx / 8);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (tid + i * NT < nvec)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(slots + (s * VPT + i) * NT)),
                       "l"(src + i * NT)
                       : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int grid = (int)gridDim.x;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch((int)blockIdx.x + s * grid, s);
  // where this thread's codes and its warp's scale words lie in a row
  uint8_t* codes0 = x4 + tid * 4;
  uint8_t* scales0 = sf + (tid >> 5) * 1024 + (lane >> 4) * 512 + ((lane >> 2) & 3);
  const int atom_row = units * 1024;  // bytes of 128 rows' scales
  int slot = 0, parity = 0;
  for (int r = (int)blockIdx.x; r < M; r += grid) {
    // the slot read last turn is free: this thread's reads of it went into values used since
    fetch(r + (STAGES - 1) * grid, slot == 0 ? STAGES - 1 : slot - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    const uint4* xs = slots + slot * VPT * NT;
    uint64_t y[KEEP ? VPT : 1][4];
    uint32_t top[VPT];
    float ss[GROUPS] = {};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      uint64_t f[4], g[4];
      unpack_pairs(xs[i * NT], f);
      if constexpr (!KEEP) unpack_pairs(wq[i], g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float lo = f32x2_lo(f[j]), hi = f32x2_hi(f[j]);
        ss[i % GROUPS] += lo * lo + hi * hi;
        f[j] = f32x2_mul(f[j], KEEP ? wf[KEEP ? i : 0][j] : g[j]);
        if (KEEP) y[KEEP ? i : 0][j] = f[j];
      }
      const float t = max_abs3(max_abs3(f32x2_lo(f[0]), f32x2_hi(f[0]), f32x2_lo(f[1])),
                               max_abs3(f32x2_hi(f[1]), f32x2_lo(f[2]), f32x2_hi(f[2])),
                               max_abs3(f32x2_lo(f[3]), f32x2_hi(f[3]), f32x2_hi(f[3])));
      top[i] = quad_max(__float_as_uint(t) & 0x7fffffffu);
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) ss[g] = warp_sum(ss[g]);
    if (lane == 0)
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) reinterpret_cast<float*>(red[parity])[(tid >> 5) + g * (NT / 32)] = ss[g];
    __syncthreads();
    const float4 a = red[parity][0], b = red[parity][1];
    const float sum = ((a.x + b.x) + (a.z + b.z)) + ((a.y + b.y) + (a.w + b.w));
    const float inv = rsqrtf(sum / (float)H + eps);
    uint8_t* codes = codes0 + (int64_t)r * ld4;
    uint8_t* scales = scales0 + (int64_t)(r >> 7) * atom_row + (16 * (r & 31) + 4 * ((r >> 5) & 3));
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if ((tid >> 5) + i * (NT / 32) >= units) break;  // the whole warp
      const bool inside = tid + i * NT < nvec;
      uint32_t byte = scale_byte(__float_as_uint(__uint_as_float(top[i]) * inv));
      byte = inside ? byte : 0u;  // past the row (whole blocks): inv is NaN in a row that is not finite
      float s = inv_scale(byte);
      uint64_t v[4], g[4];
      if constexpr (!KEEP) {
        unpack_pairs(xs[i * NT], v);
        unpack_pairs(wq[i], g);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = KEEP ? y[KEEP ? i : 0][j] : f32x2_mul(v[j], g[j]);
      if (byte < 32u) {  // inv * 2^-e may overflow
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = f32x2_mul(v[j], f32x2_pack(inv, inv));
      } else {
        s *= inv;
      }
      const uint32_t c = pack8(v, s);
      if (inside) *reinterpret_cast<uint32_t*>(codes + i * NT * 4) = byte == 255u ? 0u : c;
      // a block's lanes hold its byte alike; the first stores it
      if ((lane & 3) == 0) scales[i * (NT / 32) * 1024] = (uint8_t)byte;
      if (OUT && inside) {
        float f[8];
        unpack8(xs[i * NT], f);
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t gj = KEEP ? wf[KEEP ? i : 0][j] : g[j];
          o[j] = pack_bf16x2(__bfloat162float(__float2bfloat16_rn(f[2 * j] * inv)) * f32x2_lo(gj),
                             __bfloat162float(__float2bfloat16_rn(f[2 * j + 1] * inv)) * f32x2_hi(gj));
        }
        reinterpret_cast<uint4*>(out + (int64_t)r * ldo)[tid + i * NT] = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
    slot = slot + 1 == STAGES ? 0 : slot + 1;
    parity ^= 1;
  }
}

template <int UNITS>
__global__ void __launch_bounds__(kQuantThreads)
    dequantize_mxfp4_kernel(const uint8_t* __restrict__ x4, int64_t ld4, const uint8_t* __restrict__ sf, int K,
                            int k2s, uint32_t per_row, uint32_t warps, __nv_bfloat16* __restrict__ out, int64_t ldo) {
  // No early griddep_launch(): the rows may be the next product's weights, which the decode GEMM
  // reads before it waits for the kernel ahead of it (and for any kernel that one lets run on).
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t warp = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  if (warp >= warps) return;
  const uint32_t row = warp / per_row;
  const int first = (int)(warp - row * per_row) * UNITS;
  const uint8_t* xi = x4 + row * ld4 + lane * 4;
  uint32_t c[UNITS], b[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int k2 = first + u;
    c[u] = b[u] = 0u;
    if (k2 * 256 + lane * 8 < K) {
      c[u] = *reinterpret_cast<const uint32_t*>(xi + k2 * 128);
      b[u] = sf[sf_word(row, 2 * k2 + (lane >> 4), 2 * k2s) + ((lane >> 2) & 3)];
    }
  }
  __nv_bfloat16* oo = out + row * ldo + lane * 8;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
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
                x4.stride(1) == 1 && x4.stride(0) % 16 == 0 && (M <= 1 || x4.stride(0) >= x4.size(1)) &&
                x4.stride(0) < (int64_t(1) << 31) && aligned16(x4),
            op, ": codes must be uint8 [M, K / 2] with 16-byte aligned rows");
  GSB_CHECK(sf.scalar_type() == at::kByte && sf.is_contiguous() && aligned16(sf) &&
                sf.numel() == (M + 127) / 128 * k_tiles(K) * 512,
            op, ": scales must be uint8 atoms [ceil(M / 128), 2 ceil(K / 256), 512]");
}

void check_rows(const char* op, const char* what, const at::Tensor& x, const at::Device& dev) {
  GSB_CHECK(x.is_cuda() && x.device() == dev && x.scalar_type() == at::kBFloat16 && x.dim() == 2 &&
                (x.size(1) == 1 || x.stride(1) == 1) && (x.size(0) <= 1 || (x.stride(0) % 8 == 0 && std::abs(x.stride(0)) < (int64_t(1) << 31))) && aligned16(x),
            op, ": ", what, " must be bf16 [M, K] on one CUDA device with 16-byte aligned rows");
  GSB_CHECK(x.size(1) >= kBlock && x.size(1) % kBlock == 0 && x.size(1) < (int64_t(1) << 31) &&
                x.size(0) < (int64_t(1) << 31),
            op, ": K must be a positive multiple of 32");
}

// How a streaming kernel covers [M, K]: units of 256 values per warp, warps per row and in all, CTAs.
struct StreamPlan {
  int units;
  uint32_t per_row, warps;
  dim3 grid;
};
// Many rows are bound by memory, and four units a warp keep enough loads in flight; few are bound by
// one warp's chain of loads, shuffles and stores, which more and shorter warps take at once. us with
// 1 / 2 / 4 units, quantising: 16 x 4096 1.24 / 1.40 / 1.66, 1003 x 2080 2.4 / 3.0 / 3.1, 1537 x 2048 3.4 /
// 3.5 / 3.6, 1024 x 4096 4.0 / 3.5 / 4.3, 2048 x 4096 6.9 / 5.5 / 5.5, 8192 x 4096 22.5 / 17.5 / 15.7.
static StreamPlan stream_plan(const char* op, int64_t M, int64_t K) {
  const int64_t row_units = k_tiles(K) / 2, all = M * row_units;
  const int units = all <= 12800 ? 1 : (all <= 32000 ? 2 : 4);
  const int64_t per_row = (row_units + units - 1) / units, warps = M * per_row;
  GSB_CHECK(warps < (int64_t(1) << 32) - 64, op, ": too many rows");
  return {units, (uint32_t)per_row, (uint32_t)warps,
          dim3((unsigned)((warps + kQuantThreads / 32 - 1) / (kQuantThreads / 32)))};
}

void make_codes(int64_t M, int64_t K, const at::Device& dev, at::Tensor& x4, at::Tensor& sf) {
  const int64_t codes = (M * (K / 2) + 127) / 128 * 128, m_tiles = (M + 127) / 128;
  if (!x4.defined() && !sf.defined()) {
    // one allocation for both: a second one costs a sixth of a small call
    x4 = new_tensor({codes + m_tiles * k_tiles(K) * 512}, at::kByte, dev);
    auto scales = c10::make_intrusive<c10::TensorImpl>(c10::Storage(x4.storage()), x4.key_set(), x4.dtype());
    scales->set_storage_offset(codes);
    scales->set_sizes_contiguous({m_tiles, k_tiles(K), 512});
    sf = at::Tensor(std::move(scales));
    x4.unsafeGetTensorImpl()->set_sizes_contiguous({M, K / 2});
    return;
  }
  if (!x4.defined()) x4 = new_tensor({M, K / 2}, at::kByte, dev);
  if (!sf.defined()) sf = new_tensor({m_tiles, k_tiles(K), 512}, at::kByte, dev);
}

void quantize_launch(const void* x, int64_t ldx, int64_t M, int64_t K, uint8_t* x4, int64_t ld4, uint8_t* sf,
                     cudaStream_t st) {
  const StreamPlan g = stream_plan("quantize_mxfp4", M, K);
  const auto kernel = g.units == 1   ? quantize_mxfp4_kernel<1>
                      : g.units == 2 ? quantize_mxfp4_kernel<2>
                                     : quantize_mxfp4_kernel<4>;
  launch(kernel, g.grid, kQuantThreads, 0, 1, st, reinterpret_cast<const __nv_bfloat16*>(x), ldx, (int)K,
         (int)(k_tiles(K) / 2), g.per_row, g.warps, x4, ld4, sf);
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
  if (x4_.has_value() || sf_.has_value()) {
    f4::check_apart("quantize_mxfp4", "codes", x4, "x", x);
    f4::check_apart("quantize_mxfp4", "scales", sf, "x", x);
    f4::check_apart("quantize_mxfp4", "scales", sf, "the codes", x4);
  }
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
  if (x4_.has_value() || sf_.has_value()) {
    for (const at::Tensor* o : {&x4, &sf}) {
      f4::check_apart("rmsnorm_mxfp4", "codes and scales", *o, "x", x);
      f4::check_apart("rmsnorm_mxfp4", "codes and scales", *o, "the weight", w);
    }
    f4::check_apart("rmsnorm_mxfp4", "scales", sf, "the codes", x4);
  }
  __nv_bfloat16* op = nullptr;
  int64_t ldo = 0;
  GSB_CHECK(M < (int64_t(1) << 30), "rmsnorm_mxfp4: too many rows");
  if (out.has_value()) {
    f4::check_rows("rmsnorm_mxfp4", "out", *out, x.device());
    GSB_CHECK(out->size(0) == M && out->size(1) == H && (M <= 1 || out->stride(0) >= H),
              "rmsnorm_mxfp4: out must be [M, H] with rows of their own");
    f4::check_same_or_apart("rmsnorm_mxfp4", "out", *out, "x, unless it is x", x);
    f4::check_apart("rmsnorm_mxfp4", "out", *out, "the weight", w);
    f4::check_apart("rmsnorm_mxfp4", "out", *out, "the codes", x4);
    f4::check_apart("rmsnorm_mxfp4", "out", *out, "the scales", sf);
    op = reinterpret_cast<__nv_bfloat16*>(out->data_ptr());
    ldo = out->stride(0);
  }
  if (M == 0) return {x4, sf};
  auto st = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  auto* xp = reinterpret_cast<const __nv_bfloat16*>(x.data_ptr());
  auto* wp = reinterpret_cast<const __nv_bfloat16*>(w.data_ptr());
  const int vectors = (int)f4::k_tiles(H) * 16;  // with those that pad the row to 256 columns
  auto go = [&](auto kernel, int nt, int v) {
    const int smem = f4::norm_stages(v) * v * nt * 16;
    if (smem > 48 * 1024)  // per device and cheap: no cache
      GSB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const int64_t ctas = std::min<int64_t>(M, (int64_t)f4::norm_ctas(v, nt) * f4::kSms);
    f4::launch(kernel, dim3((unsigned)ctas), nt, smem, 1, st, xp, (int)x.stride(0), wp, (int)M, (int)H, (float)eps,
               x4.data_ptr<uint8_t>(), (int)x4.stride(0), sf.data_ptr<uint8_t>(), op, (int)ldo);
  };
  auto pick = [&](auto plain, auto with_out, int nt, int v) { op == nullptr ? go(plain, nt, v) : go(with_out, nt, v); };
  if (vectors <= 256) pick(f4::rmsnorm_mxfp4_kernel<128, 2, false>, f4::rmsnorm_mxfp4_kernel<128, 2, true>, 128, 2);
  else if (vectors <= 512) pick(f4::rmsnorm_mxfp4_kernel<128, 4, false>, f4::rmsnorm_mxfp4_kernel<128, 4, true>, 128, 4);
  else if (vectors <= 1024) pick(f4::rmsnorm_mxfp4_kernel<256, 4, false>, f4::rmsnorm_mxfp4_kernel<256, 4, true>, 256, 4);
  else pick(f4::rmsnorm_mxfp4_kernel<256, 8, false>, f4::rmsnorm_mxfp4_kernel<256, 8, true>, 256, 8);
  return {x4, sf};
}

// out [M, K] bf16 <- codes x4 and scale atoms sf.
at::Tensor gsb_dequantize_mxfp4(const at::Tensor& x4, const at::Tensor& sf, const c10::optional<at::Tensor>& out_) {
  GSB_CHECK(x4.is_cuda() && x4.dim() == 2, "dequantize_mxfp4: codes must be a CUDA matrix");
  const int64_t M = x4.size(0), K = x4.size(1) * 2;
  c10::cuda::CUDAGuard g(x4.device());
  at::Tensor out = out_.has_value() ? *out_
                                    : f4::new_tensor({M, K}, at::kBFloat16, x4.device());
  f4::check_rows("dequantize_mxfp4", "out", out, x4.device());
  GSB_CHECK(out.size(0) == M && out.size(1) == K && (M <= 1 || out.stride(0) >= K),
            "dequantize_mxfp4: out must be [M, K] with rows of their own");
  f4::check_codes("dequantize_mxfp4", x4, sf, M, K, x4.device());
  if (out_.has_value()) {
    f4::check_apart("dequantize_mxfp4", "out", out, "the codes", x4);
    f4::check_apart("dequantize_mxfp4", "out", out, "the scales", sf);
  }
  if (M == 0) return out;
  const f4::StreamPlan s = f4::stream_plan("dequantize_mxfp4", M, K);
  const auto kernel = s.units == 1   ? f4::dequantize_mxfp4_kernel<1>
                      : s.units == 2 ? f4::dequantize_mxfp4_kernel<2>
                                     : f4::dequantize_mxfp4_kernel<4>;
  f4::launch(kernel, s.grid, f4::kQuantThreads, 0, 1,
             c10::cuda::getCurrentCUDAStream(x4.device().index()).stream(), x4.data_ptr<uint8_t>(), x4.stride(0),
             sf.data_ptr<uint8_t>(), (int)K, (int)(f4::k_tiles(K) / 2), s.per_row, s.warps,
             reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), out.stride(0));
  return out;
}
