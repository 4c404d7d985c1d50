// MXFP4 products of a few tokens on CUDA cores (included by gemm_fp4.cu).
//
// A few token rows give the tensor core nothing to do: the work is one pass over the weight's
// bytes, and the operand-swapped kernel's fixed costs (tensor memory, cluster barriers, a
// quantiser in front) are several times that pass. Here a CTA takes 16 weight rows a step, each
// one bulk copy into shared memory with every row in flight at once, a warp two of them, a
// lane one block of 32 codes (16 bytes) of each at a time, K split over the lanes.
// An integer dot product is exact: twice an e2m1 value is an integer of at most 12, so a
// block's 32 products sum to at most 4608 in int32, and one fp32 multiply-add applies the two
// scales' product. Codes become bytes by table lookup (prmt): the instruction's sign mode turns a
// code of the other sign into 0xff, so two lookups and an AND give 192 + 2 v as an unsigned byte;
// the 192 times the sum of x that this adds comes off once per block.
//
// The token rows are expanded to bytes in shared memory by every CTA (from bf16, quantised on
// the way, or from codes): they are a few KB against the weight's megabytes, and a separate
// quantiser would cost a launch.
#pragma once

#include "common.cuh"
#include "fp4.cuh"

namespace gsb {
namespace f4 {

constexpr int GV_THREADS = 256;
constexpr int GV_ROWS = 2;                               // weight rows per warp and step
constexpr int GV_STEP = GV_THREADS / 32 * GV_ROWS;       // weight rows per CTA and step: 16
constexpr int GV_MAX_M = 4;
constexpr int GV_MAX_STAGES = 4;

struct GemvParams {
  int M, N, kblocks;          // K / 32
  int stages;                 // steps in flight
  const __nv_bfloat16* x;     // bf16 rows, or null:
  int64_t ldx;
  const uint8_t* x4;          // codes and scales
  int64_t ld4;
  const uint8_t* sfx;
  const uint8_t* w4;
  int64_t ldw;
  const uint8_t* sfw;
  float scale;
  __nv_bfloat16* out;
  int64_t ldo;
  const __nv_bfloat16* residual;
  int64_t ldr;
  uint8_t* a4;
  int64_t lda4;
  uint8_t* sfa_out;
  int lora;
  const __nv_bfloat16* s;
  int64_t lds;
  const __nv_bfloat16* lb;
  int64_t ldlb;
};

// Four codes (the low 16 bits) -> 192 + 2 v as unsigned bytes.
__device__ __forceinline__ uint32_t code_bytes(uint32_t w) {
  // 2 v of the magnitudes: 0 1 2 3 4 6 8 12
  constexpr uint32_t p0 = 0xc3c2c1c0u, p1 = 0xccc8c6c4u;  // 192 + 2 v
  constexpr uint32_t n0 = 0xbdbebfc0u, n1 = 0xb4b8babcu;  // 192 - 2 v
  uint32_t p, n;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(p) : "r"(p0), "r"(p1), "r"(w));
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(n) : "r"(n0), "r"(n1), "r"(w ^ 0x8888u));
  return p & n;
}
// The same as signed bytes.
__device__ __forceinline__ uint32_t code_signed(uint32_t w) { return __vsub4(code_bytes(w), 0xc0c0c0c0u); }

__device__ __forceinline__ int dp4a_us(uint32_t a, uint32_t b, int c) {  // unsigned a, signed b
  int d;
  asm("dp4a.u32.s32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// 2^(e1 + e2 - 2) for two scale bytes, given byte 1 - 129 in `a` and byte 2 in `b`; a byte of
// 255 is passed as 100000 (or 99871). Below the normal range the product flushes to zero.
__device__ __forceinline__ float scale_product(int a, int b) {
  const int t = a + b;
  return t > 50000 ? __int_as_float(0x7fc00000) : __int_as_float(min(max(t, 0), 254) << 23);
}

// Shared memory: a ring of steps, each 16 rows of codes and, per row and K tile, the word of
// four scale bytes; then the tokens: bytes of token m's block b in two 16-byte halves,
// [m][half][kblocks], and per (m, b) the scale byte - 129 and 192 times the block's sum.
__host__ __device__ constexpr int gemv_stage(int kblocks) {
  return GV_STEP * (kblocks * 16 + (kblocks + 3) / 4 * 4 + 12) / 16 * 16;
}
__host__ __device__ constexpr int gemv_tokens(int MT, int kblocks) { return MT * kblocks * (32 + 8); }

template <int MT>
__device__ __forceinline__ void gemv_expand(const GemvParams& p, uint8_t* smem) {
  uint4* xb = reinterpret_cast<uint4*>(smem);
  int2* meta = reinterpret_cast<int2*>(smem + MT * p.kblocks * 32);
  const int ktiles = (p.kblocks + 7) / 8 * 2;
  // four lanes a block, eight values a lane; whole warps run every turn for the shuffles
  const int vecs = MT * p.kblocks * 4;
  for (int i = threadIdx.x; i < (vecs + 31) / 32 * 32; i += GV_THREADS) {
    const int at = min(i, vecs - 1), m = at / (p.kblocks * 4), v = at - m * p.kblocks * 4, b = v >> 2;
    const bool real = i < vecs && m < p.M;
    uint32_t code = 0u, byte = 0u;
    if (p.x != nullptr) {
      uint4 q = make_uint4(0u, 0u, 0u, 0u);
      if (real) q = *reinterpret_cast<const uint4*>(p.x + m * p.ldx + v * 8);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = unpack_bf16x2(w[j]);
        f[2 * j] = t.x;
        f[2 * j + 1] = t.y;
      }
      byte = scale_byte(quad_max(max_abs_bits(f)));
      code = byte == 255u ? 0u : pack8(f, inv_scale(byte));
    } else if (real) {
      code = *reinterpret_cast<const uint32_t*>(p.x4 + m * p.ld4 + v * 4);
      byte = p.sfx[sf_word(m, b >> 2, ktiles) + (b & 3)];
    }
    const uint32_t lo = code_signed(code), hi = code_signed(code >> 16);
    int sum = __dp4a((int)lo, 0x01010101, __dp4a((int)hi, 0x01010101, 0));
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (i < vecs) {
      uint2* dst = reinterpret_cast<uint2*>(xb + (m * 2 + ((v >> 1) & 1)) * p.kblocks + b) + (v & 1);
      *dst = make_uint2(lo, hi);
      if ((v & 3) == 0) meta[m * p.kblocks + b] = make_int2(byte == 255u ? 100000 : (int)byte - 129, 192 * sum);
    }
  }
}

// This warp's rows of a step (`codes` and `words`, the scales, of its first row, n0 its index)
// against every token, summed over the warp; lane r * MT + m of the first GV_ROWS * MT gets its
// value.
template <int MT>
__device__ __forceinline__ float gemv_rows(const GemvParams& p, const uint8_t* tokens, const uint8_t* codes,
                                           const uint8_t* words, int n0, int lane, uint64_t amask,
                                           const LoraParams& lp) {
  const uint4* xb = reinterpret_cast<const uint4*>(tokens);
  const int2* meta = reinterpret_cast<const int2*>(tokens + MT * p.kblocks * 32);
  const int row_bytes = p.kblocks * 16, row_words = (p.kblocks + 3) / 4 * 4;
  float acc[GV_ROWS][MT];
#pragma unroll
  for (int r = 0; r < GV_ROWS; ++r)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[r][m] = 0.f;
#pragma unroll 2
  for (int b = lane; b < p.kblocks; b += 32) {
    uint4 w[GV_ROWS];
    int sb[GV_ROWS];
#pragma unroll
    for (int r = 0; r < GV_ROWS; ++r) {
      w[r] = *reinterpret_cast<const uint4*>(codes + r * row_bytes + b * 16);
      sb[r] = words[r * row_words + b];
      sb[r] = sb[r] == 255 ? 100000 : sb[r];
    }
    int dot[GV_ROWS][MT];
    int2 mt[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      mt[m] = meta[m * p.kblocks + b];
#pragma unroll
      for (int r = 0; r < GV_ROWS; ++r) dot[r][m] = -mt[m].y;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 xv[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) xv[m] = xb[(m * 2 + h) * p.kblocks + b];
#pragma unroll
      for (int r = 0; r < GV_ROWS; ++r) {
        const uint32_t w0 = h ? w[r].z : w[r].x, w1 = h ? w[r].w : w[r].y;
        const uint32_t c[4] = {code_bytes(w0), code_bytes(w0 >> 16), code_bytes(w1), code_bytes(w1 >> 16)};
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          dot[r][m] = dp4a_us(c[0], xv[m].x, dot[r][m]);
          dot[r][m] = dp4a_us(c[1], xv[m].y, dot[r][m]);
          dot[r][m] = dp4a_us(c[2], xv[m].z, dot[r][m]);
          dot[r][m] = dp4a_us(c[3], xv[m].w, dot[r][m]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < GV_ROWS; ++r)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[r][m] = fmaf((float)dot[r][m], scale_product(mt[m].x, sb[r]), acc[r][m]);
  }
  if (p.lora) {
    const int base = slice_base(lp, n0), blocks = __popcll(amask) * lp.blocks_per_adapter;
    for (int j = 0; j < blocks; ++j) {
      int bit;
      const int col = lora_column(lp, amask, j, bit) + lane;
      float sv[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) sv[m] = m < p.M ? bf2f(p.s[m * p.lds + base + col]) : 0.f;
#pragma unroll
      for (int r = 0; r < GV_ROWS; ++r) {
        const float l = bf2f(p.lb[(int64_t)(n0 + r) * p.ldlb + col]);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[r][m] = fmaf(sv[m], l, acc[r][m]);
      }
    }
  }
  float mine = 0.f;
#pragma unroll
  for (int r = 0; r < GV_ROWS; ++r)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float t = warp_sum(acc[r][m]);
      if (lane == r * MT + m) mine = t;
    }
  return mine;
}

template <int MT, int EPI>
__global__ void __launch_bounds__(GV_THREADS) mxfp4_gemv_kernel(const GemvParams p, const LoraParams lp, uint32_t* err) {
  extern __shared__ uint4 gemv_shared[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(gemv_shared);
  __shared__ uint64_t full_bar[GV_MAX_STAGES];
  __shared__ float tile[EPI == kEpiSwiGLU ? MT : 1][64];  // swiglu: 32 gate rows, 32 up rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stage_bytes = gemv_stage(p.kblocks), row_bytes = p.kblocks * 16, tiles = (p.kblocks + 3) / 4;
  uint8_t* tokens = smem + p.stages * stage_bytes;
  // A unit is 16 rows or, for swiglu, one block of 32 outputs: 32 gate rows and the 32 up rows
  // 64 further on, in four steps.
  constexpr int STEPS = EPI == kEpiSwiGLU ? 64 / GV_STEP : 1;
  const int units = EPI == kEpiSwiGLU ? p.N / 64 : (p.N + GV_STEP - 1) / GV_STEP;
  const int my_units = (units - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x, total = my_units * STEPS;
  auto first_row = [&](int i) {
    const int u = (int)blockIdx.x + i / STEPS * (int)gridDim.x, step = i % STEPS;
    if (EPI != kEpiSwiGLU) return u * GV_STEP;
    const int at = step * GV_STEP;  // 0..31 gate, 32..63 up
    return (u >> 1) * 128 + (u & 1) * 32 + (at < 32 ? at : at + 32);
  };
  // step i into its stage: one bulk copy a row, four bytes a scale word
  auto fetch = [&](int i) {
    if (i < total) {
      const int s = i % p.stages, n0 = first_row(i), rows = min(GV_STEP, p.N - n0);
      uint8_t* codes = smem + s * stage_bytes;
      if (warp == 0) {
        if (lane == 0) mbar_arrive_expect_tx(&full_bar[s], rows * row_bytes);
        __syncwarp();
        if (lane < rows)
          bulk_load(codes + lane * row_bytes, p.w4 + (int64_t)(n0 + lane) * p.ldw, row_bytes, &full_bar[s]);
      }
      const uint8_t* src = p.sfw + sf_word(n0, 0, (p.kblocks + 7) / 8 * 2);  // 16 rows of one group of 32
      const uint32_t dst = smem_u32(codes + GV_STEP * row_bytes);
      for (int j = threadIdx.x; j < tiles * GV_STEP; j += GV_THREADS) {
        const int r = j % GV_STEP, t = j / GV_STEP;  // rows past N have words too (whole atoms)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + (r * tiles + t) * 4),
                     "l"(src + (int64_t)t * 512 + r * 16)
                     : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full_bar[s], 1);
    fence_barrier_init();
  }
  // Towards L2 before the wait for the kernel before this one (reads nothing that could be stale).
  if (warp == 0 && lane < GV_STEP && first_row(0) + lane < p.N)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.w4 + (int64_t)(first_row(0) + lane) * p.ldw),
                 "r"(row_bytes)
                 : "memory");
  griddep_launch();
  griddep_wait();
  __syncthreads();
  for (int i = 0; i < GV_MAX_STAGES; ++i)
    if (i < p.stages) fetch(i);
  const uint64_t amask = p.lora ? tile_adapters(lp, 0, 1) : 0ull;
  gemv_expand<MT>(p, tokens);
  bool ok = true;
  const int64_t kt = k_tiles(p.N / 2);
  for (int i = 0; i < total; ++i) {
    const int s = i % p.stages, n0 = first_row(i) + warp * GV_ROWS;
    // all groups but the (stages - 1) youngest: this step's scales have landed
    switch (p.stages) {
      case 1: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
      case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
      case 3: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
      default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    }
    ok = ok && mbar_wait(&full_bar[s], (i / p.stages) & 1, err, kErrGemmWait);  // after one that ran out: no more waits
    __syncthreads();
    const uint8_t* codes = smem + s * stage_bytes;
    if (n0 < p.N) {  // N is a multiple of 8
      float v = gemv_rows<MT>(p, tokens, codes + warp * GV_ROWS * row_bytes,
                              codes + GV_STEP * row_bytes + warp * GV_ROWS * tiles * 4, n0, lane, amask, lp);
      const int r = lane / MT, m = lane % MT;
      if (EPI == kEpiSwiGLU) {
        if (r < GV_ROWS) tile[m][i % STEPS * GV_STEP + warp * GV_ROWS + r] = v;
      } else if (r < GV_ROWS && m < p.M) {
        v *= p.scale;
        if (EPI == kEpiResAdd) v += bf2f(p.residual[m * p.ldr + n0 + r]);
        p.out[m * p.ldo + n0 + r] = f2bf(v);
      }
    }
    if (i + p.stages < total || EPI == kEpiSwiGLU) __syncthreads();  // the stage is read, the tile written
    fetch(i + p.stages);
    if (EPI == kEpiSwiGLU && i % STEPS == STEPS - 1) {
      const int g = (int)blockIdx.x + i / STEPS * (int)gridDim.x;
      for (int m = warp; m < p.M; m += GV_THREADS / 32) {
        const float v = swiglu_f(tile[m][lane], tile[m][32 + lane]);
        uint32_t top = __float_as_uint(v) & 0x7fffffffu;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t byte = scale_byte(top);
        if (p.out != nullptr) p.out[m * p.ldo + g * 32 + lane] = f2bf(v);
        const float t = byte == 255u ? 0.f : v * inv_scale(byte);
        const uint32_t code = __nv_cvt_float_to_fp4(t, __NV_E2M1, cudaRoundNearest);
        const uint32_t next = __shfl_down_sync(0xffffffffu, code, 1);
        if ((lane & 1) == 0) p.a4[m * p.lda4 + g * 16 + lane / 2] = (uint8_t)(code | (next << 4));
        if (lane == 0) {
          p.sfa_out[sf_word(m, g >> 2, kt) + (g & 3)] = (uint8_t)byte;
          if (g == units - 1)  // scales past the row's end
            for (int b = units; b < kt * 4; ++b) p.sfa_out[sf_word(m, b >> 2, kt) + (b & 3)] = 0;
        }
      }
      // the next write to the tile is behind the next step's first barrier
    }
  }
  if (!ok) {
    // error path: copies this CTA issued may still be in flight (bounded, ~1 ms)
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) {
    }
  }
}

}  // namespace f4
}  // namespace gsb
