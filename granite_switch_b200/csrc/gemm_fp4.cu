// MXFP4 GEMM with the switched-LoRA expand in the same accumulator (tcgen05, TMEM, TMA).
//
//   out[M, N] = epi( X4 . W4^T  (e2m1, one UE8M0 scale per 32 along K)  +  S . LB^T  (bf16) )
//
// Format of X4, W4 and their scale atoms: fp4.cuh. The MMA is tcgen05.mma
// kind::mxf4.block_scale with two scales per K = 64 step, so dequantisation costs
// nothing in the main loop; the LoRA expand appends kind::f16 MMAs to the same fp32
// accumulator. Epilogues, each with one rounding:
//   store    bf16(acc * scale)
//   resadd   bf16(residual + acc * scale)
//   swiglu   silu(gate) * up quantised to MXFP4 (and, on request, stored as bf16); the
//            weight rows alternate in runs of 64: gate, up
//
// Two kernels: the split kernel for few tokens, bound by the stream of weight bytes and by its
// own latencies, and the pair kernel for many, bound by the tensor core (use_pair below).
//
// Split kernel: operands swapped, the MMA's 128-row side a tile of weight rows and its N
// side up to 128 tokens, so a weight byte is read once per token tile, whatever the tokens'
// number. The K range of a tile is split over the CTAs of a cluster when the tiles alone do not
// fill the SMs; partial sums meet in distributed shared memory in a fixed order, so results
// do not depend on timing.
//
// Warp roles (192 threads): warp 0 issues the TMA and bulk loads into a ring of
// stages (256 K elements each), warp 1 owns the tensor memory and issues the scale
// copies and MMAs, warps 2..5 drain the accumulator; all warps run the epilogue.
// Every wait is bounded; a CTA that gives up still arrives at the cluster barriers, and tells its
// cluster, which then stores nothing of that tile: its sums would lack that CTA's part.
//
// What bounds it (B200, CUDA-graph replays over rotating weights): its own chain of latencies
// more than the bytes. 1 x 4096 x 4096 takes 5.2 us (the codes' and scales' bytes 1.4 us at the
// measured copy rate), 16 x 4096 x 12800 9.3 us (4.3 us), 128 x 4096 x 4096 7.6 us, 222 x 4096 x 12800
// 13.8 us, SwiGLU over 25600 x 4096 with 1 / 64 / 128 rows 12.4 / 13.8 / 16.2 us (8.6 us). Of a
// 16 x 4096 x 4096 launch 0.7 us are set-up, 1.2 us pass until the first stage lands, 1.8 us
// stream four stages per CTA, and about 1.5 us go into the cluster's reduction and the stores.
// A plain read of the weights' bytes, launched the same way, takes 9.8 us for 25600 x 4096 and 5.6 us
// for 4096 x 12800: what is left is that chain. Three CTAs per SM (200 tiles in two K parts, evener
// over the SMs) changed nothing, a prefetch of all the weights before the wait cost 4 to 14%.
#include "common.cuh"
#include "fp4.cuh"
#include "fp4_host.h"
#include "gemm_common.cuh"
#include "tma_util.h"

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <tuple>
#include <utility>
#include <vector>

namespace gsb {
namespace f4 {

constexpr int BW = 128;        // weight rows per tile (the MMA's M)
constexpr int BT = 128;        // tokens per tile (the MMA's N), at most
constexpr int BKB = 128;       // bytes of K per stage: 256 elements
constexpr int THREADS = 192;
constexpr int MAX_STAGES = 8;
constexpr int MAX_KS = 8;      // portable cluster size
constexpr int W_BYTES = BW * BKB;
constexpr int SF_BYTES = 1024;  // a stage's two scale atoms
constexpr int SF_COLS = 16;     // tensor memory columns of a stage's scales: weights 8, tokens 8
constexpr int P_STRIDE = BW;
constexpr int SMEM_LIMIT = 227 * 1024;
constexpr int BAR_BYTES = 256;

struct LoraParams {
  int blocks_per_adapter;  // rank / 32, times the two halves for swiglu
  int rank_blocks, num_adapters, num_slices;
  int slice_bounds[5];
  const uint64_t* tile_mask;  // [ceil(M / 128)] adapters present per 128 rows, or null: all
};

struct SplitParams {
  int M, N, kstages, stages, stage_bytes;
  int mt_rows;        // tokens per tile
  int ks, rows_per;   // K parts per tile (cluster size), tokens per part in the reduction
  int tmem_cols;
  int reduce_off;     // offset of the reduction buffer: 0 (over the ring) or behind it
  int give_up;        // K part that reports a wait that ran out, at once (tests), or -1
  const uint8_t* sfx;
  const uint8_t* sfw;
  float scale;
  void* out;          // bf16 [M, N]; swiglu: bf16 [M, N / 2] or null
  int64_t ldo;
  const __nv_bfloat16* residual;
  int64_t ldr;
  uint8_t* a4;        // swiglu: codes [M, N / 4] and their scale atoms
  int64_t lda4;
  uint8_t* sfa_out;
  int lora;
  LoraParams lp;
};

// Tokens per CTA of a cluster in the reduction: a multiple of 16, so that a 16-column
// chunk of the accumulator belongs to one CTA.
__host__ __device__ constexpr int rows_per_part(int rows, int ks) { return ((rows + ks - 1) / ks + 15) / 16 * 16; }

// Instruction descriptor, kind::mxf4 with block scaling: e2m1 A and B, K-major, fp32
// accumulator, UE8M0 scales; sf_id (0 or 2) picks the byte pair of the 32-bit scale words.
__host__ __device__ constexpr uint32_t idesc_mxf4(int M, int N, int sf_id) {
  return ((uint32_t)sf_id << 4)          // B scale-factor id
         | (1u << 7) | (1u << 10)        // A, B format: E2M1
         | ((uint32_t)(N >> 3) << 17)    // N / 8
         | (1u << 23)                    // scale format: UE8M0
         | ((uint32_t)(M >> 4) << 24)    // M / 16
         | ((uint32_t)sf_id << 29);      // A scale-factor id
}

// Shared-memory descriptor of one scale atom as a tcgen05.cp source: 32 rows of 16
// bytes, no swizzle, 8-row core matrices 128 bytes apart.
__device__ __forceinline__ uint64_t sf_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(128u >> 4) << 32) | ((uint64_t)1u << 46);
}

__device__ __forceinline__ void tmem_cp_sf(uint32_t taddr, uint32_t saddr) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sf_desc(saddr)) : "memory");
}

__device__ __forceinline__ void umma_mxf4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t tsfa, uint32_t tsfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
          tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(tsfa), "r"(tsfb)
      : "memory");
}

// Untiled bulk copy global -> this CTA's shared memory (16-byte aligned, multiples of 16).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y)
               : "memory");
}

// One lane of the (converged) warp, always the same one. The issuing warps run their loops whole,
// so that addresses and descriptors stay in uniform registers, and only the issue is one lane's.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// The two halves of cluster_sync().
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// mbar_wait of a whole warp that also ends when another warp of the CTA gave up.
__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint32_t* err) {
  bool ok = mbar_try_wait(bar, parity);
  if (!__all_sync(0xffffffffu, ok)) {
    const uint64_t t0 = globaltimer_ns();
    while (!(ok = mbar_try_wait(bar, parity))) {
      if (*abort_flag) break;
      if (globaltimer_ns() - t0 > kWaitBudgetNs) {
        raise_error(err, kErrGemmWait);
        *abort_flag = 1;
        break;
      }
    }
    ok = __all_sync(0xffffffffu, ok);
  }
  return ok;
}

template <int OFF>
__device__ __forceinline__ void st_dsmem_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0+%2], %1;" ::"r"(addr), "f"(v), "n"(OFF));
}
template <int... J>
__device__ __forceinline__ void push_rows16(uint32_t addr, const uint32_t (&r)[16], std::integer_sequence<int, J...>) {
  (st_dsmem_f32<J * P_STRIDE * 4>(addr, __uint_as_float(r[J])), ...);
}

// Adapters present among the rows of 128-row tile `t` (a mask's bits past the last adapter are ignored).
__device__ __forceinline__ uint64_t tile_adapters(const LoraParams& l, int t, int tiles) {
  if (t >= tiles) return 0ull;
  const uint64_t all = (l.num_adapters >= 64) ? ~0ull : ((1ull << l.num_adapters) - 1);
  return l.tile_mask == nullptr ? all : l.tile_mask[t] & all;
}

__device__ __forceinline__ int slice_base(const LoraParams& l, int row) {
  int sl = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < l.num_slices && row >= l.slice_bounds[i]) sl = i;
  return sl * l.num_adapters * l.rank_blocks * 32;
}

// The LoRA blocks (32 columns of S and LB) of the adapters in a mask, one after the other: adapter
// by adapter its rank blocks; for swiglu each adapter has the gate's blocks, then the up's, whose
// columns start num_adapters * rank later. Advanced by the whole warp, block by block.
struct LoraWalk {
  uint64_t rem;  // adapters left, the current one lowest
  int bit, block;

  __device__ __forceinline__ void start(uint64_t mask) {
    rem = mask;
    bit = __ffsll((long long)mask) - 1;
    block = 0;
  }
  // Column from the slice's first.
  __device__ __forceinline__ int column(const LoraParams& l) const {
    const int rank = l.rank_blocks * 32;
    return bit * rank + (block >= l.rank_blocks ? l.num_adapters * rank - rank : 0) + block * 32;
  }
  __device__ __forceinline__ void next(const LoraParams& l) {
    if (++block == l.blocks_per_adapter) {
      block = 0;
      rem &= rem - 1;
      bit = __ffsll((long long)rem) - 1;
    }
  }
};

__device__ __forceinline__ float swiglu_f(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

template <int EPI>
__global__ void __launch_bounds__(THREADS, 1)
    mxfp4_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                       const __grid_constant__ CUtensorMap tm_lb, const __grid_constant__ CUtensorMap tm_s,
                       const SplitParams p, uint32_t* err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], tfull_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag, peer_abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ks = p.ks, stages = p.stages;
  const int part = ks > 1 ? (int)cluster_ctarank() : 0;
  const int tile = blockIdx.x / ks, n0 = tile * BW;
  const int m0 = blockIdx.y * p.mt_rows, rows = min(p.M - m0, p.mt_rows);  // several token tiles: 64 or 128 rows each
  const int Mp = (rows + 15) / 16 * 16, x_bytes = (p.mt_rows + 15) / 16 * 16 * BKB;
  const int mtiles128 = (p.M + 127) / 128;
  const int kb_lo = (int)((int64_t)part * p.kstages / ks), kb_hi = (int)((int64_t)(part + 1) * p.kstages / ks);
  const int n_main = kb_hi - kb_lo;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&tfull_bar, 1);
    abort_flag = part == p.give_up;
    peer_abort = 0;
    if (part == p.give_up) raise_error(err, kErrGemmWait);
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    if (p.lora) {
      tma_prefetch_desc(&tm_lb);
      tma_prefetch_desc(&tm_s);
    }
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  // a reduction buffer of its own may be written once its CTA runs
  if (ks > 1 && p.reduce_off) cluster_arrive();
  griddep_launch();

  // The first stages' weights start towards L2 before the wait for the kernel before this
  // one (a prefetch into L2 reads nothing that could be stale).
  if (warp == 0 && lane == 0)
    for (int i = 0; i < min(stages, n_main); ++i) tma_prefetch_2d(&tm_w, (kb_lo + i) * BKB, n0);
  griddep_wait();

  // adapters of the 128-row tile that holds the token tile
  const uint64_t amask = p.lora ? tile_adapters(p.lp, m0 / 128, mtiles128) : 0ull;
  const int n_lora_all = __popcll(amask) * p.lp.blocks_per_adapter;
  const int n_lora = n_lora_all > part ? (n_lora_all - part + ks - 1) / ks : 0;
  const int total = n_main + (n_lora + 1) / 2;  // a stage holds two LoRA blocks
  const int acc_cols = (p.mt_rows + 31) / 32 * 32;  // accumulator, then the ring of scales: SF_COLS columns a stage

  if (warp == 0) {
    // ---------------- producer ----------------
    const bool one = elect_one();
    const uint32_t stage_tx = W_BYTES + x_bytes + 2 * SF_BYTES;
    const uint8_t* sfw = p.sfw + ((size_t)tile * p.kstages + kb_lo) * 1024;
    const uint8_t* sfx = p.sfx + ((size_t)(m0 / 128) * p.kstages + kb_lo) * 1024;
    int issued = 0, slot = 0;
    uint32_t ph = 1;
    uint8_t* sw = smem;
    LoraWalk walk;  // this CTA takes every ks-th block, from block `part`
    walk.start(amask);
    for (int j = 0; j < part && n_lora > 0; ++j) walk.next(p.lp);
    const int s_base = p.lora ? slice_base(p.lp, n0) : 0;
    for (int i = 0; i < total; ++i) {
      if (!ring_wait(&empty_bar[slot], ph, &abort_flag, err)) break;
      uint64_t* bar = &full_bar[slot];
      uint8_t* sx = sw + W_BYTES;
      if (i < n_main) {
        if (one) {
          uint8_t* sf = sx + x_bytes;
          mbar_arrive_expect_tx(bar, stage_tx);
          tma_load_2d(sw, &tm_w, bar, (kb_lo + i) * BKB, n0);
          bulk_load(sf, sfw, 1024, bar);
          tma_load_2d(sx, &tm_x, bar, (kb_lo + i) * BKB, m0);
          bulk_load(sf + 1024, sfx, 1024, bar);
        }
        sfw += 1024;
        sfx += 1024;
      } else {
        const int nb = min(2, n_lora - 2 * (i - n_main));
        if (one) mbar_arrive_expect_tx(bar, nb * (BW * 64 + x_bytes / 2));
        for (int b = 0; b < nb; ++b) {
          if (one) {
            const int col = walk.column(p.lp);
            tma_load_2d(sw + b * BW * 64, &tm_lb, bar, col, n0);
            tma_load_2d(sx + b * (x_bytes / 2), &tm_s, bar, s_base + col, m0);
          }
          for (int j = 0; j < ks; ++j) walk.next(p.lp);
        }
      }
      ++issued;
      sw += p.stage_bytes;
      if (++slot == stages) {
        slot = 0;
        ph ^= 1;
        sw = smem;
      }
    }
    if (abort_flag) {
      // no copy may still be landing in this CTA's shared memory at exit
      for (int j = max(0, issued - stages); j < issued; ++j)
        mbar_wait(&full_bar[j % stages], (j / stages) & 1, err, kErrGemmWait);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    const bool one = elect_one();
    const uint32_t idesc_bf = umma_idesc_bf16(BW, Mp), idesc0 = idesc_mxf4(BW, Mp, 0), idesc2 = idesc_mxf4(BW, Mp, 2);
    const uint32_t base = smem_u32(smem);
    const int x_col = (m0 & 64) / 32;  // the second 64 rows' scales are the atom's columns 2 and 3
    int slot = 0;
    uint32_t ph = 0, sw = base, tw = tmem_base + acc_cols;
    bool ok = true;
    for (int i = 0; i < total; ++i) {
      if (!ring_wait(&full_bar[slot], ph, &abort_flag, err)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t sx = sw + W_BYTES;
      if (one) {
        if (i < n_main) {
          // scales: the weights' atoms of both K tiles, then the tokens'
          const uint32_t sf = sx + x_bytes, tx = tw + 8;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            tmem_cp_sf(tw + 4 * h, sf + 512 * h);
            tmem_cp_sf(tx + 4 * h, sf + 1024 + 512 * h);
          }
          const uint64_t ad = umma_desc_sw128(sw), bd = umma_desc_sw128(sx);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_mxf4(tmem_base, ad + 2 * kk, bd + 2 * kk, (kk & 1) ? idesc2 : idesc0, tw + 4 * (kk >> 1),
                      tx + x_col + 4 * (kk >> 1), (i | kk) != 0);
        } else {
          for (int b = 0; b < min(2, n_lora - 2 * (i - n_main)); ++b) {
            const uint64_t ad = umma_desc_sw64(sw + b * BW * 64), bd = umma_desc_sw64(sx + b * (x_bytes / 2));
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) umma_bf16(tmem_base, ad + 2 * kk, bd + 2 * kk, idesc_bf, 1);
          }
        }
        umma_commit(&empty_bar[slot]);
      }
      __syncwarp();
      sw += p.stage_bytes;
      tw += SF_COLS;
      if (++slot == stages) {
        slot = 0;
        ph ^= 1;
        sw = base;
        tw = tmem_base + acc_cols;
      }
    }
    if (ok && one) umma_commit(&tfull_bar);
    __syncwarp();
  }

  // Reduction over the cluster and epilogue. Token m of the tile belongs to CTA m / rows_per;
  // the drain warps push their fp32 partial rows into the owner's buffer R[part][m - first][128].
  bool ready = false;
  if (warp >= 2) {
    ready = !abort_flag && mbar_wait(&tfull_bar, 0, err, kErrGemmWait);
    if (!ready) abort_flag = 1;
    else tc_fence_after();
  }
  if (ks > 1) {
    if (!p.reduce_off) {  // over the ring: every main loop of the cluster has to be done
      __syncthreads();
      cluster_arrive();
    }
    cluster_wait();
  } else {
    __syncthreads();
  }
  const int rows_per = p.rows_per;
  float* R = reinterpret_cast<float*>(smem + p.reduce_off);
  if (warp >= 2 && ready) {
    const int q = warp & 3, n = q * 32 + lane;
    for (int c = 0, owner = 0, oc = 0; c < rows; c += 16) {
      if (c - oc >= rows_per) {
        ++owner;
        oc += rows_per;
      }
      uint32_t r[16];
      tmem_ld16(tmem_base + c + ((uint32_t)(q * 32) << 16), r);
      tmem_wait_ld();
      const int row = part * rows_per + c - oc;
      if (ks > 1) {
        push_rows16(mapa_shared(smem_u32(R + row * P_STRIDE + n), (uint32_t)owner), r,
                    std::make_integer_sequence<int, 16>{});
      } else {
        float* dst = R + row * P_STRIDE + n;
#pragma unroll
        for (int j = 0; j < 16; ++j) dst[j * P_STRIDE] = __uint_as_float(r[j]);
      }
    }
  }
  const int r0 = part * rows_per, n_rows = max(0, min(rows, r0 + rows_per) - r0);
  constexpr int GROUPS = (EPI == kEpiSwiGLU) ? 8 : 16;  // 8-column groups per token
  const int items = n_rows * GROUPS;
  // a token's eight columns from c, summed over the parts
  auto sum8 = [&](int lm, int c, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll 1
    for (int q = 0; q < ks; ++q) {
      const float* src = R + (q * rows_per + lm) * P_STRIDE + c;
      const float4 a0 = *reinterpret_cast<const float4*>(src), a1 = *reinterpret_cast<const float4*>(src + 4);
      v[0] += a0.x; v[1] += a0.y; v[2] += a0.z; v[3] += a0.w;
      v[4] += a1.x; v[5] += a1.y; v[6] += a1.z; v[7] += a1.w;
    }
  };
  // The residuals of a thread's first items are loaded before the barrier, four at a time.
  constexpr int BATCH = 4;
  uint4 res[BATCH];
  auto load_residuals = [&](int first) {
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int it = first + j * THREADS, col = n0 + (it % GROUPS) * 8;
      res[j] = make_uint4(0u, 0u, 0u, 0u);
      if (it < items && col < p.N)
        res[j] = *reinterpret_cast<const uint4*>(p.residual + (int64_t)(m0 + r0 + it / GROUPS) * p.ldr + col);
    }
  };
  if (EPI == kEpiResAdd) load_residuals(threadIdx.x);
  __syncthreads();  // abort_flag is final
  if (ks > 1) {
    if (abort_flag && threadIdx.x < ks)
      asm volatile("st.shared::cluster.u32 [%0], 1;" ::"r"(
                       mapa_shared(smem_u32(const_cast<int*>(&peer_abort)), threadIdx.x))
                   : "memory");
    cluster_sync();  // every partial row has landed
  }
  if (abort_flag || peer_abort) {
    // nothing of the tile is written, by any CTA of the cluster
  } else if constexpr (EPI == kEpiSwiGLU) {
    // four neighbouring items are one block of 32 outputs; whole warps run for the shuffles
    for (int it = threadIdx.x; it < (items + 31) / 32 * 32; it += THREADS) {
      const int lm = min(it, items - 1) / GROUPS, c = (it % GROUPS) * 8, m = m0 + r0 + lm;
      float v[8], u[8];
      sum8(lm, c, v);
      sum8(lm, c + 64, u);
      const int col = tile * 64 + c;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = swiglu_f(v[j], u[j]);
      const uint32_t byte = scale_byte(quad_max(max_abs_bits(v)));
      if (it >= items) continue;
      if (p.out != nullptr)
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.out) + (int64_t)m * p.ldo + col) = make_uint4(
            pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
      const int64_t kt = k_tiles(p.N / 2);
      if ((c & 31) == 0) p.sfa_out[sf_word(m, col >> 7, kt) + ((col >> 5) & 3)] = (uint8_t)byte;
      // the last tile also clears the scales past the row's end
      if (col + 8 == p.N / 2)
        for (int b = p.N / 64; b < kt * 4; ++b) p.sfa_out[sf_word(m, b >> 2, kt) + (b & 3)] = 0;
      *reinterpret_cast<uint32_t*>(p.a4 + (int64_t)m * p.lda4 + col / 2) =
          byte == 255u ? 0u : pack8(v, inv_scale(byte));
    }
  } else {
    for (int first = threadIdx.x; first < items; first += BATCH * THREADS) {
      if (EPI == kEpiResAdd && first != threadIdx.x) load_residuals(first);
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int it = first + j * THREADS, lm = it / GROUPS, c = (it % GROUPS) * 8, col = n0 + c;
        if (it >= items || col >= p.N) continue;
        float v[8];
        sum8(lm, c, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= p.scale;
        if (EPI == kEpiResAdd) {
          const uint32_t ww[4] = {res[j].x, res[j].y, res[j].z, res[j].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = unpack_bf16x2(ww[k]);
            v[2 * k] += f.x;
            v[2 * k + 1] += f.y;
          }
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.out) + (int64_t)(m0 + r0 + lm) * p.ldo + col) =
            make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                       pack_bf16x2(v[6], v[7]));
      }
    }
  }
  if (abort_flag) {
    // error path: MMAs and copies this CTA issued may still be in flight; give them
    // time to finish before the tensor memory is released (bounded, ~1 ms)
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, p.tmem_cols);
  }
}

// ---------------------------------------------------------------------------
// CTA-pair kernel (cta_group::2) for many tokens: a cluster of two CTAs computes
// 256 tokens x 256 weight rows. Each CTA stages its own 128 tokens and 128 weight rows
// per 256-K stage (half the weight bytes that a single CTA's 128 x 256 tile takes in per
// MMA; the 4-bit MMA eats 48 KB of operands in 512 cycles otherwise, which is the L2's
// whole rate), and the scales of its tokens and of all 256 weight rows. The leader's MMA
// thread issues the scale copies and MMAs for both CTAs. Persistent: one cluster per SM
// pair walks the tiles.
//
// One 256-column accumulator and the ring of scales fill the tensor memory, so the
// epilogue empties the accumulator into registers at once (eight warps, 128 columns each)
// and gives it back before it converts and stores: the next tile's MMAs run meanwhile.
//
// Bound by the tensor pipe and the power limit: 8192 x 4096 x 12800 takes 138 us alone (6.2
// PFLOP/s, the pipe active in 82% of all cycles) and 145 to 160 us back to back, 8192 x 4096 x 4096
// 51 us (5.4), 4096 x 6144 x 4096 40 us (5.1) and, expanding twelve adapters in every tile, 60 us. A
// stage of four MMAs issues in 0.30 us; a tile's end costs 0.8 us, from the last MMA's end to
// the next one's start. Two accumulators would hide that, but leave no columns for the scales.
// ---------------------------------------------------------------------------
struct PairCfg {
  static constexpr int THREADS = 320;  // warp 0 loads, warp 1 MMAs, warps 2..9 epilogue
  static constexpr int BN = 256;
  static constexpr int A_BYTES = 128 * BKB, B_BYTES = 128 * BKB;
  static constexpr int SFA_OFF = A_BYTES + B_BYTES, SFB_OFF = SFA_OFF + 1024;
  static constexpr int STAGE_BYTES = SFB_OFF + 2048;
  static constexpr int STAGES = 5;
  static constexpr int SF_COLS = 24;   // per stage: tokens 2 x 4 columns, weights 2 x 8
  static constexpr int STAGING_OFF = STAGES * STAGE_BYTES;
  static constexpr int STAGING = 4096;  // per epilogue warp: 32 rows x 128 bytes
  static constexpr int SMEM_BYTES = STAGING_OFF + 8 * STAGING + 1024;
};
static_assert(PairCfg::STAGE_BYTES % 1024 == 0 && PairCfg::SMEM_BYTES <= SMEM_LIMIT - BAR_BYTES, "shared memory");
static_assert(PairCfg::BN + PairCfg::STAGES * PairCfg::SF_COLS <= 512, "tensor memory");

struct PairParams {
  int M, N, kstages;
  float scale;
  void* out;
  int64_t ldo;
  const __nv_bfloat16* residual;
  int64_t ldr;
  uint8_t* a4;
  int64_t lda4;
  uint8_t* sfa_out;
  int lora;
  LoraParams lp;
};

// 3-D tiled load into this CTA's shared memory, completing on a barrier of the pair's leader.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster, int32_t x,
                                                 int32_t y, int32_t z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Arrival that orders no ordinary memory: tensor-memory reads are ordered by the tcgen05 fences on
// both sides. (With .release it took 0.8 us, during which the tensor core idled at every tile's end.)
__device__ __forceinline__ void arrive_relaxed_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Scale atoms of both CTAs (the same offset in each one's shared memory) into both tensor memories.
__device__ __forceinline__ void tmem_cp_sf_pair(uint32_t taddr, uint32_t saddr) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sf_desc(saddr)) : "memory");
}

__device__ __forceinline__ void umma_mxf4_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                               uint32_t tsfa, uint32_t tsfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
          tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(tsfa), "r"(tsfb)
      : "memory");
}

// Tile order: columns of 8 token tiles walk the weight tiles, so that concurrent clusters share both in L2.
__device__ __forceinline__ void pair_tile(int t, int m_tiles, int n_tiles, int& mt, int& nt) {
  const int group = t / (8 * n_tiles), first = group * 8, size = min(8, m_tiles - first), in = t - group * 8 * n_tiles;
  mt = first + in % size;
  nt = in / size;
}

__device__ __forceinline__ uint32_t swz128(int row, int chunk) {
  return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4));
}

template <int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg::THREADS, 1)
    mxfp4_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_sfx, const __grid_constant__ CUtensorMap tm_sfw,
                      const __grid_constant__ CUtensorMap tm_s, const __grid_constant__ CUtensorMap tm_lb,
                      const __grid_constant__ CUtensorMap tm_out, const PairParams p, uint32_t* err) {
  using C = PairCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full_bar[C::STAGES], empty_bar[C::STAGES], tfull_bar, tempty_bar;  // full, tempty: the leader's
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int mtiles128 = (p.M + 127) / 128;
  const int m_tiles = (p.M + 255) / 256, n_tiles = (p.N + C::BN - 1) / C::BN, num_tiles = m_tiles * n_tiles;
  const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&tfull_bar, 1);
    mbar_init(&tempty_bar, 16);  // one arrival per epilogue warp of both CTAs
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_sfx);
    tma_prefetch_desc(&tm_sfw);
  }
  if (warp == 1) {
    tmem_alloc_pair(&tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers are initialised before any remote arrival
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  griddep_launch();
  griddep_wait();

  if (warp == 0) {
    // ---------------- producer (both CTAs) ----------------
    const bool one = elect_one();
    const uint32_t full_leader = mapa_shared(smem_u32(full_bar), 0);
    uint32_t ph = 1, issued = 0;
    int slot = 0;
    bool stop = false;
    for (int t = cluster_id; t < num_tiles && !stop; t += num_clusters) {
      int mt, nt;
      pair_tile(t, m_tiles, n_tiles, mt, nt);
      const int own = 2 * mt + (int)rank, m0 = own * 128, n0 = nt * C::BN;
      uint64_t mask0 = 0ull, mask1 = 0ull;
      if (p.lora) {
        mask0 = tile_adapters(p.lp, 2 * mt, mtiles128);
        mask1 = tile_adapters(p.lp, 2 * mt + 1, mtiles128);
      }
      const uint64_t both = mask0 | mask1, mine = rank ? mask1 : mask0;
      const int base0 = p.lora ? slice_base(p.lp, n0) : 0, base1 = p.lora ? slice_base(p.lp, n0 + 128) : 0;
      const bool one_slice = base0 == base1;  // then a stage holds two LoRA blocks
      const int n_lora = __popcll(both) * p.lp.blocks_per_adapter, per = one_slice ? 2 : 1;
      const int total = p.kstages + (n_lora + per - 1) / per;
      LoraWalk walk;
      walk.start(both);
      for (int i = 0; i < total; ++i) {
        if (!ring_wait(&empty_bar[slot], ph, &abort_flag, err)) {
          stop = true;
          break;
        }
        uint8_t* sa = smem + slot * C::STAGE_BYTES;
        uint8_t* sb = sa + C::A_BYTES;
        const uint32_t fb = full_leader + slot * 8;
        if (i < p.kstages) {
          if (one) {
            // tiles past the last row are zeros, scales too
            if (leader) mbar_arrive_expect_tx(&full_bar[slot], 2 * C::STAGE_BYTES);
            tma_load_2d_pair(sa, &tm_x, fb, i * BKB, m0);
            tma_load_2d_pair(sb, &tm_w, fb, i * BKB, n0 + (int)rank * 128);
            tma_load_3d_pair(sa + C::SFA_OFF, &tm_sfx, fb, 0, i, own);
            tma_load_3d_pair(sa + C::SFB_OFF, &tm_sfw, fb, 0, i, 2 * nt);
          }
        } else {
          // As the main loop where the tile lies in one slice of S, else two halves of 128 weight
          // rows with their slice's columns, of which either CTA stages 64 rows of LB. A token tile
          // that lacks the adapter reads zeros.
          const int nb = min(per, n_lora - per * (i - p.kstages));
          if (one && leader) mbar_arrive_expect_tx(&full_bar[slot], 2 * ((one_slice ? nb : 2) + nb) * 128 * 64);
          for (int b = 0; b < nb; ++b) {
            if (one) {
              const int col = walk.column(p.lp);
              const int y = ((mine >> walk.bit) & 1ull) ? m0 : mtiles128 * 128;
              tma_load_2d_pair(sa + b * 128 * 64, &tm_s, fb, base0 + col, y);
              if (!one_slice) tma_load_2d_pair(sa + 128 * 64, &tm_s, fb, base1 + col, y);
              const int first = n0 + (int)rank * (one_slice ? 128 : 64);
              uint8_t* lb = sb + b * 128 * 64;
              tma_load_2d_pair(lb, &tm_lb, fb, col, first);
              tma_load_2d_pair(lb + 64 * 64, &tm_lb, fb, col, first + (one_slice ? 64 : 128));
            }
            walk.next(p.lp);
          }
        }
        __syncwarp();
        ++issued;
        if (++slot == C::STAGES) {
          slot = 0;
          ph ^= 1;
        }
      }
    }
    // the pair MMA has released every stage this CTA filled before the CTA may exit
    for (uint32_t j = issued > (uint32_t)C::STAGES ? issued - C::STAGES : 0; j < issued && !abort_flag; ++j)
      if (!mbar_wait(&empty_bar[j % C::STAGES], (j / C::STAGES) & 1, err, kErrGemmWait)) abort_flag = 1;
  } else if (warp == 1) {
    // ---------------- MMA issuer (leader only) ----------------
    if (leader) {
      const bool one = elect_one();
      const uint32_t base = smem_u32(smem);
      uint32_t ph = 0;
      int slot = 0, ltile = 0;
      bool stop = false;
      for (int t = cluster_id; t < num_tiles && !stop; t += num_clusters, ++ltile) {
        int mt, nt;
        pair_tile(t, m_tiles, n_tiles, mt, nt);
        const bool one_slice = !p.lora || slice_base(p.lp, nt * C::BN) == slice_base(p.lp, nt * C::BN + 128);
        int n_lora = 0;
        if (p.lora)
          n_lora = __popcll(tile_adapters(p.lp, 2 * mt, mtiles128) | tile_adapters(p.lp, 2 * mt + 1, mtiles128)) *
                   p.lp.blocks_per_adapter;
        const int per = one_slice ? 2 : 1, total = p.kstages + (n_lora + per - 1) / per;
        if (!ring_wait(&tempty_bar, (ltile & 1) ^ 1, &abort_flag, err)) break;
        tc_fence_after();
        for (int i = 0; i < total; ++i) {
          if (!ring_wait(&full_bar[slot], ph, &abort_flag, err)) {
            stop = true;
            break;
          }
          tc_fence_after();
          const uint32_t sa = base + slot * C::STAGE_BYTES, sb = sa + C::A_BYTES;
          if (one) {
            if (i < p.kstages) {
              const uint32_t ta = tmem_base + C::BN + slot * C::SF_COLS, tb = ta + 8;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                tmem_cp_sf_pair(ta + 4 * h, sa + C::SFA_OFF + 512 * h);
                tmem_cp_sf_pair(tb + 8 * h, sa + C::SFB_OFF + 512 * h);
                tmem_cp_sf_pair(tb + 8 * h + 4, sa + C::SFB_OFF + 1024 + 512 * h);
              }
              const uint64_t ad = umma_desc_sw128(sa), bd = umma_desc_sw128(sb);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_mxf4_pair(tmem_base, ad + 2 * kk, bd + 2 * kk, idesc_mxf4(256, C::BN, 2 * (kk & 1)),
                               ta + 4 * (kk >> 1), tb + 8 * (kk >> 1), (i | kk) != 0);
            } else {
              for (int b = 0; one_slice && b < min(2, n_lora - 2 * (i - p.kstages)); ++b) {
                const uint64_t ad = umma_desc_sw64(sa + b * 128 * 64), bd = umma_desc_sw64(sb + b * 128 * 64);
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
                  umma_bf16_pair(tmem_base, ad + 2 * kk, bd + 2 * kk, umma_idesc_bf16(256, C::BN), 1);
              }
              const uint32_t idesc = umma_idesc_bf16(256, 128);
#pragma unroll
              for (int u = 0; u < (one_slice ? 0 : 2); ++u) {
                const uint64_t ad = umma_desc_sw64(sa + u * 128 * 64), bd = umma_desc_sw64(sb + u * 64 * 64);
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) umma_bf16_pair(tmem_base + u * 128, ad + 2 * kk, bd + 2 * kk, idesc, 1);
              }
            }
            umma_commit_pair(&empty_bar[slot], 0x3);
          }
          __syncwarp();
          if (++slot == C::STAGES) {
            slot = 0;
            ph ^= 1;
          }
        }
        if (stop) break;
        if (one) umma_commit_pair(&tfull_bar, 0x3);
        __syncwarp();
      }
    }
  } else {
    // ---------------- epilogue: TMEM lane quarter warp % 4, columns 128 half .. ----------------
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t* buf = smem + C::STAGING_OFF + (warp - 2) * C::STAGING;
    const uint32_t tempty_leader = mapa_shared(smem_u32(&tempty_bar), 0);
    // the residual's 32 x 64 box at (row0, col) into the warp's buffer, which the last TMA store has read
    auto fetch_residual = [&](int row0, int col) {
      if (lane == 0) bulk_wait_group_read<0>();
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int rr = 4 * j + (lane >> 3), ch = lane & 7;
        if (row0 + rr < p.M && col + ch * 8 < p.N)
          cp_async16(buf + swz128(rr, ch), p.residual + (int64_t)(row0 + rr) * p.ldr + col + ch * 8);
      }
    };
    int ltile = 0;
    for (int t = cluster_id; t < num_tiles; t += num_clusters, ++ltile) {
      int mt, nt;
      pair_tile(t, m_tiles, n_tiles, mt, nt);
      const int row0 = mt * 256 + (int)rank * 128 + q * 32, row = row0 + lane, n0 = nt * C::BN + half * 128;
      if (EPI == kEpiResAdd) fetch_residual(row0, n0);  // while the tile's MMAs run
      if (abort_flag || !mbar_wait(&tfull_bar, ltile & 1, err, kErrGemmWait)) {
        abort_flag = 1;
        break;
      }
      tc_fence_after();
      uint32_t r[4][32];
      const uint32_t tb = tmem_base + half * 128 + ((uint32_t)(q * 32) << 16);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(tb + 32 * c, r[c]);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_relaxed_cluster(tempty_leader);
      if (row0 >= p.M || n0 >= p.N) continue;
      if constexpr (EPI == kEpiSwiGLU) {
        // columns 0..63 gate, 64..127 up: two blocks of 32 outputs of one row
        const int col = n0 / 2;
        const int64_t kt = k_tiles(p.N / 2);
        uint32_t bytes = 0;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          float v[4][8];
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            v[j / 8][j % 8] = swiglu_f(__uint_as_float(r[b][j]), __uint_as_float(r[2 + b][j]));
#pragma unroll
          for (int g = 0; g < 4; ++g) top = max(top, max_abs_bits(v[g]));
          const uint32_t byte = scale_byte(top);
          bytes |= byte << (8 * b);
          if (row >= p.M) continue;
          if (p.out != nullptr) {
            uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.out) + (int64_t)row * p.ldo + col +
                                                32 * b);
#pragma unroll
            for (int g = 0; g < 4; ++g)
              o[g] = make_uint4(pack_bf16x2(v[g][0], v[g][1]), pack_bf16x2(v[g][2], v[g][3]),
                                pack_bf16x2(v[g][4], v[g][5]), pack_bf16x2(v[g][6], v[g][7]));
          }
          const float inv = inv_scale(byte);
          const uint32_t keep = byte == 255u ? 0u : ~0u;
          *reinterpret_cast<uint4*>(p.a4 + (int64_t)row * p.lda4 + col / 2 + 16 * b) =
              make_uint4(pack8(v[0], inv) & keep, pack8(v[1], inv) & keep, pack8(v[2], inv) & keep,
                         pack8(v[3], inv) & keep);
        }
        if (row < p.M) {
          *reinterpret_cast<uint16_t*>(p.sfa_out + sf_word(row, col >> 7, kt) + ((col >> 5) & 3)) = (uint16_t)bytes;
          // the last columns' warp also clears the scales past the row's end
          if (n0 + 128 == p.N)
            for (int b = p.N / 64; b < kt * 4; ++b) p.sfa_out[sf_word(row, b >> 2, kt) + (b & 3)] = 0;
        }
      } else {
        // 64 columns at a time through a swizzled buffer: coalesced residual reads, one TMA store
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = n0 + 64 * h;
          if (col >= p.N) break;
          if (EPI == kEpiResAdd) {
            if (h == 1) fetch_residual(row0, col);
            cp_async_wait();
          } else if (lane == 0) {
            bulk_wait_group_read<0>();
          }
          __syncwarp();
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) {
            uint4* cell = reinterpret_cast<uint4*>(buf + swz128(lane, ch));
            float2 f[4] = {};
            if (EPI == kEpiResAdd) {
              const uint4 w = *cell;
              f[0] = unpack_bf16x2(w.x);
              f[1] = unpack_bf16x2(w.y);
              f[2] = unpack_bf16x2(w.z);
              f[3] = unpack_bf16x2(w.w);
            }
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int at = 8 * ch + 2 * j;
              const float a = __uint_as_float(r[2 * h + at / 32][at % 32]) * p.scale;
              const float b = __uint_as_float(r[2 * h + at / 32][at % 32 + 1]) * p.scale;
              o[j] = EPI == kEpiResAdd ? pack_bf16x2(a + f[j].x, b + f[j].y) : pack_bf16x2(a, b);
            }
            *cell = make_uint4(o[0], o[1], o[2], o[3]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tm_out, buf, col, row0);
            bulk_commit_group();
          }
        }
      }
    }
    if (EPI == kEpiResAdd) cp_async_wait();
    if (EPI != kEpiSwiGLU && lane == 0) bulk_wait_group_all();
  }

  if (abort_flag) {
    // error path: copies and MMAs may still be in flight (bounded, ~1 ms)
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) {
    }
  }
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------- host
constexpr int kMaxDevices = 64;

static int current_device() {
  int dev = 0;
  GSB_CUDA_CHECK(cudaGetDevice(&dev));
  GSB_CHECK(dev >= 0 && dev < kMaxDevices, "mxfp4_gemm: device index out of range");
  return dev;
}

static int num_sms() {
  static int cached[kMaxDevices] = {0};
  const int dev = current_device();
  if (!cached[dev])
    GSB_CUDA_CHECK(cudaDeviceGetAttribute(&cached[dev], cudaDevAttrMultiProcessorCount, dev));
  return cached[dev];
}

// Clusters of `ks` CTAs that fit on the GPU at once with one or two CTAs per SM (clusters lie
// inside one GPC, so large ones leave SMs unused). Asked once per device and size.
constexpr int HALF_SMEM = 112 * 1024;
static int max_clusters(int ks, int per_sm) {
  static int cached[kMaxDevices][MAX_KS + 1][3] = {{{0}}};
  const int dev = current_device();
  if (cached[dev][ks][per_sm]) return cached[dev][ks][per_sm];
  if (ks == 1) return cached[dev][ks][per_sm] = per_sm * num_sms();
  auto kfn = mxfp4_split_kernel<kEpiStore>;
  const int smem = per_sm == 2 ? HALF_SMEM - BAR_BYTES : SMEM_LIMIT - BAR_BYTES;
  GSB_CUDA_CHECK(cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT - BAR_BYTES));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * ks * num_sms()), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kfn, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    n = per_sm * num_sms() / ks;
  }
  return cached[dev][ks][per_sm] = n;
}

// Which kernel takes a call. The pair kernel needs about 48 tiles of 256 x 256 to be ahead
// (measured, us pair / split: 256 x 4096 x 4096 11.5 / 9.7, 512: 11.7 / 11.3, 768: 11.8 / 13; 256 x
// 25600 x 4096 20.9 / 26.9; K, at which these were taken, is not looked at); one token tile of 128 is
// always the split kernel's.
// gsb_mxfp4_pair_min_m forces a smallest M instead, for A/B runs.
static int g_pair_min_m = -1;
static bool use_pair(int M, int N) {
  if (g_pair_min_m >= 0) return M >= g_pair_min_m;
  return M > BT && (M + 255) / 256 * ((N + 255) / 256) >= 48;
}

// K part that gives up in the split kernel's calls (tests), or -1.
static int g_split_give_up = -1;

struct SplitPlan {
  int mt_rows, token_tiles, weight_tiles, ks, stages, stage_bytes, tmem_cols, smem_bytes, reduce_off;
};

// Token tiles of 128 or, where they still run in one wave of two CTAs per SM over a short K, of
// 64 (256 tokens x 2048 x 2048 8.2 -> 6.5 us; over K = 12800 they cost 20.5 against 15.6 us). Two CTAs
// per SM hide one another's barriers and latencies, but leave less for each one's ring: for
// 128-row tiles only when there are more tiles than SMs. K parts: as many as run in one wave,
// two stages each at least (measured from 1 to 8 at 18 sizes, this takes the fastest).
static SplitPlan split_plan(int M, int N, int64_t K) {
  SplitPlan s{};
  const int kstages = (int)((K + 255) / 256);
  s.weight_tiles = (N + BW - 1) / BW;
  const bool narrow = kstages <= 16 && (M + 63) / 64 * s.weight_tiles <= 2 * num_sms();
  s.mt_rows = std::min(M, narrow ? 64 : BT);
  s.token_tiles = (M + s.mt_rows - 1) / s.mt_rows;
  const int tiles = s.token_tiles * s.weight_tiles, acc = (s.mt_rows + 31) / 32 * 32;
  s.stage_bytes = W_BYTES + (s.mt_rows + 15) / 16 * 16 * BKB + 2 * SF_BYTES;
  auto reduce = [&](int ks) { return ks * rows_per_part(s.mt_rows, ks) * P_STRIDE * 4; };
  for (int per_sm = s.mt_rows <= 64 || tiles > num_sms() ? 2 : 1; per_sm >= 1; --per_sm) {
    const int room = (per_sm == 2 ? HALF_SMEM : SMEM_LIMIT) - BAR_BYTES - 1024;
    s.stages = std::min({MAX_STAGES, room / s.stage_bytes, (512 / per_sm - acc) / SF_COLS});
    if (per_sm == 2 && s.stages < 3) continue;
    s.ks = 1;
    for (int ks = 2; ks <= MAX_KS; ++ks)
      if (kstages / ks >= 2 && tiles <= max_clusters(ks, per_sm) && reduce(ks) <= room) s.ks = ks;
    // a reduction buffer of its own saves a cluster barrier, if three stages are left
    const int apart = (room - reduce(s.ks)) / s.stage_bytes;
    if (s.ks > 1 && apart >= 3) {
      s.stages = std::min(s.stages, apart);
      s.reduce_off = s.stages * s.stage_bytes;
    }
    s.smem_bytes = (s.reduce_off ? s.reduce_off + reduce(s.ks) : std::max(s.stages * s.stage_bytes, reduce(s.ks))) + 1024;
    break;
  }
  const int cols = acc + s.stages * SF_COLS;
  s.tmem_cols = 32;
  while (s.tmem_cols < cols) s.tmem_cols *= 2;
  return s;
}

// Codes and scale atoms of an operand.
struct Codes {
  uint8_t* q;
  int64_t ld;
  uint8_t* sf;
  int64_t rows;
};

static Codes check_operand(const char* what, const at::Tensor& q, const at::Tensor& sf, int64_t K,
                           const at::Device& dev) {
  GSB_CHECK(q.is_cuda() && q.device() == dev && sf.device() == dev, "mxfp4_gemm: ", what, " must be on one CUDA device");
  GSB_CHECK(q.scalar_type() == at::kByte && q.dim() == 2 && q.size(1) * 2 == K && q.stride(1) == 1 &&
                q.stride(0) % 16 == 0 && q.stride(0) >= q.size(1) && aligned16(q),
            "mxfp4_gemm: ", what, " codes must be uint8 [rows, K / 2] with 16-byte aligned rows");
  GSB_CHECK(sf.scalar_type() == at::kByte && sf.is_contiguous() && aligned16(sf) &&
                sf.numel() == (q.size(0) + 127) / 128 * k_tiles(K) * 512,
            "mxfp4_gemm: ", what, " scales must be uint8 atoms [ceil(rows / 128), 2 ceil(K / 256), 512]");
  return {q.data_ptr<uint8_t>(), q.stride(0), sf.data_ptr<uint8_t>(), q.size(0)};
}

static void check_out(const char* what, const at::Tensor& t, int64_t M, int64_t N, const at::Device& dev) {
  GSB_CHECK(t.device() == dev && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.size(0) == M &&
                t.size(1) == N && (N == 1 || t.stride(1) == 1) && (M <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= N)) &&
                aligned16(t),
            "mxfp4_gemm: ", what, " must be bf16 [", M, ", ", N, "] with 16-byte aligned rows");
}

template <int EPI>
static void launch_split(const CUtensorMap& tw, const CUtensorMap& tx, const CUtensorMap& tlb, const CUtensorMap& ts,
                         const SplitParams& p, const SplitPlan& s, uint32_t* err, cudaStream_t st) {
  auto kfn = mxfp4_split_kernel<EPI>;
  static bool set[kMaxDevices] = {false};
  const int dev = current_device();
  if (!set[dev]) {
    GSB_CUDA_CHECK(cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT - BAR_BYTES));
    set[dev] = true;
  }
  launch(kfn, dim3((unsigned)(s.weight_tiles * s.ks), (unsigned)s.token_tiles), THREADS, s.smem_bytes, s.ks, st,
         tw, tx, tlb, ts, p, err);
}

// Clusters of two of the pair kernel that fit at once (asked once per device and epilogue).
template <int EPI>
static int pair_clusters() {
  static int cached[kMaxDevices] = {0};
  const int dev = current_device();
  if (cached[dev]) return cached[dev];
  auto kfn = mxfp4_pair_kernel<EPI>;
  GSB_CUDA_CHECK(cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg::SMEM_BYTES));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(num_sms() / 2 * 2), 1, 1);
  cfg.blockDim = dim3(PairCfg::THREADS, 1, 1);
  cfg.dynamicSmemBytes = PairCfg::SMEM_BYTES;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  GSB_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kfn, &cfg));
  return cached[dev] = std::max(1, n);
}

template <int EPI>
static void launch_pair(const CUtensorMap& tx, const CUtensorMap& tw, const CUtensorMap& tsfx, const CUtensorMap& tsfw,
                        const CUtensorMap& ts, const CUtensorMap& tlb, const CUtensorMap& to, const PairParams& p,
                        uint32_t* err, cudaStream_t st) {
  const int tiles = ((p.M + 255) / 256) * ((p.N + PairCfg::BN - 1) / PairCfg::BN);
  const int clusters = std::min(tiles, pair_clusters<EPI>());  // also sets the shared-memory attribute
  launch(mxfp4_pair_kernel<EPI>, dim3(2 * clusters), PairCfg::THREADS, PairCfg::SMEM_BYTES, 1, st, tx, tw,
         tsfx, tsfw, ts, tlb, to, p, err);
}

// Scale atoms [tiles, K stages, 1024 bytes]; the box takes `tiles_per_box` row tiles of one stage.
static CUtensorMap make_tmap_sf(const Codes& c, int64_t kstages, uint32_t tiles_per_box) {
  CUtensorMap m;
  cuuint64_t dims[3] = {256, (cuuint64_t)kstages, (cuuint64_t)((c.rows + 127) / 128)};
  cuuint64_t strides[2] = {1024, (cuuint64_t)kstages * 1024};
  cuuint32_t box[3] = {256, 1, tiles_per_box};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = tma_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, c.sf, dims, strides, box, estr,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  GSB_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (scales) failed with code ", (int)r);
  return m;
}

static CUtensorMap make_tmap_codes(const Codes& c, int64_t K, uint32_t box_rows) {
  return make_tmap_2d(c.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)c.rows, (uint64_t)K / 2, (uint64_t)c.ld, BKB,
                      box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Refuses an output of a product that shares bytes with what the product reads.
static void check_output_apart(const char* what, const at::Tensor& out, const at::Tensor* x4, const at::Tensor* sfx,
                               const at::Tensor& w4, const at::Tensor& sfw, const c10::optional<at::Tensor>& s,
                               const c10::optional<at::Tensor>& lb) {
  if (x4 != nullptr) check_apart("mxfp4_gemm", what, out, "x", *x4);
  if (sfx != nullptr) check_apart("mxfp4_gemm", what, out, "x's scales", *sfx);
  check_apart("mxfp4_gemm", what, out, "the weight", w4);
  check_apart("mxfp4_gemm", what, out, "the weight's scales", sfw);
  if (s.has_value()) check_apart("mxfp4_gemm", what, out, "s", *s);
  if (lb.has_value()) check_apart("mxfp4_gemm", what, out, "lb", *lb);
}

struct LoraArgs {
  const c10::optional<at::Tensor>& s;
  const c10::optional<at::Tensor>& lb;
  const c10::optional<at::Tensor>& tile_mask;
  int64_t rank, num_adapters;
  std::vector<int64_t> slice_bounds;
};

// Tokens of a product: codes, or bf16 rows (`bf` not null, codes filled in when quantised).
struct Tokens {
  Codes c;
  const void* bf;
  int64_t ldbf;
};

// One product on the current stream of `dev`, the current device. `a4` (codes and scales of
// the output) for swiglu, `out` otherwise (for swiglu: the bf16 copy, or null).
static void run_gemm(Tokens t, const Codes& w, int64_t K, const at::Tensor* out, int epi, double scale,
                     const c10::optional<at::Tensor>& residual, const Codes* a4, const LoraArgs& la,
                     const at::Tensor& err, const at::Device& dev) {
  Codes& x = t.c;
  GSB_CHECK(K >= kBlock && K % kBlock == 0 && K < (int64_t(1) << 31), "mxfp4_gemm: K must be a positive multiple of 32");
  GSB_CHECK(w.rows > 0 && w.rows % 8 == 0, "mxfp4_gemm: N must be a positive multiple of 8");
  GSB_CHECK(x.rows < (int64_t(1) << 24) && w.rows < (int64_t(1) << 24),
            "mxfp4_gemm: at most 2^24 - 1 rows of x and of the weight");
  GSB_CHECK(err.device() == dev, "mxfp4_gemm: error word on another device");
  const int M = (int)x.rows, N = (int)w.rows;
  SplitParams p{};
  p.M = M;
  p.N = N;
  p.scale = (float)scale;
  p.kstages = (int)((K + 255) / 256);
  if (a4 != nullptr) {
    p.a4 = a4->q;
    p.lda4 = a4->ld;
    p.sfa_out = a4->sf;
  }
  if (out != nullptr) {
    check_out(epi == kEpiSwiGLU ? "act" : "out", *out, M, epi == kEpiSwiGLU ? N / 2 : N, dev);
    p.out = out->data_ptr();
    p.ldo = out->stride(0);
  }
  if (epi == kEpiResAdd) {
    GSB_CHECK(residual.has_value(), "mxfp4_gemm: the residual epilogue needs a residual");
    check_out("residual", *residual, M, N, dev);
    check_same_or_apart("mxfp4_gemm", "out", *out, "the residual, unless it is the residual", *residual);
    p.residual = reinterpret_cast<const __nv_bfloat16*>(residual->data_ptr());
    p.ldr = residual->stride(0);
  }
  const bool lora = la.s.has_value() || la.lb.has_value();
  if (lora) {
    GSB_CHECK(la.s.has_value() && la.lb.has_value(), "mxfp4_gemm: LoRA needs both s and lb");
    GSB_CHECK(la.rank > 0 && la.rank % 32 == 0 && la.rank <= 4096 && la.num_adapters >= 1 && la.num_adapters <= 64,
              "mxfp4_gemm: LoRA rank must be a multiple of 32, with 1 to 64 adapters");
    const int64_t cols = la.rank * la.num_adapters;
    const std::vector<int64_t>& b = la.slice_bounds;
    const int64_t slices = epi == kEpiSwiGLU ? 2 : (int64_t)b.size() - 1;
    if (epi != kEpiSwiGLU) {
      GSB_CHECK(b.size() >= 2 && b.size() <= 5 && b.front() == 0 && b.back() == N,
                "mxfp4_gemm: slice bounds must run from 0 to N (at most 4 slices)");
      for (size_t i = 0; i + 1 < b.size(); ++i)
        GSB_CHECK(b[i] % BW == 0 && b[i] < b[i + 1], "mxfp4_gemm: slice bounds must be rising multiples of 128");
    }
    const int64_t lb_cols = epi == kEpiSwiGLU ? 2 * cols : cols;
    GSB_CHECK(la.s->device() == dev && la.lb->device() == dev && la.s->scalar_type() == at::kBFloat16 &&
                  la.lb->scalar_type() == at::kBFloat16 && la.s->dim() == 2 && la.lb->dim() == 2 &&
                  la.s->size(0) == M && la.s->size(1) >= slices * cols && la.lb->size(0) == N &&
                  la.lb->size(1) >= lb_cols && la.s->stride(1) == 1 && la.lb->stride(1) == 1 &&
                  la.s->stride(0) % 8 == 0 && la.lb->stride(0) % 8 == 0 && aligned16(*la.s) && aligned16(*la.lb),
              "mxfp4_gemm: bf16 s [M, slices * adapters * rank] and lb [N, ", lb_cols,
              "] with 16-byte aligned rows required");
    p.lora = 1;
    p.lp.rank_blocks = (int)la.rank / 32;
    p.lp.blocks_per_adapter = p.lp.rank_blocks * (epi == kEpiSwiGLU ? 2 : 1);
    p.lp.num_adapters = (int)la.num_adapters;
    p.lp.num_slices = epi == kEpiSwiGLU ? 1 : (int)slices;
    for (int i = 0; epi != kEpiSwiGLU && i <= slices; ++i) p.lp.slice_bounds[i] = (int)b[i];
    if (la.tile_mask.has_value()) {
      GSB_CHECK(la.tile_mask->device() == dev && la.tile_mask->scalar_type() == at::kLong &&
                    la.tile_mask->is_contiguous() && la.tile_mask->numel() >= (M + 127) / 128,
                "mxfp4_gemm: tile_mask must hold one int64 per 128-row tile");
      p.lp.tile_mask = reinterpret_cast<const uint64_t*>(la.tile_mask->data_ptr());
    }
  }
  GSB_CHECK((x.rows + 255) / 256 * ((w.rows + 255) / 256) < (int64_t(1) << 31), "mxfp4_gemm: output too large");
  if (M == 0) return;
  auto st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  auto* ep = reinterpret_cast<uint32_t*>(err.data_ptr());

  at::Tensor work;  // codes and scales of bf16 rows; the stream orders its reuse
  if (t.bf != nullptr) {
    const int64_t code_bytes = (M * (K / 2) + 1023) / 1024 * 1024;
    work = new_tensor({code_bytes + (M + 127) / 128 * k_tiles(K) * 512}, at::kByte, dev);
    x = Codes{work.data_ptr<uint8_t>(), K / 2, work.data_ptr<uint8_t>() + code_bytes, M};
    quantize_launch(t.bf, t.ldbf, M, K, x.q, x.ld, x.sf, st);
  }
  auto tmap_s = [&](uint32_t rows) {
    return make_tmap_bf16_2d(la.s->data_ptr(), (uint64_t)M, (uint64_t)la.s->size(1), (uint64_t)la.s->stride(0), 32,
                             rows, CU_TENSOR_MAP_SWIZZLE_64B);
  };
  auto tmap_lb = [&](uint32_t rows) {
    return make_tmap_bf16_2d(la.lb->data_ptr(), (uint64_t)N, (uint64_t)la.lb->size(1), (uint64_t)la.lb->stride(0), 32,
                             rows, CU_TENSOR_MAP_SWIZZLE_64B);
  };

  if (use_pair(M, N)) {
    PairParams pp{};
    pp.M = M;
    pp.N = N;
    pp.kstages = p.kstages;
    pp.scale = p.scale;
    pp.out = p.out;
    pp.ldo = p.ldo;
    pp.residual = p.residual;
    pp.ldr = p.ldr;
    pp.a4 = p.a4;
    pp.lda4 = p.lda4;
    pp.sfa_out = p.sfa_out;
    pp.lora = p.lora;
    pp.lp = p.lp;
    const CUtensorMap tx = make_tmap_codes(x, K, 128), tw = make_tmap_codes(w, K, 128);
    const CUtensorMap tsfx = make_tmap_sf(x, p.kstages, 1), tsfw = make_tmap_sf(w, p.kstages, 2);
    const CUtensorMap ts = lora ? tmap_s(128) : tx, tlb = lora ? tmap_lb(64) : tw;
    const CUtensorMap to = epi == kEpiSwiGLU
                               ? tx
                               : make_tmap_bf16_2d(p.out, (uint64_t)M, (uint64_t)N, (uint64_t)p.ldo, 64, 32,
                                                   CU_TENSOR_MAP_SWIZZLE_128B);
    switch (epi) {
      case kEpiStore: launch_pair<kEpiStore>(tx, tw, tsfx, tsfw, ts, tlb, to, pp, ep, st); break;
      case kEpiResAdd: launch_pair<kEpiResAdd>(tx, tw, tsfx, tsfw, ts, tlb, to, pp, ep, st); break;
      default: launch_pair<kEpiSwiGLU>(tx, tw, tsfx, tsfw, ts, tlb, to, pp, ep, st); break;
    }
    return;
  }

  const SplitPlan s = split_plan(M, N, K);
  GSB_CHECK(s.token_tiles <= 65535, "mxfp4_gemm: too many rows");
  p.reduce_off = s.reduce_off;
  p.give_up = g_split_give_up;
  p.sfx = x.sf;
  p.sfw = w.sf;
  p.stages = s.stages;
  p.stage_bytes = s.stage_bytes;
  p.mt_rows = s.mt_rows;
  p.ks = s.ks;
  p.rows_per = rows_per_part(s.mt_rows, s.ks);
  p.tmem_cols = s.tmem_cols;
  const uint32_t mp = (uint32_t)((s.mt_rows + 15) / 16 * 16);
  const CUtensorMap tw = make_tmap_codes(w, K, BW), tx = make_tmap_codes(x, K, mp);
  const CUtensorMap tlb = lora ? tmap_lb(BW) : tw, ts = lora ? tmap_s(mp) : tx;
  switch (epi) {
    case kEpiStore: launch_split<kEpiStore>(tw, tx, tlb, ts, p, s, ep, st); break;
    case kEpiResAdd: launch_split<kEpiResAdd>(tw, tx, tlb, ts, p, s, ep, st); break;
    default: launch_split<kEpiSwiGLU>(tw, tx, tlb, ts, p, s, ep, st); break;
  }
}

static void check_epi(int64_t epi) {
  GSB_CHECK(epi == kEpiStore || epi == kEpiResAdd, "mxfp4_gemm: epilogue must be store (0) or residual add (1)");
}

}  // namespace f4
}  // namespace gsb

using namespace gsb;

// out [M, N] bf16 = epi(x4 . w4^T (+ s . lb^T)); epi 0: times scale, 1: residual + scale * that.
at::Tensor gsb_mxfp4_gemm(const at::Tensor& x4, const at::Tensor& sfx, const at::Tensor& w4, const at::Tensor& sfw,
                          const c10::optional<at::Tensor>& out_, int64_t epi, double scale,
                          const c10::optional<at::Tensor>& residual, const c10::optional<at::Tensor>& s,
                          const c10::optional<at::Tensor>& lb, const c10::optional<at::Tensor>& tile_mask, int64_t rank,
                          int64_t num_adapters, const c10::optional<std::vector<int64_t>>& slice_bounds,
                          const at::Tensor& err) {
  f4::check_epi(epi);
  GSB_CHECK(x4.dim() == 2 && w4.dim() == 2, "mxfp4_gemm: operands [M, K / 2] and [N, K / 2] required");
  const int64_t K = x4.size(1) * 2;
  const at::Device dev = x4.device();
  const f4::Codes x = f4::check_operand("x", x4, sfx, K, dev), w = f4::check_operand("w", w4, sfw, K, dev);
  c10::cuda::CUDAGuard g(dev);
  const at::Tensor out = out_.has_value() ? *out_ : f4::new_tensor({x.rows, w.rows}, at::kBFloat16, dev);
  if (out_.has_value()) f4::check_output_apart("out", out, &x4, &sfx, w4, sfw, s, lb);
  f4::run_gemm(f4::Tokens{x, nullptr, 0}, w, K, &out, (int)epi, scale, residual, nullptr,
               f4::LoraArgs{s, lb, tile_mask, rank, num_adapters,
                            slice_bounds.has_value() ? *slice_bounds : std::vector<int64_t>{0, w.rows}},
               err, dev);
  return out;
}

// The same from bf16 rows x [M, K], quantised into a workspace of the call.
at::Tensor gsb_mxfp4_linear(const at::Tensor& x, const at::Tensor& w4, const at::Tensor& sfw,
                            const c10::optional<at::Tensor>& out_, int64_t epi, double scale,
                            const c10::optional<at::Tensor>& residual, const c10::optional<at::Tensor>& s,
                            const c10::optional<at::Tensor>& lb, const c10::optional<at::Tensor>& tile_mask,
                            int64_t rank, int64_t num_adapters, const c10::optional<std::vector<int64_t>>& slice_bounds,
                            const at::Tensor& err) {
  f4::check_epi(epi);
  f4::check_rows("mxfp4_linear", "x", x, x.device());
  const int64_t M = x.size(0), K = x.size(1);
  const at::Device dev = x.device();
  const f4::Codes w = f4::check_operand("w", w4, sfw, K, dev);
  c10::cuda::CUDAGuard g(dev);
  const at::Tensor out = out_.has_value() ? *out_ : f4::new_tensor({M, w.rows}, at::kBFloat16, dev);
  // out may be x, which is quantised before the product starts
  if (out_.has_value()) f4::check_output_apart("out", out, nullptr, nullptr, w4, sfw, s, lb);
  f4::run_gemm(f4::Tokens{f4::Codes{nullptr, 0, nullptr, M}, x.data_ptr(), x.stride(0)}, w, K, &out, (int)epi, scale,
               residual, nullptr,
               f4::LoraArgs{s, lb, tile_mask, rank, num_adapters,
                            slice_bounds.has_value() ? *slice_bounds : std::vector<int64_t>{0, w.rows}},
               err, dev);
  return out;
}

// (a4, sf) <- quantised silu(gate) * up of the gate/up product; `act` also as bf16.
std::tuple<at::Tensor, at::Tensor> gsb_mxfp4_gemm_swiglu(
    const at::Tensor& x4, const at::Tensor& sfx, const at::Tensor& w4, const at::Tensor& sfw,
    const c10::optional<at::Tensor>& a4_, const c10::optional<at::Tensor>& sf_, const c10::optional<at::Tensor>& act,
    const c10::optional<at::Tensor>& s, const c10::optional<at::Tensor>& lb, const c10::optional<at::Tensor>& tile_mask,
    int64_t rank, int64_t num_adapters, const at::Tensor& err) {
  GSB_CHECK(x4.dim() == 2 && w4.dim() == 2, "mxfp4_gemm_swiglu: operands [M, K / 2] and [2 I, K / 2] required");
  const int64_t K = x4.size(1) * 2, I = w4.size(0) / 2;
  const at::Device dev = x4.device();
  const f4::Codes x = f4::check_operand("x", x4, sfx, K, dev), w = f4::check_operand("w", w4, sfw, K, dev);
  GSB_CHECK(w.rows > 0 && w.rows % 128 == 0,
            "mxfp4_gemm_swiglu: the weight must hold a multiple of 128 rows (64 gate, 64 up, ...)");
  c10::cuda::CUDAGuard g(dev);
  at::Tensor a4 = a4_.value_or(at::Tensor()), sf = sf_.value_or(at::Tensor());
  f4::make_codes(x.rows, I, dev, a4, sf);
  const f4::Codes o = f4::check_operand("output", a4, sf, I, dev);
  GSB_CHECK(o.rows == x.rows, "mxfp4_gemm_swiglu: output codes must be [M, I / 2]");
  if (a4_.has_value() || sf_.has_value()) {
    f4::check_output_apart("output codes", a4, &x4, &sfx, w4, sfw, s, lb);
    f4::check_output_apart("output scales", sf, &x4, &sfx, w4, sfw, s, lb);
    f4::check_apart("mxfp4_gemm_swiglu", "output scales", sf, "the output codes", a4);
  }
  if (act.has_value()) {
    f4::check_output_apart("act", *act, &x4, &sfx, w4, sfw, s, lb);
    f4::check_apart("mxfp4_gemm_swiglu", "act", *act, "the output codes", a4);
    f4::check_apart("mxfp4_gemm_swiglu", "act", *act, "the output scales", sf);
  }
  f4::run_gemm(f4::Tokens{x, nullptr, 0}, w, K, act.has_value() ? &*act : nullptr, kEpiSwiGLU, 1.0, c10::nullopt, &o,
               f4::LoraArgs{s, lb, tile_mask, rank, num_adapters, {}}, err, dev);
  return {a4, sf};
}

// Forces the smallest M that takes the pair kernel (-1: the measured rule); returns the previous value.
int64_t gsb_mxfp4_pair_min_m(int64_t m) {
  const int64_t old = f4::g_pair_min_m;
  f4::g_pair_min_m = (int)std::max<int64_t>(-1, std::min<int64_t>(m, 1 << 30));
  return old;
}

// The plan of an M x N x K product: {1 for the pair kernel, tokens per tile, K parts per tile, stages}.
std::vector<int64_t> gsb_mxfp4_gemm_plan(int64_t M, int64_t N, int64_t K) {
  using namespace gsb::f4;
  GSB_CHECK(M >= 1 && M < (int64_t(1) << 24) && N >= 1 && N < (int64_t(1) << 24) && K >= 1 && K < (int64_t(1) << 31),
            "mxfp4_gemm_plan: sizes out of range");
  if (use_pair((int)M, (int)N)) return {1, 256, 1, PairCfg::STAGES};
  const SplitPlan s = split_plan((int)M, (int)N, K);
  return {0, s.mt_rows, s.ks, s.stages};
}

// Makes one K part of every split-kernel cluster behave as if a wait had run out (-1: none); returns the previous
// value.
int64_t gsb_mxfp4_split_give_up(int64_t part) {
  const int64_t old = gsb::f4::g_split_give_up;
  gsb::f4::g_split_give_up = (int)std::max<int64_t>(-1, std::min<int64_t>(part, gsb::f4::MAX_KS));
  return old;
}
