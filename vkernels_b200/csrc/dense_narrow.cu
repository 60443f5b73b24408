// dense_narrow.cu - products of the dense feed-forward operators for small batches: weights as the M operand, split over k.
//
// A decode batch reads every weight once and does next to nothing with it: the time is that of the weights' way from memory.
// 128 weight rows are one tile (gated: 64 gate rows and the 64 up rows of the same features), up to 192 tokens, rounded up to
// 16, are the MMA's N. The k range of a tile is cut over the CTAs of a cluster, so that all SMs stream weights however few
// tiles there are. Every CTA leaves its partial sums [token][row] in its own shared memory, where the ring was, and after a
// cluster barrier each adds its share of the results over the cluster, rank after rank: no atomics, no scratch in memory, the
// same bits every time. (Sending the sums to their owner instead needs a barrier more - every ring has to be free first - and
// took 1 to 5 us longer.)
//
// Bound by the start (about 2 us until the first weights arrive) and the join (1 us, 2 to 3 from 64 tokens on) around the weights'
// way: 8192 -> 8192 24 us for 1 token (134 MB, 5.6 TB/s over all), 7168 -> 2 x 2048 gated 12.8 us (59 MB), 2880 -> 2880 6.4 us (17 MB).
#include <algorithm>

#include "dense_tc.cuh"

namespace vkernels::kernels::cuda {

namespace {

constexpr int kMaxStages = 12, kMaxSplit = 8;
constexpr int kMaxSmem = 232448;
constexpr int kEpiWarps = 8, kEpiThreads = 32 * kEpiWarps, kThreads = kEpiThreads + 64;   // and producer, MMA issuer
constexpr int kAhead = 4;
constexpr int kMaxTileTok = 192;
constexpr int kWeightBytes = 16384;            // 128 rows x 64 k

struct NarrowBars {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

struct NarrowParams {
  int M, N;                   // tokens, features
  int w_mn;
  int tile_tok, tok_tiles;    // tokens of a tile (a multiple of 16), tiles of tokens
  int stages, stage_bytes, tmem_cols, k_blocks;
  int act;
  GatedKind kind;
  const uint16_t* bias;
  const uint16_t* residual;
  uint16_t* out;
  float* preact;
  int64_t ldr, ldo, ldp;
  int vec_r, vec_o, vec_p, vec_p2;   // whole accesses of four values possible (vec_p2: the up half of preact)
  int* status;
};

__device__ __forceinline__ void tc_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ uint32_t cluster_ctas() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_cta(uint32_t addr, uint32_t cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
  return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// Four neighbouring 16-bit values.
__device__ __forceinline__ uint2 load_four(const uint16_t* p, int n, int vec) {
  if (vec && n >= 4) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) w[j >> 1] |= (uint32_t)p[j] << ((j & 1) * 16);
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_four(uint16_t* p, const uint16_t (&v)[4], int n, int vec) {
  if (vec && n >= 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(v[0] | ((uint32_t)v[1] << 16), v[2] | ((uint32_t)v[3] << 16));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[j] = v[j];
  }
}

__device__ __forceinline__ void store_four_f32(float* p, const float (&v)[4], int n, int vec) {
  if (vec && n >= 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[j] = v[j];
  }
}

template <int TYPE, bool GATED>
__global__ void __launch_bounds__(kThreads, 2)
dense_narrow_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const NarrowParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t ring = smem_u32(smem);
  NarrowBars* bars = reinterpret_cast<NarrowBars*>(smem + p.stages * p.stage_bytes);
  volatile int* abort_flag = &bars->abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = (int)cluster_ctas(), rank = (int)cluster_ctarank();
  const int cluster = (int)blockIdx.x / split, tile = cluster / p.tok_tiles;
  const int f0 = tile * (GATED ? 64 : 128);                     // first feature of the tile
  const int t0 = cluster % p.tok_tiles * p.tile_tok, n_tok = min(p.tile_tok, p.M - t0);
  const int kb0 = (int)((int64_t)p.k_blocks * rank / split), kb1 = (int)((int64_t)p.k_blocks * (rank + 1) / split);

  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(smem_u32(&bars->full[i]), 1);
      mbar_init(smem_u32(&bars->empty[i]), 1);
    }
    mbar_init(smem_u32(&bars->acc_full), 1);
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kEpiWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)),
                 "r"((uint32_t)p.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  wait_for_earlier_kernels();

  constexpr int F4 = GATED ? 16 : 32;         // fours of features of a token in a tile
  const int total = n_tok * F4;               // a CTA of the cluster takes every split-th group of kEpiThreads of them
  uint2 ahead[kAhead];

  if (warp == kEpiWarps) {
    // ------------------------------ producer --------------------------------
    if (elect_one()) {
      Ring s;
      int issued = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const uint32_t full = smem_u32(&bars->full[s.slot]), dst = ring + s.slot * p.stage_bytes;
        if (!mbar_wait(smem_u32(&bars->empty[s.slot]), s.phase ^ 1u, abort_flag, 61)) break;
        mbar_expect_tx(full, p.stage_bytes);
        if (GATED) {
          tma_load_2d(dst, &map_w, kb * 64, f0, full);
          tma_load_2d(dst + 8192, &map_w, kb * 64, p.N + f0, full);
        } else if (p.w_mn) {
          tma_load_2d(dst, &map_w, f0, kb * 64, full);
          tma_load_2d(dst + 8192, &map_w, f0 + 64, kb * 64, full);
        } else {
          tma_load_2d(dst, &map_w, kb * 64, f0, full);
        }
        tma_load_2d(dst + kWeightBytes, &map_x, kb * 64, t0, full);
        ++issued;
        s.advance(p.stages);
      }
      if (*abort_flag != 0) {   // gave up: the copies in flight land before anybody leaves
        const long long t0 = clock64();
        for (int i = max(0, issued - p.stages); i < issued; ++i)
          while (!mbar_test(smem_u32(&bars->full[i % p.stages]), (uint32_t)(i / p.stages) & 1u) && clock64() - t0 < 2000000ll) {
          }
      }
    }
    __syncwarp();
  } else if (warp == kEpiWarps + 1) {
    // -------------------------------- MMAs ----------------------------------
    if (elect_one()) {
      const uint32_t idesc = operand_idesc<TYPE>(128, p.tile_tok, p.w_mn, 0);
      const uint32_t w_step = p.w_mn ? 2048 >> 4 : 32 >> 4;   // 16 k on
      Ring s;
      bool go = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&bars->full[s.slot]), s.phase, abort_flag, 62)) {
          go = false;
          break;
        }
        tc_fence_after();
        const uint32_t src = ring + s.slot * p.stage_bytes;
        const uint64_t wd = operand_desc(src, p.w_mn), xd = operand_desc(src + kWeightBytes, 0);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_ss(tmem_base, wd + k * w_step, xd + k * 2, idesc, kb != kb0 || k != 0);
        tc_commit(smem_u32(&bars->empty[s.slot]));
        s.advance(p.stages);
      }
      if (go) tc_commit(smem_u32(&bars->acc_full));
    }
    __syncwarp();
  } else {
    // the residual of this thread's first results, on its way while the weights stream
    if (!GATED && p.residual) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = rank * kEpiThreads + tid + j * split * kEpiThreads, f = f0 + i % F4 * 4;
        if (i < total && f < p.N) ahead[j] = load_four(p.residual + (t0 + i / F4) * p.ldr + f, p.N - f, p.vec_r);
      }
    }
    const bool ready = mbar_wait(smem_u32(&bars->acc_full), 0, abort_flag, 63);
    if (__all_sync(0xFFFFFFFFu, ready)) {
      tc_fence_after();
      float* mine = reinterpret_cast<float*>(smem) + (warp & 3) * 32 + lane;
      const uint32_t lanes = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
      for (int c = (warp >> 2) * 16; c < n_tok; c += kEpiWarps / 4 * 16) {
        uint32_t v[16];
        tc_ld16(lanes + c, v);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < n_tok) mine[(c + j) * 128] = __uint_as_float(v[j]);
      }
    }
  }
  tc_fence_before();
  __syncwarp();   // the cluster barrier is .aligned: a warp's lanes arrive as one
  if (split > 1) cluster_sync_all();
  else __syncthreads();

  // ---------------------------- join and epilogue ----------------------------
  if (warp < kEpiWarps && *abort_flag == 0) {
#pragma unroll 1
    for (int i = rank * kEpiThreads + tid, it = 0; i < total; i += split * kEpiThreads, ++it) {
      const int64_t t = t0 + i / F4;
      const int f = f0 + i % F4 * 4, left = p.N - f;
      if (left <= 0) continue;
      const uint32_t at = ring + (uint32_t)(i / F4 * 128 + i % F4 * 4) * 4;
      uint2 r = make_uint2(0, 0);
      if (!GATED && p.residual) {
        if (it < kAhead) {
#pragma unroll
          for (int j = 0; j < kAhead; ++j)
            if (it == j) r = ahead[j];
        } else {
          r = load_four(p.residual + t * p.ldr + f, left, p.vec_r);
        }
      }
      float4 part[kMaxSplit], part_u[GATED ? kMaxSplit : 1];
#pragma unroll
      for (int c = 0; c < kMaxSplit; ++c)
        if (c < split) {
          const uint32_t from = split > 1 ? map_to_cta(at, c) : at;
          part[c] = ld_cluster4(from);
          if (GATED) part_u[GATED ? c : 0] = ld_cluster4(from + 256);
        }
      float z[4] = {}, zu[4] = {};
#pragma unroll
      for (int c = 0; c < kMaxSplit; ++c)
        if (c < split) {
          z[0] += part[c].x, z[1] += part[c].y, z[2] += part[c].z, z[3] += part[c].w;
          if (GATED) {
            const float4 v = part_u[GATED ? c : 0];
            zu[0] += v.x, zu[1] += v.y, zu[2] += v.z, zu[3] += v.w;
          }
        }
      if (p.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < left) {
            z[j] += dense_to_f32<TYPE>(p.bias[f + j]);
            if (GATED) zu[j] += dense_to_f32<TYPE>(p.bias[p.N + f + j]);
          }
      }
      uint16_t y[4];
      if (p.preact) {
        store_four_f32(p.preact + t * p.ldp + f, z, left, p.vec_p);
        if (GATED) store_four_f32(p.preact + t * p.ldp + p.N + f, zu, left, p.vec_p2);
      }
      if (GATED) {
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = dense_from_f32<TYPE>(dense_gated(p.kind.act, z[j], zu[j], p.kind));
      } else {
        const float2 r0 = dense_unpack<TYPE>(r.x), r1 = dense_unpack<TYPE>(r.y);
        const float res[4] = {r0.x, r0.y, r1.x, r1.y};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v = p.act != kActNone ? dense_act(p.act, z[j]) : z[j];
          if (p.residual) v += res[j];
          y[j] = dense_from_f32<TYPE>(v);
        }
      }
      store_four(p.out + t * p.ldo + f, y, left, p.vec_o);
    }
  }

  // ------------------------------ teardown ---------------------------------
  __syncwarp();   // lanes leave the join one by one
  if (split > 1) cluster_sync_all();   // nobody reads this CTA's partial sums any more
  else __syncthreads();
  if (warp == kEpiWarps + 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)p.tmem_cols) : "memory");
  if (tid == 0 && bars->abort_flag != 0) atomicExch(p.status, 100 + bars->abort_flag);
}

// How many clusters of `split` CTAs fit on the device with one CTA an SM (the SMs come in groups that a cluster cannot leave).
// Asked of the runtime once per device for a CTA that fills an SM; where two fit, twice as many clusters do.
int resident_clusters(int split) {
  static std::atomic<int> known[64][kMaxSplit + 1];
  int dev = 0;
  VK_CUDA_CHECK(cudaGetDevice(&dev));
  int n = dev >= 0 && dev < 64 ? known[dev][split].load() : 0;
  if (n == 0) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)split);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kMaxSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    VK_CUDA_CHECK(cudaFuncSetAttribute(dense_narrow_kernel<kDenseBf16, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    VK_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, dense_narrow_kernel<kDenseBf16, false>, &cfg));
    if (n < 1) n = 1;
    if (dev >= 0 && dev < 64) known[dev][split].store(n);
  }
  return n;
}

struct NarrowPlan {
  int per_sm, tile_tok, tok_tiles, tiles, split, stages, stage_bytes;
  float us;
};
constexpr int kExtraSmem = (int)sizeof(NarrowBars) + 1024;
NarrowPlan plan_of(const DenseGemm& g, int tok_tiles) {
  NarrowPlan n;
  n.tile_tok = ((g.M + tok_tiles - 1) / tok_tiles + 15) / 16 * 16;
  n.tok_tiles = (g.M + n.tile_tok - 1) / n.tile_tok;
  n.stage_bytes = kWeightBytes + n.tile_tok * 128;
  // Two CTAs an SM for a handful of tokens, where one starts or joins while the other streams; above, where the join counts, one
  // with the whole ring: half the clusters, and half the partial sums in flight between them. 2880 -> 2 x 2880 gated 9.0 us with two
  // and 9.4 with one for 1 token, 11.9 and 10.8 for 64; 7168 -> 2 x 2048 gated 12.8 and 13.2, 16.4 and 14.2; 2880 -> 2880 6.4 and
  // 6.4, 9.6 and 8.1.
  n.per_sm = g.M <= 8 ? 2 : 1;
  n.stages = std::min(kMaxStages, ((n.per_sm == 2 ? 113 * 1024 : kMaxSmem) - kExtraSmem) / n.stage_bytes);
  const int tile_n = g.gated ? 64 : 128;
  n.tiles = (g.N + tile_n - 1) / tile_n * n.tok_tiles;
  // the largest split whose clusters are all resident at once
  n.split = std::min(kMaxSplit, (g.K + 63) / 64);
  while (n.split > 1 && n.tiles > resident_clusters(n.split) * n.per_sm) --n.split;
  // Its time: start, the weights' way from memory or what an SM takes in of weights and tokens - whichever is longer -, join.
  // Measured: 2880 -> 2880 6.4 us for 1 token, 8.1 for 64, 9.7 for 128, 13.2 for 256; 7168 -> 2 x 2048 gated 12.8, 14.2, 16.0, 19.9;
  // 2048 -> 7168 8.4, 10.3, 13.1, 18.8; 7168 -> 2048 for 300 and 512 tokens 19.1 and 20.8 (29 as CTA pairs).
  const float rows = g.gated ? 2.0f * (float)g.N : (float)g.N, m = (float)g.M;
  const float memory = 2.0f * (rows * (float)g.K + m * (float)g.K + m * (float)g.N) / 6.5e6f;
  const int at_once = sm_count() * n.per_sm;
  const float waves = (float)(((int64_t)n.tiles * n.split + at_once - 1) / at_once);
  const float fill = waves * (float)n.per_sm * (float)g.K / (float)n.split * (256.0f + 2.0f * (float)n.tile_tok) / 130e3f;
  n.us = 3.4f + std::max(memory, fill) + (g.M > 16 ? 0.8f : 0.0f) + 0.015f * (float)n.tile_tok;
  return n;
}
// Tokens in as many tiles as take the least time: wider tiles bring the weights to fewer SMs, narrower ones join sooner. At most 192
// (256 tokens of 7168 -> 2 x 2048 gated: 19.7 us as two tiles, 22.6 as one).
NarrowPlan plan_narrow(const DenseGemm& g) {
  NarrowPlan best = plan_of(g, (g.M + kMaxTileTok - 1) / kMaxTileTok);
  for (int tiles = best.tok_tiles + 1; tiles <= (g.M + 63) / 64; ++tiles) {
    const NarrowPlan n = plan_of(g, tiles);
    if (n.us < best.us) best = n;
  }
  return best;
}

template <int TYPE, bool GATED>
void launch_narrow(const DenseGemm& g, cudaStream_t stream) {
  static std::atomic<bool> configured[64];
  int dev = 0;
  VK_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev].load()) {
    VK_CUDA_CHECK(cudaFuncSetAttribute(dense_narrow_kernel<TYPE, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    if (dev >= 0 && dev < 64) configured[dev].store(true);
  }
  const NarrowPlan n = plan_narrow(g);
  NarrowParams p{};
  p.M = g.M;
  p.N = g.N;
  p.w_mn = g.b.mn_major;
  p.tile_tok = n.tile_tok;
  p.tok_tiles = n.tok_tiles;
  p.stages = n.stages;
  p.stage_bytes = n.stage_bytes;
  p.k_blocks = (g.K + 63) / 64;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.tile_tok) p.tmem_cols *= 2;
  p.act = g.act;
  p.kind = g.kind;
  p.bias = g.bias;
  p.residual = g.residual;
  p.out = g.out;
  p.preact = g.preact;
  p.ldr = g.ldr;
  p.ldo = g.ldo;
  p.ldp = g.ldp;
  const auto aligned8 = [](const void* q, int64_t ld) { return (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ld % 4 == 0; };
  p.vec_r = aligned8(g.residual, g.ldr);
  p.vec_o = aligned8(g.out, g.ldo);
  p.vec_p = (reinterpret_cast<uintptr_t>(g.preact) & 15u) == 0 && g.ldp % 4 == 0;
  p.vec_p2 = p.vec_p && g.N % 4 == 0;
  p.status = status_address();
  const CUtensorMap w = g.b.mn_major ? sm100_make_map_bf16(g.b.p, (uint64_t)g.N, (uint64_t)g.K, (uint64_t)g.b.ld * 2, 64)
                                     : sm100_make_map_bf16(g.b.p, (uint64_t)g.K, GATED ? 2 * (uint64_t)g.N : (uint64_t)g.N,
                                                           (uint64_t)g.b.ld * 2, GATED ? 64 : 128);
  const CUtensorMap x = sm100_make_map_bf16(g.a.p, (uint64_t)g.K, (uint64_t)g.M, (uint64_t)g.a.ld * 2, (uint32_t)p.tile_tok);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(n.tiles * n.split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)(p.stages * p.stage_bytes + kExtraSmem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)n.split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  overlap_launch(attr[1]);
  cfg.numAttrs = 2;
  VK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, dense_narrow_kernel<TYPE, GATED>, w, x, p));
}

}  // namespace

float dense_narrow_us(const DenseGemm& g) { return plan_narrow(g).us; }

// A is the batch (contiguous along k), B the weight in either order.
void launch_dense_narrow(const DenseGemm& g, cudaStream_t stream) {
  expects(!g.a.mn_major, "dense product: the small-batch form reads its rows along k");
  if (g.type == kDenseBf16) {
    if (g.gated) launch_narrow<kDenseBf16, true>(g, stream);
    else launch_narrow<kDenseBf16, false>(g, stream);
  } else {
    if (g.gated) launch_narrow<kDenseFp16, true>(g, stream);
    else launch_narrow<kDenseFp16, false>(g, stream);
  }
}

}  // namespace vkernels::kernels::cuda
