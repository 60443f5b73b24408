// dense_gemm.cu - products of the dense feed-forward operators on tcgen05: CTA pairs, 256 x 256 tiles.
//
// out[m, n] = sum_k A[m, k] B[n, k] with either operand contiguous along k or along its own index (the backward products read
// the weight, x and the gradient as they lie: the tensor map brings 64 x 64 boxes, and the matrix descriptor says which index
// is contiguous). A pair of CTAs (cta_group::2) works on 256 rows of A and 256 of B: each CTA stages 128 of either in shared
// memory (64 k a stage, 128-byte swizzle), one thread of the leader issues the MMAs, each CTA holds its 128 result rows in
// tensor memory. Two accumulators of 256 columns: eight epilogue warps empty one while the other fills. Persistent, tiles
// dealt out in groups of eight row tiles by all column tiles, so that the pairs at work share their operands in L2.
//
// In the gated form a tile's 256 rows of B are 128 gate rows (staged by the leader) and the 128 up rows of the same features
// (staged by its peer): an epilogue thread finds a feature's gate and up sums 128 columns apart in its own lane.
#include <atomic>

#include "dense.hpp"
#include "dense_math.cuh"
#include "sm100.cuh"

namespace vkernels::kernels::cuda {

CUtensorMap sm100_make_map_bf16(const void* ptr, uint64_t inner, uint64_t outer, uint64_t pitch_bytes, uint32_t box_outer);
int* sm100_status_address();

namespace {

constexpr int kStages = 6, kStageBytes = 32768;        // 128 rows of A and of B, 64 k each
constexpr int kEpiWarps = 8, kThreads = 32 * (kEpiWarps + 2);
constexpr int kStagingBytes = 4096;                    // of one epilogue warp: 32 rows x 64 values
constexpr int kBn = 256;
constexpr int kGroupM = 8;

struct WideBars {
  uint64_t full[kStages], empty[kStages];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};
constexpr int kWideSmem = kStages * kStageBytes + kEpiWarps * kStagingBytes + (int)sizeof(WideBars) + 1024;

struct WideParams {
  int M, N, K;                // N: columns of the result (gated: features)
  int a_mn, b_mn;
  int tiles_m, tiles_n, n_tiles, k_blocks;
  int act;
  float limit, beta, linear_beta;
  const uint16_t* bias;
  const uint16_t* residual;
  uint16_t* out;
  uint16_t* preact;
  int64_t ldr, ldo, ldp;
  int vec_r, vec_o, vec_p, vec_p2;   // 16-byte accesses possible (vec_p2: the up half of preact)
  int* status;
};

__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(bar & 0xFEFFFFFFu)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Descriptor of a staged operand. Contiguous along k: rows of 64 k, groups of 8 rows 1024 bytes apart. Contiguous along the
// other index: chunks of 64 indexes x 64 k, 8192 bytes apart, groups of 8 k 1024 bytes apart. 128-byte swizzle either way.
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem_addr, int mn_major) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(mn_major ? 8192 >> 4 : 1) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// The staging buffer of a warp holds 32 rows x 64 values, eight units of 16 bytes a row, unit u of row r at u ^ (r % 8): a
// thread that owns a row writes its units, eight threads at a time move a row to or from memory, both without bank conflicts.
__device__ __forceinline__ uint32_t staging_at(uint32_t base, int row, int unit) { return base + row * 128 + ((unit ^ (row & 7)) << 4); }
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// rows x cols (at most 32 x 64) of a row-major matrix, from and to the staging buffer.
__device__ __forceinline__ void staging_out(uint32_t base, uint16_t* p, int64_t ld, int rows, int cols, int vec, int lane) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3), u = lane & 7;
    if (r >= rows) continue;
    const uint4 v = lds128(staging_at(base, r, u));
    uint16_t* q = p + (int64_t)r * ld + u * 8;
    if (vec && u * 8 + 8 <= cols) {
      *reinterpret_cast<uint4*>(q) = v;
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (u * 8 + j < cols) q[j] = (uint16_t)(w[j >> 1] >> ((j & 1) * 16));
    }
  }
}
__device__ __forceinline__ void staging_in(uint32_t base, const uint16_t* p, int64_t ld, int rows, int cols, int vec, int lane) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3), u = lane & 7;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const uint16_t* q = p + (int64_t)r * ld + u * 8;
      if (vec && u * 8 + 8 <= cols) {
        v = *reinterpret_cast<const uint4*>(q);
      } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (u * 8 + j < cols) w[j >> 1] |= (uint32_t)q[j] << ((j & 1) * 16);
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    sts128(staging_at(base, r, u), v);
  }
}

template <int TYPE, bool GATED>
__global__ void __cluster_dims__(2) __launch_bounds__(kThreads, 1)
dense_wide_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const WideParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t ring = smem_u32(smem);
  WideBars* bars = reinterpret_cast<WideBars*>(smem + kStages * kStageBytes + kEpiWarps * kStagingBytes);
  volatile int* abort_flag = &bars->abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&bars->full[i]), 1);
      mbar_init(smem_u32(&bars->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars->acc_full[i]), 1);
      mbar_init(smem_u32(&bars->acc_empty[i]), 2 * kEpiWarps);
    }
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kEpiWarps) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the peer's barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  const int unit = blockIdx.x >> 1, n_units = gridDim.x >> 1;
  const int per_group = kGroupM * p.tiles_n;
  const auto place = [&](int t, int& tm, int& tn) {
    const int first = t / per_group * kGroupM, in = t % per_group, high = min(kGroupM, p.tiles_m - first);
    tm = first + in % high;
    tn = in / high;
  };

  if (warp == kEpiWarps) {
    // ------------------------------ producer --------------------------------
    if (elect_one()) {
      Ring s;
      long long issued = 0;
      bool go = true;
      for (int t = unit; t < p.n_tiles && go; t += n_units) {
        int tm, tn;
        place(t, tm, tn);
        const int m0 = tm * 256 + (int)rank * 128;
        const int n0 = GATED ? tn * 128 + (int)rank * p.N : tn * kBn + (int)rank * 128;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          const uint32_t full = smem_u32(&bars->full[s.slot]), dst = ring + s.slot * kStageBytes;
          if (!mbar_wait(smem_u32(&bars->empty[s.slot]), s.phase ^ 1u, abort_flag, 51)) {
            go = false;
            break;
          }
          if (rank == 0) mbar_expect_tx(full, 2 * kStageBytes);
          if (p.a_mn) {
            tma_load_2d_pair(dst, &map_a, m0, kb * 64, full);
            tma_load_2d_pair(dst + 8192, &map_a, m0 + 64, kb * 64, full);
          } else {
            tma_load_2d_pair(dst, &map_a, kb * 64, m0, full);
          }
          if (p.b_mn) {
            tma_load_2d_pair(dst + 16384, &map_b, n0, kb * 64, full);
            tma_load_2d_pair(dst + 24576, &map_b, n0 + 64, kb * 64, full);
          } else {
            tma_load_2d_pair(dst + 16384, &map_b, kb * 64, n0, full);
          }
          ++issued;
          s.advance(kStages);
        }
      }
      if (*abort_flag != 0 && rank == 0) {   // gave up: the copies in flight land before anybody leaves
        const long long t0 = clock64();
        for (long long i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
          while (!mbar_test(smem_u32(&bars->full[i % kStages]), (uint32_t)(i / kStages) & 1u) && clock64() - t0 < 2000000ll) {
          }
      }
    }
    __syncwarp();
  } else if (warp == kEpiWarps + 1) {
    // -------------------------------- MMAs ----------------------------------
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = (1u << 4) | (TYPE == kDenseBf16 ? (1u << 7) | (1u << 10) : 0u) | (p.a_mn ? 1u << 15 : 0u) |
                             (p.b_mn ? 1u << 16 : 0u) | ((uint32_t)(kBn >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
      const uint32_t a_step = p.a_mn ? 2048 >> 4 : 32 >> 4, b_step = p.b_mn ? 2048 >> 4 : 32 >> 4;   // 16 k on
      Ring s;
      int it = 0;
      bool go = true;
      for (int t = unit; t < p.n_tiles && go; t += n_units, ++it) {
        const int buf = it & 1;
        if (!mbar_wait(smem_u32(&bars->acc_empty[buf]), ((it >> 1) & 1) ^ 1, abort_flag, 52)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + buf * 256;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(smem_u32(&bars->full[s.slot]), s.phase, abort_flag, 53)) {
            go = false;
            break;
          }
          tc_fence_after();
          const uint32_t src = ring + s.slot * kStageBytes;
          const uint64_t ad = operand_desc(src, p.a_mn), bd = operand_desc(src + 16384, p.b_mn);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_ss_pair(d, ad + k * a_step, bd + k * b_step, idesc, (kb | k) != 0);
          tc_commit_pair(smem_u32(&bars->empty[s.slot]));
          s.advance(kStages);
        }
        if (go) tc_commit_pair(smem_u32(&bars->acc_full[buf]));
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ epilogue --------------------------------
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t staging = ring + kStages * kStageBytes + warp * kStagingBytes;
    int it = 0;
    for (int t = unit; t < p.n_tiles; t += n_units, ++it) {
      int tm, tn;
      place(t, tm, tn);
      const int buf = it & 1;
      const bool ready = mbar_wait(smem_u32(&bars->acc_full[buf]), (it >> 1) & 1, abort_flag, 54, 32);
      if (!__all_sync(0xFFFFFFFFu, ready)) break;
      tc_fence_after();
      const uint32_t lanes = tmem_base + buf * 256 + ((uint32_t)(quad * 32) << 16);
      const int64_t row0 = (int64_t)tm * 256 + rank * 128 + quad * 32;
      const int rows = (int)min((int64_t)32, (int64_t)p.M - row0);
      if constexpr (GATED) {
        // 64 features of this warp: gate sums at columns half * 64, up sums 128 on
        const int col0 = tn * 128 + half * 64, cols = min(64, p.N - col0);
        const uint32_t tg = lanes + half * 64, tu = tg + 128;
        float bias_g[2] = {}, bias_u[2] = {};
        if (p.bias) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (i * 32 + lane < cols) {
              bias_g[i] = dense_to_f32<TYPE>(p.bias[col0 + i * 32 + lane]);
              bias_u[i] = dense_to_f32<TYPE>(p.bias[p.N + col0 + i * 32 + lane]);
            }
        }
        if (p.preact && rows > 0 && cols > 0) {
#pragma unroll
          for (int part = 0; part < 2; ++part) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t v[32];
              tc_ld32((part ? tu : tg) + i * 32, v);
              tc_wait_ld();
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int c = u * 8 + j * 2;
                  float z0 = __uint_as_float(v[c]), z1 = __uint_as_float(v[c + 1]);
                  if (p.bias) {
                    z0 += __shfl_sync(0xFFFFFFFFu, part ? bias_u[i] : bias_g[i], c);
                    z1 += __shfl_sync(0xFFFFFFFFu, part ? bias_u[i] : bias_g[i], c + 1);
                  }
                  w[j] = dense_round_preact<TYPE>(z0, p.limit) | ((uint32_t)dense_round_preact<TYPE>(z1, p.limit) << 16);
                }
                sts128(staging_at(staging, lane, i * 4 + u), make_uint4(w[0], w[1], w[2], w[3]));
              }
            }
            __syncwarp();
            staging_out(staging, p.preact + row0 * p.ldp + (part ? p.N : 0) + col0, p.ldp, rows, cols, part ? p.vec_p2 : p.vec_p, lane);
            __syncwarp();
          }
        }
        if (rows > 0 && cols > 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t g[32], uu[32];
            tc_ld32(tg + i * 32, g);
            tc_ld32(tu + i * 32, uu);
            tc_wait_ld();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float h[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int c = u * 8 + j * 2 + e;
                  float zg = __uint_as_float(g[c]), zu = __uint_as_float(uu[c]);
                  if (p.bias) {
                    zg += __shfl_sync(0xFFFFFFFFu, bias_g[i], c);
                    zu += __shfl_sync(0xFFFFFFFFu, bias_u[i], c);
                  }
                  h[e] = dense_gated(p.act, zg, zu, p.limit, p.beta, p.linear_beta);
                }
                w[j] = dense_pack<TYPE>(h[0], h[1]);
              }
              sts128(staging_at(staging, lane, i * 4 + u), make_uint4(w[0], w[1], w[2], w[3]));
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cta(smem_u32(&bars->acc_empty[buf]), 0);
        if (rows > 0 && cols > 0) {
          staging_out(staging, p.out + row0 * p.ldo + col0, p.ldo, rows, cols, p.vec_o, lane);
          __syncwarp();
        }
      } else {
#pragma unroll 1
        for (int chunk = 0; chunk < 2; ++chunk) {
          const int col0 = tn * kBn + half * 128 + chunk * 64, cols = min(64, p.N - col0);
          const uint32_t tz = lanes + half * 128 + chunk * 64;
          const bool any = rows > 0 && cols > 0;
          float bias[2] = {};
          if (p.bias && any) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (i * 32 + lane < cols) bias[i] = dense_to_f32<TYPE>(p.bias[col0 + i * 32 + lane]);
          }
          if (p.preact && any) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t v[32];
              tc_ld32(tz + i * 32, v);
              tc_wait_ld();
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int c = u * 8 + j * 2;
                  float z0 = __uint_as_float(v[c]), z1 = __uint_as_float(v[c + 1]);
                  if (p.bias) {
                    z0 += __shfl_sync(0xFFFFFFFFu, bias[i], c);
                    z1 += __shfl_sync(0xFFFFFFFFu, bias[i], c + 1);
                  }
                  w[j] = dense_round_preact<TYPE>(z0, p.limit) | ((uint32_t)dense_round_preact<TYPE>(z1, p.limit) << 16);
                }
                sts128(staging_at(staging, lane, i * 4 + u), make_uint4(w[0], w[1], w[2], w[3]));
              }
            }
            __syncwarp();
            staging_out(staging, p.preact + row0 * p.ldp + col0, p.ldp, rows, cols, p.vec_p, lane);
            __syncwarp();
          }
          if (p.residual && any) {
            staging_in(staging, p.residual + row0 * p.ldr + col0, p.ldr, rows, cols, p.vec_r, lane);
            __syncwarp();
          }
          if (any) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t v[32];
              tc_ld32(tz + i * 32, v);
              tc_wait_ld();
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const uint32_t at = staging_at(staging, lane, i * 4 + u);
                uint32_t r[4] = {0, 0, 0, 0}, w[4];
                if (p.residual) {
                  const uint4 q = lds128(at);
                  r[0] = q.x, r[1] = q.y, r[2] = q.z, r[3] = q.w;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int c = u * 8 + j * 2;
                  float z0 = __uint_as_float(v[c]), z1 = __uint_as_float(v[c + 1]);
                  if (p.bias) {
                    z0 += __shfl_sync(0xFFFFFFFFu, bias[i], c);
                    z1 += __shfl_sync(0xFFFFFFFFu, bias[i], c + 1);
                  }
                  if (p.act != kActNone) {
                    z0 = dense_act(p.act, z0);
                    z1 = dense_act(p.act, z1);
                  }
                  if (p.residual) {
                    const float2 q = dense_unpack<TYPE>(r[j]);
                    z0 += q.x;
                    z1 += q.y;
                  }
                  w[j] = dense_pack<TYPE>(z0, z1);
                }
                sts128(at, make_uint4(w[0], w[1], w[2], w[3]));
              }
            }
          }
          if (chunk == 1) tc_fence_before();
          __syncwarp();
          if (chunk == 1 && lane == 0) mbar_arrive_cta(smem_u32(&bars->acc_empty[buf]), 0);
          if (any) {
            staging_out(staging, p.out + row0 * p.ldo + col0, p.ldo, rows, cols, p.vec_o, lane);
            __syncwarp();
          }
        }
      }
    }
  }

  // ------------------------------ teardown ---------------------------------
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the peer no longer touches this CTA's barriers or tensor memory
  if (warp == kEpiWarps) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
  if (tid == 0 && bars->abort_flag != 0) atomicExch(p.status, 100 + bars->abort_flag);
}

bool aligned16(const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0; }

int* status_address() {
  static std::atomic<int*> known[64];
  int dev = 0;
  VK_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return sm100_status_address();
  int* p = known[dev].load();
  if (p == nullptr) known[dev].store(p = sm100_status_address());
  return p;
}

// A tensor map of one operand: boxes of 64 values along the contiguous index by 128 (k contiguous) or 64 rows.
CUtensorMap operand_map(const DenseOperand& o, int64_t rows, int K) {
  return o.mn_major ? sm100_make_map_bf16(o.p, (uint64_t)rows, (uint64_t)K, (uint64_t)o.ld * 2, 64)
                    : sm100_make_map_bf16(o.p, (uint64_t)K, (uint64_t)rows, (uint64_t)o.ld * 2, 128);
}

template <int TYPE, bool GATED>
void launch_wide(const DenseGemm& g, cudaStream_t stream) {
  static std::atomic<bool> configured[64];
  int dev = 0;
  VK_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev].load()) {
    VK_CUDA_CHECK(cudaFuncSetAttribute(dense_wide_kernel<TYPE, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWideSmem));
    if (dev >= 0 && dev < 64) configured[dev].store(true);
  }
  WideParams p{};
  p.M = g.M;
  p.N = g.N;
  p.K = g.K;
  p.a_mn = g.a.mn_major;
  p.b_mn = g.b.mn_major;
  const int tile_n = GATED ? 128 : kBn;
  p.tiles_m = (g.M + 255) / 256;
  p.tiles_n = (g.N + tile_n - 1) / tile_n;
  expects((int64_t)p.tiles_m * p.tiles_n < (1ll << 30), "dense product: more than 2^30 tiles");
  p.n_tiles = p.tiles_m * p.tiles_n;
  p.k_blocks = (g.K + 63) / 64;
  p.act = g.act;
  p.limit = g.limit;
  p.beta = g.beta;
  p.linear_beta = g.linear_beta;
  p.bias = g.bias;
  p.residual = g.residual;
  p.out = g.out;
  p.preact = g.preact;
  p.ldr = g.ldr;
  p.ldo = g.ldo;
  p.ldp = g.ldp;
  p.vec_r = g.residual != nullptr && aligned16(g.residual, g.ldr);
  p.vec_o = aligned16(g.out, g.ldo);
  p.vec_p = g.preact != nullptr && aligned16(g.preact, g.ldp);
  p.vec_p2 = p.vec_p && g.N % 8 == 0;
  p.status = status_address();
  const CUtensorMap a = operand_map(g.a, g.M, g.K), b = operand_map(g.b, GATED ? 2 * (int64_t)g.N : g.N, g.K);
  const int units = min(p.n_tiles, sm_count() / 2);
  dense_wide_kernel<TYPE, GATED><<<2 * units, kThreads, kWideSmem, stream>>>(a, b, p);
  VK_CUDA_CHECK(cudaGetLastError());
}

}  // namespace

void launch_dense_wide(const DenseGemm& g, cudaStream_t stream) {
  if (g.type == kDenseBf16) {
    if (g.gated) launch_wide<kDenseBf16, true>(g, stream);
    else launch_wide<kDenseBf16, false>(g, stream);
  } else {
    if (g.gated) launch_wide<kDenseFp16, true>(g, stream);
    else launch_wide<kDenseFp16, false>(g, stream);
  }
}

}  // namespace vkernels::kernels::cuda
