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

#include "dense_tc.cuh"

namespace vkernels::kernels::cuda {

namespace {

constexpr int kStages = 6, kStageBytes = 32768;        // 128 rows of A and of B, 64 k each
constexpr int kEpiWarps = 8, kThreads = 32 * (kEpiWarps + 2);
constexpr int kStagingBytes = 4096;                    // of one epilogue warp: 32 rows x 64 values
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
  int bn;                     // rows of B a tile: a multiple of 32 from 64 to 256
  int stage_bytes;            // of one CTA: what the copies of a stage bring
  int tiles_m, tiles_n, n_tiles, k_blocks;
  int act;
  float limit, beta, linear_beta;
  const uint16_t* bias;
  const uint16_t* residual;
  uint16_t* out;
  float* preact;
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
__device__ __forceinline__ void sts16(uint32_t addr, uint16_t v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(v) : "memory"); }
// rows x cols (at most 32 x 64) of a row-major matrix: a lane holds unit lane % 8 of rows lane / 8, 4 + lane / 8, ... The
// common case - whole units on 16 bytes - is straight code, all eight accesses in flight at once (with a test at each the
// loads wait for one another: 10 us instead of 2 for the last tile of a launch with a residual).
struct Piece {
  uint4 v[8];
};
__device__ __forceinline__ void piece_load(Piece& d, const uint16_t* p, int64_t ld, int rows, int cols, int lane) {
  const int r0 = lane >> 3, u = lane & 7;
  const uint16_t* q = p + (int64_t)r0 * ld + u * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    d.v[i] = i * 4 + r0 < rows && u * 8 + 8 <= cols ? *reinterpret_cast<const uint4*>(q + (int64_t)(i * 4) * ld) : make_uint4(0, 0, 0, 0);
}
// ... with the columns behind the last whole unit fetched one by one.
__device__ __forceinline__ void piece_to_staging(const Piece& d, uint32_t base, const uint16_t* p, int64_t ld, int rows, int cols, int lane) {
#pragma unroll
  for (int i = 0; i < 8; ++i) sts128(staging_at(base, i * 4 + (lane >> 3), lane & 7), d.v[i]);
  if ((cols & 7) == 0) return;
  __syncwarp();
  for (int c = cols & ~7; c < cols; ++c)
    if (lane < rows) sts16(staging_at(base, lane, c >> 3) + (c & 7) * 2, p[(int64_t)lane * ld + c]);
}
// Rows that start anywhere: a row at a time, a value a lane; sixteen rows on their way before the first is put down.
__device__ __forceinline__ void values_in(uint32_t base, const uint16_t* p, int64_t ld, int rows, int cols, int lane) {
#pragma unroll 1
  for (int first = 0; first < 32; first += 16) {
    uint16_t v[16][2];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) v[i][h] = first + i < rows && h * 32 + lane < cols ? p[(int64_t)(first + i) * ld + h * 32 + lane] : (uint16_t)0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) sts16(staging_at(base, first + i, (h * 32 + lane) >> 3) + (lane & 7) * 2, v[i][h]);
  }
}
__device__ __forceinline__ void staging_out(uint32_t base, uint16_t* p, int64_t ld, int rows, int cols, int vec, int lane) {
  const int r0 = lane >> 3, u = lane & 7;
  uint16_t* q = p + (int64_t)r0 * ld + u * 8;
  if (vec && (cols & 7) == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 v = lds128(staging_at(base, i * 4 + r0, u));
      if (i * 4 + r0 < rows && u * 8 < cols) *reinterpret_cast<uint4*>(q + (int64_t)(i * 4) * ld) = v;
    }
    return;
  }
#pragma unroll 8
  for (int r = 0; r < rows; ++r) {
    uint16_t* row = p + (int64_t)r * ld;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = h * 32 + lane;
      uint16_t v;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(staging_at(base, r, c >> 3) + (c & 7) * 2) : "memory");
      if (c < cols) row[c] = v;
    }
  }
}

// The epilogue's arithmetic: up to 64 columns of this thread's row, 16 at a time, into its row of the staging buffer. Rolled loops on
// purpose, and one activation to a copy of the code: unrolled over the columns with the choice of activation inside, the last
// tile of a launch waited 7 us for instructions instead of working 2.
template <int TYPE>
__device__ __forceinline__ void load_bias(float (&b)[2], const uint16_t* p, int cols, int lane) {
#pragma unroll
  for (int i = 0; i < 2; ++i) b[i] = i * 32 + lane < cols ? dense_to_f32<TYPE>(p[i * 32 + lane]) : 0.0f;
}
__device__ __forceinline__ void add_bias(float (&z)[16], const float (&b)[2], int block) {
  const float mine = block < 2 ? b[0] : b[1];
#pragma unroll
  for (int j = 0; j < 16; ++j) z[j] += __shfl_sync(0xFFFFFFFFu, mine, (block & 1) * 16 + j);
}
__device__ __forceinline__ void load_columns(float (&z)[16], uint32_t taddr) {
  uint32_t v[16];
  tc_ld16(taddr, v);
  tc_wait_ld();
#pragma unroll
  for (int j = 0; j < 16; ++j) z[j] = __uint_as_float(v[j]);
}
// The 64 pre-activations of this thread's row to memory in fp32, 32 at a time through the staging buffer.
__device__ __forceinline__ void preact_columns(uint32_t tz, int width, uint32_t staging, const float (&bias)[2], bool has_bias, float* p, int64_t ld,
                                               int rows, int cols, int vec, int lane) {
  const int r0 = lane >> 3, u = lane & 7;
#pragma unroll 1
  for (int part = 0; part * 32 < width; ++part) {
#pragma unroll 1
    for (int block = 0; block < 2 && part * 32 + block * 16 < width; ++block) {
      float z[16];
      load_columns(z, tz + part * 32 + block * 16);
      if (has_bias) add_bias(z, bias, part * 2 + block);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sts128(staging_at(staging, lane, block * 4 + j), make_uint4(__float_as_uint(z[j * 4]), __float_as_uint(z[j * 4 + 1]),
                                                                    __float_as_uint(z[j * 4 + 2]), __float_as_uint(z[j * 4 + 3])));
    }
    __syncwarp();
    const int left = min(32, cols - part * 32);
    float* q = p + part * 32;
    if (vec && (left & 3) == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint4 v = lds128(staging_at(staging, i * 4 + r0, u));
        if (i * 4 + r0 < rows && u * 4 < left) *reinterpret_cast<uint4*>(q + (int64_t)(i * 4 + r0) * ld + u * 4) = v;
      }
    } else {   // rows that start anywhere: a row at a time, a value a lane
#pragma unroll 8
      for (int r = 0; r < rows; ++r) {
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(staging_at(staging, r, lane >> 2) + (lane & 3) * 4) : "memory");
        if (lane < left) q[(int64_t)r * ld + lane] = v;
      }
    }
    __syncwarp();
  }
}
template <int TYPE, int ACT>
__device__ __forceinline__ void linear_columns(uint32_t tz, int width, uint32_t staging, const float (&bias)[2], bool has_bias, bool residual, int lane) {
#pragma unroll 1
  for (int block = 0; block * 16 < width; ++block) {
    float z[16];
    load_columns(z, tz + block * 16);
    if (has_bias) add_bias(z, bias, block);
    if (ACT != kActNone) {
#pragma unroll
      for (int j = 0; j < 16; ++j) z[j] = dense_act(ACT, z[j]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t at = staging_at(staging, lane, block * 2 + u);
      if (residual) {
        const uint4 q = lds128(at);
        const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = dense_unpack<TYPE>(r[j]);
          z[u * 8 + j * 2] += v.x;
          z[u * 8 + j * 2 + 1] += v.y;
        }
      }
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = dense_pack<TYPE>(z[u * 8 + j * 2], z[u * 8 + j * 2 + 1]);
      sts128(at, make_uint4(w[0], w[1], w[2], w[3]));
    }
  }
}
template <int TYPE, int ACT>
__device__ __forceinline__ void gated_columns(uint32_t tg, uint32_t tu, int width, uint32_t staging, const float (&bias_g)[2], const float (&bias_u)[2],
                                              bool has_bias, const WideParams& p, int lane) {
#pragma unroll 1
  for (int block = 0; block * 16 < width; ++block) {
    float g[16], u[16];
    load_columns(g, tg + block * 16);
    load_columns(u, tu + block * 16);
    if (has_bias) {
      add_bias(g, bias_g, block);
      add_bias(u, bias_u, block);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = h * 8 + j * 2;
        w[j] = dense_pack<TYPE>(dense_gated(ACT, g[c], u[c], p.limit, p.beta, p.linear_beta),
                                dense_gated(ACT, g[c + 1], u[c + 1], p.limit, p.beta, p.linear_beta));
      }
      sts128(staging_at(staging, lane, block * 2 + h), make_uint4(w[0], w[1], w[2], w[3]));
    }
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
  wait_for_earlier_kernels();
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
        const int n0 = GATED ? tn * (p.bn / 2) + (int)rank * p.N : tn * p.bn + (int)rank * (p.bn / 2);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          const uint32_t full = smem_u32(&bars->full[s.slot]), dst = ring + s.slot * kStageBytes;
          if (!mbar_wait(smem_u32(&bars->empty[s.slot]), s.phase ^ 1u, abort_flag, 51)) {
            go = false;
            break;
          }
          if (rank == 0) mbar_expect_tx(full, 2 * p.stage_bytes);
          if (p.a_mn) {
            tma_load_2d_pair(dst, &map_a, m0, kb * 64, full);
            tma_load_2d_pair(dst + 8192, &map_a, m0 + 64, kb * 64, full);
          } else {
            tma_load_2d_pair(dst, &map_a, kb * 64, m0, full);
          }
          if (p.b_mn) {
            tma_load_2d_pair(dst + 16384, &map_b, n0, kb * 64, full);
            if (p.bn > 128) tma_load_2d_pair(dst + 24576, &map_b, n0 + 64, kb * 64, full);
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
      const uint32_t idesc = operand_idesc<TYPE>(256, p.bn, p.a_mn, p.b_mn);
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
      const int64_t row0 = (int64_t)tm * 256 + rank * 128 + quad * 32;
      const int rows = (int)min((int64_t)32, (int64_t)p.M - row0);
      Piece ahead;   // the residual of the coming 64 columns, on its way while the MMAs run
      // the first four warps take the first half of a tile's columns (gated: features), the others the second, up to 64 at a time
      const int tile_cols = GATED ? p.bn / 2 : p.bn, mine = tile_cols / 2, col_first = tn * tile_cols + half * mine;
      if (!GATED && p.residual && p.vec_r && rows > 0 && col_first < p.N)
        piece_load(ahead, p.residual + row0 * p.ldr + col_first, p.ldr, rows, min(min(64, mine), p.N - col_first), lane);
      const bool ready = mbar_wait(smem_u32(&bars->acc_full[buf]), (it >> 1) & 1, abort_flag, 54, 32);
      if (!__all_sync(0xFFFFFFFFu, ready)) break;
      tc_fence_after();
      const uint32_t lanes = tmem_base + buf * 256 + ((uint32_t)(quad * 32) << 16);
      if constexpr (GATED) {
        // gate sums at columns half * mine of the accumulator, up sums half a tile on
        const int col0 = col_first, cols = min(mine, p.N - col0);
        const uint32_t tg = lanes + half * mine, tu = tg + tile_cols;
        const bool any = rows > 0 && cols > 0;
        const bool has_bias = p.bias != nullptr && any;
        float bias_g[2] = {}, bias_u[2] = {};
        if (has_bias) {
          load_bias<TYPE>(bias_g, p.bias + col0, cols, lane);
          load_bias<TYPE>(bias_u, p.bias + p.N + col0, cols, lane);
        }
        if (p.preact && any) {
#pragma unroll 1
          for (int part = 0; part < 2; ++part) {
            const float b[2] = {part ? bias_u[0] : bias_g[0], part ? bias_u[1] : bias_g[1]};
            preact_columns(part ? tu : tg, mine, staging, b, has_bias, p.preact + row0 * p.ldp + (part ? p.N : 0) + col0, p.ldp, rows, cols,
                           part ? p.vec_p2 : p.vec_p, lane);
          }
        }
        if (any) {
          if (p.act == 1) gated_columns<TYPE, 1>(tg, tu, mine, staging, bias_g, bias_u, has_bias, p, lane);
          else gated_columns<TYPE, 0>(tg, tu, mine, staging, bias_g, bias_u, has_bias, p, lane);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cta(smem_u32(&bars->acc_empty[buf]), 0);
        if (any) {
          staging_out(staging, p.out + row0 * p.ldo + col0, p.ldo, rows, cols, p.vec_o, lane);
          __syncwarp();
        }
      } else {
#pragma unroll 1
        for (int at = 0; at < mine; at += 64) {
          const int width = min(64, mine - at), col0 = col_first + at, cols = min(width, p.N - col0);
          const uint32_t tz = lanes + half * mine + at;
          const bool any = rows > 0 && cols > 0, last = at + 64 >= mine;
          const bool has_bias = p.bias != nullptr && any;
          float bias[2] = {};
          if (has_bias) load_bias<TYPE>(bias, p.bias + col0, cols, lane);
          if (p.preact && any) preact_columns(tz, width, staging, bias, has_bias, p.preact + row0 * p.ldp + col0, p.ldp, rows, cols, p.vec_p, lane);
          if (p.residual && any) {
            if (p.vec_r) {
              piece_to_staging(ahead, staging, p.residual + row0 * p.ldr + col0, p.ldr, rows, cols, lane);
              if (!last && col0 + 64 < p.N)
                piece_load(ahead, p.residual + row0 * p.ldr + col0 + 64, p.ldr, rows, min(min(64, mine - at - 64), p.N - col0 - 64), lane);
            } else {
              values_in(staging, p.residual + row0 * p.ldr + col0, p.ldr, rows, cols, lane);
            }
            __syncwarp();
          }
          if (any) {
            const bool res = p.residual != nullptr;
            switch (p.act) {
              case kActSilu: linear_columns<TYPE, kActSilu>(tz, width, staging, bias, has_bias, res, lane); break;
              case kActGelu: linear_columns<TYPE, kActGelu>(tz, width, staging, bias, has_bias, res, lane); break;
              case kActGeluTanh: linear_columns<TYPE, kActGeluTanh>(tz, width, staging, bias, has_bias, res, lane); break;
              default: linear_columns<TYPE, kActNone>(tz, width, staging, bias, has_bias, res, lane);
            }
          }
          if (last) tc_fence_before();
          __syncwarp();
          if (last && lane == 0) mbar_arrive_cta(smem_u32(&bars->acc_empty[buf]), 0);
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

// A tensor map of one operand: boxes of 64 values along the contiguous index by `box` (k contiguous) or 64 rows.
CUtensorMap operand_map(const DenseOperand& o, int64_t rows, int K, int box) {
  return o.mn_major ? sm100_make_map_bf16(o.p, (uint64_t)rows, (uint64_t)K, (uint64_t)o.ld * 2, 64)
                    : sm100_make_map_bf16(o.p, (uint64_t)K, (uint64_t)rows, (uint64_t)o.ld * 2, (uint32_t)box);
}

// How a launch is cut, and how long it takes by that (us): the width of a tile that makes waves x time of a wave smallest. A
// tile's time is its k blocks' (0.152 us each for 128 rows of B, 0.28 for 256, straight between; below 128 a stage is bound by
// bringing A) and what comes before and after them. Measured on 2880 -> 2880, widths 256, 192, 128 and 64: 512 tokens 20.1, 17.6,
// 13.4 and 19.1 us, 1024 tokens 22.3, 18.4, 21.2 and 27.0, 2047 tokens 35.2, 29.3, 30.4 and 43.3; with many waves the widest is
// best or within 4 % of it (8192 tokens 101.5, 97.9, 108.5, 161.1; 8192 x 7168 -> 2048 170, 175, 193, 296).
struct WidePlan {
  int bn;
  float us;
};
WidePlan plan_wide(int64_t M, int64_t N, int64_t K, bool gated) {
  const int64_t pairs = sm_count() / 2, tiles_m = (M + 255) / 256, blocks = (K + 63) / 64;
  WidePlan best{256, 1e30f};
  for (int bn = 256; bn >= 64; bn -= 32) {
    const int64_t tile_n = gated ? bn / 2 : bn, tiles = tiles_m * ((N + tile_n - 1) / tile_n);
    const float waves = (float)((tiles + pairs - 1) / pairs), narrower = (float)(256 - bn) / 64.0f;
    const float block_us = bn >= 128 ? 0.024f + 0.001f * (float)bn : 0.144f + 0.0001f * (float)bn;
    const float ends_us = bn >= 128 ? 3.4f + 0.0148f * (float)bn : 5.4f;
    // the more pairs are at work, the slower the narrower tiles, which bring more bytes for a product
    const float load = 1.0f + 0.06f * narrower * (waves > 1.0f ? 1.0f : (float)tiles / (float)pairs);
    const float us = ends_us + waves * ((float)blocks * block_us * load) + (waves - 1.0f) * 1.0f;
    if (us < best.us) best = {bn, us};
  }
  return best;
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
  p.bn = plan_wide(g.M, g.N, g.K, GATED).bn;
  p.stage_bytes = 16384 + (g.b.mn_major ? (p.bn > 128 ? 16384 : 8192) : p.bn * 64);
  const int tile_n = GATED ? p.bn / 2 : p.bn;
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
  p.vec_p = (reinterpret_cast<uintptr_t>(g.preact) & 15u) == 0 && g.ldp % 4 == 0;
  p.vec_p2 = p.vec_p && g.N % 4 == 0;
  p.status = status_address();
  const CUtensorMap a = operand_map(g.a, g.M, g.K, 128), b = operand_map(g.b, GATED ? 2 * (int64_t)g.N : g.N, g.K, p.bn / 2);
  const int units = min(p.n_tiles, sm_count() / 2);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(2 * units));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kWideSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  overlap_launch(attr[0]);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, dense_wide_kernel<TYPE, GATED>, a, b, p));
}

}  // namespace

float dense_wide_us(const DenseGemm& g) { return plan_wide(g.M, g.N, g.K, g.gated).us; }

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
