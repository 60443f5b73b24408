// dense_gemm.cu - products of the dense feed-forward operators on tcgen05: CTA pairs, tiles of 256 rows by 64 to 256 columns.
//
// out[m, n] = sum_k A[m, k] B[n, k] with either operand contiguous along k or along its own index (the backward products read
// the weight, x and the gradient as they lie: the tensor map brings 64 x 64 boxes, and the matrix descriptor says which index
// is contiguous). A pair of CTAs (cta_group::2) works on 256 rows of A and up to 256 of B: each CTA stages half of either in shared
// memory (64 k a stage, 128-byte swizzle), one thread of the leader issues the MMAs, each CTA holds its 128 result rows in
// tensor memory. Two accumulators of up to 256 columns: eight epilogue warps empty one while the other fills. Persistent, tiles
// dealt out in groups of eight row tiles by all column tiles, so that the pairs at work share their operands in L2. A gradient of few
// tiles and a long sum is cut along k: the parts' tiles follow one another like those of different products, and leave fp32 sums
// for dense_join_kernel (16384 tokens, the backward pass of 128 -> 128: 41 us whole, 17 in parts; 512 -> 512 45 and 28).
//
// In the gated form half of a tile's rows of B are gate rows (staged by the leader) and half the up rows of the same features
// (staged by its peer): an epilogue thread finds a feature's gate and up sums half a tile apart in its own lane.
//
// Bound by the tensor cores: 8192 x 7168 -> 2 x 2048 gated takes 299 to 310 us (1.61 to 1.55 PFLOP/s; the tensor pipe is active in
// 97 % of the SMs' active cycles, DRAM 21 %, L2 44 %), in a loop of seconds under the power cap 357 us (1.35 PFLOP/s).
#include <algorithm>

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

struct WideParams {           // one product
  int M, N;                   // N: columns of the result (gated: features)
  int a_mn, b_mn;
  int bn;                     // rows of B a tile: a multiple of 32 from 64 to 256
  int stage_bytes;            // of one CTA: what the copies of a stage bring
  int tiles_m, tiles_n, n_tiles, k_blocks;
  int part_tiles, part_blocks;   // of one part of k: its tiles (the parts' follow one another) and blocks
  int64_t plane;              // from one part's sums to the next's
  int act;
  GatedKind kind;
  const uint16_t* bias;
  const uint16_t* residual;
  uint16_t* out;              // null: the sums of every part to preact
  float* preact;
  int64_t ldr, ldo, ldp;
  int direct;                 // rows of result and residual start on 16 bytes
  int wide_o, wide_p;         // rows of the result, of preact start on 32
};
template <int COUNT>
struct WideLaunch {           // one product, or two that do not depend on each other: the tiles of the second follow the first's
  CUtensorMap a[COUNT], b[COUNT];
  WideParams p[COUNT];
  int n_tiles;                // of both
  DenseSums sums;             // two: column sums made by the epilogue's warps while the first products run
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
// Rows that start anywhere go through the staging buffer: rows x cols (at most 32 x 64), a row at a time, a value a lane; on the
// way in, sixteen rows are fetched before the first is put down. (A word a lane where the row allows it was slower: the row's
// parity makes three cases of every access.)
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
__device__ __forceinline__ void values_out(uint32_t base, uint16_t* p, int64_t ld, int rows, int cols, int lane) {
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

// Rows that start on 16 bytes are written from registers: a thread owns a row and takes 16 of its values at a time, 32 bytes, in
// one access where the row starts on 32 - whole sectors, although neighbouring threads are a row apart. (Through the staging
// buffer the same bytes cross shared memory twice, which the MMAs need for their operands: 8192 x 7168 -> 2 x 2048 gated 309 us
// instead of 299, the gradient of the weight of 8192 x 2048 -> 7168 193 instead of 181.)
__device__ __forceinline__ void stg32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// n (of 16) 16-bit values.
__device__ __forceinline__ void row_store(uint16_t* p, const uint32_t (&w)[8], int n, int wide) {
  if (wide && n >= 16) {
    stg32(p, w);
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (n >= h * 8 + 8) {
      *reinterpret_cast<uint4*>(p + h * 8) = make_uint4(w[h * 4], w[h * 4 + 1], w[h * 4 + 2], w[h * 4 + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (h * 8 + j < n) p[h * 8 + j] = (uint16_t)(w[h * 4 + (j >> 1)] >> ((j & 1) * 16));
    }
  }
}
// A residual on 16 bytes is fetched in whole lines, eight threads a row, 64 columns ahead of their use (a lane holds unit lane % 8
// of rows lane / 8, 4 + lane / 8, ...), and handed to the rows' owners through the staging buffer. (Each owner fetching its own 32
// bytes a block ahead: 8192 x 7168 -> 2048 173 us instead of 168.)
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
// n (of 16) fp32 values, p on 32 bytes.
__device__ __forceinline__ void row_store_f32(float* p, const float (&z)[16], int n) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (n >= h * 8 + 8) {
      stg32(p + h * 8, reinterpret_cast<const uint32_t*>(&z[h * 8]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (h * 8 + j < n) p[h * 8 + j] = z[h * 8 + j];
    }
  }
}

// The epilogue's arithmetic: columns of this thread's row, 16 at a time. Rolled loops on purpose, and one activation to a copy of
// the code: unrolled over the columns with the choice of activation inside, the last tile of a launch waited 7 us for
// instructions instead of working 2.
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
__device__ __forceinline__ void load_columns_two(float (&z)[16], uint32_t taddr, float (&y)[16], uint32_t uaddr) {
  uint32_t v[16], u[16];
  tc_ld16_two(taddr, v, uaddr, u);
  tc_wait_ld();
#pragma unroll
  for (int j = 0; j < 16; ++j) z[j] = __uint_as_float(v[j]), y[j] = __uint_as_float(u[j]);
}
// Up to 64 pre-activations of this thread's row to rows of memory that start anywhere, 32 at a time through the staging buffer.
__device__ __forceinline__ void preact_anywhere(uint32_t tz, int width, uint32_t staging, const float (&bias)[2], bool has_bias, float* p,
                                                int64_t ld, int rows, int cols, int lane) {
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
#pragma unroll 8
    for (int r = 0; r < rows; ++r) {
      float v;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(staging_at(staging, r, lane >> 2) + (lane & 3) * 4) : "memory");
      if (lane < left) p[(int64_t)r * ld + part * 32 + lane] = v;
    }
    __syncwarp();
  }
}
// Where a thread's row starts in the result and the pre-activations (null: not there, or a row behind the last), and how many of
// the columns exist.
struct RowPlace {
  uint16_t* out;
  float *preact, *preact_up;
  int cols;
};
template <int TYPE, int ACT, bool DIRECT>
__device__ __forceinline__ void linear_columns(uint32_t tz, int width, uint32_t staging, const float (&bias)[2], bool has_bias, bool residual,
                                               const RowPlace& at, const WideParams& p, int lane) {
#pragma unroll 1
  for (int block = 0; block * 16 < width; ++block) {
    const int n = at.cols - block * 16;
    float z[16];
    load_columns(z, tz + block * 16);
    if (has_bias) add_bias(z, bias, block);
    if (at.preact) row_store_f32(at.preact + block * 16, z, n);
    if (ACT != kActNone) {
#pragma unroll
      for (int j = 0; j < 16; ++j) z[j] = dense_act(ACT, z[j]);
    }
    if (residual) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 q = lds128(staging_at(staging, lane, block * 2 + u));
        const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = dense_unpack<TYPE>(r[j]);
          z[u * 8 + j * 2] += v.x;
          z[u * 8 + j * 2 + 1] += v.y;
        }
      }
    }
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = dense_pack<TYPE>(z[j * 2], z[j * 2 + 1]);
    if (DIRECT) {
      if (at.out && n > 0) row_store(at.out + block * 16, w, n, p.wide_o);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u) sts128(staging_at(staging, lane, block * 2 + u), make_uint4(w[u * 4], w[u * 4 + 1], w[u * 4 + 2], w[u * 4 + 3]));
    }
  }
}
template <int TYPE, int ACT, bool DIRECT>
__device__ __forceinline__ void gated_columns(uint32_t tg, uint32_t tu, int width, uint32_t staging, const float (&bias_g)[2], const float (&bias_u)[2],
                                              bool has_bias, const RowPlace& at, const WideParams& p, int lane) {
#pragma unroll 1
  for (int block = 0; block * 16 < width; ++block) {
    const int n = at.cols - block * 16;
    float g[16], u[16];
    load_columns_two(g, tg + block * 16, u, tu + block * 16);
    if (has_bias) {
      add_bias(g, bias_g, block);
      add_bias(u, bias_u, block);
    }
    if (at.preact) {
      row_store_f32(at.preact + block * 16, g, n);
      row_store_f32(at.preact_up + block * 16, u, n);
    }
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      w[j] = dense_pack<TYPE>(dense_gated(ACT, g[j * 2], u[j * 2], p.kind),
                              dense_gated(ACT, g[j * 2 + 1], u[j * 2 + 1], p.kind));
    if (DIRECT) {
      if (at.out && n > 0) row_store(at.out + block * 16, w, n, p.wide_o);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) sts128(staging_at(staging, lane, block * 2 + h), make_uint4(w[h * 4], w[h * 4 + 1], w[h * 4 + 2], w[h * 4 + 3]));
    }
  }
}
template <int TYPE, bool DIRECT>
__device__ __forceinline__ void linear_columns(uint32_t tz, int width, uint32_t staging, const float (&bias)[2], bool has_bias, bool residual,
                                               const RowPlace& at, const WideParams& p, int lane) {
  switch (p.act) {
    case kActSilu: linear_columns<TYPE, kActSilu, DIRECT>(tz, width, staging, bias, has_bias, residual, at, p, lane); break;
    case kActGelu: linear_columns<TYPE, kActGelu, DIRECT>(tz, width, staging, bias, has_bias, residual, at, p, lane); break;
    case kActGeluTanh: linear_columns<TYPE, kActGeluTanh, DIRECT>(tz, width, staging, bias, has_bias, residual, at, p, lane); break;
    default: linear_columns<TYPE, kActNone, DIRECT>(tz, width, staging, bias, has_bias, residual, at, p, lane);
  }
}

template <int TYPE, bool GATED, int COUNT>
__global__ void __cluster_dims__(2) __launch_bounds__(kThreads, 1)
dense_wide_kernel(const __grid_constant__ WideLaunch<COUNT> work) {
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
  // A pair's tile in round `it`. Of two products the rounds behind the one in which the second begins are dealt out from the other
  // end: what is left for the last goes first to pairs that had no long tile in that one (1001 tokens, 1504 -> 2 x 1027: 23.9 us
  // for the backward pass with all rounds in one order, 19.8 so; 4096 tokens, 1024 -> 1024 20.1 and 16.2).
  const int turn = COUNT > 1 ? work.p[0].n_tiles / n_units : 0;
  const auto tile_of = [&](int it) { return it * n_units + (COUNT > 1 && it > turn ? n_units - 1 - unit : unit); };
  // which product tile t belongs to, and where and of which part of k it lies there
  const auto place = [&](int t, int& tm, int& tn, int& part) {
    const int which = COUNT > 1 && t >= work.p[0].n_tiles;
    const WideParams& p = work.p[which];
    if (which) t -= work.p[0].n_tiles;
    part = 0;
    if (!GATED && t >= p.part_tiles) {
      part = t / p.part_tiles;
      t -= part * p.part_tiles;
    }
    const int per_group = kGroupM * p.tiles_n, first = t / per_group * kGroupM, in = t % per_group, high = min(kGroupM, p.tiles_m - first);
    tm = first + in % high;
    tn = in / high;
    return which;
  };

  if (warp == kEpiWarps) {
    // ------------------------------ producer --------------------------------
    if (elect_one()) {
      Ring s;
      long long issued = 0;
      bool go = true;
      for (int it = 0, t; (t = tile_of(it)) < work.n_tiles && go; ++it) {
        int tm, tn, part;
        const int which = place(t, tm, tn, part);
        const WideParams& p = work.p[which];
        const int kb0 = part * p.part_blocks, kb1 = min(kb0 + p.part_blocks, p.k_blocks);
        const CUtensorMap *map_a = &work.a[which], *map_b = &work.b[which];
        // kept in registers: of two products, each look into the parameters would be an indexed load
        const int a_mn = p.a_mn, b_mn = p.b_mn, b_wide = p.bn > 128, pair_bytes = 2 * p.stage_bytes;
        const int m0 = tm * 256 + (int)rank * 128;
        const int n0 = GATED ? tn * (p.bn / 2) + (int)rank * p.N : tn * p.bn + (int)rank * (p.bn / 2);
        for (int kb = kb0; kb < kb1; ++kb) {
          const uint32_t full = smem_u32(&bars->full[s.slot]), dst = ring + s.slot * kStageBytes;
          if (!mbar_wait(smem_u32(&bars->empty[s.slot]), s.phase ^ 1u, abort_flag, 51)) {
            go = false;
            break;
          }
          if (rank == 0) mbar_expect_tx(full, pair_bytes);
          if (a_mn) {
            tma_load_2d_pair(dst, map_a, m0, kb * 64, full);
            tma_load_2d_pair(dst + 8192, map_a, m0 + 64, kb * 64, full);
          } else {
            tma_load_2d_pair(dst, map_a, kb * 64, m0, full);
          }
          if (b_mn) {
            tma_load_2d_pair(dst + 16384, map_b, n0, kb * 64, full);
            if (b_wide) tma_load_2d_pair(dst + 24576, map_b, n0 + 64, kb * 64, full);
          } else {
            tma_load_2d_pair(dst + 16384, map_b, kb * 64, n0, full);
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
      Ring s;
      bool go = true;
      for (int it = 0, t; (t = tile_of(it)) < work.n_tiles && go; ++it) {
        int tm, tn, part;
        const WideParams& p = work.p[place(t, tm, tn, part)];
        const int kb0 = part * p.part_blocks, kb1 = min(kb0 + p.part_blocks, p.k_blocks);
        const int a_mn = p.a_mn, b_mn = p.b_mn;
        const uint32_t idesc = operand_idesc<TYPE>(256, p.bn, a_mn, b_mn);
        const uint32_t a_step = a_mn ? 2048 >> 4 : 32 >> 4, b_step = b_mn ? 2048 >> 4 : 32 >> 4;   // 16 k on
        const int buf = it & 1;
        if (!mbar_wait(smem_u32(&bars->acc_empty[buf]), ((it >> 1) & 1) ^ 1, abort_flag, 52)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + buf * 256;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(smem_u32(&bars->full[s.slot]), s.phase, abort_flag, 53)) {
            go = false;
            break;
          }
          tc_fence_after();
          const uint32_t src = ring + s.slot * kStageBytes;
          const uint64_t ad = operand_desc(src, a_mn), bd = operand_desc(src + 16384, b_mn);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_ss_pair(d, ad + k * a_step, bd + k * b_step, idesc, ((kb - kb0) | k) != 0);
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
    if constexpr (COUNT > 1) {   // (a launch of its own: 517 tokens, 1024 -> 768, 12.2 us for all gradients instead of 9.1)
      if (work.sums.db) sum_chunks<TYPE>(work.sums, blockIdx.x, gridDim.x, warp, lane, reinterpret_cast<float(*)[32]>(smem + kStages * kStageBytes));
    }
    for (int it = 0, t; (t = tile_of(it)) < work.n_tiles; ++it) {
      int tm, tn, part;
      const WideParams& p = work.p[place(t, tm, tn, part)];
      const int buf = it & 1;
      const int64_t row0 = (int64_t)tm * 256 + rank * 128 + quad * 32;
      const int rows = (int)min((int64_t)32, (int64_t)p.M - row0);
      // the first four warps take the first half of a tile's columns (gated: features), the others the second, up to 64 at a time
      const int tile_cols = GATED ? p.bn / 2 : p.bn, mine = tile_cols / 2, col_first = tn * tile_cols + half * mine;
      const int64_t row = row0 + lane;
      const bool row_ok = lane < rows;
      Piece ahead;   // the residual of the coming columns, on its way while the MMAs run
      if (!GATED && p.residual && p.direct && rows > 0 && col_first < p.N)
        piece_load(ahead, p.residual + row0 * p.ldr + col_first, p.ldr, rows, min(min(64, mine), p.N - col_first), lane);
      if (!GATED && p.residual && !p.direct && row_ok)   // rows that start anywhere are fetched later, out of the L2
        for (int c = 0; c < min(mine, p.N - col_first); c += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.residual + row * p.ldr + col_first + c));
      const bool ready = mbar_wait(smem_u32(&bars->acc_full[buf]), (it >> 1) & 1, abort_flag, 54, 32);
      if (!__all_sync(0xFFFFFFFFu, ready)) break;
      tc_fence_after();
      const uint32_t lanes = tmem_base + buf * 256 + ((uint32_t)(quad * 32) << 16);
#pragma unroll 1
      for (int first = 0; first < mine; first += 64) {
        const int width = min(64, mine - first), col0 = col_first + first, cols = min(width, p.N - col0);
        const bool any = rows > 0 && cols > 0, last = first + 64 >= mine, has_bias = p.bias != nullptr && any;
        const uint32_t tz = lanes + half * mine + first, tu = tz + tile_cols;   // gated: gate sums, up sums half a tile on
        float bias[2] = {}, bias_u[2] = {};
        if (has_bias) {
          load_bias<TYPE>(bias, p.bias + col0, cols, lane);
          if (GATED) load_bias<TYPE>(bias_u, p.bias + p.N + col0, cols, lane);
        }
        if (any) {
          RowPlace at{};
          at.cols = cols;
          if (row_ok && p.out) at.out = p.out + row * p.ldo + col0;
          float* const sums = p.preact + (GATED ? 0 : part * p.plane);
          if (row_ok && p.preact && p.wide_p) {
            at.preact = sums + row * p.ldp + col0;
            at.preact_up = at.preact + p.N;
          }
          if (p.preact && !p.wide_p) {
            preact_anywhere(tz, width, staging, bias, has_bias, sums + row0 * p.ldp + col0, p.ldp, rows, cols, lane);
            if (GATED) preact_anywhere(tu, width, staging, bias_u, has_bias, sums + row0 * p.ldp + p.N + col0, p.ldp, rows, cols, lane);
          }
          if (p.direct) {
            if constexpr (GATED) {
              if (p.kind.act == 1) gated_columns<TYPE, 1, true>(tz, tu, width, staging, bias, bias_u, has_bias, at, p, lane);
              else gated_columns<TYPE, 0, true>(tz, tu, width, staging, bias, bias_u, has_bias, at, p, lane);
            } else {
              if (p.residual) {
                piece_to_staging(ahead, staging, p.residual + row0 * p.ldr + col0, p.ldr, rows, cols, lane);
                if (!last && col0 + 64 < p.N)
                  piece_load(ahead, p.residual + row0 * p.ldr + col0 + 64, p.ldr, rows, min(min(64, mine - first - 64), p.N - col0 - 64), lane);
                __syncwarp();
              }
              linear_columns<TYPE, true>(tz, width, staging, bias, has_bias, p.residual != nullptr, at, p, lane);
            }
          } else {
            if (!GATED && p.residual) {
              values_in(staging, p.residual + row0 * p.ldr + col0, p.ldr, rows, cols, lane);
              __syncwarp();
            }
            if constexpr (GATED) {
              if (p.kind.act == 1) gated_columns<TYPE, 1, false>(tz, tu, width, staging, bias, bias_u, has_bias, at, p, lane);
              else gated_columns<TYPE, 0, false>(tz, tu, width, staging, bias, bias_u, has_bias, at, p, lane);
            } else {
              linear_columns<TYPE, false>(tz, width, staging, bias, has_bias, p.residual != nullptr, at, p, lane);
            }
            __syncwarp();
            values_out(staging, p.out + row0 * p.ldo + col0, p.ldo, rows, cols, lane);
          }
        }
        if (last) tc_fence_before();
        __syncwarp();
        if (last && lane == 0) mbar_arrive_cta(smem_u32(&bars->acc_empty[buf]), 0);
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
  if (tid == 0 && bars->abort_flag != 0) atomicExch(work.status, 100 + bars->abort_flag);
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
//
// Two products in one launch (the gradients of x and of the weight): a pair's share is worked out for both together, tiles dealt
// out one after the other.
struct WidePlan {
  int bn[2];
  float us;
};
// Tiles of a product whose k is cut are as wide as it is, up to 256.
int split_width(int N) { return N >= 256 ? 256 : std::max(64, (N + 31) / 32 * 32); }
constexpr int kWidths = 7;                             // 256, 224, .. 64
constexpr int width(int i) { return 256 - 32 * i; }
struct WideCost {
  int whole[kWidths], rest[kWidths];                   // tiles: full rounds of all pairs, and the last one
  float tile_us[kWidths], load_us[kWidths];            // time of a tile, and what is added to it with all pairs at work
};
WideCost cost_of(const DenseGemm& g, int pairs) {
  WideCost c;
  const float blocks = (float)(((g.K + 63) / 64 + g.split - 1) / g.split);
  const int tiles_m = (int)(((int64_t)g.M + 255) / 256);
  for (int i = 0; i < kWidths; ++i) {
    const int bn = g.split > 1 ? split_width(g.N) : width(i), tile_n = g.gated ? bn / 2 : bn;
    const int64_t tiles = (int64_t)tiles_m * ((g.N + tile_n - 1) / tile_n) * g.split;
    c.whole[i] = (int)std::min<int64_t>(tiles / pairs, 1 << 24);
    c.rest[i] = (int)(tiles % pairs);
    const float block_us = bn >= 128 ? 0.024f + 0.001f * (float)bn : 0.144f + 0.0001f * (float)bn;
    // B contiguous along its own index comes in boxes of 64 columns a CTA, some of them for nothing; where rows do not start on 128
    // bytes, each row of a box is two lines (5000 tokens, the gradient of a 608 x 304 weight: 0.186 us a block at 128 rows)
    const float us = blocks * block_us * (g.b.mn_major && bn % 128 != 0 ? 1.05f : 1.0f) *
                     (g.a.mn_major && g.a.ld % 64 != 0 ? 1.1f : 1.0f) * (g.a.mn_major && g.b.ld % 64 != 0 ? 1.1f : 1.0f);
    c.tile_us[i] = us + 1.0f;
    c.load_us[i] = us * 0.06f * (float)(256 - bn) / 64.0f;   // narrower tiles bring more bytes for a product
  }
  return c;
}
WidePlan plan_wide(const DenseGemm* g, int count) {
  const int pairs = sm_count() / 2;
  const WideCost first = cost_of(g[0], pairs), second = count > 1 ? cost_of(g[1], pairs) : WideCost{};
  WidePlan best{{256, 256}, 1e30f};
  for (int i = 0; i < kWidths; ++i)
    for (int j = 0; j < (count > 1 ? kWidths : 1); ++j) {
      const int q0 = first.whole[i], r0 = first.rest[i], q1 = count > 1 ? second.whole[j] : 0, r1 = count > 1 ? second.rest[j] : 0;
      const float full = (float)(q0 + q1) + (float)(r0 + r1) / (float)pairs, load = full < 1.0f ? full : 1.0f;
      const float c0 = first.tile_us[i] + load * first.load_us[i];
      const float c1 = count > 1 ? second.tile_us[j] + load * second.load_us[j] : 0.0f;
      // the busiest pair: of the r0 with a tile more of the first, or of the others, which have one of the second instead; then whole
      // rounds of the second and a rest, the others' first
      float most;
      if (count == 1 || r0 == 0) {
        most = (float)(r0 > 0 ? q0 + 1 : q0) * c0 + (float)(r1 > 0 ? q1 + 1 : q1) * c1;
      } else {
        const int over = q1 * pairs + r1 - (pairs - r0), rounds = std::max(over, 0) / pairs, rest = std::max(over, 0) % pairs;
        most = std::max((float)(q0 + 1) * c0 + (float)(rounds + (rest > pairs - r0)) * c1, (float)q0 * c0 + (float)(rounds + 1 + (rest > 0)) * c1);
      }
      // of many waves, half of what idle pairs leave undone in the last comes back as clock and bandwidth for the others (of two
      // products, whose tiles take different times, a fifth: 18 sizes by 36 pairs of widths, picked within 2 % of the best on
      // average, 8 % at worst)
      const float mean = ((float)q0 + (float)r0 / (float)pairs) * c0 + ((float)q1 + (float)r1 / (float)pairs) * c1;
      const int bn0 = g[0].split > 1 ? split_width(g[0].N) : width(i), bn1 = count == 1 ? 0 : g[1].split > 1 ? split_width(g[1].N) : width(j);
      const float ends = std::max(bn0, bn1) >= 128 ? 2.4f + 0.0148f * (float)std::max(bn0, bn1) : 4.4f, back = count > 1 ? 0.2f : 0.5f;
      const float us = ends + (full > 1.0f ? most - back * (most - mean) : most);
      if (us < best.us) best = {{bn0, bn1}, us};
    }
  return best;
}

template <bool GATED>
void describe(const DenseGemm& g, int bn, WideParams& p, CUtensorMap& a, CUtensorMap& b) {
  p.M = g.M;
  p.N = g.N;
  p.a_mn = g.a.mn_major;
  p.b_mn = g.b.mn_major;
  p.bn = bn;
  p.stage_bytes = 16384 + (g.b.mn_major ? (p.bn > 128 ? 16384 : 8192) : p.bn * 64);
  const int tile_n = GATED ? p.bn / 2 : p.bn;
  p.tiles_m = (g.M + 255) / 256;
  p.tiles_n = (g.N + tile_n - 1) / tile_n;
  expects((int64_t)p.tiles_m * p.tiles_n < (1ll << 29), "dense product: more than 2^29 tiles");
  expects(g.split == 1 || (!GATED && !g.bias && !g.residual && !g.preact && g.act == kActNone && g.parts), "dense product: only plain products are cut along k");
  p.part_tiles = p.tiles_m * p.tiles_n;
  p.n_tiles = p.part_tiles * g.split;
  p.k_blocks = (g.K + 63) / 64;
  p.part_blocks = (p.k_blocks + g.split - 1) / g.split;
  p.act = g.act;
  p.kind = g.kind;
  p.bias = g.bias;
  p.residual = g.residual;
  p.out = g.split > 1 ? nullptr : g.out;
  p.preact = g.split > 1 ? g.parts : g.preact;
  p.ldr = g.ldr;
  p.ldo = g.ldo;
  p.ldp = g.split > 1 ? dense_part_pitch(g.N) : g.ldp;
  p.plane = (int64_t)g.M * p.ldp;
  const auto on = [](const void* q, int64_t ld_bytes, int bytes) { return ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)ld_bytes) & (uintptr_t)(bytes - 1)) == 0; };
  p.direct = (g.split > 1 || on(g.out, g.ldo * 2, 16)) && (g.residual == nullptr || on(g.residual, g.ldr * 2, 16));
  p.wide_p = on(p.preact, p.ldp * 4, 32) && (!GATED || g.N % 8 == 0);
  const bool whole = (GATED ? p.bn / 4 : p.bn / 2) % 16 == 0;   // every warp's columns start on 32 bytes of a row that does
  p.wide_o = whole && on(g.out, g.ldo * 2, 32);
  a = operand_map(g.a, g.M, g.K, 128);
  b = operand_map(g.b, GATED ? 2 * (int64_t)g.N : g.N, g.K, p.bn / 2);
}

// What the parts of a cut sum cost more: a launch, and their way through the L2.
float join_us(const DenseGemm& g) { return g.split > 1 ? 2.0f + 4e-7f * (float)dense_parts_bytes(g.M, g.N, g.split) : 0.0f; }

template <int TYPE, bool GATED, int COUNT>
void launch_wide(const DenseGemm* g, cudaStream_t stream, const DenseSums& sums = {}) {
  static std::atomic<bool> configured[64];
  int dev = 0;
  VK_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev].load()) {
    VK_CUDA_CHECK(cudaFuncSetAttribute(dense_wide_kernel<TYPE, GATED, COUNT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWideSmem));
    if (dev >= 0 && dev < 64) configured[dev].store(true);
  }
  const WidePlan plan = plan_wide(g, COUNT);
  WideLaunch<COUNT> work{};
  for (int i = 0; i < COUNT; ++i) {
    describe<GATED>(g[i], plan.bn[i], work.p[i], work.a[i], work.b[i]);
    work.n_tiles += work.p[i].n_tiles;
  }
  work.sums = sums;
  work.status = status_address();
  const int units = std::min(work.n_tiles, sm_count() / 2);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(2 * units));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kWideSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  overlap_launch(attr[0]);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, dense_wide_kernel<TYPE, GATED, COUNT>, work));
}

}  // namespace

float dense_wide_us(const DenseGemm& g) { return plan_wide(&g, 1).us + join_us(g); }

void launch_dense_wide(const DenseGemm& g, cudaStream_t stream) {
  if (g.type == kDenseBf16) {
    if (g.gated) launch_wide<kDenseBf16, true, 1>(&g, stream);
    else launch_wide<kDenseBf16, false, 1>(&g, stream);
  } else {
    if (g.gated) launch_wide<kDenseFp16, true, 1>(&g, stream);
    else launch_wide<kDenseFp16, false, 1>(&g, stream);
  }
  if (g.split > 1) launch_dense_join(g, stream);
}

// As many parts as there are pairs for, of at least eight blocks of k each, where that saves a tile 32 blocks or more (9 us, of which
// the join takes back 3 to 6). The pairs are those of a B200's 148 SMs, written down because the workspace's size is asked for without a
// device; where a device has fewer, the parts are the same and take more rounds.
int dense_split(int M, int N, int K) {
  constexpr int kPairs = 74;
  const int bn = split_width(N), blocks = (K + 63) / 64;
  const int64_t tiles = ((int64_t)M + 255) / 256 * (((int64_t)N + bn - 1) / bn);
  if (tiles * 2 > kPairs) return 1;
  const int most = std::max(std::min((int)(kPairs / tiles), blocks / 8), 1), each = (blocks + most - 1) / most;
  return blocks - each >= 32 ? (blocks + each - 1) / each : 1;   // (no part is empty)
}

// Two linear products that do not depend on each other, in one launch, with the column sums that were left in chunks; the product with
// the longer tiles goes first. Either is cut only
// where the other does not fill the pairs as well (8192 tokens of 256 features, gated, 4096 wide: two products of 32 tiles take
// 136 us as they are, 156 cut in halves).
void launch_dense_wide_two(const DenseGemm& g, const DenseGemm& h, const DenseSums& sums, cudaStream_t stream) {
  DenseGemm best[2];
  float best_us = 1e30f;
  for (int cut = 3; cut >= 0; --cut) {
    if (((cut & 1) && g.split == 1) || ((cut & 2) && h.split == 1)) continue;
    DenseGemm two[2] = {g, h};
    if (!(cut & 1)) two[0].split = 1;
    if (!(cut & 2)) two[1].split = 1;
    if (two[0].K / two[0].split < two[1].K / two[1].split) std::swap(two[0], two[1]);
    const float us = g.split == 1 && h.split == 1 ? 0.0f : plan_wide(two, 2).us + join_us(two[0]) + join_us(two[1]);
    if (us < best_us) {
      best_us = us;
      best[0] = two[0], best[1] = two[1];
    }
  }
  if (g.type == kDenseBf16) launch_wide<kDenseBf16, false, 2>(best, stream, sums);
  else launch_wide<kDenseFp16, false, 2>(best, stream, sums);
  for (const DenseGemm& b : best)
    if (b.split > 1) launch_dense_join(b, stream);
}

}  // namespace vkernels::kernels::cuda
