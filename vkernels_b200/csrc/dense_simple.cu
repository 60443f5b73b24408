// dense_simple.cu - dense feed-forward operators: the cross-check product on CUDA cores and the element-wise kernels of the
// backward pass.
#include <algorithm>

#include "dense.hpp"
#include "dense_math.cuh"
#include "dense_launch.cuh"

namespace vkernels::kernels::cuda {

namespace {

__device__ __forceinline__ uint16_t operand_at(const DenseOperand& o, int i, int k) {
  return o.mn_major ? o.p[(int64_t)k * o.ld + i] : o.p[(int64_t)i * o.ld + k];
}

constexpr int kTile = 64, kStep = 16;

// One CTA per 64 x 64 tile of the result (64 x 32 gated: 32 gate rows and their 32 up rows), 16 x 16 threads with 4 x 4 sums
// each, products added in ascending k in fp32 (fused multiply-add). The cross-check of the tensor-core kernels, selected only
// explicitly: any pitch, order and alignment, about 20 TFLOP/s.
template <int TYPE, bool GATED>
__global__ void __launch_bounds__(256) dense_simt_kernel(DenseGemm g) {
  __shared__ float sa[kStep][kTile + 4], sb[kStep][kTile + 4];
  constexpr int kCols = GATED ? kTile / 2 : kTile;
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kCols;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < g.K; k0 += kStep) {
#pragma unroll
    for (int i = 0; i < kTile * kStep / 256; ++i) {
      const int e = threadIdx.x + i * 256;
      const int k = e % kStep, r = e / kStep;
      const int m = m0 + r;
      // gated: rows 0..31 of the tile are gate rows, 32..63 the up rows of the same features
      const int f = n0 + (GATED ? r % kCols : r);
      const int brow = GATED && r >= kCols ? g.N + f : f;
      sa[k][r] = m < g.M && k0 + k < g.K ? dense_to_f32<TYPE>(operand_at(g.a, m, k0 + k)) : 0.0f;
      sb[k][r] = f < g.N && k0 + k < g.K ? dense_to_f32<TYPE>(operand_at(g.b, brow, k0 + k)) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k) {
      float av[4], bv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) av[i] = sa[k][ty * 4 + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) bv[j] = sb[k][GATED ? tx * 2 + (j & 1) + (j >> 1) * kCols : tx * 4 + j];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty * 4 + i;
    if (m >= g.M) continue;
    if constexpr (GATED) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + tx * 2 + j;
        if (n >= g.N) continue;
        float zg = acc[i][j], zu = acc[i][j + 2];
        if (g.bias) {
          zg += dense_to_f32<TYPE>(g.bias[n]);
          zu += dense_to_f32<TYPE>(g.bias[g.N + n]);
        }
        if (g.preact) {
          g.preact[(int64_t)m * g.ldp + n] = zg;
          g.preact[(int64_t)m * g.ldp + g.N + n] = zu;
        }
        g.out[(int64_t)m * g.ldo + n] = dense_from_f32<TYPE>(dense_gated(g.kind.act, zg, zu, g.kind));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx * 4 + j;
        if (n >= g.N) continue;
        float z = acc[i][j] + (g.bias ? dense_to_f32<TYPE>(g.bias[n]) : 0.0f);
        if (g.preact) g.preact[(int64_t)m * g.ldp + n] = z;
        z = dense_act(g.act, z);
        if (g.residual) z += dense_to_f32<TYPE>(g.residual[(int64_t)m * g.ldr + n]);
        g.out[(int64_t)m * g.ldo + n] = dense_from_f32<TYPE>(z);
      }
    }
  }
}

// Eight neighbouring values of a row.
struct Eight {
  uint16_t v[8];
};
// Eight values from an address that is a multiple of 2: from the words around them where the row goes on behind them.
__device__ __forceinline__ Eight load_eight_words(const uint16_t* p, int n) {
  Eight e;
  if (n <= 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) e.v[j] = j < n ? p[j] : (uint16_t)0;
    return e;
  }
  const uint32_t* w = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3);
  const bool odd = (reinterpret_cast<uintptr_t>(p) & 2u) != 0;
  uint32_t v[5];
#pragma unroll
  for (int j = 1; j < 4; ++j) v[j] = w[j];
  v[0] = odd ? (uint32_t)p[0] << 16 : w[0];
  v[4] = odd ? w[4] : 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) reinterpret_cast<uint32_t*>(e.v)[j] = odd ? __funnelshift_r(v[j], v[j + 1], 16) : v[j];
  return e;
}
constexpr int copy_units(int cols) { return (cols + 15) / 16 * 2; }
// Copies of rows, as the `part`-th of `parts` CTAs of 256 threads: dst[r, c] = src[r, c], rows of dst on 32 bytes, filled up to whole
// pairs of units of 8.
__device__ __forceinline__ void copy_rows(const RowCopies& c, int part, int parts) {
  const int units = copy_units(c.cols);
  const int64_t first = c.dst[0] != nullptr ? (int64_t)c.rows[0] * units : 0;
  const int64_t all = first + (c.dst[1] != nullptr ? (int64_t)c.rows[1] * units : 0), step = (int64_t)parts * 256;
#pragma unroll 2
  for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < all; i += step) {
    const int z = i >= first;
    const int64_t at = z ? i - first : i;
    const int r = all < (1ll << 31) ? (int)((uint32_t)at / (uint32_t)units) : (int)(at / units), u = (int)(at - (int64_t)r * units);
    const Eight e = load_eight_words(c.src[z] + r * c.lds[z] + u * 8, c.cols - u * 8);
    *reinterpret_cast<uint4*>(c.dst[z] + at * 8) = *reinterpret_cast<const uint4*>(e.v);
  }
}
__global__ void __launch_bounds__(256) dense_copy_rows_kernel(RowCopies c) {
  wait_for_earlier_kernels();
  copy_rows(c, blockIdx.x, gridDim.x);
}

constexpr int kGradCols = 256, kGradThreads = 256;   // 64 threads across the columns, four each; four rows at a time
constexpr int kGradRows = 4, kGradStep = 4 * kGradRows;   // rows a thread has on their way, rows a CTA takes at once

// dz = dy * act'(z) and the column sums of a chunk of rows, in one pass: one CTA per 256 columns of dy and chunk. A column's
// sum is added by one thread per fourth row in fp32, the fourths in order, the chunks by sum_chunks: no atomics, the same
// result every time. The sums are of the unrounded gradients. Bound by memory (dy and z in, dz out), as long as enough of it is
// on its way: four rows a thread before the first is worked on, the whole launch resident at once (4096 x 2880 gated: eight
// columns a thread, one row at a time and three times as many CTAs took 41 us). VEC: a thread's four columns are neighbours, in
// whole accesses; else 64 apart, so that a warp still reads whole lines of rows that start anywhere.
// What is differentiated: the linear activations (DenseAct), then the gated ones. One to a kernel: with the choice inside, every
// element's code holds them all (4096 x 2880 gelu: 20 us).
enum GradForm { kGradSwiGlu = 4, kGradSiTu = 5 };
template <int TYPE, int FORM, bool VEC>
__global__ void __launch_bounds__(kGradThreads, 3) dense_grad_kernel(DenseGrad g, int rows_per_chunk, int chunks) {
  constexpr bool GATED = FORM >= kGradSwiGlu, BENT = FORM != kActNone;
  __shared__ float sums[GATED ? 2 : 1][4][kGradCols];
  wait_for_earlier_kernels();
  if ((int)blockIdx.y >= chunks) {   // operands of the products to rows on 32 bytes, on the way
    copy_rows(g.copies, (blockIdx.y - chunks) * gridDim.x + blockIdx.x, (gridDim.y - chunks) * gridDim.x);
    return;
  }
  const int across = threadIdx.x & 63, sub = threadIdx.x >> 6, first = blockIdx.x * kGradCols;
  const int r_end = min(g.T, (int)(blockIdx.y + 1) * rows_per_chunk);
  const auto column = [&](int j) { return VEC ? across * 4 + j : across + j * 64; };
  const int c0 = first + column(0);
  float sg[4] = {}, su[4] = {};
  if (c0 < g.N) {
    for (int r0 = blockIdx.y * rows_per_chunk + sub; r0 < r_end; r0 += kGradStep) {
      uint2 dy[kGradRows];
      float zg[kGradRows][4] = {}, zu[kGradRows][4] = {};
#pragma unroll
      for (int i = 0; i < kGradRows; ++i) {
        const int64_t r = r0 + i * 4;
        dy[i] = make_uint2(0, 0);
        if (r >= r_end) continue;
        const uint16_t* py = g.dy + r * g.lddy + c0;
        const float* pz = g.preact + r * g.ldp + c0;
        if constexpr (VEC) {
          dy[i] = *reinterpret_cast<const uint2*>(py);
          if (BENT) *reinterpret_cast<float4*>(zg[i]) = *reinterpret_cast<const float4*>(pz);
          if constexpr (GATED) *reinterpret_cast<float4*>(zu[i]) = *reinterpret_cast<const float4*>(pz + g.N);
        } else {
          uint16_t v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool in = c0 + j * 64 < g.N;
            v[j] = in ? py[j * 64] : (uint16_t)0;
            if (BENT) zg[i][j] = in ? pz[j * 64] : 0.0f;
            if constexpr (GATED) zu[i][j] = in ? pz[g.N + j * 64] : 0.0f;
          }
          dy[i] = make_uint2(v[0] | ((uint32_t)v[1] << 16), v[2] | ((uint32_t)v[3] << 16));
        }
      }
#pragma unroll
      for (int i = 0; i < kGradRows; ++i) {
        const int64_t r = r0 + i * 4;
        if (r >= r_end) break;
        const float2 lo = dense_unpack<TYPE>(dy[i].x), hi = dense_unpack<TYPE>(dy[i].y);
        float d[4] = {lo.x, lo.y, hi.x, hi.y}, du[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (GATED) {
            dense_gated_grad(FORM - kGradSwiGlu, d[j], zg[i][j], zu[i][j], g.kind, d[j], du[j]);
            su[j] += du[j];
          } else {
            if (BENT) d[j] *= dense_act_slope(FORM, zg[i][j]);
          }
          sg[j] += d[j];
        }
        if (g.dz) {
          uint16_t* pd = g.dz + r * g.ldz + c0;
          if constexpr (VEC) {
            *reinterpret_cast<uint2*>(pd) = make_uint2(dense_pack<TYPE>(d[0], d[1]), dense_pack<TYPE>(d[2], d[3]));
            if constexpr (GATED) *reinterpret_cast<uint2*>(pd + g.N) = make_uint2(dense_pack<TYPE>(du[0], du[1]), dense_pack<TYPE>(du[2], du[3]));
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c0 + j * 64 < g.N) {
                pd[j * 64] = dense_from_f32<TYPE>(d[j]);
                if constexpr (GATED) pd[g.N + j * 64] = dense_from_f32<TYPE>(du[j]);
              }
          }
        }
      }
    }
  }
  if (g.partial == nullptr && g.db == nullptr) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sums[0][sub][column(j)] = sg[j];
    if constexpr (GATED) sums[GATED ? 1 : 0][sub][column(j)] = su[j];
  }
  __syncthreads();
  const int col = first + threadIdx.x;
  if (col >= g.N) return;
  const int rows = GATED ? 2 * g.N : g.N;
#pragma unroll
  for (int h = 0; h < (GATED ? 2 : 1); ++h) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += sums[h][i][threadIdx.x];
    if (g.db) g.db[h * g.N + col] = dense_from_f32<TYPE>(s);
    else g.partial[(int64_t)blockIdx.y * rows + h * g.N + col] = s;
  }
}

// The result of a product whose k was cut: the parts' sums, in order, four columns a thread, eight parts on their way at a time. The
// parts come out of the L2 as a rule (a cut product is a small one: at most 74 tiles of parts, 19 MB).
template <int TYPE>
__global__ void __launch_bounds__(256) dense_join_kernel(DenseGemm g, int64_t pitch) {
  wait_for_earlier_kernels();
  const int64_t plane = g.M * pitch;
  const int across = (int)(pitch / 4);
  const bool vec = ((reinterpret_cast<uintptr_t>(g.out) & 7u) | (g.ldo & 3)) == 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)g.M * across; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / across;
    const int n = (int)(i - m * across) * 4, left = g.N - n;
    if (left <= 0) continue;
    const float* p = g.parts + m * pitch + n;
    float z[4] = {};
    for (int s = 0; s < g.split; s += 8) {
      float4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = s + j < g.split ? *reinterpret_cast<const float4*>(p + (s + j) * plane) : make_float4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) z[0] += v[j].x, z[1] += v[j].y, z[2] += v[j].z, z[3] += v[j].w;
    }
    uint16_t* q = g.out + m * g.ldo + n;
    if (vec && left >= 4) {
      *reinterpret_cast<uint2*>(q) = make_uint2(dense_pack<TYPE>(z[0], z[1]), dense_pack<TYPE>(z[2], z[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) q[j] = dense_from_f32<TYPE>(z[j]);
    }
  }
}

// Column sums of the chunks where no launch of products follows that takes them along.
template <int TYPE>
__global__ void __launch_bounds__(256) dense_sum_kernel(DenseSums q) {
  __shared__ float room[8][32];
  wait_for_earlier_kernels();
  sum_chunks<TYPE>(q, blockIdx.x, gridDim.x, threadIdx.x >> 5, threadIdx.x & 31, room);
}

template <class... P, class... A>
void launch_overlapped(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  overlap_launch(attr[0]);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
}

// CTAs for copies: two units of eight values a thread, eight CTAs an SM (of a B200's 148) at most.
int copy_ctas(const RowCopies& c) {
  int64_t units = 0;
  for (int i = 0; i < 2; ++i)
    if (c.dst[i] != nullptr) units += (int64_t)c.rows[i] * copy_units(c.cols);
  return (int)std::min<int64_t>((units + 511) / 512, 8 * 148);
}

template <int TYPE, int FORM>
void grad_of_form(const DenseGrad& g, int chunks, cudaStream_t stream) {
  const auto aligned = [](const void* p, int bytes, int64_t ld) { return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0 && ld % 4 == 0); };
  const bool vec = g.N % 4 == 0 && aligned(g.dy, 8, g.lddy) && aligned(g.preact, 16, g.ldp) && aligned(g.dz, 8, g.ldz);
  const int across = (g.N + kGradCols - 1) / kGradCols;
  const dim3 grid(across, chunks + (copy_ctas(g.copies) + across - 1) / across);
  const int rows = (g.T + chunks - 1) / chunks;
  if (vec) launch_overlapped(dense_grad_kernel<TYPE, FORM, true>, grid, kGradThreads, stream, g, rows, chunks);
  else launch_overlapped(dense_grad_kernel<TYPE, FORM, false>, grid, kGradThreads, stream, g, rows, chunks);
}
template <int TYPE>
void grad_of_type(const DenseGrad& g, int chunks, cudaStream_t stream) {
  switch (g.gated ? kGradSwiGlu + g.kind.act : g.preact ? g.act : (int)kActNone) {
    case kActSilu: grad_of_form<TYPE, kActSilu>(g, chunks, stream); break;
    case kActGelu: grad_of_form<TYPE, kActGelu>(g, chunks, stream); break;
    case kActGeluTanh: grad_of_form<TYPE, kActGeluTanh>(g, chunks, stream); break;
    case kGradSwiGlu: grad_of_form<TYPE, kGradSwiGlu>(g, chunks, stream); break;
    case kGradSiTu: grad_of_form<TYPE, kGradSiTu>(g, chunks, stream); break;
    default: grad_of_form<TYPE, kActNone>(g, chunks, stream);
  }
}

}  // namespace

// Chunks of rows: as many as make the launch three CTAs an SM over 256 columns each, of at least 16 rows; one, whose sums need no
// further kernel, up to 64 rows. The workspace's size follows from it and is asked for without a device: 148 SMs, a B200's.
int dense_sum_chunks(int T, int n_out) {
  if (T <= 64) return 1;
  const int across = (n_out + kGradCols - 1) / kGradCols;
  return std::max(1, std::min(std::max(1, 3 * 148 / across), (T + kGradStep - 1) / kGradStep));
}

void launch_dense_simt(const DenseGemm& g, cudaStream_t stream) {
  const dim3 grid((g.N + (g.gated ? kTile / 2 : kTile) - 1) / (g.gated ? kTile / 2 : kTile), (g.M + kTile - 1) / kTile);
  expects(grid.y <= 65535u, "dense product: at most 4194240 rows on the cross-check kernels");
  if (g.type == kDenseBf16) {
    if (g.gated) dense_simt_kernel<kDenseBf16, true><<<grid, 256, 0, stream>>>(g);
    else dense_simt_kernel<kDenseBf16, false><<<grid, 256, 0, stream>>>(g);
  } else {
    if (g.gated) dense_simt_kernel<kDenseFp16, true><<<grid, 256, 0, stream>>>(g);
    else dense_simt_kernel<kDenseFp16, false><<<grid, 256, 0, stream>>>(g);
  }
  VK_CUDA_CHECK(cudaGetLastError());
}

void launch_dense_grad(const DenseGrad& g, cudaStream_t stream) {
  const int chunks = dense_sum_chunks(g.T, g.N);
  if (g.type == kDenseBf16) grad_of_type<kDenseBf16>(g, chunks, stream);
  else grad_of_type<kDenseFp16>(g, chunks, stream);
}

void launch_dense_sum(DenseType type, const DenseSums& sums, cudaStream_t stream) {
  if (sums.db == nullptr) return;
  const dim3 grid(std::min((sums.cols + 31) / 32, 8 * 148));
  if (type == kDenseBf16) launch_overlapped(dense_sum_kernel<kDenseBf16>, grid, 256, stream, sums);
  else launch_overlapped(dense_sum_kernel<kDenseFp16>, grid, 256, stream, sums);
}

void launch_dense_join(const DenseGemm& g, cudaStream_t stream) {
  const int64_t pitch = dense_part_pitch(g.N), fours = (int64_t)g.M * (pitch / 4);
  const dim3 grid((unsigned)std::min<int64_t>((fours + 255) / 256, 16 * 148));
  if (g.type == kDenseBf16) launch_overlapped(dense_join_kernel<kDenseBf16>, grid, 256, stream, g, pitch);
  else launch_overlapped(dense_join_kernel<kDenseFp16>, grid, 256, stream, g, pitch);
}

void launch_dense_copy_rows(const RowCopies& c, cudaStream_t stream) {
  const int ctas = copy_ctas(c);
  if (ctas > 0) launch_overlapped(dense_copy_rows_kernel, dim3(ctas), 256, stream, c);
}

}  // namespace vkernels::kernels::cuda
