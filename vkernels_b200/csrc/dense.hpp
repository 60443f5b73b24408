// dense.hpp - dense feed-forward operators in 16 bits: the gated projection and the linear projection with bias, activation
// and residual in its epilogue, each with its backward pass. Host-side types and launchers.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace vkernels::kernels::cuda {

enum DenseType { kDenseBf16 = 0, kDenseFp16 = 1 };
// activation of the linear projection
enum DenseAct { kActNone = 0, kActSilu = 1, kActGelu = 2, kActGeluTanh = 3 };

// The gated activation: 0 SwiGLU with its clamp (inf: none), 1 SiTU.
struct GatedKind {
  int act;
  float limit, beta, linear_beta, inv_beta, inv_linear_beta;
  float t_beta, t_linear;     // 2 log2(e) / beta, the same of linear_beta
  float scale;                // 2^-kSituLift beta linear_beta (beta alone without a bend)
};
// Powers of two by which SiTU's denominators are taken smaller, so that their product stays in fp32's range.
constexpr int kSituLift = 60;
constexpr float kSituLifted = 1.0f / (float)(1ull << kSituLift);
inline GatedKind gated_kind(int act, float limit, float beta, float linear_beta) {
  constexpr float kTwoLog2e = 2.8853900817779268f;
  const bool bent = linear_beta > 0.0f;
  const float inv = 1.0f / beta, inv_linear = bent ? 1.0f / linear_beta : 0.0f;
  return {act, limit, beta, linear_beta, inv, inv_linear, kTwoLog2e / beta, bent ? kTwoLog2e / linear_beta : 0.0f, kSituLifted * beta * (bent ? linear_beta : 1.0f)};
}

// One 16-bit operand of a product: element (i, k) is p[i * ld + k], or p[k * ld + i] if mn_major (the index that is NOT
// reduced over is the contiguous one).
struct DenseOperand {
  const uint16_t* p;
  int64_t ld;
  bool mn_major;
};

// out[m, n] = act(sum_k A[m, k] B[n, k] + bias[n]) + residual[m, n], or the gated form: B has 2 N rows (gate rows, then up
// rows), bias 2 N entries, out[m, n] = gate(z[m, n]) * up(z[m, N + n]). preact (optional) receives z in fp32, [M, N] or [M, 2 N].
struct DenseGemm {
  DenseType type;
  DenseOperand a, b;
  int M, N, K;
  bool gated;
  int act;                    // linear: DenseAct
  GatedKind kind;             // gated
  const uint16_t* bias;       // or null
  const uint16_t* residual;   // or null
  int64_t ldr;
  uint16_t* out;
  int64_t ldo;
  float* preact;              // or null
  int64_t ldp;
  // k in `split` parts, if more than one: the sums of each part go to `parts`, [split][M, dense_part_pitch(N)] fp32, and out is made of
  // them by launch_dense_join. Plain linear products only.
  int split;
  float* parts;
};

// dst[i][r, c] = src[i][r, c] for up to two matrices (dst[i] not null), rows of dst one after the other, each on 32 bytes.
struct RowCopies {
  const uint16_t* src[2];
  uint16_t* dst[2];
  int64_t lds[2];
  int rows[2], cols;
};

// Gradient of the pre-activations: dz = dy * act'(z), [T, rows] (linear) or [T, 2 ispp] (gated) at pitch ldz; with no
// activation a copy of dy. dz may be null (only the column sums are wanted). partial (optional) receives the column sums of
// each chunk of rows in fp32, [dense_sum_chunks(T, N), rows]; of a single chunk db receives them at once, in the type.
struct DenseGrad {
  DenseType type;
  const uint16_t* dy;
  int64_t lddy;
  const float* preact;        // null: no activation
  int64_t ldp;
  uint16_t* dz;
  int64_t ldz;
  float* partial;
  uint16_t* db;
  int T, N;                   // N: columns of dy; the gated form has 2 N columns of dz
  bool gated;
  int act;                    // linear: DenseAct
  GatedKind kind;             // gated
  RowCopies copies;           // made by the same launch
};

// db[n] = sum over the chunks of partial[chunk, n] (db null: nothing to do).
struct DenseSums {
  const float* partial;
  int chunks, cols;
  uint16_t* db;
};

int dense_sum_chunks(int T, int n_out);
// Parts that k is cut into at most: more than one where a plain product has few tiles and k is long.
int dense_split(int M, int N, int K);
inline int64_t dense_part_pitch(int N) { return ((int64_t)N + 7) / 8 * 8; }
inline size_t dense_parts_bytes(int M, int N, int split) { return split > 1 ? (size_t)split * (size_t)M * (size_t)dense_part_pitch(N) * 4 : 0; }
// out = the parts' sums, added in order (split > 1).
void launch_dense_join(const DenseGemm& g, cudaStream_t stream);
void launch_dense_gemm(const DenseGemm& g, cudaStream_t stream);
void launch_dense_wide(const DenseGemm& g, cudaStream_t stream);   // dense_gemm.cu
void launch_dense_wide_two(const DenseGemm& g, const DenseGemm& h, const DenseSums& sums, cudaStream_t stream);
void launch_dense_narrow(const DenseGemm& g, cudaStream_t stream);  // dense_narrow.cu
float dense_wide_us(const DenseGemm& g);      // the time that either is expected to take
float dense_narrow_us(const DenseGemm& g);
void launch_dense_simt(const DenseGemm& g, cudaStream_t stream);
void launch_dense_grad(const DenseGrad& g, cudaStream_t stream);
void launch_dense_sum(DenseType type, const DenseSums& sums, cudaStream_t stream);
void launch_dense_copy_rows(const RowCopies& c, cudaStream_t stream);

// ---- the operators ----
struct DenseForward {
  DenseType type;
  const uint16_t *x, *w, *bias, *residual;
  int64_t ldx, ldw, ldr;
  uint16_t* y;
  float* preact;
  int64_t ldy, ldp;
  int T, n_in, n_out;
  bool gated;
  int act;
  float limit, beta, linear_beta;
  void* workspace;
  size_t workspace_bytes;
};
struct DenseBackward {
  DenseType type;
  const uint16_t *dy, *x, *w;
  const float* preact;
  int64_t lddy, ldx, ldw, ldp;
  uint16_t *dx, *dw, *db;     // each may be null
  int64_t lddx, lddw;
  int T, n_in, n_out;
  bool gated;
  int act;
  float limit, beta, linear_beta;
  void* workspace;
  size_t workspace_bytes;
};
void dense_forward(const DenseForward& f, cudaStream_t stream);
void dense_backward(const DenseBackward& f, cudaStream_t stream);
// Workspace: copies of x and w where a tensor map does not take them as they are; of the backward pass also the gradient of the
// pre-activations, the chunks' column sums and the parts of gradients that are cut along k.
size_t dense_forward_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int T, int n_in, int w_rows);
size_t dense_backward_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int T, int n_in, int n_out, bool gated);

}  // namespace vkernels::kernels::cuda
