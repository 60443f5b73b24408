// dense.cu - host side of the dense feed-forward operators: argument contract, choice of kernel, order of the backward pass.
#include <cmath>

#include "common.cuh"
#include "dense.hpp"
#include "moe_fused.hpp"

namespace vkernels::kernels::cuda {

namespace {

bool tma_ready(const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0; }
bool even(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }
size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

void check_common(DenseType type, int T, int n_in, int n_out, bool gated, int act, float limit, float beta) {
  expects(type == kDenseBf16 || type == kDenseFp16, "dense: dtype must be 0 (bf16) or 1 (fp16)");
  expects(T >= 0 && n_in > 0 && n_out > 0, "dense: T must not be negative, feature counts must be positive");
  expects(n_in <= (1 << 30) && n_out <= (1 << 29) && T <= (1 << 30), "dense: sizes beyond 2^29 features or 2^30 tokens");
  if (gated) {
    expects(act == 0 || act == 1, "gated_linear: activation must be 0 (SwiGLU) or 1 (SiTU)");
    expects(limit >= 0.0f, "gated_linear: swiglu_limit must not be negative (0 for none)");
    expects(act == 0 || beta > 0.0f, "gated_linear: SiTU needs a positive beta");
  } else {
    expects(act >= kActNone && act <= kActGeluTanh, "fused_linear: activation must be 0 (none), 1 (silu), 2 (gelu) or 3 (gelu_tanh)");
  }
}
void check_operand(const void* p, int64_t ld, int cols, const char* null_msg, const char* align_msg) {
  expects(p != nullptr, null_msg);
  expects(ld >= cols, "dense: a row pitch is smaller than its row");
  expects(tma_ready(p, ld), align_msg);
}
void check_result(const void* p, int64_t ld, int cols) {
  expects(p != nullptr && even(p), "dense: null or odd pointer");
  expects(ld >= cols, "dense: a row pitch is smaller than its row");
}
float effective_limit(bool gated, int act, float limit) { return gated && act == 0 && limit > 0.0f ? limit : INFINITY; }

}  // namespace

void launch_dense_gemm(const DenseGemm& g, cudaStream_t stream) {
  if (g.M == 0 || g.N == 0) return;
  if (get_moe_impl() == MoeImpl::kSimt) launch_dense_simt(g, stream);
  else launch_dense_wide(g, stream);
}

void dense_forward(const DenseForward& f, cudaStream_t stream) {
  check_common(f.type, f.T, f.n_in, f.n_out, f.gated, f.act, f.limit, f.beta);
  if (f.T == 0) return;
  const int rows = f.gated ? 2 * f.n_out : f.n_out;
  check_operand(f.x, f.ldx, f.n_in, "dense: x is null", "dense: x must start on 16 bytes, its row pitch must be a multiple of 8 elements");
  check_operand(f.w, f.ldw, f.n_in, "dense: w is null", "dense: w must start on 16 bytes, its row pitch must be a multiple of 8 elements");
  check_result(f.y, f.ldy, f.n_out);
  expects(f.bias == nullptr || even(f.bias), "dense: odd bias pointer");
  if (f.residual) check_result(f.residual, f.ldr, f.n_out);
  if (f.preact) check_result(f.preact, f.ldp, rows);
  DenseGemm g{};
  g.type = f.type;
  g.a = {f.x, f.ldx, false};
  g.b = {f.w, f.ldw, false};
  g.M = f.T;
  g.N = f.n_out;
  g.K = f.n_in;
  g.gated = f.gated;
  g.act = f.act;
  g.limit = effective_limit(f.gated, f.act, f.limit);
  g.beta = f.beta;
  g.linear_beta = f.linear_beta;
  g.bias = f.bias;
  g.residual = f.residual;
  g.ldr = f.ldr;
  g.out = f.y;
  g.ldo = f.ldy;
  g.preact = f.preact;
  g.ldp = f.ldp;
  launch_dense_gemm(g, stream);
}

// Workspace of the backward pass: the gradient of the pre-activations at a pitch that a tensor map takes, then the chunks'
// column sums.
size_t dense_backward_workspace_bytes(int T, int n_out, bool gated) {
  expects(T >= 0 && n_out > 0, "dense: T must not be negative, n_out must be positive");
  const size_t rows = (gated ? 2 : 1) * (size_t)n_out;
  return round_up((size_t)T * round_up(rows, 8) * 2, 256) + (size_t)dense_sum_chunks(T) * rows * 4;
}

void dense_backward(const DenseBackward& f, cudaStream_t stream) {
  check_common(f.type, f.T, f.n_in, f.n_out, f.gated, f.act, f.limit, f.beta);
  const int rows = f.gated ? 2 * f.n_out : f.n_out;
  if (f.dw) check_result(f.dw, f.lddw, f.n_in);
  if (f.T == 0) {   // no token: nothing flows back, and the sums over tokens are zero
    if (f.dw) VK_CUDA_CHECK(cudaMemset2DAsync(f.dw, (size_t)f.lddw * 2, 0, (size_t)f.n_in * 2, (size_t)rows, stream));
    if (f.db) VK_CUDA_CHECK(cudaMemsetAsync(f.db, 0, (size_t)rows * 2, stream));
    return;
  }
  const bool has_act = f.gated || f.act != kActNone;
  check_result(f.dy, f.lddy, f.n_out);
  if (has_act) {
    expects(f.preact != nullptr, "dense backward: the pre-activations of the forward pass are needed");
    check_result(f.preact, f.ldp, rows);
  }
  if (f.dx) {
    check_operand(f.w, f.ldw, f.n_in, "dense: w is null", "dense: w must start on 16 bytes, its row pitch must be a multiple of 8 elements");
    check_result(f.dx, f.lddx, f.n_in);
  }
  if (f.dw)
    check_operand(f.x, f.ldx, f.n_in, "dense: x is null", "dense: x must start on 16 bytes, its row pitch must be a multiple of 8 elements");
  expects(f.db == nullptr || even(f.db), "dense: odd bias gradient pointer");
  // dy itself is the operand where there is no activation and a tensor map takes it
  const bool products = f.dx || f.dw;
  const bool need_dz = products && (has_act || !tma_ready(f.dy, f.lddy));
  if (!products && !f.db) return;
  const int64_t ldz = (int64_t)round_up(rows, 8);
  uint16_t* dz = nullptr;
  float* partial = nullptr;
  if (need_dz || f.db) {
    expects(f.workspace != nullptr && (reinterpret_cast<uintptr_t>(f.workspace) & 15u) == 0, "dense backward: workspace must start on 16 bytes");
    expects(f.workspace_bytes >= dense_backward_workspace_bytes(f.T, f.n_out, f.gated),
            "dense backward: workspace smaller than vk_cuda_dense_backward_workspace_bytes");
    char* base = static_cast<char*>(f.workspace);
    if (need_dz) dz = reinterpret_cast<uint16_t*>(base);
    if (f.db) partial = reinterpret_cast<float*>(base + round_up((size_t)f.T * ldz * 2, 256));
    DenseGrad g{};
    g.type = f.type;
    g.dy = f.dy;
    g.lddy = f.lddy;
    g.preact = has_act ? f.preact : nullptr;
    g.ldp = f.ldp;
    g.dz = dz;
    g.ldz = ldz;
    g.partial = partial;
    g.T = f.T;
    g.N = f.n_out;
    g.gated = f.gated;
    g.act = f.act;
    g.limit = effective_limit(f.gated, f.act, f.limit);
    g.beta = f.beta;
    g.linear_beta = f.linear_beta;
    launch_dense_grad(g, stream);
    if (f.db) launch_dense_sum(f.type, partial, dense_sum_chunks(f.T), rows, f.db, stream);
  }
  const uint16_t* z = need_dz ? dz : f.dy;
  const int64_t ldzz = need_dz ? ldz : f.lddy;
  DenseGemm g{};
  g.type = f.type;
  g.limit = INFINITY;
  if (f.dx) {   // dx[t, i] = sum_n dz[t, n] w[n, i]
    g.a = {z, ldzz, false};
    g.b = {f.w, f.ldw, true};
    g.M = f.T;
    g.N = f.n_in;
    g.K = rows;
    g.out = f.dx;
    g.ldo = f.lddx;
    launch_dense_gemm(g, stream);
  }
  if (f.dw) {   // dw[n, i] = sum_t dz[t, n] x[t, i]
    g.a = {z, ldzz, true};
    g.b = {f.x, f.ldx, true};
    g.M = rows;
    g.N = f.n_in;
    g.K = f.T;
    g.out = f.dw;
    g.ldo = f.lddw;
    launch_dense_gemm(g, stream);
  }
}

}  // namespace vkernels::kernels::cuda
