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
// Rows of the workspace start on 32 bytes: a tensor map takes 16, but every box row then crosses a sector more (1001 tokens,
// 1504 -> 2 x 1027: 19.7 us for the backward pass, 21.6 with rows on 16 bytes; 517 x 1026 -> 770 forward 11.5 and 12.9).
size_t row_pitch(int64_t cols) { return round_up((size_t)cols, 16); }

void check_sizes(int T, int n_in, int n_out, bool gated) {
  expects(T >= 0 && n_in > 0 && n_out > 0, "dense: T must not be negative, feature counts must be positive");
  // (a wait inside the kernels gives up after two seconds; one tile over 2^27 values takes 0.6)
  constexpr int kMost = 1 << 27;
  expects(n_in <= kMost && n_out <= (gated ? kMost / 2 : kMost) && T <= kMost, "dense: sizes beyond 2^27 tokens, inputs or weight rows");
}
void check_common(DenseType type, int T, int n_in, int n_out, bool gated, int act, float limit, float beta) {
  expects(type == kDenseBf16 || type == kDenseFp16, "dense: dtype must be 0 (bf16) or 1 (fp16)");
  check_sizes(T, n_in, n_out, gated);
  if (gated) {
    expects(act == 0 || act == 1, "gated_linear: activation must be 0 (SwiGLU) or 1 (SiTU)");
    expects(limit >= 0.0f, "gated_linear: swiglu_limit must not be negative (0 for none)");
    expects(act == 0 || beta > 0.0f, "gated_linear: SiTU needs a positive beta");
  } else {
    expects(act >= kActNone && act <= kActGeluTanh, "fused_linear: activation must be 0 (none), 1 (silu), 2 (gelu) or 3 (gelu_tanh)");
  }
}
void check_matrix(const void* p, int64_t ld, int cols) {
  expects(p != nullptr && even(p), "dense: null or odd pointer");
  expects(ld >= cols, "dense: a row pitch is smaller than its row");
}
void check_preact(const float* p, int64_t ld, int cols) {
  expects((reinterpret_cast<uintptr_t>(p) & 3u) == 0, "dense: preact must be aligned to its fp32 values");
  expects(ld >= cols, "dense: a row pitch is smaller than its row");
}

size_t copy_bytes(const void* p, int64_t ld, int rows, int cols) {
  return p == nullptr || tma_ready(p, ld) ? 0 : round_up((size_t)rows * row_pitch(cols) * 2, 256);
}

// x and w as a tensor map takes them: as they are, or as copies in rows on 32 bytes at the start of the workspace, which the caller
// has made. Returns the bytes used; a null operand is left alone.
size_t bring_operands(const uint16_t*& x, int64_t& ldx, int T, const uint16_t*& w, int64_t& ldw, int w_rows, int cols, void* workspace,
                      size_t workspace_bytes, RowCopies& c) {
  const size_t bx = copy_bytes(x, ldx, T, cols), bw = copy_bytes(w, ldw, w_rows, cols);
  if (bx + bw == 0) return 0;
  expects(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "dense: workspace must start on 16 bytes");
  expects(workspace_bytes >= bx + bw, "dense: workspace smaller than the copies of x and w that their alignment calls for");
  char* base = static_cast<char*>(workspace);
  c = {{x, w}, {bx ? reinterpret_cast<uint16_t*>(base) : nullptr, bw ? reinterpret_cast<uint16_t*>(base + bx) : nullptr}, {ldx, ldw}, {T, w_rows}, cols};
  const int64_t pitch = (int64_t)row_pitch(cols);
  if (bx) x = c.dst[0], ldx = pitch;
  if (bw) w = c.dst[1], ldw = pitch;
  return bx + bw;
}
float effective_limit(int act, float limit) { return act == 0 && limit > 0.0f ? limit : INFINITY; }

}  // namespace

// Small batches go to the kernel that cuts k over clusters, the others to the CTA pairs: whichever takes less by the sizes. The
// line lies near 64 tokens for short reductions of many features, at some hundred for long ones of few (128 tokens: 2048 -> 7168
// 13.1 us and 11.2, 2880 -> 2880 9.7 and 12, 7168 -> 2 x 2048 gated 16.0 and 24; 256 tokens 18.8 and 11.2, 13.2 and 12.1, 19.9 and
// 24.6).
void launch_dense_gemm(const DenseGemm& g, cudaStream_t stream) {
  if (g.M == 0 || g.N == 0) return;
  if (get_moe_impl() == MoeImpl::kSimt) launch_dense_simt(g, stream);
  else if (!g.a.mn_major && g.M <= 512 && dense_narrow_us(g) < dense_wide_us(g)) launch_dense_narrow(g, stream);
  else launch_dense_wide(g, stream);
}

size_t dense_forward_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int T, int n_in, int w_rows) {
  check_sizes(T, n_in, w_rows, false);
  return T == 0 ? 0 : copy_bytes(x, ldx, T, n_in) + copy_bytes(w, ldw, w_rows, n_in);
}

void dense_forward(const DenseForward& f, cudaStream_t stream) {
  check_common(f.type, f.T, f.n_in, f.n_out, f.gated, f.act, f.limit, f.beta);
  if (f.T == 0) return;
  const int rows = f.gated ? 2 * f.n_out : f.n_out;
  check_matrix(f.x, f.ldx, f.n_in);
  check_matrix(f.w, f.ldw, f.n_in);
  check_matrix(f.y, f.ldy, f.n_out);
  expects(f.bias == nullptr || even(f.bias), "dense: odd bias pointer");
  if (f.residual) check_matrix(f.residual, f.ldr, f.n_out);
  if (f.preact) check_preact(f.preact, f.ldp, rows);
  const uint16_t *x = f.x, *w = f.w;
  int64_t ldx = f.ldx, ldw = f.ldw;
  RowCopies copies{};
  bring_operands(x, ldx, f.T, w, ldw, rows, f.n_in, f.workspace, f.workspace_bytes, copies);
  launch_dense_copy_rows(copies, stream);
  DenseGemm g{};
  g.type = f.type;
  g.a = {x, ldx, false};
  g.b = {w, ldw, false};
  g.M = f.T;
  g.N = f.n_out;
  g.K = f.n_in;
  g.gated = f.gated;
  g.act = f.act;
  if (f.gated) g.kind = gated_kind(f.act, effective_limit(f.act, f.limit), f.beta, f.linear_beta);
  g.bias = f.bias;
  g.residual = f.residual;
  g.ldr = f.ldr;
  g.out = f.y;
  g.ldo = f.ldy;
  g.preact = f.preact;
  g.ldp = f.ldp;
  g.split = 1;
  launch_dense_gemm(g, stream);
}

size_t dense_backward_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int T, int n_in, int n_out, bool gated) {
  check_sizes(T, n_in, n_out, gated);
  const size_t rows = (gated ? 2 : 1) * (size_t)n_out;
  if (T == 0) return 0;
  return copy_bytes(x, ldx, T, n_in) + copy_bytes(w, ldw, (int)rows, n_in) + round_up((size_t)T * row_pitch((int64_t)rows) * 2, 256) +
         round_up((size_t)dense_sum_chunks(T, n_out) * rows * 4, 256) + dense_parts_bytes(T, n_in, dense_split(T, n_in, (int)rows)) +
         dense_parts_bytes((int)rows, n_in, dense_split((int)rows, n_in, T));
}

void dense_backward(const DenseBackward& f, cudaStream_t stream) {
  check_common(f.type, f.T, f.n_in, f.n_out, f.gated, f.act, f.limit, f.beta);
  const int rows = f.gated ? 2 * f.n_out : f.n_out;
  if (f.dw) check_matrix(f.dw, f.lddw, f.n_in);
  expects(f.db == nullptr || even(f.db), "dense: odd bias gradient pointer");
  if (f.T == 0) {   // no token: nothing flows back, and the sums over tokens are zero
    if (f.dw) VK_CUDA_CHECK(cudaMemset2DAsync(f.dw, (size_t)f.lddw * 2, 0, (size_t)f.n_in * 2, (size_t)rows, stream));
    if (f.db) VK_CUDA_CHECK(cudaMemsetAsync(f.db, 0, (size_t)rows * 2, stream));
    return;
  }
  const bool products = f.dx || f.dw;
  if (!products && !f.db) return;
  const bool has_act = f.gated || f.act != kActNone;
  check_matrix(f.dy, f.lddy, f.n_out);
  if (has_act) {
    expects(f.preact != nullptr, "dense backward: the pre-activations of the forward pass are needed");
    check_preact(f.preact, f.ldp, rows);
  }
  if (f.dx) {
    check_matrix(f.w, f.ldw, f.n_in);
    check_matrix(f.dx, f.lddx, f.n_in);
  }
  if (f.dw) check_matrix(f.x, f.ldx, f.n_in);
  // dy itself is the operand where there is no activation and a tensor map takes it
  const bool need_dz = products && (has_act || !tma_ready(f.dy, f.lddy));
  const uint16_t *x = f.dw ? f.x : nullptr, *w = f.dx ? f.w : nullptr;
  int64_t ldx = f.ldx, ldw = f.ldw;
  const int64_t ldz = (int64_t)row_pitch(rows);
  const size_t dz_bytes = need_dz ? round_up((size_t)f.T * ldz * 2, 256) : 0;
  const size_t sums_bytes = f.db ? round_up((size_t)dense_sum_chunks(f.T, f.n_out) * rows * 4, 256) : 0;
  const size_t copies = copy_bytes(x, ldx, f.T, f.n_in) + copy_bytes(w, ldw, rows, f.n_in);
  const bool cut = get_moe_impl() != MoeImpl::kSimt;
  const int split_x = f.dx && cut ? dense_split(f.T, f.n_in, rows) : 1, split_w = f.dw && cut ? dense_split(rows, f.n_in, f.T) : 1;
  const size_t parts_x = dense_parts_bytes(f.T, f.n_in, split_x), parts_w = dense_parts_bytes(rows, f.n_in, split_w);
  const size_t needed = copies + dz_bytes + sums_bytes + parts_x + parts_w;
  if (needed > 0) {
    expects(f.workspace != nullptr && (reinterpret_cast<uintptr_t>(f.workspace) & 15u) == 0, "dense: workspace must start on 16 bytes");
    expects(f.workspace_bytes >= needed, "dense: workspace smaller than vk_cuda_dense_backward_workspace_bytes");
  }
  RowCopies made{};
  bring_operands(x, ldx, f.T, w, ldw, rows, f.n_in, f.workspace, f.workspace_bytes, made);
  uint16_t* dz = need_dz ? reinterpret_cast<uint16_t*>(static_cast<char*>(f.workspace) + copies) : nullptr;
  DenseSums sums{};
  if (need_dz || f.db) {
    float* partial = f.db ? reinterpret_cast<float*>(static_cast<char*>(f.workspace) + copies + dz_bytes) : nullptr;
    DenseGrad g{};
    g.type = f.type;
    g.dy = f.dy;
    g.lddy = f.lddy;
    g.preact = has_act ? f.preact : nullptr;
    g.ldp = f.ldp;
    g.dz = dz;
    g.ldz = ldz;
    const int chunks = dense_sum_chunks(f.T, f.n_out);
    g.partial = chunks > 1 ? partial : nullptr;
    g.db = chunks > 1 ? nullptr : f.db;
    g.T = f.T;
    g.N = f.n_out;
    g.gated = f.gated;
    g.act = f.act;
    if (f.gated) g.kind = gated_kind(f.act, effective_limit(f.act, f.limit), f.beta, f.linear_beta);
    g.copies = made;
    launch_dense_grad(g, stream);
    if (f.db && chunks > 1) sums = {partial, chunks, rows, f.db};
  } else {
    launch_dense_copy_rows(made, stream);
  }
  const uint16_t* z = need_dz ? dz : f.dy;
  const int64_t ldzz = need_dz ? ldz : f.lddy;
  DenseGemm gx{}, gw{};
  gx.type = gw.type = f.type;
  gx.split = split_x;
  gw.split = split_w;
  gx.parts = reinterpret_cast<float*>(static_cast<char*>(f.workspace) + copies + dz_bytes + sums_bytes);
  gw.parts = reinterpret_cast<float*>(reinterpret_cast<char*>(gx.parts) + parts_x);
  if (f.dx) {   // dx[t, i] = sum_n dz[t, n] w[n, i]
    gx.a = {z, ldzz, false};
    gx.b = {w, ldw, true};
    gx.M = f.T;
    gx.N = f.n_in;
    gx.K = rows;
    gx.out = f.dx;
    gx.ldo = f.lddx;
  }
  if (f.dw) {   // dw[n, i] = sum_t dz[t, n] x[t, i]
    gw.a = {z, ldzz, true};
    gw.b = {x, ldx, true};
    gw.M = rows;
    gw.N = f.n_in;
    gw.K = f.T;
    gw.out = f.dw;
    gw.ldo = f.lddw;
  }
  // both in one launch: the tiles of one fill what the other leaves idle (1001 tokens, 1504 -> 2 x 1024: 21.3 us as two)
  if (f.dx && f.dw && get_moe_impl() != MoeImpl::kSimt) {
    launch_dense_wide_two(gx, gw, sums, stream);
    return;
  }
  launch_dense_sum(f.type, sums, stream);
  if (f.dx) launch_dense_gemm(gx, stream);
  if (f.dw) launch_dense_gemm(gw, stream);
}

}  // namespace vkernels::kernels::cuda
