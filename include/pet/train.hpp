// pet/train.hpp -- what a training step adds, for a C++ caller: the norm's and a
// dense layer's parameter gradients, an attention layer's, and the norm and
// clipping of them all (pet_norm_rows_grads, pet_linear_grads,
// pet_attention_layer_grads, pet_grad_norm, pet_grad_clip). The reference
// (peterspackman/pet-kokkos) evaluates only, so none of it has a counterpart
// there; the views, the Workspace that holds the scratch and the exceptions are
// those of pet/attention.hpp. A Workspace serves one stream at a time, and a call that
// needs more of it than any before frees what it grows: a captured graph has a
// Workspace of its own, warm before the capture.
#pragma once

#include <hip/hip_runtime.h>

#include <string>
#include <vector>

#include "../pet_model.h"
#include "attention.hpp"

namespace pet {

// Rows of activations or their adjoints in fp32, bf16 or fp16 (PET_DTYPE_*).
struct Rows {
  void* ptr = nullptr;
  int rows = 0, cols = 0;
  int64_t ld = 0;  // in elements
  int dtype = PET_DTYPE_F32;
  Rows() = default;
  Rows(const View2D& v) : ptr(v.data()), rows(v.extent(0)), cols(v.extent(1)), ld(v.stride(0)) {}
  Rows(void* p, int r, int c, int type, int64_t stride = -1) : ptr(p), rows(r), cols(c), ld(stride < 0 ? c : stride), dtype(type) {}
};

inline void need(bool ok, const char* what, const char* needs) {
  if (!ok) throw std::runtime_error(std::string("pet: ") + what + ": " + needs);
}
inline void check_rows(const Rows& a, const Rows& b, const char* what) {
  need(a.dtype == b.dtype && a.rows == b.rows, what, "rows of one type and number are needed");
}
// A view that holds data has the shape that the call reads or writes (a vector may
// leave its length at 0).
inline void check_vector(const View1D& v, int n, const char* what) {
  need(!v.data() || v.n == 0 || v.n == n, what, "a vector of another length");
}
inline void check_matrix(const View2D& m, int rows, int cols, const char* what, const char* needs) {
  need(!m.data() || (m.extent(0) == rows && m.extent(1) == cols), what, needs);
}

// out = norm(in), RMSNorm or with a bias LayerNorm.
inline void norm_rows(const Rows& out, const Rows& in, View1D weight, View1D bias, hipStream_t stream = nullptr) {
  check_rows(out, in, "norm_rows");
  need(out.cols == in.cols, "norm_rows", "rows of one width are needed");
  check_vector(weight, in.cols, "norm_rows: weight");
  check_vector(bias, in.cols, "norm_rows: bias");
  check(pet_norm_rows_typed(in.dtype, in.rows, in.cols, out.ptr, out.ld, in.ptr, in.ld, weight.data(), bias.data(),
                            stream),
        "norm_rows");
}

// in_adj (may hold no pointer) = beta in_adj + the norm's adjoint, weight_adj
// and bias_adj (may hold none) onto beta_w times themselves; live: the device's
// count of rows that count, or null.
inline void norm_rows_grads(Workspace& ws, const Rows& in_adj, View1D weight_adj, View1D bias_adj, const Rows& out_adj,
                            const Rows& in, View1D weight, bool ln, Net beta = 0, Net beta_w = 0,
                            const int* live = nullptr, hipStream_t stream = nullptr) {
  check_rows(out_adj, in, "norm_rows_grads");
  if (in_adj.ptr) check_rows(in_adj, in, "norm_rows_grads");
  need(out_adj.cols == in.cols && (!in_adj.ptr || in_adj.cols == in.cols), "norm_rows_grads",
       "rows of one width are needed");
  check_vector(weight, in.cols, "norm_rows_grads: weight");
  check_vector(weight_adj, in.cols, "norm_rows_grads: weight_adj");
  check_vector(bias_adj, in.cols, "norm_rows_grads: bias_adj");
  const bool params = weight_adj.data() || bias_adj.data();
  const size_t bytes = params ? pet_norm_rows_grads_workspace(in.rows, in.cols) : 0;
  void* scratch = params ? ws.bytes("norm_rows_grads:scratch", bytes) : nullptr;
  check(pet_norm_rows_grads(in.dtype, in.rows, in.cols, in_adj.ptr, in_adj.ld, beta, out_adj.ptr, out_adj.ld, in.ptr,
                            in.ld, weight.data(), ln ? 1 : 0, weight_adj.data(), bias_adj.data(), beta_w, live,
                            scratch, bytes, stream),
        "norm_rows_grads");
}

// w_adj [N, K] = beta w_adj + out_adj^T in, b_adj (may hold none) = beta b_adj + the sum of out_adj's rows.
inline void linear_grads(Workspace& ws, const Rows& out_adj, const Rows& in, View2D w_adj, View1D b_adj, Net beta = 0,
                         const int* live = nullptr, hipStream_t stream = nullptr) {
  check_rows(out_adj, in, "linear_grads");
  need(w_adj.extent(0) == out_adj.cols && w_adj.extent(1) == in.cols, "linear_grads",
       "w_adj is not [out_adj's columns, in's columns]");
  check_vector(b_adj, out_adj.cols, "linear_grads: b_adj");
  const size_t bytes = pet_linear_grads_workspace(in.dtype, in.rows, out_adj.cols, in.cols);
  void* scratch = ws.bytes("linear_grads:scratch", bytes);
  check(pet_linear_grads(in.dtype, in.rows, out_adj.cols, in.cols, out_adj.ptr, out_adj.ld, in.ptr, in.ld, live,
                         w_adj.data(), w_adj.stride(0), b_adj.data(), beta, scratch, bytes, stream),
        "linear_grads");
}

// attention_layer_bwd with the gradients of the layer's parameters (null pointers: not made).
inline void attention_layer_grads(Workspace& ws, const std::string& key, const pet_layer_grads& grads,
                                  View2D tokens_adj, View2D cf_seq_adj, View2D out_adj, View2D tokens, View1D norm_w,
                                  View1D norm_b, const WeightRef& w_in, View1D b_in, View2D cf_seq,
                                  const WeightRef& w_out, const Tokens& tk, int S, int heads, int head_dim,
                                  double temperature, hipStream_t stream = nullptr) {
  const int T = tokens.extent(0), D = heads * head_dim;
  const char* what = "attention_layer_grads";
  check_matrix(tokens, T, D, what, "tokens are not [T, heads * head_dim]");
  check_matrix(tokens_adj, T, D, what, "tokens_adj is not [T, heads * head_dim]");
  check_matrix(out_adj, T, D, what, "out_adj is not [T, heads * head_dim]");
  check_matrix(w_in.v, 3 * D, D, what, "w_in is not [3 D, D]");
  check_matrix(w_out.v, D, D, what, "w_out is not [D, D]");
  need(w_in.v.stride(0) == D && w_out.v.stride(0) == D, what, "contiguous weights are needed");
  need(cf_seq.extent(0) == tk.N && cf_seq.extent(1) >= S && cf_seq_adj.extent(0) == tk.N && cf_seq_adj.extent(1) >= S, what,
       "cf_seq and cf_seq_adj are not [N, S] or wider");
  check_vector(norm_w, D, "attention_layer_grads: norm_w");
  check_vector(norm_b, D, "attention_layer_grads: norm_b");
  check_vector(b_in, 3 * D, "attention_layer_grads: b_in");
  const pet_attn_shape sh = make_shape(tk, T, S, heads, head_dim, temperature);
  const View2D merged = ws.peek2(key + ":merged"), ml = ws.peek2(key + ":ml");
  check_matrix(merged, T, D, what, "the saves under the key are of another shape");
  check_matrix(ml, tk.N * heads * S, 2, what, "the saves under the key are of another shape");
  const size_t bytes = pet_attention_layer_grads_workspace(&sh);
  void* scratch = ws.bytes("attention_layer_grads:scratch", bytes);
  check(pet_attention_layer_grads(&sh, &grads, tokens_adj.data(), tokens_adj.stride(0), cf_seq_adj.data(),
                                  cf_seq_adj.stride(0), out_adj.data(), out_adj.stride(0), tokens.data(),
                                  tokens.stride(0), norm_w.data(), norm_b.data(), w_in.v.data(), b_in.data(),
                                  cf_seq.data(), cf_seq.stride(0), w_out.v.data(), tk.off, merged.data(), ml.data(),
                                  scratch, bytes, stream),
        "attention_layer_grads");
}

// One tensor of a list of gradients: consecutive elements, or rows of a wider matrix.
inline pet_grad_tensor gradient(void* data, int64_t numel, int dtype = PET_DTYPE_F32) {
  return {data, 1, numel, numel, dtype};
}
inline pet_grad_tensor gradient(const View2D& v) {
  return {v.data(), v.extent(0), v.extent(1), v.stride(0), PET_DTYPE_F32};
}

// *norm (device) of all gradients times scale; p 1 or 2, or 0 for the largest magnitude.
inline void grad_norm(Workspace& ws, const std::vector<pet_grad_tensor>& grads, float* norm, int p = 2,
                      double scale = 1.0, hipStream_t stream = nullptr) {
  const size_t bytes = pet_grad_workspace(int(grads.size()));
  check(pet_grad_norm(grads.data(), int(grads.size()), p, scale, norm, ws.bytes("grads:scratch", bytes), bytes, stream),
        "grad_norm");
}
// ... and every gradient times scale min(1, max_norm / (*norm + eps)) in place.
inline void clip_grads(Workspace& ws, const std::vector<pet_grad_tensor>& grads, double max_norm, float* norm,
                       int p = 2, double scale = 1.0, double eps = 1e-6, hipStream_t stream = nullptr) {
  const size_t bytes = pet_grad_workspace(int(grads.size()));
  check(pet_grad_clip(grads.data(), int(grads.size()), p, scale, max_norm, eps, norm, ws.bytes("grads:scratch", bytes),
                      bytes, stream),
        "clip_grads");
}

}  // namespace pet
