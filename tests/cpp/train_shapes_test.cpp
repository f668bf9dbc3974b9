// The C++ training calls (include/pet/train.hpp) refuse views whose shapes do not fit
// together before any device work, so this runs without a GPU
// (tests/test_train_args.py); every address is a stand-in. Prints the calls that did
// not throw, or threw something else.
#include <cstdio>
#include <cstring>
#include <functional>
#include <string>

#include "pet/train.hpp"

using pet::Rows;
using pet::View1D;
using pet::View2D;
using pet::WeightRef;

int main() {
  float* p = reinterpret_cast<float*>(4096);
  const int T = 6, N = 2, S = 4, D = 16;
  pet::Workspace ws;
  int bad = 0;
  auto throws = [&](const char* name, const char* text, const std::function<void()>& f) {
    std::string got = "nothing";
    try {
      f();
    } catch (const std::exception& e) {
      got = e.what();
    }
    if (got.find(text) == std::string::npos) std::printf("%s: %s\n", name, got.c_str()), ++bad;
  };
  const View2D x(p, T, D), narrow(p, T, D - 1, D), few(p, T - 1, D);
  const View1D v{p, D}, s{p, D - 1};
  throws("norm_rows width", "one width", [&] { pet::norm_rows(Rows(narrow), Rows(x), v, v); });
  throws("norm_rows rows", "one type and number", [&] { pet::norm_rows(Rows(few), Rows(x), v, v); });
  throws("norm_rows weight", "weight: a vector", [&] { pet::norm_rows(Rows(x), Rows(x), s, v); });
  throws("norm_rows bias", "bias: a vector", [&] { pet::norm_rows(Rows(x), Rows(x), v, s); });
  auto ng = [&](const View2D& a, const View1D& wa, const View1D& ba, const View2D& g, const View1D& w) {
    return [=, &ws, &x] { pet::norm_rows_grads(ws, a, wa, ba, g, x, w, true); };
  };
  throws("norm_rows_grads out_adj", "one width", ng(x, v, v, narrow, v));
  throws("norm_rows_grads in_adj", "one width", ng(narrow, v, v, x, v));
  throws("norm_rows_grads rows", "one type and number", ng(few, v, v, x, v));
  throws("norm_rows_grads weight", "weight: a vector", ng(x, v, v, x, s));
  throws("norm_rows_grads weight_adj", "weight_adj: a vector", ng(x, s, v, x, v));
  throws("norm_rows_grads bias_adj", "bias_adj: a vector", ng(x, v, s, x, v));
  throws("linear_grads w_adj", "w_adj is not", [&] { pet::linear_grads(ws, x, x, narrow, v); });
  throws("linear_grads b_adj", "b_adj: a vector", [&] { pet::linear_grads(ws, x, x, View2D(p, D, D), s); });

  struct Layer {
    View2D tokens_adj, cf_adj, out_adj, tokens, w_in, cf, w_out;
    View1D norm_w, norm_b, b_in;
  };
  const Layer good{x, View2D(p, N, S), x, x, View2D(p, 3 * D, D), View2D(p, N, S), View2D(p, D, D), v, v, {p, 3 * D}};
  auto layer = [&](const char* name, const char* text, const std::function<void(Layer&)>& change) {
    Layer a = good;
    change(a);
    throws(name, text, [&] {
      pet::attention_layer_grads(ws, "l", {p, p, p, p, p, p, 0.f}, a.tokens_adj, a.cf_adj, a.out_adj, a.tokens, a.norm_w,
                                 a.norm_b, WeightRef(a.w_in), a.b_in, a.cf, WeightRef(a.w_out), {nullptr, N, false}, S, 1, D,
                                 1.0);
    });
  };
  layer("layer saves", "no buffer named", [](Layer&) {});
  layer("layer tokens", "tokens are not", [&](Layer& a) { a.tokens = narrow; });
  layer("layer tokens_adj", "tokens_adj is not", [&](Layer& a) { a.tokens_adj = few; });
  layer("layer out_adj", "out_adj is not", [&](Layer& a) { a.out_adj = few; });
  layer("layer w_in", "w_in is not", [&](Layer& a) { a.w_in = a.w_out; });
  layer("layer w_out", "w_out is not", [&](Layer& a) { a.w_out = a.w_in; });
  layer("layer w_in's rows", "contiguous", [&](Layer& a) { a.w_in.ld = D + 1; });
  layer("layer cf", "cf_seq", [&](Layer& a) { a.cf = View2D(p, N, S - 1); });
  layer("layer cf_adj", "cf_seq", [&](Layer& a) { a.cf_adj = View2D(p, N - 1, S); });
  layer("layer norm_w", "norm_w: a vector", [&](Layer& a) { a.norm_w = s; });
  layer("layer norm_b", "norm_b: a vector", [&](Layer& a) { a.norm_b = s; });
  layer("layer b_in", "b_in: a vector", [&](Layer& a) { a.b_in = v; });
  return bad;
}
