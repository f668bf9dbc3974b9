// Sizes whose products pass an int: the C++ calls (include/pet/attention.hpp,
// include/pet/train.hpp) say so before any device work, so this runs without a GPU
// (tests/test_typed_limits.py); every address is a stand-in or null. Prints the calls
// that did not throw, or threw something else.
#include <cstdint>
#include <cstdio>
#include <functional>
#include <string>

#include "pet/train.hpp"

using pet::Rows;
using pet::View1D;
using pet::View2D;
using pet::WeightRef;

int main() {
  float* const p = reinterpret_cast<float*>(4096);
  const int* const off = reinterpret_cast<const int*>(4096);
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
  // N heads S = 2^32 + 2^24, of which an int would keep 2^24
  const int N = 65536, H = 256, S = 257, bf = PET_DTYPE_BF16;
  const char* const saves = "N heads S";
  pet::Workspace ws;
  const Rows qkv(p, N, 3 * H, bf), merged(p, N, H, bf);
  const View2D ml(p, 1 << 24, 2), cf(nullptr, N, S);  // (without cutoff factors no call gets past its checks)
  const pet::TypedAttention at{pet::Tokens{off, N, false}, S, H, H, 1};
  throws("attn_fwd_typed", saves, [&] { pet::attn_fwd_typed(at, merged, ml, qkv, cf); });
  throws("attn_fwd_typed without saves", "invalid argument", [&] { pet::attn_fwd_typed(at, merged, View2D(), qkv, cf); });
  throws("attn_bwd_typed", saves, [&] { pet::attn_bwd_typed(ws, at, qkv, View2D(), View2D(), merged, qkv, merged, ml, cf); });

  const View2D x(p, N, H), x3(p, N, 3 * H), none(nullptr, N, S), w_in(p, 3 * H, H), w_out(p, H, H);
  const View1D v{p, H}, v3{p, 3 * H};
  const pet::Tokens tk{off, N, false};
  throws("attention", saves, [&] { pet::attention(ws, "k", x, x3, none, WeightRef(w_out), v, tk, S, H, 1, 1.0, true); });
  throws("attention_layer", saves, [&] {
    pet::attention_layer(ws, "k", x, x, v, v, WeightRef(w_in), v3, none, WeightRef(w_out), v, tk, S, H, 1, 1.0);
  });
  throws("attention_layer_grads", saves, [&] {
    pet::attention_layer_grads(ws, "k", {p, p, p, p, p, p, 0.f}, x, none, x, x, v, v, WeightRef(w_in), v3, none, WeightRef(w_out),
                               tk, S, H, 1, 1.0);
  });

  // (heads + 2 kv_heads) head_dim = 2^32 + 2, of which an int would keep 2
  const pet::TypedAttention wide{pet::Tokens{off, 1, false}, 1, (1 << 30), (1 << 30) + (1 << 29) + 1, 1};
  throws("columns", "[T, (heads + 2 kv_heads) head_dim]",
         [&] { pet::attn_fwd_typed(wide, Rows(p, 1, 1 << 30, bf), View2D(), Rows(p, 1, 2, bf), View2D(nullptr, 1, 1)); });
  // no atoms is no overflow
  throws("no atoms", "nothing", [&] { pet::attn_fwd_typed({pet::Tokens{off, 0, false}, S, H, H, 1}, Rows(p, 0, H, bf), View2D(),
                                                          Rows(p, 0, 3 * H, bf), View2D(p, 0, S)); });
  return bad;
}
