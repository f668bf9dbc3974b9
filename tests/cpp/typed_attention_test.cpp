// The typed attention, its backward and the dropout through the C++ interface
// (include/pet/train.hpp).
//
//   typed_attention_test                          shapes that have to throw before any GPU call
//   typed_attention_test DIR N T S H HK HD NB R   a run, for tests/test_gpu_cpp_typed.py
//
// The run reads DIR/{qkv,g}.b16 (bf16), DIR/{cf,table}.f32, DIR/{off,buckets,pos}.i32
// and DIR/state.i64; takes attn_fwd_typed of a dropout of 1/4 with call 1,
// dropout_rows of merged onto g with call 2, and attn_bwd_typed of that; writes
// DIR/{merged,rows,qkv_adj}.b16 and DIR/{ml,cf_adj,table_adj}.f32.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <string>
#include <vector>

#include "pet/train.hpp"

template <class T>
static T* upload(const std::string& path, size_t n) {
  std::vector<T> v(n);
  FILE* f = std::fopen(path.c_str(), "rb");
  if (!f || std::fread(v.data(), sizeof(T), n, f) != n) std::exit(2);
  std::fclose(f);
  void* p = nullptr;
  if (hipMalloc(&p, n * sizeof(T)) != hipSuccess) std::exit(4);
  if (hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) std::exit(4);
  return static_cast<T*>(p);
}
template <class T>
static T* empty(size_t n) {
  const std::vector<T> v(n);
  void* p = nullptr;
  if (hipMalloc(&p, n * sizeof(T)) != hipSuccess) std::exit(4);
  if (hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) std::exit(4);
  return static_cast<T*>(p);
}
static void write(const std::string& path, const void* dev, size_t bytes) {
  std::vector<char> v(bytes);
  if (hipMemcpy(v.data(), dev, bytes, hipMemcpyDeviceToHost) != hipSuccess) std::exit(4);
  FILE* f = std::fopen(path.c_str(), "wb");
  if (!f || std::fwrite(v.data(), 1, bytes, f) != bytes) std::exit(3);
  std::fclose(f);
}

template <class F>
static int throws(F&& f) {
  try {
    f();
  } catch (const std::runtime_error&) {
    return 0;
  }
  return 1;
}

// (the pointers are of host memory and never read)
static int refusals() {
  static uint16_t rows[64];
  static float floats[64];
  static int off[2] = {0, 1};
  static int64_t state[2];
  const int bf = PET_DTYPE_BF16;
  const pet::Rows qkv(rows, 2, 12, bf), merged(rows, 2, 4, bf);
  const pet::View2D cf(floats, 1, 2), ml(floats, 2, 2), table(floats, 2, 1);
  pet::Workspace ws;
  pet::TypedAttention at{pet::Tokens{off, 1, false}, 2, 1, 1, 4};
  const pet_dropout drop{state, 0.5, 0}, all{state, 1.0, 0};
  const pet::Rows none;
  int bad = 0;
  bad += throws([&] { pet::dropout_rows(merged, qkv, none, drop); });
  bad += throws([&] { pet::dropout_rows(merged, merged, qkv, drop); });
  bad += throws([&] { pet::dropout_rows(pet::Rows(rows, 2, 4, PET_DTYPE_F16), merged, none, drop); });
  bad += throws([&] { pet::dropout_rows(merged, merged, none, all); });
  bad += throws([&] { pet::attn_fwd_typed(at, qkv, ml, qkv, cf); });
  bad += throws([&] { pet::attn_fwd_typed(at, merged, ml, merged, cf); });
  bad += throws([&] { pet::attn_fwd_typed(at, merged, pet::View2D(floats, 1, 2), qkv, cf); });
  bad += throws([&] { pet::attn_fwd_typed(at, merged, ml, qkv, pet::View2D(floats, 1, 1)); });
  bad += throws([&] { pet::attn_bwd_typed(ws, at, merged, cf, pet::View2D(), merged, qkv, merged, ml, cf); });
  bad += throws([&] { pet::attn_bwd_typed(ws, at, qkv, cf, table, merged, qkv, merged, ml, cf); });
  bad += throws([&] { pet::attn_bwd_typed(ws, at, qkv, cf, pet::View2D(), merged, qkv, merged, pet::View2D(), cf); });
  bad += throws([&] { pet::attn_bwd_typed(ws, at, qkv, cf, pet::View2D(), qkv, qkv, merged, ml, cf); });
  at.heads = 3, at.kv_heads = 2;
  bad += throws([&] { pet::attn_fwd_typed(at, pet::Rows(rows, 2, 12, bf), pet::View2D(), pet::Rows(rows, 2, 28, bf), cf); });
  return bad;
}

int main(int argc, char** argv) {
  if (argc == 1) return refusals();
  if (argc != 10) return 1;
  const std::string dir = std::string(argv[1]) + "/";
  int n[8];
  for (int i = 0; i < 8; ++i) n[i] = std::atoi(argv[2 + i]);
  const int N = n[0], T = n[1], S = n[2], H = n[3], Hk = n[4], hd = n[5], nb = n[6], R = n[7], D = H * hd, W = D + 2 * Hk * hd;
  try {
    pet::Workspace ws;
    const int bf = PET_DTYPE_BF16;
    const pet_attn_bias bias{upload<float>(dir + "table.f32", size_t(nb) * H), upload<int>(dir + "buckets.i32", 2 * R + 1),
                             upload<int>(dir + "pos.i32", T), nb, R};
    const int64_t* state = upload<int64_t>(dir + "state.i64", 2);
    const pet_dropout first{state, 0.25, 1}, second{state, 0.25, 2};
    const pet::TypedAttention at{pet::Tokens{upload<int>(dir + "off.i32", N + 1), N, false}, S, H, Hk, hd, 1.0, &bias, &first};
    const pet::Rows qkv(upload<uint16_t>(dir + "qkv.b16", size_t(T) * W), T, W, bf),
        g(upload<uint16_t>(dir + "g.b16", size_t(T) * D), T, D, bf), merged(empty<uint16_t>(size_t(T) * D), T, D, bf),
        rows(empty<uint16_t>(size_t(T) * D), T, D, bf), qkv_adj(empty<uint16_t>(size_t(T) * W), T, W, bf);
    const pet::View2D cf(upload<float>(dir + "cf.f32", size_t(N) * S), N, S), ml(empty<float>(size_t(N) * H * S * 2), N * H * S, 2),
        cf_adj(empty<float>(size_t(N) * S), N, S), table_adj(empty<float>(size_t(nb) * H), nb, H);
    pet::attn_fwd_typed(at, merged, ml, qkv, cf);
    pet::dropout_rows(rows, merged, g, second);
    pet::attn_bwd_typed(ws, at, qkv_adj, cf_adj, table_adj, rows, qkv, merged, ml, cf);
    if (hipDeviceSynchronize() != hipSuccess) return 5;
    write(dir + "merged.b16", merged.ptr, size_t(T) * D * 2);
    write(dir + "rows.b16", rows.ptr, size_t(T) * D * 2);
    write(dir + "qkv_adj.b16", qkv_adj.ptr, size_t(T) * W * 2);
    write(dir + "ml.f32", ml.data(), size_t(N) * H * S * 8);
    write(dir + "cf_adj.f32", cf_adj.data(), size_t(N) * S * 4);
    write(dir + "table_adj.f32", table_adj.data(), size_t(nb) * H * 4);
  } catch (const std::exception& e) {
    std::fprintf(stderr, "%s\n", e.what());
    return 6;
  }
  return 0;
}
