// A training step of one attention block and one dense layer through the C++
// interface (include/pet/train.hpp), for tests/test_gpu_cpp_train.py:
//
//   train_test DIR N T S H HD
//
// reads DIR/{tokens,nw,nb,w_in,b_in,w_out,b_out,cf,g}.f32 and DIR/off.i32; runs
// attention_layer, attention_layer_grads (every parameter), linear_grads of a
// dense layer with the tokens as its input and g as its output's adjoint,
// norm_rows_grads of the same rows, then clip_grads (max_norm 1) over all
// gradients; writes DIR/{tokens_adj,grads,norm}.f32. A call with a wrong shape has
// to throw.
#include <cstdio>
#include <cstdlib>
#include <string>
#include <vector>

#include "pet/train.hpp"

template <class T>
static std::vector<T> read(const std::string& path, size_t n) {
  std::vector<T> v(n);
  FILE* f = std::fopen(path.c_str(), "rb");
  if (!f || std::fread(v.data(), sizeof(T), n, f) != n) {
    std::fprintf(stderr, "cannot read %s\n", path.c_str());
    std::exit(2);
  }
  std::fclose(f);
  return v;
}
static void write(const std::string& path, const float* dev, size_t n) {
  std::vector<float> v(n);
  if (hipMemcpy(v.data(), dev, 4 * n, hipMemcpyDeviceToHost) != hipSuccess) std::exit(4);
  FILE* f = std::fopen(path.c_str(), "wb");
  if (!f || std::fwrite(v.data(), 4, n, f) != n) std::exit(3);
  std::fclose(f);
}
template <class T>
static T* upload(const std::vector<T>& v) {
  void* p = nullptr;
  if (hipMalloc(&p, v.size() * sizeof(T)) != hipSuccess) std::exit(4);
  if (hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) std::exit(4);
  return static_cast<T*>(p);
}

int main(int argc, char** argv) {
  if (argc != 7) return 1;
  const std::string dir = std::string(argv[1]) + "/";
  const int N = std::atoi(argv[2]), T = std::atoi(argv[3]), S = std::atoi(argv[4]), H = std::atoi(argv[5]),
            hd = std::atoi(argv[6]), D = H * hd;
  auto f32 = [&](const char* name, size_t n) { return upload(read<float>(dir + name + ".f32", n)); };
  auto zeros = [&](size_t n) { return upload(std::vector<float>(n, 0.f)); };
  try {
    pet::Workspace ws;
    pet::View2D tokens(f32("tokens", size_t(T) * D), T, D), g(f32("g", size_t(T) * D), T, D),
        cf(f32("cf", size_t(N) * S), N, S), out(zeros(size_t(T) * D), T, D), tadj(zeros(size_t(T) * D), T, D),
        csa(zeros(size_t(N) * S), N, S);
    const pet::View1D nw{f32("nw", D), D}, nb{f32("nb", D), D}, b_in{f32("b_in", 3 * D), 3 * D}, b_out{f32("b_out", D), D};
    const pet::WeightRef w_in(pet::View2D(f32("w_in", size_t(3) * D * D), 3 * D, D)),
        w_out(pet::View2D(f32("w_out", size_t(D) * D), D, D));
    const pet::Tokens tk{upload(read<int>(dir + "off.i32", N + 1)), N, false};
    pet::attention_layer(ws, "l", out, tokens, nw, nb, w_in, b_in, cf, w_out, b_out, tk, S, H, hd, 1.0);
    // every gradient in one buffer: the layer's, the dense layer's, the norm's
    const size_t sizes[] = {size_t(D), size_t(D), size_t(3) * D * D, size_t(3) * D, size_t(D) * D, size_t(D),
                            size_t(D) * D, size_t(D), size_t(D), size_t(D)};
    size_t total = 0;
    for (size_t n : sizes) total += n;
    float* all = zeros(total);
    std::vector<float*> at;
    std::vector<pet_grad_tensor> list;
    float* p = all;
    for (size_t n : sizes) at.push_back(p), list.push_back(pet::gradient(p, int64_t(n))), p += n;
    pet::attention_layer_grads(ws, "l", {at[0], at[1], at[2], at[3], at[4], at[5], 0.f}, tadj, csa, g, tokens, nw, nb,
                               w_in, b_in, cf, w_out, tk, S, H, hd, 1.0);
    const pet::View2D w_adj(at[6], D, D);
    pet::linear_grads(ws, g, tokens, w_adj, {at[7], D});
    pet::norm_rows_grads(ws, pet::Rows(), {at[8], D}, {at[9], D}, g, tokens, nw, true);
    list[6] = pet::gradient(w_adj);
    float* norm = zeros(1);
    pet::clip_grads(ws, list, 1.0, norm);
    bool threw = false;
    try {
      pet::linear_grads(ws, g, tokens, pet::View2D(at[6], D, D - 1), pet::View1D());
    } catch (const std::runtime_error&) {
      threw = true;
    }
    if (!threw || hipDeviceSynchronize() != hipSuccess) return 5;
    write(dir + "tokens_adj.f32", tadj.data(), size_t(T) * D);
    write(dir + "grads.f32", all, total);
    write(dir + "norm.f32", norm, 1);
  } catch (const std::exception& e) {
    std::fprintf(stderr, "%s\n", e.what());
    return 6;
  }
  return 0;
}
