// Drives the embedding, the norm / gate / residual step and the grouped Adam through the C++ mirror against host loops in
// double.  Values of order one, a few dozen roundings of 2^-24 each: 1e-5 covers every comparison here.
// Prints "OK <n checks>" and exits 0, or the first mismatch and exits 1.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "../../sharpnet_b200/host/sharpnet_tensor.hpp"

using namespace SharpNet;

static int g_checks = 0;
#define EXPECT(cond, what)                                                                          \
  do {                                                                                              \
    ++g_checks;                                                                                     \
    if (!(cond)) { std::printf("FAILED line %d: %s\n", __LINE__, what); std::exit(1); }             \
  } while (0)

static std::vector<float> normal(size_t n, unsigned seed) {
  std::mt19937 g(seed);
  std::normal_distribution<float> d(0.0f, 1.0f);
  std::vector<float> v(n);
  for (auto& x : v) x = d(g);
  return v;
}
static double off(const std::vector<float>& got, const std::vector<double>& want) {
  double d = 0;
  for (size_t i = 0; i < got.size(); ++i) d = std::fmax(d, std::fabs(got[i] - want[i]));
  return d;
}

int main() {
  GPUWrapper gpu(0);
  const int V = 11, D = 24, N = 18;
  {  // lookup and gradient; word 0 is padding
    const auto table = normal(V * D, 1), dy = normal(N * D, 2);
    std::vector<float> ids(N);
    for (int i = 0; i < N; ++i) ids[i] = static_cast<float>((i * 7 + i * i) % V);
    GPUTensor x({3, 6}, ids.data(), gpu), W({V, D}, table.data(), gpu), dW({V, D}, table.data(), gpu), y({3, 6, D}, nullptr, gpu),
        g({3, 6, D}, dy.data(), gpu);
    EmbeddingLayer layer(V, D, 2.0f, 0, gpu);
    layer.ForwardPropagation(x, W, y);
    layer.BackwardPropagation(x, g, true, dW);
    std::vector<double> want_y(N * D), want(table.begin(), table.end());
    for (int i = 0; i < N; ++i)
      for (int c = 0; c < D; ++c) {
        const int w = static_cast<int>(ids[i]);
        want_y[i * D + c] = 2.0 * table[w * D + c];
        if (w != 0) want[w * D + c] += 2.0 * dy[i * D + c];
      }
    EXPECT(off(y.ContentAsFloatArray(), want_y) == 0.0, "lookup");
    EXPECT(off(dW.ContentAsFloatArray(), want) < 1e-5, "gradient");
  }
  {  // LayerNorm of x + gate * block, forward and the input gradient by differences of the host's own loss
    const auto x = normal(N * D, 3), b = normal(N * D, 4), gate = normal(D, 5), gamma = normal(D, 6), dy = normal(N * D, 7);
    auto loss = [&](const std::vector<float>& bx, std::vector<double>* yy) {
      double total = 0;
      for (int i = 0; i < N; ++i) {
        double r[64], m = 0, q = 0;
        for (int c = 0; c < D; ++c) { r[c] = static_cast<double>(x[i * D + c]) + static_cast<double>(gate[c]) * bx[i * D + c]; m += r[c] / D; }
        for (int c = 0; c < D; ++c) q += (r[c] - m) * (r[c] - m) / D;
        for (int c = 0; c < D; ++c) {
          const double y = (r[c] - m) / std::sqrt(q + 1e-5) * gamma[c];
          if (yy) (*yy)[i * D + c] = y;
          total += y * dy[i * D + c];
        }
      }
      return total;
    };
    GPUTensor X({N, D}, x.data(), gpu), B({N, D}, b.data(), gpu), G({1, D}, gate.data(), gpu), ga({D}, gamma.data(), gpu), DY({N, D}, dy.data(), gpu);
    GPUTensor R({N, D}, nullptr, gpu), Y({N, D}, nullptr, gpu), DX({N, D}, nullptr, gpu), DB({N, D}, nullptr, gpu), dga({D}, nullptr, gpu), dG({1, D}, nullptr, gpu);
    ResidualNorm layer(D, SNB200_NORM_LAYER, SNB200_NORM_NONE, 1, 1.0f, 1.0f, 1e-5f, gpu);
    const ResidualNorm::Parameters p = {&ga, nullptr, nullptr, nullptr, &G};
    layer.ForwardPropagation(X, &B, p, &R, &Y);
    layer.BackwardPropagation(R, &B, &DY, nullptr, p, {&dga, nullptr, nullptr, nullptr, &dG}, &DX, &DB);
    std::vector<double> want(N * D), grad(N * D);
    loss(b, &want);
    EXPECT(off(Y.ContentAsFloatArray(), want) < 1e-5, "norm");
    std::vector<float> moved = b;
    for (int i = 0; i < 40; ++i) {
      const int k = (i * 37) % (N * D);
      const float up = b[k] + 0.0009765625f, down = b[k] - 0.0009765625f;        // the step that 32 bits hold is what is divided by
      moved[k] = up;
      const double a = loss(moved, nullptr);
      moved[k] = down;
      const double c = loss(moved, nullptr);
      moved[k] = b[k];
      EXPECT(std::fabs(DB.ContentAsFloatArray()[k] - (a - c) / (static_cast<double>(up) - down)) < 1e-4, "gradient of the block");
    }
    std::vector<double> dgamma(D, 0.0);
    for (int i = 0; i < N; ++i)
      for (int c = 0; c < D; ++c) dgamma[c] += dy[i * D + c] * want[i * D + c] / gamma[c];
    EXPECT(off(dga.ContentAsFloatArray(), dgamma) < 1e-4, "gradient of gamma");   // 18 terms, a quotient by gamma among them
  }
  for (int bits : {32, 8}) {  // the first step moves every weight by the learning rate against its gradient's sign
    const auto w = normal(1000, 8), g = normal(1000, 9), w2 = normal(5, 10), g2 = normal(5, 11);
    GPUTensor W({1000}, w.data(), gpu), dW({1000}, g.data(), gpu), W2({5}, w2.data(), gpu), dW2({5}, g2.data(), gpu);
    AdamGroup group({{&W, &dW, 1.0}, {&W2, &dW2, 0.0}}, 0.9, 0.999, 1e-12, 0.1, bits, gpu);
    group.UpdateWeights(0.01, 0.01);
    std::vector<double> want(1000), want2(5);
    for (int i = 0; i < 1000; ++i) want[i] = w[i] - (0.01 * (g[i] > 0 ? 1 : -1) + 0.1 * w[i]);
    for (int i = 0; i < 5; ++i) want2[i] = w2[i] - 0.01 * (g2[i] > 0 ? 1 : -1);
    EXPECT(off(W.ContentAsFloatArray(), want) < 1e-5, "weights");
    EXPECT(off(W2.ContentAsFloatArray(), want2) < 1e-5, "weights without decay");
    bool threw = false;
    AdamGroup twice({{&W, &dW, 1.0}, {&W, &dW, 1.0}}, 0.9, 0.999, 1e-8, 0.1, bits, gpu);
    try { twice.UpdateWeights(0.01, 0.01); } catch (const std::runtime_error&) { threw = true; }
    EXPECT(threw, "the same tensor twice is refused");
  }
  std::printf("OK %d checks\n", g_checks);
  return 0;
}
