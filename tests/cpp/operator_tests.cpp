// Tests of the operators of language models through the C++ host layer: values that
// are exact in every type, and what the layer refuses.
//
//   operator_tests            all tests (needs a GPU)
//   operator_tests --host     only the tests that touch no device
#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "../../ilgpu_amd/host/ilgpu_hip_algorithms.hpp"

using namespace ilgpu;
using namespace ilgpu::Algorithms;

static int g_failed = 0;
#define CHECK(cond)                                                   \
  do {                                                                \
    if (!(cond)) {                                                    \
      std::printf("  FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      ++g_failed;                                                     \
    }                                                                 \
  } while (0)
#define EXPECT_THROW(stmt, Ex)                                               \
  do {                                                                       \
    bool caught = false;                                                     \
    try { stmt; } catch (const Ex&) { caught = true; } catch (...) {}        \
    if (!caught) {                                                           \
      std::printf("  FAILED %s:%d: expected %s\n", __FILE__, __LINE__, #Ex); \
      ++g_failed;                                                            \
    }                                                                        \
  } while (0)

static void ViewTests() {
  float data[20] = {};
  EXPECT_THROW(MatrixView<float>(ArrayView<float>(data, 15), 4, 4), ArgumentOutOfRangeException);
  EXPECT_THROW(MatrixView<float>(ArrayView<float>(data, 18), 4, 4, 5), ArgumentOutOfRangeException);
  EXPECT_THROW(MatrixView<float>(ArrayView<float>(data, 18), -1, 4), ArgumentOutOfRangeException);
  const MatrixView<float> m(ArrayView<float>(data, 19), 4, 4, 5);
  CHECK(m.Rows() == 4 && m.Columns() == 4 && m.RowStride() == 5);
  const MatrixView<float> one(ArrayView<float>(data, 4), 100, 4, 0);
  CHECK(one.Rows() == 100);
}

static uint16_t Bits(float v) {
  uint32_t u;
  std::memcpy(&u, &v, 4);
  return (uint16_t)(u >> 16);
}

static void EmbeddingTests(Accelerator& accl) {
  auto stream = accl.CreateStream();
  const int vocabulary = 5, dimension = 3;
  std::vector<BFloat16> table;
  for (int i = 0; i < vocabulary * dimension; ++i) table.push_back({Bits((float)i)});
  const std::vector<int64_t> tokens = {4, 0, -1, 4, 5, 2};
  auto t = accl.Allocate1D<BFloat16>(vocabulary * dimension);
  auto k = accl.Allocate1D<int64_t>(6);
  auto out = accl.Allocate1D<float>(6 * dimension);
  t->CopyFromCPU(*stream, table);
  k->CopyFromCPU(*stream, tokens);
  MatrixView<BFloat16> tv(t->View(), vocabulary, dimension);
  MatrixView<float> ov(out->View(), 6, dimension);
  Embedding(accl, *stream, tv, k->View(), ov, 0.5f);
  stream->Synchronize();
  const auto got = out->GetAsArray1D();
  for (int i = 0; i < 6; ++i)
    for (int c = 0; c < dimension; ++c) {
      const int64_t token = tokens[(size_t)i];
      const float expect = token >= 0 && token < vocabulary ? 0.5f * (float)(token * dimension + c) : 0.0f;
      CHECK(got[(size_t)(i * dimension + c)] == expect);
    }
  // the gradient of that output, added to ones
  auto grad = accl.Allocate1D<float>(vocabulary * dimension);
  grad->CopyFromCPU(*stream, std::vector<float>(vocabulary * dimension, 1.0f));
  auto temp = accl.Allocate1D<int32_t>(
      ComputeEmbeddingGradientTempStorageSize(accl, 6, vocabulary, dimension));
  MatrixView<float> gv(grad->View(), vocabulary, dimension);
  EmbeddingGradient(accl, *stream, ov, k->View(), gv, temp->View(), 2.0f, 2, true);
  stream->Synchronize();
  const auto sums = grad->GetAsArray1D();
  for (int v = 0; v < vocabulary; ++v)
    for (int c = 0; c < dimension; ++c) {
      const float times = v == 4 ? 2.0f : v == 0 ? 1.0f : 0.0f;  // 2 is the padding token
      CHECK(sums[(size_t)(v * dimension + c)] == 1.0f + times * (float)(v * dimension + c));
    }
  EXPECT_THROW(Embedding(accl, *stream, tv, k->View(), MatrixView<float>(out->View(), 5, dimension)),
               ArgumentOutOfRangeException);
  EXPECT_THROW(EmbeddingGradient(accl, *stream, ov, k->View(), gv, ArrayView<int32_t>()),
               ArgumentNullException);
  EXPECT_THROW(EmbeddingGradient(accl, *stream, ov, k->View(), gv, temp->View().SubView(0, 4)),
               ArgumentOutOfRangeException);
  auto wrong = accl.Allocate1D<uint32_t>(6);
  EXPECT_THROW(Embedding(accl, *stream, tv, wrong->View(), ov), NotSupportedException);
}

static void LayerNormTests(Accelerator& accl) {
  auto stream = accl.CreateStream();
  // Rows of a and -a: mean 0, deviation a with epsilon 0, so the normalised row is +-1.
  const int rows = 7, columns = 130;
  std::vector<float> x, w, b, dy;
  for (int r = 0; r < rows; ++r)
    for (int c = 0; c < columns; ++c) x.push_back((c % 2 ? -1.0f : 1.0f) * (float)(1 << r));
  for (int c = 0; c < columns; ++c) {
    w.push_back((float)(c % 5));
    b.push_back((float)c);
  }
  dy.assign(x.size(), 1.0f);
  auto dx = accl.Allocate1D<float>(rows * columns), dg = accl.Allocate1D<float>(rows * columns);
  auto dw = accl.Allocate1D<float>(columns), db = accl.Allocate1D<float>(columns);
  auto dout = accl.Allocate1D<float>(rows * columns);
  auto mean = accl.Allocate1D<float>(rows), rstd = accl.Allocate1D<float>(rows);
  auto gw = accl.Allocate1D<float>(columns), gb = accl.Allocate1D<float>(columns);
  dx->CopyFromCPU(*stream, x);
  dw->CopyFromCPU(*stream, w);
  db->CopyFromCPU(*stream, b);
  MatrixView<float> xv(dx->View(), rows, columns), ov(dout->View(), rows, columns);
  LayerNorm(accl, *stream, xv, ov, dw->View(), db->View(), 0.0f, mean->View(), rstd->View());
  dg->CopyFromCPU(*stream, dy);
  auto temp = accl.Allocate1D<int32_t>(
      ComputeLayerNormGradientTempStorageSize(accl, rows, columns));
  LayerNormGradient(accl, *stream, MatrixView<float>(dg->View(), rows, columns), xv,
                    ArrayView<float>(), mean->View(), rstd->View(), MatrixView<float>(),
                    gw->View(), gb->View(), temp->View());
  stream->Synchronize();
  const auto y = dout->GetAsArray1D();
  const auto m = mean->GetAsArray1D(), s = rstd->GetAsArray1D();
  const auto sums = gw->GetAsArray1D(), ones = gb->GetAsArray1D();
  for (int r = 0; r < rows; ++r) {
    CHECK(m[(size_t)r] == 0.0f && s[(size_t)r] == 1.0f / (float)(1 << r));
    for (int c = 0; c < columns; ++c)
      CHECK(y[(size_t)(r * columns + c)] == (c % 2 ? -1.0f : 1.0f) * w[(size_t)c] + b[(size_t)c]);
  }
  for (int c = 0; c < columns; ++c)
    CHECK(sums[(size_t)c] == (c % 2 ? -7.0f : 7.0f) && ones[(size_t)c] == 7.0f);
  EXPECT_THROW(LayerNorm(accl, *stream, xv, ov, dw->View().SubView(1), db->View(), 0.0f),
               ArgumentOutOfRangeException);
  EXPECT_THROW(LayerNorm(accl, *stream, xv, ov, dw->View(), db->View(), -1.0f),
               ArgumentOutOfRangeException);
  EXPECT_THROW(LayerNorm(accl, *stream, xv, ov, ArrayView<Half>(), ArrayView<Half>(), 0.0f),
               NotSupportedException);
}

static void ClipTests(Accelerator& accl) {
  auto stream = accl.CreateStream();
  auto a = accl.Allocate1D<float>(4), norm = accl.Allocate1D<float>(1);
  auto h = accl.Allocate1D<Half>(3);
  a->CopyFromCPU(*stream, {3.0f, 0.0f, 0.0f, 12.0f});
  h->CopyFromCPU(*stream, {{0x4400}, {0}, {0}});   // 4
  TensorList list;
  list.Add(a->View());
  list.Add(h->View());
  auto temp = accl.Allocate1D<int32_t>(ComputeGradientNormTempStorageSize(accl, list.Count()));
  GradientNorm(accl, *stream, list, norm->View(), temp->View());
  ClipGradients(accl, *stream, list, norm->View(), 6.5f);
  stream->Synchronize();
  CHECK(norm->GetAsArray1D()[0] == 13.0f);
  const auto scaled = a->GetAsArray1D();
  CHECK(scaled[0] == 1.5f && scaled[1] == 0.0f && scaled[3] == 6.0f);
  CHECK(h->GetAsArray1D()[0].bits == 0x4000);
  EXPECT_THROW(ClipGradients(accl, *stream, list, norm->View(), -1.0f), ArgumentOutOfRangeException);
  EXPECT_THROW(ClipGradients(accl, *stream, list, TensorList(), norm->View(), 1.0f),
               ArgumentOutOfRangeException);
  EXPECT_THROW(GradientNorm(accl, *stream, list, ArrayView<float>(), temp->View()),
               ArgumentNullException);
  auto ints = accl.Allocate1D<int32_t>(3);
  list.Add(ints->View());
  EXPECT_THROW(GradientNorm(accl, *stream, list, norm->View(), temp->View()), NotSupportedException);
}

int main(int argc, char** argv) {
  ViewTests();
  if (argc < 2 || std::strcmp(argv[1], "--host") != 0) {
    Accelerator accl(0);
    EmbeddingTests(accl);
    LayerNormTests(accl);
    ClipTests(accl);
  }
  std::printf("%d failed checks\n", g_failed);
  return g_failed == 0 ? 0 : 1;
}
