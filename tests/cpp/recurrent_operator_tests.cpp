// Tests of the gated recurrence, the residual norm and the AdamW step through the C++ host
// layer: values that are exact, and what the layer refuses.
//
//   recurrent_operator_tests            all tests (needs a GPU)
//   recurrent_operator_tests --host     only the tests that touch no device
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

// Values that are exact: decays of 1/2 (a gate of 0), and powers of two.
static void RecurrenceTests(Accelerator& accl) {
  auto stream = accl.CreateStream();
  const int rows = 7, channels = 3;
  auto gate = accl.Allocate1D<float>(rows * channels), x = accl.Allocate1D<float>(rows * channels);
  auto out = accl.Allocate1D<float>(rows * channels), gx = accl.Allocate1D<float>(rows * channels);
  auto first = accl.Allocate1D<float>(2 * channels), last = accl.Allocate1D<float>(2 * channels);
  auto offsets = accl.Allocate1D<int32_t>(3);
  gate->CopyFromCPU(*stream, std::vector<float>(rows * channels, 0.0f));
  x->CopyFromCPU(*stream, std::vector<float>(rows * channels, 1.0f));
  first->CopyFromCPU(*stream, std::vector<float>(2 * channels, 4.0f));
  offsets->CopyFromCPU(*stream, {0, 3, 7});
  const auto matrix = [&](auto& buffer, int r) { return MatrixView<float>(buffer->View(), r, channels); };
  const PackedSequences<int32_t> two{2, offsets->View()};
  const int64_t ints = ComputeGatedRecurrenceTempStorageSize(accl, rows, channels);
  CHECK(ints == 0);
  GatedRecurrence(accl, *stream, matrix(gate, rows), matrix(x, rows), matrix(out, rows), two,
                  DecayKind::Sigmoid, false, matrix(first, 2), matrix(last, 2), ArrayView<int32_t>());
  GatedRecurrenceGradient(accl, *stream, matrix(x, rows), matrix(gate, rows), matrix(x, rows),
                          matrix(out, rows), two, DecayKind::Sigmoid, false, matrix(first, 2),
                          MatrixView<float>(), MatrixView<float>(), matrix(gx, rows),
                          matrix(first, 2), ArrayView<int32_t>());
  stream->Synchronize();
  const auto h = out->GetAsArray1D(), ends = last->GetAsArray1D(), back = gx->GetAsArray1D();
  const float states[] = {3.0f, 2.5f, 2.25f, 3.0f, 2.5f, 2.25f, 2.125f};
  const float reach[] = {1.75f, 1.5f, 1.0f, 1.875f, 1.75f, 1.5f, 1.0f};
  for (int i = 0; i < rows * channels; ++i)
    CHECK(h[(size_t)i] == states[i / channels] && back[(size_t)i] == reach[i / channels]);
  for (int c = 0; c < channels; ++c)
    CHECK(ends[(size_t)c] == 2.25f && ends[(size_t)(channels + c)] == 2.125f);
  CHECK(first->GetAsArray1D()[0] == 0.875f && first->GetAsArray1D()[channels] == 0.9375f);
  EXPECT_THROW(GatedRecurrence(accl, *stream, matrix(gate, rows), matrix(x, rows), matrix(out, rows),
                               PackedSequences<int32_t>{3, offsets->View()}, DecayKind::Sigmoid,
                               false, MatrixView<float>(), MatrixView<float>(), ArrayView<int32_t>()),
               ArgumentOutOfRangeException);
  EXPECT_THROW(GatedRecurrence(accl, *stream, matrix(gate, rows), matrix(x, rows), matrix(out, rows),
                               PackedSequences<int32_t>{2}, DecayKind::Sigmoid, false,
                               MatrixView<float>(), MatrixView<float>(), ArrayView<int32_t>()),
               ArgumentOutOfRangeException);  // 7 rows are no two equal parts
}

static void ResidualNormTests(Accelerator& accl) {
  auto stream = accl.CreateStream();
  // Rows of +-2 and a residual of +-2: the total is +-4 with a scale of 1 and no norm behind the
  // block, its root mean square 4.
  const int rows = 3, columns = 70;
  std::vector<float> x, w(columns, 3.0f);
  for (int i = 0; i < rows * columns; ++i) x.push_back(i % 2 ? -2.0f : 2.0f);
  auto dx = accl.Allocate1D<float>(rows * columns), total = accl.Allocate1D<float>(rows * columns);
  auto out = accl.Allocate1D<float>(rows * columns), dw = accl.Allocate1D<float>(columns);
  auto rstd = accl.Allocate1D<float>(rows), gw = accl.Allocate1D<float>(columns);
  auto gr = accl.Allocate1D<float>(rows * columns);
  dx->CopyFromCPU(*stream, x);
  dw->CopyFromCPU(*stream, w);
  const auto matrix = [&](auto& buffer) { return MatrixView<float>(buffer->View(), rows, columns); };
  BlockOutput<float, float> block;
  ResidualNorm(accl, *stream, matrix(dx), block, matrix(dx), matrix(total), matrix(out), dw->View(),
               0.0f, ArrayView<float>(), rstd->View());
  auto temp = accl.Allocate1D<int32_t>(ComputeResidualNormGradientTempStorageSize(accl, rows, columns));
  ResidualNormGradients<float, float, float> gradients;
  gradients.Residual = matrix(gr);
  gradients.Weight = gw->View();
  // (a gradient along the row: none is left of it)
  ResidualNormGradient(accl, *stream, matrix(total), MatrixView<float>(), matrix(dx), block,
                       ArrayView<float>(), matrix(total), ArrayView<float>(), rstd->View(), gradients,
                       temp->View());
  stream->Synchronize();
  const auto t = total->GetAsArray1D(), y = out->GetAsArray1D(), d = gr->GetAsArray1D();
  const auto sums = gw->GetAsArray1D();
  for (int i = 0; i < rows * columns; ++i)
    CHECK(t[(size_t)i] == 2 * x[(size_t)i] && y[(size_t)i] == 1.5f * x[(size_t)i] && d[(size_t)i] == 0.0f);
  for (int c = 0; c < columns; ++c) CHECK(sums[(size_t)c] == 4.0f * rows);
  block.Normalized = true;
  EXPECT_THROW(ResidualNormGradient(accl, *stream, matrix(total), MatrixView<float>(), matrix(dx), block,
                                    ArrayView<float>(), matrix(total), ArrayView<float>(), rstd->View(),
                                    gradients, temp->View()),
               ArgumentNullException);  // no inputRstd
  block.Weight = dw->View().SubView(1);
  EXPECT_THROW(ResidualNorm(accl, *stream, matrix(dx), block, matrix(dx), matrix(total), matrix(out),
                            dw->View(), 0.0f),
               ArgumentOutOfRangeException);
}

static void AdamWTests(Accelerator& accl) {
  auto stream = accl.CreateStream();
  auto p = accl.Allocate1D<float>(300), g = accl.Allocate1D<float>(300), c = accl.Allocate1D<float>(300);
  auto m = accl.Allocate1D<uint8_t>(300), v = accl.Allocate1D<uint8_t>(300);
  auto ms = accl.Allocate1D<float>(2), vs = accl.Allocate1D<float>(2);
  auto step = accl.Allocate1D<int64_t>(1);
  p->CopyFromCPU(*stream, std::vector<float>(300, 1.0f));
  g->CopyFromCPU(*stream, std::vector<float>(300, -0.5f));
  m->CopyFromCPU(*stream, std::vector<uint8_t>(300, 0));
  v->CopyFromCPU(*stream, std::vector<uint8_t>(300, 0));
  ms->CopyFromCPU(*stream, {0.0f, 0.0f});
  vs->CopyFromCPU(*stream, {0.0f, 0.0f});
  step->CopyFromCPU(*stream, {1});
  TensorList parameters, gradients, copies, targets;
  Moments first, second;
  parameters.Add(p->View());
  gradients.Add(g->View());
  copies.Add(c->View());
  targets.Add(g->View());
  first.Values.Add(m->View());
  first.Scales.Add(ms->View());
  second.Values.Add(v->View());
  second.Scales.Add(vs->View());
  AdamWOptions options;
  options.Rate = 0.25;
  options.Beta1 = options.Beta2 = 0.5;
  AdamW(accl, *stream, parameters, gradients, first, second, options, step->View(), copies);
  AdamWMoments(accl, *stream, first, targets, second, copies);
  stream->Synchronize();
  // the first step goes the rate against the gradient's sign; all values are their blocks' largest
  const auto moved = p->GetAsArray1D(), m1 = g->GetAsArray1D(), m2 = c->GetAsArray1D();
  for (size_t i = 0; i < 300; ++i)
    CHECK(std::fabs(moved[i] - 1.25f) < 1e-6f && std::fabs(m1[i] + 0.25f) < 1e-6f &&
          std::fabs(m2[i] - 0.125f) < 1e-6f);
  CHECK(m->GetAsArray1D()[0] == 1 && v->GetAsArray1D()[299] == 255);
  EXPECT_THROW(AdamW(accl, *stream, parameters, gradients, first, second, options, ArrayView<int64_t>()),
               ArgumentNullException);
  EXPECT_THROW(AdamW(accl, *stream, parameters, TensorList(), first, second, options, step->View()),
               ArgumentOutOfRangeException);
  options.Beta1 = 1.0;
  EXPECT_THROW(AdamW(accl, *stream, parameters, gradients, first, second, options, step->View()),
               ArgumentOutOfRangeException);
}

// Calls with nothing to do, and calls that are refused, touch no device.
static void HostTests() {
  CHECK(ilgpu_hip_gated_recurrence_temp_bytes(1, 0, nullptr) == ILGPU_HIP_ERROR_NULL_VIEW);
  int64_t bytes = -1;
  CHECK(ilgpu_hip_gated_recurrence_temp_bytes(1, 64, &bytes) == ILGPU_HIP_SUCCESS && bytes == 0);
  CHECK(ilgpu_hip_residual_norm_gradient_temp_bytes(0, 0, &bytes) == ILGPU_HIP_ERROR_OUT_OF_RANGE);
  CHECK((int32_t)DecayKind::Exponential == 1 && (int32_t)GateKind::Silu == 1);
}

int main(int argc, char** argv) {
  HostTests();
  if (argc < 2 || std::strcmp(argv[1], "--host") != 0) {
    Accelerator accl(0);
    RecurrenceTests(accl);
    ResidualNormTests(accl);
    AdamWTests(accl);
  }
  std::printf("%d failed checks\n", g_failed);
  return g_failed == 0 ? 0 : 1;
}
