// Host tests of the linear-layer operators' planning headers (orth_plan.h, gemm16_plan.h).
#include <cmath>
#include <vector>
#include "mini_test.h"
#include "gemm16_plan.h"
#include "orth_plan.h"

using namespace rtat_native;

namespace {

bool power_of_two(double x) {
  int e;
  return std::frexp(x, &e) == 0.5;
}

// For singular values up to 60 (and no more than the steps before can reach) nothing that is stored
// in f16 passes its range, and all factors are what the formulas make of two powers of two.
void check_steps(const std::vector<float>& coeffs) {
  const int steps = (int)coeffs.size() / 3;
  std::vector<StepFactors> f(steps);
  step_factors(steps, coeffs.data(), f.data());
  double s = 1.0;
  for (int i = 0; i < steps; ++i) {
    const double a = coeffs[3 * i], b = coeffs[3 * i + 1], c = coeffs[3 * i + 2];
    const double ms = (double)f[i].m * 1048576.0, ps = 1.0 / f[i].back;
    CHECK(power_of_two(ms) && power_of_two(ps) && ms <= 1024.0 && ps <= 256.0);
    CHECK(f[i].a == (float)a && f[i].diag == (i < steps - 2 ? 0.0f : (float)(a * ps)));
    CHECK(f[i].p == (float)(c * (ps / (ms * ms))) && f[i].q == (float)(b * (ps / ms)));
    double next = 0.0;
    for (int j = 0; j <= 4000; ++j) {
      const double x = s * j / 4000.0, u = x * x;
      const double p = b * u + c * u * u + (i < steps - 2 ? 0.0 : a);
      CHECK(u * ms <= 65504.0 * 0.95);
      CHECK(std::fabs(p) * ps <= 65504.0 * 0.95);
      const double y = std::fabs(x * (a + b * u + c * u * u));
      if (y > next) next = y;
    }
    s = next < 60.0 ? next : 60.0;
  }
}

}  // namespace

TEST(orth_plan, f16_holds_every_step, false) {
  const std::vector<std::vector<float>> sets = {
      {8, 0, 0, 1.5f, -0.5f, 0},
      {4, 0, 0, 3.4445f, -4.775f, 2.0315f},
      {9, 0, 0, 1, 0, 0},
      {59, 0, 0, 0.01f, 0, 0},
      {55, 0, 0, 3.4445f, -4.775f, 2.0315f},
      {4, 0, 0, 3.4445f, -4.775f, 2.0315f, 3.4445f, -4.775f, 2.0315f, 3.4445f, -4.775f, 2.0315f},
      {8.2872f, -23.5959f, 17.3004f, 4.107f, -2.9478f, 0.5448f, 3.9487f, -2.9089f, 0.5518f, 3.3184f, -2.4885f, 0.5107f},
      {300, 0, 0},
      {1e4f, -3e4f, 2e4f},
      {-2, 3, -1, -50, 7, 0.25f, 0, 0, 0, 1e30f, 0, 0},
      {0, 0, 1e20f, 0, 1e-20f, 0}};
  for (const auto& c : sets) check_steps(c);
}

TEST(orth_plan, usual_coefficients_keep_the_largest_scales, false) {
  std::vector<float> c;
  for (int i = 0; i < 32; ++i) c.insert(c.end(), {3.4445f, -4.775f, 2.0315f});
  for (int i = 0; i < 32; ++i) {
    std::vector<StepFactors> f(i + 1);
    step_factors(i + 1, c.data(), f.data());
    for (const StepFactors& x : f) CHECK(x.m == 1.0f / 1024.0f && x.back == 1.0f / 256.0f);
  }
  const float cubic[6] = {1.5f, -0.5f, 0, 1.5f, -0.5f, 0};
  StepFactors f[2];
  step_factors(2, cubic, f);
  CHECK(f[1].m == 1.0f / 1024.0f && f[1].back == 1.0f / 256.0f);
}

TEST(orth_plan, scales_stay_finite_for_any_coefficients, false) {
  const float inf = INFINITY, nan = NAN, most = 3.4e38f;
  const float sets[][9] = {{nan, 0, 0, 1, 1, 1, 1, 1, 1}, {1, inf, 0, 1, -inf, 1, inf, 1, 1},
                           {most, most, most, -most, most, -most, most, -most, most}, {0, 0, 0, 0, 0, 0, 0, 0, 0}};
  for (const auto& c : sets) {
    StepFactors f[3];
    step_factors(3, c, f);
    for (const StepFactors& x : f) {
      CHECK(power_of_two((double)x.m) && power_of_two((double)x.back));
      CHECK(x.m >= 16.0f / 1048576.0f && x.back >= 1.0f / 256.0f && x.back <= 0x1p120f);
    }
  }
}

// ---- gemm16_plan.h -------------------------------------------------------------------------

TEST(gemm16_plan, choices_that_were_measured, false) {
  const size_t scratch = (size_t)64 << 20;
  struct Case {
    int m, n, k, tile;
    bool cut;
  };
  for (const Case& c : {Case{4096, 2048, 2048, 128, false}, Case{2048, 3584, 4096, 128, false},
                        Case{1024, 1024, 1024, 64, false}, Case{768, 768, 8192, 64, true},
                        Case{8192, 8192, 8192, 256, false}, Case{8192, 8192, 4096, 256, false}}) {
    const Plan16 p = plan16(c.m, c.n, c.k, 1, false, true, scratch, 256);
    CHECK_EQ(p.tri, 0);
    CHECK_EQ(p.slices > 1, c.cut);
    if (!c.cut) CHECK_EQ(p.tile, c.tile);
  }
  // The smaller half of a symmetric product, where its tiles fill the machine.
  CHECK_EQ(plan16(8192, 8192, 8192, 1, true, true, scratch, 256).tri, 1);
}

// What the kernels index by: slices have panels and room, halves only where they are asked for, the
// join's grid within its limit.
TEST(gemm16_plan, whatever_is_chosen_fits, false) {
  const int sizes[] = {1, 7, 16, 63, 64, 65, 129, 333, 512, 1000, 2051, 4099, 8192, 1 << 20, (1 << 30) - 1024};
  for (int m : sizes)
    for (int n : sizes)
      for (int k : {0, 1, 64, 65, 1000, 8192, 1 << 20})
        for (int batch : {1, 6})
          for (int symmetric = 0; symmetric <= (m == n ? 1 : 0); ++symmetric)
            for (int large : {0, 1})
              for (size_t scratch : {(size_t)0, (size_t)1 << 20, (size_t)64 << 20}) {
                const Plan16 p = plan16(m, n, k, batch, symmetric != 0, large != 0, scratch, 256);
                const long panels = ((long)k + PANEL16 - 1) / PANEL16;
                CHECK(p.tile == 64 || p.tile == 128 || (p.tile == 256 && large));
                CHECK(p.tri == 0 || symmetric);
                CHECK(p.slices >= 1 && p.slices <= 64);
                if (p.slices > 1) {
                  CHECK(batch == 1 && panels / p.slices >= SLICE_PANELS16);
                  CHECK((double)p.slices * slice_ld16(m) * n * 4.0 <= (double)scratch);
                  CHECK(p.tri == 0 || p.tile == 128);
                  CHECK(((long)n + 15) / 16 <= 65535);
                }
              }
}

TEST(gemm16_plan, few_columns_of_a_long_k, false) {
  const size_t scratch = (size_t)64 << 20;
  CHECK(few_columns16(8192, 1, 2048, scratch) && few_columns16(2048, 13, 8192, scratch) && few_columns16(1, 1, 8, scratch));
  CHECK(few_columns16(8192, 16, 131072, scratch) && few_columns16(16, 16, 20480, scratch));
  for (int m : {1, 16, 64, 1000, 1024})
    for (int k : {24576, 65536, 1 << 20, 1 << 29}) {
      CHECK(!few_columns16(m, 1, k, scratch) && !few_columns16(m, 16, k, scratch));
      CHECK(plan16(m, 16, k, 1, false, true, scratch, 256).slices >= 32);
      CHECK(few_columns16(m, 1, k, 0));  // nothing to cut into
    }
  CHECK(!few_columns16(2048, 4, 65536, scratch) && few_columns16(2048, 4, 32768, scratch));
  CHECK(!few_columns16(64, 17, 64, scratch) && !few_columns16(64, 1, 65, scratch) && !few_columns16(64, 1, 0, scratch));
  CHECK(!few_columns16((1 << 27) + 1, 1, 8, scratch));
}
