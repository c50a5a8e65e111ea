// Factors of the Newton-Schulz steps (orth.hip): which powers of two hold M and P = b M + c M^2 (+ a)
// in f16.  Plain arithmetic without device state, so it also compiles for the host alone.
//
// X is held times 2^10, so singular values s up to 60 fit.  M has entries up to s^2 and P up to the
// largest |b u + c u^2 (+ a)| over 0 <= u <= s^2, for s = 60 3600 and 2.6e7 with the usual quintic:
// no fixed scale suits both those and the values around one that a convergent iteration has.  So s is
// bounded before every step: it is at most 1 before the first, at most max |a x + b x^3 + c x^5| over
// 0 <= x <= s after a step, and never taken above 60.  M and P get the largest power of two that
// this bound leaves room for, up to 2^10 and 2^8, which convergent coefficients keep throughout.
#pragma once
#include <math.h>

namespace rtat_native {

constexpr float X_SCALE = 1024.0f;
constexpr float M_SCALE_MOST = 1024.0f, P_SCALE_MOST = 256.0f;
constexpr double SINGULAR_MOST = 60.0;  // 61440 of f16's 65504

struct StepFactors {
  float a;
  float m;     // M = m * X^T X
  float p, q;  // P = p * M^2 + q * M (+ diag)
  float diag;
  float back;  // X = back * X P (+ a X)
};

// The largest power of two up to `most` that keeps `top` below 60000 of f16's 65504.
inline float room16(double top, float most) {
  if (!(top > 0.0)) return top == top ? most : 1.0f;
  const double want = 60000.0 / top;
  if (want >= (double)most) return most;
  // 2^-120: what passes it has a result that no type here holds.
  return want > 0x1p-120 ? (float)ldexp(1.0, ilogb(want)) : 0x1p-120f;
}

// max |d + b u + c u^2| over 0 <= u <= end.
inline double top_of_square(double d, double b, double c, double end) {
  double top = fabs(d);
  const double last = fabs(d + (b + c * end) * end);
  if (!(last <= top)) top = last;
  const double u = -b / (2.0 * c);
  if (c != 0.0 && u > 0.0 && u < end && fabs(d + 0.5 * b * u) > top) top = fabs(d + 0.5 * b * u);
  return top;
}

// max |a x + b x^3 + c x^5| over 0 <= x <= end.
inline double top_of_step(double a, double b, double c, double end) {
  auto value = [&](double x) { return fabs(x * (a + x * x * (b + c * x * x))); };
  double top = value(end);
  auto at_square = [&](double u) {
    if (u > 0.0 && u < end * end && value(sqrt(u)) > top) top = value(sqrt(u));
  };
  const double root = 9.0 * b * b - 20.0 * a * c;  // a + 3 b u + 5 c u^2 = 0
  if (c != 0.0 && root >= 0.0) {
    at_square((-3.0 * b + sqrt(root)) / (10.0 * c));
    at_square((-3.0 * b - sqrt(root)) / (10.0 * c));
  }
  if (c == 0.0 && b != 0.0) at_square(-a / (3.0 * b));
  return top;
}

// coeffs: (a, b, c) per step.  The last two steps put a on the polynomial's diagonal.
inline void step_factors(int steps, const float* coeffs, StepFactors* out) {
  double s = 1.0;
  for (int i = 0; i < steps; ++i) {
    const float a = coeffs[3 * i], b = coeffs[3 * i + 1], c = coeffs[3 * i + 2];
    const float d = i < steps - 2 ? 0.0f : a;
    const float ms = room16(s * s, M_SCALE_MOST);
    const float ps = room16(top_of_square(d, b, c, s * s), P_SCALE_MOST);
    StepFactors& f = out[i];
    f.a = a;
    f.m = ms / (X_SCALE * X_SCALE);
    f.p = c * (ps / (ms * ms));
    f.q = b * (ps / ms);
    f.diag = d * ps;
    f.back = 1.0f / ps;
    s = 1.02 * top_of_step(a, b, c, s);  // the roundings of a step: some thousandths
    if (!(s < SINGULAR_MOST)) s = SINGULAR_MOST;
  }
}

}  // namespace rtat_native
