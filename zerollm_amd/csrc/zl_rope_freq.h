// Angles of rotary positions, host side: one place for the models' tables and for zl_rope_create.
#pragma once
#include <math.h>

#include <algorithm>
#include <vector>

#include "zl_common.h"

namespace zl {

// Radians per position of each of the n_rot / 2 pairs, and the factor of cos and sin. YaRN keeps the angles of pairs that
// turn often within the trained context (their period is well known to the model) and stretches those that never come
// round; pair i turns b times within orig_ctx positions at i = n_rot ln(orig_ctx / (2 pi b)) / (2 ln base). The ramp's ends
// are whole pairs, rounded outwards, as models fine-tuned with these settings have them.
inline void rope_angles(const zl_rope_opts &o, std::vector<double> *theta, double *gain) {
  ZL_REQUIRE(o.n_rot >= 2 && o.n_rot % 2 == 0 && o.n_rot <= 256, ZL_ERR_ARG, "rope: n_rot must be even, 2 to 256 (got " + std::to_string(o.n_rot) + ")");
  ZL_REQUIRE(o.base > 0.0 && o.base < INFINITY, ZL_ERR_ARG, "rope: the base must be positive");
  ZL_REQUIRE(o.scaling >= 0 && o.scaling <= 2, ZL_ERR_UNSUPPORTED, "rope: scaling must be 0 (none), 1 (linear) or 2 (YaRN)");
  ZL_REQUIRE(o.scaling == 0 || (o.factor >= 1.0 && o.factor < INFINITY), ZL_ERR_ARG, "rope: the scaling factor must be at least 1");
  double low = 0.0, high = 1.0;
  *gain = 1.0;
  if (o.scaling == 2) {
    const double fast = o.beta_fast != 0.0 ? o.beta_fast : 32.0, slow = o.beta_slow != 0.0 ? o.beta_slow : 1.0;
    ZL_REQUIRE(o.orig_ctx >= 1, ZL_ERR_ARG, "rope: YaRN needs the trained context");
    ZL_REQUIRE(o.base > 1.0, ZL_ERR_ARG, "rope: YaRN needs a base above 1");
    ZL_REQUIRE(fast > 0.0 && slow > 0.0 && fast >= slow && fast < INFINITY, ZL_ERR_ARG, "rope: beta_fast must be at least beta_slow, both positive");
    ZL_REQUIRE(o.attn_factor >= 0.0 && o.attn_factor < INFINITY, ZL_ERR_ARG, "rope: the attention factor must not be negative");
    auto pair_of = [&](double b) { return o.n_rot * log(o.orig_ctx / (2.0 * M_PI * b)) / (2.0 * log(o.base)); };
    low = std::max(floor(pair_of(fast)), 0.0);
    high = std::min(ceil(pair_of(slow)), o.n_rot - 1.0);
    *gain = o.attn_factor > 0.0 ? o.attn_factor : 0.1 * log(o.factor) + 1.0;
  }
  theta->resize(o.n_rot / 2);
  for (int i = 0; i < o.n_rot / 2; i++) {
    double th = pow(o.base, -2.0 * i / o.n_rot);
    if (o.freq_factors) {
      ZL_REQUIRE(o.freq_factors[i] > 0.0f && o.freq_factors[i] < INFINITY, ZL_ERR_ARG, "rope: frequency factors must be positive");
      th /= (double)o.freq_factors[i];
    }
    const double ramp = o.scaling == 2 ? std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001))) : 1.0;
    if (o.scaling) th = th * (1.0 - ramp) + th / o.factor * ramp;
    (*theta)[i] = th;
  }
}

}  // namespace zl
