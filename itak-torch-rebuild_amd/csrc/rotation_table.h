// The frequencies of a rotation, on the host: how far a position turns every pair of channels.
#pragma once

#include "../../include/itak_hip_kv.h"

#include <algorithm>
#include <cmath>
#include <vector>

namespace itak {

// The defaults of a configuration's zeros.
inline double rotation_amplitude(const itak_rotation_config &c) {
    if (c.amplitude != 0.0) return c.amplitude;
    return c.scaling == ITAK_ROTATION_YARN ? 0.1 * std::log(c.factor) + 1.0 : 1.0;
}

// Radians a position, pair by pair, by the host's libm in 64 bits. YaRN (Peng et al., 2023, "YaRN: Efficient Context Window
// Extension of Large Language Models", section 3.2): pair i turns original * f(i) / (2 pi) times over the trained length; the
// pairs' indices at which that is beta_fast and beta_slow, rounded outwards, are where the ramp begins and ends.
inline std::vector<double> rotation_frequencies(const itak_rotation_config &c) {
    const double r = double(c.rotary_dim), two_pi = 2.0 * M_PI;
    std::vector<double> f(c.rotary_dim / 2);
    for (size_t i = 0; i < f.size(); ++i) f[i] = std::pow(c.base, -2.0 * double(i) / r);
    if (c.scaling == ITAK_ROTATION_LINEAR) {
        for (double &x : f) x /= c.factor;
    } else if (c.scaling == ITAK_ROTATION_YARN) {
        auto index_of = [&](double turns) {
            return r * std::log(c.original_positions / (turns * two_pi)) / (2.0 * std::log(c.base));
        };
        const double low = std::max(std::floor(index_of(c.beta_fast != 0.0 ? c.beta_fast : 32.0)), 0.0);
        const double high = std::min(std::ceil(index_of(c.beta_slow != 0.0 ? c.beta_slow : 1.0)), r - 1.0);
        for (size_t i = 0; i < f.size(); ++i) {
            const double ramp = std::min(std::max((double(i) - low) / std::max(high - low, 0.001), 0.0), 1.0);
            f[i] = f[i] * (1.0 - ramp) + f[i] / c.factor * ramp;
        }
    }
    return f;
}

// What is wrong with a configuration, or null.
inline const char *rotation_refusal(const itak_rotation_config &c) {
    auto finite = [](double x) { return std::isfinite(x); };
    if (!finite(c.base) || !(c.base > 1.0)) return "base must be finite and > 1";
    if (c.rotary_dim < 2 || c.rotary_dim > 256 || c.rotary_dim % 2) return "rotary_dim must be even, from 2 to 256";
    if (c.interleaved > 1) return "interleaved must be 0 or 1";
    if (c.scaling > ITAK_ROTATION_YARN) return "scaling is none of ITAK_ROTATION_*";
    if (c.scaling != ITAK_ROTATION_PLAIN && (!finite(c.factor) || !(c.factor >= 1.0))) return "factor must be finite and >= 1";
    if (!finite(c.amplitude) || c.amplitude < 0.0) return "amplitude must be finite and >= 0";
    if (c.scaling == ITAK_ROTATION_YARN) {
        if (!finite(c.original_positions) || !(c.original_positions > 0.0)) return "original_positions must be finite and > 0";
        if (!finite(c.beta_fast) || !finite(c.beta_slow) || c.beta_fast < 0.0 || c.beta_slow < 0.0) return "betas must be finite and >= 0";
        if (!((c.beta_fast != 0.0 ? c.beta_fast : 32.0) > (c.beta_slow != 0.0 ? c.beta_slow : 1.0)))
            return "beta_fast must be greater than beta_slow";
    }
    return nullptr;
}

}  // namespace itak
