// Frequencies of rotary positions, for the operator's tables and the decoder's.
#pragma once

#include <vector>

#include "common.h"

namespace etc {

// Checks the configuration and fills its rotary_dim / 2 angles per position and the factor on the rotated values.
etc_status rope_frequencies(const etc_rope_config& config, const float* divisors, std::vector<double>* inv_freq, double* magnitude);

}  // namespace etc
