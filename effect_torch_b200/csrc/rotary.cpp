// Frequency tables of rotary positions: the rules by which a trained context is extended, and the handle that keeps a table on the
// device. The rules are those that checkpoints are published with: a common divisor ("linear"), one that depends on how many turns
// a pair makes within the trained context ("llama3", "yarn"), and divisors given pair by pair.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

#include "common.h"
#include "kernels.h"
#include "rotary.h"

using namespace etc;

namespace etc {

etc_status rope_frequencies(const etc_rope_config& c, const float* divisors, std::vector<double>* inv_freq, double* magnitude) {
  auto bad = [](const std::string& what) { return fail(ETC_COMPILATION, "rotary: " + what); };
  auto positive = [](double v) { return std::isfinite(v) && v > 0.0; };
  if (c.head_dim <= 0 || c.rotary_dim <= 0 || c.rotary_dim % 2 != 0 || c.rotary_dim > c.head_dim)
    return bad("the rotated part must be an even number of values in 2.." + std::to_string(c.head_dim) + ", got " + std::to_string(c.rotary_dim));
  if (c.head_dim > 65536) return bad("head dimension " + std::to_string(c.head_dim) + " exceeds limit 65536");
  if (c.layout != ETC_ROPE_HALF_SPLIT && c.layout != ETC_ROPE_INTERLEAVED_PAIRS) return bad("unknown layout " + std::to_string(c.layout));
  if (c.scaling < ETC_ROPE_SCALING_NONE || c.scaling > ETC_ROPE_SCALING_YARN) return bad("unknown scaling " + std::to_string(c.scaling));
  if (!positive(c.theta)) return bad("theta must be finite and positive");
  if (!std::isfinite(c.attention_factor) || c.attention_factor < 0.0) return bad("the attention factor must be finite and not negative");
  if (c.scaling != ETC_ROPE_SCALING_NONE && (!std::isfinite(c.factor) || c.factor < 1.0)) return bad("the scaling factor must be finite and at least 1");
  const bool by_turns = c.scaling == ETC_ROPE_SCALING_LLAMA3 || c.scaling == ETC_ROPE_SCALING_YARN;
  if (by_turns && !positive(c.original_context)) return bad("the original context must be finite and positive");
  if (c.scaling == ETC_ROPE_SCALING_LLAMA3 && !(positive(c.low_freq_factor) && positive(c.high_freq_factor) && c.low_freq_factor < c.high_freq_factor))
    return bad("the low frequency factor must be positive and below the high one");
  if (c.scaling == ETC_ROPE_SCALING_YARN && !(positive(c.beta_slow) && positive(c.beta_fast) && c.beta_slow < c.beta_fast))
    return bad("beta slow must be positive and below beta fast");
  if (c.scaling == ETC_ROPE_SCALING_YARN && c.theta <= 1.0) return bad("yarn scaling needs a theta above 1");
  const int pairs = c.rotary_dim / 2;
  const double pi = 3.14159265358979323846;
  if (divisors)
    for (int j = 0; j < pairs; ++j)
      if (!positive(divisors[j])) return bad("frequency divisor " + std::to_string(j) + " must be finite and positive");
  // yarn: the (fractional) pair that makes a given number of turns within the original context, as an index over rotary_dim
  auto pair_of = [&](double turns) { return c.rotary_dim * std::log(c.original_context / (turns * 2.0 * pi)) / (2.0 * std::log(c.theta)); };
  double low = 0.0, high = 0.0;
  if (c.scaling == ETC_ROPE_SCALING_YARN) {
    low = std::max(std::floor(pair_of(c.beta_fast)), 0.0);
    high = std::min(std::ceil(pair_of(c.beta_slow)), (double)c.rotary_dim - 1.0);
  }
  inv_freq->resize((size_t)pairs);
  for (int j = 0; j < pairs; ++j) {
    double f = std::pow(c.theta, -2.0 * (double)j / (double)c.rotary_dim);
    if (divisors) f /= (double)divisors[j];
    if (c.scaling == ETC_ROPE_SCALING_LINEAR) {
      f /= c.factor;
    } else if (c.scaling == ETC_ROPE_SCALING_LLAMA3) {
      const double turns = c.original_context * f / (2.0 * pi);
      const double kept = std::min(1.0, std::max(0.0, (turns - c.low_freq_factor) / (c.high_freq_factor - c.low_freq_factor)));
      f = f * ((1.0 - kept) / c.factor + kept);
    } else if (c.scaling == ETC_ROPE_SCALING_YARN) {
      const double stretched = std::min(1.0, std::max(0.0, ((double)j - low) / std::max(high - low, 0.001)));
      f = f / c.factor * stretched + f * (1.0 - stretched);
    }
    if (!std::isfinite(f)) return bad("the frequency of pair " + std::to_string(j) + " is not finite");
    (*inv_freq)[(size_t)j] = f;
  }
  *magnitude = c.attention_factor > 0.0 ? c.attention_factor : c.scaling == ETC_ROPE_SCALING_YARN ? 0.1 * std::log(c.factor) + 1.0 : 1.0;
  return ETC_OK;
}

}  // namespace etc

struct etc_rotary {
  uint32_t magic = kRotaryMagic;
  etc_runtime* rt = nullptr;
  etc_rope_config config{};
  double* d_half_turns = nullptr;  // [rotary_dim / 2] frequencies / pi
  float magnitude = 1.0f;
};

static bool valid_rotary(const etc_rotary* r) { return r && r->magic == kRotaryMagic; }

extern "C" {

etc_status etc_rope_frequencies(const etc_rope_config* config, const float* h_divisors, double* h_inv_freq, double* out_attention_factor) {
  if (!config || !h_inv_freq) return fail(ETC_INVALID_ARGUMENT, "rotary: config and the frequencies must not be null");
  std::vector<double> f;
  double magnitude = 1.0;
  ETC_TRY(rope_frequencies(*config, h_divisors, &f, &magnitude));
  std::memcpy(h_inv_freq, f.data(), f.size() * sizeof(double));
  if (out_attention_factor) *out_attention_factor = magnitude;
  return ETC_OK;
}

etc_status etc_rotary_create(etc_runtime* rt, const etc_rope_config* config, const float* h_divisors, etc_rotary** out) {
  ETC_TRY(activate(rt));
  if (!config || !out) return fail(ETC_INVALID_ARGUMENT, "rotary: config and out must not be null");
  *out = nullptr;
  std::vector<double> f;
  double magnitude = 1.0;
  ETC_TRY(rope_frequencies(*config, h_divisors, &f, &magnitude));
  for (double& v : f) v /= 3.14159265358979323846;
  void* table = nullptr;
  ETC_TRY(rt->device_alloc(f.size() * sizeof(double), &table));
  cudaError_t e = cudaMemcpyAsync(table, f.data(), f.size() * sizeof(double), cudaMemcpyHostToDevice, rt->stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(rt->stream);
  if (e != cudaSuccess) {
    rt->device_free(table);
    return fail(ETC_TRANSFER, std::string("rotary: table upload failed: ") + cudaGetErrorString(e));
  }
  etc_rotary* r = new etc_rotary();
  r->rt = rt;
  r->config = *config;
  r->d_half_turns = (double*)table;
  r->magnitude = (float)magnitude;
  *out = r;
  return ETC_OK;
}

etc_status etc_rotary_destroy(etc_rotary* rotary) {
  if (!valid_rotary(rotary)) return fail(ETC_INVALID_HANDLE, "rotary: the table handle is invalid or destroyed");
  ETC_TRY(activate(rotary->rt));
  cudaStreamSynchronize(rotary->rt->stream);
  rotary->rt->device_free(rotary->d_half_turns);
  rotary->magic = 0;
  delete rotary;
  return ETC_OK;
}

etc_status etc_rotary_into(etc_runtime* rt, const etc_rotary* rotary, const float* d_x, int64_t x_batch_stride, int64_t x_head_stride,
                           int64_t x_step_stride, const int64_t* d_offsets, int64_t n_offsets, int64_t batch, int64_t heads, int64_t steps,
                           float* d_out, int64_t out_batch_stride, int64_t out_head_stride, int64_t out_step_stride) {
  ETC_TRY(activate(rt));
  if (!valid_rotary(rotary) || rotary->rt != rt) return fail(ETC_INVALID_HANDLE, "rotary: the table belongs to a different runtime");
  if (batch < 0 || heads < 0 || steps < 0) return fail(ETC_INVALID_ARGUMENT, "rotary: negative sizes");
  if (batch == 0 || heads == 0 || steps == 0) return ETC_OK;
  if (heads > (1 << 20) || batch > INT32_MAX || steps > INT32_MAX || batch * steps > INT32_MAX)
    return fail(ETC_INVALID_ARGUMENT, "rotary: more than 2^20 heads or 2^31 - 1 positions in one call");
  if (n_offsets != 1 && n_offsets != batch)
    return fail(ETC_EXECUTION, "rotary embedding: " + std::to_string(n_offsets) + " offsets for batch " + std::to_string(batch));
  if (!d_x || !d_offsets || !d_out) return fail(ETC_INVALID_ARGUMENT, "rotary: x, offsets and out must be device buffers");
  RotaryArgs a;
  const int64_t x_stride[3] = {x_batch_stride, x_head_stride, x_step_stride}, out_stride[3] = {out_batch_stride, out_head_stride, out_step_stride};
  const int64_t extent[3] = {batch, heads, steps};
  a.in_place = d_x == d_out;
  for (int i = 0; i < 3; ++i) {
    // the stride of an axis of one is never used
    a.x_stride[i] = extent[i] > 1 ? x_stride[i] : 0;
    a.out_stride[i] = extent[i] > 1 ? out_stride[i] : 0;
    if (extent[i] == 1) continue;
    if (x_stride[i] < 0 || out_stride[i] < rotary->config.head_dim || std::max(x_stride[i], out_stride[i]) > INT64_MAX / 16 / extent[i])
      return fail(ETC_INVALID_ARGUMENT, "rotary: strides of x must not be negative, those of out at least a head, and addresses within 64 bits");
    if (d_x == d_out && x_stride[i] != out_stride[i])
      return fail(ETC_INVALID_ARGUMENT, "rotary: in place needs equal strides");
  }
  a.x = d_x;
  a.out = d_out;
  a.offsets = d_offsets;
  a.n_offsets = n_offsets;
  a.heads = (int)heads;
  a.steps = (int)steps;
  a.head_dim = rotary->config.head_dim;
  a.rotary_half = rotary->config.rotary_dim / 2;
  a.layout = rotary->config.layout;
  a.half_turns = rotary->d_half_turns;
  a.magnitude = rotary->magnitude;
  ETC_CUDA(launch_rotary(a, batch, rt->sm_count, rt->stream));
  rt->launches++;
  return ETC_OK;
}

}  // extern "C"
