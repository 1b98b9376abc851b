// Losses over the tokens of a language model's logits: log-probabilities, the clipped policy
// loss, the preference loss, and the gradient of the logits.
#pragma once
#include <stdint.h>

#include <cuda_runtime.h>

namespace m3 {

// (batch, positions) operand with element strides (0 where it is broadcast)
template <typename T>
struct Map2 {
  T* p;
  int64_t sb, st;
};

// The rows of the logits and what is known of each: (batch, positions, V), innermost stride 1.
struct TokenRows {
  const void* logits;
  int64_t sb, st;
  int64_t R;           // rows = batch * T
  int T, V;
  Map2<const int64_t> tok;
  Map2<const uint8_t> mask;  // p may be null: every position counts
  int64_t ignore;      // token id of positions that do not count
  double scale;        // 1 / temperature
  float c_hi, c_lo;    // scale * log2(e) in two floats; of the policy loss the nearest one, and next to nothing
};

struct PolicyArgs {
  Map2<const float> old_logp, adv, ref;  // ref.p null: no KL term
  double clip_lo, clip_hi;               // bounds of the ratio
  double kl_coef;
  int by_sequence;                       // mean of the sequences' means
};

// Nonzero once a bounded wait of the policy loss's kernel gave up on this device.
int token_error_word(bool reset, int* out);

// Workspaces of the two losses. They begin with what the gradient needs: stats (R) and the
// coefficients d loss / d logp (by position, or by sequence for the preference loss).
size_t policy_workspace_bytes(int64_t batch, int64_t rows);
size_t preference_workspace_bytes(int64_t batch, int64_t rows);

// logp (R) and, where given, stats (R) = (base, sum over it) of each row
int launch_token_logprobs(const TokenRows& p, int dtype, float* logp, float2* stats, cudaStream_t s);
// loss, mean KL, share of clipped tokens; dlogits where given
int launch_policy_loss(const TokenRows& p, int dtype, const PolicyArgs& a, int64_t batch, float* loss, float* kl,
                       float* clipped, float* logp, void* dlogits, int64_t dsb, int64_t dst, void* ws, cudaStream_t s);
// loss (1), rewards (2 N)
int launch_preference_loss(const TokenRows& p, int dtype, Map2<const float> ref, double beta, double smoothing,
                           int64_t pairs, float* loss, float* rewards, float* logp, void* ws, cudaStream_t s);
// dlogits = up * coef * scale * (one-hot - softmax); keep_if_one: leaves dlogits where *up is 1
int launch_token_grad(const TokenRows& p, int dtype, const float2* stats, Map2<const float> coef, const float* up,
                      bool keep_if_one, void* dlogits, int64_t dsb, int64_t dst, cudaStream_t s);
// stats and coefficients in a loss's workspace
const float2* workspace_stats(const void* ws);
Map2<const float> policy_coef(const void* ws, const TokenRows& p);
Map2<const float> preference_coef(const void* ws, const TokenRows& p);

}  // namespace m3
