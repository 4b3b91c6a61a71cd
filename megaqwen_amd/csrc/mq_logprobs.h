// Log probabilities of given tokens (logprobs.hip): host launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#define MQ_TOP_MAX 32     // most alternatives a row may ask for

// For every row of logits (type as MQ_DTYPE_*, rows `stride` elements apart): the log probability
// of its token, the entropy (nats) and the top_k most likely tokens with their log probabilities.
struct MqLogprobArgs {
  const void* logits;
  const void* tokens;       // int32, or int64 if tok64
  float* logprob;
  float* entropy;
  float* top_lp;            // [rows, top_k], or null with top_k = 0
  int* top_tok;
  long long stride;
  int rows, vocab, top_k, type;
  bool tok64;
};
size_t mq_logprobs_workspace(int rows, int vocab, int top_k);
// Returns 0, or -1 if the launch failed.
int mq_launch_token_logprobs(const MqLogprobArgs& a, void* ws, hipStream_t stream);
