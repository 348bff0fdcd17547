// q4_logits.cuh -- arguments of the logits kernel.
#pragma once
#include <cstdint>

namespace aria_q4 {

struct LogitArgs {
  int M, V;
  const void* logits;         // element strides throughout
  long long logits_row;
  void* out;                  // may be the logits
  long long out_row;
  const int* history;         // [M][history_cap] tokens, oldest first; may be null
  long long history_row;
  int history_cap;
  const int* history_lens;    // [M]
  const int* prompt_lens;     // [M]; null: all of it was generated
  const float* repetition;    // [M] each; null: 1, 0, 0
  const float* frequency;
  const float* presence;
  const int* bias_tokens;     // [M][biases], entries outside [0, V) are unused; may be null
  const float* bias_values;
  long long bias_row;
  int biases;
  const uint32_t* allowed;    // [M][ceil(V / 32)], bit v % 32 of word v / 32; row stride 0 = shared
  long long allowed_row;
  int* token;                 // [M]; may be null
  unsigned long long* best;   // workspace, zero between calls
  unsigned* arrived;
};

}  // namespace aria_q4
