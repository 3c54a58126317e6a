// logits.cuh -- operators on rows of logits (top_logits.cu, distill.cu, sample.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "tambear_gb.h"

namespace tbgb {

constexpr int kTopMax = 1024;                // largest k of the top-logits list and of a teacher's record
constexpr long long kVocabMax = 1ll << 22;   // 2^22 weights of at most 2^30 each sum below 2^53 (exact in f64)

constexpr long long kLogitRowsMax = 1ll << 24;  // rows x CTAs per row stays below the grid's limit

struct LogitsArgs {
  const void* logits;
  int32_t dtype;      // TBGB_F32, TBGB_F16, TBGB_BF16
  long long ld;       // elements from one row to the next
  long long rows;
  int vocab;
};

struct TopArgs {
  LogitsArgs x;
  int k;
  float temperature;
  const uint64_t* mask;
  long long mask_ld;  // words from one row's mask to the next (0: one mask for every row)
  void* values;
  int32_t* ids;
  float* lse;
};

struct DistillArgs {
  LogitsArgs x;
  const int32_t* ids;
  long long ids_ld;
  const void* teacher;
  int32_t teacher_dtype;
  long long teacher_ld;
  int k;
  const float* teacher_lse;
  float temperature;
  const float* weight;
  float* loss;
  float* stats;
  int stats_ld;  // 2 or 6 floats per row
  void* grad;
  long long grad_ld;
  uint32_t* err;
};

struct SampleArgs {
  LogitsArgs x;
  const float* u;
  tbgb_sampling p;
  const uint64_t* mask;
  long long mask_ld;
  int32_t* tokens;
  float* logprobs;
};

cudaError_t top_logits_launch(const TopArgs& a, int num_sms, cudaStream_t s, uint64_t* launches);
// loss and / or gradient; with_loss writes loss and stats, with_grad writes grad (from stats when
// with_loss is false).
cudaError_t distill_launch(const DistillArgs& a, bool with_loss, bool with_grad, int num_sms, cudaStream_t s,
                           uint64_t* launches);
cudaError_t sample_launch(const SampleArgs& a, int num_sms, cudaStream_t s, uint64_t* launches);

}  // namespace tbgb
