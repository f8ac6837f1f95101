// beam.cuh — parameter block and launcher of beam search's selection (beam.cu).
#pragma once

#include "common.cuh"

namespace bozo {

constexpr int kMaxBeams = 32;
constexpr int kMaxVocab = 1 << 20;

struct BeamP {
  const void* logits;
  long long stride;
  int dt, N, K, V, eos;
  const float* scores;
  const unsigned char* done;
  float* out_scores;
  long long* out_tokens;
  int* out_rows;
};
cudaError_t launch_beam(const BeamP& p, int sms, cudaStream_t st);

}  // namespace bozo
