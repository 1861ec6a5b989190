// What the sessions (api.cu) use of the serving operators (serving.cu).
#pragma once
#include "host_common.h"

constexpr int SAMPLE_MAX_VOCAB = 393216;
// One row of f32 logits on the current device: l2b_sample_device's choice, with settings by value; *token (device memory) receives it.
int32_t enqueue_filtered_sample(const float* logits, int vocab, float temperature, int top_k, float top_p, float min_p, double uniform, int* token, int device, cudaStream_t st);
