// The arguments of an append to the paged caches.
#pragma once

#include "dsa_rope.h"

namespace dsa {

constexpr int AP_KINDS = 4;        // rows that a call appends for each token (latent row, indexer key, ..)
constexpr int AP_MAX_WIDTH = 1024;

struct AppendRows {
  const void* x;        // [T, width] bf16 or fp32, rows x_row values apart
  long x_row;
  int fp32;
  int width;
  int rope_at;          // the first of the 2R rotated columns, -1: none
  int half;             // pairs (i, i + R)
  const void* weight;   // the norm of the first norm_width columns, null: none
  const void* bias;     // with it the layer norm, without it the root-mean-square norm
  int norm_fp32;
  int norm_width;
  float eps;
  float fp8_max;
  void* cache;          // e4m3 or bf16
  int cache_bf16;
  float* scale;         // per slot; null: none
};

struct AppendSet {
  AppendRows rows[AP_KINDS];
  int n;
};

}  // namespace dsa
