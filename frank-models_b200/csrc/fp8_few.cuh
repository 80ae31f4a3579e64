// The 8-bit MoE layer for a few tokens (few_fp8.cu): arguments and limits.
#pragma once

#include "fp8.cuh"

namespace frank {

constexpr int kFewMaxE = (int)kFp8MaxE;
constexpr int kFewMaxT = 64, kFewMaxSlots = 512;
constexpr int64_t kFewMaxBlocksH = 128, kFewMaxBlocksF = 2048;  // their K blocks are counted in 32 bits

struct FewRoute {
  const void* x;  // [T, H]
  int x_dtype;
  const float* norm_w;  // null: x is taken as it is (bf16)
  float eps;
  const void* wr;  // null: quantise only, the routing is given
  int wr_dtype;
  int T, H, E, k, normalize;
  uint8_t* xq;   // [T, H]
  float* xs;     // [ceil(H/128), kFewMaxT]
  float* w;      // [k, T]
  int32_t* ids;  // [k, T]
  int32_t* count;  // zeroed for few_product
  int n_count;
};

struct FewArgs {
  const uint8_t *w_up, *w_gate, *w_down;
  const float *s_up, *s_gate, *s_down;
  const uint8_t* xq;  // [T, H]
  const float* xs;
  uint8_t* hq;  // [few_h_rows, F], the slots sorted by expert, each expert at a multiple of 16
  float* hs;    // [ceil(F/128), few_h_rows]
  float* d;     // [k T, H]
  const float* w;
  const int32_t* ids;
  int T, E, k, H, F;
  float* partial;  // [few_partials]
  int32_t* count;  // [few_counts], zero; set by launch_few_experts:
  int64_t partial_stride;
  int n_count, h_rows;
  int32_t* err;       // device error word
};

int64_t few_counts(int64_t T, int64_t E, int64_t k, int64_t H, int64_t F);
int64_t few_partials(int64_t T);
int64_t few_h_rows(int64_t T, int64_t E, int64_t k);
int launch_few_route(const FewRoute& a, cudaStream_t st);
int launch_few_experts(const FewArgs& a, int32_t* err, cudaStream_t st);

}  // namespace frank
