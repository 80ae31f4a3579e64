// The 8-bit MoE layer for a few tokens (few_fp8.cu): arguments and limits.
#pragma once

#include "fp8.cuh"

namespace frank {

constexpr int kFewMaxE = (int)kFp8MaxE;
constexpr int kFewMaxT = 64, kFewMaxSlots = 512;
constexpr int64_t kFewMaxCounts = 1 << 16;  // E * ceil(F/128)

struct FewRoute {
  const void* x;  // [T, H]
  int x_dtype;
  const float* norm_w;  // null: x is taken as it is (bf16)
  float eps;
  const void* wr;  // null: quantise only, the routing is given
  int wr_dtype;
  int T, H, E, k, normalize;
  uint8_t* xq;   // [T, H]
  float* xs;     // [ceil(H/128), T]
  float* w;      // [k, T]
  int32_t* ids;  // [k, T]
  int32_t* count;  // [E, ceil(F/128)], zeroed
  int n_count;
};

struct FewArgs {
  const uint8_t *w_up, *w_gate, *w_down;
  const float *s_up, *s_gate, *s_down;
  const uint8_t* xq;  // [T, H]
  const float* xs;
  int32_t* count;  // items of a block of h that are done
  float* h;        // [k T, F]
  uint8_t* hq;     // [k T, F]
  float* hs;    // [ceil(F/128), k T]
  float* d;     // [k T, H]
  const float* w;
  const int32_t* ids;
  int T, E, k, H, F;
  int32_t* err;  // device error word
};

int launch_few_route(const FewRoute& a, cudaStream_t st);
int launch_few_experts(const FewArgs& a, int32_t* err, cudaStream_t st);

}  // namespace frank
