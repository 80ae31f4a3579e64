// Grouped product of block-scaled e4m3 rows and weights.
//
//   y[r, n] = sum_b a_scale[b, r] * w_scale[e, n/128, b] * sum_{k in b} a[r, k] * w[e, n, k]
//
// A block of 128 threads owns 16 rows of one expert and 128 columns, one column
// for each thread: the columns of one scale block, and with SWIGLU the values
// that share a scale of h.
#include "fp8.cuh"

namespace {
using namespace frank;

constexpr int kRows = 16;
constexpr int kLd = kQB + 4;

struct Params {
  const uint8_t* a;
  const float* a_scale;
  const uint8_t* w[2];
  const float* w_scale[2];
  const int32_t* offsets;
  int E;
  int64_t rows, N, K;
  const float* wrow;
  int out_dtype;
  void* out;
  float* h_scale;
};

template <int MODE>
__global__ void __launch_bounds__(128) fp8_gemm_simple_kernel(const Params p) {
  constexpr int NW = MODE == FP8_SWIGLU ? 2 : 1;
  __shared__ float as[kRows][kQB];
  __shared__ uint8_t ws[NW][kQB][kLd];
  __shared__ uint32_t amax[kRows];
  pdl_wait();
  pdl_launch();
  int e = 0;
  int64_t r0 = 0, r1 = 0, tile = blockIdx.x;
  for (; e < p.E; ++e) {
    r0 = p.offsets != nullptr ? p.offsets[e] : 0;
    r1 = p.offsets != nullptr ? p.offsets[e + 1] : p.rows;
    const int64_t tiles = (r1 - r0 + kRows - 1) / kRows;
    if (tile < tiles) break;
    tile -= tiles;
  }
  if (e == p.E) return;
  r0 += tile * kRows;
  const int nr = (int)min((int64_t)kRows, r1 - r0);
  const int64_t n0 = (int64_t)blockIdx.y * kQB, n = n0 + threadIdx.x;
  const int nb = (int)((p.K + kQB - 1) / kQB);
  float acc[NW][kRows] = {};
  for (int b = 0; b < nb; ++b) {
    const int64_t k0 = (int64_t)b * kQB;
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * kQB; i += 128) {
      const int r = i / kQB, c = i % kQB;
      as[r][c] = r < nr && k0 + c < p.K ? e4m3_to_f32(p.a[(r0 + r) * p.K + k0 + c]) : 0.f;
    }
    for (int m = 0; m < NW; ++m)
      for (int i = threadIdx.x; i < kQB * kQB; i += 128) {
        const int r = i / kQB, c = i % kQB;
        ws[m][r][c] = n0 + r < p.N && k0 + c < p.K ? p.w[m][((int64_t)e * p.N + n0 + r) * p.K + k0 + c] : 0;
      }
    __syncthreads();
    for (int m = 0; m < NW; ++m) {
      float part[kRows] = {};
      for (int c = 0; c < kQB; ++c) {
        const float w = e4m3_to_f32(ws[m][threadIdx.x][c]);
#pragma unroll
        for (int r = 0; r < kRows; ++r) part[r] = fmaf(as[r][c], w, part[r]);
      }
      const float sw = p.w_scale[m][((int64_t)e * gridDim.y + blockIdx.y) * nb + b];
      for (int r = 0; r < kRows; ++r)
        if (r < nr) acc[m][r] = fmaf(part[r], p.a_scale[b * p.rows + r0 + r] * sw, acc[m][r]);
    }
  }
  if (MODE == FP8_SWIGLU) {
    if (threadIdx.x < kRows) amax[threadIdx.x] = 0;
    __syncthreads();
    for (int r = 0; r < nr; ++r) {
      acc[0][r] = n < p.N ? acc[0][r] * silu_ref(acc[NW - 1][r]) : 0.f;
      atomicMax(&amax[r], abs_bits(acc[0][r]));
    }
    __syncthreads();
    for (int r = 0; r < nr; ++r) {
      const BlockScale s = block_scale(amax[r]);
      if (n < p.N)
        static_cast<uint8_t*>(p.out)[(r0 + r) * p.N + n] =
            (uint8_t)__nv_cvt_float_to_fp8(acc[0][r] * s.inv, __NV_SATFINITE, __NV_E4M3);
      if (threadIdx.x == 0) p.h_scale[blockIdx.y * p.rows + r0 + r] = s.scale;
    }
  } else if (n < p.N) {
    for (int r = 0; r < nr; ++r) {
      const float v = MODE == FP8_SCALE ? acc[0][r] * p.wrow[r0 + r] : acc[0][r];
      if (p.out_dtype == FRANK_F32)
        static_cast<float*>(p.out)[(r0 + r) * p.N + n] = v;
      else
        static_cast<__nv_bfloat16*>(p.out)[(r0 + r) * p.N + n] = __float2bfloat16_rn(v);
    }
  }
}

}  // namespace

namespace frank {

int launch_fp8_gemm(const Fp8Gemm& g, cudaStream_t st) {
  if (g.rows == 0) return FRANK_OK;
  Params p;
  p.a = (const uint8_t*)g.a;
  p.a_scale = g.a_scale;
  p.w[0] = (const uint8_t*)g.w;
  p.w[1] = (const uint8_t*)g.w2;
  p.w_scale[0] = g.w_scale;
  p.w_scale[1] = g.w2_scale;
  p.offsets = g.offsets;
  p.E = (int)g.E;
  p.rows = g.rows;
  p.N = g.N;
  p.K = g.K;
  p.wrow = g.wrow;
  p.out_dtype = g.out_dtype;
  p.out = g.out;
  p.h_scale = g.h_scale;
  const dim3 grid((unsigned)((g.rows + kRows - 1) / kRows + g.E), (unsigned)q_blocks(g.N));
  cudaError_t e;
  if (g.mode == FP8_SWIGLU) e = launch_chained(fp8_gemm_simple_kernel<FP8_SWIGLU>, grid, dim3(128), 0, st, 1, p);
  else if (g.mode == FP8_SCALE) e = launch_chained(fp8_gemm_simple_kernel<FP8_SCALE>, grid, dim3(128), 0, st, 1, p);
  else e = launch_chained(fp8_gemm_simple_kernel<FP8_PLAIN>, grid, dim3(128), 0, st, 1, p);
  FRANK_CUDA_TRY(e);
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

}  // namespace frank
