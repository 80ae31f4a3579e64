// Rows and weights to block-scaled e4m3 (the rule in fp8.cuh).
//
// Rows: bound by HBM (2 or 4 bytes in, 1 out).  16 lanes hold one block of
// 128 values, 8 each (one 16-byte load of bf16), so the maximum is four
// shuffles and a warp stores 256 consecutive bytes; a warp has 1024 values of a
// row under way, neighbouring warps have neighbouring rows, whose scales are
// neighbours.  With slot_pos a row is read once and written to each of its k
// expert-sorted places: the gather of the bf16 path costs no pass of its own.
// 8192 x 4096: bf16 24 us (15.5 for the bytes), fp32 28 us (25.6); 8192 rows of 2048 to
// 8 places each 34 us (25.6).  What is over the bytes is the start of each warp: one row
// segment, then its end.
#include "fp8.cuh"

namespace {
using namespace frank;

template <class TX>
__device__ __forceinline__ void load8(const TX* p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

constexpr int kPairs = 4;  // pairs of blocks a warp

// x and slot_pos may be written until pdl_wait returns, so neither is __restrict__ (which would
// allow reads through the read-only path).
template <class TX>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const TX* x, int64_t T, int64_t K, int nb, const int32_t* slot_pos, int k, uint8_t* q,
                     float* q_scale) {
  pdl_wait();
  pdl_launch();
  const int half = (threadIdx.x >> 4) & 1, l16 = threadIdx.x & 15;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t seg = item / T, t = item - seg * T;
  if (seg * 2 * kPairs >= nb) return;
  const int64_t R = slot_pos != nullptr ? T * k : T;
  const int b0 = (int)seg * 2 * kPairs + half;
  // lane j: the j-th place of this warp's row (k <= 32), asked for beside the row
  const int lane = threadIdx.x & 31;
  const int place = slot_pos != nullptr && lane < k ? slot_pos[lane * T + t] : 0;
  float v[kPairs][8];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int64_t c = (int64_t)(b0 + 2 * i) * kQB + l16 * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    if (c < K) load8(x + t * K + c, v[i]);
  }
  uint2 u[kPairs];
  float sc[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[i][j]));
#pragma unroll
    for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const BlockScale s = block_scale(m);
    sc[i] = s.scale;
    u[i].x = e4m3x4(v[i][0] * s.inv, v[i][1] * s.inv, v[i][2] * s.inv, v[i][3] * s.inv);
    u[i].y = e4m3x4(v[i][4] * s.inv, v[i][5] * s.inv, v[i][6] * s.inv, v[i][7] * s.inv);
  }
  for (int j = 0; j < k; ++j) {
    const int at = __shfl_sync(0xffffffffu, place, j);
    const int64_t r = slot_pos != nullptr ? at : t;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int b = b0 + 2 * i;
      const int64_t c = (int64_t)b * kQB + l16 * 8;
      if (c < K) {
        *reinterpret_cast<uint2*>(q + r * K + c) = u[i];
        if (l16 == 0) q_scale[b * R + r] = sc[i];
      }
    }
  }
}

// [O, I, E] -> [E, O, I]: one block for each 128 x 128 block of (o, i) and all
// experts.  The first pass finds each expert's maximum (values of one o are
// contiguous over (i, e)) with an atomic on shared memory a value, the second writes
// runs along i.  Done once: 768 x 2048 x 128 in 6.4 ms, 4096 x 4096 x 8 in 0.7 ms.
template <class TX>
__global__ void __launch_bounds__(256)
prepack_fp8_kernel(const TX* __restrict__ src, int64_t O, int64_t I, int64_t E, uint8_t* __restrict__ q,
                   float* __restrict__ scale) {
  extern __shared__ uint32_t amax[];  // [E], then the inverse scales
  const int64_t o0 = (int64_t)blockIdx.y * kQB, i0 = (int64_t)blockIdx.x * kQB;
  const int64_t on = min((int64_t)kQB, O - o0), in = min((int64_t)kQB, I - i0);
  for (int64_t e = threadIdx.x; e < E; e += 256) amax[e] = 0;
  __syncthreads();
  for (int64_t o = 0; o < on; ++o) {
    const TX* row = src + ((o0 + o) * I + i0) * E;
    for (int64_t j = threadIdx.x; j < in * E; j += 256) atomicMax(&amax[j % E], abs_bits(load_as_f32(row, j)));
  }
  __syncthreads();
  for (int64_t e = threadIdx.x; e < E; e += 256) {
    const BlockScale s = block_scale(amax[e]);
    scale[(e * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = s.scale;
    amax[e] = __float_as_uint(s.inv);
  }
  __syncthreads();
  for (int64_t o = 0; o < on; ++o) {
    const TX* row = src + ((o0 + o) * I + i0) * E;
    for (int64_t j = threadIdx.x; j < in * E; j += 256) {
      const int64_t e = j / in, i = j % in;
      const float v = load_as_f32(row, i * E + e) * __uint_as_float(amax[e]);
      q[(e * O + o0 + o) * I + i0 + i] = (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
    }
  }
}

}  // namespace

namespace frank {

int launch_quantize_rows(int x_dtype, const void* x, int64_t T, int64_t K, const int32_t* slot_pos, int64_t k,
                         void* q, float* q_scale, cudaStream_t st) {
  if (T == 0) return FRANK_OK;
  const int nb = (int)q_blocks(K);
  const int64_t warps = T * ((nb + 2 * kPairs - 1) / (2 * kPairs)), blocks = (warps + 7) / 8;
  if (blocks > 0x7fffffffLL) {
    set_error("quantize_fp8: T=%lld rows are too many", (long long)T);
    return FRANK_EINVAL;
  }
  const dim3 grid((unsigned)blocks);
  cudaError_t e;
  if (x_dtype == FRANK_F32)
    e = launch_chained(quantize_rows_kernel<float>, grid, dim3(256), 0, st, 1, (const float*)x, T, K, nb, slot_pos,
                       (int)k, (uint8_t*)q, q_scale);
  else
    e = launch_chained(quantize_rows_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, 1, (const __nv_bfloat16*)x, T, K,
                       nb, slot_pos, (int)k, (uint8_t*)q, q_scale);
  FRANK_CUDA_TRY(e);
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

int launch_prepack_fp8(int in_dtype, const void* src, int64_t O, int64_t I, int64_t E, void* q, float* scale,
                       cudaStream_t st) {
  if (O == 0 || I == 0 || E == 0) return FRANK_OK;
  const dim3 grid((unsigned)q_blocks(I), (unsigned)q_blocks(O));
  if (in_dtype == FRANK_F32)
    prepack_fp8_kernel<float><<<grid, 256, E * 4, st>>>((const float*)src, O, I, E, (uint8_t*)q, scale);
  else
    prepack_fp8_kernel<__nv_bfloat16><<<grid, 256, E * 4, st>>>((const __nv_bfloat16*)src, O, I, E, (uint8_t*)q,
                                                                scale);
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

}  // namespace frank
