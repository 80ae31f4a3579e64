// Block-scaled e4m3: the scale rule, conversions, and the launchers shared by
// the 8-bit kernels (declared in include/frank_fp8.h).
#pragma once

#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"
#include "frank_fp8.h"

namespace frank {

constexpr int kQB = FRANK_FP8_BLOCK;  // values that share a scale
inline int64_t q_blocks(int64_t n) { return (n + kQB - 1) / kQB; }

// Arguments of one pass over rows of H values (norm.cu): each row is read
// once, kept in registers and leaves in every form that is asked for.
struct NormRows {
  // source: y [T, H], or the sum over k slots of d (rows at slot_pos[j*T+t], or j*T+t)
  int y_dtype = FRANK_F32;
  const void* y = nullptr;
  const float* d = nullptr;
  const int32_t* slot_pos = nullptr;
  int k = 0;
  // v = residual_scale * residual + gate * (post_w ? rms_norm(v, post_w) : v)
  const float* post_w = nullptr;
  float eps = 0.f;
  const float* gate = nullptr;
  int64_t rows_per_gate = 1;
  int out_dtype = FRANK_F32;  // of residual and out
  const void* residual = nullptr;
  float residual_scale = 1.f;
  void* out = nullptr;
  // next = rms_norm(v, next_w), v rounded to out_dtype when it is stored; q / q_scale: 8-bit form of bf16(next)
  const float* next_w = nullptr;
  int next_dtype = FRANK_BF16;
  void* next = nullptr;
  uint8_t* q = nullptr;
  float* q_scale = nullptr;
  int64_t T = 0, H = 0;
};
constexpr int64_t kNormMaxH = 16384;
int launch_norm_rows(const NormRows& a, cudaStream_t st);

// slot_pos (may be null): row t goes to rows slot_pos[j*T + t], j < k, of q [k*T, K] and q_scale [ceil(K/128), k*T].
int launch_quantize_rows(int x_dtype, const void* x, int64_t T, int64_t K, const int32_t* slot_pos, int64_t k,
                         void* q, float* q_scale, cudaStream_t st);
int launch_prepack_fp8(int in_dtype, const void* src, int64_t O, int64_t I, int64_t E, void* q, float* scale,
                       cudaStream_t st);

// Grouped product of 8-bit rows and weights (gemm_fp8.cu).
//   PLAIN : out [rows, N] in out_dtype
//   SCALE : out fp32 [rows, N], row r times wrow[r]
//   SWIGLU: w = gate, w2 = up; h = gate * silu(up) quantised -> out e4m3 [rows, N], h_scale [ceil(N/128), rows]
enum Fp8Mode { FP8_PLAIN = 0, FP8_SCALE = 1, FP8_SWIGLU = 2 };
struct Fp8Gemm {
  Fp8Mode mode = FP8_PLAIN;
  const void* a = nullptr;
  const float* a_scale = nullptr;
  const void* w = nullptr;
  const float* w_scale = nullptr;
  const void* w2 = nullptr;
  const float* w2_scale = nullptr;
  const int32_t* offsets = nullptr;
  int64_t E = 1, rows = 0, N = 0, K = 0;
  const float* wrow = nullptr;
  int out_dtype = FRANK_F32;
  void* out = nullptr;
  float* h_scale = nullptr;
};
int launch_fp8_gemm(const Fp8Gemm& g, cudaStream_t st);
constexpr int64_t kFp8MaxE = 256;
constexpr int64_t kFp8MaxRows = 0x7fffff00LL;  // a tile that begins below the last row ends inside 31 bits

}  // namespace frank

// ---------------------------------------------------------------- device --

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// scale = 2^p and 1/scale for the largest |v| of a block, given as bits
// (integer maxima keep NaN above infinity above every number).  448 = 1.75 * 2^8:
// amax = 1.m * 2^e <= 448 * 2^p  <=>  p >= e - 8 + (1.m > 1.75).
// p is in [-110, 120], so scale and 1/scale are normal numbers.  A product's two scales are
// multiplied first (one FMA a value then): frank_fp8.h has the range that this leaves the
// weights' scales.
struct BlockScale {
  float scale, inv;
};
__device__ __forceinline__ BlockScale block_scale(uint32_t amax) {
  BlockScale s;
  if (amax >= 0x7f800000u) {
    s.scale = s.inv = __uint_as_float(0x7fc00000u);
    return s;
  }
  int p = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  p = p < -110 ? -110 : p;
  s.scale = __uint_as_float((uint32_t)(127 + p) << 23);
  s.inv = __uint_as_float((uint32_t)(127 - p) << 23);
  return s;
}

// silu(u) = u / (1 + 2^(-u log2 e)) by CUDA's approximate exponential and division (2 ulp
// each); 64 of them end a tile of a product.  The exponent's rounding error is put
// back as a factor 1 + ln 2 * error.  u is clamped to +-88 in the exponent, where 2^t and
// the error stay finite: above, the divisor is 1 and the result u, also for the largest
// finite u; below, the divisor is over 2^126, for which the approximate division gives 0.
// An infinite or NaN u gives infinity or NaN, and its block of 128 the scale NaN.
__device__ __forceinline__ float silu(float u) {
  const float c = fminf(fmaxf(u, -88.f), 88.f);
  const float t = c * -1.44269502f;
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  const float lost = fmaf(c, -1.92596299e-8f, fmaf(c, -1.44269502f, -t));
  return __fdividef(u, 1.f + fmaf(e * 0.693147182f, lost, e));
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}

// 32 bytes of one thread: a whole sector.
__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Programmatic dependent launch: blocks may start while the stream's previous
// kernel finishes and wait here for its results.  What that kernel may write is
// no read-only data then: it is read by plain loads, __ldcg or copies.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" :::); }

namespace frank {
// Raises a kernel's limit of dynamic shared memory, once on each device (a call costs
// about a microsecond); `done` is the kernel's own mask of devices.
template <typename Kern>
inline cudaError_t allow_smem(std::atomic<uint64_t>& done, Kern kern, size_t bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <typename... KArgs, typename... Args>
inline cudaError_t launch_chained(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                                  unsigned cluster, Args... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}
}  // namespace frank
