// One pass over rows: combine of the MoE slots, the norm after a block with its
// gate and residual scale, the norm before the next block, and its 8-bit form.
//
//   v    = y, or sum_j d[slot_pos[j]]                                (fp32, j in order)
//   v    = residual_scale * residual + gate * v / sqrt(mean v^2 + eps) * post_w
//   next = v / sqrt(mean v^2 + eps) * next_w
//
// Bound by HBM: every value is read once and kept in registers (H <= 16384:
// 16 vectors of 4 for each of 256 threads), the two sums of squares are
// reductions over the row's threads.  Rows of up to 1024 values are one warp
// each, longer ones one block of 256 threads.  Thread i of a row owns vectors
// i, i + threads, ...: the 128 values of a quantisation block are one vector of
// each of a warp's lanes, so the block's maximum is one warp reduction.
#include "fp8.cuh"

namespace {
using namespace frank;

constexpr int kThreads = 256;

__device__ __forceinline__ float4 load4(const void* p, int dtype, int64_t i) {
  if (dtype == FRANK_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
  const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + i);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ void store4(void* p, int dtype, int64_t i, float4 v) {
  if (dtype == FRANK_F32)
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = v;
  else
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + i) =
        make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}

__device__ __forceinline__ float4 round_bf16(float4 v) {
  v.x = __bfloat162float(__float2bfloat16_rn(v.x));
  v.y = __bfloat162float(__float2bfloat16_rn(v.y));
  v.z = __bfloat162float(__float2bfloat16_rn(v.z));
  v.w = __bfloat162float(__float2bfloat16_rn(v.w));
  return v;
}

// Sum over the GS threads of a row, the same in every thread; `red`: one
// array for each sum of a kernel, so that no barrier is needed before it.
template <int GS>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (GS == 32) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < GS / 32; ++w) s += red[w];
  return s;
}

template <int GS, int V>
__device__ __forceinline__ float inv_rms(const float4 (&v)[V], int64_t H, float eps, float* red) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    ss = fmaf(v[i].x, v[i].x, ss);
    ss = fmaf(v[i].y, v[i].y, ss);
    ss = fmaf(v[i].z, v[i].z, ss);
    ss = fmaf(v[i].w, v[i].w, ss);
  }
  return 1.f / sqrtf(row_sum<GS>(ss, red) / (float)H + eps);
}

template <int GS, int V, bool SLOTS>
__global__ void __launch_bounds__(kThreads) norm_rows_kernel(const NormRows a) {
  __shared__ float red[2][kThreads / 32];
  const int tid = threadIdx.x % GS;
  const int64_t t = (int64_t)blockIdx.x * (kThreads / GS) + threadIdx.x / GS;
  pdl_wait();
  pdl_launch();
  if (t >= a.T) return;  // GS < kThreads only: whole warps
  const int64_t H = a.H;
  // the row and its residual are asked for together: the sum of squares must not stand between them
  float4 v[V], x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int64_t h = 4 * (int64_t)(tid + i * GS);
    v[i] = x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!SLOTS && h < H) v[i] = load4(a.y, a.y_dtype, t * H + h);
    if (a.residual != nullptr && h < H) x[i] = load4(a.residual, a.out_dtype, t * H + h);
  }
  if (SLOTS) {
    // rows in order, the loads of several at a time
    constexpr int kAhead = V <= 2 ? 4 : V <= 4 ? 2 : 1;
    for (int j0 = 0; j0 < a.k; j0 += kAhead) {
      float4 u[kAhead][V];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int64_t s = (int64_t)(j0 + q) * a.T + t;
        int64_t row = 0;
        if (j0 + q < a.k) row = (a.slot_pos != nullptr ? (int64_t)a.slot_pos[s] : s) * H;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int64_t h = 4 * (int64_t)(tid + i * GS);
          u[q][i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (h < H && j0 + q < a.k) u[q][i] = load4(a.d, a.d_dtype, row + h);
        }
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q)
        if (j0 + q < a.k) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            v[i].x += u[q][i].x;
            v[i].y += u[q][i].y;
            v[i].z += u[q][i].z;
            v[i].w += u[q][i].w;
          }
        }
    }
  }
  float r = 1.f;
  if (a.post_w != nullptr) r = inv_rms<GS, V>(v, H, a.eps, red[0]);
  const float* gate = a.gate == nullptr ? nullptr : a.gate + t / a.rows_per_gate * H;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int64_t h = 4 * (int64_t)(tid + i * GS);
    if (h < H) {
      if (a.post_w != nullptr) {
        const float4 w = *reinterpret_cast<const float4*>(a.post_w + h);
        v[i] = make_float4(v[i].x * r * w.x, v[i].y * r * w.y, v[i].z * r * w.z, v[i].w * r * w.w);
      }
      if (gate != nullptr) {
        const float4 g = *reinterpret_cast<const float4*>(gate + h);
        v[i] = make_float4(v[i].x * g.x, v[i].y * g.y, v[i].z * g.z, v[i].w * g.w);
      }
      if (a.residual != nullptr) {
        const float s = a.residual_scale;
        v[i] = make_float4(fmaf(s, x[i].x, v[i].x), fmaf(s, x[i].y, v[i].y), fmaf(s, x[i].z, v[i].z),
                           fmaf(s, x[i].w, v[i].w));
      }
      if (a.out != nullptr) {
        if (a.out_dtype == FRANK_BF16) v[i] = round_bf16(v[i]);
        store4(a.out, a.out_dtype, t * H + h, v[i]);
      }
    }
  }
  if (a.next_w == nullptr) return;
  r = inv_rms<GS, V>(v, H, a.eps, red[1]);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int64_t h = 4 * (int64_t)(tid + i * GS);
    if (h < H) {
      const float4 w = *reinterpret_cast<const float4*>(a.next_w + h);
      v[i] = make_float4(v[i].x * r * w.x, v[i].y * r * w.y, v[i].z * r * w.z, v[i].w * r * w.w);
      if (a.next != nullptr) store4(a.next, a.next_dtype, t * H + h, v[i]);
    }
    if (a.q != nullptr) {  // lanes past H hold zeros
      v[i] = round_bf16(v[i]);
      uint32_t m = max(max(abs_bits(v[i].x), abs_bits(v[i].y)), max(abs_bits(v[i].z), abs_bits(v[i].w)));
      m = __reduce_max_sync(0xffffffffu, m);
      const BlockScale s = block_scale(m);
      if (h < H) {
        *reinterpret_cast<uint32_t*>(a.q + t * H + h) =
            e4m3x4(v[i].x * s.inv, v[i].y * s.inv, v[i].z * s.inv, v[i].w * s.inv);
        if (h % kQB == 0) a.q_scale[h / kQB * a.T + t] = s.scale;
      }
    }
  }
}

}  // namespace

namespace frank {

int launch_norm_rows(const NormRows& a, cudaStream_t st) {
  if (a.T == 0) return FRANK_OK;
  const bool warp_rows = a.H <= 1024;
  const int64_t vec = (a.H / 4 + (warp_rows ? 32 : kThreads) - 1) / (warp_rows ? 32 : kThreads);
  const int64_t per = warp_rows ? kThreads / 32 : 1;
  const dim3 grid((unsigned)((a.T + per - 1) / per)), block(kThreads);
  cudaError_t e;
#define FRANK_NORM(GS, V)                                                                      \
  e = a.d != nullptr ? launch_chained(norm_rows_kernel<GS, V, true>, grid, block, 0, st, 1, a) \
                     : launch_chained(norm_rows_kernel<GS, V, false>, grid, block, 0, st, 1, a)
  if (warp_rows) {
    if (vec <= 1) FRANK_NORM(32, 1);
    else if (vec <= 2) FRANK_NORM(32, 2);
    else if (vec <= 4) FRANK_NORM(32, 4);
    else FRANK_NORM(32, 8);
  } else {
    if (vec <= 2) FRANK_NORM(256, 2);
    else if (vec <= 4) FRANK_NORM(256, 4);
    else if (vec <= 8) FRANK_NORM(256, 8);
    else FRANK_NORM(256, 16);
  }
#undef FRANK_NORM
  FRANK_CUDA_TRY(e);
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

}  // namespace frank
