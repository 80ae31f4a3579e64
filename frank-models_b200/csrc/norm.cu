// One pass over rows: combine of the MoE slots, the norm after a block with its
// gate and residual scale, the norm before the next block, and its 8-bit form.
//
//   v    = y, or sum_j d[slot_pos[j]]                                (fp32, j in order)
//   v    = residual_scale * residual + gate * v / sqrt(mean v^2 + eps) * post_w
//   next = v / sqrt(mean v^2 + eps) * next_w
//
// Bound by HBM, and close behind by issue: every value is read once and kept in
// registers (H <= 16384: 4 vectors of 4 for each of 1024 threads), the two sums of
// squares are reductions over the row's threads.  Rows of up to 1024 values are one
// warp each, longer ones one block of 128 to 1024 threads.  Thread i of a row owns
// vectors i, i + threads, ...: the 128 values of a quantisation block are one
// vector of each of a warp's lanes, so the block's maximum is one warp reduction.
// 16384 rows of 4096, fp32 y, bf16 residual and next: 106 us,
// 6.36 TB/s.  Slower: two vectors a thread (128 us), a run of rows
// a block with the weights in shared memory and the next row on its way (217 us).
// With the 8-bit form instead, 8192 rows of 4096: bf16 in 37 us (15.5 for the bytes), fp32 in
// 38 us (25.6): two passes of reductions a row, which is short work for a block of 256 threads.
#include "fp8.cuh"

namespace {
using namespace frank;

__device__ __forceinline__ float4 unpack4(uint2 u) {
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}

// This thread's V vectors of a row, GS vectors apart (zeros past the row's n), fp32 or bf16.
template <int GS, int V>
__device__ __forceinline__ void load_row(float4 (&v)[V], const void* base, int dtype, int64_t row, int tid, int n) {
  if (dtype == FRANK_F32) {
    const float4* p = reinterpret_cast<const float4*>(base) + row + tid;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = tid + i * GS < n ? p[i * GS] : make_float4(0.f, 0.f, 0.f, 0.f);
  } else {
    const uint2* p = reinterpret_cast<const uint2*>(base) + row + tid;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = unpack4(tid + i * GS < n ? p[i * GS] : make_uint2(0u, 0u));
  }
}

// Stores them; ROUND: v becomes what the row then holds.
template <int GS, int V, bool ROUND>
__device__ __forceinline__ void store_row(float4 (&v)[V], void* base, int dtype, int64_t row, int tid, int n) {
  if (dtype == FRANK_F32) {
    float4* p = reinterpret_cast<float4*>(base) + row + tid;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (tid + i * GS < n) p[i * GS] = v[i];
  } else {
    uint2* p = reinterpret_cast<uint2*>(base) + row + tid;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint2 u = make_uint2(pack_bf16x2(v[i].x, v[i].y), pack_bf16x2(v[i].z, v[i].w));
      if (tid + i * GS < n) p[i * GS] = u;
      if (ROUND) v[i] = unpack4(u);
    }
  }
}

// Sum over the GS threads of a row, the same in every thread; `red`: one array for
// each sum of a row, so that no barrier is needed before it.
template <int GS>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (GS == 32) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < GS / 32; w += 4) {
    const float4 q = *reinterpret_cast<const float4*>(red + w);
    s += (q.x + q.y) + (q.z + q.w);
  }
  return s;
}

// 1 / sqrt(mean v^2 + eps); CUDA's rsqrtf is within 2 ulp.
template <int GS, int V>
__device__ __forceinline__ float inv_rms(const float4 (&v)[V], int n, float eps, float* red) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    ss = fmaf(v[i].x, v[i].x, ss);
    ss = fmaf(v[i].y, v[i].y, ss);
    ss = fmaf(v[i].z, v[i].z, ss);
    ss = fmaf(v[i].w, v[i].w, ss);
  }
  return rsqrtf(row_sum<GS>(ss, red) / (float)(4 * n) + eps);
}

// v *= r * w, w a row of n vectors
template <int GS, int V>
__device__ __forceinline__ void scale_row(float4 (&v)[V], float r, const float* w, int tid, int n) {
  const float4* p = reinterpret_cast<const float4*>(w) + tid;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (tid + i * GS < n) {
      const float4 q = p[i * GS];
      v[i] = make_float4(v[i].x * r * q.x, v[i].y * r * q.y, v[i].z * r * q.z, v[i].w * r * q.w);
    }
}

template <int GS, int V, bool SLOTS>
__global__ void __launch_bounds__(GS == 32 ? 256 : GS, 1)  // without the 1: 118 us
norm_rows_kernel(const NormRows a) {
  constexpr int kGroups = GS == 32 ? 8 : 1;
  __shared__ alignas(16) float red[2][GS == 32 ? 4 : GS / 32];
  const int tid = threadIdx.x % GS, n = (int)(a.H / 4);
  const int64_t t = (int64_t)blockIdx.x * kGroups + threadIdx.x / GS;
  pdl_wait();
  pdl_launch();
  if (t >= a.T) return;  // whole warps of GS = 32
  // a row and its residual are asked for together: the sum of squares must not stand between them
  float4 v[V], x[V];
  if (!SLOTS) load_row<GS, V>(v, a.y, a.y_dtype, t * n, tid, n);
  if (a.residual != nullptr) load_row<GS, V>(x, a.residual, a.out_dtype, t * n, tid, n);
  if (SLOTS) {
    // rows in order, the loads of several at a time
    constexpr int kAhead = V <= 2 ? 4 : V <= 4 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < a.k; j0 += kAhead) {
      float4 u[kAhead][V];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int64_t s = (int64_t)(j0 + q) * a.T + t;
        if (j0 + q < a.k)
          load_row<GS, V>(u[q], a.d, FRANK_F32, (a.slot_pos != nullptr ? (int64_t)a.slot_pos[s] : s) * n, tid, n);
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
  if (a.post_w != nullptr) scale_row<GS, V>(v, inv_rms<GS, V>(v, n, a.eps, red[0]), a.post_w, tid, n);
  if (a.gate != nullptr)
    scale_row<GS, V>(v, 1.f, a.gate + (int64_t)((uint32_t)t / (uint32_t)a.rows_per_gate) * a.H, tid, n);
  if (a.residual != nullptr) {
    const float s = a.residual_scale;
#pragma unroll
    for (int i = 0; i < V; ++i)
      v[i] = make_float4(fmaf(s, x[i].x, v[i].x), fmaf(s, x[i].y, v[i].y), fmaf(s, x[i].z, v[i].z),
                         fmaf(s, x[i].w, v[i].w));
  }
  if (a.out != nullptr) store_row<GS, V, true>(v, a.out, a.out_dtype, t * n, tid, n);
  if (a.next_w == nullptr) return;
  scale_row<GS, V>(v, inv_rms<GS, V>(v, n, a.eps, red[1]), a.next_w, tid, n);
  if (a.q == nullptr) {
    store_row<GS, V, false>(v, a.next, a.next_dtype, t * n, tid, n);
    return;
  }
  if (a.next != nullptr) store_row<GS, V, false>(v, a.next, a.next_dtype, t * n, tid, n);
#pragma unroll
  for (int i = 0; i < V; ++i) {  // lanes past the row hold zeros
    const int h = tid + i * GS;
    const float4 w = unpack4(make_uint2(pack_bf16x2(v[i].x, v[i].y), pack_bf16x2(v[i].z, v[i].w)));
    const BlockScale s = block_scale(
        __reduce_max_sync(0xffffffffu, max(max(abs_bits(w.x), abs_bits(w.y)), max(abs_bits(w.z), abs_bits(w.w)))));
    if (h < n) {
      *reinterpret_cast<uint32_t*>(a.q + t * a.H + 4 * h) =
          e4m3x4(w.x * s.inv, w.y * s.inv, w.z * s.inv, w.w * s.inv);
      if (h % (kQB / 4) == 0) a.q_scale[(int64_t)(h / (kQB / 4)) * a.T + t] = s.scale;
    }
  }
}

// y[t] = sum_j d[slot_pos[j]] alone: four columns a thread, eight rows at a time.
template <class TY>
__global__ void __launch_bounds__(128) combine_slots_kernel(const NormRows a) {
  pdl_wait();
  pdl_launch();
  const int64_t t = blockIdx.x;
  const int h = (blockIdx.y * 128 + threadIdx.x) * 4;
  if (h >= a.H) return;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j0 = 0; j0 < a.k; j0 += 8) {
    float4 u[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (j0 + q < a.k) {
        const int64_t s = (int64_t)(j0 + q) * a.T + t;
        const int64_t row = a.slot_pos != nullptr ? (int64_t)a.slot_pos[s] : s;
        u[q] = *reinterpret_cast<const float4*>(a.d + row * a.H + h);
      }
    }
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (j0 + q < a.k) v.x += u[q].x, v.y += u[q].y, v.z += u[q].z, v.w += u[q].w;
  }
  TY* y = static_cast<TY*>(a.out) + t * a.H + h;
  if constexpr (sizeof(TY) == 4)
    *reinterpret_cast<float4*>(y) = v;
  else
    *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}

template <int GS, int V>
cudaError_t launch_rows(const NormRows& a, cudaStream_t st) {
  constexpr int kGroups = GS == 32 ? 8 : 1;
  const dim3 grid((unsigned)((a.T + kGroups - 1) / kGroups)), block(GS == 32 ? 256 : GS);
  return a.d != nullptr ? launch_chained(norm_rows_kernel<GS, V, true>, grid, block, 0, st, 1, a)
                        : launch_chained(norm_rows_kernel<GS, V, false>, grid, block, 0, st, 1, a);
}

cudaError_t launch_combine_slots(const NormRows& a, cudaStream_t st) {
  const dim3 grid((unsigned)a.T, (unsigned)((a.H + 511) / 512));
  if (a.out_dtype == FRANK_F32)
    return launch_chained(combine_slots_kernel<float>, grid, dim3(128), 0, st, 1, a);
  return launch_chained(combine_slots_kernel<__nv_bfloat16>, grid, dim3(128), 0, st, 1, a);
}

}  // namespace

namespace frank {

int launch_norm_rows(const NormRows& a, cudaStream_t st) {
  if (a.T == 0) return FRANK_OK;
  const int64_t H4 = a.H / 4;
  cudaError_t e;
  if (a.d != nullptr && a.post_w == nullptr && a.gate == nullptr && a.residual == nullptr && a.next_w == nullptr)
    e = launch_combine_slots(a, st);
  else if (H4 <= 32) e = launch_rows<32, 1>(a, st);
  else if (H4 <= 64) e = launch_rows<32, 2>(a, st);
  else if (H4 <= 128) e = launch_rows<32, 4>(a, st);
  else if (H4 <= 256) e = launch_rows<32, 8>(a, st);
  else if (H4 <= 512) e = launch_rows<128, 4>(a, st);
  else if (H4 <= 1024) e = launch_rows<256, 4>(a, st);
  else if (H4 <= 2048) e = launch_rows<512, 4>(a, st);
  else e = launch_rows<1024, 4>(a, st);
  FRANK_CUDA_TRY(e);
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

}  // namespace frank
