// The 8-bit MoE layer for a few tokens, bound by the expert weights in HBM:
// three launches chained by programmatic dependent launch (and the combine in
// norm.cu), without a permutation, a gather or atomics.
//
//   few_route   [norm,] quantisation, router, softmax and top-k: clusters of 8
//               CTAs take 8 tokens, each CTA an eighth of H.  The sums of squares and
//               the partial logits are exchanged through distributed shared memory
//               and added in CTA order.
//   few_up      h = gate * silu(up), quantised: clusters of 4 CTAs take one expert and
//               128 columns of F, each CTA 32 of them; a block of h shares one scale, so
//               the maxima go round the cluster.
//   few_down    d[slot] = route weight * down(h[slot])
//
// The weights are read once, straight into the registers of the warps that use
// them, 16 bytes a lane and four K blocks (8 KB a warp) at a time: with two CTAs an SM
// 128 KB are under way, what 6.5 TB/s need at 3 us.  A warp multiplies 16 weight rows (8 of
// gate and the same 8 of up, or 16 of down) with 8 tokens by mma.m16n8k16 in
// fp16, into which e4m3 converts exactly, with fp32 sums; one K block is summed and
// then scaled.  Lane t of a quad holds K elements 16 t .. 16 t + 15 of a row: the
// MMA's K index is permuted alike for weights and tokens, which leaves the sum.
#include "fp8.cuh"
#include "fp8_few.cuh"

namespace {
using namespace frank;

// ------------------------------------------------------------ cluster --
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_peer(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ float ld_peer(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float4 load4(const void* p, int dtype, int64_t i) {
  if (dtype == FRANK_F32) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
  const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + i));
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}

// -------------------------------------------------------------- route --
constexpr int kRouteCtas = 8, kRouteTok = 8, kRouteThreads = 512;

__global__ void __launch_bounds__(kRouteThreads) few_route_kernel(const FewRoute a) {
  extern __shared__ float xs[];  // [8 tokens][slice]
  __shared__ float part[kFewMaxE][kRouteTok];
  __shared__ float ssq_block[kRouteTok][16], ssq[kRouteCtas][kRouteTok];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kWarps = kRouteThreads / 32;
  const uint32_t rank = cta_rank();
  const int t0 = blockIdx.x / kRouteCtas * kRouteTok, nt = min(kRouteTok, a.T - t0);
  const int nb = (a.H + kQB - 1) / kQB, sb = (nb + kRouteCtas - 1) / kRouteCtas;  // blocks of a row, of a slice
  const int slice = sb * kQB, h0 = (int)rank * slice;
  pdl_wait();
  pdl_launch();
  cluster_arrive();  // every CTA has started before its memory is written
  // one (token, block) a warp: a vector of 4 for each lane
  for (int i = warp; i < kRouteTok * sb; i += kWarps) {
    const int t = i / sb, b = i % sb, h = h0 + b * kQB + lane * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (t < nt && h < a.H) v = load4(a.x, a.x_dtype, (int64_t)(t0 + t) * a.H + h);
    *reinterpret_cast<float4*>(xs + t * slice + b * kQB + lane * 4) = v;
    if (a.norm_w != nullptr) {
      float s = fmaf(v.x, v.x, fmaf(v.y, v.y, fmaf(v.z, v.z, v.w * v.w)));
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) ssq_block[t][b] = s;
    }
  }
  cluster_wait();
  if (a.norm_w != nullptr) {
    __syncthreads();
    if (threadIdx.x < kRouteTok * kRouteCtas) {
      const int t = threadIdx.x % kRouteTok, to = threadIdx.x / kRouteTok;
      float s = 0.f;
      for (int b = 0; b < sb; ++b) s += ssq_block[t][b];
      st_peer(peer_addr(&ssq[rank][t], (uint32_t)to), __float_as_uint(s));
    }
    cluster_sync();
  }
  for (int i = warp; i < kRouteTok * sb; i += kWarps) {
    const int t = i / sb, b = i % sb, h = h0 + b * kQB + lane * 4;
    float* p = xs + t * slice + b * kQB + lane * 4;
    float4 v = *reinterpret_cast<const float4*>(p);  // written by this lane
    if (a.norm_w != nullptr && h < a.H) {
      float s = 0.f;
      for (int r = 0; r < kRouteCtas; ++r) s += ssq[r][t];
      const float inv = 1.f / sqrtf(s / (float)a.H + a.eps);
      const float4 w = __ldg(reinterpret_cast<const float4*>(a.norm_w + h));
      v = make_float4(v.x * inv * w.x, v.y * inv * w.y, v.z * inv * w.z, v.w * inv * w.w);
      v.x = __bfloat162float(__float2bfloat16_rn(v.x));
      v.y = __bfloat162float(__float2bfloat16_rn(v.y));
      v.z = __bfloat162float(__float2bfloat16_rn(v.z));
      v.w = __bfloat162float(__float2bfloat16_rn(v.w));
      *reinterpret_cast<float4*>(p) = v;
    }
    const uint32_t m = __reduce_max_sync(
        0xffffffffu, max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w))));
    const BlockScale s = block_scale(m);
    if (t < nt && h < a.H) {
      *reinterpret_cast<uint32_t*>(a.xq + (int64_t)(t0 + t) * a.H + h) =
          e4m3x4(v.x * s.inv, v.y * s.inv, v.z * s.inv, v.w * s.inv);
      if (lane == 0) a.xs[(int64_t)(h / kQB) * a.T + t0 + t] = s.scale;
    }
  }
  __syncthreads();
  // partial logits of this slice: four experts a warp, 8 tokens each
  for (int e0 = warp * 4; e0 < a.E; e0 += kWarps * 4) {
    float acc[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i] = 0.f;
#pragma unroll 2
    for (int b = 0; b < sb; ++b) {
      const int c = b * kQB + lane * 4;
      float4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (e0 + j < a.E && h0 + c < a.H) w[j] = load4(a.wr, a.wr_dtype, (int64_t)(e0 + j) * a.H + h0 + c);
      }
#pragma unroll
      for (int t = 0; t < kRouteTok; ++t) {
        if (t < nt) {
          const float4 v = *reinterpret_cast<const float4*>(xs + t * slice + c);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[j * 8 + t] =
                fmaf(v.w, w[j].w, fmaf(v.z, w[j].z, fmaf(v.y, w[j].y, fmaf(v.x, w[j].x, acc[j * 8 + t]))));
        }
      }
    }
    // 32 sums over 32 lanes: each step halves the values a lane still carries; lane l ends with sum l
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < o; ++i) {
        const float send = up ? acc[i] : acc[i + o];
        const float got = __shfl_xor_sync(0xffffffffu, send, o);
        acc[i] = (up ? acc[i + o] : acc[i]) + got;
      }
    }
    if (e0 + (lane >> 3) < a.E) part[e0 + (lane >> 3)][lane & 7] = acc[0];
  }
  cluster_sync();
  // softmax and top-k of token `rank`, one warp; ties go to the lowest index
  if (warp == 0 && (int)rank < nt) {
    constexpr int kPer = kFewMaxE / 32;
    float p[kPer];
    float mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      p[i] = -INFINITY;
      if (e < a.E) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < kRouteCtas; ++r) s += ld_peer(peer_addr(&part[e][rank], (uint32_t)r));
        p[i] = s;
      }
      mx = fmaxf(mx, p[i]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      p[i] = lane + 32 * i < a.E ? expf(p[i] - mx) : 0.f;
      sum += p[i];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // order by bits + 1 (probabilities are >= 0), 0 for no expert; a token whose logits are no numbers takes
    // experts 0 .. k-1 with weights that are none either
    const bool bad = !(sum < INFINITY);
    uint32_t key[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      p[i] = p[i] / sum;
      key[i] = lane + 32 * i < a.E ? (bad ? 1u : __float_as_uint(p[i]) + 1u) : 0u;
    }
    float mine = 0.f, wsum = 0.f;  // lane j: the weight of choice j
    int my_id = 0;
    for (int j = 0; j < a.k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      uint32_t id = 0xffffffffu;
#pragma unroll
      for (int i = kPer - 1; i >= 0; --i)
        if (key[i] == best) id = lane + 32 * i;
      id = __reduce_min_sync(0xffffffffu, id);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 32 * i == (int)id) key[i] = 0u;
      const float v = bad ? __uint_as_float(0x7fc00000u) : __uint_as_float(best - 1u);
      wsum += v;
      if (lane == j) mine = v, my_id = (int)id;
    }
    if (lane < a.k) {
      const int64_t s = (int64_t)lane * a.T + t0 + (int)rank;
      a.w[s] = a.normalize ? mine / wsum : mine;
      a.ids[s] = my_id;
    }
  }
  cluster_sync();  // the others' sums stay until they are read
}

// ------------------------------------------------------------- products --
// 16 weight rows times 8 tokens of one K block, one 64-byte half at a time.
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void to_half(const uint4& v, uint32_t (&h)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[2 * i] = e4m3x2_to_half2(w[i] & 0xffffu);
    h[2 * i + 1] = e4m3x2_to_half2(w[i] >> 16);
  }
}

// Weights are read once by one SM: past L1, first to leave L2.
__device__ __forceinline__ uint4 load_weights(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

constexpr int kGroups = kFewGroups;    // groups of 8 tokens taken at once
constexpr int kFewThreads = 256;

// acc[g][0..3] += (rows r0 and r1, this lane's two tokens of group g) over K blocks [b0, b1).
//   r0, r1      this lane's two weight rows (row g of the MMA and row g + 8)
//   s0, s1      their scales, one a K block
//   tok[g]      this lane's token row of group g for the product (lane / 4), or -1
//   col[g][2]   the rows of its two accumulator columns (2 (lane % 4) and the next), or -1
template <int G>
__device__ __forceinline__ void product(float (&acc)[G][4], const uint8_t* r0, const uint8_t* r1, const float* s0,
                                        const float* s1, const uint8_t* x, const float* x_scale, int64_t ld_scale,
                                        const int (&tok)[G], const int (&col)[G][2], int K, int b0, int b1) {
  constexpr int kBatch = G == 1 ? 4 : 2;  // K blocks under way a warp
  const int k_lane = (threadIdx.x & 3) * 16;
#pragma unroll 1
  for (int b = b0; b < b1; b += kBatch) {
    uint4 w0[kBatch][2], w1[kBatch][2];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = (b + i) * kQB + h * 64 + k_lane;
        w0[i][h] = w1[i][h] = make_uint4(0u, 0u, 0u, 0u);
        if (b + i < b1 && k < K) {
          w0[i][h] = load_weights(r0 + k);
          w1[i][h] = load_weights(r1 + k);
        }
      }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (b + i < b1) {
        float part[G][4] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = (b + i) * kQB + h * 64 + k_lane;
          uint32_t a0[8], a1[8];
          to_half(w0[i][h], a0);
          to_half(w1[i][h], a1);
#pragma unroll
          for (int g = 0; g < G; ++g) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (tok[g] >= 0 && k < K) v = *reinterpret_cast<const uint4*>(x + (int64_t)tok[g] * K + k);
            uint32_t t[8];
            to_half(v, t);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              mma_16816(part[g], a0[2 * j], a1[2 * j], a0[2 * j + 1], a1[2 * j + 1], t[2 * j], t[2 * j + 1]);
          }
        }
        const float f0 = __ldg(s0 + b + i), f1 = __ldg(s1 + b + i);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float* xs = x_scale + (int64_t)(b + i) * ld_scale;
          const float c0 = col[g][0] >= 0 ? xs[col[g][0]] : 0.f, c1 = col[g][1] >= 0 ? xs[col[g][1]] : 0.f;
          acc[g][0] = fmaf(part[g][0], c0 * f0, acc[g][0]);
          acc[g][1] = fmaf(part[g][1], c1 * f0, acc[g][1]);
          acc[g][2] = fmaf(part[g][2], c0 * f1, acc[g][2]);
          acc[g][3] = fmaf(part[g][3], c1 * f1, acc[g][3]);
        }
      }
    }
  }
}

// Expert id of a slot, inside [0, E) whatever the caller gave.
__device__ __forceinline__ int expert_of(const int32_t* ids, int s, int E) { return min(max(ids[s], 0), E - 1); }

// This unit's expert and its slots, ascending, in shared memory.  With no more slots than
// experts a unit is a slot and works if it is the first one of its expert;
// otherwise a unit is an expert.  Returns the number of slots, 0: nothing to do.
__device__ __forceinline__ int unit_slots(const FewArgs& a, int unit, int* slots, int* expert) {
  __shared__ int count;
  const int n = a.k * a.T, lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    const int e = n <= a.E ? expert_of(a.ids, unit, a.E) : unit;
    int c = 0;
    for (int base = 0; base < n; base += 32) {
      const int s = base + lane;
      const bool mine = s < n && expert_of(a.ids, s, a.E) == e;
      const uint32_t m = __ballot_sync(0xffffffffu, mine);
      if (mine) slots[c + __popc(m & ((1u << lane) - 1u))] = s;
      c += __popc(m);
    }
    __syncwarp();
    if (n <= a.E && slots[0] != unit) c = 0;
    if (lane == 0) count = c, *expert = e;
  }
  __syncthreads();
  return count;
}

template <int G>
__device__ __forceinline__ void lane_tokens(const int* slots, int c0, int c, int mod, int (&tok)[G], int (&col)[G][2]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int i = c0 + g * 8 + (lane >> 2), j = c0 + g * 8 + (lane & 3) * 2;
    tok[g] = i < c ? slots[i] % mod : -1;
    col[g][0] = j < c ? slots[j] % mod : -1;
    col[g][1] = j + 1 < c ? slots[j + 1] % mod : -1;
  }
}

// -------------------------------------------------------------- gate/up --
constexpr int kUpCtas = 4, kUpItems = 4;  // a CTA: 4 items of 8 columns of F, two warps each along K

template <int G>
__device__ __forceinline__ void up_chunk(const FewArgs& a, int e, const int* slots, int c0, int c, int fb,
                                         uint32_t rank, float (*red)[kGroups][4][32], uint32_t (*amax)[kFewChunk],
                                         uint32_t (*peers)[kFewChunk]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = warp >> 1, split = warp & 1;
  const int nbh = (a.H + kQB - 1) / kQB, nbf = (a.F + kQB - 1) / kQB;
  const int f = fb * kQB + (int)rank * 32 + item * 8 + (lane >> 2);
  const int64_t row = (int64_t)e * a.F + min(f, a.F - 1);
  int tok[G], col[G][2];
  lane_tokens<G>(slots, c0, c, a.T, tok, col);
  float acc[G][4] = {};
  const int half = (nbh + 1) / 2;
  const int64_t so = ((int64_t)e * nbf + fb) * nbh;
  product<G>(acc, a.w_gate + row * a.H, a.w_up + row * a.H, a.s_gate + so, a.s_up + so, a.xq, a.xs, a.T, tok, col,
             a.H, split * half, split ? nbh : half);
  // the second half of K, then h of 8 columns x this lane's two tokens a group
  if (split) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[item][g][i][lane] = acc[g][i];
  }
  __syncthreads();
  float h[G][2];
  if (!split) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[g][i] += red[item][g][i][lane];
      uint32_t m[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        h[g][i] = f < a.F ? acc[g][i] * silu_ref(acc[g][2 + i]) : 0.f;
        m[i] = abs_bits(h[g][i]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
        if (lane < 4) amax[item][g * 8 + lane * 2 + i] = m[i];
      }
    }
  }
  __syncthreads();
  if (c0 == 0) cluster_wait();
  if (threadIdx.x < G * 8 * kUpCtas) {
    const int t = threadIdx.x % (G * 8), to = threadIdx.x / (G * 8);
    uint32_t m = 0;
    for (int i = 0; i < kUpItems; ++i) m = max(m, amax[i][t]);
    st_peer(peer_addr(&peers[rank][t], (uint32_t)to), m);
  }
  cluster_sync();
  if (!split) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = g * 8 + (lane & 3) * 2 + i;
        if (c0 + t < c) {
          const BlockScale s = block_scale(max(max(peers[0][t], peers[1][t]), max(peers[2][t], peers[3][t])));
          const int slot = slots[c0 + t];
          if (f < a.F) {
            const float v = h[g][i] * s.inv;
            a.hq[(int64_t)slot * a.F + f] = (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
          }
          if (rank == 0 && item == 0 && lane < 4) a.hs[(int64_t)fb * a.k * a.T + slot] = s.scale;
        }
      }
  }
  cluster_sync();  // the maxima are read before the next chunk's arrive
}

__global__ void __launch_bounds__(kFewThreads, 2) few_up_kernel(const FewArgs a) {
  __shared__ int slots[kFewMaxSlots];
  __shared__ int expert;
  __shared__ float red[kUpItems][kGroups][4][32];
  __shared__ uint32_t amax[kUpItems][kFewChunk], peers[kUpCtas][kFewChunk];
  const uint32_t rank = cta_rank();
  const int nbf = (a.F + kQB - 1) / kQB;
  const int cluster = blockIdx.x / kUpCtas, unit = cluster / nbf, fb = cluster % nbf;
  pdl_wait();
  pdl_launch();
  const int c = unit_slots(a, unit, slots, &expert);
  if (c == 0) return;  // the whole cluster
  cluster_arrive();    // every CTA has started before its memory is written
  for (int c0 = 0; c0 < c; c0 += kFewChunk) {
    if (c - c0 <= 8) up_chunk<1>(a, expert, slots, c0, c, fb, rank, red, amax, peers);
    else up_chunk<kGroups>(a, expert, slots, c0, c, fb, rank, red, amax, peers);
  }
}

// ----------------------------------------------------------------- down --
// A CTA takes 128 / SPLIT rows of one expert's down matrix, SPLIT warps along K for each 16 rows.
template <int G, int SPLIT>
__device__ __forceinline__ void down_chunk(const FewArgs& a, int e, const int* slots, int c0, int c, int rb,
                                           float (*red)[kGroups][4][32]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = warp / SPLIT, split = warp % SPLIT;
  const int nbh = (a.H + kQB - 1) / kQB, nbf = (a.F + kQB - 1) / kQB;
  const int h = rb * (128 / SPLIT) + item * 16 + (lane >> 2);  // and h + 8
  const int64_t base = (int64_t)e * a.H;
  int tok[G], col[G][2];
  lane_tokens<G>(slots, c0, c, 0x7fffffff, tok, col);
  float acc[G][4] = {};
  const int per = (nbf + SPLIT - 1) / SPLIT;
  const float* sw = a.s_down + ((int64_t)e * nbh + min(h, a.H - 1) / kQB) * nbf;
  product<G>(acc, a.w_down + (base + min(h, a.H - 1)) * a.F, a.w_down + (base + min(h + 8, a.H - 1)) * a.F, sw, sw,
             a.hq, a.hs, (int64_t)a.k * a.T, tok, col, a.F, min(split * per, nbf), min((split + 1) * per, nbf));
  if (split) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[warp][g][i][lane] = acc[g][i];
  }
  __syncthreads();
  if (!split) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int s = 1; s < SPLIT; ++s) acc[g][i] += red[warp + s][g][i][lane];
        const int slot = col[g][i & 1], r = h + (i >> 1) * 8;
        if (slot >= 0 && r < a.H) a.d[(int64_t)slot * a.H + r] = acc[g][i] * a.w[slot];
      }
    }
  }
  __syncthreads();
}

template <int SPLIT>
__global__ void __launch_bounds__(kFewThreads, 2) few_down_kernel(const FewArgs a) {
  __shared__ int slots[kFewMaxSlots];
  __shared__ int expert;
  __shared__ float red[kFewThreads / 32][kGroups][4][32];
  const int nrb = (a.H + 128 / SPLIT - 1) / (128 / SPLIT);
  const int unit = blockIdx.x / nrb, rb = blockIdx.x % nrb;
  pdl_wait();
  pdl_launch();
  const int c = unit_slots(a, unit, slots, &expert);
  for (int c0 = 0; c0 < c; c0 += kFewChunk) {
    if (c - c0 <= 8) down_chunk<1, SPLIT>(a, expert, slots, c0, c, rb, red);
    else down_chunk<kGroups, SPLIT>(a, expert, slots, c0, c, rb, red);
  }
}

// Ids outside [0, E) are clamped where they are used; this records them.
__global__ void few_check_ids_kernel(const int32_t* ids, int n, int E, int32_t* err) {
  pdl_wait();
  pdl_launch();
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (ids[i] < 0 || ids[i] >= E) atomicExch(err, 1);
}

}  // namespace

namespace frank {

int launch_few_route(const FewRoute& a, cudaStream_t st) {
  const int nb = (a.H + kQB - 1) / kQB, slice = (nb + kRouteCtas - 1) / kRouteCtas * kQB;
  const size_t smem = (size_t)kRouteTok * slice * 4;
  FRANK_CUDA_TRY(cudaFuncSetAttribute(few_route_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)(kRouteTok * kNormMaxH / kRouteCtas * 4)));
  const dim3 grid((unsigned)((a.T + kRouteTok - 1) / kRouteTok * kRouteCtas));
  FRANK_CUDA_TRY(launch_chained(few_route_kernel, grid, dim3(kRouteThreads), smem, st, kRouteCtas, a));
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

int launch_few_experts(const FewArgs& a, int32_t* err, cudaStream_t st) {
  const int n = a.k * a.T, units = n <= a.E ? n : a.E;
  if (err != nullptr) {
    FRANK_CUDA_TRY(launch_chained(few_check_ids_kernel, dim3(1), dim3(256), 0, st, 1, a.ids, n, a.E, err));
    FRANK_LAUNCH_CHECK();
  }
  const unsigned nbf = (unsigned)q_blocks(a.F);
  FRANK_CUDA_TRY(
      launch_chained(few_up_kernel, dim3(units * nbf * kUpCtas), dim3(kFewThreads), 0, st, kUpCtas, a));
  FRANK_LAUNCH_CHECK();
  // long rows are split over all eight warps, so that a CTA's loads cover them sooner
  if (nbf >= 32) {
    FRANK_CUDA_TRY(
        launch_chained(few_down_kernel<8>, dim3(units * (unsigned)((a.H + 15) / 16)), dim3(kFewThreads), 0, st, 1, a));
  } else {
    FRANK_CUDA_TRY(
        launch_chained(few_down_kernel<2>, dim3(units * (unsigned)((a.H + 63) / 64)), dim3(kFewThreads), 0, st, 1, a));
  }
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

}  // namespace frank
