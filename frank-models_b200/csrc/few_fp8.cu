// The 8-bit MoE layer for a few tokens, bound by the expert weights in HBM:
// three launches chained by programmatic dependent launch (and the combine in
// norm.cu), without a permutation or a gather, each weight read once.
//
//   few_route   [norm,] quantisation, router, softmax and top-k: clusters of 8
//               CTAs take 8 tokens, each CTA an eighth of H.  The sums of squares and
//               the partial logits are exchanged through distributed shared memory
//               and added in CTA order.
//   few_up      h = gate * silu(up) for items of 8 columns of F of one expert; the
//               last of the 16 items of a quantisation block quantises it
//   few_down    d[slot] = route weight * down(h[slot]) for items of 16 rows of one expert
//
// few_up and few_down are persistent, 8 warps an SM.  A warp takes an item by itself: its
// weight rows come by TMA, 8 KB (16 rows x 512 values) a stage, three stages a warp,
// so 192 KB an SM are under way and no warp waits for another one.  A warp
// multiplies 16 weight rows (8 of gate and the same 8 of up, or 16 of down) with 8
// tokens by mma.m16n8k32 (e4m3, fp32 sums); one K block is summed and then
// scaled.  Lane t of a quad holds K elements 16 t .. 16 t + 15 of a row: the MMA's
// K index is permuted alike for weights and tokens, which leaves the sum.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "fp8.cuh"
#include "fp8_few.cuh"
#include "mbarrier.cuh"

namespace {
using namespace frank;
using namespace frank_mbar;

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
  if (a.wr != nullptr) {  // the router's slice does not wait for the stream's last kernel
    const int64_t esz = a.wr_dtype == FRANK_F32 ? 4 : 2;
    const int h0 = (int)rank * ((a.H + kQB * kRouteCtas - 1) / (kQB * kRouteCtas)) * kQB;
    const int h1 = min(h0 + (a.H + kQB * kRouteCtas - 1) / (kQB * kRouteCtas) * kQB, a.H);
    const int lines = (int)(((h1 - h0) * esz + 127) / 128);
    for (int i = threadIdx.x; i < a.E * lines; i += kRouteThreads)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(a.wr) +
                                                    ((int64_t)(i / lines) * a.H + h0) * esz + i % lines * 128));
  }
  const int nb = (a.H + kQB - 1) / kQB, sb = (nb + kRouteCtas - 1) / kRouteCtas;  // blocks of a row, of a slice
  const int slice = sb * kQB, h0 = (int)rank * slice;
  pdl_wait();
  pdl_launch();
  cluster_arrive();  // every CTA has started before its memory is written
  for (int i = blockIdx.x * kRouteThreads + threadIdx.x; i < a.n_count; i += gridDim.x * kRouteThreads) a.count[i] = 0;
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
  if (a.wr == nullptr) return;  // the routing is given
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
__device__ __forceinline__ void mma_16832(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kWarps = 8, kFewThreads = 32 * kWarps;
constexpr int kChunkK = 512, kChunkB = kChunkK / kQB;      // values and blocks along K of a stage
constexpr int kRows = 16, kStages = 3;
constexpr int kStageBytes = kRows * kChunkK;
static_assert(kFewMaxT <= 64, "an expert has at most 8 groups of 8 tokens");

struct FewMaps {
  CUtensorMap a, b;  // few_up: gate and up; few_down: down
};

// The routing as every CTA sees it: the experts that have tokens, ascending, and their slots.
struct Table {
  int nact;
  int expert[kFewMaxE];
  int start[kFewMaxE + 1];
  int slots[kFewMaxSlots];
  int tokens[kFewMaxSlots];  // of the slots
};

__device__ __forceinline__ void build_table(const FewArgs& a, Table& tb, int* sid, int* sums) {
  const int n = a.k * a.T, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int s = tid; s < n; s += kFewThreads) sid[s] = min(max(a.ids[s], 0), a.E - 1);
  __syncthreads();
  // thread e counts expert e
  int c = 0;
  for (int s = 0; s < n; ++s) c += sid[s] == tid;
  int v = c | (c != 0) << 16;  // slots and experts before this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  int before = v - (c | (c != 0) << 16), total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  if (c != 0) {
    int at = before & 0xffff;
    tb.expert[before >> 16] = tid;
    tb.start[before >> 16] = at;
    for (int s = 0; s < n; ++s)
      if (sid[s] == tid) tb.slots[at] = s, tb.tokens[at++] = s % a.T;
  }
  if (tid == 0) tb.nact = total >> 16, tb.start[total >> 16] = n;
  __syncthreads();
}

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int k8, int row, int e, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(k8), "r"(row), "r"(e), "r"(bar)
      : "memory");
}

// The stream of one warp's stages: item after item, chunk after chunk along K.  Lane 0
// issues the loads, three stages ahead; the warp that read a stage refills it.
//   UP: 8 rows of map a over 8 rows of map b; else ROWS rows of map a
template <bool UP, int ROWS>
struct Stream {
  const FewMaps* maps;
  const Table* tb;
  uint8_t* smem;      // this warp's stages
  uint32_t bar;       // this warp's barriers
  int items, per;     // items in all, items an expert
  int chunks;         // chunks of an item
  int next, chunk, step;
  uint32_t issued;

  __device__ __forceinline__ void issue() {
    if (next >= items) return;
    const uint32_t s = issued % kStages, dst = smem_u32(smem + s * kStageBytes), b = bar + 8 * s;
    const int e = tb->expert[next / per], i = next % per, k8 = chunk * (kChunkK / 8);
    mbar_expect_tx(b, (UP ? 16 : ROWS) * kChunkK);
    load_box(dst, &maps->a, k8, i * (UP ? 8 : ROWS), e, b);
    if (UP) load_box(dst + 8 * kChunkK, &maps->b, k8, i * 8, e, b);
    ++issued;
    if (++chunk == chunks) chunk = 0, next += step;
  }
};

// One stage: acc[g] += 16 rows x the tokens of group g over four blocks of K.
//   xp[g]: this lane's token row at its K elements of the first block, null: no token
//   sp[g][2]: scales of its two accumulator columns' rows at the first block, null: no column
//   FULL: all four blocks are whole; else left < 512 values of K are left
template <int G, int ROWS, bool FULL>
__device__ __forceinline__ void stage_product(float (&acc)[G][4], const uint8_t* st, const uint8_t* const (&xp)[G],
                                              const float* const (&sp)[G][2], uint32_t ld_scale, const float* s0,
                                              const float* s1, int left, uint32_t bar, uint32_t parity, bool& ok,
                                              volatile int* abort, int32_t* err) {
  const int lane = threadIdx.x & 31, k_lane = (lane & 3) * 16;
  // up to 16 tokens: everything but the weights is loaded before they are waited for
  constexpr bool kAhead = G <= 2;
  uint4 v[kAhead ? G : 1][kChunkB][2];
  float xs[kAhead ? G : 1][kChunkB][2], f0[kChunkB], f1[kChunkB];
  auto tokens = [&](int g, int i, uint4 (&q)[2], float (&sc)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      q[h] = make_uint4(0u, 0u, 0u, 0u);
      if (xp[g] != nullptr && (FULL || i * kQB + h * 64 + k_lane < left))
        q[h] = *reinterpret_cast<const uint4*>(xp[g] + i * kQB + h * 64);
      sc[h] = 0.f;
      if (sp[g][h] != nullptr && (FULL || i * kQB < left)) sc[h] = sp[g][h][i * ld_scale];
    }
  };
#pragma unroll
  for (int i = 0; i < kChunkB; ++i) {
    f0[i] = FULL || i * kQB < left ? __ldg(s0 + i) : 0.f;
    f1[i] = f0[i];
    if (s1 != s0) f1[i] = FULL || i * kQB < left ? __ldg(s1 + i) : 0.f;
    if (kAhead) {
#pragma unroll
      for (int g = 0; g < G; ++g) tokens(g, i, v[g][i], xs[g][i]);
    }
  }
  if (!mbar_wait_inline(bar, parity, abort, err)) ok = false;
  const uint8_t* w = st + (lane >> 2) * kChunkK + k_lane;
#pragma unroll
  for (int i = 0; i < kChunkB; ++i) {
    if (!FULL && i * kQB >= left) break;
    uint4 a0[2], a1[2] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      a0[h] = *reinterpret_cast<const uint4*>(w + i * kQB + h * 64);
      if (ROWS == 16) a1[h] = *reinterpret_cast<const uint4*>(w + 8 * kChunkK + i * kQB + h * 64);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float part[4] = {};
      uint4 q[2];
      float sc[2];
      if (!kAhead) tokens(g, i, q, sc);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 t = kAhead ? v[kAhead ? g : 0][i][h] : q[h];
        mma_16832(part, a0[h].x, a1[h].x, a0[h].y, a1[h].y, t.x, t.y);
        mma_16832(part, a0[h].z, a1[h].z, a0[h].w, a1[h].w, t.z, t.w);
      }
      const float x0 = kAhead ? xs[kAhead ? g : 0][i][0] : sc[0], x1 = kAhead ? xs[kAhead ? g : 0][i][1] : sc[1];
      acc[g][0] = fmaf(part[0], x0 * f0[i], acc[g][0]);
      acc[g][1] = fmaf(part[1], x1 * f0[i], acc[g][1]);
      acc[g][2] = fmaf(part[2], x0 * f1[i], acc[g][2]);
      acc[g][3] = fmaf(part[3], x1 * f1[i], acc[g][3]);
    }
  }
}

// One item: rows i * 8 .. of gate and up, or i * ROWS .. of down, of the ai-th active expert.
template <bool UP, int ROWS, int G>
__device__ __forceinline__ bool run_item(const FewArgs& a, const Table& tb, Stream<UP, ROWS>& sm, int ai, int i,
                                         uint32_t& it, volatile int* abort_flag) {
  const int lane = threadIdx.x & 31, n = a.k * a.T, K = UP ? a.H : a.F, N = UP ? a.F : a.H;
  const int nb = (K + kQB - 1) / kQB, nbn = (N + kQB - 1) / kQB;
  const int e = tb.expert[ai], c0 = tb.start[ai], c = tb.start[ai + 1] - c0;
  const int* rows = (UP ? tb.tokens : tb.slots) + c0;  // of the token operand
  const uint32_t ld = UP ? a.T : n;
  const uint8_t* xp[G];
  const float* sp[G][2];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int t = g * 8 + (lane >> 2), u = g * 8 + (lane & 3) * 2;
    xp[g] = t < c ? (UP ? a.xq : a.hq) + (int64_t)rows[t] * K + (lane & 3) * 16 : nullptr;
    sp[g][0] = u < c ? (UP ? a.xs : a.hs) + rows[u] : nullptr;
    sp[g][1] = u + 1 < c ? (UP ? a.xs : a.hs) + rows[u + 1] : nullptr;
  }
  const int64_t so = ((int64_t)e * nbn + i * (UP ? 8 : ROWS) / kQB) * nb;
  const float* s0 = (UP ? a.s_gate : a.s_down) + so;
  const float* s1 = (UP ? a.s_up : a.s_down) + so;
  float acc[G][4] = {};
  bool ok = true;
#pragma unroll 1
  for (int left = K; left > 0 && ok; left -= kChunkK, ++it) {
    const uint32_t s = it % kStages, parity = (it / kStages) & 1u;
    const uint8_t* st = sm.smem + s * kStageBytes;
    if (left >= kChunkK)
      stage_product<G, UP ? 16 : ROWS, true>(acc, st, xp, sp, ld, s0, s1, left, sm.bar + 8 * s, parity, ok, abort_flag,
                                             a.err);
    else
      stage_product<G, UP ? 16 : ROWS, false>(acc, st, xp, sp, ld, s0, s1, left, sm.bar + 8 * s, parity, ok,
                                              abort_flag, a.err);
    __syncwarp();
    if (lane == 0 && ok) sm.issue();
    s0 += kChunkB;
    s1 += kChunkB;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (xp[g] != nullptr) xp[g] += kChunkK;
      if (sp[g][0] != nullptr) sp[g][0] += kChunkB * ld;
      if (sp[g][1] != nullptr) sp[g][1] += kChunkB * ld;
    }
  }
  if (!ok) return false;
  if constexpr (UP) {
    // h of 8 columns: column lane / 4, this lane's two tokens of each group
    const int f = i * 8 + (lane >> 2), fb = i * 8 / kQB;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int t = g * 8 + (lane & 3) * 2 + j;
        if (t < c) a.h[(int64_t)tb.slots[c0 + t] * a.F + f] = acc[g][j] * silu_ref(acc[g][2 + j]);
      }
    __threadfence();
    __syncwarp();
    int old = 0;
    if (lane == 0) old = atomicAdd(a.count + (int64_t)e * nbn + fb, 1);
    old = __shfl_sync(0xffffffffu, old, 0);
    if (old == min(kQB / 8, sm.per - fb * (kQB / 8)) - 1) {
      // the block's last item: its 128 values of every slot, four a lane
      __threadfence();
      const int fq = fb * kQB + lane * 4;
#pragma unroll 4
      for (int t = 0; t < c; ++t) {
        const int slot = tb.slots[c0 + t];
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (fq < a.F) q = __ldcg(reinterpret_cast<const float4*>(a.h + (int64_t)slot * a.F + fq));
        const BlockScale sc = block_scale(__reduce_max_sync(
            0xffffffffu, max(max(abs_bits(q.x), abs_bits(q.y)), max(abs_bits(q.z), abs_bits(q.w)))));
        if (fq < a.F)
          *reinterpret_cast<uint32_t*>(a.hq + (int64_t)slot * a.F + fq) =
              e4m3x4(q.x * sc.inv, q.y * sc.inv, q.z * sc.inv, q.w * sc.inv);
        if (lane == 0) a.hs[(int64_t)fb * n + slot] = sc.scale;
      }
    }
  } else {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int t = g * 8 + (lane & 3) * 2 + j;
        if (t < c) {
          const int slot = tb.slots[c0 + t];
          const float w = a.w[slot];
          float* d = a.d + (int64_t)slot * a.H + i * ROWS + (lane >> 2);
          d[0] = acc[g][j] * w;
          if (ROWS == 16) d[8] = acc[g][2 + j] * w;
        }
      }
  }
  return true;
}

template <bool UP, int ROWS>
__global__ void __launch_bounds__(kFewThreads, 1)
few_product_kernel(const __grid_constant__ FewMaps maps, const __grid_constant__ FewArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  __shared__ Table tb;
  __shared__ int sid[kFewMaxSlots], sums[kWarps];
  __shared__ uint64_t bars[kWarps * kStages];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * kStages; ++i) mbar_init(smem_u32(&bars[i]), 1);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  pdl_wait();
  pdl_launch();
  build_table(a, tb, sid, sums);  // and the barriers are initialised

  // F and H are multiples of 16: no item is short
  const int K = UP ? a.H : a.F, N = UP ? a.F : a.H;
  Stream<UP, ROWS> sm;
  sm.maps = &maps;
  sm.tb = &tb;
  sm.smem = smem + warp * kStages * kStageBytes;
  sm.bar = smem_u32(&bars[warp * kStages]);
  sm.per = N / (UP ? 8 : ROWS);
  sm.items = tb.nact * sm.per;
  sm.chunks = (K + kChunkK - 1) / kChunkK;
  sm.step = gridDim.x * kWarps;
  sm.next = blockIdx.x + gridDim.x * warp;  // neighbouring items on different SMs
  sm.chunk = 0;
  sm.issued = 0;
  const int first = sm.next;
  if (lane == 0)
    for (int s = 0; s < kStages; ++s) sm.issue();
  uint32_t it = 0;
  bool ok = true;
  for (int item = first; item < sm.items && ok; item += sm.step) {
    const int ai = item / sm.per, i = item - ai * sm.per, c = tb.start[ai + 1] - tb.start[ai];
    if (c <= 8) ok = run_item<UP, ROWS, 1>(a, tb, sm, ai, i, it, abort_flag);
    else if (c <= 16) ok = run_item<UP, ROWS, 2>(a, tb, sm, ai, i, it, abort_flag);
    else if (c <= 32) ok = run_item<UP, ROWS, 4>(a, tb, sm, ai, i, it, abort_flag);
    else ok = run_item<UP, ROWS, 8>(a, tb, sm, ai, i, it, abort_flag);
  }
  if (!ok) {  // no copy may land after this CTA is gone; these waits are bounded too
    abort_word = 0;
    const uint32_t issued = __shfl_sync(0xffffffffu, sm.issued, 0);
    for (uint32_t s = it; s < issued; ++s)
      mbar_wait(sm.bar + 8 * (s % kStages), (s / kStages) & 1u, abort_flag, a.err);
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

// Map of e4m3 [E, N, K] as 8-byte elements, box 512 bytes x rows.
static int few_map(CUtensorMap* m, const void* base, int64_t E, int64_t N, int64_t K, uint32_t rows) {
  static PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  if (!enc) {
    set_error("cuTensorMapEncodeTiled unavailable");
    return FRANK_ECUDA;
  }
  const cuuint64_t dims[3] = {(cuuint64_t)K / 8, (cuuint64_t)N, (cuuint64_t)E};
  const cuuint64_t strides[2] = {(cuuint64_t)K, (cuuint64_t)(N * K)};
  const cuuint32_t box[3] = {kChunkK / 8, rows, 1}, estr[3] = {1, 1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_INT64, 3, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled([%lld, %lld, %lld] bytes) failed: %d", (long long)E, (long long)N, (long long)K,
              (int)r);
    return FRANK_ECUDA;
  }
  return FRANK_OK;
}

template <bool UP, int ROWS>
static int launch_few_product(const FewMaps& maps, const FewArgs& a, cudaStream_t st) {
  const size_t smem = 128 + (size_t)kWarps * kStages * kStageBytes;
  FRANK_CUDA_TRY(
      cudaFuncSetAttribute(few_product_kernel<UP, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  FRANK_CUDA_TRY(
      launch_chained(few_product_kernel<UP, ROWS>, dim3(num_sms()), dim3(kFewThreads), smem, st, 1, maps, a));
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

int launch_few_experts(const FewArgs& args, int32_t* err, cudaStream_t st) {
  FewArgs a = args;
  a.err = device_error_word();
  if (err != nullptr) {
    FRANK_CUDA_TRY(launch_chained(few_check_ids_kernel, dim3(1), dim3(256), 0, st, 1, a.ids, a.k * a.T, a.E, err));
    FRANK_LAUNCH_CHECK();
  }
  FewMaps up, down;
  FRANK_TRY(few_map(&up.a, a.w_gate, a.E, a.F, a.H, 8));
  FRANK_TRY(few_map(&up.b, a.w_up, a.E, a.F, a.H, 8));
  FRANK_TRY((launch_few_product<true, 16>(up, a, st)));
  // An item of 16 rows of 4096 values or more holds an SM's last warp too long: 8 rows then.
  const bool wide = a.F < 4096;
  FRANK_TRY(few_map(&down.a, a.w_down, a.E, a.H, a.F, wide ? 16 : 8));
  down.b = down.a;
  return wide ? launch_few_product<false, 16>(down, a, st) : launch_few_product<false, 8>(down, a, st);
}

}  // namespace frank
