// The 8-bit MoE layer for a few tokens, bound by the expert weights in HBM:
// three launches chained by programmatic dependent launch (and the combine in
// norm.cu), without a pass that sorts or copies rows: every CTA counts the slots by expert
// for itself and fetches the rows of its tiles.  A weight is read once for each 32 slots of
// its expert (16 where the call has at most 16 tokens): once for up to 32 tokens that each
// name an expert once, twice at most for 64.
//
//   few_route   [norm,] quantisation, router, softmax and top-k: clusters of 8
//               CTAs take 4 tokens, each CTA an eighth of H.  The sums of squares and
//               the partial logits are exchanged through distributed shared memory
//               and added in CTA order.
//   few_product<UP>    h = gate * silu(up), quantised: tiles of 128 columns of F (one
//               quantisation block) of one expert
//   few_product<DOWN>  d[slot] = route weight * down(h[slot]): tiles of 128 rows of H of
//               one expert
//
// Weights and tokens change places: the 128 weight rows are the M of
// tcgen05.mma.kind::f8f6f4 (UP: one MMA for gate, one for up), the expert's tokens, 16
// or 32 of them, its N.  So the weights go from TMA to the tensor core without passing
// through a register, and a K block of 128 costs the epilogue 16 or 32 columns: they
// are scaled and summed in fp32 registers from eight TMEM buffers.  The ring of K
// blocks keeps up to 190 KB an SM under way.  An MMA reads 128 weight rows in 80 ns
// whatever its N, so one SM draws 51 GB/s and all of them 7.5 TB/s: the K blocks have
// to be spread evenly over the SMs.  Where whole tiles would not, every SM takes the same
// number of K blocks in a row, and the last SM of a divided tile adds its partial sums
// in order.  (An earlier form multiplied in warps by mma.sync: 610 instructions for 8 KB
// of weights, 2.5 to 4 TB/s.)
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
// Of tensors that an earlier kernel may write while this one has started: not by __ldg, whose
// reads may come from a stale line and need not stay behind pdl_wait.
__device__ __forceinline__ float4 load4(const void* p, int dtype, int64_t i) {
  if (dtype == FRANK_F32) return __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
  const uint2 u = __ldcg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + i));
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}

// -------------------------------------------------------------- route --
constexpr int kRouteCtas = 8, kRouteTok = 4, kRouteThreads = 1024;

// PER: experts a lane of the top-k, E <= 32 PER
template <int PER>
__global__ void __launch_bounds__(kRouteThreads) few_route_kernel(const FewRoute a) {
  extern __shared__ float xs[];  // [tokens][slice]
  __shared__ float part[kRouteCtas][kFewMaxE];  // of this CTA's token, from every slice
  __shared__ float ssq_block[kRouteTok][16], ssq[kRouteCtas][kRouteTok];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kWarps = kRouteThreads / 32;
  const uint32_t rank = cta_rank();
  const int t0 = blockIdx.x / kRouteCtas * kRouteTok, nt = min(kRouteTok, a.T - t0);
  if (a.wr != nullptr) {  // the router's slice comes to L2 while the stream's last kernel ends
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
  // A warp's router weights: four experts, one block of columns a step, loaded two steps
  // ahead.
  const int steps = ((a.E + 4 * kWarps - 1) / (4 * kWarps)) * sb;
  auto router = [&](int q, float4 (&w)[4]) {
    const int e0 = (q / sb * kWarps + warp) * 4, c = h0 + q % sb * kQB + lane * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (q < steps && e0 + j < a.E && c < a.H) w[j] = load4(a.wr, a.wr_dtype, (int64_t)(e0 + j) * a.H + c);
    }
  };
  float4 w0[4], w1[4];
  pdl_wait();  // the stream's last kernel may have written the router too
  pdl_launch();
  if (a.wr != nullptr) router(0, w0), router(1, w1);
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
      const float4 w = load4(a.norm_w, FRANK_F32, h);
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
      if (lane == 0) a.xs[(int64_t)(h / kQB) * kFewMaxT + t0 + t] = s.scale;
    }
  }
  if (a.wr == nullptr) return;  // the routing is given
  __syncthreads();
  // partial logits of this slice: four experts a warp, four tokens each; the sums go to the token's CTA
  constexpr int kSums = 4 * kRouteTok;
  float acc[kSums] = {};
  auto step = [&](int q, const float4 (&w)[4]) {
    if (q >= steps) return;
    const int b = q % sb;
#pragma unroll
    for (int t = 0; t < kRouteTok; ++t) {
      if (t < nt) {
        const float4 v = *reinterpret_cast<const float4*>(xs + t * slice + b * kQB + lane * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[j * kRouteTok + t] =
              fmaf(v.w, w[j].w, fmaf(v.z, w[j].z, fmaf(v.y, w[j].y, fmaf(v.x, w[j].x, acc[j * kRouteTok + t]))));
      }
    }
    if (b < sb - 1) return;
    // kSums sums over the lanes: each step halves the values a lane still carries; lane l ends
    // with sum l % kSums of half a warp, and the last step adds the halves
#pragma unroll
    for (int o = kSums / 2; o; o >>= 1) {
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < o; ++i) {
        const float send = up ? acc[i] : acc[i + o];
        const float got = __shfl_xor_sync(0xffffffffu, send, o);
        acc[i] = (up ? acc[i + o] : acc[i]) + got;
      }
    }
    const float sum = acc[0] + __shfl_xor_sync(0xffffffffu, acc[0], 16);
    const int e = (q / sb * kWarps + warp) * 4 + (lane & (kSums - 1)) / kRouteTok, t = lane & (kRouteTok - 1);
    if (lane < kSums && e < a.E && t < nt) st_peer(peer_addr(&part[rank][e], (uint32_t)t), __float_as_uint(sum));
#pragma unroll
    for (int i = 0; i < kSums; ++i) acc[i] = 0.f;
  };
  static_assert(kSums == 16, "half a warp holds the sums");
#pragma unroll 1
  for (int q = 0; q < steps; q += 2) {
    step(q, w0);
    router(q + 2, w0);
    step(q + 1, w1);
    router(q + 3, w1);
  }
  cluster_sync();
  // softmax and top-k of token `rank`, one warp; ties go to the lowest index
  if (warp == 0 && (int)rank < nt) {
    float p[PER];
    float mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 32 * i;
      p[i] = -INFINITY;
      if (e < a.E) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < kRouteCtas; ++r) s += part[r][e];
        p[i] = s;
      }
      mx = fmaxf(mx, p[i]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      p[i] = lane + 32 * i < a.E ? expf(p[i] - mx) : 0.f;
      sum += p[i];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // order by bits + 1 (probabilities are >= 0), 0 for no expert; a token whose logits are no numbers takes
    // experts 0 .. k-1 with weights that are none either
    const bool bad = !(sum < INFINITY);
    const float inv = 1.f / sum;
    uint32_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      p[i] *= inv;
      key[i] = lane + 32 * i < a.E ? (bad ? 1u : __float_as_uint(p[i]) + 1u) : 0u;
    }
    float mine = 0.f, wsum = 0.f;  // lane j: the weight of choice j
    int my_id = 0;
    for (int j = 0; j < a.k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      uint32_t id = 0xffffffffu;
#pragma unroll
      for (int i = PER - 1; i >= 0; --i)
        if (key[i] == best) id = lane + 32 * i;
      id = __reduce_min_sync(0xffffffffu, id);
#pragma unroll
      for (int i = 0; i < PER; ++i)
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
}

// ------------------------------------------------------------- products --
// warp 0: TMA, warp 1: MMA, warp 2: scales of h (DOWN), warp 3: token rows and their scales
// (UP), warps 4..7 and 8..11: epilogue of every other tile
constexpr int kFewThreads = 384, kGroupWarps = 4;
constexpr uint32_t kTile = 128 * kQB;  // bytes of 128 weight rows of a K block
// TMEM buffers and scale slots: half of them for each epilogue group, which then sees every
// phase of its barriers (a wait by parity must not miss one)
constexpr int kMaxStages = 12, kBufs = 8, kGroupBufs = 4, kBufCols = 64, kScaleSlots = 16, kGroupSlots = 8;
constexpr int kMaxTokens = 32;  // of a tile
constexpr uint32_t kTmemCols = kBufs * kBufCols;

struct FewMaps {
  CUtensorMap w, w2;  // UP: gate and up; DOWN: down (boxes of 128 rows)
  CUtensorMap x[2];   // DOWN: rows of h, boxes of 16 and 32
};

// The slots that a tile takes at once.
__host__ __device__ __forceinline__ int tile_tokens(int T) { return T <= 16 ? 16 : kMaxTokens; }

// The routing as every CTA sees it: the experts that have tokens, ascending, and their
// slots, at most tile_tokens an entry.  An entry's rows of h start at a multiple of 16.
constexpr int kMaxEntries = kFewMaxE + kFewMaxSlots / 16;
struct Table {
  int entries;
  int expert[kMaxEntries];
  int first[kMaxEntries + 1];  // of its slots
  int row[kMaxEntries];        // of h
  int slots[kFewMaxSlots];
  int tokens[kFewMaxSlots];    // of the slots
};

// A stable counting sort of the slots: ranks inside 32 slots by a warp match, one thread
// an expert adds up the chunks.  at: scratch [kFewMaxSlots / 32][kFewMaxE].
__device__ __forceinline__ void build_table(const FewArgs& a, Table& tb, uint16_t (*at)[kFewMaxE], int* sums) {
  const int n = a.k * a.T, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kWarps = kFewMaxE / 32, kChunks = kFewMaxSlots / 32;  // of the threads that work here
  static_assert(kFewThreads >= kFewMaxE && kChunks == 2 * kWarps, "a thread an expert, two chunks a warp");
  const bool works = tid < kFewMaxE;
  const int chunks = (n + 31) / 32;
  int id[2], rank[2], size[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = (warp + i * kWarps) * 32 + lane;
    id[i] = works && s < n ? min(max(__ldcg(a.ids + s), 0), a.E - 1) : -1;
  }
  if (works)
    for (int c = 0; c < chunks; ++c) at[c][tid] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t m = __match_any_sync(0xffffffffu, id[i]);
    rank[i] = __popc(m & ((1u << lane) - 1u));
    size[i] = __popc(m);
    if (id[i] >= 0 && rank[i] == 0) at[warp + i * kWarps][id[i]] = (uint16_t)size[i];
  }
  __syncthreads();
  int c = 0;
  if (works)
    for (int i = 0; i < chunks; ++i) {
      const int t = at[i][tid];
      at[i][tid] = (uint16_t)c;
      c += t;
    }
  // before this expert: slots (bits 0..9), entries (10..18) and groups of 16 rows (19..)
  const int cap = tile_tokens(a.T), mine = c | (c + cap - 1) / cap << 10 | (c + 15) / 16 << 19;
  int v = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (works && lane == 31) sums[warp] = v;
  __syncthreads();
  int before = v - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  const int first = before & 1023;
  for (int i = 0; i * cap < c; ++i) {
    const int entry = (before >> 10 & 511) + i;
    tb.expert[entry] = tid;
    tb.first[entry] = first + i * cap;
    tb.row[entry] = (before >> 19) * 16 + i * cap;
  }
  if (c != 0)
    for (int i = 0; i < chunks; ++i) at[i][tid] += (uint16_t)first;
  if (tid == 0) tb.entries = total >> 10 & 511, tb.first[total >> 10 & 511] = n;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (id[i] >= 0) {
      const int s = (warp + i * kWarps) * 32 + lane, p = at[warp + i * kWarps][id[i]] + rank[i];
      tb.slots[p] = s;
      tb.tokens[p] = s % a.T;
    }
  }
}

__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// Weights are read once: first to leave L2.
__device__ __forceinline__ void load_weights(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar,
                                             uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, "
      "%4}], [%5], %6;" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// K-major operand, 128-byte swizzle: rows of 128 bytes, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// After the wait: keeps what uses the values behind it.
template <int N>
__device__ __forceinline__ void pin(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

// A CTA's way through the K blocks of all tiles (entry after entry, tile after tile):
// every gridDim.x-th whole tile, or an equal run of K blocks that may begin and end
// inside a tile.
// Where it stands: tile n (128 rows) of entry ai, K blocks [kb0, kb1()).
struct Walk {
  int nb, tiles, ai, n, kb0, todo, dai, dn;  // todo: K blocks; dai, dn: the step to the next tile

  // slack: K blocks that a CTA may have more than the mean before tiles are divided
  __device__ __forceinline__ Walk(int entries, int tiles_, int nb_, int slack) : nb(nb_), tiles(tiles_) {
    const int G = gridDim.x, all = entries * tiles, total = all * nb, b = blockIdx.x;
    const bool whole = total < G || (all + G - 1) / G * nb - total / G <= slack;  // a run is never empty
    const int first = whole ? b : start(b, total) / nb;
    kb0 = whole ? 0 : start(b, total) - first * nb;
    todo = whole ? (b < all ? (all - b + G - 1) / G * nb : 0) : start(b + 1, total) - start(b, total);
    ai = first / tiles;
    n = first - ai * tiles;
    dai = whole ? G / tiles : 0;
    dn = whole ? G - dai * tiles : 1;
  }
  static __device__ __forceinline__ int start(int cta, int total) {
    const int q = total / (int)gridDim.x;
    return cta * q + min(cta, total - q * (int)gridDim.x);
  }
  // The CTA whose run holds K block x (no run is empty).
  static __device__ __forceinline__ int cta_of(int x, int total) {
    const int q = total / (int)gridDim.x, r = total - q * (int)gridDim.x;
    return x < r * (q + 1) ? x / (q + 1) : r + (x - r * (q + 1)) / q;
  }
  __device__ __forceinline__ bool more() const { return todo > 0; }
  __device__ __forceinline__ int kb1() const { return min(nb, kb0 + todo); }
  __device__ __forceinline__ void advance() {
    todo -= kb1() - kb0;
    kb0 = 0;
    ai += dai;
    n += dn;
    if (n >= tiles) n -= tiles, ++ai;
  }
};

// A stage of the ring and the parity of its barriers.
struct Ring {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) s = 0, phase ^= 1u;
  }
};

// K blocks of the tiles of each epilogue group so far; tiles alternate.
struct Turns {
  uint32_t mine = 0, other = 0;
  int group = 0;
  __device__ __forceinline__ uint32_t buf() const { return group * kGroupBufs + mine % kGroupBufs; }
  __device__ __forceinline__ uint32_t buf_parity() const { return mine / kGroupBufs & 1u; }
  __device__ __forceinline__ uint32_t slot() const { return group * kGroupSlots + mine % kGroupSlots; }
  __device__ __forceinline__ uint32_t slot_parity() const { return mine / kGroupSlots & 1u; }
  __device__ __forceinline__ void next_tile() {
    const uint32_t t = mine;
    mine = other;
    other = t;
    group ^= 1;
  }
};

template <bool UP>
__global__ void __launch_bounds__(kFewThreads, 1)
few_product_kernel(const __grid_constant__ FewMaps maps, const __grid_constant__ FewArgs a, int stages,
                   uint32_t stage_bytes) {
  constexpr int kSums = UP ? 256 : 128;  // of a column: 128 rows of gate and of up, or of down
  constexpr uint32_t kWeights = (UP ? 2 : 1) * kTile;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Table tb;
  __shared__ int sums[kFewMaxE / 32];
  __shared__ uint64_t bars[2 * kMaxStages + 2 * kBufs + 2 * kScaleSlots + 2];
  __shared__ alignas(128) float scales[kScaleSlots][kMaxTokens];  // of the tokens, a slot for each K block
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word, last_word[2];
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  auto tfull_bar = [&](int b) { return bar0 + 8u * (2 * kMaxStages + b); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * kMaxStages + kBufs + b); };
  auto sfull_bar = [&](int i) { return bar0 + 8u * (2 * kMaxStages + 2 * kBufs + i); };
  auto sempty_bar = [&](int i) { return bar0 + 8u * (2 * kMaxStages + 2 * kBufs + kScaleSlots + i); };
  auto tile_bar = [&](int g) { return bar0 + 8u * (2 * kMaxStages + 2 * kBufs + 2 * kScaleSlots + g); };
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), UP ? 2 : 1);  // the bytes of TMA; UP: and the rows of warp 3
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), kGroupWarps);
    }
    for (int i = 0; i < kScaleSlots; ++i) {
      mbar_init(sfull_bar(i), 1);
      mbar_init(sempty_bar(i), kGroupWarps);
    }
    for (int g = 0; g < 2; ++g) mbar_init(tile_bar(g), kGroupWarps);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // DOWN needs nothing of UP but h.  Its table, route weights and first expert weights are read
  // before its own wait, which is more than the model promises (visibility of an earlier grid's
  // writes after griddepcontrol.wait alone).  What it relies on: every CTA of UP lets this kernel
  // start (launch_dependents) only after its own wait has returned, so the routing's grid, and all
  // before it, were complete and in L2 when the first CTA here began; and ids and route weights are
  // read past L1 (__ldcg).  Ids are clamped, so no value of them leads out of the buffers.  With a wait here
  // as in UP: one token 34.1 instead of 32.4 us, 47 tokens 130 instead of 124.
  if (UP) pdl_wait();
  pdl_launch();
  build_table(a, tb, reinterpret_cast<uint16_t(*)[kFewMaxE]>(smem), sums);
  fence_proxy_async_smem();  // the scratch becomes the ring
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;

  const int K = UP ? a.H : a.F, N = UP ? a.F : a.H;
  const int nb = (K + kQB - 1) / kQB, tiles = (N + kQB - 1) / kQB;
  // dividing a tile costs about 3 us: 5 K blocks of UP, 10 of DOWN
  const Walk walk(tb.entries, tiles, nb, UP ? 5 : 10);
  auto tokens_of = [&](const Walk& t) { return tb.first[t.ai + 1] - tb.first[t.ai]; };

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer --
      uint64_t policy;
      asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
      Ring r;
      bool ok = true;
      // One K block: the weights, and DOWN's rows of h.
      auto weights = [&](int e, int n, int kb, uint32_t x_bytes) {
        const uint32_t st = smem_u32(smem + r.s * stage_bytes);
        mbar_expect_tx(full_bar(r.s), kWeights + x_bytes);
        load_weights(st, &maps.w, kb * kQB, n * 128, e, full_bar(r.s), policy);
        if (UP) load_weights(st + kTile, &maps.w2, kb * kQB, n * 128, e, full_bar(r.s), policy);
      };
      auto rows = [&](int s, int box, int kb, int row) {
        load_2d(smem_u32(smem + s * stage_bytes) + kWeights, &maps.x[box], kb * kQB, row, full_bar(s));
      };
      Walk t = walk;
      int kb = t.kb0;
      if (!UP) {
        // the ring is filled with weights, its rows of h follow when they are there
        int n = 0;
        for (; t.more() && n < stages;) {
          weights(tb.expert[t.ai], t.n, kb, tokens_of(t) <= 16 ? 16 * kQB : 32 * kQB);
          r.next(stages);
          ++n;
          if (++kb == t.kb1()) t.advance(), kb = 0;
        }
        pdl_wait();
        Walk u = walk;
        for (int m = 0, ukb = u.kb0; m < n; ++m) {
          rows(m, tokens_of(u) <= 16 ? 0 : 1, ukb, tb.row[u.ai]);
          if (++ukb == u.kb1()) u.advance(), ukb = 0;
        }
      }
      for (; t.more() && ok; t.advance(), kb = 0) {
        const int e = tb.expert[t.ai], box = tokens_of(t) <= 16 ? 0 : 1, row = tb.row[t.ai];
        for (const int kb1 = t.kb1(); kb < kb1; ++kb, r.next(stages)) {
          if (!mbar_wait_inline(empty_bar(r.s), r.phase ^ 1u, abort_flag, a.err)) {
            ok = false;
            break;
          }
          weights(e, t.n, kb, UP ? 0 : (16u << box) * kQB);
          if (!UP) rows(r.s, box, kb, row);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // -------------------------------------------------- MMA issuer --
      Ring r;
      Turns turn;
      bool ok = true;
      for (Walk t = walk; t.more() && ok; t.advance(), turn.next_tile()) {
        // kind::f8f6f4: D fp32, A and B e4m3, N >> 3 at [17,23), M >> 4 at [24,29)
        const uint32_t cols = tokens_of(t) <= 16 ? 16 : 32;
        const uint32_t idesc = (1u << 4) | (cols >> 3 << 17) | ((uint32_t)(128 >> 4) << 24);
        for (int kb = t.kb0, kb1 = t.kb1(); kb < kb1; ++kb, r.next(stages), ++turn.mine) {
          const int s = r.s, b = turn.buf();
          if (!mbar_wait_inline(tempty_bar(b), turn.buf_parity() ^ 1u, abort_flag, a.err) ||
              !mbar_wait_inline(full_bar(s), r.phase, abort_flag, a.err)) {
            ok = false;
            break;
          }
          fence_after();
          const uint32_t st = smem_u32(smem + s * stage_bytes);
          const uint64_t wd = smem_desc(st), w2d = smem_desc(st + kTile), xd = smem_desc(st + kWeights);
#pragma unroll
          for (int j = 0; j < kQB / 32; ++j) {  // 32 bytes along K inside the swizzled row
            mma(tmem + b * kBufCols, wd + (uint64_t)(2 * j), xd + (uint64_t)(2 * j), idesc, j != 0);
            if (UP)
              mma(tmem + b * kBufCols + kMaxTokens, w2d + (uint64_t)(2 * j), xd + (uint64_t)(2 * j), idesc, j != 0);
          }
          commit(empty_bar(s));
          commit(tfull_bar(b));
        }
      }
    }
  } else if (warp == 2) {
    if (!UP && lane == 0) {
      // --------------------------------------------- scales of h --
      pdl_wait();
      Turns turn;
      bool ok = true;
      for (Walk t = walk; t.more() && ok; t.advance(), turn.next_tile()) {
        const float* src = a.hs + tb.row[t.ai];
        const uint32_t bytes = (tokens_of(t) + 15) / 16 * 64;
        for (int kb = t.kb0, kb1 = t.kb1(); kb < kb1; ++kb, ++turn.mine) {
          const int i = turn.slot();
          if (!mbar_wait_inline(sempty_bar(i), turn.slot_parity() ^ 1u, abort_flag, a.err)) {
            ok = false;
            break;
          }
          mbar_expect_tx(sfull_bar(i), bytes);
          bulk_load(smem_u32(scales[i]), src + (int64_t)kb * a.h_rows, bytes, sfull_bar(i));
        }
      }
    }
  } else if (warp == 3) {
    if (UP) {
      // ------------------------------- token rows and their scales --
      // 16 bytes a lane, eight lanes a row, into the swizzled tile; three K blocks under way
      constexpr int kAhead = 3;
      const int r0 = lane >> 3, chunk = lane & 7;
      uint32_t under_way = 0;
      Ring r, first;  // of the next K block, of the oldest one under way
      int slots_under_way[kAhead] = {};  // their scale slots, the oldest first
      Turns turn;
      bool ok = true;
      auto arrive = [&]() {  // the oldest K block is in shared memory
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full_bar(first.s)), mbar_arrive(sfull_bar(slots_under_way[0]));
        first.next(stages);
        --under_way;
#pragma unroll
        for (int i = 0; i + 1 < kAhead; ++i) slots_under_way[i] = slots_under_way[i + 1];
      };
      for (Walk t = walk; t.more() && ok; t.advance(), turn.next_tile()) {
        const int c = tokens_of(t), *tok = tb.tokens + tb.first[t.ai];
        for (int kb = t.kb0, kb1 = t.kb1(); kb < kb1; ++kb, ++turn.mine) {
          const int s = r.s, i = turn.slot();
          if (!mbar_wait_inline(empty_bar(s), r.phase ^ 1u, abort_flag, a.err) ||
              !mbar_wait_inline(sempty_bar(i), turn.slot_parity() ^ 1u, abort_flag, a.err)) {
            ok = false;
            break;
          }
          const uint32_t st = smem_u32(smem + s * stage_bytes) + kWeights;
          const int k = kb * kQB + chunk * 16;
          for (int q = r0; q < c; q += 4) {
            const uint8_t* src = a.xq + (int64_t)tok[q] * a.H + (k < a.H ? k : 0);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(st + q * kQB + ((chunk ^ (q & 7)) << 4)),
                         "l"(src), "r"(k < a.H ? 16 : 0)
                         : "memory");
          }
          if (lane < c)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&scales[i][lane])),
                         "l"(a.xs + (int64_t)kb * kFewMaxT + tok[lane])
                         : "memory");
          asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
          for (int q = 0; q < kAhead; ++q)
            if (q == (int)under_way) slots_under_way[q] = i;
          r.next(stages);
          if (++under_way >= kAhead) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
            arrive();
          }
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      while (ok && under_way > 0) arrive();
    }
  } else {
    // ---------------------------------------------------- epilogue --
    const int quad = warp & 3, group = (warp - 4) >> 2;
    const int row = quad * 32 + lane;  // this thread's weight row of the tile
    const uint32_t my_tmem = tmem + ((uint32_t)(quad * 32) << 16);
    float* sums_buf = reinterpret_cast<float*>(smem + stages * stage_bytes) + group * 16 * kSums;
    uint32_t it = 0, meets = 0;  // K blocks of this group's tiles
    bool ok = true;
    // the four warps of a group meet (bounded, unlike a named barrier)
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(tile_bar(group));
      if (!mbar_wait_inline(tile_bar(group), meets++ & 1u, abort_flag, a.err)) ok = false;
    };
    int turn = 0;
    for (Walk t = walk; t.more() && ok; t.advance()) {
      const int kb1 = t.kb1();
      if ((turn++ & 1) != group) continue;  // the other group's tile
      const int f = tb.first[t.ai], c = tokens_of(t);
      // scales of the weights: lane l holds those of K block kb0 + l, of 32 at a time
      const int64_t so = ((int64_t)tb.expert[t.ai] * tiles + t.n) * nb + lane;
      float w0s = 0.f, w1s = 0.f;
      auto weight_scales = [&](int kb) {
        w0s = kb + lane < kb1 ? __ldg((UP ? a.s_gate : a.s_down) + so + kb) : 0.f;
        if (UP) w1s = kb + lane < kb1 ? __ldg(a.s_up + so + kb) : 0.f;
      };
      weight_scales(t.kb0);
      const float route_w = !UP && lane < c ? __ldcg(a.w + tb.slots[f + lane]) : 0.f;
      float acc[UP ? 2 : 1][2][16] = {};
      // Two K blocks at a time where there are two: one round of waits and TMEM loads for both.
#pragma unroll 1
      for (int kb = t.kb0; kb < kb1;) {
        const int l = kb - t.kb0 & 31, two = l < 31 && kb + 1 < kb1;
        if (l == 0 && kb > t.kb0) weight_scales(kb);
        const uint32_t itl = it + two;
        const int b0 = group * kGroupBufs + it % kGroupBufs, b1 = group * kGroupBufs + itl % kGroupBufs;
        const int i0 = group * kGroupSlots + it % kGroupSlots, i1 = group * kGroupSlots + itl % kGroupSlots;
        if (!mbar_wait_inline(sfull_bar(i0), it / kGroupSlots & 1u, abort_flag, a.err) ||
            !mbar_wait_inline(sfull_bar(i1), itl / kGroupSlots & 1u, abort_flag, a.err) ||
            !mbar_wait_inline(tfull_bar(b0), it / kGroupBufs & 1u, abort_flag, a.err) ||
            !mbar_wait_inline(tfull_bar(b1), itl / kGroupBufs & 1u, abort_flag, a.err)) {
          ok = false;
          break;
        }
        fence_after();
        const float w00 = __shfl_sync(0xffffffffu, w0s, l), w01 = __shfl_sync(0xffffffffu, w0s, l + two);
        const float w10 = UP ? __shfl_sync(0xffffffffu, w1s, l) : 0.f;
        const float w11 = UP ? __shfl_sync(0xffffffffu, w1s, l + two) : 0.f;
        const uint32_t t0 = my_tmem + b0 * kBufCols, t1 = my_tmem + b1 * kBufCols;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (g == 0 || c > 16) {
            uint32_t v[2][UP ? 2 : 1][16];
            tmem_ld16(t0 + g * 16, v[0][0]);
            if constexpr (UP) tmem_ld16(t0 + kMaxTokens + g * 16, v[0][UP ? 1 : 0]);
            if (two) {
              tmem_ld16(t1 + g * 16, v[1][0]);
              if constexpr (UP) tmem_ld16(t1 + kMaxTokens + g * 16, v[1][UP ? 1 : 0]);
            }
            auto add = [&](const uint32_t (&u)[UP ? 2 : 1][16], const float* sc, float f0, float f1) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float4 s = *reinterpret_cast<const float4*>(sc + g * 16 + 4 * q);
                const float s4[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  acc[0][g][4 * q + j] = fmaf(__uint_as_float(u[0][4 * q + j]), s4[j] * f0, acc[0][g][4 * q + j]);
                  if constexpr (UP)
                    acc[UP ? 1 : 0][g][4 * q + j] =
                        fmaf(__uint_as_float(u[UP ? 1 : 0][4 * q + j]), s4[j] * f1, acc[UP ? 1 : 0][g][4 * q + j]);
                }
              }
            };
            tmem_wait();
            pin(v[0][0]), pin(v[0][UP ? 1 : 0]);
            add(v[0], scales[i0], w00, w10);
            if (two) {
              pin(v[1][0]), pin(v[1][UP ? 1 : 0]);
              add(v[1], scales[i1], w01, w11);
            }
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(tempty_bar(b0)), mbar_arrive(sempty_bar(i0));
          if (two) mbar_arrive(tempty_bar(b1)), mbar_arrive(sempty_bar(i1));
        }
        kb += 1 + two;
        it += 1 + two;
      }
      if (!ok) break;
      // this thread's sums of columns [16 g, c) and on, a column after the other
      auto put = [&](float* to, int g, const float (&v)[16], const float (&v2)[16]) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (g * 16 + i < c) {
            to[i * kSums] = v[i];
            if (UP) to[i * kSums + 128] = v2[i];
          }
      };
      // What becomes of the four sums (UP: of gate and of up) that a lane has of slot i: h, quantised, or d.
      const int col = t.n * 128 + lane * 4;
      const bool in = col < N;
      auto finish = [&](int i, const float4& g, const float4& p) {
        if constexpr (UP) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (in) v = make_float4(g.x * silu(p.x), g.y * silu(p.y), g.z * silu(p.z), g.w * silu(p.w));
          const BlockScale s = block_scale(__reduce_max_sync(
              0xffffffffu, max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)))));
          const int64_t r = tb.row[t.ai] + i;
          if (in)
            *reinterpret_cast<uint32_t*>(a.hq + r * a.F + col) =
                e4m3x4(v.x * s.inv, v.y * s.inv, v.z * s.inv, v.w * s.inv);
          if (lane == 0) a.hs[(int64_t)t.n * a.h_rows + r] = s.scale;
        } else {
          const float r = __shfl_sync(0xffffffffu, route_w, i);
          if (in)
            *reinterpret_cast<float4*>(a.d + (int64_t)tb.slots[f + i] * a.H + col) =
                make_float4(g.x * r, g.y * r, g.z * r, g.w * r);
        }
      };
      if (kb1 - t.kb0 < nb) {
        // A divided tile: its partial sums go to this CTA's place, the last CTA of the
        // tile adds all of them in order.  A CTA has two divided tiles at most, the
        // one its run begins in and the one it ends in.
        const int total = tb.entries * tiles * nb, tile = t.ai * tiles + t.n, from = tile * nb;
        const int cta0 = Walk::cta_of(from, total), cta1 = Walk::cta_of(from + nb - 1, total);
        auto place = [&](int cta) {
          return a.partial + (2 * cta + (Walk::start(cta, total) >= from ? 0 : 1)) * a.partial_stride;
        };
        float* mine = place(blockIdx.x) + row;
        put(mine, 0, acc[0][0], acc[UP ? 1 : 0][0]);
        if (c > 16) put(mine + 16 * kSums, 1, acc[0][1], acc[UP ? 1 : 0][1]);
        __threadfence();
        meet();
        if (!ok) break;
        if (quad == 0 && lane == 0) {
          last_word[group] = atomicAdd(a.count + (UP ? 0 : a.n_count / 2) + tile, 1) == cta1 - cta0;
          __threadfence();
        }
        meet();
        if (!ok) break;
        if (!*reinterpret_cast<volatile int*>(&last_word[group])) continue;
        for (int i = quad; i < c; i += 4) {
          float4 g = make_float4(0.f, 0.f, 0.f, 0.f), p = g;
#pragma unroll 4
          for (int cta = cta0; cta <= cta1; ++cta) {
            const float4* q = reinterpret_cast<const float4*>(place(cta) + i * kSums) + lane;
            const float4 u = __ldcg(q);
            g = make_float4(g.x + u.x, g.y + u.y, g.z + u.z, g.w + u.w);
            if (UP) {
              const float4 v = __ldcg(q + 32);
              p = make_float4(p.x + v.x, p.y + v.y, p.z + v.z, p.w + v.w);
            }
          }
          finish(i, g, p);
        }
      } else {
        // 16 columns at a time through shared memory: a warp then has the 128 sums of a slot
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (g * 16 < c && ok) {
            put(sums_buf + row, g, acc[0][g], acc[UP ? 1 : 0][g]);
            meet();
            if (!ok) break;
#pragma unroll 1
            for (int i = quad; i < min(16, c - g * 16); i += 4) {
              const float4* q = reinterpret_cast<const float4*>(sums_buf + i * kSums) + lane;
              finish(g * 16 + i, q[0], q[UP ? 32 : 0]);
            }
            meet();  // before the next values
          }
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    if (*abort_flag) outlast_copies();
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
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
  const auto kern = a.E <= 128 ? few_route_kernel<4> : few_route_kernel<8>;
  static std::atomic<uint64_t> done[2];
  FRANK_CUDA_TRY(allow_smem(done[a.E <= 128], kern, kRouteTok * kNormMaxH / kRouteCtas * 4));
  const dim3 grid((unsigned)((a.T + kRouteTok - 1) / kRouteTok * kRouteCtas));
  FRANK_CUDA_TRY(launch_chained(kern, grid, dim3(kRouteThreads), smem, st, kRouteCtas, a));
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

// Map of bytes [E, R, K] (or [R, K]), box 128 bytes x rows, 128-byte swizzle.
static int few_map(CUtensorMap* m, const void* base, int64_t E, int64_t R, int64_t K, uint32_t rows, bool three) {
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
  const cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)R, (cuuint64_t)E};
  const cuuint64_t strides[2] = {(cuuint64_t)K, (cuuint64_t)(R * K)};
  const cuuint32_t box[3] = {kQB, rows, 1}, estr[3] = {1, 1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, three ? 3 : 2, const_cast<void*>(base), dims, strides, box,
                         estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled([%lld, %lld, %lld] bytes) failed: %d", (long long)E, (long long)R, (long long)K,
              (int)r);
    return FRANK_ECUDA;
  }
  return FRANK_OK;
}

// 227 KB an SM less the static tables; the rest is the ring and the epilogue's sums.
constexpr size_t kFewSmem = 232448 - 13312;

template <bool UP>
static int launch_few_product(const FewMaps& maps, const FewArgs& a, cudaStream_t st) {
  const uint32_t stage = (UP ? 2 : 1) * kTile + tile_tokens(a.T) * kQB;
  const size_t sums = 2 * 16 * (UP ? 256 : 128) * 4;
  const int fit = (int)((kFewSmem - 1024 - sums) / stage), stages = fit < kMaxStages ? fit : kMaxStages;
  static std::atomic<uint64_t> done{0};
  FRANK_CUDA_TRY(allow_smem(done, few_product_kernel<UP>, kFewSmem));
  FRANK_CUDA_TRY(launch_chained(few_product_kernel<UP>, dim3(num_sms()), dim3(kFewThreads),
                                1024 + sums + (size_t)stages * stage, st, 1, maps, a, stages, stage));
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

// Tiles of both products, and their counters: an expert's slots may need several entries.
int64_t few_counts(int64_t T, int64_t E, int64_t k, int64_t H, int64_t F) {
  const int64_t n = k * T, entries = (n < E ? n : E) + n / 16;
  return 2 * entries * (q_blocks(F) > q_blocks(H) ? q_blocks(F) : q_blocks(H));
}

// Floats of a CTA's place for partial sums; two places a CTA.
int64_t few_partial_stride(int64_t T) { return tile_tokens((int)T) * 256; }
int64_t few_partials(int64_t T) { return 2 * num_sms() * few_partial_stride(T); }

int64_t few_h_rows(int64_t T, int64_t E, int64_t k) {
  const int64_t n = k * T;  // up to 15 rows of padding for each expert that has slots
  return (n + 15 * (n < E ? n : E) + 15) / 16 * 16;
}

int launch_few_experts(const FewArgs& args, int32_t* err, cudaStream_t st) {
  FewArgs a = args;
  a.err = device_error_word();
  a.partial_stride = few_partial_stride(a.T);
  a.n_count = (int)few_counts(a.T, a.E, a.k, a.H, a.F);
  a.h_rows = (int)few_h_rows(a.T, a.E, a.k);
  if (err != nullptr) {
    FRANK_CUDA_TRY(launch_chained(few_check_ids_kernel, dim3(1), dim3(256), 0, st, 1, a.ids, a.k * a.T, a.E, err));
    FRANK_LAUNCH_CHECK();
  }
  FewMaps up{}, down{};
  FRANK_TRY(few_map(&up.w, a.w_gate, a.E, a.F, a.H, 128, true));
  FRANK_TRY(few_map(&up.w2, a.w_up, a.E, a.F, a.H, 128, true));
  FRANK_TRY(few_map(&down.w, a.w_down, a.E, a.H, a.F, 128, true));
  down.w2 = down.w;
  for (int i = 0; i < tile_tokens(a.T) / 16; ++i)
    FRANK_TRY(few_map(&down.x[i], a.hq, 1, a.h_rows, a.F, 16u << i, false));
  FRANK_TRY(launch_few_product<true>(up, a, st));
  return launch_few_product<false>(down, a, st);
}

}  // namespace frank
