// Grouped product of block-scaled e4m3 rows and weights on the 5th-generation
// tensor cores (tcgen05 + TMEM), fed by TMA.
//
//   y[r, n] = sum_b a_scale[b, r] * w_scale[e, n/128, b] * sum_{k in b} a[r, k] * w[e, n, k]
//
// The scales differ from block to block along K, so the tensor core sums one
// block of 128 (four tcgen05.mma.kind::f8f6f4 of K = 32) into TMEM and the
// epilogue warps multiply that partial tile by the two scales and add it to
// fp32 accumulators in registers, while the tensor core fills the other of two
// TMEM buffers.  Per K block and SM the tensor core needs 512 cycles for
// 128 x 256 x 128, the eight epilogue warps read 128 KB of TMEM and issue 64
// packed FMAs each, at the same time.  Small groups are bound by the weights from HBM.
//
// Structure (persistent, 384 threads, one CTA per SM):
//   warp 0      TMA producer: A 128 x 128 bytes and B 256 x 128 bytes a stage (SWIZZLE_128B), four stages
//   warp 1      TMEM allocator and MMA issuer
//   warps 4..11 epilogue: two warps for each TMEM lane quadrant, each half of the columns;
//               128 accumulators a thread, so they take registers from the first four warps
// Tiles are (expert, m, n) with m fastest inside a band of rows that stays in L2.
//
// Measured, 8192 x 14336 x 4096: 478 to 490 us, 2.0 PFLOP/s, 1060 cycles a K block where
// the MMAs alone are 512.  Without the epilogue's loads and FMAs it takes 858 (an MMA reads
// 96 bytes a cycle from shared memory and the copies write as many, of 128), without
// MMAs and copies the epilogue takes 965; what bounds it is the way of a TMEM
// buffer from the last MMA through the loads to the next MMA, with only two buffers.
// These are times at 1965 MHz; in a row for longer than about 0.1 s the power cap takes the
// clock to 1.6 GHz and the time to 550 us, called from Python or from a graph alike.
// Pairs of CTAs (cta_group::2, 256 x 256 tiles) take 465 us here, but 719 against 671 us
// for an expert FFN of 65536 sorted rows of 128 experts, so tiles are single.  No faster:
// sixteen epilogue warps (724 us), halves of 128 columns with barriers of their own (581
// us), the next K block's TMEM loads before the last FMAs (523 us), the scales by
// warps 2 and 3 through shared memory (483 us).
// Weights' scales may be any fp32 numbers here.  Where all are powers of two, as this
// library's own quantiser makes them, the MMA could apply them itself and sum all
// of K in TMEM; there is no such form.
// Every wait is bounded (about 2 s); on expiry the CTA records FRANK_ETIMEOUT in
// the device error word and unwinds, freeing its TMEM.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "fp8.cuh"
#include "mbarrier.cuh"

namespace {
using namespace frank;
using namespace frank_mbar;

constexpr int BM = 128, BN = 256, BK = kQB;  // rows of one CTA, columns, bytes along K
constexpr int kThreads = 384, kEpiWarps = 8;
// registers a thread: 128 x 40 + 256 x 224 = 62,464 of the 384 x 168 = 64,512 at launch
constexpr int kRegsLaunch = 168, kRegsFew = 40, kRegsEpilogue = 224;
static_assert(128 * kRegsFew + 32 * kEpiWarps * kRegsEpilogue <= kThreads * kRegsLaunch, "setmaxnreg would wait");
constexpr uint32_t kTileBytes = 128 * BK;  // 16 KiB: 128 rows of A or of B
constexpr uint32_t kTmemCols = 512;
constexpr int kStages = 4;
constexpr uint32_t kStageBytes = 3 * kTileBytes;
// kind::f8f6f4: D fp32 [4,6)=1, A and B e4m3 [7,10)=[10,13)=0, N>>3 at [17,23), M>>4 at [24,29)
constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
size_t smem_bytes(int64_t E) {
  return 1024 + kStages * kStageBytes + 2048 + 8 * (2 * kStages + 8) + 16 + 8 * (E + 1) + 64;
}

// A small group needs few rows of A: boxes of 128, 64, 32 or 16 rows.
__host__ __device__ __forceinline__ int box_of(int64_t rows) {
  int box = 0;
  while (box < 3 && rows <= (64 >> box)) ++box;
  return box;
}

struct Maps {
  CUtensorMap a[4];  // boxes of 128, 64, 32 and 16 rows
  CUtensorMap w, w2;
};

struct Params {
  const float* a_scale;
  const float* w_scale;
  const float* w2_scale;
  const int32_t* offsets;
  int E, rows, n_tiles, N, nk, nb_n;
  int band;  // row tiles whose rows of A stay in L2 while the CTAs sweep the columns
  const float* wrow;
  int out_dtype;
  int wide;  // rows of out are 32-byte aligned
  void* out;
  float* h_scale;
  int32_t* err;
};

// ------------------------------------------------------------ PTX glue --
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// K-major operand, 128-byte swizzle: rows of 128 bytes, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(kIdesc), "r"(accumulate)
      : "memory");
}

// Arrives when the MMAs issued so far are done.
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// After the wait: keeps what uses the values behind it.
__device__ __forceinline__ void pin(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}

// acc[0..31] += v[0..31] * s, two lanes of the pair of floats at a time
__device__ __forceinline__ void scale_add(float* acc, const uint32_t (&v)[32], float s) {
  uint64_t s2;
  asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(s));
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    uint64_t a, b;
    asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(acc[2 * i]), "f"(acc[2 * i + 1]));
    asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "r"(v[2 * i]), "r"(v[2 * i + 1]));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(b), "l"(s2));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[2 * i]), "=f"(acc[2 * i + 1]) : "l"(a));
  }
}

// ---------------------------------------------------------------- tiles --
struct Tile {
  int e, m0, m_end, n;
};

// First row of group e; offsets outside [0, rows] cannot lead out of the buffers.
__device__ __forceinline__ int group_at(const Params& p, int e) {
  return p.offsets != nullptr ? min(max(p.offsets[e], 0), p.rows) : (e == 0 ? 0 : p.rows);
}

// prefix: tiles of the groups before each; begin: their first rows.
__device__ __forceinline__ Tile tile_at(int t, const int* prefix, const int* begin, const Params& p) {
  int lo = 0, hi = p.E;  // prefix[lo] <= t < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= t) lo = mid; else hi = mid;
  }
  const int r0 = begin[lo], r1 = begin[lo + 1];
  const int mt = (r1 - r0 + BM - 1) / BM;
  const int local = t - prefix[lo];
  const int band = local / (p.band * p.n_tiles);
  const int gm = min(p.band, mt - band * p.band);
  const int in = local - band * p.band * p.n_tiles;
  return Tile{lo, r0 + (band * p.band + in % gm) * BM, r1, in / gm};
}

// 32 bytes of this thread's row: one sector.  Every thread writes its own row; through
// shared memory, eight rows of 64 bytes an instruction, 65536 x 2048 x 768 takes
// 171 us instead of 163.
__device__ __forceinline__ void put(char* at, bool wide, const uint32_t (&v)[8]) {
  if (wide) {
    store32(at, v);
  } else {  // rows of 16-byte alignment
    reinterpret_cast<uint4*>(at)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<uint4*>(at)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// --------------------------------------------------------------- kernel --
template <int MODE>
__device__ __forceinline__ bool tile_out(const Params& p, const Tile& tl, int row0, int half, float* acc,
                                         uint32_t* amax, int quad, uint32_t parity, uint32_t row_bar,
                                         volatile int* abort_flag) {
  const int lane = threadIdx.x & 31, row = row0 + lane;
  if constexpr (MODE == FP8_SWIGLU) {
    // acc[0..63]: gate, acc[64..127]: up, columns half * 64 + 0..63 of this block of F
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
      acc[i] *= silu(acc[64 + i]);
      m = max(m, abs_bits(acc[i]));
    }
    // the row's other 64 columns are in the other warp of this quadrant
    uint32_t* mine = amax + parity * 256 + quad * 32 + lane;
    mine[half * 128] = m;
    __syncwarp();
    if (lane == 0) mbar_arrive(row_bar);
    if (!mbar_wait_inline(row_bar, parity, abort_flag, p.err)) return false;
    m = max(m, mine[(half ^ 1) * 128]);
    const BlockScale s = block_scale(m);
    if (row < tl.m_end) {
      const int col = tl.n * 128 + half * 64;
      char* out = static_cast<char*>(p.out) + (int64_t)row * p.N + col;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float* a = acc + c * 32 + j * 4;
          w[j] = e4m3x4(a[0] * s.inv, a[1] * s.inv, a[2] * s.inv, a[3] * s.inv);
        }
        if (col + c * 32 + 32 <= p.N)
          put(out + c * 32, p.wide, w);
        else if (col + c * 32 < p.N)  // N ends after 16 of them
          *reinterpret_cast<uint4*>(out + c * 32) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      if (half == 0) p.h_scale[(int64_t)tl.n * p.rows + row] = s.scale;
    }
  } else if (row < tl.m_end) {
    const float s = MODE == FP8_SCALE ? p.wrow[row] : 1.f;
    const int col = tl.n * BN + half * 128;
    if (MODE == FP8_SCALE || p.out_dtype == FRANK_F32) {
      float* out = static_cast<float*>(p.out) + (int64_t)row * p.N + col;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __float_as_uint(acc[c * 8 + j] * s);
        if (col + c * 8 < p.N) put(reinterpret_cast<char*>(out + c * 8), p.wide, v);
      }
    } else {
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + (int64_t)row * p.N + col;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = pack_bf16x2(acc[c * 16 + 2 * j], acc[c * 16 + 2 * j + 1]);
        if (col + c * 16 < p.N) put(reinterpret_cast<char*>(out + c * 16), p.wide, v);
      }
    }
  }
  return true;
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint32_t* amax = reinterpret_cast<uint32_t*>(smem + kStages * kStageBytes);  // [2 parities][2 halves][128 rows]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes + 2048);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* prefix = reinterpret_cast<int*>(tmem_slot + 4);  // [E + 1]
  int* begin = prefix + p.E + 1;                         // [E + 1]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * kStages + a); };
  auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * kStages + 2 + a); };
  auto row_bar = [&](int quad) { return bar0 + 8u * (2 * kStages + 4 + quad); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), kEpiWarps);
    }
    for (int q = 0; q < 4; ++q) mbar_init(row_bar(q), 2);  // the two warps of a quadrant
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_launch();
  for (int e = threadIdx.x; e <= p.E; e += kThreads) begin[e] = group_at(p, e);
  __syncthreads();
  if (warp == 0) {  // prefix[e] = tiles of the experts before e
    int carry = 0;
    for (int base = 0; base < p.E; base += 32) {
      const int e = base + lane;
      const int v =
          e < p.E ? (max(begin[e + 1] - begin[e], 0) + BM - 1) / BM * p.n_tiles : 0;
      int incl = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      if (e < p.E) prefix[e] = carry + incl - v;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) prefix[p.E] = carry;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  const int total = prefix[p.E];

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------- TMA producer --
      uint32_t it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        const Tile tl = tile_at(t, prefix, begin, p);
        const int box = box_of(tl.m_end - tl.m0);
        const uint32_t a_bytes = kTileBytes >> box;
        for (int kb = 0; kb < p.nk; ++kb, ++it) {
          const int s = it % kStages;
          if (!mbar_wait_inline(empty_bar(s), ((it / kStages) & 1u) ^ 1u, abort_flag, p.err)) {
            ok = false;
            break;
          }
          const uint32_t st = smem_u32(smem + s * kStageBytes);
          mbar_expect_tx(full_bar(s), a_bytes + 2 * kTileBytes);
          load_2d(st, &maps.a[box], kb * BK, tl.m0, full_bar(s));
          if constexpr (MODE == FP8_SWIGLU) {
            load_3d(st + kTileBytes, &maps.w, kb * BK, tl.n * 128, tl.e, full_bar(s));
            load_3d(st + 2 * kTileBytes, &maps.w2, kb * BK, tl.n * 128, tl.e, full_bar(s));
          } else {
            load_3d(st + kTileBytes, &maps.w, kb * BK, tl.n * BN, tl.e, full_bar(s));
            load_3d(st + 2 * kTileBytes, &maps.w, kb * BK, tl.n * BN + 128, tl.e, full_bar(s));
          }
        }
      }
    } else if (warp == 1 && lane == 0) {
      // ----------------------------------------------- MMA issuer --
      uint32_t it = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        for (int kb = 0; kb < p.nk; ++kb, ++it) {
          const int s = it % kStages;
          const uint32_t a = it & 1u;
          if (!mbar_wait_inline(tempty_bar(a), ((it >> 1) & 1u) ^ 1u, abort_flag, p.err) ||
              !mbar_wait_inline(full_bar(s), (it / kStages) & 1u, abort_flag, p.err)) {
            ok = false;
            break;
          }
          fence_after();
          const uint32_t st = smem_u32(smem + s * kStageBytes);
          const uint64_t ad = smem_desc(st), bd = smem_desc(st + kTileBytes);
#pragma unroll
          for (int j = 0; j < BK / 32; ++j)  // 32 bytes along K inside the swizzled row
            mma(tmem + a * BN, ad + (uint64_t)(2 * j), bd + (uint64_t)(2 * j), j != 0);
          commit(empty_bar(s));
          commit(tfull_bar(a));
        }
      }
    }
  } else {
    // -------------------------------------------------- epilogue --
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpilogue));
    const int quad = warp & 3, half = (warp - 4) >> 2;
    // columns of this warp: SWIGLU 64 of gate and the same 64 of up, else 128 in a row
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const uint32_t col0 = MODE == FP8_SWIGLU ? half * 64 : half * 128;
    const uint32_t col1 = MODE == FP8_SWIGLU ? 128 + half * 64 : half * 128 + 64;
    uint32_t it = 0, tiles = 0;  // K blocks; tiles with rows of this warp
    bool ok = true;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const Tile tl = tile_at(t, prefix, begin, p);
      const int row0 = tl.m0 + quad * 32;
      const bool work = row0 < tl.m_end;
      // where the next scales are: blocks of 128 bytes in 180 GB fit 32 bits
      uint32_t ia = (uint32_t)min(row0 + lane, p.rows - 1);
      uint32_t iw = (uint32_t)((tl.e * p.nb_n + (MODE == FP8_SWIGLU ? tl.n : min(2 * tl.n + half, p.nb_n - 1))) * p.nk);
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.f;
      // scales of the next two K blocks: they come from L2 while the tensor core works.  The kernel
      // before may have written those of the rows after this one started: not for __ldg.
      float a0 = 0.f, a1 = 0.f, w0 = 0.f, w1 = 0.f, u0 = 0.f, u1 = 0.f;
      auto next_scales = [&](float& fa, float& fw, float& fu) {
        fa = __ldcg(p.a_scale + ia), fw = __ldg(p.w_scale + iw);
        if (MODE == FP8_SWIGLU) fu = __ldg(p.w2_scale + iw);
        ia += (uint32_t)p.rows, ++iw;
      };
      if (work) next_scales(a0, w0, u0);
      if (work && p.nk > 1) next_scales(a1, w1, u1);
#pragma unroll 1
      for (int kb = 0; kb < p.nk; ++kb, ++it) {
        const uint32_t a = it & 1u;
        const float s0 = a0 * w0, s1 = MODE == FP8_SWIGLU ? a0 * u0 : s0;
        a0 = a1, w0 = w1, u0 = u1;
        if (work && kb + 2 < p.nk) next_scales(a1, w1, u1);
        if (!mbar_wait_inline(tfull_bar(a), (it >> 1) & 1u, abort_flag, p.err)) {
          ok = false;
          break;
        }
        fence_after();
        uint32_t v0[32], v1[32];
        if (work) {
          const uint32_t ta = tmem + a * BN + lane_base;
          tmem_ld32(ta + col0, v0);
          tmem_ld32(ta + col0 + 32, v1);
          tmem_wait();
          pin(v0), pin(v1);
          scale_add(acc, v0, s0);
          tmem_ld32(ta + col1, v0);
          scale_add(acc + 32, v1, s0);
          tmem_ld32(ta + col1 + 32, v1);
          tmem_wait();
          pin(v0), pin(v1);
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(a));
        if (work) {
          scale_add(acc + 64, v0, s1);
          scale_add(acc + 96, v1, s1);
        }
      }
      if (ok && work)
        ok = tile_out<MODE>(p, tl, row0, half, acc, amax, quad, tiles++ & 1u, row_bar(quad), abort_flag);
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

// ------------------------------------------------------------ host side --
// Map of bytes [E, R, K] (E = 1: two dimensions), box 128 bytes x box_rows, 128-byte swizzle.
int make_map(CUtensorMap* m, const void* base, int64_t E, int64_t R, int64_t K, uint32_t box_rows, bool three) {
  static PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  if (!enc) {
    frank::set_error("cuTensorMapEncodeTiled unavailable");
    return FRANK_ECUDA;
  }
  const cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)R, (cuuint64_t)E};
  const cuuint64_t strides[2] = {(cuuint64_t)K, (cuuint64_t)(R * K)};
  const cuuint32_t box[3] = {BK, box_rows, 1}, estr[3] = {1, 1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, three ? 3 : 2, const_cast<void*>(base), dims, strides, box,
                         estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    frank::set_error("cuTensorMapEncodeTiled([%lld, %lld, %lld] bytes) failed: %d", (long long)E, (long long)R,
                     (long long)K, (int)r);
    return FRANK_ECUDA;
  }
  return FRANK_OK;
}

template <int MODE>
int launch(const Maps& maps, const Params& p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const size_t smem = smem_bytes(p.E);
  FRANK_CUDA_TRY(frank::allow_smem(done, fp8_gemm_kernel<MODE>, smem_bytes(frank::kFp8MaxE)));
  FRANK_CUDA_TRY(
      frank::launch_chained(fp8_gemm_kernel<MODE>, dim3(frank::num_sms()), dim3(kThreads), smem, st, 1, maps, p));
  FRANK_LAUNCH_CHECK();
  return FRANK_OK;
}

}  // namespace

namespace frank {

int launch_fp8_gemm(const Fp8Gemm& g, cudaStream_t st) {
  if (g.rows == 0) return FRANK_OK;
  Maps maps{};
  // one group of all rows has whole tiles and one rest at most (a map costs the host 0.4 us)
  const int tail = box_of(g.rows % BM != 0 ? g.rows % BM : BM);
  for (int i = 0; i < 4; ++i)
    if (g.offsets != nullptr || i == tail || (i == 0 && g.rows > BM))
      FRANK_TRY(make_map(&maps.a[i], g.a, 1, g.rows, g.K, 128u >> i, false));
  FRANK_TRY(make_map(&maps.w, g.w, g.E, g.N, g.K, 128, true));
  maps.w2 = maps.w;
  if (g.mode == FP8_SWIGLU) FRANK_TRY(make_map(&maps.w2, g.w2, g.E, g.N, g.K, 128, true));
  Params p;
  p.a_scale = g.a_scale;
  p.w_scale = g.w_scale;
  p.w2_scale = g.mode == FP8_SWIGLU ? g.w2_scale : g.w_scale;
  p.offsets = g.offsets;
  p.E = (int)g.E;
  p.rows = (int)g.rows;
  p.n_tiles = (int)(g.mode == FP8_SWIGLU ? q_blocks(g.N) : (g.N + BN - 1) / BN);
  p.N = (int)g.N;
  p.nk = (int)q_blocks(g.K);
  p.nb_n = (int)q_blocks(g.N);
  p.wrow = g.wrow;
  p.out_dtype = g.out_dtype;
  p.out = g.out;
  p.h_scale = g.h_scale;
  const int64_t row_bytes = g.N * (g.mode == FP8_SWIGLU ? 1 : g.out_dtype == FRANK_F32 ? 4 : 2);
  p.wide = (uintptr_t)g.out % 32 == 0 && row_bytes % 32 == 0;
  p.err = device_error_word();
  // rows of A that the CTAs share through L2 while they sweep the columns: 64 MB
  const int64_t band = (64ll << 20) / g.K / BM;
  p.band = (int)(band < 1 ? 1 : (band > 64 ? 64 : band));
  switch (g.mode) {
    case FP8_SWIGLU: return launch<FP8_SWIGLU>(maps, p, st);
    case FP8_SCALE: return launch<FP8_SCALE>(maps, p, st);
    default: return launch<FP8_PLAIN>(maps, p, st);
  }
}

}  // namespace frank
