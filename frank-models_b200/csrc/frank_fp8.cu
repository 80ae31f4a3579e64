// C-ABI entry points of the 8-bit path (include/frank_fp8.h): argument checks,
// workspace layout and the order of the launches.
#include <initializer_list>

#include "fp8.cuh"
#include "fp8_few.cuh"

namespace frank {

int launch_router_topk(int, const void*, int, const void*, int64_t, int64_t, int64_t, int64_t, int, float*, int32_t*,
                       float*, cudaStream_t, const __nv_bfloat16* wr3_pre = nullptr);
size_t router_pack_offset(int64_t, int64_t);
size_t router_scratch_bytes(int, int64_t, int64_t, int64_t);
size_t permute_workspace_size(int64_t, int64_t);
int launch_permute(const int32_t*, int64_t, int64_t, int32_t*, int32_t*, int32_t*, int32_t*, void*, size_t,
                   cudaStream_t, const float* = nullptr, float* = nullptr);

static int check_float_dtype(int d, const char* what) {
  FRANK_CHECK_ARG(d == FRANK_F32 || d == FRANK_BF16, "%s: dtype %d is neither FRANK_F32 (0) nor FRANK_BF16 (1)", what,
                  d);
  return FRANK_OK;
}

// Rows are counted in 31 bits.
static int check_rows(int64_t T, const char* what) {
  FRANK_CHECK_ARG(T >= 0 && T <= 0x7fffffffLL, "%s: T=%lld out of range", what, (long long)T);
  return FRANK_OK;
}

static bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p % 16 != 0) return false;
  return true;
}

struct Fp8Weights {
  const void *up, *gate, *down;
  const float *s_up, *s_gate, *s_down;
};

// A few tokens: the weights bound the call, and few_fp8.cu reads them once for each 32 slots
// of an expert, so the experts must not have many more on average.  Graph of experts() from a
// cold L2, us there / by the sorted rows, at 8, 16, 20, 24, 26, 28 and 32 slots an expert:
//   2 of 4 of 4096 x 4096    59/72  61/72  63/72  64/72  64/72  78/72  90/74
//   8 of 16 of 2048 x 2048   61/74  63/74  66/74  66/74  66/74  82/74  88/74
//   4 of 8 of 4096 x 14336   272/287  266/274  268/272  274/274  279/279  279/274  375/276
// 8 of 128 of 2048 x 768, 64 tokens (4 an expert): 131 / 158.
static bool few_tokens(int64_t T, int64_t E, int64_t k, int64_t H, int64_t F) {
  return T <= kFewMaxT && k * T <= kFewMaxSlots && k * T <= 24 * E && q_blocks(H) <= kFewMaxBlocksH &&
         q_blocks(F) <= kFewMaxBlocksF;
}

// Workspace of one call; the same for a block, its experts and its sub-layer
// (which adds the normalised tokens).
struct Fp8MoeWs {
  float* w;               // [k, T] routing of the block
  int32_t* ids;           // [k, T]
  int32_t* sorted_slots;  // [n]
  int32_t* offsets;       // [E + 1]
  int32_t* slot_pos;      // [n]
  float* wsorted;         // [n]
  __nv_bfloat16* xn;      // [T, H]
  uint8_t* xq;            // [n, H]
  float* xs;              // [H/128, n]
  uint8_t* hq;            // [n, F]
  float* hs;              // [F/128, n]
  float* d;               // [n, H]
  float* partial;         // a few tokens: partial sums of divided tiles, and their counters
  int32_t* count;
  float* logits;
  void* perm;
  size_t perm_bytes;
};

static size_t fp8_moe_layout(int64_t T, int64_t H, int64_t F, int64_t E, int64_t k, void* base, size_t cap,
                             Fp8MoeWs* out) {
  const int64_t n = k * T;
  Carve c(base, cap);
  Fp8MoeWs l;
  l.w = c.take<float>(n);
  l.ids = c.take<int32_t>(n);
  l.sorted_slots = c.take<int32_t>(n);
  l.offsets = c.take<int32_t>(E + 1);
  l.slot_pos = c.take<int32_t>(n);
  l.wsorted = c.take<float>(n);
  l.xn = c.take<__nv_bfloat16>(T * H);
  const bool few = few_tokens(T, E, k, H, F);
  const int64_t h_rows = few ? few_h_rows(T, E, k) : n;
  l.xq = c.take<uint8_t>(n * H);
  l.xs = c.take<float>((few ? kFewMaxT : n) * q_blocks(H));
  l.hq = c.take<uint8_t>(h_rows * F);
  l.hs = c.take<float>(h_rows * q_blocks(F));
  l.d = c.take<float>(n * H);
  l.partial = c.take<float>(few ? few_partials(T) : 0);
  l.count = c.take<int32_t>(few ? few_counts(T, E, k, H, F) : 0);
  l.logits = c.take<float>(router_scratch_bytes(FRANK_BF16, T, H, E) / sizeof(float) + 1);
  l.perm_bytes = permute_workspace_size(n, E);
  l.perm = c.take<char>(l.perm_bytes);
  if (out) *out = l;
  return align_up(c.used, 256);
}

static int check_moe(const char* what, int64_t T, int64_t E, int64_t k, int64_t H, int64_t F, const Fp8Weights& w,
                     const void* workspace, size_t ws_bytes) {
  FRANK_CHECK_ARG(E >= 1 && E <= kFp8MaxE, "%s: n_expert=%lld outside [1, %lld]", what, (long long)E,
                  (long long)kFp8MaxE);
  FRANK_CHECK_ARG(k >= 1 && k <= E && k <= 32, "%s: n_expert_used=%lld outside [1, min(E, 32)]", what, (long long)k);
  FRANK_CHECK_ARG(T >= 0 && T <= kFp8MaxRows && k * T <= kFp8MaxRows, "%s: T=%lld out of range", what, (long long)T);
  FRANK_CHECK_ARG(H >= 16 && H % 16 == 0 && H <= kNormMaxH, "%s: n_embd=%lld is not a multiple of 16 in [16, %lld]",
                  what, (long long)H, (long long)kNormMaxH);
  FRANK_CHECK_ARG(F >= 16 && F % 16 == 0 && F <= 0x7fffffLL, "%s: n_ff=%lld is not a positive multiple of 16", what,
                  (long long)F);
  if (T == 0) return FRANK_OK;
  FRANK_CHECK_ARG(w.up && w.gate && w.down && w.s_up && w.s_gate && w.s_down, "%s: null weights", what);
  FRANK_CHECK_ARG(aligned16({w.up, w.gate, w.down, workspace}), "%s: weights and workspace must be 16-byte aligned",
                  what);
  const size_t need = fp8_moe_layout(T, H, F, E, k, nullptr, 0, nullptr);
  if (ws_bytes < need || workspace == nullptr) {
    set_error("%s: workspace %zu < %zu bytes", what, workspace ? ws_bytes : (size_t)0, need);
    return FRANK_ENOSPC;
  }
  return FRANK_OK;
}

static FewArgs few_args(const Fp8Weights& W, int64_t T, int64_t E, int64_t k, int64_t H, int64_t F, const float* w,
                        const int32_t* ids, const Fp8MoeWs& L) {
  FewArgs a;
  a.w_up = static_cast<const uint8_t*>(W.up);
  a.w_gate = static_cast<const uint8_t*>(W.gate);
  a.w_down = static_cast<const uint8_t*>(W.down);
  a.s_up = W.s_up;
  a.s_gate = W.s_gate;
  a.s_down = W.s_down;
  a.xq = L.xq;
  a.xs = L.xs;
  a.partial = L.partial;
  a.count = L.count;
  a.hq = L.hq;
  a.hs = L.hs;
  a.d = L.d;
  a.w = w;
  a.ids = ids;
  a.T = (int)T;
  a.E = (int)E;
  a.k = (int)k;
  a.H = (int)H;
  a.F = (int)F;
  return a;
}

static FewRoute few_route(int x_dtype, const void* x, const float* norm_w, float eps, int wr_dtype, const void* wr,
                          int64_t T, int64_t E, int64_t k, int64_t H, int64_t F, int normalize, float* w, int32_t* ids,
                          const Fp8MoeWs& L) {
  FewRoute r;
  r.x = x;
  r.x_dtype = x_dtype;
  r.norm_w = norm_w;
  r.eps = eps;
  r.wr = wr;
  r.wr_dtype = wr_dtype;
  r.T = (int)T;
  r.H = (int)H;
  r.E = (int)E;
  r.k = (int)k;
  r.normalize = normalize;
  r.xq = L.xq;
  r.xs = L.xs;
  r.w = w;
  r.ids = ids;
  r.count = L.count;
  r.n_count = (int)few_counts(T, E, k, H, F);
  return r;
}

// Routed rows through the experts: L.d[r] = w * down(q(h)) for the expert-sorted rows r, in
// fp32 whatever the result's type: the sum over a token's slots, and the norm after it, round once.
static int run_experts(const void* x, const float* w, const int32_t* ids, const Fp8Weights& W, int64_t T, int64_t E,
                       int64_t k, int64_t H, int64_t F, int32_t* err, const Fp8MoeWs& L, cudaStream_t st) {
  const int64_t n = k * T;
  if (few_tokens(T, E, k, H, F)) {
    FRANK_TRY(launch_few_route(few_route(FRANK_BF16, x, nullptr, 0.f, FRANK_F32, nullptr, T, E, k, H, F, 0, nullptr,
                                         nullptr, L), st));
    return launch_few_experts(few_args(W, T, E, k, H, F, w, ids, L), err, st);
  }
  FRANK_TRY(launch_permute(ids, n, E, L.sorted_slots, L.offsets, L.slot_pos, err, L.perm, L.perm_bytes, st, w,
                           L.wsorted));
  FRANK_TRY(launch_quantize_rows(FRANK_BF16, x, T, H, L.slot_pos, k, L.xq, L.xs, st));
  Fp8Gemm g;
  g.mode = FP8_SWIGLU;
  g.a = L.xq;
  g.a_scale = L.xs;
  g.w = W.gate;
  g.w_scale = W.s_gate;
  g.w2 = W.up;
  g.w2_scale = W.s_up;
  g.offsets = L.offsets;
  g.E = E;
  g.rows = n;
  g.N = F;
  g.K = H;
  g.out = L.hq;
  g.h_scale = L.hs;
  FRANK_TRY(launch_fp8_gemm(g, st));
  Fp8Gemm d;
  d.mode = FP8_SCALE;
  d.a = L.hq;
  d.a_scale = L.hs;
  d.w = W.down;
  d.w_scale = W.s_down;
  d.offsets = L.offsets;
  d.E = E;
  d.rows = n;
  d.N = H;
  d.K = F;
  d.wrow = L.wsorted;
  d.out = L.d;
  return launch_fp8_gemm(d, st);
}

static NormRows combine_of(const Fp8MoeWs& L, int64_t T, int64_t E, int64_t k, int64_t H, int64_t F, int out_dtype,
                           void* out) {
  NormRows a;
  a.d = L.d;
  a.slot_pos = few_tokens(T, E, k, H, F) ? nullptr : L.slot_pos;
  a.k = (int)k;
  a.T = T;
  a.H = H;
  a.out_dtype = out_dtype;
  a.out = out;
  return a;
}

// The block up to L.d: x [T, H] bf16, or with norm_w the residual it is normalised from.
static int route_and_run(int x_dtype, const void* x, const float* norm_w, float eps, int wr_dtype, const void* wr,
                         const Fp8Weights& W, int64_t T, int64_t E, int64_t k, int64_t H, int64_t F, int normalize,
                         float* w, int32_t* ids, const Fp8MoeWs& L, cudaStream_t st) {
  const __nv_bfloat16* wr3 = nullptr;
  if (wr_dtype == FRANK_ROUTER_PACKED) {
    wr3 = reinterpret_cast<const __nv_bfloat16*>(static_cast<const char*>(wr) + router_pack_offset(E, H));
    wr_dtype = FRANK_F32;
  }
  FRANK_TRY(check_float_dtype(wr_dtype, "fp8_moe router"));
  FRANK_CHECK_ARG(wr != nullptr, "fp8_moe router: null pointer");
  if (few_tokens(T, E, k, H, F)) {
    FRANK_TRY(launch_few_route(
        few_route(x_dtype, x, norm_w, eps, wr_dtype, wr, T, E, k, H, F, normalize, w, ids, L), st));
    return launch_few_experts(few_args(W, T, E, k, H, F, w, ids, L), nullptr, st);
  }
  if (norm_w != nullptr) {
    NormRows pre;
    pre.y_dtype = x_dtype;
    pre.y = x;
    pre.eps = eps;
    pre.next_w = norm_w;
    pre.next = L.xn;
    pre.T = T;
    pre.H = H;
    FRANK_TRY(launch_norm_rows(pre, st));
    x = L.xn;
  }
  FRANK_TRY(launch_router_topk(FRANK_BF16, x, wr_dtype, wr, T, H, E, k, normalize, w, ids, L.logits, st, wr3));
  return run_experts(x, w, ids, W, T, E, k, H, F, nullptr, L, st);
}

// The arguments of a product of rows x, quantised or to be quantised.
static int check_matmul(const char* what, const void* x, const void* w, const float* w_scale, const int32_t* offsets,
                        int64_t E, int64_t rows, int64_t N, int64_t K, int out_dtype, const void* out) {
  FRANK_TRY(check_float_dtype(out_dtype, what));
  FRANK_CHECK_ARG(E >= 1 && E <= kFp8MaxE, "%s: E=%lld outside [1, %lld]", what, (long long)E, (long long)kFp8MaxE);
  FRANK_CHECK_ARG(offsets != nullptr || E == 1, "%s: offsets may be omitted only for a single group", what);
  FRANK_CHECK_ARG(K >= 16 && K % 16 == 0 && K <= 0x7fffffLL && N >= 16 && N % 16 == 0 && N <= 0x7fffffLL,
                  "%s: n_in=%lld and n_out=%lld must be positive multiples of 16", what, (long long)K, (long long)N);
  FRANK_CHECK_ARG(rows >= 0 && rows <= kFp8MaxRows, "%s: rows=%lld out of range", what, (long long)rows);
  if (rows == 0) return FRANK_OK;
  FRANK_CHECK_ARG(x && w && w_scale && out, "%s: null pointer", what);
  FRANK_CHECK_ARG(aligned16({x, w, out}), "%s: rows, w and out must be 16-byte aligned", what);
  return FRANK_OK;
}

static int check_gate(const char* what, const float* gate, int64_t gate_rows, int64_t T) {
  if (gate == nullptr) return FRANK_OK;
  FRANK_CHECK_ARG(gate_rows >= 1 && T % gate_rows == 0, "%s: gate_rows=%lld does not divide T=%lld", what,
                  (long long)gate_rows, (long long)T);
  FRANK_CHECK_ARG(aligned16({gate}), "%s: gate must be 16-byte aligned", what);
  return FRANK_OK;
}

}  // namespace frank

using namespace frank;

extern "C" {

int frank_quantize_fp8(int x_dtype, const void* x, int64_t T, int64_t K, void* q, float* scale, void* stream) {
  FRANK_TRY(check_float_dtype(x_dtype, "quantize_fp8"));
  FRANK_TRY(check_rows(T, "quantize_fp8"));
  FRANK_CHECK_ARG(K >= 16 && K % 16 == 0 && K <= 0x7fffffLL, "quantize_fp8: K=%lld must be a positive multiple of 16",
                  (long long)K);
  if (T == 0) return FRANK_OK;
  FRANK_CHECK_ARG(x && q && scale, "quantize_fp8: null pointer");
  FRANK_CHECK_ARG(aligned16({x, q}), "quantize_fp8: x and q must be 16-byte aligned");
  return launch_quantize_rows(x_dtype, x, T, K, nullptr, 1, q, scale, as_stream(stream));
}

int frank_rms_norm_fp8(int x_dtype, const void* x, const float* weight, int64_t T, int64_t H, float eps, void* xn,
                       void* q, float* scale, void* stream) {
  FRANK_TRY(check_float_dtype(x_dtype, "rms_norm_fp8"));
  FRANK_TRY(check_rows(T, "rms_norm_fp8"));
  FRANK_CHECK_ARG(H >= 16 && H % 16 == 0 && H <= kNormMaxH, "rms_norm_fp8: H=%lld must be a multiple of 16 in [16, %lld]",
                  (long long)H, (long long)kNormMaxH);
  if (T == 0) return FRANK_OK;
  FRANK_CHECK_ARG(x && weight && q && scale, "rms_norm_fp8: null pointer");
  FRANK_CHECK_ARG(aligned16({x, weight, xn, q}), "rms_norm_fp8: buffers must be 16-byte aligned");
  NormRows a;
  a.y_dtype = x_dtype;
  a.y = x;
  a.eps = eps;
  a.next_w = weight;
  a.next = xn;
  a.q = static_cast<uint8_t*>(q);
  a.q_scale = scale;
  a.T = T;
  a.H = H;
  return launch_norm_rows(a, as_stream(stream));
}

int frank_prepack_experts_fp8(int in_dtype, const void* w_oie, int64_t O, int64_t I, int64_t E, void* q_eoi,
                              float* scale, void* stream) {
  FRANK_TRY(check_float_dtype(in_dtype, "prepack_fp8"));
  FRANK_CHECK_ARG(O >= 0 && I >= 0 && E >= 0 && E <= kFp8MaxE && O <= 0x7fffffLL && I <= 0x7fffffLL,
                  "prepack_fp8: bad extents [%lld, %lld, %lld]", (long long)O, (long long)I, (long long)E);
  FRANK_CHECK_ARG(O * I * E == 0 || (w_oie && q_eoi && scale), "prepack_fp8: null pointer");
  return launch_prepack_fp8(in_dtype, w_oie, O, I, E, q_eoi, scale, as_stream(stream));
}

int frank_fp8_matmul(const void* q, const float* scale, const void* w, const float* w_scale, const int32_t* offsets,
                     int64_t E, int64_t rows, int64_t N, int64_t K, int out_dtype, void* out, void* stream) {
  FRANK_TRY(check_matmul("fp8_matmul", q, w, w_scale, offsets, E, rows, N, K, out_dtype, out));
  if (rows == 0) return FRANK_OK;
  FRANK_CHECK_ARG(scale != nullptr, "fp8_matmul: null pointer");
  Fp8Gemm g;
  g.a = q;
  g.a_scale = scale;
  g.w = w;
  g.w_scale = w_scale;
  g.offsets = offsets;
  g.E = E;
  g.rows = rows;
  g.N = N;
  g.K = K;
  g.out_dtype = out_dtype;
  g.out = out;
  return launch_fp8_gemm(g, as_stream(stream));
}

size_t frank_fp8_linear_workspace_size(int64_t rows, int64_t K) {
  return align_up((size_t)rows * K, 256) + align_up((size_t)rows * q_blocks(K) * 4, 256);
}

int frank_fp8_linear(int x_dtype, const void* x, const void* w, const float* w_scale, const int32_t* offsets,
                     int64_t E, int64_t rows, int64_t N, int64_t K, int out_dtype, void* out, void* workspace,
                     size_t ws_bytes, void* stream) {
  // everything is checked before the rows are quantised: a refused call launches nothing
  FRANK_TRY(check_float_dtype(x_dtype, "fp8_linear"));
  FRANK_TRY(check_matmul("fp8_linear", x, w, w_scale, offsets, E, rows, N, K, out_dtype, out));
  if (rows == 0) return FRANK_OK;
  const size_t need = frank_fp8_linear_workspace_size(rows, K);
  if (workspace == nullptr || ws_bytes < need) {
    set_error("fp8_linear: workspace %zu < %zu bytes", workspace ? ws_bytes : (size_t)0, need);
    return FRANK_ENOSPC;
  }
  FRANK_CHECK_ARG(aligned16({workspace}), "fp8_linear: workspace must be 16-byte aligned");
  float* scale = reinterpret_cast<float*>(static_cast<char*>(workspace) + align_up((size_t)rows * K, 256));
  FRANK_TRY(frank_quantize_fp8(x_dtype, x, rows, K, workspace, scale, stream));
  return frank_fp8_matmul(workspace, scale, w, w_scale, offsets, E, rows, N, K, out_dtype, out, stream);
}

size_t frank_fp8_moe_workspace_size(int64_t T, int64_t H, int64_t F, int64_t E, int64_t k) {
  return fp8_moe_layout(T, H, F, E, k, nullptr, 0, nullptr);
}

int frank_fp8_moe_experts(const void* x, const float* route_w, const int32_t* route_ids, const void* w_up,
                          const float* s_up, const void* w_gate, const float* s_gate, const void* w_down,
                          const float* s_down, int64_t T, int64_t E, int64_t k, int64_t H, int64_t F, int y_dtype,
                          void* y, int32_t* err_flag, void* workspace, size_t ws_bytes, void* stream) {
  FRANK_TRY(check_float_dtype(y_dtype, "fp8_moe_experts"));
  const Fp8Weights W{w_up, w_gate, w_down, s_up, s_gate, s_down};
  FRANK_TRY(check_moe("fp8_moe_experts", T, E, k, H, F, W, workspace, ws_bytes));
  if (T == 0) return FRANK_OK;
  FRANK_CHECK_ARG(x && route_w && route_ids && y, "fp8_moe_experts: null pointer");
  FRANK_CHECK_ARG(aligned16({x, y}), "fp8_moe_experts: x and y must be 16-byte aligned");
  cudaStream_t st = as_stream(stream);
  Fp8MoeWs L;
  fp8_moe_layout(T, H, F, E, k, workspace, ws_bytes, &L);
  FRANK_TRY(run_experts(x, route_w, route_ids, W, T, E, k, H, F, err_flag, L, st));
  return launch_norm_rows(combine_of(L, T, E, k, H, F, y_dtype, y), st);
}

int frank_fp8_moe_block(const void* x, int wr_dtype, const void* wr, const void* w_up, const float* s_up,
                        const void* w_gate, const float* s_gate, const void* w_down, const float* s_down, int64_t T,
                        int64_t E, int64_t k, int64_t H, int64_t F, int normalize, int y_dtype, void* y,
                        float* route_w, int32_t* route_ids, void* workspace, size_t ws_bytes, void* stream) {
  FRANK_TRY(check_float_dtype(y_dtype, "fp8_moe_block"));
  const Fp8Weights W{w_up, w_gate, w_down, s_up, s_gate, s_down};
  FRANK_TRY(check_moe("fp8_moe_block", T, E, k, H, F, W, workspace, ws_bytes));
  if (T == 0) return FRANK_OK;
  FRANK_CHECK_ARG(x && y, "fp8_moe_block: null pointer");
  FRANK_CHECK_ARG(aligned16({x, y, wr}), "fp8_moe_block: x, y and wr must be 16-byte aligned");
  cudaStream_t st = as_stream(stream);
  Fp8MoeWs L;
  fp8_moe_layout(T, H, F, E, k, workspace, ws_bytes, &L);
  float* w = route_w ? route_w : L.w;
  int32_t* ids = route_ids ? route_ids : L.ids;
  FRANK_TRY(route_and_run(FRANK_BF16, x, nullptr, 0.f, wr_dtype, wr, W, T, E, k, H, F, normalize, w, ids, L, st));
  return launch_norm_rows(combine_of(L, T, E, k, H, F, y_dtype, y), st);
}

int frank_fp8_moe_sublayer(int res_dtype, const void* residual, const float* norm_w, float eps, int wr_dtype,
                           const void* wr, const void* w_up, const float* s_up, const void* w_gate,
                           const float* s_gate, const void* w_down, const float* s_down, int64_t T, int64_t E,
                           int64_t k, int64_t H, int64_t F, int normalize, const float* post_w, const float* gate,
                           int64_t gate_rows, float residual_scale, void* out, float* route_w, int32_t* route_ids,
                           void* workspace, size_t ws_bytes, void* stream) {
  FRANK_TRY(check_float_dtype(res_dtype, "fp8_moe_sublayer"));
  const Fp8Weights W{w_up, w_gate, w_down, s_up, s_gate, s_down};
  FRANK_TRY(check_moe("fp8_moe_sublayer", T, E, k, H, F, W, workspace, ws_bytes));
  if (T == 0) return FRANK_OK;
  FRANK_CHECK_ARG(residual && norm_w && out, "fp8_moe_sublayer: null pointer");
  FRANK_CHECK_ARG(aligned16({residual, norm_w, post_w, out, wr}), "fp8_moe_sublayer: buffers must be 16-byte aligned");
  FRANK_TRY(check_gate("fp8_moe_sublayer", gate, gate_rows, T));
  cudaStream_t st = as_stream(stream);
  Fp8MoeWs L;
  fp8_moe_layout(T, H, F, E, k, workspace, ws_bytes, &L);
  float* w = route_w ? route_w : L.w;
  int32_t* ids = route_ids ? route_ids : L.ids;
  FRANK_TRY(
      route_and_run(res_dtype, residual, norm_w, eps, wr_dtype, wr, W, T, E, k, H, F, normalize, w, ids, L, st));
  NormRows a = combine_of(L, T, E, k, H, F, res_dtype, out);
  a.post_w = post_w;
  a.eps = eps;
  a.gate = gate;
  a.rows_per_gate = gate ? T / gate_rows : 1;
  a.residual = residual;
  a.residual_scale = residual_scale;
  return launch_norm_rows(a, st);
}

int frank_post_norm_residual(int y_dtype, const void* y, int res_dtype, const void* residual, const float* weight,
                             float eps, const float* gate, int64_t gate_rows, float residual_scale, void* out,
                             const float* next_weight, int next_dtype, void* next, int64_t T, int64_t H,
                             void* stream) {
  FRANK_TRY(check_float_dtype(y_dtype, "post_norm_residual"));
  FRANK_TRY(check_float_dtype(res_dtype, "post_norm_residual"));
  if (next != nullptr) FRANK_TRY(check_float_dtype(next_dtype, "post_norm_residual"));
  FRANK_TRY(check_rows(T, "post_norm_residual"));
  FRANK_CHECK_ARG(H >= 4 && H % 4 == 0 && H <= kNormMaxH,
                  "post_norm_residual: H=%lld must be a multiple of 4 in [4, %lld]", (long long)H, (long long)kNormMaxH);
  if (T == 0) return FRANK_OK;
  FRANK_CHECK_ARG(y && residual && weight && out && (next == nullptr || next_weight),
                  "post_norm_residual: null pointer");
  FRANK_CHECK_ARG(aligned16({y, residual, weight, out, next_weight, next}),
                  "post_norm_residual: buffers must be 16-byte aligned");
  FRANK_TRY(check_gate("post_norm_residual", gate, gate_rows, T));
  NormRows a;
  a.y_dtype = y_dtype;
  a.y = y;
  a.post_w = weight;
  a.eps = eps;
  a.gate = gate;
  a.rows_per_gate = gate ? T / gate_rows : 1;
  a.out_dtype = res_dtype;
  a.residual = residual;
  a.residual_scale = residual_scale;
  a.out = out;
  a.next_w = next ? next_weight : nullptr;
  a.next_dtype = next_dtype;
  a.next = next;
  a.T = T;
  a.H = H;
  return launch_norm_rows(a, as_stream(stream));
}

}  // extern "C"
