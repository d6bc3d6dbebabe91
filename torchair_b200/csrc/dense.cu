// Host side of the dense 16-bit GEMMs: argument checks, tensor maps, the choice between the narrow and the pair kernel and
// how many CTAs share a tile, and the C entry points tab_dense_matmul, tab_gated_matmul_grad, tab_gated_ffn.
#include <stdlib.h>

#include <algorithm>
#include <atomic>

#include "dense_common.cuh"
#include "dense_narrow.cuh"
#include "dense_pair.cuh"

namespace tab {

typedef CUresult (*DenseEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static DenseEncodeFn dense_encode_fn() {
  static DenseEncodeFn fn = []() -> DenseEncodeFn {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<DenseEncodeFn>(ptr);
  }();
  return fn;
}

static int dense_sms() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return kNumSMs;
  if (cached[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 2) n = kNumSMs;
    cached[dev] = n;
  }
  return cached[dev];
}

static long long dense_wait_cycles() {
  static const long long cycles = []() {
    long long ms = 2000;
    if (const char* f = getenv("TAB_GMM_WAIT_MS")) {
      const long long v = atoll(f);
      if (v >= 1 && v <= 600000) ms = v;
    }
    return ms * kDnCyclesPerMs;
  }();
  return cycles;
}

// One operand: `rows` indices of the product times `depth` contraction elements, 16-bit, `ld` elements between lines.
// mn = 0: a line is one index (contiguous along the contraction); mn = 1: a line is one contraction element.
struct DenseOperand {
  const void* ptr;
  int64_t ld, rows, depth;
  int mn;
};

static int check_operand(const char* op, const char* name, const DenseOperand& o) {
  if (!o.ptr) return fail(TAB_ERR_BAD_ARG, "%s: null pointer (%s)", op, name);
  if (!aligned16(o.ptr) || o.ld % 8 != 0)
    return fail(TAB_ERR_ALIGNMENT, "%s: %s must be 16-byte aligned with a leading dimension that is a multiple of 8 (got %lld)", op, name, (long long)o.ld);
  const int64_t line = o.mn ? o.rows : o.depth, lines = o.mn ? o.depth : o.rows;
  if (o.ld < line && lines > 1) return fail(TAB_ERR_BAD_ARG, "%s: leading dimension %lld of %s is shorter than a line (%lld)", op, (long long)o.ld, name, (long long)line);
  return TAB_OK;
}

// box_rows: product indices per box (64, or the token columns of the narrow kernel)
static int make_map(const char* op, const DenseOperand& o, int box_rows, CUtensorMap* map) {
  DenseEncodeFn enc = dense_encode_fn();
  if (!enc) return fail(TAB_ERR_CUDA, "%s: cuTensorMapEncodeTiled is not available from the driver", op);
  const int64_t line = o.mn ? o.rows : o.depth, lines = o.mn ? o.depth : o.rows;
  cuuint64_t dims[2] = {(cuuint64_t)line, (cuuint64_t)lines};
  cuuint64_t strides[1] = {(cuuint64_t)((o.ld > 0 ? o.ld : 8) * 2)};
  cuuint32_t box[2] = {64, (cuuint32_t)(o.mn ? kDnBlockK : box_rows)};
  cuuint32_t es[2] = {1, 1};
  auto encode = [&]() {
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(o.ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  int dev = 0;
  if (r == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess)
    r = encode();       // the thread (an autograd worker, say) had made no runtime call yet that binds the device's context
  if (r != CUDA_SUCCESS) return fail(TAB_ERR_CUDA, "%s: tensor map rejected (CUresult %d)", op, (int)r);
  return TAB_OK;
}

// Raises a kernel's dynamic shared memory limit once per device.
template <typename F>
static int allow_smem(const char* op, F* kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return TAB_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(TAB_ERR_CUDA, "%s: shared memory opt-in failed: %s", op, cudaGetErrorString(e));
  if (dev >= 0 && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return TAB_OK;
}

template <typename F>
static int launch_cluster(const char* op, F* kernel, int ctas, int threads, int smem, int cluster, const CUtensorMap& ma,
                          const CUtensorMap& mb, const DenseParams& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, ma, mb, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(TAB_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
  }
  return check_launch(op);
}

// Pairs that share a tile's contraction in the last, partly filled turn.  The GPCs of a B200 hold 33 clusters of 4 such CTAs or 15 of
// 8 at a time; one more costs a second turn.  The join takes longer than it saves on short contractions: 14 tiles left of 88 at
// K = 3008 take 40.4 / 43.5 / 42.2 us with 1 / 2 / 4 pairs, 16 left of 90 at K = 8192 98.4 / 91.3, 2 left of 224 178.8 / 171.7 / 167.9.
static int pair_split(int64_t tiles, int num_kb) {
  if (num_kb < 64) return 1;
  return tiles <= 15 ? 4 : tiles <= 33 ? 2 : 1;
}

// Whole tiles for the turns that fill all pairs, clusters for the `rest` where that is shorter than another whole turn.
static int pair_rest(int64_t tiles, int pairs, int num_kb, int64_t& rest) {
  rest = tiles % pairs;
  const int split = rest ? pair_split(rest, num_kb) : 1;
  if (split == 1) rest = 0;
  return split;
}

template <typename T, int EPI>
static int launch_pair_t(const char* op, const CUtensorMap& ma, const CUtensorMap& mb, DenseParams& p, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0}, done_split{0};
  const int64_t tiles = static_cast<int64_t>(p.row_tiles) * p.col_tiles;
  const int pairs = dense_sms() / 2;
  int64_t rest;
  const int split = pair_rest(tiles, pairs, p.num_kb, rest);
  const int64_t whole = tiles - rest;
  int rc = TAB_OK;
  if (whole > 0) {
    if ((rc = allow_smem(op, dense_pair_kernel<T, EPI, false>, kDpSmemBytes<EPI>, done)) != TAB_OK) return rc;
    p.tile_begin = 0;
    p.tile_end = (int)whole;
    p.split = 1;
    rc = launch_cluster(op, dense_pair_kernel<T, EPI, false>, 2 * (int)(whole < pairs ? whole : pairs), kDpThreads, kDpSmemBytes<EPI>, 2, ma, mb, p, st);
    if (rc != TAB_OK) return rc;
  }
  if (rest > 0) {
    if ((rc = allow_smem(op, dense_pair_kernel<T, EPI, true>, kDpSmemBytes<EPI>, done_split)) != TAB_OK) return rc;
    p.tile_begin = (int)whole;
    p.tile_end = (int)tiles;
    p.split = split;
    if (whole > 0) p.beside = 1;      // both launches read the same operands and write different tiles: the second may fill SMs that the first has left
    rc = launch_cluster(op, dense_pair_kernel<T, EPI, true>, 2 * split * (int)rest, kDpThreads, kDpSmemBytes<EPI>, 2 * split, ma, mb, p, st);
  }
  return rc;
}

template <int EPI>
static int launch_pair_epi(const char* op, int dtype, const DenseOperand& a, const DenseOperand& b, DenseParams& p, cudaStream_t st) {
  p.num_kb = (int)((a.depth + kDnBlockK - 1) / kDnBlockK);
  p.row_tiles = (p.M + 255) / 256;
  p.col_tiles = (p.N + kDpTileCols<EPI> - 1) / kDpTileCols<EPI>;
  p.a_mn = a.mn;
  p.b_mn = b.mn;
  p.idesc = ptx::idesc_f16(256, kDpCols, dtype == TAB_BF16 ? 1 : 0, a.mn, b.mn);
  p.wait_cycles = dense_wait_cycles();
  CUtensorMap ma, mb;
  int rc = make_map(op, a, 64, &ma);
  if (rc == TAB_OK) rc = make_map(op, b, 64, &mb);
  if (rc != TAB_OK) return rc;
  return dtype == TAB_BF16 ? launch_pair_t<__nv_bfloat16, EPI>(op, ma, mb, p, st) : launch_pair_t<__half, EPI>(op, ma, mb, p, st);
}

// ---- narrow kernel ----
struct NarrowPlan {
  int nt, split, row_tiles, col_tiles;
  double cost;               // estimated SM cycles
};

// CTAs of the wide form that the GPCs of a B200 hold at a time in clusters of 1 .. 8 (occupancy queries on the GPU).
constexpr int kClusterRoom[kNwMaxSplit + 1] = {0, 148, 148, 135, 132, 130, 132, 105, 120};

static NarrowPlan narrow_plan(int64_t M, int64_t N, int num_kb, int epi, bool x_mn) {
  NarrowPlan best = {};
  const int64_t features = epi == kEpiGlu ? 64 : 128;
  const int64_t col_tiles = (N + features - 1) / features;
  if (M <= 64) {
    best.nt = x_mn ? 64 : M <= 16 ? 16 : M <= 32 ? 32 : 64;       // (boxes of 64 rows where x is contiguous along its rows)
    best.row_tiles = 1;
    best.col_tiles = (int)col_tiles;
    // CTAs per tile: the most with which all are resident at a time, two to an SM up to 32 rows, one with 64 (where the parts to exchange weigh
    // more), and parts of at least 5 blocks.  Of all numbers up to 8 at 14 tile counts from 5 to 148 and K = 1408 .. 7168, weights from HBM,
    // this one takes 2 % longer than the fastest on average.  8 rows, K = 4096, us with 1 .. 8 CTAs to one of 20 tiles: 16.3 11.4 9.7 9.1 8.8
    // 8.8 8.5 8.2; of 48: 16.7 13.3 12.2 12.2 11.9, then a second turn: 17.6 17.1 16.6; of 110: 21.6 21.5, then 26.9 .. 33.9.  64 rows, 40 tiles:
    // 18.5 14.6 12.8, then 15.0 and more.  Shorter parts: 8 rows, 40 tiles of K = 512: 4.3 with one CTA, 5.1 to 9.3 with more.
    const int per_sm = best.nt <= 32 ? 2 : 1;
    best.split = 1;
    for (int split = 2; split <= kNwMaxSplit && split * 5 <= num_kb; ++split)
      if (col_tiles * split <= per_sm * kClusterRoom[split]) best.split = split;
    best.cost = 0.0;                           // never slower than a 256-row tile: the same weights, less of everything else
    return best;
  }
  // Estimates in SM cycles: 58 bytes of operands a cycle reach an SM, a block takes at least 400; 3500 cycles until the first block and
  // after the last, 30 per row that a tile has for the epilogue; the exchange of parts 1500 and 32 per row.  At 19 shapes from 100 x 4096
  // -> 4096 to 2048 x 3008 -> 2816 the combination chosen so took at most 9 % longer than the fastest of all (400 x 4096 -> 2048: 17.3 us
  // with two CTAs to 128 rows, 19.3 with one to 64, 18.3 on CTA pairs).
  for (int nt = x_mn ? 64 : 32; nt <= kNwMaxTokens; nt *= 2) {
    const int64_t row_tiles = (M + nt - 1) / nt, tiles = row_tiles * col_tiles;
    if (tiles > 8 * 148) continue;
    const double rows = static_cast<double>(std::min<int64_t>(nt, M));
    const int per_sm = nt <= 64 ? 2 : 1;
    for (int split = 1; split <= kNwMaxSplit; ++split) {
      if (split > 1 && (nt > 128 || split * 4 > num_kb || tiles * split > kClusterRoom[split])) continue;
      const int64_t ctas = tiles * split, room = static_cast<int64_t>(kClusterRoom[split]) * per_sm;
      const double turns = static_cast<double>((ctas + room - 1) / room);
      const double together = ctas > kClusterRoom[split] ? per_sm : 1;
      const double cost = turns * ((num_kb + split - 1) / split * std::max(400.0, together * dense_narrow_stage_bytes(nt) / 58.0) + 3500.0 + 30.0 * rows * together +
                                   (split > 1 ? 1500.0 + 32.0 * rows : 0.0));
      if (best.nt == 0 || cost < best.cost) best = NarrowPlan{nt, split, (int)row_tiles, (int)col_tiles, cost};
    }
  }
  return best;
}

// The pair kernel's estimate in the same unit.
static double pair_cost(int64_t M, int64_t N, int num_kb, int epi, int pairs) {
  const int64_t cols = epi == kEpiGlu ? 128 : 256;
  const int64_t tiles = ((M + 255) / 256) * ((N + cols - 1) / cols);
  const int64_t turns = tiles / pairs, rest = tiles % pairs;
  const int split = rest ? pair_split(rest, num_kb) : 1;
  const double last = rest == 0 ? 0.0 : split > 1 ? num_kb / split * 520.0 + 9000.0 : num_kb * 520.0;
  return turns * num_kb * 520.0 + last + 11000.0;
}

template <typename T, int EPI, bool WIDE>
static int launch_narrow_t(const char* op, const CUtensorMap& mw, const CUtensorMap& mx, const DenseParams& p, cudaStream_t st) {
  const int smem = 1024 + p.stages * dense_narrow_stage_bytes(p.nt) + kNwCtrlBytes + dense_narrow_recv_bytes(p.nt, p.split);
  static std::atomic<unsigned long long> done{0};
  const int rc = allow_smem(op, dense_narrow_kernel<T, EPI, WIDE>, dense_narrow_smem(true), done);
  if (rc != TAB_OK) return rc;
  return launch_cluster(op, dense_narrow_kernel<T, EPI, WIDE>, p.row_tiles * p.col_tiles * p.split, dense_narrow_threads(WIDE), smem, p.split,
                        mw, mx, p, st);
}

template <int EPI>
static int launch_narrow_epi(const char* op, int dtype, const DenseOperand& x, const DenseOperand& w, DenseParams& p, const NarrowPlan& plan,
                             cudaStream_t st) {
  p.num_kb = (int)((x.depth + kDnBlockK - 1) / kDnBlockK);
  p.nt = plan.nt;
  p.split = plan.split;
  p.row_tiles = plan.row_tiles;
  p.col_tiles = plan.col_tiles;
  const bool wide = plan.nt > 64;
  const int recv = dense_narrow_recv_bytes(p.nt, p.split);
  const bool alone = wide || plan.row_tiles * plan.col_tiles * plan.split <= kClusterRoom[plan.split];
  p.stages = (dense_narrow_smem(alone) - 1024 - kNwCtrlBytes - recv) / dense_narrow_stage_bytes(p.nt);
  if (p.stages > kNwMaxStages) p.stages = kNwMaxStages;
  p.a_mn = w.mn;
  p.b_mn = x.mn;
  p.idesc = ptx::idesc_f16(128, p.nt, dtype == TAB_BF16 ? 1 : 0, w.mn, x.mn);
  p.wait_cycles = dense_wait_cycles();
  CUtensorMap mw, mx;
  int rc = make_map(op, w, 64, &mw);
  if (rc == TAB_OK) rc = make_map(op, x, x.mn ? 64 : p.nt, &mx);
  if (rc != TAB_OK) return rc;
  if (dtype == TAB_BF16)
    return wide ? launch_narrow_t<__nv_bfloat16, EPI, true>(op, mw, mx, p, st) : launch_narrow_t<__nv_bfloat16, EPI, false>(op, mw, mx, p, st);
  return wide ? launch_narrow_t<__half, EPI, true>(op, mw, mx, p, st) : launch_narrow_t<__half, EPI, false>(op, mw, mx, p, st);
}
constexpr bool narrow_fits(int nt, int split, int stages) {     // that many stages, and the parts of a tile overlay them
  return 1024 + stages * dense_narrow_stage_bytes(nt) + kNwCtrlBytes + dense_narrow_recv_bytes(nt, split) <= dense_narrow_smem(nt > 64) &&
         nt * 512 <= stages * dense_narrow_stage_bytes(nt);
}
static_assert(narrow_fits(16, kNwMaxSplit, 5) && narrow_fits(32, kNwMaxSplit, 4) && narrow_fits(64, kNwMaxSplit, 3) &&
              narrow_fits(128, kNwMaxSplit, 4) && narrow_fits(256, 1, 4), "shared memory of the narrow kernel");

// Which kernel: the one with the lower estimate.
static bool narrow_is_chosen(const NarrowPlan& plan, int64_t M, int64_t N, int num_kb, int epi) {
  return plan.nt != 0 && plan.cost <= pair_cost(M, N, num_kb, epi, dense_sms() / 2);
}

template <int EPI>
static int launch_dense(const char* op, int dtype, const DenseOperand& a, const DenseOperand& b, DenseParams& p, cudaStream_t st) {
  const int num_kb = (int)((a.depth + kDnBlockK - 1) / kDnBlockK);
  const NarrowPlan plan = narrow_plan(p.M, p.N, num_kb, EPI, a.mn != 0);
  if (narrow_is_chosen(plan, p.M, p.N, num_kb, EPI)) return launch_narrow_epi<EPI>(op, dtype, a, b, p, plan, st);
  return launch_pair_epi<EPI>(op, dtype, a, b, p, st);
}

// ---- checks ----
static int check_dense(const char* op, int dtype, int64_t M, int64_t N, int64_t K, int act) {
  if (M < 0 || N <= 0 || K <= 0) return fail(TAB_ERR_BAD_ARG, "%s: M=%lld N=%lld K=%lld", op, (long long)M, (long long)N, (long long)K);
  if (dtype != TAB_BF16 && dtype != TAB_F16) return fail(TAB_ERR_UNSUPPORTED, "%s: dtype %d (want 5 or 15)", op, dtype);
  if (act < TAB_ACT_NONE || act > TAB_ACT_SILU) return fail(TAB_ERR_BAD_ARG, "%s: activation %d", op, act);
  if (M > (1LL << 30) || N > (1LL << 24) || K > (1LL << 30)) return fail(TAB_ERR_UNSUPPORTED, "%s: dimension too large", op);
  if (((M + 255) / 256) * ((N + 127) / 128) > (1LL << 28)) return fail(TAB_ERR_UNSUPPORTED, "%s: too many tiles", op);
  return TAB_OK;
}

static int check_multiple(const char* op, const char* name, int64_t v) {
  return v % 8 == 0 ? TAB_OK : fail(TAB_ERR_ALIGNMENT, "%s: %s=%lld (must be a multiple of 8)", op, name, (long long)v);
}

static int check_keep(const char* op, const void* keep, const int8_t* keep_q, const float* keep_scale, int64_t keep_ld, int64_t width) {
  if (keep && keep_q) return fail(TAB_ERR_BAD_ARG, "%s: keep either 16-bit or 8-bit values", op);
  if (keep_q && !keep_scale) return fail(TAB_ERR_BAD_ARG, "%s: 8-bit values need their scales", op);
  if ((keep || keep_q) && (keep_ld < width || keep_ld > (1LL << 30))) return fail(TAB_ERR_BAD_ARG, "%s: kept rows hold %lld values, %lld are needed", op, (long long)keep_ld, (long long)width);
  if ((keep && (!aligned16(keep) || keep_ld % 8 != 0)) || (keep_q && (!aligned16(keep_q) || keep_ld % kKeepBlock != 0)))
    return fail(TAB_ERR_ALIGNMENT, "%s: kept values must be 16-byte aligned with rows of a multiple of 8 (8-bit: 64) values", op);
  return TAB_OK;
}

static int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }

static int check_epilogue_ptrs(const char* op, const void* bias, const void* residual, const void* out, bool whole = true) {
  if (!out) return fail(TAB_ERR_BAD_ARG, "%s: null output", op);
  if (whole && (!aligned16(out) || !aligned16(bias) || !aligned16(residual)))
    return fail(TAB_ERR_ALIGNMENT, "%s: bias, residual and output must be 16-byte aligned", op);
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(residual)) & 1u) != 0)
    return fail(TAB_ERR_ALIGNMENT, "%s: misaligned pointer", op);
  return TAB_OK;
}

static int gated_matmul(const char* op, const DenseOperand& x, const DenseOperand& w, int dtype, int64_t M, int64_t I, const void* bias, int act,
                        void* keep, int8_t* keep_q, float* keep_scale, int64_t keep_ld, void* h, cudaStream_t st) {
  DenseParams p = {};
  p.M = (int)M;
  p.N = (int)I;
  p.act = act;
  p.bias = bias;
  p.out = h;
  p.keep = keep;
  p.keep_q = keep_q;
  p.keep_scale = keep_scale;
  p.keep_ld = (int)keep_ld;
  p.keep_up = (int)(keep_q ? up64(I) : I);
  return launch_dense<kEpiGlu>(op, dtype, x, w, p, st);
}

static int linear_matmul(const char* op, const DenseOperand& a, const DenseOperand& b, int dtype, int64_t M, int64_t N, const void* bias,
                         const void* residual, int act, void* keep, int8_t* keep_q, float* keep_scale, int64_t keep_ld, void* out, int dependent,
                         int beside, cudaStream_t st) {
  DenseParams p = {};
  p.M = (int)M;
  p.N = (int)((N + 7) / 8 * 8);
  p.n_out = (int)N;
  p.act = act;
  p.bias = bias;
  p.residual = residual;
  p.out = out;
  p.keep = keep;
  p.keep_q = keep_q;
  p.keep_scale = keep_scale;
  p.keep_ld = (int)keep_ld;
  p.dependent = dependent;
  p.beside = beside;
  if (N % 8 != 0 || !aligned16(out) || !aligned16(bias) || !aligned16(residual)) return launch_dense<kEpiLinearAny>(op, dtype, a, b, p, st);
  return launch_dense<kEpiLinear>(op, dtype, a, b, p, st);
}

}  // namespace tab

using namespace tab;

extern "C" int tab_dense_matmul(const void* a, int64_t lda, int a_mn, const void* b, int64_t ldb, int b_mn, int dtype, int64_t M, int64_t N,
                                int64_t K, const void* bias, const void* residual, int act, void* keep, int8_t* keep_q, float* keep_scale,
                                int64_t keep_ld, void* out, int beside_previous, tab_stream_t stream) {
  const char* op = "dense_matmul";
  int rc = check_dense(op, dtype, M, N, K, act);
  if (rc != TAB_OK || M == 0) return rc;
  const DenseOperand oa = {a, lda, M, K, a_mn ? 1 : 0}, ob = {b, ldb, N, K, b_mn ? 1 : 0};
  if ((rc = check_operand(op, "a", oa)) != TAB_OK || (rc = check_operand(op, "b", ob)) != TAB_OK) return rc;
  if ((rc = check_epilogue_ptrs(op, bias, residual, out, false)) != TAB_OK) return rc;
  if ((rc = check_keep(op, keep, keep_q, keep_scale, keep_ld, keep_q ? up64(N) : (N + 7) / 8 * 8)) != TAB_OK) return rc;
  return linear_matmul(op, oa, ob, dtype, M, N, bias, residual, act, keep, keep_q, keep_scale, keep_ld, out, 0,
                       beside_previous ? 1 : 0, as_stream(stream));
}

extern "C" int tab_gated_matmul_grad(const void* dy, int64_t lddy, const void* weight, int64_t ldw, int w_mn, int dtype, int64_t M, int64_t I,
                                     int64_t K, int act, const void* keep, const int8_t* keep_q, const float* keep_scale, int64_t keep_ld,
                                     void* dz, void* h, tab_stream_t stream) {
  const char* op = "gated_matmul_grad";
  int rc = check_dense(op, dtype, M, I, K, act);
  if (rc == TAB_OK) rc = check_multiple(op, "I", I);
  if (rc != TAB_OK || M == 0) return rc;
  const DenseOperand oa = {dy, lddy, M, K, 0}, ow = {weight, ldw, I, K, w_mn ? 1 : 0};
  if ((rc = check_operand(op, "dy", oa)) != TAB_OK || (rc = check_operand(op, "weight", ow)) != TAB_OK) return rc;
  if ((rc = check_epilogue_ptrs(op, dz, nullptr, h)) != TAB_OK) return rc;
  if (!dz || (!keep && !keep_q)) return fail(TAB_ERR_BAD_ARG, "%s: null pointer", op);
  if ((rc = check_keep(op, keep, keep_q, keep_scale, keep_ld, 2 * (keep_q ? up64(I) : I))) != TAB_OK) return rc;
  DenseParams p = {};
  p.M = (int)M;
  p.N = (int)I;
  p.act = act;
  p.out = h;
  p.dgate = dz;
  p.keep = const_cast<void*>(keep);
  p.keep_q = const_cast<int8_t*>(keep_q);
  p.keep_scale = const_cast<float*>(keep_scale);
  p.keep_ld = (int)keep_ld;
  p.keep_up = (int)(keep_q ? up64(I) : I);
  return launch_dense<kEpiGluGrad>(op, dtype, oa, ow, p, as_stream(stream));
}

extern "C" int tab_gated_ffn_workspace_bytes(int64_t M, int64_t H, int64_t I, size_t* bytes) {
  if (!bytes || M < 0 || H <= 0 || I <= 0) return fail(TAB_ERR_BAD_ARG, "gated_ffn: M=%lld H=%lld I=%lld", (long long)M, (long long)H, (long long)I);
  *bytes = static_cast<size_t>(M) * I * 2;                        // the hidden rows
  return TAB_OK;
}

extern "C" int tab_gated_ffn(const void* x, int64_t ldx, const void* w1, int64_t ldw1, int w1_mn, const void* w2, int64_t ldw2, int w2_mn,
                             int64_t w2_rows, int dtype, int64_t M, int64_t H, int64_t I, const void* bias1, const void* bias2, const void* residual, int act,
                             void* keep, int8_t* keep_q, float* keep_scale, int64_t keep_ld, void* y, void* workspace,
                             size_t workspace_bytes, tab_stream_t stream) {
  const char* op = "gated_ffn";
  int rc = check_dense(op, dtype, M, I, H, act);
  if (rc == TAB_OK) rc = check_dense(op, dtype, M, H, I, act);
  if (rc == TAB_OK) rc = check_multiple(op, "I", I);
  if (rc != TAB_OK || M == 0) return rc;
  if (w2_rows > I || w2_rows <= 0) return fail(TAB_ERR_BAD_ARG, "%s: the second weight has %lld rows for I=%lld", op, (long long)w2_rows, (long long)I);
  const DenseOperand ox = {x, ldx, M, H, 0}, o1 = {w1, ldw1, 2 * I, H, w1_mn ? 1 : 0}, o2 = {w2, ldw2, H, w2_rows, w2_mn ? 1 : 0};
  if ((rc = check_operand(op, "x", ox)) != TAB_OK || (rc = check_operand(op, "weight1", o1)) != TAB_OK || (rc = check_operand(op, "weight2", o2)) != TAB_OK)
    return rc;
  if ((rc = check_epilogue_ptrs(op, bias2, residual, y, false)) != TAB_OK) return rc;
  if (!aligned16(bias1)) return fail(TAB_ERR_ALIGNMENT, "%s: bias1 must be 16-byte aligned", op);
  if ((rc = check_keep(op, keep, keep_q, keep_scale, keep_ld, 2 * (keep_q ? up64(I) : I))) != TAB_OK) return rc;
  size_t need = 0;
  tab_gated_ffn_workspace_bytes(M, H, I, &need);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return fail(TAB_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", op);
  if (workspace_bytes < need) return fail(TAB_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", op, workspace_bytes, need);
  cudaStream_t st = as_stream(stream);
  rc = gated_matmul(op, ox, o1, dtype, M, I, bias1, act, keep, keep_q, keep_scale, keep_ld, workspace, st);
  if (rc != TAB_OK) return rc;
  // the hidden columns behind w2_rows meet no row of w2 and are not read: a row of infinities leaves NaN there
  const DenseOperand oh = {workspace, I, M, w2_rows, 0};
  return linear_matmul(op, oh, o2, dtype, M, H, bias2, residual, TAB_ACT_NONE, nullptr, nullptr, nullptr, 0, y, 1, 0, st);
}

extern "C" int tab_dense_plan(int gated, int64_t M, int64_t N, int64_t K, int a_mn, int64_t* plan) {
  const char* op = "dense_plan";
  int rc = check_dense(op, TAB_BF16, M, N, K, TAB_ACT_NONE);
  if (rc != TAB_OK) return rc;
  if (!plan || gated < 0 || gated > 2 || M == 0) return fail(TAB_ERR_BAD_ARG, "%s: gated=%d M=%lld", op, gated, (long long)M);
  const int epi = gated == 0 ? kEpiLinear : gated == 1 ? kEpiGlu : kEpiGluGrad, num_kb = (int)((K + kDnBlockK - 1) / kDnBlockK);
  const int64_t n8 = (N + 7) / 8 * 8;
  const NarrowPlan narrow = narrow_plan(M, n8, num_kb, epi, a_mn != 0);
  if (narrow_is_chosen(narrow, M, n8, num_kb, epi)) {
    plan[0] = narrow.nt;
    plan[1] = static_cast<int64_t>(narrow.row_tiles) * narrow.col_tiles;
    plan[2] = narrow.split;
    plan[3] = 0;
  } else {
    const int64_t cols = epi == kEpiGlu ? 128 : 256;
    int64_t rest;
    plan[0] = 0;
    plan[1] = ((M + 255) / 256) * ((n8 + cols - 1) / cols);
    plan[2] = pair_rest(plan[1], dense_sms() / 2, num_kb, rest);
    plan[3] = rest;
  }
  return TAB_OK;
}

extern "C" int tab_dense_status_reset(tab_stream_t stream) {
  cudaError_t e = cudaStreamSynchronize(as_stream(stream));
  const int zero = 0;
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_dense_status, &zero, sizeof(int));
  if (e != cudaSuccess) return fail(TAB_ERR_CUDA, "dense_status_reset: %s", cudaGetErrorString(e));
  return TAB_OK;
}

extern "C" int tab_dense_status(int* status_host, tab_stream_t stream) {
  if (!status_host) return fail(TAB_ERR_BAD_ARG, "dense_status: null pointer");
  cudaError_t e = cudaStreamSynchronize(as_stream(stream));
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(status_host, g_dense_status, sizeof(int));
  if (e != cudaSuccess) return fail(TAB_ERR_CUDA, "dense_status: %s", cudaGetErrorString(e));
  if (*status_host != 0) return fail(TAB_ERR_TIMEOUT, "dense matmul: device-side wait %d gave up", *status_host);
  return TAB_OK;
}
