// Activations kept in 8 bits, and the elementwise half of the dense operators' backward pass.  Everything here is bound by
// HBM: a value is read once and written once.
//
// Mapping of the 8-bit kernels: 8 lanes hold the 64 values of a block, 8 each (16 bytes of 16-bit data), so the block's
// amax is three shuffles and every lane stores 8 bytes of q.  A warp takes 4 blocks side by side and kUnroll such groups in
// flight, loads first.  When rows are whole numbers of blocks and lie back to back, the matrix is one long row and no
// division is left in the loop.
#include "dense_math.cuh"

namespace tab {

constexpr int kCkThreads = 256;
constexpr int kCkUnroll = 4;
constexpr int kCkChunk = 4 * kCkUnroll;          // blocks of 64 per warp and iteration

// 8 values at column `col` of a row; columns >= cols are zero.  VEC: 16-byte loads (aligned, cols a multiple of 8).
template <typename T, bool VEC>
__device__ __forceinline__ void load_cols8(const T* row, int64_t col, int64_t cols, float (&v)[8]) {
  if constexpr (VEC) {
    if (col < cols) {
      Elem<T>::load8(row + col, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? Elem<T>::to_f32(row[col + i]) : 0.f;
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kCkThreads) checkpoint_quant_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t cols,
                                                                      int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
                                                                      int64_t lds) {
  const int lane = threadIdx.x & 31;
  const int64_t blocks = (cols + 63) / 64;
  const int64_t chunks = (blocks + kCkChunk - 1) / kCkChunk;
  const int64_t total = rows * chunks;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kCkThreads / 32);
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * (kCkThreads / 32) + (threadIdx.x >> 5); w < total; w += warps) {
    const int64_t row = chunks == 1 ? w : w / chunks;
    const int64_t b0 = (chunks == 1 ? 0 : w - row * chunks) * kCkChunk;
    const T* xr = x + row * ldx;
    float v[kCkUnroll][8];
#pragma unroll
    for (int i = 0; i < kCkUnroll; ++i) load_cols8<T, VEC>(xr, (b0 + i * 4 + (lane >> 3)) * 64 + (lane & 7) * 8, cols, v[i]);
#pragma unroll
    for (int i = 0; i < kCkUnroll; ++i) {
      const int64_t blk = b0 + i * 4 + (lane >> 3);
      const int64_t col = blk * 64 + (lane & 7) * 8;
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[i][j]) & 0x7fffffffu);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (blk >= blocks) continue;
      const RowQuant rq = make_block_quant(__uint_as_float(m), m < 0x7f800000u);
      const uint2 o = quant8(v[i], rq);
      if constexpr (VEC) {
        if (col < cols) *reinterpret_cast<uint2*>(q + row * ldq + col) = o;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < cols) q[row * ldq + col + j] = static_cast<int8_t>((j < 4 ? o.x >> (8 * j) : o.y >> (8 * j - 32)) & 0xffu);
      }
      if ((lane & 7) == 0) scale[row * lds + blk] = rq.scale;
    }
  }
}

// y = q * scale in [0, cols), 0 in [cols, pad_cols)
template <typename T, bool VEC>
__global__ void __launch_bounds__(kCkThreads) checkpoint_dequant_kernel(const int8_t* __restrict__ q, int64_t ldq, const float* __restrict__ scale,
                                                                        int64_t lds, int64_t rows, int64_t cols, T* __restrict__ y,
                                                                        int64_t ldy, int64_t pad_cols) {
  const int lane = threadIdx.x & 31;
  const int64_t blocks = (pad_cols + 63) / 64;
  const int64_t chunks = (blocks + kCkChunk - 1) / kCkChunk;
  const int64_t total = rows * chunks;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kCkThreads / 32);
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * (kCkThreads / 32) + (threadIdx.x >> 5); w < total; w += warps) {
    const int64_t row = chunks == 1 ? w : w / chunks;
    const int64_t b0 = (chunks == 1 ? 0 : w - row * chunks) * kCkChunk;
    uint2 raw[kCkUnroll];
    float s[kCkUnroll];
#pragma unroll
    for (int i = 0; i < kCkUnroll; ++i) {
      const int64_t blk = b0 + i * 4 + (lane >> 3);
      const int64_t col = blk * 64 + (lane & 7) * 8;
      raw[i] = make_uint2(0u, 0u);
      s[i] = 0.f;
      if (col < cols) {
        s[i] = __ldg(scale + row * lds + blk);
        if constexpr (VEC) {
          raw[i] = __ldg(reinterpret_cast<const uint2*>(q + row * ldq + col));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t b = col + j < cols ? static_cast<uint8_t>(q[row * ldq + col + j]) : 0u;
            if (j < 4) raw[i].x |= b << (8 * j); else raw[i].y |= b << (8 * j - 32);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kCkUnroll; ++i) {
      const int64_t col = (b0 + i * 4 + (lane >> 3)) * 64 + (lane & 7) * 8;
      if (col >= pad_cols) continue;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(static_cast<int8_t>(j < 4 ? raw[i].x >> (8 * j) : raw[i].y >> (8 * j - 32))) * s[i];
      if constexpr (VEC) {
        Elem<T>::store8(y + row * ldy + col, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < pad_cols) y[row * ldy + col + j] = Elem<T>::from_f32(col + j < cols ? v[j] : 0.f);
      }
    }
  }
}

// dz = dy act'(z) and partial column sums of dz.  A CTA owns 128 columns (16 lanes x 8) and a slice of the rows; 16 rows per
// step, so a warp reads two rows' 256-byte segments.  Column sums stay in registers over the slice and are added over the
// 16 row lanes once, in a fixed order.
constexpr int kAgThreads = 256;
constexpr int kAgCols = 128;
constexpr int kAgRows = kAgThreads / (kAgCols / 8);

template <typename T>
__global__ void __launch_bounds__(kAgThreads) act_grad_kernel(const T* __restrict__ dy, int64_t lddy, int64_t M, int64_t N, int act,
                                                              const T* __restrict__ keep, const int8_t* __restrict__ keep_q,
                                                              const float* __restrict__ keep_scale, int64_t keep_ld, T* __restrict__ dz,
                                                              float* __restrict__ sums) {
  __shared__ float red[kAgRows][kAgCols + 4];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kAgCols + cl * 8;
  const int64_t r_begin = M * blockIdx.y / gridDim.y, r_end = M * (blockIdx.y + 1) / gridDim.y;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (col < N) {
#pragma unroll 2
    for (int64_t r = r_begin + rl; r < r_end; r += kAgRows) {
      float g[8];
      Elem<T>::load8(dy + r * lddy + col, g);
      if (act != TAB_ACT_NONE) {
        float z[8];
        if (keep_q != nullptr) {
          const uint2 raw = __ldg(reinterpret_cast<const uint2*>(keep_q + r * keep_ld + col));
          const float s = __ldg(keep_scale + r * (keep_ld / kKeepBlock) + col / kKeepBlock);
#pragma unroll
          for (int j = 0; j < 8; ++j) z[j] = static_cast<float>(static_cast<int8_t>(j < 4 ? raw.x >> (8 * j) : raw.y >> (8 * j - 32))) * s;
        } else {
          Elem<T>::load8(keep + r * keep_ld + col, z);
        }
        with_act(act, [&](auto tag) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float a, d;
            act_both<decltype(tag)::value>(z[j], a, d);
            g[j] *= d;
          }
        });
      }
      if (dz != nullptr) Elem<T>::store8(dz + r * N + col, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += g[j];
    }
  }
  if (sums == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) red[rl][cl * 8 + j] = acc[j];
  __syncthreads();
  if (threadIdx.x < kAgCols) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kAgCols + threadIdx.x;
    if (c < N) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < kAgRows; ++r) s += red[r][threadIdx.x];
      sums[static_cast<int64_t>(blockIdx.y) * N + c] = s;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) column_sums_kernel(const float* __restrict__ sums, int64_t splits, int64_t N, T* __restrict__ out) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= N) return;
  float s = 0.f;
#pragma unroll 8
  for (int64_t i = 0; i < splits; ++i) s += sums[i * N + c];
  out[c] = Elem<T>::from_f32(s);
}

// 16-bit copy between any strides, 64 x 64 tiles through shared memory so that both sides run along their contiguous index.
__global__ void __launch_bounds__(256) copy_2d_kernel(const uint16_t* __restrict__ src, int64_t srs, int64_t scs, int64_t src_rows, int64_t src_cols,
                                                      uint16_t* __restrict__ dst, int64_t drs, int64_t dcs, int64_t dst_rows, int64_t dst_cols,
                                                      int64_t col_tiles, int64_t tiles) {
  __shared__ uint16_t tile[64][66];
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t rt = t / col_tiles;
    const int64_t r0 = rt * 64, c0 = (t - rt * col_tiles) * 64;
    for (int i = threadIdx.x; i < 4096; i += 256) {
      const int r = scs == 1 ? i >> 6 : i & 63, c = scs == 1 ? i & 63 : i >> 6;
      tile[r][c] = (r0 + r < src_rows && c0 + c < src_cols) ? src[(r0 + r) * srs + (c0 + c) * scs] : static_cast<uint16_t>(0);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 4096; i += 256) {
      const int r = dcs == 1 ? i >> 6 : i & 63, c = dcs == 1 ? i & 63 : i >> 6;
      if (r0 + r < dst_rows && c0 + c < dst_cols) dst[(r0 + r) * drs + (c0 + c) * dcs] = tile[r][c];
    }
    __syncthreads();
  }
}

static bool float_dtype(int dtype) { return dtype == TAB_BF16 || dtype == TAB_F16 || dtype == TAB_F32; }
static int esize(int dtype) { return dtype == TAB_F32 ? 4 : 2; }

static bool natural(const void* p, int size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) == 0; }

template <typename T, bool VEC>
static void launch_quant(const void* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* q, int64_t ldq, float* scale, int64_t lds, cudaStream_t st) {
  const int64_t chunks = ((cols + 63) / 64 + kCkChunk - 1) / kCkChunk;
  const int grid = grid_for((rows * chunks + kCkThreads / 32 - 1) / (kCkThreads / 32), 8);
  checkpoint_quant_kernel<T, VEC><<<grid, kCkThreads, 0, st>>>(static_cast<const T*>(x), ldx, rows, cols, q, ldq, scale, lds);
}

template <typename T, bool VEC>
static void launch_dequant(const int8_t* q, int64_t ldq, const float* scale, int64_t lds, int64_t rows, int64_t cols, void* y, int64_t ldy,
                           int64_t pad_cols, cudaStream_t st) {
  const int64_t chunks = ((pad_cols + 63) / 64 + kCkChunk - 1) / kCkChunk;
  const int grid = grid_for((rows * chunks + kCkThreads / 32 - 1) / (kCkThreads / 32), 8);
  checkpoint_dequant_kernel<T, VEC><<<grid, kCkThreads, 0, st>>>(q, ldq, scale, lds, rows, cols, static_cast<T*>(y), ldy, pad_cols);
}

// slices of the rows: enough CTAs for a few per SM, at least 64 rows each
static int64_t act_grad_splits(int64_t M, int64_t N) {
  const int64_t col_ctas = (N + kAgCols - 1) / kAgCols;
  int64_t s = (4 * kNumSMs + col_ctas - 1) / col_ctas;
  const int64_t most = (M + 63) / 64;
  if (s > most) s = most;
  if (s > 65535) s = 65535;
  return s < 1 ? 1 : s;
}

constexpr int64_t kMaxDim = 1LL << 40;

}  // namespace tab

using namespace tab;

extern "C" int tab_checkpoint_quant(const void* x, int dtype, int64_t ldx, int64_t rows, int64_t cols, int8_t* q, int64_t ldq, float* scale,
                                    int64_t lds, tab_stream_t stream) {
  const char* op = "checkpoint_quant";
  if (rows < 0 || cols < 0 || rows > kMaxDim || cols > kMaxDim) return fail(TAB_ERR_BAD_ARG, "%s: rows=%lld cols=%lld", op, (long long)rows, (long long)cols);
  if (!float_dtype(dtype)) return fail(TAB_ERR_UNSUPPORTED, "%s: dtype %d (want 5, 6 or 15)", op, dtype);
  if (rows == 0 || cols == 0) return TAB_OK;
  const int64_t blocks = (cols + 63) / 64;
  if (!x || !q || !scale) return fail(TAB_ERR_BAD_ARG, "%s: null pointer", op);
  if ((rows > 1 && ldx < cols) || ldq < cols || lds < blocks) return fail(TAB_ERR_BAD_ARG, "%s: rows of %lld / %lld values and %lld scales are too short for %lld columns", op, (long long)ldx, (long long)ldq, (long long)lds, (long long)cols);
  if (!natural(x, esize(dtype)) || !natural(scale, 4)) return fail(TAB_ERR_ALIGNMENT, "%s: misaligned pointer", op);
  const bool vec = cols % 8 == 0 && ldq % 8 == 0 && (ldx * esize(dtype)) % 16 == 0 && aligned16(x) && natural(q, 8);
  if (vec && cols % 64 == 0 && (rows == 1 || (ldx == cols && ldq == cols && lds == blocks))) {      // one long row
    cols *= rows;
    ldx = ldq = cols;
    lds = blocks * rows;
    rows = 1;
  }
  cudaStream_t st = as_stream(stream);
#define TAB_CQ(T) vec ? launch_quant<T, true>(x, ldx, rows, cols, q, ldq, scale, lds, st) : launch_quant<T, false>(x, ldx, rows, cols, q, ldq, scale, lds, st)
  if (dtype == TAB_BF16) TAB_CQ(__nv_bfloat16);
  else if (dtype == TAB_F16) TAB_CQ(__half);
  else TAB_CQ(float);
#undef TAB_CQ
  return check_launch(op);
}

extern "C" int tab_checkpoint_dequant(const int8_t* q, int64_t ldq, const float* scale, int64_t lds, int64_t rows, int64_t cols, void* y,
                                      int dtype, int64_t ldy, int64_t pad_cols, tab_stream_t stream) {
  const char* op = "checkpoint_dequant";
  if (rows < 0 || cols < 0 || pad_cols < cols || rows > kMaxDim || pad_cols > kMaxDim)
    return fail(TAB_ERR_BAD_ARG, "%s: rows=%lld cols=%lld pad_cols=%lld", op, (long long)rows, (long long)cols, (long long)pad_cols);
  if (!float_dtype(dtype)) return fail(TAB_ERR_UNSUPPORTED, "%s: dtype %d (want 5, 6 or 15)", op, dtype);
  if (rows == 0 || pad_cols == 0) return TAB_OK;
  const int64_t blocks = (cols + 63) / 64;
  if (!y || (cols > 0 && (!q || !scale))) return fail(TAB_ERR_BAD_ARG, "%s: null pointer", op);
  if (ldq < cols || lds < blocks || (rows > 1 && ldy < pad_cols)) return fail(TAB_ERR_BAD_ARG, "%s: rows of %lld / %lld values and %lld scales are too short for %lld columns", op, (long long)ldy, (long long)ldq, (long long)lds, (long long)pad_cols);
  if (!natural(y, esize(dtype)) || !natural(scale, 4)) return fail(TAB_ERR_ALIGNMENT, "%s: misaligned pointer", op);
  const bool vec = cols % 8 == 0 && pad_cols % 8 == 0 && ldq % 8 == 0 && (ldy * esize(dtype)) % 16 == 0 && aligned16(y) && natural(q, 8);
  if (vec && cols % 64 == 0 && cols == pad_cols && (rows == 1 || (ldy == cols && ldq == cols && lds == blocks))) {
    cols *= rows;
    pad_cols = ldy = ldq = cols;
    lds = blocks * rows;
    rows = 1;
  }
  cudaStream_t st = as_stream(stream);
#define TAB_CD(T) vec ? launch_dequant<T, true>(q, ldq, scale, lds, rows, cols, y, ldy, pad_cols, st) : launch_dequant<T, false>(q, ldq, scale, lds, rows, cols, y, ldy, pad_cols, st)
  if (dtype == TAB_BF16) TAB_CD(__nv_bfloat16);
  else if (dtype == TAB_F16) TAB_CD(__half);
  else TAB_CD(float);
#undef TAB_CD
  return check_launch(op);
}

extern "C" int tab_act_grad_splits(int64_t M, int64_t N, size_t* splits) {
  if (!splits || M < 0 || N <= 0) return fail(TAB_ERR_BAD_ARG, "act_grad: M=%lld N=%lld", (long long)M, (long long)N);
  *splits = static_cast<size_t>(act_grad_splits(M, N));
  return TAB_OK;
}

extern "C" int tab_act_grad(const void* dy, int64_t lddy, int dtype, int64_t M, int64_t N, int act, const void* keep, const int8_t* keep_q,
                            const float* keep_scale, int64_t keep_ld, void* dz, float* column_sums, tab_stream_t stream) {
  const char* op = "act_grad";
  if (M < 0 || N <= 0 || M > kMaxDim || N > (1LL << 24)) return fail(TAB_ERR_BAD_ARG, "%s: M=%lld N=%lld", op, (long long)M, (long long)N);
  if (dtype != TAB_BF16 && dtype != TAB_F16) return fail(TAB_ERR_UNSUPPORTED, "%s: dtype %d (want 5 or 15)", op, dtype);
  if (act < TAB_ACT_NONE || act > TAB_ACT_SILU) return fail(TAB_ERR_BAD_ARG, "%s: activation %d", op, act);
  if (!dz && !column_sums) return fail(TAB_ERR_BAD_ARG, "%s: nothing to compute", op);
  if (M > 0 && (!dy || (act != TAB_ACT_NONE && !keep && !keep_q) || (keep_q && !keep_scale))) return fail(TAB_ERR_BAD_ARG, "%s: null pointer", op);
  if (N % 8 != 0 || lddy % 8 != 0 || !aligned16(dy) || !aligned16(dz) || (keep && (!aligned16(keep) || keep_ld % 8 != 0)) ||
      (keep_q && (!natural(keep_q, 8) || keep_ld % kKeepBlock != 0)))
    return fail(TAB_ERR_ALIGNMENT, "%s: N=%lld and the leading dimensions must be multiples of 8 (8-bit: 64), pointers 16-byte aligned", op, (long long)N);
  if ((M > 1 && lddy < N) || (act != TAB_ACT_NONE && keep_ld < N)) return fail(TAB_ERR_BAD_ARG, "%s: a leading dimension is shorter than a row of %lld", op, (long long)N);
  if (M == 0 && !column_sums) return TAB_OK;
  const dim3 grid((unsigned)((N + kAgCols - 1) / kAgCols), (unsigned)act_grad_splits(M, N));
  cudaStream_t st = as_stream(stream);
  if (dtype == TAB_BF16)
    act_grad_kernel<__nv_bfloat16><<<grid, kAgThreads, 0, st>>>(static_cast<const __nv_bfloat16*>(dy), lddy, M, N, act, static_cast<const __nv_bfloat16*>(keep),
                                                                keep_q, keep_scale, keep_ld, static_cast<__nv_bfloat16*>(dz), column_sums);
  else
    act_grad_kernel<__half><<<grid, kAgThreads, 0, st>>>(static_cast<const __half*>(dy), lddy, M, N, act, static_cast<const __half*>(keep), keep_q,
                                                         keep_scale, keep_ld, static_cast<__half*>(dz), column_sums);
  return check_launch(op);
}

extern "C" int tab_column_sums(const float* column_sums, int64_t splits, int64_t N, void* out, int dtype, tab_stream_t stream) {
  const char* op = "column_sums";
  if (splits < 1 || N <= 0 || N > (1LL << 24)) return fail(TAB_ERR_BAD_ARG, "%s: splits=%lld N=%lld", op, (long long)splits, (long long)N);
  if (dtype != TAB_BF16 && dtype != TAB_F16) return fail(TAB_ERR_UNSUPPORTED, "%s: dtype %d (want 5 or 15)", op, dtype);
  if (!column_sums || !out) return fail(TAB_ERR_BAD_ARG, "%s: null pointer", op);
  const unsigned grid = (unsigned)((N + 255) / 256);
  if (dtype == TAB_BF16) column_sums_kernel<<<grid, 256, 0, as_stream(stream)>>>(column_sums, splits, N, static_cast<__nv_bfloat16*>(out));
  else column_sums_kernel<<<grid, 256, 0, as_stream(stream)>>>(column_sums, splits, N, static_cast<__half*>(out));
  return check_launch(op);
}

extern "C" int tab_copy_2d(const void* src, int64_t src_row_stride, int64_t src_col_stride, int64_t src_rows, int64_t src_cols, void* dst,
                           int64_t dst_row_stride, int64_t dst_col_stride, int64_t dst_rows, int64_t dst_cols, tab_stream_t stream) {
  const char* op = "copy_2d";
  if (src_rows < 0 || src_cols < 0 || dst_rows < 0 || dst_cols < 0 || src_rows > kMaxDim || src_cols > kMaxDim || dst_rows > kMaxDim || dst_cols > kMaxDim)
    return fail(TAB_ERR_BAD_ARG, "%s: negative or huge size", op);
  if (dst_rows == 0 || dst_cols == 0) return TAB_OK;
  if (!dst || (!src && src_rows > 0 && src_cols > 0)) return fail(TAB_ERR_BAD_ARG, "%s: null pointer", op);
  if (!natural(src, 2) || !natural(dst, 2)) return fail(TAB_ERR_ALIGNMENT, "%s: misaligned pointer", op);
  const int64_t col_tiles = (dst_cols + 63) / 64, tiles = (dst_rows + 63) / 64 * col_tiles;
  copy_2d_kernel<<<grid_for(tiles, 8), 256, 0, as_stream(stream)>>>(static_cast<const uint16_t*>(src), src_row_stride, src_col_stride, src_rows,
                                                                    src_cols, static_cast<uint16_t*>(dst), dst_row_stride, dst_col_stride,
                                                                    dst_rows, dst_cols, col_tiles, tiles);
  return check_launch(op);
}
