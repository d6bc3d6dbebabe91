// Activations kept in 8 bits, and the elementwise half of the dense operators' backward pass.  Everything here is bound by
// HBM: a value is read once and written once.
//
// Mapping of the 8-bit kernels: 8 lanes hold the 64 values of a block, 8 each (16 bytes of 16-bit data), so the block's
// amax is three shuffles and every lane stores 8 bytes of q.  A warp takes 4 blocks side by side and several such groups in
// flight, loads first, the values in their raw form until they are quantised.  When rows are whole numbers of blocks and lie
// back to back, the matrix is one long row and no division is left in the loop.
#include "dense_math.cuh"
#include "ptx_sm100.cuh"

namespace tab {

// Every kernel here is launched so that it may begin while the launch before it on the stream still runs, and waits for that one's end
// first of all; the launch after it may then begin in the same way.  One that runs beside the launch before it (`beside`: nothing of
// either is written by the other) fills the SMs that the other's last turn leaves idle, and waits before it ends.
__device__ __forceinline__ void after_previous(int beside = 0) {
  if (!beside) ptx::dependency_wait();
  ptx::launch_dependents();
}
__device__ __forceinline__ void end_after_previous() {
  if (threadIdx.x == 0) ptx::dependency_wait();
}

template <typename... Params, typename... Args>
static void launch(void (*kernel)(Params...), dim3 grid, int threads, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);      // errors are picked up by check_launch
}

constexpr int kCkThreads = 256;
constexpr int kCkUnroll = 4;
constexpr int kCkChunk = 4 * kCkUnroll;          // blocks of 64 per warp and iteration

// 8 values at column `col` of a row, as they lie in memory; columns >= cols are zero.  VEC: 16-byte loads (aligned, cols a
// multiple of 8).
template <typename T, bool VEC>
__device__ __forceinline__ void load_cols8(const T* row, int64_t col, int64_t cols, Raw8<T>& raw) {
  if constexpr (VEC) {
    if (col < cols) raw.load(row + col); else raw = Raw8<T>{};
  } else {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = col + i < cols ? row[col + i] : Elem<T>::from_f32(0.f);
    raw = *reinterpret_cast<const Raw8<T>*>(t);
  }
}

// largest magnitude of 8 values as fp32 bits: NaN > infinity > every finite value
__device__ __forceinline__ uint32_t raw_amax_bits(const Raw8<__nv_bfloat16>& raw) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw.r);
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
  return max(__float_as_uint(__low2float(m)) & 0x7fffffffu, __float_as_uint(__high2float(m)) & 0x7fffffffu);
}
__device__ __forceinline__ uint32_t raw_amax_bits(const Raw8<__half>& raw) {
  const __half2* h = reinterpret_cast<const __half2*>(&raw.r);
  const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
  return max(__float_as_uint(__low2float(m)) & 0x7fffffffu, __float_as_uint(__high2float(m)) & 0x7fffffffu);
}
__device__ __forceinline__ uint32_t raw_amax_bits(const Raw8<float>& raw) {
  float v[8];
  raw.unpack(v);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  return m;
}

// The next iteration's values are loaded before this one's are quantised.
constexpr int kCkQuantCtas = 4;                  // per SM, all resident
template <typename T, bool VEC>
__global__ void __launch_bounds__(kCkThreads, VEC ? kCkQuantCtas : 2) checkpoint_quant_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows,
                                                                                         int64_t cols, int8_t* __restrict__ q, int64_t ldq,
                                                                                         float* __restrict__ scale, int64_t lds) {
  after_previous();
  const int lane = threadIdx.x & 31;
  const int64_t blocks = (cols + 63) / 64;
  const int64_t chunks = (blocks + kCkChunk - 1) / kCkChunk;
  const int64_t total = rows * chunks;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kCkThreads / 32);
  const int in_chunk = lane >> 3, in_block = (lane & 7) * 8;
  int64_t w = static_cast<int64_t>(blockIdx.x) * (kCkThreads / 32) + (threadIdx.x >> 5);
  int64_t row = 0, b0 = 0;
  Raw8<T> next[kCkUnroll];
  auto load = [&]() {
    row = chunks == 1 ? w : rows == 1 ? 0 : w / chunks;
    b0 = (w - row * chunks) * kCkChunk;
    const T* xr = x + row * ldx;
#pragma unroll
    for (int i = 0; i < kCkUnroll; ++i) load_cols8<T, VEC>(xr, (b0 + i * 4 + in_chunk) * 64 + in_block, cols, next[i]);
  };
  if (w < total) load();
  while (w < total) {
    Raw8<T> raw[kCkUnroll];
#pragma unroll
    for (int i = 0; i < kCkUnroll; ++i) raw[i] = next[i];
    const int64_t r = row, c0 = b0;
    w += warps;
    if (w < total) load();
#pragma unroll
    for (int i = 0; i < kCkUnroll; ++i) {
      const int64_t blk = c0 + i * 4 + in_chunk;
      const int64_t col = blk * 64 + in_block;
      uint32_t m = raw_amax_bits(raw[i]);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (blk >= blocks) continue;
      const RowQuant rq = make_block_quant(__uint_as_float(m), m < 0x7f800000u);
      float v[8];
      raw[i].unpack(v);
      const uint2 o = block_quant8(v, rq);
      if constexpr (VEC) {
        if (col < cols) *reinterpret_cast<uint2*>(q + r * ldq + col) = o;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < cols) q[r * ldq + col + j] = static_cast<int8_t>((j < 4 ? o.x >> (8 * j) : o.y >> (8 * j - 32)) & 0xffu);
      }
      if ((lane & 7) == 0) scale[r * lds + blk] = rq.scale;
    }
  }
}

// The same for 16-bit values that are one long row of whole blocks: no bounds within a block, 32-bit block numbers, the amax on
// packed 16-bit magnitudes (their bits are ordered as the values are, NaN above infinity).  The general kernel needs 154
// instructions for a lane's 8 values and is bound by their issue: 8192 x 7168 took 45.7 us with it, 30.7 with this one (bytes: 27.5).
template <typename T>
__global__ void __launch_bounds__(kCkThreads, kCkQuantCtas) checkpoint_quant_flat_kernel(const T* __restrict__ x, int blocks, int8_t* __restrict__ q,
                                                                              float* __restrict__ scale) {
  after_previous();
  const int lane = threadIdx.x & 31;
  const int sub = lane >> 3, part = lane & 7;
  const int step = gridDim.x * (kCkThreads / 32) * kCkChunk;
  const uint4* src = reinterpret_cast<const uint4*>(x) + part;
  uint2* dst = reinterpret_cast<uint2*>(q) + part;
  int blk = (blockIdx.x * (kCkThreads / 32) + (threadIdx.x >> 5)) * kCkChunk + sub;
  uint4 next[kCkUnroll];
#pragma unroll
  for (int i = 0; i < kCkUnroll; ++i)
    if (blk + 4 * i < blocks) next[i] = __ldcs(src + static_cast<int64_t>(blk + 4 * i) * 8);
  for (; blk - sub < blocks; blk += step) {
    uint4 raw[kCkUnroll];
#pragma unroll
    for (int i = 0; i < kCkUnroll; ++i) raw[i] = next[i];
#pragma unroll
    for (int i = 0; i < kCkUnroll; ++i)
      if (blk - blocks + step + 4 * i < 0) next[i] = __ldcs(src + static_cast<int64_t>(blk + step + 4 * i) * 8);
#pragma unroll
    for (int i = 0; i < kCkUnroll; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float2 two = unpack2<T>(m);
      const uint32_t bits = max(__float_as_uint(two.x), __float_as_uint(two.y));
      const RowQuant rq = make_block_quant(__uint_as_float(bits), bits < 0x7f800000u);
      float v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2<T>(w[j]);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
      const uint2 o = block_quant8(v, rq);
      if (blk + 4 * i < blocks) {
        dst[static_cast<int64_t>(blk + 4 * i) * 8] = o;
        if (part == 0) scale[blk + 4 * i] = rq.scale;
      }
    }
  }
}

// y = q * scale in [0, cols), 0 in [cols, pad_cols)
template <typename T, bool VEC>
__global__ void __launch_bounds__(kCkThreads) checkpoint_dequant_kernel(const int8_t* __restrict__ q, int64_t ldq, const float* __restrict__ scale,
                                                                        int64_t lds, int64_t rows, int64_t cols, T* __restrict__ y,
                                                                        int64_t ldy, int64_t pad_cols, int beside) {
  after_previous(beside);
  const int lane = threadIdx.x & 31;
  const int64_t blocks = (pad_cols + 63) / 64;
  const int64_t chunks = (blocks + kCkChunk - 1) / kCkChunk;
  const int64_t total = rows * chunks;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kCkThreads / 32);
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * (kCkThreads / 32) + (threadIdx.x >> 5); w < total; w += warps) {
    const int64_t row = chunks == 1 ? w : rows == 1 ? 0 : w / chunks;
    const int64_t b0 = (w - row * chunks) * kCkChunk;
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
  end_after_previous();
}

// dz = dy act'(z) and partial column sums of dz (and of a second matrix: a block's two bias gradients in one launch).  A CTA owns 128 columns (16 lanes x 8) and a slice of the rows; 16 rows per
// step, so a warp reads two rows' 256-byte segments.  The next step's values are loaded before this step's are used.  Column sums
// stay in registers over the slice and are added over the 16 row lanes once, in a fixed order.  The slices are chosen so that all
// CTAs are resident at once: with 1.4 turns of CTAs and no load ahead, 8192 x 7168 with GELU took 171 us, now 60 (its bytes: 54).
constexpr int kAgThreads = 256;
constexpr int kAgCols = 128;
constexpr int kAgRows = kAgThreads / (kAgCols / 8);
constexpr int kAgCtasPerSm = 4;

// what one step reads of the activation's argument
template <typename T, bool KEEP8>
struct KeptArg {
  Raw8<T> raw;
  uint2 q;
  float s;
  __device__ __forceinline__ void load(const T* keep, const int8_t* keep_q, const float* keep_scale, int64_t keep_ld, int64_t r, int64_t col) {
    if constexpr (KEEP8) {
      q = __ldg(reinterpret_cast<const uint2*>(keep_q + r * keep_ld + col));
      s = __ldg(keep_scale + r * (keep_ld / kKeepBlock) + col / kKeepBlock);
    } else {
      raw.load(keep + r * keep_ld + col);
    }
  }
  __device__ __forceinline__ void unpack(float (&z)[8]) const {
    if constexpr (KEEP8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = static_cast<float>(static_cast<int8_t>(j < 4 ? q.x >> (8 * j) : q.y >> (8 * j - 32))) * s;
    } else {
      raw.unpack(z);
    }
  }
};

template <typename T, bool KEEP8>
__global__ void __launch_bounds__(kAgThreads, kAgCtasPerSm) act_grad_kernel(const T* __restrict__ dy, int64_t lddy, int64_t M, int64_t N, int act,
                                                              const T* __restrict__ keep, const int8_t* __restrict__ keep_q,
                                                              const float* __restrict__ keep_scale, int64_t keep_ld, T* __restrict__ dz,
                                                              float* __restrict__ sums, const T* __restrict__ more, int64_t ld_more, int64_t n_more,
                                                              int beside) {
  after_previous(beside);
  __shared__ float red[kAgRows][kAgCols + 4];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
  // CTAs behind those of dy take the columns of `more`, whose sums follow those of dy in a row of `sums`
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kAgCols, width = N + n_more;
  const int64_t own = (N + kAgCols - 1) / kAgCols * kAgCols, behind = N;
  const bool is_more = first >= own;
  const int64_t begin = is_more ? first - own : first;
  if (is_more) {
    dy = more;
    lddy = ld_more;
    N = n_more;
  }
  const int64_t col = begin + cl * 8;
  const int64_t r_begin = M * blockIdx.y / gridDim.y, r_end = M * (blockIdx.y + 1) / gridDim.y;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (col < N && r_begin + rl < r_end) {
    with_act(act, [&](auto tag) {
      constexpr int ACT = decltype(tag)::value;
      int64_t r = r_begin + rl;
      Raw8<T> g_next;
      KeptArg<T, KEEP8> z_next;
      g_next.load(dy + r * lddy + col);
      if constexpr (ACT != TAB_ACT_NONE) z_next.load(keep, keep_q, keep_scale, keep_ld, r, col);
      for (; r < r_end; r += kAgRows) {
        const Raw8<T> g_raw = g_next;
        const KeptArg<T, KEEP8> z_raw = z_next;
        if (r + kAgRows < r_end) {
          g_next.load(dy + (r + kAgRows) * lddy + col);
          if constexpr (ACT != TAB_ACT_NONE) z_next.load(keep, keep_q, keep_scale, keep_ld, r + kAgRows, col);
        }
        float g[8];
        g_raw.unpack(g);
        if constexpr (ACT != TAB_ACT_NONE) {
          float z[8];
          z_raw.unpack(z);
          act_slope<ACT>(g, z);
        }
        if (dz != nullptr) Elem<T>::store8(dz + r * N + col, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += g[j];
      }
    });
  }
  if (sums == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) red[rl][cl * 8 + j] = acc[j];
  __syncthreads();
  if (threadIdx.x < kAgCols) {
    const int64_t c = begin + threadIdx.x;
    if (c < N) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < kAgRows; ++r) s += red[r][threadIdx.x];
      sums[blockIdx.y * width + (is_more ? behind : 0) + c] = s;
    }
  }
  end_after_previous();
}

template <typename T>
__global__ void __launch_bounds__(256) column_sums_kernel(const float* __restrict__ sums, int64_t splits, int64_t N, T* __restrict__ out,
                                                          int64_t n_out, T* __restrict__ out_more) {
  after_previous();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= N) return;
  float s = 0.f;
#pragma unroll 8
  for (int64_t i = 0; i < splits; ++i) s += sums[i * N + c];
  (c < n_out ? out + c : out_more + (c - n_out))[0] = Elem<T>::from_f32(s);
}

// Up to kMaxCopies 16-bit copies between any strides in one launch, 64 x 64 tiles through shared memory so that both sides run
// along their contiguous index; rows that begin anywhere are read 2 bytes per lane, 16 loads of a thread in flight, and
// 16-byte aligned destination rows are written 16 bytes per lane.
constexpr int kMaxCopies = 8;
struct CopyItem {
  const uint16_t* src;
  uint16_t* dst;
  int64_t srs, scs, drs, dcs;
  int src_rows, src_cols, dst_rows, dst_cols, col_tiles, first_tile;
};
struct CopyList {
  CopyItem item[kMaxCopies];
  int count, tiles;
};

__global__ void __launch_bounds__(256) copy_2d_kernel(const __grid_constant__ CopyList list) {
  after_previous();
  __shared__ __align__(16) uint16_t tile[64][72];
  for (int t = blockIdx.x; t < list.tiles; t += gridDim.x) {
    int k = 0;
    while (k + 1 < list.count && list.item[k + 1].first_tile <= t) ++k;
    const CopyItem& it = list.item[k];
    const int local = t - it.first_tile;
    const int rt = local / it.col_tiles;
    const int r0 = rt * 64, c0 = (local - rt * it.col_tiles) * 64;
    const bool along_cols = it.scs == 1;
    uint16_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int e = i * 256 + threadIdx.x;
      const int r = along_cols ? e >> 6 : e & 63, c = along_cols ? e & 63 : e >> 6;
      v[i] = (r0 + r < it.src_rows && c0 + c < it.src_cols) ? it.src[(r0 + r) * it.srs + (c0 + c) * it.scs] : static_cast<uint16_t>(0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int e = i * 256 + threadIdx.x;
      tile[along_cols ? e >> 6 : e & 63][along_cols ? e & 63 : e >> 6] = v[i];
    }
    __syncthreads();
    if (it.dcs == 1 && (it.drs & 7) == 0 && (it.dst_cols & 7) == 0 && (reinterpret_cast<uintptr_t>(it.dst) & 15u) == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = i * 256 + threadIdx.x;
        const int r = e >> 3, c = (e & 7) * 8;
        if (r0 + r < it.dst_rows && c0 + c < it.dst_cols)
          *reinterpret_cast<uint4*>(it.dst + (r0 + r) * it.drs + c0 + c) = *reinterpret_cast<const uint4*>(&tile[r][c]);
      }
    } else {
      const bool out_cols = it.dcs == 1;
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const int e = i * 256 + threadIdx.x;
        const int r = out_cols ? e >> 6 : e & 63, c = out_cols ? e & 63 : e >> 6;
        if (r0 + r < it.dst_rows && c0 + c < it.dst_cols) it.dst[(r0 + r) * it.drs + (c0 + c) * it.dcs] = tile[r][c];
      }
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
  const int grid = grid_for((rows * chunks + kCkThreads / 32 - 1) / (kCkThreads / 32), VEC ? kCkQuantCtas : 2);
  launch(checkpoint_quant_kernel<T, VEC>, grid, kCkThreads, st, static_cast<const T*>(x), ldx, rows, cols, q, ldq, scale, lds);
}

template <typename T, bool VEC>
static void launch_dequant(const int8_t* q, int64_t ldq, const float* scale, int64_t lds, int64_t rows, int64_t cols, void* y, int64_t ldy,
                           int64_t pad_cols, int beside, cudaStream_t st) {
  const int64_t chunks = ((pad_cols + 63) / 64 + kCkChunk - 1) / kCkChunk;
  const int grid = grid_for((rows * chunks + kCkThreads / 32 - 1) / (kCkThreads / 32), 8);
  launch(checkpoint_dequant_kernel<T, VEC>, grid, kCkThreads, st, q, ldq, scale, lds, rows, cols, static_cast<T*>(y), ldy, pad_cols, beside);
}

// slices of the rows: as many as keep all CTAs resident at once, at least 64 rows each
static int64_t act_grad_splits(int64_t M, int64_t N) {
  const int64_t col_ctas = (N + kAgCols - 1) / kAgCols;
  int64_t s = kAgCtasPerSm * kNumSMs / col_ctas;
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
  if (vec && rows == 1 && cols % 64 == 0 && cols / 64 < (1LL << 30) && dtype != TAB_F32) {
    const int n = (int)(cols / 64);
    const int grid = grid_for((n + kCkChunk * (kCkThreads / 32) - 1) / (kCkChunk * (kCkThreads / 32)), kCkQuantCtas);
    if (dtype == TAB_BF16) launch(checkpoint_quant_flat_kernel<__nv_bfloat16>, grid, kCkThreads, st, static_cast<const __nv_bfloat16*>(x), n, q, scale);
    else launch(checkpoint_quant_flat_kernel<__half>, grid, kCkThreads, st, static_cast<const __half*>(x), n, q, scale);
    return check_launch(op);
  }
#define TAB_CQ(T) vec ? launch_quant<T, true>(x, ldx, rows, cols, q, ldq, scale, lds, st) : launch_quant<T, false>(x, ldx, rows, cols, q, ldq, scale, lds, st)
  if (dtype == TAB_BF16) TAB_CQ(__nv_bfloat16);
  else if (dtype == TAB_F16) TAB_CQ(__half);
  else TAB_CQ(float);
#undef TAB_CQ
  return check_launch(op);
}

extern "C" int tab_checkpoint_dequant(const int8_t* q, int64_t ldq, const float* scale, int64_t lds, int64_t rows, int64_t cols, void* y,
                                      int dtype, int64_t ldy, int64_t pad_cols, int beside_previous, tab_stream_t stream) {
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
#define TAB_CD(T) vec ? launch_dequant<T, true>(q, ldq, scale, lds, rows, cols, y, ldy, pad_cols, beside_previous ? 1 : 0, st) : launch_dequant<T, false>(q, ldq, scale, lds, rows, cols, y, ldy, pad_cols, beside_previous ? 1 : 0, st)
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
#define TAB_AG(T, K8) \
  launch(act_grad_kernel<T, K8>, grid, kAgThreads, st, static_cast<const T*>(dy), lddy, M, N, act, static_cast<const T*>(keep), keep_q, keep_scale, \
         keep_ld, static_cast<T*>(dz), column_sums, nullptr, 0, 0, 0)
  if (dtype == TAB_BF16) {
    if (keep_q) TAB_AG(__nv_bfloat16, true); else TAB_AG(__nv_bfloat16, false);
  } else {
    if (keep_q) TAB_AG(__half, true); else TAB_AG(__half, false);
  }
#undef TAB_AG
  return check_launch(op);
}

extern "C" int tab_column_sums(const float* column_sums, int64_t splits, int64_t N, void* out, int dtype, tab_stream_t stream) {
  const char* op = "column_sums";
  if (splits < 1 || N <= 0 || N > (1LL << 24)) return fail(TAB_ERR_BAD_ARG, "%s: splits=%lld N=%lld", op, (long long)splits, (long long)N);
  if (dtype != TAB_BF16 && dtype != TAB_F16) return fail(TAB_ERR_UNSUPPORTED, "%s: dtype %d (want 5 or 15)", op, dtype);
  if (!column_sums || !out) return fail(TAB_ERR_BAD_ARG, "%s: null pointer", op);
  const unsigned grid = (unsigned)((N + 255) / 256);
  if (dtype == TAB_BF16) launch(column_sums_kernel<__nv_bfloat16>, grid, 256, as_stream(stream), column_sums, splits, N, static_cast<__nv_bfloat16*>(out), N, nullptr);
  else launch(column_sums_kernel<__half>, grid, 256, as_stream(stream), column_sums, splits, N, static_cast<__half*>(out), N, nullptr);
  return check_launch(op);
}

extern "C" int tab_two_column_sums(const void* a, int64_t lda, int64_t Na, const void* b, int64_t ldb, int64_t Nb, int dtype, int64_t M, float* sums,
                                   int64_t splits, void* out_a, void* out_b, int beside_previous, tab_stream_t stream) {
  const char* op = "two_column_sums";
  if (M < 0 || Na <= 0 || Nb < 0 || M > kMaxDim || Na > (1LL << 24) || Nb > (1LL << 24) || splits < 1 || splits > 65535)
    return fail(TAB_ERR_BAD_ARG, "%s: M=%lld Na=%lld Nb=%lld splits=%lld", op, (long long)M, (long long)Na, (long long)Nb, (long long)splits);
  if (dtype != TAB_BF16 && dtype != TAB_F16) return fail(TAB_ERR_UNSUPPORTED, "%s: dtype %d (want 5 or 15)", op, dtype);
  if ((M > 0 && (!a || (Nb > 0 && !b))) || !sums || !out_a || (Nb > 0 && !out_b)) return fail(TAB_ERR_BAD_ARG, "%s: null pointer", op);
  if (Na % 8 != 0 || Nb % 8 != 0 || lda % 8 != 0 || ldb % 8 != 0 || !aligned16(a) || !aligned16(b))
    return fail(TAB_ERR_ALIGNMENT, "%s: widths and leading dimensions must be multiples of 8, pointers 16-byte aligned", op);
  if (M > 1 && (lda < Na || ldb < Nb)) return fail(TAB_ERR_BAD_ARG, "%s: a leading dimension is shorter than a row", op);
  const dim3 grid((unsigned)((Na + kAgCols - 1) / kAgCols + (Nb + kAgCols - 1) / kAgCols), (unsigned)splits);
  const unsigned grid2 = (unsigned)((Na + Nb + 255) / 256);
  cudaStream_t st = as_stream(stream);
#define TAB_TS(T)                                                                                                                                  \
  launch(act_grad_kernel<T, false>, grid, kAgThreads, st, static_cast<const T*>(a), lda, M, Na, TAB_ACT_NONE, nullptr, nullptr, nullptr, 0, nullptr, \
         sums, static_cast<const T*>(b), ldb, Nb, beside_previous ? 1 : 0);                                                                                                 \
  launch(column_sums_kernel<T>, grid2, 256, st, sums, splits, Na + Nb, static_cast<T*>(out_a), Na, static_cast<T*>(out_b))
  if (dtype == TAB_BF16) {
    TAB_TS(__nv_bfloat16);
  } else {
    TAB_TS(__half);
  }
#undef TAB_TS
  return check_launch(op, 2);
}

extern "C" int tab_copy_2d(const tab_copy* copies, int count, tab_stream_t stream) {
  const char* op = "copy_2d";
  if (count < 0 || count > kMaxCopies || (count > 0 && !copies)) return fail(TAB_ERR_BAD_ARG, "%s: %d copies (at most %d)", op, count, kMaxCopies);
  CopyList list = {};
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i) {
    const tab_copy& c = copies[i];
    if (c.src_rows < 0 || c.src_cols < 0 || c.dst_rows < 0 || c.dst_cols < 0) return fail(TAB_ERR_BAD_ARG, "%s: negative size", op);
    const int64_t most = 1LL << 30;
    if (c.src_rows > most || c.src_cols > most || c.dst_rows > most || c.dst_cols > most) return fail(TAB_ERR_UNSUPPORTED, "%s: dimension too large", op);
    if (c.dst_rows == 0 || c.dst_cols == 0) continue;
    if (!c.dst || (!c.src && c.src_rows > 0 && c.src_cols > 0)) return fail(TAB_ERR_BAD_ARG, "%s: null pointer", op);
    if (!natural(c.src, 2) || !natural(c.dst, 2)) return fail(TAB_ERR_ALIGNMENT, "%s: misaligned pointer", op);
    CopyItem& it = list.item[list.count++];
    it.src = static_cast<const uint16_t*>(c.src);
    it.dst = static_cast<uint16_t*>(c.dst);
    it.srs = c.src_row_stride;
    it.scs = c.src_col_stride;
    it.drs = c.dst_row_stride;
    it.dcs = c.dst_col_stride;
    it.src_rows = (int)c.src_rows;
    it.src_cols = (int)c.src_cols;
    it.dst_rows = (int)c.dst_rows;
    it.dst_cols = (int)c.dst_cols;
    it.col_tiles = (int)((c.dst_cols + 63) / 64);
    it.first_tile = (int)tiles;
    tiles += (c.dst_rows + 63) / 64 * it.col_tiles;
    if (tiles > (1LL << 30)) return fail(TAB_ERR_UNSUPPORTED, "%s: too many elements", op);
  }
  if (tiles == 0) return TAB_OK;
  list.tiles = (int)tiles;
  launch(copy_2d_kernel, grid_for(tiles, 8), 256, as_stream(stream), list);
  return check_launch(op);
}
