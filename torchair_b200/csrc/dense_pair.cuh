// Dense 16-bit GEMM on CTA pairs: out[i, j] = sum_k A[i, k] B[j, k] for bf16 or fp16 operands with fp32 accumulators, in
// tiles of 256 x 256 computed by tcgen05.mma.cta_group::2 on two SMs, with the epilogues of a feed-forward block and of its
// backward pass.
//
// What bounds it.  Per 64-wide block of the contraction a pair reads 64 KB of operands and issues 256 x 256 x 64
// multiply-adds, 512 tensor cycles: the tensor pipe is the limit as long as the ring of six stages stays full.  Every CTA
// brings its own 128 rows of A and half of the tile's 256 rows of B (32 KB per stage); the MMA reads the other half out
// of the peer's shared memory.  Two accumulator buffers (2 x 256 of the 512 TMEM columns) let the epilogue of a tile run
// under the MMAs of the next.
//
// Operand layouts.  Either operand may be contiguous along the contraction (K-major) or along its own index (MN-major):
// the backward pass needs x^T dz and dz W^T of the same row-major tensors, and no transposed copy is ever made.  Both
// kinds of stage consist of 8 KB TMA boxes of 64 rows x 128 bytes with the 128-byte swizzle; only the coordinates, the
// matrix descriptors and the step from one 16-wide MMA slice to the next differ.
//
// Split tiles.  With one tile per pair and turn, the last turn leaves pairs idle (88 tiles on 74 pairs take two turns).
// The host may hand the first sk_tiles tiles out by contraction blocks instead: pair p takes blocks [p U / P, (p+1) U / P)
// of the U = sk_tiles * num_kb blocks.  A CTA that holds only part of a tile stores its fp32 accumulators to a slot of its
// own and counts its arrival; the CTA that arrives last adds all parts in the order of the contraction (so the result does
// not depend on who came last) and runs the epilogue.  Nobody waits for anybody: the kernel needs no co-residency.
//
// Protocol of the pair: as in gmm_i8_pair.cuh (loads of both CTAs complete on the leader's full barrier, the leader issues
// the MMAs and commits to both CTAs' empty / accumulator-full barriers, a bounded hand-shake ends the kernel).
#pragma once

#include "dense_common.cuh"

namespace tab {

constexpr int kDpStageBytes = 2 * kDnOperandBytes;     // 16 KB of A + 16 KB of B per CTA
constexpr int kDpStages = 6;
constexpr int kDpBufs = 2;
constexpr int kDpCols = 256;
constexpr int kDpEpiWarps = 8;                         // two per TMEM lane quarter, each takes half of the columns
constexpr int kDpThreads = 64 + kDpEpiWarps * 32;
constexpr int kDpCtrlBytes = 256;
constexpr int kDpPitch = 80;                           // staged row: 32 16-bit values + 16 bytes of padding
constexpr int kDpPatchBytes = 32 * kDpPitch;           // one epilogue warp's 32 rows
constexpr int kDpSmemBytes = 1024 + kDpStages * kDpStageBytes + kDpCtrlBytes + kDpEpiWarps * kDpPatchBytes;
static_assert(kDpSmemBytes <= kDnSmemLimit, "dense pair GEMM shared memory");
constexpr int64_t kDpPartFloats = 128 * kDpCols;       // accumulators of one CTA and tile

// Work of one pair: segments of tiles.  Split tiles come first, so that their joins run under the whole tiles behind them.
struct DenseWork {
  int tile, kb0, kb1;
};
__host__ __device__ __forceinline__ int64_t dense_unit_begin(int p, int64_t units, int pairs) { return p * units / pairs; }
// pair that holds unit u
__host__ __device__ __forceinline__ int dense_unit_owner(int64_t u, int64_t units, int pairs) {
  int p = static_cast<int>(u * pairs / units);
  while (p + 1 < pairs && dense_unit_begin(p + 1, units, pairs) <= u) ++p;
  while (p > 0 && dense_unit_begin(p, units, pairs) > u) --p;
  return p;
}
struct DenseSched {
  int64_t u, u_end;
  int next_tile, tiles, num_kb, pairs;
  __host__ __device__ DenseSched(int pair, int pairs_, int sk_tiles, int tiles_, int num_kb_) {
    const int64_t units = static_cast<int64_t>(sk_tiles) * num_kb_;
    u = dense_unit_begin(pair, units, pairs_);
    u_end = dense_unit_begin(pair + 1, units, pairs_);
    next_tile = sk_tiles + pair;
    tiles = tiles_;
    num_kb = num_kb_;
    pairs = pairs_;
  }
  __host__ __device__ bool next(DenseWork& w) {
    if (u < u_end) {
      w.tile = static_cast<int>(u / num_kb);
      w.kb0 = static_cast<int>(u - static_cast<int64_t>(w.tile) * num_kb);
      const int64_t left = u_end - u;
      w.kb1 = left < num_kb - w.kb0 ? w.kb0 + static_cast<int>(left) : num_kb;
      u += w.kb1 - w.kb0;
      return true;
    }
    if (next_tile < tiles) {
      w.tile = next_tile;
      w.kb0 = 0;
      w.kb1 = num_kb;
      next_tile += pairs;
      return true;
    }
    return false;
  }
};
// A pair has at most one part that does not begin its tile (slot 0) and one that does but does not end it (slot 1).
__host__ __device__ __forceinline__ int dense_slot(int pair, int kb0) { return 2 * pair + (kb0 == 0 ? 1 : 0); }

// Tiles are numbered so that the tiles in flight share operands: column by column inside bands of kDpBand row tiles.
constexpr int kDpBand = 8;
__device__ __forceinline__ void dense_tile_coord(int t, int row_tiles, int col_tiles, int& rt, int& ct) {
  const int per_band = kDpBand * col_tiles;
  const int band = t / per_band;
  const int in = t - band * per_band;
  const int h = min(kDpBand, row_tiles - band * kDpBand);
  ct = in / h;
  rt = band * kDpBand + (in - ct * h);
}

__device__ __forceinline__ void dense_epi_bar() { asm volatile("bar.sync 1, %0;" ::"n"(kDpEpiWarps * 32) : "memory"); }

// ---- moving 32 rows x 32 columns of 16-bit values between registers (thread = row) and row-major memory, through the warp's
// patch: global accesses are 16 bytes per lane, four lanes to a row's 64 bytes.  Rows >= rows_end and columns >= cols are left
// alone (loads give zeros); cols and col are multiples of 8, so a 16-byte piece is never cut.
template <typename T>
__device__ __forceinline__ void store_rows32(uint8_t* patch, int lane, const float (&v)[32], T* base, int64_t ld, int row_base, int rows_end,
                                             int col, int cols) {
  uint4* prow = reinterpret_cast<uint4*>(patch + lane * kDpPitch);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    prow[k] = make_uint4(pack2<T>(v[8 * k], v[8 * k + 1]), pack2<T>(v[8 * k + 2], v[8 * k + 3]), pack2<T>(v[8 * k + 4], v[8 * k + 5]),
                         pack2<T>(v[8 * k + 6], v[8 * k + 7]));
  __syncwarp();
  const int c = col + (lane & 3) * 8;
  if (c < cols) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 2);
      if (row_base + r < rows_end)
        *reinterpret_cast<uint4*>(base + static_cast<int64_t>(row_base + r) * ld + c) =
            *reinterpret_cast<const uint4*>(patch + r * kDpPitch + (lane & 3) * 16);
    }
  }
  __syncwarp();
}

template <typename T>
__device__ __forceinline__ void load_rows32(uint8_t* patch, int lane, uint32_t (&v)[16], const T* base, int64_t ld, int row_base, int rows_end,
                                            int col, int cols) {
  const int c = col + (lane & 3) * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (c < cols && row_base + r < rows_end) x = __ldg(reinterpret_cast<const uint4*>(base + static_cast<int64_t>(row_base + r) * ld + c));
    *reinterpret_cast<uint4*>(patch + r * kDpPitch + (lane & 3) * 16) = x;
  }
  __syncwarp();
  const uint4* prow = reinterpret_cast<const uint4*>(patch + lane * kDpPitch);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint4 x = prow[k];
    v[4 * k] = x.x;
    v[4 * k + 1] = x.y;
    v[4 * k + 2] = x.z;
    v[4 * k + 3] = x.w;
  }
  __syncwarp();
}

// v[0..31] += bias[col .. col + 31] (columns beyond cols hold nothing that is stored)
template <typename T>
__device__ __forceinline__ void add_bias32(float (&v)[32], const void* bias, int col, int cols) {
  if (bias == nullptr) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (col + 8 * k < cols) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(bias) + col + 8 * k));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(w[i]);
        v[8 * k + 2 * i] += f.x;
        v[8 * k + 2 * i + 1] += f.y;
      }
    }
  }
}

// largest magnitude of a chunk as bits (NaN > infinity > every finite value); columns beyond cols do not count
__device__ __forceinline__ uint32_t chunk_amax_bits(const float (&v)[32], int col, int cols) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (col + (j & ~7) < cols) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  return m;
}

// 32 values of this thread's row -> 32 int8 at q (16-byte aligned); columns beyond cols become 0
__device__ __forceinline__ void store_q32(const float (&v)[32], const RowQuant& rq, int8_t* q, int col, int cols) {
  uint32_t w[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint2 o = make_uint2(0u, 0u);
    if (col + 8 * k < cols) {
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = v[8 * k + i];
      o = quant8(t, rq);
    }
    w[2 * k] = o.x;
    w[2 * k + 1] = o.y;
  }
  *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(q + 16) = make_uint4(w[4], w[5], w[6], w[7]);
}

// 32 kept int8 of this thread's row as fp32
__device__ __forceinline__ void load_q32(float (&v)[32], const int8_t* q, float scale) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(q)), b = __ldg(reinterpret_cast<const uint4*>(q + 16));
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int k = 0; k < 8; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * k + i] = static_cast<float>(static_cast<int8_t>(w[k] >> (8 * i))) * scale;
}

// Where the epilogue takes a tile's accumulators from: tensor memory, or (split tiles) the parts of all contributors in the
// order of the contraction, its own part from tensor memory.
struct DenseAcc {
  uint32_t taddr;          // this warp's lanes, first column of the buffer
  const float* parts;      // null: whole tile in tensor memory
  int64_t units;
  int pairs, num_kb, tile, self, first, last;
  int rank, row_local;
  __device__ __forceinline__ void fetch(int c, float (&v)[32]) const {
    __syncwarp();
    if (parts == nullptr) {
      ptx::tmem_ld32f(taddr + c, v);
      ptx::tmem_ld_wait();
      return;
    }
    const int64_t tile_u = static_cast<int64_t>(tile) * num_kb;
    for (int p = first; p <= last; ++p) {
      float t[32];
      if (p == self) {
        ptx::tmem_ld32f(taddr + c, t);
        ptx::tmem_ld_wait();
      } else {
        const int64_t b = dense_unit_begin(p, units, pairs);
        const int kb0 = b > tile_u ? static_cast<int>(b - tile_u) : 0;
        const float4* src = reinterpret_cast<const float4*>(parts + (static_cast<int64_t>(dense_slot(p, kb0)) * 2 + rank) * kDpPartFloats) +
                            static_cast<int64_t>(c >> 2) * 128 + row_local;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float4 x = __ldcg(src + k * 128);
          t[4 * k] = x.x;
          t[4 * k + 1] = x.y;
          t[4 * k + 2] = x.z;
          t[4 * k + 3] = x.w;
        }
      }
      if (p == first) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = t[j];
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] += t[j];
      }
    }
  }
};

// Epilogue of one warp: 32 rows (row_base ..) x half of the tile's accumulator columns.
template <typename T, int EPI>
__device__ __forceinline__ void dense_epilogue(const DenseParams& p, const DenseAcc& acc, uint8_t* patch, int lane, int row_base, int ct,
                                               int chalf) {
  const int row = row_base + lane;
  const bool rvalid = row < p.M;
  if constexpr (EPI == kEpiLinear) {
#pragma unroll 1
    for (int blk = chalf * 128; blk < chalf * 128 + 128; blk += 64) {       // 64 columns: one 8-bit block
      const int col0 = ct * 256 + blk;
      if (col0 >= p.N) break;
      RowQuant rq;
      if (p.keep_q != nullptr) {
        uint32_t m = 0;
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          float v[32];
          acc.fetch(blk + c, v);
          add_bias32<T>(v, p.bias, col0 + c, p.N);
          m = max(m, chunk_amax_bits(v, col0 + c, p.N));
        }
        rq = make_block_quant(__uint_as_float(m), m < 0x7f800000u);
        if (rvalid) p.keep_scale[static_cast<int64_t>(row) * (p.keep_ld / kKeepBlock) + col0 / kKeepBlock] = rq.scale;
      }
#pragma unroll 1
      for (int c = 0; c < 64; c += 32) {
        const int col = col0 + c;
        if (col >= p.N && p.keep_q == nullptr) break;
        float v[32];
        acc.fetch(blk + c, v);
        add_bias32<T>(v, p.bias, col, p.N);
        if (p.keep_q != nullptr) {
          if (rvalid) store_q32(v, rq, p.keep_q + static_cast<int64_t>(row) * p.keep_ld + col, col, p.N);
        } else if (p.keep != nullptr) {
          store_rows32<T>(patch, lane, v, static_cast<T*>(p.keep), p.keep_ld, row_base, p.M, col, p.N);
        }
        if (col >= p.N) continue;
        if (p.act != TAB_ACT_NONE)
          with_act(p.act, [&](auto tag) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = act_value<decltype(tag)::value>(v[j]);
          });
        if (p.residual != nullptr) {
          uint32_t r[16];
          load_rows32<T>(patch, lane, r, static_cast<const T*>(p.residual), p.N, row_base, p.M, col, p.N);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 f = unpack2<T>(r[j]);
            v[2 * j] += f.x;
            v[2 * j + 1] += f.y;
          }
        }
        store_rows32<T>(patch, lane, v, static_cast<T*>(p.out), p.N, row_base, p.M, col, p.N);
      }
    }
  } else if constexpr (EPI == kEpiGlu) {
    // accumulator columns [128 chalf, +64) are gate features col0 .., [128 chalf + 64, +64) the matching up features
    const int col0 = ct * 128 + chalf * 64;
    if (col0 >= p.N) return;
    const T* bias_up = p.bias ? static_cast<const T*>(p.bias) + p.N : nullptr;
    RowQuant rg, ru;
    if (p.keep_q != nullptr) {
      uint32_t mg = 0, mu = 0;
#pragma unroll 1
      for (int c = 0; c < 64; c += 32) {
        float v[32];
        acc.fetch(chalf * 128 + c, v);
        add_bias32<T>(v, p.bias, col0 + c, p.N);
        mg = max(mg, chunk_amax_bits(v, col0 + c, p.N));
        acc.fetch(chalf * 128 + 64 + c, v);
        add_bias32<T>(v, bias_up, col0 + c, p.N);
        mu = max(mu, chunk_amax_bits(v, col0 + c, p.N));
      }
      rg = make_block_quant(__uint_as_float(mg), mg < 0x7f800000u);
      ru = make_block_quant(__uint_as_float(mu), mu < 0x7f800000u);
      if (rvalid) {
        float* s = p.keep_scale + static_cast<int64_t>(row) * (p.keep_ld / kKeepBlock) + col0 / kKeepBlock;
        s[0] = rg.scale;
        s[p.keep_up / kKeepBlock] = ru.scale;
      }
    }
#pragma unroll 1
    for (int c = 0; c < 64; c += 32) {
      const int col = col0 + c;
      if (col >= p.N && p.keep_q == nullptr) break;
      float g[32], u[32];
      acc.fetch(chalf * 128 + c, g);
      acc.fetch(chalf * 128 + 64 + c, u);
      add_bias32<T>(g, p.bias, col, p.N);
      add_bias32<T>(u, bias_up, col, p.N);
      if (p.keep_q != nullptr) {
        if (rvalid) {
          int8_t* q = p.keep_q + static_cast<int64_t>(row) * p.keep_ld + col;
          store_q32(g, rg, q, col, p.N);
          store_q32(u, ru, q + p.keep_up, col, p.N);
        }
      } else if (p.keep != nullptr) {
        store_rows32<T>(patch, lane, g, static_cast<T*>(p.keep), p.keep_ld, row_base, p.M, col, p.N);
        store_rows32<T>(patch, lane, u, static_cast<T*>(p.keep) + p.keep_up, p.keep_ld, row_base, p.M, col, p.N);
      }
      if (col >= p.N) continue;
      with_act(p.act, [&](auto tag) {
#pragma unroll
        for (int j = 0; j < 32; ++j) g[j] = act_value<decltype(tag)::value>(g[j]) * u[j];
      });
      store_rows32<T>(patch, lane, g, static_cast<T*>(p.out), p.N, row_base, p.M, col, p.N);
    }
  } else {
#pragma unroll 1
    for (int c = chalf * 128; c < chalf * 128 + 128; c += 32) {
      const int col = ct * 256 + c;
      if (col >= p.N) break;
      float g[32], u[32], dh[32];
      if (p.keep_q != nullptr) {
        if (rvalid) {
          const int8_t* q = p.keep_q + static_cast<int64_t>(row) * p.keep_ld + col;
          const float* s = p.keep_scale + static_cast<int64_t>(row) * (p.keep_ld / kKeepBlock) + col / kKeepBlock;
          load_q32(g, q, __ldg(s));
          load_q32(u, q + p.keep_up, __ldg(s + p.keep_up / kKeepBlock));
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) g[j] = u[j] = 0.f;
        }
      } else {
        uint32_t r[16];
        load_rows32<T>(patch, lane, r, static_cast<const T*>(p.keep), p.keep_ld, row_base, p.M, col, p.N);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 f = unpack2<T>(r[j]);
          g[2 * j] = f.x;
          g[2 * j + 1] = f.y;
        }
        load_rows32<T>(patch, lane, r, static_cast<const T*>(p.keep) + p.keep_up, p.keep_ld, row_base, p.M, col, p.N);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 f = unpack2<T>(r[j]);
          u[2 * j] = f.x;
          u[2 * j + 1] = f.y;
        }
      }
      acc.fetch(c, dh);
      // h = a u, d(gate) = dh u a', d(up) = dh a; g, u and dh are overwritten in turn
      with_act(p.act, [&](auto tag) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          float a, d;
          act_both<decltype(tag)::value>(g[j], a, d);
          const float h = a * u[j];
          g[j] = dh[j] * u[j] * d;
          u[j] = dh[j] * a;
          dh[j] = h;
        }
      });
      store_rows32<T>(patch, lane, g, static_cast<T*>(p.dgate), 2 * static_cast<int64_t>(p.N), row_base, p.M, col, p.N);
      store_rows32<T>(patch, lane, u, static_cast<T*>(p.dgate) + p.N, 2 * static_cast<int64_t>(p.N), row_base, p.M, col, p.N);
      store_rows32<T>(patch, lane, dh, static_cast<T*>(p.out), p.N, row_base, p.M, col, p.N);
    }
  }
}

template <typename T, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kDpThreads, 1)
dense_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const DenseParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const uint32_t tiles_addr = ptx::smem_u32(smem);
  uint8_t* ctrl = smem + kDpStages * kDpStageBytes;
  const uint32_t bar0 = ptx::smem_u32(ctrl);
  auto bar_full = [&](int s) { return bar0 + 8u * s; };
  auto bar_empty = [&](int s) { return bar0 + 8u * (kDpStages + s); };
  auto bar_tfull = [&](int b) { return bar0 + 8u * (2 * kDpStages + b); };
  auto bar_tempty = [&](int b) { return bar0 + 8u * (2 * kDpStages + kDpBufs + b); };
  const uint32_t bar_drain = bar0 + 8u * (2 * kDpStages + 2 * kDpBufs);
  const uint32_t bar_done = bar_drain + 8u;            // the peer no longer touches this CTA's shared state
  static_assert(8 * (2 * kDpStages + 2 * kDpBufs + 2) <= 224, "barriers overflow the control block");
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(ctrl + 224);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  volatile int* s_got = reinterpret_cast<volatile int*>(s_tmem + 2);     // [2] outcome of the epilogue's wait, per buffer
  volatile int* s_last = reinterpret_cast<volatile int*>(s_tmem + 4);    // this CTA arrived last at the split tile
  uint8_t* s_out = ctrl + kDpCtrlBytes;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = p.row_tiles * p.col_tiles;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kDpStages; ++s) {
      ptx::mbar_init(bar_full(s), 1);                      // armed by the leader's producer for the bytes of both CTAs
      ptx::mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < kDpBufs; ++b) {
      ptx::mbar_init(bar_tfull(b), 1);
      ptx::mbar_init(bar_tempty(b), 2 * kDpEpiWarps);      // epilogue warps of both CTAs
    }
    ptx::mbar_init(bar_drain, 1);
    ptx::mbar_init(bar_done, 1);
    *s_abort = 0;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&tm_a);
    ptx::prefetch_tensormap(&tm_b);
  }
  if (warp == 1) ptx::tmem_alloc_pair<kDpBufs * kDpCols>(ptx::smem_u32(s_tmem));
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync_all();          // both CTAs' barriers exist before anything signals across the pair
  ptx::tc_fence_after();
  const uint32_t tmem_base = *s_tmem;

  if (warp == 0) {
    // ---------------- TMA producer (one per CTA): own 128 rows of A, own half of the tile's rows of B ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      DenseSched sched(pair, pairs, p.sk_tiles, tiles, p.num_kb);
      DenseWork w;
      while (ok && sched.next(w)) {
        int rt, ct;
        dense_tile_coord(w.tile, p.row_tiles, p.col_tiles, rt, ct);
        const int a0 = rt * 256 + rank * 128;
        const int b0 = EPI == kEpiGlu ? ct * 128 + rank * 64 : ct * 256 + rank * 128;
        const int b1 = EPI == kEpiGlu ? p.N + b0 : b0 + 64;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!dense_wait(bar_empty(stage), phase ^ 1u, s_abort, 31, p.wait_cycles)) { ok = false; break; }
          const uint32_t st = tiles_addr + stage * kDpStageBytes;
          const uint32_t full_leader = ptx::mapa(bar_full(stage), 0);
          if (leader) ptx::mbar_expect_tx(bar_full(stage), 2 * kDpStageBytes);
          const int k = kb * kDnBlockK;
          if (p.a_mn) {
            ptx::tma_load_2d_pair(st, &tm_a, full_leader, a0, k);
            ptx::tma_load_2d_pair(st + kDnBoxBytes, &tm_a, full_leader, a0 + 64, k);
          } else {
            ptx::tma_load_2d_pair(st, &tm_a, full_leader, k, a0);
            ptx::tma_load_2d_pair(st + kDnBoxBytes, &tm_a, full_leader, k, a0 + 64);
          }
          const uint32_t sb = st + kDnOperandBytes;
          if (p.b_mn) {
            ptx::tma_load_2d_pair(sb, &tm_b, full_leader, b0, k);
            ptx::tma_load_2d_pair(sb + kDnBoxBytes, &tm_b, full_leader, b1, k);
          } else {
            ptx::tma_load_2d_pair(sb, &tm_b, full_leader, k, b0);
            ptx::tma_load_2d_pair(sb + kDnBoxBytes, &tm_b, full_leader, k, b1);
          }
          if (++stage == kDpStages) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer: the leader's warp, for both CTAs ----------------
    if (lane == 0 && leader) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, tphase = 0;
      bool ok = true;
      const uint32_t a_step = p.a_mn ? 128u : 2u, b_step = p.b_mn ? 128u : 2u;    // 16 contraction elements, in 16-byte units
      DenseSched sched(pair, pairs, p.sk_tiles, tiles, p.num_kb);
      DenseWork w;
      while (sched.next(w)) {
        if (!dense_wait(bar_tempty(buf), tphase ^ 1u, s_abort, 32, p.wait_cycles)) { ok = false; break; }
        ptx::tc_fence_after();
        const uint32_t d = tmem_base + buf * kDpCols;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!dense_wait(bar_full(stage), phase, s_abort, 33, p.wait_cycles)) { ok = false; break; }
          ptx::tc_fence_after();
          const uint32_t st = tiles_addr + stage * kDpStageBytes;
          const uint64_t a = p.a_mn ? ptx::smem_desc_mn128(st, kDnBoxBytes) : ptx::smem_desc_k128(st);
          const uint64_t b = p.b_mn ? ptx::smem_desc_mn128(st + kDnOperandBytes, kDnBoxBytes) : ptx::smem_desc_k128(st + kDnOperandBytes);
#pragma unroll
          for (int k = 0; k < kDnBlockK / 16; ++k)
            ptx::mma_f16_pair(d, a + k * a_step, b + k * b_step, p.idesc, (kb > w.kb0 || k > 0) ? 1u : 0u);
          ptx::mma_commit_pair(bar_empty(stage));
          if (++stage == kDpStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        ptx::mma_commit_pair(bar_tfull(buf));
        if (++buf == kDpBufs) { buf = 0; tphase ^= 1u; }
      }
      if (!ok) {
        ptx::mma_commit_pair(bar_drain);
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait(bar_drain, 0) && clock64() - t0 < p.wait_cycles) {}
      }
    }
  } else {
    // ---------------- epilogue: warps 2..9, thread = row, two warps split the columns of a row ----------------
    const int quarter = warp & 3;
    const int chalf = (warp - 2) >> 2;
    const int et = threadIdx.x - 64;
    uint8_t* patch = s_out + (warp - 2) * kDpPatchBytes;
    int buf = 0;
    uint32_t tphase = 0;
    DenseAcc acc;
    acc.units = static_cast<int64_t>(p.sk_tiles) * p.num_kb;
    acc.pairs = pairs;
    acc.num_kb = p.num_kb;
    acc.self = pair;
    acc.rank = rank;
    acc.row_local = quarter * 32 + lane;
    DenseSched sched(pair, pairs, p.sk_tiles, tiles, p.num_kb);
    DenseWork w;
    while (sched.next(w)) {
      if (et == 0) s_got[buf] = dense_wait(bar_tfull(buf), tphase, s_abort, 34, p.wait_cycles) ? 1 : 0;
      dense_epi_bar();
      if (!s_got[buf]) break;
      ptx::tc_fence_after();
      int rt, ct;
      dense_tile_coord(w.tile, p.row_tiles, p.col_tiles, rt, ct);
      acc.taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * kDpCols;
      acc.parts = nullptr;
      acc.tile = w.tile;
      bool finish = true;
      if (w.kb1 - w.kb0 < p.num_kb) {
        // part of a split tile: store it, count the arrival, and only the last CTA to arrive goes on
        float4* dst = reinterpret_cast<float4*>(p.partials + (static_cast<int64_t>(dense_slot(pair, w.kb0)) * 2 + rank) * kDpPartFloats);
#pragma unroll 1
        for (int c = chalf * 128; c < chalf * 128 + 128; c += 32) {
          float v[32];
          acc.fetch(c, v);
#pragma unroll
          for (int k = 0; k < 8; ++k) __stcg(dst + ((c >> 2) + k) * 128 + acc.row_local, make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
        }
        const int64_t u0 = static_cast<int64_t>(w.tile) * p.num_kb;
        acc.first = dense_unit_owner(u0, acc.units, pairs);
        acc.last = dense_unit_owner(u0 + p.num_kb - 1, acc.units, pairs);
        __threadfence();
        dense_epi_bar();
        if (et == 0) {
          const int before = atomicAdd(p.arrivals + w.tile * 2 + rank, 1);
          *s_last = before == acc.last - acc.first ? 1 : 0;
          __threadfence();
        }
        dense_epi_bar();
        finish = *s_last != 0;
        acc.parts = p.partials;
      }
      const int row_base = rt * 256 + rank * 128 + quarter * 32;
      if (finish && row_base < p.M) dense_epilogue<T, EPI>(p, acc, patch, lane, row_base, ct, chalf);
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa(bar_tempty(buf), 0));   // the leader counts both CTAs' warps
      if (++buf == kDpBufs) { buf = 0; tphase ^= 1u; }
    }
  }

  // End of the pair's work: tell the peer, wait (bounded) for the peer, then release tensor memory (gmm_i8_pair.cuh).
  ptx::tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    ptx::mbar_arrive_cluster(ptx::mapa(bar_done, static_cast<uint32_t>(rank) ^ 1u));
    const long long t0 = clock64();
    while (!ptx::mbar_try_wait(bar_done, 0)) {
      if (clock64() - t0 > p.wait_cycles) {
        atomicCAS(&g_dense_status, 0, 35);
        break;
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair<kDpBufs * kDpCols>(tmem_base);
  }
}

}  // namespace tab
