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
// Few tiles.  A product with fewer tiles than pairs leaves SMs idle, and so does the last, partly filled turn of a larger one.
// SPLIT launches give such tiles to clusters of `split` pairs: each pair takes a part of the contraction, leaves its fp32
// accumulators in its own shared memory, and after a cluster barrier finishes its share of the tile's columns, adding the
// parts from distributed shared memory in the order of the contraction.  No workspace, no atomics, no waiting for CTAs that may
// not be resident.  (An earlier form handed out blocks of the contraction evenly over all pairs and joined the parts through
// global memory: 136.9 us instead of 104.5 us for 4096 x 2048 x 8192, where whole tiles fill 1.73 turns.)
//
// Issue.  The producer and MMA loops run on whole warps and elect a lane around the issuing instructions.  Run by a single
// lane, the same loops took 640 cycles per block of the contraction, the MMAs themselves 512 (now 520; 8192^3: 762 -> 728 us).
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
static_assert(128 * kDpCols * 4 <= kDpStages * kDpStageBytes, "a CTA's accumulators fit into its ring");

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

// Where the epilogue takes a tile's accumulators from: tensor memory, or (split tiles) the parts of all pairs of the cluster,
// added in the order of the contraction.
struct DenseAcc {
  uint32_t taddr;          // this warp's lanes, first column of the buffer
  uint32_t part;           // 0, or the shared-memory address of this thread's row in the parts: float4 [column / 4][128 rows]
  int split, parity;       // pairs of the cluster, which CTA of its pair this is
  __device__ __forceinline__ void fetch(int c, float (&v)[32]) const {
    __syncwarp();
    if (part == 0) {
      ptx::tmem_ld32f(taddr + c, v);
      ptx::tmem_ld_wait();
      return;
    }
    const uint32_t at = part + static_cast<uint32_t>(c >> 2) * 2048u;
#pragma unroll 1
    for (int s = 0; s < split; ++s) {
      const uint32_t from = ptx::mapa(at, static_cast<uint32_t>(2 * s + parity));
      float4 t[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = ptx::ld_cluster_f4(from + k * 2048u);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x[4] = {t[k].x, t[k].y, t[k].z, t[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * k + j] = s == 0 ? x[j] : v[4 * k + j] + x[j];
      }
    }
  }
};

// Epilogue of one warp: 32 rows (row_base ..) x the output columns [col_begin, col_end) of the tile (multiples of 32; of 64
// where 8-bit blocks are written).
template <typename T, int EPI>
__device__ __forceinline__ void dense_epilogue(const DenseParams& p, const DenseAcc& acc, uint8_t* patch, int lane, int row_base, int ct,
                                               int col_begin, int col_end) {
  const int row = row_base + lane;
  const bool rvalid = row < p.M;
  if constexpr (EPI == kEpiLinear) {
    RowQuant rq;
#pragma unroll 1
    for (int c = col_begin; c < col_end; c += 32) {
      const int col = ct * 256 + c;
      if (col >= p.N && (p.keep_q == nullptr || (col & ~63) >= p.N)) break;
      if (p.keep_q != nullptr && (c & 63) == 0) {                        // amax of the 64-value block first
        uint32_t m = 0;
#pragma unroll 1
        for (int h = 0; h < 64; h += 32) {
          float v[32];
          acc.fetch(c + h, v);
          add_bias32<T>(v, p.bias, col + h, p.N);
          m = max(m, chunk_amax_bits(v, col + h, p.N));
        }
        rq = make_block_quant(__uint_as_float(m), m < 0x7f800000u);
        if (rvalid) p.keep_scale[static_cast<int64_t>(row) * (p.keep_ld / kKeepBlock) + col / kKeepBlock] = rq.scale;
      }
      float v[32];
      acc.fetch(c, v);
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
  } else if constexpr (EPI == kEpiGlu) {
    // output column c of the tile: its gate is accumulator column (c / 64) * 128 + c % 64, its up value 64 columns further
    const T* bias_up = p.bias ? static_cast<const T*>(p.bias) + p.N : nullptr;
    RowQuant rg, ru;
#pragma unroll 1
    for (int c = col_begin; c < col_end; c += 32) {
      const int col = ct * 128 + c;
      if (col >= p.N && (p.keep_q == nullptr || (col & ~63) >= p.N)) break;
      const int at = (c >> 6) * 128 + (c & 63);
      if (p.keep_q != nullptr && (c & 63) == 0) {
        uint32_t mg = 0, mu = 0;
#pragma unroll 1
        for (int h = 0; h < 64; h += 32) {
          float v[32];
          acc.fetch(at + h, v);
          add_bias32<T>(v, p.bias, col + h, p.N);
          mg = max(mg, chunk_amax_bits(v, col + h, p.N));
          acc.fetch(at + 64 + h, v);
          add_bias32<T>(v, bias_up, col + h, p.N);
          mu = max(mu, chunk_amax_bits(v, col + h, p.N));
        }
        rg = make_block_quant(__uint_as_float(mg), mg < 0x7f800000u);
        ru = make_block_quant(__uint_as_float(mu), mu < 0x7f800000u);
        if (rvalid) {
          float* s = p.keep_scale + static_cast<int64_t>(row) * (p.keep_ld / kKeepBlock) + col / kKeepBlock;
          s[0] = rg.scale;
          s[p.keep_up / kKeepBlock] = ru.scale;
        }
      }
      float g[32], u[32];
      acc.fetch(at, g);
      acc.fetch(at + 64, u);
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
    for (int c = col_begin; c < col_end; c += 32) {
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

// Output columns of a tile: 256, or 128 where gate and up share the accumulator.
template <int EPI>
constexpr int kDpTileCols = EPI == kEpiGlu ? 128 : 256;

template <typename T, int EPI, bool SPLIT>
__global__ void __launch_bounds__(kDpThreads, 1)
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
  uint8_t* s_out = ctrl + kDpCtrlBytes;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = ptx::cluster_ctarank();
  const int rank = static_cast<int>(cta & 1u);           // within the pair
  const uint32_t leader_cta = cta & ~1u;
  const bool leader = rank == 0;
  // this pair's tiles: one of them for the whole cluster, or every `step`-th one
  const int split = SPLIT ? p.split : 1, part = SPLIT ? static_cast<int>(cta >> 1) : 0;
  const int first = p.tile_begin + static_cast<int>(blockIdx.x) / (2 * split);
  const int step = SPLIT ? p.tile_end : static_cast<int>(gridDim.x >> 1);
  const int kb_begin = SPLIT ? static_cast<int>(static_cast<int64_t>(part) * p.num_kb / split) : 0;
  const int kb_end = SPLIT ? static_cast<int>(static_cast<int64_t>(part + 1) * p.num_kb / split) : p.num_kb;

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
  ptx::launch_dependents();

  if (warp == 0) {
    // ---------------- TMA producer (one per CTA): own 128 rows of A, own half of the tile's rows of B ----------------
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full0 = ptx::mapa(bar_full(0), leader_cta);
    for (int tile = first; ok && tile < p.tile_end; tile += step) {
      int rt, ct;
      dense_tile_coord(tile, p.row_tiles, p.col_tiles, rt, ct);
      const int a0 = rt * 256 + rank * 128;
      const int b0 = EPI == kEpiGlu ? ct * 128 + rank * 64 : ct * 256 + rank * 128;
      const int b1 = EPI == kEpiGlu ? p.N + b0 : b0 + 64;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        ok = __all_sync(0xffffffffu, dense_wait(bar_empty(stage), phase ^ 1u, s_abort, 31, p.wait_cycles));
        if (!ok) break;
        const uint32_t st = tiles_addr + stage * kDpStageBytes;
        const uint32_t sb = st + kDnOperandBytes;
        const uint32_t full_leader = full0 + 8u * stage;
        const int k = kb * kDnBlockK;
        if (ptx::elect_one()) {
          if (leader) ptx::mbar_expect_tx(bar_full(stage), 2 * kDpStageBytes);
          // coordinates: contiguous index first
          ptx::tma_load_2d_pair(st, &tm_a, full_leader, p.a_mn ? a0 : k, p.a_mn ? k : a0);
          ptx::tma_load_2d_pair(st + kDnBoxBytes, &tm_a, full_leader, p.a_mn ? a0 + 64 : k, p.a_mn ? k : a0 + 64);
          ptx::tma_load_2d_pair(sb, &tm_b, full_leader, p.b_mn ? b0 : k, p.b_mn ? k : b0);
          ptx::tma_load_2d_pair(sb + kDnBoxBytes, &tm_b, full_leader, p.b_mn ? b1 : k, p.b_mn ? k : b1);
        }
        __syncwarp();
        if (++stage == kDpStages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer: the leader's warp, for both CTAs ----------------
    if (leader) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, tphase = 0;
      bool ok = true;
      const uint16_t both = static_cast<uint16_t>(3u << leader_cta);
      const uint32_t a_step = p.a_mn ? 128u : 2u, b_step = p.b_mn ? 128u : 2u;    // 16 contraction elements, in 16-byte units
      const uint64_t a_first = p.a_mn ? ptx::smem_desc_mn128(tiles_addr, kDnBoxBytes) : ptx::smem_desc_k128(tiles_addr);
      const uint64_t b_first = p.b_mn ? ptx::smem_desc_mn128(tiles_addr + kDnOperandBytes, kDnBoxBytes) : ptx::smem_desc_k128(tiles_addr + kDnOperandBytes);
      for (int tile = first; ok && tile < p.tile_end; tile += step) {
        ok = __all_sync(0xffffffffu, dense_wait(bar_tempty(buf), tphase ^ 1u, s_abort, 32, p.wait_cycles));
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t d = tmem_base + buf * kDpCols;
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          ok = __all_sync(0xffffffffu, dense_wait(bar_full(stage), phase, s_abort, 33, p.wait_cycles));
          if (!ok) break;
          ptx::tc_fence_after();
          const uint64_t a = a_first + static_cast<uint64_t>(stage * (kDpStageBytes >> 4));
          const uint64_t b = b_first + static_cast<uint64_t>(stage * (kDpStageBytes >> 4));
          if (ptx::elect_one()) {
#pragma unroll
            for (int k = 0; k < kDnBlockK / 16; ++k)
              ptx::mma_f16_pair(d, a + k * a_step, b + k * b_step, p.idesc, (kb > kb_begin || k > 0) ? 1u : 0u);
            ptx::mma_commit_mask(bar_empty(stage), both);
          }
          __syncwarp();
          if (++stage == kDpStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if (ptx::elect_one()) ptx::mma_commit_mask(bar_tfull(buf), both);
        __syncwarp();
        if (++buf == kDpBufs) { buf = 0; tphase ^= 1u; }
      }
      if (!ok && lane == 0) {
        ptx::mma_commit_mask(bar_drain, both);
        const long long t0 = clock64();
        while (!ptx::mbar_try_wait(bar_drain, 0) && clock64() - t0 < p.wait_cycles) {}
      }
    }
  } else {
    // ---------------- epilogue: warps 2..9, thread = row, two warps share the columns of a row ----------------
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    const int et = threadIdx.x - 64;
    int buf = 0;
    uint32_t tphase = 0;
    DenseAcc acc;
    acc.part = 0;
    for (int tile = first; tile < p.tile_end; tile += step) {
      if (et == 0) s_got[buf] = dense_wait(bar_tfull(buf), tphase, s_abort, 34, p.wait_cycles) ? 1 : 0;
      dense_epi_bar();
      if (!s_got[buf]) break;
      ptx::tc_fence_after();
      acc.taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * kDpCols;
      if constexpr (SPLIT) {
        // all MMAs of this pair are done, so its ring is free: it takes the 128 x 256 accumulators
        const uint32_t dst = tiles_addr + static_cast<uint32_t>(quarter * 32 + lane) * 16u;
#pragma unroll 1
        for (int c = half * 128; c < half * 128 + 128; c += 32) {
          float v[32];
          acc.fetch(c, v);
#pragma unroll
          for (int k = 0; k < 8; ++k) ptx::st_shared_f4(dst + static_cast<uint32_t>((c >> 2) + k) * 2048u, make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
        }
      } else {
        int rt, ct;
        dense_tile_coord(tile, p.row_tiles, p.col_tiles, rt, ct);
        const int row_base = rt * 256 + rank * 128 + quarter * 32;
        constexpr int kHalf = kDpTileCols<EPI> / 2;
        if (row_base < p.M) dense_epilogue<T, EPI>(p, acc, s_out + (warp - 2) * kDpPatchBytes, lane, row_base, ct, half * kHalf, half * kHalf + kHalf);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa(bar_tempty(buf), leader_cta));   // the leader counts both CTAs' warps
      if (++buf == kDpBufs) { buf = 0; tphase ^= 1u; }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (SPLIT) {
    ptx::cluster_sync_all();          // every pair's part is in place
    if (warp >= 2) {
      // this pair's share of the tile's columns, halved again between the two warps of a row; 64-value blocks are not cut, so
      // with four pairs some hold no share (which pairs share a tile must not depend on what is kept: the sums would differ)
      int rt, ct;
      dense_tile_coord(first, p.row_tiles, p.col_tiles, rt, ct);
      const int quarter = warp & 3, half = (warp - 2) >> 2;
      const int unit = p.keep_q != nullptr && EPI != kEpiGluGrad ? 64 : 32;
      const int share = max(kDpTileCols<EPI> / split, unit);
      const int mid = share / 2 % unit == 0 ? share / 2 : share;
      const int begin = part * share + (half ? mid : 0);
      const int end = min(part * share + (half ? share : mid), kDpTileCols<EPI>);
      const int row_base = rt * 256 + rank * 128 + quarter * 32;
      DenseAcc acc;
      acc.taddr = 0;
      acc.part = tiles_addr + static_cast<uint32_t>(quarter * 32 + lane) * 16u;
      acc.split = split;
      acc.parity = rank;
      if (row_base < p.M) dense_epilogue<T, EPI>(p, acc, s_out + (warp - 2) * kDpPatchBytes, lane, row_base, ct, begin, end);
    }
    __syncthreads();
    ptx::cluster_sync_all();          // nobody leaves while another still reads its part or its operands
  } else {
    // The peer may still read this CTA's shared memory (its MMAs) or signal its barriers: tell the peer, wait (bounded) for it.
    if (threadIdx.x == 0) {
      ptx::mbar_arrive_cluster(ptx::mapa(bar_done, cta ^ 1u));
      const long long t0 = clock64();
      while (!ptx::mbar_try_wait(bar_done, 0)) {
        if (clock64() - t0 > p.wait_cycles) {
          atomicCAS(&g_dense_status, 0, 35);
          break;
        }
      }
    }
    __syncthreads();
  }
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair<kDpBufs * kDpCols>(tmem_base);
  }
  // a launch that was allowed to start under the one before it ends only after that one has
  if (threadIdx.x == 0) ptx::dependency_wait();
}

}  // namespace tab
