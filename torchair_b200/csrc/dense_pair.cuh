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
// The epilogue of kEpiGluGrad stages three streams of values instead of two, at the price of one stage of the ring.
template <int EPI>
constexpr int kDpStages = EPI == kEpiGluGrad ? 5 : 6;
constexpr int kDpBufs = 2;
constexpr int kDpCols = 256;
constexpr int kDpEpiWarps = 16;                        // four per TMEM lane quarter, each takes a quarter of the columns
constexpr int kDpThreads = 64 + kDpEpiWarps * 32;
constexpr int kDpCtrlBytes = 256;
constexpr int kDpPatch = 1024;                         // staging area of an epilogue warp: 32 rows x 16 16-bit values
template <int EPI>
constexpr int kDpPatches = EPI == kEpiGluGrad ? 3 : 2;
template <int EPI>
constexpr int kDpSmemBytes = 1024 + kDpStages<EPI> * kDpStageBytes + kDpCtrlBytes + kDpEpiWarps * kDpPatches<EPI> * kDpPatch;
static_assert(kDpSmemBytes<kEpiLinear> <= kDnSmemLimit && kDpSmemBytes<kEpiGluGrad> <= kDnSmemLimit, "dense pair GEMM shared memory");
static_assert(128 * kDpCols * 4 <= 5 * kDpStageBytes, "a CTA's accumulators fit into its ring");

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

// ---- epilogue ------------------------------------------------------------------------------------------------------------
// Sixteen warps, four to a scheduler: a step (16 accumulator columns of a row per thread: read, bias, activation, pack, store) is
// a chain of latencies, and with half the warps a tile's plain epilogue took 6400 cycles, its silu 11300, against 8300 for the
// main loop at K = 1024.  16-bit values pass between registers and row-major memory through patches of 32 rows x 16 columns, so
// that global accesses are 16 bytes per lane, two lanes to a row's 32-byte sector.  Rows >= M and columns >= N are left alone
// (loads give zeros); N is a multiple of 8, no 16-byte piece is ever cut.  (kEpiLinearAny moves results, residuals and biases
// element by element instead.)
__device__ __forceinline__ uint32_t patch_at(int row, int piece) { return static_cast<uint32_t>(row * 32 + ((piece ^ ((row >> 2) & 1)) << 4)); }

template <typename T>
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& x, float* v) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ void patch_put(uint8_t* patch, int lane, const float (&v)[16]) {
  *reinterpret_cast<uint4*>(patch + patch_at(lane, 0)) = pack8<T>(v);
  *reinterpret_cast<uint4*>(patch + patch_at(lane, 1)) = pack8<T>(v + 8);
}
template <typename T>
__device__ __forceinline__ void patch_get(const uint8_t* patch, int lane, float (&v)[16]) {
  unpack8<T>(*reinterpret_cast<const uint4*>(patch + patch_at(lane, 0)), v);
  unpack8<T>(*reinterpret_cast<const uint4*>(patch + patch_at(lane, 1)), v + 8);
}

// patch -> memory; the warp has met since the patch was written and meets again before it is written anew
template <typename T>
__device__ __forceinline__ void patch_store(const uint8_t* patch, int lane, T* base, int64_t ld, int row_base, int rows_end, int col, int cols) {
  const int c = col + (lane & 1) * 8;
  if (c < cols) {
    T* dst = base + static_cast<int64_t>(row_base + (lane >> 1)) * ld + c;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = i * 16 + (lane >> 1);
      if (row_base + r < rows_end) *reinterpret_cast<uint4*>(dst + i * 16 * ld) = *reinterpret_cast<const uint4*>(patch + patch_at(r, lane & 1));
    }
  }
}

// The same for rows that begin anywhere: element by element, 16 lanes to a row.
template <typename T>
__device__ __forceinline__ void patch_store_any(const uint8_t* patch, int lane, T* base, int64_t ld, int row_base, int rows_end, int col, int cols) {
  const int c = lane & 15;
  if (col + c >= cols) return;
#pragma unroll 4
  for (int r = lane >> 4; r < 32; r += 2)
    if (row_base + r < rows_end)
      base[static_cast<int64_t>(row_base + r) * ld + col + c] = *reinterpret_cast<const T*>(patch + patch_at(r, c >> 3) + (c & 7) * 2);
}
template <typename T>
__device__ __forceinline__ void patch_load_any(uint8_t* patch, int lane, const T* base, int64_t ld, int row_base, int rows_end, int col, int cols) {
  const int c = lane & 15;
#pragma unroll 4
  for (int r = lane >> 4; r < 32; r += 2)
    *reinterpret_cast<T*>(patch + patch_at(r, c >> 3) + (c & 7) * 2) =
        col + c < cols && row_base + r < rows_end ? base[static_cast<int64_t>(row_base + r) * ld + col + c] : Elem<T>::from_f32(0.f);
}

// memory -> registers, as the patch will be filled from them
struct Ahead {
  uint4 x[2];
  template <typename T>
  __device__ __forceinline__ void load(int lane, const T* base, int64_t ld, int row_base, int rows_end, int col, int cols) {
    const int c = col + (lane & 1) * 8;
    const T* src = base + static_cast<int64_t>(row_base + (lane >> 1)) * ld + c;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[i] = make_uint4(0u, 0u, 0u, 0u);
      if (c < cols && row_base + i * 16 + (lane >> 1) < rows_end) x[i] = __ldg(reinterpret_cast<const uint4*>(src + i * 16 * ld));
    }
  }
  __device__ __forceinline__ void put(uint8_t* patch, int lane) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) *reinterpret_cast<uint4*>(patch + patch_at(i * 16 + (lane >> 1), lane & 1)) = x[i];
  }
};

// v[0..15] += bias[col .. col + 15]; the loads are asked for before the accumulators (columns beyond cols are not stored)
template <typename T>
struct Bias16 {
  uint4 x[2];
  __device__ __forceinline__ void load(const void* bias, int col, int cols, bool ragged) {
    const T* b = static_cast<const T*>(bias);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      x[k] = make_uint4(0u, 0u, 0u, 0u);
      if (ragged) {
        float v[8];
        load8_any(b, col + 8 * k, cols, v);
        x[k] = pack8<T>(v);
      } else if (col + 8 * k < cols) {
        x[k] = __ldg(reinterpret_cast<const uint4*>(b + col + 8 * k));
      }
    }
  }
  __device__ __forceinline__ void add(float (&v)[16]) const {
    float b[16];
    unpack8<T>(x[0], b);
    unpack8<T>(x[1], b + 8);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += b[i];
  }
};

// largest magnitude as bits (NaN > infinity > every finite value); columns beyond cols do not count
__device__ __forceinline__ uint32_t amax_bits16(const float (&v)[16], int col, int cols) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (col + (j & ~7) < cols) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  return m;
}

// 16 values of this thread's row -> 16 int8 at q (16-byte aligned); columns beyond cols become 0
__device__ __forceinline__ void store_q16(const float (&v)[16], const RowQuant& rq, int8_t* q, int col, int cols) {
  uint2 o[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    o[k] = make_uint2(0u, 0u);
    if (col + 8 * k < cols) {
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = v[8 * k + i];
      o[k] = block_quant8(t, rq);
    }
  }
  *reinterpret_cast<uint4*>(q) = make_uint4(o[0].x, o[0].y, o[1].x, o[1].y);
}

__device__ __forceinline__ void unpack_q16(const uint4& a, float scale, float (&v)[16]) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * k + i] = static_cast<float>(static_cast<int8_t>(w[k] >> (8 * i))) * scale;
}

// Where the epilogue takes a tile's accumulators from: tensor memory, or (split tiles) the parts of all pairs of the cluster,
// added in the order of the contraction.
struct DenseAcc {
  uint32_t taddr;          // this warp's lanes, first column of the buffer
  uint32_t part;           // 0, or the shared-memory address of this thread's row in the parts: float4 [column / 4][128 rows]
  int split, parity;       // pairs of the cluster, which CTA of its pair this is
  uint32_t release_bar;    // the leader's barrier that counts this buffer's readers (0: nothing to release)

  __device__ __forceinline__ void fetch(int c, float (&v)[16]) const {
    __syncwarp();
    if (part == 0) {
      ptx::tmem_ld16f(taddr + c, v);
      ptx::tmem_ld_wait();
      return;
    }
    const uint32_t at = part + static_cast<uint32_t>(c >> 2) * 2048u;
#pragma unroll 1
    for (int s = 0; s < split; ++s) {
      const uint32_t from = ptx::mapa(at, static_cast<uint32_t>(2 * s + parity));
      float4 t[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] = ptx::ld_cluster_f4(from + k * 2048u);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float x[4] = {t[k].x, t[k].y, t[k].z, t[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * k + j] = s == 0 ? x[j] : v[4 * k + j] + x[j];
      }
    }
  }
  // this warp has read all it needs: the next tile's MMAs may overwrite the buffer while its results are still being stored
  __device__ __forceinline__ void release(int lane) {
    if (release_bar == 0) return;
    ptx::tc_fence_before();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive_cluster_relaxed(release_bar);
    release_bar = 0;
  }
};

// Epilogue of one warp: 32 rows (row_base ..) x the output columns [col_begin, col_end) of the tile (multiples of 16).  What it
// reads from global memory (residual, kept values) is asked for before the accumulators are waited for, then one step ahead.
//
// Rounding.  The kept values of kEpiGlu and kEpiLinear, the hidden rows of kEpiGlu and the three results of kEpiGluGrad go to HBM
// in the operands' 16 bits: the next product takes 16-bit operands anyway, and the values that only the backward pass reads would
// cost twice the bytes in fp32 (3001 x 2 x 1408 of them: 17 MB more per direction) for an error that stays below that of the
// operands' own rounding.  The activation and the products of the epilogue see the fp32 accumulator, not its rounded copy.
template <typename T, int EPI>
struct TileEpilogue {
  const DenseParams& p;
  uint8_t* patch;
  int lane, row_base, ct, col_begin, col_end;
  bool rvalid;
  Ahead r0, r1;            // residual (kEpiLinear); kept gate and up (kEpiGluGrad)
  uint32_t bias_pair;      // lane l: two bias values of this warp's columns (kEpiGlu: lanes 16.. those of the up values)

  __device__ __forceinline__ TileEpilogue(const DenseParams& p_, uint8_t* patch_, int lane_, int row_base_, int ct_, int begin, int end)
      : p(p_), patch(patch_), lane(lane_), row_base(row_base_), ct(ct_), col_begin(begin), col_end(end), rvalid(row_base_ + lane_ < p_.M) {}

  __device__ __forceinline__ void look_ahead(int c) {
    const int col = ct * 256 + c;
    if constexpr (EPI == kEpiLinear) {
      if (p.residual != nullptr) r0.load(lane, static_cast<const T*>(p.residual), p.N, row_base, p.M, col, p.N);
    }
    if constexpr (EPI == kEpiGluGrad) {
      if (p.keep_q == nullptr) {
        r0.load(lane, static_cast<const T*>(p.keep), p.keep_ld, row_base, p.M, col, p.N);
        r1.load(lane, static_cast<const T*>(p.keep) + p.keep_up, p.keep_ld, row_base, p.M, col, p.N);
      }
    }
  }

  // Before the wait for the accumulators.  The bias of all of a warp's columns (64, or 32 pairs) fits one register per lane and is
  // handed out by shuffles: asked for step by step, every step waited for L2.
  __device__ __forceinline__ void prefetch() {
    if (row_base >= p.M || col_begin >= col_end) return;
    look_ahead(col_begin);
    bias_pair = 0u;
    if (EPI != kEpiGluGrad && p.bias != nullptr) {
      const bool up = EPI == kEpiGlu && lane >= 16;
      const int col = ct * (EPI == kEpiGlu ? 128 : 256) + col_begin + 2 * (up ? lane - 16 : lane);
      const T* b = static_cast<const T*>(p.bias) + (up ? p.N : 0);
      if (EPI == kEpiLinearAny)
        bias_pair = pack2<T>(col < p.n_out ? Elem<T>::to_f32(b[col]) : 0.f, col + 1 < p.n_out ? Elem<T>::to_f32(b[col + 1]) : 0.f);
      else if (col < p.N)
        bias_pair = __ldg(reinterpret_cast<const uint32_t*>(b + col));
    }
  }
  // v[0..15] += bias of the 16 columns from c on (first_lane: where the pair of col_begin is held)
  __device__ __forceinline__ void add_bias(float (&v)[16], int c, int first_lane) const {
    const int from = first_lane + ((c - col_begin) >> 1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 b = unpack2<T>(__shfl_sync(0xffffffffu, bias_pair, from + i));
      v[2 * i] += b.x;
      v[2 * i + 1] += b.y;
    }
  }

  __device__ __forceinline__ void run(DenseAcc& acc) {
    if (row_base < p.M && col_begin < col_end) {
      if constexpr (epi_linear(EPI)) linear(acc);
      if constexpr (EPI == kEpiGlu) glu(acc);
      if constexpr (EPI == kEpiGluGrad) glu_grad(acc);
    }
    acc.release(lane);
  }

  // The quantiser of the 64 columns from accumulator column `at` on, whose output columns begin at col.  A block may be shared by
  // several warps: each takes the amax of all of it, the one that holds its first column stores the scale.
  __device__ __forceinline__ RowQuant block_quant(const DenseAcc& acc, const void* bias, int at, int col, float* scale, bool first) const {
    uint32_t m = 0;
#pragma unroll 1
    for (int h = 0; h < 64; h += 16) {
      float v[16];
      Bias16<T> b;
      if (bias != nullptr) b.load(bias, col + h, EPI == kEpiLinearAny ? p.n_out : p.N, EPI == kEpiLinearAny);
      acc.fetch(at + h, v);
      if (bias != nullptr) b.add(v);
      m = max(m, amax_bits16(v, col + h, p.N));
    }
    const RowQuant rq = make_block_quant(__uint_as_float(m), m < 0x7f800000u);
    if (rvalid && first) *scale = rq.scale;
    return rq;
  }

  __device__ __forceinline__ void linear(DenseAcc& acc) {
    const int64_t row = row_base + lane;
    const bool has_bias = p.bias != nullptr, has_res = p.residual != nullptr, keep8 = p.keep_q != nullptr, keep16 = !keep8 && p.keep != nullptr;
    const int act = p.act;
    constexpr bool ragged = EPI == kEpiLinearAny;
    uint8_t *main_patch = patch, *side_patch = patch + kDpPatch;
    RowQuant rq;
#pragma unroll 1
    for (int c = col_begin; c < col_end; c += 16) {
      const int col = ct * 256 + c;
      if (col >= p.N && (!keep8 || (col & ~63) >= p.N)) break;
      if (keep8 && ((c & 63) == 0 || c == col_begin))
        rq = block_quant(acc, p.bias, c & ~63, col & ~63, p.keep_scale + row * (p.keep_ld / kKeepBlock) + col / kKeepBlock, (c & 63) == 0);
      float v[16];
      if (has_res) {
        if (ragged) patch_load_any<T>(main_patch, lane, static_cast<const T*>(p.residual), p.n_out, row_base, p.M, col, p.n_out);
        else r0.put(main_patch, lane);
      }
      acc.fetch(c, v);                                   // (the warp meets in there)
      if (c + 16 >= col_end) acc.release(lane);
      if (has_bias) add_bias(v, c, 0);
      if (keep8) {
        if (rvalid) store_q16(v, rq, p.keep_q + row * p.keep_ld + col, col, p.N);
      } else if (keep16) {
        patch_put<T>(side_patch, lane, v);
      }
      if (act != TAB_ACT_NONE)
        with_act(act, [&](auto tag) { act_values<decltype(tag)::value>(v); });
      if (has_res) {
        float r[16];
        patch_get<T>(main_patch, lane, r);
        if (c + 16 < col_end) look_ahead(c + 16);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] += r[j];
      }
      patch_put<T>(main_patch, lane, v);
      __syncwarp();
      if (keep16) patch_store<T>(side_patch, lane, static_cast<T*>(p.keep), p.keep_ld, row_base, p.M, col, p.N);
      if (ragged) patch_store_any<T>(main_patch, lane, static_cast<T*>(p.out), p.n_out, row_base, p.M, col, p.n_out);
      else patch_store<T>(main_patch, lane, static_cast<T*>(p.out), p.N, row_base, p.M, col, p.N);
      __syncwarp();
    }
  }

  __device__ __forceinline__ void glu(DenseAcc& acc) {
    // output column c of the tile: its gate is accumulator column (c / 64) * 128 + c % 64, its up value 64 columns further
    const int64_t row = row_base + lane;
    const bool has_bias = p.bias != nullptr, keep8 = p.keep_q != nullptr, keep16 = !keep8 && p.keep != nullptr;
    const T* bias_up = static_cast<const T*>(p.bias) + p.N;
    uint8_t *pg = patch, *pu = patch + kDpPatch;
    RowQuant rg, ru;
#pragma unroll 1
    for (int c = col_begin; c < col_end; c += 16) {
      const int col = ct * 128 + c;
      if (col >= p.N && (!keep8 || (col & ~63) >= p.N)) break;
      const int at = (c >> 6) * 128 + (c & 63);
      if (keep8 && ((c & 63) == 0 || c == col_begin)) {
        float* scale = p.keep_scale + row * (p.keep_ld / kKeepBlock) + col / kKeepBlock;
        const int block_at = (c >> 6) * 128;
        rg = block_quant(acc, p.bias, block_at, col & ~63, scale, (c & 63) == 0);
        ru = block_quant(acc, has_bias ? bias_up : nullptr, block_at + 64, col & ~63, scale + p.keep_up / kKeepBlock, (c & 63) == 0);
      }
      float g[16], u[16];
      acc.fetch(at, g);
      acc.fetch(at + 64, u);
      if (c + 16 >= col_end) acc.release(lane);
      if (has_bias) {
        add_bias(g, c, 0);
        add_bias(u, c, 16);
      }
      if (keep8) {
        if (rvalid) {
          int8_t* q = p.keep_q + row * p.keep_ld + col;
          store_q16(g, rg, q, col, p.N);
          store_q16(u, ru, q + p.keep_up, col, p.N);
        }
      } else if (keep16) {
        patch_put<T>(pg, lane, g);
        patch_put<T>(pu, lane, u);
        __syncwarp();
        patch_store<T>(pg, lane, static_cast<T*>(p.keep), p.keep_ld, row_base, p.M, col, p.N);
        patch_store<T>(pu, lane, static_cast<T*>(p.keep) + p.keep_up, p.keep_ld, row_base, p.M, col, p.N);
        __syncwarp();
      }
      with_act(p.act, [&](auto tag) { act_gate<decltype(tag)::value>(g, u); });
      patch_put<T>(pg, lane, g);
      __syncwarp();
      patch_store<T>(pg, lane, static_cast<T*>(p.out), p.N, row_base, p.M, col, p.N);
      __syncwarp();
    }
  }

  __device__ __forceinline__ void glu_grad(DenseAcc& acc) {
    const int64_t row = row_base + lane;
    const int64_t ld2 = 2 * static_cast<int64_t>(p.N);
    const bool keep8 = p.keep_q != nullptr;
    uint8_t *pg = patch, *pu = patch + kDpPatch, *ph = patch + 2 * kDpPatch;
#pragma unroll 1
    for (int c = col_begin; c < col_end; c += 16) {
      const int col = ct * 256 + c;
      if (col >= p.N) break;
      float g[16], u[16], dh[16];
      if (keep8) {
        uint4 qg = make_uint4(0u, 0u, 0u, 0u), qu = qg;
        float sg = 0.f, su = 0.f;
        if (rvalid) {
          const int8_t* q = p.keep_q + row * p.keep_ld + col;
          const float* s = p.keep_scale + row * (p.keep_ld / kKeepBlock) + col / kKeepBlock;
          qg = __ldg(reinterpret_cast<const uint4*>(q));
          qu = __ldg(reinterpret_cast<const uint4*>(q + p.keep_up));
          sg = __ldg(s);
          su = __ldg(s + p.keep_up / kKeepBlock);
        }
        unpack_q16(qg, sg, g);
        unpack_q16(qu, su, u);
        acc.fetch(c, dh);
      } else {
        r0.put(pg, lane);
        r1.put(pu, lane);
        acc.fetch(c, dh);                                // (the warp meets in there)
        patch_get<T>(pg, lane, g);
        patch_get<T>(pu, lane, u);
        if (c + 16 < col_end) look_ahead(c + 16);
      }
      if (c + 16 >= col_end) acc.release(lane);
      with_act(p.act, [&](auto tag) { act_gate_grad<decltype(tag)::value>(g, u, dh); });
      patch_put<T>(pg, lane, g);
      patch_put<T>(pu, lane, u);
      patch_put<T>(ph, lane, dh);
      __syncwarp();
      patch_store<T>(pg, lane, static_cast<T*>(p.dgate), ld2, row_base, p.M, col, p.N);
      patch_store<T>(pu, lane, static_cast<T*>(p.dgate) + p.N, ld2, row_base, p.M, col, p.N);
      patch_store<T>(ph, lane, static_cast<T*>(p.out), p.N, row_base, p.M, col, p.N);
      __syncwarp();
    }
  }
};

// Output columns of a tile: 256, or 128 where gate and up share the accumulator.
template <int EPI>
constexpr int kDpTileCols = EPI == kEpiGlu ? 128 : 256;

// The part of a pair's columns [from, to) that warp `share` of the four warps of a lane quarter takes.
__device__ __forceinline__ void dense_columns(int from, int to, int share, int& begin, int& end) {
  const int each = max((to - from) / 4, 16);
  begin = min(from + share * each, to);
  end = min(begin + each, to);
}

template <typename T, int EPI, bool SPLIT>
__global__ void __launch_bounds__(kDpThreads, 1)
dense_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const DenseParams p) {
  constexpr int kStages = kDpStages<EPI>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const uint32_t tiles_addr = ptx::smem_u32(smem);
  uint8_t* ctrl = smem + kStages * kDpStageBytes;
  const uint32_t bar0 = ptx::smem_u32(ctrl);
  auto bar_full = [&](int s) { return bar0 + 8u * s; };
  auto bar_empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto bar_tfull = [&](int b) { return bar0 + 8u * (2 * kStages + b); };
  auto bar_tempty = [&](int b) { return bar0 + 8u * (2 * kStages + kDpBufs + b); };
  const uint32_t bar_drain = bar0 + 8u * (2 * kStages + 2 * kDpBufs);
  const uint32_t bar_done = bar_drain + 8u;            // the peer no longer touches this CTA's shared state
  static_assert(8 * (2 * kStages + 2 * kDpBufs + 2) <= 224, "barriers overflow the control block");
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(ctrl + 224);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
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
    for (int s = 0; s < kStages; ++s) {
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
  if (!p.beside) ptx::dependency_wait();
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
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
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
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
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
    // ---------------- epilogue: warps 2..17, thread = row, four warps share the columns of a row ----------------
    const int quarter = warp & 3;
    const int share = (warp - 2) >> 2;
    int buf = 0;
    uint32_t tphase = 0;
    DenseAcc acc;
    acc.part = 0;
    for (int tile = first; tile < p.tile_end; tile += step) {
      acc.taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * kDpCols;
      acc.release_bar = ptx::mapa(bar_tempty(buf), leader_cta);          // the leader counts both CTAs' warps
      if constexpr (SPLIT) {
        if (!__all_sync(0xffffffffu, dense_wait(bar_tfull(buf), tphase, s_abort, 34, p.wait_cycles))) break;
        ptx::tc_fence_after();
        // all MMAs of this pair are done, so its ring is free: it takes the 128 x 256 accumulators
        const uint32_t dst = tiles_addr + static_cast<uint32_t>(quarter * 32 + lane) * 16u;
#pragma unroll 1
        for (int c = share * 64; c < share * 64 + 64; c += 16) {
          float v[16];
          acc.fetch(c, v);
#pragma unroll
          for (int k = 0; k < 4; ++k) ptx::st_shared_f4(dst + static_cast<uint32_t>((c >> 2) + k) * 2048u, make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
        }
        acc.release(lane);
      } else {
        int rt, ct;
        dense_tile_coord(tile, p.row_tiles, p.col_tiles, rt, ct);
        int begin, end;
        dense_columns(0, kDpTileCols<EPI>, share, begin, end);
        TileEpilogue<T, EPI> epi(p, s_out + (warp - 2) * kDpPatches<EPI> * kDpPatch, lane, rt * 256 + rank * 128 + quarter * 32, ct, begin, end);
        epi.prefetch();
        if (!__all_sync(0xffffffffu, dense_wait(bar_tfull(buf), tphase, s_abort, 34, p.wait_cycles))) break;
        ptx::tc_fence_after();
        epi.run(acc);
      }
      if (++buf == kDpBufs) { buf = 0; tphase ^= 1u; }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (SPLIT) {
    ptx::cluster_sync_all();          // every pair's part is in place
    if (warp >= 2) {
      int rt, ct, begin, end;
      dense_tile_coord(first, p.row_tiles, p.col_tiles, rt, ct);
      const int quarter = warp & 3;
      const int cols = kDpTileCols<EPI> / split;             // this pair's columns of the tile
      dense_columns(part * cols, part * cols + cols, (warp - 2) >> 2, begin, end);
      DenseAcc acc;
      acc.taddr = 0;
      acc.part = tiles_addr + static_cast<uint32_t>(quarter * 32 + lane) * 16u;
      acc.split = split;
      acc.parity = rank;
      acc.release_bar = 0;
      TileEpilogue<T, EPI> epi(p, s_out + (warp - 2) * kDpPatches<EPI> * kDpPatch, lane, rt * 256 + rank * 128 + quarter * 32, ct, begin, end);
      epi.prefetch();
      epi.run(acc);
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
