// Dense 16-bit GEMM for few rows or few tiles: out[m, n] = sum_k x[m, k] W[k, n] in tiles of 128 output features x NT rows, one CTA
// or one cluster to a tile.
//
// The features are the stationary 128-row operand of tcgen05.mma (for the gated form 64 gate features and the matching 64 up
// features), the rows of x its narrow N operand (NT = 16 .. 256 columns): a decode batch pads no MMA work beyond 16 rows, and the
// weights stream from HBM once.  What bounds it: the bytes of W for a handful of rows, the operand bytes from L2 (NT = 128: 32 KB per
// 256 tensor cycles) where there are many; the pair kernel needs half of those, but only 74 tiles of its 256 x 256 fill the GPU.
//
// One tile holds too little work for an SM when there are few: a cluster of `split` CTAs shares it, each taking a part of the
// contraction.  The parts meet in distributed shared memory: every CTA copies the rows of its fp32 accumulators to the CTAs that
// finish them (one bulk copy each, counted on a barrier of the receiver), which add them in the order of the contraction and
// run the epilogue.  No workspace, no atomics, the same bits every time.  Cluster barriers are only arrived at early and
// waited for late; reading the parts remotely between two full barriers cost some 2 us more per launch.
//
// A launch of this kernel is over in 5 to 15 us, so its start counts: the producer sets up its barriers and asks for the first
// weights before the CTA's threads have met and tensor memory is allocated.
//
// A launch marked `dependent` (the second projection of a feed-forward block) asks for weights before it waits for the kernel that writes
// x, in those of its CTAs that find room beside that kernel's.  Those are few when the first projection has no more CTAs than SMs, for
// each then takes all of its SM's shared memory: 37 rows, 4096 -> 1408: 132 of them leave 16 SMs to the second one's 128 CTAs; one row of
// 7168 -> 2048: 192 half-SM places of 296 are taken, 104 of the second one's 224 CTAs find room.
#pragma once

#include "dense_common.cuh"

namespace tab {

constexpr int kNwMaxTokens = 256;
constexpr int kNwMaxStages = 12;
constexpr int kNwCtrlBytes = 512;                        // barriers, control words, from 256 on the bias of kEpiLinearAny
constexpr int kNwMaxSplit = 8;

// Up to 64 rows two CTAs may share an SM, each with a ring of about 110 KB: the one streams weights while the other is in its
// prologue or epilogue.  A CTA that has its SM to itself (wider tiles, or no more CTAs than SMs) takes all of the shared memory:
// a block of the contraction then takes some 550 cycles with five stages of 20 KB in flight, less with eleven.
__host__ __device__ constexpr int dense_narrow_threads(bool wide) { return wide ? 320 : 192; }
__host__ __device__ constexpr int dense_narrow_smem(bool alone) { return alone ? kDnSmemLimit : 113 * 1024; }
__host__ __device__ constexpr int dense_narrow_stage_bytes(int nt) { return kDnOperandBytes + nt * 128; }
// where a CTA of a cluster receives the parts of the rows that it finishes: rows x 128 fp32 of a tile in all, up to one more
// group of 64 or 128 from each of the CTAs where the rows do not divide evenly
__host__ __device__ constexpr int dense_narrow_recv_bytes(int nt, int split) { return split > 1 ? (nt + split) * 512 : 0; }

// 8 consecutive fp32 values at `src` of the first part, summed over the parts in order
__device__ __forceinline__ void sum_parts8(const float* src, int part_floats, int parts, float (&v)[8]) {
  float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
#pragma unroll 1
  for (int r = 1; r < parts; ++r) {
    src += part_floats;
    const float4 c = *reinterpret_cast<const float4*>(src), d = *reinterpret_cast<const float4*>(src + 4);
    a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
    b.x += d.x; b.y += d.y; b.z += d.z; b.w += d.w;
  }
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// Keeps 8 values of a row for the backward pass; the 8 lanes of an aligned group hold one 64-value block.  Every lane of the
// warp calls it; `in` = these values exist, `live` = this lane's group of 64 has a place in the kept row.
template <typename T>
__device__ __forceinline__ void keep8(const DenseParams& p, const float (&v)[8], int64_t row, int col, bool in, bool live) {
  if (p.keep_q != nullptr) {
    uint32_t m = 0;
    if (in) {
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (live) {
      const RowQuant rq = make_block_quant(__uint_as_float(m), m < 0x7f800000u);
      const uint2 q = in ? block_quant8(v, rq) : make_uint2(0u, 0u);
      *reinterpret_cast<uint2*>(p.keep_q + row * p.keep_ld + col) = q;
      if ((threadIdx.x & 7) == 0) p.keep_scale[row * (p.keep_ld / kKeepBlock) + col / kKeepBlock] = rq.scale;
    }
  } else if (p.keep != nullptr && in) {
    Elem<T>::store8(static_cast<T*>(p.keep) + row * p.keep_ld + col, v);
  }
}

// 8 kept values of a row
template <typename T>
__device__ __forceinline__ void kept8(const DenseParams& p, int64_t row, int col, float (&v)[8]) {
  if (p.keep_q != nullptr) {
    const uint2 q = __ldg(reinterpret_cast<const uint2*>(p.keep_q + row * p.keep_ld + col));
    const float s = __ldg(p.keep_scale + row * (p.keep_ld / kKeepBlock) + col / kKeepBlock);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(static_cast<int8_t>(j < 4 ? q.x >> (8 * j) : q.y >> (8 * j - 32))) * s;
  } else {
    Elem<T>::load8(static_cast<const T*>(p.keep) + row * p.keep_ld + col, v);
  }
}

template <typename T, int EPI, bool WIDE>
__global__ void __launch_bounds__(dense_narrow_threads(WIDE), WIDE ? 1 : 2)
dense_narrow_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const DenseParams p) {
  constexpr int kThreads = dense_narrow_threads(WIDE);
  constexpr int kTmemCols = WIDE ? 256 : 64;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const uint32_t tiles_addr = ptx::smem_u32(smem);
  const int stage_bytes = dense_narrow_stage_bytes(p.nt);
  uint8_t* ctrl = smem + p.stages * stage_bytes;
  float* recv = reinterpret_cast<float*>(ctrl + kNwCtrlBytes);         // parts of this CTA's groups, one after another
  const uint32_t bar0 = ptx::smem_u32(ctrl);
  auto bar_full = [&](int s) { return bar0 + 8u * s; };
  auto bar_empty = [&](int s) { return bar0 + 8u * (kNwMaxStages + s); };
  const uint32_t bar_tfull = bar0 + 8u * (2 * kNwMaxStages);
  const uint32_t bar_recv = bar_tfull + 8u;
  static_assert(8 * (2 * kNwMaxStages + 2) <= 224 && 2 * kNwMaxStages + 2 <= 32, "barriers: one per lane, ahead of the control words");
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(ctrl + 224);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  float* part = reinterpret_cast<float*>(smem);          // [rows][128], over the stages once the MMAs are done

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const int rank = split > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int tile = blockIdx.x / split;
  const int ft = tile / p.row_tiles;                     // CTAs that follow one another read the same features
  const int row0 = (tile - ft * p.row_tiles) * p.nt;
  const int rows = min(p.nt, p.M - row0);
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * p.num_kb / split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * p.num_kb / split);
  const int n_kb = kb1 - kb0;                            // >= 1: the host keeps split <= num_kb
  const int head = min(p.stages, n_kb);

  // groups of 64 output features of one row; CTA r finishes groups [r G / split, (r + 1) G / split)
  constexpr int kGroups = EPI == kEpiGlu ? 1 : 2;        // per row
  constexpr int kGroupFloats = 128 / kGroups;            // accumulators of a group (gate and up together)
  const int groups = rows * kGroups;
  auto group_begin = [&](int r) { return r * groups / split; };

  const int f0 = EPI == kEpiGlu ? ft * 64 : ft * 128;
  const int f1 = EPI == kEpiGlu ? p.N + f0 : f0 + 64;
  auto load_w = [&](int s, int kb) {                     // by the elected lane of the producer warp
    const uint32_t st = tiles_addr + s * stage_bytes;
    const int k = kb * kDnBlockK;
    ptx::mbar_expect_tx(bar_full(s), static_cast<uint32_t>(stage_bytes));
    ptx::tma_load_2d(st, &tm_w, bar_full(s), p.a_mn ? f0 : k, p.a_mn ? k : f0);
    ptx::tma_load_2d(st + kDnBoxBytes, &tm_w, bar_full(s), p.a_mn ? f1 : k, p.a_mn ? k : f1);
  };
  auto load_x = [&](int s, int kb) {
    const uint32_t st = tiles_addr + s * stage_bytes + kDnOperandBytes;
    if (p.b_mn) {                                        // 64 rows per box
      for (int r = 0; r < p.nt; r += 64) ptx::tma_load_2d(st + r * 128, &tm_x, bar_full(s), row0 + r, kb * kDnBlockK);
    } else {
      ptx::tma_load_2d(st, &tm_x, bar_full(s), kb * kDnBlockK, row0);
    }
  };

  if (warp == 0) {
    if (lane < 2 * kNwMaxStages + 2) ptx::mbar_init(bar0 + 8u * lane, 1);
    if (lane == 0) *s_abort = 0;
    ptx::fence_barrier_init();
    __syncwarp();
    if (ptx::elect_one()) {
      if (!p.beside && !p.dependent) ptx::dependency_wait();
      const int mine = group_begin(rank + 1) - group_begin(rank);
      if (split > 1 && mine > 0) ptx::mbar_expect_tx(bar_recv, static_cast<uint32_t>(mine * split * kGroupFloats * 4));
      for (int i = 0; i < min(head, 2); ++i) load_w(i, kb0 + i);
    }
    __syncwarp();
  } else if (warp == 1) {
    ptx::tmem_alloc<kTmemCols>(ptx::smem_u32(s_tmem));
  } else if (threadIdx.x == 64) {
    ptx::prefetch_tensormap(&tm_w);
    ptx::prefetch_tensormap(&tm_x);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (split > 1) ptx::cluster_arrive();                  // this CTA runs and its barriers exist
  const uint32_t tmem_base = *s_tmem;
  if (!p.dependent) {
    if (!p.beside) ptx::dependency_wait();
    ptx::launch_dependents();
  }

  // What this thread will need in the epilogue: its columns are the same in every step (a step is an even number of groups), so the
  // bias is fetched once, and the residual of the first step with it, while the products run.  (Element by element the values would
  // be waited for here, ahead of the products: kEpiLinearAny has one warp put the bias into shared memory.)
  constexpr bool ragged = EPI == kEpiLinearAny;
  static_assert(kThreads / 8 % 2 == 0, "steps of an even number of groups");
  const bool has_bias = p.bias != nullptr, has_res = epi_linear(EPI) && p.residual != nullptr;
  const int n_out = ragged ? p.n_out : p.N;
  const int64_t ld = n_out;
  const T *bias = static_cast<const T*>(p.bias), *res = static_cast<const T*>(p.residual);
  const int g_begin = group_begin(rank), g_end = group_begin(rank + 1), g_first = g_begin + static_cast<int>(threadIdx.x >> 3);
  const int col = ft * (EPI == kEpiGlu ? 64 : 128) + (kGroups == 2 ? (g_first & 1) * 64 : 0) + static_cast<int>(threadIdx.x & 7) * 8;
  const bool col_in = col < p.N;
  auto unpack_8 = [](const uint4& x, float (&v)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  };
  uint4 bias_v = make_uint4(0u, 0u, 0u, 0u), bias_up = bias_v, res_v = bias_v;
  T* s_bias = reinterpret_cast<T*>(ctrl + 256);
  if constexpr (ragged) {
    if (has_bias && warp == 3) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = ft * 128 + i * 32 + lane;
        s_bias[i * 32 + lane] = c < n_out ? bias[c] : Elem<T>::from_f32(0.f);
      }
    }
  } else if (col_in) {
    if (EPI != kEpiGluGrad && has_bias) {
      bias_v = __ldcg(reinterpret_cast<const uint4*>(bias + col));
      if (EPI == kEpiGlu) bias_up = __ldcg(reinterpret_cast<const uint4*>(bias + p.N + col));
    }
    if (has_res && g_first < g_end) res_v = __ldcg(reinterpret_cast<const uint4*>(res + (row0 + g_first / kGroups) * ld + col));
  }

  // Two producer warps (the second is one that has nothing to do before the epilogue) take the blocks in turn: one alone needs
  // some 400 cycles for a block's wait and copies, more than the bytes do.
  if (warp == 0 || warp == 2) {
    const int odd = warp >> 1;
    if (ptx::elect_one()) {
      if (!p.dependent && odd < head) load_x(odd, kb0 + odd);
      for (int i = 2 + odd; i < head; i += 2) {
        load_w(i, kb0 + i);
        if (!p.dependent) load_x(i, kb0 + i);
      }
      if (p.dependent) {
        ptx::dependency_wait();
        ptx::launch_dependents();
        for (int i = odd; i < head; i += 2) load_x(i, kb0 + i);
      }
    }
    __syncwarp();
    int i = odd, stage = odd;
    uint32_t phase = 1;                                  // of the first use; later ones wait for the MMAs of the use before
    while (stage >= p.stages) stage -= p.stages;
    for (; i < n_kb; i += 2) {
      if (i >= head) {
        if (!__all_sync(0xffffffffu, dense_wait(bar_empty(stage), phase, s_abort, 41, p.wait_cycles))) break;
        if (ptx::elect_one()) {
          load_w(stage, kb0 + i);
          load_x(stage, kb0 + i);
        }
        __syncwarp();
      }
      stage += 2;
      if (stage >= p.stages) { stage -= p.stages; phase ^= 1u; }
    }
  }
  if (warp == 0) {
    // nothing until the parts are exchanged
  } else if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t a_step = p.a_mn ? 128u : 2u, b_step = p.b_mn ? 128u : 2u, idesc = p.idesc;
    const uint64_t a_first = p.a_mn ? ptx::smem_desc_mn128(tiles_addr, kDnBoxBytes) : ptx::smem_desc_k128(tiles_addr);
    const uint64_t b_first = p.b_mn ? ptx::smem_desc_mn128(tiles_addr + kDnOperandBytes, kDnBoxBytes) : ptx::smem_desc_k128(tiles_addr + kDnOperandBytes);
    const uint32_t stage_step = static_cast<uint32_t>(stage_bytes) >> 4;
    uint32_t off = 0;
    for (int i = 0; i < n_kb; ++i) {
      ok = __all_sync(0xffffffffu, dense_wait(bar_full(stage), phase, s_abort, 42, p.wait_cycles));
      if (!ok) break;
      ptx::tc_fence_after();
      if (ptx::elect_one()) {
        const uint64_t a = a_first + off, b = b_first + off;
#pragma unroll
        for (int k = 0; k < kDnBlockK / 16; ++k) ptx::mma_f16(tmem_base, a + k * a_step, b + k * b_step, idesc, (i | k) != 0 ? 1u : 0u);
        ptx::mma_commit(bar_empty(stage));
      }
      __syncwarp();
      off += stage_step;
      if (++stage == p.stages) { stage = 0; phase ^= 1u; off = 0; }
    }
    // also after a wait that gave up: the barrier then says that no MMA is in flight any more
    if (ptx::elect_one()) ptx::mma_commit(bar_tfull);
    __syncwarp();
    if (!ok) {
      const long long t0 = clock64();
      while (!ptx::mbar_try_wait(bar_tfull, 0) && clock64() - t0 < p.wait_cycles) {}
      __syncwarp();
    }
  } else {
    const bool got = dense_wait(bar_tfull, 0, s_abort, 43, p.wait_cycles) && *s_abort == 0;
    __syncwarp();
    if (__all_sync(0xffffffffu, got)) {
      ptx::tc_fence_after();
      const int quarter = warp & 3, group = (warp - 2) >> 2;       // warps of one lane quarter take the 16-row steps in turn
      const uint32_t t0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      for (int c = group * 16; c < rows; c += (kThreads / 32 - 2) / 4 * 16) {
        float v[16];
        __syncwarp();
        ptx::tmem_ld16f(t0 + c, v);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < rows) part[(c + j) * 128 + quarter * 32 + lane] = v[j];
      }
    }
    ptx::tc_fence_before();
    if (split > 1) ptx::fence_async_shared();            // the copies below read what this thread wrote
  }
  __syncthreads();

  // ---- the parts go to the CTAs that finish their rows ----
  const int part_floats = split > 1 ? (g_end - g_begin) * kGroupFloats : 0;
  float* sums = part + g_begin * kGroupFloats;           // this CTA's groups in the first part
  if (split > 1) {
    ptx::cluster_wait();                                 // every CTA of the cluster runs
    if (warp == 0 && lane < split) {
      const int b = group_begin(lane), n = group_begin(lane + 1) - b;
      if (n > 0)
        ptx::copy_to_cluster(ptx::mapa(ptx::smem_u32(recv) + static_cast<uint32_t>(rank * n * kGroupFloats * 4), static_cast<uint32_t>(lane)),
                             tiles_addr + static_cast<uint32_t>(b * kGroupFloats * 4), static_cast<uint32_t>(n * kGroupFloats * 4),
                             ptx::mapa(bar_recv, static_cast<uint32_t>(lane)));
    }
    __syncwarp();
    if (part_floats > 0) dense_wait(bar_recv, 0, s_abort, 44, p.wait_cycles);
    sums = recv;
    __syncthreads();
    ptx::cluster_arrive();                               // what was sent here has arrived: the senders may leave
  }

  // ---- add up and finish: 8 lanes x 8 features to a group ----
  const bool keeps = p.keep != nullptr || p.keep_q != nullptr;
  const int act = p.act;
  T* out = static_cast<T*>(p.out);
  const int lane8 = (threadIdx.x & 7) * 8;
#pragma unroll 2
  for (int g0 = g_begin; g0 < g_end; g0 += kThreads / 8) {
    const int g = g0 + static_cast<int>(threadIdx.x >> 3);
    const bool mine = g < g_end;
    const int64_t row = row0 + (mine ? g / kGroups : 0);
    const bool in = mine && col_in;
    float* src = sums + (mine ? g - g_begin : 0) * kGroupFloats + lane8;
    float v[8];
    if constexpr (EPI == kEpiGluGrad) {
      if (in) {
        float gate[8], up[8];
        kept8<T>(p, row, col, gate);
        kept8<T>(p, row, p.keep_up + col, up);
        sum_parts8(src, part_floats, split, v);
        with_act(act, [&](auto tag) { act_gate_grad<decltype(tag)::value>(gate, up, v); });
        T* dz = static_cast<T*>(p.dgate) + row * 2 * ld + col;
        Elem<T>::store8(dz, gate);
        Elem<T>::store8(dz + p.N, up);
        Elem<T>::store8(out + row * ld + col, v);
      }
    } else {
      float u[8], r[8];
      if (in) {
        if (has_res) {
          if constexpr (ragged) {
            load8_any(res + row * ld, col, n_out, r);
          } else {
            if (g0 > g_begin) res_v = __ldcg(reinterpret_cast<const uint4*>(res + row * ld + col));
            unpack_8(res_v, r);
          }
        }
        sum_parts8(src, part_floats, split, v);
        if constexpr (EPI == kEpiGlu) sum_parts8(src + 64, part_floats, split, u);
        if (has_bias) {
          float b[8];
          if constexpr (ragged) Elem<T>::load8(s_bias + (col - ft * 128), b); else unpack_8(bias_v, b);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += b[i];
          if constexpr (EPI == kEpiGlu) {
            unpack_8(bias_up, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] += b[i];
          }
        }
      }
      if (keeps) {
        const bool live = mine && (col & ~63) < p.N;
        keep8<T>(p, v, row, col, in, live);
        if constexpr (EPI == kEpiGlu) keep8<T>(p, u, row, p.keep_up + col, in, live);
      }
      if (in) {
        if constexpr (EPI == kEpiGlu) {
          with_act(act, [&](auto tag) { act_gate<decltype(tag)::value>(v, u); });
        } else if (act != TAB_ACT_NONE) {
          with_act(act, [&](auto tag) { act_values<decltype(tag)::value>(v); });
        }
        if (has_res) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += r[i];
        }
        // rows that begin anywhere leave through shared memory (over the sums just read), so that lanes run along them
        if (ragged) Elem<T>::store8(reinterpret_cast<T*>(src), v); else Elem<T>::store8(out + row * ld + col, v);
      }
    }
  }
  if constexpr (ragged) {
    // A warp to a group of 64 values, two values to a lane where they lie on a 4-byte boundary of the result.  These stores end in sectors
    // that are written in part: 777 x 1003 -> 1501 takes 13.7 us with them, 9.5 without, 9.4 with whole rows of 1504.
    __syncthreads();
#pragma unroll 4
    for (int g = g_begin + warp; g < g_end; g += kThreads / 32) {
      const unsigned short* from = reinterpret_cast<const unsigned short*>(sums + (g - g_begin) * kGroupFloats);     // value c at (c / 8) * 16 + c % 8
      const int col0 = ft * 128 + (g & 1) * 64;
      unsigned short* to = reinterpret_cast<unsigned short*>(out) + (row0 + (g >> 1)) * ld + col0;
      const int odd = static_cast<int>((reinterpret_cast<uintptr_t>(to) >> 1) & 1u), n = n_out - col0;
      auto value = [&](int c) { return static_cast<uint32_t>(from[(c & ~7) * 2 + (c & 7)]); };
      const int c = 2 * lane + odd;
      if (c + 1 < n && c + 1 < 64) {
        *reinterpret_cast<uint32_t*>(to + c) = value(c) | value(c + 1) << 16;
      } else if (c < n && c < 64) {
        to[c] = static_cast<unsigned short>(value(c));
      }
      if (odd && lane == 0 && n > 0) to[0] = static_cast<unsigned short>(value(0));
    }
  }
  if (split > 1) {
    __syncwarp();
    ptx::cluster_wait();              // what this CTA sent has arrived
  }
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<kTmemCols>(tmem_base);
  }
  // a launch that was allowed to start under the one before it ends only after that one has
  if (threadIdx.x == 0) ptx::dependency_wait();
}

}  // namespace tab
