// Dense 16-bit GEMM for few rows (decode): out[m, n] = sum_k x[m, k] W[k, n] with at most 128 rows, weights streamed once.
//
// What bounds it: the bytes of W.  The weights are the stationary 128-row operand of tcgen05.mma (128 output features; for the
// gated form 64 gate features and the matching 64 up features), the rows of x its narrow N operand (16 .. 128 columns), so
// no MMA work is padded beyond 16 rows.  One tile of 128 features holds far too little work for an SM when N is a few
// thousand: a cluster of `split` CTAs shares a tile, each taking a part of the contraction.  The parts meet in distributed
// shared memory: every CTA leaves its fp32 accumulators in its own shared memory, and after a cluster barrier each CTA adds
// up, in the order of the contraction, the groups of 64 features that are its to finish, and runs the epilogue on them.  No
// workspace, no atomics, the same bits every time.  Two CTAs share an SM, each with a ring of about 100 KB.
//
// A launch marked `dependent` (the second projection of a feed-forward block) may start while the kernel before it still
// runs: it fills its ring with weights first and waits for that kernel only before it touches x.
#pragma once

#include "dense_common.cuh"

namespace tab {

constexpr int kNwThreads = 192;               // producer warp, MMA warp, 4 warps that empty tensor memory; all of them add up
constexpr int kNwMaxTokens = 128;
constexpr int kNwMaxStages = 8;
constexpr int kNwCtrlBytes = 256;
constexpr int kNwSmemTarget = 113 * 1024;     // two CTAs per SM
constexpr int kNwMaxSplit = 8;

__host__ __device__ constexpr int dense_narrow_stage_bytes(int nt) { return kDnOperandBytes + nt * 128; }

// 8 consecutive features of one token, summed over the cluster in rank order
__device__ __forceinline__ void sum_parts8(uint32_t part_addr, int token, int feature, int split, float (&v)[8]) {
  const uint32_t off = part_addr + static_cast<uint32_t>(token * 128 + feature) * 4u;
  float4 a[kNwMaxSplit], b[kNwMaxSplit];
#pragma unroll
  for (int r = 0; r < kNwMaxSplit; ++r)
    if (r < split) {
      const uint32_t at = ptx::mapa(off, static_cast<uint32_t>(r));
      a[r] = ptx::ld_cluster_f4(at);
      b[r] = ptx::ld_cluster_f4(at + 16);
    }
  v[0] = a[0].x; v[1] = a[0].y; v[2] = a[0].z; v[3] = a[0].w;
  v[4] = b[0].x; v[5] = b[0].y; v[6] = b[0].z; v[7] = b[0].w;
#pragma unroll
  for (int r = 1; r < kNwMaxSplit; ++r)
    if (r < split) {
      v[0] += a[r].x; v[1] += a[r].y; v[2] += a[r].z; v[3] += a[r].w;
      v[4] += b[r].x; v[5] += b[r].y; v[6] += b[r].z; v[7] += b[r].w;
    }
}

template <typename T>
__device__ __forceinline__ void add8(float (&v)[8], const T* src) {
  float t[8];
  Elem<T>::load8(src, t);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += t[i];
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
      const uint2 q = in ? quant8(v, rq) : make_uint2(0u, 0u);
      *reinterpret_cast<uint2*>(p.keep_q + row * p.keep_ld + col) = q;
      if ((threadIdx.x & 7) == 0) p.keep_scale[row * (p.keep_ld / kKeepBlock) + col / kKeepBlock] = rq.scale;
    }
  } else if (p.keep != nullptr && in) {
    Elem<T>::store8(static_cast<T*>(p.keep) + row * p.keep_ld + col, v);
  }
}

template <typename T, int EPI>
__global__ void __launch_bounds__(kNwThreads, 2)
dense_narrow_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const DenseParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const uint32_t tiles_addr = ptx::smem_u32(smem);
  const int stage_bytes = dense_narrow_stage_bytes(p.nt);
  uint8_t* ctrl = smem + p.stages * stage_bytes;
  const uint32_t bar0 = ptx::smem_u32(ctrl);
  auto bar_full = [&](int s) { return bar0 + 8u * s; };
  auto bar_empty = [&](int s) { return bar0 + 8u * (kNwMaxStages + s); };
  const uint32_t bar_tfull = bar0 + 8u * (2 * kNwMaxStages);
  static_assert(8 * (2 * kNwMaxStages + 1) <= 224, "barriers overflow the control block");
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(ctrl + 224);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  float* part = reinterpret_cast<float*>(smem);          // [tokens][128], over the stages once the MMAs are done

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int tile = blockIdx.x / p.split;
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * p.num_kb / p.split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * p.num_kb / p.split);
  const int n_kb = kb1 - kb0;                            // >= 1: the host keeps split <= num_kb

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      ptx::mbar_init(bar_full(s), 1);
      ptx::mbar_init(bar_empty(s), 1);
    }
    ptx::mbar_init(bar_tfull, 1);
    *s_abort = 0;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&tm_w);
    ptx::prefetch_tensormap(&tm_x);
  }
  if (warp == 1) ptx::tmem_alloc<kNwMaxTokens>(ptx::smem_u32(s_tmem));
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *s_tmem;
  ptx::launch_dependents();

  if (warp == 0) {
    const int f0 = EPI == kEpiGlu ? tile * 64 : tile * 128;
    const int f1 = EPI == kEpiGlu ? p.N + f0 : f0 + 64;
    auto load_w = [&](int s, int kb) {                   // by the elected lane
      const uint32_t st = tiles_addr + s * stage_bytes;
      const int k = kb * kDnBlockK;
      ptx::mbar_expect_tx(bar_full(s), static_cast<uint32_t>(stage_bytes));
      ptx::tma_load_2d(st, &tm_w, bar_full(s), p.a_mn ? f0 : k, p.a_mn ? k : f0);
      ptx::tma_load_2d(st + kDnBoxBytes, &tm_w, bar_full(s), p.a_mn ? f1 : k, p.a_mn ? k : f1);
    };
    auto load_x = [&](int s, int kb) {
      ptx::tma_load_2d(tiles_addr + s * stage_bytes + kDnOperandBytes, &tm_x, bar_full(s), kb * kDnBlockK, 0);
    };
    const int head = min(p.stages, n_kb);
    if (ptx::elect_one()) {
      for (int i = 0; i < head; ++i) load_w(i, kb0 + i);
      ptx::dependency_wait();
      for (int i = 0; i < head; ++i) load_x(i, kb0 + i);
    }
    __syncwarp();
    int stage = 0;
    uint32_t phase = 0;
    for (int i = head; i < n_kb; ++i) {
      if (!__all_sync(0xffffffffu, dense_wait(bar_empty(stage), phase, s_abort, 41, p.wait_cycles))) break;
      if (ptx::elect_one()) {
        load_w(stage, kb0 + i);
        load_x(stage, kb0 + i);
      }
      __syncwarp();
      if (++stage == p.stages) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t a_step = p.a_mn ? 128u : 2u;
    for (int i = 0; i < n_kb; ++i) {
      ok = __all_sync(0xffffffffu, dense_wait(bar_full(stage), phase, s_abort, 42, p.wait_cycles));
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t st = tiles_addr + stage * stage_bytes;
      const uint64_t a = p.a_mn ? ptx::smem_desc_mn128(st, kDnBoxBytes) : ptx::smem_desc_k128(st);
      const uint64_t b = ptx::smem_desc_k128(st + kDnOperandBytes);
      if (ptx::elect_one()) {
#pragma unroll
        for (int k = 0; k < kDnBlockK / 16; ++k) ptx::mma_f16(tmem_base, a + k * a_step, b + k * 2, p.idesc, (i | k) != 0 ? 1u : 0u);
        ptx::mma_commit(bar_empty(stage));
      }
      __syncwarp();
      if (++stage == p.stages) { stage = 0; phase ^= 1u; }
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
      const int quarter = warp & 3;
      const uint32_t t0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      for (int c = 0; c < p.M; c += 16) {
        int v[16];
        __syncwarp();
        ptx::tmem_ld16(t0 + c, v);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < p.M) part[(c + j) * 128 + quarter * 32 + lane] = __int_as_float(v[j]);
      }
    }
    ptx::tc_fence_before();
  }
  __syncthreads();
  ptx::cluster_sync_all();            // every CTA's part is in place

  // ---- add up and finish: groups of 64 output features of one token, 8 lanes x 8 features each ----
  constexpr int kGroupsPerToken = EPI == kEpiGlu ? 1 : 2;
  const int groups = p.M * kGroupsPerToken;
  const int g_begin = static_cast<int>(static_cast<int64_t>(rank) * groups / p.split);
  const int g_end = static_cast<int>(static_cast<int64_t>(rank + 1) * groups / p.split);
  const uint32_t part_addr = tiles_addr;
  for (int g0 = g_begin; g0 < g_end; g0 += kNwThreads / 8) {
    const int g = g0 + static_cast<int>(threadIdx.x >> 3);
    const bool mine = g < g_end;
    const int token = mine ? g / kGroupsPerToken : 0;
    const int in_tile = (mine ? g % kGroupsPerToken : 0) * 64 + (threadIdx.x & 7) * 8;
    const int col = tile * (EPI == kEpiGlu ? 64 : 128) + in_tile;
    const bool in = mine && col < p.N;
    const bool live = mine && (col & ~63) < p.N;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (in) {
      sum_parts8(part_addr, token, in_tile, p.split, v);
      if (p.bias != nullptr) add8(v, static_cast<const T*>(p.bias) + col);
    }
    keep8<T>(p, v, token, col, in, live);
    if constexpr (EPI == kEpiGlu) {
      float u[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (in) {
        sum_parts8(part_addr, token, 64 + in_tile, p.split, u);
        if (p.bias != nullptr) add8(u, static_cast<const T*>(p.bias) + p.N + col);
      }
      keep8<T>(p, u, token, p.keep_up + col, in, live);
      with_act(p.act, [&](auto tag) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_value<decltype(tag)::value>(v[i]) * u[i];
      });
    } else if (p.act != TAB_ACT_NONE) {
      with_act(p.act, [&](auto tag) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_value<decltype(tag)::value>(v[i]);
      });
    }
    if (in) {
      const int64_t at = static_cast<int64_t>(token) * p.N + col;
      if constexpr (EPI == kEpiLinear) {
        if (p.residual != nullptr) add8(v, static_cast<const T*>(p.residual) + at);
      }
      Elem<T>::store8(static_cast<T*>(p.out) + at, v);
    }
  }
  ptx::cluster_sync_all();            // no CTA leaves while another still reads its part
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<kNwMaxTokens>(tmem_base);
  }
}

}  // namespace tab
