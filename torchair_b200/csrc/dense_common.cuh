// Pieces shared by the dense 16-bit GEMM kernels (dense_pair.cuh, dense_narrow.cuh): launch parameters and the
// bounded wait.
#pragma once

#include <cuda.h>

#include "dense_math.cuh"
#include "ptx_sm100.cuh"

namespace tab {

// Status word of the dense GEMMs on this device: 0, or the code of the bounded wait that gave up (tab_dense_status).
// This header is included by exactly one translation unit (dense.cu).
__device__ int g_dense_status = 0;

constexpr int kDnBlockK = 64;                 // contraction elements per stage = one 128-byte swizzle span of 16-bit values
constexpr int kDnBoxBytes = 64 * 128;         // every TMA box of the 128-row operands: 64 rows x 128 bytes
constexpr int kDnOperandBytes = 2 * kDnBoxBytes;
constexpr int kDnSmemLimit = 232448;
constexpr long long kDnCyclesPerMs = 2000000LL;

enum DenseEpilogue {
  kEpiLinear = 0,   // out = act(acc + bias) + residual, optionally keeping acc + bias for the backward pass
  kEpiGlu = 1,      // out = act(gate) * up, optionally keeping gate and up
  kEpiGluGrad = 2,  // acc = d(act(gate) * up): writes d(gate), d(up) and act(gate) * up from the kept gate and up
  kEpiLinearAny = 3 // kEpiLinear whose bias, residual and out are accessed element by element: rows of any length, anywhere.  A kind
                    // of its own: the checks for it inside the loops of kEpiLinear cost 10 % of a 4096 x 4096 x 1024 product
};
__host__ __device__ constexpr bool epi_linear(int epi) { return epi == kEpiLinear || epi == kEpiLinearAny; }

struct DenseParams {
  int M;             // rows of the product
  int N;             // columns of the product (kEpiGlu, kEpiGluGrad: inner features I), rounded up to a multiple of 8
  int n_out;         // columns of bias, residual and out of kEpiLinearAny
  int num_kb;        // blocks of 64 along the contraction
  int row_tiles, col_tiles;
  int tile_begin, tile_end;   // tiles of this launch (dense_pair.cuh)
  int a_mn, b_mn;    // operand is contiguous along the product's rows / columns instead of along the contraction
  uint32_t idesc;
  int act;           // TAB_ACT_*
  const void* bias;      // [N] (kEpiGlu: [2 N]) or null
  const void* residual;  // [M, N] or null
  void* out;             // [M, N]
  // activations kept for the backward pass: 16-bit [M, keep_ld], or int8 [M, keep_ld] with fp32 scales [M, keep_ld / 64].
  // kEpiGlu / kEpiGluGrad: gate in columns [0, ..), up from keep_up on.
  void* keep;
  int8_t* keep_q;
  float* keep_scale;
  int keep_ld, keep_up;
  void* dgate;           // kEpiGluGrad: d(gate) in columns [0, N), d(up) in [N, 2 N) of rows of 2 N values
  int split;             // CTAs (dense_pair.cuh: pairs) of a cluster that share one tile's contraction
  int stages, nt;        // dense_narrow.cuh: shared-memory stages, token columns of a tile
  // Every launch of these kernels may begin while the one before it on the stream still runs: it sets up its barriers and tensor
  // memory, then waits for that one to end before it touches global memory, and only then lets the next launch begin.  (linear
  // layers one after the other, 8 x 2048 -> 7168: 11.0 -> 9.6 us.)  Two kinds wait later:
  int dependent;         // the launch before writes the token operand and nothing else of this one: weights are loaded ahead of the wait
  int beside;            // nothing of this one is written or read by the launch before: waits only before it ends
  long long wait_cycles;
};

// Waits for a phase of an mbarrier; gives up after `limit` clock ticks or when another role already gave up.
__device__ __forceinline__ bool dense_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code, long long limit) {
  if (ptx::mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  unsigned spins = 0;
  while (!ptx::mbar_try_wait(bar, parity)) {
    if ((++spins & 255u) == 0) {
      if (*abort_flag != 0) return false;
      if (clock64() - t0 > limit) {
        *abort_flag = code;
        atomicCAS(&g_dense_status, 0, code);
        return false;
      }
    }
  }
  return true;
}

}  // namespace tab
