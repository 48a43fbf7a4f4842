// The kernels of gated_matmul.h for one data type, and their launch; a source file of
// each type includes this so that they compile beside one another.
#ifndef PORTDNN_AMD_CSRC_GATED_MATMUL_RUN_H_
#define PORTDNN_AMD_CSRC_GATED_MATMUL_RUN_H_

#include "gated_matmul.h"
#include "snn_kernels.h"

namespace snn {
namespace gated {

template <typename T, bool GATED, bool QK, int BM, int BN, int WM, int WN, int CB,
          int STAGES>
__global__ void __launch_bounds__(64 * WM * WN) tile_kernel(Pair g) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int kStage = epi::Space<BM, BN, WM * WN, CB>::kStage;
  // (an array of its own for each chunk)
  __shared__ __align__(1024) char ring0[kStage];
  __shared__ __align__(1024) char ring1[kStage];
  char *r2 = nullptr, *r3 = nullptr, *r4 = nullptr;
  if constexpr (STAGES > 2) {
    __shared__ __align__(1024) char ring2[kStage];
    r2 = ring2;
  }
  if constexpr (STAGES > 3) {
    __shared__ __align__(1024) char ring3[kStage];
    r3 = ring3;
  }
  if constexpr (STAGES > 4) {
    __shared__ __align__(1024) char ring4[kStage];
    r4 = ring4;
  }
  tile_body<T, GATED, QK, BM, BN, WM, WN, CB, STAGES>(g, ring0, ring1, r2, r3, r4);
#endif
}

template <typename T, bool GATED, bool QK, int BM, int BN, int WM, int WN, int CB,
          int STAGES>
int launch_as(const Pair& g, hipStream_t stream) {
  hipLaunchKernelGGL(
      (tile_kernel<T, GATED, QK, BM, BN, WM, WN, CB, STAGES>),
      dim3(static_cast<unsigned>(g.tiles_m) * g.tiles_n * g.splits),
      dim3(64 * WM * WN), 0, stream, g);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T, bool GATED, bool QK, int BM, int BN, int WAVES, int STAGES,
          bool DIRECT>
__global__ void __launch_bounds__(64 * WAVES) few_kernel(Pair g) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int kStage = (BM + BN) * kChunkBytes * WAVES;
  __shared__ __align__(1024) char ring0[kStage];
  char *r1 = nullptr, *r2 = nullptr, *r3 = nullptr;
  if constexpr (DIRECT) {
    __shared__ __align__(1024) char ring1[kStage];
    r1 = ring1;
  }
  if constexpr (DIRECT && STAGES > 2) {
    __shared__ __align__(1024) char ring2[kStage];
    r2 = ring2;
  }
  if constexpr (DIRECT && STAGES > 3) {
    __shared__ __align__(1024) char ring3[kStage];
    r3 = ring3;
  }
  few_body<T, GATED, QK, BM, BN, WAVES, STAGES, DIRECT>(g, ring0, r1, r2, r3);
#endif
}

template <typename T, bool GATED, bool QK, int BM, int BN, int WAVES, int STAGES,
          bool DIRECT>
int launch_few(const Pair& g, hipStream_t stream) {
  hipLaunchKernelGGL(
      (few_kernel<T, GATED, QK, BM, BN, WAVES, STAGES, DIRECT>),
      dim3(static_cast<unsigned>(g.tiles_m) * g.tiles_n * g.splits),
      dim3(64 * WAVES), 0, stream, g);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T, bool GATED, bool QK>
int launch_tile(const Pair& g, int kernel, hipStream_t stream) {
  switch (kernel) {
    case kFew16x32:
      return launch_few<T, GATED, QK, 16, 32, 4, 3, true>(g, stream);
    case kFew16x64:
      return launch_few<T, GATED, QK, 16, 64, 4, 3, true>(g, stream);
    case kFew32x32:
      return launch_few<T, GATED, QK, 32, 32, 4, 2, true>(g, stream);
    case kFew32x64:
      return launch_few<T, GATED, QK, 32, 64, 4, 3, true>(g, stream);
    case kTile64x128:
      return launch_as<T, GATED, QK, 64, 128, 2, 4, 128, 5>(g, stream);
    case kAny16x32:
      return launch_few<T, GATED, QK, 16, 32, 4, 2, false>(g, stream);
    default:
      break;
  }
  if constexpr (sizeof(T) == 2) {
    switch (kernel) {
      case kFew64x32:
        return launch_few<T, GATED, QK, 64, 32, 4, 2, true>(g, stream);
      case kTile128:
        return launch_as<T, GATED, QK, 128, 128, 2, 4, 128, 4>(g, stream);
      case kTile128Pair:
        return launch_as<T, GATED, QK, 128, 128, 2, 4, 128, 2>(g, stream);
      case kTile256:
        return launch_as<T, GATED, QK, 256, 256, 4, 4, 64, 4>(g, stream);
      default:
        break;
    }
  } else if (kernel == kTile128) {
    return launch_as<T, GATED, QK, 128, 128, 2, 4, 64, 4>(g, stream);
  }
  return SNN_HIP_INVALID_ALGORITHM;
}

// Up to four operands on their way to rows that start at multiples of 16 bytes.
struct Copies {
  const void* in[4];
  void* out[4];
  long in_stride[4], out_stride[4];
  int rows[4], cols[4];
  unsigned groups[4];  // work-groups up to an operand's last
};
template <typename T>
__global__ void __launch_bounds__(256) copy_rows_kernel(Copies c) {
  constexpr int kPiece = 16 / sizeof(T);
  int o = 0;
  while (blockIdx.x >= c.groups[o]) ++o;
  const unsigned group = blockIdx.x - (o > 0 ? c.groups[o - 1] : 0);
  const int pieces = static_cast<int>(c.out_stride[o] / kPiece);
  const long at = static_cast<long>(group) * 256 + threadIdx.x;
  const long row = at / pieces;
  const int col = static_cast<int>(at - row * pieces) * kPiece;
  if (row >= c.rows[o]) return;
  const T* const from =
      static_cast<const T*>(c.in[o]) + row * c.in_stride[o] + col;
  T part[kPiece];
  if (col + kPiece <= c.cols[o]) {
    __builtin_memcpy(part, from, 16);
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
      part[i] = col + i < c.cols[o] ? from[i] : T(0);
  }
  __builtin_memcpy(
      __builtin_assume_aligned(
          static_cast<T*>(c.out[o]) + row * c.out_stride[o] + col, 16),
      part, 16);
}

template <typename T>
int run(Pair& g, void* workspace, size_t bytes, hipStream_t stream) {
  auto both_aligned = [](const void* const (&at)[2]) {
    return seq::aligned(static_cast<const T*>(at[0]), 16) &&
           (at[1] == nullptr || seq::aligned(static_cast<const T*>(at[1]), 16));
  };
  const Plan plan =
      make_plan(g, sizeof(T), bytes, both_aligned(g.p), both_aligned(g.q));
  if (plan.splits == 0) return SNN_HIP_INDEX_EXCEEDED;
  g.tiles_m = plan.tiles_m;
  g.tiles_n = plan.tiles_n;
  g.splits = plan.splits;
  // (in chunks of the kernel's; those of 64 bytes are half of the plan's)
  const int chunk = chunk_bytes(sizeof(T), plan.kernel) / static_cast<int>(sizeof(T));
  g.chunks = ceil_div(g.k, chunk);
  g.split_chunks = plan.splits == 1
                       ? 2 * g.chunks
                       : plan.split_chunks * (kChunkBytes / sizeof(T) / chunk);
  char* space = static_cast<char*>(workspace);
  if (plan.copy_p || plan.copy_q) {
    Copies c = {};
    unsigned groups = 0;
    int n = 0;
    auto copy = [&](const void** at, long stride, bool k_inner, int rows,
                    size_t size) {
      c.in[n] = *at;
      c.out[n] = space;
      c.in_stride[n] = stride;
      c.rows[n] = epi::memory_rows(k_inner, rows, g.k);
      c.cols[n] = epi::memory_cols(k_inner, rows, g.k);
      c.out_stride[n] = epi::copied_stride(c.cols[n], sizeof(T));
      const size_t pieces =
          static_cast<size_t>(c.rows[n]) * c.out_stride[n] * sizeof(T) / 16;
      groups += static_cast<unsigned>(ceil_div(pieces, size_t{256}));
      c.groups[n] = groups;
      *at = space;
      space += size;
      return c.out_stride[n++];
    };
    if (plan.copy_p) {
      const long stride = g.p_stride;
      for (int i = 0; i < (g.gated ? 1 : 2); ++i)
        g.p_stride = copy(&g.p[i], stride, true, g.m, plan.p_bytes);
    }
    if (plan.copy_q) {
      const long stride = g.q_stride;
      for (int i = 0; i < 2; ++i)
        g.q_stride = copy(&g.q[i], stride, g.q_k_inner, g.n, plan.q_bytes);
    }
    hipLaunchKernelGGL(copy_rows_kernel<T>, dim3(groups), dim3(256), 0, stream, c);
    SNN_HIP_CHECK_LAUNCH();
  }
  g.partial = reinterpret_cast<float*>(space);
  int status;
  if (g.gated)
    status = g.q_k_inner ? launch_tile<T, true, true>(g, plan.kernel, stream)
                         : launch_tile<T, true, false>(g, plan.kernel, stream);
  else
    status = g.q_k_inner ? launch_tile<T, false, true>(g, plan.kernel, stream)
                         : launch_tile<T, false, false>(g, plan.kernel, stream);
  if (status != SNN_HIP_OK || g.splits == 1) return status;
  const size_t threads = static_cast<size_t>(g.m) * ceil_div(g.n, 8);
  hipLaunchKernelGGL(join_kernel<T>,
                     dim3(static_cast<unsigned>(ceil_div(threads, size_t{256}))),
                     dim3(256), 0, stream, g);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

}  // namespace gated
}  // namespace snn

#endif  // PORTDNN_AMD_CSRC_GATED_MATMUL_RUN_H_
