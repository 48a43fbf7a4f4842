// The kernels of gemm_epilogue.h for one data type, and their launch; a source
// file of each type includes this so that they compile beside one another.
#ifndef PORTDNN_AMD_CSRC_GEMM_EPILOGUE_RUN_H_
#define PORTDNN_AMD_CSRC_GEMM_EPILOGUE_RUN_H_

#include "gemm_epilogue.h"
#include "snn_kernels.h"

namespace snn {
namespace epi {

template <typename T, bool PK, bool QK, int BM, int BN, int WM, int WN,
          int STAGES, bool DIRECT>
__global__ void __launch_bounds__(64 * WM * WN) gemm_kernel(Product g) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int kStage = Space<BM, BN, WM * WN, STAGES>::kStage;
  __shared__ __align__(1024) char ring0[kStage];
  __shared__ __align__(1024) char ring1[kStage];
  if constexpr (STAGES == 2) {
    gemm_body<T, PK, QK, BM, BN, WM, WN, 2, DIRECT>(g, ring0, ring1, nullptr,
                                                    nullptr);
  } else {
    __shared__ __align__(1024) char ring2[kStage];
    if constexpr (STAGES == 3) {
      gemm_body<T, PK, QK, BM, BN, WM, WN, 3, DIRECT>(g, ring0, ring1, ring2,
                                                      nullptr);
    } else {
      static_assert(STAGES == 4, "two to four chunks");
      __shared__ __align__(1024) char ring3[kStage];
      gemm_body<T, PK, QK, BM, BN, WM, WN, 4, DIRECT>(g, ring0, ring1, ring2,
                                                      ring3);
    }
  }
#endif
}

template <typename T, bool PK, bool QK, int BM, int BN, int WM, int WN,
          int STAGES, bool DIRECT>
int launch_as(const Product& g, hipStream_t stream) {
  const auto kernel = gemm_kernel<T, PK, QK, BM, BN, WM, WN, STAGES, DIRECT>;
  hipLaunchKernelGGL(
      kernel,
      dim3(static_cast<unsigned>(g.tiles_m) * g.tiles_n * g.splits),
      dim3(64 * WM * WN), 0, stream, g);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T, bool PK, bool QK>
int launch_tile(const Product& g, const Plan& p, bool direct,
                hipStream_t stream) {
  if (p.bm == 16)
    return direct ? launch_as<T, PK, QK, 16, 128, 1, 4, 4, true>(g, stream)
                  : launch_as<T, PK, QK, 16, 128, 1, 4, 2, false>(g, stream);
  if (p.bm == 64)
    return direct ? launch_as<T, PK, QK, 64, 128, 1, 4, 3, true>(g, stream)
                  : launch_as<T, PK, QK, 64, 128, 1, 4, 2, false>(g, stream);
  if constexpr (sizeof(T) == 2) {
    if (p.bm == 256)
      return launch_as<T, PK, QK, 256, 256, 2, 4, 2, true>(g, stream);
  }
  return direct ? launch_as<T, PK, QK, 128, 128, 2, 2, 2, true>(g, stream)
                : launch_as<T, PK, QK, 128, 128, 2, 2, 2, false>(g, stream);
}

template <typename T>
int run(Product& g, void* workspace, size_t bytes, hipStream_t stream) {
  auto fits = [&](const void* p, long stride) {
    return p == nullptr ||
           seq::rows_aligned(static_cast<const T*>(p), stride, 16);
  };
  // Straight to LDS: whole 16-byte pieces, and a tile's rows within 31 bits.
  constexpr int kPiece = 16 / sizeof(T);
  auto reach = [&](bool k_inner, long stride) {
    return (k_inner ? 256 : kChunkBytes / static_cast<int>(sizeof(T))) *
               stride * static_cast<long>(sizeof(T)) <
           0x7FFF0000l;
  };
  const bool direct = fits(g.p, g.p_stride) && fits(g.q, g.q_stride) &&
                      (g.p_k_inner ? g.k : g.m) % kPiece == 0 &&
                      (g.q_k_inner ? g.k : g.n) % kPiece == 0 &&
                      reach(g.p_k_inner, g.p_stride) &&
                      reach(g.q_k_inner, g.q_stride);
  const Plan plan = make_plan(g.m, g.n, g.k, sizeof(T), direct, bytes);
  if (static_cast<size_t>(plan.tiles_m) * plan.tiles_n * plan.splits > INT_MAX)
    return SNN_HIP_INDEX_EXCEEDED;
  g.tiles_m = plan.tiles_m;
  g.tiles_n = plan.tiles_n;
  g.splits = plan.splits;
  g.split_chunks = plan.split_chunks;
  g.partial = static_cast<float*>(workspace);
  g.wide = g.n % 8 == 0 && fits(g.out, g.out_stride) &&
           fits(g.pre, g.pre_stride) && fits(g.residual, g.residual_stride) &&
           fits(g.bias, 0);
  int status;
  if (g.p_k_inner)
    status = g.q_k_inner ? launch_tile<T, true, true>(g, plan, direct, stream)
                         : launch_tile<T, true, false>(g, plan, direct, stream);
  else
    status = g.q_k_inner ? launch_tile<T, false, true>(g, plan, direct, stream)
                         : launch_tile<T, false, false>(g, plan, direct, stream);
  if (status != SNN_HIP_OK || g.splits == 1) return status;
  const size_t threads = static_cast<size_t>(g.m) * ceil_div(g.n, 8);
  hipLaunchKernelGGL(gemm_join_kernel<T>,
                     dim3(static_cast<unsigned>(ceil_div(threads, size_t{256}))),
                     dim3(256), 0, stream, g);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

}  // namespace epi
}  // namespace snn

#endif  // PORTDNN_AMD_CSRC_GEMM_EPILOGUE_RUN_H_
