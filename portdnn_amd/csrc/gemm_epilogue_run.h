// The kernels of gemm_epilogue.h for one data type, and their launch; a source
// file of each type includes this so that they compile beside one another.
#ifndef PORTDNN_AMD_CSRC_GEMM_EPILOGUE_RUN_H_
#define PORTDNN_AMD_CSRC_GEMM_EPILOGUE_RUN_H_

#include "gemm_epilogue.h"
#include "snn_kernels.h"

namespace snn {
namespace epi {

template <typename T, bool PK, bool QK, int BM, int BN, int WM, int WN, int CB,
          int STAGES, int HELD>
__global__ void __launch_bounds__(64 * WM * WN) gemm_kernel(Product g) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int kStage = Space<BM, BN, WM * WN, CB>::kStage;
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
  gemm_body<T, PK, QK, BM, BN, WM, WN, CB, STAGES, HELD>(g, ring0, ring1, r2, r3,
                                                         r4);
#endif
}

template <typename T, bool PK, bool QK, int BM, int BN, int WM, int WN, int CB,
          int STAGES, int HELD = 0>
int launch_as(const Product& g, hipStream_t stream) {
  hipLaunchKernelGGL((gemm_kernel<T, PK, QK, BM, BN, WM, WN, CB, STAGES, HELD>),
                     dim3(static_cast<unsigned>(g.tiles_m) * g.tiles_n * g.splits),
                     dim3(64 * WM * WN), 0, stream, g);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T, bool PK, bool QK, int BM, int BN, int WAVES, int STAGES,
          bool DIRECT>
__global__ void __launch_bounds__(64 * WAVES) gemm_few_kernel(Product g) {
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
  gemm_few_body<T, PK, QK, BM, BN, WAVES, STAGES, DIRECT>(g, ring0, r1, r2, r3);
#endif
}

template <typename T, bool PK, bool QK, int BM, int BN, int WAVES, int STAGES,
          bool DIRECT>
int launch_few(const Product& g, hipStream_t stream) {
  hipLaunchKernelGGL(
      (gemm_few_kernel<T, PK, QK, BM, BN, WAVES, STAGES, DIRECT>),
      dim3(static_cast<unsigned>(g.tiles_m) * g.tiles_n * g.splits),
      dim3(64 * WAVES), 0, stream, g);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T, bool PK, bool QK>
int launch_tile(const Product& g, int kernel, hipStream_t stream) {
  switch (kernel) {
    case kFew16x16:
      return launch_few<T, PK, QK, 16, 16, 4, 4, true>(g, stream);
    case kFew16x32:
      return launch_few<T, PK, QK, 16, 32, 4, 4, true>(g, stream);
    case kFew32x32:
      return launch_few<T, PK, QK, 32, 32, 4, 2, true>(g, stream);
    case kTile64x128:
      return launch_as<T, PK, QK, 64, 128, 2, 4, 128, 5>(g, stream);
    case kAny16x16:
      return launch_few<T, PK, QK, 16, 16, 4, 4, false>(g, stream);
    case kAny32x32:
      return launch_few<T, PK, QK, 32, 32, 8, 2, false>(g, stream);
    case kAny64x32:
      return launch_few<T, PK, QK, 64, 32, 4, 2, false>(g, stream);
    case kAnyTile128:
      // (4095 x 1023 x 1001 binary16, the product alone: sixteen waves 18.4 us, eight
      // 19.9, four 26; four chunks under way 21; copies of both operands and their
      // products 25.7.  8191 x 4095 x 4095: 462 against 266 with copies)
      return launch_as<T, PK, QK, 128, 128, 4, 4, 128, 2, 2>(g, stream);
    default:
      break;
  }
  if constexpr (sizeof(T) == 2) {
    switch (kernel) {
      case kFew64x32:
        return launch_few<T, PK, QK, 64, 32, 4, 2, true>(g, stream);
      case kTile128:
        return launch_as<T, PK, QK, 128, 128, 2, 4, 128, 4>(g, stream);
      case kTile128Pair:
        return launch_as<T, PK, QK, 128, 128, 2, 4, 128, 2>(g, stream);
      case kTile256:
        // (eight waves where both operands' fragments are transposing reads, whose
        // addresses take sixteen waves' registers: 361 -> 201 us for 2048x8192x8192;
        // sixteen elsewhere: 203 against 208 and 217 against 220)
        if constexpr (!PK && !QK)
          return launch_as<T, PK, QK, 256, 256, 2, 4, 64, 4>(g, stream);
        return launch_as<T, PK, QK, 256, 256, 4, 4, 64, 4>(g, stream);
      default:
        break;
    }
  } else if (kernel == kTile128) {
    return launch_as<T, PK, QK, 128, 128, 2, 4, 64, 4>(g, stream);
  }
  return SNN_HIP_INVALID_ALGORITHM;
}

// One operand on its way to rows that start at multiples of 16 bytes.  (4095 x 1023
// and 1023 x 1001 binary16: 5.5-10 us, 21 MB read and written.)
struct Copy {
  const void* in;
  void* out;
  long in_stride, out_stride;
  int rows, cols;
  unsigned groups;  // work-groups
};

// Copies up to two operands; behind a row's end are zeros.
template <typename T>
__global__ void __launch_bounds__(256) copy_rows_kernel(Copy a, Copy b) {
  constexpr int kPiece = 16 / sizeof(T);
  const bool first = blockIdx.x < a.groups;
  const Copy c = first ? a : b;
  const unsigned group = first ? blockIdx.x : blockIdx.x - a.groups;
  const int pieces = static_cast<int>(c.out_stride / kPiece);
  const long at = static_cast<long>(group) * 256 + threadIdx.x;
  const long row = at / pieces;
  const int col = static_cast<int>(at - row * pieces) * kPiece;
  if (row >= c.rows) return;
  const T* const from = static_cast<const T*>(c.in) + row * c.in_stride + col;
  T part[kPiece];
  if (col + kPiece <= c.cols) {
    __builtin_memcpy(part, from, 16);
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
      part[i] = col + i < c.cols ? from[i] : T(0);
  }
  __builtin_memcpy(__builtin_assume_aligned(
                       static_cast<T*>(c.out) + row * c.out_stride + col, 16),
                   part, 16);
}

template <typename T>
int run(Product& g, void* workspace, size_t bytes, hipStream_t stream) {
  const Plan plan = make_plan(g, sizeof(T), bytes,
                              seq::aligned(static_cast<const T*>(g.p), 16),
                              seq::aligned(static_cast<const T*>(g.q), 16));
  if (plan.splits == 0) return SNN_HIP_INDEX_EXCEEDED;
  g.tiles_m = plan.tiles_m;
  g.tiles_n = plan.tiles_n;
  g.splits = plan.splits;
  g.split_chunks = plan.split_chunks;
  char* const space = static_cast<char*>(workspace);
  g.partial = reinterpret_cast<float*>(space + plan.p_bytes + plan.q_bytes);
  if (plan.copy_p || plan.copy_q) {
    Copy copies[2] = {};
    auto copy = [&](const void** at, long* stride, bool k_inner, int rows,
                    char* to, Copy* c) {
      c->in = *at;
      c->out = to;
      c->in_stride = *stride;
      c->rows = memory_rows(k_inner, rows, g.k);
      c->cols = memory_cols(k_inner, rows, g.k);
      c->out_stride = copied_stride(c->cols, sizeof(T));
      const size_t pieces = static_cast<size_t>(c->rows) * c->out_stride *
                            sizeof(T) / 16;
      c->groups = static_cast<unsigned>(ceil_div(pieces, size_t{256}));
      *at = to;
      *stride = c->out_stride;
    };
    if (plan.copy_p)
      copy(&g.p, &g.p_stride, g.p_k_inner, g.m, space, &copies[0]);
    if (plan.copy_q)
      copy(&g.q, &g.q_stride, g.q_k_inner, g.n, space + plan.p_bytes,
           &copies[1]);
    hipLaunchKernelGGL(copy_rows_kernel<T>,
                       dim3(copies[0].groups + copies[1].groups), dim3(256), 0,
                       stream, copies[0], copies[1]);
    SNN_HIP_CHECK_LAUNCH();
  }
  int status;
  if (g.p_k_inner)
    status = g.q_k_inner ? launch_tile<T, true, true>(g, plan.kernel, stream)
                         : launch_tile<T, true, false>(g, plan.kernel, stream);
  else
    status = g.q_k_inner ? launch_tile<T, false, true>(g, plan.kernel, stream)
                         : launch_tile<T, false, false>(g, plan.kernel, stream);
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
