// Device helpers of the operators of a residual block over sequences
// (residual_norm*.hip, linear_recurrence.hip, gemm_epilogue*.hip): vector
// accesses of float, binary16 and bfloat16, the logistic function, sums over a
// wave.
#ifndef PORTDNN_AMD_CSRC_SEQUENCE_H_
#define PORTDNN_AMD_CSRC_SEQUENCE_H_

#include <algorithm>
#include <type_traits>

#include "snn_common.h"

namespace snn {
namespace seq {

// VEC values of T as one access of VEC * sizeof(T) bytes at any address: the
// memory takes 16-byte accesses wherever a value may start, so that rows of any
// length and stride are read and written alike.
template <typename T, int VEC>
struct Pack {
  typedef T type __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
};
template <typename T>
struct Pack<T, 1> {
  typedef T type;
};

// Where a lane's VEC neighbouring channels begin: at `c`, or as far in front of
// it as the row's end asks for; `skip` of them are then the lane's before it and
// are neither summed nor stored twice.  (Rows of VEC channels at least.)
template <int VEC>
struct Group {
  int c, skip;
  __device__ __forceinline__ Group(int first, int channels)
      : c(min(first, channels - VEC)), skip(first - c) {}
};

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const typename Pack<T, VEC>::type& p,
                                       float (&out)[VEC]) {
  if constexpr (VEC == 1) {
    out[0] = static_cast<float>(p);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = static_cast<float>(p[i]);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ typename Pack<T, VEC>::type pack(
    const float (&in)[VEC]) {
  typename Pack<T, VEC>::type p;
  if constexpr (VEC == 1) {
    p = static_cast<T>(in[0]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = static_cast<T>(in[i]);
  }
  return p;
}

// sigmoid(z) and 1 - sigmoid(z), both to full relative precision: e = exp(-|z|)
// is at most 1, so neither overflows nor cancels.  The 16-bit types take the
// hardware's exponential, whose error of |z| 2^-23 is far below theirs.
template <typename T>
__device__ __forceinline__ void sigmoid(float z, float* s, float* rest) {
  const float e = sizeof(T) == 2 ? __expf(-fabsf(z)) : expf(-fabsf(z));
  const float large = __builtin_amdgcn_rcpf(1.f + e);
  const float small = e * large;
  *s = z >= 0.f ? large : small;
  *rest = z >= 0.f ? small : large;
}

// sigmoid(z) where the rest is not needed: an exponential that overflows gives
// the zero that it stands for.
template <typename T>
__device__ __forceinline__ float sigmoid_alone(float z) {
  return __builtin_amdgcn_rcpf(1.f + (sizeof(T) == 2 ? __expf(-z) : expf(-z)));
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// A dimension of a grid holds at most 2^32 - 1 work-items.
inline bool grid_fits(size_t groups, unsigned threads) {
  return groups <= UINT_MAX / threads;
}
// Where there may be more work-groups than that, they continue along y, 2^20 at a
// time; the last of these may not exist.
constexpr unsigned kGroupsOfX = 1u << 20;
inline dim3 grid_of(size_t groups) {
  return dim3(static_cast<unsigned>(std::min(groups, size_t{kGroupsOfX})),
              static_cast<unsigned>(ceil_div(groups, size_t{kGroupsOfX})));
}
__device__ __forceinline__ unsigned group_of_grid() {
  return blockIdx.x + blockIdx.y * kGroupsOfX;
}

// Adds up partial sums: out[c] = sum over `count` rows of `in`, `stride` floats
// apart.  blockIdx.y is the output, `step` floats behind the one before: row
// blockIdx.y of `rows_out`, or one of `outputs` (null: not wanted).  16 waves
// share a column's rows, and their sums are added in order.  Columns continue along
// z (columns_grid).
constexpr int kMaxSums = 5;
struct SumOutputs {
  void* out[kMaxSums];
};
template <typename T>
__global__ void __launch_bounds__(1024)
    add_rows_kernel(const float* __restrict__ in, SumOutputs outputs,
                    T* rows_out, int channels, int count, long stride,
                    long step) {
  __shared__ float part[16][64];
  T* const out = rows_out != nullptr
                     ? rows_out + static_cast<long>(blockIdx.y) * channels
                     : static_cast<T*>(outputs.out[blockIdx.y]);
  if (out == nullptr) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (blockIdx.x + blockIdx.z * kGroupsOfX) * 64 + lane;
  in += blockIdx.y * step + c;
  const int each = (count + 15) / 16;
  const int begin = min(count, wave * each), end = min(count, begin + each);
  float s = 0.f;
  if (c < channels) {
#pragma unroll 8
    for (int i = begin; i < end; ++i) s += in[i * stride];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= channels) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += part[w][lane];
  out[c] = static_cast<T>(s);
}

inline dim3 columns_grid(int channels, int outputs) {
  const dim3 columns = grid_of(ceil_div(channels, 64));
  return dim3(columns.x, static_cast<unsigned>(outputs), columns.y);
}

template <typename T>
inline bool aligned(const T* p, unsigned bytes) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0;
}

}  // namespace seq
}  // namespace snn

#endif  // PORTDNN_AMD_CSRC_SEQUENCE_H_
