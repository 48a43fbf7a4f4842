// What the kernels of residual_norm.hip and residual_norm_grad.hip share.
#ifndef PORTDNN_AMD_CSRC_RESIDUAL_NORM_H_
#define PORTDNN_AMD_CSRC_RESIDUAL_NORM_H_

#include "sequence.h"

namespace snn {
namespace norm {

// Rows of up to kMaxChannels values stay in registers: PT of them per lane.
constexpr int kMaxChannels = 16384;

// The operands as a kernel takes them: strides filled in.
struct Rows {
  snn_hip_residual_norm_tensors t;
  int rows, channels, post, pre, gate, gate_rows;
  long x_stride, gate_stride;
  float epsilon;
};

inline Rows rows_of(const snn_hip_residual_norm_tensors& t,
                    const snn_hip_residual_norm_params& p) {
  Rows r = {};
  r.t = t;
  r.rows = p.rows;
  r.channels = p.channels;
  r.post = p.post_norm;
  r.pre = p.pre_norm;
  r.gate = p.gate;
  r.gate_rows = p.gate_rows;
  r.x_stride = p.x_stride == 0 ? p.channels : p.x_stride;
  r.gate_stride = p.gate_stride == 0 ? p.channels : p.gate_stride;
  r.epsilon = p.epsilon;
  return r;
}

inline int check_params(const snn_hip_residual_norm_params* p) {
  if (p == nullptr) return SNN_HIP_INVALID_PARAMETER;
  SNN_REQUIRE(p->rows > 0 && p->channels > 0 && p->channels <= kMaxChannels);
  SNN_REQUIRE(p->post_norm >= SNN_HIP_NORM_NONE &&
              p->post_norm <= SNN_HIP_NORM_LAYER);
  SNN_REQUIRE(p->pre_norm >= SNN_HIP_NORM_NONE &&
              p->pre_norm <= SNN_HIP_NORM_LAYER);
  SNN_REQUIRE(p->gate >= SNN_HIP_GATE_NONE && p->gate <= SNN_HIP_GATE_SILU);
  SNN_REQUIRE(p->gate == SNN_HIP_GATE_NONE || p->gate_rows > 0);
  SNN_REQUIRE(p->x_stride == 0 || p->x_stride >= p->channels);
  SNN_REQUIRE(p->gate_stride == 0 || p->gate_stride >= p->channels);
  SNN_REQUIRE(p->epsilon >= 0.f);  // (a NaN is not)
  return SNN_HIP_OK;
}

inline int check_operands(const snn_hip_residual_norm_tensors* t,
                          const snn_hip_residual_norm_params& p) {
  if (t == nullptr) return SNN_HIP_INVALID_PARAMETER;
  SNN_REQUIRE(t->x != nullptr);
  SNN_REQUIRE((t->gate != nullptr) == (p.gate != SNN_HIP_GATE_NONE));
  SNN_REQUIRE(p.post_norm != SNN_HIP_NORM_NONE ||
              (t->post_weight == nullptr && t->post_bias == nullptr));
  SNN_REQUIRE(p.pre_norm != SNN_HIP_NORM_NONE ||
              (t->pre_weight == nullptr && t->pre_bias == nullptr));
  return SNN_HIP_OK;
}

// Sums over the lanes that share a row: a wave, or all waves of the work-group
// through LDS.  Two slots in turn, so that one barrier a sum is enough: a wave
// is past the reads of a slot when it has passed the next sum's barrier.
template <int WAVES, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* lds, int* turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = seq::wave_sum(v[i]);
  if constexpr (WAVES > 1) {
    float* const slot = lds + *turn * (2 * WAVES);
    *turn ^= 1;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) slot[i * WAVES + wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += slot[i * WAVES + w];
      v[i] = s;
    }
  }
}

// PT values of a row per lane, as PT / VEC accesses: access j of lane l is for
// the channels (j * lanes + l) * VEC ... + VEC - 1 and begins in front of them
// where the row ends before (see Group).  Values that are another lane's or behind
// the row's end are zero and are not stored.  WHOLE: rows are a multiple of VEC,
// so that an access is inside as a whole or not at all.
template <typename T, int VEC, int PT, int WAVES, bool WHOLE>
struct Slice {
  static constexpr int kLanes = 64 * WAVES;
  typedef typename seq::Pack<T, VEC>::type V;

  static __device__ __forceinline__ int lane() {
    return WAVES == 1 ? static_cast<int>(threadIdx.x & 63)
                      : static_cast<int>(threadIdx.x);
  }
  static __device__ __forceinline__ int first(int j) {
    return (j * kLanes + lane()) * VEC;
  }
  // the channel of value i
  static __device__ __forceinline__ int start(int j, int channels) {
    return WHOLE ? first(j) : min(first(j), channels - VEC);
  }
  static __device__ __forceinline__ int channel(int i, int channels) {
    return start(i / VEC, channels) + i % VEC;
  }
  static __device__ __forceinline__ bool inside(int i, int channels) {
    const int c = first(i / VEC);
    return c < channels && (WHOLE || start(i / VEC, channels) + i % VEC >= c);
  }
  static constexpr int kAccesses = PT / VEC;
  // As they are in memory, which takes fewer registers; `absent` where there is
  // no row.
  static __device__ __forceinline__ void fetch(const void* row, int channels,
                                               V (&raw)[kAccesses],
                                               float absent = 0.f) {
#pragma unroll
    for (int j = 0; j < kAccesses; ++j) {
      float part[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) part[k] = absent;
      raw[j] = seq::pack<T, VEC>(part);
      if (row != nullptr && first(j) < channels)
        raw[j] = *reinterpret_cast<const V*>(static_cast<const T*>(row) +
                                             start(j, channels));
    }
  }
  static __device__ __forceinline__ void expand(const V (&raw)[kAccesses],
                                                int channels,
                                                float (&out)[PT]) {
#pragma unroll
    for (int j = 0; j < kAccesses; ++j) {
      float part[VEC];
      seq::unpack<T, VEC>(raw[j], part);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const int i = j * VEC + k;
        // (an access that is outside has not been made)
        out[i] = WHOLE || inside(i, channels) ? part[k] : 0.f;
      }
    }
  }
  static __device__ __forceinline__ void load(const void* row, int channels,
                                              float (&out)[PT]) {
    V raw[kAccesses];
    fetch(row, channels, raw);
    expand(raw, channels, out);
  }
  static __device__ __forceinline__ void store(void* row, int channels,
                                               const float (&in)[PT]) {
#pragma unroll
    for (int j = 0; j < PT / VEC; ++j) {
      T* const at = static_cast<T*>(row) + first(j);
      const int skip = first(j) + VEC - channels;  // above zero at the row's end
      if (WHOLE ? first(j) < channels : skip <= 0) {
        float part[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) part[k] = in[j * VEC + k];
        *reinterpret_cast<V*>(at) = seq::pack<T, VEC>(part);
      } else if (!WHOLE) {
#pragma unroll
        for (int k = 1; k < VEC; ++k)
          if (k >= skip) at[k - skip] = static_cast<T>(in[j * VEC + k]);
      }
    }
  }
};

// At most PT = 8 values per lane up to 8192 channels, 16 beyond.
template <typename Go>
int by_length(int channels, Go go) {
  using std::integral_constant;
  if (channels <= 512)
    return go(integral_constant<int, 1>(), integral_constant<int, 8>());
  if (channels <= 1024)
    return go(integral_constant<int, 2>(), integral_constant<int, 8>());
  if (channels <= 2048)
    return go(integral_constant<int, 4>(), integral_constant<int, 8>());
  if (channels <= 4096)
    return go(integral_constant<int, 8>(), integral_constant<int, 8>());
  if (channels <= 8192)
    return go(integral_constant<int, 16>(), integral_constant<int, 8>());
  return go(integral_constant<int, 16>(), integral_constant<int, 16>());
}

// Calls `go` with the waves that share a row, the values per lane, and whether
// rows are a multiple of VEC.
template <int VEC, typename Go>
int by_channels(int channels, Go go) {
  return channels % VEC == 0
             ? by_length(channels, [&](auto waves, auto values) {
                 return go(waves, values, std::true_type());
               })
             : by_length(channels, [&](auto waves, auto values) {
                 return go(waves, values, std::false_type());
               });
}

}  // namespace norm
}  // namespace snn

#endif  // PORTDNN_AMD_CSRC_RESIDUAL_NORM_H_
