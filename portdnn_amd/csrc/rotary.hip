// Positions by rotation (gfx950): pair i of a token at position p is turned by
// 2 pi p f_i, f in turns,
//
//   (a, b) -> magnitude (a cos - b sin, a sin + b cos)
//
// and by the negative angle for the inverse, which is also the gradient.
//
// Bound by memory: a value is read and written once, and an angle serves all of a
// token's heads.  p f_i is taken in 64 bits and only its fraction, below half a turn,
// goes on in fp32: at position 10^6 an angle that was held in fp32 throughout would
// be off by 0.06.  A lane holds the sines and cosines of VEC pairs of a token and
// walks every `slices`-th of its heads.
//
// bfloat16, 4 x 4096 tokens of 32 heads of 128 channels: 54 us, 268 MB, 5.0 TB/s; fp32,
// 2 x 5001 tokens of 12 heads of 100 channels, 64 of them turned as neighbours: 28.6 us,
// 96 MB, 3.4 TB/s, with angles that memory waits for (31.2 us while the first heads were
// asked for behind them).  A token of 16 sequences is the time of a launch.
#include <algorithm>
#include <cmath>

#include "sequence.h"
#include "snn_kernels.h"

namespace snn {
namespace {

using seq::Group;
using seq::Pack;
using seq::pack;
using seq::unpack;

struct Rotary {
  const void* in;
  void* out;
  const double* frequencies;
  const int* positions;
  long in_stride, out_stride;
  int steps, heads, channels, turned, kind;
  int turns, copies;  // lanes for a head: of pairs, of channels that stay
  int slices;         // lanes that share a token's heads
  unsigned lanes;
  float magnitude;
  bool inverse;
};

// Sine and cosine of a fraction of a turn.  The 16-bit types take the hardware's,
// whose errors of 2^-20 are far below theirs.
template <typename T>
__device__ __forceinline__ void turn_of(float fraction, float* s, float* c) {
  if constexpr (sizeof(T) == 2) {
    *s = __builtin_amdgcn_sinf(fraction);
    *c = __builtin_amdgcn_cosf(fraction);
  } else {
    sincospif(2.f * fraction, s, c);
  }
}

// A lane's own of VEC values, from `skip` on.
template <typename T, int VEC>
__device__ __forceinline__ void put(T* at, const float (&v)[VEC], int skip) {
  if (skip == 0) {
    *reinterpret_cast<typename Pack<T, VEC>::type*>(at) = pack<T, VEC>(v);
  } else {
#pragma unroll
    for (int k = 1; k < VEC; ++k)
      if (k >= skip) at[k] = static_cast<T>(v[k]);
  }
}

// VEC pairs of each head: two groups of VEC channels half of `turned` apart, or 2 VEC
// channels in a row.  (Lanes whose groups overlap at the end compute the same values
// of those that they share, and one of them stores, so that in place works too.)
template <typename T, int VEC, bool PAIRS>
__global__ void __launch_bounds__(256) rotary_kernel(Rotary r) {
  typedef typename Pack<T, VEC>::type V;
  const unsigned lane = blockIdx.x * 256u + threadIdx.x;
  if (lane >= r.lanes) return;
  const unsigned units = r.turns + r.copies;
  const unsigned unit = lane % units, rest = lane / units;
  const unsigned slice = rest % r.slices, row = rest / r.slices;
  const T* in = static_cast<const T*>(r.in) + row * r.in_stride +
                static_cast<long>(slice) * r.channels;
  T* out = static_cast<T*>(r.out) + row * r.out_stride +
           static_cast<long>(slice) * r.channels;
  const long step = static_cast<long>(r.slices) * r.channels;

  if (unit >= static_cast<unsigned>(r.turns)) {  // channels that stay
    const int first = r.turned + (unit - r.turns) * VEC;
    const int stay = r.channels - r.turned;
    const int c = stay >= VEC ? min(first, r.channels - VEC) : first;
    constexpr int kAhead = 4;  // heads under way at once
    for (int h = slice; h < r.heads; h += kAhead * r.slices) {
      if (stay >= VEC) {
        V some[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (h + u * r.slices < r.heads)
            some[u] = *reinterpret_cast<const V*>(in + u * step + c);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (h + u * r.slices < r.heads)
            *reinterpret_cast<V*>(out + u * step + c) = some[u];
      } else {
        for (int u = 0; u < kAhead && h + u * r.slices < r.heads; ++u)
          for (int k = c; k < r.channels; ++k)
            out[u * step + k] = in[u * step + k];
      }
      in += kAhead * step;
      out += kAhead * step;
    }
    return;
  }

  const int half = r.turned / 2;
  const Group<VEC> at(static_cast<int>(unit) * VEC, half);
  const int c0 = PAIRS ? 2 * at.c : at.c;
  const int c1 = PAIRS ? c0 + VEC : c0 + half;
  // (two heads' values are on their way while the angles are worked out, and then while
  // the ones before are turned)
  V ahead[2][2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (slice + u * r.slices < static_cast<unsigned>(r.heads)) {
      ahead[u][0] = *reinterpret_cast<const V*>(in + u * step + c0);
      ahead[u][1] = *reinterpret_cast<const V*>(in + u * step + c1);
    }
  const unsigned b = row / r.steps, t = row - b * r.steps;
  const int kind = r.kind;
  const long p = kind == SNN_HIP_ROTARY_POSITIONS_NONE ? static_cast<long>(t)
                 : kind == SNN_HIP_ROTARY_POSITIONS_FIRST
                     ? static_cast<long>(r.positions[b]) + t
                     : static_cast<long>(r.positions[row]);
  float sine[VEC], cosine[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const double turns = static_cast<double>(p) * r.frequencies[at.c + i];
    turn_of<T>(static_cast<float>(turns - __builtin_rint(turns)), &sine[i],
               &cosine[i]);
    sine[i] *= r.inverse ? -r.magnitude : r.magnitude;
    cosine[i] *= r.magnitude;
  }
  auto turn = [&](V (&held)[2], bool more) {
    float x[2][VEC], y[2][VEC];
    unpack<T, VEC>(held[0], x[0]);
    unpack<T, VEC>(held[1], x[1]);
    if (more) {
      held[0] = *reinterpret_cast<const V*>(in + 2 * step + c0);
      held[1] = *reinterpret_cast<const V*>(in + 2 * step + c1);
    }
    if constexpr (PAIRS) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int e = 2 * i, o = 2 * i + 1;
        const float a = x[e / VEC][e % VEC], v = x[o / VEC][o % VEC];
        y[e / VEC][e % VEC] = a * cosine[i] - v * sine[i];
        y[o / VEC][o % VEC] = a * sine[i] + v * cosine[i];
      }
      put<T, VEC>(out + c0, y[0], min(2 * at.skip, VEC));
      put<T, VEC>(out + c1, y[1], max(2 * at.skip - VEC, 0));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        y[0][i] = x[0][i] * cosine[i] - x[1][i] * sine[i];
        y[1][i] = x[0][i] * sine[i] + x[1][i] * cosine[i];
      }
      put<T, VEC>(out + c0, y[0], at.skip);
      put<T, VEC>(out + c1, y[1], at.skip);
    }
    in += step;
    out += step;
  };
  for (int h = slice; h < r.heads; h += 2 * r.slices) {
    turn(ahead[0], h + 2 * r.slices < r.heads);
    if (h + r.slices < r.heads) turn(ahead[1], h + 3 * r.slices < r.heads);
  }
}

template <typename T, int VEC>
int launch_rotary(const Rotary& r, int layout, hipStream_t stream) {
  const dim3 grid((r.lanes - 1) / 256 + 1);
  if (layout == SNN_HIP_ROTARY_PAIRS)
    hipLaunchKernelGGL((rotary_kernel<T, VEC, true>), grid, dim3(256), 0,
                       stream, r);
  else
    hipLaunchKernelGGL((rotary_kernel<T, VEC, false>), grid, dim3(256), 0,
                       stream, r);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T>
int rotary(const void* input, const double* frequencies, const int* positions,
           void* output, const snn_hip_rotary_params* params,
           void* stream_arg) {
  if (params == nullptr) return SNN_HIP_INVALID_PARAMETER;
  const snn_hip_rotary_params& p = *params;
  SNN_REQUIRE(p.batch > 0 && p.steps > 0 && p.heads > 0 && p.channels > 0);
  SNN_REQUIRE(p.turned >= 2 && p.turned <= p.channels && p.turned % 2 == 0);
  SNN_REQUIRE(p.layout == SNN_HIP_ROTARY_HALVES ||
              p.layout == SNN_HIP_ROTARY_PAIRS);
  SNN_REQUIRE(p.positions >= SNN_HIP_ROTARY_POSITIONS_NONE &&
              p.positions <= SNN_HIP_ROTARY_POSITIONS_EACH);
  SNN_REQUIRE(std::isfinite(p.magnitude));
  const long width = static_cast<long>(p.heads) * p.channels;
  SNN_REQUIRE(p.row_stride == 0 || p.row_stride >= width);
  SNN_REQUIRE(p.output_row_stride == 0 || p.output_row_stride >= width);
  SNN_REQUIRE(input != nullptr && output != nullptr && frequencies != nullptr);
  SNN_REQUIRE((positions != nullptr) ==
              (p.positions != SNN_HIP_ROTARY_POSITIONS_NONE));
  Rotary r = {};
  r.in = input;
  r.out = output;
  r.frequencies = frequencies;
  r.positions = positions;
  r.in_stride = p.row_stride == 0 ? width : p.row_stride;
  r.out_stride = p.output_row_stride == 0 ? width : p.output_row_stride;
  SNN_REQUIRE(input != output || r.in_stride == r.out_stride);
  r.steps = p.steps;
  r.heads = p.heads;
  r.channels = p.channels;
  r.turned = p.turned;
  r.kind = p.positions;
  r.magnitude = p.magnitude;
  r.inverse = p.inverse != 0;
  constexpr int kWide = 16 / sizeof(T);
  const bool wide = p.turned / 2 >= kWide;
  const int vec = wide ? kWide : 1;
  r.turns = ceil_div(p.turned / 2, vec);
  r.copies = input == output ? 0 : ceil_div(p.channels - p.turned, vec);
  // Lanes for the GPU's 256 CUs, as long as a lane's angles serve some heads.
  const size_t rows = static_cast<size_t>(p.batch) * p.steps;
  const size_t tokens = rows * (r.turns + r.copies);
  constexpr size_t kLanes = 256 * 2048;
  r.slices = static_cast<int>(std::min<size_t>(
      p.heads, std::max<size_t>(1, kLanes / tokens)));
  if (tokens >= UINT_MAX - 255 || rows > UINT_MAX) return SNN_HIP_INDEX_EXCEEDED;
  r.lanes = static_cast<unsigned>(tokens * r.slices);
  const hipStream_t stream = as_stream(stream_arg);
  KernelTimer timer(stream);
  return wide ? launch_rotary<T, kWide>(r, p.layout, stream)
              : launch_rotary<T, 1>(r, p.layout, stream);
}

}  // namespace
}  // namespace snn

extern "C" {

int snn_hip_rotary_f32(const void* input, const double* frequencies,
                       const int* positions, void* output,
                       const snn_hip_rotary_params* params, void* stream) {
  return snn::rotary<float>(input, frequencies, positions, output, params,
                            stream);
}
int snn_hip_rotary_f16(const void* input, const double* frequencies,
                       const int* positions, void* output,
                       const snn_hip_rotary_params* params, void* stream) {
  return snn::rotary<_Float16>(input, frequencies, positions, output, params,
                               stream);
}
int snn_hip_rotary_bf16(const void* input, const double* frequencies,
                        const int* positions, void* output,
                        const snn_hip_rotary_params* params, void* stream) {
  return snn::rotary<__bf16>(input, frequencies, positions, output, params,
                             stream);
}

int snn_hip_rotary_frequencies(int turned, double base, int scaling,
                               double factor, double context, double low,
                               double high, double* frequencies) {
  SNN_REQUIRE(turned >= 2 && turned % 2 == 0 && frequencies != nullptr);
  SNN_REQUIRE(std::isfinite(base) && base > 0.0);
  SNN_REQUIRE(scaling >= SNN_HIP_ROTARY_SCALING_NONE &&
              scaling <= SNN_HIP_ROTARY_SCALING_BANDS);
  if (scaling != SNN_HIP_ROTARY_SCALING_NONE)
    SNN_REQUIRE(std::isfinite(factor) && factor > 0.0);
  if (scaling == SNN_HIP_ROTARY_SCALING_BANDS)
    SNN_REQUIRE(std::isfinite(context) && context > 0.0 &&
                std::isfinite(low) && std::isfinite(high) && low < high);
  constexpr double kTurn = 6.283185307179586476925;
  if (scaling == SNN_HIP_ROTARY_SCALING_BASE && turned > 2)
    base *= std::pow(factor, static_cast<double>(turned) / (turned - 2));
  for (int i = 0; i < turned / 2; ++i) {
    double f = std::pow(base, -2.0 * i / turned) / kTurn;
    if (scaling == SNN_HIP_ROTARY_SCALING_POSITIONS) f /= factor;
    if (scaling == SNN_HIP_ROTARY_SCALING_BANDS) {
      const double keep =
          std::min(1.0, std::max(0.0, (f * context - low) / (high - low)));
      f *= keep + (1.0 - keep) / factor;
    }
    frequencies[i] = f;
  }
  return SNN_HIP_OK;
}

}  // extern "C"
