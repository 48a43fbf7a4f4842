// Gated linear recurrence over the steps of a sequence, channel by channel, and
// its gradients (gfx950):
//
//   a_t = sigmoid(f_t),  b_t = w_t x_t,  w_t = sigmoid(i_t) or 1 - a_t
//   h_t = a_t h_{t-1} + b_t
//
// Steps compose: a run of them is h -> A h + S with A = a_t ... a_s, and two
// runs in turn are (A, S) then (A', S') = (A' A, A' S + S').  A lane owns a few
// neighbouring channels and walks the steps of a piece of the sequence.  Where
// the sequences and channels do not fill the GPU, a sequence is divided into
// pieces: one launch finds every piece's (A, S), a second the state in front
// of every piece, a third walks the pieces from there.  The gradients run the
// other way: with D_t = a_t G_t, the gradient that step t hands to step t - 1,
//
//   G_t = dh_t + D_{t+1}   D_t = a_t dh_t + a_t D_{t+1}
//   dx_t = G_t w_t   df_t = G_t (h_{t-1} [- x_t]) a_t (1 - a_t)
//   di_t = G_t x_t w_t (1 - w_t)
//
// All of it is bound by memory: a step is about ten operations on the values
// that it reads and writes once (the inputs of the recurrence itself twice where
// a sequence is divided).  States and pieces are fp32.
//
// A reset leaves h_{t-1} out by selection and not by a factor of zero, so that
// an infinite state does not survive it; steps behind a sequence's length are
// not read (a = 1, b = 0).
#include <algorithm>

#include "sequence.h"
#include "snn_kernels.h"

namespace snn {
namespace {

using seq::Pack;
using seq::pack;
using seq::sigmoid;
using seq::sigmoid_alone;
using seq::unpack;

// Steps whose loads are in flight together: 8 forward; the gradients, with five
// operands, keep more waves on a SIMD with 4 (4 x 4096 x 2048 binary16: 176 ->
// 147 us).
template <bool BACK>
constexpr int kSteps = BACK ? 4 : 8;

struct Recurrence {
  int batch, steps, channels;
  long stride, grad_stride;  // of x and the gates, of their gradients
  int pieces, piece_steps;
  const void *x, *f, *i, *h, *dh;
  const unsigned char* resets;
  const int* lengths;
  const float* initial;  // the state in front of the first step
  const float* first;    // the state (gradient) that the walk starts from
  float* last;           // ... and ends with
  void *out_h, *dx, *df, *di;
  float *A, *S;  // [batch][pieces][channels]
};

template <typename T>
constexpr int kVec = sizeof(T) == 2 ? 4 : 2;

// A piece with a reset has A = -0, which the factors behind it leave as it is; a
// product that has only become too small is +0.
__device__ __forceinline__ bool is_reset(float a) {
  return __float_as_uint(a) == 0x80000000u;
}

// What a wave needs of its place: sequence, piece, first channel of the lane.
struct Place {
  int b, piece, c, skip, begin, end, length;
  bool on;
};

// With `turned` the last come first: the walk behind a launch over the same
// pieces then begins with what that has read last and the caches still hold.
template <int VEC>
__device__ __forceinline__ Place place_of(const Recurrence& r, bool turned) {
  Place p;
  const int blocks = (r.channels + 64 * VEC - 1) / (64 * VEC);
  const unsigned place = turned ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const unsigned at = place * (blockDim.x / 64) + threadIdx.x / 64;
  const unsigned row = at / blocks;
  const int first =
      static_cast<int>(at - row * blocks) * 64 * VEC + (threadIdx.x & 63) * VEC;
  // (a row's last channels: see Group; what is before them is not stored)
  const seq::Group<VEC> group(first, r.channels);
  p.c = group.c;
  p.skip = group.skip;
  p.b = static_cast<int>(row / r.pieces);
  p.piece = static_cast<int>(row - static_cast<unsigned>(p.b) * r.pieces);
  p.on = p.b < r.batch && first < r.channels;
  if (p.b >= r.batch) p.b = 0;
  p.begin = p.piece * r.piece_steps;
  p.end = min(r.steps, p.begin + r.piece_steps);
  p.length = r.lengths == nullptr
                 ? r.steps
                 : max(0, min(r.steps, r.lengths[p.b]));
  return p;
}

// Stores the lane's own of VEC values.
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

// (A, S) of a piece, forward: S behind the piece's steps from a zero state;
// backward: the gradient in front of it from a zero gradient behind.
template <typename T, int VEC, bool GATE, bool BACK>
__global__ void __launch_bounds__(256)
    recurrence_pieces_kernel(Recurrence r) {
  typedef typename Pack<T, VEC>::type V;
  constexpr int kGroup = kSteps<BACK>;
  const Place p = place_of<VEC>(r, false);
  if (!p.on) return;
  const long row = static_cast<long>(p.b) * r.steps;
  const T* const f = static_cast<const T*>(r.f) + row * r.stride + p.c;
  const T* const x = static_cast<const T*>(r.x) + row * r.stride + p.c;
  const T* const ig = GATE ? static_cast<const T*>(r.i) + row * r.stride + p.c
                           : nullptr;
  const T* const dh =
      BACK ? static_cast<const T*>(r.dh) + row * r.channels + p.c : nullptr;
  float A[VEC], S[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    A[k] = 1.f;
    S[k] = 0.f;
  }
  const int end = min(p.end, p.length);
  const int groups = (end - p.begin + kGroup - 1) / kGroup;
  for (int g = 0; g < groups; ++g) {
    V fv[kGroup], xv[kGroup], iv[kGroup];
    unsigned char fresh[kGroup];
    const int first = BACK ? p.begin + (groups - 1 - g) * kGroup
                           : p.begin + g * kGroup;
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      const int t = min(first + u, end - 1);
      fv[u] = *reinterpret_cast<const V*>(f + t * r.stride);
      if (BACK) {
        xv[u] = *reinterpret_cast<const V*>(dh + static_cast<long>(t) *
                                                     r.channels);
      } else {
        xv[u] = *reinterpret_cast<const V*>(x + t * r.stride);
        if (GATE) iv[u] = *reinterpret_cast<const V*>(ig + t * r.stride);
      }
      fresh[u] = r.resets == nullptr ? 0 : r.resets[row + t];
    }
#pragma unroll
    for (int n = 0; n < kGroup; ++n) {
      const int u = BACK ? kGroup - 1 - n : n;
      if (first + u >= end) continue;
      float fs[VEC], xs[VEC], is[VEC];
      unpack<T, VEC>(fv[u], fs);
      unpack<T, VEC>(xv[u], xs);
      if (GATE && !BACK) unpack<T, VEC>(iv[u], is);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float a, w;
        if (BACK || GATE)
          a = sigmoid_alone<T>(fs[k]);
        else
          sigmoid<T>(fs[k], &a, &w);
        if (BACK) {
          S[k] = fresh[u] ? 0.f : a * (xs[k] + S[k]);
          A[k] = fresh[u] ? -0.f : a * A[k];
        } else {
          if (GATE) w = sigmoid_alone<T>(is[k]);
          S[k] = w * xs[k] + (fresh[u] ? 0.f : a * S[k]);
          A[k] = fresh[u] ? -0.f : a * A[k];
        }
      }
    }
  }
  const long at = (static_cast<long>(p.b) * r.pieces + p.piece) * r.channels +
                  p.c;
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    r.A[at + k] = A[k];
    r.S[at + k] = S[k];
  }
}

// The state in front of every piece, over S; `last` behind the last one.  A
// work-group takes 64 channels of a sequence; each of its 16 waves composes a
// run of the pieces, the runs' results are composed in turn by every wave up to
// its own, and the wave walks its run from there.
template <bool BACK>
__global__ void __launch_bounds__(1024)
    recurrence_join_kernel(Recurrence r) {
  constexpr int kRuns = 16;
  __shared__ float run_a[kRuns][64], run_s[kRuns][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
  const int blocks = (r.channels + 63) / 64;
  const int b = blockIdx.x / blocks;
  const int c = (blockIdx.x - b * blocks) * 64 + lane;
  const bool on = c < r.channels;
  const int each = (r.pieces + kRuns - 1) / kRuns;
  const int begin = min(r.pieces, run * each), end = min(r.pieces, begin + each);
  const long base = static_cast<long>(b) * r.pieces * r.channels + c;
  auto at = [&](int n) {  // the n-th piece in the walk's order
    return base + static_cast<long>(BACK ? r.pieces - 1 - n : n) * r.channels;
  };
  // (eight pieces' pairs are under way together)
  constexpr int kBatch = 8;
  auto walk = [&](auto step) {
    for (int n = begin; n < end; n += kBatch) {
      float a[kBatch], s[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const long where = at(min(n + u, end - 1));
        a[u] = r.A[where];
        s[u] = r.S[where];
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (n + u < end) step(n + u, a[u], s[u]);
    }
  };
  float A = 1.f, S = 0.f;
  if (on)
    walk([&](int, float a, float s) {
      S = is_reset(a) ? s : a * S + s;
      A = is_reset(a) ? a : A * a;
    });
  run_a[run][lane] = A;
  run_s[run][lane] = S;
  // (read in front of the barrier: `last` may be the same buffer)
  const long state_at = static_cast<long>(b) * r.channels + c;
  float state = !on || r.first == nullptr ? 0.f : r.first[state_at];
  __syncthreads();
  if (!on) return;
  for (int q = 0; q < run; ++q) {
    const float a = run_a[q][lane];
    state = is_reset(a) ? run_s[q][lane] : a * state + run_s[q][lane];
  }
  walk([&](int n, float a, float s) {
    r.S[at(n)] = state;
    state = is_reset(a) ? s : a * state + s;
  });
  if (run == kRuns - 1 && r.last != nullptr) r.last[state_at] = state;
}

// The walk over a piece from the state in front of it.
template <typename T, int VEC, bool GATE>
__global__ void __launch_bounds__(256) recurrence_walk_kernel(Recurrence r) {
  typedef typename Pack<T, VEC>::type V;
  constexpr int kGroup = kSteps<false>;
  const Place p = place_of<VEC>(r, r.pieces > 1);
  if (!p.on) return;
  const long row = static_cast<long>(p.b) * r.steps;
  const T* const f = static_cast<const T*>(r.f) + row * r.stride + p.c;
  const T* const x = static_cast<const T*>(r.x) + row * r.stride + p.c;
  const T* const ig = GATE ? static_cast<const T*>(r.i) + row * r.stride + p.c
                           : nullptr;
  T* const h = static_cast<T*>(r.out_h) + row * r.channels + p.c;
  const long state_at = static_cast<long>(p.b) * r.channels + p.c;
  const float* const from =
      r.pieces > 1 ? r.S + (static_cast<long>(p.b) * r.pieces + p.piece) *
                               r.channels + p.c
                   : r.first == nullptr ? nullptr : r.first + state_at;
  float state[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) state[k] = from == nullptr ? 0.f : from[k];
  const int end = min(p.end, p.length);
  for (int first = p.begin; first < end; first += kGroup) {
    V fv[kGroup], xv[kGroup], iv[kGroup];
    unsigned char fresh[kGroup];
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      const int t = min(first + u, end - 1);
      fv[u] = *reinterpret_cast<const V*>(f + t * r.stride);
      xv[u] = *reinterpret_cast<const V*>(x + t * r.stride);
      if (GATE) iv[u] = *reinterpret_cast<const V*>(ig + t * r.stride);
      fresh[u] = r.resets == nullptr ? 0 : r.resets[row + t];
    }
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      if (first + u >= end) break;
      float fs[VEC], xs[VEC], is[VEC];
      unpack<T, VEC>(fv[u], fs);
      unpack<T, VEC>(xv[u], xs);
      if (GATE) unpack<T, VEC>(iv[u], is);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float a, w;
        if (GATE) {
          a = sigmoid_alone<T>(fs[k]);
          w = sigmoid_alone<T>(is[k]);
        } else {
          sigmoid<T>(fs[k], &a, &w);
        }
        state[k] = w * xs[k] + (fresh[u] ? 0.f : a * state[k]);
      }
      put<T, VEC>(h + static_cast<long>(first + u) * r.channels, state, p.skip);
    }
  }
  float zero[VEC] = {};
  for (int t = max(p.begin, end); t < p.end; ++t)
    put<T, VEC>(h + static_cast<long>(t) * r.channels, zero, p.skip);
  if (r.pieces == 1 && r.last != nullptr)
    put<float, VEC>(r.last + state_at, state, p.skip);
}

// The gradients' walk over a piece, from its end, with the gradient that the
// step behind it hands over.
template <typename T, int VEC, bool GATE>
__global__ void __launch_bounds__(256) recurrence_grad_kernel(Recurrence r) {
  typedef typename Pack<T, VEC>::type V;
  constexpr int kGroup = kSteps<true>;
  const Place p = place_of<VEC>(r, r.pieces > 1);
  if (!p.on) return;
  const long row = static_cast<long>(p.b) * r.steps;
  const T* const f = static_cast<const T*>(r.f) + row * r.stride + p.c;
  const T* const x = static_cast<const T*>(r.x) + row * r.stride + p.c;
  const T* const ig = GATE ? static_cast<const T*>(r.i) + row * r.stride + p.c
                           : nullptr;
  const T* const h = static_cast<const T*>(r.h) + row * r.channels + p.c;
  const T* const dh = static_cast<const T*>(r.dh) + row * r.channels + p.c;
  T* const dx = static_cast<T*>(r.dx) + row * r.grad_stride + p.c;
  T* const df = static_cast<T*>(r.df) + row * r.grad_stride + p.c;
  T* const di =
      GATE ? static_cast<T*>(r.di) + row * r.grad_stride + p.c : nullptr;
  const long state_at = static_cast<long>(p.b) * r.channels + p.c;
  const float* const from =
      r.pieces > 1 ? r.S + (static_cast<long>(p.b) * r.pieces + p.piece) *
                               r.channels + p.c
                   : r.first == nullptr ? nullptr : r.first + state_at;
  float D[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) D[k] = from == nullptr ? 0.f : from[k];
  const int end = min(p.end, p.length);
  const float zero[VEC] = {};
  for (int t = max(p.begin, end); t < p.end; ++t) {
    put<T, VEC>(dx + t * r.grad_stride, zero, p.skip);
    put<T, VEC>(df + t * r.grad_stride, zero, p.skip);
    if (GATE) put<T, VEC>(di + t * r.grad_stride, zero, p.skip);
  }
  const int groups = (end - p.begin + kGroup - 1) / kGroup;
  for (int g = groups - 1; g >= 0; --g) {
    V fv[kGroup], xv[kGroup], iv[kGroup], hv[kGroup], dv[kGroup];
    unsigned char fresh[kGroup];
    const int first = p.begin + g * kGroup;
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      const int t = min(first + u, end - 1);
      fv[u] = *reinterpret_cast<const V*>(f + t * r.stride);
      xv[u] = *reinterpret_cast<const V*>(x + t * r.stride);
      if (GATE) iv[u] = *reinterpret_cast<const V*>(ig + t * r.stride);
      hv[u] = *reinterpret_cast<const V*>(
          h + static_cast<long>(max(t - 1, 0)) * r.channels);
      dv[u] = *reinterpret_cast<const V*>(dh + static_cast<long>(t) *
                                                   r.channels);
      fresh[u] = r.resets == nullptr ? 0 : r.resets[row + t];
    }
#pragma unroll
    for (int u = kGroup - 1; u >= 0; --u) {
      const int t = first + u;
      if (t >= end) continue;
      float fs[VEC], xs[VEC], is[VEC], before[VEC], ds[VEC];
      float gx[VEC], gf[VEC], gi[VEC];
      unpack<T, VEC>(fv[u], fs);
      unpack<T, VEC>(xv[u], xs);
      if (GATE) unpack<T, VEC>(iv[u], is);
      unpack<T, VEC>(hv[u], before);
      unpack<T, VEC>(dv[u], ds);
      if (t == 0) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          before[k] = r.initial == nullptr ? 0.f : r.initial[state_at + k];
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float a, rest, w, w_rest;
        sigmoid<T>(fs[k], &a, &rest);
        if (GATE) {
          sigmoid<T>(is[k], &w, &w_rest);
        } else {
          w = rest;
        }
        const float G = ds[k] + D[k];
        const float prior = fresh[u] ? 0.f : before[k];
        gx[k] = G * w;
        gf[k] = G * (GATE ? prior : prior - xs[k]) * (a * rest);
        if (GATE) gi[k] = G * xs[k] * (w * w_rest);
        D[k] = fresh[u] ? 0.f : a * G;
      }
      put<T, VEC>(dx + t * r.grad_stride, gx, p.skip);
      put<T, VEC>(df + t * r.grad_stride, gf, p.skip);
      if (GATE) put<T, VEC>(di + t * r.grad_stride, gi, p.skip);
    }
  }
  if (r.pieces == 1 && r.last != nullptr)
    put<float, VEC>(r.last + state_at, D, p.skip);
}

// How many pieces a sequence is divided into: as many as give the GPU
// kWantedWaves waves, of kLeastSteps steps at least so that a piece's fp32
// pair costs little beside its steps.
constexpr int kWantedWaves = 4096;
constexpr int kLeastSteps = 32;

template <typename T>
void divide_steps(const snn_hip_linear_recurrence_params& p, int* pieces,
                  int* piece_steps) {
  const long waves =
      static_cast<long>(p.batch) * ceil_div(p.channels, 64 * kVec<T>);
  const long want = std::max(1l, kWantedWaves / waves);
  const long most = std::max(1, p.steps / kLeastSteps);
  const int n = static_cast<int>(std::min(want, most));
  *piece_steps = ceil_div(ceil_div(p.steps, n), kSteps<false>) * kSteps<false>;
  *pieces = ceil_div(p.steps, *piece_steps);
}

size_t pair_floats(const snn_hip_linear_recurrence_params& p, int pieces) {
  return pieces < 2 ? 0
                    : size_t{2} * static_cast<size_t>(p.batch) * pieces *
                          p.channels;
}

template <typename T, int VEC, bool GATE, bool BACK>
int launch_recurrence_as(const Recurrence& r, hipStream_t stream) {
  const long waves = static_cast<long>(r.batch) * r.pieces *
                     ceil_div(r.channels, 64 * VEC);
  if (waves > INT_MAX) return SNN_HIP_INDEX_EXCEEDED;
  const dim3 grid(static_cast<unsigned>((waves + 3) / 4)), threads(256);
  KernelTimer timer(stream);
  if (r.pieces > 1) {
    hipLaunchKernelGGL((recurrence_pieces_kernel<T, VEC, GATE, BACK>), grid,
                       threads, 0, stream, r);
    SNN_HIP_CHECK_LAUNCH();
    hipLaunchKernelGGL(
        (recurrence_join_kernel<BACK>),
        dim3(static_cast<unsigned>(r.batch * ceil_div(r.channels, 64))),
        dim3(1024), 0, stream, r);
    SNN_HIP_CHECK_LAUNCH();
  }
  if (BACK)
    hipLaunchKernelGGL((recurrence_grad_kernel<T, VEC, GATE>), grid, threads, 0,
                       stream, r);
  else
    hipLaunchKernelGGL((recurrence_walk_kernel<T, VEC, GATE>), grid, threads, 0,
                       stream, r);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T, bool BACK>
int launch_recurrence(Recurrence r, const snn_hip_linear_recurrence_params& p,
                      void* workspace, size_t elems, hipStream_t stream) {
  r.batch = p.batch;
  r.steps = p.steps;
  r.channels = p.channels;
  r.stride = p.row_stride == 0 ? p.channels : p.row_stride;
  r.grad_stride = p.grad_row_stride == 0 ? p.channels : p.grad_row_stride;
  divide_steps<T>(p, &r.pieces, &r.piece_steps);
  const size_t floats = pair_floats(p, r.pieces);
  if (workspace == nullptr || elems * sizeof(T) < floats * sizeof(float)) {
    r.pieces = 1;
    r.piece_steps = p.steps;
  } else {
    r.A = static_cast<float*>(workspace);
    r.S = r.A + floats / 2;
  }
  constexpr int VEC = kVec<T>;
  if (p.channels >= VEC)
    return r.i != nullptr ? launch_recurrence_as<T, VEC, true, BACK>(r, stream)
                          : launch_recurrence_as<T, VEC, false, BACK>(r, stream);
  return r.i != nullptr ? launch_recurrence_as<T, 1, true, BACK>(r, stream)
                        : launch_recurrence_as<T, 1, false, BACK>(r, stream);
}

int check_recurrence(const snn_hip_linear_recurrence_params* p,
                     const void* workspace) {
  if (p == nullptr) return SNN_HIP_INVALID_PARAMETER;
  SNN_REQUIRE(p->batch > 0 && p->steps > 0 && p->channels > 0);
  SNN_REQUIRE(p->row_stride == 0 || p->row_stride >= p->channels);
  SNN_REQUIRE(p->grad_row_stride == 0 || p->grad_row_stride >= p->channels);
  SNN_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0);
  // (the grids count waves and 64-channel blocks in 31 bits)
  if (static_cast<size_t>(p->batch) * ceil_div(p->channels, 64) > INT_MAX)
    return SNN_HIP_INDEX_EXCEEDED;
  return SNN_HIP_OK;
}

template <typename T>
int forward(const void* x, const void* forget, const void* input_gate,
            const unsigned char* resets, const int* lengths,
            const float* initial, void* h, float* final_state,
            const snn_hip_linear_recurrence_params* params, void* workspace,
            size_t elems, void* stream) {
  const int v = check_recurrence(params, workspace);
  if (v != SNN_HIP_OK) return v;
  SNN_REQUIRE(x != nullptr && forget != nullptr && h != nullptr);
  Recurrence r = {};
  r.x = x;
  r.f = forget;
  r.i = input_gate;
  r.resets = resets;
  r.lengths = lengths;
  r.first = initial;
  r.last = final_state;
  r.out_h = h;
  return launch_recurrence<T, false>(r, *params, workspace, elems,
                                     as_stream(stream));
}

template <typename T>
int backward(const void* grad_h, const float* grad_final, const void* x,
             const void* forget, const void* input_gate,
             const unsigned char* resets, const int* lengths,
             const float* initial, const void* h, void* grad_x,
             void* grad_forget, void* grad_input_gate, float* grad_initial,
             const snn_hip_linear_recurrence_params* params, void* workspace,
             size_t elems, void* stream) {
  const int v = check_recurrence(params, workspace);
  if (v != SNN_HIP_OK) return v;
  SNN_REQUIRE(grad_h != nullptr && x != nullptr && forget != nullptr &&
              h != nullptr && grad_x != nullptr && grad_forget != nullptr);
  SNN_REQUIRE((input_gate == nullptr) == (grad_input_gate == nullptr));
  Recurrence r = {};
  r.dh = grad_h;
  r.first = grad_final;
  r.x = x;
  r.f = forget;
  r.i = input_gate;
  r.resets = resets;
  r.lengths = lengths;
  r.initial = initial;
  r.h = h;
  r.dx = grad_x;
  r.df = grad_forget;
  r.di = grad_input_gate;
  r.last = grad_initial;
  return launch_recurrence<T, true>(r, *params, workspace, elems,
                                    as_stream(stream));
}

}  // namespace
}  // namespace snn

#define SNN_RECURRENCE(suffix, T)                                              \
  int snn_hip_linear_recurrence_##suffix(                                      \
      const void* x, const void* forget, const void* input_gate,               \
      const unsigned char* resets, const int* lengths,                         \
      const float* initial_state, void* h, float* final_state,                 \
      const snn_hip_linear_recurrence_params* params, void* workspace,         \
      size_t workspace_elems, void* stream) {                                  \
    return snn::forward<T>(x, forget, input_gate, resets, lengths,             \
                           initial_state, h, final_state, params, workspace,   \
                           workspace_elems, stream);                           \
  }                                                                            \
  int snn_hip_linear_recurrence_grad_##suffix(                                 \
      const void* grad_h, const float* grad_final_state, const void* x,        \
      const void* forget, const void* input_gate, const unsigned char* resets, \
      const int* lengths, const float* initial_state, const void* h,           \
      void* grad_x, void* grad_forget, void* grad_input_gate,                  \
      float* grad_initial_state,                                               \
      const snn_hip_linear_recurrence_params* params, void* workspace,         \
      size_t workspace_elems, void* stream) {                                  \
    return snn::backward<T>(grad_h, grad_final_state, x, forget, input_gate,   \
                            resets, lengths, initial_state, h, grad_x,         \
                            grad_forget, grad_input_gate, grad_initial_state,  \
                            params, workspace, workspace_elems, stream);       \
  }

extern "C" {

SNN_RECURRENCE(f32, float)
SNN_RECURRENCE(f16, _Float16)
SNN_RECURRENCE(bf16, __bf16)

int snn_hip_linear_recurrence_workspace_size(
    const snn_hip_linear_recurrence_params* params, int dtype,
    size_t* required_elems, size_t* recommended_elems) {
  const int v = snn::check_recurrence(params, nullptr);
  if (v != SNN_HIP_OK) return v;
  if (required_elems == nullptr || recommended_elems == nullptr ||
      dtype < SNN_HIP_DTYPE_F32 || dtype > SNN_HIP_DTYPE_BF16)
    return SNN_HIP_INVALID_PARAMETER;
  int pieces, piece_steps;
  if (dtype == SNN_HIP_DTYPE_F32)
    snn::divide_steps<float>(*params, &pieces, &piece_steps);
  else
    snn::divide_steps<_Float16>(*params, &pieces, &piece_steps);
  *required_elems = 0;
  *recommended_elems = snn::pair_floats(*params, pieces) *
                       (dtype == SNN_HIP_DTYPE_F32 ? 1 : 2);
  return SNN_HIP_OK;
}

}  // extern "C"
