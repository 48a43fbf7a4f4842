// Gated linear recurrence over the steps of a sequence, channel by channel, and
// its gradients (gfx950):
//
//   a_t = sigmoid(f_t),  b_t = w_t x_t,  w_t = sigmoid(i_t) or 1 - a_t
//   h_t = a_t h_{t-1} + b_t
//
// and backwards, with D_t = a_t G_t the gradient that step t hands to step t - 1,
//
//   G_t = dh_t + D_{t+1}   D_t = a_t dh_t + a_t D_{t+1}
//   dx_t = G_t w_t   df_t = G_t (h_{t-1} [- x_t]) a_t (1 - a_t)
//   di_t = G_t x_t w_t (1 - w_t)
//
// Bound by memory: a step is some twenty operations on values that are read and
// written once.  A lane owns a few neighbouring channels and walks the steps.
// Where sequences and channels do not fill the GPU with lanes, a sequence is
// divided: steps compose, a run of them is h -> A h + S, and two runs in turn are
// (A, S), (A', S') -> (A' A, A' S + S').  A work-group takes a piece of the
// sequence, every wave a segment of it, which it holds in registers:
//
//   1  every wave finds (A, S) of its segment, the work-group's are composed;
//   2  the piece's (A, S) is published for the pieces behind it;
//   3  the state in front of the piece is found: the nearest piece before it whose
//      state behind it is known already, and (A, S) of those between, in turn;
//   4  the state behind the piece is published, and every wave walks its segment
//      from the state in front of that.
//
// so that every operand is read once all the same.  Pieces are handed out by a
// counter in their order: a work-group waits only for pieces whose work-groups
// have begun before it, which therefore end.  The state behind a piece is A s + S
// of the state in front of it wherever it is computed, so that results do not
// depend on who waits for whom.  States and pieces are fp32.
//
// One sequence of 32768 x 2048 bfloat16: 121.5 us, 403 MB at 3.3 TB/s (with two passes
// over the operands 151); a gradient of 4 x 4096 x 2048 binary16 with both gates 131
// us, 537 MB at 4.1 TB/s.  What is left is the wait of a CU's few waves for the
// states, as their segments fill the registers.  A token of 64 x 4096 fp32: 3.8-4.6 us,
// a launch's latency.
//
// A reset leaves h_{t-1} out by selection and not by a factor of zero, so that
// an infinite state does not survive it; steps behind a sequence's length do not
// count (a = 1, b = 0).
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

struct Recurrence {
  int batch, steps, channels;
  long stride, grad_stride;  // of x and the gates, of their gradients
  const void *x, *f, *i, *h, *dh;
  const unsigned char* resets;
  const int* lengths;
  const float* initial;  // the state in front of the first step
  const float* first;    // the state (gradient) that the walk starts from
  float* last;           // ... and ends with
  void *out_h, *dx, *df, *di;
  // The divided walk: pieces, in the walk's order, of `segments` segments.
  int segments, pieces;
  unsigned* counter;          // of the pieces handed out
  unsigned* flags;            // [batch x channel blocks][pieces]: see kNothing
  unsigned long long* pairs;  // [as flags][64 VEC]: (A, S)
  unsigned* states;           // [as flags][64 VEC]: behind the piece
};

template <typename T>
constexpr int kVec = sizeof(T) == 2 ? 4 : 2;

// The gate a of a logit, with 1 - a where it is asked for.  Above zero, as sigmoid
// is: an infinite state stays infinite behind a gate that fp32 has no value for.
template <typename T>
__device__ __forceinline__ float gate_of(float z) {
  return sigmoid_alone<T>(z) + 0x1p-126f;
}
template <typename T>
__device__ __forceinline__ void gate_of(float z, float* a, float* rest) {
  sigmoid<T>(z, a, rest);
  *a += 0x1p-126f;
}

// A run of steps with a reset has A = -0, which the factors behind it leave as it
// is; products that become too small are the smallest value above zero, for the same
// reason (as bits: zero has none set).
__device__ __forceinline__ bool is_reset(float a) {
  return __float_as_uint(a) == 0x80000000u;
}
__device__ __forceinline__ float above_zero(float a) {
  return __uint_as_float(max(__float_as_uint(a), 1u));
}
__device__ __forceinline__ float composed(float a, float s, float state) {
  return is_reset(a) ? s : a * state + s;
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

__device__ __forceinline__ int length_of(const Recurrence& r, int b) {
  return r.lengths == nullptr ? r.steps
                              : max(0, min(r.steps, r.lengths[b]));
}

// Which of the steps `first` ... `first` + n - 1 (n <= 64; as far as they are
// before `end`) are resets, a bit each: one load for all.
__device__ __forceinline__ unsigned long long resets_of(const Recurrence& r,
                                                        long row, int first,
                                                        int n, int end) {
  if (r.resets == nullptr) return 0;
  const int lane = threadIdx.x & 63;
  const int t = first + lane;
  const bool on = lane < n && t < end;
  return __ballot(on && r.resets[row + (on ? t : 0)] != 0);
}

// ---- undivided ---------------------------------------------------------------

// Steps whose loads are in flight together.  (64 sequences of 48 x 256 bfloat16
// forward, whole: 15 us, with 8 of them 16.4.)
constexpr int kSteps = 4;

// What a wave needs of its place: sequence and first channel of the lane.  (Lanes
// behind a row's channels stay, and store nothing.)
struct Place {
  int b, c, skip;
};
template <int VEC>
__device__ __forceinline__ Place place_of(const Recurrence& r) {
  Place p;
  const int blocks = (r.channels + 64 * VEC - 1) / (64 * VEC);
  const unsigned at = seq::group_of_grid() * (blockDim.x / 64) + threadIdx.x / 64;
  const unsigned b = at / blocks;
  p.b = static_cast<int>(min(b, static_cast<unsigned>(r.batch)));
  const int first = static_cast<int>(at - b * blocks) *
                        64 * VEC +
                    (threadIdx.x & 63) * VEC;
  // (a row's last channels: see Group; what is before them is not stored)
  const seq::Group<VEC> group(first, r.channels);
  p.c = group.c;
  p.skip = group.skip;
  return p;
}

// The walk over a sequence.
template <typename T, int VEC, bool GATE>
__global__ void __launch_bounds__(256) recurrence_walk_kernel(Recurrence r) {
  typedef typename Pack<T, VEC>::type V;
  constexpr int kGroup = kSteps;
  const Place p = place_of<VEC>(r);
  if (p.b >= r.batch) return;
  const long row = static_cast<long>(p.b) * r.steps;
  const T* const f = static_cast<const T*>(r.f) + row * r.stride + p.c;
  const T* const x = static_cast<const T*>(r.x) + row * r.stride + p.c;
  const T* const ig = GATE ? static_cast<const T*>(r.i) + row * r.stride + p.c
                           : nullptr;
  T* const h = static_cast<T*>(r.out_h) + row * r.channels + p.c;
  const long state_at = static_cast<long>(p.b) * r.channels + p.c;
  const float* const from = r.first == nullptr ? nullptr : r.first + state_at;
  float state[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) state[k] = from == nullptr ? 0.f : from[k];
  const int end = length_of(r, p.b);
  for (int first = 0; first < end; first += kGroup) {
    V fv[kGroup], xv[kGroup], iv[kGroup];
    const unsigned long long resets = resets_of(r, row, first, kGroup, end);
    auto fresh = [&](int u) { return (resets >> u & 1) != 0; };
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      const int t = min(first + u, end - 1);
      fv[u] = *reinterpret_cast<const V*>(f + t * r.stride);
      xv[u] = *reinterpret_cast<const V*>(x + t * r.stride);
      if (GATE) iv[u] = *reinterpret_cast<const V*>(ig + t * r.stride);
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
          a = gate_of<T>(fs[k]);
          w = sigmoid_alone<T>(is[k]);
        } else {
          gate_of<T>(fs[k], &a, &w);
        }
        state[k] = w * xs[k] + (fresh(u) ? 0.f : a * state[k]);
      }
      put<T, VEC>(h + static_cast<long>(first + u) * r.channels, state, p.skip);
    }
  }
  float zero[VEC] = {};
  for (int t = end; t < r.steps; ++t)
    put<T, VEC>(h + static_cast<long>(t) * r.channels, zero, p.skip);
  if (r.last != nullptr)
    put<float, VEC>(r.last + state_at, state, p.skip);
}

// The gradients' walk over a sequence, from its end.
template <typename T, int VEC, bool GATE>
__global__ void __launch_bounds__(256) recurrence_grad_kernel(Recurrence r) {
  typedef typename Pack<T, VEC>::type V;
  constexpr int kGroup = kSteps;
  const Place p = place_of<VEC>(r);
  if (p.b >= r.batch) return;
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
  const float* const from = r.first == nullptr ? nullptr : r.first + state_at;
  float D[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) D[k] = from == nullptr ? 0.f : from[k];
  const int end = length_of(r, p.b);
  const float zero[VEC] = {};
  for (int t = end; t < r.steps; ++t) {
    put<T, VEC>(dx + t * r.grad_stride, zero, p.skip);
    put<T, VEC>(df + t * r.grad_stride, zero, p.skip);
    if (GATE) put<T, VEC>(di + t * r.grad_stride, zero, p.skip);
  }
  const int groups = (end + kGroup - 1) / kGroup;
  for (int g = groups - 1; g >= 0; --g) {
    V fv[kGroup], xv[kGroup], iv[kGroup], hv[kGroup], dv[kGroup];
    const int first = g * kGroup;
    const unsigned long long resets = resets_of(r, row, first, kGroup, end);
    auto fresh = [&](int u) { return (resets >> u & 1) != 0; };
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
        gate_of<T>(fs[k], &a, &rest);
        if (GATE) {
          sigmoid<T>(is[k], &w, &w_rest);
        } else {
          w = rest;
        }
        const float G = ds[k] + D[k];
        const float prior = fresh(u) ? 0.f : before[k];
        gx[k] = G * w;
        gf[k] = G * (GATE ? prior : prior - xs[k]) * (a * rest);
        if (GATE) gi[k] = G * xs[k] * (w * w_rest);
        D[k] = fresh(u) ? 0.f : a * G;
      }
      put<T, VEC>(dx + t * r.grad_stride, gx, p.skip);
      put<T, VEC>(df + t * r.grad_stride, gf, p.skip);
      if (GATE) put<T, VEC>(di + t * r.grad_stride, gi, p.skip);
    }
  }
  if (r.last != nullptr)
    put<float, VEC>(r.last + state_at, D, p.skip);
}

// ---- divided -----------------------------------------------------------------

// What the flag of a piece says: hints for those that wait, which take nothing
// but words that have arrived.  Not arrived: all bits set, which no value is
// published as.
enum : unsigned { kNothing = 0, kPair = 1, kState = 2 };
constexpr unsigned kNotYet = 0xFFFFFFFFu;

__device__ __forceinline__ unsigned published(float v) {
  const unsigned bits = __float_as_uint(v);
  return bits == kNotYet ? 0x7FC00000u : bits;  // (another NaN)
}
// Work-groups on other XCDs see these accesses without their L2s in between.
template <typename W>
__device__ __forceinline__ void publish(W* at, W v) {
  __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename W>
__device__ __forceinline__ W look(const W* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sets the counter and the flags to zero, the words to "not arrived".
__global__ void __launch_bounds__(256)
    recurrence_clear_kernel(unsigned* zeros, size_t n_zeros,
                            seq::Pack<unsigned, 4>::type* words,
                            size_t n_words) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n_zeros) zeros[i] = 0u;
  if (i < n_words)
    words[i] = seq::Pack<unsigned, 4>::type{kNotYet, kNotYet, kNotYet, kNotYet};
}

// The state in front of piece `piece` of a row of flags, by the wave that calls.
template <int VEC>
__device__ __forceinline__ void state_before(const Recurrence& r, long row,
                                             int piece, float (&state)[VEC]) {
  const int lane = threadIdx.x & 63;
  const long base = row * r.pieces;
  // The nearest of the 64 pieces before this one with a state, if all between
  // have pairs: lane l looks at the piece l + 1 before.
  int back;
  for (;;) {
    const int at = piece - 1 - lane;
    const unsigned flag = at >= 0 ? look(r.flags + base + at) : kNothing;
    const unsigned long long with_state = __ballot(flag == kState);
    const unsigned long long with_pair = __ballot(flag != kNothing);
    back = with_state == 0 ? 64 : __builtin_ctzll(with_state);
    const unsigned long long between = (1ull << (back & 63)) - 1;
    if (back < 64 && (with_pair & between) == between) break;
    __builtin_amdgcn_s_sleep(1);
  }
  const long word = static_cast<long>(lane) * VEC;
  const unsigned* const known =
      r.states + (base + piece - 1 - back) * (64 * VEC) + word;
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    unsigned v;
    while ((v = look(known + k)) == kNotYet) __builtin_amdgcn_s_sleep(1);
    state[k] = __uint_as_float(v);
  }
  // (four pieces' pairs are under way together)
  constexpr int kBatch = 4;
  for (int n = back; n > 0; n -= kBatch) {
    unsigned long long pair[kBatch][VEC];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        pair[u][k] = look(r.pairs + (base + piece - max(n - u, 1)) * (64 * VEC) +
                          word + k);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (n - u < 1) break;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        unsigned long long v = pair[u][k];
        while (v == ~0ull) {
          __builtin_amdgcn_s_sleep(1);
          v = look(r.pairs + (base + piece - (n - u)) * (64 * VEC) + word + k);
        }
        state[k] = composed(__uint_as_float(static_cast<unsigned>(v)),
                            __uint_as_float(static_cast<unsigned>(v >> 32)),
                            state[k]);
      }
    }
  }
}

// WAVES segments of L steps each are a piece.
template <typename T, int VEC, bool GATE, bool BACK, int WAVES, int L>
__global__ void __launch_bounds__(64 * WAVES)
    __attribute__((amdgpu_waves_per_eu(BACK ? 4 : 2)))
    recurrence_pass_kernel(Recurrence r) {
  typedef typename Pack<T, VEC>::type V;
  __shared__ unsigned handed_out;
  __shared__ float seg_a[WAVES][VEC][64], seg_s[WAVES][VEC][64];
  __shared__ float front[VEC][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (threadIdx.x == 0)
    handed_out = __hip_atomic_fetch_add(r.counter, 1u, __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const unsigned tile = __builtin_amdgcn_readfirstlane(handed_out);
  const int blocks = (r.channels + 64 * VEC - 1) / (64 * VEC);
  const unsigned rows = static_cast<unsigned>(r.batch) * blocks;
  const int piece = static_cast<int>(tile / rows);
  const unsigned row = tile - piece * rows;
  const int b = static_cast<int>(row / blocks);
  const int block = static_cast<int>(row - static_cast<unsigned>(b) * blocks);
  // (a row's last channels: see Group; lanes behind them store nothing)
  const seq::Group<VEC> group((block * 64 + lane) * VEC, r.channels);
  const int c = group.c, skip = group.skip;
  const int length = length_of(r, b);
  const int segment = piece * WAVES + wave;
  const int begin =
      segment >= r.segments
          ? r.steps
          : (BACK ? r.segments - 1 - segment : segment) * L;
  const int stop = min(begin + L, r.steps);  // the segment's end
  const int end = min(stop, length);         // ... of the steps that count

  // Rows are addressed by the wave (a scalar), channels by the lane's offset.
  const long at0 = static_cast<long>(b) * r.steps;
  const unsigned offset = static_cast<unsigned>(c) * sizeof(T);
  auto load = [&](const void* p, long stride, long t) {
    return *reinterpret_cast<const V*>(
        static_cast<const char*>(p) + (at0 + t) * stride * sizeof(T) + offset);
  };
  auto store = [&](void* p, long stride, long t, const float (&v)[VEC]) {
    put<T, VEC>(reinterpret_cast<T*>(static_cast<char*>(p) +
                                     (at0 + t) * stride * sizeof(T) + offset),
                v, skip);
  };
  auto step_of = [&](int u) { return min(begin + u, max(end, 1) - 1); };
  V fv[L], xv[L], iv[L], dv[L], hv[L];
  const unsigned long long resets = resets_of(r, at0, begin, L, end);
  auto fresh = [&](int u) { return (resets >> u & 1) != 0; };
#pragma unroll
  for (int u = 0; u < L; ++u) {
    const long t = step_of(u);
    fv[u] = load(r.f, r.stride, t);
    if (BACK) {
      dv[u] = load(r.dh, r.channels, t);
    } else {
      xv[u] = load(r.x, r.stride, t);
      if (GATE) iv[u] = load(r.i, r.stride, t);
    }
  }
  // Backwards what only the walk needs is loaded there, kLate steps at a time: held
  // from the start it takes the registers of a second work-group on the CU
  // (4 x 4096 x 2048 binary16: 175 -> 129 us).
  constexpr int kLate = 4;
  auto load_rest = [&](int u) {
    const long t = step_of(u);
    xv[u] = load(r.x, r.stride, t);
    if (GATE) iv[u] = load(r.i, r.stride, t);
    hv[u] = load(r.h, r.channels, max(t - 1, 0l));
  };

  // (A, S) of the segment.  Forward a_t and b_t are kept for the walk: working them
  // out again leaves room for more waves and is slower (32768 x 2048 bfloat16: 138
  // against 121 us).
  float A[VEC], S[VEC];
  float keep_a[BACK ? 1 : L][VEC], keep_b[BACK ? 1 : L][VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    A[k] = 1.f;
    S[k] = 0.f;
  }
#pragma unroll
  for (int n = 0; n < L; ++n) {
    const int u = BACK ? L - 1 - n : n;
    float fs[VEC], xs[VEC], is[VEC];
    unpack<T, VEC>(fv[u], fs);
    unpack<T, VEC>(BACK ? dv[u] : xv[u], xs);
    if (GATE && !BACK) unpack<T, VEC>(iv[u], is);
    const bool counts = begin + u < end;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      float a, w;
      if (BACK || GATE)
        a = gate_of<T>(fs[k]);
      else
        gate_of<T>(fs[k], &a, &w);
      if (BACK) {
        if (counts) {
          S[k] = fresh(u) ? 0.f : a * (xs[k] + S[k]);
          A[k] = fresh(u) ? -0.f : a * A[k];
        }
      } else {
        if (GATE) w = sigmoid_alone<T>(is[k]);
        const float add = w * xs[k];
        keep_a[u][k] = a;
        keep_b[u][k] = add;
        if (counts) {
          S[k] = add + (fresh(u) ? 0.f : a * S[k]);
          A[k] = fresh(u) ? -0.f : a * A[k];
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    A[k] = above_zero(A[k]);
    seg_a[wave][k][lane] = A[k];
    seg_s[wave][k][lane] = S[k];
  }
  __syncthreads();

  const long state_at = static_cast<long>(b) * r.channels + c;
  if (wave == 0) {
    // the piece's pair
#pragma unroll
    for (int w = 1; w < WAVES; ++w)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float a = seg_a[w][k][lane];
        S[k] = composed(a, seg_s[w][k][lane], S[k]);
        A[k] = is_reset(a) ? a : above_zero(a * A[k]);
      }
    const long place = static_cast<long>(row) * r.pieces + piece;
    const long word = place * (64 * VEC) + static_cast<long>(lane) * VEC;
    const bool others = piece + 1 < r.pieces;
    float state[VEC];
    if (piece == 0) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        state[k] = r.first == nullptr ? 0.f : r.first[state_at + k];
    } else {
      if (others) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          publish(r.pairs + word + k,
                  static_cast<unsigned long long>(published(A[k])) |
                      static_cast<unsigned long long>(published(S[k])) << 32);
        if (lane == 0) publish(r.flags + place, static_cast<unsigned>(kPair));
      }
      state_before<VEC>(r, row, piece, state);
    }
    if (others) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        publish(r.states + word + k, published(composed(A[k], S[k], state[k])));
      if (lane == 0) publish(r.flags + place, static_cast<unsigned>(kState));
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) front[k][lane] = state[k];
  }
  __syncthreads();
  float state[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) state[k] = front[k][lane];
  for (int w = 0; w < wave; ++w)
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      state[k] = composed(seg_a[w][k][lane], seg_s[w][k][lane], state[k]);

  // (Backwards the gates are worked out again: the barrier keeps the compiler from
  // holding them, which takes twice the registers of what they come from.)
  if (BACK) {
#pragma unroll
    for (int u = 0; u < L; ++u) {
      typedef typename Pack<unsigned, sizeof(V) / 4>::type Bits;
      Bits bits = __builtin_bit_cast(Bits, fv[u]);
      asm volatile("" : "+v"(bits));
      fv[u] = __builtin_bit_cast(V, bits);
    }
  }

  // the walk over the segment
  if (!BACK) {
#pragma unroll
    for (int u = 0; u < L; ++u) {
      const int t = begin + u;
      if (t < end) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          state[k] = keep_b[u][k] + (fresh(u) ? 0.f : keep_a[u][k] * state[k]);
        store(r.out_h, r.channels, t, state);
      } else if (t < stop) {
        const float zero[VEC] = {};
        store(r.out_h, r.channels, t, zero);
      }
    }
  } else {
#pragma unroll
    for (int u = L - 1; u >= 0; --u) {
      if ((L - 1 - u) % kLate == 0) {
#pragma unroll
        for (int q = 0; q < kLate; ++q)
          if (u - q >= 0) load_rest(u - q);
      }
      const int t = begin + u;
      float gx[VEC] = {}, gf[VEC] = {}, gi[VEC] = {};
      if (t < end) {
        float fs[VEC], xs[VEC], is[VEC], before[VEC], ds[VEC];
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
          gate_of<T>(fs[k], &a, &rest);
          if (GATE)
            sigmoid<T>(is[k], &w, &w_rest);
          else
            w = rest;
          const float G = ds[k] + state[k];
          const float prior = fresh(u) ? 0.f : before[k];
          gx[k] = G * w;
          gf[k] = G * (GATE ? prior : prior - xs[k]) * (a * rest);
          if (GATE) gi[k] = G * xs[k] * (w * w_rest);
          state[k] = fresh(u) ? 0.f : a * G;
        }
      }
      if (t < stop) {
        store(r.dx, r.grad_stride, t, gx);
        store(r.df, r.grad_stride, t, gf);
        if (GATE) store(r.di, r.grad_stride, t, gi);
      }
    }
  }
  // (behind the last segment there are none, or empty ones)
  if (r.last != nullptr && piece == r.pieces - 1 && wave == WAVES - 1)
    put<float, VEC>(r.last + state_at, state, skip);
}

// ---- the choice ----------------------------------------------------------------

// A piece: waves of a work-group, and the steps of a segment.  Longer pieces make a
// shorter chain of them, larger segments take registers from the waves of a CU.
// Forward, 32768 x 2048 bfloat16: 12 x 12 122 us, 16 x 8 126, 16 x 12 130, 8 x 16 135,
// 8 x 8 159, 12 x 16 170.  Gradients, 4 x 4096 x 2048 binary16: 16 x 8 132 us, 8 x 8
// 131, 16 x 4 137, 8 x 12 138, 12 x 12 144.  fp32, two channels a lane, is within a
// seventh of the best of these on four sizes: 32768 x 2048 188 us (8 x 16 170),
// gradients 320 (8 x 8 311); 8192 x 1024 33 (16 x 8 32) and 50 (16 x 4 55).
template <bool BACK>
constexpr int kWaves = BACK ? 16 : 12;
template <bool BACK>
constexpr int kSegment = BACK ? 8 : 12;

// A sequence is divided where there are fewer waves of lanes than this, and where
// it is long enough for the second launch.  bfloat16 of 1024 channels, four waves a
// sequence, us divided and whole, forward | gradients; in brackets with an input gate:
//
//   4 sequences of 32 steps    12, 10 |  12,  18
//   4 of 64                    13, 19 |  14,  32
//   64 of 66                   17, 26 |  20,  39
//   128 of 128                 33, 49 |  54,  93   (39,  67 |  62, 116)
//   128 of 512               119, 272 | 206, 357
//   256 of 128                 61, 78 | 102, 104   (73,  80 | 121, 135)
//   512 of 128               111, 101 | 187, 176  (133, 115 | 227, 231)
//   1000 of 128              205, 161 | 352, 318  (248, 214 | 433, 432)
//
// (by which the forward walk would be divided up to 1024 waves: its threshold is from
// kernels before these)
template <bool BACK>
constexpr int kWantedWaves = BACK ? 2048 : 512;
template <bool BACK>
constexpr int kLeastSteps = BACK ? 24 : 48;

struct Division {
  int segments, pieces;  // pieces == 0: undivided
  size_t rows, zeros, words, bytes;
};
template <typename T, bool BACK>
Division divide(const snn_hip_linear_recurrence_params& p) {
  Division d = {};
  constexpr int VEC = kVec<T>;
  d.rows = static_cast<size_t>(p.batch) * ceil_div(p.channels, 64 * VEC);
  d.segments = ceil_div(p.steps, kSegment<BACK>);
  if (p.channels < VEC || d.rows >= kWantedWaves<BACK> ||
      p.steps < kLeastSteps<BACK>)
    return d;
  const int pieces = ceil_div(d.segments, kWaves<BACK>);
  const size_t places = d.rows * pieces;
  if (!seq::grid_fits(places, 64 * kWaves<BACK>)) return d;
  d.pieces = pieces;
  // the counter and the flags, then the states and the pairs
  d.zeros = (places + 1 + 3) / 4 * 4;
  d.words = places * (64 * VEC) * 3;
  d.bytes = (d.zeros + d.words) * sizeof(unsigned);
  return d;
}

template <typename T, int VEC, bool GATE, bool BACK>
int launch_undivided(const Recurrence& r, hipStream_t stream) {
  const size_t waves =
      static_cast<size_t>(r.batch) * ceil_div(r.channels, 64 * VEC);
  const dim3 grid = seq::grid_of(ceil_div(waves, size_t{4})), threads(256);
  if (BACK)
    hipLaunchKernelGGL((recurrence_grad_kernel<T, VEC, GATE>), grid, threads, 0,
                       stream, r);
  else
    hipLaunchKernelGGL((recurrence_walk_kernel<T, VEC, GATE>), grid, threads, 0,
                       stream, r);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T, bool GATE, bool BACK>
int launch_divided(Recurrence r, const Division& d, void* workspace,
                   hipStream_t stream) {
  r.segments = d.segments;
  r.pieces = d.pieces;
  unsigned* const at = static_cast<unsigned*>(workspace);
  r.counter = at;
  r.flags = at + 1;
  r.states = at + d.zeros;
  const size_t slots = d.words / 3;
  r.pairs = reinterpret_cast<unsigned long long*>(r.states + slots);
  const size_t most = std::max(d.zeros, d.words / 4);
  hipLaunchKernelGGL(
      recurrence_clear_kernel,
      dim3(static_cast<unsigned>(ceil_div(most, size_t{256}))), dim3(256), 0,
      stream, at, d.zeros,
      reinterpret_cast<seq::Pack<unsigned, 4>::type*>(at + d.zeros),
      d.words / 4);
  SNN_HIP_CHECK_LAUNCH();
  hipLaunchKernelGGL(
      (recurrence_pass_kernel<T, kVec<T>, GATE, BACK, kWaves<BACK>,
                              kSegment<BACK>>),
      dim3(static_cast<unsigned>(d.rows * d.pieces)), dim3(64 * kWaves<BACK>), 0,
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
  KernelTimer timer(stream);
  const Division d = divide<T, BACK>(p);
  if (d.pieces > 0 && workspace != nullptr && elems * sizeof(T) >= d.bytes) {
    return r.i != nullptr
               ? launch_divided<T, true, BACK>(r, d, workspace, stream)
               : launch_divided<T, false, BACK>(r, d, workspace, stream);
  }
  constexpr int VEC = kVec<T>;
  if (p.channels >= VEC)
    return r.i != nullptr ? launch_undivided<T, VEC, true, BACK>(r, stream)
                          : launch_undivided<T, VEC, false, BACK>(r, stream);
  return r.i != nullptr ? launch_undivided<T, 1, true, BACK>(r, stream)
                        : launch_undivided<T, 1, false, BACK>(r, stream);
}

template <typename T>
size_t workspace_bytes(const snn_hip_linear_recurrence_params& p) {
  return std::max(divide<T, false>(p).bytes, divide<T, true>(p).bytes);
}

int check_recurrence(const snn_hip_linear_recurrence_params* p,
                     const void* workspace) {
  if (p == nullptr) return SNN_HIP_INVALID_PARAMETER;
  SNN_REQUIRE(p->batch > 0 && p->steps > 0 && p->channels > 0);
  SNN_REQUIRE(p->row_stride == 0 || p->row_stride >= p->channels);
  SNN_REQUIRE(p->grad_row_stride == 0 || p->grad_row_stride >= p->channels);
  SNN_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0);
  // (waves, and steps and channels of a group behind the last one, are counted in 31
  // bits)
  if (static_cast<size_t>(p->batch) * ceil_div(p->channels, 64) > INT_MAX ||
      p->steps > INT_MAX - 64 || p->channels > INT_MAX - 1024)
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
  *required_elems = 0;
  *recommended_elems = dtype == SNN_HIP_DTYPE_F32
                           ? snn::workspace_bytes<float>(*params) / 4
                           : snn::workspace_bytes<_Float16>(*params) / 2;
  return SNN_HIP_OK;
}

}  // extern "C"
