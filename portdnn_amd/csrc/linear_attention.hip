// The entry points of linear attention (the walks over blocks of steps:
// linear_attention.h), the walk over a few steps and the sums along pieces.
#include <algorithm>
#include <cmath>

#include "linear_attention.h"

namespace snn {
namespace {

using att::Problem;
using att::Walk;
using seq::Pack;

// ---- a few steps ---------------------------------------------------------------

// (bfloat16, 64 sequences of 16 heads of 128 x 128, call after call on the same states,
// which are partly in the last cache: 1 step 22 us, 4 29, 12 48, 16 59; 17 steps in a block
// 50)
constexpr int kFewSteps = 12;

struct Few {
  const void *q, *k, *v;
  void* out;
  long q_row, k_row, v_row;
  int batch, heads, share, steps, keys, values, slices;
  const float* decay;
  const unsigned char* resets;
  const int* lengths;
  const float* initial;
  float* final;
  float scale;
};

// One step after the other, all in fp32: a work-group owns 64 values of a head's
// state, a lane four neighbouring values of every sixteenth key.  Bound by the state,
// which is read and written once: one step of 64 sequences of 16 heads of 128 x 128, among
// other calls, in 27.5 us, 135 MB, 4.9 TB/s.
template <typename T, int R>
__global__ void __launch_bounds__(256) few_steps_kernel(Few p) {
  __shared__ float q_of[kFewSteps][16 * R], k_of[kFewSteps][16 * R];
  __shared__ float sums[kFewSteps][4][64];
  typedef Pack<float, 4>::type F;
  const unsigned at = seq::group_of_grid();
  const unsigned bh = at / p.slices, slice = at - bh * p.slices;
  const unsigned b = bh / p.heads, h = bh - b * p.heads;
  if (b >= static_cast<unsigned>(p.batch)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int first_key = tid / 16;
  const int col = slice * 64 + tid % 16 * 4;
  const int cols = max(0, min(4, p.values - col));
  const long row = static_cast<long>(b) * p.steps;
  const long state_at =
      static_cast<long>(bh) * p.keys * p.values + min(col, p.values - 1);
  const int length = p.lengths == nullptr
                         ? p.steps
                         : max(0, min(p.steps, p.lengths[b]));

  float state[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int key = first_key + 16 * i;
#pragma unroll
    for (int c = 0; c < 4; ++c) state[i][c] = 0.f;
    if (p.initial != nullptr && key < p.keys) {
      const float* const from =
          p.initial + state_at + static_cast<long>(key) * p.values;
      if (cols == 4) {
        const F f = *reinterpret_cast<const F*>(from);
#pragma unroll
        for (int c = 0; c < 4; ++c) state[i][c] = f[c];
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (c < cols) state[i][c] = from[c];
      }
    }
  }
  const T* const q = static_cast<const T*>(p.q) + row * p.q_row +
                     static_cast<long>(h / p.share) * p.keys;
  const T* const k = static_cast<const T*>(p.k) + row * p.k_row +
                     static_cast<long>(h / p.share) * p.keys;
  const T* const v = static_cast<const T*>(p.v) + row * p.v_row +
                     static_cast<long>(h) * p.values + col;
  for (int e = tid; e < length * 16 * R; e += 256) {
    const int t = e / (16 * R), key = e % (16 * R);
    const bool in = key < p.keys;
    q_of[t][key] = in ? static_cast<float>(q[t * p.q_row + key]) : 0.f;
    k_of[t][key] = in ? static_cast<float>(k[t * p.k_row + key]) : 0.f;
  }
  // (above zero, as in the walks over blocks)
  const float a = expf(att::log_decay(p.decay, h)) + 0x1p-126f;
  __syncthreads();
  for (int t = 0; t < length; ++t) {
    float x[4] = {};
    const T* const from = v + t * p.v_row;
    if (cols == 4) {
      seq::unpack<T, 4>(
          *reinterpret_cast<const typename Pack<T, 4>::type*>(from), x);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c < cols) x[c] = static_cast<float>(from[c]);
    }
    const bool fresh = p.resets != nullptr && p.resets[row + t] != 0;
    float sum[4] = {};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float key = k_of[t][first_key + 16 * i];
      const float query = q_of[t][first_key + 16 * i];
      // (keys that do not exist hold zeros, also beside an infinite v)
      const bool in = first_key + 16 * i < p.keys;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float now = key * x[c] + (fresh ? 0.f : a * state[i][c]);
        state[i][c] = in ? now : 0.f;
        sum[c] += query * state[i][c];
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      sum[c] += __shfl_xor(sum[c], 16);
      sum[c] += __shfl_xor(sum[c], 32);
      if (lane < 16) sums[t][wave][lane * 4 + c] = sum[c];
    }
  }
  __syncthreads();
  T* const out = static_cast<T*>(p.out) +
                 (row * p.heads + h) * static_cast<long>(p.values) + slice * 64;
  for (int e = tid; e < p.steps * 64; e += 256) {
    const int t = e / 64, c = e % 64;
    if (static_cast<int>(slice * 64) + c >= p.values) continue;
    float s = 0.f;
    if (t < length) {
#pragma unroll
      for (int u = 0; u < 4; ++u) s += sums[t][u][c];
    }
    out[t * static_cast<long>(p.heads) * p.values + c] =
        static_cast<T>(s * p.scale);
  }
  if (p.final == nullptr) return;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int key = first_key + 16 * i;
    if (key >= p.keys) continue;
    float* const to = p.final + state_at + static_cast<long>(key) * p.values;
    if (cols == 4) {
      *reinterpret_cast<F*>(to) =
          F{state[i][0], state[i][1], state[i][2], state[i][3]};
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c < cols) to[c] = state[i][c];
    }
  }
}

template <typename T>
int run_few(const Few& f, hipStream_t stream) {
  const dim3 grid = seq::grid_of(static_cast<size_t>(f.batch) * f.heads *
                                 f.slices);
  if (f.keys <= 64)
    hipLaunchKernelGGL((few_steps_kernel<T, 4>), grid, dim3(256), 0, stream, f);
  else if (f.keys <= 128)
    hipLaunchKernelGGL((few_steps_kernel<T, 8>), grid, dim3(256), 0, stream, f);
  else
    hipLaunchKernelGGL((few_steps_kernel<T, 16>), grid, dim3(256), 0, stream, f);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

// ---- along the pieces ------------------------------------------------------------

// The pieces' own states become the states in front of them, in the walk's order: each
// lane has one of a state's values and adds the pieces up, eight under way at once.  It
// waits for memory: 10 us for 16 pieces of 16 heads of 128 x 128, 34 MB read and
// written; 18 us with one under way.
struct Chain {
  float* states;
  const int* carries;
  const float* initial;
};
struct Chains {
  Chain chain[2];
  int heads, pieces, piece_steps, steps;
  long size;  // of a state
  const float* decay;
  const int* lengths;
};
constexpr int kChained = 8;  // pieces under way at once
__global__ void __launch_bounds__(256) chain_kernel(Chains p) {
  const Chain& c = p.chain[blockIdx.z];
  const int bh = blockIdx.y;
  const long at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= p.size) return;
  const int b = bh / p.heads, h = bh - b * p.heads;
  const int length = p.lengths == nullptr
                         ? p.steps
                         : max(0, min(p.steps, p.lengths[b]));
  const float log_a = att::log_decay(p.decay, h);
  const float whole = expf(p.piece_steps * log_a) + 0x1p-126f;
  float state = c.initial == nullptr ? 0.f : c.initial[bh * p.size + at];
  float* to = c.states + static_cast<long>(bh) * p.pieces * p.size + at;
  const int* const carries = c.carries + static_cast<long>(bh) * p.pieces;
  // (the last piece has left no state of its own, and those behind it none at all)
  const int on = length == 0 ? 0 : (length - 1) / p.piece_steps;
  for (int first = 0; first <= on; first += kChained, to += kChained * p.size) {
    float own[kChained];
    bool carried[kChained];
#pragma unroll
    for (int i = 0; i < kChained; ++i) {
      const int piece = min(first + i, on);
      own[i] = piece < on ? to[(piece - first) * p.size] : 0.f;
      carried[i] = piece < on && carries[piece] != 0;
    }
#pragma unroll
    for (int i = 0; i < kChained; ++i) {
      if (first + i > on) break;
      to[i * p.size] = state;
      state = (carried[i] ? whole * state : 0.f) + own[i];
    }
  }
}

// ---- gradients of shared heads ---------------------------------------------------

// out[row][g][c] = sum over the group's heads of in[row][g * share + i][c], VEC
// neighbouring c at a time, for q's and k's gradients beside one another.  Bound by
// memory: bfloat16, 4 x 4096 steps of 16 heads of 128 channels, four of which share: 51
// us for both, 302 MB, partly from the last cache (51 for each, one value at a time), of
// 309 for the call; 240 where no heads share.
struct Shared {
  const float* in[2];
  void* out[2];
  long out_row[2];
  size_t rows;
  int groups, share, keys;
};
template <typename T, int VEC>
__global__ void __launch_bounds__(256) share_kernel(Shared p) {
  const bool second = blockIdx.y != 0;
  const float* const in = p.in[second];
  T* const out = static_cast<T*>(p.out[second]);
  const long out_row = p.out_row[second];
  const unsigned pieces = static_cast<unsigned>(p.keys) / VEC;
  const unsigned units = static_cast<unsigned>(p.groups) * pieces;
  // (a lane's place goes on by the same rows and units of a row each time)
  const size_t first = blockIdx.x * size_t{256} + threadIdx.x;
  const size_t all = gridDim.x * size_t{256};
  size_t row = first / units;
  unsigned unit = static_cast<unsigned>(first - row * units);
  const size_t on_rows = all / units;
  const unsigned on_units = static_cast<unsigned>(all - on_rows * units);
  while (row < p.rows) {
    const unsigned g = unit / pieces, c = (unit - g * pieces) * VEC;
    const float* const from =
        in + ((row * p.groups + g) * p.share) * p.keys + c;
    float sum[VEC] = {};
    for (int i = 0; i < p.share; ++i) {
      float x[VEC];
      seq::unpack<float, VEC>(*reinterpret_cast<const typename Pack<float, VEC>::type*>(
                                  from + static_cast<long>(i) * p.keys),
                              x);
#pragma unroll
      for (int u = 0; u < VEC; ++u) sum[u] += x[u];
    }
    *reinterpret_cast<typename Pack<T, VEC>::type*>(
        out + row * out_row + static_cast<long>(g) * p.keys + c) =
        seq::pack<T, VEC>(sum);
    row += on_rows;
    unit += on_units;
    if (unit >= units) {
      unit -= units;
      ++row;
    }
  }
}

// ---- entry points ------------------------------------------------------------------

int check(const snn_hip_linear_attention_params* p, const void* workspace) {
  if (p == nullptr) return SNN_HIP_INVALID_PARAMETER;
  SNN_REQUIRE(p->batch > 0 && p->steps > 0 && p->heads > 0 &&
              p->key_heads > 0 && p->keys > 0 && p->values > 0);
  SNN_REQUIRE(p->heads % p->key_heads == 0);
  SNN_REQUIRE(p->keys <= 256 && p->values <= 256);
  SNN_REQUIRE(std::isfinite(p->scale));
  const long of_keys = static_cast<long>(p->key_heads) * p->keys;
  const long of_values = static_cast<long>(p->heads) * p->values;
  auto stride_ok = [](int stride, long row) {
    return stride == 0 || stride >= row;
  };
  SNN_REQUIRE(stride_ok(p->q_stride, of_keys) && stride_ok(p->k_stride, of_keys) &&
              stride_ok(p->v_stride, of_values));
  SNN_REQUIRE(stride_ok(p->grad_q_stride, of_keys) &&
              stride_ok(p->grad_k_stride, of_keys) &&
              stride_ok(p->grad_v_stride, of_values));
  SNN_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0);
  // (steps and places of pieces are counted in 31 bits, a block's rows in 31 bits of
  // bytes)
  const size_t heads = static_cast<size_t>(p->batch) * p->heads;
  constexpr int kStride = 1 << 22;
  if (p->steps > (1 << 30) || heads > (1u << 20) || of_keys > kStride ||
      of_values > kStride || p->q_stride > kStride || p->k_stride > kStride ||
      p->v_stride > kStride || p->grad_q_stride > kStride ||
      p->grad_k_stride > kStride || p->grad_v_stride > kStride)
    return SNN_HIP_INDEX_EXCEEDED;
  return SNN_HIP_OK;
}
// ... and of the gradients: where heads share queries and keys, a row of their fp32
// sums is that of all heads, and a block's rows of them are counted in 31 bits of
// bytes as well.
int check_grad(const snn_hip_linear_attention_params* p, const void* workspace) {
  const int valid = check(p, workspace);
  if (valid != SNN_HIP_OK) return valid;
  constexpr long kMostSums = 1 << 23;
  static_assert(63 * kMostSums * 4 + 1024 < 0x7FFFFFF0l, "beyond a buffer's range");
  if (p->heads != p->key_heads &&
      static_cast<long>(p->heads) * p->keys > kMostSums)
    return SNN_HIP_INDEX_EXCEEDED;
  return SNN_HIP_OK;
}

long or_else(int stride, long row) { return stride == 0 ? row : stride; }
size_t round16(size_t bytes) { return (bytes + 15) / 16 * 16; }
int block_of(int elem_size) { return elem_size == 2 ? 64 : 32; }
int class_of(int keys) { return keys <= 64 ? 64 : keys <= 128 ? 128 : 256; }

// Waves of a work-group, 16 values each, and the work-groups that share the values.
// With eight, q, k and their products serve twice as many values.  (us, four and eight:
// bfloat16, 1 x 32768 steps of 16 heads of 128 x 128 258, 219, gradients of 4 x 4096
// steps 339, 256; 1 x 8192 steps of 16 heads of 256 x 256 266, 199, gradients 634, 510.
// In fp32 a block of 32 steps has four tiles of q k, one for each of four waves.)
int waves_of(int size, int values) {
  return size == 2 && values > 64 ? 8 : 4;
}
int slices_of(int size, int values) {
  return ceil_div(values, 16 * waves_of(size, values));
}

// How a sequence is divided into pieces that are walked beside one another: as this
// estimate says, in times of a block, where the work-groups of a CU wait for one another.
// A piece costs four blocks for its states.  Work-groups of eight waves, or with states
// of more than 128 keys, have a CU to themselves; of the others up to three share one,
// and each further one takes 0.4 of the first's time.  The walk that leaves only states
// takes 0.4 of one with outputs; it and the chain behind it cost their launches.
// (us for 1, 2, 4, 8, 16, 32 pieces; * is what is taken.  bfloat16, 1 x 32768 steps of
// 16 heads of 128 x 128: 1787, 1311, 663, 349, 222*, 248; gradients of 4 x 4096 steps
// of such heads: 237*, 325, 304, 349, 461, 643; 1 x 16384 steps of 16 heads of 64 x 64:
// 638, 490, 253, 134, 79, 60*; 1 x 8192 steps of 16 heads of 256 x 256: 759, 603, 335,
// 202*, 221, 275.  fp32, 1 x 8192 steps of 8 heads of 128 x 128: 1007, 774, 396, 208,
// 121, 103*)
struct Division {
  int pieces, piece_steps;
};
constexpr int kCus = 256, kMostPieces = 128;
double rounds_of(size_t groups, int of_cu) {
  const size_t each = (groups + kCus - 1) / kCus;  // for the CU that has most
  const size_t rest = each % of_cu;
  return each / of_cu * (0.6 + 0.4 * of_cu) + (rest == 0 ? 0. : 0.6 + 0.4 * rest);
}
Division divide(const snn_hip_linear_attention_params& p, int units, int block,
                int of_cu, size_t bytes, int states) {
  const int blocks = ceil_div(p.steps, block);
  const size_t heads = static_cast<size_t>(p.batch) * p.heads;
  auto need = [&](int pieces) {
    return states * (round16(heads * pieces * p.keys * p.values * sizeof(float)) +
                     round16(heads * pieces * sizeof(int)));
  };
  Division best = {1, blocks * block};
  double least = rounds_of(heads * units, of_cu) * (blocks + 4);
  // (many work-groups fill the GPU evenly enough, and pieces would take half as long again
  // and more.  us for 1, 2, 4 pieces: bfloat16, 64 x 1024 steps of 32 heads of 64 x 64 263,
  // 418, 474; 128 x 1024 of 16 heads of 128 x 128 630, 1148, 1409, gradients of 48 x 512
  // 346, 709, 906; fp32, 64 x 256 of 16 heads of 128 x 128 227, 493, 574)
  const int most = heads * units >= 8 * kCus ? 1 : std::min(blocks, kMostPieces);
  for (int want = 2; want <= most; ++want) {
    const int each = ceil_div(blocks, want), pieces = ceil_div(blocks, each);
    if (pieces != want || need(pieces) > bytes) continue;
    // (of the gradients' three walks two leave states)
    const size_t all = heads * units * pieces;
    const double time =
        (rounds_of(all, of_cu) + 0.4 * rounds_of(states == 1 ? all : all * 2 / 3, of_cu)) *
            (each + 4) + 2 + pieces / 16.;
    if (time < least) {
      least = time;
      best = {pieces, each * block};
    }
  }
#ifdef SNN_HIP_TUNING
  if (const char* want = std::getenv("SNN_HIP_ATT_PIECES")) {
    const int each = ceil_div(blocks, std::max(1, std::min(std::atoi(want), blocks)));
    best = {ceil_div(blocks, each), each * block};
    if (best.pieces == 1 || need(best.pieces) > bytes) best = {1, blocks * block};
  }
#endif
  return best;
}
size_t division_bytes(const snn_hip_linear_attention_params& p,
                      const Division& d, int states) {
  if (d.pieces == 1) return 0;
  const size_t heads = static_cast<size_t>(p.batch) * p.heads * d.pieces;
  return states * (round16(heads * p.keys * p.values * sizeof(float)) +
                   round16(heads * sizeof(int)));
}

// Work-groups of a pass over the whole sequence, and how many of them share a CU.
int forward_units(const snn_hip_linear_attention_params& p, int size) {
  return slices_of(size, p.values);
}
int grad_units(const snn_hip_linear_attention_params& p, int size) {
  return 2 * slices_of(size, p.keys) + slices_of(size, p.values);
}
Division forward_division(const snn_hip_linear_attention_params& p, int size,
                          size_t bytes) {
  const bool alone =
      class_of(p.keys) == 256 || waves_of(size, p.values) == 8;
  return divide(p, forward_units(p, size), block_of(size), alone ? 1 : 3, bytes, 1);
}
Division grad_division(const snn_hip_linear_attention_params& p, int size,
                       size_t bytes) {
  const bool alone =
      class_of(std::max(p.keys, p.values)) == 256 ||
      waves_of(size, p.values) == 8 || waves_of(size, p.keys) == 8;
  return divide(p, grad_units(p, size), block_of(size), alone ? 1 : 3, bytes, 2);
}

// fp32 gradients of q and k by heads, where heads share them.
size_t shared_bytes(const snn_hip_linear_attention_params& p) {
  return p.heads == p.key_heads
             ? 0
             : round16(static_cast<size_t>(p.batch) * p.steps * p.heads *
                       p.keys * sizeof(float));
}

template <typename T>
int run_class(const Problem& p, int keys_class, int waves, bool outputs,
              hipStream_t stream) {
  const size_t groups =
      static_cast<size_t>(p.units) * p.batch * p.heads * p.pieces;
  if (!seq::grid_fits(groups, 64 * waves)) return SNN_HIP_INDEX_EXCEEDED;
  if (std::is_same<T, float>::value)
    return att::run_walks_f32(p, keys_class, waves, outputs, stream);
  if (std::is_same<T, _Float16>::value)
    return att::run_walks_f16(p, keys_class, waves, outputs, stream);
  return att::run_walks_bf16(p, keys_class, waves, outputs, stream);
}

Problem problem_of(const snn_hip_linear_attention_params& p, const Division& d,
                   const float* decay, const unsigned char* resets,
                   const int* lengths) {
  Problem g = {};
  g.batch = p.batch;
  g.heads = p.heads;
  g.steps = p.steps;
  g.pieces = d.pieces;
  g.piece_steps = d.piece_steps;
  g.decay = decay;
  g.resets = resets;
  g.lengths = lengths;
  return g;
}
void add(Problem* g, const Walk& w, int size) {
  g->walk[g->walks] = w;
  g->walk[g->walks].slices = slices_of(size, w.values);
  g->units += g->walk[g->walks].slices;
  ++g->walks;
}
// Walks of one class of keys and one width of slices go together.
template <typename T>
int run_all(const Problem& base, const Walk* walks, int n, bool outputs,
            hipStream_t stream) {
  bool done[att::kMostWalks] = {};
  for (int i = 0; i < n; ++i) {
    if (done[i]) continue;
    const int keys = class_of(walks[i].keys);
    const int waves = waves_of(sizeof(T), walks[i].values);
    Problem g = base;
    for (int j = i; j < n; ++j) {
      if (done[j] || class_of(walks[j].keys) != keys ||
          waves_of(sizeof(T), walks[j].values) != waves)
        continue;
      add(&g, walks[j], sizeof(T));
      done[j] = true;
    }
    const int s = run_class<T>(g, keys, waves, outputs, stream);
    if (s != SNN_HIP_OK) return s;
  }
  return SNN_HIP_OK;
}
// The states in front of the pieces of one or two walks.
template <typename T>
int run_pieces(const snn_hip_linear_attention_params& p, const Problem& base,
               const Walk* walks, int n, hipStream_t stream) {
  const int s = run_all<T>(base, walks, n, false, stream);
  if (s != SNN_HIP_OK) return s;
  Chains c = {};
  for (int i = 0; i < n; ++i)
    c.chain[i] = {walks[i].states, walks[i].carries, walks[i].initial};
  c.heads = p.heads;
  c.pieces = base.pieces;
  c.piece_steps = base.piece_steps;
  c.steps = p.steps;
  c.size = static_cast<long>(p.keys) * p.values;
  c.decay = base.decay;
  c.lengths = base.lengths;
  hipLaunchKernelGGL(
      chain_kernel,
      dim3(static_cast<unsigned>(ceil_div(static_cast<size_t>(c.size), size_t{256})),
           static_cast<unsigned>(p.batch) * p.heads, static_cast<unsigned>(n)),
      dim3(256), 0, stream, c);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}
// Places of a walk's states and carries.
char* place_states(const snn_hip_linear_attention_params& p, int pieces,
                   char* at, Walk* w) {
  const size_t heads = static_cast<size_t>(p.batch) * p.heads * pieces;
  w->states = reinterpret_cast<float*>(at);
  at += round16(heads * p.keys * p.values * sizeof(float));
  w->carries = reinterpret_cast<int*>(at);
  return at + round16(heads * sizeof(int));
}

template <typename T>
int forward(const void* q, const void* k, const void* v, const float* decay,
            const unsigned char* resets, const int* lengths,
            const float* initial, void* output, float* final,
            const snn_hip_linear_attention_params* params, void* workspace,
            size_t elems, void* stream_arg) {
  const int valid = check(params, workspace);
  if (valid != SNN_HIP_OK) return valid;
  const snn_hip_linear_attention_params& p = *params;
  SNN_REQUIRE(q != nullptr && k != nullptr && v != nullptr && decay != nullptr &&
              output != nullptr);
  const hipStream_t stream = as_stream(stream_arg);
  const long of_keys = static_cast<long>(p.key_heads) * p.keys;
  const long of_values = static_cast<long>(p.heads) * p.values;
  KernelTimer timer(stream);
  if (p.steps <= kFewSteps) {
    Few f = {};
    f.q = q;
    f.k = k;
    f.v = v;
    f.out = output;
    f.q_row = or_else(p.q_stride, of_keys);
    f.k_row = or_else(p.k_stride, of_keys);
    f.v_row = or_else(p.v_stride, of_values);
    f.batch = p.batch;
    f.heads = p.heads;
    f.share = p.heads / p.key_heads;
    f.steps = p.steps;
    f.keys = p.keys;
    f.values = p.values;
    f.slices = ceil_div(p.values, 64);
    f.decay = decay;
    f.resets = resets;
    f.lengths = lengths;
    f.initial = initial;
    f.final = final;
    f.scale = p.scale;
    return run_few<T>(f, stream);
  }
  Walk w = {};
  w.q = q;
  w.k = k;
  w.v = v;
  w.out = output;
  w.q_row = or_else(p.q_stride, of_keys);
  w.k_row = or_else(p.k_stride, of_keys);
  w.v_row = or_else(p.v_stride, of_values);
  w.out_row = of_values;
  w.q_share = w.k_share = p.heads / p.key_heads;
  w.v_share = 1;
  w.keys = p.keys;
  w.values = p.values;
  w.initial = initial;
  w.final = final;
  w.weight = p.scale;
  w.reach_weight = p.scale;
  w.state_weight = 1.f;
  const Division d =
      forward_division(p, sizeof(T), workspace == nullptr ? 0 : elems * sizeof(T));
  const Problem base = problem_of(p, d, decay, resets, lengths);
  if (d.pieces > 1) {
    place_states(p, d.pieces, static_cast<char*>(workspace), &w);
    const int s = run_pieces<T>(p, base, &w, 1, stream);
    if (s != SNN_HIP_OK) return s;
  }
  return run_all<T>(base, &w, 1, true, stream);
}

template <typename T>
int share_sums(const snn_hip_linear_attention_params& p, const float* q_sums,
               void* grad_q, const float* k_sums, void* grad_k, hipStream_t stream) {
  const long width = static_cast<long>(p.key_heads) * p.keys;
  Shared g = {};
  unsigned n = 0;
  auto add = [&](const float* in, void* out, int stride) {
    if (in == nullptr) return;
    g.in[n] = in;
    g.out[n] = out;
    g.out_row[n++] = or_else(stride, width);
  };
  add(q_sums, grad_q, p.grad_q_stride);
  add(k_sums, grad_k, p.grad_k_stride);
  g.rows = static_cast<size_t>(p.batch) * p.steps;
  g.groups = p.key_heads;
  g.share = p.heads / p.key_heads;
  g.keys = p.keys;
  const int vec = p.keys % 4 == 0 ? 4 : 1;
  const dim3 grid(static_cast<unsigned>(std::min<size_t>(
                      ceil_div(g.rows * static_cast<size_t>(width) / vec,
                               size_t{256}),
                      4096)),
                  n);
  if (n == 0) return SNN_HIP_OK;
  if (vec == 4)
    hipLaunchKernelGGL((share_kernel<T, 4>), grid, dim3(256), 0, stream, g);
  else
    hipLaunchKernelGGL((share_kernel<T, 1>), grid, dim3(256), 0, stream, g);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T>
int backward(const void* grad, const float* grad_final, const void* q,
             const void* k, const void* v, const float* decay,
             const unsigned char* resets, const int* lengths,
             const float* initial, void* grad_q, void* grad_k, void* grad_v,
             float* grad_initial, const snn_hip_linear_attention_params* params,
             void* workspace, size_t elems, void* stream_arg) {
  const int valid = check_grad(params, workspace);
  if (valid != SNN_HIP_OK) return valid;
  const snn_hip_linear_attention_params& p = *params;
  SNN_REQUIRE(grad != nullptr && q != nullptr && k != nullptr && v != nullptr &&
              decay != nullptr);
  SNN_REQUIRE(grad_q != nullptr || grad_k != nullptr || grad_v != nullptr ||
              grad_initial != nullptr);
  const hipStream_t stream = as_stream(stream_arg);
  const long of_keys = static_cast<long>(p.key_heads) * p.keys;
  const long of_values = static_cast<long>(p.heads) * p.values;
  const int share = p.heads / p.key_heads;
  const size_t each = shared_bytes(p);
  const size_t shared = each * ((grad_q != nullptr) + (grad_k != nullptr));
  const size_t bytes = workspace == nullptr ? 0 : elems * sizeof(T);
  if (bytes < shared) return SNN_HIP_INSUFFICIENT_WORKSPACE;
  char* at = static_cast<char*>(workspace);
  float *q_sums = nullptr, *k_sums = nullptr;
  if (each > 0 && grad_q != nullptr) {
    q_sums = reinterpret_cast<float*>(at);
    at += each;
  }
  if (each > 0 && grad_k != nullptr) {
    k_sums = reinterpret_cast<float*>(at);
    at += each;
  }
  const long q_row = or_else(p.q_stride, of_keys);
  const long k_row = or_else(p.k_stride, of_keys);
  const long v_row = or_else(p.v_stride, of_values);

  Walk of_q = {}, of_k = {}, of_v = {}, front = {};
  of_q.q = grad;
  of_q.q_row = of_values;
  of_q.q_share = 1;
  of_q.k = v;
  of_q.k_row = v_row;
  of_q.k_share = 1;
  of_q.v = k;
  of_q.v_row = k_row;
  of_q.v_share = share;
  of_q.keys = p.values;
  of_q.values = p.keys;
  of_q.initial = initial;
  of_q.transposed = 1;
  of_q.weight = of_q.reach_weight = p.scale;
  of_q.state_weight = 1.f;

  of_k.q = v;
  of_k.q_row = v_row;
  of_k.q_share = 1;
  of_k.k = grad;
  of_k.k_row = of_values;
  of_k.k_share = 1;
  of_k.v = q;
  of_k.v_row = q_row;
  of_k.v_share = share;
  of_k.keys = p.values;
  of_k.values = p.keys;
  of_k.initial = grad_final;
  of_k.transposed = 1;
  of_k.from_end = 1;
  of_k.weight = of_k.state_weight = p.scale;
  of_k.reach_weight = 1.f;

  of_v.q = k;
  of_v.q_row = k_row;
  of_v.q_share = share;
  of_v.k = q;
  of_v.k_row = q_row;
  of_v.k_share = share;
  of_v.v = grad;
  of_v.v_row = of_values;
  of_v.v_share = 1;
  of_v.out = grad_v;
  of_v.out_row = or_else(p.grad_v_stride, of_values);
  of_v.keys = p.keys;
  of_v.values = p.values;
  of_v.initial = grad_final;
  of_v.final = grad_initial;
  of_v.from_end = 1;
  of_v.weight = of_v.state_weight = p.scale;
  of_v.reach_weight = 1.f;

  auto output = [&](Walk* w, void* out, int stride, float* sums) {
    w->out = sums != nullptr ? sums : out;
    w->out_float = sums != nullptr;
    w->out_row = sums != nullptr ? static_cast<long>(p.heads) * p.keys
                                 : or_else(stride, of_keys);
  };
  output(&of_q, grad_q, p.grad_q_stride, q_sums);
  output(&of_k, grad_k, p.grad_k_stride, k_sums);

  KernelTimer timer(stream);
  const Division d = grad_division(p, sizeof(T), bytes - shared);
  const Problem base = problem_of(p, d, decay, resets, lengths);
  if (d.pieces > 1) {
    // the states from the front, as the forward pass has them, and from the end
    front = {};
    front.k = k;
    front.k_row = k_row;
    front.k_share = share;
    front.v = v;
    front.v_row = v_row;
    front.v_share = 1;
    front.q_share = 1;
    front.keys = p.keys;
    front.values = p.values;
    front.initial = initial;
    front.state_weight = 1.f;
    at = place_states(p, d.pieces, at, &front);
    place_states(p, d.pieces, at, &of_v);
    of_q.states = front.states;
    of_k.states = of_v.states;
    Walk both[2];
    int n = 0;
    if (grad_q != nullptr) both[n++] = front;
    if (grad_k != nullptr || grad_v != nullptr || grad_initial != nullptr)
      both[n++] = of_v;
    const int s = run_pieces<T>(p, base, both, n, stream);
    if (s != SNN_HIP_OK) return s;
  }
  Walk walks[att::kMostWalks];
  int n = 0;
  if (grad_q != nullptr) walks[n++] = of_q;
  if (grad_k != nullptr) walks[n++] = of_k;
  if (grad_v != nullptr || grad_initial != nullptr) walks[n++] = of_v;
  int s = run_all<T>(base, walks, n, true, stream);
  if (s == SNN_HIP_OK) s = share_sums<T>(p, q_sums, grad_q, k_sums, grad_k, stream);
  return s;
}

}  // namespace
}  // namespace snn

namespace snn {
namespace {

// The launches that run_all makes of walks over these keys and values.
struct Sizes {
  int keys, values;
};
void add_launches(const snn_hip_linear_attention_params& p, const Sizes* walks, int n,
                  bool outputs, bool direct, int size,
                  snn_hip_linear_attention_plan* plan) {
  bool done[att::kMostWalks] = {};
  for (int i = 0; i < n; ++i) {
    if (done[i]) continue;
    const int keys = class_of(walks[i].keys);
    const int waves = waves_of(size, walks[i].values);
    size_t units = 0;
    for (int j = i; j < n; ++j) {
      if (done[j] || class_of(walks[j].keys) != keys ||
          waves_of(size, walks[j].values) != waves)
        continue;
      units += slices_of(size, walks[j].values);
      done[j] = true;
    }
    const unsigned groups = static_cast<unsigned>(
        units * p.batch * p.heads * static_cast<size_t>(plan->pieces));
    plan->launch[plan->launches++] = {
        outputs, keys, waves, att::ring_of(keys, waves, outputs, direct, groups),
        static_cast<int>(groups)};
  }
}

}  // namespace
}  // namespace snn

#define SNN_LINEAR_ATTENTION(suffix, T)                                        \
  int snn_hip_linear_attention_##suffix(                                       \
      const void* q, const void* k, const void* v, const float* decay,         \
      const unsigned char* resets, const int* lengths,                         \
      const float* initial_state, void* output, float* final_state,            \
      const snn_hip_linear_attention_params* params, void* workspace,          \
      size_t workspace_elems, void* stream) {                                  \
    return snn::forward<T>(q, k, v, decay, resets, lengths, initial_state,     \
                           output, final_state, params, workspace,             \
                           workspace_elems, stream);                           \
  }                                                                            \
  int snn_hip_linear_attention_grad_##suffix(                                  \
      const void* grad_output, const float* grad_final_state, const void* q,   \
      const void* k, const void* v, const float* decay,                        \
      const unsigned char* resets, const int* lengths,                         \
      const float* initial_state, void* grad_q, void* grad_k, void* grad_v,    \
      float* grad_initial_state,                                               \
      const snn_hip_linear_attention_params* params, void* workspace,          \
      size_t workspace_elems, void* stream) {                                  \
    return snn::backward<T>(grad_output, grad_final_state, q, k, v, decay,     \
                            resets, lengths, initial_state, grad_q, grad_k,    \
                            grad_v, grad_initial_state, params, workspace,     \
                            workspace_elems, stream);                          \
  }

extern "C" {

SNN_LINEAR_ATTENTION(f32, float)
SNN_LINEAR_ATTENTION(f16, _Float16)
SNN_LINEAR_ATTENTION(bf16, __bf16)

int snn_hip_linear_attention_workspace_size(
    const snn_hip_linear_attention_params* params, int grad, int dtype,
    size_t* required_elems, size_t* recommended_elems) {
  if (dtype < SNN_HIP_DTYPE_F32 || dtype > SNN_HIP_DTYPE_BF16 ||
      required_elems == nullptr || recommended_elems == nullptr)
    return SNN_HIP_INVALID_PARAMETER;
  const int valid = grad != 0 ? snn::check_grad(params, nullptr)
                              : snn::check(params, nullptr);
  if (valid != SNN_HIP_OK) return valid;
  const int size = dtype == SNN_HIP_DTYPE_F32 ? 4 : 2;
  size_t all = 0;
  *required_elems = 0;
  if (grad != 0) {
    all = 2 * snn::shared_bytes(*params);
    *required_elems = all / size;
    all += snn::division_bytes(*params, snn::grad_division(*params, size, ~size_t{0}), 2);
  } else if (params->steps > snn::kFewSteps) {
    all = snn::division_bytes(*params, snn::forward_division(*params, size, ~size_t{0}), 1);
  }
  *recommended_elems = all / size;
  return SNN_HIP_OK;
}

int snn_hip_linear_attention_planned(
    const snn_hip_linear_attention_params* params, int grad, int dtype,
    int aligned, size_t workspace_elems, snn_hip_linear_attention_plan* plan) {
  if (dtype < SNN_HIP_DTYPE_F32 || dtype > SNN_HIP_DTYPE_BF16 || plan == nullptr)
    return SNN_HIP_INVALID_PARAMETER;
  const int valid = grad != 0 ? snn::check_grad(params, nullptr)
                              : snn::check(params, nullptr);
  if (valid != SNN_HIP_OK) return valid;
  const snn_hip_linear_attention_params& p = *params;
  const int size = dtype == SNN_HIP_DTYPE_F32 ? 4 : 2, piece = 16 / size;
  *plan = {};
  plan->pieces = 1;
  if (grad == 0 && p.steps <= snn::kFewSteps) return SNN_HIP_OK;
  bool direct = aligned != 0;
  for (const int n : {p.keys, p.values, p.q_stride, p.k_stride, p.v_stride,
                      p.grad_q_stride, p.grad_k_stride, p.grad_v_stride})
    direct = direct && n % piece == 0;
  size_t bytes = workspace_elems * size;
  snn::Division d;
  if (grad != 0) {
    const size_t shared = 2 * snn::shared_bytes(p);
    if (bytes < shared) return SNN_HIP_INSUFFICIENT_WORKSPACE;
    d = snn::grad_division(p, size, bytes - shared);
  } else {
    d = snn::forward_division(p, size, bytes);
  }
  plan->pieces = d.pieces;
  plan->piece_steps = d.piece_steps;
  const snn::Sizes across = {p.keys, p.values}, back = {p.values, p.keys};
  const snn::Sizes states[] = {across, across}, walks[] = {back, back, across};
  if (d.pieces > 1)
    snn::add_launches(p, states, grad != 0 ? 2 : 1, false, direct, size, plan);
  if (grad != 0)
    snn::add_launches(p, walks, 3, true, direct, size, plan);
  else
    snn::add_launches(p, &across, 1, true, direct, size, plan);
  return SNN_HIP_OK;
}

}  // extern "C"
