// Linear attention with a decay for each head, and its gradients (gfx950):
//
//   S_t = a S_{t-1} + k_t^T v_t,  o_t = scale q_t S_t
//
// All of it is one operation, a walk over the sequence with operands in turn:
//
//   walk(q, k, v)_t = q_t X_t,  X_t = a X_{t-1} + k_t^T v_t
//
//   o   walk(q, k, v) from the front
//   dq  walk(do, v, k) from the front, whose state is S transposed
//   dk  walk(v, do, q) and
//   dv  walk(k, q, do) from the end, whose state is the gradient that the steps
//       behind hand to those in front
//
// From the end the state is handed on decayed, X'_t = a (X'_{t+1} + ...), so that
// the exponents of a are one less where it comes in and one more where it goes out.
//
// A walk goes in blocks of C steps.  Within a block (row r of the walk's order, n
// rows) and the state X in front of it
//
//   out_r = a^(r + 1) q_r X + sum over s <= r of a^(r - s) (q_r k_s) v_s
//   X'    = a^n X + sum over s of a^(n - 1 - s) k_s^T v_s
//
// are four products of the matrix instructions.  All exponents are at least zero, so
// that nothing overflows.  A work-group of four waves owns a piece of a head's
// sequence and a slice of its values, which the waves divide.  The state stays in
// registers: its accumulators' layout is that of the first operand of q X, as the
// reduction's order is free as long as both operands agree.  The next block's rows
// are on their way while one is multiplied.
//
// Sequences that do not fill the GPU are divided into pieces: a first pass walks them
// without outputs from a state of zero (k and v alone are read), the states are added
// up along the sequence, and the second pass starts each piece from its own.
//
// The 16-bit types: q_r k_s and its decay are rounded to the type, as the softmax
// weights of other attentions are; the state and the decayed v are held in two values
// of the type (16 bits of a bfloat16 pair), as the state is an fp32 result.
// Rows that may not count, those of later steps and those in front of a reset, are left
// out by selection.  The matrix instructions would multiply their v by zero, which an
// infinity or NaN survives: blocks that hold one (a product with zero tells) are
// summed value by value instead.
#ifndef PORTDNN_AMD_CSRC_LINEAR_ATTENTION_H_
#define PORTDNN_AMD_CSRC_LINEAR_ATTENTION_H_

#include "gemm_epilogue.h"
#include "snn_kernels.h"

namespace snn {
namespace att {

using epi::float4v;
using epi::lds_short4_ptr;
using epi::short4v;
using epi::uint4v;

struct Walk {
  const void *q, *k, *v;
  void* out;                          // null: the state alone
  long q_row, k_row, v_row, out_row;  // elements from step to step
  int q_share, k_share, v_share;      // heads that share one of the operand's
  int keys, values;                   // channels of q and k, of v and out
  int from_end;
  int out_float;       // out holds floats, whatever T is
  const float* initial;
  float* final;
  int transposed;      // initial and states are stored [values][keys]
  float weight;        // of q_r k_s
  float state_weight;  // of k_s^T v_s in the state
  float reach_weight;  // of q_r X
  int slices;          // work-groups that share the values
  float* states;       // [batch * heads][pieces][keys][values]
  int* carries;        // [batch * heads][pieces]: no reset in the piece
};

constexpr int kMostWalks = 3;
struct Problem {
  Walk walk[kMostWalks];
  int walks, units;  // units: slices of all walks
  int batch, heads, steps, pieces, piece_steps;
  const float* decay;
  const unsigned char* resets;
  const int* lengths;
};

// One launch for all walks; `outputs`: the second pass.
int run_walks_f32(const Problem& p, int keys_class, int waves, bool outputs,
                  hipStream_t stream);
int run_walks_f16(const Problem& p, int keys_class, int waves, bool outputs,
                  hipStream_t stream);
int run_walks_bf16(const Problem& p, int keys_class, int waves, bool outputs,
                   hipStream_t stream);

template <typename T>
constexpr int kBlock = sizeof(T) == 2 ? 64 : 32;  // C

__device__ __forceinline__ float log_decay(const float* decay, int head) {
  const float d = decay[head];
  return d > 0.f ? 0.f : d < -1e4f ? -1e4f : d;  // (a NaN stays)
}

__device__ __forceinline__ int length_of(const Problem& p, int b) {
  return p.lengths == nullptr ? p.steps : max(0, min(p.steps, p.lengths[b]));
}

// Tiles in LDS: rows of 16-byte pieces, piece c of row r at c ^ swizzle(r), so that
// neither the 16 rows of a fragment along the row nor the four rows of a transposing
// read (the four lane groups' rows of a transposed fragment of floats) meet in a bank.
template <int E, int PITCH>
__device__ __forceinline__ constexpr unsigned swizzle(unsigned r) {
  const unsigned low = r & 3u, high = (r >> 2) & 3u;
  if (PITCH == 128) return E == 4 ? (r >> 1) & 7u : ((r & 2u) << 1) | high;
  return E == 4 ? (high << 2) | low : (low << 2) | high;
}

template <typename T, int COLS>
struct Tile {
  static constexpr int E = sizeof(T);
  static constexpr int kPitch = COLS * E;
  static constexpr int kPieces = kPitch / 16;  // of a row
  static constexpr int kPer = 16 / E;          // values of a piece
  static __device__ __forceinline__ unsigned at(unsigned row, unsigned piece) {
    return row * kPitch + ((piece ^ swizzle<E, kPitch>(row)) << 4);
  }
  static __device__ __forceinline__ float value(const char* tile, int row,
                                                int col) {
    return static_cast<float>(*reinterpret_cast<const T*>(
        tile + at(row, col / kPer) + col % kPer * E));
  }
  // The lane's part of a fragment: row 16 t + lane % 16, reductions along the row,
  // piece 4 b + lane / 16.  A tile's row enters its swizzle by its last four bits
  // and b enters the swizzled place by its last two, so that four (two) addresses of
  // the lane's, `along`, and constants make all of them.
  static constexpr int kAlong = kPieces < 16 ? kPieces / 4 : 4;
  static __device__ __forceinline__ void start_rows(unsigned (&along)[kAlong],
                                                    int lane) {
#pragma unroll
    for (int b = 0; b < kAlong; ++b)
      along[b] = at(lane & 15, 4 * b + (lane >> 4));
  }
  static __device__ __forceinline__ uint4v rows(const char* tile,
                                                const unsigned (&along)[kAlong],
                                                int t, int b) {
    return *reinterpret_cast<const uint4v*>(tile + along[b % kAlong] +
                                            16 * t * kPitch +
                                            b / kAlong * 256);
  }
  // Reductions are rows: those of block b (32 or 16 of them) for a column of the
  // lane's.  16-bit types: columns 32 i + 4 half + 8 (c / 4) + c % 4 for c = lane %
  // 16, so that two such fragments share out 32 columns in runs of eight; fp32:
  // columns 16 i + c.
  static constexpr int kDown = E == 2 ? 2 : 4;
  static constexpr int kAcross = kAlong;
  static __device__ __forceinline__ void start_columns(
      unsigned (&down)[kAcross][kDown], int lane) {
#pragma unroll
    for (int i = 0; i < kAcross; ++i)
#pragma unroll
      for (int u = 0; u < kDown; ++u) {
        if constexpr (E == 2)
          down[i][u] = at(8 * (lane >> 4) + ((lane & 15) >> 2) + 4 * u,
                          4 * i + (lane & 3));
        else
          down[i][u] = at(4 * (lane >> 4) + u, 4 * i + ((lane & 15) >> 2)) +
                       (lane & 3) * 4;
      }
  }
  static __device__ __forceinline__ uint4v columns(
      const char* tile, const unsigned (&down)[kAcross][kDown], int i, int half,
      int b) {
    return fragment(tile + i / kAcross * 256 + half * 8, down[i % kAcross], b);
  }
  // The same of the 16 neighbouring columns from `first` on.
  static __device__ __forceinline__ void start_columns(unsigned (&down)[kDown],
                                                       int first, int lane) {
#pragma unroll
    for (int u = 0; u < kDown; ++u) {
      if constexpr (E == 2) {
        const unsigned col = first + 4 * (lane & 3);
        down[u] = at(8 * (lane >> 4) + ((lane & 15) >> 2) + 4 * u, col >> 3) +
                  ((col & 4) << 1);
      } else {
        const unsigned col = first + (lane & 15);
        down[u] = at(4 * (lane >> 4) + u, col >> 2) + (col & 3) * 4;
      }
    }
  }
  // (transposing reads: within 16 lanes, lane 4 j + i supplies the address of four
  // values of row j and lane t receives column t of rows 0 ... 3)
  static __device__ __forceinline__ uint4v fragment(
      const char* tile, const unsigned (&down)[kDown], int b) {
    if constexpr (E == 2) {
      const char* const from = tile + 32 * b * kPitch;
      const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_short4_ptr)(const_cast<char*>(from) + down[0]));
      const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_short4_ptr)(const_cast<char*>(from) + down[1]));
      return __builtin_bit_cast(
          uint4v, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      uint4v v;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        v[u] = *reinterpret_cast<const unsigned*>(tile + 16 * b * kPitch +
                                                  down[u]);
      return v;
    }
  }
};

// Eight (four) floats as values of T, and what those leave of them; fp32 leaves none.
template <typename T>
struct Split {
  static constexpr int N = 16 / sizeof(T);
  typedef T V __attribute__((ext_vector_type(N)));
  static __device__ __forceinline__ void split(const float (&v)[N], uint4v* high,
                                               uint4v* low) {
    V t;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = static_cast<T>(v[i]);
    *high = __builtin_bit_cast(uint4v, t);
    if constexpr (sizeof(T) == 2) {
      // (the rounded values themselves: worked out anew from a product, with one
      // rounding less, one in two thousand would be another than the one taken off)
      asm volatile("" : "+v"(*high));
      t = __builtin_bit_cast(V, *high);
#pragma unroll
      for (int i = 0; i < N; ++i)
        t[i] = static_cast<T>(v[i] - static_cast<float>(t[i]));
      *low = __builtin_bit_cast(uint4v, t);
    }
  }
  static __device__ __forceinline__ void floats(uint4v f, float (&v)[N]) {
    const V t = __builtin_bit_cast(V, f);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<float>(t[i]);
  }
};

// What a work-group is given.
struct Part {
  int walk, slice, bh, b, h, piece;
};
__device__ __forceinline__ Part part_of(const Problem& p) {
  // (an XCD takes slices and walks of one head and piece beside one another: they
  // read the same rows)
  const unsigned at = gemm::xcd_remap(blockIdx.x, gridDim.x);
  Part r;
  unsigned unit = at % p.units;
  const unsigned rest = at / p.units, heads = p.batch * p.heads;
  r.bh = static_cast<int>(rest % heads);
  r.piece = static_cast<int>(rest / heads);
  r.b = r.bh / p.heads;
  r.h = r.bh - r.b * p.heads;
  r.walk = 0;
  while (unit >= static_cast<unsigned>(p.walk[r.walk].slices)) {
    unit -= p.walk[r.walk].slices;
    ++r.walk;
  }
  r.slice = static_cast<int>(unit);
  return r;
}

// D: the keys, rounded up; WAVES: of a work-group, with 16 values each.
template <typename T, int D, int WAVES, bool OUTPUT>
__global__ void __launch_bounds__(64 * WAVES, 2)
    walk_kernel(Problem p) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int E = sizeof(T), C = kBlock<T>, BV = 16 * WAVES;
  constexpr int kThreads = 64 * WAVES;
  constexpr int KB = 64 / E;      // reductions of a fragment
  constexpr int HALVES = KB / 16;  // state tiles of a block of KB keys
  constexpr int BLOCKS = D / KB, TT = C / 16, SB = C / KB;
  constexpr int PT = (TT * TT + WAVES - 1) / WAVES;  // tiles of q k of a wave
  typedef Tile<T, D> Keys;
  typedef Tile<T, BV> Values;
  typedef Tile<T, C> Weights;
  constexpr int kLoadsK = C * Keys::kPieces / kThreads;
  constexpr int kLoadsV = C * Values::kPieces / kThreads;
  __shared__ __align__(1024) char q_tile[OUTPUT ? C * Keys::kPitch : 16];
  __shared__ __align__(1024) char k_tile[C * Keys::kPitch];
  __shared__ __align__(1024) char v_tile[C * Values::kPitch];
  __shared__ __align__(1024) char p_tile[OUTPUT ? C * Weights::kPitch : 16];
  __shared__ float power[C + 1];
  __shared__ int resets_to[C];  // in front of a row that count against it

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, group = lane >> 4;
  const Part part = part_of(p);
  const Walk& w = p.walk[part.walk];
  const int length = length_of(p, part.b);
  const int first = part.piece * p.piece_steps;  // in the walk's order
  const int last = min(first + p.piece_steps, length);
  const bool from_end = w.from_end != 0;
  // (the last piece's state is the second pass's to find)
  if (!OUTPUT && first + p.piece_steps >= length) return;
  const float log_a = log_decay(p.decay, part.h);
  if (tid <= C) power[tid] = tid == 0 ? 1.f : expf(tid * log_a);
  __syncthreads();

  const int col0 = part.slice * BV + wave * 16;  // of the wave's values
  const long row_base = static_cast<long>(part.b) * p.steps;
  const T* const q = OUTPUT ? static_cast<const T*>(w.q) +
                                  row_base * w.q_row +
                                  static_cast<long>(part.h / w.q_share) * w.keys
                            : nullptr;
  const T* const k = static_cast<const T*>(w.k) + row_base * w.k_row +
                     static_cast<long>(part.h / w.k_share) * w.keys;
  const T* const v = static_cast<const T*>(w.v) + row_base * w.v_row +
                     static_cast<long>(part.h / w.v_share) * w.values;
  // the step of a place in the walk's order
  auto step_of = [&](int place) {
    return from_end ? length - 1 - place : place;
  };

  // The state: tile i, values 16 j: the lane's column of it is its value lane % 16,
  // its rows the keys key_of(i) + 0 ... 3.
  float4v state[D / 16];
  auto key_of = [&](int i) {
    return i / HALVES * KB + group * (KB / 4) + i % HALVES * 4;
  };
  const long state_size = static_cast<long>(w.keys) * w.values;
  const long state_at =
      (static_cast<long>(part.bh) * p.pieces + part.piece) * state_size;
  {
    const float* from = nullptr;
    bool transposed = false;
    if (OUTPUT) {
      if (p.pieces > 1)
        from = w.states + state_at;
      else if (w.initial != nullptr)
        from = w.initial + part.bh * state_size;
      transposed = w.transposed != 0;
    }
    const int value = col0 + c16;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      state[i] = float4v{0.f, 0.f, 0.f, 0.f};
      if (from != nullptr && value < w.values) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = key_of(i) + r;
          if (key < w.keys)
            state[i][r] =
                from[transposed ? static_cast<long>(value) * w.keys + key
                                : static_cast<long>(key) * w.values + value];
        }
      }
    }
  }

  // A block's rows on their way, in pieces of 16 bytes.  Rows behind the last are that
  // one again and pieces that would reach behind a head's channels begin before, so
  // that every load is of values that exist; on their way into LDS the one become
  // zeros and the others are shifted to where the piece begins.
  constexpr int kPer = 16 / E;
  auto load_piece = [&](const T* base, long stride, int row, int place, int col,
                        int cols) {
    const T* const at = base + step_of(min(place + row, last - 1)) * stride;
    uint4v f;
    if (cols >= kPer) {
      __builtin_memcpy(&f, at + min(col, cols - kPer), 16);
    } else {
      T some[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) some[i] = at[min(i, cols - 1)];
      __builtin_memcpy(&f, some, 16);
    }
    return f;
  };
  auto whole_piece = [&](uint4v f, int row, int n, int col, int cols) {
    if (row >= n || col >= cols) return uint4v{0u, 0u, 0u, 0u};
    if (cols >= kPer)
      return epi::shifted_down(f, max(0, col + kPer - cols) * E);
    typedef T V __attribute__((ext_vector_type(kPer)));
    V some = __builtin_bit_cast(V, f);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i >= cols) some[i] = T(0);
    return __builtin_bit_cast(uint4v, some);
  };
  const int value0 = part.slice * BV;
  const bool whole_keys = w.keys == D, whole_values = w.values - value0 >= BV;
  uint4v held_q[OUTPUT ? kLoadsK : 1], held_k[kLoadsK], held_v[kLoadsV];
  unsigned held_reset = 0;
  auto load = [&](int place) {
#pragma unroll
    for (int l = 0; l < kLoadsK; ++l) {
      const int at = tid + kThreads * l, row = at / Keys::kPieces;
      const int col = at % Keys::kPieces * kPer;
      held_k[l] = load_piece(k, w.k_row, row, place, col, w.keys);
      if (OUTPUT) held_q[l] = load_piece(q, w.q_row, row, place, col, w.keys);
    }
#pragma unroll
    for (int l = 0; l < kLoadsV; ++l) {
      const int at = tid + kThreads * l, row = at / Values::kPieces;
      const int col = at % Values::kPieces * kPer;
      held_v[l] = load_piece(v, w.v_row, row, place, value0 + col, w.values);
    }
    if (p.resets != nullptr)
      held_reset = lane < C && place + lane < last
                       ? p.resets[row_base + step_of(place + lane)]
                       : 0u;
  };

  // The weights of the wave's tiles of q k: of row (column of the tile) 16 t + c16
  // and the four s from 16 x + 4 group on.
  float weight[PT][4], reach[TT];
  if constexpr (OUTPUT) {
#pragma unroll
    for (int x = 0; x < PT; ++x) {
      const int t = (wave * PT + x) / TT % TT, s = (wave * PT + x) % TT;
      const int apart = 16 * (t - s) + c16 - 4 * group;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        weight[x][r] = apart >= r ? w.weight * power[apart - r] : 0.f;
    }
#pragma unroll
    for (int t = 0; t < TT; ++t)
      reach[t] = w.reach_weight * power[16 * t + c16 + (from_end ? 0 : 1)];
  }
  bool carried = true;  // no reset so far
  unsigned along[Keys::kAlong], along_p[Weights::kAlong];
  unsigned down_k[Keys::kAcross][Keys::kDown], down_v[Values::kDown];
  Keys::start_rows(along, lane);
  Weights::start_rows(along_p, lane);
  Keys::start_columns(down_k, lane);
  Values::start_columns(down_v, wave * 16, lane);

  if (first < last) load(first);
  for (int place = first; place < last; place += C) {
    const int n = min(C, last - place);
    if (n < C || !whole_keys) {
#pragma unroll
      for (int l = 0; l < kLoadsK; ++l) {
        const int at = tid + kThreads * l, row = at / Keys::kPieces;
        const int col = at % Keys::kPieces * kPer;
        held_k[l] = whole_piece(held_k[l], row, n, col, w.keys);
        if (OUTPUT) held_q[l] = whole_piece(held_q[l], row, n, col, w.keys);
      }
    }
    if (n < C || !whole_values) {
#pragma unroll
      for (int l = 0; l < kLoadsV; ++l) {
        const int at = tid + kThreads * l, row = at / Values::kPieces;
        const int col = value0 + at % Values::kPieces * kPer;
        held_v[l] = whole_piece(held_v[l], row, n, col, w.values);
      }
    }
#pragma unroll
    for (int l = 0; l < kLoadsK; ++l) {
      const int at = tid + kThreads * l;
      const unsigned to = Keys::at(at / Keys::kPieces, at % Keys::kPieces);
      *reinterpret_cast<uint4v*>(k_tile + to) = held_k[l];
      if (OUTPUT) *reinterpret_cast<uint4v*>(q_tile + to) = held_q[l];
    }
#pragma unroll
    for (int l = 0; l < kLoadsV; ++l) {
      const int at = tid + kThreads * l;
      *reinterpret_cast<uint4v*>(
          v_tile + Values::at(at / Values::kPieces, at % Values::kPieces)) =
          held_v[l];
    }
    // Which of the block's rows are resets.  Rows s < r (in the walk's order) count
    // for one another where none is among s + 1 ... r, or s ... r - 1 from the end:
    // where as many are in front of both.
    const unsigned long long resets = __ballot(held_reset != 0);
    if (p.resets != nullptr && wave == 0 && lane < C) {
      const unsigned long long before = (1ull << lane) - 1;
      resets_to[lane] = static_cast<int>(__popcll(
          resets & (from_end ? before : before | 1ull << lane)));
    }
    const int all_resets = static_cast<int>(__popcll(resets));
    __syncthreads();
    if (place + C < last) load(place + C);

    if constexpr (OUTPUT) {
#pragma unroll
      for (int x = 0; x < PT; ++x) {
        const int t = (wave * PT + x) / TT, s = (wave * PT + x) % TT;
        if (t >= TT) continue;  // (blocks of fewer tiles than waves)
        float4v acc = {0.f, 0.f, 0.f, 0.f};
        if (s <= t) {
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b)
            acc = epi::multiply<T>(Keys::rows(k_tile, along, s, b),
                                   Keys::rows(q_tile, along, t, b), acc);
        }
        typedef T Four __attribute__((ext_vector_type(4)));
        Four to;
        const int row = 16 * t + c16, col = 16 * s + 4 * group;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          bool on = col + r <= row;
          if (resets != 0) on = on && resets_to[col + r] == resets_to[row];
          to[r] = static_cast<T>(on ? acc[r] * weight[x][r] : 0.f);
        }
        *reinterpret_cast<Four*>(p_tile +
                                 Weights::at(row, col / Weights::kPer) +
                                 col % Weights::kPer * E) = to;
      }
      __syncthreads();
    }

    uint4v v_part[SB];
    bool finite = true;
    {
      float4v zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        v_part[b] = Values::fragment(v_tile, down_v, b);
        zero = epi::multiply<T>(v_part[b], uint4v{0u, 0u, 0u, 0u}, zero);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) finite = finite && zero[r] == 0.f;
    }
    finite = __all(finite);

    if constexpr (OUTPUT) {
      // q X of all rows, and the sums over the block's v
      float scale = 1.f, unscale[4] = {1.f, 1.f, 1.f, 1.f};
      if constexpr (std::is_same<T, _Float16>::value) {
        // (a value's column of the state times a power of two that brings it close to
        // binary16's largest values)
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = fabsf(state[i][r]);
            most = x < INFINITY ? fmaxf(most, x) : most;
          }
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        const int exponent = min(
            126,
            max(-100, static_cast<int>(__float_as_uint(most) >> 23) - 141));
        scale = __uint_as_float(static_cast<unsigned>(127 - exponent) << 23);
        const float back =
            __uint_as_float(static_cast<unsigned>(127 + exponent) << 23);
#pragma unroll
        for (int r = 0; r < 4; ++r) unscale[r] = __shfl(back, 4 * group + r);
      }
      float4v acc[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[t] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        float x[4 * HALVES];
#pragma unroll
        for (int i = 0; i < 4 * HALVES; ++i)
          x[i] = state[b * HALVES + i / 4][i % 4] * scale;
        uint4v high, low;
        Split<T>::split(x, &high, &low);
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          const uint4v of_q = Keys::rows(q_tile, along, t, b);
          acc[t] = epi::multiply<T>(high, of_q, acc[t]);
          if constexpr (E == 2) acc[t] = epi::multiply<T>(low, of_q, acc[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const int row = 16 * t + c16;
        const bool reached = resets == 0 || resets_to[row] == 0;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[t][r] = reached ? acc[t][r] * reach[t] * unscale[r] : 0.f;
        if (finite) {
#pragma unroll
          for (int b = 0; b < SB; ++b) {
            if (b * KB > 16 * t + 15) continue;
            acc[t] = epi::multiply<T>(
                v_part[b], Weights::rows(p_tile, along_p, t, b), acc[t]);
          }
        } else {
          int to = row, first_value = wave * 16 + 4 * group;
          // (not worked out in front of the blocks, where it would take registers)
          asm volatile("" : "+v"(to), "+v"(first_value));
          for (int s = 0; s <= to; ++s) {
            if (resets != 0 && resets_to[s] != resets_to[to]) continue;
            const float x = Weights::value(p_tile, to, s);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[t][r] += x * Values::value(v_tile, s, first_value + r);
          }
        }
        if (w.out != nullptr && row < n) {
          const long at =
              (row_base + step_of(place + row)) * w.out_row +
              static_cast<long>(part.h) * w.values;
          const int col = col0 + 4 * group;
          auto store = [&](auto* out) {
            typedef std::remove_pointer_t<decltype(out)> O;
            out += at + col;
            if (col + 4 <= w.values) {
              float x[4] = {acc[t][0], acc[t][1], acc[t][2], acc[t][3]};
              *reinterpret_cast<typename seq::Pack<O, 4>::type*>(out) =
                  seq::pack<O, 4>(x);
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (col + r < w.values) out[r] = static_cast<O>(acc[t][r]);
            }
          };
          if (w.out_float)
            store(static_cast<float*>(w.out));
          else
            store(static_cast<T*>(w.out));
        }
      }
    }

    // The state behind the block.
    const float carry = power[n];
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        state[i][r] = all_resets == 0 ? state[i][r] * carry : 0.f;
    carried = carried && all_resets == 0;
    const int to_end = from_end ? n : n - 1;
    // (rows in front of a reset may hold a k that a weight of zero leaves infinite)
    bool by_products = finite;
    if (finite && resets != 0) {
#pragma unroll
      for (int b = 0; b < SB; ++b)
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const float4v zero = epi::multiply<T>(
              Keys::columns(k_tile, down_k, i / HALVES, i % HALVES, b),
              uint4v{0u, 0u, 0u, 0u}, float4v{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int r = 0; r < 4; ++r)
            by_products = by_products && zero[r] == 0.f;
        }
      by_products = __all(by_products);
    }
    if (by_products) {
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        float by[16 / E];
#pragma unroll
        for (int i = 0; i < 16 / E; ++i)
        {
          const int row = b * KB + group * (KB / 4) + i;
          by[i] = w.state_weight * power[max(0, to_end - row)];
          if (resets != 0 && resets_to[row] != all_resets) by[i] = 0.f;
        }
        float x[16 / E];
        Split<T>::floats(v_part[b], x);
#pragma unroll
        for (int i = 0; i < 16 / E; ++i) x[i] *= by[i];
        uint4v high, low;
        Split<T>::split(x, &high, &low);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint4v of_k =
              Keys::columns(k_tile, down_k, i / HALVES, i % HALVES, b);
          state[i] = epi::multiply<T>(of_k, high, state[i]);
          if constexpr (E == 2) state[i] = epi::multiply<T>(of_k, low, state[i]);
        }
      }
    } else {
      int value = wave * 16 + c16, key = group * (KB / 4);
      asm volatile("" : "+v"(value), "+v"(key));
      for (int s = 0; s < n; ++s) {
        if (resets != 0 && resets_to[s] != all_resets) continue;
        const float x =
            w.state_weight * power[to_end - s] * Values::value(v_tile, s, value);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            state[i][r] += x * Keys::value(k_tile, s, key + i / HALVES * KB +
                                                          i % HALVES * 4 + r);
      }
    }
    __syncthreads();  // the tiles have been read
  }

  if (OUTPUT && w.out != nullptr) {  // rows behind the sequence's length
    const int end = min(first + p.piece_steps, p.steps);
    const int columns = min(BV, w.values - part.slice * BV);
    const long rows = end - max(first, length);
    for (long at = tid; at < rows * columns; at += kThreads) {
      const long to =
          (row_base + max(first, length) + at / columns) * w.out_row +
          static_cast<long>(part.h) * w.values + part.slice * BV + at % columns;
      if (w.out_float)
        static_cast<float*>(w.out)[to] = 0.f;
      else
        static_cast<T*>(w.out)[to] = T(0);
    }
  }
  // The state behind the sequence, or behind the piece.
  float* to = nullptr;
  if (!OUTPUT) {
    to = w.states + state_at;
    if (part.slice == 0 && tid == 0)
      w.carries[static_cast<long>(part.bh) * p.pieces + part.piece] = carried;
  } else if (w.final != nullptr &&
             (length == 0 ? part.piece == 0 : first < length && last == length)) {
    to = w.final + part.bh * state_size;
  }
  if (to == nullptr) return;
  const int value = col0 + c16;
  if (value >= w.values) return;
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int key = key_of(i) + r;
      if (key < w.keys)
        to[static_cast<long>(key) * w.values + value] = state[i][r];
    }
#endif
}

template <typename T, int D, int WAVES>
int launch_walk(const Problem& p, bool outputs, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.units) * p.batch * p.heads * p.pieces);
  if (outputs)
    hipLaunchKernelGGL((walk_kernel<T, D, WAVES, true>), grid,
                       dim3(64 * WAVES), 0, stream, p);
  else
    hipLaunchKernelGGL((walk_kernel<T, D, WAVES, false>), grid,
                       dim3(64 * WAVES), 0, stream, p);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T>
int run_walks(const Problem& p, int keys_class, int waves, bool outputs,
              hipStream_t stream) {
  switch (keys_class) {
    case 64:
      return waves == 8 ? launch_walk<T, 64, 8>(p, outputs, stream)
                        : launch_walk<T, 64, 4>(p, outputs, stream);
    case 128:
      return waves == 8 ? launch_walk<T, 128, 8>(p, outputs, stream)
                        : launch_walk<T, 128, 4>(p, outputs, stream);
    default:
      return waves == 8 ? launch_walk<T, 256, 8>(p, outputs, stream)
                        : launch_walk<T, 256, 4>(p, outputs, stream);
  }
}

}  // namespace att
}  // namespace snn

#endif  // PORTDNN_AMD_CSRC_LINEAR_ATTENTION_H_
