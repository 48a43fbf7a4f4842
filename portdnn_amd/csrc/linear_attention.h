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
// that nothing overflows.  A work-group of four or eight waves owns a piece of a head's
// sequence and a slice of its values, 16 for each wave.  The state stays in registers:
// its accumulators' layout is that of the first operand of q X, as the reduction's order
// is free as long as both operands agree.  The next blocks' rows are on their way while
// one is multiplied.
//
// What bounds it: neither memory nor the matrix unit, but the chain of a block.  A block
// of 64 steps and 128 channels takes a work-group 3.5 us alone on its CU: q k, its weights
// by way of LDS, q X and the splits of X, the sums over v, the split of the weighted v,
// its products; waits at two barriers lie between, and the vector unit is busy with
// splits, weights and carries about half of the time.  bfloat16, 1 x 32768 steps of 16
// heads of 128 channels: 228 us, of them 70 for the pass that leaves states, 10 for their
// sums, 151 for the outputs (537 MB in all, 2.4 TB/s; 34 GFLOP by the formula of the steps,
// 150 TFLOP/s); binary16 249.  Left out, of the 166 us that the outputs took before blocks
// were asked for three ahead: loads 31, stores 44, the state's update 64, q X 90 us.
// Gradients of 4 x 4096 steps, three walks of 64 heads in one launch: 254 us.  fp32, 1 x
// 8192 steps of 8 heads: 98 us, gradients 206.
//
// Sequences that do not fill the GPU are divided into pieces: a first pass walks them
// without outputs from a state of zero (k and v alone are read), the states are added
// up along the sequence, and the second pass starts each piece from its own.
//
// The 16-bit types: q_r k_s and its decay are rounded to the type, once, as an output
// is: a product of two more values would cost as much again.  The state is held in two
// values of the type for q X (an output is rounded to 8 or 11 bits of the sum), and the
// weighted v in three, as states are fp32 results (binary16: two, of 22 bits together,
// where a value's column of the block takes a power of two into the type's range).
// Rows that may not count, those of later steps and those in front of a reset, are left
// out by selection.  The matrix instructions would multiply their v by zero, which an
// infinity or NaN survives: where there is one (a product with zero tells) they are
// summed value by value instead, in a second walk of the work-group's piece, and so they
// are where a state of a 16-bit walk is infinite.  That walk is slow: with one such value in
// a sequence, or in all, bfloat16 calls of 228 us (above) take 2990, gradients of 240 3760,
// 64 x 512 steps of 16 heads of 64 channels 679 for 80; fp32 calls of 98 us 331.
#ifndef PORTDNN_AMD_CSRC_LINEAR_ATTENTION_H_
#define PORTDNN_AMD_CSRC_LINEAR_ATTENTION_H_

#include "gemm_epilogue.h"
#include "snn_kernels.h"

namespace snn {
namespace att {

using epi::float4v;
using epi::lds_ptr;
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

// Eight (four) floats as a sum of values of T, each what those before leave of them:
// three of bfloat16 and two of binary16 hold 24 and 22 bits, fp32 needs one.
template <typename T>
struct Split {
  static constexpr int N = 16 / sizeof(T);
  static constexpr int kWhole = sizeof(T) == 4 ? 1 : std::is_same<T, _Float16>::value ? 2 : 3;
  typedef T V __attribute__((ext_vector_type(N)));
  // ANY: values that are infinite, which leave nothing, and that would be when rounded.
  template <bool ANY = false, int PARTS>
  static __device__ __forceinline__ void split(float (&v)[N], uint4v (&parts)[PARTS]) {
    constexpr float kMost = std::is_same<T, _Float16>::value ? 65504.f : 0x1.fep127f;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      V t;
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = static_cast<T>(v[i]);
      if constexpr (ANY && PARTS > 1) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (fabsf(v[i]) < INFINITY && fabsf(v[i]) > kMost)
            t[i] = static_cast<T>(copysignf(kMost, v[i]));
      }
      parts[p] = __builtin_bit_cast(uint4v, t);
      if (p + 1 == PARTS) break;
      // (the rounded values themselves: worked out anew from a product, with one
      // rounding less, one in two thousand would be another than the one taken off)
      asm volatile("" : "+v"(parts[p]));
      t = __builtin_bit_cast(V, parts[p]);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float rest = v[i] - static_cast<float>(t[i]);
        v[i] = ANY && fabsf(v[i]) == INFINITY ? 0.f : rest;
      }
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
  // (divisions are the vector unit's, their results the same for all lanes)
  auto same = [](unsigned x) {
    return static_cast<int>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
  };
  unsigned unit = same(at % p.units);
  const unsigned rest = same(at / p.units), heads = p.batch * p.heads;
  r.bh = same(rest % heads);
  r.piece = same(rest / heads);
  r.b = same(r.bh / p.heads);
  r.h = r.bh - r.b * p.heads;
  r.walk = 0;
  while (unit >= static_cast<unsigned>(p.walk[r.walk].slices)) {
    unit -= p.walk[r.walk].slices;
    ++r.walk;
  }
  r.slice = static_cast<int>(unit);
  return r;
}

// D: the keys, rounded up; WAVES: of a work-group, with 16 values each.  STAGES: blocks
// in a ring of LDS, to which rows of whole 16-byte pieces at aligned addresses go
// straight; 0: rows pass through registers, where one block is under way.
//
// Waves that share a SIMD's registers: as many as need not put many of their own into
// memory.  (2 x 4096 steps of 16 heads of 127 x 63 in bfloat16, three and two: 174 and 69
// us, gradients 353 and 169; of 128 x 64 64 and 57, 147 and 137.  fp32 gradients of 1 x
// 8192 steps of 8 heads of 128 x 128: 212 and 228.)
template <typename T, int D, int WAVES, bool OUTPUT, int RING>
constexpr int kWavesOfSimd =
    D == 256     ? WAVES / 4
    : WAVES == 8 ? (OUTPUT || (D == 128 && RING == 0) ? 2 : 4)
    : !OUTPUT    ? (D == 128 ? 3 : 4)
    : RING == 2  ? 2
    : D == 128   ? (sizeof(T) == 4 && RING == 1 ? 3 : 2)
                 : 3;

template <typename T, int D, int WAVES, bool OUTPUT, int RING>
__device__ __forceinline__ void walk_body(const Problem& p, char* ring0, char* ring1,
                                          char* ring2, char* p_tile, float* power,
                                          int* all_resets_to) {
  constexpr int E = sizeof(T), C = kBlock<T>, BV = 16 * WAVES;
  constexpr int kThreads = 64 * WAVES;
  constexpr int KB = 64 / E;       // reductions of a fragment
  constexpr int HALVES = KB / 16;  // state tiles of a block of KB keys
  constexpr int BLOCKS = D / KB, TT = C / 16, SB = C / KB;
  constexpr int PT = TT * TT / WAVES;  // tiles of q k of a wave
  constexpr int kPer = 16 / E;
  constexpr bool DIRECT = RING > 0;
  constexpr int STAGES = DIRECT ? RING : 1;
  typedef Tile<T, D> Keys;
  typedef Tile<T, BV> Values;
  typedef Tile<T, C> Weights;
  constexpr int kLoadsK = C * Keys::kPieces / kThreads;
  constexpr int kLoadsV = C * Values::kPieces / kThreads;
  // a block in LDS: k, v, q
  constexpr int kVAt = C * Keys::kPitch, kQAt = kVAt + C * Values::kPitch;
  auto ring = [&](int u) { return u == 0 ? ring0 : u == 1 ? ring1 : ring2; };

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, group = lane >> 4;
  const Part part = part_of(p);
  const Walk& w = p.walk[part.walk];
  const int length = __builtin_amdgcn_readfirstlane(length_of(p, part.b));
  const int first = part.piece * p.piece_steps;  // in the walk's order
  const int last = min(first + p.piece_steps, length);
  const bool from_end = w.from_end != 0;
  // (the last piece's state is the second pass's to find)
  if (!OUTPUT && first + p.piece_steps >= length) return;
  // (what the blocks need stays in scalar registers: read anew from the arguments it
  // would hold up every block)
  auto pin = [](auto x) {
    asm volatile("" : "+s"(x));
    return x;
  };
  auto same = [](unsigned x) {
    return static_cast<unsigned>(
        __builtin_amdgcn_readfirstlane(static_cast<int>(x)));
  };
  const float log_a = log_decay(p.decay, part.h);
  // (above zero: an infinite state stays infinite behind decays that fp32 has no value
  // for)
  if (tid <= C) power[tid] = tid == 0 ? 1.f : expf(tid * log_a) + 0x1p-126f;
  __syncthreads();
  // Tables by row: what a block's v and the state in front of it enter with, and the v of
  // a block that is not whole, two in turn.
  float *const into = power + C + 4, *const reach = into + C,
               *const into_parts = reach + C;
  if (tid < C) {
    into[tid] = w.state_weight * power[C - (from_end ? 0 : 1) - tid];
    reach[tid] = w.reach_weight * power[tid + (from_end ? 0 : 1)];
  }
  const float state_weight = pin(w.state_weight);
  __syncthreads();

  const int value0 = part.slice * BV, col0 = value0 + wave * 16;
  const long row_base = static_cast<long>(part.b) * p.steps;
  auto share_of = [&](int heads) {
    return __builtin_amdgcn_readfirstlane(part.h / heads);
  };
  const T* const q = OUTPUT ? static_cast<const T*>(w.q) +
                                  row_base * w.q_row +
                                  static_cast<long>(share_of(w.q_share)) * w.keys
                            : nullptr;
  const T* const k = static_cast<const T*>(w.k) + row_base * w.k_row +
                     static_cast<long>(share_of(w.k_share)) * w.keys;
  const T* const v = static_cast<const T*>(w.v) + row_base * w.v_row +
                     static_cast<long>(share_of(w.v_share)) * w.values + value0;
  // The step of a place in the walk's order; a block's lowest step (which may be in
  // front of the sequence, where the block's rows do not exist).
  auto step_of = [&](int place) {
    return from_end ? length - 1 - place : place;
  };
  auto lowest = [&](int place) {
    return from_end ? static_cast<long>(length) - C - place
                    : static_cast<long>(place);
  };

  // The state: tile i's column of the lane is its value lane % 16, its rows are the keys
  // key_of(i) + 0 ... 3.
  float4v state[D / 16];
  auto key_of = [&](int i) {
    return i / HALVES * KB + group * (KB / 4) + i % HALVES * 4;
  };
  const long state_size = static_cast<long>(w.keys) * w.values;
  const long state_at =
      (static_cast<long>(part.bh) * p.pieces + part.piece) * state_size;
  const int my_value = col0 + c16;
  // (through a buffer of the state's size, keys and values behind its own out of range:
  // as bits and not as a choice, which would be a branch around every access, and a wait)
  auto state_buffer = [&](const float* at) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(at), 0,
                                             static_cast<int>(state_size * 4),
                                             0x00020000);
  };
  auto state_offset = [&](int key, int of_key, int of_value) {
    const int out = (w.keys - 1 - key) | (w.values - 1 - my_value);
    return static_cast<unsigned>(key * of_key + my_value * of_value) |
           (static_cast<unsigned>(out >> 31) & epi::kOob);
  };
  auto start = [&] {
    const float* from = nullptr;
    if (OUTPUT)
      from = p.pieces > 1           ? w.states + state_at
             : w.initial != nullptr ? w.initial + part.bh * state_size
                                    : nullptr;
    if (from == nullptr) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) state[i] = float4v{0.f, 0.f, 0.f, 0.f};
      return;
    }
    const __amdgpu_buffer_rsrc_t rsrc = state_buffer(from);
    if (w.transposed && w.keys % 4 == 0) {
      // (a value's keys lie beside one another: gradients of 64 x 64 steps of 16 heads of
      // 128 channels, whose time is their states', 167 us one by one, 127 by four)
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        state[i] = __builtin_bit_cast(
            float4v, __builtin_amdgcn_raw_buffer_load_b128(
                         rsrc, state_offset(key_of(i), 4, 4 * w.keys), 0, 0));
      return;
    }
    const int of_key = w.transposed ? 4 : 4 * w.values;
    const int of_value = w.transposed ? 4 * w.keys : 4;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        state[i][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
            rsrc, state_offset(key_of(i) + r, of_key, of_value), 0, 0));
  };

  // A block's rows on their way, where they pass through registers.  Rows behind the
  // last are that one again and pieces that would reach behind a head's channels begin
  // before, so that every load is of values that exist; on their way into LDS the one
  // become zeros and the others are shifted to where the piece begins.
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
    if (n >= C && cols >= col + kPer) return f;
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
  const int there = w.values - value0;  // values from the slice's first on
  uint4v held_q[OUTPUT && !DIRECT ? kLoadsK : 1], held_k[DIRECT ? 1 : kLoadsK],
      held_v[DIRECT ? 1 : kLoadsV];
  unsigned held_reset = 0;
  auto load = [&](int place) {
    if constexpr (!DIRECT) {
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
        held_v[l] = load_piece(v, w.v_row, row, place, col, there);
      }
    }
  };
  auto put = [&](int place, char* to) {
    if constexpr (!DIRECT) {
      const int n = min(C, last - place);
#pragma unroll
      for (int l = 0; l < kLoadsK; ++l) {
        const int at = tid + kThreads * l, row = at / Keys::kPieces;
        const int piece = at % Keys::kPieces;
        const unsigned where = Keys::at(row, piece);
        *reinterpret_cast<uint4v*>(to + where) =
            whole_piece(held_k[l], row, n, piece * kPer, w.keys);
        if (OUTPUT)
          *reinterpret_cast<uint4v*>(to + kQAt + where) =
              whole_piece(held_q[l], row, n, piece * kPer, w.keys);
      }
#pragma unroll
      for (int l = 0; l < kLoadsV; ++l) {
        const int at = tid + kThreads * l, row = at / Values::kPieces;
        const int piece = at % Values::kPieces;
        *reinterpret_cast<uint4v*>(to + kVAt + Values::at(row, piece)) =
            whole_piece(held_v[l], row, n, piece * kPer, there);
      }
    }
  };
  // (every lane loads a byte that exists)
  const unsigned char* const resets_of =
      p.resets == nullptr ? nullptr : p.resets + row_base;
  auto load_reset = [&](int place) {
    if (resets_of != nullptr)
      held_reset = resets_of[step_of(min(place + lane % C, last - 1))];
  };

  // ... and straight to LDS, a KiB of neighbouring places for each load: the row and
  // the piece that belong there.
  // (a load of all threads is a number of rows; every sixteen rows, where the swizzle
  // comes again, a scalar offset moves: from the lowest step on)
  constexpr int kTurnsK =
      16 * Keys::kPieces > kThreads ? 16 * Keys::kPieces / kThreads : 1;
  constexpr int kTurnsV =
      16 * Values::kPieces > kThreads ? 16 * Values::kPieces / kThreads : 1;
  unsigned from_k[kTurnsK], from_q[kTurnsK], from_v[kTurnsV];
  auto moves = [&](auto tile) {  // rows of such a move, and how many there are
    typedef decltype(tile) Of;
    constexpr int kTurns =
        16 * Of::kPieces > kThreads ? 16 * Of::kPieces / kThreads : 1;
    constexpr int kRows = kThreads * kTurns / Of::kPieces;
    return std::integral_constant<int, kRows>();
  };
  constexpr int kMoveK = decltype(moves(Keys()))::value,
                kMoveV = decltype(moves(Values()))::value;
  const unsigned move_k = pin(static_cast<unsigned>(kMoveK * w.k_row * E)),
                 move_q = pin(static_cast<unsigned>(kMoveK * w.q_row * E)),
                 move_v = pin(static_cast<unsigned>(kMoveV * w.v_row * E));
  // the block that is issued next, and from block to block
  const char *at_k = nullptr, *at_q = nullptr, *at_v = nullptr;
  const long step_k = pin((from_end ? -C : C) * w.k_row * E),
             step_q = pin((from_end ? -C : C) * w.q_row * E),
             step_v = pin((from_end ? -C : C) * w.v_row * E);
  if constexpr (DIRECT) {
    auto places_of = [&](auto tile, long stride, int cols, int move, auto& from) {
      typedef decltype(tile) Of;
      constexpr int kTurns = sizeof(from) / sizeof(unsigned);
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        const int row = (tid + kThreads * u) / Of::kPieces;
        const int col = static_cast<int>(
            (tid % Of::kPieces ^ swizzle<E, Of::kPitch>(row)) * kPer);
        const int up = from_end ? move - 1 - row : row;
        from[u] = col < cols ? static_cast<unsigned>((up * stride + col) * E)
                             : epi::kOob;
      }
    };
    places_of(Keys(), w.k_row, w.keys, kMoveK, from_k);
    if (OUTPUT) places_of(Keys(), w.q_row, w.keys, kMoveK, from_q);
    places_of(Values(), w.v_row, there, kMoveV, from_v);
  }
  auto issue = [&](int place, char* to) {
    if constexpr (DIRECT) {
      const int n = last - place;  // (none: nothing but zeros comes)
      auto some = [&](const char* base, const auto& from, unsigned move, auto tile,
                      char* at) {
        typedef decltype(tile) Of;
        constexpr int kLoads = C * Of::kPieces / kThreads;
        constexpr int kRows = kThreads / Of::kPieces;
        constexpr int kTurns = sizeof(from) / sizeof(unsigned);
        constexpr int kMoves = kLoads / kTurns;
        const __amdgpu_buffer_rsrc_t rsrc = epi::make_rsrc(base);
        auto all = [&](auto offset_of) {
#pragma unroll
          for (int l = 0; l < kLoads; ++l)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rsrc, (lds_ptr)(at + (kThreads * l + 64 * wave) * 16), 16,
                offset_of(l),
                same((from_end ? kMoves - 1 - l / kTurns : l / kTurns) * move), 0,
                0);
        };
        if (n >= C)
          all([&](int l) { return from[l % kTurns]; });
        else
          all([&](int l) {
            return tid / Of::kPieces + kRows * l >= n ? epi::kOob
                                                      : from[l % kTurns];
          });
      };
      some(at_k, from_k, move_k, Keys(), to);
      some(at_v, from_v, move_v, Values(), to + kVAt);
      if (OUTPUT) some(at_q, from_q, move_q, Keys(), to + kQAt);
      at_k += step_k;
      at_v += step_v;
      at_q += step_q;
    }
  };

  // The wave's tiles of q k: rows 16 t, s from 16 (t + x) % TT on.  Their weights: a power
  // of the decay for the tile's distance from the diagonal, times the lane's four within
  // a tile.
  const int t_tile = wave * PT / TT;
  auto s_tile = [&](int x) { return (t_tile + wave * PT % TT + x) % TT; };
  // (the first of them is on the diagonal where a wave has all of a row)
  constexpr int kWords = E;  // of four weights
  float within[4], diagonal[4], beyond[PT];
  unsigned counts[PT][kWords];  // bits of the weights that count
  if constexpr (OUTPUT) {
    const int apart = c16 - 4 * group;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      within[r] = power[16 + apart - r];
      diagonal[r] = w.weight * power[max(0, apart - r)];
    }
#pragma unroll
    for (int x = 0; x < PT; ++x) {
      const int rows = 16 * (t_tile - s_tile(x));
      beyond[x] = rows < 0 ? 0.f : w.weight * power[max(0, rows - 16)];
#pragma unroll
      for (int u = 0; u < kWords; ++u) {
        counts[x][u] = 0;
#pragma unroll
        for (int r = u * 4 / kWords; r < (u + 1) * 4 / kWords; ++r)
          if (rows + apart >= r)
            counts[x][u] |= E == 4 ? ~0u : 0xFFFFu << 16 * (r % 2);
      }
    }
  }
  auto weight_of = [&](int x, int r) {
    const int rows = 16 * (t_tile - s_tile(x));
    return rows > 0 ? within[r] * beyond[x]
                    : diagonal[r];
  };
  bool carried = true;  // no reset so far
  unsigned along[Keys::kAlong], along_p[Weights::kAlong];
  unsigned down_k[Keys::kAcross][Keys::kDown], down_v[Values::kDown];
  Keys::start_rows(along, lane);
  Weights::start_rows(along_p, lane);
  Keys::start_columns(down_k, lane);
  Values::start_columns(down_v, wave * 16, lane);
  // Where the lane's row c16 of the result goes, and its other rows 16 further, from the
  // lowest step on.
  const bool out_float = pin(w.out_float) != 0;
  const int out_size = out_float ? 4 : E;
  const unsigned out_at =
      w.out != nullptr && my_value - c16 + 4 * group < w.values
          ? static_cast<unsigned>(
                ((from_end ? 15 - c16 : c16) * w.out_row + col0 + 4 * group) *
                out_size)
          : epi::kOob;
  const unsigned out_move = pin(static_cast<unsigned>(16 * w.out_row * out_size));
  char* at_out = nullptr;
  const long out_step = pin((from_end ? -C : C) * w.out_row * out_size);
  auto rewind = [&] {
    at_k = pin(reinterpret_cast<const char*>(k + lowest(first) * w.k_row));
    at_v = pin(reinterpret_cast<const char*>(v + lowest(first) * w.v_row));
    if (OUTPUT) {
      at_q = pin(reinterpret_cast<const char*>(q + lowest(first) * w.q_row));
      at_out = pin(static_cast<char*>(w.out) +
                   ((row_base + lowest(first)) * w.out_row +
                    static_cast<long>(part.h) * w.values) *
                       out_size);
    }
  };

  // The power of two that brings the largest value of a column of the wave's, of which
  // each lane has seen a part, close to binary16's largest; returns its inverse.
  auto range_of = [&](float most, float* scale) {
    // (rows of 16 lanes change places with their neighbours', halves with each other)
    const unsigned bits = __float_as_uint(most);
    const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
    most = fmaxf(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
    const unsigned pair = __float_as_uint(most);
    const auto halves = __builtin_amdgcn_permlane32_swap(pair, pair, false, false);
    most = fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
    const int exponent =
        min(126, max(-100, static_cast<int>(__float_as_uint(most) >> 23) - 141));
    *scale = __uint_as_float(static_cast<unsigned>(127 - exponent) << 23);
    return __uint_as_float(static_cast<unsigned>(127 + exponent) << 23);
  };

  // One block, whose rows are in `tile`.
  // CAREFUL: rows that do not count are left out one by one; otherwise by weights of
  // zero, after which `clean` tells whether that was enough.
  float4v clean = {0.f, 0.f, 0.f, 0.f};  // stays zero while every v is finite
  bool clean_k = true;
  // (... and while no state is infinite or would be when rounded: what the first of its
  // two values leaves is no number then.  Looked at in front of a reset and behind the
  // last block, as what is infinite stays so in between; bfloat16, which rounds the largest
  // states to infinity, also in front of the first)
  auto look = [&] {
    if constexpr (OUTPUT && E == 2) {
      unsigned most = 0;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          most = max(most, __float_as_uint(fabsf(state[i][r])));
      if (most >= __float_as_uint(0x1.ffp127f)) clean[0] = NAN;
    }
  };
  auto look_first = [&] {
    if constexpr (std::is_same<T, __bf16>::value) look();
  };
  auto walk = [&](const char* tile, int place, auto careful, auto next) {
    constexpr bool CAREFUL = decltype(careful)::value;
    // (two tables in turn: waves may still read the ones of the block before)
    const int turn = (place - first) / C % 2 * C;
    int* const resets_to = all_resets_to + turn;
    float* const into_part = into_parts + turn;
    const int n = min(C, last - place);
    const char *const k_tile = tile, *const v_tile = tile + kVAt,
                      *const q_tile = tile + kQAt;
    // Which of the block's rows are resets.  Rows s < r (in the walk's order) count
    // for one another where none is among s + 1 ... r, or s ... r - 1 from the end:
    // where as many are in front of both.
    unsigned long long resets = 0;
    if (resets_of != nullptr)
      resets = __ballot(held_reset != 0 && lane < C && place + lane < last);
    const int all_resets = static_cast<int>(__popcll(resets));
    const int to_end = from_end ? n : n - 1;
    const bool whole = n == C && resets == 0;
    if (!whole && wave == 0 && lane < C) {
      const unsigned long long before = (1ull << lane) - 1;
      const int mine = static_cast<int>(
          __popcll(resets & (from_end ? before : before | 1ull << lane)));
      resets_to[lane] = mine;
      into_part[lane] = lane < n && mine == all_resets
                           ? state_weight * power[to_end - lane]
                           : 0.f;
    }
    const float* const into_state = whole ? into : into_part;
    __builtin_amdgcn_s_waitcnt(epi::kLgkm0 & epi::vmcnt_imm(63));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    next();

    if constexpr (OUTPUT) {
      // (tiles of later s are worked out as well and left out: no branches)
      float4v acc[PT];
      uint4v of_q[2], of_k[2][PT];
      auto fetch = [&](int b) {
        of_q[b % 2] = Keys::rows(q_tile, along, t_tile, b);
#pragma unroll
        for (int x = 0; x < PT; ++x)
          of_k[b % 2][x] = Keys::rows(k_tile, along, s_tile(x), b);
      };
      fetch(0);
#pragma unroll
      for (int x = 0; x < PT; ++x) acc[x] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        if (b + 1 < BLOCKS) fetch(b + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < PT; ++x)
          acc[x] = epi::multiply<T>(of_k[b % 2][x], of_q[b % 2], acc[x]);
        __builtin_amdgcn_sched_barrier(0);
      }
      typedef unsigned int Words __attribute__((ext_vector_type(kWords)));
      const int row = 16 * t_tile + c16;
      unsigned bits[PT][kWords];
#pragma unroll
      for (int x = 0; x < PT; ++x)
#pragma unroll
        for (int u = 0; u < kWords; ++u) bits[x][u] = counts[x][u];
      if (resets != 0) {
        const int mine = resets_to[row];
#pragma unroll
        for (int x = 0; x < PT; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (resets_to[16 * s_tile(x) + 4 * group + r] != mine)
              bits[x][r * kWords / 4] &= E == 4 ? 0u : ~(0xFFFFu << 16 * (r % 2));
      }
#pragma unroll
      for (int x = 0; x < PT; ++x) {
        const int col = 16 * s_tile(x) + 4 * group;
        float to[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) to[r] = acc[x][r] * weight_of(x, r);
        Words words = __builtin_bit_cast(Words, seq::pack<T, 4>(to));
#pragma unroll
        for (int u = 0; u < kWords; ++u) words[u] &= bits[x][u];
        // (in assembly, as in front of a store that it knows the compiler waits for all
        // loads into LDS, those of the blocks under way too; the wait is below)
        const lds_ptr to_at = (lds_ptr)(p_tile + Weights::at(row, col / kPer) +
                                        col % kPer * E);
        if constexpr (E == 4)
          asm volatile("ds_write_b128 %0, %1" ::"v"(to_at), "v"(words) : "memory");
        else
          asm volatile("ds_write_b64 %0, %1" ::"v"(to_at), "v"(words) : "memory");
      }
      __builtin_amdgcn_s_waitcnt(epi::kLgkm0 & epi::vmcnt_imm(63));
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }

    uint4v v_part[SB];
    auto weighted = [&](int b, float (&x)[kPer]) {
      Split<T>::floats(v_part[b], x);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        x[i] *= into_state[b * KB + group * (KB / 4) + i];
    };
    constexpr bool kScaled = std::is_same<T, _Float16>::value;
    float range = 1.f, range_back = 1.f;  // of the weighted values
    auto fetch_v = [&] {
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        v_part[b] = Values::fragment(v_tile, down_v, b);
        if (!CAREFUL)
          clean = epi::multiply<T>(v_part[b], uint4v{0u, 0u, 0u, 0u}, clean);
      }
      if constexpr (kScaled && !CAREFUL) {
        float most = 0.f;
#pragma unroll
        for (int b = 0; b < SB; ++b) {
          float x[kPer];
          weighted(b, x);
#pragma unroll
          for (int i = 0; i < kPer; ++i) most = fmaxf(most, fabsf(x[i]));
        }
        range_back = range_of(most, &range);
      }
    };
    if constexpr (!OUTPUT) fetch_v();
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
        const float back = range_of(most, &scale);
#pragma unroll
        for (int r = 0; r < 4; ++r) unscale[r] = __shfl(back, 4 * group + r);
      }
      float4v acc[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[t] = float4v{0.f, 0.f, 0.f, 0.f};
      uint4v of_q[2][TT];
      auto fetch = [&](int b) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
          of_q[b % 2][t] = Keys::rows(q_tile, along, t, b);
      };
      fetch(0);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        if (b + 1 < BLOCKS) fetch(b + 1);
        float x[4 * HALVES];
#pragma unroll
        for (int i = 0; i < 4 * HALVES; ++i)
          x[i] = state[b * HALVES + i / 4][i % 4] * scale;
        uint4v parts[E == 4 ? 1 : 2];
        Split<T>::template split<CAREFUL>(x, parts);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (const uint4v& part : parts)
#pragma unroll
          for (int t = 0; t < TT; ++t)
            acc[t] = epi::multiply<T>(part, of_q[b % 2][t], acc[t]);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const float by = reach[16 * t + c16];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // (the two factors together may be zero, which no infinity survives)
          if (CAREFUL)
            acc[t][r] = acc[t][r] * unscale[r] * by;
          else
            acc[t][r] *= by * unscale[r];
        }
        if (resets != 0) {
          const bool reached = resets_to[16 * t + c16] == 0;
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[t][r] = reached ? acc[t][r] : 0.f;
        }
      }
      fetch_v();
      if constexpr (!CAREFUL) {
#pragma unroll
        for (int b = 0; b < SB; ++b)
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            if (b * KB > 16 * t + 15) continue;
            acc[t] = epi::multiply<T>(
                v_part[b], Weights::rows(p_tile, along_p, t, b), acc[t]);
          }
      } else {
        const int first_value = wave * 16 + 4 * group;
        for (int r = 0; r < n; ++r) {
          typedef T Four __attribute__((ext_vector_type(4)));
          const Four x = *reinterpret_cast<const Four*>(
              v_tile + Values::at(r, first_value / kPer) + first_value % kPer * E);
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            const int to = 16 * t + c16;
            if (r > to || (resets != 0 && resets_to[r] != resets_to[to])) continue;
            const float by = Weights::value(p_tile, to, r);
#pragma unroll
            for (int c = 0; c < 4; ++c)
              acc[t][c] += by * static_cast<float>(x[c]);
          }
        }
      }
      if constexpr (DIRECT) {
        const __amdgpu_buffer_rsrc_t rsrc = epi::make_rsrc(at_out);
        auto all = [&](auto store) {
#pragma unroll
          for (int t = 0; t < TT; ++t)
            store(acc[t], 16 * t + c16 < n ? out_at : epi::kOob,
                  same((from_end ? TT - 1 - t : t) * out_move));
        };
        // (16-byte stores without a scalar offset: with one, registers were written anew
        // before the store had read them, and no wait is put between the two)
        auto floats = [&](float4v x, unsigned at, unsigned up) {
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint4v, x), rsrc,
                                                 at + up, 0, 0);
        };
        if constexpr (E == 4) {
          all(floats);
        } else if (out_float) {
          all(floats);
        } else {
          all([&](float4v x, unsigned at, unsigned up) {
            const float v[4] = {x[0], x[1], x[2], x[3]};
            typedef unsigned int uint2v __attribute__((ext_vector_type(2)));
            __builtin_amdgcn_raw_buffer_store_b64(
                __builtin_bit_cast(uint2v, seq::pack<T, 4>(v)), rsrc, at, up, 0);
          });
        }
      } else if (out_at != epi::kOob) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          if (16 * t + c16 >= n) continue;
          auto store = [&](auto* out) {
            typedef std::remove_pointer_t<decltype(out)> O;
            if (col0 + 4 * group + 4 <= w.values) {
              float x[4] = {acc[t][0], acc[t][1], acc[t][2], acc[t][3]};
              *reinterpret_cast<typename seq::Pack<O, 4>::type*>(out) =
                  seq::pack<O, 4>(x);
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (col0 + 4 * group + r < w.values)
                  out[r] = static_cast<O>(acc[t][r]);
            }
          };
          char* const at =
              at_out + ((from_end ? TT - 1 - t : t) * static_cast<long>(out_move) +
                        out_at);
          if (out_float)
            store(reinterpret_cast<float*>(at));
          else
            store(reinterpret_cast<T*>(at));
        }
      }
      at_out += out_step;
    }

    // The state behind the block.
    carried = carried && all_resets == 0;
    const float carry = power[n];
    if (!CAREFUL && all_resets != 0) look();
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) state[i][r] *= carry;
    if (all_resets != 0) {  // by selection: no infinity passes a reset
      unsigned none = 0;
      asm volatile("" : "+s"(none));  // (or zeros for this would be made in every block)
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          state[i][r] = __uint_as_float(__float_as_uint(state[i][r]) & none);
    }
    if constexpr (!CAREFUL) {
      // (rows in front of a reset may hold a k that a weight of zero leaves infinite)
      if (resets != 0) {
#pragma unroll
        for (int u = 0; u < Keys::kPieces / WAVES; ++u) {
          float x[kPer];
          Split<T>::floats(*reinterpret_cast<const uint4v*>(
                               k_tile + Keys::at(lane % C, wave + u * WAVES)),
                           x);
#pragma unroll
          for (int i = 0; i < kPer; ++i) clean_k = clean_k && x[i] * 0.f == 0.f;
        }
      }
      // (weighted values in full, as the states that leave the kernel are fp32.  With two
      // parts of bfloat16 these were off by 2.4e-6 instead of 2e-7, and 1 x 32768 steps of
      // 16 heads of 128 channels took 215 us instead of 224)
      // (binary16: a value's column times a power of two, which its sums of the block
      // lose again, as the second part of small values would be below the type's
      // smallest: gradients of 1e-3 left states that were off by 4e-4.  1 x 32768 steps of
      // 16 heads of 128 channels 247 us, 229 without, gradients of 4 x 4096 294 and 270; 64 x
      // 512 of 64 channels 84 and 81, gradients 181 and 172)
      constexpr int kParts = Split<T>::kWhole;
      uint4v parts[SB][kParts];
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        if (kScaled) asm volatile("" : "+v"(v_part[b]));  // (worked out again, not kept)
        float x[kPer];
        weighted(b, x);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (kScaled) x[i] *= range;
        Split<T>::split(x, parts[b]);
      }
      // (two tiles' fragments are read while those before are multiplied, and no more of
      // them: they would take the registers that the loads' and sums' need.  Scaled sums
      // join the state while the next are multiplied; without outputs, where twice as many
      // waves share a SIMD's registers, a tile at a time and at once)
      constexpr bool kFewer = kScaled && !OUTPUT;
      constexpr int kStep = kFewer ? 1 : 2, kBehind = kFewer ? 0 : kStep;
      uint4v of_k[2][kStep][SB];
      float4v sums[2][kStep];
      auto fetch = [&](int i) {
#pragma unroll
        for (int u = 0; u < kStep; ++u)
#pragma unroll
          for (int b = 0; b < SB; ++b)
            of_k[i / kStep % 2][u][b] = Keys::columns(
                k_tile, down_k, (i + u) / HALVES, (i + u) % HALVES, b);
      };
      auto join = [&](int i) {
#pragma unroll
        for (int u = 0; u < kStep; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            state[i + u][r] += range_back * sums[i / kStep % 2][u][r];
      };
      fetch(0);
#pragma unroll
      for (int i = 0; i < D / 16; i += kStep) {
        if (i + kStep < D / 16) fetch(i + kStep);
        __builtin_amdgcn_sched_barrier(0);
        float4v (&to)[kStep] = sums[i / kStep % 2];
#pragma unroll
        for (int u = 0; u < kStep; ++u)
          to[u] = kScaled ? float4v{0.f, 0.f, 0.f, 0.f} : state[i + u];
#pragma unroll
        for (int b = 0; b < SB; ++b)
#pragma unroll
          for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int u = 0; u < kStep; ++u)
              to[u] = epi::multiply<T>(of_k[i / kStep % 2][u][b], parts[b][part], to[u]);
        if constexpr (kScaled) {
          if (i >= kBehind) join(i - kBehind);
        } else {
#pragma unroll
          for (int u = 0; u < kStep; ++u) state[i + u] = to[u];
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (kScaled && kBehind > 0) join(D / 16 - kBehind);
    } else {
      const int value = wave * 16 + c16;
      for (int r = 0; r < n; ++r) {
        if (resets != 0 && resets_to[r] != all_resets) continue;
        const float x = into_state[r] * Values::value(v_tile, r, value);
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
          float of_k[kPer];  // the lane's keys of the block: a piece
          Split<T>::floats(*reinterpret_cast<const uint4v*>(
                               k_tile + Keys::at(r, 4 * b + group)),
                           of_k);
#pragma unroll
          for (int i = 0; i < kPer; ++i)  // (keys that do not exist stay zero)
            if (b * KB + group * kPer + i < w.keys)
              state[b * HALVES + i / 4][i % 4] += x * of_k[i];
        }
      }
    }
  };

  constexpr auto kFast = std::false_type();
  constexpr auto kCareful = std::true_type();
  start();
  rewind();
  if constexpr (DIRECT && STAGES == 1) {
    for (int place = first; place < last; place += C) {
      load_reset(place);
      issue(place, ring0);
      __builtin_amdgcn_s_waitcnt(epi::vmcnt_imm(0));
      asm volatile("" ::: "memory");
      if (place == first) look_first();
      walk(ring0, place, kFast, [] {});
      __syncthreads();  // the tiles have been read
    }
  } else if constexpr (DIRECT) {
    constexpr int kLoads = kLoadsV + kLoadsK * (OUTPUT ? 2 : 1);
    if (first < last) load_reset(first);
#pragma unroll
    for (int u = 0; u < STAGES - 1; ++u) issue(first + u * C, ring(u));
    // (the state has come: the compiler would wait for it inside of the loop, in every
    // block, and so for the blocks under way)
    __builtin_amdgcn_s_waitcnt(epi::vmcnt_imm(0));
    look_first();
    auto step = [&](int place, int u) {
      // (loads come in order: where no more accesses are under way than the loads of the
      // blocks behind, the block's own have come, whatever has become of stores)
      __builtin_amdgcn_s_waitcnt(epi::vmcnt_imm((STAGES - 2) * kLoads));
      asm volatile("" ::: "memory");
      walk(ring(u), place, kFast, [&] {
        load_reset(place + C);
        issue(place + (STAGES - 1) * C, ring((u + STAGES - 1) % STAGES));
      });
    };
    for (int place = first; place < last; place += STAGES * C) {
#pragma unroll
      for (int u = 0; u < STAGES; ++u)
        if (place + u * C < last) step(place + u * C, u);
    }
  } else {
    if (first < last) {
      load_reset(first);
      load(first);
    }
    for (int place = first; place < last; place += C) {
      if (place == first) look_first();
      put(place, ring0);
      walk(ring0, place, kFast, [&] {
        if (place + C < last) {
          load_reset(place + C);
          load(place + C);
        }
      });
      __syncthreads();  // the tiles have been read
    }
  }
  // Values that are not finite: once more, and with care.
  look();
  const bool all_clean = clean_k && clean[0] == 0.f && clean[1] == 0.f &&
                         clean[2] == 0.f && clean[3] == 0.f;
  if (__builtin_amdgcn_readfirstlane(__syncthreads_and(all_clean)) == 0) {
    start();
    rewind();
    carried = true;
#pragma unroll 1
    for (int place = first; place < last; place += C) {
      load_reset(place);
      if constexpr (DIRECT) {
        issue(place, ring0);
        __builtin_amdgcn_s_waitcnt(epi::vmcnt_imm(0));
        asm volatile("" ::: "memory");
      } else {
        load(place);
        put(place, ring0);
      }
      walk(ring0, place, kCareful, [] {});
      __syncthreads();  // the tiles have been read
    }
  }

  if (OUTPUT && w.out != nullptr) {  // rows behind the sequence's length
    const int end = min(first + p.piece_steps, p.steps);
    const int columns = min(BV, there);
    const long rows = end - max(first, length);
    for (long at = tid; at < rows * columns; at += kThreads) {
      const long to =
          (row_base + max(first, length) + at / columns) * w.out_row +
          static_cast<long>(part.h) * w.values + value0 + at % columns;
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
  const __amdgpu_buffer_rsrc_t rsrc = state_buffer(to);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      __builtin_amdgcn_raw_buffer_store_b32(
          __float_as_uint(state[i][r]), rsrc,
          state_offset(key_of(i) + r, 4 * w.values, 4), 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <typename T, int D, int WAVES, bool OUTPUT, int RING>
__global__ void __launch_bounds__(64 * WAVES, (kWavesOfSimd<T, D, WAVES, OUTPUT, RING>))
    walk_kernel(Problem p) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int E = sizeof(T), C = kBlock<T>;
  constexpr int kStage = C * E * ((OUTPUT ? 2 : 1) * D + 16 * WAVES);
  // (an array of its own for each block)
  __shared__ __align__(1024) char ring0[kStage];
  char *r1 = nullptr, *r2 = nullptr;
  if constexpr (RING > 1) {
    __shared__ __align__(1024) char ring1[kStage];
    r1 = ring1;
  }
  if constexpr (RING > 2) {
    __shared__ __align__(1024) char ring2[kStage];
    r2 = ring2;
  }
  __shared__ __align__(1024) char p_tile[OUTPUT ? C * C * E : 16];
  __shared__ __align__(16) float power[5 * C + 4];
  __shared__ int resets_to[2 * C];  // in front of a row that count against it
  walk_body<T, D, WAVES, OUTPUT, RING>(p, ring0, r1, r2, p_tile, power, resets_to);
#endif
}

template <typename T, int D, int WAVES, bool OUTPUT, int RING>
int launch_ring(const Problem& p, unsigned groups, hipStream_t stream) {
  hipLaunchKernelGGL((walk_kernel<T, D, WAVES, OUTPUT, RING>), dim3(groups),
                     dim3(64 * WAVES), 0, stream, p);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}
// The blocks of the ring.  LDS holds three of 128 keys, q and 128 values, and for walks
// without q two work-groups of a CU with two each (outputs of 1 x 32768 steps of 16 heads
// of 128 channels in bfloat16: 166 us while every block waited for the next as well, 149
// with three under way).  Work-groups of four waves have two where they do not fill the
// CUs three deep, otherwise one, loaded when the one before has been used.  (us for 256,
// 512, 640, 768, 1024, 2048 work-groups with 1024 steps of 64 channels, one and two:
// bfloat16 46 and 40, 65 and 58, 86 and 102, 97 and 107, 149 and 125, 250 and 239; gradients
// 44 and 40, 53 and 51, 65 and 82, 74 and 85, 120 and 106, 217 and 214; fp32 101 and 81, 145
// and 137, 187 and 198, 203 and 209, 286 and 273, 529 and 535.  The rule leaves a sixth of
// the time around 1024.  fp32 heads of 128 channels, one work-group a CU: 105 and 107.)
inline int ring_of(int keys_class, int waves, bool outputs, bool direct,
                   unsigned groups) {
  if (!direct) return 0;
  if (waves == 8 && keys_class <= 128) return outputs ? 3 : 2;
  return keys_class > 64 || groups > 512 ? 1 : 2;
}
template <typename T, int D, int WAVES, bool OUTPUT, bool DIRECT>
int launch_as(const Problem& p, hipStream_t stream) {
  const unsigned groups =
      static_cast<unsigned>(p.units) * p.batch * p.heads * p.pieces;
  if constexpr (!DIRECT) {
    return launch_ring<T, D, WAVES, OUTPUT, 0>(p, groups, stream);
  } else if constexpr (WAVES == 8 && D <= 128) {
    return launch_ring<T, D, WAVES, OUTPUT, OUTPUT ? 3 : 2>(p, groups, stream);
  } else if constexpr (D > 64) {
    return launch_ring<T, D, WAVES, OUTPUT, 1>(p, groups, stream);
  } else {
    return ring_of(D, WAVES, OUTPUT, DIRECT, groups) == 2
               ? launch_ring<T, D, WAVES, OUTPUT, 2>(p, groups, stream)
               : launch_ring<T, D, WAVES, OUTPUT, 1>(p, groups, stream);
  }
}
template <typename T, int D, int WAVES, bool DIRECT>
int launch_walk(const Problem& p, bool outputs, hipStream_t stream) {
  return outputs ? launch_as<T, D, WAVES, true, DIRECT>(p, stream)
                 : launch_as<T, D, WAVES, false, DIRECT>(p, stream);
}

// Whether all walks' rows go straight to LDS and from registers in whole pieces.
template <typename T>
bool is_direct(const Problem& p, bool outputs) {
  constexpr int kPer = 16 / sizeof(T);
  auto ok = [](const void* at, long stride) {
    return seq::aligned(static_cast<const char*>(at), 16) && stride % kPer == 0;
  };
  for (int i = 0; i < p.walks; ++i) {
    const Walk& w = p.walk[i];
    if (w.keys % kPer != 0 || w.values % kPer != 0 || !ok(w.k, w.k_row) ||
        !ok(w.v, w.v_row))
      return false;
    if (outputs && (!ok(w.q, w.q_row) || !ok(w.out, w.out_row))) return false;
  }
  return true;
}

template <typename T, bool DIRECT>
int run_class(const Problem& p, int keys_class, int waves, bool outputs,
              hipStream_t stream) {
  switch (keys_class) {
    case 64:
      if constexpr (sizeof(T) == 2)
        if (waves == 8) return launch_walk<T, 64, 8, DIRECT>(p, outputs, stream);
      return launch_walk<T, 64, 4, DIRECT>(p, outputs, stream);
    case 128:
      if constexpr (sizeof(T) == 2)
        if (waves == 8) return launch_walk<T, 128, 8, DIRECT>(p, outputs, stream);
      return launch_walk<T, 128, 4, DIRECT>(p, outputs, stream);
    default:
      if constexpr (sizeof(T) == 2)
        if (waves == 8) return launch_walk<T, 256, 8, DIRECT>(p, outputs, stream);
      return launch_walk<T, 256, 4, DIRECT>(p, outputs, stream);
  }
}
template <typename T>
int run_walks(const Problem& p, int keys_class, int waves, bool outputs,
              hipStream_t stream) {
  return is_direct<T>(p, outputs)
             ? run_class<T, true>(p, keys_class, waves, outputs, stream)
             : run_class<T, false>(p, keys_class, waves, outputs, stream);
}

}  // namespace att
}  // namespace snn

#endif  // PORTDNN_AMD_CSRC_LINEAR_ATTENTION_H_
