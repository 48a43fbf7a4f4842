// Matrix product with its epilogue, and the product of its gradients:
//
//   C[m][n] = act(sum over r of P[m][r] Q[n][r] + bias[n]) + residual[m][n]
//
// on the matrix instructions of gfx950: v_mfma_f32_16x16x32_{f16,bf16} for the
// 16-bit types, v_mfma_f32_16x16x4_f32 for fp32, sums in fp32.  Both operands
// come in either order in memory, the reduction contiguous ("K inner") or the
// row, so that the forward product of any transposition and the two products of
// its gradients, whose operands are the forward ones read the other way, run on
// the same kernel without a copy.
//
// A work-group owns a BM x BN tile of C and a range of the reduction, which it
// walks in chunks of CB = 128 or 64 bytes (64 or 32 16-bit values).  A chunk of P and Q
// goes to LDS, STAGES chunks in a ring:
//
//   K inner    [BM rows][CB bytes]; a fragment is one 16-byte read per lane
//   row inner  [reductions][BM values]; 16-bit fragments are two
//              transposing reads (ds_read_b64_tr_b16: within 16 lanes, lane
//              4 j + i supplies the address of four values of reduction j and
//              lane t receives column t of reductions 0 ... 3), floats four
//              4-byte reads
//
// 16-byte pieces are XOR-swizzled so that lanes that read together fall into
// different banks (swizzle() below).  Where rows start at multiples of 16 bytes
// the loads go from memory straight to LDS and the swizzle is applied to their
// source; elsewhere they pass through registers, or the operand is copied first to
// aligned rows, whichever the estimate finds faster.
//
// Q is the instruction's A operand, so a lane ends up with four neighbouring
// columns of a row.  The tile leaves through LDS, each wave's part in its own
// place: there a lane picks up eight neighbouring columns, for which the bias, the
// residual, the activation and the rounding are one piece of code, and stores
// whole rows.
//
// Products of a few rows are bound by the bytes of Q, large ones by the matrix
// instructions, those between by their first chunks' way from memory and by the
// way out, which nothing overlaps where the tiles fill the GPU once.  Measured:
//
//   1 x 2048 x 8192 bfloat16, silu      9.5 us    34 MB at 3.5 TB/s
//   24 x 4096 x 4096 binary16           8.8 us    34 MB at 3.9 TB/s
//   4095 x 1023 x 1001 binary16, gelu  21.2 us    396 TFLOP/s
//   4096 x 1024 x 1024 fp32            68.7 us    125 TFLOP/s
//   8192 x 4096 x 8192 bfloat16        411-441 us 1.25-1.34 PFLOP/s; 468 with
//                                      gelu_tanh and what it is taken of stored
#ifndef PORTDNN_AMD_CSRC_GEMM_EPILOGUE_H_
#define PORTDNN_AMD_CSRC_GEMM_EPILOGUE_H_

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gemm_tile.h"
#include "sequence.h"

namespace snn {
namespace epi {

typedef float float4v __attribute__((ext_vector_type(4)));
typedef unsigned int uint4v __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(3))) short4v* lds_short4_ptr;

// One product with its epilogue.  Sizes and strides in elements.
struct Product {
  const void *p, *q;
  long p_stride, q_stride;
  int m, n, k;  // k: the reduction
  bool p_k_inner, q_k_inner;
  const void *bias, *residual;
  void *out, *pre;
  long residual_stride, out_stride, pre_stride;
  int activation;
  // division of the work
  int tiles_m, tiles_n, splits, split_chunks;  // chunks of a share
  float* partial;                              // [splits][m][n]
};

int run_f32(Product& g, void* workspace, size_t bytes, hipStream_t stream);
int run_f16(Product& g, void* workspace, size_t bytes, hipStream_t stream);
int run_bf16(Product& g, void* workspace, size_t bytes, hipStream_t stream);
// Bytes of workspace that a product makes use of; goes by its sizes, strides and
// orders alone.
size_t workspace_bytes(const Product& g, int elem_size);

// Phi(-|z|), the normal distribution's tail, and e = exp(-z^2 / 2) of it.  With
// t = |z| / sqrt(2) the tail is e erfcx(t) / 2, and erfcx(t) = u P(u) with
// u = 1 / (1 + 0.48 t): a polynomial that was fitted to the least relative error
// over 0 <= t <= 11, 4.5e-8 (the tail's own rounding, t^2 2^-24, is above that from
// |z| = 1 on).  A third of erff's instructions, and no cancellation for negative z:
// the way out of a 4095 x 1023 x 1001 product waited for them.
__device__ __forceinline__ float normal_tail(float z, float* e) {
  const float t = fabsf(z) * 0.70710678118654752f;
  const float u = __builtin_amdgcn_rcpf(1.f + 0.48f * t);
  float q = -0.0501767740f;
  q = q * u + 0.270425839f;
  q = q * u - 0.532466997f;
  q = q * u + 0.392529913f;
  q = q * u - 0.0812016915f;
  q = q * u + 0.227616447f;
  q = q * u + 0.230840945f;
  q = q * u + 0.271655724f;
  q = q * u + 0.270776638f;
  *e = __expf(-t * t);
  return 0.5f * q * u * *e;
}

template <int KIND>
__device__ __forceinline__ float activate(float z) {
  if constexpr (KIND == SNN_HIP_ACTIVATION_RELU) {
    return z < 0.f ? 0.f : z;  // (a NaN stays)
  } else if constexpr (KIND == SNN_HIP_ACTIVATION_GELU) {
    float e;
    const float tail = normal_tail(z, &e);
    return z * (z > 0.f ? 1.f - tail : tail);
  } else {
    // (1 + tanh(u)) / 2 = sigmoid(2 u)
    float s, rest;
    seq::sigmoid<float>(
        KIND == SNN_HIP_ACTIVATION_SILU
            ? z
            : 1.5957691216057308f * (z + 0.044715f * z * z * z),
        &s, &rest);
    return z * s;
  }
}
// (the kind is the same for all lanes: one branch for all N)
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int kind) {
  auto all = [&](auto k) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = activate<decltype(k)::value>(v[i]);
  };
  switch (kind) {
    case SNN_HIP_ACTIVATION_RELU:
      all(std::integral_constant<int, SNN_HIP_ACTIVATION_RELU>());
      break;
    case SNN_HIP_ACTIVATION_GELU:
      all(std::integral_constant<int, SNN_HIP_ACTIVATION_GELU>());
      break;
    case SNN_HIP_ACTIVATION_GELU_TANH:
      all(std::integral_constant<int, SNN_HIP_ACTIVATION_GELU_TANH>());
      break;
    case SNN_HIP_ACTIVATION_SILU:
      all(std::integral_constant<int, SNN_HIP_ACTIVATION_SILU>());
      break;
    default:
      break;
  }
}

__device__ __forceinline__ float activation_slope(float z, int kind) {
  switch (kind) {
    case SNN_HIP_ACTIVATION_RELU:
      return z > 0.f ? 1.f : 0.f;
    case SNN_HIP_ACTIVATION_GELU: {
      float e;
      const float tail = normal_tail(z, &e);
      return (z > 0.f ? 1.f - tail : tail) + z * 0.39894228040143268f * e;
    }
    case SNN_HIP_ACTIVATION_GELU_TANH: {
      float s, rest;
      seq::sigmoid<float>(
          1.5957691216057308f * (z + 0.044715f * z * z * z), &s, &rest);
      // (s * rest is exactly zero long before |z| = 64, and would be multiplied by an
      // infinite z^2 from 1.8e19 on)
      const float near = fminf(fmaxf(z, -64.f), 64.f);
      return s + near * s * rest * 1.5957691216057308f *
                     (1.f + 0.134145f * near * near);
    }
    case SNN_HIP_ACTIVATION_SILU: {
      float s, rest;
      seq::sigmoid<float>(z, &s, &rest);
      return s + z * s * rest;
    }
    default:
      return 1.f;
  }
}

// Eight neighbouring columns of a row: bias, activation, residual, one rounding.
// Rows may start anywhere (see Pack).
template <typename T>
__device__ __forceinline__ void finish8(const Product& g, int row, int col,
                                        float (&v)[8]) {
  constexpr int VEC = 16 / sizeof(T);
  typedef typename seq::Pack<T, VEC>::type V;
  const T* const bias = static_cast<const T*>(g.bias);
  const T* const residual =
      g.residual == nullptr
          ? nullptr
          : static_cast<const T*>(g.residual) + row * g.residual_stride;
  T* const pre =
      g.pre == nullptr ? nullptr : static_cast<T*>(g.pre) + row * g.pre_stride;
  T* const out = static_cast<T*>(g.out) + row * g.out_stride;
  if (col + 8 <= g.n) {
    auto load = [&](const T* from, float (&to)[8]) {
#pragma unroll
      for (int j = 0; j < 8; j += VEC) {
        float part[VEC];
        seq::unpack<T, VEC>(*reinterpret_cast<const V*>(from + col + j), part);
#pragma unroll
        for (int i = 0; i < VEC; ++i) to[j + i] = part[i];
      }
    };
    auto store = [&](T* to, const float (&from)[8]) {
#pragma unroll
      for (int j = 0; j < 8; j += VEC) {
        float part[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) part[i] = from[j + i];
        *reinterpret_cast<V*>(to + col + j) = seq::pack<T, VEC>(part);
      }
    };
    float add[8];
    if (bias != nullptr) {
      load(bias, add);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += add[i];
    }
    if (pre != nullptr) store(pre, v);
    if (residual != nullptr) load(residual, add);
    activate(v, g.activation);
    if (residual != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += add[i];
    }
    store(out, v);
    return;
  }
  // (a row's last columns, one at a time; the values move up, as an index that is
  // not known when compiled would put them into LDS)
#pragma unroll 1
  for (; col < g.n; ++col) {
    float z[1] = {v[0]};
#pragma unroll
    for (int i = 0; i < 7; ++i) v[i] = v[i + 1];
    if (bias != nullptr) z[0] += static_cast<float>(bias[col]);
    if (pre != nullptr) pre[col] = static_cast<T>(z[0]);
    activate(z, g.activation);
    if (residual != nullptr) z[0] += static_cast<float>(residual[col]);
    out[col] = static_cast<T>(z[0]);
  }
}

// Shares of a reduction are multiples of this many bytes of a row.
constexpr int kChunkBytes = 128;
constexpr unsigned kOob = 0x80000000u;  // beyond every buffer's range

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0x7FFFFFF0,
                                           0x00020000);
}

constexpr int vmcnt_imm(int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); }
constexpr int kLgkm0 = ~0x0F00;  // ... and all LDS reads, by &

// Eight neighbouring columns of a tile: the result, or a share of its sums.
template <typename T>
__device__ __forceinline__ void leave(const Product& g, unsigned split, int row,
                                      int col, float (&v)[8]) {
  if (g.splits == 1) {
    finish8<T>(g, row, col, v);
    return;
  }
  float* const to =
      g.partial + (static_cast<long>(split) * g.m + row) * g.n + col;
  if (col + 8 <= g.n) {
    typedef seq::Pack<float, 4>::type F;  // (rows may start anywhere)
    *reinterpret_cast<F*>(to) = F{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<F*>(to + 4) = F{v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < g.n) to[i] = v[i];
  }
}

// Which 16-byte position of its row holds piece c: c ^ swizzle(row).
//   K inner: the 16 rows of a fragment, two (four) of which fill the 64 banks.
//   Lanes that read together are rows 0 ... 3 and 12 ... 15 of one piece and 4 ...
//   11 of the next; with four rows a bank row that takes the order 0, 2, 3, 1.
//   row inner, 16-bit: the four reductions of a transposing read by the two
//   blocks of eight, 32 bytes each.
//   row inner, floats: four blocks of four reductions, 64 bytes each.
template <int E, bool K_INNER, int ROWS, int CB>
__device__ __forceinline__ constexpr unsigned swizzle(unsigned row) {
  if (K_INNER) {
    if (CB == 128) return (row >> 1) & 7u;
    const unsigned four = (row >> 2) & 3u;
    return (((four ^ (four >> 1)) & 1u) << 1) | (four >> 1);
  }
  constexpr int kPitch = ROWS * E;
  if (E == 2) {
    if (kPitch >= 256) return 2u * ((row & 3u) | (((row >> 3) & 1u) << 2));
    if (kPitch == 128)
      return 2u * (((row >> 1) & 1u) | (((row >> 3) & 1u) << 1));
    return 0;
  }
  if (kPitch >= 256) return 4u * ((row >> 2) & 3u);
  if (kPitch == 128) return 4u * ((row >> 2) & 1u);
  return 0;
}

// One operand's tile: ROWS rows of the result's dimension by a chunk of CB bytes
// of the reduction.
template <typename T, bool K_INNER, int ROWS, int CB>
struct Operand {
  static constexpr int E = sizeof(T);
  static constexpr bool kInner = K_INNER;
  static constexpr int kRows = ROWS;
  static constexpr int kBlocks = ROWS * CB / 1024;  // of 1 KiB
  static constexpr int kPitch = K_INNER ? CB : ROWS * E;
  static constexpr int kPiece = 16 / E;  // values
  static constexpr int kChunk = CB / E;

  // Row and column (in values) of the tile's memory that LDS position `pos`
  // holds.
  static __device__ __forceinline__ void source(unsigned pos, int* row,
                                                int* col) {
    const unsigned r = pos / kPitch;
    const unsigned piece = (pos % kPitch) >> 4;
    *row = static_cast<int>(r);
    *col = static_cast<int>((piece ^ swizzle<E, K_INNER, ROWS, CB>(r)) * kPiece);
  }
  static __device__ __forceinline__ const T* at(const void* p, long stride,
                                                int row0, int k0) {
    return static_cast<const T*>(p) +
           (K_INNER ? row0 * stride + k0 : k0 * stride + row0);
  }

  // LDS address of the lane's part of the fragment of rows row0 ... row0 + 15
  // (step 0); K inner: step s is at the address ^ 64 s, row inner:
  // at + s * kStep.
  static __device__ __forceinline__ unsigned fragment(int row0, int lane) {
    if (K_INNER) {
      const unsigned row = row0 + (lane & 15);
      return row * CB +
             (((lane >> 4) ^ swizzle<E, true, ROWS, CB>(row)) << 4);
    }
    if (E == 2) {
      const unsigned k = 8 * (lane >> 4) + ((lane >> 2) & 3);
      const unsigned piece = row0 / 8 + ((lane & 3) >> 1);
      return k * kPitch + ((piece ^ swizzle<E, false, ROWS, CB>(k)) << 4) +
             ((lane & 1) << 3);
    }
    const unsigned k = 4 * (lane >> 4);
    const unsigned piece = row0 / 4 + ((lane & 15) >> 2);
    return k * kPitch + ((piece ^ swizzle<E, false, ROWS, CB>(k)) << 4) +
           ((lane & 3) << 2);
  }
  static __device__ __forceinline__ uint4v read(const char* tile, unsigned at,
                                                int s) {
    if constexpr (K_INNER) {
      return *reinterpret_cast<const uint4v*>(tile + (at ^ (s << 6)));
    } else if constexpr (E == 2) {
      const char* const from = tile + at + s * (32 * kPitch);
      const short4v lo =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_ptr)(from));
      const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_short4_ptr)(from + 4 * kPitch));
      return __builtin_bit_cast(
          uint4v, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const char* const from = tile + at + s * (16 * kPitch);
      uint4v v;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        v[t] = *reinterpret_cast<const unsigned*>(from + t * kPitch);
      return v;
    }
  }
};

template <typename T>
__device__ __forceinline__ float4v multiply(uint4v q, uint4v p, float4v acc);
template <>
__device__ __forceinline__ float4v multiply<_Float16>(uint4v q, uint4v p,
                                                      float4v acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(
      __builtin_bit_cast(half8, q), __builtin_bit_cast(half8, p), acc, 0, 0, 0);
}
template <>
__device__ __forceinline__ float4v multiply<__bf16>(uint4v q, uint4v p,
                                                    float4v acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      __builtin_bit_cast(bf16x8, q), __builtin_bit_cast(bf16x8, p), acc, 0, 0,
      0);
}
// (four instructions over four reductions each: lane group g holds reductions
// 4 g ... 4 g + 3 of the step's 16, instruction t takes the t-th of each)
template <>
__device__ __forceinline__ float4v multiply<float>(uint4v q, uint4v p,
                                                   float4v acc) {
  const float4v a = __builtin_bit_cast(float4v, q);
  const float4v b = __builtin_bit_cast(float4v, p);
#pragma unroll
  for (int t = 0; t < 4; ++t)
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], b[t], acc, 0, 0, 0);
  return acc;
}

// LDS of a work-group: the ring of chunks, rounded up so that every wave issues
// the same number of loads, or the tile on its way out.
template <int BM, int BN, int WAVES, int CB>
struct Space {
  static constexpr int kBlocks = (BM + BN) * CB / 1024;
  static constexpr int kLoads = (kBlocks + WAVES - 1) / WAVES;  // per wave
  static constexpr int kStage = kLoads * WAVES * 1024;
};

// (v >> 8 * bytes), zeros from above.
__device__ __forceinline__ uint4v shifted_down(uint4v v, int bytes) {
  typedef unsigned long long Two __attribute__((ext_vector_type(2)));
  Two w = __builtin_bit_cast(Two, v);
  if (bytes >= 8) {
    w = Two{w[1], 0ull};
    bytes -= 8;
  }
  if (bytes >= 8) w = Two{0ull, 0ull};
  if (bytes > 0 && bytes < 8) {
    w[0] = w[0] >> (8 * bytes) | w[1] << (64 - 8 * bytes);
    w[1] >>= 8 * bytes;
  }
  return __builtin_bit_cast(uint4v, w);
}

// The product of a tile by waves that walk the reduction together.  HELD = 0: whole
// 16-byte pieces at aligned addresses, which go straight to a ring of STAGES chunks
// in LDS.  Otherwise rows of at least 16 bytes at any address by way of registers,
// where HELD chunks are under way; LDS holds STAGES = 2.
template <typename T, bool PK, bool QK, int BM, int BN, int WM, int WN,
          int CB, int STAGES, int HELD>
__device__ __forceinline__ void gemm_body(const Product& g, char* r0, char* r1,
                                          char* r2, char* r3, char* r4) {
  typedef Operand<T, PK, BM, CB> OP;
  typedef Operand<T, QK, BN, CB> OQ;
  constexpr int WAVES = WM * WN;
  typedef Space<BM, BN, WAVES, CB> S;
  constexpr int TM = BM / WM, TN = BN / WN, IM = TM / 16, IN = TN / 16;
  constexpr int kPBytes = BM * CB;
  constexpr int kChunk = OP::kChunk;
  auto ring = [&](int u) {
    return u == 0 ? r0 : u == 1 ? r1 : u == 2 ? r2 : u == 3 ? r3 : r4;
  };
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;

  // Every XCD takes a run of tiles, in bands of eight tiles of rows, so that the
  // tiles it works on at a time share both operands in its L2.
  const unsigned tiles = static_cast<unsigned>(g.tiles_m) * g.tiles_n;
  const unsigned lin = gemm::xcd_remap(blockIdx.x, tiles * g.splits);
  const unsigned split = lin / tiles, tile = lin - split * tiles;
  constexpr unsigned kBand = 8;
  const unsigned band = tile / (kBand * g.tiles_n);
  const unsigned in_band = tile - band * kBand * g.tiles_n;
  const unsigned height = min(kBand, g.tiles_m - band * kBand);
  const int row0 = static_cast<int>(band * kBand + in_band % height) * BM;
  const int col0 = static_cast<int>(in_band / height) * BN;
  const int share = g.split_chunks * (kChunkBytes / static_cast<int>(sizeof(T)));
  const int k_begin = static_cast<int>(split) * share;
  const int k_end = min(g.k, k_begin + share);
  const int chunks = (k_end - k_begin + kChunk - 1) / kChunk;
  const int rows_left = g.m - row0, cols_left = g.n - col0;

  unsigned at_p[IM], at_q[IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
    at_p[i] = OP::fragment(wm * TM + 16 * i, lane);
#pragma unroll
  for (int j = 0; j < IN; ++j)
    at_q[j] = kPBytes + OQ::fragment(wn * TN + 16 * j, lane);

  float4v acc[IM][IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < IN; ++j) acc[i][j] = float4v{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](const char* tile_at) {
#pragma unroll
    for (int s = 0; s < CB / 64; ++s) {
      uint4v p[IM], q[IN];
#pragma unroll
      for (int j = 0; j < IN; ++j) q[j] = OQ::read(tile_at, at_q[j], s);
#pragma unroll
      for (int i = 0; i < IM; ++i) p[i] = OP::read(tile_at, at_p[i], s);
#pragma unroll
      for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j) acc[i][j] = multiply<T>(q[j], p[i], acc[i][j]);
    }
  };

  int left = chunks;
  if constexpr (HELD == 0) {
    // Offsets of the lane's loads within a chunk; the chunk's own place is in
    // the buffer's base, so that operands may be of any size.
    unsigned offset[S::kLoads];
    int order[S::kLoads];  // its reduction index
#pragma unroll
    for (int l = 0; l < S::kLoads; ++l) {
      const int block = wave + l * WAVES;
      int row, col;
      bool in;
      long stride;
      if (block < OP::kBlocks) {
        OP::source(block * 1024 + lane * 16, &row, &col);
        in = PK ? row < rows_left : col < rows_left;
        stride = g.p_stride;
        order[l] = PK ? col : row;
      } else {
        OQ::source((block - OP::kBlocks) * 1024 + lane * 16, &row, &col);
        in = block < S::kBlocks && (QK ? row < cols_left : col < cols_left);
        stride = g.q_stride;
        order[l] = QK ? col : row;
      }
      offset[l] = in ? static_cast<unsigned>((row * stride + col) * sizeof(T))
                     : kOob;
    }
    const char* from_p =
        reinterpret_cast<const char*>(OP::at(g.p, g.p_stride, row0, k_begin));
    const char* from_q =
        reinterpret_cast<const char*>(OQ::at(g.q, g.q_stride, col0, k_begin));
    const long step_p = PK ? CB : CB * g.p_stride;
    const long step_q = QK ? CB : CB * g.q_stride;
    int k_left = k_end - k_begin;
    auto issue = [&](char* to) {  // the next chunk
      const __amdgpu_buffer_rsrc_t p = make_rsrc(from_p), q = make_rsrc(from_q);
#pragma unroll
      for (int l = 0; l < S::kLoads; ++l) {
        const int block = wave + l * WAVES;
        const unsigned from = order[l] < k_left ? offset[l] : kOob;
        if (block < OP::kBlocks)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              p, (lds_ptr)(to + block * 1024), 16, from, 0, 0, 0);
        else
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              q, (lds_ptr)(to + block * 1024), 16, from, 0, 0, 0);
      }
      from_p += step_p;
      from_q += step_q;
      k_left -= kChunk;
    };
    // STAGES - 1 chunks are under way while one is multiplied; behind the last
    // one the loads are out of range, so that there is always the same number.  A
    // chunk's place is loaded again behind the barrier that every wave reaches
    // when it has read it.  (The places are arrays of their own: the compiler
    // waits for all loads into an array before it reads from it.)
#pragma unroll
    for (int c = 0; c < STAGES - 1; ++c) issue(ring(c));
    auto step = [&](int u) {
      // the chunk is here, and the reads of the one before have returned
      __builtin_amdgcn_s_waitcnt(kLgkm0 & vmcnt_imm((STAGES - 2) * S::kLoads));
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      issue(ring((u + STAGES - 1) % STAGES));
      compute(ring(u));
    };
    for (; left >= STAGES; left -= STAGES) {
#pragma unroll
      for (int u = 0; u < STAGES; ++u) step(u);
    }
#pragma unroll
    for (int u = 0; u < STAGES - 1; ++u)
      if (u < left) step(u);
  } else {
    // Where a piece would reach behind its row's end the row's last 16 bytes are
    // loaded and, on their way into LDS, shifted to where the piece begins: zeros
    // behind the end of a reduction, anything in columns that are not kept.
    constexpr int kLoadsP = OP::kBlocks / WAVES;
    static_assert(OP::kBlocks % WAVES == 0 && OQ::kBlocks % WAVES == 0,
                  "waves load the same number of blocks of each operand");
    int offset[S::kLoads], order[S::kLoads], late[S::kLoads];
#pragma unroll
    for (int l = 0; l < S::kLoads; ++l) {
      auto place = [&](auto o, unsigned pos, bool inner, int there, long stride) {
        typedef decltype(o) O;
        int row, col;
        O::source(pos, &row, &col);
        order[l] = inner ? col : row;
        const int r = inner ? min(row, there - 1) : row;
        const int c = inner ? col : min(col, there - O::kPiece);
        late[l] = (col - c) * static_cast<int>(sizeof(T));
        offset[l] = static_cast<int>((r * stride + c) * sizeof(T));
      };
      const int block = wave + l * WAVES;
      if (l < kLoadsP)
        place(OP(), block * 1024 + lane * 16, PK, rows_left, g.p_stride);
      else
        place(OQ(), (block - OP::kBlocks) * 1024 + lane * 16, QK, cols_left,
              g.q_stride);
    }
    const char* from_p =
        reinterpret_cast<const char*>(OP::at(g.p, g.p_stride, row0, k_begin));
    const char* from_q =
        reinterpret_cast<const char*>(OQ::at(g.q, g.q_stride, col0, k_begin));
    const long step_p = PK ? CB : CB * g.p_stride;
    const long step_q = QK ? CB : CB * g.q_stride;
    int k_left = k_end - k_begin, k_here = k_left;  // to be loaded, to be stored
    uint4v held[HELD][S::kLoads];
    auto load = [&](uint4v (&to)[S::kLoads]) {
      if (k_left > 0) {
#pragma unroll
        for (int l = 0; l < S::kLoads; ++l) {
          const bool of_p = l < kLoadsP;
          const bool inner = of_p ? PK : QK;
          long from = offset[l];
          if (k_left < kChunk) {
            const int over =
                max(0, order[l] - (k_left - (inner ? OP::kPiece : 1)));
            from -= over * (inner ? 1l : of_p ? g.p_stride : g.q_stride) *
                    static_cast<long>(sizeof(T));
          }
          __builtin_memcpy(&to[l], (of_p ? from_p : from_q) + from, 16);
        }
      }
      from_p += step_p;
      from_q += step_q;
      k_left -= kChunk;
    };
    auto step = [&](uint4v (&from)[S::kLoads], char* to) {
#pragma unroll
      for (int l = 0; l < S::kLoads; ++l) {
        const bool of_p = l < kLoadsP;
        uint4v v = from[l];
        if (of_p ? PK : QK) {
          if (k_here < kChunk)
            v = shifted_down(v, max(0, order[l] + OP::kPiece - k_here) *
                                    static_cast<int>(sizeof(T)));
        } else {
          if ((of_p ? rows_left < BM : cols_left < BN))
            v = shifted_down(v, late[l]);
          if (order[l] >= k_here) v = uint4v{0u, 0u, 0u, 0u};
        }
        *reinterpret_cast<uint4v*>(to + (wave + l * WAVES) * 1024 + lane * 16) = v;
      }
      k_here -= kChunk;
      load(from);
      // every wave has stored the chunk, and has read the one before
      __builtin_amdgcn_s_waitcnt(kLgkm0 & vmcnt_imm(63));
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      compute(to);
    };
    static_assert(STAGES == 2 && HELD % 2 == 0, "two chunks in LDS");
#pragma unroll
    for (int u = 0; u < HELD; ++u) load(held[u]);
    for (; left >= HELD; left -= HELD) {
#pragma unroll
      for (int u = 0; u < HELD; ++u) step(held[u], ring(u % 2));
    }
#pragma unroll
    for (int u = 0; u < HELD - 1; ++u)
      if (u < left) step(held[u], ring(u % 2));
  }
  __builtin_amdgcn_s_waitcnt(kLgkm0 & vmcnt_imm(0));

  // The way out.  A wave's part of the tile in passes of kRows rows, a 16-byte
  // piece c of row r at c ^ (r & 15) (& 7 for rows of 32 columns).
  __syncthreads();
  constexpr int kSharers = (WAVES + STAGES - 1) / STAGES;  // of a chunk's place
  constexpr int kSpace = S::kStage / kSharers / 1024 * 1024;
  constexpr int kFit = kSpace / (TN * 4) / 16 * 16;
  constexpr int kRows = TM <= kFit       ? TM
                        : TM / 2 <= kFit ? TM / 2
                                         : TM / 4;
  static_assert(kRows <= kFit && kRows % 16 == 0, "no room for the way out");
  constexpr unsigned kMask = TN / 4 - 1 < 15 ? TN / 4 - 1 : 15;
  char* own = ring(0);
#pragma unroll
  for (int u = 1; u < STAGES; ++u)
    if (wave / kSharers == u) own = ring(u);
  own += wave % kSharers * kSpace;
  constexpr int kLanes = TN / 8;          // of a row
  constexpr int kTurnRows = 64 / kLanes;  // rows at a time
#pragma unroll
  for (int pass = 0; pass < TM / kRows; ++pass) {
#pragma unroll
    for (int i = 0; i < kRows / 16; ++i) {
      const unsigned r = 16 * i + (lane & 15);
#pragma unroll
      for (int j = 0; j < IN; ++j) {
        const unsigned piece = (4 * j + (lane >> 4)) ^ (r & kMask);
        *reinterpret_cast<float4v*>(own + r * (TN * 4) + piece * 16) =
            acc[pass * (kRows / 16) + i][j];
      }
    }
    const int col = col0 + wn * TN + (lane % kLanes) * 8;
#pragma unroll 1
    for (int t = 0; t < kRows; t += kTurnRows) {
      const unsigned r = t + lane / kLanes;
      const int row = row0 + wm * TM + pass * kRows + static_cast<int>(r);
      if (row >= g.m || col >= g.n) continue;
      float v[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned piece = (2 * (lane % kLanes) + h) ^ (r & kMask);
        const float4v f =
            *reinterpret_cast<const float4v*>(own + r * (TN * 4) + piece * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * h + i] = f[i];
      }
      leave<T>(g, split, row, col, v);
    }
  }
}

// A 16-byte piece of an operand's tile from any address, by way of registers.
// Rows (or columns) beyond the operand are others of its rows, whose results are
// not kept; reductions beyond `k_end` are zero.  Where the piece does not exist
// as a whole it is put together from single values, all of them loads of
// existing ones, so that no load waits for another.
template <typename O, typename T>
__device__ __forceinline__ uint4v load_piece(const void* base, long stride,
                                             int left, int first, int k0,
                                             int k_end, unsigned pos) {
  int row, col;
  O::source(pos, &row, &col);
  const int k_left = k_end - k0;
  const T* const from = O::at(base, stride, first, k0);
  uint4v v = {0u, 0u, 0u, 0u};
  if (k_left <= 0) return v;
  // what exists of the tile, rows and columns of memory
  const int rows = O::kInner ? left : k_left;
  const int cols = O::kInner ? k_left : left;
  const T* const line = from + min(row, rows - 1) * stride;
  if (k_left >= O::kChunk && (O::kInner || left >= O::kRows)) {
    __builtin_memcpy(&v, line + col, 16);
    return v;
  }
  T part[O::kPiece];
#pragma unroll
  for (int i = 0; i < O::kPiece; ++i) part[i] = line[min(col + i, cols - 1)];
#pragma unroll
  for (int i = 0; i < O::kPiece; ++i)
    if ((O::kInner ? col + i : row) >= k_left) part[i] = T(0);
  __builtin_memcpy(&v, part, 16);
  return v;
}

// Products of a few rows, which are bound by the bytes of Q.  The work-group's
// waves share the reduction of a BM x BN tile, chunk by chunk in turn, and every
// wave has a ring of its own, so that nothing but its own loads holds it up:
// STAGES chunks of each wave are under way.  Their sums meet in LDS at the end.
template <typename T, bool PK, bool QK, int BM, int BN, int WAVES, int STAGES,
          bool DIRECT>
__device__ __forceinline__ void gemm_few_body(const Product& g, char* r0,
                                              char* r1, char* r2, char* r3) {
  constexpr int CB = kChunkBytes;
  typedef Operand<T, PK, BM, CB> OP;
  typedef Operand<T, QK, BN, CB> OQ;
  constexpr int IM = BM / 16, IN = BN / 16;
  constexpr int kPBytes = BM * CB, kOwn = (BM + BN) * CB;
  constexpr int kLoads = kOwn / 1024, kChunk = OP::kChunk;
  auto ring = [&](int u) { return u == 0 ? r0 : u == 1 ? r1 : u == 2 ? r2 : r3; };
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned tiles = static_cast<unsigned>(g.tiles_m) * g.tiles_n;
  const unsigned lin = gemm::xcd_remap(blockIdx.x, tiles * g.splits);
  const unsigned split = lin / tiles, tile = lin - split * tiles;
  const int row0 = static_cast<int>(tile % g.tiles_m) * BM;
  const int col0 = static_cast<int>(tile / g.tiles_m) * BN;
  const int share = g.split_chunks * kChunk;
  const int k_begin = static_cast<int>(split) * share + wave * kChunk;
  const int k_end = min(g.k, static_cast<int>(split) * share + share);
  const int rows_left = g.m - row0, cols_left = g.n - col0;

  unsigned at_p[IM], at_q[IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
    at_p[i] = wave * kOwn + OP::fragment(16 * i, lane);
#pragma unroll
  for (int j = 0; j < IN; ++j)
    at_q[j] = wave * kOwn + kPBytes + OQ::fragment(16 * j, lane);
  float4v acc[IM][IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < IN; ++j) acc[i][j] = float4v{0.f, 0.f, 0.f, 0.f};

  // The fragments of a chunk, and what becomes of them.
  uint4v p[2][IM], q[2][IN];
  auto fetch = [&](const char* place) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int j = 0; j < IN; ++j) q[s][j] = OQ::read(place, at_q[j], s);
#pragma unroll
      for (int i = 0; i < IM; ++i) p[s][i] = OP::read(place, at_p[i], s);
    }
  };
  auto multiply_all = [&]() {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j)
          acc[i][j] = multiply<T>(q[s][j], p[s][i], acc[i][j]);
  };
  int k_left = k_end - k_begin;  // at the chunk that is loaded next
  int left = (k_left + WAVES * kChunk - 1) / (WAVES * kChunk);

  if constexpr (DIRECT) {
    unsigned offset[kLoads];
    int order[kLoads];
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      int row, col;
      bool in;
      long stride;
      if (l < OP::kBlocks) {
        OP::source(l * 1024 + lane * 16, &row, &col);
        in = PK ? row < rows_left : col < rows_left;
        stride = g.p_stride;
        order[l] = PK ? col : row;
      } else {
        OQ::source((l - OP::kBlocks) * 1024 + lane * 16, &row, &col);
        in = QK ? row < cols_left : col < cols_left;
        stride = g.q_stride;
        order[l] = QK ? col : row;
      }
      offset[l] =
          in ? static_cast<unsigned>((row * stride + col) * sizeof(T)) : kOob;
    }
    const char* from_p =
        reinterpret_cast<const char*>(OP::at(g.p, g.p_stride, row0, k_begin));
    const char* from_q =
        reinterpret_cast<const char*>(OQ::at(g.q, g.q_stride, col0, k_begin));
    const long step_p = WAVES * (PK ? CB : CB * g.p_stride);
    const long step_q = WAVES * (QK ? CB : CB * g.q_stride);
    auto issue = [&](char* to) {
      const __amdgpu_buffer_rsrc_t p = make_rsrc(from_p), q = make_rsrc(from_q);
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const unsigned from = order[l] < k_left ? offset[l] : kOob;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            l < OP::kBlocks ? p : q, (lds_ptr)(to + wave * kOwn + l * 1024), 16,
            from, 0, 0, 0);
      }
      from_p += step_p;
      from_q += step_q;
      k_left -= WAVES * kChunk;
    };
    auto step = [&](char* place) {
      __builtin_amdgcn_s_waitcnt(vmcnt_imm((STAGES - 1) * kLoads));
      asm volatile("" ::: "memory");
      fetch(place);
      // the chunk is in registers before its place is loaded again
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(kLgkm0 & vmcnt_imm(63));
      asm volatile("" ::: "memory");
      issue(place);
      multiply_all();
    };
#pragma unroll
    for (int u = 0; u < STAGES; ++u) issue(ring(u));
    for (; left >= STAGES; left -= STAGES) {
#pragma unroll
      for (int u = 0; u < STAGES; ++u) step(ring(u));
    }
#pragma unroll
    for (int u = 0; u < STAGES - 1; ++u)
      if (u < left) step(ring(u));
  } else {
    // Through registers, STAGES chunks of which are under way; LDS holds one.
    uint4v held[STAGES][kLoads];
    int k0 = k_begin;
    auto load = [&](uint4v (&to)[kLoads]) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        if (l < OP::kBlocks)
          to[l] = load_piece<OP, T>(g.p, g.p_stride, rows_left, row0, k0, k_end,
                                    l * 1024 + lane * 16);
        else
          to[l] = load_piece<OQ, T>(g.q, g.q_stride, cols_left, col0, k0, k_end,
                                    (l - OP::kBlocks) * 1024 + lane * 16);
      }
      k0 += WAVES * kChunk;
    };
    auto step = [&](uint4v (&from)[kLoads]) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l)
        *reinterpret_cast<uint4v*>(r0 + wave * kOwn + l * 1024 + lane * 16) =
            from[l];
      fetch(r0);
      load(from);
      multiply_all();
    };
#pragma unroll
    for (int u = 0; u < STAGES; ++u) load(held[u]);
    for (; left >= STAGES; left -= STAGES) {
#pragma unroll
      for (int u = 0; u < STAGES; ++u) step(held[u]);
    }
#pragma unroll
    for (int u = 0; u < STAGES - 1; ++u)
      if (u < left) step(held[u]);
  }
  __builtin_amdgcn_s_waitcnt(kLgkm0 & vmcnt_imm(0));

  // The waves' tiles, [wave][BM][BN], over the first ring; their sums eight
  // columns at a time.
  __syncthreads();
  static_assert(BM * BN * 4 <= kOwn, "no room for the sums");
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < IN; ++j)
      *reinterpret_cast<float4v*>(r0 + ((wave * BM + 16 * i + (lane & 15)) * BN +
                                        16 * j + 4 * (lane >> 4)) *
                                           4) = acc[i][j];
  __syncthreads();
  for (int e = tid; e < BM * BN / 8; e += 64 * WAVES) {
    const int r = e / (BN / 8), c = e % (BN / 8) * 8;
    const int row = row0 + r, col = col0 + c;
    if (row >= g.m || col >= g.n) continue;
    float v[8] = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float4v* const f = reinterpret_cast<const float4v*>(
          r0 + ((w * BM + r) * BN + c) * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] += f[0][i];
        v[4 + i] += f[1][i];
      }
    }
    leave<T>(g, split, row, col, v);
  }
}

// Adds the shares of a divided reduction in their order and finishes.  (14 x 3490 x
// 876 fp32 in eight shares 13.7 us; one share after another 19.1)
template <typename T>
__global__ void __launch_bounds__(256) gemm_join_kernel(Product g) {
  const int groups = (g.n + 7) / 8;
  const long at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
  const int row = static_cast<int>(at / groups);
  const int col = static_cast<int>(at - static_cast<long>(row) * groups) * 8;
  if (row >= g.m) return;
  const long size = static_cast<long>(g.m) * g.n;
  const float* from = g.partial + static_cast<long>(row) * g.n + col;
  // Four shares at a time, all of whose loads are under way together: behind the
  // last share that one again, which is not added.
  constexpr int kBatch = 4;
  const int last = g.n - 1 - col;
  float v[8] = {};
  auto add = [&](auto fetch) {
    for (int s0 = 0; s0 < g.splits; s0 += kBatch) {
      float part[kBatch][8];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        fetch(from + min(s0 + u, g.splits - 1) * size, part[u]);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (s0 + u < g.splits) v[i] += part[u][i];
    }
  };
  if (last >= 7)
    add([](const float* share, float (&to)[8]) {
      typedef seq::Pack<float, 4>::type F;  // (rows may start anywhere)
      const F a = *reinterpret_cast<const F*>(share);
      const F b = *reinterpret_cast<const F*>(share + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        to[i] = a[i];
        to[4 + i] = b[i];
      }
    });
  else
    add([&](const float* share, float (&to)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) to[i] = share[min(i, last)];
    });
  finish8<T>(g, row, col, v);
}

// The kernels of a product: tiles of work-groups that walk the reduction
// together, tiles whose waves share it (for few rows), and those that take rows at
// any address.
enum Kernel {
  kFew16x16,
  kFew16x32,
  kFew32x32,
  kFew64x32,
  kTile64x128,
  kTile128,
  kTile128Pair,  // two work-groups of a CU
  kTile256,
  kAny16x16,
  kAny32x32,
  kAny64x32,
  kAnyTile128,  // rows of 16 bytes at least, tiles within 31 bits
  kKernels
};

// What the choice goes by, measured: microseconds of a round of `slots`
// work-groups that does not go into its steps, and of a step (`chunks` 128-byte
// chunks of the reduction) with Q K inner and row inner; 0: not for this type.
// `waves` of a work-group, at most.
struct Shape {
  int bm, bn, chunks, slots, waves;
  float fixed, step_k, step_row;
};
constexpr Shape kShapes16[kKernels] = {
    {16, 16, 4, 384, 4, 2.3f, 0.43f, 0.6f}, {16, 32, 4, 256, 4, 2.5f, 0.49f, 0.62f},
    {32, 32, 4, 256, 4, 2.5f, 0.42f, 0.7f}, {64, 32, 4, 256, 4, 2.8f, 0.55f, 0.88f},
    {64, 128, 1, 256, 8, 4.3f, 0.24f, 0.24f}, {128, 128, 1, 256, 8, 5.2f, 0.42f, 0.42f},
    {128, 128, 1, 512, 8, 5.0f, 0.92f, 0.92f}, {256, 256, 1, 256, 16, 8.0f, 1.5f, 1.5f},
    {16, 16, 4, 768, 4, 3.0f, 0.6f, 1.2f}, {32, 32, 8, 256, 8, 3.0f, 1.8f, 5.5f},
    {64, 32, 4, 256, 4, 3.0f, 1.55f, 3.6f}, {128, 128, 1, 256, 16, 5.0f, 0.78f, 0.78f}};
constexpr Shape kShapes32[kKernels] = {
    {16, 16, 4, 384, 4, 2.3f, 0.33f, 0.5f}, {16, 32, 4, 256, 4, 2.5f, 0.45f, 0.72f},
    {32, 32, 4, 256, 4, 2.5f, 0.6f, 0.8f}, {64, 32, 4, 256, 4, 0.f, 0.f, 0.f},
    {64, 128, 1, 256, 8, 4.3f, 1.0f, 1.0f}, {128, 128, 1, 256, 8, 5.0f, 1.9f, 1.9f},
    {128, 128, 1, 512, 8, 0.f, 0.f, 0.f}, {256, 256, 1, 256, 8, 0.f, 0.f, 0.f},
    {16, 16, 4, 768, 4, 3.0f, 0.9f, 1.2f}, {32, 32, 8, 256, 8, 3.0f, 2.0f, 5.5f},
    {64, 32, 4, 256, 4, 3.0f, 2.0f, 4.0f}, {128, 128, 1, 256, 16, 5.0f, 2.15f, 2.15f}};

inline const Shape& shape_of(int elem_size, int kernel) {
  return (elem_size == 2 ? kShapes16 : kShapes32)[kernel];
}

// How a product is run: the kernel, which operands are copied to rows that start
// at multiples of 16 bytes, the shares of the reduction.
struct Plan {
  int kernel;
  bool copy_p, copy_q;
  size_t p_bytes, q_bytes;  // of the copies
  int tiles_m, tiles_n, splits, split_chunks;
};

// Rows of an operand in memory, and their length.
inline int memory_rows(bool k_inner, int rows, int k) { return k_inner ? rows : k; }
inline int memory_cols(bool k_inner, int rows, int k) { return k_inner ? k : rows; }
inline long copied_stride(int cols, int elem_size) {
  const int piece = 16 / elem_size;
  return (cols + piece - 1) / piece * piece;
}

// The kernel and the shares with the least time by the table above; the shares'
// sums cost a launch and their bytes; below zero: no grid holds the tiles.  `direct`: whole 16-byte pieces at aligned
// addresses; `tiled`: what kAnyTile128 takes.  `bytes`: the workspace that is left
// for the shares.
inline float choose(const Product& g, int elem_size, bool direct, bool tiled,
                    size_t bytes, Plan* p) {
  const int chunks = ceil_div(g.k, kChunkBytes / elem_size);
  // (operands that an L2 holds)
  const bool cached = (static_cast<double>(g.m) + g.n) * g.k * elem_size < 4e6;
  const float share_mb = static_cast<float>(g.m) * g.n * 4e-6f;
  // (the operands at 4.2 TB/s, which no division makes faster: 24 x 4096 x 4096
  // binary16 takes 8.7 us whole, 10.7 in two shares)
  const float memory =
      1.f + (static_cast<float>(g.m) + g.n) * g.k * elem_size / 4.2e6f;
  float best = -1.f;
  for (int kernel = direct ? 0 : kAny16x16;
       kernel < (direct ? kAny16x16 : kKernels); ++kernel) {
    const Shape& s = shape_of(elem_size, kernel);
    if (s.fixed == 0.f || (kernel == kAnyTile128 && !tiled)) continue;
#ifdef SNN_HIP_TUNING
    if (const char* only = std::getenv("SNN_HIP_EPI_KERNEL"))
      if (std::atoi(only) % kAny16x16 != kernel % kAny16x16) continue;
#endif
    const int tiles_m = ceil_div(g.m, s.bm), tiles_n = ceil_div(g.n, s.bn);
    const double tiles = static_cast<double>(tiles_m) * tiles_n;
    for (int want = 1; want <= 32; want *= 2) {
#ifdef SNN_HIP_TUNING
      if (const char* only = std::getenv("SNN_HIP_EPI_SPLITS"))
        if (std::atoi(only) != want) continue;
#endif
      if (want > 1 && (want > chunks / s.chunks || tiles * want > 1024 ||
                       static_cast<size_t>(g.m) * g.n * 4 * want > bytes))
        break;
      const int split_chunks = ceil_div(chunks, want);
      const int splits = ceil_div(chunks, split_chunks);
      if (tiles * splits > UINT_MAX / (64u * s.waves)) break;
      double rounds = std::ceil(tiles * splits / s.slots);
      if (s.slots == 512)  // work-groups that are alone on their CU are faster
        rounds += std::max(0.55, std::min(1.0, tiles * splits / 512 -
                                                   (rounds - 1.0))) -
                  1.0;
      const float steps =
          static_cast<float>(ceil_div(split_chunks, s.chunks));
      float step = g.q_k_inner ? s.step_k : s.step_row;
      if (s.chunks > 1 && cached) step *= 0.6f;
      const float time =
          std::max(static_cast<float>(std::ceil(rounds)) * s.fixed +
                       static_cast<float>(rounds) * steps * step,
                   memory) +
          (splits > 1 ? 2.2f + (0.2f + 0.5f * share_mb) * splits : 0.f);
      if (best < 0.f || time < best) {
        best = time;
        p->kernel = kernel;
        p->tiles_m = tiles_m;
        p->tiles_n = tiles_n;
        p->splits = splits;
        p->split_chunks = split_chunks;
      }
    }
  }
  return best;
}

// `bytes`: the workspace.  `p_aligned`, `q_aligned`: of the pointers.  No shares
// (splits == 0): no grid holds the tiles.
inline Plan make_plan(const Product& g, int elem_size, size_t bytes,
                      bool p_aligned, bool q_aligned) {
  Plan p = {};
  const int m = g.m, n = g.n, k = g.k;
  // Straight to LDS go whole 16-byte pieces, and tiles within 31 bits.
  const int chunk = kChunkBytes / elem_size;
  auto tile = [&](bool k_inner, int rows, long stride) {
    return memory_cols(k_inner, rows, k) * static_cast<long>(elem_size) >= 16 &&
           (k_inner ? 256 : chunk) * stride * elem_size < 0x7FFF0000l;
  };
  auto direct = [&](bool k_inner, bool aligned, int rows, long stride) {
    return aligned && stride * elem_size % 16 == 0 &&
           memory_cols(k_inner, rows, k) * static_cast<long>(elem_size) % 16 ==
               0 &&
           tile(k_inner, rows, stride);
  };
  const bool p_direct = direct(g.p_k_inner, p_aligned, m, g.p_stride);
  const bool q_direct = direct(g.q_k_inner, q_aligned, n, g.q_stride);
  if (p_direct && q_direct) {
    choose(g, elem_size, true, false, bytes, &p);
    return p;
  }
  const float any = choose(g, elem_size, false,
                           tile(g.p_k_inner, m, g.p_stride) &&
                               tile(g.q_k_inner, n, g.q_stride),
                           bytes, &p);
  auto copy_bytes = [&](bool k_inner, int rows) {
    return static_cast<size_t>(memory_rows(k_inner, rows, k)) *
           copied_stride(memory_cols(k_inner, rows, k), elem_size) * elem_size;
  };
  const size_t p_bytes = p_direct ? 0 : copy_bytes(g.p_k_inner, m);
  const size_t q_bytes = q_direct ? 0 : copy_bytes(g.q_k_inner, n);
  const int reach = 0x7FFF0000 / 256 / elem_size;
  if (p_bytes + q_bytes > bytes || m >= reach || n >= reach || k >= reach ||
      !seq::grid_fits((p_bytes + q_bytes) / 4096 + 2, 256))
    return p;
  Plan copied = {};
  copied.copy_p = !p_direct;
  copied.copy_q = !q_direct;
  copied.p_bytes = p_bytes;
  copied.q_bytes = q_bytes;
  // (a launch, and the operands read and written)
  const float product =
      choose(g, elem_size, true, false, bytes - p_bytes - q_bytes, &copied);
  const float with_copies =
      product + 3.f + static_cast<float>(p_bytes + q_bytes) * 0.5e-6f;
  if (product < 0.f) return p;
#ifdef SNN_HIP_TUNING
  if (const char* copy = std::getenv("SNN_HIP_EPI_COPY"))
    return std::atoi(copy) != 0 ? copied : p;
#endif
  return any < 0.f || with_copies < any ? copied : p;
}

}  // namespace epi
}  // namespace snn

#endif  // PORTDNN_AMD_CSRC_GEMM_EPILOGUE_H_
