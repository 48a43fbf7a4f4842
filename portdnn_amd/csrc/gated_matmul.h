// Two products at a time, in two forms, on the tiles of gemm_epilogue.h:
//
//   GATED   C[m][n] = act(sum P[m][r] G[n][r] + b[n]) (sum P[m][r] U[n][r] + c[n])
//   SUM     C[m][n] = sum P[m][r] G[n][r] + sum P'[m][r] U[n][r]
//
// the first half of a gated feed-forward part, and the gradient of its input, with
// P and P' the gradients of the two factors.  P's reduction is contiguous, G and U
// come in either order.
//
// GATED is one product with twice the columns: half of a tile's columns are G's, half
// U's, and both halves of a column are the same lane's on the way out, so that the
// factors meet in registers and P is read once.  SUM is one product with twice the
// reduction, whose chunks change operands halfway: nothing is rounded in between.
//
// Many rows are bound by the matrix unit, few by reading the weights.  bfloat16, 8192
// rows, k 2048, n 8192, both factors kept: 530 us, 1.04 PFLOP/s (256 x 256 tiles; a
// library's product of these sizes reaches 1.35); SUM of 4096 rows, 2 x 8192 to 2048
// columns: 249 us, 1.1 PFLOP/s (128 tiles of 256 x 256 in two shares, and their join).
// 1 row, k 2048, n 8192: 15.2 us, 67 MB, 4.4 TB/s; binary16, 32 rows, k 4096, n 8192,
// weights by column: 29.4 us, 134 MB, 4.6 TB/s; fp32, 1 row or 16, k 2048, n 8192: 30.8
// us, 134 MB, 4.4 TB/s.
#ifndef PORTDNN_AMD_CSRC_GATED_MATMUL_H_
#define PORTDNN_AMD_CSRC_GATED_MATMUL_H_

#include "gemm_epilogue.h"

namespace snn {
namespace gated {

using epi::float4v;
using epi::kChunkBytes;
using epi::lds_ptr;
using epi::Operand;
using epi::uint4v;

struct Pair {
  const void *p[2], *q[2];  // GATED: one p
  long p_stride, q_stride;
  int m, n, k;
  bool gated, q_k_inner;
  const void* bias[2];
  void *out, *pre[2];
  long out_stride;
  int activation;
  // division of the work
  int tiles_m, tiles_n, splits, split_chunks, chunks;  // chunks of one operand
  float* partial;  // [splits][GATED: 2][m][n]
};

int run_f32(Pair& g, void* workspace, size_t bytes, hipStream_t stream);
int run_f16(Pair& g, void* workspace, size_t bytes, hipStream_t stream);
int run_bf16(Pair& g, void* workspace, size_t bytes, hipStream_t stream);
// Bytes of workspace that a pair makes use of, by its sizes, strides and order.
size_t workspace_bytes(const Pair& g, int elem_size);

// N neighbouring columns of a row to or from memory, at any address, as far as the
// row goes.
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* from, int there, float (&to)[N]) {
  if (there >= N) {
    constexpr int VEC = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
#pragma unroll
    for (int j = 0; j < N; j += VEC) {
      float part[VEC];
      seq::unpack<T, VEC>(
          *reinterpret_cast<const typename seq::Pack<T, VEC>::type*>(from + j),
          part);
#pragma unroll
      for (int i = 0; i < VEC; ++i) to[j + i] = part[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      to[i] = i < there ? static_cast<float>(from[i]) : 0.f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_row(T* to, int there, const float (&from)[N]) {
  if (there >= N) {
    constexpr int VEC = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
#pragma unroll
    for (int j = 0; j < N; j += VEC) {
      float part[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) part[i] = from[j + i];
      *reinterpret_cast<typename seq::Pack<T, VEC>::type*>(to + j) =
          seq::pack<T, VEC>(part);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < there) to[i] = static_cast<T>(from[i]);
  }
}

// Eight neighbouring columns of a row: biases, activation, product, one rounding.
template <typename T>
__device__ __forceinline__ void finish(const Pair& p, int row, int col,
                                       float (&g)[8], float (&u)[8]) {
  const int there = p.n - col;
  if (p.gated) {
    auto add = [&](const void* bias, float (&to)[8]) {
      if (bias == nullptr) return;
      float b[8];
      load_row<T, 8>(static_cast<const T*>(bias) + col, there, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) to[i] += b[i];
    };
    add(p.bias[0], g);
    add(p.bias[1], u);
    if (p.pre[0] != nullptr) {
      const long at = static_cast<long>(row) * p.n + col;
      store_row<T, 8>(static_cast<T*>(p.pre[0]) + at, there, g);
      store_row<T, 8>(static_cast<T*>(p.pre[1]) + at, there, u);
    }
    epi::activate(g, p.activation);
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] *= u[i];
  }
  store_row<T, 8>(static_cast<T*>(p.out) + row * p.out_stride + col, there, g);
}

// ... of a tile: the result, or a share of its sums.
template <typename T>
__device__ __forceinline__ void leave(const Pair& p, unsigned split, int row,
                                      int col, float (&g)[8], float (&u)[8]) {
  if (p.splits == 1) {
    finish<T>(p, row, col, g, u);
    return;
  }
  const long size = static_cast<long>(p.m) * p.n;
  float* const to = p.partial + split * (p.gated ? 2 : 1) * size +
                    static_cast<long>(row) * p.n + col;
  store_row<float, 8>(to, p.n - col, g);
  if (p.gated) store_row<float, 8>(to + size, p.n - col, u);
}

// A chunk of the reduction: which operands, and where.
struct Chunk {
  int of, k0, left;  // operands, first reduction, reductions from there on
};
template <int CHUNK, bool GATED>
__device__ __forceinline__ Chunk chunk_of(const Pair& g, int c) {
  Chunk r;
  r.of = !GATED && c >= g.chunks ? 1 : 0;
  r.k0 = (c - r.of * g.chunks) * CHUNK;
  r.left = g.k - r.k0;
  return r;
}

// The tile of a work-group whose waves walk the reduction together: see gemm_body.
template <typename T, bool GATED, bool QK, int BM, int BN, int WM, int WN, int CB,
          int STAGES>
__device__ __forceinline__ void tile_body(const Pair& g, char* r0, char* r1,
                                          char* r2, char* r3, char* r4) {
  constexpr int H = GATED ? BN / 2 : BN;  // columns of one operand's tile
  constexpr int N = GATED ? 2 : 1;        // such tiles
  typedef Operand<T, true, BM, CB> OP;
  typedef Operand<T, QK, H, CB> OQ;
  constexpr int WAVES = WM * WN;
  typedef epi::Space<BM, BN, WAVES, CB> S;
  constexpr int TM = BM / WM, TN = BN / WN, IM = TM / 16, IN = TN / 16;
  constexpr int TH = TN / N, JN = IN / N;  // a wave's columns of one operand
  constexpr int kPBytes = BM * CB, kQBytes = H * CB;
  constexpr int kChunk = OP::kChunk;
  auto ring = [&](int u) {
    return u == 0 ? r0 : u == 1 ? r1 : u == 2 ? r2 : u == 3 ? r3 : r4;
  };
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;

  const unsigned tiles = static_cast<unsigned>(g.tiles_m) * g.tiles_n;
  const unsigned lin = gemm::xcd_remap(blockIdx.x, tiles * g.splits);
  const unsigned split = lin / tiles, tile = lin - split * tiles;
  constexpr unsigned kBand = 8;
  const unsigned band = tile / (kBand * g.tiles_n);
  const unsigned in_band = tile - band * kBand * g.tiles_n;
  const unsigned height = min(kBand, g.tiles_m - band * kBand);
  const int row0 = static_cast<int>(band * kBand + in_band % height) * BM;
  const int col0 = static_cast<int>(in_band / height) * H;
  const int all = N == 2 ? g.chunks : 2 * g.chunks;
  int at = static_cast<int>(split) * g.split_chunks;  // the chunk loaded next
  int left = min(all, at + g.split_chunks) - at;
  const int rows_left = g.m - row0, cols_left = g.n - col0;

  unsigned at_p[IM], at_q[IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
    at_p[i] = OP::fragment(wm * TM + 16 * i, lane);
#pragma unroll
  for (int j = 0; j < IN; ++j)
    at_q[j] = kPBytes + j / JN * kQBytes +
              OQ::fragment(wn * TH + 16 * (j % JN), lane);
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
        for (int j = 0; j < IN; ++j)
          acc[i][j] = epi::multiply<T>(q[j], p[i], acc[i][j]);
    }
  };

  // Offsets of the lane's loads within a chunk, and their reductions.
  unsigned offset[S::kLoads];
  int order[S::kLoads];
#pragma unroll
  for (int l = 0; l < S::kLoads; ++l) {
    const int block = wave + l * WAVES;
    int row, col;
    bool in;
    long stride;
    if (block < OP::kBlocks) {
      OP::source(block * 1024 + lane * 16, &row, &col);
      in = row < rows_left;
      stride = g.p_stride;
      order[l] = col;
    } else {
      OQ::source((block - OP::kBlocks) % OQ::kBlocks * 1024 + lane * 16, &row,
                 &col);
      in = block < S::kBlocks && (QK ? row < cols_left : col < cols_left);
      stride = g.q_stride;
      order[l] = QK ? col : row;
    }
    offset[l] =
        in ? static_cast<unsigned>((row * stride + col) * sizeof(T)) : epi::kOob;
  }
  auto issue = [&](char* to) {  // the next chunk; behind the last, any or none
    const Chunk c = chunk_of<kChunk, GATED>(g, at++);
    const __amdgpu_buffer_rsrc_t p =
        epi::make_rsrc(OP::at(g.p[c.of], g.p_stride, row0, c.k0));
    const __amdgpu_buffer_rsrc_t q =
        epi::make_rsrc(OQ::at(g.q[c.of], g.q_stride, col0, c.k0));
    const __amdgpu_buffer_rsrc_t u =
        GATED ? epi::make_rsrc(OQ::at(g.q[1], g.q_stride, col0, c.k0)) : q;
#pragma unroll
    for (int l = 0; l < S::kLoads; ++l) {
      const int block = wave + l * WAVES;
      const unsigned from = order[l] < c.left ? offset[l] : epi::kOob;
      if (block < OP::kBlocks)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            p, (lds_ptr)(to + block * 1024), 16, from, 0, 0, 0);
      else if (!GATED || block < OP::kBlocks + OQ::kBlocks)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            q, (lds_ptr)(to + block * 1024), 16, from, 0, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            u, (lds_ptr)(to + block * 1024), 16, from, 0, 0, 0);
    }
  };
#pragma unroll
  for (int c = 0; c < STAGES - 1; ++c) issue(ring(c));
  auto step = [&](int u) {
    // the chunk is here, and the reads of the one before have returned
    __builtin_amdgcn_s_waitcnt(epi::kLgkm0 &
                               epi::vmcnt_imm((STAGES - 2) * S::kLoads));
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
  __builtin_amdgcn_s_waitcnt(epi::kLgkm0 & epi::vmcnt_imm(0));

  // The way out, each wave's part in a place of its own: see gemm_body.
  __syncthreads();
  constexpr int kSharers = (WAVES + STAGES - 1) / STAGES;
  constexpr int kSpace = S::kStage / kSharers / 1024 * 1024;
  constexpr int kFit = kSpace / (TN * 4) / 16 * 16;
  constexpr int kRows = TM <= kFit ? TM : TM / 2 <= kFit ? TM / 2 : TM / 4;
  static_assert(kRows <= kFit && kRows % 16 == 0, "no room for the way out");
  constexpr unsigned kMask = TN / 4 - 1 < 15 ? TN / 4 - 1 : 15;
  char* own = ring(0);
#pragma unroll
  for (int u = 1; u < STAGES; ++u)
    if (wave / kSharers == u) own = ring(u);
  own += wave % kSharers * kSpace;
  constexpr int kLanes = TH / 8, kTurnRows = 64 / kLanes;
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
    const int col = col0 + wn * TH + (lane % kLanes) * 8;
#pragma unroll 1
    for (int t = 0; t < kRows; t += kTurnRows) {
      const unsigned r = t + lane / kLanes;
      const int row = row0 + wm * TM + pass * kRows + static_cast<int>(r);
      if (static_cast<int>(r) >= kRows || row >= g.m || col >= g.n) continue;
      float v[2][8];
#pragma unroll
      for (int o = 0; o < N; ++o)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned piece =
              (o * (TH / 4) + 2 * (lane % kLanes) + h) ^ (r & kMask);
          const float4v f =
              *reinterpret_cast<const float4v*>(own + r * (TN * 4) + piece * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[o][4 * h + i] = f[i];
        }
      leave<T>(g, split, row, col, v[0], v[1]);
    }
  }
}

// Few rows: the waves share the reduction, each with a ring of its own: see
// gemm_few_body.  DIRECT: whole 16-byte pieces at aligned addresses, straight to
// LDS; otherwise operands at any address by way of registers.
template <typename T, bool GATED, bool QK, int BM, int BN, int WAVES, int STAGES,
          bool DIRECT>
__device__ __forceinline__ void few_body(const Pair& g, char* r0, char* r1,
                                         char* r2, char* r3) {
  constexpr int CB = kChunkBytes;
  constexpr int H = GATED ? BN / 2 : BN, N = GATED ? 2 : 1;
  typedef Operand<T, true, BM, CB> OP;
  typedef Operand<T, QK, H, CB> OQ;
  constexpr int IM = BM / 16, IN = BN / 16, JN = IN / N;
  constexpr int kPBytes = BM * CB, kQBytes = H * CB, kOwn = (BM + BN) * CB;
  constexpr int kLoads = kOwn / 1024, kChunk = OP::kChunk;
  auto ring = [&](int u) { return u == 0 ? r0 : u == 1 ? r1 : u == 2 ? r2 : r3; };
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned tiles = static_cast<unsigned>(g.tiles_m) * g.tiles_n;
  const unsigned lin = gemm::xcd_remap(blockIdx.x, tiles * g.splits);
  const unsigned split = lin / tiles, tile = lin - split * tiles;
  const int row0 = static_cast<int>(tile % g.tiles_m) * BM;
  const int col0 = static_cast<int>(tile / g.tiles_m) * H;
  const int all = N == 2 ? g.chunks : 2 * g.chunks;
  const int begin = static_cast<int>(split) * g.split_chunks;
  const int end = min(all, begin + g.split_chunks);
  int at = begin + wave;  // the chunk that is loaded next
  int left = (end - at + WAVES - 1) / WAVES;
  const int rows_left = g.m - row0, cols_left = g.n - col0;

  unsigned at_p[IM], at_q[IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
    at_p[i] = wave * kOwn + OP::fragment(16 * i, lane);
#pragma unroll
  for (int j = 0; j < IN; ++j)
    at_q[j] = wave * kOwn + kPBytes + j / JN * kQBytes +
              OQ::fragment(16 * (j % JN), lane);
  float4v acc[IM][IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < IN; ++j) acc[i][j] = float4v{0.f, 0.f, 0.f, 0.f};
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
          acc[i][j] = epi::multiply<T>(q[s][j], p[s][i], acc[i][j]);
  };

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
        in = row < rows_left;
        stride = g.p_stride;
        order[l] = col;
      } else {
        OQ::source((l - OP::kBlocks) % OQ::kBlocks * 1024 + lane * 16, &row, &col);
        in = QK ? row < cols_left : col < cols_left;
        stride = g.q_stride;
        order[l] = QK ? col : row;
      }
      offset[l] = in ? static_cast<unsigned>((row * stride + col) * sizeof(T))
                     : epi::kOob;
    }
    auto issue = [&](char* to) {
      const Chunk c = chunk_of<kChunk, GATED>(g, min(at, all - 1));
      const int there = at < end ? c.left : 0;
      at += WAVES;
      const __amdgpu_buffer_rsrc_t p_at =
          epi::make_rsrc(OP::at(g.p[c.of], g.p_stride, row0, c.k0));
      const __amdgpu_buffer_rsrc_t q_at =
          epi::make_rsrc(OQ::at(g.q[c.of], g.q_stride, col0, c.k0));
      const __amdgpu_buffer_rsrc_t u_at =
          GATED ? epi::make_rsrc(OQ::at(g.q[1], g.q_stride, col0, c.k0)) : q_at;
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const unsigned from = order[l] < there ? offset[l] : epi::kOob;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            l < OP::kBlocks                              ? p_at
            : !GATED || l < OP::kBlocks + OQ::kBlocks ? q_at
                                                         : u_at,
            (lds_ptr)(to + wave * kOwn + l * 1024), 16, from, 0, 0, 0);
      }
    };
    auto step = [&](char* place) {
      __builtin_amdgcn_s_waitcnt(epi::vmcnt_imm((STAGES - 1) * kLoads));
      asm volatile("" ::: "memory");
      fetch(place);
      // the chunk is in registers before its place is loaded again
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(epi::kLgkm0 & epi::vmcnt_imm(63));
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
    uint4v held[STAGES][kLoads];
    auto load = [&](uint4v (&to)[kLoads]) {
      const Chunk c = chunk_of<kChunk, GATED>(g, min(at, all - 1));
      const int k_end = at < end ? g.k : 0;
      at += WAVES;
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        if (l < OP::kBlocks)
          to[l] = epi::load_piece<OP, T>(g.p[c.of], g.p_stride, rows_left, row0,
                                         c.k0, k_end, l * 1024 + lane * 16);
        else
          to[l] = epi::load_piece<OQ, T>(
              g.q[GATED ? (l - OP::kBlocks) / OQ::kBlocks : c.of], g.q_stride,
              cols_left, col0, c.k0, k_end,
              (l - OP::kBlocks) % OQ::kBlocks * 1024 + lane * 16);
      }
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
  __builtin_amdgcn_s_waitcnt(epi::kLgkm0 & epi::vmcnt_imm(0));

  // The waves' tiles, [wave][BM][BN], over the first ring; their sums eight columns
  // at a time.
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
  for (int e = tid; e < BM * H / 8; e += 64 * WAVES) {
    const int r = e / (H / 8), c = e % (H / 8) * 8;
    const int row = row0 + r, col = col0 + c;
    if (row >= g.m || col >= g.n) continue;
    float v[2][8] = {};
#pragma unroll
    for (int o = 0; o < N; ++o)
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float4v* const f = reinterpret_cast<const float4v*>(
            r0 + ((w * BM + r) * BN + o * H + c) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[o][i] += f[0][i];
          v[o][4 + i] += f[1][i];
        }
      }
    leave<T>(g, split, row, col, v[0], v[1]);
  }
}

// Adds the shares of a divided reduction in their order and finishes.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(Pair g) {
  const int groups = (g.n + 7) / 8;
  const long at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
  const int row = static_cast<int>(at / groups);
  const int col = static_cast<int>(at - static_cast<long>(row) * groups) * 8;
  if (row >= g.m) return;
  const long size = static_cast<long>(g.m) * g.n;
  const int n = g.gated ? 2 : 1;
  const float* from = g.partial + static_cast<long>(row) * g.n + col;
  float v[2][8] = {};
  constexpr int kBatch = 4;  // shares whose loads are under way together
  for (int s0 = 0; s0 < g.splits; s0 += kBatch) {
    float part[kBatch][2][8];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float* const share = from + min(s0 + u, g.splits - 1) * n * size;
      load_row<float, 8>(share, g.n - col, part[u][0]);
      if (n == 2) load_row<float, 8>(share + size, g.n - col, part[u][1]);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s0 + u < g.splits) {
          v[0][i] += part[u][0][i];
          if (n == 2) v[1][i] += part[u][1][i];
        }
  }
  finish<T>(g, row, col, v[0], v[1]);
}

// The kernels: those of gemm_epilogue.h that have a form for pairs, and one for
// operands at any address.
enum Kernel {
  kFew16x32,
  kFew16x64,
  kFew32x32,
  kFew32x64,
  kFew64x32,
  kTile64x128,
  kTile128,
  kTile128Pair,
  kTile256,
  kDirectKernels,
  kAny16x32 = kDirectKernels,
};
inline epi::Shape shape_of(int elem_size, int kernel) {
  constexpr int kSame[] = {epi::kFew16x32, -1, epi::kFew32x32, -1, epi::kFew64x32,
                           epi::kTile64x128, epi::kTile128,  epi::kTile128Pair,
                           epi::kTile256};
  if (kernel == kAny16x32)
    return {16, 32, 4, 512, 4, 3.0f, 1.2f, 2.4f};
  const bool f32 = elem_size == 4;
  if (kernel == kFew16x64)
    return {16, 64, 4, 256, 4, 2.6f, f32 ? 0.8f : 0.6f, f32 ? 1.1f : 0.9f};
  if (kernel == kFew32x64)
    return {32, 64, 4, 256, 4, 2.8f, f32 ? 1.3f : 0.7f, f32 ? 1.6f : 1.1f};
  epi::Shape s = epi::shape_of(elem_size, kSame[kernel]);
  // (sums of 2 x 8192 products in bfloat16, at the clocks of long calls: 4096 x 2048 in
  // 512 tiles of 128 x 128 281 us; in 128 of 256 x 256, in two shares, 233 and 16 for
  // their join.  GATED has hardly a use for them; us in tiles of 128 x 128, two such to a
  // CU, 256 x 256, * is what is taken: 2048 x 2048 x 8192 158, 149, 119*; 4096 x 1024 x 4096
  // 100, 85, 74*; 1024 x 4096 x 4096 74, 68*, 79; 512 x 2048 x 8192 42, 42*, 46.  SUM, with
  // the pass over the factors: 155*, 205, 165; 94*, 126, 108; 77*, 109, 90; 56, 71, 68 (64 x
  // 128: 59*).  6000 x 2000 x 3000 takes two of 128 x 128 to a CU, 197, SUM 238, where 256 x
  // 256 would take 170 and 195)
  if (kernel == kTile128 && elem_size == 2) s.step_k = s.step_row = 0.48f;
  return s;
}

// Bytes of a row in one of a kernel's chunks.
inline int chunk_bytes(int elem_size, int kernel) {
  return kernel == kTile256 || (kernel == kTile128 && elem_size == 4)
             ? kChunkBytes / 2
             : kChunkBytes;
}

// How a pair is run.
struct Plan {
  int kernel;
  bool copy_p, copy_q;
  size_t p_bytes, q_bytes;  // of a copy of one operand
  int tiles_m, tiles_n, splits, split_chunks;
};

// The kernel and the shares with the least time by epi's estimates, of a product with
// twice the columns or twice the reduction; below zero: no grid holds the tiles.
// `bytes`: the workspace that is left for the shares.
inline float choose(const Pair& g, int elem_size, bool direct, size_t bytes,
                    Plan* p) {
  const int each = ceil_div(g.k, kChunkBytes / elem_size);
  const int factors = g.gated ? 2 : 1;
  const double values = (g.gated ? g.m + 2.0 * g.n : 2.0 * g.m + 2.0 * g.n) * g.k;
  const bool cached = values * elem_size < 4e6;
  const float share_mb = static_cast<float>(g.m) * g.n * factors * 4e-6f;
  const double weights = 2.0 * g.n * g.k * elem_size;
  float best = -1.f;
  for (int kernel = direct ? 0 : kAny16x32;
       kernel < (direct ? kDirectKernels : kAny16x32 + 1); ++kernel) {
    const epi::Shape s = shape_of(elem_size, kernel);
    if (s.fixed == 0.f) continue;
#ifdef SNN_HIP_TUNING
    if (const char* only = std::getenv("SNN_HIP_GATED_KERNEL"))
      if (std::atoi(only) != kernel && direct) continue;
#endif
    const int tiles_m = ceil_div(g.m, s.bm);
    const int tiles_n = ceil_div(g.n, s.bn / factors);
    const double tiles = static_cast<double>(tiles_m) * tiles_n;
    // Reading from memory: pieces of 16 columns cost a sixth more, weights that are
    // read once more a quarter of a time, or a tenth where their rows are the
    // reduction's.  (bfloat16, k 2048, n 8192, us beside a cold cache: 1 row 16x32 38.4,
    // 16x64 33.2; 32 rows 16x64 41.6, 32x32 41.6, 32x64 33.8; transposed, 1 row
    // 30.8, 31.2, 32 rows 34.4, 31.0, 32.0)
    const bool narrow = !g.q_k_inner && s.bn / factors == 16;
    const float memory = 1.f + static_cast<float>(
        (values * elem_size * (narrow ? 1.17 : 1.0) +
         weights * std::min(tiles_m - 1, 4) * (g.q_k_inner ? 0.1 : 0.25)) / 4.2e6);
    const int chunks = g.gated ? each : 2 * each;
    for (int want = 1; want <= 32; want *= 2) {
#ifdef SNN_HIP_TUNING
      if (const char* only = std::getenv("SNN_HIP_GATED_SPLITS"))
        if (std::atoi(only) != want) continue;
#endif
      if (want > 1 && (want > chunks / s.chunks || tiles * want > 1024 ||
                       static_cast<size_t>(g.m) * g.n * factors * 4 * want >
                           bytes))
        break;
      const int split_chunks = ceil_div(chunks, want);
      const int splits = ceil_div(chunks, split_chunks);
      if (tiles * splits > UINT_MAX / (64u * s.waves)) break;
      double rounds = std::ceil(tiles * splits / s.slots);
      if (s.slots == 512)  // work-groups that are alone on their CU are faster
        rounds += std::max(0.55, std::min(1.0, tiles * splits / 512 -
                                                   (rounds - 1.0))) -
                  1.0;
      const float steps = static_cast<float>(ceil_div(split_chunks, s.chunks));
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
inline Plan make_plan(const Pair& g, int elem_size, size_t bytes, bool p_aligned,
                      bool q_aligned) {
  Plan p = {};
  const int chunk = kChunkBytes / elem_size;
  // Straight to LDS go whole 16-byte pieces, and tiles within 31 bits.
  auto direct = [&](bool k_inner, bool aligned, int rows, long stride) {
    const long cols = epi::memory_cols(k_inner, rows, g.k);
    return aligned && stride * elem_size % 16 == 0 && cols * elem_size % 16 == 0 &&
           (k_inner ? 256 : chunk) * stride * elem_size < 0x7FFF0000l;
  };
  const bool p_direct = direct(true, p_aligned, g.m, g.p_stride);
  const bool q_direct = direct(g.q_k_inner, q_aligned, g.n, g.q_stride);
  if (p_direct && q_direct) {
    choose(g, elem_size, true, bytes, &p);
    return p;
  }
  const float any = choose(g, elem_size, false, bytes, &p);
  auto copy_bytes = [&](bool k_inner, int rows) {
    return static_cast<size_t>(epi::memory_rows(k_inner, rows, g.k)) *
           epi::copied_stride(epi::memory_cols(k_inner, rows, g.k), elem_size) *
           elem_size;
  };
  const size_t p_bytes = p_direct ? 0 : copy_bytes(true, g.m);
  const size_t q_bytes = q_direct ? 0 : copy_bytes(g.q_k_inner, g.n);
  const size_t all = (g.gated ? 1 : 2) * p_bytes + 2 * q_bytes;
  const int reach = 0x7FFF0000 / 256 / elem_size;
  if (all > bytes || g.m >= reach || g.n >= reach || g.k >= reach ||
      !seq::grid_fits(all / 4096 + 4, 256))
    return p;
  Plan copied = {};
  copied.copy_p = !p_direct;
  copied.copy_q = !q_direct;
  copied.p_bytes = p_bytes;
  copied.q_bytes = q_bytes;
  // (a launch, and the operands read and written)
  const float product = choose(g, elem_size, true, bytes - all, &copied);
  if (product < 0.f) return p;
  const float with_copies = product + 3.f + static_cast<float>(all) * 0.5e-6f;
  return any < 0.f || with_copies < any ? copied : p;
}

}  // namespace gated
}  // namespace snn

#endif  // PORTDNN_AMD_CSRC_GATED_MATMUL_H_
