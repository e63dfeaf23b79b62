// Matrix product of eight-bit rows (mk_gemm_int8):
//   C[m][n] = (sum_k A[m][k] B[k][n]) a_scale[m] b_scale[n] (+ bias[n]) (ReLU)
// with A and B whole numbers of 8 bits, k contiguous in both, summed exactly in
// 32 bits (K <= 131071: 131071 * 128 * 128 < 2^31), so that no order of the sum
// changes it; the scales and the bias are applied to it in fp32 and rounded once.
//
// v_mfma_i32_32x32x32_i8 and v_mfma_i32_16x16x64_i8 give lane (c, g) of an
// operand row c and 16 consecutive k of group g.  They are issued with B's rows
// first, so that a lane's accumulator holds 4 consecutive columns of one row of
// C (lane (c, g), reg r of the 32 x 32 form: row c, column 8 (r / 4) + 4 g + r % 4).
//
// Bound: the matrix cores at the power limit for many rows (8192 x 4096 x 16384, M x K x N,
// 466 to 505 us by the card, 2180 to 2360 TOP/s), HBM for few, where the weights
// are the traffic (16 x 4096 x 16384 13.9 us, 67 MB), launches and latency for one (1 x
// 768 x 2304 3.2 to 3.8 us).
#include "attn_common.h"

#include <algorithm>
#include <string>
#include <type_traits>

namespace mk {
namespace {

using namespace attn;

typedef int i32x16_t __attribute__((ext_vector_type(16)));

constexpr int64_t kMaxK = 131071;

struct Int8Gemm {
  const int8_t *A, *B;
  const float *a_scale, *b_scale;
  void* C;
  const void* bias;
  int64_t M, N, K;
  int64_t lda, ldb, ldc;
  int tiles_m, tiles_n;
  int k_waves;   // few rows: waves of a workgroup that share a column block
  int c_type, epilogue;
  int stream_c;  // C goes past the caches
};

// one value of C from its sum
__device__ inline float finish(const Int8Gemm& p, int sum, float sa, int64_t n) {
  const float b = (p.epilogue & 3) != 0 ? load_as_f32(p.bias, n, (p.epilogue & 4) ? int(MK_F32) : p.c_type) : 0.f;
  float v = fmaf(float(sum) * sa, p.b_scale[n], b);
  if ((p.epilogue & 3) == 2) v = v < 0.f ? 0.f : v;  // keeps a NaN
  return v;
}

// 16 bytes from any address, one instruction on gfx950
struct __attribute__((packed, aligned(1))) Any16 { i32x4_t v; };
__device__ inline i32x4_t load16(const int8_t* p) { return reinterpret_cast<const Any16*>(p)->v; }
// bytes 0 .. n - 1 of 16, zeros past them
__device__ inline i32x4_t load16_upto(const int8_t* p, int64_t n) {
  if (n >= 16) return load16(p);
  uint8_t b[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) b[e] = e < n ? uint8_t(p[e]) : uint8_t(0);
  return __builtin_bit_cast(i32x4_t, b);
}

// ---------------------------------------------------------------- few rows
// At most 64 rows: reading B (the weights) once is the work.  A wave has 16 VN columns
// and all rows, and every k_waves-th step of 128 bytes of k, kD steps ahead in
// registers; the sums of the k_waves waves of a column block meet in LDS (whole
// numbers: in any order).  Nothing is staged.  A lane (c, g) of v_mfma_i32_16x16x64_i8
// loads 32 consecutive bytes of row c at k = 32 g, so that 4 lanes take a whole line of
// a row, and they are the operands of two MFMAs: which k an MFMA's slots mean is free
// as long as A and B agree.  Rows need no alignment.
constexpr int kStep = 128;

template <int VN, int MT, int NW, int kD>
__global__ __launch_bounds__(64 * NW) void gemm_int8_rows_kernel(const Int8Gemm p) {
  constexpr int NT = 16 * VN;
  __shared__ __attribute__((aligned(16))) int red[NW][16][NT + 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int kw = p.k_waves, k_wave = wave % kw, blocks = NW / kw;  // of columns, in this workgroup
  const int64_t n_first = int64_t(blockIdx.x) * blocks * NT, n0 = n_first + wave / kw * NT;
  const int64_t m_first = int64_t(blockIdx.y) * 16 * MT;
  // rows past the operands' repeat the last and are not stored
  const int8_t *ap[MT], *bp[VN];
#pragma unroll
  for (int m = 0; m < MT; ++m) ap[m] = p.A + std::min<int64_t>(m_first + 16 * m + c, p.M - 1) * p.lda + 32 * g;
#pragma unroll
  for (int j = 0; j < VN; ++j) bp[j] = p.B + std::min<int64_t>(n0 + 16 * j + c, p.N - 1) * p.ldb + 32 * g;
  struct Step {
    i32x4_t a[MT][2], b[VN][2];
  };
  auto load = [&](Step& s, int64_t step) __attribute__((always_inline)) {
    const int64_t k = step * kStep;
#pragma unroll
    for (int j = 0; j < VN; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) s.b[j][h] = load16(bp[j] + k + 16 * h);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) s.a[m][h] = load16(ap[m] + k + 16 * h);
  };
  i32x4_t acc[MT][VN] = {};
  auto multiply = [&](const Step& s) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < VN; ++j)
          acc[m][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.b[j][h], s.a[m][h], acc[m][j], 0, 0, 0);
  };
  // the loop's loads are unconditional: with a branch around them the compiler
  // waits for every load at the loop's head
  const int full = int(p.K) / kStep, n = full > k_wave ? (full - k_wave + kw - 1) / kw : 0;
  Step s[kD];
  auto fetch = [&](int d, int i) __attribute__((always_inline)) { load(s[d], k_wave + kw * i); };
  if (n >= kD) {
    int i = 0;
#pragma unroll
    for (int d = 0; d < kD; ++d) fetch(d, d);
    for (; i + 2 * kD <= n; i += kD) {
#pragma unroll
      for (int d = 0; d < kD; ++d) {
        multiply(s[d]);
        fetch(d, i + kD + d);
      }
    }
#pragma unroll
    for (int d = 0; d < kD; ++d) {
      multiply(s[d]);
      if (i + kD + d < n) fetch(d, i + kD + d);
    }
#pragma unroll
    for (int d = 0; d < kD; ++d)
      if (i + kD + d < n) multiply(s[d]);
  } else {
#pragma unroll
    for (int d = 0; d < kD - 1; ++d)
      if (d < n) fetch(d, d);
#pragma unroll
    for (int d = 0; d < kD - 1; ++d)
      if (d < n) multiply(s[d]);
  }
  if (p.K % kStep != 0 && full % kw == k_wave) {  // the last, shorter step: zeros past K
    const int64_t k = int64_t(full) * kStep, left = p.K - k - 32 * g;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < VN; ++j) s[0].b[j][h] = load16_upto(bp[j] + k + 16 * h, left - 16 * h);
#pragma unroll
      for (int m = 0; m < MT; ++m) s[0].a[m][h] = load16_upto(ap[m] + k + 16 * h, left - 16 * h);
    }
    multiply(s[0]);
  }
  // acc[m][j] reg r of lane (c, g): row 16 m + c, column 16 j + 4 g + r
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < VN; ++j) *reinterpret_cast<i32x4_t*>(&red[wave][c][16 * j + 4 * g]) = acc[m][j];
    __syncthreads();
    const int width = blocks * NT;
    for (int e = threadIdx.x; e < 16 * width; e += 64 * NW) {
      const int row = e / width, col = e % width, w0 = col / NT * kw;
      int sum = red[w0][row][col % NT];
      for (int w = 1; w < kw; ++w) sum += red[w0 + w][row][col % NT];
      const int64_t mrow = m_first + 16 * m + row, nc = n_first + col;
      if (mrow < p.M && nc < p.N)
        store_from_f32(p.C, mrow * p.ldc + nc, p.c_type, finish(p, sum, p.a_scale[mrow], nc));
    }
  }
}

template <int VN, int MT>
void launch_rows(hipStream_t s, Int8Gemm a, int k_waves) {
  constexpr int kWords = 8 * (VN + MT), kSums = 4 * VN * MT;
  // steps in flight within 128 registers (sixteen waves a CU) where two fit, else 256
  constexpr bool kSlim = 2 * kWords + kSums <= 72;
  constexpr int kFit = ((kSlim ? 72 : 192) - kSums) / kWords, kD = kFit > 4 ? 4 : kFit;
  static_assert(kD >= 2, "two steps in flight");
  constexpr int kMost = kSlim && VN == 1 ? 16 : 8;  // (32 columns a wave and more are never cut further)
  a.k_waves = std::min(k_waves, kMost);
  const int64_t blocks = (a.N + 16 * VN - 1) / (16 * VN);
  auto go = [&](auto nw) {
    constexpr int NW = decltype(nw)::value;
    const int64_t per = NW / a.k_waves;
    const dim3 g{unsigned((blocks + per - 1) / per), unsigned((a.M + 16 * MT - 1) / (16 * MT))};
    hipLaunchKernelGGL((gemm_int8_rows_kernel<VN, MT, NW, kD>), g, dim3(64 * NW), 0, s, a);
  };
  if (a.k_waves == 16) go(Int<kMost>{});
  else go(Int<8>{});
}

// Waves enough to fill the chip, from the columns (64 or 32 a wave where they are
// many: less of A is read) and then from k.  us, by columns a wave and waves along
// k: 16 x 4096 x 16384 (M x K x N) 16: 17.5 / 17.6 (2, 4), 32: 15.1 / 15.8 (4, 8),
// 64: 14.0 (8); 16 x 512 x 16384 16: 4.6 (4), 32: 4.6 (4); 16 x 4096 x 4096 16: 17.4,
// 10.3, 7.2, 7.2 (2, 4, 8, 16), 32: 8.7 (8); 1 x 768 x 2304 16: 3.2 (8).
template <int VN>
void launch_few_rows(hipStream_t s, const Int8Gemm& a) {
  const int64_t blocks = (a.N + 16 * VN - 1) / (16 * VN);
  int kw = 1;
  while (kw < 16 && kw * blocks < (VN == 1 ? 4096 : 2048) && kw * kStep < a.K) kw *= 2;
  if (a.M <= 16) launch_rows<VN, 1>(s, a, kw);
  else if (a.M <= 32) launch_rows<VN, 2>(s, a, kw);
  else launch_rows<VN, 4>(s, a, kw);
}
void launch_few_rows(hipStream_t s, const Int8Gemm& a) {
  if (a.N >= 12288 && a.K >= 2048) launch_few_rows<4>(s, a);
  else if (a.N >= 8192) launch_few_rows<2>(s, a);
  else launch_few_rows<1>(s, a);
}

// A small C: 16 x 16 blocks, k over the waves of a workgroup each.  Where those find
// a CU each they are ahead of the tiles, whose few workgroups have all of k in
// series; off the 16-byte grid for longer.  us, so / else: 64 x 16384 x 256 16.8 / 27.6;
// 256 x 4096 x 256 6.7 / 9.6; 128 x 2048 x 512 (256 blocks) 4.8 / 6.5; 106 x 4720 x 857
// (378) 10.3 / 11.0; 128 x 4096 x 1024 (512) 11.2 / 9.7; 42 x 6055 x 208 18 / 37.
bool small_c(const Int8Gemm& a, bool grid) {
  return (a.M + 15) / 16 * ((a.N + 15) / 16) <= (grid ? 256 : 512);
}
void launch_small(hipStream_t s, const Int8Gemm& a) {
  int kw = 1;
  while (kw < 16 && kw * kStep < a.K) kw *= 2;
  launch_rows<1, 1>(s, a, kw);
}

// ---------------------------------------------------------------- tiles
// Workgroup tile TM x TN, k in tiles of 128 bytes, WGM x WGN waves of 32 x 32 blocks.
// Tiles of rows on the 16-byte grid go straight into LDS (buffer_load ... lds,
// attn_common.h) in S stages: the copies of k tile t + S - 1 are issued while tile t is
// multiplied, one barrier a tile.  An LDS row is
// 128 bytes, its 16-byte chunk c at position c ^ ((row >> 1) & 7), so that the
// 16 rows a ds_read_b128 takes at one chunk lie on 16 different bank groups.
// Chunks past M, N or K are loaded from an out-of-range offset, which reads
// zeros.  Where K is no multiple of 16 the last chunk of a row is loaded whole
// (16 aligned bytes, so on the row's last page) and A's bytes past K are then
// cleared in LDS: what B holds there is multiplied by zero.
//
// Tile order: workgroups are dealt round-robin to the 8 XCDs, each with its own
// L2; workgroup i takes tile (i % 8) (tiles / 8) + i / 8 of an order that walks
// groups of 4 tile rows column by column, so that an XCD's tiles are a compact block.
constexpr int kBK = 128;
constexpr int kGroupM = 4;
constexpr int kInvalid = int(0x80000000u);  // buffer offset past every accepted range

// The copies one wave makes of an operand tile of W * kC * 8 rows: copy c is 1 KB,
// 8 rows, lane l of it writes chunk position l % 8 of row l / 8.
template <int kC, int W>
struct Copies {
  uint32_t off[kC];
  int32_t k[kC];
  __device__ inline Copies(int wave, int lane, int64_t r0, int64_t rows, int64_t ld) {
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const int row = 8 * (wave + W * c) + lane / 8;
      k[c] = 16 * ((lane % 8) ^ ((row >> 1) & 7));
      off[c] = r0 + row < rows ? uint32_t((r0 + row) * ld + k[c]) : uint32_t(kInvalid);
    }
  }
  // Clears what this wave copied of the last k tile (at k0, K no multiple of 16) past K.
  __device__ inline void clear_past(int8_t* tile, int wave, int lane, int k0, int64_t K) const {
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const int left = int(K) - k0 - k[c];
      if (left <= 0 || left >= 16) continue;
      u32x4_t* at = reinterpret_cast<u32x4_t*>(tile + (wave + W * c) * 1024 + 16 * lane);
      u32x4_t v = *at;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = left - 4 * q;
        v[q] &= n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1;
      }
      *at = v;
    }
  }
  // offset for the k tile at k0, or one that reads zeros once the chunk lies past K
  __device__ inline int at(int c, int k0, int64_t K) const {
    return off[c] != uint32_t(kInvalid) && k[c] + k0 < K ? int(off[c] + uint32_t(k0)) : kInvalid;
  }
};

// The same chunks of rows at any address and pitch, through registers: rows past
// the operand repeat its last one, k past K is zeros.
template <int kC, int W>
struct Loads {
  const int8_t* at[kC];
  int32_t k[kC];
  i32x4_t v[kC];
  __device__ inline Loads(const int8_t* base, int wave, int lane, int64_t r0, int64_t rows, int64_t ld) {
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const int row = 8 * (wave + W * c) + lane / 8;
      k[c] = 16 * ((lane % 8) ^ ((row >> 1) & 7));
      at[c] = base + std::min<int64_t>(r0 + row, rows - 1) * ld + k[c];
    }
  }
  __device__ inline void load(int k0, int K) {
    if (k0 + kBK <= K) {
#pragma unroll
      for (int c = 0; c < kC; ++c) v[c] = load16(at[c] + k0);
    } else {
#pragma unroll
      for (int c = 0; c < kC; ++c) v[c] = load16_upto(at[c] + k0, K - k0 - k[c]);
    }
  }
  __device__ inline void store(int8_t* tile, int wave, int lane) const {
#pragma unroll
    for (int c = 0; c < kC; ++c) *reinterpret_cast<i32x4_t*>(tile + (wave + W * c) * 1024 + 16 * lane) = v[c];
  }
};

// MFMA operand for rows rb .. rb + 31 and k 32 ks .. 32 ks + 31 of a tile
__device__ inline i32x4_t read_operand(const int8_t* t, int rb, int ks, int lane) {
  const int row = rb + (lane & 31), ch = (2 * ks + (lane >> 5)) ^ ((row >> 1) & 7);
  return *reinterpret_cast<const i32x4_t*>(t + row * kBK + 16 * ch);
}

template <int N>
__device__ inline void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// Workgroup tile, wave grid, LDS stages; DIRECT: rows on the 16-byte grid go straight
// into LDS, any others through registers.
template <int TM_, int TN_, int WGM_, int WGN_, int S_, bool DIRECT = true>
struct Shape {
  static constexpr int TM = TM_, TN = TN_, WGM = WGM_, WGN = WGN_, S = S_;
  static constexpr bool kDirect = DIRECT;
};

typedef uint32_t u32x4_by4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_by2_t __attribute__((ext_vector_type(4), aligned(2)));

// C's tile through LDS, each wave for itself and without barriers: 32 rows of its
// columns at a time, in its part of the operand stages (8192 x 768 x 50304 in bf16, with
// ordinary stores: 6% less than with the workgroup storing whole rows of the tile between
// barriers).  A lane writes 4 consecutive columns, chunk c of staging row r at position
// c ^ (r & 15) (rows of 8 and 4 chunks: c ^ ((r >> 1) & 7), c ^ ((r >> 2) & 3)), and the
// wave stores runs of 16 bytes (of whole rows; they need no alignment past an element's).
template <int CT, bool STREAM, int kWM, int kWN, int kI, int kJ>
__device__ __attribute__((always_inline)) inline void store_tile(const Int8Gemm& p, const i32x16_t (&acc)[kI][kJ],
                                                                 int8_t* stage, const float* sa, const float* sb,
                                                                 const float* bias, int64_t m0, int64_t n0, int wm,
                                                                 int wn, int lane) {
  constexpr int kSz = CT == MK_F32 ? 4 : 2, kPer = 16 / kSz, kCpr = kWN / kPer;
  static_assert(kCpr % 4 == 0 && 32 * kCpr % 64 == 0, "whole chunks, evenly over the lanes");
  using out_t = std::conditional_t<CT == MK_F32, u32x4_by4_t, u32x4_by2_t>;
  auto pos = [](int row, int cn) {
    return cn ^ (kCpr % 16 == 0 ? row & 15 : kCpr % 8 == 0 ? (row >> 1) & 7 : (row >> 2) & 3);
  };
  const int c = lane & 31, g = lane >> 5;
  char* C = static_cast<char*>(p.C);
  // this lane's scales and biases
  float s[kI];
  f32x4 t[kJ][4], u[kJ][4];
#pragma unroll
  for (int a = 0; a < kI; ++a) s[a] = sa[wm * kWM + 32 * a + c];
#pragma unroll
  for (int b = 0; b < kJ; ++b)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
      const int nl = wn * kWN + 32 * b + 8 * rg + 4 * g;
      t[b][rg] = *reinterpret_cast<const f32x4*>(sb + nl);
      u[b][rg] = *reinterpret_cast<const f32x4*>(bias + nl);
    }
#pragma unroll
  for (int a = 0; a < kI; ++a) {
#pragma unroll
    for (int b = 0; b < kJ; ++b)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const int nl = 32 * b + 8 * rg + 4 * g;
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = fmaf(float(acc[a][b][4 * rg + q]) * s[a], t[b][rg].v[q], u[b][rg].v[q]);
        if ((p.epilogue & 3) == 2) {
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = v[q] < 0.f ? 0.f : v[q];
        }
        int8_t* to = stage + c * kWN * kSz + 16 * pos(c, nl / kPer) + nl % kPer * kSz;
        if constexpr (CT == MK_F32) {
          *reinterpret_cast<f32x4*>(to) = f32x4{{v[0], v[1], v[2], v[3]}};
        } else {
          uint16_t h[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) h[q] = CT == MK_BF16 ? f32_to_bf16(v[q]) : f32_to_f16(v[q]);
          __builtin_memcpy(to, h, 8);
        }
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int it = 0; it < 32 * kCpr / 64; ++it) {
      const int e = it * 64 + lane;
      const int row = e / kCpr, cn = e % kCpr;
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(stage + row * kWN * kSz + 16 * pos(row, cn));
      const int64_t m = m0 + wm * kWM + 32 * a + row, n = n0 + wn * kWN + cn * kPer;
      if (m >= p.M || n >= p.N) continue;
      char* to = C + kSz * (m * p.ldc + n);
      if (n + kPer <= p.N) {
        if constexpr (STREAM) __builtin_nontemporal_store(out_t(v), reinterpret_cast<out_t*>(to));
        else *reinterpret_cast<out_t*>(to) = v;
      } else {  // the chunk that straddles N
#pragma unroll
        for (int q = 0; q < kPer; ++q)
          if (n + q < p.N) {
            if constexpr (CT == MK_F32) reinterpret_cast<uint32_t*>(to)[q] = v[q];
            else reinterpret_cast<uint16_t*>(to)[q] = uint16_t(v[q / 2] >> (16 * (q & 1)));
          }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

template <class Sh, int CT>
__global__ __launch_bounds__(64 * Sh::WGM * Sh::WGN, 1) void gemm_int8_tiled_kernel(const Int8Gemm p) {
  constexpr int TM = Sh::TM, TN = Sh::TN, WGN = Sh::WGN, S = Sh::S, kW = Sh::WGM * WGN;
  constexpr int kWM = TM / Sh::WGM, kWN = TN / WGN, kI = kWM / 32, kJ = kWN / 32;
  constexpr int kCa = TM / 8 / kW, kCb = TN / 8 / kW, kNC = kCa + kCb;
  static_assert(kI * 32 * Sh::WGM == TM && kJ * 32 * WGN == TN, "wave blocks tile the workgroup tile");
  static_assert(kCa * kW * 8 == TM && kCb * kW * 8 == TN, "copies split evenly over the waves");
  __shared__ __attribute__((aligned(1024))) int8_t lds[S * kBK * (TM + TN)];
  __shared__ __attribute__((aligned(16))) float sa[TM], sb[TN], bias[TN];
  int8_t (*As)[TM * kBK] = reinterpret_cast<int8_t (*)[TM * kBK]>(lds);
  int8_t (*Bs)[TN * kBK] = reinterpret_cast<int8_t (*)[TN * kBK]>(lds + S * TM * kBK);

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const uint32_t nt = gridDim.x, per = nt / 8, i = blockIdx.x;
  const uint32_t t = i < 8 * per ? (i % 8) * per + i / 8 : i;
  const uint32_t group = t / (kGroupM * uint32_t(p.tiles_n)), first_m = group * kGroupM;
  const uint32_t gm = min(uint32_t(kGroupM), uint32_t(p.tiles_m) - first_m);
  const uint32_t w_in = t - group * kGroupM * uint32_t(p.tiles_n);
  const int64_t m0 = int64_t(first_m + w_in % gm) * TM, n0 = int64_t(w_in / gm) * TN;
  // the last row's last chunk whole: to the next multiple of 16 bytes
  const i32x4_t ra = tile_desc(p.A, uint32_t(((p.M - 1) * p.lda + p.K + 15) & ~int64_t(15)));
  const i32x4_t rb = tile_desc(p.B, uint32_t(((p.N - 1) * p.ldb + p.K + 15) & ~int64_t(15)));
  const Copies<kCa, kW> ca(wave, lane, m0, p.M, p.lda);
  const Copies<kCb, kW> cb(wave, lane, n0, p.N, p.ldb);
  const int K = int(p.K);
  // this wave's copies [lo, hi) of k tile kt (A's, then B's): of a tile wholly below
  // K, and of the one that crosses it
  auto issue = [&](int kt, int lo, int hi) __attribute__((always_inline)) {
    const int st = kt % S;
#pragma unroll
    for (int c = 0; c < kNC; ++c) {
      if (c < lo || c >= hi) continue;
      const uint32_t at = uint32_t(kBK * kt);
      if (c < kCa) copy_to_lds_so(ra, lds_addr(&As[st][(wave + kW * c) * 1024]), int(ca.off[c < kCa ? c : 0]), at);
      else copy_to_lds_so(rb, lds_addr(&Bs[st][(wave + kW * (c - kCa)) * 1024]), int(cb.off[c < kCa ? 0 : c - kCa]), at);
    }
  };
  auto issue_last = [&](int kt) __attribute__((always_inline)) {
    const int st = kt % S;
#pragma unroll
    for (int c = 0; c < kCa; ++c) copy_to_lds(ra, lds_addr(&As[st][(wave + kW * c) * 1024]), ca.at(c, kBK * kt, K));
#pragma unroll
    for (int c = 0; c < kCb; ++c) copy_to_lds(rb, lds_addr(&Bs[st][(wave + kW * c) * 1024]), cb.at(c, kBK * kt, K));
  };
  i32x16_t acc[kI][kJ] = {};
  const int nk = (K + kBK - 1) / kBK, full = K / kBK;
  if constexpr (Sh::kDirect) {
#pragma unroll
    for (int kt = 0; kt < S - 1; ++kt) {
      if (kt < full) issue(kt, 0, kNC);
      else if (kt < nk) issue_last(kt);
    }
  }
  // the scales and the bias of the tile, for the end (after the first copies, so
  // that these go first)
  for (int e = threadIdx.x; e < TM; e += 64 * kW) sa[e] = m0 + e < p.M ? p.a_scale[m0 + e] : 0.f;
  for (int e = threadIdx.x; e < TN; e += 64 * kW) {
    sb[e] = n0 + e < p.N ? p.b_scale[n0 + e] : 0.f;
    bias[e] = 0.f;
    if ((p.epilogue & 3) != 0)
      bias[e] = n0 + e < p.N ? load_as_f32(p.bias, n0 + e, (p.epilogue & 4) ? int(MK_F32) : CT) : 0.f;
  }
  // Tile kt from stage kt % S, a step's operands read while the step before is
  // multiplied; MORE: the copies of tile kt + S - 1 in two parts between the first
  // steps (all at once they fill the memory queue with the MFMAs behind them).
  auto multiply = [&](int kt, auto more) __attribute__((always_inline)) {
    const int8_t *at = As[kt % S], *bt = Bs[kt % S];
    constexpr bool kAhead = kI * kJ == 1;
    i32x4_t af[2][kI], bf[2][kJ];
    auto read = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < kI; ++a) {
        af[ks % 2][a] = read_operand(at, wm * kWM + 32 * a, ks, lane);
      }
#pragma unroll
      for (int b = 0; b < kJ; ++b) bf[ks % 2][b] = read_operand(bt, wn * kWN + 32 * b, ks, lane);
    };
    if constexpr (kAhead) read(0);
#pragma unroll
    for (int ks = 0; ks < kBK / 32; ++ks) {
      if constexpr (!kAhead) read(ks);
      else if (ks + 1 < kBK / 32) read(ks + 1);
      if constexpr (decltype(more)::value)
        if (ks < 2) issue(kt + S - 1, ks * kNC / 2, (ks + 1) * kNC / 2);
#pragma unroll
      for (int a = 0; a < kI; ++a)
#pragma unroll
        for (int b = 0; b < kJ; ++b)
          acc[a][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bf[ks % 2][b], af[ks % 2][a], acc[a][b], 0, 0, 0);
    }
  };
  if constexpr (Sh::kDirect) {
    // Each turn waits for this wave's copies of its tile (those of the S - 2 tiles
    // after it may still be in flight), then for everyone's; the stage of the tile
    // before is then free for the tile S - 1 further on.
    int kt = 0;
    for (; kt + S - 1 < full; ++kt) {
      wait_vm<(S - 2) * kNC>();
      lds_barrier();
      multiply(kt, Flag<true>{});
    }
    for (; kt < nk; ++kt) {
      wait_vm<0>();
      lds_barrier();
      if (kt + S - 1 == full && full < nk) issue_last(full);
      if (kt == nk - 1 && K % 16 != 0) {
        ca.clear_past(As[kt % S], wave, lane, kBK * kt, K);
        lds_barrier();
      }
      multiply(kt, Flag<false>{});
    }
  } else {
    // the next tile's loads are in flight while this one is multiplied; a stage is
    // written again two barriers after its last reader began
    static_assert(S == 2 || Sh::kDirect, "two stages");
    Loads<kCa, kW> la(p.A, wave, lane, m0, p.M, p.lda);
    Loads<kCb, kW> lb(p.B, wave, lane, n0, p.N, p.ldb);
    if (nk > 0) la.load(0, K), lb.load(0, K);
    for (int kt = 0; kt < nk; ++kt) {
      la.store(As[kt % S], wave, lane);
      lb.store(Bs[kt % S], wave, lane);
      __syncthreads();
      if (kt + 1 < nk) la.load(kBK * (kt + 1), K), lb.load(kBK * (kt + 1), K);
      multiply(kt, Flag<false>{});
    }
  }
  lds_barrier();  // every wave is done with the operand stages before they hold C
  constexpr int kStage = 32 * kWN * (CT == MK_F32 ? 4 : 2);  // bytes a wave
  static_assert(kStage * kW <= S * kBK * (TM + TN), "room for C");
  int8_t* stage = lds + wave * kStage;
  if (p.stream_c) store_tile<CT, true, kWM, kWN>(p, acc, stage, sa, sb, bias, m0, n0, wm, wn, lane);
  else store_tile<CT, false, kWM, kWN>(p, acc, stage, sa, sb, bias, m0, n0, wm, wn, lane);
}

template <class Sh>
void launch_tiled(hipStream_t s, Int8Gemm a) {
  a.tiles_m = int((a.M + Sh::TM - 1) / Sh::TM);
  a.tiles_n = int((a.N + Sh::TN - 1) / Sh::TN);
  const dim3 g{unsigned(int64_t(a.tiles_m) * a.tiles_n)}, b{unsigned(64 * Sh::WGM * Sh::WGN)};
  auto go = [&](auto ct) {
    constexpr int CT = decltype(ct)::value;
    hipLaunchKernelGGL((gemm_int8_tiled_kernel<Sh, CT>), g, b, 0, s, a);
  };
  if (a.c_type == MK_BF16) go(Int<MK_BF16>{});
  else if (a.c_type == MK_F16) go(Int<MK_F16>{});
  else go(Int<MK_F32>{});
}

// The tile with the least estimated time: rounds of workgroups of nk + e k tiles, e the
// first copies and the epilogue; a last round that leaves every workgroup alone on its
// CU runs each k tile in `alone`, and 256 x 256 tiles, one on a CU, in a time that
// grows with their number (the power limit).  us, fitted to the shapes' times on 166
// products of 17 .. 8192 rows with both C types; the choice costs 1.0% over the fastest
// on average (1.6% without that last term).  In the order below, us: bf16 C (M x K x N):
// 8192 x 4096 x 16384 467, 578, 773, 895, 1120; 2048 x 4096 x 4096 54, 43, 58, 67, 83; 512 x
// 4096 x 4096 41, 23, 18, 18, 24; 64 x 768 x 50257 18, 14, 12.7, 15.5, 17.5; 128 x 768 x 768
// 12.2, 5.7, 5.1, 4.3, 4.3.
void launch_best_tile(hipStream_t s, Int8Gemm& a, bool grid) {
  struct Option {
    int tm, tn, per_cu;
    double each, alone, e16, e32;
  };
  static const Option options[] = {{256, 256, 1, 2.04, 1.21, 3.2, 5.1},
                                   {128, 128, 2, 1.40, 0.70, 2.3, 3.0},
                                   {64, 128, 2, 0.86, 0.45, 3.1, 3.7},
                                   {64, 64, 2, 0.50, 0.31, 4.3, 5.1},
                                   {64, 32, 3, 0.45, 0.27, 4.6, 5.4}};
  const double nk = double((a.K + kBK - 1) / kBK);
  int best = 0;
  double least = 0;
  for (int o = 0; o < 5; ++o) {
    if (!grid && o != 1 && o != 3) continue;
    const Option& q = options[o];
    const int64_t tiles = ((a.M + q.tm - 1) / q.tm) * ((a.N + q.tn - 1) / q.tn), slots = 256 * q.per_cu;
    const double work = nk + (a.c_type == MK_F32 ? q.e32 : q.e16);
    double t = double(tiles / slots) * work * q.each;
    const int64_t rem = tiles % slots;
    if (q.per_cu == 1) t += rem ? work * (q.alone + (q.each - q.alone) * double(rem) / 256) : 0;
    else if (rem) t += work * (rem <= 256 ? q.alone : q.each);
    if (least == 0 || t < least) best = o, least = t;
  }
  // C past the caches where it is most of the last-level cache and its rows lie on the
  // 128-byte lines; us, so / with ordinary stores: bf16 8192 x 768 x 50304 394 / 473,
  // 8192 x 4096 x 16384 475 / 490, fp32 8192 x 768 x 50304 482 / 590, 8192 x 2048 x 16384
  // 291 / 326.  Off the lines not every C gains: fp32 8192 x 768 x 50257 680 / 672, x 50260
  // 632 / 655, bf16 x 50264 402 / 494; all of those take ordinary stores
  const int64_t pitch = a.ldc * dtype_bytes(a.c_type);
  a.stream_c = a.M * a.N * dtype_bytes(a.c_type) >= int64_t(192) << 20 && pitch % 128 == 0 &&
               reinterpret_cast<uintptr_t>(a.C) % 128 == 0;
  if (!grid && best == 1) launch_tiled<Shape<128, 128, 2, 4, 2, false>>(s, a);
  else if (!grid) launch_tiled<Shape<64, 64, 2, 2, 2, false>>(s, a);
  else if (best == 0) launch_tiled<Shape<256, 256, 2, 4, 2>>(s, a);
  else if (best == 1) launch_tiled<Shape<128, 128, 2, 4, 2>>(s, a);
  else if (best == 2) launch_tiled<Shape<64, 128, 2, 4, 3>>(s, a);
  else if (best == 3) launch_tiled<Shape<64, 64, 2, 2, 4>>(s, a);
  else launch_tiled<Shape<64, 32, 2, 1, 4>>(s, a);
}

// rows on the 16-byte grid that do not overlap, below the 2^31 bytes of a buffer's offsets
// (an operand of more is loaded through registers: 131056 x 16384 x 4096 7.0 ms, 131088
// rows 10.9)
bool on_grid(const int8_t* p, int64_t rows, int64_t K, int64_t ld) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 16 == 0 && ld >= K && ld < (int64_t(1) << 31) &&
         (rows - 1) * ld + K + 16 < (int64_t(1) << 31);
}

}  // namespace
}  // namespace mk

using namespace mk;

extern "C" int mk_gemm_int8(void* stream, int c_type, int64_t M, int64_t N, int64_t K, const int8_t* A, int64_t a_ms,
                            const float* a_scale, const int8_t* B, int64_t b_ns, const float* b_scale, void* C,
                            int64_t c_ms, const void* bias, int epilogue) {
  clear_error();
  if (c_type != MK_BF16 && c_type != MK_F16 && c_type != MK_F32)
    return fail(MK_ERR_UNSUPPORTED, "mk_gemm_int8: c_type must be bf16/f16/f32");
  if (M < 0 || N < 0 || K < 0) return fail(MK_ERR_INVALID, "mk_gemm_int8: negative shape");
  if (K > kMaxK) return fail(MK_ERR_UNSUPPORTED, "mk_gemm_int8: K past 131071: the 32-bit sums could overflow");
  // a workgroup of 256 threads per 64 x 64 tile, or of 512 per two, below HIP's 2^32 threads
  if (M >> 30 || N >> 30 || (M + 63) / 64 * ((N + 63) / 64) >= (int64_t(1) << 24) - 1)
    return fail(MK_ERR_UNSUPPORTED, "mk_gemm_int8: 2^24 - 1 or more tiles of 64 x 64");
  const int epi = epilogue & 3;
  if (epilogue < 0 || epilogue > 6 || epi == 3 || (epilogue == 4))
    return fail(MK_ERR_INVALID, "mk_gemm_int8: epilogue must be 0, 1, 2, 5 or 6");
  if (M == 0 || N == 0) return MK_OK;
  if ((K > 0 && (!A || !B)) || !a_scale || !b_scale || !C || (epi != 0 && !bias))
    return fail(MK_ERR_INVALID, "mk_gemm_int8: null pointer");
  if ((M > 1 && (a_ms < 0 || c_ms < N)) || (N > 1 && b_ns < 0)) return fail(MK_ERR_INVALID, "mk_gemm_int8: bad stride");
  if (reinterpret_cast<uintptr_t>(C) % dtype_bytes(c_type) || reinterpret_cast<uintptr_t>(a_scale) % 4 ||
      reinterpret_cast<uintptr_t>(b_scale) % 4 ||
      (epi != 0 && reinterpret_cast<uintptr_t>(bias) % ((epilogue & 4) ? 4 : dtype_bytes(c_type))))
    return fail(MK_ERR_INVALID, "mk_gemm_int8: an operand is not aligned to its elements");
  // one row's pitch says nothing
  if (M == 1) a_ms = (K + 15) & ~int64_t(15);
  if (N == 1) b_ns = (K + 15) & ~int64_t(15);
  if (M == 1) c_ms = N;
  Int8Gemm a{A, B, a_scale, b_scale, C, bias, M, N, K, a_ms, b_ns, c_ms, 0, 0, 1,
             c_type, epilogue, 0};
  hipStream_t s = as_stream(stream);
  const bool grid = K > 0 && on_grid(A, M, K, a_ms) && on_grid(B, N, K, b_ns);
  // few rows off the grid, or up to where the tiles are ahead (from 17 rows on they share
  // A's reads; for wide weights they are from one row on).  us, rows kernel / tiles:
  // 32 x 4096 x 16384 16.9 / 13.4; 32 x 4096 x 4096 9.5 / 10.0; 32 x 4096 x 8192 11.7 / 10.3;
  // fp32 C 1 x 768 x 50257 10.5 / 9.1, 16 rows 13.0 / 9.6; 1 x 4096 x 128256 118 / 108, 16 rows
  // 126 / 113; bf16 C 1 x 4096 x 32768 30 / 33
  if (small_c(a, grid)) launch_small(s, a);
  else if (M <= 64 && (!grid || (M <= 16 && N < 32768) || (M <= 32 && N <= 8192))) launch_few_rows(s, a);
  else launch_best_tile(s, a, grid);
  return check_launch("mk_gemm_int8");
}
