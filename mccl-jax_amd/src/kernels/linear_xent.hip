// Softmax cross entropy over a large vocabulary from the hidden rows and the
// embedding (mk_linear_xent), and its gradient (mk_linear_xent_bwd), without
// the logits in memory.
//
//   s[n][v] = x[n] . w[v];  lse[n] = log sum_v exp s[n][v];  loss[n] = lse[n] - s[n][label]
//   g[n][v] = (exp(s[n][v] - lse[n]) - [v == label]) row_grad[n] grad_scale
//   dx = g w,  dw = gᵀ x
//
// Forward: one product, tile by tile; a tile ends with each of its rows' maximum
// and sum of exponentials (8 bytes a row for TN logits), and a second launch joins
// a row's tiles.  Up to 32 rows have kernels of their own.  Backward, piece by piece
// of the vocabulary: the same product again, ending with g in the operands' type (a
// matrix product reads it next; it is formed from fp32 logits, and what its rounding
// leaves of the labels' elements is kept beside it), then dx and dw of the piece in
// one launch.  g is the only large thing that goes through memory, 512 MB at a time.
//
// Many rows are bound by the matrix rate: 8192 x 768 x 50257 bf16 takes 570 us
// forward (1.11 PFLOP/s; the library's product of the logits alone 597) and 1866
// backward (three products, 1.02 PFLOP/s; the library's three 2008, without the
// softmax), 8192 x 4096 x 65536 11.1 ms backward (1.19).  Twelve k tiles of 768 are short
// beside a tile's end.  Few rows are bound by w: 16 rows of it 20.4 us forward (16 us
// of products, 4.8 TB/s), 100 rows 70 backward, where w is read twice and dw written.
// The products are tiles as in gemm_tiled.hip (copies HBM -> LDS, two stages, k
// tiles of 128 bytes a row); fp32 operands take the same bytes and the fp32 MFMA.
// Operand bases move along k in 64 bits, so no operand's size is limited by a
// buffer's 32-bit offsets.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <numeric>
#include <string>
#include <type_traits>

#include "gemm_tile.h"

namespace mk {
namespace {

using namespace attn;

constexpr int kGroupM = 4;                  // tile rows per group of the tile order
constexpr int kInvalid = int(0x80000000u);  // buffer offset past the range of every copy
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kThreads = 256;               // of the kernels without products

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// Element types: bytes, elements of a 16-byte chunk, and the MFMA step of one
// chunk an operand: 16 k of 16 bits, or 8 k of 32 bits in four instructions of 2
// (lane half g has k 4 g .. 4 g + 3 of them, in both operands).
struct Bf16 {
  static constexpr int esz = 2, mk = MK_BF16;
  static __device__ inline f32x16_t mma(const u32x4_t& b, const u32x4_t& a, const f32x16_t& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(b), as_bf16x8(a), c, 0, 0, 0);
  }
};
struct F16 {
  static constexpr int esz = 2, mk = MK_F16;
  static __device__ inline f32x16_t mma(const u32x4_t& b, const u32x4_t& a, const f32x16_t& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, b), __builtin_bit_cast(f16x8_t, a), c, 0,
                                                  0, 0);
  }
};
struct F32 {
  static constexpr int esz = 4, mk = MK_F32;
  static __device__ inline f32x16_t mma(const u32x4_t& b, const u32x4_t& a, f32x16_t c) {
    const f32x4_t bf = __builtin_bit_cast(f32x4_t, b), af = __builtin_bit_cast(f32x4_t, a);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(bf[e], af[e], c, 0, 0, 0);
    return c;
  }
};

// BK: 16-bit elements of a k tile (2 BK bytes a row whatever the type)
using Big = Shape<256, 256, 2, 4, 64, 2>;
using Mid = Shape<128, 128, 4, 2, 64, 2>;

template <class Sh>
struct Geo {
  static constexpr int W = Sh::WGM * Sh::WGN, threads = 64 * W;
  static constexpr int WM = Sh::TM / Sh::WGM, WN = Sh::TN / Sh::WGN;  // wave block
  static constexpr int I = WM / 32, J = WN / 32;                      // MFMA blocks of it
  static constexpr int row_bytes = 2 * Sh::BK, steps = row_bytes / 32;  // of a k tile; its MFMA steps
  static constexpr int stage = row_bytes * (Sh::TM + Sh::TN), lds_bytes = Sh::S * stage;
  static_assert(Sh::TM * Sh::TN * 2 <= lds_bytes, "a 16-bit tile is staged where the operands were");
};
template <class Sh>
using Acc = f32x16_t[Geo<Sh>::I][Geo<Sh>::J];

// ---------------------------------------------------------------- operand copies
// The 1 KB copies one wave makes of one operand's k tile (gemm_tiled.hip's
// Copies): their byte offsets from the tile's base, and the first k each reads.
// `base` is the tile's first row (KC) or column (!KC) at its first k; rows: those
// of the tile inside the operand.
template <class T, bool KC, int R, int W, int BK>
struct Operand {
  static constexpr int kRow = 2 * BK;  // bytes of k a tile row has
  static constexpr int kE = 16 / T::esz, kDeep = kRow / T::esz, kC = R * kRow / (1024 * W);
  static constexpr int kCpr = KC ? kRow / 16 : R / kE;  // chunks of an LDS row
  static_assert(kC * 1024 * W == R * kRow, "copies split evenly over the waves");
  const char* base;
  int64_t step;  // bytes from a k tile to the next
  uint32_t off[kC];
  // the tile row and the k of this lane's chunk of copy c
  static __device__ inline void chunk(int c, int wave, int lane, int& row, int& k) {
    const int u = 64 * (wave + W * c) + lane, r = u / kCpr;
    row = KC ? r : kE * ((u % kCpr) ^ (T::esz == 2 ? nc_swizzle<R>(r) : 0));
    k = KC ? kE * ((u % kCpr) ^ kc_swizzle<BK>(r)) : r;
  }
  __device__ inline Operand(int wave, int lane, const char* base, int64_t rows, int64_t ld)
      : base(base), step(KC ? kRow : kDeep * ld * T::esz) {
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      int row, k;
      chunk(c, wave, lane, row, k);
      off[c] = row < rows ? uint32_t((KC ? row * ld + k : k * ld + row) * T::esz) : uint32_t(kInvalid);
    }
  }
  // the copies of k tile kt, of which the operand has `left` k
  __device__ inline void issue(int kt, int64_t left, char* tile, int wave, int lane) const {
    const i32x4_t r = tile_desc(base + kt * step, uint32_t(kInvalid));
    if (left >= kDeep) {
#pragma unroll
      for (int c = 0; c < kC; ++c) copy_to_lds_so(r, lds_addr(tile + 1024 * (wave + W * c)), int(off[c]), 0);
      return;
    }
    asm volatile("" : "+v"(lane));  // nothing of the last tile's is held through the loop
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      int row, k;
      chunk(c, wave, lane, row, k);
      copy_to_lds(r, lds_addr(tile + 1024 * (wave + W * c)), k < left ? int(off[c]) : kInvalid);
    }
  }
};

template <class T, bool KC, int R, int BK>
__device__ inline u32x4_t read_chunk(const char* t, int rb, int ks, int lane) {
  if constexpr (KC || T::esz == 2) {  // a k-contiguous row is chunks of 16 bytes in either width
    return read_operand16<KC, R, BK>(reinterpret_cast<const uint16_t*>(t), rb, ks, lane);
  } else {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(t) + (8 * ks + 4 * (lane >> 5)) * R + rb + (lane & 31);
    return u32x4_t{p[0], p[R], p[2 * R], p[3 * R]};
  }
}

// ---------------------------------------------------------------- labels
struct Labels {
  const void* p;
  int wide;  // int64
  int has_ignore;
  int64_t ignore;
  __device__ inline int64_t at(int64_t n) const {
    return wide ? static_cast<const int64_t*>(p)[n] : int64_t(static_cast<const int32_t*>(p)[n]);
  }
  __device__ inline bool ignored(int64_t label) const { return has_ignore && label == ignore; }
};

// acc += A B of one workgroup tile over K: the k loop of gemm_tiled.hip.  A wave
// waits for its own copies of tile kt, the barrier publishes all and frees the
// other stage, whose next copies are issued beside the first k-steps' MFMAs.
// start() issues the first k tile's copies, into the first stage; run() ends with a
// barrier: the operands' LDS is free, and start() of the next product may follow.
// rest: what is added beside the operands' k tiles (LabelRest).
struct NoRest {
  __device__ inline void load(int) const {}
  __device__ inline void arrived() const {}
  template <class A>
  __device__ inline void add(int, A&) const {}
};
template <class T, class Sh, bool AKC, bool BKC>
struct Product {
  using G = Geo<Sh>;
  using OA = Operand<T, AKC, Sh::TM, G::W, Sh::BK>;
  using OB = Operand<T, BKC, Sh::TN, G::W, Sh::BK>;
  static constexpr int kA = Sh::TM * G::row_bytes;
  static_assert(Sh::S == 2, "two stages");
  OA oa;
  OB ob;
  int64_t K;
  int nk;
  __device__ inline Product(const char* A, int64_t lda, int64_t a_rows, const char* B, int64_t ldb, int64_t b_rows,
                            int64_t K, int wave, int lane)
      : oa(wave, lane, A, a_rows, lda), ob(wave, lane, B, b_rows, ldb), K(K), nk(int((K + OA::kDeep - 1) / OA::kDeep)) {}
  // A's second k tile, as long as the first (at most a k tile), with B's first again
  __device__ inline void twice() { nk = 2, ob.step = 0; }
  __device__ inline void issue(int kt, char* to, int wave, int lane, bool a, bool b) const {
    const int64_t left = K <= OA::kDeep ? K : K - int64_t(OA::kDeep) * kt;
    if (a) oa.issue(kt, left, to, wave, lane);
    if (b) ob.issue(kt, left, to + kA, wave, lane);
  }
  __device__ inline void start(char* lds, int wave, int lane) const {
    if (nk > 0) issue(0, lds, wave, lane, true, true);
  }
  // LATE: stores that may still be on their way when the first k tile is there (late: so many
  // or more came after its copies)
  template <int LATE = 0, class Beside = NoRest>
  __device__ __attribute__((always_inline)) inline void run(char* lds, int wave, int lane, Acc<Sh>& acc,
                                                            bool late = false, Beside&& rest = {}) const {
    const int wm = wave / Sh::WGN, wn = wave % Sh::WGN;
    for (int kt = 0; kt < nk; ++kt) {
      if (LATE > 0 && late && kt == 0) wait_vm<LATE>();
      else wait_vm<0>();
      lds_barrier();
      rest.arrived();
      const char* at = lds + (kt & 1) * G::stage;
      char* next = lds + ((kt + 1) & 1) * G::stage;
      const bool more = kt + 1 < nk;
#pragma unroll
      for (int ks = 0; ks < G::steps; ++ks) {
        u32x4_t af[G::I], bf[G::J];
#pragma unroll
        for (int a = 0; a < G::I; ++a) af[a] = read_chunk<T, AKC, Sh::TM, Sh::BK>(at, wm * G::WM + 32 * a, ks, lane);
#pragma unroll
        for (int b = 0; b < G::J; ++b) bf[b] = read_chunk<T, BKC, Sh::TN, Sh::BK>(at + kA, wn * G::WN + 32 * b, ks, lane);
        if (more && ks < 2) issue(kt + 1, next, wave, lane, ks == 0, ks == 1);
        if (more && ks == 1) rest.load(kt + 1);
#pragma unroll
        for (int a = 0; a < G::I; ++a)
#pragma unroll
          for (int b = 0; b < G::J; ++b) acc[a][b] = T::mma(bf[b], af[a], acc[a][b]);
      }
      rest.add(kt, acc);
    }
    lds_barrier();
  }
};

template <class Sh>
__device__ inline void zero(Acc<Sh>& acc) {
#pragma unroll
  for (int a = 0; a < Geo<Sh>::I; ++a)
#pragma unroll
    for (int b = 0; b < Geo<Sh>::J; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
}

// The tile of a tiles_m x tiles_n grid that workgroup i of nt has: an XCD (i % 8)
// has a run of tiles, which walk groups of 4 tile rows column by column.  False:
// there are fewer than nt.
__device__ inline bool tile_of(uint32_t i, uint32_t nt, uint32_t tiles_m, uint32_t tiles_n, uint32_t& tm, uint32_t& tn) {
  if (nt == 0) return false;
  const uint32_t per = nt / 8, t = i < 8 * per ? (i % 8) * per + i / 8 : i;
  if (t >= tiles_m * tiles_n) return false;
  const uint32_t first = t / (kGroupM * tiles_n) * kGroupM, gm = min(uint32_t(kGroupM), tiles_m - first);
  const uint32_t in = t - first * tiles_n;
  tm = first + in % gm;
  tn = in / gm;
  return t < tiles_m * tiles_n;
}

// ---------------------------------------------------------------- forward
struct LossArgs {
  const char *x, *w;       // w: of this piece
  int64_t rows, width, vocab;  // vocab: of this piece
  int64_t ld_x, ld_w;
  int64_t v0;              // the piece's first class
  int tiles_m, tiles_n;
  Labels labels;
  float2* part;            // [tiles_n][rows]: the maximum and the sum of e^(s - maximum)
  float* target;           // [rows]: the label's logit
};

// Exponentials are of base 2, of s log2(e) - t in one instruction, with t the rounded
// product of the row's maximum and log2(e); the sum is then made relative to the
// maximum itself, which undoes t's rounding.  That is at most 2^-15 where t is below 2^10;
// past that (weights of a type's lowest value give logits up to the end of fp32's
// range, where it is more than an exponent can hold) differences are taken first, an
// instruction more.
__device__ inline float base2(float top, bool& plain) {
  const float t = top * kLog2e;
  plain = fabsf(t) < 1024.f;
  return plain ? t : 0.f;
}
// e^(top - to): what a sum relative to top weighs among those relative to `to`, the largest
// top, or 0 where that is -inf (all sums are 0 then)
__device__ inline float weight(float top, float to) { return __builtin_amdgcn_exp2f((top - to) * kLog2e); }
__device__ inline float or_zero(float top) { return top == -INFINITY ? 0.f : top; }

// A workgroup has every gridDim-th tile, and the next one's first copies in flight
// while it ends a tile.
template <class T, class Sh>
__global__ __launch_bounds__(Geo<Sh>::threads, 2) void loss_kernel(const LossArgs p) {
  using G = Geo<Sh>;
  using P = Product<T, Sh, true, true>;
  __shared__ __attribute__((aligned(1024))) char lds[G::lds_bytes];
  __shared__ float2 red[Sh::WGN * Sh::TM];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / Sh::WGN, wn = wave % Sh::WGN, c = lane & 31, g = lane >> 5;
  const uint32_t nt = uint32_t(p.tiles_m) * uint32_t(p.tiles_n);
  auto tile = [&](uint32_t i, int64_t& m0, int64_t& n0) __attribute__((always_inline)) {
    uint32_t tm, tn;
    tile_of(i, nt, uint32_t(p.tiles_m), uint32_t(p.tiles_n), tm, tn);
    m0 = int64_t(tm) * Sh::TM, n0 = int64_t(tn) * Sh::TN;
    return P(p.x + m0 * p.ld_x * T::esz, p.ld_x, p.rows - m0, p.w + n0 * p.ld_w * T::esz, p.ld_w, p.vocab - n0, p.width,
             wave, lane);
  };
  int64_t m0, n0;
  P now = tile(blockIdx.x, m0, n0);
  now.start(lds, wave, lane);
  for (uint32_t i = blockIdx.x;;) {
    int rel[G::I];  // the label's column of this wave's, -1: none
#pragma unroll
    for (int a = 0; a < G::I; ++a) {
      const int64_t m = m0 + wm * G::WM + 32 * a + c;
      const int64_t at = m < p.rows ? p.labels.at(m) - p.v0 - n0 - wn * G::WN : -1;
      rel[a] = at >= 0 && at < G::WN ? int(at) : -1;
    }
    Acc<Sh> acc;
    zero<Sh>(acc);
    now.run(lds, wave, lane, acc);
    const int64_t m_now = m0, n_now = n0;
    i += gridDim.x;
    if (i < nt) {
      now = tile(i, m0, n0);
      now.start(lds, wave, lane);
    }
    // a lane has, of row 32 a + c, the columns 32 b + 8 (r / 4) + 4 g + r % 4
    if (n_now + Sh::TN > p.vocab) {
      const int64_t left = p.vocab - n_now - wn * G::WN - 4 * g;
#pragma unroll
      for (int b = 0; b < G::J; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * b + 8 * (r / 4) + r % 4 >= left)
#pragma unroll
            for (int a = 0; a < G::I; ++a) acc[a][b][r] = -INFINITY;
    }
#pragma unroll
    for (int a = 0; a < G::I; ++a) {
      const int ml = wm * G::WM + 32 * a + c;
      if (rel[a] >= 0) {
#pragma unroll
        for (int b = 0; b < G::J; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (rel[a] == 32 * b + 8 * (r / 4) + 4 * g + r % 4) p.target[m_now + ml] = acc[a][b][r];
      }
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < G::J; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[a][b][r]);
      float lo, hi;
      lane_halves_sched(top, lo, hi);
      top = fmaxf(lo, hi);
      bool plain;
      const float from = base2(top, plain);
      if (!plain && top != -INFINITY) {
#pragma unroll
        for (int b = 0; b < G::J; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[a][b][r] -= top;
      }
      float sum = 0.f;
#pragma unroll
      for (int b = 0; b < G::J; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(fmaf(acc[a][b][r], kLog2e, -from));
      lane_halves_sched(sum, lo, hi);
      sum = lo + hi;
      if (plain) sum *= __builtin_amdgcn_exp2f(fmaf(top, -kLog2e, from));
      if (g == 0) red[wn * Sh::TM + ml] = float2{top, sum};
    }
    lds_barrier();
    for (int e = int(threadIdx.x); e < Sh::TM; e += G::threads) {
      if (m_now + e >= p.rows) break;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int q = 0; q < Sh::WGN; ++q) top = fmaxf(top, red[q * Sh::TM + e].x);
#pragma unroll
      for (int q = 0; q < Sh::WGN; ++q) sum += red[q * Sh::TM + e].y * weight(red[q * Sh::TM + e].x, or_zero(top));
      p.part[n_now / Sh::TN * p.rows + m_now + e] = float2{top, sum};
    }
    if (i >= nt) return;
  }
}

// A row's tiles joined: 16 rows a block, 16 threads a row over the tiles (64 where there are
// few rows), 8 of them loaded at a time (one after the other a row's 393 tiles took 9 us).
template <int NT>
__global__ __launch_bounds__(16 * NT) void loss_final_kernel(const float2* part, const float* target, int64_t rows,
                                                              int64_t vocab, int64_t tiles, Labels labels, float* loss,
                                                              float* lse) {
  constexpr int kAt = 8;
  __shared__ float2 red[NT / 4][16];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t n = int64_t(blockIdx.x) * 16 + tx;
  float top = -INFINITY, sum = 0.f;
  if (n < rows) {
    for (int64_t t = ty; t < tiles; t += NT * kAt) {
      float2 v[kAt];
#pragma unroll
      for (int i = 0; i < kAt; ++i) v[i] = t + NT * i < tiles ? part[(t + NT * i) * rows + n] : float2{-INFINITY, 0.f};
      float to = top;
#pragma unroll
      for (int i = 0; i < kAt; ++i) to = fmaxf(to, v[i].x);
      const float from = or_zero(to);
      sum *= weight(top, from);
#pragma unroll
      for (int i = 0; i < kAt; ++i) sum += v[i].y * weight(v[i].x, from);
      top = to;
    }
  }
  // 4 of them are lanes of a wave
#pragma unroll
  for (int d = 16; d < 64; d *= 2) {
    const float t = __shfl_xor(top, d), more = __shfl_xor(sum, d), to = fmaxf(top, t), from = or_zero(to);
    const float mine = sum * weight(top, from), its = more * weight(t, from);
    sum = mine + its;  // the same in both lanes
    top = to;
  }
  if (ty % 4 == 0) red[ty / 4][tx] = float2{top, sum};
  __syncthreads();
  if (ty != 0 || n >= rows) return;
#pragma unroll
  for (int i = 1; i < NT / 4; ++i) top = fmaxf(top, red[i][tx].x);
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 4; ++i) sum += red[i][tx].y * weight(red[i][tx].x, or_zero(top));
  const float z = top + log2f(sum) * kLn2;
  if (lse) lse[n] = z;
  if (!loss) return;
  const int64_t label = labels.at(n);
  loss[n] = labels.ignored(label) ? 0.f : (label >= 0 && label < vocab ? z - target[n] : z);
}

// ---------------------------------------------------------------- operands off the 16-byte boundaries
// Rows copied to a pitch of whole 16-byte chunks with zeros past their end, and
// (has_ignore) zeros for ignored rows, which g's zeros would not keep out of dw
// if they held infinities.  again > 0: every `again` rows anew, zeros past `held` of them.
struct PackArgs {
  const void* src;
  int64_t ld, rows, cols;
  void* dst;
  int64_t ld_dst;
  Labels labels;
  int64_t held;
  int again;
};
template <typename U, int THREADS>
__device__ inline void pack_block(const PackArgs& p, int64_t block) {
  constexpr int kE = 16 / int(sizeof(U));
  struct __attribute__((packed, aligned(sizeof(U)))) Any { U v[kE]; };  // 16 bytes at any element
  struct alignas(16) Chunk { U v[kE]; };
  const int64_t chunks = p.ld_dst / kE, first = block * THREADS;
  const uint32_t in = uint32_t(first % chunks) + threadIdx.x;
  const int64_t to = first / chunks + in / uint32_t(chunks), col = int64_t(in % uint32_t(chunks)) * kE;
  const int64_t row = p.again ? to % p.again : to;
  if (to >= p.rows) return;
  const U* src = static_cast<const U*>(p.src) + row * p.ld + col;
  Chunk c;
  if (row >= p.held || (p.labels.has_ignore && p.labels.ignored(p.labels.at(row)))) {
#pragma unroll
    for (int e = 0; e < kE; ++e) c.v[e] = U(0);
  } else if (col + kE <= p.cols) {
    const Any l = *reinterpret_cast<const Any*>(src);
#pragma unroll
    for (int e = 0; e < kE; ++e) c.v[e] = l.v[e];
  } else {
#pragma unroll
    for (int e = 0; e < kE; ++e) c.v[e] = col + e < p.cols ? src[e] : U(0);
  }
  *reinterpret_cast<Chunk*>(static_cast<U*>(p.dst) + to * p.ld_dst + col) = c;
}

// ---------------------------------------------------------------- backward: g
struct Rest {
  int label;   // -1: outside the vocabulary, or the row is ignored
  float left;  // what the rounding of g leaves of the label's element, in g's scale
};
struct GradArgs {
  const char *x, *w;
  int64_t rows, width, vocab;  // vocab: of this piece
  int64_t ld_x, ld_w, v0, all;  // all: classes of the vocabulary
  int tiles_m, tiles_n;
  Labels labels;
  const float *lse, *row_grad;
  const float* dyn;  // {factor of g, factor of the products} on the device, or null: `unit`
  float unit;        // factor of g
  char* g;           // [rows][ld_g], columns past vocab up to a whole chunk are zeros
  int64_t ld_g;
  int low;           // what g's rounding leaves goes to the rows kLow further on
  Rest* rest;        // [rows] (16 bits without those rows), or null
  PackArgs pack;     // of few rows: dw's x, by the workgroups past the tiles
};

__device__ inline uint32_t pack2(Bf16, float a, float b) {
  return uint32_t(f32_to_bf16(a)) | (uint32_t(f32_to_bf16(b)) << 16);
}
__device__ inline uint32_t pack2(F16, float a, float b) { return uint32_t(f32_to_f16(a)) | (uint32_t(f32_to_f16(b)) << 16); }

// of the low 16 bits
__device__ inline float widened(Bf16, uint32_t a) { return bf16_to_f32(uint16_t(a)); }
__device__ inline float widened(F16, uint32_t a) { return f16_to_f32(uint16_t(a)); }

__device__ inline float rounded(Bf16, float a) { return bf16_to_f32(f32_to_bf16(a)); }
__device__ inline float rounded(F32, float a) { return a; }
__device__ inline float rounded(F16, float a) { return f16_to_f32(f32_to_f16(a)); }

// 16 bits: the 8 columns 32 b + 16 h + 8 g .. + 7 of a lane's row 32 a + c as one
// chunk.  value(a, b, rg, v) gives the 4 columns 32 b + 8 rg + 4 g .. + 3; lanes l
// and l + 32 trade halves of them.
template <class T, class V>
__device__ __attribute__((always_inline)) inline u32x4_t chunk16(int a, int b, int h, V&& value) {
  uint2 w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float v[4];
    value(a, b, 2 * h + e, v);
    w[e] = uint2{pack2(T{}, v[0], v[1]), pack2(T{}, v[2], v[3])};
  }
  const auto s0 = __builtin_amdgcn_permlane32_swap(w[0].x, w[1].x, false, false);
  const auto s1 = __builtin_amdgcn_permlane32_swap(w[0].y, w[1].y, false, false);
  return u32x4_t{static_cast<uint32_t>(s0[0]), static_cast<uint32_t>(s1[0]), static_cast<uint32_t>(s0[1]),
                 static_cast<uint32_t>(s1[1])};
}

// 16 bytes at an element's alignment: one instruction, whatever the address
template <class T> using Elem = std::conditional_t<T::esz == 2, uint16_t, uint32_t>;
template <class T> struct __attribute__((packed, aligned(sizeof(Elem<T>)))) Loose { u32x4_t v; };
template <class T>
__device__ inline u32x4_t loose16(const char* p) {
  return reinterpret_cast<const Loose<T>*>(p)->v;
}
// The same to a row's elements, of which `left` are inside.
template <class T>
__device__ inline void store_chunk(char* to, const u32x4_t& v, int64_t left) {
  constexpr int kE = 16 / T::esz;
  if (left >= kE) {
    reinterpret_cast<Loose<T>*>(to)->v = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < kE; ++e)
    if (e < left)
      reinterpret_cast<Elem<T>*>(to)[e] = T::esz == 2 ? Elem<T>(v[e / 2] >> 16 * (e & 1)) : Elem<T>(v[e % 4]);
}

// A tile of 16-bit results, whole chunks of rows (cols a multiple of 8), through a part of
// LDS that is the wave's own: a row of its block is one line, and 8 of them go out in an
// instruction (straight from the accumulators each would have 32 bytes of 32 rows:
// 403 us against 392 for g of 8192 x 768 x 26624).  Rows and cols: what of the tile is stored.
template <class T, class Sh, class V>
__device__ __attribute__((always_inline)) inline void store16_wave(char* lds, int wave, int lane, char* out, int64_t ld,
                                                                   int64_t rows, int64_t cols, V&& value) {
  using G = Geo<Sh>;
  static_assert(G::WN == 64, "a line a row");
  constexpr int kRows = std::min(G::WM, G::stage / G::W / 128);  // at a time
  const int wm = wave / Sh::WGN, wn = wave % Sh::WGN, c = lane & 31, g = lane >> 5, row = lane >> 3, nl = wn * 64 + 8 * (lane & 7);
  char* st = lds + wave * (kRows * 128);
  char* to = out + (int64_t(wm * G::WM + row) * ld + nl) * 2;
#pragma unroll
  for (int r0 = 0; r0 < G::WM; r0 += kRows) {
#pragma unroll
    for (int a = 0; a < kRows / 32; ++a)
#pragma unroll
      for (int b = 0; b < G::J; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<u32x4_t*>(st + (32 * a + c) * 128 + 16 * ((4 * b + 2 * h + g) ^ (c & 7))) =
              chunk16<T>(r0 / 32 + a, b, h, value);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < kRows / 8; ++i) {
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(st + (8 * i + row) * 128 + 16 * ((lane & 7) ^ row));
      if (wm * G::WM + r0 + 8 * i + row < rows && nl < cols) *reinterpret_cast<u32x4_t*>(to) = v;
      to += 16 * ld;
    }
    asm volatile("" ::: "memory");
  }
}

// A tile of 16-bit results of any alignment through LDS (gemm_tiled.hip's
// store_staged): rows go out in runs of 16 bytes.
template <class T, class Sh, class V>
__device__ __attribute__((always_inline)) inline void store16(char* lds, int wave, int lane, char* out, int64_t ld,
                                                              int64_t rows, int64_t cols, V&& value) {
  using G = Geo<Sh>;
  constexpr int kCpr = Sh::TN / 8;
  static_assert(kCpr % 16 == 0, "staging rows of whole 16-chunk groups");
  const int wm = wave / Sh::WGN, wn = wave % Sh::WGN, c = lane & 31, g = lane >> 5;
  uint16_t* st = reinterpret_cast<uint16_t*>(lds);
#pragma unroll
  for (int a = 0; a < G::I; ++a) {
    const int ml = wm * G::WM + 32 * a + c;
#pragma unroll
    for (int b = 0; b < G::J; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int cn = (wn * G::WN + 32 * b + 16 * h + 8 * g) >> 3;
        *reinterpret_cast<u32x4_t*>(st + ml * Sh::TN + 8 * (cn ^ (ml & 15))) = chunk16<T>(a, b, h, value);
      }
  }
  lds_barrier();
#pragma unroll 4
  for (int it = 0; it < Sh::TM * kCpr / G::threads; ++it) {
    const int e = it * G::threads + int(threadIdx.x), row = e / kCpr, cn = e % kCpr;
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(st + row * Sh::TN + 8 * (cn ^ (row & 15)));
    if (row < rows) store_chunk<T>(out + (row * ld + 8 * cn) * 2, v, cols - 8 * cn);
  }
}

// A tile of fp32 results of any alignment straight from the accumulators: 16 bytes a
// lane (two lanes' are neighbours).
template <class Sh, class V>
__device__ __attribute__((always_inline)) inline void store32(int wave, int lane, float* out, int64_t ld,
                                                              int64_t rows, int64_t cols, V&& value) {
  using G = Geo<Sh>;
  const int wm = wave / Sh::WGN, wn = wave % Sh::WGN, c = lane & 31, g = lane >> 5;
#pragma unroll
  for (int a = 0; a < G::I; ++a) {
    const int ml = wm * G::WM + 32 * a + c;
#pragma unroll
    for (int b = 0; b < G::J; ++b)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const int nl = wn * G::WN + 32 * b + 8 * rg + 4 * g;
        float v[4];
        value(a, b, rg, v);
        if (ml < rows)
          store_chunk<F32>(reinterpret_cast<char*>(out + ml * ld + nl),
                           __builtin_bit_cast(u32x4_t, f32x4{{v[0], v[1], v[2], v[3]}}), cols - nl);
      }
  }
}

// What the rounding of g to 16 bits leaves.  A row of g is its label's element, near
// -1, and many small ones, and a class that one token has as its label gets its
// gradient from that one product: the rounding of this element would be the error of
// the whole rows of dx and dw.  So what it leaves of it is kept (Rest, fp32) and
// added to both: to dw by its tiles (LabelRest), to dx where its sums are joined.  Errors
// against 64 bits, without it and with it: 100 x 768 x 50257 bf16 0.00188, 0.00165; 1777
// x 1001 x 30011 fp16 0.000279, 0.000207, both then those of fp32 products.  Times:
// 8192 x 768 x 50257 1848 us, 1880; 1777 x 1001 x 30011 393, 400; 100 x 768 x 50257 68,
// 70; of few classes, each with many labels, 2000 x 2048 x 1500 61, 68.  (Another
// class with much of a row's probability is rounded with the rest of g.)  At most
// kLow rows have a second operand row each, what the rounding leaves of every
// element; their tiles have the room (16 bits: half of dx's 128 rows, and of dw's
// two k tiles the second), so that it costs nothing.
constexpr int kLow = 64;

// 256 x 256: a workgroup has every gridDim-th tile, as in loss_kernel: the next
// tile's first copies are issued before this one ends, and their wait leaves this
// one's stores on their way (a tile a workgroup: all store at once and then all
// wait, 388 us against 336 for g of 8192 x 768 x 23633).  What a tile needs of its rows
// lies in LDS, since registers are full.  Of 128 x 128, two workgroups a CU hide
// each other's stores.
template <class T, class Sh>
__global__ __launch_bounds__(Geo<Sh>::threads, 2) void grad_kernel(const GradArgs p) {
  using G = Geo<Sh>;
  using P = Product<T, Sh, true, true>;
  constexpr bool kOn = Sh::TM == 256;
  constexpr int kLate = kOn ? G::WM / 8 : 0;
  __shared__ __attribute__((aligned(1024))) char lds[G::lds_bytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / Sh::WGN, wn = wave % Sh::WGN, c = lane & 31, g = lane >> 5;
  const uint32_t nt = uint32_t(p.tiles_m) * uint32_t(p.tiles_n);
  auto tile = [&](uint32_t i, int64_t& m0, int64_t& n0) __attribute__((always_inline)) {
    uint32_t tm, tn;
    tile_of(i, nt, uint32_t(p.tiles_m), uint32_t(p.tiles_n), tm, tn);
    m0 = int64_t(tm) * Sh::TM, n0 = int64_t(tn) * Sh::TN;
    return P(p.x + m0 * p.ld_x * T::esz, p.ld_x, p.rows - m0, p.w + n0 * p.ld_w * T::esz, p.ld_w, p.vocab - n0, p.width,
             wave, lane);
  };
  const float unit = p.dyn ? p.dyn[0] : p.unit;
  // of a tile's rows: lse, factor, the label's column of the tile or -1, or -2: the row is ignored
  __shared__ float row_lse[2][Sh::TM], row_factor[2][Sh::TM];
  __shared__ int row_rel[2][Sh::TM];
  __shared__ float row_label[Sh::TM];  // the label's element without its factor, for the lane that had it
  static_assert(Sh::TM <= G::threads, "a thread a row");
  const int t = int(threadIdx.x);
  int64_t label;
  float z, f;
  auto rows_load = [&](int64_t m0) __attribute__((always_inline)) {
    label = -1, z = f = 0.f;
    if (t < Sh::TM && m0 + t < p.rows) {
      label = p.labels.at(m0 + t);
      z = p.lse[m0 + t];
      f = p.row_grad ? p.row_grad[m0 + t] : 1.f;
    }
  };
  auto rows_keep = [&](int at, int64_t n0) __attribute__((always_inline)) {
    if (t >= Sh::TM) return;
    const int64_t col = label - p.v0 - n0;
    const bool ignored = p.labels.ignored(label);
    row_lse[at][t] = z;
    row_factor[at][t] = ignored ? 0.f : unit * f;
    row_rel[at][t] = ignored ? -2 : col >= 0 && col < Sh::TN ? int(col) : -1;
  };
  int64_t m0, n0;
  P now = tile(blockIdx.x, m0, n0);
  now.start(lds, wave, lane);
  rows_load(m0);
  rows_keep(0, n0);
  if constexpr (T::esz == 2) {
    if (p.rest && p.v0 == 0) {
      for (int64_t n = int64_t(blockIdx.x) * G::threads + t; n < p.rows; n += int64_t(gridDim.x) * G::threads) {
        const int64_t l = p.labels.at(n);
        p.rest[n].label = l >= 0 && l < p.all && !p.labels.ignored(l) ? int(l) : -1;
      }
    }
  }
  bool late = false;
  int at = 0;
  for (uint32_t i = blockIdx.x;;) {
    Acc<Sh> acc;
    if constexpr (T::esz == 2) {
      // from -lse on: the difference costs no instruction, and holds where lse log2(e) would not
      lds_barrier();
#pragma unroll
      for (int a = 0; a < G::I; ++a) {
        const float from = -row_lse[at][wm * G::WM + 32 * a + c];
#pragma unroll
        for (int b = 0; b < G::J; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[a][b][r] = from;
      }
    } else {
      zero<Sh>(acc);
    }
    now.template run<kLate>(lds, wave, lane, acc, late);
    const int64_t m_now = m0, n_now = n0;
    i += gridDim.x;
    if (kOn && i < nt) {
      now = tile(i, m0, n0);
      now.start(lds, wave, lane);
      rows_load(m0);
    }
    int rel[G::I];
    bool counts = true;
#pragma unroll
    for (int a = 0; a < G::I; ++a) {
      rel[a] = row_rel[at][wm * G::WM + 32 * a + c];
      if (rel[a] == -2) counts = false;
    }
    // Most tiles have every class, and waves no ignored row: an exponential, its
    // exponent and a factor for each element.  The label's -1 is put in afterwards
    // by the few lanes that have one.
    const bool some = !__all(counts) || n_now + Sh::TN > p.vocab;
    const int64_t left = p.vocab - n_now - wn * G::WN - 4 * g;  // columns below it exist
    bool found = false;  // a label's element
#pragma unroll
    for (int a = 0; a < G::I; ++a) {
      const float lse = T::esz == 4 ? row_lse[at][wm * G::WM + 32 * a + c] : 0.f;
      const int mine = rel[a] - wn * G::WN - 4 * g;
#pragma unroll
      for (int b = 0; b < G::J; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          // 32-bit results: the difference of whole sums, which is exact where it is small
          acc[a][b][r] = __builtin_amdgcn_exp2f((T::esz == 4 ? acc[a][b][r] - lse : acc[a][b][r]) * kLog2e);
      if (rel[a] >= 0 && mine >= 0 && mine < G::WN && !(mine & 4)) {
        found = true;
#pragma unroll
        for (int b = 0; b < G::J; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (mine == 32 * b + 8 * (r / 4) + r % 4) row_label[wm * G::WM + 32 * a + c] = acc[a][b][r] -= 1.f;
      }
    }
    if (some) {
#pragma unroll
      for (int a = 0; a < G::I; ++a)
#pragma unroll
        for (int b = 0; b < G::J; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            // selected: an ignored row's logits may be anything
            if (rel[a] == -2 || 32 * b + 8 * (r / 4) + r % 4 >= left) acc[a][b][r] = 0.f;
    }
#pragma unroll
    for (int a = 0; a < G::I; ++a) {
      const float factor = row_factor[at][wm * G::WM + 32 * a + c];
#pragma unroll
      for (int b = 0; b < G::J; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[a][b][r] *= factor;
    }
    at ^= 1;
    if (kOn && i < nt) rows_keep(at, n0);
    auto value = [&](int a, int b, int rg, float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = acc[a][b][4 * rg + q];
    };
    constexpr int kE = 16 / T::esz;
    const int64_t rows = p.rows - m_now, cols = (p.vocab + kE - 1) / kE * kE - n_now;
    char* out = p.g + (m_now * p.ld_g + n_now) * T::esz;
    if constexpr (T::esz == 2) {
      store16_wave<T, Sh>(lds + G::stage, wave, lane, out, p.ld_g, rows, cols, value);
      late = rows >= Sh::TM && cols >= Sh::TN;  // every lane stored
      if constexpr (Sh::TM == 128) {
        if (p.low) {
          store16_wave<T, Sh>(lds + G::stage, wave, lane, out + kLow * p.ld_g * T::esz, p.ld_g, rows, cols,
                              [&](int a, int b, int rg, float (&v)[4]) __attribute__((always_inline)) {
                                value(a, b, rg, v);
#pragma unroll
                                for (int q = 0; q < 4; ++q) v[q] -= rounded(T{}, v[q]);
                              });
        }
      }
    } else {
      store32<Sh>(wave, lane, reinterpret_cast<float*>(out), p.ld_g, rows, cols, value);
    }
    if constexpr (T::esz == 2) {
      if (p.rest && __any(found)) {  // now that the accumulators' registers are free
#pragma unroll
        for (int a = 0; a < G::I; ++a) {
          const int row = wm * G::WM + 32 * a + c, rel_at = row_rel[at ^ 1][row], mine = rel_at - wn * G::WN - 4 * g;
          if (rel_at < 0 || mine < 0 || mine >= G::WN || (mine & 4)) continue;
          const float v = row_label[row] * row_factor[at ^ 1][row];
          p.rest[m_now + row].left = v - rounded(T{}, v);
        }
      }
    }
    if (!kOn || i >= nt) return;
  }
}

// ---------------------------------------------------------------- backward: dx and dw of a piece
struct ProductsArgs {
  const char *g, *x, *w;
  int64_t rows, width, vocab;  // vocab: of this piece
  int64_t ld_g, ld_x, ld_w;
  // dx: tiles of rows x width, the piece's classes cut into `slices` runs of `run`
  int dx_m, dx_n, slices;
  int64_t run;
  int dx_first;    // dx's runs before dw's tiles
  int first;       // the first piece: sums start from zero
  float* sums;     // [slices][dx tile][accumulators]
  // dw: tiles of classes x width; where they are few their rows are cut too
  int dw_m, dw_n, dw_slices;
  int64_t dw_run;
  float* dw_sums;  // as sums, of more than one slice
  int low;         // g has its second rows
  const Rest* rest;  // GradArgs' rest
  int64_t v0;        // the piece's first class
  char* dw;        // the piece's rows
  int64_t ld_dw;
  int dw_f32;
  const float* dyn;
  float unit;      // factor of dw
};

// a tile's accumulators as they lie in a slice's sums
template <class Sh>
__device__ __attribute__((always_inline)) inline void keep_sums(const Acc<Sh>& acc, f32x4* sums) {
  using G = Geo<Sh>;
#pragma unroll
  for (int a = 0; a < G::I; ++a)
#pragma unroll
    for (int b = 0; b < G::J; ++b)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg)
        sums[((a * G::J + b) * 4 + rg) * G::threads + threadIdx.x] =
            f32x4{{acc[a][b][4 * rg], acc[a][b][4 * rg + 1], acc[a][b][4 * rg + 2], acc[a][b][4 * rg + 3]}};
}
template <class Sh>
__device__ __attribute__((always_inline)) inline void take_sums(Acc<Sh>& acc, const f32x4* sums) {
  using G = Geo<Sh>;
#pragma unroll
  for (int a = 0; a < G::I; ++a)
#pragma unroll
    for (int b = 0; b < G::J; ++b)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const f32x4 v = sums[((a * G::J + b) * 4 + rg) * G::threads + threadIdx.x];
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[a][b][4 * rg + q] = v.v[q];
      }
}

// dw's share of `rest`: row n adds left x[n] to its label's class.  A wave lists the rows
// with a label in its classes as the k loop passes them (lane l has row l of a k tile's
// 64), and multiplies 64 of them, or what there is at the end, as four more steps of
// 16 rows: their x comes from memory as a lane needs it, and A holds each row's rest at
// its label and zeros.  (Multiplied within the k tile that has them, dx's and dw's launch
// of 8192 x 768 x 26624 took 34 us of 580 more, so 14: a wait is the whole workgroup's.)
template <class T, class Sh>
struct LabelRest {
  using G = Geo<Sh>;
  struct Entry {
    int row;        // of the run
    uint32_t part;  // its label's class of the wave's, and in the low half what is left, rounded to T
  };
  static constexpr int kMost = 128;  // 63 kept and a k tile's
  Entry* list;       // in LDS, the wave's own
  const Rest* rows;  // the run's first row; null: none (nor where the wave has no columns)
  int64_t count;     // its rows
  int first, classes;  // the wave's first class of the vocabulary, and those of its classes that are the piece's
  const char* x;       // the run's first row of x, at the wave's first column
  int64_t ld_x, cols;  // cols: those from there on
  int lane;
  Rest next, now;  // of the k tile on its way, and of the one that is multiplied
  int n = 0;
  __device__ inline void load(int kt) {
    const int64_t at = 64 * int64_t(kt) + lane;
    next = Rest{-1, 0.f};
    if (rows && at < count) next = rows[at];
  }
  __device__ inline void arrived() {
    now = next;
    asm volatile("" : "+v"(now.label), "+v"(now.left));  // waited for here, not past the next copies
  }
  __device__ inline void add(int kt, Acc<Sh>& acc) {
    const unsigned at = unsigned(now.label) - unsigned(first);
    const bool mine = now.label >= 0 && at < unsigned(classes);
    const uint64_t all = __ballot(mine);
    if (all == 0) return;
    const int before = __builtin_amdgcn_mbcnt_hi(uint32_t(all >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(all), 0));
    if (mine) list[n + before] = Entry{64 * kt + lane, at << 16 | (pack2(T{}, now.left, 0.f) & 0xFFFFu)};
    n += __builtin_popcountll(all);
    if (n < 64) return;
    multiply(64, acc);
    list[lane] = list[64 + lane];
    n -= 64;
  }
  __device__ __attribute__((always_inline)) inline void multiply(int most, Acc<Sh>& acc) const {
    const int c = lane & 31, g = lane >> 5;
    asm volatile("" ::: "memory");  // what other lanes listed: LDS is in order
#pragma unroll 1
    for (int k0 = 0; k0 < most; k0 += 16) {
      uint32_t part[8], v[G::J][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int e = k0 + 8 * g + j;
        const Entry at = list[min(e, most - 1)];
        part[j] = e < most ? at.part : 0xFFFF0000u;  // no class
        const uint16_t* row = reinterpret_cast<const uint16_t*>(x + int64_t(at.row) * ld_x * 2);
#pragma unroll
        for (int b = 0; b < G::J; ++b) v[b][j] = row[min(int64_t(32 * b + c), cols - 1)];
      }
      u32x4_t bf[G::J];
#pragma unroll
      for (int b = 0; b < G::J; ++b)
#pragma unroll
        for (int w = 0; w < 4; ++w) bf[b][w] = v[b][2 * w] | v[b][2 * w + 1] << 16;
#pragma unroll
      for (int a = 0; a < G::I; ++a) {
        u32x4_t af;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t mine = uint32_t(32 * a + c);
          af[w] = (part[2 * w] >> 16 == mine ? part[2 * w] & 0xFFFFu : 0u) |
                  (part[2 * w + 1] >> 16 == mine ? part[2 * w + 1] << 16 : 0u);
        }
#pragma unroll
        for (int b = 0; b < G::J; ++b) acc[a][b] = T::mma(bf[b], af, acc[a][b]);
      }
    }
  }
};

// REST: of more than kLow rows of 16 bits; the others do without its lists (32 x 768 x 50257
// 62.8 us with them, 61.8 without)
template <class T, class Sh, bool REST>
__global__ __launch_bounds__(Geo<Sh>::threads, 2) void products_kernel(const ProductsArgs p) {
  using G = Geo<Sh>;
  constexpr int64_t kTile = Sh::TM * Sh::TN / 4;  // of a slice's sums, in f32x4
  __shared__ __attribute__((aligned(1024))) char lds[G::lds_bytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The longer ones first mostly, and the others fill the last round (1000 x 768 x
  // 50257: dx's runs first 266 us, dw's tiles 305).  Both start at a multiple of 8, an
  // XCD each.
  const uint32_t n_dw = (uint32_t(p.dw_m) * p.dw_n * p.dw_slices + 7) / 8 * 8;
  const uint32_t n_dx = uint32_t(p.dx_m) * p.dx_n * p.slices, dx_at = p.dx_first ? 0 : n_dw;
  const uint32_t dw_at = p.dx_first ? (n_dx + 7) / 8 * 8 : 0;
  Acc<Sh> acc;
  uint32_t tm, tn;
  if (p.dx_first ? blockIdx.x < dw_at : blockIdx.x >= n_dw) {
    // a slice of the classes is one XCD's (of 8 slices), with all of dx's tiles
    const uint32_t j = blockIdx.x - dx_at, slice = j % p.slices, tile = j / p.slices;
    if (j >= n_dx) return;
    tm = tile / p.dx_n, tn = tile % p.dx_n;
    const int64_t m0 = int64_t(tm) * Sh::TM, n0 = int64_t(tn) * Sh::TN, k0 = slice * p.run;
    f32x4* sums = reinterpret_cast<f32x4*>(p.sums) + (int64_t(slice) * p.dx_m * p.dx_n + tile) * kTile;
    if (p.first) zero<Sh>(acc);
    else take_sums<Sh>(acc, sums);
    const Product<T, Sh, true, false> dx(p.g + (m0 * p.ld_g + k0) * T::esz, p.ld_g, p.rows + (p.low ? kLow : 0) - m0,
                                         p.w + (k0 * p.ld_w + n0) * T::esz, p.ld_w, p.width - n0,
                                         min(p.run, p.vocab - k0), wave, lane);
    dx.start(lds, wave, lane);
    dx.run(lds, wave, lane, acc);
    keep_sums<Sh>(acc, sums);
    return;
  }
  if (!tile_of(blockIdx.x - dw_at, n_dw, uint32_t(p.dw_m), uint32_t(p.dw_n) * p.dw_slices, tm, tn)) return;
  const uint32_t slice = tn / p.dw_n;
  tn %= p.dw_n;
  const int64_t m0 = int64_t(tm) * Sh::TM, n0 = int64_t(tn) * Sh::TN, k0 = slice * p.dw_run;
  zero<Sh>(acc);
  Product<T, Sh, false, false> dw(p.g + (k0 * p.ld_g + m0) * T::esz, p.ld_g, p.vocab - m0,
                                  p.x + (k0 * p.ld_x + n0) * T::esz, p.ld_x, p.width - n0, min(p.dw_run, p.rows - k0), wave,
                                  lane);
  static_assert(128 / Bf16::esz == kLow, "g's second rows are the second k tile");
  if (p.low) dw.twice();
  dw.start(lds, wave, lane);
  if constexpr (REST) {
    using L = LabelRest<T, Sh>;
    __shared__ typename L::Entry lists[G::W][L::kMost];
    const int64_t c0 = m0 + wave / Sh::WGN * G::WM, d0 = n0 + wave % Sh::WGN * G::WN;
    L rest{lists[wave], d0 < p.width ? p.rest + k0 : nullptr, min(p.dw_run, p.rows - k0), int(p.v0 + c0),
           int(max(int64_t(0), min(int64_t(G::WM), p.vocab - c0))), p.x + (k0 * p.ld_x + d0) * 2, p.ld_x,
           p.width - d0, lane};
    rest.load(0);
    dw.template run<0>(lds, wave, lane, acc, false, rest);
    rest.multiply(rest.n, acc);
  } else {
    dw.run(lds, wave, lane, acc);
  }
  if (p.dw_slices > 1) {
    keep_sums<Sh>(acc, reinterpret_cast<f32x4*>(p.dw_sums) +
                           ((int64_t(slice) * p.dw_m + tm) * p.dw_n + tn) * kTile);
    return;
  }
  const float unit = p.dyn ? p.dyn[1] : p.unit;
  auto value = [&](int a, int b, int rg, float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = acc[a][b][4 * rg + q] * unit;
  };
  const int64_t rows = p.vocab - m0, cols = p.width - n0;
  if constexpr (T::esz == 2) {
    if (!p.dw_f32) {
      store16<T, Sh>(lds, wave, lane, p.dw + (m0 * p.ld_dw + n0) * 2, p.ld_dw, rows, cols, value);
      return;
    }
  }
  store32<Sh>(wave, lane, reinterpret_cast<float*>(p.dw) + m0 * p.ld_dw + n0, p.ld_dw, rows, cols, value);
}

// dx, or dw = the slices' sums times the factor.  A block has the 32 rows x WN columns of
// one of a wave's accumulator rows, as they lay, and stores them in rows through
// LDS.  Many slices are added by NG groups of threads, each every NG-th slice in
// order, then the groups in order (64 slices by one group: 12 us of latency).  REST: of
// dx with what is left of the labels; a kernel of its own, since the labels' loads beside
// the slices' cost calls without them too (40 x 2048 x 32000 11.9 us, 5.4).
struct SumsArgs {
  const float* sums;
  int64_t rows, width;
  int tiles_m, tiles_n, slices;
  int low;  // of rows kLow further on too
  const float* dyn;
  float unit;
  char* out;
  int64_t ld;
  const Rest* rest;  // of dx (REST): what is left times w's row of the label is added
  const char* w;
  int64_t ld_w;
};

template <class T, class Sh, int NG, bool REST>
__global__ __launch_bounds__(kThreads* NG) void sums_kernel(const SumsArgs p) {
  using G = Geo<Sh>;
  constexpr int kPitch = G::WN + 4, kSize = 32 * kPitch;
  __shared__ float lds[NG * kSize];
  const int group = int(threadIdx.x) / kThreads, tid = int(threadIdx.x) % kThreads;
  const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n, tile = blockIdx.x / (G::W * G::I);
  const int part = int(blockIdx.x % (G::W * G::I)), wave = part / G::I, a = part % G::I;
  const f32x4* from = reinterpret_cast<const f32x4*>(p.sums) + tile * (Sh::TM * Sh::TN / 4);
  const int64_t m0 = tile / p.tiles_n * Sh::TM + wave / Sh::WGN * G::WM + 32 * a;
  const int64_t n0 = tile % p.tiles_n * Sh::TN + wave % Sh::WGN * G::WN;
  // what a thread stores: 4 columns of a row each
  constexpr int kItems = 32 * G::WN / 4, kMine = (kItems + kThreads * NG - 1) / (kThreads * NG);
  struct __attribute__((packed, aligned(sizeof(Elem<T>)))) Half { uint2 v; };
  float left[kMine];
  uint32_t wrow[kMine][2];  // w's row of the label, 4 columns
  if constexpr (REST) {
    Rest rest[kMine];
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int i = int(threadIdx.x) + k * kThreads * NG;
      rest[k] = p.rest[min(m0 + i / (G::WN / 4), p.rows - 1)];
    }
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int64_t n = n0 + (int(threadIdx.x) + k * kThreads * NG) % (G::WN / 4) * 4;
      const bool labelled = rest[k].label >= 0;
      left[k] = labelled ? rest[k].left : 0.f;
      wrow[k][0] = wrow[k][1] = 0;
      if (labelled && n < p.width) {
        const char* w = p.w + (rest[k].label * p.ld_w + n) * T::esz;
        if (n + 4 <= p.width) {
          const uint2 v = reinterpret_cast<const Half*>(w)->v;
          wrow[k][0] = v.x, wrow[k][1] = v.y;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < p.width) wrow[k][e / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(w)[e]) << (16 * (e & 1));
        }
      }
    }
  }
  // the waves kLow rows further on, in the same tile (128 rows, 32 a wave)
  const int64_t low = kLow / G::WM * Sh::WGN * 64;
#pragma unroll
  for (int i = tid; i < G::J * 4 * 64; i += kThreads) {
    const int lane = i & 63, br = i >> 6;  // accumulator group: b, rg
    const f32x4* at = from + (a * G::J * 4 + br) * G::threads + wave * 64 + lane;
    f32x4 s = {{0.f, 0.f, 0.f, 0.f}};
    auto add = [&](const f32x4* at) __attribute__((always_inline)) {
#pragma unroll 8
      for (int q = group; q < p.slices; q += NG) {
        const f32x4 v = at[q * tiles * (Sh::TM * Sh::TN / 4)];
#pragma unroll
        for (int e = 0; e < 4; ++e) s.v[e] += v.v[e];
      }
    };
    if (p.low && wave / Sh::WGN * G::WM < kLow) add(at + low);
    add(at);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      lds[group * kSize + (lane & 31) * kPitch + 32 * (br >> 2) + 8 * (br & 3) + 4 * (lane >> 5) + e] = s.v[e];
  }
  __syncthreads();
  const float f = p.dyn ? p.dyn[1] : p.unit;
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int i = int(threadIdx.x) + k * kThreads * NG, row = i / (G::WN / 4), col = i % (G::WN / 4) * 4;
    const int64_t m = m0 + row, n = n0 + col;
    if (i >= kItems || m >= p.rows || n >= p.width) continue;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = lds[row * kPitch + col + e];
#pragma unroll
      for (int q = 1; q < NG; ++q) v[e] += lds[q * kSize + row * kPitch + col + e];
      if constexpr (REST) v[e] += left[k] * widened(T{}, wrow[k][e / 2] >> (16 * (e & 1)));
      v[e] *= f;
    }
    char* to = p.out + (m * p.ld + n) * T::esz;
    if (n + 4 <= p.width) {
      if constexpr (T::esz == 2) reinterpret_cast<Half*>(to)->v = uint2{pack2(T{}, v[0], v[1]), pack2(T{}, v[2], v[3])};
      else store_chunk<T>(to, __builtin_bit_cast(u32x4_t, f32x4{{v[0], v[1], v[2], v[3]}}), 4);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.width) store_from_f32(to, e, T::mk, v[e]);
    }
  }
}

// ---------------------------------------------------------------- few rows
// Up to 32 rows: one MFMA block of them, so that a call is the reading of w, and a tile of
// 128 rows would have most of the matrix rate for nothing (fp32) and, of few
// classes, few workgroups.  The waves of a workgroup share the k of their tile, each
// with a part of LDS that no barrier guards, and w is read where it lies, whatever its
// alignment; their accumulators are added through LDS.  Measured, tiles of 128
// rows and here: forward 1 x 3680 x 1313 bf16 31 us, 15; 6 x 3686 x 16342 fp32 313, 59;
// 8 x 769 x 50257 bf16 52, 30; 1 x 4096 x 65536 127, 117; 16 x 768 x 50257 20.2, 20.7;
// backward of the second 574, 242, of the last 61, 61.  The rule looks at the rows alone:
// where the classes fill the chip and rows lie on the 16-byte boundaries both are the
// reading of w, and within 3%.
constexpr int kThinRows = 32, kThinClasses = 64;

// the same of a row of `n` elements from element `at` on, zeros past its end
template <class T>
__device__ inline u32x4_t row_end16(const char* row, int64_t at, int64_t n) {
  constexpr int kE = 16 / T::esz;
  if (at + kE <= n) return loose16<T>(row + at * T::esz);
  struct alignas(16) { Elem<T> v[kE]; } c;
#pragma unroll
  for (int e = 0; e < kE; ++e) c.v[e] = at + e < n ? reinterpret_cast<const Elem<T>*>(row)[at + e] : Elem<T>(0);
  return __builtin_bit_cast(u32x4_t, c);
}

// The accumulators of two blocks of W waves, added: wave q gets quads q, q + W .. of 8,
// quad t the four columns 32 (t / 4) + 8 (t % 4) + 4 g .. + 3 of row lane % 32.
template <int W>
struct ThinSums { f32x4 v[W][8][64]; };
template <int W>
__device__ __attribute__((always_inline)) inline void join_waves(ThinSums<W>& red, const f32x16_t& a, const f32x16_t& b,
                                                                 int wave, int lane, f32x4 (&s)[8 / W]) {
#pragma unroll
  for (int rg = 0; rg < 4; ++rg) {
    red.v[wave][rg][lane] = f32x4{{a[4 * rg], a[4 * rg + 1], a[4 * rg + 2], a[4 * rg + 3]}};
    red.v[wave][4 + rg][lane] = f32x4{{b[4 * rg], b[4 * rg + 1], b[4 * rg + 2], b[4 * rg + 3]}};
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8 / W; ++i) {
    s[i] = red.v[0][wave + W * i][lane];
#pragma unroll
    for (int q = 1; q < W; ++q) {
      const f32x4 v = red.v[q][wave + W * i][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i].v[e] += v.v[e];
    }
  }
}

// The logits of 64 classes, and their end: LossArgs, each row's maximum and sum; GradArgs, g.
template <class T, int W, class Args>
__global__ __launch_bounds__(64 * W) void thin_logits_kernel(const Args p) {
  constexpr int kE = 16 / T::esz, kChunk = 8 * kE;  // 128 bytes of a row
  constexpr int kRows = kThinRows + kThinClasses;  // of a wave's part of LDS, a chunk each
  __shared__ __attribute__((aligned(16))) char lds[W * kRows * 128];
  static_assert(sizeof(ThinSums<W>) <= sizeof(lds), "the sums lie where the operands were");
  if constexpr (std::is_same_v<Args, GradArgs>) {
    if (int(blockIdx.x) >= p.tiles_n) {
      pack_block<Elem<T>, 64 * W>(p.pack, int(blockIdx.x) - p.tiles_n);
      return;
    }
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, g = lane >> 5;
  const int64_t v0 = int64_t(blockIdx.x) * kThinClasses;
  // 8 lanes a row load whole lines (lanes as the MFMA has them would load 32 bytes of
  // 32 lines: 94 us against 70 for 247 MB of w); the wave's own LDS turns them
  const int part = lane & 7, sub = lane >> 3;
  const char* from[kRows / 8];
#pragma unroll
  for (int i = 0; i < kRows / 8; ++i)
    from[i] = i < kThinRows / 8 ? p.x + min(int64_t(8 * i + sub), p.rows - 1) * p.ld_x * T::esz
                                : p.w + min(v0 + 8 * i - kThinRows + sub, p.vocab - 1) * p.ld_w * T::esz;
  u32x4_t next[kRows / 8];
  auto load = [&](int64_t k) __attribute__((always_inline)) {
    if (k + kChunk <= p.width) {
#pragma unroll
      for (int i = 0; i < kRows / 8; ++i) next[i] = loose16<T>(from[i] + (k + part * kE) * T::esz);
    } else {
#pragma unroll
      for (int i = 0; i < kRows / 8; ++i) next[i] = row_end16<T>(from[i], k + part * kE, p.width);
    }
  };
  f32x16_t acc[2];
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[0][r] = acc[1][r] = 0.f;
  char* st = lds + wave * (kRows * 128);
  int64_t k = int64_t(wave) * kChunk;
  if (k < p.width) load(k);
  while (k < p.width) {
#pragma unroll
    for (int i = 0; i < kRows / 8; ++i)
      *reinterpret_cast<u32x4_t*>(st + (8 * i + sub) * 128 + 16 * (part ^ sub)) = next[i];
    k += W * kChunk;
    if (k < p.width) load(k);
    asm volatile("" ::: "memory");  // what another lane of the wave wrote: LDS is in order
    auto read = [&](int row, int s) __attribute__((always_inline)) {
      return *reinterpret_cast<const u32x4_t*>(st + (row + c) * 128 + 16 * ((2 * s + g) ^ (c & 7)));
    };
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const u32x4_t a = read(0, s);
      acc[0] = T::mma(read(kThinRows, s), a, acc[0]);
      acc[1] = T::mma(read(kThinRows + 32, s), a, acc[1]);
    }
    asm volatile("" ::: "memory");
  }
  __syncthreads();
  ThinSums<W>& red = *reinterpret_cast<ThinSums<W>*>(lds);
  f32x4 sums[8 / W];
  join_waves<W>(red, acc[0], acc[1], wave, lane, sums);
  const int64_t label = c < p.rows ? p.labels.at(c) : -1;
  if constexpr (std::is_same_v<Args, LossArgs>) {
    __shared__ float2 ends[8][32];
#pragma unroll
    for (int i = 0; i < 8 / W; ++i) {
      const int t = wave + W * i;
      const int64_t col = v0 + 32 * (t / 4) + 8 * (t % 4) + 4 * g, left = p.vocab - col, at = label - p.v0 - col;
      f32x4& z = sums[i];
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e >= left) z.v[e] = -INFINITY;
        else if (c < p.rows && at == e) p.target[c] = z.v[e];
        top = fmaxf(top, z.v[e]);
      }
      float lo, hi;
      lane_halves_sched(top, lo, hi);
      top = fmaxf(lo, hi);
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += weight(z.v[e], or_zero(top));
      lane_halves_sched(sum, lo, hi);
      if (g == 0) ends[t][c] = float2{top, lo + hi};
    }
    __syncthreads();
    if (int(threadIdx.x) >= p.rows) return;
    float most = -INFINITY, all = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) most = fmaxf(most, ends[q][threadIdx.x].x);
#pragma unroll
    for (int q = 0; q < 8; ++q) all += ends[q][threadIdx.x].y * weight(ends[q][threadIdx.x].x, or_zero(most));
    p.part[int64_t(blockIdx.x) * p.rows + threadIdx.x] = float2{most, all};
  } else {
    // 16 bits: all of the 64 rows are written, what the rounding leaves 32 rows further on:
    // they are one k tile of dw
    const bool here = c < p.rows;
    if (!here && T::esz == 4) return;
    const float lse = here ? p.lse[c] : 0.f;
    const float factor = here ? (p.dyn ? p.dyn[0] : p.unit) * (p.row_grad ? p.row_grad[c] : 1.f) : 0.f;
    const bool none = !here || p.labels.ignored(label);
#pragma unroll
    for (int i = 0; i < 8 / W; ++i) {
      const int t = wave + W * i;
      const int64_t col = v0 + 32 * (t / 4) + 8 * (t % 4) + 4 * g, left = p.vocab - col, at = label - p.v0 - col;
      float v[4], rest[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z = sums[i].v[e];
        v[e] = weight(z, lse);
        if (at == e) v[e] -= 1.f;
        v[e] = none || e >= left ? 0.f : v[e] * factor;  // whole tiles are written, zeros past the classes
        rest[e] = v[e] - rounded(T{}, v[e]);
      }
      char* to = p.g + (c * p.ld_g + col) * T::esz;
      if constexpr (T::esz == 2) {
        *reinterpret_cast<uint2*>(to) = uint2{pack2(T{}, v[0], v[1]), pack2(T{}, v[2], v[3])};
        *reinterpret_cast<uint2*>(to + kThinRows * p.ld_g * 2) =
            uint2{pack2(T{}, rest[0], rest[1]), pack2(T{}, rest[2], rest[3])};
      } else {
        *reinterpret_cast<f32x4*>(to) = f32x4{{v[0], v[1], v[2], v[3]}};
      }
    }
  }
}

// dx: a workgroup has a run of classes and 32 chunks of 16 bytes of w's rows (256 columns
// of 16 bits, 128 of 32).  A lane takes a chunk from each of the kE classes its
// half of an MFMA step has, and a block of the MFMA is element j of all lanes' chunks:
// turning them by kE x kE is two bytes picked from two registers each (16 bits), or
// nothing (32 bits).
struct ThinDxArgs {
  const char *g, *w;
  int64_t rows, width, vocab;  // vocab: of this piece
  int64_t ld_g, ld_w;
  int slices;
  int64_t run;
  int first;
  float* sums;  // [slices][groups of columns][j][4][64 lanes][4]
};

template <class T>
__global__ __launch_bounds__(512, 2) void thin_dx_kernel(const ThinDxArgs p) {
  constexpr int kE = 16 / T::esz, kStep = 2 * kE, W = 8;
  __shared__ ThinSums<W> red;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, g = lane >> 5;
  const uint32_t slice = blockIdx.x % p.slices, group = blockIdx.x / p.slices;
  const int64_t col = (int64_t(group) * 32 + c) * kE, k0 = slice * p.run, k1 = min(k0 + p.run, p.vocab);
  const char* ga = p.g + min(int64_t(c), p.rows - 1) * p.ld_g * T::esz;
  f32x16_t acc[kE];
#pragma unroll
  for (int j = 0; j < kE; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[j][r] = 0.f;
  for (int64_t k = k0 + wave * kStep; k < k1; k += W * kStep) {
    const int64_t v = k + kE * g;
    u32x4_t raw[kE];
    const char* w = p.w + v * p.ld_w * T::esz;
    if (k + kStep <= p.vocab && col + kE <= p.width) {
#pragma unroll
      for (int e = 0; e < kE; ++e) raw[e] = loose16<T>(w + (e * p.ld_w + col) * T::esz);
    } else {
#pragma unroll
      for (int e = 0; e < kE; ++e)
        raw[e] = v + e < p.vocab ? row_end16<T>(w + e * p.ld_w * T::esz, col, p.width) : u32x4_t{0, 0, 0, 0};
    }
    const u32x4_t a = *reinterpret_cast<const u32x4_t*>(ga + v * T::esz);
    u32x4_t low = a;
    if constexpr (T::esz == 2) low = *reinterpret_cast<const u32x4_t*>(ga + (kThinRows * p.ld_g + v) * 2);
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      u32x4_t b;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if constexpr (T::esz == 2) b[h] = __builtin_amdgcn_perm(raw[2 * h + 1][j / 2], raw[2 * h][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
        else b[h] = raw[h][j];
      }
      acc[j] = T::mma(b, a, acc[j]);
      if constexpr (T::esz == 2) acc[j] = T::mma(b, low, acc[j]);
    }
  }
  f32x4* to = reinterpret_cast<f32x4*>(p.sums) + (int64_t(slice) * (gridDim.x / p.slices) + group) * kE * 256;
#pragma unroll
  for (int j = 0; j < kE; j += 2) {
    f32x4 sum[1];
    join_waves<W>(red, acc[j], acc[j + 1], wave, lane, sum);
    f32x4& s = sum[0];
    f32x4* at = to + (4 * j + wave) * 64 + lane;
    if (!p.first) {
      const f32x4 v = *at;
#pragma unroll
      for (int e = 0; e < 4; ++e) s.v[e] += v.v[e];
    }
    *at = s;
    __syncthreads();
  }
}

// The slices' sums, 16 runs of them in order, times the factor, to dx.
template <class T>
__global__ __launch_bounds__(1024) void thin_sums_kernel(const SumsArgs p) {
  constexpr int kE = 16 / T::esz;
  __shared__ f32x4 red[16][64];
  const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int64_t all = int64_t(p.tiles_n) * kE * 256;  // f32x4 of a slice
  const f32x4* at = reinterpret_cast<const f32x4*>(p.sums) + int64_t(blockIdx.x) * 64 + lane;
  f32x4 s = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
  for (int i = q; i < p.slices; i += 16) {
    const f32x4 v = at[i * all];
#pragma unroll
    for (int e = 0; e < 4; ++e) s.v[e] += v.v[e];
  }
  red[q][lane] = s;
  __syncthreads();
  const int row = lane & 31, g = lane >> 5, rg = blockIdx.x % 4, j = blockIdx.x / 4 % kE;
  if (q > 0 || row >= p.rows) return;
#pragma unroll
  for (int i = 1; i < 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) s.v[e] += red[i][lane].v[e];
  const float f = p.dyn ? p.dyn[1] : p.unit;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t col = (int64_t(blockIdx.x / (4 * kE)) * 32 + 8 * rg + 4 * g + e) * kE + j;
    if (col < p.width) store_from_f32(p.out + row * p.ld * T::esz, col, T::mk, s.v[e] * f);
  }
}

template <typename U>
__global__ __launch_bounds__(kThreads) void pack_kernel(const PackArgs p) { pack_block<U, kThreads>(p, blockIdx.x); }

// rows x cols of zeros (words of U): the gradient of no rows
template <typename U>
__global__ __launch_bounds__(kThreads) void zero_kernel(U* p, int64_t ld, int64_t rows, int64_t cols) {
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < rows * cols; i += int64_t(gridDim.x) * kThreads)
    p[i / cols * ld + i % cols] = U(0);
}

// dyn = {factor of g, factor of the products} for fp16: |g| <= max |row_grad| of the rows
// that count (an ignored row's may be anything), and
// 2^15 times that over its power of two is below fp16's largest value, while the
// smallest normal value is 2^-29 of it.
constexpr int kFactorThreads = 1024;
__global__ __launch_bounds__(kFactorThreads) void factor_kernel(const float* row_grad, int64_t rows, Labels labels, float scale, float* dyn) {
  __shared__ float red[kFactorThreads / kWave];
  float top = 0.f;
#pragma unroll 4
  for (int64_t n = threadIdx.x; n < rows; n += kFactorThreads) {
    const float v = fabsf(row_grad[n]);
    if (v < INFINITY && !(labels.has_ignore && labels.ignored(labels.at(n)))) top = fmaxf(top, v);
  }
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x) return;
#pragma unroll
  for (int i = 1; i < kFactorThreads / kWave; ++i) top = fmaxf(top, red[i]);
  int e = 0;
  if (top > 0.f) (void)frexpf(top, &e);  // top <= 2^e
  e = max(-112, e);  // 2^127 at most
  dyn[0] = ldexpf(1.f, 15 - e);
  dyn[1] = ldexpf(scale, e - 15);
}

// ---------------------------------------------------------------- host
constexpr int64_t kGBytes = int64_t(512) << 20;     // of g a piece
constexpr int64_t kPackBytes = int64_t(256) << 20;  // of w copied a piece

// compute units of the current device (cached per device)
int64_t cu_count() {
  static std::atomic<int> cache[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cache[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

bool on_grid(const void* p, int64_t ld, int64_t width, int esz) {
  // 256 rows of a tile lie within a buffer's 32-bit offsets
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld * esz % 16 == 0 && width * esz % 16 == 0 && ld >= width &&
         ld * esz < (int64_t(1) << 23);
}

// One call's sizes and its workspace, from the shapes and the operands' alignment alone.
enum { kBig, kMid };
struct Plan {
  int esz;
  int64_t rows, width, vocab;
  int logits, products;           // shapes of the kernels that form the logits, and of dx's and dw's
  int64_t tm, tn, pm, pn;         // their tiles
  bool pack_x, pack_w;
  int64_t pitch;                  // of packed rows, elements
  int64_t piece, pieces;          // classes of a piece
  int64_t ld_g;
  int64_t slices, dw_slices;      // runs of dx's classes and of dw's rows
  bool dx_first;                  // dx's runs before dw's tiles
  bool thin, twice;               // the kernels of few rows; their g and x have 64 rows
  bool low;                       // g has its second rows
  bool rest;                      // what g's rounding leaves of the labels' elements is kept
  int64_t x_at, w_at, part_at, target_at, g_at, rest_at, sums_at, dw_sums_at, dyn_at, bytes;
};

// k tiles that the last of the chip's workgroups ends with, of n workgroups of kn k
// tiles and then m of km, an XCD's share on its `slots` of them: each takes the
// next one when it is free.
int64_t ends(int64_t n, int64_t kn, int64_t m, int64_t km, int64_t slots) {
  const int64_t rounds = n / slots, more = n % slots, most = (m + slots - 1) / slots;
  int64_t lo = (rounds + (more > 0)) * kn, hi = lo + most * km;
  auto fits = [&](int64_t t) {
    const int64_t late = std::max<int64_t>(0, t - (rounds + 1) * kn) / km, early = std::max<int64_t>(0, t - rounds * kn) / km;
    return more * late + (slots - more) * early >= m;
  };
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (fits(mid)) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Tile shapes: a k tile of 256 x 256 takes 1.75 us on a CU, one of 128 x 128 with
// another beside it on the CU 1.12 us, alone 0.78 of that; of 32 bits what the fp32
// MFMA takes.  A tile's begin and end count as more k tiles.
constexpr int64_t kSizes[2][2] = {{256, 256}, {128, 128}};
double step_time(int shape, int esz) { return esz == 4 ? 3.5 : shape == kBig ? 1.75 : 1.12; }

// Estimated us of the logits' tiles, kt k tiles each.  Measured, 256 and 128: loss of
// 300 x 768 x 50257 51, 39, of 1000 94, 88 (here it is 6% off); gradient of 300 (with the
// same products) 136, 125, of 1000 263, 266, of 2048 x 1024 x 32000 383, 417, of 187 x
// 2409 x 4098 96, 71.
double logits_time(int shape, int esz, int64_t rows, int64_t classes, int64_t kt) {
  const int64_t tm = kSizes[shape][0], tn = kSizes[shape][1];
  const int64_t tiles = (rows + tm - 1) / tm * ((classes + tn - 1) / tn);
  const int64_t cus = cu_count(), slots = shape == kBig ? cus : 2 * cus, rest = tiles % slots;
  const double last = rest == 0 ? 0.0 : shape == kMid && rest <= cus ? 0.78 : 1.0;
  return (double(tiles / slots) + last) * step_time(shape, esz) * (double(kt) + 1.5);
}

struct Cuts {
  double time;
  int shape;
  int64_t dx, dw;  // runs
  bool dx_first;
};

// The shape of dx's and dw's tiles of a piece, their order, and the runs that dx's
// classes and (where dw's tiles are few) dw's rows are cut into, by estimated us: fewer k
// tiles one after the other against a tile of sums a run, written and read again at
// about 3.8 TB/s.  A k tile of the last workgroup costs less than it takes alone
// (step_time), since those that have ended leave it the power and the bandwidth;
// the tiles' ends count as more k tiles.  Measured, up to 28 ways each of twelve sizes (100
// to 8192 rows, 64 to 4096 wide, 2148 to 50257 classes): it takes the fastest or one
// within 3% at ten, 4% slower at 4527 x 1328 x 7316 bf16, 8% at 560 x 284 x 28975 fp32.
Cuts products_cuts(int shape, int esz, int64_t rows, int64_t width, int64_t classes) {
  const int64_t end_w = shape == kBig ? 7 : 5, end_x = shape == kBig ? 7 : 6;
  const double last = shape == kBig ? 1.06 : 0.51, all = shape == kBig ? 0.0 : 0.24, slower = esz == 4 ? 2.4 : 1.0;
  const int64_t tm = kSizes[shape][0], tn = kSizes[shape][1], across = (width + tn - 1) / tn, deep = 128 / esz;
  const int64_t dx = (rows + tm - 1) / tm * across, dw = (classes + tm - 1) / tm * across;
  const int64_t kx = (classes + deep - 1) / deep, kw = (rows + deep - 1) / deep;
  const int64_t slots = std::max<int64_t>(1, cu_count() / 8 * (shape == kBig ? 1 : 2));
  Cuts best{};
  for (int64_t w = 1; w == 1 || (w <= 16 && dw * w <= 16 * slots && kw >= 4 * w); w *= 2)
    for (int64_t n = 1; n <= 64 && n <= kx; n *= 2) {
      const double sums = double((dx * n + (w > 1 ? dw * w : 0)) * tm * tn * 4);
      const int64_t w1 = (dw * w + 7) / 8, wt = (kw + w - 1) / w + end_w;
      const int64_t x1 = (dx * n + 7) / 8, xt = (kx + n - 1) / n + end_x;
      const double t = slower * all * double(w1 * wt + x1 * xt) / double(slots) + sums * 2 / 7.6e6 + (w > 8 ? 12.0 : w > 1 ? 4.0 : 0.0);
      const double dw_first = t + slower * last * double(ends(w1, wt, x1, xt, slots));
      const double dx_first = t + slower * last * double(ends(x1, xt, w1, wt, slots)) * (shape == kBig ? 1.03 : 1.01);
      if (best.dx == 0 || std::min(dw_first, dx_first) < best.time)
        best = {std::min(dw_first, dx_first), shape, n, w, dx_first < dw_first};
    }
  return best;
}

Plan plan(bool bwd, int io_type, int64_t rows, int64_t width, int64_t vocab, const void* x, int64_t ld_x, const void* w,
          int64_t ld_w, bool has_ignore) {
  Plan q{};
  q.esz = dtype_bytes(io_type);
  q.rows = rows, q.width = width, q.vocab = vocab;
  const int64_t deep = 128 / q.esz;
  const int64_t kt = (width + deep - 1) / deep;
  q.thin = rows <= kThinRows;
  q.low = bwd && q.esz == 2 && rows <= kLow && !q.thin;
  q.rest = bwd && q.esz == 2 && rows > kLow;
  const double mid = logits_time(kMid, q.esz, rows, vocab, kt), big = logits_time(kBig, q.esz, rows, vocab, kt);
  q.logits = q.esz == 4 || q.low || mid < big ? kMid : kBig;
  q.tm = q.thin ? kThinRows : kSizes[q.logits][0], q.tn = q.thin ? kThinClasses : kSizes[q.logits][1];
  // few rows are read as they lie, but by dw's tiles (16 bits: twice, beside both rows of g)
  q.twice = q.thin && bwd && q.esz == 2;
  q.pack_x = q.thin && !bwd ? false : q.twice || !on_grid(x, ld_x, width, q.esz) || (bwd && has_ignore);
  q.pack_w = !q.thin && !on_grid(w, ld_w, width, q.esz);
  q.pitch = up(width, 16 / q.esz);
  int64_t most = vocab;
  if (q.pack_w) most = std::min(most, std::max<int64_t>(q.tn, kPackBytes / (q.pitch * q.esz)));
  if (bwd) most = std::min(most, std::max<int64_t>(q.tn, std::min<int64_t>(kGBytes / (rows * q.esz), int64_t(1) << 20)));
  q.pieces = (vocab + most - 1) / most;
  q.piece = up((vocab + q.pieces - 1) / q.pieces, 256);
  if (q.pieces > 1) {  // whole rounds of tiles in all but the last piece, where they fit
    const int64_t tiles_m = (rows + q.tm - 1) / q.tm, round = cu_count() / std::gcd(tiles_m, cu_count()) * q.tn;
    if (up(q.piece, round) <= most) q.piece = up(q.piece, round);
  }
  q.pieces = (vocab + q.piece - 1) / q.piece;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t here = at; at += align256(bytes); return here; };
  const int64_t kept = q.twice ? 2 * kThinRows : rows;
  if (q.pack_x) q.x_at = take(kept * q.pitch * q.esz);
  if (q.pack_w) q.w_at = take(std::min(vocab, q.piece) * q.pitch * q.esz);
  if (!bwd) {
    q.part_at = take(((vocab + q.tn - 1) / q.tn + q.pieces) * rows * 8);
    q.target_at = take(rows * 4);
  } else {
    const int64_t classes = std::min(vocab, q.piece);
    q.ld_g = up(classes, 64);
    q.g_at = take((kept + (q.low ? kLow : 0)) * q.ld_g * q.esz);
    if (q.rest) q.rest_at = take(rows * sizeof(Rest));
    const Cuts small = products_cuts(kMid, q.esz, rows, width, classes);
    const Cuts large = products_cuts(kBig, q.esz, rows, width, classes);
    const Cuts& cuts = q.esz == 4 || rows <= kLow || small.time < large.time ? small : large;  // low: 128 rows a tile
    q.products = cuts.shape, q.slices = cuts.dx, q.dw_slices = cuts.dw, q.dx_first = cuts.dx_first;
    q.pm = kSizes[q.products][0], q.pn = kSizes[q.products][1];
    int64_t tiles = (rows + q.pm - 1) / q.pm * ((width + q.pn - 1) / q.pn) * q.pm * q.pn;
    if (q.thin) {  // a workgroup a CU, or 8 MFMA steps of its waves
      const int64_t columns = 512 / q.esz, groups = (width + columns - 1) / columns, step = 8 * 32 / q.esz;
      q.slices = std::max<int64_t>(1, std::min(cu_count() / groups, (classes + step - 1) / step));
      tiles = groups * kThinRows * columns;
    }
    q.sums_at = take(q.slices * tiles * 4);
    if (q.dw_slices > 1)
      q.dw_sums_at = take(q.dw_slices * ((classes + q.pm - 1) / q.pm) * ((width + q.pn - 1) / q.pn) * q.pm * q.pn * 4);
    q.dyn_at = take(8);
  }
  q.bytes = at;
  return q;
}

int check_shapes(const std::string& what, int io_type, int64_t rows, int64_t width, int64_t vocab, int64_t ld_x,
                 int64_t ld_w, int label_type) {
  if (io_type != MK_BF16 && io_type != MK_F16 && io_type != MK_F32)
    return fail(MK_ERR_UNSUPPORTED, what + ": io_type must be bf16, f16 or f32");
  if (label_type != MK_S32 && label_type != MK_S64) return fail(MK_ERR_UNSUPPORTED, what + ": label_type must be s32 or s64");
  if (rows < 0 || width <= 0 || vocab <= 0) return fail(MK_ERR_INVALID, what + ": bad shape");
  if (ld_x < 0 || ld_w < 0) return fail(MK_ERR_INVALID, what + ": negative pitch");
  if (rows >= int64_t(1) << 31 || vocab >= int64_t(1) << 31 || width > int64_t(1) << 20)
    return fail(MK_ERR_UNSUPPORTED, what + ": rows and vocab must be below 2^31, width at most 2^20");
  return MK_OK;
}

int check_pointer(const std::string& what, const char* name, const void* p, int bytes, bool needed) {
  if (!p) return needed ? fail(MK_ERR_INVALID, what + ": null " + name) : MK_OK;
  if (reinterpret_cast<uintptr_t>(p) % bytes) return fail(MK_ERR_INVALID, what + ": not aligned: " + name);
  return MK_OK;
}

int check_tiles(const std::string& what, int64_t tiles, int threads) {
  if (tiles * threads >= int64_t(1) << 32) return fail(MK_ERR_UNSUPPORTED, what + ": too many tiles");
  return MK_OK;
}

int pack(const char* what, hipStream_t s, const Plan& q, const PackArgs& p) {
  const int64_t blocks = (p.rows * (p.ld_dst * q.esz / 16) + kThreads - 1) / kThreads;
  if (int rc = check_tiles(what, blocks, kThreads)) return rc;
  const dim3 g{unsigned(blocks)}, b{kThreads};
  if (q.esz == 2) hipLaunchKernelGGL(pack_kernel<uint16_t>, g, b, 0, s, p);
  else hipLaunchKernelGGL(pack_kernel<uint32_t>, g, b, 0, s, p);
  return check_launch(what);
}

// Workgroups of a kernel whose workgroups go on from tile to tile: those that the
// chip holds at once (multiples of 8, so that a workgroup's tiles are one XCD's).
template <class Sh>
unsigned resident(int64_t tiles) {
  const int64_t most = cu_count() * (Geo<Sh>::lds_bytes <= 80 * 1024 ? 2 : 1) / 8 * 8;
  return unsigned(std::min(tiles, std::max<int64_t>(8, most)));
}

// f(type, shape) of a kernel; fp32 has the small shape alone (measured: 512 x 768 x 50257 983 us,
// with 256 x 256 1076; 560 x 284 x 28975 347, 554)
template <class T, class F>
int with_shape(T t, int shape, F&& f) {
  return shape == kBig ? f(t, Big{}) : f(t, Mid{});
}
template <class F>
int with_kernels(int io_type, int shape, F&& f) {
  if (io_type == MK_BF16) return with_shape(Bf16{}, shape, f);
  if (io_type == MK_F16) return with_shape(F16{}, shape, f);
  return f(F32{}, Mid{});
}
// the same of results of type `to`, an fp32 gradient of 16-bit operands too
template <class F>
int with_results(int to, int shape, F&& f) {
  if (to == MK_F32) return with_shape(F32{}, shape, f);
  return with_kernels(to, shape, f);
}

// 4 waves a tile where the tiles fill the chip, else 8
template <class T, class Args>
int thin_logits(const char* what, hipStream_t s, const Args& a) {
  const int waves = a.tiles_n > 2 * cu_count() ? 4 : 8;
  int64_t more = 0;
  if constexpr (std::is_same_v<Args, GradArgs>)
    if (a.v0 == 0) more = (a.pack.rows * (a.pack.ld_dst * T::esz / 16) + 64 * waves - 1) / (64 * waves);
  const dim3 g{unsigned(a.tiles_n + more)}, b{unsigned(64 * waves)};
  if (waves == 4) hipLaunchKernelGGL((thin_logits_kernel<T, 4, Args>), g, b, 0, s, a);
  else hipLaunchKernelGGL((thin_logits_kernel<T, 8, Args>), g, b, 0, s, a);
  return check_launch(what);
}

}  // namespace
}  // namespace mk

using namespace mk;

extern "C" size_t mk_linear_xent_workspace_bytes(int io_type, int64_t rows, int64_t width, int64_t vocab, const void* x,
                                                 int64_t ld_x, const void* w, int64_t ld_w) {
  if (check_shapes("", io_type, rows, width, vocab, ld_x, ld_w, MK_S32) || rows == 0) return 0;
  return size_t(plan(false, io_type, rows, width, vocab, x, ld_x, w, ld_w, false).bytes);
}

extern "C" int mk_linear_xent(void* stream, int io_type, int64_t rows, int64_t width, int64_t vocab, const void* x,
                              int64_t ld_x, const void* w, int64_t ld_w, int label_type, const void* labels,
                              int has_ignore, int64_t ignore_index, float* loss_rows, float* lse, void* workspace) {
  clear_error();
  const char* what = "mk_linear_xent";
  if (int rc = check_shapes(what, io_type, rows, width, vocab, ld_x, ld_w, label_type)) return rc;
  if (rows == 0) return MK_OK;
  const int esz = dtype_bytes(io_type);
  const struct { const char* name; const void* p; int bytes; bool needed; } ptrs[] = {
      {"x", x, esz, true}, {"w", w, esz, true}, {"labels", labels, dtype_bytes(label_type), true},
      {"loss_rows", loss_rows, 4, false}, {"lse", lse, 4, false}, {"workspace", workspace, 16, true}};
  for (const auto& e : ptrs)
    if (int rc = check_pointer(what, e.name, e.p, e.bytes, e.needed)) return rc;
  const Plan q = plan(false, io_type, rows, width, vocab, x, ld_x, w, ld_w, false);
  hipStream_t s = as_stream(stream);
  char* ws = static_cast<char*>(workspace);
  LossArgs a{};
  a.labels = {labels, label_type == MK_S64, has_ignore != 0, ignore_index};
  a.x = static_cast<const char*>(x), a.ld_x = ld_x;
  a.rows = rows, a.width = width;
  a.part = reinterpret_cast<float2*>(ws + q.part_at);
  a.target = reinterpret_cast<float*>(ws + q.target_at);
  a.tiles_m = int((rows + q.tm - 1) / q.tm);
  if (int rc = check_tiles(what, std::max(a.tiles_m * ((q.piece + q.tn - 1) / q.tn), (rows + 15) / 16), 512)) return rc;
  if (q.pack_x) {
    if (int rc = pack(what, s, q, {x, ld_x, rows, width, ws + q.x_at, q.pitch, Labels{}, rows, 0})) return rc;
    a.x = ws + q.x_at, a.ld_x = q.pitch;
  }
  const float2* part = a.part;
  int64_t tiles = 0;
  for (int64_t v0 = 0; v0 < vocab; v0 += q.piece) {
    a.v0 = v0;
    a.vocab = std::min(q.piece, vocab - v0);
    a.w = static_cast<const char*>(w) + v0 * ld_w * esz, a.ld_w = ld_w;
    if (q.pack_w) {
      if (int rc = pack(what, s, q, {a.w, ld_w, a.vocab, width, ws + q.w_at, q.pitch, Labels{}, a.vocab, 0})) return rc;
      a.w = ws + q.w_at, a.ld_w = q.pitch;
    }
    a.tiles_n = int((a.vocab + q.tn - 1) / q.tn);
    const int rc = with_kernels(io_type, q.logits, [&](auto t, auto sh) {
      using T = decltype(t);
      using Sh = decltype(sh);
      if (q.thin) {
        return thin_logits<T>(what, s, a);
      }
      hipLaunchKernelGGL((loss_kernel<T, Sh>), dim3(resident<Sh>(int64_t(a.tiles_m) * a.tiles_n)), dim3(Geo<Sh>::threads),
                         0, s, a);
      return check_launch(what);
    });
    if (rc) return rc;
    a.part += a.tiles_n * rows;
    tiles += a.tiles_n;
  }
  const dim3 joins{unsigned((rows + 15) / 16)};
  if (rows <= 1024)
    hipLaunchKernelGGL(loss_final_kernel<64>, joins, dim3(1024), 0, s, part, a.target, rows, vocab, tiles, a.labels,
                       loss_rows, lse);
  else
    hipLaunchKernelGGL(loss_final_kernel<16>, joins, dim3(256), 0, s, part, a.target, rows, vocab, tiles, a.labels,
                       loss_rows, lse);
  return check_launch(what);
}

extern "C" size_t mk_linear_xent_bwd_workspace_bytes(int io_type, int64_t rows, int64_t width, int64_t vocab,
                                                     const void* x, int64_t ld_x, const void* w, int64_t ld_w,
                                                     int has_ignore) {
  if (check_shapes("", io_type, rows, width, vocab, ld_x, ld_w, MK_S32) || rows == 0) return 0;
  return size_t(plan(true, io_type, rows, width, vocab, x, ld_x, w, ld_w, has_ignore != 0).bytes);
}

extern "C" int mk_linear_xent_bwd(void* stream, int io_type, int dw_type, int64_t rows, int64_t width, int64_t vocab,
                                  const void* x, int64_t ld_x, const void* w, int64_t ld_w, int label_type,
                                  const void* labels, int has_ignore, int64_t ignore_index, const float* lse,
                                  const float* row_grad, float grad_scale, void* dx, int64_t ld_dx, void* dw,
                                  int64_t ld_dw, void* workspace) {
  clear_error();
  const char* what = "mk_linear_xent_bwd";
  if (int rc = check_shapes(what, io_type, rows, width, vocab, ld_x, ld_w, label_type)) return rc;
  if (dw && dw_type != io_type && dw_type != MK_F32)
    return fail(MK_ERR_UNSUPPORTED, std::string(what) + ": dw_type must be io_type or f32");
  const int esz = dtype_bytes(io_type), dwsz = dw ? dtype_bytes(dw_type) : 1;
  if ((dx && rows > 1 && ld_dx < width) || (dw && vocab > 1 && ld_dw < width))
    return fail(MK_ERR_INVALID, std::string(what) + ": rows of dx or dw overlap");
  if (int rc = check_pointer(what, "dw", dw, dwsz, false)) return rc;
  hipStream_t s = as_stream(stream);
  if (!dx && !dw) return MK_OK;
  const struct { const char* name; const void* p; int bytes; bool needed; } ptrs[] = {
      {"x", x, esz, true}, {"w", w, esz, true}, {"labels", labels, dtype_bytes(label_type), true}, {"lse", lse, 4, true},
      {"row_grad", row_grad, 4, false}, {"dx", dx, esz, false}, {"workspace", workspace, 16, true}};
  if (rows == 0) {
    if (!dw) return MK_OK;
    const int64_t blocks = std::min<int64_t>((vocab * width + kThreads - 1) / kThreads, 1 << 16);
    if (dwsz == 2)
      hipLaunchKernelGGL(zero_kernel<uint16_t>, dim3(unsigned(blocks)), dim3(kThreads), 0, s, static_cast<uint16_t*>(dw),
                         ld_dw, vocab, width);
    else
      hipLaunchKernelGGL(zero_kernel<uint32_t>, dim3(unsigned(blocks)), dim3(kThreads), 0, s, static_cast<uint32_t*>(dw),
                         ld_dw, vocab, width);
    return check_launch(what);
  }
  for (const auto& e : ptrs)
    if (int rc = check_pointer(what, e.name, e.p, e.bytes, e.needed)) return rc;
  if (dx == x || dx == w || dw == w || dw == x || dx == dw)
    return fail(MK_ERR_INVALID, std::string(what) + ": dx or dw over x, over w or one over the other");
  const Plan q = plan(true, io_type, rows, width, vocab, x, ld_x, w, ld_w, has_ignore != 0);
  char* ws = static_cast<char*>(workspace);
  const Labels lab = {labels, label_type == MK_S64, has_ignore != 0, ignore_index};
  GradArgs a{};
  ProductsArgs b{};
  a.rows = rows, b.rows = q.twice ? 2 * kThinRows : rows, a.width = b.width = width;
  a.labels = lab;
  a.lse = lse, a.row_grad = row_grad;
  a.x = static_cast<const char*>(x), a.ld_x = ld_x;
  a.g = ws + q.g_at, a.ld_g = q.ld_g;
  a.all = vocab;
  if (q.rest) b.rest = a.rest = reinterpret_cast<Rest*>(ws + q.rest_at);
  a.tiles_m = int((rows + q.tm - 1) / q.tm);
  b.dx_m = dx && !q.thin ? int((rows + q.pm - 1) / q.pm) : 0;
  b.dx_n = b.dw_n = int((width + q.pn - 1) / q.pn);
  const int64_t thin_groups = (width + 512 / esz - 1) / (512 / esz);
  b.slices = int(q.slices), b.dw_slices = int(q.dw_slices);
  b.dw_run = up((b.rows + q.dw_slices - 1) / q.dw_slices, 128 / esz);
  a.low = b.low = q.low, b.dx_first = q.dx_first;
  const int64_t most = a.tiles_m * ((q.piece + q.tn - 1) / q.tn),
                most2 = int64_t(b.dx_m) * b.dx_n * q.slices + (q.piece + q.pm - 1) / q.pm * b.dw_n * q.dw_slices + 16;
  // the sums' blocks have 32 rows and a wave's columns, and at most 1024 threads
  const int64_t most3 = int64_t(b.dx_m) * b.dx_n * (q.products == kBig ? 32 : 8) * 2;
  if (int rc = check_tiles(what, std::max({most, most2, most3}), 512)) return rc;
  // fp16: g out of the subnormals, by a power of two of the largest row_grad
  a.unit = io_type == MK_F16 ? 32768.f : 1.f;
  b.unit = io_type == MK_F16 ? grad_scale / 32768.f : grad_scale;
  if (io_type == MK_F16 && row_grad) {
    float* dyn = reinterpret_cast<float*>(ws + q.dyn_at);
    hipLaunchKernelGGL(factor_kernel, dim3(1), dim3(kFactorThreads), 0, s, row_grad, rows, lab, grad_scale, dyn);
    if (int rc = check_launch(what)) return rc;
    a.dyn = b.dyn = dyn;
  }
  b.g = a.g, b.ld_g = a.ld_g;
  b.x = a.x, b.ld_x = a.ld_x;
  if (q.pack_x) {
    const PackArgs c{x, ld_x, b.rows, width, ws + q.x_at, q.pitch, lab, rows, q.twice ? kThinRows : 0};
    b.x = ws + q.x_at, b.ld_x = q.pitch;
    if (q.thin) {
      a.pack = c;
    } else {
      if (int rc = pack(what, s, q, c)) return rc;
      a.x = b.x, a.ld_x = b.ld_x;
    }
  }
  b.sums = reinterpret_cast<float*>(ws + q.sums_at), b.dw_sums = reinterpret_cast<float*>(ws + q.dw_sums_at);
  b.dw_f32 = dw_type == MK_F32;
  b.ld_dw = ld_dw;
  // the sums of slices, dx's or a piece's dw's, into rows of type `to`
  auto join = [&](int to, const SumsArgs& c) {
    return with_results(to, q.products, [&](auto t, auto sh) {
      using T = decltype(t);
      using Sh = decltype(sh);
      const dim3 g{unsigned(c.tiles_m) * unsigned(c.tiles_n) * Geo<Sh>::W * Geo<Sh>::I};
      if constexpr (T::esz == 2) {
        if (c.rest) {
          if (c.slices > 8) hipLaunchKernelGGL((sums_kernel<T, Sh, 4, true>), g, dim3(4 * kThreads), 0, s, c);
          else hipLaunchKernelGGL((sums_kernel<T, Sh, 1, true>), g, dim3(kThreads), 0, s, c);
          return check_launch(what);
        }
      }
      if (c.slices > 8) hipLaunchKernelGGL((sums_kernel<T, Sh, 4, false>), g, dim3(4 * kThreads), 0, s, c);
      else hipLaunchKernelGGL((sums_kernel<T, Sh, 1, false>), g, dim3(kThreads), 0, s, c);
      return check_launch(what);
    });
  };
  for (int64_t v0 = 0; v0 < vocab; v0 += q.piece) {
    a.v0 = b.v0 = v0;
    a.vocab = b.vocab = std::min(q.piece, vocab - v0);
    a.w = static_cast<const char*>(w) + v0 * ld_w * esz, a.ld_w = ld_w;
    if (q.pack_w) {
      if (int rc = pack(what, s, q, {a.w, ld_w, a.vocab, width, ws + q.w_at, q.pitch, Labels{}, a.vocab, 0})) return rc;
      a.w = ws + q.w_at, a.ld_w = q.pitch;
    }
    b.w = a.w, b.ld_w = a.ld_w;
    b.first = v0 == 0;
    const int64_t deep = 128 / esz;
    b.run = up((a.vocab + q.slices - 1) / q.slices, deep);
    b.dw = static_cast<char*>(dw) + v0 * ld_dw * dwsz;
    a.tiles_n = int((a.vocab + q.tn - 1) / q.tn);
    b.dw_m = dw ? int((a.vocab + q.pm - 1) / q.pm) : 0;
    int rc = with_kernels(io_type, q.logits, [&](auto t, auto sh) {
      using T = decltype(t);
      using Sh = decltype(sh);
      if (q.thin) {
        return thin_logits<T>(what, s, a);
      }
      const int64_t tiles = int64_t(a.tiles_m) * a.tiles_n;
      hipLaunchKernelGGL((grad_kernel<T, Sh>), dim3(q.logits == kBig ? resident<Sh>(tiles) : unsigned(tiles)),
                         dim3(Geo<Sh>::threads), 0, s, a);
      return check_launch(what);
    });
    if (rc) return rc;
    if (dx && q.thin) {
      const ThinDxArgs c{b.g, b.w, rows, width, b.vocab, b.ld_g, b.ld_w, b.slices, up((a.vocab + q.slices - 1) / q.slices, 8 * 32 / esz),
                         b.first, b.sums};
      rc = with_kernels(io_type, q.products, [&](auto t, auto) {
        using T = decltype(t);
        hipLaunchKernelGGL(thin_dx_kernel<T>, dim3(unsigned(thin_groups * q.slices)), dim3(512), 0, s, c);
        return check_launch(what);
      });
      if (rc) return rc;
    }
    if (q.thin && !dw) continue;
    rc = with_kernels(io_type, q.products, [&](auto t, auto sh) {
      using T = decltype(t);
      using Sh = decltype(sh);
      const unsigned tiles = (unsigned(b.dx_m) * b.dx_n * b.slices + 7) / 8 * 8 + (unsigned(b.dw_m) * b.dw_n * b.dw_slices + 7) / 8 * 8;
      const dim3 n{tiles}, threads{Geo<Sh>::threads};
      if constexpr (T::esz == 4) {
        hipLaunchKernelGGL((products_kernel<T, Sh, false>), n, threads, 0, s, b);
      } else if constexpr (Sh::TM == 256) {  // never of up to kLow rows
        hipLaunchKernelGGL((products_kernel<T, Sh, true>), n, threads, 0, s, b);
      } else {
        if (q.rest) hipLaunchKernelGGL((products_kernel<T, Sh, true>), n, threads, 0, s, b);
        else hipLaunchKernelGGL((products_kernel<T, Sh, false>), n, threads, 0, s, b);
      }
      return check_launch(what);
    });
    if (rc) return rc;
    if (dw && b.dw_slices > 1) {
      const SumsArgs c{b.dw_sums, b.vocab, width, b.dw_m, b.dw_n, b.dw_slices, 0, b.dyn, b.unit, b.dw, ld_dw};
      if (int r = join(dw_type, c)) return r;
    }
  }
  if (!dx) return MK_OK;
  if (q.thin) {
    const SumsArgs c{b.sums, rows, width, 1, int(thin_groups), b.slices, 0, b.dyn, b.unit, static_cast<char*>(dx), ld_dx};
    return with_kernels(io_type, q.products, [&](auto t, auto) {
      using T = decltype(t);
      hipLaunchKernelGGL(thin_sums_kernel<T>, dim3(unsigned(thin_groups) * (64 / T::esz)), dim3(1024), 0, s, c);
      return check_launch(what);
    });
  }
  return join(io_type, SumsArgs{b.sums, rows, width, b.dx_m, b.dx_n, b.slices, b.low, b.dyn, b.unit,
                                static_cast<char*>(dx), ld_dx, b.rest, static_cast<const char*>(w), ld_w});
}
