// Dropout with its mask regenerated instead of stored: the branch's way into
// the residual stream (mk_dropout_add) and its gradient with the bias's
// (mk_dropout_add_bwd).
//
//   out = residual + keep (x + bias) 65536 / (65536 - T);   dx = keep dy 65536 / (65536 - T)
//
// keep(r, c) comes from a counter: Philox-4x32 of 10 rounds on (c / 8, r, o),
// whose 128 bits are the 16-bit fields of 8 neighbouring columns.  A round is
// two products of 32 by 32 bits, which run at a quarter of the vector rate:
// 8 columns cost 20 of them, so that a field of 16 bits an element keeps the
// generator (15 operations an element, the rest about 8) below the memory's
// time, where 32 bits an element would not (bf16: 4 bytes moved an element).
// p is then a multiple of 2^-16, and the scale is that of the rounded p.
// The rows start at field 0, so the mask does not depend on their pitch.
//
// A thread has a group of 8 columns and walks down the rows, with the bias of its
// columns (forward) or their sums (backward) in registers; a block is CT groups
// wide (a power of two that wastes little of the last tile) and 256 / CT rows
// high.  Sums of columns go through LDS, then as one partial row a block to the
// workspace, and a second launch adds the partial rows in order.
#include "mk_common.h"

#include <algorithm>
#include <cmath>
#include <string>

namespace mk {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 8;         // columns a thread has: one draw of the generator
constexpr int64_t kMaxParts = 256;  // partial rows of the column sums

struct DropArgs {
  const void *x, *bias, *residual;
  void* out;
  float* part;  // backward: partial column sums, or null
  const uint64_t* step;
  int64_t ld_x, ld_r, ld_out;
  int64_t rows, cols, rows_per_block;
  uint64_t offset;
  uint32_t k0, k1;
  uint32_t cut;  // T
  float scale;
  int ct_log2;
  uint32_t col_tiles;
};

struct F16 { uint16_t bits; };
template <typename T> __device__ inline float widen(T v);
template <> __device__ inline float widen<float>(float v) { return v; }
template <> __device__ inline float widen<uint16_t>(uint16_t v) { return bf16_to_f32(v); }
template <> __device__ inline float widen<F16>(F16 v) { return f16_to_f32(v.bits); }
template <typename T> __device__ inline T narrow(float v);
template <> __device__ inline float narrow<float>(float v) { return v; }
template <> __device__ inline uint16_t narrow<uint16_t>(float v) { return f32_to_bf16(v); }
template <> __device__ inline F16 narrow<F16>(float v) { return F16{f32_to_f16(v)}; }

// 16 bytes of T at an element-aligned address (one instruction on gfx950)
template <typename T> constexpr int kE = 16 / int(sizeof(T));
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Chunk { T v[kE<T>]; };

// the group's n columns at p (n < 8: the row's last)
template <typename T>
__device__ inline void load8(const T* p, int n, float (&v)[kGroup]) {
  if (n == kGroup) {
#pragma unroll
    for (int h = 0; h < kGroup / kE<T>; ++h) {
      const Chunk<T> c = *reinterpret_cast<const Chunk<T>*>(p + kE<T> * h);
#pragma unroll
      for (int e = 0; e < kE<T>; ++e) v[kE<T> * h + e] = widen(c.v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kGroup; ++e) v[e] = e < n ? widen(p[e]) : 0.f;
  }
}
template <typename T>
__device__ inline void store8(T* p, int n, const float (&v)[kGroup]) {
  if (n == kGroup) {
#pragma unroll
    for (int h = 0; h < kGroup / kE<T>; ++h) {
      Chunk<T> c;
#pragma unroll
      for (int e = 0; e < kE<T>; ++e) c.v[e] = narrow<T>(v[kE<T> * h + e]);
      *reinterpret_cast<Chunk<T>*>(p + kE<T> * h) = c;
    }
  } else {
#pragma unroll
    for (int e = 0; e < kGroup; ++e)
      if (e < n) p[e] = narrow<T>(v[e]);
  }
}

// The 8 fields of group g of row r: Philox-4x32, 10 rounds.
struct Fields { uint32_t w[4]; };
__device__ inline Fields philox(uint32_t g, uint32_t r, uint32_t o0, uint32_t o1, uint32_t k0, uint32_t k1) {
  uint32_t c0 = g, c1 = r, c2 = o0, c3 = o1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = uint64_t(c0) * 0xD2511F53u, p1 = uint64_t(c2) * 0xCD9E8D57u;
    c0 = uint32_t(p1 >> 32) ^ c1 ^ k0;
    c1 = uint32_t(p1);
    c2 = uint32_t(p0 >> 32) ^ c3 ^ k1;
    c3 = uint32_t(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

template <typename T, bool BWD>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const DropArgs a) {
  const int ct = 1 << a.ct_log2;
  const int tx = int(threadIdx.x) & (ct - 1), ty = int(threadIdx.x) >> a.ct_log2, high = kThreads >> a.ct_log2;
  const uint32_t tile = blockIdx.x % a.col_tiles;
  const int64_t block_row = blockIdx.x / a.col_tiles;
  const int64_t g = int64_t(tile) * ct + tx;
  const int64_t col = g * kGroup;
  const int n = int(std::min<int64_t>(a.cols - col, kGroup));  // below 1: no columns here
  const uint64_t o = a.offset + (a.step ? *a.step : 0);
  const uint32_t o0 = uint32_t(o), o1 = uint32_t(o >> 32);
  const T* x = static_cast<const T*>(a.x) + col;
  const T* res = static_cast<const T*>(a.residual) + col;
  T* out = static_cast<T*>(a.out) + col;
  float bias[kGroup], sum[kGroup];
#pragma unroll
  for (int e = 0; e < kGroup; ++e) bias[e] = sum[e] = 0.f;
  if (!BWD && a.bias && n > 0) load8(static_cast<const T*>(a.bias) + col, n, bias);
  const int64_t r0 = block_row * a.rows_per_block, r1 = std::min(a.rows, r0 + a.rows_per_block);
  if (n > 0) {
#pragma unroll 2
    for (int64_t r = r0 + ty; r < r1; r += high) {
      float v[kGroup], rv[kGroup];
      load8(x + r * a.ld_x, n, v);
      if (!BWD && a.residual) {
        load8(res + r * a.ld_r, n, rv);
      } else {
#pragma unroll
        for (int e = 0; e < kGroup; ++e) rv[e] = 0.f;
      }
      const Fields f = philox(uint32_t(g), uint32_t(r), o0, o1, a.k0, a.k1);
#pragma unroll
      for (int e = 0; e < kGroup; ++e) {
        const uint32_t field = e & 1 ? f.w[e / 2] >> 16 : f.w[e / 2] & 0xFFFFu;
        // selected, not multiplied: a dropped infinity or NaN is dropped
        const bool keep = field >= a.cut;
        if (BWD) {
          v[e] = keep ? v[e] : 0.f;
          sum[e] += v[e];
          v[e] *= a.scale;
        } else {
          v[e] = keep ? fmaf(v[e] + bias[e], a.scale, rv[e]) : rv[e];
        }
      }
      store8(out + r * a.ld_out, n, v);
    }
  }
  if (!BWD || !a.part) return;
  // column sums: the block's rows in order of ty
  __shared__ float lds[kThreads * kGroup];
#pragma unroll
  for (int e = 0; e < kGroup; ++e) lds[e * kThreads + threadIdx.x] = sum[e];
  __syncthreads();
  float* part = a.part + block_row * a.cols;
  for (int i = int(threadIdx.x); i < ct * kGroup; i += kThreads) {
    const int e = i & (kGroup - 1), t = i / kGroup;
    float s = 0.f;
    for (int y = 0; y < high; ++y) s += lds[e * kThreads + (y << a.ct_log2) + t];
    const int64_t c = (int64_t(tile) * ct + t) * kGroup + e;
    if (c < a.cols) part[c] = s;
  }
}

// y[c] = scale * (the partial rows' sum, 8 runs of them in order)
__global__ __launch_bounds__(kThreads) void colsum_final_kernel(const float* part, int64_t parts, int64_t cols, float scale,
                                                                float* y) {
  __shared__ float lds[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = int64_t(blockIdx.x) * 32 + tx;
  const int64_t run = (parts + 7) / 8, p0 = ty * run, p1 = std::min(parts, p0 + run);
  float s = 0.f;
  if (c < cols)
    for (int64_t p = p0; p < p1; ++p) s += part[p * cols + c];
  lds[ty][tx] = s;
  __syncthreads();
  if (ty != 0 || c >= cols) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += lds[i][tx];
  y[c] = s * scale;
}

// Groups a block is wide: the widest power of two that pads the row least.
int ct_log2(int64_t groups) {
  int best = 0;
  int64_t best_pad = -1;
  for (int l = 8; l >= 3 || (int64_t(1) << l) >= groups; --l) {
    const int64_t ct = int64_t(1) << l, pad = (groups + ct - 1) / ct * ct;
    if (best_pad < 0 || pad * 16 < best_pad * 15) best = l, best_pad = pad;
    if (l == 0) break;
  }
  return best;
}

int64_t row_parts(int64_t rows, int high) { return std::min(kMaxParts, (rows + high - 1) / high); }

const char* bad_pointer(const void* p, int bytes, bool needed) {
  if (!p) return needed ? "null " : nullptr;
  return reinterpret_cast<uintptr_t>(p) % bytes ? "not aligned to its elements: " : nullptr;
}

int check(const char* what, int io_type, int64_t rows, int64_t cols, double p) {
  const std::string w(what);
  if (io_type != MK_BF16 && io_type != MK_F16 && io_type != MK_F32)
    return fail(MK_ERR_UNSUPPORTED, w + ": io_type must be bf16, f16 or f32");
  if (rows < 0 || cols < 0) return fail(MK_ERR_INVALID, w + ": negative shape");
  if (rows >= int64_t(1) << 32 || cols > int64_t(1) << 31)
    return fail(MK_ERR_UNSUPPORTED, w + ": rows must be below 2^32 and cols at most 2^31");
  if (!(p >= 0.0 && p <= 1.0)) return fail(MK_ERR_INVALID, w + ": p must be in [0, 1]");
  return MK_OK;
}

void draw_args(DropArgs& a, int64_t rows, int64_t cols, double p, uint64_t seed, uint64_t offset, const uint64_t* step) {
  a.rows = rows, a.cols = cols;
  a.k0 = uint32_t(seed), a.k1 = uint32_t(seed >> 32);
  a.offset = offset, a.step = step;
  a.cut = uint32_t(std::nearbyint(p * 65536.0));
  a.scale = a.cut < 65536u ? float(65536.0 / (65536.0 - a.cut)) : 0.f;
  const int64_t groups = (cols + kGroup - 1) / kGroup;
  a.ct_log2 = ct_log2(groups);
  a.col_tiles = uint32_t((groups + (int64_t(1) << a.ct_log2) - 1) >> a.ct_log2);
}

template <bool BWD>
int launch(const char* what, hipStream_t s, int io_type, DropArgs& a, int64_t parts) {
  a.rows_per_block = (a.rows + parts - 1) / parts;
  parts = (a.rows + a.rows_per_block - 1) / a.rows_per_block;
  const uint64_t blocks = uint64_t(parts) * a.col_tiles;
  if (blocks >= uint64_t(1) << 24) return fail(MK_ERR_UNSUPPORTED, std::string(what) + ": too many elements");
  const dim3 g{unsigned(blocks)}, b{kThreads};
  if (io_type == MK_BF16) hipLaunchKernelGGL((dropout_kernel<uint16_t, BWD>), g, b, 0, s, a);
  else if (io_type == MK_F16) hipLaunchKernelGGL((dropout_kernel<F16, BWD>), g, b, 0, s, a);
  else hipLaunchKernelGGL((dropout_kernel<float, BWD>), g, b, 0, s, a);
  return check_launch(what);
}

}  // namespace
}  // namespace mk

using namespace mk;

extern "C" int mk_dropout_add(void* stream, int io_type, int64_t rows, int64_t cols, const void* x, int64_t ld_x,
                              const void* bias, const void* residual, int64_t ld_residual, double p, uint64_t seed,
                              uint64_t offset, const uint64_t* step, void* out, int64_t ld_out) {
  clear_error();
  const char* what = "mk_dropout_add";
  if (int rc = check(what, io_type, rows, cols, p)) return rc;
  if (rows == 0 || cols == 0) return MK_OK;
  const int esz = dtype_bytes(io_type);
  const struct { const char* name; const void* ptr; int bytes; bool needed; } ptrs[] = {
      {"x", x, esz, true}, {"out", out, esz, true}, {"bias", bias, esz, false}, {"residual", residual, esz, false},
      {"step", step, 8, false}};
  for (const auto& q : ptrs)
    if (const char* why = bad_pointer(q.ptr, q.bytes, q.needed))
      return fail(MK_ERR_INVALID, std::string(what) + ": " + why + q.name);
  if (ld_x < 0 || ld_residual < 0 || (rows > 1 && ld_out < cols))
    return fail(MK_ERR_INVALID, std::string(what) + ": a pitch below 0, or rows of out that overlap");
  DropArgs a{};
  draw_args(a, rows, cols, p, seed, offset, step);
  a.x = x, a.bias = bias, a.residual = residual, a.out = out;
  a.ld_x = ld_x, a.ld_r = ld_residual, a.ld_out = ld_out;
  // a row a thread until 16 blocks a CU are there, then longer walks
  const int high = kThreads >> a.ct_log2;
  const int64_t most = (rows + high - 1) / high, want = std::max<int64_t>(1, 8192 / a.col_tiles);
  return launch<false>(what, as_stream(stream), io_type, a, std::min(most, want));
}

extern "C" size_t mk_dropout_add_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return size_t(std::min(kMaxParts, rows) * cols * 4);
}

extern "C" int mk_dropout_add_bwd(void* stream, int io_type, int64_t rows, int64_t cols, const void* dy, int64_t ld_dy,
                                  double p, uint64_t seed, uint64_t offset, const uint64_t* step, void* dx,
                                  int64_t ld_dx, float* dx_colsum, void* workspace) {
  clear_error();
  const char* what = "mk_dropout_add_bwd";
  if (int rc = check(what, io_type, rows, cols, p)) return rc;
  if (cols == 0) return MK_OK;
  const int esz = dtype_bytes(io_type);
  if (const char* why = bad_pointer(dx_colsum, 4, false))
    return fail(MK_ERR_INVALID, std::string(what) + ": " + why + "dx_colsum");
  if (rows == 0) return dx_colsum ? mk_fill(stream, 4, cols, 0, dx_colsum) : MK_OK;
  const struct { const char* name; const void* ptr; int bytes; bool needed; } ptrs[] = {
      {"dy", dy, esz, true}, {"dx", dx, esz, true}, {"step", step, 8, false},
      {"workspace", workspace, 4, dx_colsum != nullptr}};
  for (const auto& q : ptrs)
    if (const char* why = bad_pointer(q.ptr, q.bytes, q.needed))
      return fail(MK_ERR_INVALID, std::string(what) + ": " + why + q.name);
  if (ld_dy < 0 || (rows > 1 && ld_dx < cols))
    return fail(MK_ERR_INVALID, std::string(what) + ": a pitch below 0, or rows of dx that overlap");
  DropArgs a{};
  draw_args(a, rows, cols, p, seed, offset, step);
  a.x = dy, a.out = dx;
  a.ld_x = ld_dy, a.ld_out = ld_dx;
  a.part = dx_colsum ? static_cast<float*>(workspace) : nullptr;
  hipStream_t s = as_stream(stream);
  if (int rc = launch<true>(what, s, io_type, a, row_parts(rows, kThreads >> a.ct_log2))) return rc;
  if (!dx_colsum) return MK_OK;
  const int64_t parts = (rows + a.rows_per_block - 1) / a.rows_per_block;
  hipLaunchKernelGGL(colsum_final_kernel, dim3(unsigned((cols + 31) / 32)), dim3(kThreads), 0, s, a.part, parts, cols,
                     a.scale, dx_colsum);
  return check_launch(what);
}
