// Rows to eight bits: residual add + RMS norm + rounding (mk_add_rmsnorm_int8),
// rounding of rows or of their GELU (mk_quantize_rows), and the way back
// (mk_dequantize_rows).  The operands of mk_gemm_int8.
//
//   s = x + r (one rounding, stored);  y = s rstd gamma,  rstd = 1 / sqrt(mean(s^2) + eps)
//   scale = max |y| / 127,  q = rint(y / scale)
// rstd cancels out of y / scale: with t = s gamma and top = max |t|,
//   q = rint(t 127 / top),  scale = rstd top / 127,
// so the sum of squares and the maximum are reduced together, in one round,
// and a row is read once and stays in registers.
//
// The squares are summed in 64 bits: an fp32 or bf16 value above 2^64 has no
// square in 32.  The maximum is taken over the bits of |t| as whole numbers,
// where NaN is above infinity is above every number, so neither is lost.
//
// Bound: HBM, each operand once, at the 5.4 MB a us of a 200 MiB copy: the norm of 8192 x
// 4096 in bf16 (235 MB) takes 43 us, rounding 50257 x 768 of fp32 (193 MB) 34 us, the way
// back 36 us (operands of three calls in turn; of one call, part of them stays in the
// last-level cache: 37, 28, 29 us).  One row is a launch and two round trips to memory: 768 in
// 2.8 us.  A team of W waves has a row; its lanes hold up to NV chunks of 16 bytes each.
// The last chunk of a row that is no whole number of chunks is the row's last 16 bytes:
// what it shares with the chunk before it is left out of the sum and written twice
// with the same values (after every load of the row, so that the sum may be x or r).
#include "mk_common.h"

#include <algorithm>
#include <string>

namespace mk {
namespace {

enum Mode { kAddNorm, kNorm, kPlain, kGelu };

struct RowsArgs {
  const void *x, *r, *gamma;
  void* sum;
  int8_t* q;
  float* scale;
  int64_t rows, cols, ld_x, ld_r, ld_sum, ld_q;
  float eps;
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
template <int N> struct __attribute__((packed, aligned(1))) Bytes { uint32_t v[N / 4]; };

// the row's value that is rounded
template <Mode M, typename T>
__device__ inline float value(T s, T gamma, bool has_gamma) {
  if constexpr (M == kGelu) return gelu_tanh_f32(widen(s));
  if constexpr (M == kPlain) return widen(s);
  return has_gamma ? widen(s) * widen(gamma) : widen(s);
}

struct Stats {
  double squares;
  uint32_t top;  // bits of the largest |t|
};

__device__ inline Stats join(Stats a, Stats b) { return {a.squares + b.squares, max(a.top, b.top)}; }

__device__ inline Stats wave_join(Stats s) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1)
    s = join(s, {__shfl_xor(s.squares, m, kWave), uint32_t(__shfl_xor(int(s.top), m, kWave))});
  return s;
}

// over the waves of a team, in wave order
template <int W>
__device__ inline Stats team_join(Stats s, Stats* lds) {
  s = wave_join(s);
  if constexpr (W == 1) return s;
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = s;
  __syncthreads();
  s = lds[0];
#pragma unroll
  for (int w = 1; w < W; ++w) s = join(s, lds[w]);
  return s;
}

// What a row's t are multiplied by, 127 / top = hi + lo to 2^-45 of itself (2^-28 above
// 2^100, where lo is no normal number), and its scale.
struct Steps {
  float hi, lo, scale;
};

// Below 2^-119 the scale is no normal fp32 number: such a row is all zeros.  A
// row with a NaN or an infinity has scale NaN and zeros, so that whatever is
// multiplied by it is NaN.
template <Mode M>
__device__ inline Steps steps(const Stats& s, const RowsArgs& p) {
  if (s.top >= 0x7f800000u) return {0.f, 0.f, __builtin_nanf("")};
  const float top = __builtin_bit_cast(float, s.top);
  if (top < 0x1p-119f) return {0.f, 0.f, 0.f};
  const float hi = 127.f / top, lo = fmaf(-hi, top, 127.f) * (hi * (1.f / 127.f));
  if constexpr (M == kPlain || M == kGelu) return {hi, lo, top / 127.f};
  const double rstd = 1.0 / sqrt(s.squares / double(p.cols) + double(p.eps));
  return {hi, lo, float(rstd * double(top) / 127.0)};
}

// rint(t 127 / top) in a float's low byte: 1.5 2^23 + n holds the whole number n in
// its low bits, and the addition rounds to nearest even.  The quotient is rounded to
// fp32 first, once: with hi alone the rounding of the reciprocal, the same for the whole
// row, decided the exact halves, which rows of 16-bit values hold often (t = top / 2; of
// 512 x 768 bf16 values 290 were a step off for it).  A GELU has no exact values to
// keep, and is rounded in one step (8192 x 16384 80 us, 86 in two); plain rows of 16 x
// 16384 take 3.2 us, 3.1 in one, 8192 x 4096 and its norm the same.
template <Mode M>
__device__ inline uint32_t in_low_byte(float t, const Steps& step) {
  if constexpr (M == kGelu) return __builtin_bit_cast(uint32_t, fmaf(t, step.hi, 12582912.f));
  return __builtin_bit_cast(uint32_t, fmaf(t, step.hi, t * step.lo) + 12582912.f);
}
// the low bytes of four words, a to d from the lowest up (selector 0x0c: zeros);
// zeros for a step of 0, where t may be NaN
__device__ inline uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d, const Steps& step) {
  const uint32_t w = __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
  return step.hi != 0.f ? w : 0u;
}

// Rows of E to 64 W NV E elements in registers.
template <typename T, Mode M, int W, int NV>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void rows_int8_kernel(const RowsArgs p) {
  constexpr int E = kE<T>, S = 64 * W, kRows = W == 1 ? 4 : 1;
  constexpr bool kIsNorm = M == kAddNorm || M == kNorm;
  __shared__ Stats lds[W];
  const int t = int(threadIdx.x) % S;
  const int64_t row = (int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * kRows + int(threadIdx.x) / S;
  if (row >= p.rows) return;  // whole teams
  const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
  const T* gamma = static_cast<const T*>(p.gamma);
  const bool has_gamma = kIsNorm && gamma;
  const int cols = int(p.cols), chunks = (cols + E - 1) / E;
  // lanes past the last chunk load it too (and neither count nor store it)
  int at[NV];
  Chunk<T> s[NV], g[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    at[v] = min(min(t + S * v, chunks - 1) * E, cols - E);
    s[v] = *reinterpret_cast<const Chunk<T>*>(x + at[v]);
  }
  if constexpr (M == kAddNorm) {
    const T* r = static_cast<const T*>(p.r) + row * p.ld_r;
    Chunk<T> b[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) b[v] = *reinterpret_cast<const Chunk<T>*>(r + at[v]);
    if (has_gamma) {
#pragma unroll
      for (int v = 0; v < NV; ++v) g[v] = *reinterpret_cast<const Chunk<T>*>(gamma + at[v]);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < E; ++e) s[v].v[e] = narrow<T>(widen(s[v].v[e]) + widen(b[v].v[e]));
  } else if (has_gamma) {
#pragma unroll
    for (int v = 0; v < NV; ++v) g[v] = *reinterpret_cast<const Chunk<T>*>(gamma + at[v]);
  }
  if (!has_gamma) {
#pragma unroll
    for (int v = 0; v < NV; ++v) g[v] = s[v];  // not used
  }
  Stats st{0.0, 0u};
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int shared = (t + S * v) * E - at[v];  // elements the chunk before holds too; all E past the last chunk
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (kIsNorm) {
        const double f = e >= shared ? double(widen(s[v].v[e])) : 0.0;
        st.squares = fma(f, f, st.squares);
      }
      st.top = max(st.top, __builtin_bit_cast(uint32_t, value<M>(s[v].v[e], g[v].v[e], has_gamma)) & 0x7fffffffu);
    }
  }
  st = team_join<W>(st, lds);
  const Steps step = steps<M>(st, p);
  T* sum = static_cast<T*>(p.sum) + row * p.ld_sum;
  int8_t* q = p.q + row * p.ld_q;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (t + S * v >= chunks) continue;
    if constexpr (M == kAddNorm) *reinterpret_cast<Chunk<T>*>(sum + at[v]) = s[v];
    Bytes<E> out;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = in_low_byte<M>(value<M>(s[v].v[e + k], g[v].v[e + k], has_gamma), step);
      out.v[e / 4] = low_bytes(w[0], w[1], w[2], w[3], step);
    }
    *reinterpret_cast<Bytes<E>*>(q + at[v]) = out;
  }
  if (t == 0) p.scale[row] = step.scale;
}

// Rows of any length, read twice, element by element: those too short for a
// chunk and those too long for the registers (a lane reads the sum that it
// stored itself).
template <typename T, Mode M, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void rows_int8_any_kernel(const RowsArgs p) {
  constexpr int S = 64 * W, kRows = W == 1 ? 4 : 1;
  constexpr bool kIsNorm = M == kAddNorm || M == kNorm;
  __shared__ Stats lds[W];
  const int t = int(threadIdx.x) % S;
  const int64_t row = (int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * kRows + int(threadIdx.x) / S;
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
  const T* r = static_cast<const T*>(p.r) + row * p.ld_r;
  const T* gamma = static_cast<const T*>(p.gamma);
  T* sum = static_cast<T*>(p.sum) + row * p.ld_sum;
  int8_t* q = p.q + row * p.ld_q;
  const bool has_gamma = kIsNorm && gamma;
  Stats st{0.0, 0u};
  for (int64_t c = t; c < p.cols; c += S) {
    T s = x[c];
    if constexpr (M == kAddNorm) {
      s = narrow<T>(widen(s) + widen(r[c]));
      sum[c] = s;
    }
    if constexpr (kIsNorm) st.squares = fma(double(widen(s)), double(widen(s)), st.squares);
    const float y = value<M>(s, has_gamma ? gamma[c] : s, has_gamma);
    st.top = max(st.top, __builtin_bit_cast(uint32_t, y) & 0x7fffffffu);
  }
  st = team_join<W>(st, lds);
  const Steps step = steps<M>(st, p);
  for (int64_t c = t; c < p.cols; c += S) {
    const T s = M == kAddNorm ? sum[c] : x[c];
    const uint32_t w = in_low_byte<M>(value<M>(s, has_gamma ? gamma[c] : s, has_gamma), step);
    q[c] = int8_t(step.hi != 0.f ? w & 0xffu : 0u);
  }
  if (t == 0) p.scale[row] = step.scale;
}

// y = q scale: a lane writes 16 bytes of four places of the row in a step, all four
// loaded first; the elements behind the last whole chunk one by one
template <typename T, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void dequantize_kernel(int64_t rows, int64_t cols, const int8_t* q,
                                                                           int64_t ld_q, const float* scale, T* y,
                                                                           int64_t ld_y) {
  constexpr int E = kE<T>, S = 64 * W, kRows = W == 1 ? 4 : 1, kSteps = 4;
  struct __attribute__((packed, aligned(1))) In { int8_t v[E]; };
  const int t = int(threadIdx.x) % S;
  const int64_t row = (int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * kRows + int(threadIdx.x) / S;
  if (row >= rows) return;
  const float f = scale[row];
  q += row * ld_q;
  y += row * ld_y;
  const int64_t whole = cols / E;
  for (int64_t i = t; i < whole; i += S * kSteps) {
    In in[kSteps];
#pragma unroll
    for (int v = 0; v < kSteps; ++v) in[v] = *reinterpret_cast<const In*>(q + E * std::min(i + S * v, whole - 1));
#pragma unroll
    for (int v = 0; v < kSteps; ++v) {
      if (i + S * v >= whole) continue;
      Chunk<T> out;
#pragma unroll
      for (int e = 0; e < E; ++e) out.v[e] = narrow<T>(float(in[v].v[e]) * f);
      *reinterpret_cast<Chunk<T>*>(y + E * (i + S * v)) = out;
    }
  }
  if (const int64_t c = E * whole + t; c < cols) y[c] = narrow<T>(float(q[c]) * f);
}

// teams of W waves over `rows` rows: below HIP's 2^32 threads an axis
template <int W>
dim3 row_grid(int64_t rows) {
  const int64_t blocks = W == 1 ? (rows + 3) / 4 : rows, wide = int64_t(1) << 21;
  return blocks <= wide ? dim3(unsigned(blocks)) : dim3(unsigned(wide), unsigned((blocks + wide - 1) / wide));
}
constexpr int64_t kMaxRows = int64_t(1) << 36;

template <typename T, Mode M, int W, int NV>
void launch_held(hipStream_t s, const RowsArgs& a) {
  hipLaunchKernelGGL((rows_int8_kernel<T, M, W, NV>), row_grid<W>(a.rows), dim3(W == 1 ? 256 : 64 * W), 0, s, a);
}

// Teams by the row's chunks: as few waves as hold the row in 2 to 4 chunks a lane, more
// where they would leave CUs idle.  us, for W x NV, bf16 (every sum to the same memory,
// which stays in the last-level cache): norm of 8192 x 768 1 x 2: 11.2, 2 x 1: 12.7, 4 x 1:
// 18.6; of 8192 x 2048 2 x 2: 21.2, 1 x 4: 22.2, 4 x 1: 22.2; of 256 x 2048 2 x 2: 3.8, 4 x 1:
// 3.6; of 8192 x 4096 4 x 2: 38.1, 1 x 8: 42.9, 8 x 1: 43.8, 16 x 1: 72; of 1 x 8192 4 x 4:
// 3.6, 8 x 2: 3.6, 16 x 1: 4.0; of 4096 x 16384 8 x 4: 91, 4 x 8: 88, 16 x 2: 99; of 64 x 16384
// 5.5, 6.0, 6.0.  50257 x 768 of fp32 to 8 bits 2 x 2: 34, 4 x 1: 46.
// Longer rows than 16 x 4 holds are read twice: 1024 x 16384 of fp32 47 us held, 69 so.
template <typename T, Mode M>
int launch_rows(hipStream_t s, const RowsArgs& a, const char* what) {
  const int64_t chunks = (a.cols + kE<T> - 1) / kE<T>;
  if (a.cols < kE<T>)
    hipLaunchKernelGGL((rows_int8_any_kernel<T, M, 1>), row_grid<1>(a.rows), dim3(256), 0, s, a);
  else if (chunks > 4096)
    hipLaunchKernelGGL((rows_int8_any_kernel<T, M, 16>), row_grid<16>(a.rows), dim3(1024), 0, s, a);
  else if (chunks <= 64) launch_held<T, M, 1, 1>(s, a);
  else if (chunks <= 128) launch_held<T, M, 1, 2>(s, a);
  else if (chunks <= 256 && a.rows >= 1024) launch_held<T, M, 2, 2>(s, a);
  else if (chunks <= 256) launch_held<T, M, 4, 1>(s, a);
  else if (chunks <= 512) launch_held<T, M, 4, 2>(s, a);
  else if (chunks <= 1024) launch_held<T, M, 4, 4>(s, a);
  else if (chunks <= 2048) launch_held<T, M, 8, 4>(s, a);
  else launch_held<T, M, 16, 4>(s, a);
  return check_launch(what);
}

template <Mode M>
int launch_typed(hipStream_t s, int io_type, const RowsArgs& a, const char* what) {
  if (io_type == MK_BF16) return launch_rows<uint16_t, M>(s, a, what);
  if (io_type == MK_F16) return launch_rows<F16, M>(s, a, what);
  return launch_rows<float, M>(s, a, what);
}

template <typename T>
int launch_dequantize(hipStream_t s, int64_t rows, int64_t cols, const int8_t* q, int64_t ld_q, const float* scale,
                      void* y, int64_t ld_y) {
  // us, 1, 4 and 16 waves a row: 8192 x 2048 of bf16 11.3, 14.8, 17.5; 8192 x 4096 21.6,
  // 20.0, 27.5; 1 x 8192 3.1, 2.1, 2.2; 64 x 40000 16.1, 5.8, 4.6; 50257 x 768 of fp32 36, 43, 80
  const int64_t chunks = cols / kE<T>;
  if (chunks <= 256)
    hipLaunchKernelGGL((dequantize_kernel<T, 1>), row_grid<1>(rows), dim3(256), 0, s, rows, cols, q, ld_q, scale,
                       static_cast<T*>(y), ld_y);
  else if (chunks <= 2048)
    hipLaunchKernelGGL((dequantize_kernel<T, 4>), row_grid<4>(rows), dim3(256), 0, s, rows, cols, q, ld_q, scale,
                       static_cast<T*>(y), ld_y);
  else
    hipLaunchKernelGGL((dequantize_kernel<T, 16>), row_grid<16>(rows), dim3(1024), 0, s, rows, cols, q, ld_q, scale,
                       static_cast<T*>(y), ld_y);
  return check_launch("mk_dequantize_rows");
}

// What every entry point of this file asks of its shape, and of one operand of
// it; null when it holds.
const char* bad_shape(int type, int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1) return "need rows >= 0 and cols >= 1";
  if (type != MK_BF16 && type != MK_F16 && type != MK_F32) return "type must be bf16/f16/f32";
  if (rows > kMaxRows) return "more than 2^36 rows";
  return nullptr;
}
const char* bad_operand(const void* p, int bytes, int64_t rows, int64_t cols, int64_t ld, bool written) {
  if (!p) return "null ";
  if (reinterpret_cast<uintptr_t>(p) % bytes) return "not aligned to its elements: ";
  if (ld < 0 || (written && rows > 1 && ld < cols)) return "row pitch below the columns: ";
  return nullptr;
}
int refuse(const char* entry, const char* why, const char* operand = "") {
  return fail(MK_ERR_INVALID, std::string(entry) + ": " + why + operand);
}
int refuse_shape(const char* entry, const char* why, int64_t rows, int64_t cols) {
  return fail(rows < 0 || cols < 1 ? MK_ERR_INVALID : MK_ERR_UNSUPPORTED, std::string(entry) + ": " + why);
}

}  // namespace
}  // namespace mk

using namespace mk;

extern "C" int mk_add_rmsnorm_int8(void* stream, int io_type, int64_t rows, int64_t cols, const void* x, int64_t ld_x,
                                   const void* residual, int64_t ld_residual, const void* gamma, float eps, void* sum,
                                   int64_t ld_sum, int8_t* q, int64_t ld_q, float* scale) {
  clear_error();
  const char* at = "mk_add_rmsnorm_int8";
  if (const char* w = bad_shape(io_type, rows, cols)) return refuse_shape(at, w, rows, cols);
  if (!(eps >= 0.f)) return refuse(at, "eps must be a number >= 0");
  if (rows == 0) return MK_OK;
  const int bytes = dtype_bytes(io_type);
  if (const char* w = bad_operand(x, bytes, rows, cols, ld_x, false)) return refuse(at, w, "x");
  if (residual) {
    if (const char* w = bad_operand(residual, bytes, rows, cols, ld_residual, false)) return refuse(at, w, "residual");
    if (const char* w = bad_operand(sum, bytes, rows, cols, ld_sum, true)) return refuse(at, w, "sum");
  }
  if (gamma)
    if (const char* w = bad_operand(gamma, bytes, 1, cols, cols, false)) return refuse(at, w, "gamma");
  if (const char* w = bad_operand(q, 1, rows, cols, ld_q, true)) return refuse(at, w, "q");
  if (const char* w = bad_operand(scale, 4, 1, 1, 1, true)) return refuse(at, w, "scale");
  const RowsArgs a{x, residual, gamma, sum, q, scale, rows, cols, ld_x, ld_residual, ld_sum, ld_q, eps};
  return residual ? launch_typed<kAddNorm>(as_stream(stream), io_type, a, at)
                  : launch_typed<kNorm>(as_stream(stream), io_type, a, at);
}

extern "C" int mk_quantize_rows(void* stream, int io_type, int64_t rows, int64_t cols, const void* x, int64_t ld_x,
                                int gelu, int8_t* q, int64_t ld_q, float* scale) {
  clear_error();
  const char* at = "mk_quantize_rows";
  if (const char* w = bad_shape(io_type, rows, cols)) return refuse_shape(at, w, rows, cols);
  if (rows == 0) return MK_OK;
  if (const char* w = bad_operand(x, dtype_bytes(io_type), rows, cols, ld_x, false)) return refuse(at, w, "x");
  if (const char* w = bad_operand(q, 1, rows, cols, ld_q, true)) return refuse(at, w, "q");
  if (const char* w = bad_operand(scale, 4, 1, 1, 1, true)) return refuse(at, w, "scale");
  const RowsArgs a{x, nullptr, nullptr, nullptr, q, scale, rows, cols, ld_x, 0, 0, ld_q, 0.f};
  return gelu ? launch_typed<kGelu>(as_stream(stream), io_type, a, at)
              : launch_typed<kPlain>(as_stream(stream), io_type, a, at);
}

extern "C" int mk_dequantize_rows(void* stream, int out_type, int64_t rows, int64_t cols, const int8_t* q,
                                  int64_t ld_q, const float* scale, void* y, int64_t ld_y) {
  clear_error();
  const char* at = "mk_dequantize_rows";
  if (const char* w = bad_shape(out_type, rows, cols)) return refuse_shape(at, w, rows, cols);
  if (rows == 0) return MK_OK;
  if (const char* w = bad_operand(q, 1, rows, cols, ld_q, false)) return refuse(at, w, "q");
  if (const char* w = bad_operand(scale, 4, 1, 1, 1, false)) return refuse(at, w, "scale");
  if (const char* w = bad_operand(y, dtype_bytes(out_type), rows, cols, ld_y, true)) return refuse(at, w, "y");
  hipStream_t s = as_stream(stream);
  if (out_type == MK_BF16) return launch_dequantize<uint16_t>(s, rows, cols, q, ld_q, scale, y, ld_y);
  if (out_type == MK_F16) return launch_dequantize<F16>(s, rows, cols, q, ld_q, scale, y, ld_y);
  return launch_dequantize<float>(s, rows, cols, q, ld_q, scale, y, ld_y);
}
