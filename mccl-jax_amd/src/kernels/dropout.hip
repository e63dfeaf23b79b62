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
// A thread has 16 bytes of a row (8 columns of 16 bits, or half a draw's 4 of 32:
// lanes that are neighbours read neighbouring bytes) and walks down the rows, with
// the bias of its columns (forward) or their sums (backward) in registers; a block
// is CT chunks wide (a power of two that wastes little of the last tile) and 256 /
// CT rows high.  Sums of columns go through LDS, then as one partial row a block to
// the workspace, and a second launch adds the partial rows in order.
//
// Memory bounds the large ones: 20011 x 4097 fp32 116 us (5.7 TB/s of the bytes read
// and written, some of them in the last-level cache; a copy 5.4).  8192 x 768 bf16 with
// bias and residual 7.4 us (5.1 TB/s), its gradient 11.5 with the sums, of which 2 to 4
// are the second launch.  64 x 768 is a launch: 2.8 us on the GPU, 7 with the call.
#include "mk_common.h"

#include <algorithm>
#include <cmath>
#include <string>

namespace mk {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 8;  // columns of one draw of the generator
constexpr int64_t kEach = 4;

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

// The 8 fields of group g of row r: Philox-4x32, 10 rounds.
struct Fields { uint32_t w[4]; };
__device__ inline Fields philox(uint32_t g, uint32_t r, uint32_t o0, uint32_t o1, uint32_t k0, uint32_t k1) {
  uint32_t c0 = g, c1 = r, c2 = o0, c3 = o1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = uint64_t(c0) * 0xD2511F53u, p1 = uint64_t(c2) * 0xCD9E8D57u;
    c0 = __builtin_amdgcn_bitop3_b32(uint32_t(p1 >> 32), c1, k0, 0x96);  // three-way exclusive or
    c1 = uint32_t(p1);
    c2 = __builtin_amdgcn_bitop3_b32(uint32_t(p0 >> 32), c3, k1, 0x96);
    c3 = uint32_t(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// One element from x (or dy), its bias and residual.
template <bool BWD>
__device__ inline float drop(bool keep, float x, float bias, float residual, float scale) {
  // selected, not multiplied: a dropped infinity or NaN is dropped
  return BWD ? (keep ? x : 0.f) : (keep ? fmaf(x + bias, scale, residual) : residual);
}
__device__ inline uint32_t field(const Fields& f, int e) {
  return e & 1 ? f.w[e / 2] >> 16 : f.w[e / 2] & 0xFFFFu;
}

// NR: rows a thread has in flight.  Their loads come first: a row after the other
// would wait for memory each time, since a store may be what the next load reads
// as far as the compiler knows.
template <typename T, bool BWD, int NR>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const DropArgs a) {
  constexpr int E = kE<T>;
  const int ct = 1 << a.ct_log2;
  const int tx = int(threadIdx.x) & (ct - 1), ty = int(threadIdx.x) >> a.ct_log2, high = kThreads >> a.ct_log2;
  // a run of rows is one XCD's (workgroups are dealt to the 8 of them in turn): rows
  // off the 128-byte lines have lines that two tiles write
  const uint32_t turn = blockIdx.x / 8, tile = turn % a.col_tiles;
  const int64_t block_row = int64_t(turn / a.col_tiles) * 8 + blockIdx.x % 8;
  const int64_t chunk = int64_t(tile) * ct + tx, col = chunk * E, chunks = a.cols / E;  // whole ones
  const bool upper = E < kGroup && (chunk & 1);  // of the group's fields
  const uint64_t o = a.offset + (a.step ? *a.step : 0);
  const uint32_t o0 = uint32_t(o), o1 = uint32_t(o >> 32);
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  const T* bias_p = static_cast<const T*>(a.bias);
  T* out = static_cast<T*>(a.out);
  const int64_t r0 = block_row * a.rows_per_block, r1 = std::min(a.rows, r0 + a.rows_per_block);
  if (r0 >= a.rows) return;
  float bias[E], sum[E];
#pragma unroll
  for (int e = 0; e < E; ++e) bias[e] = sum[e] = 0.f;
  if (chunk < chunks) {
    if (!BWD && a.bias) {
      const Chunk<T> b = *reinterpret_cast<const Chunk<T>*>(bias_p + col);
#pragma unroll
      for (int e = 0; e < E; ++e) bias[e] = widen(b.v[e]);
    }
    for (int64_t r = r0 + ty; r < r1; r += int64_t(high) * NR) {
      Chunk<T> xv[NR], rv[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int64_t row = r + int64_t(high) * i;
        if (i > 0 && row >= r1) break;
        xv[i] = *reinterpret_cast<const Chunk<T>*>(x + row * a.ld_x + col);
        if (!BWD && a.residual) rv[i] = *reinterpret_cast<const Chunk<T>*>(res + row * a.ld_r + col);
      }
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int64_t row = r + int64_t(high) * i;
        if (i > 0 && row >= r1) break;
        const Fields f = philox(uint32_t(col / kGroup), uint32_t(row), o0, o1, a.k0, a.k1);
        Chunk<T> c;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t at = E < kGroup && upper ? field(f, e + E) : field(f, e);
          float v = drop<BWD>(at >= a.cut, widen(xv[i].v[e]), bias[e], !BWD && a.residual ? widen(rv[i].v[e]) : 0.f, a.scale);
          if (BWD) sum[e] += v, v *= a.scale;
          c.v[e] = narrow<T>(v);
        }
        *reinterpret_cast<Chunk<T>*>(out + row * a.ld_out + col) = c;
      }
    }
  }
  // what is left of the rows past their whole chunks: a thread a row (beside the
  // chunks, their element loads would be another path through every wave that ends a row)
  const int left = int(a.cols - chunks * E);
  const bool has_left = left > 0 && tile + 1 == a.col_tiles;
  float last[E];
#pragma unroll
  for (int e = 0; e < E; ++e) last[e] = 0.f;
  if (has_left) {
    const int64_t c0 = chunks * E;
    for (int64_t row = r0 + threadIdx.x; row < r1; row += kThreads) {
      const Fields f = philox(uint32_t(c0 / kGroup), uint32_t(row), o0, o1, a.k0, a.k1);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (e >= left) break;
        const uint32_t at = E < kGroup && (chunks & 1) ? field(f, e + E) : field(f, e);
        float v = drop<BWD>(at >= a.cut, widen(x[row * a.ld_x + c0 + e]), !BWD && a.bias ? widen(bias_p[c0 + e]) : 0.f,
                            !BWD && a.residual ? widen(res[row * a.ld_r + c0 + e]) : 0.f, a.scale);
        if (BWD) last[e] += v, v *= a.scale;
        out[row * a.ld_out + c0 + e] = narrow<T>(v);
      }
    }
  }
  if (!BWD || !a.part) return;
  // column sums: the block's rows in order of ty, the last columns' in the order of the waves
  __shared__ float lds[kThreads * E];
  __shared__ float ends[kThreads / kWave][E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    lds[threadIdx.x * E + e] = sum[e];
    last[e] = wave_sum_dpp(last[e]);
    if ((threadIdx.x & 63) == 0) ends[threadIdx.x >> 6][e] = last[e];
  }
  __syncthreads();
  float* part = a.part + block_row * a.cols;
  for (int i = int(threadIdx.x); i < ct * E; i += kThreads) {
    float s = 0.f;
    for (int y = 0; y < high; ++y) s += lds[y * ct * E + i];
    const int64_t c = int64_t(tile) * ct * E + i;
    if (c < chunks * E) part[c] = s;
  }
  if (has_left && int(threadIdx.x) < left) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) s += ends[w][threadIdx.x];
    part[chunks * E + threadIdx.x] = s;
  }
}

// y[c] = scale * (the partial rows' sum, 32 runs of them in order)
__global__ __launch_bounds__(1024) void colsum_final_kernel(const float* part, int64_t parts, int64_t cols, float scale,
                                                            float* y) {
  __shared__ float lds[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t run = (parts + 31) / 32, p0 = ty * run, p1 = std::min(parts, p0 + run);
  for (int64_t c0 = int64_t(blockIdx.x) * 32; c0 < cols; c0 += int64_t(gridDim.x) * 32) {
    const int64_t c = c0 + tx;
    float s = 0.f;
    if (c < cols) {
#pragma unroll 8
      for (int64_t p = p0; p < p1; ++p) s += part[p * cols + c];
    }
    lds[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < cols) {
#pragma unroll
      for (int i = 1; i < 32; ++i) s += lds[i][tx];
      y[c] = s * scale;
    }
    __syncthreads();
  }
}

// Chunks a block is wide: the widest power of two that pads the row least.
int ct_log2(int64_t chunks) {
  int best = 0;
  int64_t best_pad = -1;
  for (int l = 8; l >= 3 || (int64_t(1) << l) >= chunks; --l) {
    const int64_t ct = int64_t(1) << l, pad = (chunks + ct - 1) / ct * ct;
    if (best_pad < 0 || pad * 16 < best_pad * 15) best = l, best_pad = pad;
    if (l == 0) break;
  }
  return best;
}

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

void draw_args(DropArgs& a, int io_type, int64_t rows, int64_t cols, double p, uint64_t seed, uint64_t offset, const uint64_t* step) {
  a.rows = rows, a.cols = cols;
  a.k0 = uint32_t(seed), a.k1 = uint32_t(seed >> 32);
  a.offset = offset, a.step = step;
  a.cut = uint32_t(std::nearbyint(p * 65536.0));
  a.scale = a.cut < 65536u ? float(65536.0 / (65536.0 - a.cut)) : 0.f;
  const int64_t each = io_type == MK_F32 ? 4 : 8, chunks = std::max<int64_t>(1, cols / each);
  a.ct_log2 = ct_log2(chunks);
  a.col_tiles = uint32_t((chunks + (int64_t(1) << a.ct_log2) - 1) >> a.ct_log2);
}

// Rows a thread walks down.  One until the chip is full, then up to 4, which are in
// flight together; more only with sums of columns, for fewer partial rows.
int64_t rows_each(const DropArgs& a, bool sums) {
  const int64_t high = kThreads >> a.ct_log2, deep = (a.rows + high - 1) / high;  // rows of a column of threads
  auto cut = [&](int64_t blocks) { return (deep + std::max<int64_t>(1, blocks / a.col_tiles) - 1) / std::max<int64_t>(1, blocks / a.col_tiles); };
  if (!sums) return std::min<int64_t>(kEach, cut(2048));
  const int64_t each = cut(1024);
  return each < 8 ? each : cut(512);
}

template <typename T, bool BWD>
void launch_rows(hipStream_t s, const DropArgs& a, dim3 g, int64_t each) {
  const dim3 b{kThreads};
  if (each >= 4) hipLaunchKernelGGL((dropout_kernel<T, BWD, 4>), g, b, 0, s, a);
  else if (each >= 2) hipLaunchKernelGGL((dropout_kernel<T, BWD, 2>), g, b, 0, s, a);
  else hipLaunchKernelGGL((dropout_kernel<T, BWD, 1>), g, b, 0, s, a);
}

int64_t row_parts(const DropArgs& a) { return (a.rows + a.rows_per_block - 1) / a.rows_per_block; }

template <bool BWD>
int launch(const char* what, hipStream_t s, int io_type, DropArgs& a) {
  const int64_t each = rows_each(a, a.part != nullptr), parts = (a.rows_per_block = each * (kThreads >> a.ct_log2), row_parts(a));
  const uint64_t blocks = uint64_t((parts + 7) / 8 * 8) * a.col_tiles;
  if (blocks >= uint64_t(1) << 24) return fail(MK_ERR_UNSUPPORTED, std::string(what) + ": too many elements");
  const dim3 g{unsigned(blocks)};
  if (io_type == MK_BF16) launch_rows<uint16_t, BWD>(s, a, g, each);
  else if (io_type == MK_F16) launch_rows<F16, BWD>(s, a, g, each);
  else launch_rows<float, BWD>(s, a, g, each);
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
  if (rows > 1 && ((out == x && ld_out != ld_x) || (out == residual && ld_out != ld_residual)))
    return fail(MK_ERR_INVALID, std::string(what) + ": out over x or residual at another pitch");
  DropArgs a{};
  draw_args(a, io_type, rows, cols, p, seed, offset, step);
  a.x = x, a.bias = bias, a.residual = residual, a.out = out;
  a.ld_x = ld_x, a.ld_r = ld_residual, a.ld_out = ld_out;
  return launch<false>(what, as_stream(stream), io_type, a);
}

extern "C" size_t mk_dropout_add_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  DropArgs a{};
  int64_t parts = 0;
  for (int t : {MK_BF16, MK_F32}) {  // 8 or 4 columns a thread
    draw_args(a, t, rows, cols, 0.0, 0, 0, nullptr);
    a.rows_per_block = rows_each(a, true) * (kThreads >> a.ct_log2);
    parts = std::max(parts, row_parts(a));
  }
  return size_t(parts * cols * 4);
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
  if (rows > 1 && dx == dy && ld_dx != ld_dy)
    return fail(MK_ERR_INVALID, std::string(what) + ": dx over dy at another pitch");
  DropArgs a{};
  draw_args(a, io_type, rows, cols, p, seed, offset, step);
  a.x = dy, a.out = dx;
  a.ld_x = ld_dy, a.ld_out = ld_dx;
  a.part = dx_colsum ? static_cast<float*>(workspace) : nullptr;
  hipStream_t s = as_stream(stream);
  if (int rc = launch<true>(what, s, io_type, a)) return rc;
  if (!dx_colsum) return MK_OK;
  hipLaunchKernelGGL(colsum_final_kernel, dim3(unsigned(std::min<int64_t>((cols + 31) / 32, 1 << 16))), dim3(1024), 0, s, a.part, row_parts(a), cols,
                     a.scale, dx_colsum);
  return check_launch(what);
}
