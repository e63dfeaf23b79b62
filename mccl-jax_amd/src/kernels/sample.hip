// The next token from a row of logits (mk_sample_rows): temperature, top-k,
// top-p and min-p, drawn with a random number that the caller gives.
//
//   w_i = exp((x_i - max x) / T);  tokens are ranked by x, larger first, ties by
//   lower index; every limit keeps a run of ranks from the first on, and the
//   token is the first index i whose kept weights w_0 + .. + w_i exceed u times
//   all of them.
//
// What is kept is one cut (key, ties): the tokens whose x is above a value, and
// the first `ties` of those equal to it, in the order of the vocabulary.  So no
// row is sorted: the cut's value is found digit by digit from a histogram of
// counts (top-k) or of weights (top-p) over x's bits, taken as a whole number
// that orders as x does.
//
// Weights are whole numbers: w 2^s rounded, from an exponential in 64 bits, s
// such that a row's sum stays below 2^63 (47 bits for 50257 tokens).  Their sums
// are exact, whatever order the atomics take, and a token is the one that sums
// in 64 bits give but for u within about 2^-40 of a border.
//
// A workgroup has a row.  Bound: a few passes over the row, from L2 after the
// first, at what one CU takes in.
#include "mk_common.h"

#include <algorithm>
#include <string>

namespace mk {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kBins = 4096;                 // 12 bits: a level of the histogram
constexpr int kLane = 8;                    // elements a lane takes at once
constexpr int kChunk = kLane * kWave;       // elements a wave takes at once
constexpr int64_t kMaxVocab = int64_t(kBins) * kChunk;

typedef unsigned long long u64;

struct SampleArgs {
  const void* x;
  int64_t rows, V, ld;
  const float *u, *temperature, *top_p, *min_p;  // null (but u): the value below for every row
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int index_type;
  void* token;
  float* logprob;
  int shift;  // s
};

// An element type's values as whole numbers that order as they do, -0 as +0.
// Finite values and infinities are at least 1.
template <typename T> struct Order;
template <> struct Order<float> {
  static constexpr int kLevels = 3;
  static constexpr int kShift[3] = {20, 10, 0}, kBits[3] = {12, 10, 10};
  static __device__ inline float value(float v) { return v; }
  static __device__ inline uint32_t key(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
  }
  static __device__ inline float of_key(uint32_t k) {
    return __builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
  }
};
struct F16 { uint16_t bits; };
__device__ inline uint32_t key16(uint32_t b) {
  b = b == 0x8000u ? 0u : b;
  return b ^ (b >> 15 ? 0xffffu : 0x8000u);
}
__device__ inline uint16_t of_key16(uint32_t k) { return uint16_t(k ^ (k >> 15 ? 0x8000u : 0xffffu)); }
template <> struct Order<uint16_t> {
  static constexpr int kLevels = 2;
  static constexpr int kShift[2] = {4, 0}, kBits[2] = {12, 4};
  static __device__ inline float value(uint16_t v) { return bf16_to_f32(v); }
  static __device__ inline uint32_t key(uint16_t v) { return key16(v); }
  static __device__ inline float of_key(uint32_t k) { return bf16_to_f32(of_key16(k)); }
};
template <> struct Order<F16> {
  static constexpr int kLevels = 2;
  static constexpr int kShift[2] = {4, 0}, kBits[2] = {12, 4};
  static __device__ inline float value(F16 v) { return f16_to_f32(v.bits); }
  static __device__ inline uint32_t key(F16 v) { return key16(v.bits); }
  static __device__ inline float of_key(uint32_t k) { return f16_to_f32(of_key16(k)); }
};

template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Run { T v[kLane]; };

struct Shared {
  u64 mass[kBins];      // a level's weights by digit; then the chunks' weights
  uint32_t count[kBins];  // a level's counts by digit; then the chunks' ties
  u64 wave_sum[kWaves];
  uint32_t top, bad;
  // what the one thread that found a place leaves for the others
  int found;
  u64 before, total;
  uint32_t ties_before;
};

__device__ inline u64 shfl_up(u64 v, int d) { return __shfl_up(v, d, kWave); }

// sum of v over the threads before this one (and all of them, in total)
__device__ inline u64 scan(u64 v, Shared& sh, u64& total) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  u64 s = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const u64 o = shfl_up(s, d);
    if (lane >= d) s += o;
  }
  __syncthreads();
  if (lane == kWave - 1) sh.wave_sum[wave] = s;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) before = all;
    all += sh.wave_sum[w];
  }
  total = all;
  return before + s - v;
}

template <typename T>
struct Row {
  using O = Order<T>;
  const T* x;
  int64_t V;
  double top, per;  // the largest value; log2(e) / temperature
  double least;     // min-p
  int shift;
  uint32_t cut;     // kept: keys above cut, and the first `ties` equal to it
  u64 ties;

  // weight of a value, 2^shift for the largest
  __device__ inline u64 weight(float v) const {
    const double z = (double(v) - top) * per;
    if (!(z > -double(shift) - 2.0)) return 0;  // rounds to 0 (z may be -inf)
    const double w = exp2(z);
    if (w < least) return 0;
    // 2^52 + n holds the whole number n in its low bits
    return __builtin_bit_cast(u64, ldexp(w, shift) + 0x1p52) & ((u64(1) << 52) - 1);
  }
  // f(index, element) over the row, kLane consecutive elements per lane
  template <class F>
  __device__ inline void each(F f) const {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    for (int64_t c = wave; c * kChunk < V; c += kWaves) {
      const int64_t i = c * kChunk + lane * kLane;
      chunk(c, i, f);
    }
  }
  template <class F>
  __device__ inline void chunk(int64_t c, int64_t i, F f) const {
    if (i + kLane <= V) {
      const Run<T> r = *reinterpret_cast<const Run<T>*>(x + i);
#pragma unroll
      for (int e = 0; e < kLane; ++e) f(c, i + e, r.v[e]);
    } else {
      for (int64_t k = i; k < V; ++k) f(c, k, x[k]);
    }
  }

  // The digit of a level in which the running sum from the largest digit down
  // reaches `target`: sh.found, and sh.before, the sum above it.  The total of
  // the level is returned first to `aim`, which says what the target is.
  template <bool MASS, class Aim>
  __device__ inline void place(Shared& sh, int bits, u64 above, Aim aim) {
    const int bins = 1 << bits, per_thread = bins > kThreads ? bins / kThreads : 1;
    u64 own = 0;
    const int first = bins - 1 - int(threadIdx.x) * per_thread;
    for (int k = 0; k < per_thread; ++k)
      if (first - k >= 0) own += MASS ? sh.mass[first - k] : u64(sh.count[first - k]);
    u64 total;
    u64 before = above + scan(own, sh, total);
    const u64 target = aim(above + total);
    if (before < target && target <= before + own) {
      for (int k = 0; k < per_thread; ++k) {
        const u64 n = MASS ? sh.mass[first - k] : u64(sh.count[first - k]);
        if (before + n >= target) {
          sh.found = first - k;
          sh.before = before;
          break;
        }
        before += n;
      }
    }
    __syncthreads();
  }

  // Moves the cut to where the kept counts (or weights) from the largest value
  // down reach aim(their total), and keeps as many ties there as that takes.
  template <bool MASS, class Aim>
  __device__ inline void select(Shared& sh, Aim aim) {
    uint32_t prefix = 0;
    u64 above = 0, target = 0;
    const u64 tie_weight = MASS && cut != 0 ? weight(O::of_key(cut)) : 0;
    for (int level = 0; level < O::kLevels; ++level) {
      const int shift_by = O::kShift[level], bits = O::kBits[level];
      const uint32_t mask = (1u << bits) - 1;
      __syncthreads();
      for (int b = threadIdx.x; b <= int(mask); b += kThreads) {
        if (MASS) sh.mass[b] = 0;
        else sh.count[b] = 0;
      }
      __syncthreads();
      each([&](int64_t, int64_t, T v) {
        const uint32_t key = O::key(v);
        if (level > 0 && (key >> (shift_by + bits)) != prefix) return;
        if (MASS) {
          if (key > cut)
            if (const u64 w = weight(O::value(v))) atomicAdd(&sh.mass[(key >> shift_by) & mask], w);
        } else {
          atomicAdd(&sh.count[(key >> shift_by) & mask], 1u);
        }
      });
      if (MASS && cut != 0 && threadIdx.x == 0 && (level == 0 || (cut >> (shift_by + bits)) == prefix))
        atomicAdd(&sh.mass[(cut >> shift_by) & mask], ties * tie_weight);
      __syncthreads();
      place<MASS>(sh, bits, above, [&](u64 total) {
        if (level == 0) target = aim(total);
        return target;
      });
      prefix = (prefix << bits) | uint32_t(sh.found);
      above = sh.before;
    }
    u64 need = target - above;
    if (MASS) {
      const u64 w = weight(O::of_key(prefix));
      need = w ? (need + w - 1) / w : 0;
    }
    ties = prefix == cut ? min(ties, need) : need;
    cut = prefix;
  }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs p) {
  using O = Order<T>;
  __shared__ Shared sh;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1);
  Row<T> r;
  r.x = static_cast<const T*>(p.x) + row * p.ld;
  r.V = p.V;
  r.shift = p.shift;
  const float u = p.u[row];
  float t = p.temperature ? p.temperature[row] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[row] : p.min_p_all;
  int64_t k = p.top_k ? p.top_k[row] : p.top_k_all;
  bool bad = !(t >= 0.f) || t == INFINITY || top_p != top_p || min_p != min_p || u != u;

  // the largest value, and whether there is a NaN
  if (threadIdx.x == 0) sh.top = 0, sh.bad = 0;
  __syncthreads();
  uint32_t top = 0, nan = 0;
  r.each([&](int64_t, int64_t, T v) {
    const float f = O::value(v);
    nan |= f != f;
    top = max(top, O::key(v));
  });
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    top = max(top, uint32_t(__shfl_xor(int(top), m, kWave)));
    nan |= uint32_t(__shfl_xor(int(nan), m, kWave));
  }
  if (lane == 0) {
    atomicMax(&sh.top, top);
    atomicOr(&sh.bad, nan);
  }
  __syncthreads();
  const float largest = O::of_key(sh.top);
  bad = bad || sh.bad || largest == INFINITY || largest == -INFINITY;
  if (bad) {  // the whole workgroup
    if (threadIdx.x == 0) {
      if (p.index_type == MK_S64) static_cast<int64_t*>(p.token)[row] = -1;
      else static_cast<int32_t*>(p.token)[row] = -1;
      if (p.logprob) p.logprob[row] = __builtin_nanf("");
    }
    return;
  }
  const bool greedy = t == 0.f;
  if (greedy) t = 1.f, k = 1;
  r.top = largest;
  r.per = 1.4426950408889634 / double(t);
  r.least = greedy ? 0.0 : min(double(min_p), 1.0);
  r.cut = 0;
  r.ties = 0;
  if (k == 1) {
    r.cut = sh.top;
    r.ties = 1;
  } else if (k > 0 && k < p.V) {
    r.template select<false>(sh, [&](u64) { return u64(k); });
  }
  if (!greedy && top_p < 1.f && k != 1) {
    // top-p counts what top-k kept, before min-p
    const double least = r.least;
    r.least = 0.0;
    r.template select<true>(sh, [&](u64 total) {
      const double aim = ceil(double(top_p) * double(total));
      return aim >= 1.0 ? min(u64(aim), total) : u64(1);
    });
    r.least = least;
  }

  // weights and ties of each chunk
  const u64 tie_weight = r.cut != 0 ? r.weight(O::of_key(r.cut)) : 0;
  const int chunks = int((p.V + kChunk - 1) / kChunk);
  __syncthreads();
  for (int b = threadIdx.x; b < chunks; b += kThreads) sh.mass[b] = 0, sh.count[b] = 0;
  __syncthreads();
  r.each([&](int64_t c, int64_t, T v) {
    const uint32_t key = O::key(v);
    if (key > r.cut) {
      if (const u64 w = r.weight(O::value(v))) atomicAdd(&sh.mass[c], w);
    } else if (key == r.cut) {
      atomicAdd(&sh.count[c], 1u);
    }
  });
  __syncthreads();
  // chunks in order: the ties that each still keeps, then the weights before it
  const int each = (chunks + kThreads - 1) / kThreads, first = int(threadIdx.x) * each;
  u64 own_ties = 0;
  for (int b = first; b < min(first + each, chunks); ++b) own_ties += sh.count[b];
  u64 all;
  u64 ties_before = scan(own_ties, sh, all);
  u64 own = 0, seen = ties_before;
  for (int b = first; b < min(first + each, chunks); ++b) {
    const u64 left = r.ties > seen ? r.ties - seen : 0;
    own += sh.mass[b] + min(left, u64(sh.count[b])) * tie_weight;
    seen += sh.count[b];
  }
  u64 total;
  u64 before = scan(own, sh, total);
  // the first token whose sum exceeds u total: whole numbers exceed its floor
  const double aim = floor(double(u) * double(total));
  const u64 goal = aim > 0.0 ? min(u64(min(aim, 0x1p63)), total - 1) : 0;
  if (before <= goal && goal < before + own) {
    seen = ties_before;
    for (int b = first; b < min(first + each, chunks); ++b) {
      const u64 left = r.ties > seen ? r.ties - seen : 0;
      const u64 n = sh.mass[b] + min(left, u64(sh.count[b])) * tie_weight;
      if (goal < before + n) {
        sh.found = b;
        sh.before = goal - before;
        sh.ties_before = uint32_t(min(seen, u64(0xffffffffu)));
        break;
      }
      before += n;
      seen += sh.count[b];
    }
  }
  __syncthreads();
  if (threadIdx.x >= kWave) return;

  // within the chunk, one wave
  const u64 rest = sh.before;
  const int64_t i0 = int64_t(sh.found) * kChunk + lane * kLane;
  T v[kLane];
  uint32_t mine = 0;
#pragma unroll
  for (int e = 0; e < kLane; ++e) {
    v[e] = r.x[min(i0 + e, p.V - 1)];
    mine += i0 + e < p.V && O::key(v[e]) == r.cut;
  }
  uint32_t tie = mine;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t o = uint32_t(__shfl_up(int(tie), d, kWave));
    if (lane >= d) tie += o;
  }
  tie += sh.ties_before - mine;  // ties before this lane's elements
  u64 w[kLane], sum = 0;
#pragma unroll
  for (int e = 0; e < kLane; ++e) {
    const uint32_t key = O::key(v[e]);
    w[e] = 0;
    if (i0 + e < p.V) {
      if (key > r.cut) w[e] = r.weight(O::value(v[e]));
      else if (key == r.cut && u64(tie++) < r.ties) w[e] = tie_weight;
    }
    sum += w[e];
  }
  u64 upto = sum;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const u64 o = shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  u64 at = upto - sum;
  if (at <= rest && rest < upto) {
    bool done = false;
#pragma unroll
    for (int e = 0; e < kLane; ++e) {
      at += w[e];
      if (!done && rest < at) {
        done = true;
        if (p.index_type == MK_S64) static_cast<int64_t*>(p.token)[row] = i0 + e;
        else static_cast<int32_t*>(p.token)[row] = int32_t(i0 + e);
        if (p.logprob) {
          const double z = (double(O::value(v[e])) - r.top) / double(t);
          p.logprob[row] = float(z - log(ldexp(double(total), -r.shift)));
        }
      }
    }
  }
}

}  // namespace
}  // namespace mk

using namespace mk;

extern "C" int mk_sample_rows(void* stream, int io_type, int64_t rows, int64_t vocab, const void* logits,
                              int64_t ld_logits, const float* u, const float* temperature, float temperature_all,
                              const int32_t* top_k, int top_k_all, const float* top_p, float top_p_all,
                              const float* min_p, float min_p_all, int index_type, void* tokens, float* logprobs) {
  clear_error();
  const std::string at = "mk_sample_rows: ";
  if (io_type != MK_BF16 && io_type != MK_F16 && io_type != MK_F32)
    return fail(MK_ERR_UNSUPPORTED, at + "io_type must be bf16/f16/f32");
  if (index_type != MK_S32 && index_type != MK_S64)
    return fail(MK_ERR_UNSUPPORTED, at + "index_type must be s32/s64");
  if (rows < 0 || vocab < 1) return fail(MK_ERR_INVALID, at + "need rows >= 0 and vocab >= 1");
  if (vocab > kMaxVocab) return fail(MK_ERR_UNSUPPORTED, at + "more than 2097152 tokens");
  if (rows >= int64_t(1) << 22) return fail(MK_ERR_UNSUPPORTED, at + "2^22 rows or more");
  if (!temperature && !(temperature_all >= 0.f && temperature_all < INFINITY))
    return fail(MK_ERR_INVALID, at + "temperature must be a number >= 0");
  if ((!top_p && top_p_all != top_p_all) || (!min_p && min_p_all != min_p_all))
    return fail(MK_ERR_INVALID, at + "top_p and min_p must be numbers");
  if (rows == 0) return MK_OK;
  if (!logits || !u || !tokens) return fail(MK_ERR_INVALID, at + "null pointer");
  if (ld_logits < 0) return fail(MK_ERR_INVALID, at + "negative row pitch");
  if (reinterpret_cast<uintptr_t>(logits) % dtype_bytes(io_type) ||
      reinterpret_cast<uintptr_t>(tokens) % dtype_bytes(index_type) || reinterpret_cast<uintptr_t>(u) % 4 ||
      reinterpret_cast<uintptr_t>(temperature) % 4 || reinterpret_cast<uintptr_t>(top_k) % 4 ||
      reinterpret_cast<uintptr_t>(top_p) % 4 || reinterpret_cast<uintptr_t>(min_p) % 4 ||
      reinterpret_cast<uintptr_t>(logprobs) % 4)
    return fail(MK_ERR_INVALID, at + "an operand is not aligned to its elements");
  int bits = 0;
  while ((int64_t(1) << bits) < vocab) ++bits;
  const SampleArgs a{logits, rows, vocab, ld_logits, u, temperature, top_p, min_p, top_k, temperature_all, top_p_all,
                     min_p_all, top_k_all, index_type, tokens, logprobs, std::min(51, 62 - bits)};
  const dim3 g{unsigned(rows)}, b{kThreads};
  hipStream_t s = as_stream(stream);
  if (io_type == MK_BF16) hipLaunchKernelGGL((sample_kernel<uint16_t>), g, b, 0, s, a);
  else if (io_type == MK_F16) hipLaunchKernelGGL((sample_kernel<F16>), g, b, 0, s, a);
  else hipLaunchKernelGGL((sample_kernel<float>), g, b, 0, s, a);
  return check_launch("mk_sample_rows");
}
