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
// row is sorted: in general the cut's value is found digit by digit from a histogram
// of counts (top-k) or of weights (top-p) over x's bits, taken as a whole number that
// orders as x does.
//
// Weights are whole numbers: w 2^s, with 2^z to 2^-33 of itself in 64 bits, s
// such that a row's sum stays below 2^63 (46 bits for 50257 tokens).  Their sums
// are exact, whatever order the atomics take, so a result is the same on every
// run, and errors of single weights cancel in them: for 50257 tokens a token is
// the one that real numbers give but for about one u in a million.
//
// A workgroup has a row and reads it two or three times (from L2 after the first):
//   for the largest value, which also is the whole of a greedy choice;
//   top-k: the k-th largest of the lanes' own maxima is below the row's k-th
//   largest value, so what is at or above it holds the first k and is seldom much
//   more: a second pass puts those tokens into a list in LDS;
//   top-p alone: a second pass for the weights by 64ths of a power of two, a third for
//   the list of the tokens from the cut's step up or, where they are many, for their
//   weights by 512 tokens;
//   min-p alone: a second pass for the list of what is above it;
//   no limit: a second pass for the weights of each 512 tokens.
// What remains happens on the list (12288 tokens; where it is longer the row is read
// again).  A list of at most 256 tokens is ranked by comparing each with each, and
// one wave does the rest; a longer one is summed by 512 tokens of the row, and one
// wave finds the token in its 512.
//
// Bound: one CU's work on a row.  50257 tokens, one row of bf16 / 256 rows of fp32,
// us: greedy 7.0 / 12.9 (the first pass: one CU takes in a line every 8 clocks),
// top-k 50 and top-p 0.9 15 / 24 (two passes and 20 barriers), top-p 0.95 39 / 49 and
// no limit 20 / 28 (an exponential in 64 bits for each token, 10 us a pass).  Loops are
// kept short on purpose: with the row in registers and each pass unrolled over it
// the same steps took 35, 59 and 34 us, waiting for instructions.
#include "mk_common.h"

#include <algorithm>
#include <string>
#include <type_traits>

namespace mk {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kBins = 4096;                 // 12 bits: a level of the histogram
constexpr int kLane = 8;                    // elements a lane takes at once
constexpr int kChunk = kLane * kWave;       // elements a wave takes at once
constexpr int kList = 12288;                // tokens of the list
constexpr int kFew = 256;                   // ... of one that is ranked by comparing each with each
constexpr int kStep = 512;                  // tokens of a step of find_top that are compared so
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
// No number and no infinity is 0.  Places past the row's end hold -inf, which
// weighs nothing.
template <typename T> struct Order;
template <> struct Order<float> {
  static constexpr int kLevels = 3;
  static constexpr int kShift[3] = {20, 10, 0}, kBits[3] = {12, 10, 10};
  static constexpr int kFine = 17;  // 64 steps from a power of two to the next
  static __device__ inline float none() { return -INFINITY; }
  static __device__ inline float value(float v) { return v; }
  static __device__ inline uint32_t key(float v) {
    uint32_t b = __builtin_bit_cast(uint32_t, v);
    b = b == 0x80000000u ? 0u : b;
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
  }
  static __device__ inline uint32_t nearest(float v) { return key(v); }
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
  static constexpr int kShift[2] = {4, 0}, kBits[2] = {12, 4}, kFine = 1;
  static __device__ inline uint16_t none() { return 0xff80u; }
  static __device__ inline float value(uint16_t v) { return bf16_to_f32(v); }
  static __device__ inline uint32_t key(uint16_t v) { return key16(v); }
  static __device__ inline uint32_t nearest(float v) { return key(f32_to_bf16(v)); }
  static __device__ inline float of_key(uint32_t k) { return bf16_to_f32(of_key16(k)); }
};
template <> struct Order<F16> {
  static constexpr int kLevels = 2;
  static constexpr int kShift[2] = {4, 0}, kBits[2] = {12, 4}, kFine = 4;
  static __device__ inline F16 none() { return F16{0xfc00u}; }
  static __device__ inline float value(F16 v) { return f16_to_f32(v.bits); }
  static __device__ inline uint32_t key(F16 v) { return key16(v.bits); }
  static __device__ inline uint32_t nearest(float v) { return key(F16{f32_to_f16(v)}); }
  static __device__ inline float of_key(uint32_t k) { return f16_to_f32(of_key16(k)); }
};

template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Run { T v[kLane]; };

// A list of at most 256 tokens, in the two orders that count.
struct Few {
  u64 weight[kFew];           // by rank
  uint32_t rank[4][kFew], place[4][kFew];  // partial counts of the tokens before one
  uint32_t rank_at[kFew], index_at[kFew];  // by place in the vocabulary
};

struct Shared {
  union {
    struct {
      u64 mass[kBins];        // a level's weights by digit; then the chunks' weights
      uint32_t count[kBins];  // a level's counts by digit; then the chunks' ties
    };
    Few few;
  };
  uint32_t key[kList], index[kList];  // the list
  u64 step_weight[kStep];            // of a step's tokens
  uint32_t step_key[kStep], step_chunk[kStep];
  u64 wave_sum[2][kWaves];
  uint32_t n;
  // what the one thread that found a place leaves for the others
  int found;
  u64 before;
  uint32_t ties_before, kept, in_step;
};

// v of the lane that a DPP control word names, 0 where there is none
template <int CTRL, int ROWS = 0xF>
__device__ inline uint32_t dpp(uint32_t v) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS = 0xF>
__device__ inline u64 dpp(u64 v) {
  return (u64(dpp<CTRL, ROWS>(uint32_t(v >> 32))) << 32) | dpp<CTRL, ROWS>(uint32_t(v));
}
// sum of v over the lanes up to and with this one: within rows of 16 (row_shr 1, 2,
// 4, 8), then the last lane of a row to the next row and of two rows to the next two
template <typename V>
__device__ inline V upto(V v) {
  v += dpp<0x111>(v);
  v += dpp<0x112>(v);
  v += dpp<0x114>(v);
  v += dpp<0x118>(v);
  v += dpp<0x142, 0xA>(v);
  v += dpp<0x143, 0xC>(v);
  return v;
}
__device__ inline u64 last_lane(u64 v) {
  return (u64(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v >> 32)), 63))) << 32) |
         uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), 63));
}

__device__ inline uint32_t wave_max(uint32_t v) {
  v = max(v, dpp<0x111>(v));
  v = max(v, dpp<0x112>(v));
  v = max(v, dpp<0x114>(v));
  v = max(v, dpp<0x118>(v));
  v = max(v, dpp<0x142, 0xA>(v));
  v = max(v, dpp<0x143, 0xC>(v));
  return uint32_t(__builtin_amdgcn_readlane(int(v), 63));
}

// Sum of v over the threads before this one (and all of them, in total), one
// barrier.  Two scans in a row take different `turn`s.
__device__ inline u64 scan(u64 v, Shared& sh, int turn, u64& total) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const u64 s = upto(v);
  if (lane == kWave - 1) sh.wave_sum[turn][wave] = s;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const u64 n = sh.wave_sum[turn][w];
    before += w < wave ? n : 0;
    all += n;
  }
  total = all;
  return before + s - v;
}

// sum over 16 lanes, in each of them: quad_perm [1,0,3,2] and [2,3,0,1], half_mirror, mirror
__device__ inline u64 row_sum(u64 v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  v += dpp<0x140>(v);
  return v;
}
// v of all lanes added to *to
__device__ inline void add_all(u64* to, u64 v) {
  v = row_sum(v);
  if (threadIdx.x % 16 == 0 && v) atomicAdd(to, v);
}

// The first sum that exceeds u times the total exceeds this: whole numbers
// exceed the product's floor.
__device__ inline u64 goal_of(float u, u64 total) {
  const double aim = floor(double(u) * double(total));
  return aim > 0.0 ? min(u64(min(aim, 0x1p63)), total - 1) : 0;
}
// The weight that a cut by top-p reaches: a rank is kept while less than this is
// before it.
__device__ inline u64 cut_of(float top_p, u64 all) {
  const double aim = ceil(double(top_p) * double(all));
  return aim >= 1.0 ? min(u64(aim), all) : u64(1);
}

template <typename T>
struct Row {
  using O = Order<T>;
  const T* x;
  int V;
  double top, per;  // the largest value; log2(e) / temperature
  int shift;
  uint32_t lightest;  // keys below it weigh nothing (masked tokens, above all)
  uint32_t cut;     // kept: keys above cut, and the first `ties` equal to it
  u64 ties;
  int listed;       // tokens in the list, -1: there is none
  bool whole;       // the list holds everything that is kept
  bool summed;      // sh.mass and sh.count hold what is kept of each chunk

  // log2 of a weight, at least -64 (weights below 2^-52 are 0)
  __device__ inline double log2_weight(float v) const { return max((double(v) - top) * per, -64.0); }
  // The weight, 2^shift for the largest.  2^z = 2^n 2^f, n the nearest whole number
  // (1.5 2^52 + n holds it in its low bits); 2^f is the polynomial through it at 8
  // Chebyshev points of [-1/2, 1/2], its constant made 1, 2^-33 of itself off;
  // 2^52 + w holds the rounded weight in its low bits.
  static constexpr u64 kRaw = u64(0x433) << 52;  // the bits of 2^52, which raw_weight is above its weight
  __device__ inline u64 raw_weight(double z) const {
    const double t = z + 0x1.8p52, f = z - (t - 0x1.8p52);
    const int n = int(uint32_t(__builtin_bit_cast(u64, t)));
    double e = 1.5303699001378845e-05;
    e = fma(e, f, 0.00015469729140704658);
    e = fma(e, f, 0.0013333478480888061);
    e = fma(e, f, 0.0096180256135980358);
    e = fma(e, f, 0.055504109063177154);
    e = fma(e, f, 0.24022651213495422);
    e = fma(e, f, 0.69314718055683411);
    e = fma(e, f, 1.0);
    return __builtin_bit_cast(u64, ldexp(e, shift + n) + 0x1p52);
  }
  __device__ inline u64 weight_of(double z) const { return raw_weight(z) - kRaw; }
  __device__ inline u64 weight(float v) const { return weight_of(log2_weight(v)); }

  // where load(i) takes its elements from
  __device__ inline int start(int i) const { return V >= kLane ? min(i, V - kLane) : i; }
  // The elements at i .. i + kLane - 1.  Where the row ends among or before them
  // they are the row's last kLane, with none() for those before i: which of its
  // chunk's elements a lane holds is all that counts.
  __device__ inline Run<T> load(int i) const {
    Run<T> r;
    if (V >= kLane) {
      const int from = start(i);
      r = *reinterpret_cast<const Run<T>*>(x + from);
      if (from < i) {
#pragma unroll
        for (int e = 0; e < kLane; ++e) r.v[e] = from + e < i ? O::none() : r.v[e];
      }
    } else {
      for (int e = 0; e < kLane; ++e) r.v[e] = i + e < V ? x[i + e] : O::none();
    }
    return r;
  }
  static __device__ inline int lane() { return threadIdx.x & (kWave - 1); }
  static __device__ inline int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }

  // f(chunk, its kLane elements of this lane) over the row, kAhead chunks loaded ahead
  template <int kAhead, class F>
  __device__ inline void each(F f) const {
    const int chunks = (V + kChunk - 1) / kChunk;
    auto at = [&](int c) { return load(c * kChunk + lane() * kLane); };
    Run<T> next[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) next[a] = at(wave() + kWaves * a);
#pragma unroll 1
    for (int c = wave(); c < chunks; c += kAhead * kWaves) {
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const Run<T> r = next[a];
        next[a] = at(c + kWaves * (a + kAhead));
        if (c + kWaves * a < chunks) f(c + kWaves * a, r);
      }
    }
  }
  // f(chunk, key) over the list, or over the row
  template <class F>
  __device__ inline void over(const Shared& sh, F f) const {
    if (listed >= 0) {
#pragma unroll 1
      for (int e = threadIdx.x; e < listed; e += kThreads) f(int(sh.index[e] / kChunk), sh.key[e]);
    } else {
      each<1>([&](int c, const Run<T>& r) {
#pragma unroll
        for (int e = 0; e < kLane; ++e) f(c, O::key(r.v[e]));
      });
    }
  }
  // Puts the elements that the lanes take, a bit each, into the list: one atomic a
  // wave (one a lane, all on one address, took 7 clocks each; 18 us for the list of
  // 5000 of 50257 tokens).
  __device__ inline void append(Shared& sh, int c, const Run<T>& r, uint32_t mine) const {
    if (!__ballot(mine != 0)) return;
    const uint32_t n = uint32_t(__popc(mine)), s = upto(n);
    uint32_t base = 0;
    if (lane() == kWave - 1) base = atomicAdd(&sh.n, s);
    uint32_t at = uint32_t(__builtin_amdgcn_readlane(int(base), kWave - 1)) + s - n;
    if (at > uint32_t(kList - kLane)) return;
    const uint32_t i = uint32_t(start(c * kChunk + lane() * kLane));
#pragma unroll
    for (int e = 0; e < kLane; ++e)
      if (mine >> e & 1) {
        sh.key[at] = O::key(r.v[e]);
        sh.index[at] = i + e;
        ++at;
      }
  }
  // whether what was put into it fits, behind a barrier
  __device__ inline bool end_list(const Shared& sh) {
    __syncthreads();
    listed = sh.n <= uint32_t(kList - kLane) ? int(sh.n) : -1;
    return listed >= 0;
  }
  // The list of the tokens from value lo to hi; whether they fit.  sh.n is 0 before it.
  __device__ inline bool make_list(Shared& sh, float lo, float hi) {
    each<3>([&](int c, const Run<T>& r) {
      uint32_t mine = 0;
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        const float v = O::value(r.v[e]);
        mine |= uint32_t(v >= lo && v <= hi) << e;
      }
      append(sh, c, r, mine);
    });
    return end_list(sh);
  }

  // The digit of a level in which the running sum from the largest digit down
  // (`above` before the level) reaches aim(sum of all): left in sh.found, and the
  // sum above it in sh.before.
  template <bool MASS, class Aim>
  __device__ inline void place(Shared& sh, int bits, u64 above, int turn, Aim aim) const {
    constexpr int kPer = kBins / kThreads;
    const int bins = 1 << bits, per_thread = bins > kThreads ? kPer : 1;
    const int first = bins - 1 - int(threadIdx.x) * per_thread;
    u64 n[kPer], own = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const bool in = k < per_thread && first - k >= 0;
      n[k] = in ? (MASS ? sh.mass[in ? first - k : 0] : u64(sh.count[in ? first - k : 0])) : 0;
      own += n[k];
    }
    u64 total;
    u64 before = above + scan(own, sh, turn, total);
    const u64 target = aim(above + total);
    if (before < target && target <= before + own) {
      int at = 0;
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        if (at == k && before + n[k] < target) before += n[k], ++at;
      sh.found = first - at;
      sh.before = before;
    }
    __syncthreads();
  }
  // an empty level and list, behind a barrier
  template <bool MASS>
  __device__ inline void clear(Shared& sh, int n) const {
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    for (int b = threadIdx.x; b < n; b += kThreads) {
      if (MASS) sh.mass[b] = 0;
      else sh.count[b] = 0;
    }
    __syncthreads();
  }

  // which 64th of a power of two below the largest a weight is
  static __device__ inline int step_of(double z) { return min(int(-64.0 * z), kBins - 1); }
  // Top-p of a row without a top-k: its weights by their logarithm, in steps of
  // 1 / 64, say in which step the cut is, and about how many tokens are above it.  Few
  // are in the step itself, and are compared with each other.  Where little is kept, a
  // list of the tokens from that step up holds all of it; else another pass sums the
  // weights above the step by chunk and puts the step's own tokens aside.  Returns the
  // weight that the cut reaches where the cut is still to be found: on a short list, or
  // where many are in the step.  us, list / pass by tokens kept: 5000 of 50257 39.1 /
  // 40.3, 13000 57.7 (more than the list holds) / 42; 2000 of 32000 64.5 / 64.8, 7000
  // 78 / 68; 8000 of 128000 77 / 89.
  __device__ inline u64 find_top(Shared& sh, float top_p, u64 least) {
    clear<true>(sh, kBins);
    // the last 64 steps weigh nothing: a lane's own there for what is masked (all on one
    // address: 58 us, 25 so, for 50257 tokens of which 10 are left)
    const int farthest = kBins - 1 - lane();
    each<1>([&](int, const Run<T>& r) {
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        const double z = log2_weight(O::value(r.v[e]));
        atomicAdd(&sh.mass[kBins - 1 - min(int(-64.0 * z), farthest)], weight_of(z));
      }
    });
    __syncthreads();
    // each thread's steps from the largest weight down: their weights, and how many
    // tokens that is (the weight over one of the step's)
    constexpr int kPer = kBins / kThreads;
    u64 mass[kPer], own = 0, all;
    uint32_t tokens[kPer], some = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int j = int(threadIdx.x) * kPer + k;
      own += mass[k] = sh.mass[kBins - 1 - j];
      some += tokens[k] = uint32_t(float(mass[k]) * exp2f(float(j) / 64.f - float(shift)) + 0.5f);
    }
    some = upto(some) - some;
    if (lane() == kWave - 1) sh.wave_sum[1][wave()] = some + tokens[0] + tokens[1] + tokens[2] + tokens[3];
    u64 above = scan(own, sh, 0, all);
    const u64 target = cut_of(top_p, all);
    if (above < target && target <= above + own) {
      for (int w = 0; w < int(threadIdx.x) / kWave; ++w) some += uint32_t(sh.wave_sum[1][w]);
      int at = 0;
      uint32_t in_step = 0;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        if (at == k) some += tokens[k], in_step = tokens[k];
        if (at == k && above + mass[k] < target) above += mass[k], ++at;
      }
      sh.found = int(threadIdx.x) * kPer + at;
      sh.before = above;
      sh.kept = some;
      sh.in_step = in_step;
    }
    __syncthreads();
    const int step = sh.found;
    const uint32_t kept = sh.kept;
    const bool many = sh.in_step > uint32_t(kStep);  // at least as many are in the step
    above = sh.before;
    clear<true>(sh, (V + kChunk - 1) / kChunk);
    clear<false>(sh, (V + kChunk - 1) / kChunk);
    if (kept <= uint32_t(min(V / 8, kList - kList / 32))) {
      // a little past the step's end: what is past it does no harm on the list
      const float end = float(top - (step + 1) / 64.0 / per);
      whole = make_list(sh, end - fabsf(end) * 0x1p-22f - float(fabs(top)) * 0x1p-40f, INFINITY);
      if (whole && listed <= kFew) return target;
      if (!whole || many) return target;
      __syncthreads();  // everyone has read the list's length
      if (threadIdx.x == 0) sh.n = 0;
      __syncthreads();
      over(sh, [&](int c, uint32_t key) {
        const double z = log2_weight(O::of_key(key));
        if (step_of(z) == step) put_aside(sh, c, key, weight_of(z));
      });
    } else {
      if (many) return target;
      const double from = -(step + 1) / 64.0, to = -step / 64.0;  // z in (from, to]
      const u64 low = kRaw + least;
      each<1>([&](int c, const Run<T>& r) {
        u64 own = 0;
#pragma unroll
        for (int e = 0; e < kLane; ++e) {
          const float v = O::value(r.v[e]);
          const double z = log2_weight(v);
          const u64 w = raw_weight(z);
          own += z > to && w >= low ? w : kRaw;
          if (z > from && z <= to) put_aside(sh, c, O::key(r.v[e]), w - kRaw);
        }
        add_all(&sh.mass[c], own - kLane * kRaw);
      });
    }
    __syncthreads();
    const int n = int(sh.n);
    if (n > kStep) return target;
    if (int(threadIdx.x) < n) {
      const uint32_t key = sh.step_key[threadIdx.x];
      const u64 w = sh.step_weight[threadIdx.x];
      u64 same = 0;
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const uint32_t k = sh.step_key[i];
        const u64 v = sh.step_weight[i];
        above += k > key ? v : 0;
        same += k == key ? v : 0;
      }
      if (above < target && target <= above + same) {  // the same for all of one key
        sh.found = int(key);
        sh.before = (target - above + w - 1) / w;
      }
    }
    __syncthreads();
    cut = uint32_t(sh.found);
    ties = sh.before;
    summed = !whole;
    if (summed && int(threadIdx.x) < n) {
      const uint32_t key = sh.step_key[threadIdx.x], c = sh.step_chunk[threadIdx.x];
      const u64 w = sh.step_weight[threadIdx.x];
      if (key > cut && w >= least) atomicAdd(&sh.mass[c], w);
      if (key == cut) atomicAdd(&sh.count[c], 1u);
    }
    return 0;
  }
  // one of the step's tokens
  __device__ inline void put_aside(Shared& sh, int c, uint32_t key, u64 w) const {
    const uint32_t at = atomicAdd(&sh.n, 1u);
    if (at >= uint32_t(kStep)) return;
    sh.step_key[at] = key;
    sh.step_chunk[at] = uint32_t(c);
    sh.step_weight[at] = w;
  }

  // Moves the cut to where the kept counts (or weights) from the largest value
  // down reach aim(their total), and keeps as many ties there as that takes.
  template <bool MASS, class Aim>
  __device__ inline void select(Shared& sh, Aim aim) {
    uint32_t prefix = 0;
    u64 above = 0, target = 0;
    const u64 tie_weight = MASS && cut != 0 ? weight(O::of_key(cut)) : 0;
#pragma unroll 1
    for (int level = 0; level < O::kLevels; ++level) {
      const int by = O::kShift[level], bits = O::kBits[level];
      const uint32_t mask = (1u << bits) - 1;
      clear<MASS>(sh, int(mask) + 1);
      over(sh, [&](int, uint32_t key) {
        if (key < lightest || (MASS && key <= cut) || (level > 0 && (key >> (by + bits)) != prefix)) return;
        if (MASS) atomicAdd(&sh.mass[(key >> by) & mask], weight(O::of_key(key)));
        else atomicAdd(&sh.count[(key >> by) & mask], 1u);
      });
      if (MASS && cut != 0 && threadIdx.x == 0 && (level == 0 || (cut >> (by + bits)) == prefix))
        atomicAdd(&sh.mass[(cut >> by) & mask], ties * tie_weight);
      __syncthreads();
      place<MASS>(sh, bits, above, level & 1, [&](u64 total) {
        if (level == 0) target = aim(total);
        return target;
      });
      prefix = (prefix << bits) | uint32_t(sh.found);
      above = sh.before;
      // the other digits on the tokens of this one, with those above where they fit
      if (level == 0 && listed < 0) {
        const uint32_t least = prefix << by, width = (1u << by) - 1;
        for (int only = 0; only < 2 && listed < 0; ++only) {
          clear<MASS>(sh, 0);
          const float from = O::of_key(max(least, O::key(O::none()))), to = only ? O::of_key(least + width) : INFINITY;
          whole = make_list(sh, from, to) && !only;
        }
      }
    }
    if (!whole) listed = -1;
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
__device__ inline void put(const SampleArgs& p, const Row<T>& r, int64_t row, float t, int i, float x, u64 total) {
  if (p.index_type == MK_S64) static_cast<int64_t*>(p.token)[row] = i;
  else static_cast<int32_t*>(p.token)[row] = i;
  if (p.logprob)
    p.logprob[row] = float((double(x) - r.top) / double(t) - log(ldexp(double(total), -p.shift)));
}

// The token of a list of at most kFew that holds all that is kept: the first k
// ranks of it, cut at `target` or by top-p, and by min-p.  Four threads compare a
// token with a quarter of the others each; then one wave sums in both orders.
template <typename T>
__device__ inline void take_few(const SampleArgs& p, const Row<T>& r, Shared& sh, int64_t row, float u, float t,
                                int64_t k, u64 target, float top_p, u64 least) {
  const int n = r.listed, j = threadIdx.x % kFew, part = threadIdx.x / kFew;
  const int q = (n + 3) / 4, lo = part * q, hi = min(lo + q, n);
  Few& few = sh.few;
  uint32_t key = 0, index = 0;
  if (j < n) {
    key = sh.key[j];
    index = sh.index[j];
    uint32_t rank = 0, place = 0;
#pragma unroll 4
    for (int i = lo; i < hi; ++i) {
      const uint32_t ki = sh.key[i], ii = sh.index[i];
      rank += ki > key || (ki == key && ii < index);
      place += ii < index;
    }
    few.rank[part][j] = rank;
    few.place[part][j] = place;
  }
  __syncthreads();
  if (part == 0 && j < n) {
    const uint32_t rank = few.rank[0][j] + few.rank[1][j] + few.rank[2][j] + few.rank[3][j];
    const uint32_t place = few.place[0][j] + few.place[1][j] + few.place[2][j] + few.place[3][j];
    few.weight[rank] = r.weight(Order<T>::of_key(key));
    few.rank_at[place] = rank;
    few.index_at[place] = index;
  }
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  constexpr int kPer = kFew / kWave;
  const int first = threadIdx.x * kPer;
  u64 w[kPer], sum = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) sum += w[e] = first + e < n && first + e < k ? few.weight[first + e] : 0;
  u64 s = upto(sum);
  const u64 all = last_lane(s), limit = target ? target : top_p < 1.f ? cut_of(top_p, all) : ~u64(0);
  uint32_t mine = 0;  // kept ranks: a run from the first on
  s -= sum;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    mine += w[e] != 0 && s < limit && w[e] >= least;
    s += w[e];
  }
  const uint32_t kept = uint32_t(__builtin_amdgcn_readlane(int(upto(mine)), 63));
  sum = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const uint32_t rank = first + e < n ? few.rank_at[first + e] : kept;
    sum += w[e] = rank < kept ? few.weight[rank] : 0;
  }
  s = upto(sum);
  const u64 total = last_lane(s), goal = goal_of(u, total);
  s -= sum;
  if (s <= goal && goal < s + sum) {
    int at = -1;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      s += w[e];
      if (at < 0 && goal < s) at = first + e;
    }
    const int i = int(few.index_at[at]);
    put(p, r, row, t, i, Order<T>::value(r.x[i]), total);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs p) {
  using O = Order<T>;
  __shared__ Shared sh;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1);
  Row<T> r;
  r.x = static_cast<const T*>(p.x) + row * p.ld;
  r.V = int(p.V);
  r.shift = p.shift;
  r.listed = -1;
  r.whole = r.summed = false;
  const float u = p.u[row];
  float t = p.temperature ? p.temperature[row] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[row] : p.min_p_all;
  int64_t k = p.top_k ? p.top_k[row] : p.top_k_all;
  bool bad = !(t >= 0.f) || t == INFINITY || top_p != top_p || min_p != min_p || u != u;
  if (threadIdx.x == 0) sh.n = 0;
  sh.count[threadIdx.x] = 0;

  // The largest value, of this lane's and of all, with the first chunk that holds
  // it; and whether there is a NaN.
  float lane_top = -INFINITY;
  bool nan = false;
  int mine_at = 0;
  r.template each<3>([&](int c, const Run<T>& v) {
    float m = O::value(v.v[0]);
    nan |= m != m;
#pragma unroll
    for (int e = 1; e < kLane; ++e) {
      const float f = O::value(v.v[e]);
      nan |= f != f;
      m = f > m ? f : m;
    }
    if (m > lane_top) lane_top = m, mine_at = c;
  });
  const uint32_t mine = O::nearest(lane_top);  // its key
  const uint32_t wave_top = __ballot(nan) ? 0xffffffffu : wave_max(mine);
  const uint32_t wave_at = wave_max(mine == wave_top ? uint32_t(~mine_at) : 0u);
  if (lane == 0) sh.wave_sum[0][threadIdx.x / kWave] = (u64(wave_top) << 32) | wave_at;
  __syncthreads();
  u64 best = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) best = max(best, sh.wave_sum[0][w]);
  const uint32_t top_key = uint32_t(best >> 32);
  const float largest = O::of_key(top_key);
  bad = bad || top_key == 0xffffffffu || largest == INFINITY || largest == -INFINITY;
  if (bad) {  // the whole workgroup
    if (threadIdx.x == 0) {
      if (p.index_type == MK_S64) static_cast<int64_t*>(p.token)[row] = -1;
      else static_cast<int32_t*>(p.token)[row] = -1;
      if (p.logprob) p.logprob[row] = __builtin_nanf("");
    }
    return;
  }
  if (t == 0.f) t = 1.f, k = 1;  // (one token is kept whatever the others say)
  r.top = largest;
  r.per = 1.4426950408889634 / double(t);
  r.lightest = max(O::nearest(float(r.top - double(p.shift + 2) / r.per)) - 1, O::key(O::none()) + 1);
  r.cut = 0;
  r.ties = 0;
  u64 total, rest;
  int chunk;
  uint32_t ties_before;
  // min-p as a weight
  const u64 least = u64(ceil(ldexp(max(0.0, min(double(min_p), 1.0)), p.shift)));
  u64 tie_weight;
  if (k == 1) {
    r.cut = top_key;
    r.ties = 1;
    tie_weight = total = u64(1) << p.shift;
    rest = 0;
    chunk = int(~uint32_t(best));
    ties_before = 0;
  } else {
    if (k > 0 && k < r.V) {
      // k lanes have a maximum at most so many steps below the top: so is the
      // row's k-th largest value.  Each wave finds the step for itself.
      const int lanes = min((r.V + kLane - 1) / kLane, kThreads);  // that hold anything
      if (k <= lanes / 2) {
        // (step b at (b % 16) 64 + b / 16: lane l reads steps 16 l .. side by side)
        constexpr int kPer = kThreads / kWave;
        const uint32_t my_step = min((top_key - mine) >> O::kFine, uint32_t(kThreads - 1));
        if (mine) atomicAdd(&sh.count[my_step % kPer * kWave + my_step / kPer], 1u);
        __syncthreads();
        uint32_t n[kPer], own = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) own += n[e] = sh.count[kWave * e + lane];
        uint32_t s = upto(own) - own;
        const u64 here = __ballot(s < k && k <= s + own);
        uint32_t step = uint32_t(kPer * lane);
#pragma unroll
        for (int e = 0; e < kPer - 1; ++e)
          if (step == uint32_t(kPer * lane + e) && s + n[e] < k) s += n[e], ++step;
        step = uint32_t(__builtin_amdgcn_readlane(int(step), __ffsll(here) - 1));
        // where the steps end before the k-th: all that weighs anything (10 of 50257 tokens
        // left, top-k 50: 14.5 us, 139 with the masked ones counted)
        uint32_t bound = r.lightest;
        if (step < uint32_t(kThreads - 1)) bound = max(bound, top_key - min(((step + 1) << O::kFine) - 1, top_key));
        r.whole = r.make_list(sh, O::of_key(bound), INFINITY);
      }
      if (!r.whole || r.listed > kFew) r.template select<false>(sh, [&](u64 all) { return min(u64(k), all); });
    }
    const bool few_k = r.whole && r.listed <= kFew && r.cut == 0;  // top-k is still to be taken
    u64 target = 0;
    if (top_p < 1.f && !few_k) {  // of what top-k kept, before min-p
      const bool top_k = r.cut != 0;
      if (!top_k) target = r.find_top(sh, top_p, least);
      if (top_k || (target != 0 && !(r.whole && r.listed <= kFew)))
        r.template select<true>(sh, [&](u64 all) { return target ? target : cut_of(top_p, all); });
    }
    if (r.cut == 0 && r.listed < 0 && least > 0) {  // min-p alone: what may be above it, a little below it
      r.template clear<true>(sh, 0);
      const double lo = r.top + double(log2f(fminf(min_p, 1.f))) / r.per;
      r.whole = r.make_list(sh, float(lo - (fabs(lo) + fabs(r.top)) * 0x1p-20 - 0x1p-10 / r.per), INFINITY);
    }
    if (r.whole && r.listed <= kFew && r.cut == 0)
      return take_few(p, r, sh, row, u, t, few_k ? k : int64_t(kFew), target, top_p, least);
    // weights and ties of each chunk
    tie_weight = r.cut != 0 ? r.weight(O::of_key(r.cut)) : 0;
    if (tie_weight < least) tie_weight = 0;
    const int chunks = (r.V + kChunk - 1) / kChunk;
    if (!r.summed) {
      r.template clear<true>(sh, chunks);
      if (r.cut != 0) r.template clear<false>(sh, chunks);
    }
    if (r.summed) {
      // by find_top
    } else if (r.listed >= 0) {
      r.over(sh, [&](int c, uint32_t key) {
        if (key > r.cut) {
          const u64 w = r.weight(O::of_key(key));
          if (w >= least) atomicAdd(&sh.mass[c], w);
        } else if (key == r.cut) {
          atomicAdd(&sh.count[c], 1u);
        }
      });
    } else if (r.cut == 0 && least == 0) {
      r.template each<1>([&](int c, const Run<T>& v) {
        u64 own = 0;
#pragma unroll
        for (int e = 0; e < kLane; ++e) own += r.raw_weight(r.log2_weight(O::value(v.v[e])));
        add_all(&sh.mass[c], own - kLane * r.kRaw);
      });
    } else {
      r.template each<1>([&](int c, const Run<T>& v) {
        u64 own = 0;
        uint32_t ties = 0;
#pragma unroll
        for (int e = 0; e < kLane; ++e) {
          const uint32_t key = O::key(v.v[e]);
          const u64 w = r.weight(O::value(v.v[e]));
          own += key > r.cut && w >= least ? w : 0;
          ties += key == r.cut;
        }
        add_all(&sh.mass[c], own);
        if (ties) atomicAdd(&sh.count[c], ties);
      });
    }
    __syncthreads();
    // chunks in order: the ties that each still keeps, then the weights before it
    const int each = (chunks + kThreads - 1) / kThreads, first = int(threadIdx.x) * each;
    const int last = min(first + each, chunks);
    u64 before_ties = 0;
    if (r.cut != 0) {
      u64 own_ties = 0, all;
      for (int b = first; b < last; ++b) own_ties += sh.count[b];
      before_ties = scan(own_ties, sh, 0, all);
    }
    u64 own = 0, seen = before_ties;
    auto kept = [&](int b) {  // a chunk's weight, `seen` ties before it
      if (r.cut == 0) return sh.mass[b];
      const u64 n = sh.count[b], left = r.ties > seen ? r.ties - seen : 0;
      seen += n;
      return sh.mass[b] + min(left, n) * tie_weight;
    };
    for (int b = first; b < last; ++b) own += kept(b);
    u64 before = scan(own, sh, 1, total);
    const u64 goal = goal_of(u, total);
    if (before <= goal && goal < before + own) {
      seen = before_ties;
      for (int b = first; b < last; ++b) {
        const u64 ties = seen, n = kept(b);
        if (goal < before + n) {
          sh.found = b;
          sh.before = goal - before;
          sh.ties_before = uint32_t(ties);
          break;
        }
        before += n;
      }
    }
    __syncthreads();
    rest = sh.before;
    chunk = sh.found;
    ties_before = sh.ties_before;
  }
  if (threadIdx.x >= kWave) return;

  // within the chunk, one wave
  const int i0 = chunk * kChunk + lane * kLane;
  const int from = r.start(i0);  // places before i0 hold -inf
  const Run<T> v = r.load(i0);
  uint32_t equal = 0;
#pragma unroll
  for (int e = 0; e < kLane; ++e) equal += O::key(v.v[e]) == r.cut;
  uint32_t tie = ties_before + upto(equal) - equal;  // before this lane's elements
  u64 w[kLane], sum = 0;
#pragma unroll
  for (int e = 0; e < kLane; ++e) {
    const uint32_t key = O::key(v.v[e]);
    w[e] = r.weight(O::value(v.v[e]));
    w[e] = key > r.cut && w[e] >= least ? w[e] : 0;
    if (key == r.cut) w[e] = u64(tie++) < r.ties ? tie_weight : 0;
    sum += w[e];
  }
  const u64 s = upto(sum);
  u64 at = s - sum;
  if (at <= rest && rest < s) {
    int e_at = kLane;
    float x_at = 0.f;
#pragma unroll
    for (int e = 0; e < kLane; ++e) {
      at += w[e];
      if (e_at == kLane && rest < at) e_at = e, x_at = O::value(v.v[e]);
    }
    put(p, r, row, t, from + e_at, x_at, total);
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
  if (io_type != MK_BF16 && io_type != MK_F16 && io_type != MK_F32)
    return fail(MK_ERR_UNSUPPORTED, "mk_sample_rows: io_type must be bf16/f16/f32");
  if (index_type != MK_S32 && index_type != MK_S64)
    return fail(MK_ERR_UNSUPPORTED, "mk_sample_rows: index_type must be s32/s64");
  if (rows < 0 || vocab < 1) return fail(MK_ERR_INVALID, "mk_sample_rows: need rows >= 0 and vocab >= 1");
  if (vocab > kMaxVocab) return fail(MK_ERR_UNSUPPORTED, "mk_sample_rows: more than 2097152 tokens");
  if (rows >= int64_t(1) << 22) return fail(MK_ERR_UNSUPPORTED, "mk_sample_rows: 2^22 rows or more");
  if (!temperature && !(temperature_all >= 0.f && temperature_all < INFINITY))
    return fail(MK_ERR_INVALID, "mk_sample_rows: temperature must be a number >= 0");
  if ((!top_p && top_p_all != top_p_all) || (!min_p && min_p_all != min_p_all))
    return fail(MK_ERR_INVALID, "mk_sample_rows: top_p and min_p must be numbers");
  if (rows == 0) return MK_OK;
  if (!logits || !u || !tokens) return fail(MK_ERR_INVALID, "mk_sample_rows: null pointer");
  if (ld_logits < 0) return fail(MK_ERR_INVALID, "mk_sample_rows: negative row pitch");
  if (reinterpret_cast<uintptr_t>(logits) % dtype_bytes(io_type) ||
      reinterpret_cast<uintptr_t>(tokens) % dtype_bytes(index_type) || reinterpret_cast<uintptr_t>(u) % 4 ||
      reinterpret_cast<uintptr_t>(temperature) % 4 || reinterpret_cast<uintptr_t>(top_k) % 4 ||
      reinterpret_cast<uintptr_t>(top_p) % 4 || reinterpret_cast<uintptr_t>(min_p) % 4 ||
      reinterpret_cast<uintptr_t>(logprobs) % 4)
    return fail(MK_ERR_INVALID, "mk_sample_rows: an operand is not aligned to its elements");
  int bits = 0;
  while ((int64_t(1) << bits) < vocab) ++bits;
  const SampleArgs a{logits, rows, vocab, ld_logits, u, temperature, top_p, min_p, top_k, temperature_all, top_p_all,
                     min_p_all, top_k_all, index_type, tokens, logprobs, std::min(51, 62 - bits)};
  hipStream_t s = as_stream(stream);
  const dim3 g{unsigned(rows)}, b{kThreads};
  if (io_type == MK_BF16) hipLaunchKernelGGL((sample_kernel<uint16_t>), g, b, 0, s, a);
  else if (io_type == MK_F16) hipLaunchKernelGGL((sample_kernel<F16>), g, b, 0, s, a);
  else hipLaunchKernelGGL((sample_kernel<float>), g, b, 0, s, a);
  return check_launch("mk_sample_rows");
}
