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
#include "attn_common.h"

#include <algorithm>
#include <string>

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
  int c_type, epilogue;
};

// one value of C from its sum
__device__ inline float finish(const Int8Gemm& p, int sum, float sa, int64_t n) {
  float v = float(sum) * sa * p.b_scale[n];
  if ((p.epilogue & 3) != 0) v += load_as_f32(p.bias, n, (p.epilogue & 4) ? int(MK_F32) : p.c_type);
  if ((p.epilogue & 3) == 2) v = v < 0.f ? 0.f : v;  // keeps a NaN
  return v;
}

// 16 bytes from any address
struct __attribute__((packed, aligned(1))) Any16 { u32x4_t v; };

// Any shape, pitch and alignment: 64 x 64 tiles, 4 waves of 32 x 32, k 64 deep
// through registers and LDS.
__global__ __launch_bounds__(256) void gemm_int8_any_kernel(const Int8Gemm p) {
  constexpr int T = 64, BK = 64, kPitch = BK + 16;  // rows 80 bytes apart: 16 lanes of a read on different banks
  __shared__ __attribute__((aligned(16))) int8_t lds[2][T * kPitch];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 31, g = lane >> 5;
  const int64_t m0 = int64_t(blockIdx.x / p.tiles_n) * T, n0 = int64_t(blockIdx.x % p.tiles_n) * T;
  // this thread's chunk of either tile; rows past the operand repeat its last
  const int row = threadIdx.x / 4, at = 16 * (threadIdx.x % 4);
  const int8_t* src[2] = {p.A + std::min<int64_t>(m0 + row, p.M - 1) * p.lda + at,
                          p.B + std::min<int64_t>(n0 + row, p.N - 1) * p.ldb + at};
  i32x16_t acc = {};
  for (int64_t k0 = 0; k0 < p.K; k0 += BK) {
    u32x4_t v[2];
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const int64_t left = p.K - k0 - at;
      if (left >= 16) {
        v[o] = reinterpret_cast<const Any16*>(src[o] + k0)->v;
      } else {
        uint8_t b[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) b[e] = e < left ? uint8_t(src[o][k0 + e]) : 0;
        __builtin_memcpy(&v[o], b, 16);
      }
    }
    __syncthreads();
#pragma unroll
    for (int o = 0; o < 2; ++o) *reinterpret_cast<u32x4_t*>(&lds[o][row * kPitch + at]) = v[o];
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      const i32x4_t a = *reinterpret_cast<const i32x4_t*>(&lds[0][(32 * (wave / 2) + c) * kPitch + 32 * ks + 16 * g]);
      const i32x4_t b = *reinterpret_cast<const i32x4_t*>(&lds[1][(32 * (wave % 2) + c) * kPitch + 32 * ks + 16 * g]);
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(b, a, acc, 0, 0, 0);
    }
  }
  const int64_t m = m0 + 32 * (wave / 2) + c;
  if (m >= p.M) return;
  const float sa = p.a_scale[m];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t n = n0 + 32 * (wave % 2) + 8 * (r / 4) + 4 * g + r % 4;
    if (n < p.N) store_from_f32(p.C, m * p.ldc + n, p.c_type, finish(p, acc[r], sa, n));
  }
}

}  // namespace
}  // namespace mk

using namespace mk;

extern "C" int mk_gemm_int8(void* stream, int c_type, int64_t M, int64_t N, int64_t K, const int8_t* A, int64_t a_ms,
                            const float* a_scale, const int8_t* B, int64_t b_ns, const float* b_scale, void* C,
                            int64_t c_ms, const void* bias, int epilogue) {
  clear_error();
  const std::string at = "mk_gemm_int8: ";
  if (c_type != MK_BF16 && c_type != MK_F16 && c_type != MK_F32)
    return fail(MK_ERR_UNSUPPORTED, at + "c_type must be bf16/f16/f32");
  if (M < 0 || N < 0 || K < 0) return fail(MK_ERR_INVALID, at + "negative shape");
  if (K > kMaxK) return fail(MK_ERR_UNSUPPORTED, at + "K past 131071: the 32-bit sums could overflow");
  // a workgroup of 256 threads per 64 x 64 tile, below HIP's 2^32 threads
  if (M >> 30 || N >> 30 || (M + 63) / 64 * ((N + 63) / 64) >= int64_t(1) << 24)
    return fail(MK_ERR_UNSUPPORTED, at + "2^24 or more tiles of 64 x 64");
  const int epi = epilogue & 3;
  if (epilogue < 0 || epilogue > 6 || epi == 3 || (epilogue == 4))
    return fail(MK_ERR_INVALID, at + "epilogue must be 0, 1, 2, 5 or 6");
  if (M == 0 || N == 0) return MK_OK;
  if ((K > 0 && (!A || !B)) || !a_scale || !b_scale || !C || (epi != 0 && !bias))
    return fail(MK_ERR_INVALID, at + "null pointer");
  if ((M > 1 && (a_ms < 0 || c_ms < N)) || (N > 1 && b_ns < 0)) return fail(MK_ERR_INVALID, at + "bad stride");
  if (reinterpret_cast<uintptr_t>(C) % dtype_bytes(c_type) || reinterpret_cast<uintptr_t>(a_scale) % 4 ||
      reinterpret_cast<uintptr_t>(b_scale) % 4 ||
      (epi != 0 && reinterpret_cast<uintptr_t>(bias) % ((epilogue & 4) ? 4 : dtype_bytes(c_type))))
    return fail(MK_ERR_INVALID, at + "an operand is not aligned to its elements");
  Int8Gemm a{A, B, a_scale, b_scale, C, bias, M, N, K, a_ms, b_ns, c_ms, int((M + 63) / 64), int((N + 63) / 64),
             c_type, epilogue};
  hipLaunchKernelGGL(gemm_int8_any_kernel, dim3(unsigned(int64_t(a.tiles_m) * a.tiles_n)), dim3(256), 0,
                     as_stream(stream), a);
  return check_launch("mk_gemm_int8");
}
