// The host side of the eight-bit entry points (src/kernels/rows_int8.hip,
// gemm_int8.hip, sample.hip) against a HIP runtime that only writes down its
// launches: the largest shapes they take must stay within the 2^32 - 1 threads
// per grid axis that HIP launches, and a product must run on the kernel that the
// dispatch rule names.  Nothing is allocated and nothing runs on a GPU.
// Prints "ok".
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <map>
#include <string>

#include "mk_kernels.h"

namespace {
std::map<const void*, std::string> g_names;
std::string g_kernel;
uint64_t g_x = 0, g_y = 0, g_block_size = 0, g_launched = 0;
dim3 g_grid, g_block;

void expect(bool ok, const std::string& what) {
  if (ok) return;
  std::printf("FAILED: %s\n", what.c_str());
  std::exit(1);
}
void* ptr(uint64_t v) { return reinterpret_cast<void*>(v); }
void launched(const std::string& what, int rc) {
  expect(rc == MK_OK && g_launched == 1, what + ": not launched once");
  expect(g_x * g_block_size < (uint64_t(1) << 32) && g_y < 65536, what + ": too large a grid");
  g_launched = 0;
}
}  // namespace

extern "C" {
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
void** __hipRegisterFatBinary(const void*) { return nullptr; }
void __hipRegisterFunction(void**, const void* f, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
  g_names[f] = name;
}
void __hipUnregisterFatBinary(void**) {}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t) { return g_grid = g, g_block = b, hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* s) {
  return *g = g_grid, *b = g_block, *lds = 0, *s = nullptr, hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3 g, dim3 b, void**, size_t, hipStream_t) {
  expect(g.x > 0 && g.y > 0, "an empty grid");
  g_kernel = g_names[f], g_x = g.x, g_y = g.y, g_block_size = b.x, ++g_launched;
  return hipSuccess;
}
}

namespace mk {
void clear_error() {}
int fail(int code, const std::string& what) { return std::printf("%s\n", what.c_str()), code; }
int check_launch(const char*) { return MK_OK; }
}  // namespace mk

int main() {
  void *X = ptr(uint64_t(1) << 44), *Y = ptr(uint64_t(1) << 46);  // never touched
  auto i8 = [](void* p) { return static_cast<int8_t*>(p); };
  auto f32 = [](void* p) { return static_cast<float*>(p); };

  // rows of every team, up to the most
  for (int64_t rows : {int64_t(1), (int64_t(1) << 21) - 1, (int64_t(1) << 21) + 1, (int64_t(1) << 23) + 5, int64_t(1) << 36})
    for (int64_t cols : {1, 7, 64, 512, 1024, 2048, 4096, 8192, 16384, 32768, 32769, 200000})
      for (int t : {MK_BF16, MK_F16, MK_F32}) {
        const std::string at = " of " + std::to_string(rows) + " x " + std::to_string(cols);
        launched("norm" + at, mk_add_rmsnorm_int8(nullptr, t, rows, cols, X, cols, X, cols, X, 1e-6f, Y, cols, i8(Y), cols, f32(Y)));
// waves a row: the number after the mode, ...ModeE0ELi<W>E
        const int waves = std::atoi(g_kernel.c_str() + g_kernel.find("ModeE") + 9);
        const uint64_t teams = g_x * g_y * (waves == 1 ? 4 : 1);
        expect(g_block_size == (waves == 1 ? 256 : 64 * waves), "norm" + at + ": threads of " + g_kernel);
        expect(teams >= uint64_t(rows), "norm" + at + ": rows left out");
        launched("rows" + at, mk_quantize_rows(nullptr, t, rows, cols, X, cols, 1, i8(Y), cols, f32(Y)));
        launched("values" + at, mk_dequantize_rows(nullptr, t, rows, cols, i8(X), cols, f32(X), Y, cols));
      }

  for (int64_t rows : {int64_t(1), (int64_t(1) << 22) - 1})
    launched("sampling", mk_sample_rows(nullptr, MK_F32, rows, 2097152, X, 2097152, f32(X), nullptr, 1.f, nullptr, 0, nullptr,
                                        1.f, nullptr, 0.f, MK_S64, Y, f32(Y)));

  auto product = [&](int64_t M, int64_t K, int64_t N, int64_t lda, int64_t ldb, int t = MK_BF16) {
    const std::string at = "product of " + std::to_string(M) + " x " + std::to_string(K) + " x " + std::to_string(N);
    launched(at, mk_gemm_int8(nullptr, t, M, N, K, i8(X), lda, f32(X), i8(X), ldb, f32(X), Y, N, nullptr, 0));
    return at;
  };
  // the largest: long rows of C, long columns, both orders of the grid, off it too
  const int64_t big = (int64_t(1) << 30) - 128, half = int64_t(1) << 18;
  for (int64_t K : {1, 16, 768, 4096, 131071})
    for (int64_t ld : {(K + 15) / 16 * 16, K + 1})
      for (int t : {MK_BF16, MK_F32}) {
        for (int64_t few : {1, 16, 17, 32, 33, 64}) product(few, K, big, ld, ld, t);
        for (int64_t few : {1, 33, 64}) product(big, K, few, ld, ld, t);
        product(half - 64, K, half - 64, ld, ld, t);
        product((int64_t(1) << 29) - 128, K, 128, ld, ld, t);
        product(128, K, (int64_t(1) << 29) - 128, ld, ld, t);
      }

  // which kernel: what its name holds
  struct { int64_t M, K, N, lda, ldb; const char* name; } routes[] = {
      {1, 768, 2304, 768, 768, "rows_kernelILi1ELi1ELi8E"},      // waves along k as K needs
      {16, 4096, 4096, 4096, 4096, "rows_kernelILi1ELi1ELi16E"},
      {16, 4096, 16384, 4096, 4096, "rows_kernelILi4ELi1E"},     // 64 columns a wave
      {16, 1024, 8192, 1024, 1024, "rows_kernelILi2ELi1E"},
      {32, 4096, 8192, 4096, 4096, "rows_kernelILi2ELi2E"},
      {60, 4097, 9000, 4097, 4097, "rows_kernelILi2ELi4E"},      // off the 16-byte grid
      {256, 4096, 256, 4096, 4096, "rows_kernelILi1ELi1ELi16E"}, // a small C
      {256, 4096, 512, 4096, 4096, "tiled_kernel"},
      {16, 768, 50257, 768, 768, "tiled_kernel"},
      {8192, 4096, 16384, 4096, 4096, "ShapeILi256ELi256E"},
      {2048, 4096, 4096, 4096, 4096, "ShapeILi"},
      {8192, 768, 768, 768, 768, "ShapeILi128ELi128E"},
      {128, 4096, 4096, 4096, 4096, "ShapeILi64ELi32E"},
      {8192, 4095, 4096, 4095, 4095, "ShapeILi128ELi128ELi2ELi4ELi2ELb0E"},
      {8192, 4096, 4096, 4096, 0, "ELb0E"},                      // one row of B for every column
      {8192, 4095, 4096, 4096, 4096, "ELb1E"}};                  // K off the grid, rows on it
  for (const auto& r : routes) {
    const std::string at = product(r.M, r.K, r.N, r.lda, r.ldb);
    expect(g_kernel.find(r.name) != std::string::npos, at + " on " + g_kernel);
  }
  std::printf("ok\n");
}
