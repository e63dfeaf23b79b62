// Which kernel mk_gemm_int8 launches for a product, and whether its C goes past the
// caches: the host code of gemm_int8.hip against a HIP runtime that only writes down
// its launches.  Nothing is allocated and nothing runs on a GPU.
//
// Reads products from stdin, "c_type M K N lda ldb ldc", and prints one line each,
// "rows<VN, MT, NW>" or "tiled<TM, TN, direct, CT> cached|streamed"; then a line
// "compiled <kernel>" for every kernel there is.
#include "gemm_int8.hip"

#include <cstdio>
#include <cstdlib>
#include <cxxabi.h>
#include <map>

namespace {
std::map<const void*, std::string> g_names;
std::string g_kernel;
bool g_streamed = false;
dim3 g_grid, g_block;

std::string short_name(const char* mangled) {
  int status = 0;
  char* text = abi::__cxa_demangle(mangled, nullptr, nullptr, &status);
  const std::string name = status == 0 ? text : mangled;
  std::free(text);
  int v[7], ct;
  char direct[6];
  size_t at = name.find("gemm_int8_rows_kernel<");
  if (at != std::string::npos &&
      std::sscanf(name.c_str() + at, "gemm_int8_rows_kernel<%d, %d, %d, %d>", v, v + 1, v + 2, v + 3) == 4)
    return "rows<" + std::to_string(v[0]) + ", " + std::to_string(v[1]) + ", " + std::to_string(v[2]) + ">";
  at = name.find("Shape<");
  if (at != std::string::npos && std::sscanf(name.c_str() + at, "Shape<%d, %d, %d, %d, %d, %5[a-z]>, %d>", v, v + 1,
                                             v + 2, v + 3, v + 4, direct, &ct) == 7)
    return "tiled<" + std::to_string(v[0]) + ", " + std::to_string(v[1]) + ", " + direct + ", " + std::to_string(ct) + ">";
  return name;
}
}  // namespace

extern "C" {
hipError_t hipGetLastError() { return hipSuccess; }
void** __hipRegisterFatBinary(const void*) { return nullptr; }
void __hipRegisterFunction(void**, const void* f, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
  g_names[f] = short_name(name);
}
void __hipUnregisterFatBinary(void**) {}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t) { return g_grid = g, g_block = b, hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* s) {
  return *g = g_grid, *b = g_block, *lds = 0, *s = nullptr, hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3, dim3, void** args, size_t, hipStream_t) {
  g_kernel += g_names[f];
  g_streamed = static_cast<const mk::Int8Gemm*>(args[0])->stream_c != 0;
  return hipSuccess;
}
}

namespace mk {
void clear_error() {}
int fail(int code, const std::string& what) { return std::printf("%s\n", what.c_str()), code; }
int check_launch(const char*) { return MK_OK; }
}  // namespace mk

int main() {
  int8_t* x = reinterpret_cast<int8_t*>(uint64_t(1) << 44);  // never touched
  float* s = reinterpret_cast<float*>(x);
  void* c = reinterpret_cast<void*>(uint64_t(1) << 46);
  int t;
  long long M, K, N, lda, ldb, ldc;
  while (std::scanf("%d %lld %lld %lld %lld %lld %lld", &t, &M, &K, &N, &lda, &ldb, &ldc) == 7) {
    g_kernel.clear();
    if (mk_gemm_int8(nullptr, t, M, N, K, x, lda, s, x, ldb, s, c, ldc, nullptr, 0) != MK_OK) return 1;
    std::printf("%s%s\n", g_kernel.c_str(), g_kernel[0] != 't' ? "" : g_streamed ? " streamed" : " cached");
  }
  for (const auto& n : g_names) std::printf("compiled %s\n", n.second.c_str());
}
