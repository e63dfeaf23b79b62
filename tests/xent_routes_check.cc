// Which kernels mk_linear_xent, mk_linear_xent_bwd, mk_dropout_add and
// mk_dropout_add_bwd launch: the host code of linear_xent.hip (and of dropout.hip,
// linked) against a HIP runtime that only writes down its launches, of a GPU of
// 256 compute units.  Nothing is allocated and nothing runs on a GPU.
//
// Reads calls from stdin, a line each,
//   loss|grad type dw_type rows width vocab pitch_x pitch_w offset ignore    (offset: of both bases, elements)
//   drop|dropgrad type rows cols sums
// and prints a line of their launches, "kernel" or, of those that go from tile to
// tile, "kernel:tiles/workgroups/k tiles"; then a line "compiled <kernel>" for every kernel there is.
#include "linear_xent.hip"

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <cxxabi.h>
#include <map>

namespace {
std::map<const void*, std::string> g_names;
std::string g_line;
dim3 g_grid, g_block;

std::string short_name(const char* mangled) {
  int status = 0;
  char* text = abi::__cxa_demangle(mangled, nullptr, nullptr, &status);
  std::string s = status == 0 ? text : mangled;
  std::free(text);
  auto drop = [&](const std::string& what, const std::string& by) {
    for (size_t at; (at = s.find(what)) != std::string::npos;) s.replace(at, what.size(), by);
  };
  drop("mk::", ""), drop("(anonymous namespace)::", ""), drop("void ", ""), drop(", 2, 4, 64, 2>", ">"),
      drop(", 4, 2, 64, 2>", ">"), drop(" ", ""), drop("_kernel", "");
  return s.substr(0, s.find('('));
}

template <class A>
std::string tiles(const void* p, unsigned grid, int deep) {
  const A& a = *static_cast<const A*>(p);
  return ":" + std::to_string(int64_t(a.tiles_m) * a.tiles_n) + "/" + std::to_string(grid) + "/" +
         std::to_string((a.width + deep - 1) / deep);
}
}  // namespace

extern "C" {
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
void** __hipRegisterFatBinary(const void*) { return nullptr; }
void __hipRegisterFunction(void**, const void* f, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
  g_names[f] = short_name(name);
}
void __hipUnregisterFatBinary(void**) {}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t) { return g_grid = g, g_block = b, hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* s) {
  return *g = g_grid, *b = g_block, *lds = 0, *s = nullptr, hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3 g, dim3 b, void** args, size_t, hipStream_t) {
  if (uint64_t(g.x) * b.x >= uint64_t(1) << 32) g_line += "too-large:";
  const std::string& name = g_names[f];
  g_line += name;
  const int deep = name.find("<F32") != std::string::npos ? 32 : 64;
  if (name.compare(0, 5, "loss<") == 0) g_line += tiles<mk::LossArgs>(args[0], g.x, deep);
  if (name.compare(0, 5, "grad<") == 0) g_line += tiles<mk::GradArgs>(args[0], g.x, deep);
  g_line += " ";
  return hipSuccess;
}
}

namespace mk {
void clear_error() {}
int fail(int code, const std::string& what) { return std::printf("refused %s\n", what.c_str()), code; }
int check_launch(const char*) { return MK_OK; }
}  // namespace mk

extern "C" int mk_fill(void*, int, int64_t, uint64_t, void*) { return MK_OK; }

int main() {
  char kind[16];
  auto ptr = [](uint64_t v) { return reinterpret_cast<void*>(v); };
  while (std::scanf("%15s", kind) == 1) {
    g_line.clear();
    const std::string k = kind;
    long long type, dw, rows, width, vocab, px, pw, off, ignore, sums;
    if (k == "loss" || k == "grad") {
      if (std::scanf("%lld %lld %lld %lld %lld %lld %lld %lld %lld", &type, &dw, &rows, &width, &vocab, &px, &pw, &off, &ignore) != 9)
        return 1;
      const int64_t shift = off * mk::dtype_bytes(int(type));
      void *x = ptr((1ull << 40) + shift), *w = ptr((1ull << 41) + shift), *other = ptr(1ull << 42);
      const int rc = k == "loss" ? mk_linear_xent(nullptr, int(type), rows, width, vocab, x, px, w, pw, MK_S32, other, int(ignore), -100,
                                                  static_cast<float*>(other), static_cast<float*>(other), other)
                                 : mk_linear_xent_bwd(nullptr, int(type), int(dw), rows, width, vocab, x, px, w, pw, MK_S32, other,
                                                      int(ignore), -100, static_cast<float*>(other), static_cast<float*>(other), 1.f,
                                                      ptr(1ull << 43), width, ptr(1ull << 44), width, other);
      if (rc) return 1;
    } else {
      if (std::scanf("%lld %lld %lld %lld", &type, &rows, &width, &sums) != 4) return 1;
      void *a = ptr(1ull << 40), *b = ptr(1ull << 41), *c = ptr(1ull << 42);
      const int rc = k == "drop" ? mk_dropout_add(nullptr, int(type), rows, width, a, width, nullptr, nullptr, 0, 0.1, 1, 2, nullptr, b, width)
                                 : mk_dropout_add_bwd(nullptr, int(type), rows, width, a, width, 0.1, 1, 2, nullptr, b, width,
                                                      sums ? static_cast<float*>(c) : nullptr, c);
      if (rc) return 1;
    }
    std::printf("%s\n", g_line.c_str());
  }
  for (const auto& e : g_names) std::printf("compiled %s\n", e.second.c_str());
}
