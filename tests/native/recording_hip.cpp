// Stands in front of the HIP runtime and writes down what a library asks of it: "attr <kernel> <bytes>" for every grant of dynamic LDS,
// "launch <kernel> <bytes>" for every launch.  Nothing runs.  refuse_grants(n): the next n grants fail.
#include <cstddef>
#include <cstdio>
struct Dim3 { unsigned x, y, z; };
static Dim3 grid, block;
static size_t lds;
static void* stream;
static int refuse = 0;
extern "C" {
void refuse_grants(int n) { refuse = n; }
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipGetLastError() { return 0; }
int hipFuncSetAttribute(const void* f, int, int bytes) {
  if (refuse > 0) { --refuse; return 1; }
  std::printf("attr %p %d\n", f, bytes);
  return 0;
}
int __hipPushCallConfiguration(Dim3 g, Dim3 b, size_t s, void* st) { grid = g; block = b; lds = s; stream = st; return 0; }
int __hipPopCallConfiguration(Dim3* g, Dim3* b, size_t* s, void** st) { *g = grid; *b = block; *s = lds; *st = stream; return 0; }
int hipLaunchKernel(const void* f, Dim3, Dim3, void**, size_t s, void*) { std::printf("launch %p %zu\n", f, s); return 0; }
}
