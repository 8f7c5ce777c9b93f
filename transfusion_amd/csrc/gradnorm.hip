// Global norm over many tensors, and clipping (torch.nn.utils.clip_grad_norm_'s arithmetic):
//   total = sqrt(sum over all tensors of g^2)   or   max |g|;      g *= min(1, max_norm / (total + 1e-6))
// Two passes over the bytes are the floor when the norm exceeds the limit (one read for the norm, one read + write for the scale), one
// when it does not.  A launch carries up to 192 tensors in its kernel arguments (address, length, first workgroup), so hundreds of
// gradients take a few launches instead of several per tensor, nothing is copied to the device, and a captured graph holds the table.
//
// Every workgroup of the first pass writes ONE 64-bit partial; every workgroup of the second pass adds all of them up again in index
// order (a few thousand values from L2) -- no atomics, no counter to reset, the same bits on every run and rank, and no third launch.
// Squares are accumulated in 64 bits: neither the length of the sum nor a gradient beyond 2^64 costs anything, and the kernel stays
// bound by its loads: they bring 1.2 (fp32) to 2.4 (bf16) elements a picosecond, the card forms up to 39 fp64 FMAs in that time.
#include "tf_common.h"
#include "tf_kernels.h"
#include <algorithm>
#include <vector>

namespace {

constexpr int GN_TAB = 192;                              // tensors of one launch: 192 * 20 bytes of kernel arguments
constexpr int GN_CHUNK = 16384;                          // elements of a workgroup, at least
constexpr int GN_BLOCKS = 2048;                          // workgroups beyond which the chunk grows

struct GnTab {
  void* p[GN_TAB];
  long long n[GN_TAB];
  int blk0[GN_TAB];                                      // (bit 31: the tensor is bf16)
};

__device__ __forceinline__ int gn_find(const GnTab& t, int count, int blk) {
  int lo = 0, hi = count - 1;                            // the last tensor whose first workgroup is <= blk
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((t.blk0[mid] & 0x7fffffff) <= blk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// inf norm: the largest |g| as an integer; the bits of a NaN are above those of infinity, so a NaN wins as it does in torch
template <bool INF> __device__ __forceinline__ void gn_add(double& s, unsigned& m, float x) {
  if (INF) m = max(m, __builtin_bit_cast(unsigned, x) & 0x7fffffffu);
  else s = __builtin_fma((double)x, (double)x, s);
}

// f over n values from x on (STORE: x = f(x)), by 256 threads: 16-byte accesses from the first aligned address on, four in flight a thread,
// single elements before and behind
template <class T, class F> __device__ __forceinline__ void gn_each(const T* xc, long long n, int tid, F&& f, bool store) {
  constexpr int N = 16 / sizeof(T);
  T* x = const_cast<T*>(xc);
  auto one = [&](long long i) {
    if constexpr (sizeof(T) == 2) { const float y = f(bf2f(x[i])); if (store) x[i] = f2bf(y); }
    else { const float y = f(x[i]); if (store) x[i] = y; }
  };
  const long long head = min(n, (long long)(((16 - ((size_t)x & 15)) & 15) / sizeof(T)));
  if (tid < head) one(tid);
  u32x4* v = (u32x4*)(x + head);
  const long long nv = (n - head) / N;
  auto vec = [&](const u32x4& u) {
    u32x4 r;
    if constexpr (sizeof(T) == 2) {
      float e[8];
      unpack8(u, e);
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = f(e[k]);
      r = pack8(e);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) { const unsigned w = u[k]; r[k] = __builtin_bit_cast(unsigned, f(__builtin_bit_cast(float, w))); }
    }
    return r;
  };
  long long i = tid;
  for (; i + 3 * 256 < nv; i += 4 * 256) {
    u32x4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = v[i + k * 256];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const u32x4 r = vec(u[k]);
      if (store) v[i + k * 256] = r;
    }
  }
  for (; i < nv; i += 256) {
    const u32x4 r = vec(v[i]);
    if (store) v[i] = r;
  }
  const long long t0 = head + nv * N;
  if (t0 + tid < n) one(t0 + tid);
}

template <bool INF> __device__ __forceinline__ double gn_block_reduce(double s, unsigned m, double* sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    if (INF) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
    else s += __shfl_xor(s, o, 64);
  }
  if (lane == 0) sh[wave] = INF ? (double)m : s;
  __syncthreads();
  const double r = INF ? fmax(fmax(sh[0], sh[1]), fmax(sh[2], sh[3])) : (sh[0] + sh[1]) + (sh[2] + sh[3]);
  __syncthreads();
  return r;
}

template <bool INF>
__global__ __launch_bounds__(256) void grad_norm_part_kernel(const GnTab tab, int count, long long chunk, double* __restrict__ part) {
  __shared__ double sh[4];
  const int t = gn_find(tab, count, (int)blockIdx.x), tid = threadIdx.x;
  const bool bf = tab.blk0[t] < 0;
  const long long b = (long long)((int)blockIdx.x - (tab.blk0[t] & 0x7fffffff));
  const long long lo = b * chunk, hi = min(tab.n[t], lo + chunk);
  double s = 0.0;
  unsigned m = 0u;
  if (bf) gn_each<u16>((const u16*)tab.p[t] + lo, hi - lo, tid, [&](float x) { gn_add<INF>(s, m, x); return x; }, false);
  else gn_each<float>((const float*)tab.p[t] + lo, hi - lo, tid, [&](float x) { gn_add<INF>(s, m, x); return x; }, false);
  const double r = gn_block_reduce<INF>(s, m, sh);
  if (tid == 0) part[blockIdx.x] = r;
}

// total and, with a limit, g *= coef.  `first`: this launch's workgroup 0 writes the norm.
template <bool INF>
__global__ __launch_bounds__(256) void grad_clip_kernel(const GnTab tab, int count, long long chunk, const double* __restrict__ part, int nparts,
                                                        float max_norm, float* __restrict__ norm, int first) {
  __shared__ double sh[4];
  const int tid = threadIdx.x;
  double s = 0.0;
  unsigned m = 0u;
  for (int i = tid; i < nparts; i += 256) {
    if (INF) m = max(m, (unsigned)part[i]);
    else s += part[i];
  }
  const double r = gn_block_reduce<INF>(s, m, sh);
  const float total = INF ? __builtin_bit_cast(float, (unsigned)r) : (float)sqrt(r);
  if (first && blockIdx.x == 0 && tid == 0) norm[0] = total;
  if (count == 0) return;
  float coef = max_norm / (total + 1e-6f);
  if (coef > 1.0f) coef = 1.0f;                          // (a NaN stays)
  if (coef == 1.0f) return;                              // times one is the same bits: nothing to write
  const int blk = (int)(gridDim.x - 1 - blockIdx.x);     // from the end: what the first pass read last is still in the caches
  const int t = gn_find(tab, count, blk);
  const bool bf = tab.blk0[t] < 0;
  const long long b = (long long)(blk - (tab.blk0[t] & 0x7fffffff));
  const long long lo = b * chunk, hi = min(tab.n[t], lo + chunk);
  if (bf) gn_each<u16>((const u16*)tab.p[t] + lo, hi - lo, tid, [&](float x) { return x * coef; }, true);
  else gn_each<float>((const float*)tab.p[t] + lo, hi - lo, tid, [&](float x) { return x * coef; }, true);
}

struct GnPlan {
  long long chunk;
  int blocks;
};
bool gn_plan(const long long* n, int count, GnPlan* out) {
  long long total = 0;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0 || n[i] > (1ll << 42) || total > (1ll << 42)) return false;
    total += n[i];
  }
  const long long grow = (total / GN_BLOCKS + 255) / 256 * 256;
  out->chunk = std::max((long long)GN_CHUNK, grow);
  long long blocks = 0;
  for (int i = 0; i < count; ++i) blocks += (n[i] + out->chunk - 1) / out->chunk;
  if (blocks > 0x3fffffff) return false;
  out->blocks = (int)blocks;
  return true;
}

}  // namespace

extern "C" long long tf_grad_clip_parts(const long long* n, int count) {
  GnPlan pl;
  if (count < 0 || (count > 0 && n == nullptr) || !gn_plan(n, count, &pl)) return -1;
  return std::max(1, pl.blocks);
}

extern "C" int tf_launch_grad_clip(const TfGradClipArgs* a, hipStream_t st) {
  if (a->count < 0 || (a->count > 0 && (a->grads == nullptr || a->n == nullptr || a->is_bf16 == nullptr))) return -1;
  if (a->work == nullptr || a->norm == nullptr || (a->norm_type != 0 && a->norm_type != 1)) return -2;
  GnPlan pl;
  if (!gn_plan(a->n, a->count, &pl) || a->parts < std::max(1, pl.blocks)) return -3;
  // one memory may not be scaled twice: no two tensors overlap
  std::vector<std::pair<uintptr_t, uintptr_t>> span;
  double bytes = 0.0;
  for (int i = 0; i < a->count; ++i) {
    if (a->n[i] == 0) continue;
    if (a->grads[i] == nullptr) return -4;
    const int e = a->is_bf16[i] ? 2 : 4;
    const uintptr_t p = (uintptr_t)a->grads[i];
    if (p % e != 0) return -4;
    span.emplace_back(p, p + (uintptr_t)a->n[i] * e);
    bytes += (double)a->n[i] * e;
  }
  std::sort(span.begin(), span.end());
  for (size_t i = 1; i < span.size(); ++i)
    if (span[i].first < span[i - 1].second) return -5;

  double* part = (double*)a->work;
  auto each = [&](auto&& launch) -> int {                // tables of up to GN_TAB tensors; blk_base counts the workgroups before them
    GnTab tab;
    int k = 0, nblk = 0, base = 0;
    for (int i = 0; i <= a->count; ++i) {
      if (k == GN_TAB || (i == a->count && k > 0)) {
        const int rc = launch(tab, k, nblk, base);
        if (rc != 0) return rc;
        base += nblk;
        k = nblk = 0;
      }
      if (i == a->count || a->n[i] == 0) continue;
      tab.p[k] = a->grads[i];
      tab.n[k] = a->n[i];
      tab.blk0[k] = nblk | (a->is_bf16[i] ? (int)0x80000000 : 0);
      nblk += (int)((a->n[i] + pl.chunk - 1) / pl.chunk);
      ++k;
    }
    return 0;
  };
  int rc = each([&](const GnTab& tab, int k, int nblk, int base) {
    TfTraceScope tr("grad_norm_part_kernel", st, 0.0, bytes);
    if (a->norm_type == 1) hipLaunchKernelGGL(grad_norm_part_kernel<true>, dim3(nblk), dim3(256), 0, st, tab, k, pl.chunk, part + base);
    else hipLaunchKernelGGL(grad_norm_part_kernel<false>, dim3(nblk), dim3(256), 0, st, tab, k, pl.chunk, part + base);
    return (int)hipGetLastError();
  });
  if (rc != 0) return rc;
  const int nparts = pl.blocks;
  auto finish = [&](const GnTab& tab, int k, int nblk, int first) {
    TfTraceScope tr("grad_clip_kernel", st, 0.0, k ? 2 * bytes : 0.0);
    if (a->norm_type == 1) hipLaunchKernelGGL(grad_clip_kernel<true>, dim3(nblk), dim3(256), 0, st, tab, k, pl.chunk, part, nparts, a->max_norm, a->norm, first);
    else hipLaunchKernelGGL(grad_clip_kernel<false>, dim3(nblk), dim3(256), 0, st, tab, k, pl.chunk, part, nparts, a->max_norm, a->norm, first);
    return (int)hipGetLastError();
  };
  if (!a->clip || pl.blocks == 0) return finish(GnTab{}, 0, 1, 1);
  return each([&](const GnTab& tab, int k, int nblk, int base) { return finish(tab, k, nblk, base == 0); });
}
