// Rotary positions with several axes (time, height, width, ...): channel pair p of every head turns by the angle
//   theta[token, p] = pos[token, axis(p)] * inv_freq[p]            (a, b) -> (a cos - b sin, a sin + b cos)
// pairs (p, P + p) of the first 2 P channels, or, interleaved, (2 p, 2 p + 1); channels behind 2 P pass through.  The gradient is the
// turn by -theta: the same kernel with the sign of the sine changed.
//
// Angles: the table holds inv_freq / (2 pi) in 64 bits; position times frequency gives REVOLUTIONS, whose whole part is dropped in 64
// bits before the fraction is rounded to fp32 -- a position of 2^20 keeps 2^-33 of a revolution, where an fp32 product would keep 2^-4.
// Sine and cosine are formed once per (token, pair) into LDS and shared by all heads of Q and K: the kernel is then one read and one
// write of the rows, which is its floor.
#include "tf_common.h"
#include "tf_kernels.h"
#include <algorithm>

namespace {

template <bool F32> struct RVec;
template <> struct RVec<false> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const void* p, size_t off, float (&f)[8]) { unpack8(*(const u32x4*)((const u16*)p + off), f); }
  static __device__ __forceinline__ void store(void* p, size_t off, const float (&f)[8]) { *(u32x4*)((u16*)p + off) = pack8(f); }
  static __device__ __forceinline__ float get(const void* p, size_t off) { return bf2f(((const u16*)p)[off]); }
  static __device__ __forceinline__ void put(void* p, size_t off, float v) { ((u16*)p)[off] = f2bf(v); }
};
template <> struct RVec<true> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const void* p, size_t off, float (&f)[4]) {
    const f32x4 v = *(const f32x4*)((const float*)p + off);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = v[i];
  }
  static __device__ __forceinline__ void store(void* p, size_t off, const float (&f)[4]) { *(f32x4*)((float*)p + off) = f32x4{f[0], f[1], f[2], f[3]}; }
  static __device__ __forceinline__ float get(const void* p, size_t off) { return ((const float*)p)[off]; }
  static __device__ __forceinline__ void put(void* p, size_t off, float v) { ((float*)p)[off] = v; }
};

constexpr int ROT_MAX_PAIRS = 256;

__device__ __forceinline__ double rot_pos(const TfRotaryArgs& a, size_t i) {
  if (a.pos_type == 0) return (double)((const int*)a.pos)[i];
  if (a.pos_type == 1) return (double)((const long long*)a.pos)[i];
  return (double)((const float*)a.pos)[i];
}

// n / d for n < 2^16 (m = ceil(2^32 / d), d < 2^16): one high multiplication
__device__ __forceinline__ int div16(int n, unsigned m) { return (int)__umulhi((unsigned)n, m); }
unsigned div16_of(int d) { return d == 1 ? 0u : (unsigned)((0x100000000ull + d - 1) / d); }
struct RotGeo {
  int tt;                      // tokens of a workgroup; tt * (H + Hk) * units < 2^16
  int units;                   // pieces of a head's row (see the kernel)
  int Pp;                      // pairs, rounded up to 4: the tables' row length
  unsigned m_units, m_heads, m_pairs;
};
__device__ __forceinline__ int div_u(int n, int d, unsigned m) { return d == 1 ? n : div16(n, m); }

// A workgroup turns g.tt tokens of the [B * S]: the table of their angles first, then pieces of rows, neighbours in memory by neighbouring
// threads.  VEC: a piece is a 16-byte vector of an interleaved row, or the two vectors of a row's halves that turn together, or a vector
// that passes through (the launcher checked that no pair straddles vectors); else one pair or one channel.
template <bool F32, bool VEC>
__global__ __launch_bounds__(256) void rotary_kernel(const TfRotaryArgs a, const RotGeo g) {
  using V = RVec<F32>;
  constexpr int N = V::N;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int P = a.pairs, Pp = g.Pp, tid = threadIdx.x, HT = a.H + a.Hk;
  long long* tq = (long long*)smem;                      // [tt] offsets of the token's first Q row / K row, in elements
  long long* tk = tq + g.tt;
  float* cs = (float*)(tk + g.tt);                       // [tt][2][Pp]: cosines, then sines
  const long long tokens = (long long)a.B * a.S, t0 = (long long)blockIdx.x * g.tt;
  const int nt = (int)min((long long)g.tt, tokens - t0);
  if (tid < nt) {
    const long long tok = t0 + tid, b = tok / a.S, s = tok - b * a.S;
    tq[tid] = b * a.q_sb + s * a.q_ss;
    tk[tid] = b * a.k_sb + s * a.k_ss;
  }
  for (int i = tid; i < nt * P; i += 256) {
    const int t = div_u(i, P, g.m_pairs), p = i - t * P;
    const long long tok = t0 + t;
    const size_t row = a.pos_batched ? (size_t)tok : (size_t)(tok % a.S);
    const double rev = rot_pos(a, row * a.n_axes + a.axis[p]) * a.inv_freq[p];
    float s, c;
    sincospif(2.0f * (float)(rev - rint(rev)), &s, &c);
    cs[2 * t * Pp + p] = c;
    cs[(2 * t + 1) * Pp + p] = a.inverse ? -s : s;
  }
  __syncthreads();
  const int W = HT * g.units;
#pragma unroll 2
  for (int i = tid; i < nt * W; i += 256) {
    const int th = div_u(i, g.units, g.m_units), u = i - th * g.units, t = div_u(th, HT, g.m_heads), h = th - t * HT;
    const bool isq = h < a.H;
    const int hh = isq ? h : h - a.H;
    const void* x = isq ? a.q : a.k;
    void* y = isq ? a.q_out : a.k_out;
    const size_t xo = isq ? tq[t] + hh * a.q_sh : tk[t] + hh * a.k_sh;
    const size_t yo = ((size_t)(t0 + t) * (isq ? a.H : a.Hk) + hh) * a.D;
    const float* c = cs + 2 * t * Pp;
    const float* sn = c + Pp;
    if (VEC) {
      float f[N], w[N];
      if (a.interleaved) {
        V::load(x, xo + u * N, f);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          const int p = u * (N / 2) + e, pc = min(p, P - 1);
          const float cc = c[pc], ss = sn[pc];
          w[2 * e] = p < P ? f[2 * e] * cc - f[2 * e + 1] * ss : f[2 * e];
          w[2 * e + 1] = p < P ? f[2 * e] * ss + f[2 * e + 1] * cc : f[2 * e + 1];
        }
        V::store(y, yo + u * N, w);
      } else if (u * N < P) {
        V::load(x, xo + u * N, f);
        V::load(x, xo + P + u * N, w);
        float r0[N], r1[N];
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          const f32x4 cc = *(const f32x4*)(c + u * N + e), ss = *(const f32x4*)(sn + u * N + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            r0[e + k] = f[e + k] * cc[k] - w[e + k] * ss[k];
            r1[e + k] = f[e + k] * ss[k] + w[e + k] * cc[k];
          }
        }
        V::store(y, yo + u * N, r0);
        V::store(y, yo + P + u * N, r1);
      } else {
        const int c0 = P + u * N;
        V::load(x, xo + c0, f);
        V::store(y, yo + c0, f);
      }
    } else if (u < P) {
      const float cc = c[u], ss = sn[u];
      const int c0 = a.interleaved ? 2 * u : u, c1 = a.interleaved ? 2 * u + 1 : P + u;
      const float f = V::get(x, xo + c0), w = V::get(x, xo + c1);
      V::put(y, yo + c0, f * cc - w * ss);
      V::put(y, yo + c1, f * ss + w * cc);
    } else {
      V::put(y, yo + P + u, V::get(x, xo + P + u));
    }
  }
}

bool vec_ok(const void* x, const void* y, long long sb, long long ss, long long sh, int n) {
  return (((uintptr_t)x | (uintptr_t)y) & 15) == 0 && sb % n == 0 && ss % n == 0 && sh % n == 0;
}

}  // namespace

extern "C" int tf_launch_rotary(const TfRotaryArgs* a, hipStream_t st) {
  if (a->B < 0 || a->S < 0 || a->H < 0 || a->Hk < 0 || a->D <= 0 || a->pairs <= 0 || a->pairs > ROT_MAX_PAIRS || 2 * a->pairs > a->D) return -1;
  if (a->n_axes <= 0 || a->pos_type < 0 || a->pos_type > 2) return -2;
  const long long tokens = (long long)a->B * a->S;
  const int HT = a->H + a->Hk;
  if (tokens == 0 || HT == 0) return 0;
  if (a->pos == nullptr || a->inv_freq == nullptr || a->axis == nullptr) return -3;
  if ((a->H > 0 && (a->q == nullptr || a->q_out == nullptr)) || (a->Hk > 0 && (a->k == nullptr || a->k_out == nullptr))) return -3;
  const int n = a->is_f32 ? 4 : 8;
  bool vec = a->D % n == 0 && (a->interleaved || a->pairs % n == 0);
  if (a->H > 0) vec = vec && vec_ok(a->q, a->q_out, a->q_sb, a->q_ss, a->q_sh, n);
  if (a->Hk > 0) vec = vec && vec_ok(a->k, a->k_out, a->k_sb, a->k_ss, a->k_sh, n);
  RotGeo g;
  g.units = vec ? (a->interleaved ? a->D / n : (a->D - a->pairs) / n) : a->D - a->pairs;
  g.Pp = (a->pairs + 3) / 4 * 4;
  const long long W = (long long)HT * g.units;
  if (W > 0xffff || a->D > 0xffff) return -5;
  // eight pieces a thread where that still leaves four workgroups a CU, fewer tokens a workgroup otherwise; the tables stay in 16 KiB
  long long tt = std::max(1ll, std::min({2048 / W, tokens / 1024, 0xffff / std::max<long long>(W, a->pairs), 2048ll / g.Pp, 64ll}));
  g.tt = (int)tt;
  g.m_units = div16_of(g.units);
  g.m_heads = div16_of(HT);
  g.m_pairs = div16_of(a->pairs);
  const long long blocks = (tokens + tt - 1) / tt;
  if (blocks > 0x7fffffffll) return -4;
  const size_t lds = (size_t)tt * (16 + 2 * g.Pp * sizeof(float));
  const double bytes = 2.0 * tokens * HT * a->D * (a->is_f32 ? 4 : 2);
  TfTraceScope tr("rotary_kernel", st, 3.0 * tokens * HT * 2 * a->pairs, bytes);
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), lds, st, *a, g); };
  if (a->is_f32) vec ? go(rotary_kernel<true, true>) : go(rotary_kernel<true, false>);
  else vec ? go(rotary_kernel<false, true>) : go(rotary_kernel<false, false>);
  return (int)hipGetLastError();
}
