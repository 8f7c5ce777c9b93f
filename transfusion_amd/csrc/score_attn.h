// Attention whose scores are changed before the softmax: capped by a tanh, biased by distance, masked by documents and by a causal
// horizon with a bidirectional prefix.  For query i at position p and key j of one head
//   s = scale * q.k ;  s = cap * tanh(s / cap) (cap > 0) ;  s -= slope_h * |p - j| ;
//   hidden unless  doc_q == doc_k >= 0  and  (not causal or j <= p or j < prefix) ;   P = softmax_j(s) ;  o = P v .
// A row that attends nothing gives o = 0 and no gradient.  Heads may share keys and values (H / Hk heads each).
//
// No [Sq, Sk] tensor reaches memory: the forward keeps a running maximum and sum and stores one log-sum-exp a row, the backward forms P
// again from it.  Orientation as in attn_bf16.hip: the score tile is computed transposed (keys in the accumulator registers, the query
// on the lane), so a row's statistics are one scalar a lane and the tile is the next product's operand as it stands.
//   score_attn_fwd.hip   score_fwd_kernel: 128 queries a workgroup;  score_few16 / few32_kernel: single tokens, the keys split over the chip
//   score_attn_bwd.hip   score_dq_kernel: query on the lane -> dq, delta = rowsum(dO o), the slopes' row sums;
//                        score_dkv_kernel: key on the lane, loops over the heads of its group and their queries -> dk, dv
// Where there are too few workgroups, a kernel splits its loop and writes fp32 parts that a second kernel adds up in order: no atomics.
// Scores, statistics and accumulators are fp32.  P and dS are rounded to the operand type of the next product (bf16: at most half a step,
// 2^-8 of each term, as every product of bf16 operands has it already); fp32 tensors run on the fp32 matrix instructions throughout.
#pragma once
#include "tf_common.h"
#include "tf_kernels.h"
#include "attn_common.h"
#include <algorithm>
#include <atomic>

namespace {

// ---- operand fragments: 8 consecutive channels of one row per lane (half h of the wave holds channels 16 ks + 8 h ..) ----
template <bool F32> struct SFrag;
template <> struct SFrag<false> { u32x4 v; };
template <> struct SFrag<true> { f32x4 a, b; };

template <bool F32> __device__ __forceinline__ f32x16 smma(const SFrag<F32>& A, const SFrag<F32>& B, f32x16 c) {
  if constexpr (F32) {
    // step e multiplies channel e of both halves: the k order inside the 16 channels is the same for both operands, so any will do
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(A.a[e], B.a[e], c, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(A.b[e], B.b[e], c, 0, 0, 0);
    return c;
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(A.v), as_bf16x8(B.v), c, 0, 0, 0);
  }
}

// fragment of one row straight from memory; `ok` false: zeros
template <bool F32> __device__ __forceinline__ SFrag<F32> gfrag(const char* row, int ks, int h, int D, bool ok) {
  SFrag<F32> f;
  const int c0 = ks * 16 + 8 * h;
  ok = ok && c0 < D;
  if constexpr (F32) {
    f.a = ok ? *(const f32x4*)(row + c0 * 4) : f32x4{0, 0, 0, 0};
    f.b = ok ? *(const f32x4*)(row + c0 * 4 + 16) : f32x4{0, 0, 0, 0};
  } else {
    f.v = ok ? *(const u32x4*)(row + c0 * 2) : u32x4{0, 0, 0, 0};
  }
  return f;
}
// Loads that have to be back here: a value still under way when a loop with LDS-DMA begins makes the compiler wait for ALL transfers in front
// of its first use in the loop, on every turn -- the transfers ahead would never be ahead
__device__ __forceinline__ void landed(SFrag<false>& f) { asm volatile("" : "+v"(f.v)); }
__device__ __forceinline__ void landed(SFrag<true>& f) { asm volatile("" : "+v"(f.a), "+v"(f.b)); }
__device__ __forceinline__ void landed(float& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void landed(int& x) { asm volatile("" : "+v"(x)); }

// ---- the change of a score, in the log2 domain ----
struct SMod {
  float sc;          // no cap: scale * log2 e;  cap: 2 log2 e * scale / cap (the exponent of the tanh)
  float capl;        // cap * log2 e, or 0
  float slope2;      // slope * log2 e
  float zs, zlim;    // cap: scores (before the scale, times zs) up to zlim take the polynomial below
  float small;       // zlim where zs is 1, else -1
  float c0, c1, c2, c3;
};
__device__ __forceinline__ float uniform(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x))); }
__device__ __forceinline__ SMod smod(const TfScoreAttnArgs& a, int head) {
  SMod m;
  m.capl = uniform(a.softcap > 0.f ? a.softcap * LOG2E : 0.f);
  m.sc = uniform(a.softcap > 0.f ? 2.f * LOG2E * a.scale / a.softcap : a.scale * LOG2E);
  m.slope2 = a.slopes != nullptr ? uniform(a.slopes[head] * LOG2E) : 0.f;
  // tanh y = y (1 - y^2 / 3 ...) for |y| <= 1/2: a least-maximum fit of degree 3 in y^2, relative error 5e-7.  Scores are mostly far below the
  // cap, and five multiplications cost less than half of an exponential and a reciprocal (two quarter-rate instructions).  The powers of y / score
  // are folded into the coefficients; where they leave fp32's range the polynomial takes s * sc = 2 log2(e) y instead of s.
  const float g = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
  const float last = fabsf(m.capl * g * (g * g) * (g * g) * (g * g));
  const bool in = last > 1e-36f && last < 1e36f;         // (a coefficient that is infinite makes a NaN of a score of 0)
  const float y = in ? g : 0.5f / LOG2E, y2 = y * y;
  m.zs = uniform(in ? 1.f : m.sc);
  m.zlim = uniform(0.5f / fabsf(y));
  m.small = in ? m.zlim : -1.f;
  m.c0 = uniform(0.99999946f * m.capl * y);
  m.c1 = uniform(-0.33326318f * m.capl * y * y2);
  m.c2 = uniform(0.13190297f * m.capl * y * y2 * y2);
  m.c3 = uniform(-0.04440223f * m.capl * y * y2 * y2 * y2);
  return m;
}
__device__ __forceinline__ float capped_poly(float s, float c0, float c1, float c2, float c3) {
  const float u = s * s;
  return s * fmaf(u, fmaf(u, fmaf(u, c3, c2), c1), c0);
}
// cap * tanh(scale s / cap) in the log2 domain, to 2^-20 of its value.  1 - 2 / (1 + e^2y) alone (+-inf give +-1, no NaN in between) is off by 2e-7
// whatever its size: under a cap of 1e6 that is 0.2 of every score, however small.
template <bool F32> __device__ __forceinline__ float capped(const SMod& m, float s) {
  if constexpr (F32) return m.capl * tanhf(s * m.sc * 0.34657359027997264f);
  const float z = s * m.zs, low = capped_poly(z, m.c0, m.c1, m.c2, m.c3);
  const float high = m.capl * (1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + fast_exp2(s * m.sc)));
  return fabsf(z) <= m.zlim ? low : high;
}
// are all scores of a tile small enough for the polynomial as they stand?  (wave-uniform; a NaN stays one either way)
template <bool F32, int N> __device__ __forceinline__ bool all_small(const SMod& m, const f32x16 (&st)[N]) {
  if (F32) return false;                  // (fp32: the polynomial's 5e-7 would show)
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(st[k][r]));
  return __all(top <= m.small);
}
// Beyond this size (log2 domain) what rounding takes from a score is more than a small part of its probability: there every kernel forms the same
// rounded score and only then takes the row's maximum or log-sum-exp off it.  Left to itself, a product that rides in an FMA with the maximum is not
// rounded: at 10^10 the largest score then lies up to 512 beyond "itself", an infinity or a zero in place of a one.
constexpr float S_BIG = 4096.f;
__device__ __forceinline__ bool big(float x) { return fabsf(x) > S_BIG && fabsf(x) < INFINITY; }
// (no FMA across it)
__device__ __forceinline__ float rounded(float x) { asm("" : "+v"(x)); return x; }
// score by score, in place: capped, or only scaled
template <bool F32> __device__ __forceinline__ void cap_each(const SMod& m, f32x16& st) {
  if (m.capl != 0.f) {
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = rounded(capped<F32>(m, st[r]));
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = rounded(st[r] * m.sc);
  }
}
// the capped scores of a forward's tile, in place.  (One branch that rewrites the scores; as two arms the forms cost a second set of registers.)
template <bool F32, int N> __device__ __forceinline__ void cap_scores(const SMod& m, f32x16 (&st)[N]) {
  float c0 = m.c0, c1 = m.c1, c2 = m.c2, c3 = m.c3;
  if (__builtin_expect(!all_small<F32, N>(m, st), F32)) {         // the polynomial below becomes the identity
#pragma unroll
    for (int k = 0; k < N; ++k) cap_each<F32>(m, st[k]);
    c0 = 1.f;
    c1 = c2 = c3 = 0.f;
  }
  if (!F32) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int r = 0; r < 16; ++r) st[k][r] = capped_poly(st[k][r], c0, c1, c2, c3);
  }
}
// position of query 0 (bounded so that sums with a query number stay in 32 bits) and the prefix length of sample b
__device__ __forceinline__ int q_pos0(const TfScoreAttnArgs& a, int b) {
  const int p = a.q_start != nullptr ? a.q_start[b] : a.Sk - a.Sq;
  return min(max(p, -(1 << 30)), 1 << 30);
}
__device__ __forceinline__ int prefix_of(const TfScoreAttnArgs& a, int b) { return a.prefix != nullptr ? min(max(a.prefix[b], 0), a.Sk) : 0; }

// (by value: a bit cast of a vector's element in place takes the vector's first)
__device__ __forceinline__ float f_of(unsigned u) { return __builtin_bit_cast(float, u); }
// two values -> one register of bf16 in one instruction (spelt so that the compiler keeps the wait between an exponential and its use)
__device__ __forceinline__ unsigned pk2(float lo, float hi) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  const f32x2 v = {lo, hi};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}
constexpr float S_NEG = -1.0e38f;          // the running maximum before the first visible key

// ---- LDS tiles ----
// Rows of HDP channels.  bf16: a stride of an ODD multiple of 64 bytes, 16-byte piece ^= (row >> 2) & 3: four consecutive rows start 16
// banks apart in some order, so row reads (ds_read_b128) and transposed reads (ds_read_b64_tr_b16) are both free of conflicts, at the
// smallest such stride (192 bytes for 64 channels, 448 for 192).  fp32: rows 4 banks apart.
template <bool F32, int HDP> struct SGeo {
  static constexpr int ESZ = F32 ? 4 : 2, KS = HDP / 16, DB = HDP / 32, CPR = HDP * ESZ / 16;
  static constexpr int STR = F32 ? HDP * 4 + 16 : ((HDP * 2 + 63) / 64 | 1) * 64;
  static constexpr int FR = F32 ? 2 : 1;                 // LDS reads of a row fragment
};
// LDS-DMA of a tile of ROWS rows by NW waves: the image is linear in the lane, so the layout lives on the source side.  Pieces at or beyond
// D get an offset behind the buffer's end and arrive as zeros, as do rows beyond its last.
template <bool F32, int HDP, int ROWS, int NW> struct SDma {
  using G = SGeo<F32, HDP>;
  static constexpr int T = G::STR, NI = (ROWS * T + NW * 1024 - 1) / (NW * 1024), BYTES = NI * NW * 1024;
  static constexpr unsigned OUT = 0x7fffff00u;
  unsigned off[NI], rb;       // offsets for rows of rb bytes; a matrix with other rows has them formed where it is read
  int wave, lane;
  __device__ __forceinline__ int slot(int i) const { return (wave * NI + i) * 1024 + lane * 16; }
  __device__ __forceinline__ unsigned offset(int i, unsigned row_bytes, int D) const {
    const int pos = slot(i), r = pos / T, cp = (pos % T) >> 4, c = F32 ? cp : cp ^ ((r >> 2) & 3);
    return r >= ROWS || cp >= G::CPR || c * (16 / G::ESZ) >= D ? OUT : (unsigned)r * row_bytes + c * 16;
  }
  __device__ __forceinline__ SDma(int wave_, int lane_, unsigned row_bytes, int D) : rb(row_bytes), wave(wave_), lane(lane_) {
#pragma unroll
    for (int i = 0; i < NI; ++i) off[i] = offset(i, row_bytes, D);
  }
  // rows row0 .. of the matrix at base, row_end excluded (row0 < row_end); doc != null: rows of negative documents are zeros too
  __device__ __forceinline__ void issue(const char* base, unsigned row_bytes, int row0, int row_end, int D, const int* doc, unsigned char* tile) const {
    const int n = min(ROWS, row_end - row0);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(base + (long long)row0 * row_bytes), 0,
                                                                         (int)((unsigned)(n - 1) * row_bytes + D * G::ESZ), 0x00020000);
    unsigned char* dst = tile + wave * NI * 1024;
    if (doc == nullptr && row_bytes == rb) {
#pragma unroll
      for (int i = 0; i < NI; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, TF_LDS_PTR(dst + i * 1024), 16, (int)off[i], 0, 0, 0);
    } else {
      // (a lane a row and one ballot: a load a piece, each waited for, took as long as the tile's products)
      const u64 neg = doc != nullptr ? __ballot(doc[row0 + min(lane, n - 1)] < 0) : 0ull;
#pragma unroll 1
      for (int i = 0; i < NI; ++i) {
        const unsigned o = (neg >> min(slot(i) / T, 63)) & 1ull ? OUT : offset(i, row_bytes, D);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, TF_LDS_PTR(dst + i * 1024), 16, (int)o, 0, 0, 0);
      }
    }
  }
};

template <int OFF> __device__ __forceinline__ unsigned rd32_asm(unsigned addr) {
  unsigned d;
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(d) : "v"(addr), "n"(OFF) : "memory");
  return d;
}
template <int N> __device__ __forceinline__ void lgkm_wait32(unsigned& f) { asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(f) : "n"(N)); }

// values of an accumulator tile as the next product's operand
template <bool F32> struct SPack;
template <> struct SPack<false> {
  unsigned v[8];
  __device__ __forceinline__ void set2(int r, float x0, float x1) { v[r >> 1] = pk2(x0, x1); }
};
template <> struct SPack<true> {
  float v[16];
  __device__ __forceinline__ void set2(int r, float x0, float x1) { v[r] = x0; v[r + 1] = x1; }
};

// A matrix instruction may not sink below the waits that follow it: left to itself the scheduler gathers the waits of a product in front of
// its matrix instructions, and every read is waited for before the first of them starts
#define SCORE_PIN() __builtin_amdgcn_sched_barrier(0)

// Reads of a tile: row fragments (32 rows x 16 channels) and the products whose operand is the tile transposed.  All reads are issued from
// inline asm a few fragments ahead of the matrix instruction that takes them, each wait names the fragment it releases (attn_common.h).
template <bool F32, int HDP> struct SAddr;
template <int HDP> struct SAddr<false, HDP> {
  static constexpr int T = SGeo<false, HDP>::STR, DB = HDP / 32;
  unsigned row_e, row_o, tr_a, tr_b;
  __device__ __forceinline__ SAddr(unsigned tile, int lane) {
    const int r = lane & 31, x = (r >> 2) & 3, hh = lane >> 5;
    row_e = tile + r * T + ((hh ^ x) << 4);
    row_o = tile + r * T + (((2 + hh) ^ x) << 4);
    const int li = lane & 15, q4 = li >> 2, p = li & 3, cb = (lane >> 4) & 1, low2 = 2 * cb + (p >> 1);
    tr_a = tile + (4 * hh + q4) * T + ((low2 ^ hh) << 4) + (p & 1) * 8;
    tr_b = tile + (4 * hh + q4 + 8) * T + ((low2 ^ (hh + 2)) << 4) + (p & 1) * 8;
  }
  __device__ __forceinline__ SAddr shifted(unsigned bytes) const {
    SAddr g = *this;
    g.row_e += bytes; g.row_o += bytes; g.tr_a += bytes; g.tr_b += bytes;
    return g;
  }
  // OFF: bytes from the address to a tile behind it, a compile-time constant in every form
  template <int KS, int OFF> __device__ __forceinline__ void row(SFrag<false>& f) const { f.v = rd128_asm<OFF + 64 * (KS >> 1)>((KS & 1) ? row_o : row_e); }
  template <int N> static __device__ __forceinline__ void wait(SFrag<false>& f) { lgkm_wait<N>(f.v); }
  // acc[channel][lane] += sum over 32 NP rows of tile[row][channel] * p[row]
  template <int OFF, int NP> __device__ __forceinline__ void mul_t(const SPack<false> (&p)[NP], f32x16 (&acc)[DB]) const {
    constexpr int NF = 2 * NP * DB, PF = 2;
    u64 fa[NF], fb[NF];
    static_for<PF>([&](auto I) { tr<I, OFF>(fa[I], fb[I]); });
    static_for<NF>([&](auto I) {
      constexpr int i = I, nx = i + PF, k = i / DB, s = 4 * (k & 1);
      if constexpr (nx < NF) tr<nx, OFF>(fa[nx], fb[nx]);
      lgkm_wait<2 * (NF - 1 - i < PF ? NF - 1 - i : PF)>(fa[i], fb[i]);
      acc[i % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(join_tr64(fa[i], fb[i]), as_bf16x8(u32x4{p[k / 2].v[s], p[k / 2].v[s + 1], p[k / 2].v[s + 2], p[k / 2].v[s + 3]}), acc[i % DB], 0, 0, 0);
      SCORE_PIN();
    });
  }
  template <int I, int OFF> __device__ __forceinline__ void tr(u64& a, u64& b) const {
    a = tr_read_asm<OFF + (I / DB) * 16 * T + (I % DB) * 64>(tr_a);
    b = tr_read_asm<OFF + (I / DB) * 16 * T + (I % DB) * 64>(tr_b);
  }
};
template <int HDP> struct SAddr<true, HDP> {
  static constexpr int T = SGeo<true, HDP>::STR, DB = HDP / 32;
  unsigned r0, t0;
  __device__ __forceinline__ SAddr(unsigned tile, int lane) {
    r0 = tile + (lane & 31) * T + (lane >> 5) * 32;
    t0 = tile + 4 * (lane >> 5) * T + (lane & 31) * 4;
  }
  __device__ __forceinline__ SAddr shifted(unsigned bytes) const {
    SAddr g = *this;
    g.r0 += bytes; g.t0 += bytes;
    return g;
  }
  template <int KS, int OFF> __device__ __forceinline__ void row(SFrag<true>& f) const {
    f.a = __builtin_bit_cast(f32x4, rd128_asm<OFF + 64 * KS>(r0));
    f.b = __builtin_bit_cast(f32x4, rd128_asm<OFF + 64 * KS + 16>(r0));
  }
  template <int N> static __device__ __forceinline__ void wait(SFrag<true>& f) { asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(f.a), "+v"(f.b) : "n"(N)); }
  template <int OFF, int NP> __device__ __forceinline__ void mul_t(const SPack<true> (&p)[NP], f32x16 (&acc)[DB]) const {
    static_for<NP>([&](auto P) { (P == 0 ? *this : shifted(P * 32 * T)).template one_t<OFF>(p[P], acc); });
  }
  template <int OFF> __device__ __forceinline__ void one_t(const SPack<true>& p, f32x16 (&acc)[DB]) const {
    constexpr int NF = 16 * DB, PF = 6;
    unsigned fr[NF];
    static_for<PF>([&](auto I) { fr[I] = col<I, OFF>(); });
    static_for<NF>([&](auto I) {
      constexpr int i = I, nx = i + PF;
      if constexpr (nx < NF) fr[nx] = col<nx, OFF>();
      lgkm_wait32<(NF - 1 - i < PF ? NF - 1 - i : PF)>(fr[i]);
      acc[i % DB] = __builtin_amdgcn_mfma_f32_32x32x2f32(f_of(fr[i]), p.v[i / DB], acc[i % DB], 0, 0, 0);
    });
  }
  template <int I, int OFF> __device__ __forceinline__ unsigned col() const {
    constexpr int r = I / DB;
    return rd32_asm<OFF + ((r & 3) + 8 * (r >> 2)) * T + (I % DB) * 128>(t0);
  }
};
// st += tile . x ; x(ks) gives the other operand's fragment
template <bool F32, int HDP, class X> __device__ __forceinline__ void mul_rows(const SAddr<F32, HDP>& f, X&& x, f32x16& st) {
  constexpr int NF = HDP / 16, PF = NF < 4 ? NF : (F32 ? 2 : 4), R = SGeo<F32, HDP>::FR;
  SFrag<F32> fr[NF];
  static_for<PF>([&](auto I) { f.template row<I, 0>(fr[I]); });
  static_for<NF>([&](auto I) {
    constexpr int i = I, nx = i + PF;
    if constexpr (nx < NF) f.template row<nx, 0>(fr[nx]);
    SAddr<F32, HDP>::template wait<R * (NF - 1 - i < PF ? NF - 1 - i : PF)>(fr[i]);
    st = smma<F32>(fr[i], x(I), st);
    if (!F32) SCORE_PIN();
  });
}
// st += X . x and dp += Y . y of two tiles OFF bytes apart, the two accumulators in turn
template <bool F32, int HDP, int OFF, class X, class Y>
__device__ __forceinline__ void mul_rows2(const SAddr<F32, HDP>& f, X&& x, Y&& y, f32x16& st, f32x16& dp) {
  constexpr int NF = 2 * (HDP / 16), PF = F32 ? 2 : 4, R = SGeo<F32, HDP>::FR;
  SFrag<F32> fr[NF];
  auto get = [&](auto I) { f.template row<(I >> 1), (I & 1) * OFF>(fr[I]); };
  static_for<PF>(get);
  static_for<NF>([&](auto I) {
    constexpr int i = I, nx = i + PF;
    if constexpr (nx < NF) get(std::integral_constant<int, nx>{});
    SAddr<F32, HDP>::template wait<R * (NF - 1 - i < PF ? NF - 1 - i : PF)>(fr[i]);
    if constexpr (i & 1) dp = smma<F32>(fr[i], y(std::integral_constant<int, (i >> 1)>{}), dp);
    else st = smma<F32>(fr[i], x(std::integral_constant<int, (i >> 1)>{}), st);
    if (!F32) SCORE_PIN();
  });
}

// 4 channels c .. c + 3 of a row of T
template <bool F32> __device__ __forceinline__ void put4(void* base, long long off, float x0, float x1, float x2, float x3) {
  if constexpr (F32) *(f32x4*)((float*)base + off) = f32x4{x0, x1, x2, x3};
  else *(u32x2*)((u16*)base + off) = u32x2{pk2(x0, x1), pk2(x2, x3)};
}
// what rounding to bf16 took from 4 values, as bf16
__device__ __forceinline__ void put4_lo(void* base, long long off, float x0, float x1, float x2, float x3) {
  auto lo = [](float x) { return x - bf2f(f2bf(x)); };
  *(u32x2*)((u16*)base + off) = u32x2{pk2(lo(x0), lo(x1)), pk2(lo(x2), lo(x3))};
}
// A lane's row: x[d][4 g + e] is channel 32 d + 8 g + 4 h + e.  bf16: lane and lane ^ 32 hold 4 channels each of every 8; they swap one
// group of a pair, then 16-byte stores.  All lanes of the wave take part; ok false: nothing is written.
template <bool F32, int DB> __device__ __forceinline__ void store_row(void* base, long long off, const f32x16 (&x)[DB], float scale, int h, int D, bool ok) {
#pragma unroll
  for (int d = 0; d < DB; ++d) {
    if constexpr (F32) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = d * 32 + 8 * g + 4 * h;
        if (ok && c < D) put4<true>(base, off + c, x[d][4 * g] * scale, x[d][4 * g + 1] * scale, x[d][4 * g + 2] * scale, x[d][4 * g + 3] * scale);
      }
    } else {
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        const int ge = 8 * pr, go = 8 * pr + 4;
        const unsigned e0 = pk2(x[d][ge] * scale, x[d][ge + 1] * scale), e1 = pk2(x[d][ge + 2] * scale, x[d][ge + 3] * scale);
        const unsigned o0 = pk2(x[d][go] * scale, x[d][go + 1] * scale), o1 = pk2(x[d][go + 2] * scale, x[d][go + 3] * scale);
        const u32x2 s0 = __builtin_amdgcn_permlane32_swap(e0, o0, false, false);
        const u32x2 s1 = __builtin_amdgcn_permlane32_swap(e1, o1, false, false);
        const int c = d * 32 + 8 * (2 * pr + h);
        if (ok && c < D) *(u32x4*)((u16*)base + off + c) = u32x4{s0[0], s1[0], s0[1], s1[1]};
      }
    }
  }
}
template <int DB> __device__ __forceinline__ void store_part(float* base, long long off, const f32x16 (&x)[DB], int h, int D) {
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = d * 32 + 8 * g + 4 * h;
      if (c < D) *(f32x4*)(base + off + c) = f32x4{x[d][4 * g], x[d][4 * g + 1], x[d][4 * g + 2], x[d][4 * g + 3]};
    }
}

__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ u64 scalar64(u64 v) {
  return ((u64)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)v);
}
// the keys of a tile (document of key kv0 + lane in kd) that belong to this lane's document: one ballot per document among the lanes
__device__ __forceinline__ u64 doc_bits(int qd, int kd) {
  u64 bits = 0ull, todo = ~0ull;
  while (todo != 0ull) {
    const int d = __builtin_amdgcn_readlane(qd, __builtin_ctzll(todo));
    const u64 hit = __ballot(kd == d && kd >= 0);
    const bool mine = qd == d;
    if (mine) bits = hit;
    todo &= ~__ballot(mine);
  }
  return bits;
}

// Up to 64 tiles of 64 items against the range of documents [dmin, dmax] of the other side: which tiles hold an item that may be inside
// the range (vis), only items of the range's one document (full), an item of a negative document (neg).  Four threads a tile, 16 items
// each; all four waves take part.
struct DocChunk { u64 vis, full, neg; };
__device__ __forceinline__ DocChunk doc_chunk(const int* __restrict__ doc, int tile0, int tiles, int items, int dmin, int dmax, u64 (*sh)[3], int wave, int lane) {
  const int t = wave * 16 + (lane >> 2), i0 = (tile0 + t) * 64 + (lane & 3) * 16;
  int lo = 0x7fffffff, up = -1, any = 0;                 // of the documents that are not negative; negative ones seen
  if (t < tiles && i0 < items) {
    if (i0 + 16 <= items) {
      struct __attribute__((packed, aligned(4))) I4 { int v[4]; };
      I4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = *(const I4*)(doc + i0 + 4 * k);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int d = x[k >> 2].v[k & 3];
        lo = (int)min((unsigned)lo, (unsigned)d);
        up = max(up, d);
        any |= d;
      }
    } else {
      for (int k = 0; k < items - i0; ++k) {
        const int d = doc[i0 + k];
        lo = (int)min((unsigned)lo, (unsigned)d);
        up = max(up, d);
        any |= d;
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min(lo, __shfl_xor(lo, o, 64));
    up = max(up, __shfl_xor(up, o, 64));
    any |= __shfl_xor(any, o, 64);
  }
  const bool in = t < tiles, first = (lane & 3) == 0;
  // bit 4 k of a ballot is tile 16 wave + k: every fourth bit is gathered to the low 16
  auto gather = [](u64 b) {
    b &= 0x1111111111111111ull;
    b = (b | b >> 3) & 0x0303030303030303ull;
    b = (b | b >> 6) & 0x000f000f000f000full;
    b = (b | b >> 12) & 0x000000ff000000ffull;
    return (b | b >> 24) & 0xffffull;
  };
  const u64 vis = gather(__ballot(first && in && lo <= dmax && up >= dmin)), full = gather(__ballot(first && in && lo == up && up == dmin && dmin == dmax && any >= 0)),
            neg = gather(__ballot(first && in && any < 0));
  __syncthreads();
  if (lane == 0) { sh[wave][0] = vis << (16 * wave); sh[wave][1] = full << (16 * wave); sh[wave][2] = neg << (16 * wave); }
  __syncthreads();
  DocChunk c;
  c.vis = scalar64(sh[0][0] | sh[1][0] | sh[2][0] | sh[3][0]);
  c.full = scalar64(sh[0][1] | sh[1][1] | sh[2][1] | sh[3][1]);
  c.neg = scalar64(sh[0][2] | sh[1][2] | sh[2][2] | sh[3][2]);
  return c;
}
// the tiles t of [t_lo, t_end) a workgroup visits, in order: all of them, or, with documents, those whose range meets the workgroup's own
template <bool DOC> struct TileWalk {
  const int* doc;
  int t_end, items, dmin, dmax, base;       // base: first tile of the chunk in hand
  DocChunk c;
  bool full, neg;
  __device__ __forceinline__ int chunk_from(int t, u64 (*sh)[3], int wave, int lane) {
    for (base = t; base < t_end; base += 64) {
      c = doc_chunk(doc, base, min(64, t_end - base), items, dmin, dmax, sh, wave, lane);
      if (c.vis != 0ull) return take();
    }
    return -1;
  }
  __device__ __forceinline__ int take() {
    const int i = __builtin_ctzll(c.vis);
    c.vis &= c.vis - 1ull;
    full = (c.full >> i) & 1ull;
    neg = (c.neg >> i) & 1ull;
    return base + i;
  }
  __device__ __forceinline__ int first(int t_lo, u64 (*sh)[3], int wave, int lane) {
    full = true;
    neg = false;
    if (!DOC) return t_lo < t_end ? t_lo : -1;
    return dmin > dmax ? -1 : chunk_from(t_lo, sh, wave, lane);
  }
  __device__ __forceinline__ int next(int t, u64 (*sh)[3], int wave, int lane) {
    if (!DOC) return t + 1 < t_end ? t + 1 : -1;
    return c.vis != 0ull ? take() : chunk_from(base + 64, sh, wave, lane);
  }
};

// A walk over the halves (32 items) [s_lo, items / 32) of 64-item tiles in steps of T = 64 or 32 items.  s: the step in hand starts at item 32 s
// (a step of 64 at an even half, whether or not the range holds both of its halves: see `mine`), -1 at the end.
template <bool DOC, int T> struct StepWalk {
  TileWalk<DOC> w;
  int s, s_lo, items;
  bool full, neg;
  __device__ __forceinline__ void first(u64 (*sh)[3], int wave, int lane) {
    const int t = w.first(s_lo >> 1, sh, wave, lane);
    s = t < 0 ? -1 : T == 64 ? 2 * t : max(2 * t, s_lo);
    if (s >= 0 && s * 32 >= items) s = -1;
    full = w.full;
    neg = w.neg;
  }
  __device__ __forceinline__ void next(u64 (*sh)[3], int wave, int lane) {
    if (T == 32 && !(s & 1) && (s + 1) * 32 < items) { ++s; return; }
    const int t = w.next(s >> 1, sh, wave, lane);
    s = t < 0 ? -1 : 2 * t;
    full = w.full;
    neg = w.neg;
  }
  __device__ __forceinline__ bool mine(int half) const { return half >= s_lo && half * 32 < items; }
};

// range of the documents of a workgroup's 128 rows (d: this lane's row, live: it takes part) for a walk
__device__ __forceinline__ void doc_range(int d, bool live, int* sh, int wave, int lane, int& dmin, int& dmax) {
  const int lo = wave_min_i(live ? d : 0x7fffffff), up = -wave_min_i(live ? -d : 0x7fffffff);
  if (lane == 0) { sh[wave] = lo; sh[4 + wave] = up; }
  __syncthreads();
  dmin = __builtin_amdgcn_readfirstlane(min(min(sh[0], sh[1]), min(sh[2], sh[3])));
  dmax = __builtin_amdgcn_readfirstlane(max(max(sh[4], sh[5]), max(sh[6], sh[7])));
}
// Which block of rows (0: the one that sees most) and which group this workgroup has; `per` consecutive groups share keys.  Where the blocks differ
// in work (causal), the heaviest of ALL groups come first, so that the light ones fill up the end.  A chiplet keeps the groups that share
// keys (workgroups are dealt to the 8 chiplets in turn) and, where they divide evenly, takes samples with stride 8, for the sake of ragged lengths.
// Against one head after the other (heaviest block first within each): 4 x 4096 causal, 8 heads of 128, forward 170 -> 152 us; 32 x 708 with a
// prefix, 4 heads of 192, backward 272 -> 226; documents in 8192 tokens, 16 heads of 64, forward 107 -> 92, backward 349 -> 294.
__device__ __forceinline__ void order_blocks(int nb, int per, bool uneven, int& block, int& group) {
  const int n = gridDim.x / nb;
  if (!uneven) {
    const int l = xcd_remap(blockIdx.x, gridDim.x);
    block = l % nb;
    group = l / nb;
    return;
  }
  const int g = blockIdx.x % n, y = g >> 3;
  block = blockIdx.x / n;
  group = n / per % 8 == 0 ? (8 * (y / per) + (g & 7)) * per + y % per : n % 8 == 0 ? (g & 7) * (n >> 3) + y : g;
}
// Distances count from the position among the keys that is nearest to the query's: the rest is the same for every key of the row, so the softmax
// and its gradients do not know it, and beside it -- 2^20 positions times a slope -- fp32 would lose the scores (slope 0.5 at position 10^6 on 300
// keys: probabilities off by several per cent).  The stored log-sum-exp lacks it as well.
__device__ __forceinline__ int near_pos(const TfScoreAttnArgs& a, int p) { return min(max(p, 0), a.Sk - 1); }
// what a query row may see: everything below follows from these
struct QRow { int p, lim, lim_lo, lim_hi; };       // position for distances; last visible key of this row, of the wave's first row, of its last
__device__ __forceinline__ QRow q_row(const TfScoreAttnArgs& a, int p0, int pfx, int w0, int i) {
  QRow q;
  q.p = near_pos(a, p0 + i);
  q.lim = a.causal ? min(max(p0 + i, pfx - 1), a.Sk - 1) : a.Sk - 1;
  q.lim_lo = a.causal ? min(max(p0 + w0, pfx - 1), a.Sk - 1) : a.Sk - 1;
  q.lim_hi = a.causal ? min(max(p0 + min(w0 + 31, a.Sq - 1), pfx - 1), a.Sk - 1) : a.Sk - 1;
  return q;
}
// one past the last key that query i_last (or an earlier one) sees
__device__ __forceinline__ int key_end(const TfScoreAttnArgs& a, int p0, int pfx, int i_last) {
  return a.causal ? max(0, min(max(p0 + i_last + 1, pfx), a.Sk)) : a.Sk;
}
__device__ __forceinline__ unsigned low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// body(FULL, CAP, SLP) with the flags (all uniform over the wave) as compile-time constants: the loops over a tile's scores stay free of
// branches and of registers that only one of their forms needs.  CAP: 0 none, 1 score by score (cap_each), 2 the cap's polynomial
template <class F> __device__ __forceinline__ void by_flags(bool full, int cap, bool slp, F&& body) {
  auto three = [&](auto FULL, auto CAP) { if (slp) body(FULL, CAP, std::true_type{}); else body(FULL, CAP, std::false_type{}); };
  auto two = [&](auto FULL) {
    if (cap == 2) three(FULL, std::integral_constant<int, 2>{});
    else if (__builtin_expect(cap == 1, false)) three(FULL, std::integral_constant<int, 1>{});
    else three(FULL, std::integral_constant<int, 0>{});
  };
  if (full) two(std::true_type{}); else two(std::false_type{});
}

// Launches KERN with `bytes` of dynamic LDS (always the same for a kernel).  What lies beyond the default limit is granted per kernel and device: a
// kernel is a template value here, so each has a flag of its own (a flag per type would be shared by all widths), set once the runtime has agreed.
template <auto KERN, class... Args> int launch_lds(int blocks, size_t bytes, hipStream_t st, Args... args) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return (int)e;
  if (dev > 63 || !(done.load(std::memory_order_relaxed) >> dev & 1ull)) {
    e = hipFuncSetAttribute((const void*)KERN, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) return (int)e;
    if (dev <= 63) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  hipLaunchKernelGGL(KERN, dim3(blocks), dim3(256), bytes, st, args...);
  return (int)hipGetLastError();
}

// Ways to split the `units` (tiles of keys or queries) of a loop that `blocks` workgroups run.  bf16: until two workgroups a CU are there, `least` units
// each.  fp32, where a unit is sixteen times the matrix work: down to one unit, as long as all workgroups run at once (two a CU up to 64 channels, then
// one) and only if that shortens the longest loop.  2 x 355 x 417, 6 heads of 88, fp32 (36 workgroups): forward 54 -> 24 us with the join, dq 34 -> 26, dk / dv 38 -> 30.
inline int split_ways(bool f32, int D, long long blocks, long long units, int least) {
  if (blocks == 0 || units <= 1) return 1;
  if (!f32) return (int)std::max(1ll, blocks >= 256 ? 1ll : std::min((512 + blocks - 1) / blocks, units / least));
  const long long ways = std::max(1ll, std::min((D <= 64 ? 512 : 256) / blocks, units)), each = (units + ways - 1) / ways;
  return (int)((units + each - 1) / each);
}

inline int score_check(const TfScoreAttnArgs* a) {
  if (a->B < 0 || a->Sq < 0 || a->Sk < 0 || a->H <= 0 || a->Hk <= 0 || a->H % a->Hk != 0) return -1;
  if (a->D <= 0 || a->D > 256 || a->D % 8 != 0) return -2;
  // (their quotient and its square stay finite)
  if (!(fabsf(a->scale) <= 1e10f) || !(a->softcap == 0.f || (a->softcap >= 1e-10f && a->softcap <= 1e10f))) return -3;
  if ((a->k_doc == nullptr) != (a->q_doc == nullptr) && a->Sq > 0 && a->Sk > 0) return -4;
  const long long blocks = (long long)a->B * std::max(a->H * ((a->Sq + 127ll) / 128), (long long)a->Hk * ((a->Sk + 127) / 128));
  if (blocks > 0x3fffff || (long long)a->Sq + a->Sk > (1ll << 30)) return -5;
  return 0;
}
// (64 rows of a tile are addressed with 32-bit offsets)
inline bool score_aligned(const void* p, long long sb, long long ss, long long sh, int e) {
  return (((uintptr_t)p) & 15) == 0 && sb >= 0 && ss >= 0 && sh >= 0 && ss < (1ll << 30) / 64 / e && sb * e % 16 == 0 && ss * e % 16 == 0 && sh * e % 16 == 0;
}


inline int hdp_of(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : D <= 192 ? 192 : 256; }
template <class Fn> int by_head_dim(const TfScoreAttnArgs* a, Fn&& fn) {
  auto pick = [&](auto f32) {
    switch (hdp_of(a->D)) {
      case 32: return fn(f32, std::integral_constant<int, 32>{});
      case 64: return fn(f32, std::integral_constant<int, 64>{});
      case 96: return fn(f32, std::integral_constant<int, 96>{});
      case 128: return fn(f32, std::integral_constant<int, 128>{});
      case 192: return fn(f32, std::integral_constant<int, 192>{});
      default: return fn(f32, std::integral_constant<int, 256>{});
    }
  };
  return a->is_f32 ? pick(std::true_type{}) : pick(std::false_type{});
}


}  // namespace
