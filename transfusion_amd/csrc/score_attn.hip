// Attention whose scores are changed before the softmax: capped by a tanh, biased by distance, masked by documents and by a causal
// horizon with a bidirectional prefix.  For query i at position p and key j of one head
//   s = scale * q.k ;  s = cap * tanh(s / cap) (cap > 0) ;  s -= slope_h * |p - j| ;
//   hidden unless  doc_q == doc_k >= 0  and  (not causal or j <= p or j < prefix) ;   P = softmax_j(s) ;  o = P v .
// A row that attends nothing gives o = 0 and no gradient.  Heads may share keys and values (H / Hk heads each).
//
// No [Sq, Sk] tensor reaches memory: the forward keeps a running maximum and sum and stores one log-sum-exp a row, the backward forms P
// again from it.  Orientation as in attn_bf16.hip: the score tile is computed transposed (keys in the accumulator registers, the query
// on the lane), so a row's statistics are one scalar a lane and the tile is the next product's operand as it stands.
//   score_fwd_kernel   query on the lane, loops over key tiles                       -> o, lse
//   score_dq_kernel    query on the lane, loops over key tiles                       -> dq, delta = rowsum(dO o), the slopes' row sums
//   score_dkv_kernel   key on the lane, loops over the heads of its group and their query tiles -> dk, dv (no atomics)
// Scores, statistics and accumulators are fp32.  P and dS are rounded to the operand type of the next product (bf16: half a step, 2^-9
// of each term); fp32 tensors run on the fp32 matrix instructions throughout.
#include "tf_common.h"
#include "tf_kernels.h"
#include "attn_common.h"
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

template <bool F32, int HDP> struct STile {
  static constexpr int ESZ = F32 ? 4 : 2;
  static constexpr int STR = F32 ? HDP * 4 + 16 : Geo<HDP>::TSTR;       // fp32: rows 4 banks apart
  static constexpr int CPR = HDP * ESZ / 16;                            // 16-byte pieces of a row
  static __device__ __forceinline__ int off(int row, int c) {
    if constexpr (F32) return row * STR + c * 16;
    else return tile_off(row, c, STR);
  }
  // rows row0 .. row0 + ROWS - 1 of a [*, row_bytes] matrix into LDS; rows at or beyond row_end, rows whose document is negative and
  // channels at or beyond D arrive as zeros, whatever memory holds there
  template <int ROWS> static __device__ __forceinline__ void stage(unsigned char* lds, const char* base, long long row_bytes, int row0, int row_end,
                                                                   const int* doc, int D, int tid) {
    for (int id = tid; id < ROWS * CPR; id += 256) {
      const int r = id / CPR, c = id % CPR, gr = row0 + r;
      u32x4 v = {0, 0, 0, 0};
      if (gr < row_end && c * (16 / ESZ) < D && (doc == nullptr || doc[gr] >= 0)) v = *(const u32x4*)(base + (long long)gr * row_bytes + c * 16);
      *(u32x4*)(lds + off(r, c)) = v;
    }
  }
  static __device__ __forceinline__ SFrag<F32> row(const unsigned char* tile, int row0, int ks, int lane) {
    SFrag<F32> f;
    if constexpr (F32) {
      const unsigned char* p = tile + (row0 + (lane & 31)) * STR + (ks * 16 + 8 * (lane >> 5)) * 4;
      f.a = *(const f32x4*)p;
      f.b = *(const f32x4*)(p + 16);
    } else {
      f.v = *(const u32x4*)(tile + tile_off(row0 + (lane & 31), 2 * ks + (lane >> 5), STR));
    }
    return f;
  }
  // c[channel col0 + ..][lane's row] += sum over 32 tile rows (krow0 ..) of tile[row][channel] * p[row]: p is an accumulator tile
  static __device__ __forceinline__ f32x16 mma_t(const unsigned char* tile, int krow0, int col0, const f32x16& p, f32x16 c, int lane) {
    if constexpr (F32) {
      const float* t = (const float*)(tile + (krow0 + 4 * (lane >> 5)) * STR) + col0 + (lane & 31);
#pragma unroll
      for (int r = 0; r < 16; ++r) c = __builtin_amdgcn_mfma_f32_32x32x2f32(t[((r & 3) + 8 * (r >> 2)) * (STR / 4)], p[r], c, 0, 0, 0);
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_frag<HDP>(tile, krow0 + 16 * s, col0, lane), acc_frag(p, s), c, 0, 0, 0);
    }
    return c;
  }
};

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
template <bool F32> __device__ __forceinline__ float frag_dot(const SFrag<F32>& x, const SFrag<F32>& y) {
  float s = 0.f;
  if constexpr (F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s += x.a[e] * y.a[e] + x.b[e] * y.b[e];
  } else {
    float a[8], b[8];
    unpack8(x.v, a);
    unpack8(y.v, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += a[e] * b[e];
  }
  return s;
}

// ---- the change of a score, in the log2 domain ----
struct SMod {
  float sc;          // no cap: scale * log2 e;  cap: 2 log2 e * scale / cap (the exponent of the tanh)
  float capl;        // cap * log2 e, or 0
  float slope2;      // slope * log2 e
};
template <bool F32> __device__ __forceinline__ float tanh_of(float y2) {       // y2 = 2 log2(e) y
  if constexpr (F32) return tanhf(y2 * 0.34657359027997264f);
  // 1 - 2 / (1 + e^2y): absolute error ~1e-7 (the bf16 product's own error is larger); +-inf give +-1, no NaN in between
  return 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + fast_exp2(y2));
}
__device__ __forceinline__ SMod smod(const TfScoreAttnArgs& a, int head) {
  SMod m;
  m.capl = a.softcap > 0.f ? a.softcap * LOG2E : 0.f;
  m.sc = a.softcap > 0.f ? 2.f * LOG2E * a.scale / a.softcap : a.scale * LOG2E;
  m.slope2 = a.slopes != nullptr ? a.slopes[head] * LOG2E : 0.f;
  return m;
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

// ================================================================================================
// forward
// ================================================================================================
template <bool F32, int HDP>
__global__ __launch_bounds__(256, 1) void score_fwd_kernel(const TfScoreAttnArgs a, int nqb, int nsplit, int split_tiles) {
  using T = STile<F32, HDP>;
  constexpr int KT = F32 ? 32 : 64, NKB = KT / 32, KS = HDP / 16, DB = HDP / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* kt = smem;
  unsigned char* vt = smem + KT * T::STR;
  int* docs = (int*)(smem + 2 * KT * T::STR);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const int logical = xcd_remap(blockIdx.x, gridDim.x);
  const int split = logical % nsplit, t1 = logical / nsplit;
  const int qb = nqb - 1 - t1 % nqb, bh = t1 / nqb, b = bh / a.H, head = bh % a.H, kvh = head / (a.H / a.Hk);
  const char* qbase = (const char*)a.q + ((long long)b * a.q_sb + (long long)head * a.q_sh) * T::ESZ;
  const char* kbase = (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * T::ESZ;
  const char* vbase = (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * T::ESZ;
  const int* kdoc = a.k_doc != nullptr ? a.k_doc + (size_t)b * a.Sk : nullptr;
  const SMod m = smod(a, head);
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const int i = qb * 128 + wave * 32 + (lane & 31);
  const int qd = kdoc != nullptr && i < a.Sq ? a.q_doc[(size_t)b * a.Sq + i] : 0;
  const bool live = i < a.Sq && qd >= 0;
  const int p = p0 + i;
  const int lim = !live ? -1 : (a.causal ? min(max(p, pfx - 1), a.Sk - 1) : a.Sk - 1);       // last key this row may see
  const int i_last = min(qb * 128 + 127, a.Sq - 1);
  const int hi = a.causal ? min(max(p0 + i_last + 1, pfx), a.Sk) : a.Sk;                      // one past the block's last
  const int tile_end = (max(hi, 0) + KT - 1) / KT;
  const int t_lo = split * split_tiles, t_hi = min(tile_end, t_lo + split_tiles);
  SFrag<F32> qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = gfrag<F32>(qbase + (long long)min(i, a.Sq - 1) * a.q_ss * T::ESZ, ks, h, a.D, live);
  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m_run = S_NEG, l_run = 0.f;
  for (int t = t_lo; t < t_hi; ++t) {
    const int kv0 = t * KT;
    __syncthreads();
    T::template stage<KT>(kt, kbase, a.k_ss * T::ESZ, kv0, hi, kdoc, a.D, tid);
    T::template stage<KT>(vt, vbase, a.v_ss * T::ESZ, kv0, hi, kdoc, a.D, tid);
    if (kdoc != nullptr && tid < KT) docs[tid] = kv0 + tid < a.Sk ? kdoc[kv0 + tid] : -1;
    __syncthreads();
    f32x16 st[NKB];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) st[kb][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) st[kb] = smma<F32>(T::row(kt, kb * 32, ks, lane), qf[ks], st[kb]);
    }
    const float pd = (float)(p - kv0 - 4 * h);
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = kb * 32 + (r & 3) + 8 * (r >> 2);
        float x = m.capl != 0.f ? m.capl * tanh_of<F32>(st[kb][r] * m.sc) : st[kb][r] * m.sc;
        if (m.slope2 != 0.f) x -= m.slope2 * fabsf(pd - (float)j);
        bool vis = kv0 + j + 4 * h <= lim;
        if (kdoc != nullptr) vis = vis && docs[j + 4 * h] == qd;
        st[kb][r] = vis ? x : -INFINITY;
      }
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[kb][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float m_new = fmaxf(m_run, mx), alpha = fast_exp2(m_run - m_new);
    m_run = m_new;
    l_run *= alpha;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        st[kb][r] = fast_exp2(st[kb][r] - m_run);
        l_run += st[kb][r];
      }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) o[d] = T::mma_t(vt, kb * 32, d * 32, st[kb], o[d], lane);
  }
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  if (i >= a.Sq) return;
  const long long rows = (long long)a.B * a.H * a.Sq, row = (long long)bh * a.Sq + i;
  if (nsplit > 1) {                       // unnormalised part of this range of keys; score_join_kernel adds them up
    float* po = (float*)a.work + ((long long)split * rows + row) * a.D;
    float* pml = (float*)a.work + (long long)nsplit * rows * a.D + ((long long)split * rows + row) * 2;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = d * 32 + 8 * g + 4 * h;
        if (c < a.D) *(f32x4*)(po + c) = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
      }
    if (h == 0) { pml[0] = m_run; pml[1] = l_tot; }
    return;
  }
  const float inv = l_tot == 0.f ? 0.f : 1.0f / l_tot;
  char* orow = (char*)a.out + (((long long)b * a.Sq + i) * a.H + head) * a.D * T::ESZ;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = d * 32 + 8 * g + 4 * h;
      if (c >= a.D) continue;
      const float x0 = o[d][4 * g] * inv, x1 = o[d][4 * g + 1] * inv, x2 = o[d][4 * g + 2] * inv, x3 = o[d][4 * g + 3] * inv;
      if constexpr (F32) *(f32x4*)(orow + c * 4) = f32x4{x0, x1, x2, x3};
      else *(u32x2*)(orow + c * 2) = u32x2{pack2bf(x0, x1), pack2bf(x2, x3)};
    }
  // rows without keys: +inf, so that every probability formed from it again is 0
  if (h == 0 && a.lse != nullptr) a.lse[row] = l_tot == 0.f ? INFINITY : m_run + log2f(l_tot);
}

// ================================================================================================
// forward, bf16
// ================================================================================================
// LDS tiles of the bf16 kernels: 64 rows of HDP channels at a stride of an ODD multiple of 64 bytes, 16-byte piece ^= (row >> 2) & 3:
// four consecutive rows start 16 banks apart in some order, so row reads (ds_read_b128) and transposed reads (ds_read_b64_tr_b16) are
// both free of conflicts -- at the smallest such stride (192 bytes for 64 channels, 448 for 192).
template <int HDP> struct SGeo {
  static constexpr int STR = ((HDP * 2 + 63) / 64 | 1) * 64;
  static constexpr int KS = HDP / 16, DB = HDP / 32, TILE = 64 * STR;
};
// LDS-DMA of a 64-row tile by four waves: the image is linear in the lane, so the layout lives on the source side.  Pieces at or beyond D
// get an offset behind the buffer's end and arrive as zeros, as do rows beyond its last.
template <int HDP> struct SDma {
  static constexpr int T = SGeo<HDP>::STR, NI = 64 * T / 4096;
  static constexpr unsigned OUT = 0x7fffff00u;
  unsigned off[NI], rb;       // offsets for rows of rb bytes; a matrix with other rows has them formed where it is read
  int wave, lane;
  __device__ __forceinline__ unsigned offset(int i, unsigned row_bytes, int D) const {
    const int pos = (wave * NI + i) * 1024 + lane * 16, r = pos / T, cp = (pos % T) >> 4, c = cp ^ ((r >> 2) & 3);
    return cp >= HDP / 8 || c * 8 >= D ? OUT : (unsigned)r * row_bytes + c * 16;
  }
  __device__ __forceinline__ SDma(int wave_, int lane_, unsigned row_bytes, int D) : rb(row_bytes), wave(wave_), lane(lane_) {
#pragma unroll
    for (int i = 0; i < NI; ++i) off[i] = offset(i, row_bytes, D);
  }
  __device__ __forceinline__ int row(int i) const { return ((wave * NI + i) * 1024 + lane * 16) / T; }
  // rows row0 .. of the matrix at base, row_end excluded; doc != null: rows of negative documents are zeros too (few tiles hold any)
  __device__ __forceinline__ void issue(const char* base, unsigned row_bytes, int row0, int row_end, int D, const int* doc, unsigned char* tile) const {
    const int n = min(64, row_end - row0);
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)(base + (long long)row0 * row_bytes), 0, (int)((unsigned)(n - 1) * row_bytes + D * 2), 0x00020000);
    if (doc == nullptr && row_bytes == rb) {
#pragma unroll
      for (int i = 0; i < NI; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, TF_LDS_PTR(tile + (wave * NI + i) * 1024), 16, (int)off[i], 0, 0, 0);
    } else {
      for (int i = 0; i < NI; ++i) {
        const unsigned o = doc != nullptr && doc[row0 + min(row(i), n - 1)] < 0 ? OUT : offset(i, row_bytes, D);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, TF_LDS_PTR(tile + (wave * NI + i) * 1024), 16, (int)o, 0, 0, 0);
      }
    }
  }
};
// per-lane LDS addresses of row fragments (32 rows x 16 channels) and transposed fragments of such a tile; see attn_common.h FragAddr
template <int HDP> struct SAddr {
  static constexpr int T = SGeo<HDP>::STR;
  unsigned row_e, row_o, tr_a, tr_b;
  __device__ __forceinline__ SAddr(unsigned tile, int lane) {
    const int r = lane & 31, x = (r >> 2) & 3, hh = lane >> 5;
    row_e = tile + r * T + ((hh ^ x) << 4);
    row_o = tile + r * T + (((2 + hh) ^ x) << 4);
    const int li = lane & 15, q4 = li >> 2, p = li & 3, cb = (lane >> 4) & 1, low2 = 2 * cb + (p >> 1);
    tr_a = tile + (4 * hh + q4) * T + ((low2 ^ hh) << 4) + (p & 1) * 8;
    tr_b = tile + (4 * hh + q4 + 8) * T + ((low2 ^ (hh + 2)) << 4) + (p & 1) * 8;
  }
  template <int ROW0, int KS> __device__ __forceinline__ u32x4 row() const { return rd128_asm<ROW0 * T + 64 * (KS >> 1)>((KS & 1) ? row_o : row_e); }
  template <int KROW0, int COL0> __device__ __forceinline__ void tr(u64& a, u64& b) const {
    a = tr_read_asm<KROW0 * T + 2 * COL0>(tr_a);
    b = tr_read_asm<KROW0 * T + 2 * COL0>(tr_b);
  }
};

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

// 64-tile chunks of a row of 64-item tiles against a range of documents [dmin, dmax] of the other side: which tiles hold an item inside the
// range (vis), only items of the range's one document (full), an item of a negative document (neg).  Called by all four waves.
struct DocChunk { u64 vis, full, neg; };
__device__ __forceinline__ DocChunk doc_chunk(const int* __restrict__ doc, int tile0, int tiles, int items, int dmin, int dmax, u64 (*sh)[3], int wave, int lane) {
  u64 vis = 0ull, full = 0ull, neg = 0ull;
#pragma unroll 4
  for (int s = 0; s < 16; ++s) {
    const int t = s * 4 + wave;
    if (t >= tiles) break;
    const int i = (tile0 + t) * 64 + lane;
    const bool in = i < items;
    const int d = in ? doc[i] : -1;
    if (__any(d >= dmin && d <= dmax)) vis |= 1ull << t;
    if (__all(!in || d == dmin) && dmin == dmax) full |= 1ull << t;
    if (__any(in && d < 0)) neg |= 1ull << t;
  }
  __syncthreads();
  if (lane == 0) { sh[wave][0] = vis; sh[wave][1] = full; sh[wave][2] = neg; }
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

// 128 queries a workgroup (32 a wave, on the lane), 64-key tiles by LDS-DMA: V(t) travels under S(t) and the softmax, K(t + 1) under PV(t).
// Two workgroups a CU (heads <= 192) hide the barriers of one behind the matrix work of the other.
// DOC: documents are given.
template <int HDP, bool DOC>
__global__ __launch_bounds__(256, (HDP <= 192 ? 2 : 1)) void score_fwd16_kernel(const TfScoreAttnArgs a, int nqb, int nsplit, int split_tiles) {
  using G = SGeo<HDP>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* kt = smem;
  unsigned char* vt = smem + G::TILE;
  u64 (*dsh)[3] = (u64 (*)[3])(smem + 2 * G::TILE);
  int* rsh = (int*)(smem + 2 * G::TILE + 96);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int logical = xcd_remap(blockIdx.x, gridDim.x);
  const int split = logical % nsplit, t1 = logical / nsplit;
  const int qb = nqb - 1 - t1 % nqb, bh = t1 / nqb, b = bh / a.H, head = bh % a.H, kvh = head / (a.H / a.Hk);
  const char* qbase = (const char*)a.q + ((long long)b * a.q_sb + (long long)head * a.q_sh) * 2;
  const char* kbase = (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * 2;
  const char* vbase = (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * 2;
  const unsigned krb = (unsigned)a.k_ss * 2, vrb = (unsigned)a.v_ss * 2;
  const int* kdoc = DOC ? a.k_doc + (size_t)b * a.Sk : nullptr;
  const SMod m = smod(a, head);
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const int w0 = qb * 128 + wave * 32, i = w0 + (lane & 31), ic = min(i, a.Sq - 1);
  const int qd = DOC ? a.q_doc[(size_t)b * a.Sq + ic] : 0;
  const bool live = i < a.Sq && qd >= 0, wave_live = w0 < a.Sq;
  const int p = p0 + i;
  const int lim = a.causal ? min(max(p, pfx - 1), a.Sk - 1) : a.Sk - 1;
  const int lim_lo = a.causal ? min(max(p0 + w0, pfx - 1), a.Sk - 1) : a.Sk - 1;                       // of the wave's first row
  const int lim_hi = a.causal ? min(max(p0 + min(w0 + 31, a.Sq - 1), pfx - 1), a.Sk - 1) : a.Sk - 1;   // of its last
  const int hi = a.causal ? min(max(p0 + min(qb * 128 + 127, a.Sq - 1) + 1, pfx), a.Sk) : a.Sk;
  TileWalk<DOC> walk{kdoc, min((max(hi, 0) + 63) / 64, (split + 1) * split_tiles), a.Sk, 0, 0, 0, {}, true, false};
  if (DOC) {                  // the documents of the block's rows
    const int lo = wave_min_i(live ? qd : 0x7fffffff), up = -wave_min_i(live ? -qd : 0x7fffffff);
    if (lane == 0) { rsh[wave] = lo; rsh[4 + wave] = up; }
    __syncthreads();
    walk.dmin = __builtin_amdgcn_readfirstlane(min(min(rsh[0], rsh[1]), min(rsh[2], rsh[3])));
    walk.dmax = __builtin_amdgcn_readfirstlane(max(max(rsh[4], rsh[5]), max(rsh[6], rsh[7])));
  }
  u32x4 qf[G::KS];
#pragma unroll
  for (int ks = 0; ks < G::KS; ++ks) qf[ks] = gfrag<false>(qbase + (long long)ic * a.q_ss * 2, ks, h, a.D, live).v;
  f32x16 o[G::DB];
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m_run = S_NEG, l_run = 0.f;
  const bool changed = m.capl != 0.f || m.slope2 != 0.f || !(m.sc > 0.f);      // else the scale rides in the exponent's FMA
  const float scf = changed ? 1.0f : m.sc;
  const SAddr<HDP> fk(lds_addr_of(kt), lane), fv(lds_addr_of(vt), lane);
  const SDma<HDP> dma(wave, lane, krb, a.D);
  int t = walk.first(split * split_tiles, dsh, wave, lane);
  bool full = walk.full, neg = walk.neg;
  int kd_n = 0;
  if (t >= 0) {
    if (DOC) kd_n = t * 64 + lane < a.Sk ? kdoc[t * 64 + lane] : -1;
    dma.issue(kbase, krb, t * 64, hi, a.D, DOC && neg ? kdoc : nullptr, kt);
  }
  while (t >= 0) {
    const int kv0 = t * 64;
    const bool full_t = full && kv0 + 63 <= lim_lo, work = wave_live && kv0 <= lim_hi;
    const int kd = kd_n;
    dma_wait_barrier();                   // K(t) is there; every wave is done with V(t - 1)
    dma.issue(vbase, vrb, kv0, hi, a.D, DOC && neg ? kdoc : nullptr, vt);
    unsigned pk[2][8];
    if (work) {
      f32x16 st[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[kb][r] = 0.f;
      {
        constexpr int NF = 2 * G::KS, PF = 3;
        u32x4 fr[NF];
        static_for<(PF < NF ? PF : NF)>([&](auto I) { fr[I] = fk.template row<(I & 1) * 32, (I >> 1)>(); });
        static_for<NF>([&](auto I) {
          constexpr int x = I, nx = x + PF;
          if constexpr (nx < NF) fr[nx] = fk.template row<(nx & 1) * 32, (nx >> 1)>();
          lgkm_wait<(NF - 1 - x < PF ? NF - 1 - x : PF)>(fr[x]);
          st[x & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(fr[x]), as_bf16x8(qf[x >> 1]), st[x & 1], 0, 0, 0);
        });
      }
      if (changed) {                      // (workgroup-uniform)
        if (m.capl != 0.f) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) st[kb][r] = m.capl * tanh_of<false>(st[kb][r] * m.sc);
        } else {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) st[kb][r] *= m.sc;
        }
        if (m.slope2 != 0.f) {
          const float pd = (float)(p - kv0 - 4 * h);
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) st[kb][r] -= m.slope2 * fabsf(pd - (float)(kb * 32 + (r & 3) + 8 * (r >> 2)));
        }
      }
      if (!full_t) {
        const int n = lim - kv0 + 1;
        u64 bits = n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull;
        if (DOC) bits &= doc_bits(qd, kd);
        bits >>= 4 * h;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!((bits >> (kb * 32 + (r & 3) + 8 * (r >> 2))) & 1ull)) st[kb][r] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[kb][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * scf;
      const bool need = mx - m_run > RESCALE_THR;        // per row; the wave only skips the multiplication when no row needs it
      if (__any(need)) {
        const float m_new = need ? fmaxf(m_run, mx) : m_run, alpha = need ? fast_exp2(m_run - m_new) : 1.0f;
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < G::DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
      }
      float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float e0 = fast_exp2(fmaf(st[kb][r], scf, -m_run)), e1 = fast_exp2(fmaf(st[kb][r + 1], scf, -m_run));
          ps0 += e0;
          ps1 += e1;
          pk[kb][r >> 1] = pk2(e0, e1);
        }
      l_run += ps0 + ps1;
    }
    const int tn = walk.next(t, dsh, wave, lane);        // (may scan documents, with barriers of its own: all waves take part)
    full = walk.full;
    neg = walk.neg;
    dma_wait_barrier();                   // V(t) is there; every wave is done with K(t)
    if (tn >= 0) {
      if (DOC) kd_n = tn * 64 + lane < a.Sk ? kdoc[tn * 64 + lane] : -1;
      dma.issue(kbase, krb, tn * 64, hi, a.D, DOC && neg ? kdoc : nullptr, kt);
    }
    if (work) {
      constexpr int NF = 4 * G::DB, PF = 2;
      u64 fa[NF], fb[NF];
      bf16x8 pf[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int kb = g >> 1, s4 = 4 * (g & 1);
        pf[g] = as_bf16x8(u32x4{pk[kb][s4], pk[kb][s4 + 1], pk[kb][s4 + 2], pk[kb][s4 + 3]});
      }
      static_for<PF>([&](auto I) { fv.template tr<(I / G::DB) * 16, (I % G::DB) * 32>(fa[I], fb[I]); });
      static_for<NF>([&](auto I) {
        constexpr int x = I, nx = x + PF;
        if constexpr (nx < NF) fv.template tr<(nx / G::DB) * 16, (nx % G::DB) * 32>(fa[nx], fb[nx]);
        lgkm_wait<2 * (NF - 1 - x < PF ? NF - 1 - x : PF)>(fa[x], fb[x]);
        o[x % G::DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(join_tr64(fa[x], fb[x]), pf[x / G::DB], o[x % G::DB], 0, 0, 0);
      });
    }
    t = tn;
  }
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  const long long rows = (long long)a.B * a.H * a.Sq, row = (long long)bh * a.Sq + i;
  const bool none = !live || l_tot == 0.f;
  if (nsplit > 1) {
    if (i >= a.Sq) return;
    float* po = (float*)a.work + ((long long)split * rows + row) * a.D;
    float* pml = (float*)a.work + (long long)nsplit * rows * a.D + ((long long)split * rows + row) * 2;
#pragma unroll
    for (int d = 0; d < G::DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = d * 32 + 8 * g + 4 * h;
        if (c < a.D) *(f32x4*)(po + c) = none ? f32x4{0, 0, 0, 0} : f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
      }
    if (h == 0) { pml[0] = none ? S_NEG : m_run; pml[1] = none ? 0.f : l_tot; }
    return;
  }
  const float inv = 1.0f / l_tot;
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = none ? 0.f : o[d][r] * inv;
  u16* orow = (u16*)a.out + (((long long)b * a.Sq + ic) * a.H + head) * a.D;
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {      // lane and lane ^ 32 hold 4 channels each of every 8: they swap one group of a pair, then 16-byte stores
      const int ge = 2 * pr, go = 2 * pr + 1;
      const unsigned e0 = pack2bf(o[d][4 * ge] , o[d][4 * ge + 1]), e1 = pack2bf(o[d][4 * ge + 2] , o[d][4 * ge + 3]);
      const unsigned o0 = pack2bf(o[d][4 * go] , o[d][4 * go + 1]), o1 = pack2bf(o[d][4 * go + 2] , o[d][4 * go + 3]);
      const u32x2 s0 = __builtin_amdgcn_permlane32_swap(e0, o0, false, false);
      const u32x2 s1 = __builtin_amdgcn_permlane32_swap(e1, o1, false, false);
      const int c = d * 32 + 8 * (2 * pr + h);
      if (i < a.Sq && c < a.D) *(u32x4*)(orow + c) = u32x4{s0[0], s1[0], s0[1], s1[1]};
    }
  if (i < a.Sq && h == 0 && a.lse != nullptr) a.lse[row] = none ? INFINITY : m_run + log2f(l_tot);
}

// Two 32-row tiles that are used together (K and V, or Q and dO), staged as one image of 64 rows: waves 0 and 1 fetch the first matrix,
// 2 and 3 the second.  Two images: the next pair travels under the whole of this one's work, one barrier a pair.
template <int HDP> struct PairDma {
  static constexpr int T = SGeo<HDP>::STR, NI = 64 * T / 4096, HALF = 32 * T, BUF = 64 * T;
  unsigned off[NI];
  int wave, lane;
  __device__ __forceinline__ int row(int i) const { return ((wave & 1) * NI * 1024 + i * 1024 + lane * 16) / T; }
  __device__ __forceinline__ PairDma(int wave_, int lane_, unsigned row_bytes, int D) : wave(wave_), lane(lane_) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int pos = (wave & 1) * NI * 1024 + i * 1024 + lane * 16, r = pos / T, cp = (pos % T) >> 4, c = cp ^ ((r >> 2) & 3);
      off[i] = cp >= HDP / 8 || c * 8 >= D ? SDma<HDP>::OUT : (unsigned)r * row_bytes + c * 16;
    }
  }
  // base, row_bytes: of the matrix this wave fetches.  Rows at or beyond row_end and (doc != null) rows of negative documents: zeros
  __device__ __forceinline__ void issue(const char* base, unsigned row_bytes, int row0, int row_end, int D, const int* doc, unsigned char* image) const {
    const int n = min(32, row_end - row0);
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)(base + (long long)row0 * row_bytes), 0, (int)((unsigned)(n - 1) * row_bytes + D * 2), 0x00020000);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      unsigned o = off[i];
      if (doc != nullptr && doc[row0 + min(row(i), n - 1)] < 0) o = SDma<HDP>::OUT;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, TF_LDS_PTR(image + (wave * NI + i) * 1024), 16, (int)o, 0, 0, 0);
    }
  }
};
// st += X . x and dp += Y . y of a pair image: row fragments PF ahead of their matrix instruction, the two accumulators in turn
template <int HDP> __device__ __forceinline__ void pair_rows(const SAddr<HDP>& fx, const SAddr<HDP>& fy, const u32x4 (&x)[HDP / 16], const u32x4 (&y)[HDP / 16],
                                                             f32x16& st, f32x16& dp) {
  constexpr int NF = 2 * (HDP / 16), PF = 4;
  u32x4 fr[NF];
  static_for<PF>([&](auto I) { if constexpr (I & 1) fr[I] = fy.template row<0, (I >> 1)>(); else fr[I] = fx.template row<0, (I >> 1)>(); });
  static_for<NF>([&](auto I) {
    constexpr int i = I, nx = i + PF;
    if constexpr (nx < NF) { if constexpr (nx & 1) fr[nx] = fy.template row<0, (nx >> 1)>(); else fr[nx] = fx.template row<0, (nx >> 1)>(); }
    lgkm_wait<(NF - 1 - i < PF ? NF - 1 - i : PF)>(fr[i]);
    if constexpr (i & 1) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(fr[i]), as_bf16x8(y[i >> 1]), dp, 0, 0, 0);
    else st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(fr[i]), as_bf16x8(x[i >> 1]), st, 0, 0, 0);
  });
}
template <int HDP> __device__ __forceinline__ void one_rows(const SAddr<HDP>& fx, const u32x4 (&x)[HDP / 16], f32x16& st) {
  constexpr int NF = HDP / 16, PF = NF < 4 ? NF : 4;
  u32x4 fr[NF];
  static_for<PF>([&](auto I) { fr[I] = fx.template row<0, I>(); });
  static_for<NF>([&](auto I) {
    constexpr int i = I, nx = i + PF;
    if constexpr (nx < NF) fr[nx] = fx.template row<0, nx>();
    lgkm_wait<(NF - 1 - i < PF ? NF - 1 - i : PF)>(fr[i]);
    st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(fr[i]), as_bf16x8(x[i]), st, 0, 0, 0);
  });
}
// acc[channel][lane] += sum over the 32 rows of a tile of tile[row][channel] * p[row]; p: 16 values packed as they lie in the accumulator
template <int HDP> __device__ __forceinline__ void tile_t(const SAddr<HDP>& f, const unsigned (&p)[8], f32x16 (&acc)[HDP / 32]) {
  constexpr int DB = HDP / 32, NF = 2 * DB, PF = 2;
  u64 fa[NF], fb[NF];
  static_for<PF>([&](auto I) { f.template tr<(I / DB) * 16, (I % DB) * 32>(fa[I], fb[I]); });
  static_for<NF>([&](auto I) {
    constexpr int i = I, nx = i + PF, s = 4 * (i / DB);
    if constexpr (nx < NF) f.template tr<(nx / DB) * 16, (nx % DB) * 32>(fa[nx], fb[nx]);
    lgkm_wait<2 * (NF - 1 - i < PF ? NF - 1 - i : PF)>(fa[i], fb[i]);
    acc[i % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(join_tr64(fa[i], fb[i]), as_bf16x8(u32x4{p[s], p[s + 1], p[s + 2], p[s + 3]}), acc[i % DB], 0, 0, 0);
  });
}
template <int HDP> __device__ __forceinline__ SAddr<HDP> shifted(const SAddr<HDP>& f, unsigned bytes) {
  SAddr<HDP> g = f;
  g.row_e += bytes; g.row_o += bytes; g.tr_a += bytes; g.tr_b += bytes;
  return g;
}

// ================================================================================================
// forward of few rows (single tokens): Sq * H / Hk <= 32
// ================================================================================================
// Bound by the bytes of K and V.  The rows of all heads that share a key head are one 32-column tile, so every key is read once; each of
// the four waves walks key tiles of its own (32 keys) and the workgroup's keys are a range of the sample's (the launcher splits the keys
// until the chip is full).  bf16: no barrier in the loop -- a wave waits for its own transfers by count: K(t + 1) is under way from the
// moment S(t) has been read, V(t + 1) from the end of PV(t), so one tile is always in flight.  The waves' parts are joined in LDS.
struct FewRows { int i, head, lim, qd; bool ok, live; float slope2; };
__device__ __forceinline__ FewRows few_rows(const TfScoreAttnArgs& a, int b, int kvh, int p0, int pfx, int lane) {
  FewRows w;
  const int G = a.H / a.Hk, r = lane & 31;
  w.ok = r < a.Sq * G;
  const int rc = w.ok ? r : 0;
  w.i = rc / G;
  w.head = kvh * G + rc % G;
  w.qd = a.k_doc != nullptr ? a.q_doc[(size_t)b * a.Sq + w.i] : 0;
  w.live = w.ok && w.qd >= 0;
  w.lim = a.causal ? min(max(p0 + w.i, pfx - 1), a.Sk - 1) : a.Sk - 1;
  w.slope2 = a.slopes != nullptr ? a.slopes[w.head] * LOG2E : 0.f;
  return w;
}
// the changed and masked scores of a 32-key tile (kd: document of key kv0 + (lane & 31))
template <bool F32, bool DOC> __device__ __forceinline__ void few_change(const TfScoreAttnArgs& a, const FewRows& w, const SMod& m, int p0, int kv0, int kd, int h,
                                                                         f32x16& st) {
  if (m.capl != 0.f) {
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = m.capl * tanh_of<F32>(st[r] * m.sc);
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] *= m.sc;
  }
  if (a.slopes != nullptr) {
    const float pd = (float)(p0 + w.i - kv0 - 4 * h);
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] -= w.slope2 * fabsf(pd - (float)((r & 3) + 8 * (r >> 2)));
  }
  const int n = w.lim - kv0 + 1;
  unsigned bits = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
  if (DOC) bits &= (unsigned)doc_bits(w.qd, kd);
  if (__any(bits != 0xffffffffu)) {
    bits >>= 4 * h;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (!((bits >> ((r & 3) + 8 * (r >> 2))) & 1u)) st[r] = -INFINITY;
  }
}
// one step of the running softmax over a 32-key tile: st becomes the probabilities
template <int DB> __device__ __forceinline__ void few_softmax(f32x16& st, float& m_run, float& l_run, f32x16 (&o)[DB]) {
  float mx = -INFINITY;
#pragma unroll
  for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[r]);
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
  const bool need = mx - m_run > RESCALE_THR;
  if (__any(need)) {
    const float m_new = need ? fmaxf(m_run, mx) : m_run, alpha = need ? fast_exp2(m_run - m_new) : 1.0f;
    m_run = m_new;
    l_run *= alpha;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    st[r] = fast_exp2(st[r] - m_run);
    l_run += st[r];
  }
}
// joins the four waves' parts (smem: 4 * 32 * D + 256 floats) and writes the rows, or this split's part of them
template <bool F32, int DB> __device__ __forceinline__ void few_finish(const TfScoreAttnArgs& a, const FewRows& w, int b, int kvh, float m_run, float l_run,
                                                                       f32x16 (&o)[DB], float* smem, int nsplit, int split, int wave, int lane) {
  const int h = lane >> 5, r = lane & 31, G = a.H / a.Hk, R = a.Sq * G;
  float* ml = smem + 128 * a.D;                          // [4 waves][32][2]
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  const bool none = !w.live || l_tot == 0.f;
  __syncthreads();
  if (h == 0) { ml[(wave * 32 + r) * 2] = none ? S_NEG : m_run; ml[(wave * 32 + r) * 2 + 1] = none ? 0.f : l_tot; }
  __syncthreads();
  float mx = S_NEG;
#pragma unroll
  for (int v = 0; v < 4; ++v) mx = fmaxf(mx, ml[(v * 32 + r) * 2]);
  const float s = none ? 0.f : fast_exp2(m_run - mx);
  if (w.ok) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = d * 32 + 8 * g + 4 * h;
        if (c < a.D) *(f32x4*)(smem + (wave * 32 + r) * a.D + c) = none ? f32x4{0, 0, 0, 0} : f32x4{o[d][4 * g] * s, o[d][4 * g + 1] * s, o[d][4 * g + 2] * s, o[d][4 * g + 3] * s};
      }
  }
  __syncthreads();
  const int d4 = a.D / 4;
  const long long rows = (long long)a.B * a.H * a.Sq;
  for (int x = wave * 64 + lane; x < R * d4; x += 256) {
    const int q = x / d4, c = x % d4 * 4, i = q / G, head = kvh * G + q % G;
    float top = S_NEG, l = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) top = fmaxf(top, ml[(v * 32 + q) * 2]);
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      l += ml[(v * 32 + q) * 2 + 1] * fast_exp2(ml[(v * 32 + q) * 2] - top);
      acc += *(const f32x4*)(smem + (v * 32 + q) * a.D + c);
    }
    const long long row = ((long long)b * a.H + head) * a.Sq + i;
    if (nsplit > 1) {
      *(f32x4*)((float*)a.work + ((long long)split * rows + row) * a.D + c) = acc;
      if (c == 0) {
        float* pml = (float*)a.work + (long long)nsplit * rows * a.D + ((long long)split * rows + row) * 2;
        pml[0] = top;
        pml[1] = l;
      }
    } else {
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const long long oo = (((long long)b * a.Sq + i) * a.H + head) * a.D + c;
      if constexpr (F32) *(f32x4*)((float*)a.out + oo) = acc * inv;
      else *(u32x2*)((u16*)a.out + oo) = u32x2{pk2(acc[0] * inv, acc[1] * inv), pk2(acc[2] * inv, acc[3] * inv)};
      if (c == 0 && a.lse != nullptr) a.lse[row] = l == 0.f ? INFINITY : top + log2f(l);
    }
  }
}
// keys of a workgroup: an equal share of the tiles this sample's rows can see
struct FewRange { int lo, end, hi; };
__device__ __forceinline__ FewRange few_range(const TfScoreAttnArgs& a, int p0, int pfx, int nsplit, int split) {
  FewRange f;
  f.hi = a.causal ? max(0, min(max(p0 + a.Sq, pfx), a.Sk)) : a.Sk;
  const int tiles = (f.hi + 31) / 32;
  f.lo = (int)((long long)tiles * split / nsplit);
  f.end = (int)((long long)tiles * (split + 1) / nsplit);
  return f;
}

template <int N> __device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <int HDP, bool DOC>
__global__ __launch_bounds__(256, (HDP <= 128 ? 2 : 1)) void score_few16_kernel(const TfScoreAttnArgs a, int nsplit) {
  using G = SGeo<HDP>;
  constexpr int T = G::STR, NI = 32 * T / 1024;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  unsigned char* kt = smem + wave * 64 * T;
  unsigned char* vt = kt + 32 * T;
  const int logical = xcd_remap(blockIdx.x, gridDim.x), split = logical % nsplit, bk = logical / nsplit, b = bk / a.Hk, kvh = bk % a.Hk;
  const char* kbase = (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * 2;
  const char* vbase = (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * 2;
  const unsigned krb = (unsigned)a.k_ss * 2, vrb = (unsigned)a.v_ss * 2;
  const int* kdoc = DOC ? a.k_doc + (size_t)b * a.Sk : nullptr;
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const FewRows w = few_rows(a, b, kvh, p0, pfx, lane);
  SMod m = smod(a, kvh * (a.H / a.Hk));
  const FewRange f = few_range(a, p0, pfx, nsplit, split);
  unsigned koff[NI], voff[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int pos = i * 1024 + lane * 16, r = pos / T, cp = (pos % T) >> 4, c = cp ^ ((r >> 2) & 3);
    const bool out = cp >= HDP / 8 || c * 8 >= a.D;
    koff[i] = out ? SDma<HDP>::OUT : (unsigned)r * krb + c * 16;
    voff[i] = out ? SDma<HDP>::OUT : (unsigned)r * vrb + c * 16;
  }
  auto issue = [&](const char* base, unsigned rb, const unsigned (&off)[NI], int t, unsigned char* tile, bool neg) {
    const int n = min(32, f.hi - t * 32);
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)(base + (long long)t * 32 * rb), 0, (int)((unsigned)(n - 1) * rb + a.D * 2), 0x00020000);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      unsigned x = off[i];
      if (DOC && neg && kdoc[t * 32 + min((i * 1024 + lane * 16) / T, n - 1)] < 0) x = SDma<HDP>::OUT;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, TF_LDS_PTR(tile + i * 1024), 16, (int)x, 0, 0, 0);
    }
  };
  // documents: the tile's ids are read a tile ahead of its transfer; tiles without one of the rows' documents are passed over
  const int dmin = DOC ? wave_min_i(w.live ? w.qd : 0x7fffffff) : 0, dmax = DOC ? -wave_min_i(w.live ? -w.qd : 0x7fffffff) : 0;
  auto doc_of = [&](int t) { const int j = t * 32 + (lane & 31); return j < a.Sk ? kdoc[j] : -1; };
  bool neg = false;
  int kd = 0, kd_n = 0, kd_nn = 0;                       // of the tile in hand, the tile under way, the tile after it
  auto seek = [&](int t) {                               // first visible tile from t on; leaves its documents in kd_n
    if (!DOC) return t < f.end ? t : -1;
    for (; t < f.end; t += 4) {
      kd_n = kd_nn;
      if (t + 4 < f.end) kd_nn = doc_of(t + 4);
      if (__any(kd_n >= dmin && kd_n <= dmax)) { neg = __any(kd_n < 0); return t; }
    }
    return -1;
  };
  u32x4 qf[G::KS];
  {
    const char* qrow = (const char*)a.q + ((long long)b * a.q_sb + (long long)w.i * a.q_ss + (long long)w.head * a.q_sh) * 2;
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) qf[ks] = gfrag<false>(qrow, ks, h, a.D, w.live).v;
  }
  f32x16 o[G::DB];
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m_run = S_NEG, l_run = 0.f;
  const SAddr<HDP> fk(lds_addr_of(kt), lane), fv(lds_addr_of(vt), lane);
  if (DOC && f.lo + wave < f.end) kd_nn = doc_of(f.lo + wave);
  int t = seek(f.lo + wave);
  bool neg_t = neg;
  if (t >= 0) {
    kd = kd_n;
    issue(kbase, krb, koff, t, kt, neg);
    issue(vbase, vrb, voff, t, vt, neg);
  }
  while (t >= 0) {
    const int tn = seek(t + 4), kd_next = kd_n;
    neg_t = neg;
    vm_wait<NI>();                        // K(t); V(t)'s NI transfers may still be out
    f32x16 st;
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = 0.f;
    one_rows<HDP>(fk, qf, st);
    if (tn >= 0) issue(kbase, krb, koff, tn, kt, neg_t);
    few_change<false, DOC>(a, w, m, p0, t * 32, kd, h, st);
    few_softmax<G::DB>(st, m_run, l_run, o);
    unsigned pk[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) pk[r] = pk2(st[2 * r], st[2 * r + 1]);
    if (tn >= 0) vm_wait<NI>(); else vm_wait<0>();       // V(t); K(t + 1)'s may still be out
    tile_t<HDP>(fv, pk, o);
    if (tn >= 0) issue(vbase, vrb, voff, tn, vt, neg_t);
    kd = kd_next;
    t = tn;
  }
  few_finish<false, G::DB>(a, w, b, kvh, m_run, l_run, o, (float*)smem, nsplit, split, wave, lane);
}

// fp32: K fragments and V rows come straight from memory (V's are whole 128-byte lines a half-wave, the fp32 matrix instruction takes them
// untransposed), so nothing is staged; many waves hide the latency
template <int HDP, bool DOC>
__global__ __launch_bounds__(256, 1) void score_few32_kernel(const TfScoreAttnArgs a, int nsplit) {
  constexpr int KS = HDP / 16, DB = HDP / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int logical = xcd_remap(blockIdx.x, gridDim.x), split = logical % nsplit, bk = logical / nsplit, b = bk / a.Hk, kvh = bk % a.Hk;
  const char* kbase = (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * 4;
  const char* vbase = (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * 4;
  const int* kdoc = DOC ? a.k_doc + (size_t)b * a.Sk : nullptr;
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const FewRows w = few_rows(a, b, kvh, p0, pfx, lane);
  const SMod m = smod(a, kvh * (a.H / a.Hk));
  const FewRange f = few_range(a, p0, pfx, nsplit, split);
  const int dmin = DOC ? wave_min_i(w.live ? w.qd : 0x7fffffff) : 0, dmax = DOC ? -wave_min_i(w.live ? -w.qd : 0x7fffffff) : 0;
  constexpr bool REREAD = HDP > 192;      // Q does not fit beside the accumulators: read again (from L1) for every tile
  const char* qrow = (const char*)a.q + ((long long)b * a.q_sb + (long long)w.i * a.q_ss + (long long)w.head * a.q_sh) * 4;
  SFrag<true> qf[REREAD ? 1 : KS];
  if constexpr (!REREAD) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = gfrag<true>(qrow, ks, h, a.D, w.live);
  }
  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m_run = S_NEG, l_run = 0.f;
  for (int t = f.lo + wave; t < f.end; t += 4) {
    const int kv0 = t * 32, j = kv0 + (lane & 31);
    int kd = 0;
    if (DOC) {
      kd = j < a.Sk ? kdoc[j] : -1;
      if (!__any(kd >= dmin && kd <= dmax)) continue;
    }
    f32x16 st;
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = 0.f;
    const char* krow = kbase + (long long)min(j, f.hi - 1) * a.k_ss * 4;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const SFrag<true> x = gfrag<true>(krow, ks, h, a.D, j < f.hi && (!DOC || kd >= 0));
      if constexpr (REREAD) st = smma<true>(x, gfrag<true>(qrow, ks, h, a.D, w.live), st);
      else st = smma<true>(x, qf[ks], st);
    }
    few_change<true, DOC>(a, w, m, p0, kv0, kd, h, st);
    few_softmax<DB>(st, m_run, l_run, o);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int jj = (r & 3) + 8 * (r >> 2) + 4 * h;
      const bool in = kv0 + jj < f.hi && (!DOC || __shfl(kd, jj, 64) >= 0);
      const float* vrow = (const float*)(vbase + (long long)min(kv0 + jj, f.hi - 1) * a.v_ss * 4) + (lane & 31);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const float v = in && d * 32 + (lane & 31) < a.D ? vrow[d * 32] : 0.f;
        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, st[r], o[d], 0, 0, 0);
      }
    }
  }
  few_finish<true, DB>(a, w, b, kvh, m_run, l_run, o, (float*)smem, nsplit, split, wave, lane);
}

// joins the parts of a split forward, one workgroup a row: the parts' weights first (one thread a part), then every wave adds up a quarter
// of the parts (four channels a lane, the loads of several parts in flight).  At 32 parts of 64 rows a wave that walked all parts by
// itself took 23 us, as long as the product; this form takes 5.
constexpr int JOIN_MAX = 512;
template <bool F32> __global__ __launch_bounds__(256) void score_join_kernel(const TfScoreAttnArgs a, int nsplit) {
  __shared__ float wgt[JOIN_MAX], red[8];
  __shared__ f32x4 part[256];
  const long long rows = (long long)a.B * a.H * a.Sq, row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* po = (const float*)a.work + row * a.D;
  const float* pml = (const float*)a.work + (long long)nsplit * rows * a.D + row * 2;
  float mx = S_NEG;
  for (int s = tid; s < nsplit; s += 256) mx = fmaxf(mx, pml[(long long)s * rows * 2]);
  mx = wave_max(mx);
  if (lane == 0) red[wave] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float l = 0.f;
  for (int s = tid; s < nsplit; s += 256) {
    const float w = fast_exp2(pml[(long long)s * rows * 2] - mx);
    wgt[s] = w;
    l += w * pml[(long long)s * rows * 2 + 1];
  }
  l = wave_sum(l);
  if (lane == 0) red[4 + wave] = l;
  __syncthreads();
  l = (red[4] + red[5]) + (red[6] + red[7]);
  f32x4 acc = {0, 0, 0, 0};
  if (lane * 4 < a.D) {
#pragma unroll 8
    for (int s = wave; s < nsplit; s += 4) acc += wgt[s] * *(const f32x4*)(po + (long long)s * rows * a.D + lane * 4);
  }
  part[tid] = acc;
  __syncthreads();
  if (wave != 0) return;
  acc = (part[lane] + part[64 + lane]) + (part[128 + lane] + part[192 + lane]);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int i = (int)(row % a.Sq), bh = (int)(row / a.Sq), b = bh / a.H, head = bh % a.H;
  const long long oo = (((long long)b * a.Sq + i) * a.H + head) * a.D + lane * 4;
  if (lane * 4 < a.D) {
    if constexpr (F32) *(f32x4*)((float*)a.out + oo) = acc * inv;
    else *(u32x2*)((u16*)a.out + oo) = u32x2{pk2(acc[0] * inv, acc[1] * inv), pk2(acc[2] * inv, acc[3] * inv)};
  }
  if (lane == 0 && a.lse != nullptr) a.lse[row] = l == 0.f ? INFINITY : mx + log2f(l);
}

// ================================================================================================
// backward: dq
// ================================================================================================
template <bool F32, int HDP>
__global__ __launch_bounds__(256, 1) void score_dq_kernel(const TfScoreAttnArgs a, int nqb) {
  using T = STile<F32, HDP>;
  constexpr int KT = 32, KS = HDP / 16, DB = HDP / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* kt = smem;
  unsigned char* vt = smem + KT * T::STR;
  int* docs = (int*)(smem + 2 * KT * T::STR);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const int logical = xcd_remap(blockIdx.x, gridDim.x);
  const int qb = nqb - 1 - logical % nqb, bh = logical / nqb, b = bh / a.H, head = bh % a.H, kvh = head / (a.H / a.Hk);
  const char* qbase = (const char*)a.q + ((long long)b * a.q_sb + (long long)head * a.q_sh) * T::ESZ;
  const char* kbase = (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * T::ESZ;
  const char* vbase = (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * T::ESZ;
  const int* kdoc = a.k_doc != nullptr ? a.k_doc + (size_t)b * a.Sk : nullptr;
  const SMod m = smod(a, head);
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const int i = qb * 128 + wave * 32 + (lane & 31), ic = min(i, a.Sq - 1);
  const int qd = kdoc != nullptr && i < a.Sq ? a.q_doc[(size_t)b * a.Sq + i] : 0;
  const bool live = i < a.Sq && qd >= 0;
  const int p = p0 + i;
  const int lim = !live ? -1 : (a.causal ? min(max(p, pfx - 1), a.Sk - 1) : a.Sk - 1);
  const int i_last = min(qb * 128 + 127, a.Sq - 1);
  const int hi = a.causal ? min(max(p0 + i_last + 1, pfx), a.Sk) : a.Sk;
  const int tile_end = (max(hi, 0) + KT - 1) / KT;
  const long long row = (long long)bh * a.Sq + ic;
  // fp32 heads of 256: Q, dO and dq together do not fit the register file, Q is read again (from L1 / L2) for every tile
  constexpr bool REREAD = F32 && HDP > 192;
  const char* qrow = qbase + (long long)ic * a.q_ss * T::ESZ;
  SFrag<F32> qf[REREAD ? 1 : KS], dof[KS];
  float delta = 0.f;
  {
    const char* orow = (const char*)a.out + (((long long)b * a.Sq + ic) * a.H + head) * a.D * T::ESZ;
    const char* drow = (const char*)a.dout + ((long long)b * a.do_sb + (long long)ic * a.do_ss + (long long)head * a.do_sh) * T::ESZ;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if constexpr (!REREAD) qf[ks] = gfrag<F32>(qrow, ks, h, a.D, live);
      dof[ks] = gfrag<F32>(drow, ks, h, a.D, live);
      delta += frag_dot<F32>(dof[ks], gfrag<F32>(orow, ks, h, a.D, live));
    }
    delta += __shfl_xor(delta, 32, 64);
  }
  const float lse = live ? a.lse[row] : INFINITY;
  f32x16 dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
  float dsl = 0.f;
  for (int t = 0; t < tile_end; ++t) {
    const int kv0 = t * KT;
    __syncthreads();
    T::template stage<KT>(kt, kbase, a.k_ss * T::ESZ, kv0, hi, kdoc, a.D, tid);
    T::template stage<KT>(vt, vbase, a.v_ss * T::ESZ, kv0, hi, kdoc, a.D, tid);
    if (kdoc != nullptr && tid < KT) docs[tid] = kv0 + tid < a.Sk ? kdoc[kv0 + tid] : -1;
    __syncthreads();
    f32x16 st, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) { st[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if constexpr (REREAD) st = smma<F32>(T::row(kt, 0, ks, lane), gfrag<F32>(qrow, ks, h, a.D, live), st);
      else st = smma<F32>(T::row(kt, 0, ks, lane), qf[ks], st);
      dp = smma<F32>(T::row(vt, 0, ks, lane), dof[ks], dp);
    }
    const float pd = (float)(p - kv0 - 4 * h);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = (r & 3) + 8 * (r >> 2);
      const float th = m.capl != 0.f ? tanh_of<F32>(st[r] * m.sc) : 0.f, dist = fabsf(pd - (float)j);
      float x = m.capl != 0.f ? m.capl * th : st[r] * m.sc;
      if (m.slope2 != 0.f) x -= m.slope2 * dist;
      bool vis = kv0 + j + 4 * h <= lim;
      if (kdoc != nullptr) vis = vis && docs[j + 4 * h] == qd;
      const float ds = vis ? fast_exp2(x - lse) * (dp[r] - delta) : 0.f;
      dsl -= ds * dist;
      st[r] = ds * (1.f - th * th);
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) dq[d] = T::mma_t(kt, 0, d * 32, st, dq[d], lane);
  }
  dsl += __shfl_xor(dsl, 32, 64);
  if (i >= a.Sq) return;
  if (h == 0) {
    a.delta[row] = delta;
    if (a.dslopes != nullptr) a.dslope_rows[row] = dsl;
  }
  char* grow = (char*)a.dq + (((long long)b * a.Sq + i) * a.H + head) * a.D * T::ESZ;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = d * 32 + 8 * g + 4 * h;
      if (c >= a.D) continue;
      const float x0 = dq[d][4 * g] * a.scale, x1 = dq[d][4 * g + 1] * a.scale, x2 = dq[d][4 * g + 2] * a.scale, x3 = dq[d][4 * g + 3] * a.scale;
      if constexpr (F32) *(f32x4*)(grow + c * 4) = f32x4{x0, x1, x2, x3};
      else *(u32x2*)(grow + c * 2) = u32x2{pack2bf(x0, x1), pack2bf(x2, x3)};
    }
}

// the slopes' gradient: one workgroup a head adds the rows of all samples up, in 64 bits and in one order
__global__ __launch_bounds__(256) void score_dslope_kernel(const float* __restrict__ rows, float* __restrict__ out, int B, int H, int Sq) {
  __shared__ double sh[256];
  const int head = blockIdx.x, tid = threadIdx.x;
  double s = 0.0;
  for (int b = 0; b < B; ++b) {
    const float* r = rows + ((size_t)b * H + head) * Sq;
    for (int i = tid; i < Sq; i += 256) s += (double)r[i];
  }
  sh[tid] = s;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (tid < o) sh[tid] += sh[tid + o];
    __syncthreads();
  }
  if (tid == 0) out[head] = (float)sh[0];
}

// ================================================================================================
// backward: dk, dv.  PART 0: dv, 1: dk, 2: both (wide heads do not hold both accumulators beside the operands)
// ================================================================================================
template <bool F32, int HDP, int PART>
__global__ __launch_bounds__(256, 1) void score_dkv_kernel(const TfScoreAttnArgs a, int nkb) {
  using T = STile<F32, HDP>;
  constexpr int QT = 32, KS = HDP / 16, DB = HDP / 32;
  constexpr bool DK = PART != 0, DV = PART != 1;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* qt = smem;
  unsigned char* dot = smem + QT * T::STR;
  float* lse_s = (float*)(smem + 2 * QT * T::STR);
  float* del_s = lse_s + QT;
  int* lim_s = (int*)(del_s + QT);
  int* doc_s = lim_s + QT;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const int logical = xcd_remap(blockIdx.x, gridDim.x);
  const int kb = logical % nkb, bk = logical / nkb, b = bk / a.Hk, kvh = bk % a.Hk, G = a.H / a.Hk;
  const char* kbase = (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * T::ESZ;
  const char* vbase = (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * T::ESZ;
  const int* kdoc = a.k_doc != nullptr ? a.k_doc + (size_t)b * a.Sk : nullptr;
  const int* qdoc = a.k_doc != nullptr ? a.q_doc + (size_t)b * a.Sq : nullptr;
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const int k0 = kb * 128, j = k0 + wave * 32 + (lane & 31), jc = min(j, a.Sk - 1);
  const int kd = kdoc != nullptr ? (j < a.Sk ? kdoc[j] : -1) : 0;
  const bool live = j < a.Sk && kd >= 0;
  constexpr bool REREAD = F32 && HDP > 192;                   // as in score_dq_kernel: V is read again for every tile
  const char* vrow = vbase + (long long)jc * a.v_ss * T::ESZ;
  SFrag<F32> kf[KS], vf[DK && !REREAD ? KS : 1];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    kf[ks] = gfrag<F32>(kbase + (long long)jc * a.k_ss * T::ESZ, ks, h, a.D, live);
    if constexpr (DK && !REREAD) vf[ks] = gfrag<F32>(vrow, ks, h, a.D, live);
  }
  f32x16 dk[DK ? DB : 1], dv[DV ? DB : 1];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if (DK) dk[d][r] = 0.f;
      if (DV) dv[d][r] = 0.f;
    }
  // the first query that may see a key of this block
  const int i_lo = a.causal && k0 >= pfx ? min(max(k0 - p0, 0), a.Sq) : 0;
  for (int g = 0; g < G; ++g) {
    const int head = kvh * G + g;
    const SMod m = smod(a, head);
    const char* qbase = (const char*)a.q + ((long long)b * a.q_sb + (long long)head * a.q_sh) * T::ESZ;
    const char* dbase = (const char*)a.dout + ((long long)b * a.do_sb + (long long)head * a.do_sh) * T::ESZ;
    const long long row0 = ((long long)b * a.H + head) * a.Sq;
    for (int i0 = i_lo / QT * QT; i0 < a.Sq; i0 += QT) {
      __syncthreads();
      T::template stage<QT>(qt, qbase, a.q_ss * T::ESZ, i0, a.Sq, qdoc, a.D, tid);
      T::template stage<QT>(dot, dbase, a.do_ss * T::ESZ, i0, a.Sq, qdoc, a.D, tid);
      if (tid < QT) {
        const int i = i0 + tid, p = p0 + i, qd = qdoc != nullptr && i < a.Sq ? qdoc[i] : 0;
        const bool ok = i < a.Sq && qd >= 0;
        lse_s[tid] = ok ? a.lse[row0 + i] : INFINITY;
        del_s[tid] = ok ? a.delta[row0 + i] : 0.f;
        lim_s[tid] = !ok ? -1 : (a.causal ? max(p, pfx - 1) : a.Sk - 1);
        doc_s[tid] = qd;
      }
      __syncthreads();
      f32x16 st, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) { st[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        st = smma<F32>(T::row(qt, 0, ks, lane), kf[ks], st);
        if constexpr (DK && REREAD) dp = smma<F32>(T::row(dot, 0, ks, lane), gfrag<F32>(vrow, ks, h, a.D, live), dp);
        else if constexpr (DK) dp = smma<F32>(T::row(dot, 0, ks, lane), vf[ks], dp);
      }
      const float pd = (float)(p0 + i0 + 4 * h - j);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int q = (r & 3) + 8 * (r >> 2), qq = q + 4 * h;
        const float th = m.capl != 0.f ? tanh_of<F32>(st[r] * m.sc) : 0.f;
        float x = m.capl != 0.f ? m.capl * th : st[r] * m.sc;
        if (m.slope2 != 0.f) x -= m.slope2 * fabsf(pd + (float)q);
        const bool vis = live && j <= lim_s[qq] && doc_s[qq] == kd;
        const float pr = vis ? fast_exp2(x - lse_s[qq]) : 0.f;
        if (DK) dp[r] = vis ? pr * (dp[r] - del_s[qq]) * (1.f - th * th) : 0.f;
        st[r] = pr;
      }
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        if (DV) dv[d] = T::mma_t(dot, 0, d * 32, st, dv[d], lane);
        if (DK) dk[d] = T::mma_t(qt, 0, d * 32, dp, dk[d], lane);
      }
    }
  }
  if (j >= a.Sk) return;
  const long long go = (((long long)b * a.Sk + j) * a.Hk + kvh) * a.D;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = d * 32 + 8 * g + 4 * h;
      if (c >= a.D) continue;
      if (DK) {
        const float x0 = dk[d][4 * g] * a.scale, x1 = dk[d][4 * g + 1] * a.scale, x2 = dk[d][4 * g + 2] * a.scale, x3 = dk[d][4 * g + 3] * a.scale;
        if constexpr (F32) *(f32x4*)((float*)a.dk + go + c) = f32x4{x0, x1, x2, x3};
        else *(u32x2*)((u16*)a.dk + go + c) = u32x2{pack2bf(x0, x1), pack2bf(x2, x3)};
      }
      if (DV) {
        const float x0 = dv[d][4 * g], x1 = dv[d][4 * g + 1], x2 = dv[d][4 * g + 2], x3 = dv[d][4 * g + 3];
        if constexpr (F32) *(f32x4*)((float*)a.dv + go + c) = f32x4{x0, x1, x2, x3};
        else *(u32x2*)((u16*)a.dv + go + c) = u32x2{pack2bf(x0, x1), pack2bf(x2, x3)};
      }
    }
}

// ================================================================================================
// backward, bf16
// ================================================================================================
// [rows of a 32-row accumulator tile][channels] of one lane -> 16-byte stores (see the forward's epilogue)
template <int DB> __device__ __forceinline__ void store_lane_row(u16* row, const f32x16 (&x)[DB], float scale, int h, int D, bool ok) {
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {
      const int ge = 8 * pr, go = 8 * pr + 4;
      const unsigned e0 = pk2(x[d][ge] * scale, x[d][ge + 1] * scale), e1 = pk2(x[d][ge + 2] * scale, x[d][ge + 3] * scale);
      const unsigned o0 = pk2(x[d][go] * scale, x[d][go + 1] * scale), o1 = pk2(x[d][go + 2] * scale, x[d][go + 3] * scale);
      const u32x2 s0 = __builtin_amdgcn_permlane32_swap(e0, o0, false, false);
      const u32x2 s1 = __builtin_amdgcn_permlane32_swap(e1, o1, false, false);
      const int c = d * 32 + 8 * (2 * pr + h);
      if (ok && c < D) *(u32x4*)(row + c) = u32x4{s0[0], s1[0], s0[1], s1[1]};
    }
}

// body(FULL, CAP, SLP) with the flags (all uniform over the wave) as compile-time constants: the loops over a tile's scores stay free of
// branches and of registers that only one of their forms needs
template <class F> __device__ __forceinline__ void by_flags(bool full, bool cap, bool slp, F&& body) {
  auto two = [&](auto FULL) {
    if (cap) { if (slp) body(FULL, std::true_type{}, std::true_type{}); else body(FULL, std::true_type{}, std::false_type{}); }
    else { if (slp) body(FULL, std::false_type{}, std::true_type{}); else body(FULL, std::false_type{}, std::false_type{}); }
  };
  if (full) two(std::true_type{}); else two(std::false_type{});
}

// One step of a walk over 64-item tiles in halves of 32 items.
template <bool DOC> struct HalfWalk {
  TileWalk<DOC> w;
  int s, items;                           // s: the half in hand (items 32 s ..), -1 at the end
  bool full, neg;
  __device__ __forceinline__ void first(int s0, u64 (*sh)[3], int wave, int lane) {
    const int t = w.first(s0 >> 1, sh, wave, lane);
    s = t < 0 ? -1 : max(2 * t, s0);
    if (s >= 0 && s * 32 >= items) s = -1;
    full = w.full;
    neg = w.neg;
  }
  __device__ __forceinline__ void next(u64 (*sh)[3], int wave, int lane) {
    if (!(s & 1) && (s + 1) * 32 < items) { ++s; return; }
    const int t = w.next(s >> 1, sh, wave, lane);
    s = t < 0 ? -1 : 2 * t;
    full = w.full;
    neg = w.neg;
  }
};

// dq: query on the lane, 128 queries a workgroup; also delta = rowsum(dO o) and the slopes' row sums
template <int HDP, bool DOC>
__global__ __launch_bounds__(256, (HDP <= 128 ? 2 : 1)) void score_dq16_kernel(const TfScoreAttnArgs a, int nqb) {
  using G = SGeo<HDP>;
  using PD = PairDma<HDP>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  u64 (*dsh)[3] = (u64 (*)[3])(smem + 2 * PD::BUF);
  int* rsh = (int*)(smem + 2 * PD::BUF + 96);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int logical = xcd_remap(blockIdx.x, gridDim.x);
  const int qb = nqb - 1 - logical % nqb, bh = logical / nqb, b = bh / a.H, head = bh % a.H, kvh = head / (a.H / a.Hk);
  const char* qbase = (const char*)a.q + ((long long)b * a.q_sb + (long long)head * a.q_sh) * 2;
  // this wave's matrix of the pair: K (waves 0, 1) or V
  const char* xbase = wave < 2 ? (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * 2
                               : (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * 2;
  const unsigned xrb = (unsigned)(wave < 2 ? a.k_ss : a.v_ss) * 2;
  const int* kdoc = DOC ? a.k_doc + (size_t)b * a.Sk : nullptr;
  const SMod m = smod(a, head);
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const int w0 = qb * 128 + wave * 32, i = w0 + (lane & 31), ic = min(i, a.Sq - 1);
  const int qd = DOC ? a.q_doc[(size_t)b * a.Sq + ic] : 0;
  const bool live = i < a.Sq && qd >= 0, wave_live = w0 < a.Sq;
  const int p = p0 + i;
  const int lim = a.causal ? min(max(p, pfx - 1), a.Sk - 1) : a.Sk - 1;
  const int lim_lo = a.causal ? min(max(p0 + w0, pfx - 1), a.Sk - 1) : a.Sk - 1;
  const int lim_hi = a.causal ? min(max(p0 + min(w0 + 31, a.Sq - 1), pfx - 1), a.Sk - 1) : a.Sk - 1;
  const int hi = a.causal ? min(max(p0 + min(qb * 128 + 127, a.Sq - 1) + 1, pfx), a.Sk) : a.Sk;
  HalfWalk<DOC> walk{{kdoc, (max(hi, 0) + 63) / 64, a.Sk, 0, 0, 0, {}, true, false}, -1, max(hi, 0), true, false};
  if (DOC) {
    const int lo = wave_min_i(live ? qd : 0x7fffffff), up = -wave_min_i(live ? -qd : 0x7fffffff);
    if (lane == 0) { rsh[wave] = lo; rsh[4 + wave] = up; }
    __syncthreads();
    walk.w.dmin = __builtin_amdgcn_readfirstlane(min(min(rsh[0], rsh[1]), min(rsh[2], rsh[3])));
    walk.w.dmax = __builtin_amdgcn_readfirstlane(max(max(rsh[4], rsh[5]), max(rsh[6], rsh[7])));
  }
  walk.first(0, dsh, wave, lane);
  const PD dma(wave, lane, xrb, a.D);
  int kd_n = -1;
  if (walk.s >= 0) {
    if (DOC) kd_n = walk.s * 32 + (lane & 31) < a.Sk ? kdoc[walk.s * 32 + (lane & 31)] : -1;
    dma.issue(xbase, xrb, walk.s * 32, hi, a.D, DOC && walk.neg ? kdoc : nullptr, smem);
  }
  const long long row = (long long)bh * a.Sq + ic;
  u32x4 qf[G::KS], dof[G::KS];
  float delta = 0.f;
  {
    const char* orow = (const char*)a.out + (((long long)b * a.Sq + ic) * a.H + head) * a.D * 2;
    const char* drow = (const char*)a.dout + ((long long)b * a.do_sb + (long long)ic * a.do_ss + (long long)head * a.do_sh) * 2;
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) {
      qf[ks] = gfrag<false>(qbase + (long long)ic * a.q_ss * 2, ks, h, a.D, live).v;
      const SFrag<false> g = gfrag<false>(drow, ks, h, a.D, live);
      dof[ks] = g.v;
      delta += frag_dot<false>(g, gfrag<false>(orow, ks, h, a.D, live));
    }
    delta += __shfl_xor(delta, 32, 64);
  }
  const float lse = live ? a.lse[row] : INFINITY;
  f32x16 dq[G::DB];
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
  float dsl = 0.f;
  const SAddr<HDP> fk0(lds_addr_of(smem), lane);
  int buf = 0;
  while (walk.s >= 0) {
    const int kv0 = walk.s * 32;
    const bool full_t = walk.full && kv0 + 31 <= lim_lo, work = wave_live && kv0 <= lim_hi;
    const int kd = kd_n;
    walk.next(dsh, wave, lane);
    dma_wait_barrier();                   // this pair is there; every wave is done with the one before
    if (walk.s >= 0) {
      if (DOC) kd_n = walk.s * 32 + (lane & 31) < a.Sk ? kdoc[walk.s * 32 + (lane & 31)] : -1;
      dma.issue(xbase, xrb, walk.s * 32, hi, a.D, DOC && walk.neg ? kdoc : nullptr, smem + (buf ^ 1) * PD::BUF);
    }
    if (work) {
      const SAddr<HDP> fk = shifted(fk0, buf * PD::BUF), fv = shifted(fk, PD::HALF);
      f32x16 st, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) { st[r] = 0.f; dp[r] = 0.f; }
      pair_rows<HDP>(fk, fv, qf, dof, st, dp);
      unsigned bits = 0xffffffffu;
      if (!full_t) {
        const int n = lim - kv0 + 1;
        bits = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
        if (DOC) bits &= (unsigned)doc_bits(qd, kd);
        bits >>= 4 * h;
      }
      const float pd = (float)(p - kv0 - 4 * h), ncap = m.capl != 0.f ? -1.0f / (m.capl * m.capl) : 0.f;
      unsigned pk[8];
      by_flags(full_t, m.capl != 0.f, m.slope2 != 0.f || a.dslopes != nullptr, [&](auto FULL, auto CAP, auto SLP) {
        auto one = [&](int r) {
          const int j = (r & 3) + 8 * (r >> 2);
          float t = CAP ? m.capl * tanh_of<false>(st[r] * m.sc) : st[r] * m.sc, x = t;
          const float dist = SLP ? fabsf(pd - (float)j) : 0.f;
          if (SLP) x -= m.slope2 * dist;
          x = fast_exp2(x - lse) * (dp[r] - delta);
          if (!FULL) x = (bits >> j) & 1u ? x : 0.f;
          if (SLP) dsl -= x * dist;
          return CAP ? x * fmaf(t * t, ncap, 1.0f) : x;           // the cap's derivative: 1 - (t / cap)^2
        };
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float x0 = one(r), x1 = one(r + 1);
          pk[r >> 1] = pk2(x0, x1);
        }
      });
      tile_t<HDP>(fk, pk, dq);
    }
    buf ^= 1;
  }
  dsl += __shfl_xor(dsl, 32, 64);
  if (i < a.Sq && h == 0) {
    a.delta[row] = delta;
    if (a.dslopes != nullptr) a.dslope_rows[row] = live ? dsl : 0.f;
  }
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = live ? dq[d][r] : 0.f;
  store_lane_row<G::DB>((u16*)a.dq + (((long long)b * a.Sq + ic) * a.H + head) * a.D, dq, a.scale, h, a.D, i < a.Sq);
}

// dk, dv: key on the lane, 128 keys a workgroup.  PART 0: dv, 1: dk, 2: both
template <int HDP, int PART, bool DOC>
__global__ __launch_bounds__(256, (HDP <= (PART == 2 ? (DOC ? 64 : 96) : PART == 1 ? 128 : 192) ? 2 : 1)) void score_dkv16_kernel(const TfScoreAttnArgs a, int nkb) {
  using G = SGeo<HDP>;
  using PD = PairDma<HDP>;
  constexpr bool DK = PART != 0, DV = PART != 1;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float* stat = (float*)(smem + 2 * PD::BUF);             // [2 images][32 lse, 32 delta]
  u64 (*dsh)[3] = (u64 (*)[3])(smem + 2 * PD::BUF + 512);
  int* rsh = (int*)(smem + 2 * PD::BUF + 512 + 96);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int logical = xcd_remap(blockIdx.x, gridDim.x);
  const int kb = logical % nkb, bk = logical / nkb, b = bk / a.Hk, kvh = bk % a.Hk, G_ = a.H / a.Hk;
  const char* kbase = (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * 2;
  const char* vbase = (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * 2;
  const int* qdoc = DOC ? a.q_doc + (size_t)b * a.Sq : nullptr;
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const int k0 = kb * 128, w0 = k0 + wave * 32, j = w0 + (lane & 31), jc = min(j, a.Sk - 1);
  const int kd = DOC ? a.k_doc[(size_t)b * a.Sk + jc] : 0;
  const bool live = j < a.Sk && kd >= 0, wave_live = w0 < a.Sk;
  u32x4 kf[G::KS], vf[DK ? G::KS : 1];
#pragma unroll
  for (int ks = 0; ks < G::KS; ++ks) {
    kf[ks] = gfrag<false>(kbase + (long long)jc * a.k_ss * 2, ks, h, a.D, live).v;
    if constexpr (DK) vf[ks] = gfrag<false>(vbase + (long long)jc * a.v_ss * 2, ks, h, a.D, live).v;
  }
  f32x16 dk[DK ? G::DB : 1], dv[DV ? G::DB : 1];
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if constexpr (DK) dk[d][r] = 0.f;
      if constexpr (DV) dv[d][r] = 0.f;
    }
  // queries from q_lane on see this lane's key; the block's first key is seen from i_lo on, the wave's last key by all from q_full on
  const int q_lane = a.causal && j >= pfx ? j - p0 : -(1 << 30);
  const int i_lo = a.causal && k0 >= pfx ? min(max(k0 - p0, 0), a.Sq) : 0;
  const int w_last = min(w0 + 31, a.Sk - 1);
  const int q_full = a.causal && w_last >= pfx ? w_last - p0 : -(1 << 30), q_any = a.causal && w0 >= pfx ? w0 - p0 : -(1 << 30);
  HalfWalk<DOC> walk{{qdoc, (a.Sq + 63) / 64, a.Sq, 0, 0, 0, {}, true, false}, -1, a.Sq, true, false};
  if (DOC) {
    const int lo = wave_min_i(live ? kd : 0x7fffffff), up = -wave_min_i(live ? -kd : 0x7fffffff);
    if (lane == 0) { rsh[wave] = lo; rsh[4 + wave] = up; }
    __syncthreads();
    walk.w.dmin = __builtin_amdgcn_readfirstlane(min(min(rsh[0], rsh[1]), min(rsh[2], rsh[3])));
    walk.w.dmax = __builtin_amdgcn_readfirstlane(max(max(rsh[4], rsh[5]), max(rsh[6], rsh[7])));
  }
  const unsigned xrb = (unsigned)(wave < 2 ? a.q_ss : a.do_ss) * 2;
  const PD dma(wave, lane, xrb, a.D);
  const SAddr<HDP> fq0(lds_addr_of(smem), lane);
  const unsigned stat0 = lds_addr_of(stat) + 16 * h;
  for (int g = 0; g < G_; ++g) {
    const int head = kvh * G_ + g;
    const SMod m = smod(a, head);
    const char* xbase = wave < 2 ? (const char*)a.q + ((long long)b * a.q_sb + (long long)head * a.q_sh) * 2
                                 : (const char*)a.dout + ((long long)b * a.do_sb + (long long)head * a.do_sh) * 2;
    const long long row0 = ((long long)b * a.H + head) * a.Sq;
    int qd_n = -1;
    auto fetch = [&](int buf) {           // the pair in walk.s, its rows' statistics (wave 0: 32 of each, 4 bytes a lane) and documents
      const int i0 = walk.s * 32;
      if (DOC) qd_n = i0 + (lane & 31) < a.Sq ? qdoc[i0 + (lane & 31)] : -1;
      dma.issue(xbase, xrb, i0, a.Sq, a.D, DOC && walk.neg ? qdoc : nullptr, smem + buf * PD::BUF);
      if (wave == 0) {
        const float* src = (lane < 32 ? a.lse : a.delta) + row0 + min(i0 + (lane & 31), a.Sq - 1);
        __builtin_amdgcn_global_load_lds(TF_GLB_PTR(src), TF_LDS_PTR(stat + buf * 64), 4, 0, 0);
      }
    };
    walk.first(i_lo / 32, dsh, wave, lane);
    int buf = 0;
    if (g > 0) __syncthreads();           // every wave is done with the images of the head before
    if (walk.s >= 0) fetch(0);
    while (walk.s >= 0) {
      const int i0 = walk.s * 32;
      const bool full_t = walk.full && i0 >= q_full && i0 + 32 <= a.Sq, work = wave_live && i0 + 31 >= q_any;
      const int qd = qd_n;
      walk.next(dsh, wave, lane);
      dma_wait_barrier();
      if (walk.s >= 0) fetch(buf ^ 1);
      if (work) {
        const SAddr<HDP> fq = shifted(fq0, buf * PD::BUF), fd = shifted(fq, PD::HALF);
        f32x16 st, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { st[r] = 0.f; dp[r] = 0.f; }
        if constexpr (DK) pair_rows<HDP>(fq, fd, kf, vf, st, dp);
        else one_rows<HDP>(fq, kf, st);
        u32x4 ls[4], de[4];               // register 4 g + e is query 8 g + 4 h + e
        const unsigned sa = stat0 + buf * 256;
        static_for<4>([&](auto I) { ls[I] = rd128_asm<32 * I>(sa); });
        if constexpr (DK) static_for<4>([&](auto I) { de[I] = rd128_asm<128 + 32 * I>(sa); });
        unsigned bits = 0xffffffffu;
        if (!full_t) {
          const int n = max(q_lane - i0, 0), e = a.Sq - i0;
          bits = n >= 32 ? 0u : 0xffffffffu << n;
          if (e < 32) bits &= (1u << e) - 1u;
          if (DOC) bits &= (unsigned)doc_bits(kd, qd);
          bits >>= 4 * h;
        }
        static_for<4>([&](auto I) { lgkm_wait<0>(ls[I]); });
        if constexpr (DK) static_for<4>([&](auto I) { lgkm_wait<0>(de[I]); });
        const float pd = (float)(p0 + i0 + 4 * h - j), ncap = m.capl != 0.f ? -1.0f / (m.capl * m.capl) : 0.f;
        unsigned pp[8], ps[8];
        by_flags(full_t, m.capl != 0.f, m.slope2 != 0.f, [&](auto FULL, auto CAP, auto SLP) {
          auto one = [&](int r, float& pr, float& ds) {
            const int q = (r & 3) + 8 * (r >> 2);
            float t = CAP ? m.capl * tanh_of<false>(st[r] * m.sc) : st[r] * m.sc, x = t;
            if (SLP) x -= m.slope2 * fabsf(pd + (float)q);
            pr = fast_exp2(x - f_of(ls[r >> 2][r & 3]));
            if (!FULL) pr = (bits >> q) & 1u ? pr : 0.f;
            if constexpr (DK) {
              ds = pr * (dp[r] - f_of(de[r >> 2][r & 3]));
              if (CAP) ds *= fmaf(t * t, ncap, 1.0f);
              if (!FULL) ds = (bits >> q) & 1u ? ds : 0.f;        // (a hidden pair's product may not be finite)
            }
          };
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            float p0_, p1_, s0_ = 0.f, s1_ = 0.f;
            one(r, p0_, s0_);
            one(r + 1, p1_, s1_);
            if constexpr (DV) pp[r >> 1] = pk2(p0_, p1_);
            if constexpr (DK) ps[r >> 1] = pk2(s0_, s1_);
          }
        });
        if constexpr (DV) tile_t<HDP>(fd, pp, dv);
        if constexpr (DK) tile_t<HDP>(fq, ps, dk);
      }
      buf ^= 1;
    }
  }
  const long long go = (((long long)b * a.Sk + jc) * a.Hk + kvh) * a.D;
  if constexpr (DK) {
#pragma unroll
    for (int d = 0; d < G::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dk[d][r] = live ? dk[d][r] : 0.f;
    store_lane_row<G::DB>((u16*)a.dk + go, dk, a.scale, h, a.D, j < a.Sk);
  }
  if constexpr (DV) {
#pragma unroll
    for (int d = 0; d < G::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dv[d][r] = live ? dv[d][r] : 0.f;
    store_lane_row<G::DB>((u16*)a.dv + go, dv, 1.0f, h, a.D, j < a.Sk);
  }
}

// ================================================================================================
// launchers
// ================================================================================================
// dynamic LDS beyond the default limit is granted per device
template <class K> void allow_lds(K kern, size_t bytes) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev > 63) dev = 0;
  if (done.load(std::memory_order_relaxed) >> dev & 1ull) return;
  (void)hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  done.fetch_or(1ull << dev, std::memory_order_relaxed);
}

int hdp_of(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : D <= 192 ? 192 : 256; }

struct FwdPlan { bool few; int nqb, nsplit, split_tiles; };
FwdPlan fwd_plan(const TfScoreAttnArgs* a) {
  FwdPlan f;
  f.few = (long long)a->Sq * (a->H / a->Hk) <= 32;
  if (f.few) {                            // two workgroups a CU, each with at least two tiles a wave
    const long long groups = (long long)a->B * a->Hk, tiles = (a->Sk + 31) / 32;
    f.nqb = f.split_tiles = 0;
    f.nsplit = (int)std::max(1ll, std::min((512 + groups - 1) / groups, tiles / 8));
    return f;
  }
  const int kt = a->is_f32 ? 32 : 64;
  f.nqb = (a->Sq + 127) / 128;
  const long long blocks = (long long)a->B * a->H * f.nqb;
  const int tiles = std::max(1, (a->Sk + kt - 1) / kt);
  long long want = blocks >= 256 ? 1 : std::min<long long>((512 + blocks - 1) / blocks, tiles / 4);
  if (want < 1) want = 1;
  f.split_tiles = (int)((tiles + want - 1) / want);
  f.nsplit = (tiles + f.split_tiles - 1) / f.split_tiles;
  return f;
}

int check(const TfScoreAttnArgs* a) {
  if (a->B < 0 || a->Sq < 0 || a->Sk < 0 || a->H <= 0 || a->Hk <= 0 || a->H % a->Hk != 0) return -1;
  if (a->D <= 0 || a->D > 256 || a->D % 8 != 0) return -2;
  if (!(a->softcap >= 0.f)) return -3;
  if ((a->k_doc == nullptr) != (a->q_doc == nullptr) && a->Sq > 0 && a->Sk > 0) return -4;
  const long long blocks = (long long)a->B * std::max(a->H * ((a->Sq + 127ll) / 128), (long long)a->Hk * ((a->Sk + 127) / 128));
  if (blocks > 0x3fffff || (long long)a->Sq + a->Sk > (1ll << 30)) return -5;
  return 0;
}
// (64 rows of a tile are addressed with 32-bit offsets)
bool aligned(const void* p, long long sb, long long ss, long long sh, int e) {
  return (((uintptr_t)p) & 15) == 0 && sb >= 0 && ss >= 0 && sh >= 0 && ss < (1ll << 30) / 64 / e && sb * e % 16 == 0 && ss * e % 16 == 0 && sh * e % 16 == 0;
}

template <bool F32, int HDP> int launch_fwd(const TfScoreAttnArgs* a, hipStream_t st) {
  const FwdPlan f = fwd_plan(a);
  if (f.few) {
    TfTraceScope tr(F32 ? "score_few32_kernel" : "score_few16_kernel", st, 4.0 * a->B * a->H * (double)a->Sq * a->Sk * a->D);
    const size_t join = (128 * (size_t)a->D + 256) * 4;
    auto go = [&](auto kern, size_t lds) {
      allow_lds(kern, std::max(lds, (size_t)(128 * HDP + 256) * 4));
      hipLaunchKernelGGL(kern, dim3(a->B * a->Hk * f.nsplit), dim3(256), std::max(lds, join), st, *a, f.nsplit);
    };
    if constexpr (F32) a->k_doc != nullptr ? go(score_few32_kernel<HDP, true>, 0) : go(score_few32_kernel<HDP, false>, 0);
    else a->k_doc != nullptr ? go(score_few16_kernel<HDP, true>, 256 * SGeo<HDP>::STR) : go(score_few16_kernel<HDP, false>, 256 * SGeo<HDP>::STR);
  } else {
    TfTraceScope tr(F32 ? "score_fwd_kernel" : "score_fwd16_kernel", st, 4.0 * a->B * a->H * (double)a->Sq * a->Sk * a->D);
    auto go = [&](auto kern, size_t lds) {
      allow_lds(kern, lds);
      hipLaunchKernelGGL(kern, dim3(a->B * a->H * f.nqb * f.nsplit), dim3(256), lds, st, *a, f.nqb, f.nsplit, f.split_tiles);
    };
    if constexpr (F32) go(score_fwd_kernel<true, HDP>, 2 * 32 * STile<true, HDP>::STR + 32 * 4);
    else if (a->k_doc != nullptr) go(score_fwd16_kernel<HDP, true>, 2 * SGeo<HDP>::TILE + 128);
    else go(score_fwd16_kernel<HDP, false>, 2 * SGeo<HDP>::TILE + 128);
  }
  if (f.nsplit > 1) {
    TfTraceScope tr("score_join_kernel", st);
    hipLaunchKernelGGL(score_join_kernel<F32>, dim3((unsigned)((long long)a->B * a->H * a->Sq)), dim3(256), 0, st, *a, f.nsplit);
  }
  return (int)hipGetLastError();
}

template <bool F32, int HDP> int launch_bwd(const TfScoreAttnArgs* a, hipStream_t st) {
  const double fl = 4.0 * a->B * a->H * (double)a->Sq * a->Sk * a->D;
  const int nqb = (a->Sq + 127) / 128, nkb = (a->Sk + 127) / 128;
  const bool doc = a->k_doc != nullptr;
  const size_t lds = F32 ? 64 * STile<true, HDP>::STR + 32 * 16 : 2 * PairDma<HDP>::BUF + 512 + 128;
  auto go = [&](auto kern, int blocks, int n) {
    allow_lds(kern, lds);
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), lds, st, *a, n);
  };
  if (nqb > 0) {
    TfTraceScope tr(F32 ? "score_dq_kernel" : "score_dq16_kernel", st, 1.5 * fl);
    const int blocks = a->B * a->H * nqb;
    if constexpr (F32) go(score_dq_kernel<true, HDP>, blocks, nqb);
    else doc ? go(score_dq16_kernel<HDP, true>, blocks, nqb) : go(score_dq16_kernel<HDP, false>, blocks, nqb);
  }
  if (a->dslopes != nullptr) {
    TfTraceScope tr("score_dslope_kernel", st);
    hipLaunchKernelGGL(score_dslope_kernel, dim3(a->H), dim3(256), 0, st, (const float*)a->dslope_rows, a->dslopes, a->B, a->H, a->Sq);
  }
  if (nkb > 0) {
    TfTraceScope tr(F32 ? "score_dkv_kernel" : "score_dkv16_kernel", st, 2.0 * fl);
    const int blocks = a->B * a->Hk * nkb;
    auto part = [&](auto which) {
      constexpr int PART = decltype(which)::value;
      if constexpr (F32) go(score_dkv_kernel<true, HDP, PART>, blocks, nkb);
      else doc ? go(score_dkv16_kernel<HDP, PART, true>, blocks, nkb) : go(score_dkv16_kernel<HDP, PART, false>, blocks, nkb);
    };
    if constexpr (HDP <= (F32 ? 128 : 192)) part(std::integral_constant<int, 2>{});
    else { part(std::integral_constant<int, 0>{}); part(std::integral_constant<int, 1>{}); }
  }
  return (int)hipGetLastError();
}

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

// bytes of TfScoreAttnArgs.work for the forward; the backward needs none
static size_t work_bytes(const TfScoreAttnArgs* a) {
  if (check(a) != 0 || a->B == 0 || a->Sq == 0) return 0;
  const FwdPlan f = fwd_plan(a);
  return f.nsplit > 1 ? (size_t)f.nsplit * a->B * a->H * a->Sq * (a->D + 2) * sizeof(float) : 0;
}

extern "C" size_t tf_score_attn_work(int B, int Sq, int Sk, int H, int Hk, int D, int is_f32) {
  TfScoreAttnArgs a{};
  a.B = B; a.Sq = Sq; a.Sk = Sk; a.H = H; a.Hk = Hk; a.D = D; a.is_f32 = is_f32;
  return work_bytes(&a);
}

extern "C" int tf_launch_score_fwd(const TfScoreAttnArgs* a, hipStream_t st) {
  const int rc = check(a);
  if (rc != 0) return rc;
  if (a->B == 0 || a->Sq == 0) return 0;
  const int e = a->is_f32 ? 4 : 2;
  if (a->q == nullptr || a->out == nullptr || (a->Sk > 0 && (a->k == nullptr || a->v == nullptr))) return -6;
  if (!aligned(a->q, a->q_sb, a->q_ss, a->q_sh, e) || !aligned(a->k, a->k_sb, a->k_ss, a->k_sh, e) || !aligned(a->v, a->v_sb, a->v_ss, a->v_sh, e) ||
      !aligned(a->out, 0, 0, 0, e)) return -7;
  const size_t need = work_bytes(a);
  if (need > 0 && (a->work == nullptr || a->work_bytes < need || ((uintptr_t)a->work & 15) != 0)) return -8;
  return by_head_dim(a, [&](auto f32, auto hdp) { return launch_fwd<decltype(f32)::value, decltype(hdp)::value>(a, st); });
}

extern "C" int tf_launch_score_bwd(const TfScoreAttnArgs* a, hipStream_t st) {
  const int rc = check(a);
  if (rc != 0) return rc;
  if (a->B == 0) {
    if (a->dslopes != nullptr) hipLaunchKernelGGL(score_dslope_kernel, dim3(a->H), dim3(256), 0, st, (const float*)nullptr, a->dslopes, 0, a->H, 0);
    return (int)hipGetLastError();
  }
  const int e = a->is_f32 ? 4 : 2;
  if (a->Sq > 0 && (a->q == nullptr || a->out == nullptr || a->dout == nullptr || a->dq == nullptr || a->lse == nullptr || a->delta == nullptr)) return -6;
  if (a->Sk > 0 && (a->k == nullptr || a->v == nullptr || a->dk == nullptr || a->dv == nullptr)) return -6;
  if (a->dslopes != nullptr && (a->slopes == nullptr || (a->Sq > 0 && a->dslope_rows == nullptr))) return -6;
  if (!aligned(a->q, a->q_sb, a->q_ss, a->q_sh, e) || !aligned(a->k, a->k_sb, a->k_ss, a->k_sh, e) || !aligned(a->v, a->v_sb, a->v_ss, a->v_sh, e) ||
      !aligned(a->dout, a->do_sb, a->do_ss, a->do_sh, e) || !aligned(a->out, 0, 0, 0, e) || !aligned(a->dq, 0, 0, 0, e) ||
      !aligned(a->dk, 0, 0, 0, e) || !aligned(a->dv, 0, 0, 0, e)) return -7;
  return by_head_dim(a, [&](auto f32, auto hdp) { return launch_bwd<decltype(f32)::value, decltype(hdp)::value>(a, st); });
}
