// Forward of attention with changed scores (score_attn.h has the mathematics).
#include "score_attn.h"

namespace {

// 128 queries a workgroup (32 a wave, on the lane), 64-key tiles by LDS-DMA into one slot for K and one for V: V(t) travels under S(t), K(t + 1)
// under PV(t).  Several workgroups a CU hide the barriers of one behind the matrix work of the others.  (A third slot, which gives a transfer a
// whole tile's work to travel under, costs a workgroup a CU or gains nothing: 4 x 4096 causal, 8 heads of 128, 177 against 168 us; 4 x 2048, 16
// heads of 64, 87 against 84.)  DOC: documents are given.
// Bound by the vector work between the two products (exponential, cap, masks, rounding) and by the barriers: matrix and vector pipes are busy 45 % of
// the time each at 128 channels, 42 and 70 % at 64.  A causal prompt of 16384 tokens, 8 heads of 128: 620 us = 890 TFLOP/s (a large library product
// reaches 1215 on this card); 4 x 2048, 16 heads of 64: 83 us = 830 TFLOP/s; 32 x 708, 4 heads of 192: 64 us = 770 TFLOP/s.
// RIDE (bf16, no cap, no slopes, a scale > 0, which leaves the order of the scores as it is): the scale rides in the exponent's FMA, until a row's maximum
// is large (see S_BIG).  A form of its own: the same switch in the loop of all forms cost a causal prompt of 16384 with slopes, 8 heads of 128, 2 % (600 -> 612 us).
template <bool F32, int HDP, bool DOC, bool RIDE>
__global__ __launch_bounds__(256, (!F32 && HDP <= 64 && !DOC ? 4 : !F32 && HDP <= 96 ? 3 : HDP <= (F32 ? 64 : 192) ? 2 : 1)) void score_fwd_kernel(const TfScoreAttnArgs a, int nqb, int nsplit, int split_tiles) {
  using G = SGeo<F32, HDP>;
  using Dma = SDma<F32, HDP, 64, 4>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  u64 (*dsh)[3] = (u64 (*)[3])(smem + 2 * Dma::BYTES);
  int* rsh = (int*)(smem + 2 * Dma::BYTES + 96);
  int* kds = (int*)(smem + 2 * Dma::BYTES + 128);         // [2][64] documents of the keys of two tiles
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  int block, group;
  order_blocks(nqb, a.H / a.Hk * nsplit, a.causal, block, group);
  const int qb = nqb - 1 - block, split = group % nsplit, bh = group / nsplit, b = bh / a.H, head = bh % a.H, kvh = head / (a.H / a.Hk);
  const char* qbase = (const char*)a.q + ((long long)b * a.q_sb + (long long)head * a.q_sh) * G::ESZ;
  const char* kbase = (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * G::ESZ;
  const char* vbase = (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * G::ESZ;
  const unsigned krb = (unsigned)a.k_ss * G::ESZ, vrb = (unsigned)a.v_ss * G::ESZ;
  const int* kdoc = DOC ? a.k_doc + (size_t)b * a.Sk : nullptr;
  const SMod m = smod(a, head);
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const int w0 = qb * 128 + wave * 32, i = w0 + (lane & 31), ic = min(i, a.Sq - 1);
  const int qd = DOC ? a.q_doc[(size_t)b * a.Sq + ic] : 0;
  const bool live = i < a.Sq && qd >= 0, wave_live = w0 < a.Sq;
  const QRow row_ = q_row(a, p0, pfx, w0, i);
  const int hi = key_end(a, p0, pfx, min(qb * 128 + 127, a.Sq - 1));
  TileWalk<DOC> walk{kdoc, min((hi + 63) / 64, (split + 1) * split_tiles), a.Sk, 0, 0, 0, {}, true, false};
  if (DOC) doc_range(qd, live, rsh, wave, lane, walk.dmin, walk.dmax);
  // fp32 heads of 256: Q does not fit the register file beside the accumulators; it is read again (from the caches) for every tile
  constexpr bool REREAD = F32 && HDP > 192;
  const char* qrow = qbase + (long long)ic * a.q_ss * G::ESZ;
  SFrag<F32> qf[REREAD ? 1 : G::KS];
  if constexpr (!REREAD) {
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) qf[ks] = gfrag<F32>(qrow, ks, h, a.D, live);
  }
  f32x16 o[G::DB];
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m_run = S_NEG, l_run = 0.f;
  bool scaled = !RIDE && m.capl == 0.f;
  float scf = RIDE ? m.sc : 1.0f;
  const SAddr<F32, HDP> f0(lds_addr_of(smem), lane);
  const Dma dma(wave, lane, krb, a.D);
  int t = walk.first(split * split_tiles, dsh, wave, lane);
  bool full = walk.full, neg = walk.neg;
  int dslot = 0;                          // of the documents of K(t)
  auto issue_k = [&](int tile, bool ng) {
    // (keys behind the last are hidden by the row's limit, whatever document they show)
    if (DOC && wave == 0) __builtin_amdgcn_global_load_lds(TF_GLB_PTR(kdoc + min(tile * 64 + lane, a.Sk - 1)), TF_LDS_PTR(kds + dslot * 64), 4, 0, 0);
    dslot ^= 1;
    dma.issue(kbase, krb, tile * 64, hi, a.D, DOC && ng ? kdoc : nullptr, smem);
  };
  auto issue_v = [&](int tile, bool ng) { dma.issue(vbase, vrb, tile * 64, hi, a.D, DOC && ng ? kdoc : nullptr, smem + Dma::BYTES); };
  if constexpr (!REREAD) {
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) landed(qf[ks]);
  }
  if (t >= 0) issue_k(t, neg);
  while (t >= 0) {
    const int kv0 = t * 64;
    const bool full_t = full && kv0 + 63 <= row_.lim_lo, work = wave_live && kv0 <= row_.lim_hi;
    const unsigned kd_at = lds_addr_of(kds + (dslot ^ 1) * 64) + lane * 4;
    const int tn = walk.next(t, dsh, wave, lane);        // (may scan documents, with barriers of its own: all waves take part)
    const bool neg_t = neg;
    full = walk.full;
    neg = walk.neg;
    dma_wait_barrier();                   // K(t) is there; every wave is done with V(t - 1)
    issue_v(t, neg_t);
    SPack<F32> pk[2];
    if (work) {
      f32x16 st[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[kb][r] = 0.f;
      auto qx = [&](auto I) { if constexpr (REREAD) return gfrag<F32>(qrow, I, h, a.D, live); else return qf[I]; };
      mul_rows2<F32, HDP, 32 * G::STR>(f0, qx, qx, st[0], st[1]);
      // each change is a branch that rewrites the scores in place (uniform; as two arms of one branch they cost a second set of registers)
      if (!RIDE && m.capl != 0.f) cap_scores<F32, 2>(m, st);
      if (scaled) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) st[kb][r] *= m.sc;
      }
      if (!RIDE && m.slope2 != 0.f) {
        const float pd = (float)(row_.p - kv0 - 4 * h);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) st[kb][r] = fmaf(-m.slope2, fabsf(pd - (float)(kb * 32 + (r & 3) + 8 * (r >> 2))), st[kb][r]);
      }
      if (!full_t) {
        const int n = row_.lim - kv0 + 1;
        u64 bits = n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull;
        if (DOC) {
          unsigned kd = rd32_asm<0>(kd_at);
          lgkm_wait32<0>(kd);
          bits &= doc_bits(qd, (int)kd);
        }
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
        if (RIDE && scf != 1.0f && __any(big(m_run) && m_run != S_NEG)) {        // from here on the scores are rounded first
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) st[kb][r] *= scf;
          scaled = true;
          scf = 1.0f;
        }
      }
      float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float e0 = fast_exp2(fmaf(st[kb][r], scf, -m_run)), e1 = fast_exp2(fmaf(st[kb][r + 1], scf, -m_run));
          ps0 += e0;
          ps1 += e1;
          pk[kb].set2(r, e0, e1);
        }
      l_run += ps0 + ps1;
    }
    dma_wait_barrier();                   // V(t) is there; every wave is done with K(t)
    if (tn >= 0) issue_k(tn, neg);
    if (work) {
      if constexpr (!F32) f0.template mul_t<Dma::BYTES>(pk, o);
      else f0.shifted(Dma::BYTES).template mul_t<0>(pk, o);
    }
    t = tn;
  }
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  const long long rows = (long long)a.B * a.H * a.Sq, row = (long long)bh * a.Sq + i;
  const bool none = !live || l_tot == 0.f;
  const float inv = nsplit > 1 ? 1.0f : 1.0f / l_tot;
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = none ? 0.f : o[d][r] * inv;
  if (nsplit > 1) {                       // unnormalised part of this range of keys; score_join_kernel adds them up
    if (i >= a.Sq) return;
    store_part<G::DB>((float*)a.work, ((long long)split * rows + row) * a.D, o, h, a.D);
    float* pml = (float*)a.work + (long long)nsplit * rows * a.D + ((long long)split * rows + row) * 2;
    if (h == 0) { pml[0] = none ? S_NEG : m_run; pml[1] = none ? 0.f : l_tot; }
    return;
  }
  const long long oo = (((long long)b * a.Sq + ic) * a.H + head) * a.D;
  store_row<F32, G::DB>(a.out, oo, o, 1.0f, h, a.D, i < a.Sq);
  if (!F32 && a.out_lo != nullptr) {      // what the rounding took, for the backward's delta
#pragma unroll
    for (int d = 0; d < G::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] -= bf2f(f2bf(o[d][r]));
    store_row<F32, G::DB>(a.out_lo, oo, o, 1.0f, h, a.D, i < a.Sq);
  }
  // rows without keys: +inf, so that every probability formed from it again is 0
  if (i < a.Sq && h == 0 && a.lse != nullptr) a.lse[row] = none ? INFINITY : m_run + log2f(l_tot);
}

// ================================================================================================
// forward of few rows (single tokens): Sq * H / Hk <= 32
// ================================================================================================
// Bound by the bytes of K and V: 4 x 16411 keys, 16 heads of 128 on 4, take 25.7 us = 5.2 TB/s (a large copy reaches 4.87), and 4 us the join.  The
// rows of all heads that share a key head are one 32-column tile, so every key is read once; each of the four waves walks key tiles of its own
// (32 keys) and the workgroup's keys are a range of the sample's (the launcher splits the keys until the chip is full).  bf16: no barrier in the loop -- a wave waits for its own transfers by count: K(t + 1) is under way from the
// moment S(t) has been read, V(t + 1) from the end of PV(t), so one tile is always in flight.  The waves' parts are joined in LDS.
struct FewRows { int i, head, p, lim, qd; bool ok, live; float slope2; };       // (p: see near_pos)
__device__ __forceinline__ FewRows few_rows(const TfScoreAttnArgs& a, int b, int kvh, int p0, int pfx, int lane) {
  FewRows w;
  const int G = a.H / a.Hk, r = lane & 31;
  w.ok = r < a.Sq * G;
  const int rc = w.ok ? r : 0;
  w.i = rc / G;
  w.head = kvh * G + rc % G;
  w.qd = a.k_doc != nullptr ? a.q_doc[(size_t)b * a.Sq + w.i] : 0;
  w.live = w.ok && w.qd >= 0;
  w.p = near_pos(a, p0 + w.i);
  w.lim = a.causal ? min(max(p0 + w.i, pfx - 1), a.Sk - 1) : a.Sk - 1;
  w.slope2 = a.slopes != nullptr ? a.slopes[w.head] * LOG2E : 0.f;
  return w;
}
// the changed and masked scores of a 32-key tile (kd: document of key kv0 + (lane & 31))
template <bool F32, bool DOC> __device__ __forceinline__ void few_change(const TfScoreAttnArgs& a, const FewRows& w, const SMod& m, int kv0, int kd, int h,
                                                                         f32x16& st) {
  if (m.capl != 0.f) {
    cap_scores<F32, 1>(m, reinterpret_cast<f32x16 (&)[1]>(st));
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] *= m.sc;
  }
  if (a.slopes != nullptr) {
    const float pd = (float)(w.p - kv0 - 4 * h);
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = fmaf(-w.slope2, fabsf(pd - (float)((r & 3) + 8 * (r >> 2))), st[r]);
  }
  unsigned bits = low_bits(w.lim - kv0 + 1);
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
#pragma clang fp contract(off)            // (the maximum comes off the rounded score: see S_BIG)
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
      else {
        put4<false>(a.out, oo, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
        if (a.out_lo != nullptr) put4_lo(a.out_lo, oo, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
      }
      if (c == 0 && a.lse != nullptr) a.lse[row] = l == 0.f ? INFINITY : top + log2f(l);
    }
  }
}
// keys of a workgroup: an equal share of the tiles this sample's rows can see
struct FewRange { int lo, end, hi; };
__device__ __forceinline__ FewRange few_range(const TfScoreAttnArgs& a, int p0, int pfx, int nsplit, int split) {
  FewRange f;
  f.hi = key_end(a, p0, pfx, a.Sq - 1);
  const int tiles = (f.hi + 31) / 32;
  f.lo = (int)((long long)tiles * split / nsplit);
  f.end = (int)((long long)tiles * (split + 1) / nsplit);
  return f;
}

template <int N> __device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <int HDP, bool DOC>
__global__ __launch_bounds__(256, (HDP <= 128 ? 2 : 1)) void score_few16_kernel(const TfScoreAttnArgs a, int nsplit) {
  using G = SGeo<false, HDP>;
  using Dma = SDma<false, HDP, 32, 1>;
  constexpr int NI = Dma::NI;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  unsigned char* kt = smem + wave * 2 * Dma::BYTES;
  unsigned char* vt = kt + Dma::BYTES;
  const int logical = xcd_remap(blockIdx.x, gridDim.x), split = logical % nsplit, bk = logical / nsplit, b = bk / a.Hk, kvh = bk % a.Hk;
  const char* kbase = (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * 2;
  const char* vbase = (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * 2;
  const unsigned krb = (unsigned)a.k_ss * 2, vrb = (unsigned)a.v_ss * 2;
  const int* kdoc = DOC ? a.k_doc + (size_t)b * a.Sk : nullptr;
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const FewRows w = few_rows(a, b, kvh, p0, pfx, lane);
  SMod m = smod(a, kvh * (a.H / a.Hk));
  const FewRange f = few_range(a, p0, pfx, nsplit, split);
  const Dma kdma(0, lane, krb, a.D), vdma(0, lane, vrb, a.D);
  auto issue = [&](const Dma& dma, const char* base, unsigned rb, int t, unsigned char* tile, bool neg) {
    dma.issue(base, rb, t * 32, f.hi, a.D, DOC && neg ? kdoc : nullptr, tile);
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
  SFrag<false> qf[G::KS];
  {
    const char* qrow = (const char*)a.q + ((long long)b * a.q_sb + (long long)w.i * a.q_ss + (long long)w.head * a.q_sh) * 2;
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) qf[ks] = gfrag<false>(qrow, ks, h, a.D, w.live);
  }
  f32x16 o[G::DB];
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m_run = S_NEG, l_run = 0.f;
  const SAddr<false, HDP> fk(lds_addr_of(kt), lane), fv(lds_addr_of(vt), lane);
#pragma unroll
  for (int ks = 0; ks < G::KS; ++ks) landed(qf[ks]);
  if (DOC && f.lo + wave < f.end) kd_nn = doc_of(f.lo + wave);
  int t = seek(f.lo + wave);
  bool neg_t = neg;
  if (t >= 0) {
    kd = kd_n;
    issue(kdma, kbase, krb, t, kt, neg);
    issue(vdma, vbase, vrb, t, vt, neg);
  }
  while (t >= 0) {
    const int tn = seek(t + 4), kd_next = kd_n;
    neg_t = neg;
    vm_wait<NI>();                        // K(t); V(t)'s NI transfers may still be out
    f32x16 st;
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = 0.f;
    mul_rows<false, HDP>(fk, [&](auto I) { return qf[I]; }, st);
    if (tn >= 0) issue(kdma, kbase, krb, tn, kt, neg_t);
    few_change<false, DOC>(a, w, m, t * 32, kd, h, st);
    few_softmax<G::DB>(st, m_run, l_run, o);
    SPack<false> pk[1];
#pragma unroll
    for (int r = 0; r < 16; r += 2) pk[0].set2(r, st[r], st[r + 1]);
    if (tn >= 0) vm_wait<NI>(); else vm_wait<0>();       // V(t); K(t + 1)'s may still be out
    fv.template mul_t<0>(pk, o);
    if (tn >= 0) issue(vdma, vbase, vrb, tn, vt, neg_t);
    kd = kd_next;
    t = tn;
  }
  few_finish<false, G::DB>(a, w, b, kvh, m_run, l_run, o, (float*)smem, nsplit, split, wave, lane);
}

// fp32: K fragments and V rows come straight from memory (V's are whole 128-byte lines a half-wave, the fp32 matrix instruction takes them
// untransposed), so nothing is staged and a wave waits for its loads tile by tile: the same size takes 313 us = 0.86 TB/s
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
    few_change<true, DOC>(a, w, m, kv0, kd, h, st);
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
// (With 4260 rows of 7 parts a workgroup a row takes 8.7 us and score_join_rows_kernel 4.7.)
template <bool F32> __device__ __forceinline__ void join_store(const TfScoreAttnArgs& a, long long row, int lane, f32x4 acc, float mx, float l) {
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int i = (int)(row % a.Sq), bh = (int)(row / a.Sq), b = bh / a.H, head = bh % a.H;
  const long long oo = (((long long)b * a.Sq + i) * a.H + head) * a.D + lane * 4;
  if (lane * 4 < a.D) {
    if constexpr (F32) *(f32x4*)((float*)a.out + oo) = acc * inv;
    else {
      put4<false>(a.out, oo, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
      if (a.out_lo != nullptr) put4_lo(a.out_lo, oo, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    }
  }
  if (lane == 0 && a.lse != nullptr) a.lse[row] = l == 0.f ? INFINITY : mx + log2f(l);
}
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
  join_store<F32>(a, row, lane, (part[lane] + part[64 + lane]) + (part[128 + lane] + part[192 + lane]), mx, l);
}
// the same with a wave a row, a lane a part: for many rows of at most 64 parts each.  Up to 128 channels the halves of a wave take every other part
template <bool F32> __global__ __launch_bounds__(256) void score_join_rows_kernel(const TfScoreAttnArgs a, int nsplit) {
  const int lane = threadIdx.x & 63;
  const long long rows = (long long)a.B * a.H * a.Sq, row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const float* po = (const float*)a.work + row * a.D;
  const float* pml = (const float*)a.work + (long long)nsplit * rows * a.D + ((long long)min(lane, nsplit - 1) * rows + row) * 2;
  const float m = pml[0], mx = wave_max(m), w = lane < nsplit ? fast_exp2(m - mx) : 0.f, l = wave_sum(w * pml[1]);
  const bool two = a.D <= 128;
  const int step = two ? 2 : 1, first = two ? lane >> 5 : 0, c = (two ? lane & 31 : lane) * 4;
  f32x4 acc = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = 0; s < nsplit; s += step) {
    const float ws = __shfl(w, s + first, 64);           // (0 behind the last part)
    if (c < a.D) acc += ws * *(const f32x4*)(po + (long long)min(s + first, nsplit - 1) * rows * a.D + c);
  }
  if (two) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], 32, 64);
  }
  join_store<F32>(a, row, lane, acc, mx, l);
}

// ================================================================================================
// launchers
// ================================================================================================
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
  f.nqb = (a->Sq + 127) / 128;
  const long long blocks = (long long)a->B * a->H * f.nqb;
  const int tiles = std::max(1, (a->Sk + 63) / 64);
  const int want = split_ways(a->is_f32, a->D, blocks, tiles, 4);
  f.split_tiles = (tiles + want - 1) / want;
  f.nsplit = (tiles + f.split_tiles - 1) / f.split_tiles;
  return f;
}

template <bool F32, int HDP> int launch_fwd(const TfScoreAttnArgs* a, hipStream_t st) {
  const FwdPlan f = fwd_plan(a);
  const bool doc = a->k_doc != nullptr;
  const double fl = 4.0 * a->B * a->H * (double)a->Sq * a->Sk * a->D;
  int rc;
  if (f.few) {
    TfTraceScope tr(F32 ? "score_few32_kernel" : "score_few16_kernel", st, fl);
    const int blocks = a->B * a->Hk * f.nsplit;
    constexpr size_t join = (128 * (size_t)HDP + 256) * 4;
    if constexpr (F32) {
      rc = doc ? launch_lds<score_few32_kernel<HDP, true>>(blocks, join, st, *a, f.nsplit) : launch_lds<score_few32_kernel<HDP, false>>(blocks, join, st, *a, f.nsplit);
    } else {
      constexpr size_t lds = std::max<size_t>(8 * SDma<false, HDP, 32, 1>::BYTES, join);
      rc = doc ? launch_lds<score_few16_kernel<HDP, true>>(blocks, lds, st, *a, f.nsplit) : launch_lds<score_few16_kernel<HDP, false>>(blocks, lds, st, *a, f.nsplit);
    }
  } else {
    TfTraceScope tr(F32 ? "score_fwd_kernel<fp32>" : "score_fwd_kernel<bf16>", st, fl);
    const int blocks = a->B * a->H * f.nqb * f.nsplit;
    constexpr size_t lds = 2 * SDma<F32, HDP, 64, 4>::BYTES + 640;
    auto go = [&](auto ride) {
      return doc ? launch_lds<score_fwd_kernel<F32, HDP, true, decltype(ride)::value>>(blocks, lds, st, *a, f.nqb, f.nsplit, f.split_tiles)
                 : launch_lds<score_fwd_kernel<F32, HDP, false, decltype(ride)::value>>(blocks, lds, st, *a, f.nqb, f.nsplit, f.split_tiles);
    };
    if constexpr (F32) rc = go(std::false_type{});
    else rc = a->softcap == 0.f && a->slopes == nullptr && a->scale > 0.f ? go(std::true_type{}) : go(std::false_type{});
  }
  if (rc != 0) return rc;
  if (f.nsplit > 1) {
    TfTraceScope tr("score_join_kernel", st);
    const unsigned rows = (unsigned)((long long)a->B * a->H * a->Sq);
    if (rows >= 1024 && f.nsplit <= 64) hipLaunchKernelGGL(score_join_rows_kernel<F32>, dim3((rows + 3) / 4), dim3(256), 0, st, *a, f.nsplit);
    else hipLaunchKernelGGL(score_join_kernel<F32>, dim3(rows), dim3(256), 0, st, *a, f.nsplit);
  }
  return (int)hipGetLastError();
}

size_t work_bytes(const TfScoreAttnArgs* a) {
  if (score_check(a) != 0 || a->B == 0 || a->Sq == 0) return 0;
  const FwdPlan f = fwd_plan(a);
  return f.nsplit > 1 ? (size_t)f.nsplit * a->B * a->H * a->Sq * (a->D + 2) * sizeof(float) : 0;
}

}  // namespace

// bytes of TfScoreAttnArgs.work for the forward
extern "C" size_t tf_score_attn_work(int B, int Sq, int Sk, int H, int Hk, int D, int is_f32) {
  TfScoreAttnArgs a{};
  a.B = B; a.Sq = Sq; a.Sk = Sk; a.H = H; a.Hk = Hk; a.D = D; a.is_f32 = is_f32;
  return work_bytes(&a);
}

extern "C" int tf_launch_score_fwd(const TfScoreAttnArgs* a, hipStream_t st) {
  const int rc = score_check(a);
  if (rc != 0) return rc;
  if (a->B == 0 || a->Sq == 0) return 0;
  const int e = a->is_f32 ? 4 : 2;
  if (a->q == nullptr || a->out == nullptr || (a->Sk > 0 && (a->k == nullptr || a->v == nullptr))) return -6;
  if (!score_aligned(a->q, a->q_sb, a->q_ss, a->q_sh, e) || !score_aligned(a->k, a->k_sb, a->k_ss, a->k_sh, e) || !score_aligned(a->v, a->v_sb, a->v_ss, a->v_sh, e) ||
      !score_aligned(a->out, 0, 0, 0, e) || !score_aligned(a->out_lo, 0, 0, 0, e)) return -7;
  const size_t need = work_bytes(a);
  if (need > 0 && (a->work == nullptr || a->work_bytes < need || ((uintptr_t)a->work & 15) != 0)) return -8;
  return by_head_dim(a, [&](auto f32, auto hdp) { return launch_fwd<decltype(f32)::value, decltype(hdp)::value>(a, st); });
}
