// Backward of attention with changed scores (score_attn.h has the mathematics).  With P formed again from the log-sum-exp:
//   dV = P^T dO ;  dP = dO V^T ;  dS = P (dP - delta), delta = rowsum(dO o) ;  dslope = -sum dS |p - j| ;  dS *= 1 - tanh^2 ;
//   dQ = scale dS K ;  dK = scale dS^T Q .
// Two kernels, each with every score of its own rows or keys: seven products where five would do, but no gradient is touched by two
// workgroups, nothing is atomic, and the [Sq, Sk] tensor dS stays out of memory.
//
// Bound by the registers: accumulators and row operands leave room for one wave a SIMD from 96 channels (dk / dv) or 192 (dq) on, so the products,
// the exponentials and the barriers of a tile follow each other more than they overlap (dk / dv at 128 channels: matrix pipe busy 31 % of the
// time, vector pipe 25 %).  4 x 4096 causal, 8 heads of 128: 557 us = 617 TFLOP/s (five products credited, seven computed); 4 x 2048, 16 heads of
// 64: 281 us = 611; 32 x 708, 4 heads of 192: 274 us = 450.  Two forms that were no faster: a tile shared by two waves of a SIMD, P handed over
// through LDS (the first size 606 us where this form took 603), and the next tile's scores formed under this one's products (spilled).
#include "score_attn.h"

namespace {

// Two tiles of T rows that are used together (K and V, or Q and dO) as one image: waves 0 and 1 fetch the first, 2 and 3 the second.  Two
// images, one barrier a pair: the next pair is under way while one is worked on, 32 rows at a time.  WG workgroups share a CU's LDS; T is 64
// where that leaves the room, which halves the barriers (32 x 708, 4 heads of 192: 301 -> 276 us; elsewhere 1 to 2 %).
// (A third image, transfers waited for by count, gained nothing: 4 x 4096 causal, 8 heads of 128, 653 against 603 us, and 4 x 2048, 16 heads of
// 64, 308 either way.)
template <bool F32, int HDP, int WG> struct Pair {
  static constexpr int EXTRA = 6144;      // statistics and documents of the rows, scan of the documents; from 2048 on the slopes' sums
  static constexpr int T = 4 * SDma<F32, HDP, 64, 2>::BYTES + EXTRA <= 160 * 1024 / WG ? 64 : 32;
  using Dma = SDma<F32, HDP, T, 2>;
  static constexpr int HALF = Dma::BYTES, BUF = 2 * HALF, IMAGES = 2 * BUF, LDS = IMAGES + EXTRA;
};
// workgroups a CU (what the registers allow)
constexpr int dq_wgs(bool f32, int hdp) { return hdp <= (f32 ? 64 : 128) ? 2 : 1; }
constexpr int dkv_wgs(bool f32, int hdp, int part) { return hdp <= (f32 ? 32 : part == 2 ? 64 : part == 1 ? 128 : 192) ? 2 : 1; }

// a pair under way: half-tile number (-1: none), full (see TileWalk)
struct Coming { int s = -1; bool full = false; };

// A workgroup's part of the rows: parts [nsplit] of fp32 in the layout of the result, added up by score_finish_kernel
template <bool F32, int DB> __device__ __forceinline__ void store_grad(void* out, float* parts, long long n, int split, int nsplit, long long off,
                                                                       const f32x16 (&x)[DB], float scale, int h, int D, bool ok) {
  if (nsplit > 1) {
    if (ok) store_part<DB>(parts, split * n + off, x, h, D);
  } else {
    store_row<F32, DB>(out, off, x, scale, h, D, ok);
  }
}

// where the parts of the three gradients and of the slopes' row sums lie in the workspace
struct BwdPlan {
  unsigned chunks;                       // of the slopes' rows
  int nqb, nkb, sq, sg, sk;              // splits of dq (keys); of dk / dv: groups of heads x ranges of queries
  size_t o_dk, o_dv, o_rows, o_part, o_far, floats;       // o_far: a word per 32 queries of a head, is one of their log-sum-exps big (see S_BIG)
};

// ================================================================================================
// dq: query on the lane, 128 queries a workgroup; also delta, and the slopes' row sums
// ================================================================================================
template <bool F32, int HDP, bool DOC>
__global__ __launch_bounds__(256, dq_wgs(F32, HDP)) void score_dq_kernel(const TfScoreAttnArgs a, const BwdPlan pl) {
  using G = SGeo<F32, HDP>;
  using PR = Pair<F32, HDP, dq_wgs(F32, HDP)>;
  // fp32 heads of 256 (of 192 with documents): Q, dO and dq do not fit the register file together; Q and dO are read again (from the caches) for every tile
  constexpr bool REREAD = F32 && (HDP > 192 || (HDP > 128 && DOC));
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  u64 (*dsh)[3] = (u64 (*)[3])(smem + PR::IMAGES + 1536);
  int* rsh = (int*)(smem + PR::IMAGES + 1536 + 96);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  int block, group;
  order_blocks(pl.nqb, a.H / a.Hk * pl.sq, a.causal, block, group);
  const int qb = pl.nqb - 1 - block, split = group % pl.sq, bh = group / pl.sq, b = bh / a.H, head = bh % a.H, kvh = head / (a.H / a.Hk);
  const char* qbase = (const char*)a.q + ((long long)b * a.q_sb + (long long)head * a.q_sh) * G::ESZ;
  // this wave's matrix of the pair: K (waves 0, 1) or V
  const char* xbase = wave < 2 ? (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * G::ESZ
                               : (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * G::ESZ;
  const unsigned xrb = (unsigned)(wave < 2 ? a.k_ss : a.v_ss) * G::ESZ;
  const int* kdoc = DOC ? a.k_doc + (size_t)b * a.Sk : nullptr;
  const SMod m = smod(a, head);
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const int w0 = qb * 128 + wave * 32, i = w0 + (lane & 31), ic = min(i, a.Sq - 1);
  const int qd = DOC ? a.q_doc[(size_t)b * a.Sq + ic] : 0;
  const bool live = i < a.Sq && qd >= 0, wave_live = w0 < a.Sq;
  const QRow qr = q_row(a, p0, pfx, w0, i);
  const int hi = key_end(a, p0, pfx, min(qb * 128 + 127, a.Sq - 1));
  const int units = (hi + 31) / 32, u_lo = (int)((long long)units * split / pl.sq), u_hi = (int)((long long)units * (split + 1) / pl.sq);
  StepWalk<DOC, PR::T> walk{{kdoc, (u_hi + 1) / 2, a.Sk, 0, 0, 0, {}, true, false}, -1, u_lo, min(hi, u_hi * 32), true, false};
  if (DOC) doc_range(qd, live, rsh, wave, lane, walk.w.dmin, walk.w.dmax);
  walk.first(dsh, wave, lane);
  const typename PR::Dma dma(wave & 1, lane, xrb, a.D);
  int* kds = (int*)(smem + PR::IMAGES);    // [2 images][64] documents of the keys
  auto fetch = [&](int buf) {
    // (keys behind the last are hidden by the row's limit, whatever document they show)
    if (DOC && wave == 0) __builtin_amdgcn_global_load_lds(TF_GLB_PTR(kdoc + min(walk.s * 32 + lane, a.Sk - 1)), TF_LDS_PTR(kds + buf * 64), 4, 0, 0);
    dma.issue(xbase, xrb, walk.s * 32, hi, a.D, DOC && walk.neg ? kdoc : nullptr, smem + buf * PR::BUF + (wave >> 1) * PR::HALF);
  };
  const long long row = (long long)bh * a.Sq + ic, orow = (((long long)b * a.Sq + ic) * a.H + head) * a.D;
  const char* qrow = qbase + (long long)ic * a.q_ss * G::ESZ;
  SFrag<F32> qf[REREAD ? 1 : G::KS], dof[REREAD ? 1 : G::KS];
  const char* drow = (const char*)a.dout + ((long long)b * a.do_sb + (long long)ic * a.do_ss + (long long)head * a.do_sh) * G::ESZ;
  // delta by the matrix instructions that form dP, from the diagonal of dO O^T: a row that sees one key (o = v) gets dP - delta = 0 exactly
  float delta = 0.f;
  {
    f32x16 dd;
#pragma unroll
    for (int r = 0; r < 16; ++r) dd[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) {
      const SFrag<F32> d = gfrag<F32>(drow, ks, h, a.D, live);
      dd = smma<F32>(gfrag<F32>((const char*)a.out + orow * G::ESZ, ks, h, a.D, live), d, dd);
      if (!F32 && a.out_lo != nullptr) dd = smma<F32>(gfrag<F32>((const char*)a.out_lo + orow * G::ESZ, ks, h, a.D, live), d, dd);
      if constexpr (!REREAD) {
        qf[ks] = gfrag<F32>(qrow, ks, h, a.D, live);
        dof[ks] = d;
      }
      if (F32 && HDP > 128) asm volatile("" ::: "memory");        // (a few loads at a time: the rows of O are not to lie in registers as a whole)
    }
    // element (r & 3) + 8 (r >> 2) + 4 h of column lane & 31
    const int c = lane & 31;
#pragma unroll
    for (int r = 0; r < 16; ++r) delta = h == ((c >> 2) & 1) && r == ((c & 3) | (c >> 3) << 2) ? dd[r] : delta;
    delta += __shfl_xor(delta, 32, 64);
  }
  auto qx = [&](auto I) { if constexpr (REREAD) return gfrag<F32>(qrow, I, h, a.D, live); else return qf[I]; };
  auto dx = [&](auto I) { if constexpr (REREAD) return gfrag<F32>(drow, I, h, a.D, live); else return dof[I]; };
  float lse = live ? a.lse[row] : INFINITY;
  const bool far = !F32 && __any(big(lse));              // (uniform: see S_BIG)
  const int mode = far ? 1 : m.capl == 0.f ? 0 : F32 || a.dslopes != nullptr ? 1 : 2;        // by_flags' CAP; 2: where a tile's scores allow it
  landed(lse);
  landed(delta);
  if constexpr (!REREAD) {
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) { landed(qf[ks]); landed(dof[ks]); }
  }
  Coming cur{};
  auto take = [&](int image) {            // the pair the walk stands at goes to `image`
    if (walk.s < 0) return Coming{};
    fetch(image);
    return Coming{walk.s, walk.full};
  };
  auto go_on = [&](int image) {
    if (walk.s < 0) return Coming{};
    walk.next(dsh, wave, lane);
    return take(image);
  };
  cur = take(0);
  f32x16 dq[G::DB];
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
  // The slopes' gradient of a row is -cov(dP, dist) under P.  Its own sums of P, P e, P dist and P e dist (e = dP - delta) make it exact to fp32: delta
  // holds the roundings of P and of the output, and the mean distance -- hundreds -- would multiply them (2e-3 of the gradient)
  // (in LDS, a tile's sums at a time: the registers are taken)
  f32x4* const sums = (f32x4*)(smem + PR::IMAGES + 2048) + tid;
  if (a.dslopes != nullptr) *sums = f32x4{0, 0, 0, 0};
  const SAddr<F32, HDP> fk0(lds_addr_of(smem), lane);
  int buf = 0;
  while (cur.s >= 0) {
    unsigned todo = 0;                   // (uniform) halves this wave has work in; 4: all of it is visible
#pragma unroll
    for (int hf = 0; hf < PR::T / 32; ++hf) {
      const int kv0 = (cur.s + hf) * 32;
      if (wave_live && kv0 <= qr.lim_hi && (PR::T == 32 || walk.mine(cur.s + hf))) todo |= (cur.full && kv0 + 31 <= qr.lim_lo ? 5u : 1u) << hf;
    }
    dma_wait_barrier();                  // the pair in hand is there, and every wave is done with the one before
    const Coming nxt = go_on(buf ^ 1);
    auto rows32 = [&](int hf) __attribute__((always_inline)) {
      const int kv0 = (cur.s + hf) * 32;
      if ((todo >> hf) & 1u) {
        const bool full_t = (todo >> hf) & 4u;
        const SAddr<F32, HDP> fk = fk0.shifted(buf * PR::BUF + hf * 32 * G::STR);
        f32x16 st, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { st[r] = 0.f; dp[r] = 0.f; }
        mul_rows2<F32, HDP, PR::HALF>(fk, qx, dx, st, dp);
        unsigned bits = 0xffffffffu;
        if (!full_t) {
          bits = low_bits(qr.lim - kv0 + 1);
          if (DOC) {
            unsigned kd = rd32_asm<0>(lds_addr_of(kds + buf * 64 + hf * 32) + (lane & 31) * 4);
            lgkm_wait32<0>(kd);
            bits &= (unsigned)doc_bits(qd, (int)kd);
          }
          bits >>= 4 * h;
        }
        const float pd = (float)(qr.p - kv0 - 4 * h), ncap = m.capl != 0.f ? -1.0f / (m.capl * m.capl) : 0.f;
        SPack<F32> pk[1];
        const f32x16 (&raw)[1] = reinterpret_cast<const f32x16 (&)[1]>(st);
        const int cap = mode == 2 && !all_small<F32, 1>(m, raw) ? 1 : mode;
        auto form = [&](auto FULL, auto CAP, auto SLP, auto SUMS) {
          f32x4 t4 = {0, 0, 0, 0};
          if (!F32 && CAP == 1) {
            if (SUMS && !far) cap_each<SUMS>(m, st);              // (sums: the cap as exactly as fp32 has it)
            else cap_each<false>(m, st);
          }
          auto one = [&](int r) {
            const int j = (r & 3) + 8 * (r >> 2);
            float t = CAP == 2 ? capped_poly(st[r], m.c0, m.c1, m.c2, m.c3) : CAP == 1 ? (F32 ? rounded(capped<true>(m, st[r])) : st[r]) : F32 ? rounded(st[r] * m.sc) : st[r] * m.sc, x = t;
            const float dist = SLP ? fabsf(pd - (float)j) : 0.f;
            if (SLP) x = fmaf(-m.slope2, dist, x);
            float pr = fast_exp2(x - lse);
            x = pr * (dp[r] - delta);
            if (!FULL) x = (bits >> j) & 1u ? x : 0.f;
            if (SUMS) {
              pr = (bits >> j) & 1u ? pr : 0.f;
              t4[0] += pr;
              t4[1] += x;
              t4[2] = fmaf(pr, dist, t4[2]);
              t4[3] = fmaf(x, dist, t4[3]);
            }
            return CAP ? x * fmaf(t * ncap, t, 1.0f) : x;           // the cap's derivative: 1 - (t / cap)^2
          };
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            const float x0 = one(r), x1 = one(r + 1);
            pk[0].set2(r, x0, x1);
          }
          if (SUMS) *sums += t4;
        };
        if (a.dslopes != nullptr) {           // (one form for full and masked tiles)
          if (cap != 0) form(std::false_type{}, std::integral_constant<int, 1>{}, std::true_type{}, std::true_type{});
          else form(std::false_type{}, std::integral_constant<int, 0>{}, std::true_type{}, std::true_type{});
        } else by_flags(full_t, cap, m.slope2 != 0.f, [&](auto FULL, auto CAP, auto SLP) { form(FULL, CAP, SLP, std::false_type{}); });
        fk.template mul_t<0>(pk, dq);
      }
    };
    if constexpr (PR::T == 32) rows32(0);
    else {
#pragma unroll 1
      for (int hf = 0; hf < 2; ++hf) rows32(hf);
    }
    cur = nxt;
    buf ^= 1;
  }
  const long long rows = (long long)a.B * a.H * a.Sq;
  if (a.dslopes != nullptr) {
    f32x4 t = *sums;
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] += __shfl_xor(t[e], 32, 64);
    if (i < a.Sq && h == 0) {
      float* r = (float*)a.work + pl.o_rows + 4 * split * rows + row;
      r[0] = live ? t[0] : 0.f;
      r[rows] = t[1];
      r[2 * rows] = t[2];
      r[3 * rows] = t[3];
    }
  }
  if (i < a.Sq && h == 0 && split == 0) a.delta[row] = delta;
  if (!F32 && lane == 0 && split == 0) ((int*)a.work + pl.o_far)[((size_t)bh * pl.nqb + qb) * 4 + wave] = far;
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = live ? dq[d][r] : 0.f;
  store_grad<F32, G::DB>(a.dq, (float*)a.work, rows * a.D, split, pl.sq, orow, dq, a.scale, h, a.D, i < a.Sq);
}

// ================================================================================================
// dk, dv: key on the lane, 128 keys a workgroup, over the heads that share them and their queries.  PART 0: dv, 1: dk, 2: both
// ================================================================================================
template <bool F32, int HDP, int PART, bool DOC>
__global__ __launch_bounds__(256, dkv_wgs(F32, HDP, PART)) void score_dkv_kernel(const TfScoreAttnArgs a, const BwdPlan pl) {
  using G = SGeo<F32, HDP>;
  using PR = Pair<F32, HDP, dkv_wgs(F32, HDP, PART)>;
  constexpr bool DK = PART != 0, DV = PART != 1;
  constexpr bool REREAD = F32 && HDP > 192;              // as in score_dq_kernel: V is read again for every tile
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float* stat = (float*)(smem + PR::IMAGES);             // [2 images][64 lse, 64 delta]
  int* qds = (int*)(smem + PR::IMAGES + 1024);            // [2 images][64] documents of the queries
  u64 (*dsh)[3] = (u64 (*)[3])(smem + PR::IMAGES + 1536);
  int* rsh = (int*)(smem + PR::IMAGES + 1536 + 96);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int nsplit = pl.sg * pl.sk;
  int kb, group;
  order_blocks(pl.nkb, nsplit, a.causal, kb, group);
  const int split = group % nsplit, bk = group / nsplit, b = bk / a.Hk, kvh = bk % a.Hk, G_ = a.H / a.Hk;
  const char* kbase = (const char*)a.k + ((long long)b * a.k_sb + (long long)kvh * a.k_sh) * G::ESZ;
  const char* vbase = (const char*)a.v + ((long long)b * a.v_sb + (long long)kvh * a.v_sh) * G::ESZ;
  const int* qdoc = DOC ? a.q_doc + (size_t)b * a.Sq : nullptr;
  const int p0 = q_pos0(a, b), pfx = prefix_of(a, b);
  const int k0 = kb * 128, w0 = k0 + wave * 32, j = w0 + (lane & 31), jc = min(j, a.Sk - 1);
  const int kd = DOC ? a.k_doc[(size_t)b * a.Sk + jc] : 0;
  const bool live = j < a.Sk && kd >= 0, wave_live = w0 < a.Sk;
  const char* vrow = vbase + (long long)jc * a.v_ss * G::ESZ;
  SFrag<F32> kf[G::KS], vf[DK && !REREAD ? G::KS : 1];
  // (keys no query sees may hold anything)
  const bool seen = live && (!a.causal || j < pfx || j <= p0 + a.Sq - 1);
#pragma unroll
  for (int ks = 0; ks < G::KS; ++ks) {
    kf[ks] = gfrag<F32>(kbase + (long long)jc * a.k_ss * G::ESZ, ks, h, a.D, seen);
    if constexpr (DK && !REREAD) vf[ks] = gfrag<F32>(vrow, ks, h, a.D, seen);
  }
#pragma unroll
  for (int ks = 0; ks < G::KS; ++ks) {
    landed(kf[ks]);
    if constexpr (DK && !REREAD) landed(vf[ks]);
  }
  auto kx = [&](auto I) { return kf[I]; };
  auto vx = [&](auto I) { if constexpr (REREAD) return gfrag<F32>(vrow, I, h, a.D, seen); else return vf[I]; };
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
  const int s_g = split / pl.sk, s_k = split % pl.sk, g_lo = G_ * s_g / pl.sg, g_hi = G_ * (s_g + 1) / pl.sg;
  const int u0 = i_lo / 32, units = (a.Sq + 31) / 32 - u0;
  const int u_lo = u0 + (int)((long long)units * s_k / pl.sk), u_hi = u0 + (int)((long long)units * (s_k + 1) / pl.sk);
  StepWalk<DOC, PR::T> walk{{qdoc, (u_hi + 1) / 2, a.Sq, 0, 0, 0, {}, true, false}, -1, u_lo, min(a.Sq, u_hi * 32), true, false};
  if (DOC) doc_range(kd, live, rsh, wave, lane, walk.w.dmin, walk.w.dmax);
  const unsigned xrb = (unsigned)(wave < 2 ? a.q_ss : a.do_ss) * G::ESZ;
  const typename PR::Dma dma(wave & 1, lane, xrb, a.D);
  const SAddr<F32, HDP> fq0(lds_addr_of(smem), lane);
  const unsigned stat0 = lds_addr_of(stat) + 16 * h;
  for (int g = g_lo; g < g_hi; ++g) {
    const int head = kvh * G_ + g;
    const SMod m = smod(a, head);
    const char* xbase = wave < 2 ? (const char*)a.q + ((long long)b * a.q_sb + (long long)head * a.q_sh) * G::ESZ
                                 : (const char*)a.dout + ((long long)b * a.do_sb + (long long)head * a.do_sh) * G::ESZ;
    const long long row0 = ((long long)b * a.H + head) * a.Sq;
    bool far = false;                     // as in score_dq_kernel, for all queries of the head
    if (!F32) {
      const int* flag = (const int*)a.work + pl.o_far + ((size_t)b * a.H + head) * pl.nqb * 4;
      int any = 0;
      for (int x = lane; x < pl.nqb * 4; x += 64) any |= flag[x];
      far = __any(any != 0);
    }
    const int mode = far ? 1 : m.capl == 0.f ? 0 : F32 ? 1 : 2;
    auto fetch = [&](int buf) {           // the pair in walk.s, its rows' statistics (waves 0 and 1) and documents, 4 bytes a lane
      const int i0 = walk.s * 32;
      // (queries behind the last are hidden by number, whatever document they show)
      if (DOC && wave == 2) __builtin_amdgcn_global_load_lds(TF_GLB_PTR(qdoc + min(i0 + lane, a.Sq - 1)), TF_LDS_PTR(qds + buf * 64), 4, 0, 0);
      if (wave < 2) {
        const float* src = (wave == 0 ? a.lse : a.delta) + row0 + min(i0 + lane, a.Sq - 1);
        __builtin_amdgcn_global_load_lds(TF_GLB_PTR(src), TF_LDS_PTR(stat + buf * 128 + wave * 64), 4, 0, 0);
      }
      dma.issue(xbase, xrb, i0, a.Sq, a.D, DOC && walk.neg ? qdoc : nullptr, smem + buf * PR::BUF + (wave >> 1) * PR::HALF);
    };
    Coming cur{};
    auto take = [&](int image) {
      if (walk.s < 0) return Coming{};
      fetch(image);
      return Coming{walk.s, walk.full};
    };
    auto go_on = [&](int image) {
      if (walk.s < 0) return Coming{};
      walk.next(dsh, wave, lane);
      return take(image);
    };
    walk.first(dsh, wave, lane);
    if (g > g_lo) __syncthreads();        // every wave is done with the images of the head before
    int buf = 0;
    cur = take(0);
    while (cur.s >= 0) {
      unsigned todo = 0;                 // as in score_dq_kernel
#pragma unroll
      for (int hf = 0; hf < PR::T / 32; ++hf) {
        const int i0 = (cur.s + hf) * 32;
        if (wave_live && i0 + 31 >= q_any && (PR::T == 32 || walk.mine(cur.s + hf))) todo |= (cur.full && i0 >= q_full && i0 + 32 <= a.Sq ? 5u : 1u) << hf;
      }
      dma_wait_barrier();                // the pair in hand is there, and every wave is done with the one before
      const Coming nxt = go_on(buf ^ 1);
      auto rows32 = [&](int hf) __attribute__((always_inline)) {
        const int i0 = (cur.s + hf) * 32;
        if ((todo >> hf) & 1u) {
          const bool full_t = (todo >> hf) & 4u;
          const SAddr<F32, HDP> fq = fq0.shifted(buf * PR::BUF + hf * 32 * G::STR);
          f32x16 st, dp;
#pragma unroll
          for (int r = 0; r < 16; ++r) st[r] = 0.f;
          u32x4 ls[4];                      // register 4 g + e is query 8 g + 4 h + e
          const unsigned sa = stat0 + buf * 512 + hf * 128;
          static_for<4>([&](auto I) { ls[I] = rd128_asm<32 * I>(sa); });
          u32x4 de[4];
          if constexpr (DK) {               // (dP starts at 0 and delta comes off behind it, as in score_dq_kernel)
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] = 0.f;
            mul_rows2<F32, HDP, PR::HALF>(fq, kx, vx, st, dp);
            static_for<4>([&](auto I) { de[I] = rd128_asm<256 + 32 * I>(sa); });
          } else mul_rows<F32, HDP>(fq, kx, st);
          unsigned bits = 0xffffffffu;
          if (!full_t) {
            bits = ~low_bits(max(q_lane - i0, 0)) & low_bits(a.Sq - i0);
            if (DOC) {
              unsigned qd = rd32_asm<0>(lds_addr_of(qds + buf * 64 + hf * 32) + (lane & 31) * 4);
              lgkm_wait32<0>(qd);
              bits &= (unsigned)doc_bits(kd, (int)qd);
            }
            bits >>= 4 * h;
          }
          static_for<4>([&](auto I) { lgkm_wait<0>(ls[I]); if constexpr (DK) lgkm_wait<0>(de[I]); });
          const float pd = (float)(p0 + i0 + 4 * h - j), ncap = m.capl != 0.f ? -1.0f / (m.capl * m.capl) : 0.f;
          SPack<F32> pp[1], ps[1];
          const f32x16 (&raw)[1] = reinterpret_cast<const f32x16 (&)[1]>(st);
          const int cap = mode == 2 && !all_small<F32, 1>(m, raw) ? 1 : mode;
          by_flags(full_t, cap, m.slope2 != 0.f, [&](auto FULL, auto CAP, auto SLP) {
            if (!F32 && CAP == 1) cap_each<false>(m, st);
            // distances: near_pos of the query, less the key
            auto bias = [&](int r, float x, float slope2) {
              return fmaf(slope2, fabsf(__builtin_amdgcn_fmed3f(pd + (float)((r & 3) + 8 * (r >> 2)), (float)-j, (float)(a.Sk - 1 - j))), x);
            };
            constexpr bool EACH = F32 || CAP == 1;       // the bias comes off the score, as in the forward; else it goes to the log-sum-exp (fewer registers)
            float ll[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              ll[r] = f_of(ls[r >> 2][r & 3]);
              if (SLP && !EACH) ll[r] = bias(r, ll[r], m.slope2);
            }
            auto one = [&](int r, float& pr, float& ds) {
              const int q = (r & 3) + 8 * (r >> 2);
              const float t = CAP == 2 ? capped_poly(st[r], m.c0, m.c1, m.c2, m.c3) : CAP == 1 ? (F32 ? rounded(capped<true>(m, st[r])) : st[r]) : F32 ? rounded(st[r] * m.sc) : st[r] * m.sc;
              pr = fast_exp2((SLP && EACH ? bias(r, t, -m.slope2) : t) - ll[r]);
              if (!FULL) pr = (bits >> q) & 1u ? pr : 0.f;
              if constexpr (DK) {
                ds = pr * (dp[r] - f_of(de[r >> 2][r & 3]));
                if (CAP) ds *= fmaf(t * ncap, t, 1.0f);
                if (!FULL) ds = (bits >> q) & 1u ? ds : 0.f;        // (a hidden pair's product may not be finite)
              }
            };
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
              float p0_, p1_, s0_ = 0.f, s1_ = 0.f;
              one(r, p0_, s0_);
              one(r + 1, p1_, s1_);
              if constexpr (DV) pp[0].set2(r, p0_, p1_);
              if constexpr (DK) ps[0].set2(r, s0_, s1_);
            }
          });
          if constexpr (DV) fq.template mul_t<PR::HALF>(pp, dv);
          if constexpr (DK) fq.template mul_t<0>(ps, dk);
        }
      };
      if constexpr (PR::T == 32) rows32(0);
      else {
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) rows32(hf);
      }
      cur = nxt;
      buf ^= 1;
    }
  }
  const long long go = (((long long)b * a.Sk + jc) * a.Hk + kvh) * a.D, n = (long long)a.B * a.Sk * a.Hk * a.D;
  if constexpr (DK) {
#pragma unroll
    for (int d = 0; d < G::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dk[d][r] = live ? dk[d][r] : 0.f;
    store_grad<F32, G::DB>(a.dk, (float*)a.work + pl.o_dk, n, split, nsplit, go, dk, a.scale, h, a.D, j < a.Sk);
  }
  if constexpr (DV) {
#pragma unroll
    for (int d = 0; d < G::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dv[d][r] = live ? dv[d][r] : 0.f;
    store_grad<F32, G::DB>(a.dv, (float*)a.work + pl.o_dv, n, split, nsplit, go, dv, 1.0f, h, a.D, j < a.Sk);
  }
}

// What is left when dq, dk and dv are there, in one launch: the sums of a split gradient's parts (out = scale * (part 0 + part 1 + ...), rounded once; 1024
// values a workgroup) and, by the first H workgroups, the slopes' gradient: from the four sums of each of its rows, in 64 bits and one order.
struct Finish {
  struct Sum { const float* parts; void* out; long long n; int nsplit; unsigned blocks; float scale; } sum[3];
  const float* rows;
  float* dslopes;
  double* part;
  // heads: H, or 0 without slopes; rows: [parts][P, P e, P dist, P e dist][B][H][Sq]; part: [H][chunks] sums of SLOPE_CHUNK rows each where there
  // are more than one
  unsigned heads, B, H, Sq, parts, chunks;
};
// adds up what 256 threads hold, in one order
__device__ __forceinline__ double block_sum(double s, int tid) {
  __shared__ double sh[256];
  sh[tid] = s;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (tid < o) sh[tid] += sh[tid + o];
    __syncthreads();
  }
  return sh[0];
}
// rows lo .. hi - 1 of the B * Sq of a head
__device__ __forceinline__ double slope_rows(const Finish& f, unsigned head, unsigned lo, unsigned hi, int tid) {
  const size_t rows = (size_t)f.B * f.Sq * f.H;
  double s = 0.0;
#pragma unroll 2
  for (unsigned i = lo + tid; i < hi; i += 256) {
    const float* r = f.rows + ((size_t)(i / f.Sq) * f.H + head) * f.Sq + i % f.Sq;
    double p = 0.0, e = 0.0, d = 0.0, ed = 0.0;
#pragma unroll 4
    for (unsigned k = 0; k < f.parts; ++k, r += 4 * rows) {
      p += (double)r[0];
      e += (double)r[rows];
      d += (double)r[2 * rows];
      ed += (double)r[3 * rows];
    }
    if (p != 0.0) s -= (ed - e * d / p) / p;              // -cov(e, dist); a row that sees nothing has none (its p is 0), a NaN goes on
  }
  return block_sum(s, tid);
}
// many rows: a workgroup takes SLOPE_CHUNK rows of a head (one workgroup a head would need half a microsecond for 256 of them)
constexpr unsigned SLOPE_CHUNK = 1024;
__global__ __launch_bounds__(256) void score_slope_kernel(const Finish f) {
  const unsigned head = blockIdx.x / f.chunks, c = blockIdx.x % f.chunks;
  const double s = slope_rows(f, head, c * SLOPE_CHUNK, min(f.B * f.Sq, (c + 1) * SLOPE_CHUNK), threadIdx.x);
  if (threadIdx.x == 0) f.part[blockIdx.x] = s;
}
template <bool F32> __global__ __launch_bounds__(256) void score_finish_kernel(const Finish f) {
  const int tid = threadIdx.x;
  unsigned block = blockIdx.x;
  if (block < f.heads) {
    double s = 0.0;
    if (f.chunks > 1) {
      for (unsigned c = tid; c < f.chunks; c += 256) s += f.part[block * f.chunks + c];
      s = block_sum(s, tid);
    } else s = slope_rows(f, block, 0, f.B * f.Sq, tid);
    if (tid == 0) f.dslopes[block] = (float)s;
    return;
  }
  block -= f.heads;
  int w = 0;
  while (w < 2 && block >= f.sum[w].blocks) block -= f.sum[w++].blocks;
  const Finish::Sum& u = f.sum[w];
  const long long i = ((long long)block * 256 + tid) * 4;
  if (i >= u.n) return;
  f32x4 s = *(const f32x4*)(u.parts + i);
#pragma unroll 4
  for (int k = 1; k < u.nsplit; ++k) s += *(const f32x4*)(u.parts + (long long)k * u.n + i);
  put4<F32>(u.out, i, s[0] * u.scale, s[1] * u.scale, s[2] * u.scale, s[3] * u.scale);
}

// ================================================================================================
// launchers
// ================================================================================================
BwdPlan bwd_plan(const TfScoreAttnArgs* a, bool slopes) {
  BwdPlan p;
  const int G = a->H / a->Hk;
  p.nqb = (a->Sq + 127) / 128;
  p.nkb = (a->Sk + 127) / 128;
  // Too few workgroups for 256 CUs: the loops are split.  dk / dv are split by heads first (each is a loop of its own), and up to four a CU:
  // with shared heads a workgroup's loop is long and uneven.
  const long long bq = (long long)a->B * a->H * p.nqb, bk = (long long)a->B * a->Hk * p.nkb;
  p.sq = split_ways(a->is_f32, a->D, bq, (a->Sk + 31) / 32, 4);
  p.sg = bk == 0 ? 1 : (int)std::max(1ll, std::min({(1024 + bk - 1) / bk, (long long)G, (long long)G * ((a->Sq + 31) / 32) / 8}));
  p.sk = split_ways(a->is_f32, a->D, bk * p.sg, (a->Sq + 31) / 32, 4);
  const size_t nq = (size_t)a->B * a->Sq * a->H * a->D, nk = (size_t)a->B * a->Sk * a->Hk * a->D, ns = (size_t)p.sg * p.sk;
  p.o_dk = p.sq > 1 ? p.sq * nq : 0;
  p.o_dv = p.o_dk + (ns > 1 ? ns * nk : 0);
  p.o_rows = p.o_dv + (ns > 1 ? ns * nk : 0);
  p.chunks = slopes ? (unsigned)(((long long)a->B * a->Sq + SLOPE_CHUNK - 1) / SLOPE_CHUNK) : 0;
  p.o_part = (p.o_rows + (slopes ? 4 * (size_t)p.sq * a->B * a->H * a->Sq : 0) + 1) / 2 * 2;
  p.o_far = p.o_part + (p.chunks > 1 ? 2 * (size_t)p.chunks * a->H : 0);
  p.floats = p.o_far + (a->is_f32 ? 0 : 4 * (size_t)a->B * a->H * p.nqb);
  return p;
}

template <bool F32, int HDP> int launch_bwd(const TfScoreAttnArgs* a, hipStream_t st) {
  const double fl = 4.0 * a->B * a->H * (double)a->Sq * a->Sk * a->D;
  const BwdPlan pl = bwd_plan(a, a->dslopes != nullptr);
  const bool doc = a->k_doc != nullptr;
  int rc = 0;
  if (const int blocks = a->B * a->H * pl.nqb * pl.sq; blocks > 0) {
    TfTraceScope tr(F32 ? "score_dq_kernel<fp32>" : "score_dq_kernel<bf16>", st, 1.5 * fl);
    constexpr size_t lds = Pair<F32, HDP, dq_wgs(F32, HDP)>::LDS;
    rc = doc ? launch_lds<score_dq_kernel<F32, HDP, true>>(blocks, lds, st, *a, pl) : launch_lds<score_dq_kernel<F32, HDP, false>>(blocks, lds, st, *a, pl);
  }
  if (rc != 0) return rc;
  if (const int blocks = a->B * a->Hk * pl.nkb * pl.sg * pl.sk; blocks > 0) {
    TfTraceScope tr(F32 ? "score_dkv_kernel<fp32>" : "score_dkv_kernel<bf16>", st, 2.0 * fl);
    auto part = [&](auto which) {
      constexpr int PART = decltype(which)::value;
      constexpr size_t lds = Pair<F32, HDP, dkv_wgs(F32, HDP, PART)>::LDS;
      return doc ? launch_lds<score_dkv_kernel<F32, HDP, PART, true>>(blocks, lds, st, *a, pl) : launch_lds<score_dkv_kernel<F32, HDP, PART, false>>(blocks, lds, st, *a, pl);
    };
    if constexpr (HDP <= (F32 ? 128 : 192)) rc = part(std::integral_constant<int, 2>{});
    else {
      rc = part(std::integral_constant<int, 0>{});
      if (rc == 0) rc = part(std::integral_constant<int, 1>{});
    }
  }
  if (rc != 0) return rc;
  const int ns = pl.sg * pl.sk;
  Finish f{};
  f.rows = (const float*)a->work + pl.o_rows;
  f.dslopes = a->dslopes;
  f.heads = a->dslopes != nullptr ? a->H : 0;
  f.H = a->H;
  f.Sq = a->Sq;
  f.B = a->B;
  f.parts = pl.sq;
  f.chunks = pl.chunks;
  f.part = (double*)((float*)a->work + pl.o_part);
  unsigned blocks = f.heads;
  auto add = [&](int w, size_t off, long long n, int nsplit, float scale, void* out) {
    const unsigned need = nsplit > 1 ? (unsigned)((n / 4 + 255) / 256) : 0;
    f.sum[w] = {(const float*)a->work + off, out, n, nsplit, need, scale};
    blocks += need;
  };
  add(0, 0, (long long)a->B * a->Sq * a->H * a->D, pl.sq, a->scale, a->dq);
  add(1, pl.o_dk, (long long)a->B * a->Sk * a->Hk * a->D, ns, a->scale, a->dk);
  add(2, pl.o_dv, (long long)a->B * a->Sk * a->Hk * a->D, ns, 1.0f, a->dv);
  if (f.heads > 0 && f.chunks > 1) {
    TfTraceScope tr("score_slope_kernel", st);
    hipLaunchKernelGGL(score_slope_kernel, dim3(f.heads * f.chunks), dim3(256), 0, st, f);
  }
  if (blocks > 0) {
    TfTraceScope tr("score_finish_kernel", st);
    hipLaunchKernelGGL(score_finish_kernel<F32>, dim3(blocks), dim3(256), 0, st, f);
  }
  return (int)hipGetLastError();
}

}  // namespace

// bytes of TfScoreAttnArgs.work for the backward
extern "C" size_t tf_score_attn_bwd_work(int B, int Sq, int Sk, int H, int Hk, int D, int is_f32, int slopes) {
  TfScoreAttnArgs a{};
  a.B = B; a.Sq = Sq; a.Sk = Sk; a.H = H; a.Hk = Hk; a.D = D; a.is_f32 = is_f32;
  return score_check(&a) != 0 ? 0 : bwd_plan(&a, slopes != 0).floats * sizeof(float);
}

extern "C" int tf_launch_score_bwd(const TfScoreAttnArgs* a, hipStream_t st) {
  const int rc = score_check(a);
  if (rc != 0) return rc;
  const int e = a->is_f32 ? 4 : 2;
  if (a->B > 0 && a->Sq > 0 && (a->q == nullptr || a->out == nullptr || a->dout == nullptr || a->dq == nullptr || a->lse == nullptr || a->delta == nullptr)) return -6;
  if (a->B > 0 && a->Sk > 0 && (a->k == nullptr || a->v == nullptr || a->dk == nullptr || a->dv == nullptr)) return -6;
  if (a->dslopes != nullptr && a->slopes == nullptr) return -6;
  if (!score_aligned(a->q, a->q_sb, a->q_ss, a->q_sh, e) || !score_aligned(a->k, a->k_sb, a->k_ss, a->k_sh, e) || !score_aligned(a->v, a->v_sb, a->v_ss, a->v_sh, e) ||
      !score_aligned(a->dout, a->do_sb, a->do_ss, a->do_sh, e) || !score_aligned(a->out, 0, 0, 0, e) || !score_aligned(a->out_lo, 0, 0, 0, e) ||
      !score_aligned(a->dq, 0, 0, 0, e) || !score_aligned(a->dk, 0, 0, 0, e) || !score_aligned(a->dv, 0, 0, 0, e)) return -7;
  const size_t need = bwd_plan(a, a->dslopes != nullptr).floats * sizeof(float);
  if (need > 0 && (a->work == nullptr || a->work_bytes < need || ((uintptr_t)a->work & 15) != 0)) return -8;
  return by_head_dim(a, [&](auto f32, auto hdp) { return launch_bwd<decltype(f32)::value, decltype(hdp)::value>(a, st); });
}
