// Backward of the attention to encoder states for few keys (up to 96 at the narrow heads: a caption's 77 tokens): one pass.
//
// With so few keys a wave holds ALL probabilities and score gradients of its 32 queries in registers (queries on the lanes,
// KT tiles of 32 keys), so the scores are computed once -- two kernels, one per operand side, would compute them twice --
// and delta = sum_k P dP comes from the very values it is subtracted from: O is not read, and its rounding to bf16 is in no
// gradient.  dS^T is directly the operand of dQ^T = K^T dS^T.  dV and dK reduce over the queries, so P and dS go through a
// small LDS tile of the wave's own (written [query][key], read transposed), against dO and Q from a second one.  The waves
// of a workgroup keep dK and dV in registers over all their query tiles, add them up in wave order at the end, and leave
// one fp32 partial per workgroup, which cross_gather_kernel sums in a fixed order: no atomics.
//
// Bound by the vector work per score at two waves per SIMD (the registers of dK and dV).  64 x 2304 queries, 8 heads of 16, 77
// tokens: bf16 48 us (55.8 with all 77 valid); 8 x 576, 8 heads of 32, fp32 32 us with the sum.
#include "dm_cross.h"

namespace {

using namespace dm_cross;

template <typename T> constexpr int patch_stride() { return sizeof(T) == 2 ? 72 : 144; }   // 32 keys + padding: writes without conflicts
// P / dS tile pairs that go through LDS together: all of them in bf16, one at a time in fp32 (twice the bytes, and bound by
// its matrix instructions anyway)
template <typename T, int KT> constexpr int pairs() { return sizeof(T) == 2 ? KT : 1; }
// In bf16 the operands P and dS are rounded (half a step, 2^-8 of each value).  Sums over few queries or keys do not even that
// out, so for one tile of keys both go in as two bf16 numbers, the value and what its rounding left: one more matrix
// instruction per product where these are few.  With more tiles it would be a fifth of the kernel's work.
template <typename T, int KT> constexpr bool two_terms() { return sizeof(T) == 2 && KT == 1; }
template <typename T, int HDP, int KT> constexpr int wave_lds() {
  return 2 * 32 * Geo<T, HDP>::ST + (pairs<T, KT>() + two_terms<T, KT>()) * 2 * 32 * patch_stride<T>();
}
template <typename T, int HDP, int KT> constexpr int few_lds() {
  const int keys = KT * 32 * (2 * Geo<T, HDP>::SR + 4) + 32, loop = keys + 4 * wave_lds<T, HDP, KT>();
  const int sums = 2 * KT * 32 * (HDP + 4) * 4;
  return loop > sums ? loop : sums;
}

// waves per SIMD that the registers allow (dK and dV alone take 32 KT HDP / 32)
template <typename T, int HDP, int KT> constexpr int few_waves() {
  return HDP * KT <= (sizeof(T) == 2 ? 64 : 32) ? 2 : 1;
}

// dK^T or dV^T of one tile of 32 keys, and what is added to it: X^T (LDS, 32 queries) times the P or dS tile (LDS patch).
// 16-wide heads in bf16 use the 16x16 tiles, which they fill: half the registers of a 32x32 one.
template <typename T, int HDP> struct KvAcc {
  static constexpr int N = Geo<T, HDP>::DT;
  f32x16 a[N];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int d = 0; d < N; ++d) a[d] = zero16();
  }
  __device__ __forceinline__ void add(const char* x, const char* patch, int f, int lane) {
    const typename Cr<T>::frag pf = tr_frag<T, 32>(patch, patch_stride<T>(), f, 0, lane);
#pragma unroll
    for (int d = 0; d < N; ++d) a[d] = Cr<T>::mma(tr_frag<T, HDP>(x, Geo<T, HDP>::ST, f, d, lane), pf, a[d]);
  }
  // four consecutive channels at a time: f(key in the tile, channel, values)
  template <typename F> __device__ __forceinline__ void each(int lane, const F& f) {
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
      for (int i = 0; i < (HDP < 32 ? 2 : 4); ++i)
        f(lane & 31, d * 32 + 8 * i + 4 * (lane >> 5), f32x4{a[d][4 * i], a[d][4 * i + 1], a[d][4 * i + 2], a[d][4 * i + 3]});
  }
};
template <> struct KvAcc<bf16, 16> {
  f32x4 a[2];      // keys 0..15 and 16..31
  __device__ __forceinline__ void clear() { a[0] = a[1] = f32x4{0.f, 0.f, 0.f, 0.f}; }
  static __device__ __forceinline__ bf16x8 operand(const char* tile, int stride, int lane) {
    typedef s16x4 __attribute__((address_space(3))) * lds_ptr;
    const char* at = tile + (8 * (lane >> 4) + ((lane & 15) >> 2)) * stride + (lane & 3) * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 4 * stride));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  __device__ __forceinline__ void add(const char* x, const char* patch, int f, int lane) {
    if (f) return;      // (one instruction reduces over all 32 queries)
    const bf16x8 xt = operand(x, Geo<bf16, 16>::ST, lane);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      a[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xt, operand(patch + 32 * k, patch_stride<bf16>(), lane), a[k], 0, 0, 0);
  }
  template <typename F> __device__ __forceinline__ void each(int lane, const F& f) {
#pragma unroll
    for (int k = 0; k < 2; ++k) f(16 * k + (lane & 15), 4 * (lane >> 4), a[k]);
  }
};

// N of the tile's 32 rows (keys)
template <typename T, int N> __device__ __forceinline__ void put_tile(char* patch, const f32x16& s, int lane) {
#pragma unroll
  for (int i = 0; i < N / 8; ++i)
    store4<T>(patch + (lane & 31) * patch_stride<T>() + (8 * i + 4 * (lane >> 5)) * (int)sizeof(T), s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
}

// NT tiles of 32 keys against the wave's 32 queries: dk, dv += ..., dq = ... .  All tiles go through each stage together, so
// that one tile's exponentials run beside the next one's matrix instructions.  HALF: the last tile has at most 16 keys; what
// its other columns of dk and dv become is nothing that is kept.
template <typename T, int HDP, int KT, int NT, bool HALF, bool DROP, typename Next>
__device__ __forceinline__ void few_step(const CrossParams& p, const char* sK, const char* sV, const float* bias, const char* sQ,
                                         const char* sD, char* patch, const typename Cr<T>::frag (&qf)[Geo<T, HDP>::NC],
                                         const typename Cr<T>::frag (&df)[Geo<T, HDP>::NC], float lse2, float c, uint32_t rs,
                                         KvAcc<T, HDP> (&dk)[KT], KvAcc<T, HDP> (&dv)[KT],
                                         f32x16 (&dq)[Geo<T, HDP>::DT], int lane, const Next& next) {
  typedef Geo<T, HDP> Gm;
  typedef typename Cr<T>::frag frag;
  constexpr int PS = patch_stride<T>(), NF = Cr<T>::NF, PT = pairs<T, KT>();
  const int half = lane >> 5;
  f32x16 pr[NT], dp[NT];
  uint32_t keep[NT];
  float delta = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    f32x16 s = score_init(bias + t * 32, half), e = zero16();
#pragma unroll
    for (int kc = 0; kc < Gm::NC; ++kc) {
      s = Cr<T>::mma(row_frag<T>(sK + t * 32 * Gm::SR, Gm::SR, kc, lane), qf[kc], s);
      e = Cr<T>::mma(row_frag<T>(sV + t * 32 * Gm::SR, Gm::SR, kc, lane), df[kc], e);
    }
    pr[t] = s;
    dp[t] = e;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (DROP) {
      keep[t] = 0;
#pragma unroll
      for (int i = 0; i < (HALF && t == NT - 1 ? 8 : 16); i += 2) {
        const uint32_t z = dm_drop_bits(rs, (uint32_t)(t * 32 + tile_row(i, half)) >> 1);
        const bool k0 = dm_keep16(z, 0, p.thresh), k1 = dm_keep16(z, 1, p.thresh);
        keep[t] |= (k0 ? 1u : 0u) << i | (k1 ? 2u : 0u) << i;
        dp[t][i] = k0 ? dp[t][i] * p.inv_keep : 0.f;
        dp[t][i + 1] = k1 ? dp[t][i + 1] * p.inv_keep : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < (HALF && t == NT - 1 ? 8 : 16); ++i) {
      pr[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(pr[t][i], c, -lse2));
      delta = __builtin_fmaf(pr[t][i], dp[t][i], delta);
    }
  }
  delta = half_sum(delta);
  next();                       // the next tile's rows fly during the products below
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < (HALF && t == NT - 1 ? 8 : 16); ++i) dp[t][i] = pr[t][i] * (dp[t][i] - delta);
    if (DROP) {
#pragma unroll
      for (int i = 0; i < (HALF && t == NT - 1 ? 8 : 16); ++i) pr[t][i] = keep[t] >> i & 1u ? pr[t][i] * p.inv_keep : 0.f;
    }
  }
  f32x16 rest, prest;  // of dS and P, where they have two terms (of the rows that hold no key: nothing that is kept)
  if constexpr (two_terms<T, KT>()) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      rest[i] = dp[0][i] - (float)(T)dp[0][i];
      prest[i] = pr[0][i] - (float)(T)pr[0][i];
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int f = 0; f < (HALF && t == NT - 1 ? NF / 2 : NF); ++f) {
      const frag sf = Cr<T>::pack(dp[t], f);
      if constexpr (two_terms<T, KT>()) {
        const frag rf = Cr<T>::pack(rest, f);
#pragma unroll
        for (int d = 0; d < Gm::DT; ++d)
          dq[d] = Cr<T>::mma(tr_frag<T, HDP>(sK, Gm::SR, f, d, lane), rf, f == 0 ? zero16() : dq[d]);
      }
#pragma unroll
      for (int d = 0; d < Gm::DT; ++d)
        dq[d] = Cr<T>::mma(tr_frag<T, HDP>(sK + t * 32 * Gm::SR, Gm::SR, f, d, lane), sf,
                           t == 0 && f == 0 && !two_terms<T, KT>() ? zero16() : dq[d]);
      if (KT > 1 && HDP > 16) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
  for (int t0 = 0; t0 < NT; t0 += PT) {
#pragma unroll
    for (int t = t0; t < NT && t < t0 + PT; ++t) {
      constexpr int ALL = 32, SOME = 16;
      if (HALF && t == NT - 1) {
        put_tile<T, SOME>(patch + 2 * (t - t0) * 32 * PS, pr[t], lane);
        put_tile<T, SOME>(patch + (2 * (t - t0) + 1) * 32 * PS, dp[t], lane);
      } else {
        put_tile<T, ALL>(patch + 2 * (t - t0) * 32 * PS, pr[t], lane);
        put_tile<T, ALL>(patch + (2 * (t - t0) + 1) * 32 * PS, dp[t], lane);
      }
    }
    if constexpr (two_terms<T, KT>()) {
      put_tile<T, HALF ? 16 : 32>(patch + 2 * 32 * PS, prest, lane);
      put_tile<T, HALF ? 16 : 32>(patch + 3 * 32 * PS, rest, lane);
    }
    wave_lds_order();
#pragma unroll
    for (int f = 0; f < NF; ++f) {
#pragma unroll
      for (int t = t0; t < NT && t < t0 + PT; ++t) {
        dv[t].add(sD, patch + 2 * (t - t0) * 32 * PS, f, lane);
        dk[t].add(sQ, patch + (2 * (t - t0) + 1) * 32 * PS, f, lane);
        if constexpr (two_terms<T, KT>()) {
          dv[t].add(sD, patch + 2 * 32 * PS, f, lane);
          dk[t].add(sQ, patch + 3 * 32 * PS, f, lane);
        }
      }
      if (KT > 1 && HDP > 16) __builtin_amdgcn_sched_barrier(0);      // (all operand reads at once would not fit the registers)
    }
    wave_lds_order();
  }
}

// HEADS: a workgroup takes every query head of its key / value head (small calls), not a share of one head's queries.
template <typename T, int HDP, int KT, bool DROP, bool HEADS>
__global__ __launch_bounds__(256, (few_waves<T, HDP, KT>())) void cross_few_kernel(const CrossParams p) {
  typedef Geo<T, HDP> Gm;
  typedef typename Cr<T>::frag frag;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* sK = smem;
  char* sV = sK + KT * 32 * Gm::SR;
  float* bias = reinterpret_cast<float*>(sV + KT * 32 * Gm::SR);
  uint32_t* bits = reinterpret_cast<uint32_t*>(bias + KT * 32);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  char* sQ = reinterpret_cast<char*>(bits + 8) + wave * wave_lds<T, HDP, KT>();
  char* sD = sQ + 32 * Gm::ST;
  char* patch = sD + 32 * Gm::ST;
  // a workgroup's units are tiles of 32 queries
  const int HB = HEADS ? p.H / p.G : 1;
  uint32_t id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int h0 = (int)(id % (uint32_t)(p.H / HB)) * HB;
  id /= (uint32_t)(p.H / HB);
  const int qb = id % p.nqb, b = id / p.nqb;
  const int ctx = context_of(p, b), kn = keys_of(p, ctx);
  const int hdb = p.hd * (int)sizeof(T), g = h0 / (p.H / p.G);
  const int tiles_q = (p.Nq + 31) >> 5, units = HEADS ? HB * tiles_q : min(tiles_q, (qb + 1) * p.iters * 4);
  const long krow = (long)(ctx < 0 ? 0 : ctx) * p.Nk;
  const unsigned char* mask = p.mask ? p.mask + krow : nullptr;
  const float c = p.scale * CR_LOG2E;
  const uint32_t seed = DROP ? dm_eff_seed(p.seed, p.seed_ctr) : 0u;
  const long tok = (long)b * p.Nq;

  frag qf[Gm::NC], df[Gm::NC];
  float L2;
  auto fetch = [&](int unit) {
    const int hh = HEADS ? unit / tiles_q : 0, h = h0 + hh, q = (unit - hh * tiles_q) * 32, left = p.Nq - q;
    load_frags<T, HDP>(rows_of(p.q + (tok + q) * p.ldq + h * hdb, p.ldq, left, hdb, lane), hdb, lane, qf);
    load_frags<T, HDP>(rows_of(p.d_o + (tok + q) * p.lddo + h * hdb, p.lddo, left, hdb, lane), hdb, lane, df);
    L2 = p.lse[((long)b * p.H + h) * p.Nq + min(q + (lane & 31), p.Nq - 1)];
  };
  const int first = qb * p.iters * 4 + wave;
  fetch(min(first, units - 1));
  stage_rows2<T, HDP>(sK, Gm::SR, p.k + krow * p.ldk + g * hdb, p.ldk, sV, Gm::SR, p.v + krow * p.ldv + g * hdb, p.ldv, 0,
                      KT * 32, kn, mask, hdb, tid);
  stage_valid(bits, bias, 0, KT * 32, kn, mask, tid);
  __syncthreads();
  int tiles = 0;       // up to the last one with a valid key
  bool some = false;   // which has none past its first 16
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane((int)bits[t]);
    if (w) { tiles = t + 1; some = (w >> 16) == 0; }
  }
  KvAcc<T, HDP> dk[KT], dv[KT];
#pragma unroll
  for (int t = 0; t < KT; ++t) { dk[t].clear(); dv[t].clear(); }

  // one loop for each number of tiles, so that each keeps only its own LDS addresses in registers
  auto each = [&](auto step) {
    for (int unit = first; unit < units; unit += 4) {
      const int hh = HEADS ? unit / tiles_q : 0, hq = h0 + hh, q0 = (unit - hh * tiles_q) * 32;
      const long row = ((long)b * p.H + hq) * p.Nq;
      // a query past the end, and one without a finite score, has no probabilities
      const float lse2 = L2 == -INFINITY || q0 + (lane & 31) >= p.Nq ? INFINITY : L2 * CR_LOG2E;
#pragma unroll
      for (int kc = 0; kc < Gm::NC; ++kc) {
        *reinterpret_cast<frag*>(sQ + (lane & 31) * Gm::ST + kc * 32 + half * 16) = qf[kc];
        *reinterpret_cast<frag*>(sD + (lane & 31) * Gm::ST + kc * 32 + half * 16) = df[kc];
      }
      const uint32_t rs = DROP ? dm_drop_row(seed, (uint32_t)(row + q0 + (lane & 31))) : 0u;
      f32x16 dq[Gm::DT];
      wave_lds_order();
      step(lse2, rs, dq, [&]() { if (unit + 4 < units) fetch(unit + 4); });
      const Rows dst = rows_of(p.dq + (tok + q0) * p.lddq + hq * hdb, p.lddq, p.Nq - q0, hdb, lane);
#pragma unroll
      for (int d = 0; d < Gm::DT; ++d) store_tile<T>(dst, dq[d], p.scale, d * 32, hdb, lane);
    }
  };
#define DM_FEW(NT, HALF) each([&](float lse2, uint32_t rs, f32x16 (&dq)[Gm::DT], const auto& next) { \
    few_step<T, HDP, KT, NT, HALF, DROP>(p, sK, sV, bias, sQ, sD, patch, qf, df, lse2, c, rs, dk, dv, dq, lane, next); })
  if (tiles == 0) {
    each([&](float, uint32_t, f32x16 (&dq)[Gm::DT], const auto&) {
#pragma unroll
      for (int d = 0; d < Gm::DT; ++d) dq[d] = zero16();
    });
  } else if (tiles == 1) {
    if (some) DM_FEW(1, true); else DM_FEW(1, false);
  } else if (KT > 1 && tiles == 2) {
    constexpr int N2 = KT > 1 ? 2 : 1;
    if (some) DM_FEW(N2, true); else DM_FEW(N2, false);
  } else if (KT > 2) {
    constexpr int N3 = KT > 2 ? 3 : 1;
    if (some) DM_FEW(N3, true); else DM_FEW(N3, false);
  }
#undef DM_FEW

  // dK, dV of the four waves, added in wave order: [dk | dv][key][channel]
  constexpr int RS = HDP + 4;
  float* sum = reinterpret_cast<float*>(smem);
#pragma unroll 1
  for (int turn = 0; turn < 4; ++turn) {
    __syncthreads();
    if (turn != wave) continue;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int which = 0; which < 2; ++which)
        (which ? dv[t] : dk[t]).each(lane, [&](int key, int col, f32x4 v) {
          f32x4* at = reinterpret_cast<f32x4*>(sum + ((which * KT + t) * 32 + key) * RS + col);
          if (turn) v += *at;
          *at = v;
        });
  }
  __syncthreads();
  if (ctx < 0) return;
  const int per = p.hd >> 2, n = p.Nk * per;
  for (int i = tid; i < 2 * n; i += 256) {
    const int which = i >= n, e = which ? i - n : i, key = e / per, col = (e - key * per) * 4;
    const bool counts = key < kn && (!mask || mask[key]);
    const f32x4 v = counts ? *reinterpret_cast<const f32x4*>(sum + (which * KT * 32 + key) * RS + col) : f32x4{0.f, 0.f, 0.f, 0.f};
    if (p.nsplit) {
      *reinterpret_cast<f32x4*>(p.part + ((((long)b * p.H + h0) * p.nqb + qb) * 2 + which) * p.Nk * p.hd + (long)key * p.hd + col) = v;
    } else {
      const float f = which ? 1.f : p.scale;
      char* dst = which ? p.dv + (krow + key) * p.lddv : p.dk + (krow + key) * p.lddk;
      store4<T>(dst + g * hdb + col * (int)sizeof(T), v[0] * f, v[1] * f, v[2] * f, v[3] * f);
    }
  }
}

// dk, dv of context c: the partials of every sample that uses it (in order), of the heads of the group and of the query
// shares.  SL lanes split the list of one result (4 channels) and join by a fixed tree: 8 for long lists, 1 for short ones.
template <typename T, int SL>
__global__ __launch_bounds__(256) void cross_gather_kernel(const CrossParams p) {
  constexpr int RPW = 64 / SL;                             // results per wave
  const int lane = threadIdx.x & 63, slice = lane / RPW;
  const int per = p.hd >> 2, HG = p.H / p.G, U = HG * p.nqb;
  const long n = (long)p.G * 2 * p.Nk * per;               // results of a context; p.iters workgroups share one
  const int ctx = blockIdx.x / p.iters;
  const long i = ((long)(blockIdx.x % p.iters) * 4 + (threadIdx.x >> 6)) * RPW + lane % RPW;
  const long r = i < n ? i : n - 1;
  const long gw = r / per, kw = gw / p.Nk;
  const int col = (int)(r - gw * per) * 4, key = (int)(gw - kw * p.Nk), which = (int)(kw & 1), g = (int)(kw >> 1);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  int m = 0;
  auto add = [&](int b) {
    for (int u = (slice - m * U) & (SL - 1); u < U; u += SL) {
      const long src = (((long)b * p.H + g * HG) * p.nqb + u) * 2 + which;      // (a head's shares are adjacent: hh * nqb + share)
      s += *reinterpret_cast<const f32x4*>(p.part + (src * p.Nk + key) * p.hd + col);
    }
    ++m;
  };
  if (!p.index) {
    if (p.Bc == 1) for (int b = 0; b < p.B; ++b) add(b);
    else add(ctx);
  } else {
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      unsigned long long hit = __ballot(b0 + lane < p.B && p.index[min(b0 + lane, p.B - 1)] == ctx);
      for (; hit; hit &= hit - 1) add(b0 + __builtin_ctzll(hit));
    }
  }
  if (SL > 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int o = RPW; o < 64; o <<= 1) s[j] += __shfl_xor(s[j], o, 64);
  }
  if (i >= n || slice) return;
  const float f = which ? 1.f : p.scale;
  const long krow = (long)ctx * p.Nk + key;
  char* dst = which ? p.dv + krow * p.lddv : p.dk + krow * p.lddk;
  store4<T>(dst + (g * p.hd + col) * (long)sizeof(T), s[0] * f, s[1] * f, s[2] * f, s[3] * f);
}

template <typename T, int HDP, int KT, bool DROP, bool HEADS>
int launch(const CrossParams& p, hipStream_t st) {
  auto kern = cross_few_kernel<T, HDP, KT, DROP, HEADS>;
  constexpr int lds = few_lds<T, HDP, KT>();
  static_assert(lds <= 160 * 1024, "LDS");
  const long blocks = (long)p.B * p.nqb * (HEADS ? p.G : p.H);
  if (blocks > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
  static unsigned long long attr_devs = 0ull;
  if (dm_first_on_device(attr_devs) &&
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
    return DM_ERR_LAUNCH;
  static const DmVariantName nm("cross_bwd_few<%s,%d,KT=%d>", sizeof(T) == 2 ? "bf16" : "fp32", HDP, KT);
  dm_set_variant(nm.s);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), lds, st, p);
  DM_LAUNCH_CHECK();
  if (p.nsplit) {
    const long n = (long)p.G * 2 * p.Nk * (p.hd >> 2);
    const bool wide = (long)((p.B + p.Bc - 1) / p.Bc) * (p.H / p.G) * p.nqb > 4;
    CrossParams g = p;
    g.iters = (int)((n + (wide ? 31 : 255)) / (wide ? 32 : 256));
    const long gb = (long)p.Bc * g.iters;
    if (gb > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
    if (wide) hipLaunchKernelGGL((cross_gather_kernel<T, 8>), dim3((unsigned)gb), dim3(256), 0, st, g);
    else hipLaunchKernelGGL((cross_gather_kernel<T, 1>), dim3((unsigned)gb), dim3(256), 0, st, g);
    DM_LAUNCH_CHECK();
  }
  return DM_OK;
}
// tiles of 32 keys that a wave's registers hold beside the rest
constexpr int most_tiles(int hdp, int esize) { return hdp <= 32 ? 3 : (esize == 2 && hdp == 64 ? 2 : 1); }
template <typename T, int HDP, int KT, bool HEADS> int pick_drop(const CrossParams& p, hipStream_t st) {
  return p.thresh ? launch<T, HDP, KT, true, HEADS>(p, st) : launch<T, HDP, KT, false, HEADS>(p, st);
}
template <typename T, int HDP> int pick(const CrossParams& p, const FewPlan& f, hipStream_t st) {
  if constexpr (HDP <= 32)
    if (f.heads) return pick_drop<T, HDP, 1, true>(p, st);
  if (f.kt == 1) return pick_drop<T, HDP, 1, false>(p, st);
  constexpr int KT = most_tiles(HDP, sizeof(T));
  if constexpr (KT > 1) return pick_drop<T, HDP, KT, false>(p, st);
  return DM_ERR_ARG;
}

}  // namespace

namespace dm_cross {

bool few_plan(const dm_cross_args* a, FewPlan& f) {
  const int hdp = cross_hdp(a->hd);
  const int most = most_tiles(hdp, a->dtype == 0 ? 2 : 4);
  if (a->Nk < 1 || a->Nk > 32 * most || (a->dtype != 0 && hdp > 64)) return false;
  f.kt = a->Nk <= 32 ? 1 : most;
  const long pairs = (long)a->B * a->heads, groups = ((long)a->Nq + 127) / 128;      // one tile per wave of a workgroup
  // one round of workgroups over the device: a second one would stage the keys and add up dK / dV again (B=64, 8 heads of 16,
  // 2304 queries, 77 tokens: 55.8 us at one round, 61.2 at two; fp32, 64 pairs of 576 queries: 32.3 at one, 42.5 at two)
  const int cap = 256 * (hdp * f.kt <= (a->dtype == 0 ? 64 : 32) ? 2 : 1);
  long nqb = cap / pairs;
  if (nqb < 1) nqb = 1;
  if (nqb > groups) nqb = groups;
  f.iters = (int)((groups + nqb - 1) / nqb);
  f.nqb = (int)((groups + f.iters - 1) / f.iters);
  // a small call lets one workgroup take all the heads that share a key / value head: nothing is left to add up afterwards,
  // which saves a launch
  const int HG = a->heads / a->kv_heads;
  const bool own = !a->index && a->Bc == a->B;
  f.heads = own && hdp <= 32 && f.kt == 1 && HG > 1 && (long)HG * ((a->Nq + 31) / 32) <= 32;
  if (f.heads) f.nqb = 1;
  f.direct = own && f.nqb == 1 && (f.heads || HG == 1);
  f.ws = f.direct ? 0 : pairs * f.nqb * 2 * a->Nk * a->hd * 4;
  return f.ws <= (1L << 29);
}

int few_launch(const CrossParams& p, const FewPlan& f, int dtype, hipStream_t st) {
  const int hdp = cross_hdp(p.hd);
  if (dtype == 0) {
    switch (hdp) {
      case 16: return pick<bf16, 16>(p, f, st);
      case 32: return pick<bf16, 32>(p, f, st);
      case 64: return pick<bf16, 64>(p, f, st);
      case 96: return pick<bf16, 96>(p, f, st);
      default: return pick<bf16, 128>(p, f, st);
    }
  }
  switch (hdp) {
    case 16: return pick<float, 16>(p, f, st);
    case 32: return pick<float, 32>(p, f, st);
    default: return pick<float, 64>(p, f, st);
  }
}

}  // namespace dm_cross
