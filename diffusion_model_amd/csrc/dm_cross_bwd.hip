// Attention to an encoder's states of another length, backward (include/dm_hip.h: dm_cross_bwd).
//
//   P = exp2(c S - lse log2(e)),  dP = dO V^T,  dS = P (dP - delta),  delta = sum_d dO * O,
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K.
// dQ runs with the queries on the lanes (as the forward), dK / dV with the keys on the lanes; each probability tile is then
// already the operand of the product that reduces over its rows.  S and dP are computed in both kernels, seven products in all:
// one kernel for both sides would have to add dQ up over its key blocks in memory, 4 bytes per channel and block. The pipes
// (vector, matrix, LDS) are 40, 25 and 26 % busy in dQ, 33, 31 and 35 % in dK / dV at two waves per SIMD; more waves, or two
// query tiles at a time, were not faster.  delta reads O as the forward rounded it.  bf16, 16 x 1024 queries, 8 heads of 64 on
// 333 states (2 key / value heads, a tenth masked): dQ 36 us, dK and dV 41 us; fp32, 8 key / value heads: 477 us together (82
// TFLOP/s).
#include "dm_cross.h"

namespace {

using namespace dm_cross;

// ---------------------------------------------------------------- dQ (and delta)
// as the forward: resident keys, or two images of 64 keys in turn
template <typename T, int HDP> constexpr int image_bytes() { return 64 * (2 * Geo<T, HDP>::SR + 4) + 16; }

template <typename T, int HDP, bool RES, bool SPLIT, bool DROP>
__global__ __launch_bounds__(256, (HDP * (int)sizeof(T) < 384 ? 2 : 1)) void cross_dq_kernel(const CrossParams p) {
  typedef Geo<T, HDP> Gm;
  typedef typename Cr<T>::frag frag;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* sK = smem;
  char* sV = sK + p.kb * Gm::SR;
  float* bias = reinterpret_cast<float*>(sV + p.kb * Gm::SR);
  uint32_t* bits = reinterpret_cast<uint32_t*>(bias + p.kb);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  uint32_t id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int h = id % p.H;
  id /= p.H;
  const int qb = id % p.nqb;
  id /= p.nqb;
  const int split = id % p.qsplit, b = id / p.qsplit;
  const int ctx = context_of(p, b);
  const int k0 = split * p.qksplit, kn = min(keys_of(p, ctx), k0 + p.qksplit);
  const int hdb = p.hd * (int)sizeof(T), g = h / (p.H / p.G);
  const long krow = (long)(ctx < 0 ? 0 : ctx) * p.Nk;
  const char* kbase = p.k + krow * p.ldk + g * hdb;
  const char* vbase = p.v + krow * p.ldv + g * hdb;
  const unsigned char* mask = p.mask ? p.mask + krow : nullptr;
  const float c = p.scale * CR_LOG2E;
  const uint32_t seed = DROP ? dm_eff_seed(p.seed, p.seed_ctr) : 0u;
  frag qf[Gm::NC], df[Gm::NC];
  f32x16 acc[Gm::DT];
  float L2 = 0.f, delta = 0.f;
  uint32_t rs = 0;
  auto begin = [&](int q0) {                   // q0: the wave's first query
    const int q = q0 + (lane & 31), left = p.Nq - q0;
    const bool ok = q < p.Nq;
    const long tok = (long)b * p.Nq + q0, row = ((long)b * p.H + h) * p.Nq + q;
    load_frags<T, HDP>(rows_of(p.q + tok * p.ldq + h * hdb, p.ldq, left, hdb, lane), hdb, lane, qf);
    load_frags<T, HDP>(rows_of(p.d_o + tok * p.lddo + h * hdb, p.lddo, left, hdb, lane), hdb, lane, df);
    frag of[Gm::NC];
    load_frags<T, HDP>(rows_of(p.o + tok * p.ldo + h * hdb, p.ldo, left, hdb, lane), hdb, lane, of);
    float s = 0.f;
#pragma unroll
    for (int kc = 0; kc < Gm::NC; ++kc)
#pragma unroll
      for (int j = 0; j < (int)(16 / sizeof(T)); ++j) s += (float)df[kc][j] * (float)of[kc][j];
    delta = half_sum(s);
    L2 = ok ? p.lse[row] * CR_LOG2E : INFINITY;
    if (L2 == -INFINITY) L2 = INFINITY;        // no probability without a finite score, nor past the last query
    if (ok && half == 0 && split == 0) p.delta[row] = delta;
    if (DROP) rs = dm_drop_row(seed, (uint32_t)row);
#pragma unroll
    for (int d = 0; d < Gm::DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  };
  auto stage = [&](int from, int n) {
    stage_rows2<T, HDP>(sK, Gm::SR, kbase, p.ldk, sV, Gm::SR, vbase, p.ldv, from, n, kn, mask, hdb, tid);
    stage_valid(bits, bias, from, n, kn, mask, tid);
  };
  auto sweep = [&](int from, int tiles, int first, int step) {
    for (int t = first; t < tiles; t += step) {
      const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane((int)bits[t]);
      if (w == 0) continue;
      f32x16 s = score_init(bias + t * 32, half), dp = zero16();      // (masked keys: exp2(-inf) = 0)
#pragma unroll
      for (int kc = 0; kc < Gm::NC; ++kc) {
        s = Cr<T>::mma(row_frag<T>(sK + t * 32 * Gm::SR, Gm::SR, kc, lane), qf[kc], s);
        dp = Cr<T>::mma(row_frag<T>(sV + t * 32 * Gm::SR, Gm::SR, kc, lane), df[kc], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -L2));
      if (DROP) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const uint32_t key = from + t * 32 + tile_row(i, half), z = dm_drop_bits(rs, key >> 1);
          dp[i] = dm_keep16(z, 0, p.thresh) ? dp[i] * p.inv_keep : 0.f;
          dp[i + 1] = dm_keep16(z, 1, p.thresh) ? dp[i + 1] * p.inv_keep : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] *= dp[i] - delta;
#pragma unroll
      for (int f = 0; f < Cr<T>::NF; ++f) {
        const frag sf = Cr<T>::pack(s, f);
#pragma unroll
        for (int d = 0; d < Gm::DT; ++d)
          acc[d] = Cr<T>::mma(tr_frag<T, HDP>(sK + t * 32 * Gm::SR, Gm::SR, f, d, lane), sf, acc[d]);
      }
    }
  };
  auto finish = [&](int q) {
    if (p.qsplit > 1) {
      const long row = (((long)split * p.B + b) * p.H + h) * p.Nq + q;
      const Rows dst = rows_of((char*)(p.qpart + row * p.hd), p.hd * 4, p.Nq - q, p.hd * 4, lane);
#pragma unroll
      for (int d = 0; d < Gm::DT; ++d) store_tile<float>(dst, acc[d], 1.f, d * 32, p.hd * 4, lane);
      return;
    }
    const Rows dst = rows_of(p.dq + ((long)b * p.Nq + q) * p.lddq + h * hdb, p.lddq, p.Nq - q, hdb, lane);
#pragma unroll
    for (int d = 0; d < Gm::DT; ++d) store_tile<T>(dst, acc[d], p.scale, d * 32, hdb, lane);
  };
  if (SPLIT) {
    // one or two query tiles: the waves that share a tile take its keys' tiles in turn, and their sums are added in order
    const int WK = p.wk, n = max(0, (kn - k0 + 31) & ~31);
    begin(wave / WK * 32);
    stage(k0, n);
    __syncthreads();
    sweep(k0, n >> 5, wave % WK, WK);
    __syncthreads();
    constexpr int RS = HDP + 4;
    float* sum = reinterpret_cast<float*>(smem);
    put_rows<HDP>(sum + wave * 32 * RS, acc, lane);
    __syncthreads();
    const int per = p.hd >> 2;
    for (int i = tid; i < min(p.Nq, 128 / WK) * per; i += 256) {
      const int q = i / per, col = (i - q * per) * 4;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < WK; ++k) x += *reinterpret_cast<const f32x4*>(sum + (((q >> 5) * WK + k) * 32 + (q & 31)) * RS + col);
      if (p.qsplit > 1)
        *reinterpret_cast<f32x4*>(p.qpart + ((((long)split * p.B + b) * p.H + h) * p.Nq + q) * p.hd + col) = x;
      else
        store4<T>(p.dq + ((long)b * p.Nq + q) * p.lddq + h * hdb + col * (int)sizeof(T), x[0] * p.scale, x[1] * p.scale, x[2] * p.scale, x[3] * p.scale);
    }
    return;
  }
  const int q0 = qb * p.iters * 128 + wave * 32;
  if (RES) {
    const int n = max(0, (kn - k0 + 31) & ~31);
    stage(k0, n);
    __syncthreads();
    for (int it = 0; it < p.iters; ++it) {
      const int q = q0 + it * 128;
      if (q >= p.Nq) break;
      begin(q);
      sweep(k0, n >> 5, 0, 1);
      finish(q);
    }
  } else {
    Stager<T, HDP, 64> next;
    bool in = false;
    unsigned char byte = 1;
    auto load = [&](int from) {
      next.load(kbase, p.ldk, vbase, p.ldv, from, kn, mask, hdb, tid);
      in = load_valid(from, kn, mask, tid, byte);
    };
    auto store = [&]() {
      next.store(sK, Gm::SR, sV, Gm::SR, 64, mask != nullptr, tid);
      store_valid(bits, bias, in, byte, tid);
    };
    char* const image = smem;
    auto use = [&](int i) {
      sK = image + (i & 1) * image_bytes<T, HDP>();
      sV = sK + 64 * Gm::SR;
      bias = reinterpret_cast<float*>(sV + 64 * Gm::SR);
      bits = reinterpret_cast<uint32_t*>(bias + 64);
    };
    if (k0 < kn) load(k0);
    begin(q0);
    use(0);
    if (k0 < kn) store();
    __syncthreads();
    for (int from = k0, i = 0; from < kn; from += 64, ++i) {
      const bool more = from + 64 < kn;
      if (more) load(from + 64);
      use(i);
      sweep(from, 2, 0, 1);
      use(i + 1);
      if (more) store();
      __syncthreads();
    }
    finish(q0);
  }
}

// ---------------------------------------------------------------- dK, dV
// A workgroup owns 128 keys (32 per wave, on the lanes) of one (context, key / value head) and walks a share of the
// context's query list: every sample that uses the context, every query head of the group, 64 queries at a time.  The
// blocks of that list go to the p.nsplit shares in turn, each share leaves one fp32 partial, and cross_sum_kernel adds
// them in order: no atomics, the same inputs give the same bits.
constexpr int QS = 64;

// one image: 64 queries, their output gradients, and per query the log-sum-exp (base 2), delta and the dropout word
template <typename T, int HDP> constexpr int list_bytes() { return QS * (2 * Geo<T, HDP>::SR + 12); }

// walks the share's blocks of 64 queries
struct QueryList : Samples {
  uint32_t u, per;            // block of the present sample; blocks per sample
  __device__ __forceinline__ void settle(const CrossParams& p, int lane) {
    while (!done && u >= per) {
      u -= per;
      sample(p, lane);
    }
  }
  __device__ __forceinline__ void start(const CrossParams& p, int c, uint32_t blocks, int share, int lane) {
    per = blocks; u = (uint32_t)share;
    first(p, c, lane);
    settle(p, lane);
  }
  __device__ __forceinline__ void next(const CrossParams& p, int lane) {
    u += p.nsplit;
    settle(p, lane);
  }
};

template <typename T, int HDP, bool DROP>
__global__ __launch_bounds__(256, HDP * (int)sizeof(T) < 192 ? 2 : 1) void cross_dkv_kernel(const CrossParams p) {
  typedef Geo<T, HDP> Gm;
  typedef typename Cr<T>::frag frag;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  const int nkb = (p.Nk + 127) / 128;
  uint32_t id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int g = id % p.G;
  id /= p.G;
  const int kblk = id % nkb;
  id /= nkb;
  const int split = id % p.nsplit, ctx = id / p.nsplit;
  const int kn = keys_of(p, ctx), hdb = p.hd * (int)sizeof(T), HG = p.H / p.G;
  const int key = kblk * 128 + wave * 32 + (lane & 31);
  const long krow = (long)ctx * p.Nk + key;
  const bool valid = key < kn && (!p.mask || p.mask[krow]);
  const bool active = __any(valid);
  const float c = p.scale * CR_LOG2E;
  const uint32_t seed = DROP ? dm_eff_seed(p.seed, p.seed_ctr) : 0u;
  frag kf[Gm::NC], vf[Gm::NC];
  load_frags<T, HDP>(p.k + krow * p.ldk + g * hdb, valid, hdb, lane, kf);
  load_frags<T, HDP>(p.v + krow * p.ldv + g * hdb, valid, hdb, lane, vf);
  f32x16 dk[Gm::DT], dv[Gm::DT];
#pragma unroll
  for (int d = 0; d < Gm::DT; ++d) { dk[d] = zero16(); dv[d] = zero16(); }

  const int nqc = (p.Nq + QS - 1) / QS;
  Stager<T, HDP, QS> next;
  float nl = 0.f, nd = 0.f;
  uint32_t nrow = 0;
  auto load = [&](const QueryList& at) {
    const int h = g * HG + (int)(at.u / (uint32_t)nqc), r0 = (int)(at.u % (uint32_t)nqc) * QS;
    const long tok = (long)at.b * p.Nq, row = ((long)at.b * p.H + h) * p.Nq;
    next.load(p.q + tok * p.ldq + h * hdb, p.ldq, p.d_o + tok * p.lddo + h * hdb, p.lddo, r0, p.Nq, nullptr, hdb, tid);
    if (tid < QS) {
      const int q = min(r0 + tid, p.Nq - 1);
      const float l = p.lse[row + q] * CR_LOG2E;
      nl = r0 + tid >= p.Nq || l == -INFINITY ? INFINITY : l;      // no probability for queries past the end
      nd = r0 + tid < p.Nq ? p.delta[row + q] : 0.f;
      nrow = (uint32_t)(row + q);
    }
  };
  char *sQ, *sD;
  float *sL, *sDelta;
  uint32_t* sRow;
  auto use = [&](int i) {
    sQ = smem + (i & 1) * list_bytes<T, HDP>();
    sD = sQ + QS * Gm::SR;
    sL = reinterpret_cast<float*>(sD + QS * Gm::SR);
    sDelta = sL + QS;
    sRow = reinterpret_cast<uint32_t*>(sDelta + QS);
  };
  auto store = [&]() {
    next.store(sQ, Gm::SR, sD, Gm::SR, QS, false, tid);
    if (tid < QS) {
      sL[tid] = nl;
      sDelta[tid] = nd;
      if (DROP) sRow[tid] = dm_drop_row(seed, nrow);
    }
  };
  auto block = [&](int rows) {
    if (!active) return;
    for (int t = 0; t < QS / 32; ++t) {
      if (t * 32 >= rows) break;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int kc = 0; kc < Gm::NC; ++kc) {
        s = Cr<T>::mma(row_frag<T>(sQ + t * 32 * Gm::SR, Gm::SR, kc, lane), kf[kc], s);
        dp = Cr<T>::mma(row_frag<T>(sD + t * 32 * Gm::SR, Gm::SR, kc, lane), vf[kc], dp);
      }
      f32x16 pd;      // what multiplies dO: the probability, dropped
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(sL + t * 32 + 8 * i + 4 * half);
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(sDelta + t * 32 + 8 * i + 4 * half);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i + r], c, -l4[r]));
          float z = 1.f;
          if (DROP) z = dm_keep16(dm_drop_bits(sRow[t * 32 + 8 * i + 4 * half + r], (uint32_t)key >> 1), (uint32_t)key, p.thresh) ? p.inv_keep : 0.f;
          pd[4 * i + r] = DROP ? pr * z : pr;
          s[4 * i + r] = pr * ((DROP ? dp[4 * i + r] * z : dp[4 * i + r]) - d4[r]);
        }
      }
#pragma unroll
      for (int f = 0; f < Cr<T>::NF; ++f) {
        const frag pf = Cr<T>::pack(pd, f), sf = Cr<T>::pack(s, f);
#pragma unroll
        for (int d = 0; d < Gm::DT; ++d) {
          dv[d] = Cr<T>::mma(tr_frag<T, HDP>(sD + t * 32 * Gm::SR, Gm::SR, f, d, lane), pf, dv[d]);
          dk[d] = Cr<T>::mma(tr_frag<T, HDP>(sQ + t * 32 * Gm::SR, Gm::SR, f, d, lane), sf, dk[d]);
        }
      }
    }
  };
  if (kblk * 128 < kn) {
    QueryList at;
    at.start(p, ctx, (uint32_t)HG * nqc, split, lane);
    if (!at.done) {
      load(at);
      use(0);
      store();
    }
    __syncthreads();
    for (int i = 0; !at.done; ++i) {
      const int rows = p.Nq - (int)(at.u % (uint32_t)nqc) * QS;
      at.next(p, lane);
      if (!at.done) load(at);          // the next block's rows fly while this one is used
      use(i);
      block(rows);
      use(i + 1);
      if (!at.done) store();
      __syncthreads();
    }
  }
  if (key >= p.Nk) return;
  const float osc = valid ? p.scale : 0.f;
  if (p.nsplit > 1) {
    const long n = (long)p.Bc * p.Nk * p.G * p.hd;
    float* dst = p.part + (long)split * 2 * n + (krow * p.G + g) * p.hd;
#pragma unroll
    for (int d = 0; d < Gm::DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = d * 32 + 8 * i + 4 * half;
        if (col < p.hd) {
          *reinterpret_cast<f32x4*>(dst + col) = valid ? f32x4{dk[d][4 * i], dk[d][4 * i + 1], dk[d][4 * i + 2], dk[d][4 * i + 3]} : f32x4{0.f, 0.f, 0.f, 0.f};
          *reinterpret_cast<f32x4*>(dst + n + col) = valid ? f32x4{dv[d][4 * i], dv[d][4 * i + 1], dv[d][4 * i + 2], dv[d][4 * i + 3]} : f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
    return;
  }
  char* ok = p.dk + krow * p.lddk + g * hdb;
  char* ov = p.dv + krow * p.lddv + g * hdb;
#pragma unroll
  for (int d = 0; d < Gm::DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = d * 32 + 8 * i + 4 * half;
      if (col >= p.hd) continue;
      if (valid) {
        store4<T>(ok + col * sizeof(T), dk[d][4 * i] * osc, dk[d][4 * i + 1] * osc, dk[d][4 * i + 2] * osc, dk[d][4 * i + 3] * osc);
        store4<T>(ov + col * sizeof(T), dv[d][4 * i], dv[d][4 * i + 1], dv[d][4 * i + 2], dv[d][4 * i + 3]);
      } else {
        store4<T>(ok + col * sizeof(T), 0.f, 0.f, 0.f, 0.f);
        store4<T>(ov + col * sizeof(T), 0.f, 0.f, 0.f, 0.f);
      }
    }
}

// Adds the shares of dK / dV: SL lanes split the list of one result (4 channels of one key) and join by a fixed tree, 8 for
// long lists, 1 for short ones.
template <typename T, int SL>
__global__ __launch_bounds__(256) void cross_sum_kernel(const CrossParams p) {
  constexpr int RPW = 64 / SL;
  const int lane = threadIdx.x & 63, slice = lane / RPW;
  const long n = (long)p.Bc * p.Nk * p.G * p.hd;
  const long r = (((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * RPW + lane % RPW) * 4, i = r < 2 * n ? r : 0;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = slice; k < p.nsplit; k += SL) s += *reinterpret_cast<const f32x4*>(p.part + (long)k * 2 * n + i);
  if (SL > 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int o = RPW; o < 64; o <<= 1) s[j] += __shfl_xor(s[j], o, 64);
  }
  if (r >= 2 * n || slice) return;
  const bool is_v = i >= n;
  const long e = is_v ? i - n : i, w = (long)p.G * p.hd, row = e / w, col = e - row * w;
  const float f = is_v ? 1.f : p.scale;
  store4<T>((is_v ? p.dv + row * p.lddv : p.dk + row * p.lddk) + col * (long)sizeof(T), s[0] * f, s[1] * f, s[2] * f, s[3] * f);
}

constexpr int LDS_IMAGE = 80 * 1024;

struct BwdPlan { int kb, iters, nqb, wk, qsplit, qksplit, nsplit; bool res; long delta_bytes, part_bytes, ws; };
int row_bytes(const dm_cross_args* a) { return cross_hdp(a->hd) * (a->dtype == 0 ? 2 : 4) + 16; }
BwdPlan bwd_plan(const dm_cross_args* a) {
  BwdPlan f{};
  const int image = (LDS_IMAGE - 64) / (2 * row_bytes(a) + 5) / 64 * 64;
  f.wk = cross_wk(a);
  const long groups = ((long)a->Nq + 127) / 128, blocks = cross_groups(a) * a->B * a->heads;
  // dQ with few rows: the keys are split as in the forward (B=1, 3 heads of 40, 40 queries on 1031 states, fp32, backward: 28
  // us, 128 without)
  const long qs = cross_splits(a, blocks, image, a->hd * 4L);
  f.qksplit = qs > 1 ? (int)((((long)a->Nk + qs - 1) / qs + 63) & ~63L) : a->Nk;
  f.qsplit = qs > 1 ? (a->Nk + f.qksplit - 1) / f.qksplit : 1;
  const int need = (f.qksplit + 63) & ~63;
  f.res = need <= image;
  if (!f.res) f.wk = 1;
  f.kb = need > 0 ? need : 64;
  f.iters = 1;
  if (f.res && f.wk == 1) {
    long it = blocks * f.qsplit / 512;
    if (it > 8) it = 8;
    if (it > groups) it = groups;
    f.iters = it < 1 ? 1 : (int)it;
  }
  f.nqb = f.wk > 1 ? 1 : (int)((groups + f.iters - 1) / f.iters);
  f.iters = f.wk > 1 ? 1 : (int)((groups + f.nqb - 1) / f.nqb);
  f.delta_bytes = (((long)a->B * a->heads * a->Nq + 3) & ~3L) * 4;
  // shares of a context's query list: two workgroups per CU, at least two blocks of queries each, partials of at most 256 MiB
  const long used = cross_used(a), owners = used * a->kv_heads * ((a->Nk + 127) / 128);
  const long list = (a->B + used - 1) / used * (a->heads / a->kv_heads) * ((a->Nq + QS - 1) / QS);
  long ns = owners > 0 ? 512 / owners : 1;
  if (ns > list / 2) ns = list / 2;
  const double part = 8.0 * a->Bc * a->Nk * a->kv_heads * a->hd;
  if (ns * part > (double)(1L << 28)) ns = (long)((double)(1L << 28) / part);
  f.nsplit = ns < 1 ? 1 : (int)ns;
  f.part_bytes = f.nsplit > 1 ? (long)f.nsplit * 2 * a->Bc * a->Nk * a->kv_heads * a->hd * 4 : 0;
  f.ws = f.delta_bytes + f.part_bytes + (f.qsplit > 1 ? (long)f.qsplit * a->B * a->heads * a->Nq * a->hd * 4 : 0);
  return f;
}

template <typename T, int HDP, bool RES, bool SPLIT, bool DROP>
int launch_dq(const CrossParams& p, hipStream_t st) {
  auto kern = cross_dq_kernel<T, HDP, RES, SPLIT, DROP>;
  const long blocks = (long)p.B * p.qsplit * p.nqb * p.H;
  if (blocks > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
  static unsigned long long attr_devs = 0ull;
  if (dm_first_on_device(attr_devs) &&
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                          RES ? LDS_IMAGE : 2 * image_bytes<T, HDP>()) != hipSuccess)
    return DM_ERR_LAUNCH;
  size_t lds = RES ? (size_t)p.kb * (2 * Geo<T, HDP>::SR + 4) + (p.kb / 32 + 2) * 4 : 2 * image_bytes<T, HDP>();
  if (SPLIT && lds < 4 * 32 * (HDP + 4) * 4) lds = 4 * 32 * (HDP + 4) * 4;
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), lds, st, p);
  DM_LAUNCH_CHECK();
  return p.qsplit > 1 ? dqsum_launch(p, sizeof(T) == 2 ? 0 : 1, st) : DM_OK;
}
template <typename T, int HDP, bool DROP>
int launch_dkv(const CrossParams& p, hipStream_t st) {
  auto kern = cross_dkv_kernel<T, HDP, DROP>;
  const int lds = 2 * list_bytes<T, HDP>();
  const long blocks = (long)p.Bc * p.nsplit * ((p.Nk + 127) / 128) * p.G;
  if (blocks == 0) return DM_OK;
  if (blocks > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
  static unsigned long long attr_devs = 0ull;
  if (dm_first_on_device(attr_devs) &&
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
    return DM_ERR_LAUNCH;
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), lds, st, p);
  DM_LAUNCH_CHECK();
  if (p.nsplit > 1) {
    const long n = (long)2 * p.Bc * p.Nk * p.G * (p.hd >> 2);
    const bool wide = p.nsplit > 8;
    const long jb = (n + (wide ? 31 : 255)) / (wide ? 32 : 256);
    if (jb > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
    if (wide) hipLaunchKernelGGL((cross_sum_kernel<T, 8>), dim3((unsigned)jb), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((cross_sum_kernel<T, 1>), dim3((unsigned)jb), dim3(256), 0, st, p);
    DM_LAUNCH_CHECK();
  }
  return DM_OK;
}
template <typename T, int HDP, bool DROP> int run_bwd(const CrossParams& p, bool res, hipStream_t st) {
  const int rc = !res ? launch_dq<T, HDP, false, false, DROP>(p, st)
                      : (p.wk > 1 ? launch_dq<T, HDP, true, true, DROP>(p, st) : launch_dq<T, HDP, true, false, DROP>(p, st));
  if (rc != DM_OK) return rc;
  static const DmVariantName nm("cross_bwd<%s,%d>", sizeof(T) == 2 ? "bf16" : "fp32", HDP);
  dm_set_variant(nm.s);
  return launch_dkv<T, HDP, DROP>(p, st);
}
template <typename T, int HDP> int pick_bwd(const CrossParams& p, bool res, hipStream_t st) {
  return p.thresh ? run_bwd<T, HDP, true>(p, res, st) : run_bwd<T, HDP, false>(p, res, st);
}
template <typename T> int pick_width(const CrossParams& p, bool res, hipStream_t st) {
  switch (cross_hdp(p.hd)) {
    case 16: return pick_bwd<T, 16>(p, res, st);
    case 32: return pick_bwd<T, 32>(p, res, st);
    case 64: return pick_bwd<T, 64>(p, res, st);
    case 96: return pick_bwd<T, 96>(p, res, st);
    default: return pick_bwd<T, 128>(p, res, st);
  }
}

}  // namespace

extern "C" long dm_cross_bwd_workspace_bytes(const dm_cross_args* a) {
  if (!dm_cross::cross_sizes_ok(a)) return 0;
  dm_cross::FewPlan few;
  dm_cross::OneBwdPlan one;
  if (dm_cross::onebwd_plan(a, one)) return one.ws;
  if (dm_cross::few_plan(a, few)) return few.ws;
  return dm_cross::rowsbwd_plan(a, one) ? one.ws : bwd_plan(a).ws;
}

extern "C" int dm_cross_bwd(const dm_cross_args* a, dm_stream_t stream) {
  CrossParams p{};
  const int rc = cross_fill(p, a, true);
  if (rc != DM_OK) return rc;
  OneBwdPlan one;
  if (onebwd_plan(a, one)) {
    DM_REQUIRE(one.ws == 0 || (a->workspace && a->ws_bytes >= one.ws && (uintptr_t)a->workspace % 16 == 0));
    p.qsplit = one.tiles; p.nsplit = one.ws ? 1 : 0;
    p.qpart = (float*)a->workspace;
    return onebwd_launch(p, a->dtype, (hipStream_t)stream);
  }
  FewPlan few;
  if (few_plan(a, few)) {
    DM_REQUIRE(few.ws == 0 || (a->workspace && a->ws_bytes >= few.ws && (uintptr_t)a->workspace % 16 == 0));
    p.iters = few.iters; p.nqb = few.nqb; p.nsplit = few.direct ? 0 : 1;
    p.part = (float*)a->workspace;
    return few_launch(p, few, a->dtype, (hipStream_t)stream);
  }
  if (rowsbwd_plan(a, one)) {
    DM_REQUIRE(one.ws == 0 || (a->workspace && a->ws_bytes >= one.ws && (uintptr_t)a->workspace % 16 == 0));
    p.qsplit = one.tiles; p.nsplit = one.ws ? 1 : 0;
    p.qpart = (float*)a->workspace;
    return rowsbwd_launch(p, a->dtype, (hipStream_t)stream);
  }
  const BwdPlan f = bwd_plan(a);
  DM_REQUIRE(a->workspace && a->ws_bytes >= f.ws && (uintptr_t)a->workspace % 16 == 0);
  p.kb = f.kb; p.iters = f.iters; p.nqb = f.nqb; p.nsplit = f.nsplit; p.wk = f.wk; p.qsplit = f.qsplit; p.qksplit = f.qksplit;
  p.delta = (float*)a->workspace;
  p.part = (float*)((char*)a->workspace + f.delta_bytes);
  p.qpart = (float*)((char*)a->workspace + f.delta_bytes + f.part_bytes);
  return a->dtype == 0 ? pick_width<bf16>(p, f.res, (hipStream_t)stream) : pick_width<float>(p, f.res, (hipStream_t)stream);
}
