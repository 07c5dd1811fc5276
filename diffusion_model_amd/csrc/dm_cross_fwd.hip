// Attention to an encoder's states of another length, forward (include/dm_hip.h: dm_cross_fwd).
//
//   S^T = K Q^T (keys on the rows of the tile, queries on the lanes), P = exp2(c S - c m), c = scale log2(e), m the running
//   maximum of the lane's query;  O^T += V^T P^T;  l += sum P;  o = O / l, lse = scale m + ln l.
// The row sum takes the fp32 probabilities before they are rounded for the second product, so lse is an fp32 value.
//
// Narrow heads are bound by the vector work per score (an exponential, a maximum, two adds and half a conversion against 64
// matrix flops; vector units 67 % busy at 16-wide heads), which is why masks cost none of it and empty half tiles are left out;
// wide ones by the chain of scores, softmax and products of the one tile that a wave has (vector units 40 % busy, matrix units
// 32, LDS 28 at 128-wide heads).  bf16, ragged lengths: 64 x 2304 queries, 8 heads of 16, 77 tokens 27 us; 64 x 576, 8 heads of
// 32, 77 tokens 12.5 us (3.3 TB/s); 16 x 1024, 8 heads of 128, 512 states 49 us (700 TFLOP/s).  fp32: 16 x 1024, 8 heads of 64,
// 333 states 118 us (95 TFLOP/s).
#include "dm_cross.h"

namespace {

using namespace dm_cross;

template <typename T, int HDP> struct FwdState {
  f32x16 acc[Geo<T, HDP>::DT];
  float m, l;
};

// NT tiles of 32 keys (LDS rows t0..) against the wave's 32 queries.  FIRST: the state is not read but begun, with the
// maximum of these tiles, so nothing is cleared or rescaled (up to 96 keys need no other step).
// HALF: the last tile has at most 16 keys, which are the lower halves of the registers; the upper ones are left out.
template <typename T, int HDP, int NT, bool FIRST, bool HALF, bool DROP>
__device__ __forceinline__ void fwd_step(const CrossParams& p, FwdState<T, HDP>& st, const char* sK, const char* sV,
                                         const uint32_t* bits, const float* bias, int t0, int key0, float c,
                                         const typename Cr<T>::frag (&qf)[Geo<T, HDP>::NC], uint32_t rs, int lane) {
  typedef Geo<T, HDP> Gm;
  const int half = lane >> 5;
  if (!FIRST) {
    uint32_t any = bits[t0];
    if (NT > 1) any |= bits[t0 + 1];
    if (__builtin_amdgcn_readfirstlane((int)any) == 0) return;
  }
  f32x16 s[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    s[t] = score_init(bias + (t0 + t) * 32, half);
#pragma unroll
    for (int kc = 0; kc < Gm::NC; ++kc)
      s[t] = Cr<T>::mma(row_frag<T>(sK + (t0 + t) * 32 * Gm::SR, Gm::SR, kc, lane), qf[kc], s[t]);
  }
  float mx = s[0][0];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < (HALF && t == NT - 1 ? 8 : 16); ++i) mx = fmaxf(mx, s[t][i]);
  mx = half_max(mx);
  if (FIRST) {
    st.m = mx;
    st.l = 0.f;
  } else {
    // the reference maximum moves only when a block exceeds it by more than 2^8 in the probability: exact all the same
    // (numerator and denominator share it), and the common block rescales nothing
    const bool up = (mx - st.m) * c > 8.f;
    if (__any(up)) {
      const float alpha = up ? __builtin_amdgcn_exp2f((st.m - mx) * c) : 1.f;
      st.m = up ? mx : st.m;
      st.l *= alpha;
#pragma unroll
      for (int d = 0; d < Gm::DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.acc[d][i] *= alpha;
    }
  }
  const float mc = st.m == -INFINITY ? 0.f : st.m * c;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int i = 0; i < (HALF && t == NT - 1 ? 8 : 16); ++i) {
      s[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], c, -mc));
      st.l += s[t][i];
    }
    if (DROP) {
#pragma unroll
      for (int i = 0; i < (HALF && t == NT - 1 ? 8 : 16); i += 2) {
        const uint32_t key = key0 + t * 32 + tile_row(i, half), z = dm_drop_bits(rs, key >> 1);
        if (!dm_keep16(z, 0, p.thresh)) s[t][i] = 0.f;
        if (!dm_keep16(z, 1, p.thresh)) s[t][i + 1] = 0.f;
      }
    }
#pragma unroll
    for (int f = 0; f < (HALF && t == NT - 1 ? Cr<T>::NF / 2 : Cr<T>::NF); ++f) {
      const typename Cr<T>::frag pf = Cr<T>::pack(s[t], f);
#pragma unroll
      for (int d = 0; d < Gm::DT; ++d)
        st.acc[d] = Cr<T>::mma(tr_frag<T, HDP>(sV + (t0 + t) * 32 * Gm::ST, Gm::ST, f, d, lane), pf,
                               FIRST && t == 0 && f == 0 ? zero16() : st.acc[d]);
    }
  }
}

template <typename T, int HDP>
__device__ __forceinline__ void fwd_finish(const CrossParams& p, const FwdState<T, HDP>& st, int b, int h, int q0, int split,
                                           float c, int lane) {      // q0: the wave's first query (uniform)
  typedef Geo<T, HDP> Gm;
  const int q = q0 + (lane & 31);
  const float l = half_sum(st.l);
  const float mc = st.m == -INFINITY ? 0.f : st.m * c;
  const bool mine = q < p.Nq && lane < 32;
  const long row = ((long)b * p.H + h) * p.Nq + q0;
  if (p.nsplit > 1) {
    const long rows = (long)p.B * p.H * p.Nq;
    const Rows o = rows_of((char*)(p.part + (split * rows + row) * p.hd), p.hd * 4, p.Nq - q0, p.hd * 4, lane);
#pragma unroll
    for (int d = 0; d < Gm::DT; ++d) store_tile<float>(o, st.acc[d], 1.f, d * 32, p.hd * 4, lane);
    if (mine) {
      float* ml = p.part + p.nsplit * rows * p.hd + (split * rows + row + lane) * 2;
      ml[0] = mc;
      ml[1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : p.inv_keep * __builtin_amdgcn_rcpf(l);      // (v_rcp_f32: 1 ulp)
  const int hdb = p.hd * (int)sizeof(T);
  const Rows o = rows_of(p.o + ((long)b * p.Nq + q0) * p.ldo + h * hdb, p.ldo, p.Nq - q0, hdb, lane);
#pragma unroll
  for (int d = 0; d < Gm::DT; ++d) store_tile<T>(o, st.acc[d], inv, d * 32, hdb, lane);
  if (mine) p.lse[row + lane] = l == 0.f ? -INFINITY : (mc + __builtin_amdgcn_logf(l)) * CR_LN2;
}

// one image of the streamed kernel: 64 keys, values, starts and validity words
template <typename T, int HDP> constexpr int image_bytes() { return 64 * (Geo<T, HDP>::SR + Geo<T, HDP>::ST + 4) + 16; }

// A workgroup: 4 waves x p.iters tiles of 32 queries of one (sample, head, key split).  RES: the keys of the split fit one
// LDS image, which is staged once for all the tiles; otherwise two images of 64 keys take turns (iters is 1).
template <typename T, int HDP, bool RES, bool SPLIT, bool DROP>
__global__ __launch_bounds__(256, (HDP * (int)sizeof(T) <= 64 ? 4 : (HDP * (int)sizeof(T) < 384 ? 2 : 1))) void cross_fwd_kernel(const CrossParams p) {
  typedef Geo<T, HDP> Gm;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* sK = smem;
  char* sV = sK + p.kb * Gm::SR;
  float* bias = reinterpret_cast<float*>(sV + p.kb * Gm::ST);
  uint32_t* bits = reinterpret_cast<uint32_t*>(bias + p.kb);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int h = id % p.H;
  id /= p.H;
  const int qb = id % p.nqb;
  id /= p.nqb;
  const int split = id % p.nsplit, b = id / p.nsplit;
  const int ctx = context_of(p, b), kn = keys_of(p, ctx);
  const int k0 = p.nsplit > 1 ? split * p.ksplit : 0;
  const int k1 = p.nsplit > 1 ? min(kn, k0 + p.ksplit) : kn;
  const int hdb = p.hd * (int)sizeof(T), g = h / (p.H / p.G);
  const long krow = (long)(ctx < 0 ? 0 : ctx) * p.Nk;
  const char* kbase = p.k + krow * p.ldk + g * hdb;
  const char* vbase = p.v + krow * p.ldv + g * hdb;
  const unsigned char* mask = p.mask ? p.mask + krow : nullptr;
  const float c = p.scale * CR_LOG2E;
  const uint32_t seed = DROP ? dm_eff_seed(p.seed, p.seed_ctr) : 0u;

  FwdState<T, HDP> st;
  typename Cr<T>::frag qf[Gm::NC], nf[Gm::NC];
  uint32_t rs = 0;
  constexpr bool AHEAD = Gm::NC <= 4;          // (wider rows would not fit the registers twice)
  auto fetch = [&](int q) {                    // q: the wave's first query
    load_frags<T, HDP>(rows_of(p.q + ((long)b * p.Nq + q) * p.ldq + h * hdb, p.ldq, p.Nq - q, hdb, lane), hdb, lane, nf);
  };
  auto begin = [&](int q) {
    if (!AHEAD && RES && !SPLIT) fetch(q);
#pragma unroll
    for (int kc = 0; kc < Gm::NC; ++kc) qf[kc] = nf[kc];
    if (DROP) rs = dm_drop_row(seed, (uint32_t)(((long)b * p.H + h) * p.Nq + q + (lane & 31)));
  };
  auto clear = [&]() {
    st.m = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int d = 0; d < Gm::DT; ++d) st.acc[d] = zero16();
  };
  auto stage = [&](int from, int n) {
    stage_rows2<T, HDP>(sK, Gm::SR, kbase, p.ldk, sV, Gm::ST, vbase, p.ldv, from, n, k1, mask, hdb, tid);
    stage_valid(bits, bias, from, n, k1, mask, tid);
  };
#define DM_STEP(NT, FIRST, t, from) DM_STEP_H(NT, FIRST, false, t, from)
#define DM_STEP_H(NT, FIRST, HALF, t, from) \
  fwd_step<T, HDP, NT, FIRST, HALF, DROP>(p, st, sK, sV, bits, bias, t, (from) + (t) * 32, c, qf, rs, lane)
  if (SPLIT) {
    // one or two query tiles: the waves that share a tile take its keys' tiles in turn and join through LDS
    const int WK = p.wk, wq = wave / WK, w = wave % WK, n = max(0, (k1 - k0 + 31) & ~31), tiles = n >> 5, q = wq * 32;
    fetch(q);
    stage(k0, n);
    __syncthreads();
    begin(q);
    clear();
    for (int t = w; t < tiles; t += WK) DM_STEP(1, false, t, k0);
    const float l = half_sum(st.l);
    __syncthreads();
    constexpr int RS = HDP + 4;
    float* o = reinterpret_cast<float*>(smem);
    float* ml = o + 4 * 32 * RS;             // [wave][query] {maximum (base 2), sum}
    put_rows<HDP>(o + wave * 32 * RS, st.acc, lane);
    if (lane < 32) {
      ml[(wave * 32 + lane) * 2] = st.m == -INFINITY ? -INFINITY : st.m * c;
      ml[(wave * 32 + lane) * 2 + 1] = l;
    }
    __syncthreads();
    const int per = p.hd >> 2;
    const long rows = (long)p.B * p.H * p.Nq;
    for (int i = tid; i < min(p.Nq, 128 / WK) * per; i += 256) {
      const int qq = i / per, col = (i - qq * per) * 4, base = (qq >> 5) * WK, r = qq & 31;
      float m = -INFINITY;
      for (int k = 0; k < WK; ++k) m = fmaxf(m, ml[((base + k) * 32 + r) * 2]);
      const float ref = m == -INFINITY ? 0.f : m;
      float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < WK; ++k) {
        const float f = __builtin_amdgcn_exp2f(ml[((base + k) * 32 + r) * 2] - ref);
        const f32x4 a = *reinterpret_cast<const f32x4*>(o + ((base + k) * 32 + r) * RS + col);
        sum += f * ml[((base + k) * 32 + r) * 2 + 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += f * a[j];
      }
      const long row = ((long)b * p.H + h) * p.Nq + qq;
      if (p.nsplit > 1) {
        *reinterpret_cast<f32x4*>(p.part + (split * rows + row) * p.hd + col) = f32x4{x[0], x[1], x[2], x[3]};
        if (col == 0) {
          float* at = p.part + p.nsplit * rows * p.hd + (split * rows + row) * 2;
          at[0] = ref;
          at[1] = sum;
        }
      } else {
        const float inv = sum == 0.f ? 0.f : p.inv_keep * __builtin_amdgcn_rcpf(sum);
        store4<T>(p.o + ((long)b * p.Nq + qq) * p.ldo + h * hdb + col * (int)sizeof(T), x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        if (col == 0) p.lse[row] = sum == 0.f ? -INFINITY : (ref + __builtin_amdgcn_logf(sum)) * CR_LN2;
      }
    }
    return;
  }
  const int q0 = qb * p.iters * 128 + wave * 32;
  if (AHEAD) fetch(q0);
  if (RES) {
    const int n = max(0, (k1 - k0 + 31) & ~31), tiles = n >> 5;
    const bool half = n - (k1 - k0) >= 16;
    stage(k0, n);
    __syncthreads();
    // the first step looks at no validity word, and a masked key's score is -infinity only under a finite query (its product
    // with the zeroed key is not zero under a NaN or an infinity): without any valid key there is no step
    bool some = !mask;
    if (mask)
      for (int t = 0; t < tiles; ++t) some = some || __builtin_amdgcn_readfirstlane((int)bits[t]) != 0;
    // one loop for each number of tiles, so that each keeps only its own LDS addresses in registers
    auto each = [&](auto step) {
      for (int it = 0; it < p.iters; ++it) {
        const int q = q0 + it * 128;
        if (q >= p.Nq) break;                    // (wave-uniform)
        begin(q);
        if (AHEAD && it + 1 < p.iters) fetch(q + 128);      // the next tile's queries fly while this one is computed
        step();
        fwd_finish<T, HDP>(p, st, b, h, q, split, c, lane);
      }
    };
    if (tiles == 0 || !some) each([&]() { clear(); });
    else if (tiles == 1 && half) each([&]() { DM_STEP_H(1, true, true, 0, k0); });
    else if (tiles == 1) each([&]() { DM_STEP(1, true, 0, k0); });
    else if (tiles == 2 && half) each([&]() { DM_STEP_H(2, true, true, 0, k0); });
    else if (tiles == 3 && half && HDP <= 64) each([&]() { DM_STEP_H(3, true, true, 0, k0); });
    else if (tiles == 3 && HDP <= 64) each([&]() { DM_STEP(3, true, 0, k0); });
    else each([&]() {
      int t = 2;
      DM_STEP(2, true, 0, k0);
      for (; t + 2 <= tiles; t += 2) DM_STEP(2, false, t, k0);
      if (t < tiles) DM_STEP(1, false, t, k0);
    });
  } else {
    // two images of 64 keys in turn: the next one's rows fly while the present one is used
    Stager<T, HDP, 64> next;
    bool in = false;
    unsigned char byte = 1;
    auto load = [&](int from) {
      next.load(kbase, p.ldk, vbase, p.ldv, from, k1, mask, hdb, tid);
      in = load_valid(from, k1, mask, tid, byte);
    };
    auto store = [&]() {
      next.store(sK, Gm::SR, sV, Gm::ST, 64, mask != nullptr, tid);
      store_valid(bits, bias, in, byte, tid);
    };
    char* const image = smem;
    auto use = [&](int i) {
      sK = image + (i & 1) * image_bytes<T, HDP>();
      sV = sK + 64 * Gm::SR;
      bias = reinterpret_cast<float*>(sV + 64 * Gm::ST);
      bits = reinterpret_cast<uint32_t*>(bias + 64);
    };
    if (k0 < k1) load(k0);
    if (!AHEAD) fetch(q0);
    begin(q0);
    clear();
    use(0);
    if (k0 < k1) store();
    __syncthreads();
    for (int from = k0, i = 0; from < k1; from += 64, ++i) {
      const bool more = from + 64 < k1;
      if (more) load(from + 64);
      use(i);
      DM_STEP(2, false, 0, from);
      use(i + 1);
      if (more) store();
      __syncthreads();
    }
    fwd_finish<T, HDP>(p, st, b, h, q0, split, c, lane);
  }
#undef DM_STEP
#undef DM_STEP_H
}

constexpr int LDS_IMAGE = 80 * 1024;     // two workgroups per CU

int key_bytes(const dm_cross_args* a) {
  const int hdp = cross_hdp(a->hd);
#define DM_KEYB(HDP) if (hdp == HDP) return a->dtype == 0 ? Geo<bf16, HDP>::SR + Geo<bf16, HDP>::ST : Geo<float, HDP>::SR + Geo<float, HDP>::ST
  DM_KEYB(16); DM_KEYB(32); DM_KEYB(64); DM_KEYB(96); DM_KEYB(128);
#undef DM_KEYB
  return 0;
}

struct FwdPlan { int nsplit, ksplit, kb, iters, nqb, wk; bool res; long ws; };
FwdPlan fwd_plan(const dm_cross_args* a) {
  FwdPlan f{};
  const int kbytes = key_bytes(a);
  const int image = (LDS_IMAGE - 64) / (kbytes + 5) / 64 * 64;     // keys per LDS image
  f.wk = cross_wk(a);
  const long groups = cross_groups(a);                        // workgroups along the queries at one tile per wave
  const long blocks = groups * a->B * a->heads;
  // fewer workgroups than CUs: the keys are split (at least 128 each) until there are two per CU (at 336 workgroups the join
  // cost more than the split gave)
  const long ns = cross_splits(a, blocks, image, (a->hd + 2) * 4L);
  f.ksplit = ns > 1 ? (int)((((long)a->Nk + ns - 1) / ns + 63) & ~63L) : a->Nk;
  f.nsplit = ns > 1 ? (a->Nk + f.ksplit - 1) / f.ksplit : 1;
  const int need = (f.ksplit + 63) & ~63;
  f.res = need <= image;
  if (!f.res) f.wk = 1;
  f.kb = need > 0 ? need : 64;
  // resident keys serve several query tiles per wave, as long as there are two workgroups per CU (B=64, 8 heads of 32, 576
  // queries, 77 tokens: 14.4 us at two, 16.7 at six)
  const long g1 = ((long)a->Nq + 127) / 128;
  f.iters = 1;
  if (f.res && f.wk == 1) {
    long it = blocks * f.nsplit / 512;
    if (it > 8) it = 8;
    if (it > g1) it = g1;
    f.iters = it < 1 ? 1 : (int)it;
  }
  f.nqb = f.wk > 1 ? 1 : (int)((g1 + f.iters - 1) / f.iters);
  f.iters = f.wk > 1 ? 1 : (int)((g1 + f.nqb - 1) / f.nqb);   // (evenly)
  f.ws = f.nsplit > 1 ? (long)f.nsplit * a->B * a->heads * a->Nq * (a->hd + 2) * 4 : 0;
  return f;
}

template <typename T, int HDP, bool RES, bool SPLIT, bool DROP>
int launch_fwd(const CrossParams& p, hipStream_t st) {
  auto kern = cross_fwd_kernel<T, HDP, RES, SPLIT, DROP>;
  const long blocks = (long)p.B * p.nsplit * p.nqb * p.H;
  if (blocks > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
  static unsigned long long attr_devs = 0ull;
  if (dm_first_on_device(attr_devs) &&
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                          RES ? LDS_IMAGE : 2 * image_bytes<T, HDP>()) != hipSuccess)
    return DM_ERR_LAUNCH;
  size_t lds = RES ? (size_t)p.kb * (Geo<T, HDP>::SR + Geo<T, HDP>::ST + 4) + (p.kb / 32 + 2) * 4 : 2 * image_bytes<T, HDP>();
  if (SPLIT && lds < 4 * 32 * ((HDP + 4) * 4 + 8)) lds = 4 * 32 * ((HDP + 4) * 4 + 8);
  static const DmVariantName nm("cross_fwd<%s,%d,%s>", sizeof(T) == 2 ? "bf16" : "fp32", HDP, SPLIT ? "split" : (RES ? "resident" : "streamed"));
  dm_set_variant(nm.s);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), lds, st, p);
  DM_LAUNCH_CHECK();
  return p.nsplit > 1 ? join_launch(p, sizeof(T) == 2 ? 0 : 1, st) : DM_OK;
}
template <typename T, int HDP, bool RES, bool SPLIT> int pick_drop(const CrossParams& p, hipStream_t st) {
  return p.thresh ? launch_fwd<T, HDP, RES, SPLIT, true>(p, st) : launch_fwd<T, HDP, RES, SPLIT, false>(p, st);
}
template <typename T, int HDP> int pick_fwd(const CrossParams& p, bool res, hipStream_t st) {
  if (!res) return pick_drop<T, HDP, false, false>(p, st);
  return p.wk > 1 ? pick_drop<T, HDP, true, true>(p, st) : pick_drop<T, HDP, true, false>(p, st);
}
template <typename T> int pick_width(const CrossParams& p, bool res, hipStream_t st) {
  switch (cross_hdp(p.hd)) {
    case 16: return pick_fwd<T, 16>(p, res, st);
    case 32: return pick_fwd<T, 32>(p, res, st);
    case 64: return pick_fwd<T, 64>(p, res, st);
    case 96: return pick_fwd<T, 96>(p, res, st);
    default: return pick_fwd<T, 128>(p, res, st);
  }
}

}  // namespace

extern "C" long dm_cross_fwd_workspace_bytes(const dm_cross_args* a) {
  if (!dm_cross::cross_sizes_ok(a)) return 0;
  dm_cross::OnePlan one;
  const long ws = fwd_plan(a).ws;                              // (with dropout single queries take the tiles, too)
  return dm_cross::one_plan(a, one) && one.ws > ws ? one.ws : ws;
}

extern "C" int dm_cross_fwd(const dm_cross_args* a, dm_stream_t stream) {
  CrossParams p{};
  const int rc = cross_fill(p, a, false);
  if (rc != DM_OK) return rc;
  OnePlan one;
  if (p.thresh == 0 && one_plan(a, one)) {
    DM_REQUIRE(one.ws == 0 || (a->workspace && a->ws_bytes >= one.ws && (uintptr_t)a->workspace % 16 == 0));
    p.nsplit = one.nsplit; p.ksplit = one.ksplit;
    p.part = (float*)a->workspace;
    return one_launch(p, a->dtype, (hipStream_t)stream);
  }
  const FwdPlan f = fwd_plan(a);
  DM_REQUIRE(f.ws == 0 || (a->workspace && a->ws_bytes >= f.ws && (uintptr_t)a->workspace % 16 == 0));
  p.nsplit = f.nsplit; p.ksplit = f.ksplit; p.kb = f.kb; p.iters = f.iters; p.nqb = f.nqb; p.wk = f.wk;
  p.part = (float*)a->workspace;
  return a->dtype == 0 ? pick_width<bf16>(p, f.res, (hipStream_t)stream) : pick_width<float>(p, f.res, (hipStream_t)stream);
}
