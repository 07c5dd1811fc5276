// Backward for the lists of rows between a few and a few tiles (dm_cross_onebwd.hip's, where they are too many for the vector
// units): 32 rows at a time -- queries of any of the samples that use the context, under any head of the group -- against 128
// states per workgroup, 32 on the lanes of each wave.  The rows are gathered into LDS, so short queries of many samples fill
// the matrix tiles; the states are read once, their dK and dV stay in registers over the whole list, and
// dQ^T = K^T dS^T takes dS through a small LDS tile (written [state][row], read transposed).  The waves add dQ up in wave order,
// the workgroups of a list through fp32 partials: no atomics.  Against the two kernels of dm_cross_bwd.hip that is five products
// instead of seven, the states read once and one launch less; past a tile or two the partials of dQ cost more than that.
// bf16, 38 samples of 10 queries, 2 heads on 1 of 24, 1894 states, forward and backward: 23.2 us (28.7 with two kernels);
// 2 samples of 5, 32 heads on 8 of 24, 2501 states: 23.7 (31.2).
#include "dm_cross.h"

namespace {

using namespace dm_cross;

constexpr int ROWS = 32, STATES = 128;
template <typename T> constexpr int patch_stride() { return sizeof(T) == 2 ? 72 : 144; }
template <typename T, int HDP> constexpr int lds_bytes() {
  return 2 * ROWS * Geo<T, HDP>::SR + 4 * 32 * (Geo<T, HDP>::ST + patch_stride<T>()) + ROWS * (HDP + 4) * 4 + ROWS * 20;
}

template <typename T, int HDP, bool DROP>
__global__ __launch_bounds__(256, HDP * (int)sizeof(T) < 192 ? 2 : 1) void cross_rows_kernel(const CrossParams p) {
  typedef Geo<T, HDP> Gm;
  typedef typename Cr<T>::frag frag;
  constexpr int PS = patch_stride<T>(), NF = Cr<T>::NF, E = 16 / (int)sizeof(T), RS = HDP + 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  char* sQ = smem;
  char* sD = sQ + ROWS * Gm::SR;
  char* sK = sD + ROWS * Gm::SR + wave * 32 * Gm::ST;
  char* patch = sD + ROWS * Gm::SR + 4 * 32 * Gm::ST + wave * 32 * PS;
  float* sum = reinterpret_cast<float*>(sD + ROWS * Gm::SR + 4 * 32 * (Gm::ST + PS));
  float* sL = sum + ROWS * RS;
  float* sDelta = sL + ROWS;
  uint32_t* sWord = reinterpret_cast<uint32_t*>(sDelta + ROWS);
  int* sSample = reinterpret_cast<int*>(sWord + ROWS);
  int* sOf = sSample + ROWS;                     // row of the sample (head of the group * Nq + query)
  uint32_t id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int g = id % p.G;
  id /= p.G;
  const int tile = id % p.qsplit, ctx = id / p.qsplit;
  const int kn = keys_of(p, ctx), HG = p.H / p.G, per_sample = HG * p.Nq, hdb = p.hd * (int)sizeof(T);
  const int key = tile * STATES + wave * 32 + (lane & 31);
  const long krow = (long)ctx * p.Nk + key;
  const bool valid = key < kn && (!p.mask || p.mask[krow]);
  const bool active = __any(valid), some = tile * STATES < kn;      // (of this wave, of the workgroup)
  const float c = p.scale * CR_LOG2E;
  const uint32_t seed = DROP ? dm_eff_seed(p.seed, p.seed_ctr) : 0u;
  frag kf[Gm::NC], vf[Gm::NC];
  load_frags<T, HDP>(p.k + krow * p.ldk + g * hdb, valid, hdb, lane, kf);
  load_frags<T, HDP>(p.v + krow * p.ldv + g * hdb, valid, hdb, lane, vf);
#pragma unroll
  for (int kc = 0; kc < Gm::NC; ++kc) *reinterpret_cast<frag*>(sK + (lane & 31) * Gm::ST + kc * 32 + half * 16) = kf[kc];
  f32x16 dk[Gm::DT], dv[Gm::DT];
#pragma unroll
  for (int d = 0; d < Gm::DT; ++d) { dk[d] = zero16(); dv[d] = zero16(); }

  Samples at;
  at.first(p, ctx, lane);
  int next = 0;                                  // row of the present sample that comes next
  while (!at.done) {
    const int slot = tid >> 3;                   // 8 threads per row
    int count = 0, b = 0, of = 0;
    for (; count < ROWS && !at.done; ++count) {
      if (count == slot) { b = at.b; of = next; }
      if (++next == per_sample) {
        next = 0;
        at.sample(p, lane);
      }
    }
    __syncthreads();                             // (the rows and sums before have been read)
    if (some) {
      const bool have = slot < count;
      const int h = g * HG + of / p.Nq, n = of % p.Nq;
      const long tok = (long)b * p.Nq + n, row = ((long)b * p.H + h) * p.Nq + n;
      float delta = 0.f;
#pragma unroll
      for (int pc = tid & 7; pc < Gm::PPR; pc += 8) {
        const bool in = have && pc * 16 < hdb;
        const long off = (long)h * hdb + pc * 16;
        const u32x4 zero = {0u, 0u, 0u, 0u};
        const u32x4 qw = in ? *reinterpret_cast<const u32x4*>(p.q + tok * p.ldq + off) : zero;
        const u32x4 dw = in ? *reinterpret_cast<const u32x4*>(p.d_o + tok * p.lddo + off) : zero;
        const u32x4 ow = in ? *reinterpret_cast<const u32x4*>(p.o + tok * p.ldo + off) : zero;
        float x[E], y[E];
        widen<T>(dw, x);
        widen<T>(ow, y);
#pragma unroll
        for (int e = 0; e < E; ++e) delta = __builtin_fmaf(x[e], y[e], delta);
        *reinterpret_cast<u32x4*>(sQ + slot * Gm::SR + pc * 16) = qw;
        *reinterpret_cast<u32x4*>(sD + slot * Gm::SR + pc * 16) = dw;
      }
      delta = row_sum<8>(delta);
      if ((tid & 7) == 0) {
        const float l = have ? p.lse[row] * CR_LOG2E : INFINITY;
        sL[slot] = l == -INFINITY ? INFINITY : l;      // (no probability without a finite score, nor past the list)
        sDelta[slot] = delta;
        if (DROP) sWord[slot] = dm_drop_row(seed, (uint32_t)row);
      }
    }
    if ((tid & 7) == 0 && slot < count) { sSample[slot] = b; sOf[slot] = of; }
    __syncthreads();
    f32x16 dq[Gm::DT];
    if (active) {
      f32x16 s = zero16(), dp = zero16(), pd;    // pd: what multiplies dO, the probability, dropped
#pragma unroll
      for (int kc = 0; kc < Gm::NC; ++kc) {
        s = Cr<T>::mma(row_frag<T>(sQ, Gm::SR, kc, lane), kf[kc], s);
        dp = Cr<T>::mma(row_frag<T>(sD, Gm::SR, kc, lane), vf[kc], dp);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(sL + 8 * i + 4 * half);
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(sDelta + 8 * i + 4 * half);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float pr = valid ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i + r], c, -l4[r])) : 0.f;
          float z = 1.f;
          if (DROP) z = dm_keep16(dm_drop_bits(sWord[8 * i + 4 * half + r], (uint32_t)key >> 1), (uint32_t)key, p.thresh) ? p.inv_keep : 0.f;
          pd[4 * i + r] = DROP ? pr * z : pr;
          s[4 * i + r] = valid ? pr * ((DROP ? dp[4 * i + r] * z : dp[4 * i + r]) - d4[r]) : 0.f;      // (masked: also under a NaN)
        }
        store4<T>(patch + (lane & 31) * PS + (8 * i + 4 * half) * (int)sizeof(T), s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
      }
      wave_lds_order();
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const frag pf = Cr<T>::pack(pd, f), sf = Cr<T>::pack(s, f), tf = tr_frag<T, 32>(patch, PS, f, 0, lane);
#pragma unroll
        for (int d = 0; d < Gm::DT; ++d) {
          dv[d] = Cr<T>::mma(tr_frag<T, HDP>(sD, Gm::SR, f, d, lane), pf, dv[d]);
          dk[d] = Cr<T>::mma(tr_frag<T, HDP>(sQ, Gm::SR, f, d, lane), sf, dk[d]);
          dq[d] = Cr<T>::mma(tr_frag<T, HDP>(sK, Gm::ST, f, d, lane), tf, f == 0 ? zero16() : dq[d]);
        }
      }
    } else {
#pragma unroll
      for (int d = 0; d < Gm::DT; ++d) dq[d] = zero16();
    }
    // dQ of the four waves, added in wave order
    if (some) {
#pragma unroll 1
      for (int turn = 0; turn < 4; ++turn) {
        if (turn == wave && (turn == 0 || active)) {
#pragma unroll
          for (int d = 0; d < Gm::DT; ++d)
#pragma unroll
            for (int i = 0; i < (HDP < 32 ? 2 : 4); ++i) {
              f32x4* to = reinterpret_cast<f32x4*>(sum + (lane & 31) * RS + d * 32 + 8 * i + 4 * half);
              f32x4 v = {dq[d][4 * i], dq[d][4 * i + 1], dq[d][4 * i + 2], dq[d][4 * i + 3]};
              if (turn) v += *to;
              *to = v;
            }
        }
        __syncthreads();
      }
    }
    const int per = p.hd >> 2;
    const long rows = (long)p.B * p.H * p.Nq;
    for (int i = tid; i < count * per; i += 256) {
      const int r = i / per, col = (i - r * per) * 4, bb = sSample[r], h = g * HG + sOf[r] / p.Nq, n = sOf[r] % p.Nq;
      const f32x4 x = some ? *reinterpret_cast<const f32x4*>(sum + r * RS + col) : f32x4{0.f, 0.f, 0.f, 0.f};
      if (p.nsplit)
        *reinterpret_cast<f32x4*>(p.qpart + (tile * rows + ((long)bb * p.H + h) * p.Nq + n) * p.hd + col) = x;
      else
        store4<T>(p.dq + ((long)bb * p.Nq + n) * p.lddq + (h * p.hd + col) * (int)sizeof(T), x[0] * p.scale, x[1] * p.scale, x[2] * p.scale, x[3] * p.scale);
    }
  }
  if (key >= p.Nk) return;
  char* ok = p.dk + krow * p.lddk + g * hdb;
  char* ov = p.dv + krow * p.lddv + g * hdb;
#pragma unroll
  for (int d = 0; d < Gm::DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = d * 32 + 8 * i + 4 * half;
      if (col >= p.hd) continue;
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      const f32x4 a = valid ? f32x4{dk[d][4 * i], dk[d][4 * i + 1], dk[d][4 * i + 2], dk[d][4 * i + 3]} : zero;
      const f32x4 e = valid ? f32x4{dv[d][4 * i], dv[d][4 * i + 1], dv[d][4 * i + 2], dv[d][4 * i + 3]} : zero;
      store4<T>(ok + col * sizeof(T), a[0] * p.scale, a[1] * p.scale, a[2] * p.scale, a[3] * p.scale);
      store4<T>(ov + col * sizeof(T), e[0], e[1], e[2], e[3]);
    }
}

template <typename T, int HDP, bool DROP> int launch(const CrossParams& p, hipStream_t st) {
  auto kern = cross_rows_kernel<T, HDP, DROP>;
  constexpr int lds = lds_bytes<T, HDP>();
  static_assert(lds <= 160 * 1024, "LDS");
  const long blocks = (long)p.Bc * p.qsplit * p.G;
  if (blocks > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
  static unsigned long long attr_devs = 0ull;
  if (dm_first_on_device(attr_devs) &&
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
    return DM_ERR_LAUNCH;
  static const DmVariantName nm("cross_bwd_rows<%s,%d>", sizeof(T) == 2 ? "bf16" : "fp32", HDP);
  dm_set_variant(nm.s);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), lds, st, p);
  DM_LAUNCH_CHECK();
  return p.nsplit ? dqsum_launch(p, sizeof(T) == 2 ? 0 : 1, st) : DM_OK;
}
template <typename T, int HDP> int pick_drop(const CrossParams& p, hipStream_t st) {
  return p.thresh ? launch<T, HDP, true>(p, st) : launch<T, HDP, false>(p, st);
}
template <typename T> int pick_width(const CrossParams& p, hipStream_t st) {
  switch (cross_hdp(p.hd)) {
    case 16: return pick_drop<T, 16>(p, st);
    case 32: return pick_drop<T, 32>(p, st);
    case 64: return pick_drop<T, 64>(p, st);
    case 96: return pick_drop<T, 96>(p, st);
    default: return pick_drop<T, 128>(p, st);
  }
}

}  // namespace

namespace dm_cross {

bool rowsbwd_plan(const dm_cross_args* a, OneBwdPlan& f) {
  // rows per context, on average: one tile in bf16, two in fp32 (32 samples, 8 heads of 64, 500 states: bf16 36.0 us here and
  // 38.4 with two kernels at 32 rows, 44.6 and 41.8 at 48; fp32 78 and 90 at 32, 122 and 122 at 64, 165 and 156 at 96; 16
  // samples, 8 heads on 2 of 96, 77 states, 32 rows: bf16 12.1 and 19.0, fp32 19.5 and 39.0; 16 samples, 8 heads of 128, 1000
  // states, fp32, 32 rows: 145 and 244)
  // Shared contexts make some lists longer than the average; the widest heads in bf16 (one wave per SIMD)
  // lose by that (97 samples of 20 rows on 79 contexts of 917 states, 3 heads of 128, forward and backward: 205 us
  // here, 180 with two kernels; 27 samples on 20 contexts, 8 heads on 4 of 64: 38 and 48).
  const double rows = (double)a->B * (a->heads / a->kv_heads) * a->Nq;
  if (a->Nk < 1 || rows > (a->dtype == 0 ? 32.0 : 64.0) * cross_used(a)) return false;
  if (a->dtype == 0 && a->hd > 96 && a->index) return false;
  const long tiles = ((long)a->Nk + STATES - 1) / STATES;
  f.tiles = (int)tiles;
  f.ws = tiles > 1 || a->index ? tiles * a->B * a->heads * a->Nq * a->hd * 4 : 0;      // (as in onebwd_plan)
  return true;
}

int rowsbwd_launch(const CrossParams& p, int dtype, hipStream_t st) {
  return dtype == 0 ? pick_width<bf16>(p, st) : pick_width<float>(p, st);
}

}  // namespace dm_cross
