// Backward for single queries (a pooled token) and other short row lists: few rows -- the queries of every sample that uses a
// context, times the query heads of a key / value head -- against many states.  Matrix tiles of 32 queries would be mostly
// empty and read the states twice, so this streams them once: LPR lanes hold the 16-byte pieces of a state's key and value
// (as the forward of single queries does), U states per lane, whose dK and dV stay in the same lane's registers while the
// workgroup walks ALL rows of the context, 16 at a time out of LDS: no partials of dK and dV, whatever shares the context.
//   s = q k, dp = dO v (sums over the LPR lanes), P = exp2(c s - lse log2(e)), dS = P (dp - delta),
//   dK += dS q, dV += P dO (in the lane), dQ += dS k: over the lanes, then the waves through LDS, then the workgroups.
// Bound by the states' bytes at one row (8 queries, 8 heads of 64, 4096 states, bf16: 34 us, 4.0 TB/s), by the work per row past
// three or four.
#include "dm_cross.h"

namespace {

using namespace dm_cross;

constexpr int ROWS = 16;       // rows in LDS at a time
// states in a lane's registers, in 32 bits with their gradients (two instead of four for wide heads: 49 us, not 40, for 8 rows
// on 32 x 500 states, 8 heads of 64, bf16: what each row costs a wave is spread over fewer states)
constexpr int states_per_lane(int lpr) { return lpr >= 8 ? 4 : (lpr == 4 ? 2 : 1); }
constexpr int states_per_wg(int lpr) { return 4 * (64 / lpr) * states_per_lane(lpr); }

// Sum over the 64 / LPR lane groups.  Each step halves the elements a lane still holds until one is left: 7 exchanges for 8
// elements over 8 groups, not 24.  Afterwards the lane holds x[0..n) = elements [off, off + n).
template <int LPR, int E> __device__ __forceinline__ int group_sum(float (&x)[E], int lane) {
  int off = 0, n = E;
#pragma unroll
  for (int w = LPR; w < 64; w <<= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = lane & w;
#pragma unroll
      for (int j = 0; j < E / 2; ++j)
        if (j < n) {
          const float give = up ? x[j] : x[j + n], keep = up ? x[j + n] : x[j];
          x[j] = keep + __shfl_xor(give, w, 64);
        }
      off += up ? n : 0;
    } else {
      x[0] += __shfl_xor(x[0], w, 64);
    }
  }
  return off;
}
template <int LPR, int E> constexpr int group_left() {
  int n = E;
  for (int w = LPR; w < 64; w <<= 1) n = n > 1 ? n / 2 : 1;
  return n;
}

template <typename T, int LPR, bool DROP>
__global__ __launch_bounds__(256) void cross_onebwd_kernel(const CrossParams p) {
  constexpr int E = 16 / (int)sizeof(T), RPS = 64 / LPR, U = states_per_lane(LPR), DS = LPR * E + 4;
  __shared__ __attribute__((aligned(16))) u32x4 sQ[ROWS][LPR], sD[ROWS][LPR];
  __shared__ __attribute__((aligned(16))) float sDq[4][ROWS][DS];
  __shared__ float sL[ROWS], sDelta[ROWS];
  __shared__ uint32_t sWord[ROWS];
  __shared__ int sSample[ROWS], sOf[ROWS];       // sample, row of the sample (head of the group * Nq + query)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), piece = lane % LPR, group = lane / LPR;
  uint32_t id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int g = id % p.G;
  id /= p.G;
  const int tile = id % p.qsplit, ctx = id / p.qsplit;
  const int kn = keys_of(p, ctx), HG = p.H / p.G, per_sample = HG * p.Nq, hdb = p.hd * (int)sizeof(T);
  const int k0 = tile * states_per_wg(LPR);
  const bool active = k0 < kn, mine = piece * 16 < hdb;
  const long krow = (long)ctx * p.Nk;
  const float c = p.scale * CR_LOG2E;
  const uint32_t seed = DROP ? dm_eff_seed(p.seed, p.seed_ctr) : 0u;
  bool ok[U];
  float kf[U][E], vf[U][E], dk[U][E], dv[U][E];
  auto key_of = [&](int u) { return k0 + (wave * U + u) * RPS + group; };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int key = key_of(u);
    ok[u] = key < kn && (!p.mask || p.mask[krow + key]);
    const bool get = ok[u] && mine;      // (what invalid states hold is not read)
    const u32x4 kw = get ? *reinterpret_cast<const u32x4*>(p.k + (krow + key) * p.ldk + g * hdb + piece * 16) : u32x4{0u, 0u, 0u, 0u};
    const u32x4 vw = get ? *reinterpret_cast<const u32x4*>(p.v + (krow + key) * p.ldv + g * hdb + piece * 16) : u32x4{0u, 0u, 0u, 0u};
    widen<T>(kw, kf[u]);
    widen<T>(vw, vf[u]);
#pragma unroll
    for (int e = 0; e < E; ++e) dk[u][e] = dv[u][e] = 0.f;
  }

  Samples at;
  at.first(p, ctx, lane);
  int next = 0;                        // row of the present sample that comes next
  while (!at.done) {
    // 16 rows: 16 threads each
    const int slot = tid >> 4;
    int count = 0, b = 0, of = 0;
    for (; count < ROWS && !at.done; ++count) {
      if (count == slot) { b = at.b; of = next; }
      if (++next == per_sample) {
        next = 0;
        at.sample(p, lane);
      }
    }
    __syncthreads();                   // (the sums of the rows before have been read)
    if (slot < count) {
      const int h = g * HG + of / p.Nq, n = of % p.Nq;
      const long tok = (long)b * p.Nq + n, row = ((long)b * p.H + h) * p.Nq + n;
      if (active) {
        float delta = 0.f;
        for (int pc = tid & 15; pc < LPR; pc += 16) {
          const bool in = pc * 16 < hdb;
          const long off = (long)h * hdb + pc * 16;
          const u32x4 zero = {0u, 0u, 0u, 0u};
          const u32x4 qw = in ? *reinterpret_cast<const u32x4*>(p.q + tok * p.ldq + off) : zero;
          const u32x4 dw = in ? *reinterpret_cast<const u32x4*>(p.d_o + tok * p.lddo + off) : zero;
          const u32x4 ow = in ? *reinterpret_cast<const u32x4*>(p.o + tok * p.ldo + off) : zero;
          float df[E], of_[E];
          widen<T>(dw, df);
          widen<T>(ow, of_);
#pragma unroll
          for (int e = 0; e < E; ++e) delta = __builtin_fmaf(df[e], of_[e], delta);
          sQ[slot][pc] = qw;
          sD[slot][pc] = dw;
        }
        delta = row_sum<16>(delta);
        if ((tid & 15) == 0) {
          const float l = p.lse[row] * CR_LOG2E;
          sL[slot] = l == -INFINITY ? INFINITY : l;      // (no probability without a finite score)
          sDelta[slot] = delta;
          if (DROP) sWord[slot] = dm_drop_row(seed, (uint32_t)row);
        }
      }
      if ((tid & 15) == 0) { sSample[slot] = b; sOf[slot] = of; }
    }
    __syncthreads();
    if (active) {
      for (int r = 0; r < count; ++r) {
        float qf[E], df[E], dq[E];
        widen<T>(sQ[r][piece], qf);
        widen<T>(sD[r][piece], df);
        const float L2 = sL[r], delta = sDelta[r];
#pragma unroll
        for (int e = 0; e < E; ++e) dq[e] = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float s = 0.f, dp = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            s = __builtin_fmaf(qf[e], kf[u][e], s);
            dp = __builtin_fmaf(df[e], vf[u][e], dp);
          }
          s = row_sum<LPR>(s);
          dp = row_sum<LPR>(dp);
          float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, -L2)), z = 1.f;
          if (DROP) {
            const uint32_t key = (uint32_t)key_of(u);
            z = dm_keep16(dm_drop_bits(sWord[r], key >> 1), key, p.thresh) ? p.inv_keep : 0.f;
          }
          const float ds = ok[u] ? pr * ((DROP ? dp * z : dp) - delta) : 0.f;
          pr = ok[u] ? (DROP ? pr * z : pr) : 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            dk[u][e] = __builtin_fmaf(ds, qf[e], dk[u][e]);
            dv[u][e] = __builtin_fmaf(pr, df[e], dv[u][e]);
            dq[e] = __builtin_fmaf(ds, kf[u][e], dq[e]);
          }
        }
        const int off = group_sum<LPR, E>(dq, lane);
#pragma unroll
        for (int j = 0; j < group_left<LPR, E>(); ++j) sDq[wave][r][piece * E + off + j] = dq[j];
      }
    }
    __syncthreads();
    const int per = p.hd >> 2;
    const long rows = (long)p.B * p.H * p.Nq;
    for (int i = tid; i < count * per; i += 256) {
      const int r = i / per, col = (i - r * per) * 4, bb = sSample[r], h = g * HG + sOf[r] / p.Nq, n = sOf[r] % p.Nq;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      if (active) {
#pragma unroll
        for (int w = 0; w < 4; ++w) x += *reinterpret_cast<const f32x4*>(&sDq[w][r][col]);
      }
      if (p.nsplit)
        *reinterpret_cast<f32x4*>(p.qpart + (tile * rows + ((long)bb * p.H + h) * p.Nq + n) * p.hd + col) = x;
      else
        store4<T>(p.dq + ((long)bb * p.Nq + n) * p.lddq + (h * p.hd + col) * (int)sizeof(T), x[0] * p.scale, x[1] * p.scale, x[2] * p.scale, x[3] * p.scale);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int key = key_of(u);
    if (key >= p.Nk || !mine) continue;
    char* ok_ = p.dk + (krow + key) * p.lddk + g * hdb + piece * 16;
    char* ov_ = p.dv + (krow + key) * p.lddv + g * hdb + piece * 16;
#pragma unroll
    for (int e = 0; e < E; e += 4) {      // (a NaN among the rows reaches no invalid state)
      store4<T>(ok_ + e * sizeof(T), ok[u] ? dk[u][e] * p.scale : 0.f, ok[u] ? dk[u][e + 1] * p.scale : 0.f, ok[u] ? dk[u][e + 2] * p.scale : 0.f, ok[u] ? dk[u][e + 3] * p.scale : 0.f);
      store4<T>(ov_ + e * sizeof(T), ok[u] ? dv[u][e] : 0.f, ok[u] ? dv[u][e + 1] : 0.f, ok[u] ? dv[u][e + 2] : 0.f, ok[u] ? dv[u][e + 3] : 0.f);
    }
  }
}

// Adds the partials of dQ: SL lanes split the list of one result (4 channels of one row) and join by a fixed tree, 8 for long
// lists, 1 for short ones.  A sample without a context has none.
template <typename T, int SL>
__global__ __launch_bounds__(256) void cross_dqsum_kernel(const CrossParams p) {
  constexpr int RPW = 64 / SL;
  const int lane = threadIdx.x & 63, slice = lane / RPW;
  const long rows = (long)p.B * p.H * p.Nq, n = rows * p.hd;
  const long r = (((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * RPW + lane % RPW) * 4, i = r < n ? r : 0;
  const long row = i / p.hd, bh = row / p.Nq, b = bh / p.H;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (context_of(p, (int)b) >= 0) {
#pragma unroll 4
    for (int k = slice; k < p.qsplit; k += SL) s += *reinterpret_cast<const f32x4*>(p.qpart + k * n + i);
  }
  if (SL > 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int o = RPW; o < 64; o <<= 1) s[j] += __shfl_xor(s[j], o, 64);
  }
  if (r >= n || slice) return;
  const int col = (int)(i - row * p.hd), h = (int)(bh - b * p.H);
  store4<T>(p.dq + (b * p.Nq + (row - bh * p.Nq)) * p.lddq + (h * p.hd + col) * (long)sizeof(T), s[0] * p.scale, s[1] * p.scale,
            s[2] * p.scale, s[3] * p.scale);
}
template <typename T> int launch_sum(const CrossParams& p, hipStream_t st) {
  const long n = (long)p.B * p.H * p.Nq * (p.hd >> 2);
  const bool wide = p.qsplit > 8;
  const long blocks = (n + (wide ? 31 : 255)) / (wide ? 32 : 256);
  if (blocks > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
  if (wide) hipLaunchKernelGGL((cross_dqsum_kernel<T, 8>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((cross_dqsum_kernel<T, 1>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  DM_LAUNCH_CHECK();
  return DM_OK;
}

template <typename T, int LPR, bool DROP> int launch(const CrossParams& p, hipStream_t st) {
  const long blocks = (long)p.Bc * p.qsplit * p.G;
  if (blocks > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
  static const DmVariantName nm("cross_bwd_one<%s,LPR=%d>", sizeof(T) == 2 ? "bf16" : "fp32", LPR);
  dm_set_variant(nm.s);
  hipLaunchKernelGGL((cross_onebwd_kernel<T, LPR, DROP>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  DM_LAUNCH_CHECK();
  return p.nsplit ? launch_sum<T>(p, st) : DM_OK;
}
template <typename T, int LPR> int pick_drop(const CrossParams& p, hipStream_t st) {
  return p.thresh ? launch<T, LPR, true>(p, st) : launch<T, LPR, false>(p, st);
}
int lanes_per_row(int hd, int esize) {
  const int pieces = hd * esize / 16;
  int l = 1;
  while (l < pieces) l *= 2;
  return l;
}
template <typename T> int pick_width(const CrossParams& p, hipStream_t st) {
  constexpr int least = 8 * (int)sizeof(T) / 16;      // pieces of the narrowest head; the widest has 16 times as many
  switch (lanes_per_row(p.hd, sizeof(T))) {
    case least: return pick_drop<T, least>(p, st);
    case 2 * least: return pick_drop<T, 2 * least>(p, st);
    case 4 * least: return pick_drop<T, 4 * least>(p, st);
    case 8 * least: return pick_drop<T, 8 * least>(p, st);
    default: return pick_drop<T, 16 * least>(p, st);
  }
}

}  // namespace

namespace dm_cross {

bool onebwd_plan(const dm_cross_args* a, OneBwdPlan& f) {
  // rows per context, on average, up to which this beats the matrix tiles, whose time hardly depends on them (16 samples, 8
  // heads of 128, 1000 states, backward: bf16 34 us here and 74 with tiles at 1 row, 56 and 76 at 6, 86 and 79 at 12; fp32 49
  // and 194 at 1, 107 and 218 at 16; 32 samples, 8 heads of 32, 77 states: bf16 4.8 and 10.3 at 1, 9.0 and 10.5 at 6, fp32
  // 4.8 and 17.3 at 1, 13.0 and 18.3 at 16)
  const int e = a->dtype == 0 ? 2 : 4;
  const double rows = (double)a->B * (a->heads / a->kv_heads) * a->Nq;
  if (a->Nk < 1 || rows > (e == 2 ? 6.0 : 16.0) * cross_used(a)) return false;
  const int keys = states_per_wg(lanes_per_row(a->hd, e));
  const long tiles = ((long)a->Nk + keys - 1) / keys;
  f.tiles = (int)tiles;
  // (with an index a sample may have no context, whose dQ the sum kernel writes)
  f.ws = tiles > 1 || a->index ? tiles * a->B * a->heads * a->Nq * a->hd * 4 : 0;
  return true;
}

int onebwd_launch(const CrossParams& p, int dtype, hipStream_t st) {
  return dtype == 0 ? pick_width<bf16>(p, st) : pick_width<float>(p, st);
}

int dqsum_launch(const CrossParams& p, int dtype, hipStream_t st) {
  return dtype == 0 ? launch_sum<bf16>(p, st) : launch_sum<float>(p, st);
}

}  // namespace dm_cross
