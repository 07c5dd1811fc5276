// Single queries (a pooled token, a decoder's next token) against an encoder's states: up to four rows -- queries times the
// query heads of one key / value head -- share every state.  A matrix tile would be 31/32 empty, and the bytes of the states
// are the whole cost, so this is a stream: LPR lanes hold the 16-byte pieces of a state's row, 64 / LPR states per wave and
// step, four steps in flight; the scores are reduced over the LPR lanes, and every group of lanes keeps its own running
// maximum, sum and output, joined at the end (lanes, then the four waves through LDS, then the key splits).
// 8 queries, 8 heads of 64, up to 4096 states, bf16: 15.7 us with the join (2.7 TB/s; half of it is the ramp and the join).
#include "dm_cross.h"

namespace {

using namespace dm_cross;

template <typename T, int LPR, int R>
__global__ __launch_bounds__(256) void cross_one_kernel(const CrossParams p) {
  constexpr int E = 16 / (int)sizeof(T), RPS = 64 / LPR, U = 4;
  __shared__ float sO[4][R][LPR * E + 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, piece = lane % LPR, group = lane / LPR;
  uint32_t id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int g = id % p.G;
  id /= p.G;
  const int split = id % p.nsplit, b = id / p.nsplit;
  const int ctx = context_of(p, b), kn = keys_of(p, ctx), HG = p.H / p.G, rows = HG * p.Nq;
  const int k0 = split * p.ksplit, k1 = min(kn, k0 + p.ksplit);
  const int hdb = p.hd * (int)sizeof(T);
  const long krow = (long)(ctx < 0 ? 0 : ctx) * p.Nk;
  const bool mine = piece * 16 < hdb;
  const char* kbase = p.k + krow * p.ldk + g * hdb + (mine ? piece * 16 : 0);
  const char* vbase = p.v + krow * p.ldv + g * hdb + (mine ? piece * 16 : 0);
  const unsigned char* mask = p.mask ? p.mask + krow : nullptr;
  const float c = p.scale * CR_LOG2E;
  // row r: query r % Nq of the group's head r / Nq
  float q[R][E], o[R][E], m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int rr = min(r, rows - 1), h = g * HG + rr / p.Nq, n = rr % p.Nq;
    const u32x4 w = mine ? *reinterpret_cast<const u32x4*>(p.q + ((long)b * p.Nq + n) * p.ldq + h * hdb + piece * 16) : u32x4{0u, 0u, 0u, 0u};
    widen<T>(w, q[r]);
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[r][e] = 0.f;
  }
  for (int base = k0 + wave * RPS * U; base < k1; base += 4 * RPS * U) {
    u32x4 kw[U], vw[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = base + u * RPS + group, at = min(key, k1 - 1);      // (a state that exists; the surplus is masked below)
      kw[u] = *reinterpret_cast<const u32x4*>(kbase + at * p.ldk);
      vw[u] = *reinterpret_cast<const u32x4*>(vbase + at * p.ldv);
      ok[u] = key < k1 && (!mask || mask[at]);
    }
    float s[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float kf[E];
      widen<T>(kw[u], kf);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) x = __builtin_fmaf(q[r][e], kf[e], x);
        x = row_sum<LPR>(mine ? x : 0.f);    // (lanes past the head width hold a copy of its first piece)
        s[u][r] = ok[u] ? x : -INFINITY;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mx = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[u][r]);
      // exactly 1 while the maximum stays: from m[r] * c - mc, contracted, the rounding of mc would be left, a factor on l and
      // o in every step
      const float ref = mx == -INFINITY ? 0.f : mx, mc = ref * c;
      const float alpha = __builtin_amdgcn_exp2f((m[r] - ref) * c);      // (m = -inf: 0)
      m[r] = mx;
      l[r] *= alpha;
#pragma unroll
      for (int e = 0; e < E; ++e) o[r][e] *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], c, -mc));
        l[r] += s[u][r];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float vf[E];
      widen<T>(ok[u] ? vw[u] : u32x4{0u, 0u, 0u, 0u}, vf);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] = __builtin_fmaf(s[u][r], vf[e], o[r][e]);
    }
  }
  // the groups of the wave, then the waves: [E channels of each piece][maximum (base 2)][sum]
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float mx = m[r];
#pragma unroll
    for (int w = LPR; w < 64; w <<= 1) mx = fmaxf(mx, __shfl_xor(mx, w, 64));
    const float ref = mx == -INFINITY ? 0.f : mx, mc = ref * c, f = __builtin_amdgcn_exp2f((m[r] - ref) * c);      // (as alpha)
    float x = l[r] * f;
#pragma unroll
    for (int w = LPR; w < 64; w <<= 1) x += __shfl_xor(x, w, 64);
    if (lane == 0) { sO[wave][r][LPR * E] = mx == -INFINITY ? -INFINITY : mc; sO[wave][r][LPR * E + 1] = x; }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float y = o[r][e] * f;
#pragma unroll
      for (int w = LPR; w < 64; w <<= 1) y += __shfl_xor(y, w, 64);
      if (group == 0) sO[wave][r][piece * E + e] = y;
    }
  }
  __syncthreads();
  const int per = p.hd >> 2;
  const long all = (long)p.B * p.H * p.Nq;
  for (int i = tid; i < rows * per; i += 256) {
    const int r = i / per, col = (i - r * per) * 4, h = g * HG + r / p.Nq, n = r % p.Nq;
    float mx = sO[0][r][LPR * E];
#pragma unroll
    for (int w = 1; w < 4; ++w) mx = fmaxf(mx, sO[w][r][LPR * E]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(sO[w][r][LPR * E] - ref);
      sum += f * sO[w][r][LPR * E + 1];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] += f * sO[w][r][col + j];
    }
    const long row = ((long)b * p.H + h) * p.Nq + n;
    if (p.nsplit > 1) {
      *reinterpret_cast<f32x4*>(p.part + (split * all + row) * p.hd + col) = f32x4{x[0], x[1], x[2], x[3]};
      if (col == 0) {
        float* ml = p.part + p.nsplit * all * p.hd + (split * all + row) * 2;
        ml[0] = ref;
        ml[1] = sum;
      }
    } else {
      const float inv = sum == 0.f ? 0.f : __builtin_amdgcn_rcpf(sum);
      store4<T>(p.o + ((long)b * p.Nq + n) * p.ldo + (h * p.hd + col) * (long)sizeof(T), x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
      if (col == 0) p.lse[row] = sum == 0.f ? -INFINITY : (ref + __builtin_amdgcn_logf(sum)) * CR_LN2;
    }
  }
}

// Joins the key splits, one wave per row: the splits' maxima and sums sit on the lanes, the weights are exchanged once, and
// the partial outputs are then independent loads.
template <typename T>
__global__ __launch_bounds__(256) void cross_join_kernel(const CrossParams p) {
  const long rows = (long)p.B * p.H * p.Nq, row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= rows) return;
  const float* ml = p.part + p.nsplit * rows * p.hd + row * 2;
  const bool have = lane < p.nsplit;
  const float mine = have ? ml[lane * rows * 2] : 0.f, ls = have ? ml[lane * rows * 2 + 1] : 0.f;
  float m = ls != 0.f ? mine : -INFINITY;
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) m = fmaxf(m, __shfl_xor(m, w, 64));
  const float f = ls != 0.f ? __builtin_amdgcn_exp2f(mine - m) : 0.f;      // (an empty split's partial is zero, too)
  float l = f * ls;
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) l += __shfl_xor(l, w, 64);
  const float inv = l == 0.f ? 0.f : p.inv_keep * __builtin_amdgcn_rcpf(l);
  // 16 lanes of 4 channels per quarter of the splits (two rounds of channels past 64)
  const int quarter = lane >> 4;
  const long bh = row / p.Nq, b = bh / p.H;
  const int h = (int)(bh - b * p.H);
  char* dst = p.o + (b * p.Nq + (row - bh * p.Nq)) * p.ldo + h * p.hd * (long)sizeof(T);
  for (int c0 = 0; c0 < p.hd; c0 += 64) {
    const int col = c0 + (lane & 15) * 4;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < p.nsplit; s0 += 4) {
      const int s = s0 + quarter;
      const float w = __shfl(f, s & 63, 64);
      if (s < p.nsplit && col < p.hd) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p.part + (s * rows + row) * p.hd + col);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += w * a[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] += __shfl_xor(x[j], 16, 64);
      x[j] += __shfl_xor(x[j], 32, 64);
    }
    if (quarter == 0 && col < p.hd) store4<T>(dst + col * sizeof(T), x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  }
  if (lane == 0) p.lse[row] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * CR_LN2;
}

template <typename T, int LPR, int R> int launch(const CrossParams& p, hipStream_t st) {
  const long blocks = (long)p.B * p.nsplit * p.G;
  if (blocks > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
  static const DmVariantName nm("cross_one<%s,LPR=%d,R=%d>", sizeof(T) == 2 ? "bf16" : "fp32", LPR, R);
  dm_set_variant(nm.s);
  hipLaunchKernelGGL((cross_one_kernel<T, LPR, R>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  DM_LAUNCH_CHECK();
  return p.nsplit > 1 ? join_launch(p, sizeof(T) == 2 ? 0 : 1, st) : DM_OK;
}
template <typename T, int LPR> int pick_rows(const CrossParams& p, hipStream_t st) {
  const int rows = p.H / p.G * p.Nq;
  if (rows == 1) return launch<T, LPR, 1>(p, st);
  return rows == 2 ? launch<T, LPR, 2>(p, st) : launch<T, LPR, 4>(p, st);
}
template <typename T> int pick_width(const CrossParams& p, hipStream_t st) {
  constexpr int least = 8 * (int)sizeof(T) / 16;      // pieces of the narrowest head; the widest has 16 times as many
  const int pieces = p.hd * (int)sizeof(T) / 16;
  if (pieces <= least) return pick_rows<T, least>(p, st);
  if (pieces <= 2 * least) return pick_rows<T, 2 * least>(p, st);
  if (pieces <= 4 * least) return pick_rows<T, 4 * least>(p, st);
  if (pieces <= 8 * least) return pick_rows<T, 8 * least>(p, st);
  return pick_rows<T, 16 * least>(p, st);
}

}  // namespace

namespace dm_cross {

bool one_plan(const dm_cross_args* a, OnePlan& f) {
  if ((long)a->heads / a->kv_heads * a->Nq > 4 || a->Nk < 1) return false;
  // splits of at least 256 states (64 per wave) until there are two workgroups per CU (8 queries, 8 heads of 64, 4096
  // states: 15.3 us with the join at two, 15.9 at one, 16.1 at four)
  const long blocks = (long)a->B * a->kv_heads;
  long ns = (512 + blocks - 1) / blocks;
  if (ns > a->Nk / 256) ns = a->Nk / 256;
  if (ns > MAX_SPLITS) ns = MAX_SPLITS;
  if (ns < 1) ns = 1;
  f.ksplit = (int)((a->Nk + ns - 1) / ns);
  f.nsplit = (a->Nk + f.ksplit - 1) / f.ksplit;
  f.ws = f.nsplit > 1 ? (long)f.nsplit * a->B * a->heads * a->Nq * (a->hd + 2) * 4 : 0;
  return true;
}

int one_launch(const CrossParams& p, int dtype, hipStream_t st) {
  return dtype == 0 ? pick_width<bf16>(p, st) : pick_width<float>(p, st);
}

int join_launch(const CrossParams& p, int dtype, hipStream_t st) {
  const long blocks = ((long)p.B * p.H * p.Nq + 3) / 4;
  if (blocks > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
  if (dtype == 0) hipLaunchKernelGGL((cross_join_kernel<bf16>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((cross_join_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, st, p);
  DM_LAUNCH_CHECK();
  return DM_OK;
}

}  // namespace dm_cross
