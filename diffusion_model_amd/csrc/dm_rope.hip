// Rotary positions with several axes (time, height, width) on the heads of a query / key projection.
//
// Pair p of a head belongs to one axis a(p) and has a frequency f(p) = theta^(-2i/d_a) (i: the pair's place inside its
// axis, d_a: the channels of that axis).  For a token at position x_a the pair (u, w) becomes
//   (u cos t - w sin t,  w cos t + u sin t),   t = x_a f(p)       (t -> -t: the inverse, which is also the backward),
// channels past the rotated width are copied.  Pairs are neighbours (2p, 2p+1) or half the rotated width apart (p, p + R/2).
//
// Angles: far positions lose their fraction in 32 bits (x = 1e5 leaves 2^-7 of a radian), so the frequency is kept in TURNS per
// unit of position as a double; x f is reduced to a fraction of a turn in 64 bits and only then rounded to 32 (at most pi 2^-24
// of a radian, of the size of sincospif's own error) for sincospif.  A workgroup computes each (token, pair) angle ONCE into an
// LDS table and uses it for every head, so the 64-bit work is 1/heads of the elements and the kernel is a pure stream: one
// 16-byte load, one 16-byte store. bf16, 64 x 576 tokens, 16 heads of 32: 14.3 us (5.3 TB/s; a copy of these 75 MB, which the
// last-level cache holds, 11.7 us); 2 x 16384 tokens, 16 heads of 128, forward and inverse: 103 us (5.2 TB/s; two such copies
// 75 us); fp32, 8 x 1371 tokens, 16 heads of 40, positions of their own per sample, both ways: 30 us (3.8 TB/s).
#include "dm_common.h"

namespace {

struct FastDiv {          // n / d for n, d < 65536: (n * m) >> 32 with m = floor(2^32 / d) + 1 is exact there
  uint32_t d, m;
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, m); }
};

struct RopeParams {
  const char* x; char* y;
  long ldx, ldy;                  // row strides, elements
  long rows;                      // B * N
  uint32_t N;                     // tokens per sample
  int RT;                         // rows per workgroup
  uint32_t upr;                   // units per row = heads * uph
  FastDiv by_upr, by_uph, by_np;
  uint32_t hd, rot, uph;          // head width, rotated channels, units per head
  uint32_t ru;                    // half pairing: rotated units per head (the rest are copies)
  const double* freq; const int* axis; uint32_t np;     // per pair: turns per unit of position, axis
  const void* pos; int pos_f32; long pos_bs; uint32_t axes;   // explicit positions (NULL: the grid)
  uint32_t g1, g2;                // grid extents of the last two axes (row-major token order)
  int inverse;
};

template <typename T, int V> struct Vec { T v[V]; };
// V elements; one access where they make 8 or 16 bytes (the host has checked the alignment), element by element otherwise
template <typename T, int V> __device__ __forceinline__ Vec<T, V> ld_vec(const T* p) {
  Vec<T, V> r;
  if constexpr (V * sizeof(T) == 16) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
    __builtin_memcpy(&r, &w, 16);
  } else if constexpr (V * sizeof(T) == 8 && sizeof(T) == 2) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(p);
    __builtin_memcpy(&r, &w, 8);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = p[j];
  }
  return r;
}
template <typename T, int V> __device__ __forceinline__ void st_vec(T* p, const Vec<T, V>& r) {
  if constexpr (V * sizeof(T) == 16) {
    u32x4 w;
    __builtin_memcpy(&w, &r, 16);
    *reinterpret_cast<u32x4*>(p) = w;
  } else if constexpr (V * sizeof(T) == 8 && sizeof(T) == 2) {
    u32x2 w;
    __builtin_memcpy(&w, &r, 8);
    *reinterpret_cast<u32x2*>(p) = w;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] = r.v[j];
  }
}

// cos / sin of every (row, pair) of this workgroup
__device__ __forceinline__ void fill_table(const RopeParams& p, float2* tab, long row0, uint32_t rows) {
  const long b0 = row0 / p.N;
  const uint32_t n0 = (uint32_t)(row0 - b0 * p.N);
  for (uint32_t i = threadIdx.x; i < rows * p.np; i += 256) {
    const uint32_t r = p.by_np.div(i), pr = i - r * p.np;
    const uint32_t nn = n0 + r, bq = nn / p.N, n = nn - bq * p.N;
    const uint32_t a = (uint32_t)p.axis[pr];
    double pos;
    if (p.pos) {
      const long o = (b0 + bq) * p.pos_bs + (long)n * p.axes + a;
      pos = p.pos_f32 ? (double)((const float*)p.pos)[o] : (double)((const int*)p.pos)[o];
    } else {
      const uint32_t last = n % p.g2, up = n / p.g2;       // (row-major grid: the last axis is the fastest)
      pos = (double)(a + 1 == p.axes ? last : (a + 2 == p.axes ? up % p.g1 : up / p.g1));
    }
    double turns = pos * p.freq[pr];
    turns -= __builtin_rint(turns);
    float s, c;
    sincospif(2.f * (float)turns, &s, &c);
    tab[i] = float2{c, p.inverse ? -s : s};
  }
}

// A unit is V channels (interleaved) or V channels and their partners R/2 further on (half).  U units are loaded per
// thread before the table is built, so that the loads fly while the angles are computed.
template <typename T, bool HALF, int V>
__global__ __launch_bounds__(256) void rope_kernel(const RopeParams p) {
  extern __shared__ float2 tab[];
  constexpr int U = HALF ? 2 : 4;
  const long row0 = (long)blockIdx.x * p.RT;
  const uint32_t rows = (uint32_t)(p.rows - row0 < p.RT ? p.rows - row0 : p.RT);
  const uint32_t total = rows * p.upr;
  const T* x = (const T*)p.x + row0 * p.ldx;
  T* y = (T*)p.y + row0 * p.ldy;
  bool ready = false;
  for (uint32_t base = 0; base < total; base += 256 * U) {
    Vec<T, V> a[U], b[U];
    uint32_t row[U], col[U], pr[U];
    bool rot[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t id = base + u * 256 + threadIdx.x;
      const uint32_t k = id < total ? id : total - 1;
      row[u] = p.by_upr.div(k);
      const uint32_t j = k - row[u] * p.upr, h = p.by_uph.div(j), c = j - h * p.uph;
      rot[u] = HALF ? c < p.ru : c * V < p.rot;
      pr[u] = HALF ? c * V : c * (V / 2);
      col[u] = h * p.hd + (HALF && !rot[u] ? p.rot + (c - p.ru) * V : c * V);
      a[u] = ld_vec<T, V>(x + (long)row[u] * p.ldx + col[u]);
      if (HALF && rot[u]) b[u] = ld_vec<T, V>(x + (long)row[u] * p.ldx + col[u] + p.rot / 2);
    }
    if (!ready) {
      fill_table(p, tab, row0, rows);
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + u * 256 + threadIdx.x >= total) continue;
      const float2* cs = tab + row[u] * p.np + pr[u];
      T* dst = y + (long)row[u] * p.ldy + col[u];
      if constexpr (HALF) {
        if (rot[u]) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float2 t = cs[j];
            const float e = (float)a[u].v[j], o = (float)b[u].v[j];
            a[u].v[j] = (T)(e * t.x - o * t.y);
            b[u].v[j] = (T)(o * t.x + e * t.y);
          }
          st_vec<T, V>(dst + p.rot / 2, b[u]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
          if (pr[u] + j >= p.np) continue;      // channels past the rotated width pass through unread by the arithmetic
          const float2 t = cs[j];
          const float e = (float)a[u].v[2 * j], o = (float)a[u].v[2 * j + 1];
          a[u].v[2 * j] = (T)(e * t.x - o * t.y);
          a[u].v[2 * j + 1] = (T)(o * t.x + e * t.y);
        }
      }
      st_vec<T, V>(dst, a[u]);
    }
  }
}

FastDiv fast_div(uint32_t d) {
  FastDiv f;
  f.d = d;
  f.m = d > 1 ? (uint32_t)((1ull << 32) / d + 1) : 0u;
  return f;
}

template <typename T, bool HALF, int V>
int launch(RopeParams& p, int heads, hipStream_t st) {
  p.ru = HALF ? p.rot / 2 / V : 0;
  p.uph = HALF ? p.ru + (p.hd - p.rot) / V : (p.hd + V - 1) / V;
  p.upr = p.uph * heads;
  if (p.upr >= 65536u) return DM_ERR_ARG;       // (FastDiv's range)
  // rows per workgroup: a full strip of loads per thread (4 x 16 bytes), fewer when the call is too small to give every
  // CU a workgroup; the table (8 bytes per row and pair) stays within 16 KiB
  const int strip = 256 * (HALF ? 2 : 4);
  long rt = (strip + p.upr - 1) / p.upr;
  const long spread = p.rows / 512;
  if (rt > spread) rt = spread < 1 ? 1 : spread;
  const long fit = 16384 / 8 / p.np;
  if (rt > fit) rt = fit < 1 ? 1 : fit;
  p.RT = (int)rt;
  p.by_upr = fast_div(p.upr);
  p.by_uph = fast_div(p.uph);
  p.by_np = fast_div(p.np);
  const long blocks = (p.rows + rt - 1) / rt;
  if (blocks > DM_MAX_GRID256) return DM_ERR_TOO_LARGE;
  static const DmVariantName nm("rope<%s,%s,V=%d>", sizeof(T) == 2 ? "bf16" : "fp32", HALF ? "half" : "interleaved", V);
  dm_set_variant(nm.s);
  hipLaunchKernelGGL((rope_kernel<T, HALF, V>), dim3((unsigned)blocks), dim3(256), (size_t)rt * p.np * 8, st, p);
  DM_LAUNCH_CHECK();
  return DM_OK;
}

}  // namespace

extern "C" int dm_rope(const dm_rope_args* a, dm_stream_t stream) {
  DM_REQUIRE(a && a->x && a->y && a->freq && a->axis);
  DM_REQUIRE(a->B > 0 && a->N > 0 && a->heads > 0 && a->hd >= 2 && a->hd <= 2048 && a->hd % 2 == 0);
  DM_REQUIRE((long)a->heads * a->hd < 65536);
  DM_REQUIRE(a->rot >= 2 && a->rot % 2 == 0 && a->rot <= a->hd);
  DM_REQUIRE(a->axes >= 1 && a->axes <= 3 && (a->dtype == 0 || a->dtype == 1) && (a->pairing == 0 || a->pairing == 1));
  DM_REQUIRE(a->ldx >= (long)a->heads * a->hd && a->ldy >= (long)a->heads * a->hd);
  DM_REQUIRE(a->x != a->y || a->ldx == a->ldy);       // (in place: the same rows)
  if (!a->pos) {
    long n = 1;
    for (int i = 0; i < a->axes; ++i) {
      DM_REQUIRE(a->grid[i] > 0);
      n *= a->grid[i];
      DM_REQUIRE(n <= a->N);
    }
    DM_REQUIRE(n == a->N);
  }
  RopeParams p{};
  p.x = (const char*)a->x; p.y = (char*)a->y; p.ldx = a->ldx; p.ldy = a->ldy;
  p.rows = (long)a->B * a->N; p.N = (uint32_t)a->N;
  p.hd = a->hd; p.rot = a->rot; p.np = a->rot / 2;
  p.freq = a->freq; p.axis = a->axis; p.axes = a->axes;
  p.pos = a->pos; p.pos_f32 = a->pos_f32; p.pos_bs = a->pos_batch_stride;
  p.g2 = a->pos ? 1 : a->grid[a->axes - 1];
  p.g1 = (a->pos || a->axes < 2) ? 1 : a->grid[a->axes - 2];
  p.inverse = a->inverse;
  const hipStream_t st = (hipStream_t)stream;
  const int e = a->dtype == 0 ? 2 : 4;
  // widest unit that every head, the two halves of a pair and both tensors are aligned for
  auto fits = [&](int V) {
    const long bytes = (long)V * e;
    if (a->hd % V || a->ldx % V || a->ldy % V || (uintptr_t)a->x % bytes || (uintptr_t)a->y % bytes) return false;
    return a->pairing == 0 || (a->rot / 2 % V == 0 && (a->hd - a->rot) % V == 0);
  };
  if (a->dtype == 0) {
    if (a->pairing == 0) {
      if (fits(8)) return launch<bf16, false, 8>(p, a->heads, st);
      if (fits(4)) return launch<bf16, false, 4>(p, a->heads, st);
      return launch<bf16, false, 2>(p, a->heads, st);
    }
    if (fits(8)) return launch<bf16, true, 8>(p, a->heads, st);
    if (fits(4)) return launch<bf16, true, 4>(p, a->heads, st);
    return launch<bf16, true, 1>(p, a->heads, st);
  }
  if (a->pairing == 0) {
    if (fits(4)) return launch<float, false, 4>(p, a->heads, st);
    return launch<float, false, 2>(p, a->heads, st);
  }
  if (fits(4)) return launch<float, true, 4>(p, a->heads, st);
  return launch<float, true, 1>(p, a->heads, st);
}
