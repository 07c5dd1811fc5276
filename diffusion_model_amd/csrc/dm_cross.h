// Shared pieces of the cross-attention kernels (dm_cross_*.hip).
//
// One source serves bf16 and fp32.  Everything runs on the 32x32 MFMA tiles (32x32x16 bf16, four 32x32x2 fp32): in both
// types a FRAGMENT is 16 bytes per lane, the reduction chunk of one fragment is 32 bytes of a row (16 bf16 or 8 fp32), and
// lane l holds row l % 32, bytes [16 (l / 32), +16) of the chunk.  For fp32 that assigns the reduction indices to the four
// MFMAs in another order than memory's, the same for both operands, so the sum is the same.
//
// A 32x32 result tile puts column l % 32 and rows 8 i + 4 (l / 32) + r (register 4 i + r) into lane l.  Scores are computed
// with the softmax axis on the registers (forward, dq) or the lanes (dk, dv), and the probability tile is then, register by
// register, already the second product's operand over the reduction order "rows 8 i + 4 half + r"; the other operand takes
// that order through the row addresses of its transposing LDS reads (tr_frag).  Where one pass computes the products of both axes,
// a probability tile is also turned through LDS.
#pragma once
#include "dm_common.h"

namespace dm_cross {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float CR_LOG2E = 1.4426950408889634f;
constexpr float CR_LN2 = 0.6931471805599453f;

struct CrossParams {
  const char *q, *k, *v, *d_o;
  char *o, *dq, *dk, *dv;
  long ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;    // row strides, BYTES
  float* lse;
  float* delta;                                       // [B, heads, Nq]: sum_d dO * O (dq kernel -> dk / dv kernel)
  const int* lens; const unsigned char* mask; const int* index;
  int B, Bc, H, G, Nq, Nk, hd;
  float scale;
  uint32_t seed, thresh; float inv_keep; const uint32_t* seed_ctr;   // dropout (dm_common.h); thresh 0 = none
  int kb;                      // keys staged per LDS image (a multiple of 64)
  int iters;                   // query tiles per wave and workgroup
  int nqb;                     // workgroups along the queries
  int wk;                      // waves of a workgroup that share a query tile, each with its own keys (1, 2 or 4)
  int nsplit, ksplit;          // forward: key splits and keys per split; dk / dv: splits of the query list
  float* part;                 // split results
  int qsplit, qksplit;         // dq: key splits and keys per split
  float* qpart;                // [qsplit][B, heads, Nq][hd]
};

// context of a sample, or -1 (no keys)
__device__ __forceinline__ int context_of(const CrossParams& p, int b) {
  if (!p.index) return p.Bc == 1 ? 0 : b;
  const int c = p.index[b];
  return c >= 0 && c < p.Bc ? c : -1;
}
__device__ __forceinline__ int keys_of(const CrossParams& p, int c) {
  if (c < 0) return 0;
  const int n = p.lens ? p.lens[c] : p.Nk;
  return n < 0 ? 0 : (n > p.Nk ? p.Nk : n);
}

template <typename T> struct Cr;
template <> struct Cr<bf16> {
  typedef bf16x8 frag;
  static constexpr int NF = 2;      // fragments that a 32-row reduction takes
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // operand fragment f of a result tile (its rows are the reduction axis); in bf16 the probabilities and the score gradients are
  // rounded here, half a step (2^-8) of each value: the matrix units take no wider operand at their rate, and fp32 sums follow
  static __device__ __forceinline__ frag pack(const f32x16& s, int f) {
    frag r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (bf16)s[8 * f + j];
    return r;
  }
};
template <> struct Cr<float> {
  typedef f32x4 frag;
  static constexpr int NF = 4;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ frag pack(const f32x16& s, int f) {
    return frag{s[4 * f], s[4 * f + 1], s[4 * f + 2], s[4 * f + 3]};
  }
};

// Head width HDP: hd rounded up to 16, 32, 64, 96 or 128; the padding is zero in LDS and in the registers.
template <typename T, int HDP> struct Geo {
  static constexpr int RB = HDP * (int)sizeof(T);          // row bytes
  static constexpr int NC = RB / 32;                       // reduction chunks of a row
  static constexpr int DT = HDP < 32 ? 1 : HDP / 32;       // 32-channel tiles of a head-dim-major result
  static constexpr int PPR = RB / 16;                      // 16-byte pieces of a row
  // LDS row strides.  SR (rows read as operand rows, 16 bytes per lane and row): an odd number of 16-byte units, so that
  // any 16 consecutive rows start in different banks.  ST (rows read through the transposing loads, 64 bytes of each of
  // four rows at a time): 4 or 12 units modulo 16; 48 bytes where a row has only 32.
  static constexpr int SR = RB + 16;
  static constexpr int units = RB / 16;
  static constexpr int ST = sizeof(T) == 4 ? RB + 16 : (units < 4 ? 48 : (units == 8 ? 192 : (units == 16 ? 320 : RB)));
};

template <typename T, int HDP>
__device__ __forceinline__ typename Cr<T>::frag tr_frag(const char* tile, int stride, int f, int dt, int lane) {
  const int h = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    typedef s16x4 __attribute__((address_space(3))) * lds_ptr;
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const int qq = (lane & 15) >> 2, pp = lane & 3, c16 = HDP < 32 ? 0 : (lane >> 4) & 1;
    const char* a = tile + (16 * f + 4 * h + qq) * stride + dt * 64 + c16 * 32 + pp * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(a));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(a + 8 * stride));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    const int d = HDP < 32 ? lane & 15 : lane & 31;
    const char* a = tile + (8 * f + 4 * h) * stride + (dt * 32 + d) * 4;
    f32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = *reinterpret_cast<const float*>(a + j * stride);
    return r;
  }
}
template <typename T>
__device__ __forceinline__ typename Cr<T>::frag row_frag(const char* tile, int stride, int kc, int lane) {
  return *reinterpret_cast<const typename Cr<T>::frag*>(tile + (lane & 31) * stride + kc * 32 + (lane >> 5) * 16);
}
template <typename T> __device__ __forceinline__ typename Cr<T>::frag zero_frag() {
  return __builtin_bit_cast(typename Cr<T>::frag, u32x4{0u, 0u, 0u, 0u});
}
// the row fragments of one row straight from global memory (zero past the head width, and altogether if !ok)
template <typename T, int HDP>
__device__ __forceinline__ void load_frags(const char* row, bool ok, int hdb, int lane,
                                           typename Cr<T>::frag (&f)[Geo<T, HDP>::NC]) {
#pragma unroll
  for (int kc = 0; kc < Geo<T, HDP>::NC; ++kc) {
    const int off = kc * 32 + (lane >> 5) * 16;
    f[kc] = ok && off < hdb ? *reinterpret_cast<const typename Cr<T>::frag*>(row + off) : zero_frag<T>();
  }
}
// 32 rows from `first` (wave-uniform) of one head as a buffer: rows past `n` rows and pieces past the head width read as
// zero and are not written, without a branch or a 64-bit address per lane (rows are below 64 MiB apart: cross_fill)
struct Rows { __amdgpu_buffer_rsrc_t r; uint32_t at; };
__device__ __forceinline__ Rows rows_of(const char* first, long ld, int n, int hdb, int lane) {
  Rows x;
  x.r = __builtin_amdgcn_make_buffer_rsrc((void*)first, 0, n <= 0 ? 0 : (int)((n > 32 ? 31 : n - 1) * ld + hdb), 0x00020000);
  x.at = (uint32_t)((lane & 31) * ld);
  return x;
}
template <typename T, int HDP>
__device__ __forceinline__ void load_frags(const Rows& x, int hdb, int lane, typename Cr<T>::frag (&f)[Geo<T, HDP>::NC]) {
#pragma unroll
  for (int kc = 0; kc < Geo<T, HDP>::NC; ++kc) {
    const int off = kc * 32 + (lane >> 5) * 16;
    f[kc] = __builtin_bit_cast(typename Cr<T>::frag, __builtin_amdgcn_raw_buffer_load_b128(x.r, off < hdb ? (int)(x.at + off) : 0x7FFFFFFF, 0, 0));
  }
}
// Rows of two tensors of one shape (keys and values, queries and their gradients) on their way into LDS, N rows at a time:
// load() asks for all of a thread's pieces, store() puts them down, so the next rows fly while the present ones are used.
// Loads go through buffer descriptors, one address register per thread: rows from `valid` on and the padding of a head read
// as zero, without a clamp, a select or a branch (a branch around each load would wait for each in turn: B=16, 8 heads of
// 128, 1024 queries on 512 keys, forward: 92 us that way, 49 with clamped addresses).  Masked rows are zeroed on the way.
template <typename T, int HDP, int N> struct Stager {
  static constexpr int PPR = Geo<T, HDP>::PPR, RPS = 256 / PPR;            // pieces per row, rows per step of the workgroup
  static constexpr int U = (N + RPS - 1) / RPS;
  u32x4 a[U], b[U];
  unsigned char keep[U];      // mask bytes, looked at only when the rows are put down
  __device__ __forceinline__ void load(const char* srcA, long ldA, const char* srcB, long ldB, int r0, int valid,
                                       const unsigned char* mask, int hdb, int tid) {
    const int r = tid / PPR, pc = tid % PPR, left = min(valid - r0, N);
    const bool mine = r < RPS && pc * 16 < hdb;
    // a descriptor covers one step of RPS rows and ends with the tensor; rows too far apart for its 32-bit range take the
    // plain loads
    if ((long)RPS * ldA < 0x7FFFFFFFL && (long)RPS * ldB < 0x7FFFFFFFL) {
      const int va = mine ? (int)(r * ldA) + pc * 16 : 0x7FFFFFFF, vb = mine ? (int)(r * ldB) + pc * 16 : 0x7FFFFFFF;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int rows = min(left - u * RPS, RPS);
        const auto ra = __builtin_amdgcn_make_buffer_rsrc((void*)(srcA + (long)(r0 + u * RPS) * ldA), 0, rows > 0 ? (int)((rows - 1) * ldA) + hdb : 0, 0x00020000);
        const auto rb = __builtin_amdgcn_make_buffer_rsrc((void*)(srcB + (long)(r0 + u * RPS) * ldB), 0, rows > 0 ? (int)((rows - 1) * ldB) + hdb : 0, 0x00020000);
        a[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, va, 0, 0));
        b[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rb, vb, 0, 0));
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool in = mine && r + u * RPS < left;
        a[u] = in ? *reinterpret_cast<const u32x4*>(srcA + (r0 + r + u * RPS) * ldA + pc * 16) : u32x4{0u, 0u, 0u, 0u};
        b[u] = in ? *reinterpret_cast<const u32x4*>(srcB + (r0 + r + u * RPS) * ldB + pc * 16) : u32x4{0u, 0u, 0u, 0u};
      }
    }
    if (mask) {
#pragma unroll
      for (int u = 0; u < U; ++u) keep[u] = mask[min(r0 + u * RPS + r, valid - 1)];
    }
  }
  // n <= N: rows that the image has room for
  __device__ __forceinline__ void store(char* dstA, int strideA, char* dstB, int strideB, int n, bool masked, int tid) {
    const int r = tid / PPR, pc = tid % PPR;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (masked && keep[u] == 0) { a[u] = u32x4{0u, 0u, 0u, 0u}; b[u] = a[u]; }
      if (r >= RPS || r + u * RPS >= n) break;
      *reinterpret_cast<u32x4*>(dstA + (r + u * RPS) * strideA + pc * 16) = a[u];
      *reinterpret_cast<u32x4*>(dstB + (r + u * RPS) * strideB + pc * 16) = b[u];
    }
  }
};
// rows [r0, r0 + n) of a resident image
template <typename T, int HDP>
__device__ __forceinline__ void stage_rows2(char* dstA, int strideA, const char* srcA, long ldA, char* dstB, int strideB,
                                            const char* srcB, long ldB, int r0, int n, int valid, const unsigned char* mask,
                                            int hdb, int tid) {
  constexpr int N = Geo<T, HDP>::RB >= 512 ? 64 : 128;      // (at most 16 pieces in flight per thread)
  for (int at = 0; at < n; at += N) {
    const unsigned char* m = r0 + at < valid ? mask : nullptr;      // (rows past the end are zero anyway)
    Stager<T, HDP, N> st;
    st.load(srcA, ldA, srcB, ldB, r0 + at, valid, m, hdb, tid);
    st.store(dstA + at * strideA, strideA, dstB + at * strideB, strideB, min(N, n - at), m != nullptr, tid);
  }
}
// Validity of keys [r0, r0 + n): one word per 32 keys (empty tiles are skipped) and, per key, what its score starts from:
// 0 or -infinity.  A score tile always starts its accumulators from the latter: four broadcast LDS reads per tile, where
// clearing the registers or masking the scores would be 16 to 64 vector instructions of a loop that is bound by them.
__device__ __forceinline__ void stage_valid(uint32_t* bits, float* bias, int r0, int n, int valid, const unsigned char* mask, int tid) {
  for (int i = tid; i < ((n + 63) & ~63); i += 256) {
    const bool ok = i < n && r0 + i < valid && (!mask || mask[r0 + i]);
    const unsigned long long w = __ballot(ok);
    if ((tid & 63) == 0) { bits[i >> 5] = (uint32_t)w; bits[(i >> 5) + 1] = (uint32_t)(w >> 32); }
    if (i < n) bias[i] = ok ? 0.f : -INFINITY;
  }
}
// the same for an image of 64 keys that is asked for early and put down late (one wave's work)
__device__ __forceinline__ bool load_valid(int r0, int valid, const unsigned char* mask, int tid, unsigned char& byte) {
  const int key = r0 + (tid & 63);
  byte = 1;
  if (mask && tid < 64) byte = mask[min(key, valid - 1)];
  return key < valid;
}
__device__ __forceinline__ void store_valid(uint32_t* bits, float* bias, bool in, unsigned char byte, int tid) {
  if (tid >= 64) return;
  const bool ok = in && byte != 0;
  const unsigned long long w = __ballot(ok);
  bias[tid] = ok ? 0.f : -INFINITY;
  if (tid == 0) { bits[0] = (uint32_t)w; bits[1] = (uint32_t)(w >> 32); }
}
// start of a score tile whose rows are the 32 keys of `bias`
__device__ __forceinline__ f32x16 score_init(const float* bias, int half) {
  f32x16 s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 b = *reinterpret_cast<const f32x4*>(bias + 8 * i + 4 * half);
#pragma unroll
    for (int r = 0; r < 4; ++r) s[4 * i + r] = b[r];
  }
  return s;
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.f;
  return s;
}
// x of this lane and of its partner 32 lanes on (in the order of the halves)
__device__ __forceinline__ void half_swap(float x, float& a, float& b) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned r0 = r[0], r1 = r[1];     // (copied out: a bit cast of a vector's element reads the vector's first)
  a = __builtin_bit_cast(float, r0);
  b = __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ float half_max(float x) {
  float a, b;
  half_swap(x, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float half_sum(float x) {
  float a, b;
  half_swap(x, a, b);
  return a + b;
}
__device__ __forceinline__ int tile_row(int reg, int half) { return 8 * (reg >> 2) + 4 * half + (reg & 3); }
template <typename T> __device__ __forceinline__ void store4(char* dst, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 2) {
    const bf16x4 w = {(bf16)a, (bf16)b, (bf16)c, (bf16)d};
    *reinterpret_cast<bf16x4*>(dst) = w;
  } else {
    *reinterpret_cast<f32x4*>(dst) = f32x4{a, b, c, d};
  }
}
// Orders this wave's LDS accesses for the compiler (the hardware keeps one wave's in order): what a lane wrote before is
// what the others read after.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// A head-dim-major result tile (columns = rows of dst, this lane's row given; 32 channels from col0) times f, 16 bytes of
// bf16 per store: the two halves of a wave exchange registers so that each lane has 8 consecutive channels.
template <typename T>
__device__ __forceinline__ void store_tile(const Rows& x, const f32x16& a, float f, int col0, int hdb, int lane) {
#pragma unroll
  for (int pair = 0; pair < 2; ++pair) {
    const int off = (col0 + 16 * pair + 8 * (lane >> 5)) * (int)sizeof(T);
    if ((col0 + 16 * pair) * (int)sizeof(T) >= hdb) break;      // (uniform)
    const int at = off < hdb ? (int)(x.at + off) : 0x7FFFFFFF;
    unsigned w[8];
#pragma unroll
    for (int j = 0; j < (sizeof(T) == 2 ? 2 : 4); ++j) {
      unsigned lo, hi;
      if constexpr (sizeof(T) == 2) {
        const bf16x2 l2 = {(bf16)(a[8 * pair + 2 * j] * f), (bf16)(a[8 * pair + 2 * j + 1] * f)};
        const bf16x2 h2 = {(bf16)(a[8 * pair + 4 + 2 * j] * f), (bf16)(a[8 * pair + 5 + 2 * j] * f)};
        lo = __builtin_bit_cast(unsigned, l2);
        hi = __builtin_bit_cast(unsigned, h2);
      } else {
        const float l1 = a[8 * pair + j] * f, h1 = a[8 * pair + 4 + j] * f;
        lo = __builtin_bit_cast(unsigned, l1);
        hi = __builtin_bit_cast(unsigned, h1);
      }
      const auto r = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
      w[j] = r[0];
      w[(sizeof(T) == 2 ? 2 : 4) + j] = r[1];
    }
    __builtin_amdgcn_raw_buffer_store_b128(u32x4{w[0], w[1], w[2], w[3]}, x.r, at, 0, 0);
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b128(u32x4{w[4], w[5], w[6], w[7]}, x.r, at + 16, 0, 0);
  }
}
// Consecutive workgroups go to the eight XCDs in turn; this gives each XCD a contiguous run of logical ids, so that the
// workgroups that share cache lines (the narrow heads of one query block) and keys share an L2.
__device__ __forceinline__ uint32_t xcd_contiguous(uint32_t id, uint32_t n) {
  const uint32_t per = n >> 3;
  return id < per * 8 ? (id & 7) * per + (id >> 3) : id;
}

// A query tile's result (head-dim-major, queries on the lanes) into LDS rows of HDP + 4 floats, one row per query
template <int HDP, int DT>
__device__ __forceinline__ void put_rows(float* rows, const f32x16 (&acc)[DT], int lane) {
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < (HDP < 32 ? 2 : 4); ++i)
      *reinterpret_cast<f32x4*>(rows + (lane & 31) * (HDP + 4) + d * 32 + 8 * i + 4 * (lane >> 5)) =
          f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
}

// ---------------------------------------------------------------- single queries: 16-byte pieces of a row on LPR lanes
template <typename T> __device__ __forceinline__ void widen(u32x4 w, float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {      // bf16 -> fp32: the upper half of the word
      const unsigned lo = w[j] << 16, hi = w[j] & 0xFFFF0000u;
      f[2 * j] = __builtin_bit_cast(float, lo);
      f[2 * j + 1] = __builtin_bit_cast(float, hi);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned x = w[j];
      f[j] = __builtin_bit_cast(float, x);
    }
  }
}

// sum over the LPR lanes of a row, in every one of them: lane exchanges inside the adds (rows of 16 lanes), no LDS
template <int CTRL> __device__ __forceinline__ float dpp_add(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
template <int LPR> __device__ __forceinline__ float row_sum(float x) {
  if (LPR > 1) x = dpp_add<0xB1>(x);       // neighbours
  if (LPR > 2) x = dpp_add<0x4E>(x);       // pairs
  if (LPR > 4) x = dpp_add<0x141>(x);      // mirrored in 8
  if (LPR > 8) x = dpp_add<0x140>(x);      // mirrored in 16
  if (LPR > 16) x += __shfl_xor(x, 16, 64);
  return x;
}

// The samples that use a context, in order: every step is wave- and workgroup-uniform.
struct Samples {
  int b0, b;                  // next sample to look at (a scan position in the index), the present one
  unsigned long long hit;     // samples of the scanned 64 that use the context
  int ctx;
  bool done;
  __device__ __forceinline__ void first(const CrossParams& p, int c, int lane) {
    ctx = c; b0 = 0; b = 0; hit = 0; done = false;
    sample(p, lane);
  }
  __device__ __forceinline__ bool sample(const CrossParams& p, int lane) {
    if (!p.index) {
      if (p.Bc != 1) { b = ctx; done = b0 > 0; b0 = 1; }
      else { b = b0++; done = b >= p.B; }
      return !done;
    }
    while (!hit) {
      if (b0 >= p.B) { done = true; return false; }
      hit = __ballot(b0 + lane < p.B && p.index[min(b0 + lane, p.B - 1)] == ctx);
      b0 += 64;
    }
    b = b0 - 64 + __builtin_ctzll(hit);
    hit &= hit - 1;
    return true;
  }
};

// ---------------------------------------------------------------- host side
inline int cross_hdp(int hd) { return hd <= 16 ? 16 : (hd <= 32 ? 32 : (hd <= 64 ? 64 : (hd <= 96 ? 96 : 128))); }

// contexts that can have a sample at all (a table may hold many more than a batch uses)
inline long cross_used(const dm_cross_args* a) { return a->B < a->Bc ? a->B : a->Bc; }

// waves that share a query tile: with one or two tiles of 32 queries the others would have none
inline int cross_wk(const dm_cross_args* a) { return a->Nq <= 32 ? 4 : (a->Nq <= 64 ? 2 : 1); }
inline long cross_groups(const dm_cross_args* a) { const long per = 32 * (4 / cross_wk(a)); return (a->Nq + per - 1) / per; }

// Key splits in units of workgroups.  With one or two query tiles the keys of a split also fit one image (`image` keys), as
// long as the splits' partial results (`row` bytes per query and head) stay below 1 GiB; beyond, or past MAX_SPLITS images,
// the keys are streamed by workgroups of one wave per query tile.
constexpr int MAX_SPLITS = 64;
inline long cross_splits(const dm_cross_args* a, long blocks, int image, long row) {
  long ns = 1;
  if (blocks < 256 && a->Nk >= 256) {
    ns = (512 + blocks - 1) / blocks;
    if (ns > a->Nk / 128) ns = a->Nk / 128;
  }
  if (cross_wk(a) > 1 && (long)a->Nk > ns * image) {
    const long fit = ((long)a->Nk + image - 1) / image;
    if (fit <= MAX_SPLITS && (double)fit * a->B * a->heads * a->Nq * row <= (double)(1L << 30)) ns = fit;
  }
  return ns < MAX_SPLITS ? ns : MAX_SPLITS;
}

inline bool cross_sizes_ok(const dm_cross_args* a) {
  return a && a->B > 0 && a->Bc > 0 && a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0 && a->Nq > 0 &&
         a->Nk >= 0 && a->hd >= 8 && a->hd <= 128 && a->hd % 8 == 0 && (a->dtype == 0 || a->dtype == 1) &&
         (long)a->B * a->heads * a->Nq < (1L << 40) && a->Nq < (1 << 30) && a->Nk < (1 << 30);
}
inline int cross_fill(CrossParams& p, const dm_cross_args* a, bool bwd) {
  DM_REQUIRE(cross_sizes_ok(a));
  DM_REQUIRE(a->index || a->Bc == a->B || a->Bc == 1);
  DM_REQUIRE(a->q && a->o && a->lse && (a->Nk == 0 || (a->k && a->v)));
  DM_REQUIRE(a->scale > 0.f && a->scale < 1e30f && a->drop_p >= 0.f && a->drop_p < 1.f);
  const long e = a->dtype == 0 ? 2 : 4;
  const long qw = (long)a->heads * a->hd, kw = (long)a->kv_heads * a->hd;
  auto rows_ok = [&](const void* ptr, long ld, long width) {
    return (uintptr_t)ptr % 16 == 0 && ld * e % 16 == 0 && ld >= width && ld * e < (1L << 26);
  };
  DM_REQUIRE(rows_ok(a->q, a->ldq, qw) && rows_ok(a->o, a->ldo, qw));
  DM_REQUIRE(a->Nk == 0 || (rows_ok(a->k, a->ldk, kw) && rows_ok(a->v, a->ldv, kw)));
  if (bwd) {
    DM_REQUIRE(a->d_o && a->dq && rows_ok(a->d_o, a->lddo, qw) && rows_ok(a->dq, a->lddq, qw));
    DM_REQUIRE(a->Nk == 0 || (a->dk && a->dv && rows_ok(a->dk, a->lddk, kw) && rows_ok(a->dv, a->lddv, kw)));
  }
  p.q = (const char*)a->q; p.k = (const char*)a->k; p.v = (const char*)a->v; p.d_o = (const char*)a->d_o;
  p.o = (char*)a->o; p.dq = (char*)a->dq; p.dk = (char*)a->dk; p.dv = (char*)a->dv;
  p.ldq = a->ldq * e; p.ldk = a->ldk * e; p.ldv = a->ldv * e; p.ldo = a->ldo * e;
  p.lddo = a->lddo * e; p.lddq = a->lddq * e; p.lddk = a->lddk * e; p.lddv = a->lddv * e;
  p.lse = a->lse; p.lens = a->lens; p.mask = a->mask; p.index = a->index;
  p.B = a->B; p.Bc = a->Bc; p.H = a->heads; p.G = a->kv_heads; p.Nq = a->Nq; p.Nk = a->Nk; p.hd = a->hd;
  p.scale = a->scale;
  uint32_t t15 = a->drop_p > 0.f ? (uint32_t)((double)a->drop_p * 32768.0 + 0.5) : 0u;   // as dm_attn_fwd
  if (t15 > 32767u) t15 = 32767u;
  p.thresh = 2u * t15;
  p.inv_keep = 32768.f / (32768.f - (float)t15);
  p.seed = dm_seed32(a->drop_seed);
  p.seed_ctr = a->drop_p > 0.f ? dm_dropout_counter() : nullptr;
  return DM_OK;
}

// ---------------------------------------------------------------- the one-kernel backward of few keys (dm_cross_few.hip)
struct FewPlan { int kt, iters, nqb; bool heads, direct; long ws; };
bool few_plan(const dm_cross_args* a, FewPlan& f);          // false: these sizes take the two kernels of dm_cross_bwd.hip
int few_launch(const CrossParams& p, const FewPlan& f, int dtype, hipStream_t st);

// ---------------------------------------------------------------- the forward of single queries (dm_cross_one.hip)
struct OnePlan { int nsplit, ksplit; long ws; };
bool one_plan(const dm_cross_args* a, OnePlan& f);          // false: too many rows share a key / value head
int one_launch(const CrossParams& p, int dtype, hipStream_t st);
int join_launch(const CrossParams& p, int dtype, hipStream_t st);      // joins the key splits of either forward

// ---------------------------------------------------------------- the backward of single queries (dm_cross_onebwd.hip)
struct OneBwdPlan { int tiles; long ws; };                  // workgroups along the states, scratch
bool onebwd_plan(const dm_cross_args* a, OneBwdPlan& f);    // false: too many rows share a key / value head
int onebwd_launch(const CrossParams& p, int dtype, hipStream_t st);
// ---------------------------------------------------------------- the backward of longer row lists (dm_cross_rowsbwd.hip)
bool rowsbwd_plan(const dm_cross_args* a, OneBwdPlan& f);
int rowsbwd_launch(const CrossParams& p, int dtype, hipStream_t st);
int dqsum_launch(const CrossParams& p, int dtype, hipStream_t st);     // adds the p.qsplit partials of dQ

}  // namespace dm_cross
