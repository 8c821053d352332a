// Paged key / value cache (gfx950): write (with quantisation), read back, and attention of a few new tokens over it.
//
// Layout (include/dsrg_hip.h, dsrg_kv_cache_t).  A page holds S tokens of every head; inside (page, head) the keys of 16
// tokens and the values of 32 tokens lie in the order in which an MFMA operand fragment wants them, so that a wave's load of
// one fragment is one contiguous run of 64 x 16 bytes (8-bit codes: 64 x 8) and needs neither LDS nor a transposition:
//   K  [S/16][D/8][16 tokens][8 dims]                    A operand of S^T = K . Q^T: lane (g, r) = token r, dims 32 s + 8 g ..
//   V  [S/32][D/16][4 g][16 dims][2 m][4 i]              A operand of O^T = V^T . P^T: lane (g, d) = dim d, tokens 16 m + 4 g + i
// The second one follows from the first product's result: lane (g, c) holds the scores of query c against tokens 4 g + i of each
// 16-token tile, so two tiles' registers ARE the B operand of the second product if the contraction index runs over the tokens
// in the order (m, i) per g - and V is stored in that order.  fp32 (v_mfma_f32_16x16x4_f32, one token or dim per step and lane
// group): 4-element chunks, K [S/16][D/4][16][4], V [S/16][D/16][4 g][16][4 i].
#include "common.h"
#include <math.h>
#include <algorithm>
#include <type_traits>

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint8_t u8;

namespace {

constexpr float KV_TINY = 1.17549435e-38f;      // smallest scale (2^-126): a row of zeros has it
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

template <int KV> struct KvT;
template <> struct KvT<DSRG_F32> { typedef float type; static constexpr int SZ = 4, E = 4; };
template <> struct KvT<DSRG_BF16> { typedef bf16_t type; static constexpr int SZ = 2, E = 8; };
template <> struct KvT<DSRG_I8> { typedef u8 type; static constexpr int SZ = 1, E = 8; };
template <> struct KvT<DSRG_E4M3> { typedef u8 type; static constexpr int SZ = 1, E = 8; };

struct Pool {
  void* k; void* v; float* ks; float* vs;
  int P, S, lgS, H;
};

// element offset of dim d of token r (within a page's head) in K / V
template <int KV, int D> __device__ __forceinline__ int k_off(int r, int d) {
  constexpr int E = KvT<KV>::E;
  return (r >> 4) * 16 * D + ((d / E) * 16 + (r & 15)) * E + d % E;
}
template <int KV, int D> __device__ __forceinline__ int v_off(int r, int d) {
  if (KvT<KV>::E == 4) return (r >> 4) * 16 * D + (((d >> 4) * 4 + ((r & 15) >> 2)) * 16 + (d & 15)) * 4 + (r & 3);
  return (r >> 5) * 32 * D + (((d >> 4) * 4 + ((r & 15) >> 2)) * 16 + (d & 15)) * 8 + ((r >> 4) & 1) * 4 + (r & 3);
}

// ---- 8-bit codes ---------------------------------------------------------------------------------------------------------
// scale = max(amax * (1 / most), 2^-126), code = round-to-nearest-even(x / scale), clamped (amax / scale can round past `most`).
// A row with a NaN or an infinity has no scale: it gets NaN, so that every value read back from it is NaN, not a wrong number.
template <int KV> __device__ __forceinline__ float kv_scale(float amax, bool finite) {
  const float s = fmaxf(amax * (KV == DSRG_I8 ? (float)(1.0 / 127.0) : (float)(1.0 / 448.0)), KV_TINY);
  return finite ? s : __builtin_nanf("");
}
// x / scale by the row's reciprocal and one correction of the quotient (P. Markstein's scheme: with the reciprocal rounded correctly the
// result is the correctly rounded quotient), 3 instructions an element for the 10 of a division: a prompt's write was bound by them.
struct Divisor { float s, r; };
__device__ __forceinline__ Divisor divisor(float s) {
  const float r = __builtin_amdgcn_rcpf(s);
  return Divisor{s, fmaf(fmaf(-s, r, 1.0f), r, r)};
}
template <int KV> __device__ __forceinline__ float kv_quotient(float x, Divisor d) {
  const float q = x * d.r, y = fmaf(fmaf(-q, d.s, x), d.r, q);
  // |x| <= amax, so |y| is past 127 (448) by less than 2^-21 of it, which rounds back; a row without a scale (y NaN) gets any valid code.  int8:
  // y + 1.5 * 2^23 is rounded to a whole number, whose two's complement is in the low byte.
  if (KV == DSRG_I8) return y + 0x1.8p23f;
  return __builtin_amdgcn_fmed3f(y, -448.f, 448.f);
}
template <int KV> __device__ __forceinline__ float kv_value(unsigned code) {
  if (KV == DSRG_I8) return (float)(int)(int8_t)code;
  return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
}

template <typename T> __device__ __forceinline__ void ld8(const T* p, float (&x)[8]) {      // 16-byte aligned
  const float4 a = ld4(p), b = ld4(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// maximum over the D / 8 lanes (8 or 16, aligned) that hold one row
template <int D> __device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp_mov_f32<0xB1>(v));
  v = fmaxf(v, dpp_mov_f32<0x4E>(v));
  v = fmaxf(v, dpp_mov_f32<0x141>(v));
  if (D == 128) v = fmaxf(v, dpp_mov_f32<0x140>(v));
  return v;
}

// What is stored of 8 dims of a row (its D / 8 lanes call this together), and the row's scale
template <int KV, int D, typename TS> __device__ __forceinline__ void encode(const float (&x)[8], TS (&w)[8], int d0, float* scale, long long at) {
  if constexpr (KvT<KV>::SZ == 1) {
    float m = 0.f;
    bool fin = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) { m = fmaxf(m, fabsf(x[j])); fin = fin && fabsf(x[j]) <= 3.4028235e38f; }
    m = row_max<D>(fin ? m : INFINITY);
    const float s = kv_scale<KV>(m, m <= 3.4028235e38f);
    if (d0 == 0) scale[at] = s;
    const Divisor d = divisor(s);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float y0 = kv_quotient<KV>(x[j], d), y1 = kv_quotient<KV>(x[j + 1], d);
      if (KV == DSRG_I8) { w[j] = (TS)__float_as_uint(y0); w[j + 1] = (TS)__float_as_uint(y1); }
      else { const unsigned c = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y0, y1, 0, false); w[j] = (TS)c; w[j + 1] = (TS)(c >> 8); }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) Elem<TS>::st(&w[j], x[j]);
  }
}

// ---- write ---------------------------------------------------------------------------------------------------------------
struct AppendArgs {
  Pool c;
  const void *k, *v;
  long long k_bs, v_bs;
  int k_rs, v_rs;
  const int32_t *table, *start, *count;
  int table_ld, width, B, T;
};

// D / 8 lanes per (sequence, token, head) row, 8 dims each, K and V of the row by the same lanes.  For few tokens of a sequence: bound by
// the launch (64 tokens of 12 heads of 64: 4.2 us), V's scattered elements do not show.
template <int KV, int D, typename TI>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs a) {
  typedef typename KvT<KV>::type TS;
  constexpr int LPR = D / 8;
  const long long row = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int d0 = (threadIdx.x % LPR) * 8, H = a.c.H;
  if (row >= (long long)a.B * a.T * H) return;          // whole rows leave together: the DPP steps below stay inside a row's lanes
  const int h = (int)(row % H);
  const long long bt = row / H;
  const int b = (int)(bt / a.T), t = (int)(bt % a.T);
  if (a.count && t >= a.count[b]) return;
  const long long pos = (long long)a.start[b] + t;
  if (pos < 0 || pos >= (long long)a.width * a.c.S) return;
  const int page = a.table[(long long)b * a.table_ld + (pos >> a.c.lgS)], r = (int)pos & (a.c.S - 1);
  if (page < 0 || page >= a.c.P) return;
  const long long ph = (long long)page * H + h;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const TI* src = (const TI*)(which ? a.v : a.k) + b * (which ? a.v_bs : a.k_bs) + (long long)t * (which ? a.v_rs : a.k_rs) + h * D + d0;
    float x[8];
    ld8(src, x);
    TS* dst = (TS*)(which ? a.c.v : a.c.k) + ph * a.c.S * D;
    TS w[8];
    encode<KV, D>(x, w, d0, which ? a.c.vs : a.c.ks, ph * a.c.S + r);
    if (which == 0) {
#pragma unroll
      for (int j = 0; j < 8; j += KvT<KV>::E) __builtin_memcpy(__builtin_assume_aligned(dst + k_off<KV, D>(r, d0 + j), KvT<KV>::E * KvT<KV>::SZ), &w[j], KvT<KV>::E * KvT<KV>::SZ);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) dst[v_off<KV, D>(r, d0 + j)] = w[j];
    }
  }
}

// A 32-token block of values on its way between rows and the pool's order: runs of 16 dims (one lane group of one dim tile) lie 16
// (8-bit: 8) bytes further apart than in the pool, so that the lanes of a row write to different LDS banks.
template <int KV, int D> struct VTile {
  static constexpr int E = KvT<KV>::E, RUN = 16 * E, STRIDE = RUN + (KvT<KV>::SZ == 4 ? 4 : 8), SIZE = 32 * D / RUN * STRIDE;
  __device__ static __forceinline__ int at(int off) { return off / RUN * STRIDE + off % RUN; }
};

// Many tokens of a sequence: one workgroup per (sequence, aligned 32-token block, head).  The block's rows are read whole, go through LDS
// into the pool's order and leave as whole chunks; a chunk of 8 (4) tokens that the call covers in part is written element by
// element, so that its other tokens stay.  16.5 thousand tokens of 8 heads of 128, bf16 to int8: 102 MB in 27 us (3.7 TB/s), bound by the
// encoding's instructions beside HBM (35 us with a division an element).
template <int KV, int D, typename TI>
__global__ __launch_bounds__(256) void kv_append_block_kernel(const AppendArgs a) {
  typedef typename KvT<KV>::type TS;
  typedef VTile<KV, D> VT;
  constexpr int LPR = D / 8, RPP = 256 / LPR, E = KvT<KV>::E, SZ = KvT<KV>::SZ;
  __shared__ __attribute__((aligned(16))) TS sk[32 * D];
  __shared__ __attribute__((aligned(16))) TS sv[VT::SIZE];
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const long long start = a.start[b], lo = max(start, 0ll);
  const long long hi = min(start + (a.count ? min(a.count[b], a.T) : a.T), (long long)a.width * a.c.S);
  const long long pos0 = (lo & ~31ll) + 32ll * blockIdx.x;
  if (pos0 >= hi) return;
  const int page = a.table[(long long)b * a.table_ld + (pos0 >> a.c.lgS)];
  if (page < 0 || page >= a.c.P) return;
  const long long ph = (long long)page * a.c.H + h;
  const int in_page = (int)pos0 & (a.c.S - 1);
  const int v0 = (int)max(lo - pos0, 0ll), v1 = (int)min(hi - pos0, 32ll);          // the block's rows that the call writes
  if (v0 >= v1) return;                                                              // (a sequence with nothing to write may start inside a block)
  const int d0 = (tid % LPR) * 8;
  float x[2][32 / RPP][8];
#pragma unroll
  for (int which = 0; which < 2; ++which)              // (every load of the block first)
#pragma unroll
    for (int q = 0; q < 32 / RPP; ++q) {
      const int r = q * RPP + tid / LPR;
      const TI* src = (const TI*)(which ? a.v : a.k) + b * (which ? a.v_bs : a.k_bs) + (pos0 + min(max(r, v0), v1 - 1) - start) * (which ? a.v_rs : a.k_rs) + h * D + d0;
      ld8(src, x[which][q]);
    }
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int q = 0; q < 32 / RPP; ++q) {
      const int r = q * RPP + tid / LPR;
      if (r < v0 || r >= v1) continue;
      TS w[8];
      encode<KV, D>(x[which][q], w, d0, (which ? a.c.vs : a.c.ks), ph * a.c.S + in_page + r);
      if (which == 0) {
#pragma unroll
        for (int j = 0; j < 8; j += E) __builtin_memcpy(__builtin_assume_aligned(sk + k_off<KV, D>(r, d0 + j), E * SZ), &w[j], E * SZ);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) sv[VT::at(v_off<KV, D>(r, d0 + j))] = w[j];
      }
    }
  __syncthreads();
  const unsigned vm = (v1 >= 32 ? ~0u : (1u << v1) - 1) & ~((1u << v0) - 1);
  TS* kd = (TS*)a.c.k + (ph * a.c.S + in_page) * D;
  TS* vd = (TS*)a.c.v + (ph * a.c.S + in_page) * D;
  for (int q = tid; q < 32 * D / E; q += 256) {
    const int r = q / (D / E * 16) * 16 + q % 16;
    if (vm >> r & 1) __builtin_memcpy(__builtin_assume_aligned(kd + q * E, E * SZ), __builtin_assume_aligned(sk + q * E, E * SZ), E * SZ);
    const int g = q / 16 % 4;
    const unsigned m = E == 8 ? (vm >> 4 * g & 15) | (vm >> (16 + 4 * g) & 15) << 4 : vm >> (q / (D * 4) * 16 + 4 * g) & 15;
    const TS* from = sv + VT::at(q * E);
    if (m == (1u << E) - 1) __builtin_memcpy(__builtin_assume_aligned(vd + q * E, E * SZ), __builtin_assume_aligned(from, E * SZ), E * SZ);
    else if (m)
      for (int j = 0; j < E; ++j)
        if (m >> j & 1) vd[q * E + j] = from[j];
  }
}

// ---- read back -----------------------------------------------------------------------------------------------------------
struct ReadArgs {
  Pool c;
  void *k, *v;
  long long k_bs, v_bs;
  int k_rs, v_rs;
  const int32_t *table, *start, *count;
  int table_ld, width, B, N;
};

// One workgroup per (sequence, aligned 32-token block, head): values come as whole chunks and are turned into rows through LDS, a
// key chunk is a piece of a row already.  A row past the sequence's count (or on no page) is zero.  Bound by HBM: 35 thousand rows of 8 heads
// of 128, int8 to bf16, 217 MB in 39 us (5.5 TB/s).
template <int KV, int D, typename TO>
__global__ __launch_bounds__(256) void kv_read_kernel(const ReadArgs a) {
  typedef typename KvT<KV>::type TS;
  typedef VTile<KV, D> VT;
  constexpr int LPR = D / 8, RPP = 256 / LPR, E = KvT<KV>::E, SZ = KvT<KV>::SZ;       // (RPP rows at a time: all 32, or 16)
  __shared__ __attribute__((aligned(16))) TS sv[VT::SIZE];
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const long long start = a.start ? a.start[b] : 0, pos0 = (start & ~31ll) + 32ll * blockIdx.x;
  if (pos0 - start >= a.N) return;
  const int count = min(a.count[b], a.N);
  int page = -1;
  if (pos0 >= 0 && pos0 < (long long)a.width * a.c.S && pos0 - start < count) page = a.table[(long long)b * a.table_ld + (pos0 >> a.c.lgS)];
  const bool there = page >= 0 && page < a.c.P;
  const long long ph = (long long)page * a.c.H + h, row0 = ph * a.c.S + ((int)pos0 & (a.c.S - 1));
  const int d0 = (tid % LPR) * 8;
  TS ek[32 / RPP][8];
  float sc[2][32 / RPP];
  if (there) {                                          // (every load of the block first)
    const TS *ks = (const TS*)a.c.k + row0 * D, *vs = (const TS*)a.c.v + row0 * D;
    TS ev[32 * D / E / 256][E];
#pragma unroll
    for (int q = 0; q < 32 * D / E / 256; ++q) __builtin_memcpy(ev[q], __builtin_assume_aligned(vs + (q * 256 + tid) * E, E * SZ), E * SZ);
#pragma unroll
    for (int q = 0; q < 32 / RPP; ++q) {
      const int r = q * RPP + tid / LPR;
#pragma unroll
      for (int j = 0; j < 8; j += E) __builtin_memcpy(&ek[q][j], __builtin_assume_aligned(ks + k_off<KV, D>(r, d0 + j), E * SZ), E * SZ);
      if constexpr (SZ == 1) { sc[0][q] = a.c.ks[row0 + r]; sc[1][q] = a.c.vs[row0 + r]; }
    }
#pragma unroll
    for (int q = 0; q < 32 * D / E / 256; ++q) __builtin_memcpy(__builtin_assume_aligned(sv + VT::at((q * 256 + tid) * E), E * SZ), ev[q], E * SZ);
    __syncthreads();
  }
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int q = 0; q < 32 / RPP; ++q) {
      const int r = q * RPP + tid / LPR;
      const long long t = pos0 + r - start;
      if (t < 0 || t >= a.N) continue;
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.f;
      if (there && t < count) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const TS e = which ? sv[VT::at(v_off<KV, D>(r, d0 + j))] : ek[q][j];
          if constexpr (SZ == 1) x[j] = kv_value<KV>(e) * sc[which][q];
          else x[j] = Elem<TS>::ld(&e);
        }
      }
      TO* dst = (TO*)(which ? a.v : a.k) + b * (which ? a.v_bs : a.k_bs) + t * (which ? a.v_rs : a.k_rs) + h * D + d0;
      st4(dst, make_float4(x[0], x[1], x[2], x[3]));
      st4(dst + 4, make_float4(x[4], x[5], x[6], x[7]));
    }
}

// ---- attention over the cache ----------------------------------------------------------------------------------------------
//   o[b, i, h] = sum_t softmax_t(scale * q[b, i, h] . k[t, h / G]) v[t, h / G]     over the tokens t that row i sees
// The Nq * G query rows that share a key / value head are the columns of S^T = K . Q^T (16 per MFMA tile; one new token with
// G = 1 fills one of them, which costs nothing: the loop waits for memory).  A wave takes 32 tokens a time: two score tiles,
// the running maximum and sum per column (maximum of a lane's 8 scores, then over the four lane groups; O is rescaled only when a
// maximum rises), P straight from the score registers into the B operand of O^T += V^T . P^T.  Waves share nothing until the end: they
// take blocks in turn and are joined in LDS.  Few sequences: the tokens are also split over workgroups, whose (maximum, sum, O) are joined
// by a second kernel.
// Bound by HBM where there is enough to read: 32 sequences of 1000-32768 tokens, 64 / 8 heads of 128, bf16: 2.21 GB in 430 us (5.15 TB/s; a 4 GiB
// copy moves 4.75); 3 of 40-60 thousand in e4m3: 317 MB in 65 us with the join.  64 of 1-2011 tokens, 12 heads of 64, int8: 105 MB in
// 28 us, the longest first.  One of 200 tokens: 4.5 us, the chain launch - length - page - keys - output.
struct PagedArgs {
  Pool c;
  const void* q; void* o; float* lse;
  long long q_bs, o_bs;
  int q_rs, o_rs;
  const int32_t *table, *lens;
  int table_ld, width, B, nh, G, Nq, NC;       // NC = Nq * G columns per (sequence, key / value head)
  int window, nsplit, bps;                     // bps: 32-token blocks per split
  float sl2;                                   // scale * log2(e)
  float* ws_o; float2* ws_ml;                  // [B, H, NC, nsplit, D], [B, H, NC, nsplit]
};

// maximum / sum over the four lanes (one per 16-lane row) of a column
__device__ __forceinline__ float col_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float col_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

using u32x2 = __attribute__((ext_vector_type(2))) unsigned;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
__device__ __forceinline__ bf16x8 codes_to_bf16(u32x2 u, int kv) {
  bf16x8 r;
  if (kv == DSRG_E4M3) {
    bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.x, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.x, 1.0f, true);
    bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.y, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.y, 1.0f, true);
    r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1]; r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r[j] = (__bf16)(float)((int)(u.x << (24 - 8 * j)) >> 24);
      r[4 + j] = (__bf16)(float)((int)(u.y << (24 - 8 * j)) >> 24);
    }
  }
  return r;
}

// Waves that a SIMD holds: bounded by the registers of O, of the step's keys and values and of the queries.
constexpr int resident(int kv, int D, int CT) {
  return D == 64 ? (CT == 1 ? 4 : 3) - (kv == DSRG_F32) : kv == DSRG_F32 ? 1 : kv != DSRG_BF16 && CT == 1 ? 3 : 2;
}
// Waves of a large workgroup (one column tile): all that a CU holds, so that a sequence's tokens are joined in LDS as far as that goes
constexpr int most_waves(int kv, int D, int CT) { return CT > 1 ? 4 : 4 * resident(kv, D, 1); }
// MIX: the columns see different tokens (causal with several rows); otherwise all see [lo, len) and no per-column bounds are kept.
template <int KV, int D, int CT, int NW, bool MIX, bool LF>
__global__ __launch_bounds__(NW * 64, resident(KV, D, CT)) void attention_paged_kernel(const PagedArgs a) {
  typedef typename KvT<KV>::type TS;
  typedef typename std::conditional<KV == DSRG_F32, float, bf16_t>::type TQ;
  constexpr bool F = KV == DSRG_F32, Q8 = KvT<KV>::SZ == 1;
  constexpr int KS = F ? D / 16 : D / 32;        // 16-byte (8-byte) key chunks of a lane per 16-token tile
  constexpr int DT = D / 16;
  constexpr int OLD = D + 4;
  extern __shared__ __attribute__((aligned(16))) float smem[];               // [NW][nc][OLD], then the waves' maxima and sums [NW][nc] each
  const int nc = min(16, a.NC);
  float* const so = smem;
  float* const sm = so + NW * nc * OLD;
  float* const sl = sm + NW * nc;
  const int lane = threadIdx.x & 63, c16 = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cap = a.width * a.c.S, sp = blockIdx.x, H = a.c.H;
  int y = blockIdx.y, b = blockIdx.z;
  if constexpr (LF) {
    // Several workgroups a CU and sequences of different lengths: the longest sequences' workgroups come first, every second round of 256 the
    // other way round, so that a CU (workgroups go round the 256 in turn) gets long and short ones.  Every wave ranks lens for itself and gets
    // the same answer; where none is long or all are alike that would only cost.  (64 x 12 heads of 64, int8, 1-2011 tokens: 33.2 -> 28.5 us;
    // 64 x 8 heads of 128, bf16, 1-4000: 111 -> 96; all of 2011 tokens, ranked all the same: 43.5 -> 45.1.)
    const int mine = lane < a.B ? min(max(a.lens[lane], 0), cap) : -1;
    const float longest = wave_max((float)mine), shortest = -wave_max(lane < a.B ? -(float)mine : -INFINITY);
    if (longest >= 1024.f && shortest < 0.5f * longest) {
      const unsigned gy = gridDim.y, total = gy * gridDim.z;
      unsigned at = y + gy * b;
      if ((at & 256) && (at | 255) < total) at ^= 255;
      y = at % gy;
      int rank = 0;
      for (int j = 0; j < a.B; ++j) {
        const int o = __builtin_amdgcn_readlane(mine, j);
        rank += o > mine || (o == mine && j < lane);
      }
      b = __builtin_ctzll(__ballot(lane < a.B && rank == (int)(at / gy)));
    }
  }
  const int kh = y % H, cg = y / H;
  const int len = min(max(a.lens[b], 0), cap);
  const int lo_all = a.window ? max(0, len - a.Nq - a.window + 1) : 0;       // first token any row sees
  const int blk0 = lo_all >> 5, blk_end = (len + 31) >> 5;
  const int bbeg = blk0 + sp * a.bps, bend = min(bbeg + a.bps, blk_end);
  if (a.nsplit > 1 && bbeg >= bend) return;                                  // (the joining kernel skips the split as well)

  // queries and what each column sees: [lo, hi)
  int hi[CT], lo[CT];
  using QF = typename std::conditional<F, f32x4, bf16x8>::type;
  QF qf[CT][KS];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int n = (cg * CT + ct) * 16 + c16;
    const bool live = n < a.NC;
    const int i = live ? n / a.G : 0, h = kh * a.G + (live ? n - i * a.G : 0);
    hi[ct] = !MIX ? len : !live ? 0 : max(0, len - a.Nq + i + 1);
    lo[ct] = !MIX ? lo_all : a.window ? max(0, hi[ct] - a.window) : 0;
    const TQ* qp = (const TQ*)a.q + b * a.q_bs + (long long)i * a.q_rs + (long long)h * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if constexpr (F) qf[ct][s] = live ? *reinterpret_cast<const f32x4*>(qp + 16 * s + 4 * g) : f32x4{0.f, 0.f, 0.f, 0.f};
      else {
        const u32x4 u = live ? *reinterpret_cast<const u32x4*>(qp + 32 * s + 8 * g) : u32x4{0, 0, 0, 0};
        qf[ct][s] = __builtin_bit_cast(bf16x8, u);
      }
    }
  }
  // blocks in [full_lo, full_hi) are seen whole by every live column
  const int full_hi = (MIX ? max(0, len - a.Nq + 1) : len) >> 5, full_lo = a.window ? (max(0, len - a.window) + 31) >> 5 : 0;

  f32x4 o[CT][DT];
  float m[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY; l[ct] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[ct][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t* trow = a.table + (long long)b * a.table_ld;
  const int lgB = a.c.lgS - 5, bmask = (1 << lgB) - 1;
  // The compiler's own vectors, not HIP's float4 and uint4: those come apart into scalars that this compiler (ROCm 7.2) has put into registers
  // of tuples that it took for dead (values' second to fourth elements overwritten before their products, in one instantiation for fp32).
  using RF = typename std::conditional<F, f32x4, typename std::conditional<Q8, u32x2, u32x4>::type>::type;
  constexpr int E = KvT<KV>::E, VN = F ? 2 * DT : DT;
  RF kr[2][KS], vr[VN];
  f32x4 ksc[2], vsc[2];
  // Where a step's block lies: its first row in the pools (times D: its elements).  A block on no page is read from page 0 and counts as
  // masked.
  struct Step { long long row0; bool there; };
  auto locate = [&](int blk) {
    Step st;
    const int page = __builtin_amdgcn_readfirstlane(trow[blk >> lgB]);
    st.there = page >= 0 && page < a.c.P;
    st.row0 = ((long long)(st.there ? page : 0) * H + kh) * a.c.S + (blk & bmask) * 32;
    return st;
  };
  auto load_k = [&](const Step& st) {
    const TS* kb = (const TS*)a.c.k + st.row0 * D;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < KS; ++s) kr[t][s] = *reinterpret_cast<const RF*>(kb + t * 16 * D + (s * 64 + lane) * E);
    if constexpr (Q8) {
#pragma unroll
      for (int t = 0; t < 2; ++t) ksc[t] = *reinterpret_cast<const f32x4*>(a.c.ks + st.row0 + 16 * t + 4 * g);
    }
  };
  auto load_v = [&](const Step& st) {
    const TS* vb = (const TS*)a.c.v + st.row0 * D;
    if constexpr (Q8) {
#pragma unroll
      for (int t = 0; t < 2; ++t) vsc[t] = *reinterpret_cast<const f32x4*>(a.c.vs + st.row0 + 16 * t + 4 * g);
    }
#pragma unroll
    for (int dt = 0; dt < VN; ++dt) vr[dt] = *reinterpret_cast<const RF*>(vb + (dt * 64 + lane) * E);
  };

  // The keys of the next step are fetched as soon as this step's are used, the values likewise: a wave always has one of the two in
  // flight and needs no second set of registers.
  int blk = bbeg + w;
  Step cur{}, nxt{};
  if (blk < bend) { cur = locate(blk); load_k(cur); load_v(cur); }
  for (; blk < bend; blk += NW) {
    const bool more = blk + NW < bend;
    if (more) nxt = locate(blk + NW);
    f32x4 s_[CT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) s_[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if constexpr (F) {
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int j = 0; j < 4; ++j) s_[ct][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[t][s][j], qf[ct][s][j], s_[ct][t], 0, 0, 0);
        } else {
          bf16x8 kf;
          if constexpr (Q8) kf = codes_to_bf16(kr[t][s], KV);
          else kf = __builtin_bit_cast(bf16x8, kr[t][s]);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) s_[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[ct][s], s_[ct][t], 0, 0, 0);
        }
      }
    }
    if constexpr (Q8) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s_[ct][t][i] *= ksc[t][i];
    }
    if (more) load_k(nxt);

    const bool full = blk >= full_lo && blk < full_hi && cur.there;
    const int key0 = blk * 32 + 4 * g;
    unsigned vis[CT];                      // MIX and 8 bits: a bit per score of the lane, of a block that is not seen whole
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      vis[ct] = 0;
      if (!full) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 16 * t + i;
            const bool in = cur.there && key < hi[ct] && key >= lo[ct];
            s_[ct][t][i] = in ? s_[ct][t][i] * a.sl2 : -INFINITY;
            if (MIX || Q8) vis[ct] |= in ? 1u << (4 * t + i) : 0u;
          }
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t) s_[ct][t] *= a.sl2;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t) mx = fmaxf(mx, fmaxf(fmaxf(s_[ct][t][0], s_[ct][t][1]), fmaxf(s_[ct][t][2], s_[ct][t][3])));
      const float mn = fmaxf(m[ct], col_max(mx));
      if (__any(mn > m[ct])) {
        const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[ct] - mn);
        l[ct] *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[ct][dt] *= f;
        m[ct] = mn;
      }
      const float mb = m[ct] == -INFINITY ? 0.f : m[ct];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s_[ct][t][i] = __builtin_amdgcn_exp2f(s_[ct][t][i] - mb);
        l[ct] += (s_[ct][t][0] + s_[ct][t][1]) + (s_[ct][t][2] + s_[ct][t][3]);
        if constexpr (Q8) {                // (the scale of what is seen counts, also with a weight of 0: it may be NaN)
#pragma unroll
          for (int i = 0; i < 4; ++i) s_[ct][t][i] = (full || (vis[ct] >> (4 * t + i) & 1)) ? s_[ct][t][i] * vsc[t][i] : 0.f;
        }
      }
    }

    // Tokens that not every column sees may hold anything, and 0 * NaN is NaN: what no column sees is zeroed here, what only some
    // columns see is looked at below (8-bit codes of a written row are finite, and its scale is only taken where it is seen).
    bool odd = false;
    if (!full) {
#pragma unroll
      for (int dt = 0; dt < VN; ++dt)
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const int key = key0 + (F ? 16 * (dt / DT) + j : 16 * (j >> 2) + (j & 3));
          const bool in = cur.there && key < len && key >= lo_all;
          if constexpr (F) {
            const float x = in ? vr[dt][j] : 0.f;
            vr[dt][j] = x;
            if (MIX) odd = odd || !(fabsf(x) <= 3.4028235e38f);
          } else if constexpr (Q8) {
            const unsigned x = vr[dt][j >> 2];
            vr[dt][j >> 2] = in ? x : x & ~(0xffu << (8 * (j & 3)));
          } else {
            const unsigned half = j & 1 ? 0xffff0000u : 0x0000ffffu, x = in ? vr[dt][j >> 1] : vr[dt][j >> 1] & ~half;
            vr[dt][j >> 1] = x;
            if (MIX) odd = odd || (x & half & 0x7f807f80u) == (half & 0x7f807f80u);
          }
        }
    }
    if constexpr (MIX && !Q8) {
      if (__any(odd)) {
        // An infinity or NaN among the values: it leaves V for 0, and three products of 0 / 1 matrices say which columns see a +inf, a -inf or
        // a NaN of a dim, which is what then goes into the sum.
#pragma unroll
        for (int dt = 0; dt < VN; ++dt) {
          float x[E];
#pragma unroll
          for (int j = 0; j < E; ++j) {
            if constexpr (F) x[j] = vr[dt][j];
            else { const unsigned v = vr[dt][j >> 1]; x[j] = __uint_as_float(j & 1 ? v & 0xffff0000u : v << 16); }
          }
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int kind = 0; kind < 3; ++kind) {
              f32x4 r = {0.f, 0.f, 0.f, 0.f};
              auto flag = [&](int j) { return (kind == 0 ? x[j] == INFINITY : kind == 1 ? x[j] == -INFINITY : x[j] != x[j]) ? 1.f : 0.f; };
              if constexpr (F) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  r = __builtin_amdgcn_mfma_f32_16x16x4f32(flag(j), (float)(vis[ct] >> (4 * (dt / DT) + j) & 1), r, 0, 0, 0);
              } else {
                bf16x8 fa, fb;
#pragma unroll
                for (int j = 0; j < 8; ++j) { fa[j] = (__bf16)flag(j); fb[j] = (__bf16)(float)(vis[ct] >> j & 1); }
                r = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa, fb, r, 0, 0, 0);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) o[ct][dt % DT][i] += r[i] > 0.f ? (kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("")) : 0.f;
            }
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (!(fabsf(x[j]) <= 3.4028235e38f)) {
              if constexpr (F) vr[dt][j] = 0.f;
              else vr[dt][j >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
            }
        }
      }
    }
    if constexpr (F) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[t * DT + dt][i], s_[ct][t][i], o[ct][dt], 0, 0, 0);
    } else {
      // P as the sum of two bf16 numbers (16 bits of it): the matrix units wait for memory, and one rounding of P to 8 bits would be as
      // large an error as the output's own
      bf16x8 pf[CT], pl[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = s_[ct][j >> 2][j & 3];
          pf[ct][j] = (__bf16)x;
          pl[ct][j] = (__bf16)(x - (float)pf[ct][j]);
        }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        bf16x8 vf;
        if constexpr (Q8) vf = codes_to_bf16(vr[dt], KV);
        else vf = __builtin_bit_cast(bf16x8, vr[dt]);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[ct], o[ct][dt], 0, 0, 0);
          o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl[ct], o[ct][dt], 0, 0, 0);
        }
      }
    }
    if (more) { load_v(nxt); cur = nxt; }
  }

  // join the waves, one 16-column tile at a time
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int n0 = (cg * CT + ct) * 16, nv = min(16, a.NC - n0);
    if (ct) __syncthreads();
    const float ls = col_sum(l[ct]);
    if (c16 < nv) {
      if (g == 0) { sm[w * nc + c16] = ls == ls ? m[ct] : ls; sl[w * nc + c16] = ls; }          // (all that it saw may be NaN: no maximum)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(so + (w * nc + c16) * OLD + dt * 16 + 4 * g) = o[ct][dt];
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < nv * (D / 4); idx += NW * 64) {
      const int c = idx / (D / 4), d = (idx % (D / 4)) * 4, n = n0 + c;
      float M = -INFINITY;
#pragma unroll
      for (int ww = 0; ww < NW; ++ww) M = fmaxf(M, sm[ww * nc + c]);
      float L = 0.f;
      f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ww = 0; ww < NW; ++ww) {
        // (a factor of 0 is multiplied too: an infinity or NaN among the values that a wave saw shows, whatever they weigh)
        const float mw = sm[ww * nc + c], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M);
        L += f * sl[ww * nc + c];
        O += f * *reinterpret_cast<const f32x4*>(so + (ww * nc + c) * OLD + d);
      }
      if (a.nsplit == 1) {
        const int i = n / a.G, h = kh * a.G + n - i * a.G;
        const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);       // (a NaN sum stays one)
        st4((TQ*)a.o + b * a.o_bs + (long long)i * a.o_rs + (long long)h * D + d, make_float4(O[0] * inv, O[1] * inv, O[2] * inv, O[3] * inv));
        if (a.lse && d == 0) a.lse[((long long)b * a.nh + h) * a.Nq + i] = L == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * LN2;
      } else {
        const long long row = ((long long)b * H + kh) * a.NC + n;
        *reinterpret_cast<f32x4*>(a.ws_o + (row * a.nsplit + sp) * D + d) = O;
        if (d == 0) a.ws_ml[row * a.nsplit + sp] = make_float2(L == L ? M : L, L);
      }
    }
  }
}

// Joins the splits of a row: one wave per row, D / 64 dims a lane.
template <int D, typename TQ>
__global__ __launch_bounds__(256) void attention_paged_join_kernel(const PagedArgs a) {
  const int lane = threadIdx.x & 63, H = a.c.H;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (long long)a.B * H * a.NC) return;
  const int n = (int)(row % a.NC), kh = (int)(row / a.NC % H), b = (int)(row / a.NC / H);
  const int len = min(max(a.lens[b], 0), a.width * a.c.S);
  const int lo_all = a.window ? max(0, len - a.Nq - a.window + 1) : 0;
  const int nb = ((len + 31) >> 5) - (lo_all >> 5);
  const int ns = min(a.nsplit, (nb + a.bps - 1) / a.bps);
  const float2* ml = a.ws_ml + row * a.nsplit;
  float M = -INFINITY;
  for (int s = lane; s < ns; s += 64) M = fmaxf(M, ml[s].x);
  M = wave_max(M);
  float L = 0.f, O[D / 64];
#pragma unroll
  for (int j = 0; j < D / 64; ++j) O[j] = 0.f;
  for (int s0 = 0; s0 < ns; s0 += 64) {
    // lane s has the factor of split s0 + s (0 past the end and for splits that saw nothing); then 8 splits' partial sums at a time, those with
    // a factor of 0 as well (as above)
    const float2 v = s0 + lane < ns ? ml[s0 + lane] : make_float2(-INFINITY, 0.f);
    const float f = v.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - M);
    L += wave_sum(f * v.y);
    const int cnt = min(64, ns - s0);
    for (int s = 0; s < cnt; s += 8) {
      float p[8][D / 64];
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < D / 64; ++j) p[t][j] = a.ws_o[(row * a.nsplit + s0 + min(s + t, cnt - 1)) * D + lane + 64 * j];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const float ft = s + t < cnt ? lane_f32(f, s + t) : 0.f;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) O[j] += s + t < cnt ? ft * p[t][j] : 0.f;
      }
    }
  }
  const int i = n / a.G, h = kh * a.G + n - i * a.G;
  const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);
  TQ* op = (TQ*)a.o + b * a.o_bs + (long long)i * a.o_rs + (long long)h * D;
#pragma unroll
  for (int j = 0; j < D / 64; ++j) Elem<TQ>::st(op + lane + 64 * j, O[j] * inv);
  if (a.lse && lane == 0) a.lse[((long long)b * a.nh + h) * a.Nq + i] = L == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * LN2;
}

// ---- host ----------------------------------------------------------------------------------------------------------------
int check_cache(const dsrg_kv_cache_t* c, const char* who, Pool& p) {
  DSRG_CHECK(c && c->k_pool && c->v_pool, "%s: cache pools are NULL", who);
  DSRG_CHECK(c->dtype == DSRG_F32 || c->dtype == DSRG_BF16 || c->dtype == DSRG_I8 || c->dtype == DSRG_E4M3, "%s: unknown cache dtype %d", who, c->dtype);
  DSRG_CHECK(c->head_dim == 64 || c->head_dim == 128, "%s: head dim %d is not built (64, 128)", who, c->head_dim);
  DSRG_CHECK(c->page_size >= 32 && c->page_size <= 65536 && (c->page_size & (c->page_size - 1)) == 0, "%s: page size %d must be a power of two from 32 to 65536", who, c->page_size);
  DSRG_CHECK(c->n_pages >= 1 && c->n_kv_heads >= 1, "%s: a cache needs pages and heads (%d, %d)", who, c->n_pages, c->n_kv_heads);
  const bool q8 = c->dtype == DSRG_I8 || c->dtype == DSRG_E4M3;
  DSRG_CHECK(q8 == (c->k_scale != nullptr) && q8 == (c->v_scale != nullptr), "%s: 8-bit caches need both scale tables, the others none", who);
  DSRG_CHECK(((uintptr_t)c->k_pool | (uintptr_t)c->v_pool | (uintptr_t)c->k_scale | (uintptr_t)c->v_scale) % 16 == 0, "%s: cache buffers must be 16-byte aligned", who);
  int lg = 5;
  while ((1 << lg) < c->page_size) ++lg;
  p = Pool{c->k_pool, c->v_pool, c->k_scale, c->v_scale, c->n_pages, c->page_size, lg, c->n_kv_heads};
  return DSRG_OK;
}
constexpr long long MAX_TOKENS = 1ll << 30;       // that a table reaches: positions and their differences fit 32 bits
int check_table(const char* who, const int32_t* table, int ld, int width, int S, int B) {
  DSRG_CHECK(table && width >= 1 && (ld >= width || B <= 1) && (long long)width * S <= MAX_TOKENS, "%s: bad page table (width %d, stride %d)", who, width, ld);
  return DSRG_OK;
}
bool rows16(const void* p, long long bs, long long rs, int size) { return (uintptr_t)p % 16 == 0 && bs * size % 16 == 0 && rs * size % 16 == 0; }

struct Split { int nw, nsplit, bps; };
// How many waves share a sequence's tokens (per key / value head and column group): as many as fill the chip's places (1024 SIMDs) about
// once (more than fit would wait for a second round), each with 64 tokens at least; at most 16384 tokens a workgroup, so that one long
// sequence among short ones does not run alone for long.  Waves of a workgroup are joined in LDS, workgroups by a second kernel (4 to 5 us
// more): large workgroups where four waves are not enough, and splits only where one of them is not.  (26 thousand tokens of one sequence, two
// heads of 128: 51 workgroups of 8 waves 14.3 us, 102 of 4 17.4; 16 sequences of up to 999, 12 fp32 heads: one of 12 waves each 17.2 us, 5 of 4
// waves and the join 18.6; 264 workgroups instead of 240 on 256 CUs: 101 us instead of 66 for three sequences of 60 thousand.)
// The tokens are those that the table reaches, since the host knows no lengths: a table much wider than its sequences costs a join and
// leaves waves without work (one of 200 tokens, 12 heads of 64: 4.7 us, in a table of 8192 8.8; 8 of 1000, 8 heads of 128: 10.6 and 20.1; 64 of
// 1-2011 int8 tokens: 24.2, in a table of 32768 44.2).
Split plan_split(int kv, int D, int ct, int B, int H, int cgs, long long max_tokens) {
  const long long blocks = std::max((max_tokens + 31) / 32, 1ll), have = (long long)B * H * cgs, places = 1024ll * resident(kv, D, ct), most = most_waves(kv, D, ct);
  const long long waves = std::max(std::min(places / have, (blocks + 1) / 2), 4ll);
  const long long nw = waves >= 6 ? most : 4;
  long long ns = std::max(waves / nw, (blocks + 511) / 512);
  ns = std::min(std::max(ns, 1ll), 1024ll);
  const long long bps = (blocks + ns - 1) / ns;
  return Split{(int)nw, (int)((blocks + bps - 1) / bps), (int)bps};
}
long long seen_tokens(int width, int S, int Nq, int window) {
  const long long cap = (long long)width * S;
  if (!window || window >= cap) return cap;
  const long long w = (long long)window + Nq - 1 + 31;       // the first block may start up to 31 tokens early
  return w < cap ? w : cap;
}
int col_tiles(int NC) { return NC > 16 ? 2 : 1; }

}  // namespace

template <int KV, int D, int CT, int NW, bool MIX, bool LF = false> static void launch_paged(const PagedArgs& a, dim3 grid, int lds, hipStream_t st) {
  if (NW * 16 * (D + 6) * 4 > 65536) DSRG_SET_MAX_LDS_ONCE((attention_paged_kernel<KV, D, CT, NW, MIX, LF>), NW * 16 * (D + 6) * 4);
  hipLaunchKernelGGL((attention_paged_kernel<KV, D, CT, NW, MIX, LF>), grid, dim3(NW * 64), lds, st, a);
}

#define KV_SWITCH(DT, ...)                                               \
  switch (DT) {                                                          \
    case DSRG_F32: { constexpr int KV = DSRG_F32; __VA_ARGS__; } break;  \
    case DSRG_BF16: { constexpr int KV = DSRG_BF16; __VA_ARGS__; } break;\
    case DSRG_I8: { constexpr int KV = DSRG_I8; __VA_ARGS__; } break;    \
    default: { constexpr int KV = DSRG_E4M3; __VA_ARGS__; } break;       \
  }
#define D_SWITCH(HD, ...)                                \
  if ((HD) == 64) { constexpr int D = 64; __VA_ARGS__; } \
  else { constexpr int D = 128; __VA_ARGS__; }

static int kv_types_ok(const char* who, int kv, int io) {
  DSRG_CHECK(io == DSRG_F32 || io == DSRG_BF16, "%s: unsupported dtype %d", who, io);
  DSRG_CHECK(kv == DSRG_I8 || kv == DSRG_E4M3 || kv == io, "%s: rows of dtype %d for a cache of dtype %d", who, io, kv);
  return DSRG_OK;
}

extern "C" int dsrg_kv_append(const dsrg_kv_cache_t* cache, const void* k, int64_t k_bs, int k_rs, const void* v, int64_t v_bs, int v_rs, int dtype,
                              const int32_t* table, int table_ld, int width, const int32_t* start, const int32_t* count, int B, int T, void* stream) {
  AppendArgs a;
  int rc = check_cache(cache, "dsrg_kv_append", a.c);
  if (rc) return rc;
  if ((rc = kv_types_ok("dsrg_kv_append", cache->dtype, dtype))) return rc;
  if (B == 0 || T == 0) return DSRG_OK;
  DSRG_CHECK(k && v && start && B > 0 && T > 0, "dsrg_kv_append: bad arguments");
  if ((rc = check_table("dsrg_kv_append", table, table_ld, width, a.c.S, B))) return rc;
  const int size = dtype == DSRG_F32 ? 4 : 2;
  DSRG_CHECK(rows16(k, k_bs, k_rs, size) && rows16(v, v_bs, v_rs, size), "dsrg_kv_append: rows must be 16-byte aligned");
  a.k = k; a.v = v; a.k_bs = k_bs; a.v_bs = v_bs; a.k_rs = k_rs; a.v_rs = v_rs;
  a.table = table; a.start = start; a.count = count; a.table_ld = table_ld; a.width = width; a.B = B; a.T = T;
  DSRG_CHECK(B <= 65535 && a.c.H <= 65535, "dsrg_kv_append: %d sequences of %d heads in one call", B, a.c.H);
  // (64 sequences, 12 bf16 heads of 64: T = 1 4.2 us either way, 8 5.6 against 4.4, 32 13.3 against 5.6; 8 int8 heads of 128: T = 1 4.7 by rows against
  // 5.4 by blocks, 4 5.7 against 6.3, 8 7.0 against 6.6)
  const bool rows = T < 8;
  const long long threads = (long long)B * T * a.c.H * (cache->head_dim / 8);
  const dim3 grid = rows ? dim3((unsigned)((threads + 255) / 256)) : dim3((T + 31) / 32 + 1, a.c.H, B), block(256);
  const hipStream_t st = (hipStream_t)stream;
  KV_SWITCH(cache->dtype, D_SWITCH(cache->head_dim, {
    auto go = [&](auto ti) {
      typedef decltype(ti) TI;
      if (rows) hipLaunchKernelGGL((kv_append_kernel<KV, D, TI>), grid, block, 0, st, a);
      else hipLaunchKernelGGL((kv_append_block_kernel<KV, D, TI>), grid, block, 0, st, a);
    };
    if constexpr (KV == DSRG_F32) go(0.f);
    else if constexpr (KV == DSRG_BF16) go((bf16_t)0);
    else if (dtype == DSRG_F32) go(0.f);
    else go((bf16_t)0);
  }))
  DSRG_LAUNCH_CHECK("dsrg_kv_append");
  return DSRG_OK;
}

extern "C" int dsrg_kv_read(const dsrg_kv_cache_t* cache, void* k, int64_t k_bs, int k_rs, void* v, int64_t v_bs, int v_rs, int dtype,
                            const int32_t* table, int table_ld, int width, const int32_t* start, const int32_t* count, int B, int N, void* stream) {
  ReadArgs a;
  int rc = check_cache(cache, "dsrg_kv_read", a.c);
  if (rc) return rc;
  if ((rc = kv_types_ok("dsrg_kv_read", cache->dtype, dtype))) return rc;
  if (B == 0 || N == 0) return DSRG_OK;
  DSRG_CHECK(k && v && count && B > 0 && N > 0, "dsrg_kv_read: bad arguments");
  if ((rc = check_table("dsrg_kv_read", table, table_ld, width, a.c.S, B))) return rc;
  const int size = dtype == DSRG_F32 ? 4 : 2;
  DSRG_CHECK(rows16(k, k_bs, k_rs, size) && rows16(v, v_bs, v_rs, size), "dsrg_kv_read: rows must be 16-byte aligned");
  a.k = k; a.v = v; a.k_bs = k_bs; a.v_bs = v_bs; a.k_rs = k_rs; a.v_rs = v_rs;
  a.table = table; a.start = start; a.count = count; a.table_ld = table_ld; a.width = width; a.B = B; a.N = N;
  DSRG_CHECK(B <= 65535 && a.c.H <= 65535, "dsrg_kv_read: %d sequences of %d heads in one call", B, a.c.H);
  const dim3 grid((N + 31) / 32 + 1, a.c.H, B), block(256);
  KV_SWITCH(cache->dtype, D_SWITCH(cache->head_dim, {
    if constexpr (KV == DSRG_F32) hipLaunchKernelGGL((kv_read_kernel<KV, D, float>), grid, block, 0, (hipStream_t)stream, a);
    else if constexpr (KV == DSRG_BF16) hipLaunchKernelGGL((kv_read_kernel<KV, D, bf16_t>), grid, block, 0, (hipStream_t)stream, a);
    else if (dtype == DSRG_F32) hipLaunchKernelGGL((kv_read_kernel<KV, D, float>), grid, block, 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((kv_read_kernel<KV, D, bf16_t>), grid, block, 0, (hipStream_t)stream, a);
  }))
  DSRG_LAUNCH_CHECK("dsrg_kv_read");
  return DSRG_OK;
}

extern "C" int64_t dsrg_attention_paged_workspace(const dsrg_kv_cache_t* cache, int width, int B, int nh, int Nq, int window) {
  Pool p;
  const int rc = check_cache(cache, "dsrg_attention_paged_workspace", p);
  if (rc) return rc;
  DSRG_CHECK(width >= 1 && B >= 0 && nh >= 1 && nh % p.H == 0 && Nq >= 0 && window >= 0 && (long long)width * p.S <= MAX_TOKENS, "dsrg_attention_paged_workspace: bad arguments");
  if (B == 0 || Nq == 0) return 0;
  const long long NC = (long long)Nq * (nh / p.H);
  DSRG_CHECK(NC <= (1 << 20), "dsrg_attention_paged_workspace: %lld query rows per key / value head", NC);
  const int ct = col_tiles((int)NC), cgs = (int)((NC + 16 * ct - 1) / (16 * ct));
  const Split s = plan_split(cache->dtype, cache->head_dim, ct, B, p.H, cgs, seen_tokens(width, p.S, Nq, window));
  return s.nsplit > 1 ? (int64_t)B * p.H * NC * s.nsplit * (cache->head_dim * 4 + 8) : 0;
}

extern "C" int dsrg_attention_paged(const dsrg_kv_cache_t* cache, const void* q, int64_t q_bs, int q_rs, void* o, int64_t o_bs, int o_rs, float* lse,
                                    const int32_t* table, int table_ld, int width, const int32_t* lens, int B, int nh, int Nq, float scale,
                                    int causal, int window, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  PagedArgs a;
  int rc = check_cache(cache, "dsrg_attention_paged", a.c);
  if (rc) return rc;
  DSRG_CHECK(dtype == (cache->dtype == DSRG_F32 ? DSRG_F32 : DSRG_BF16), "dsrg_attention_paged: queries of dtype %d for a cache of dtype %d", dtype, cache->dtype);
  DSRG_CHECK(nh >= 1 && nh % a.c.H == 0, "dsrg_attention_paged: %d query heads over %d key / value heads", nh, a.c.H);
  DSRG_CHECK(window >= 0 && (causal || !window), "dsrg_attention_paged: a window needs causal = 1 (window %d)", window);
  if (B == 0 || Nq == 0) return DSRG_OK;
  DSRG_CHECK(q && o && lens && B > 0 && B <= 65535 && Nq > 0, "dsrg_attention_paged: bad arguments");
  if ((rc = check_table("dsrg_attention_paged", table, table_ld, width, a.c.S, B))) return rc;
  const int size = dtype == DSRG_F32 ? 4 : 2, D_ = cache->head_dim;
  DSRG_CHECK(rows16(q, q_bs, q_rs, size) && rows16(o, o_bs, o_rs, size), "dsrg_attention_paged: rows must be 16-byte aligned");
  const int64_t need = dsrg_attention_paged_workspace(cache, width, B, nh, Nq, window);
  if (need < 0) return (int)need;
  DSRG_CHECK(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), "dsrg_attention_paged: workspace of %lld bytes needed, %lld given",
             (long long)need, (long long)workspace_bytes);
  a.G = nh / a.c.H;
  a.NC = Nq * a.G;
  const int ct = col_tiles(a.NC), cgs = (a.NC + 16 * ct - 1) / (16 * ct);
  DSRG_CHECK((long long)a.c.H * cgs <= 65535, "dsrg_attention_paged: %d query rows per key / value head", a.NC);
  const Split s = plan_split(cache->dtype, D_, ct, B, a.c.H, cgs, seen_tokens(width, a.c.S, Nq, window));
  a.q = q; a.o = o; a.lse = lse; a.q_bs = q_bs; a.o_bs = o_bs; a.q_rs = q_rs; a.o_rs = o_rs;
  a.table = table; a.lens = lens; a.table_ld = table_ld; a.width = width; a.B = B; a.nh = nh; a.Nq = Nq;
  a.window = window < (long long)width * a.c.S ? window : 0; a.nsplit = s.nsplit; a.bps = s.bps; a.sl2 = scale * LOG2E;
  a.ws_o = (float*)workspace;
  a.ws_ml = need ? (float2*)((float*)workspace + (int64_t)B * a.c.H * a.NC * s.nsplit * D_) : nullptr;
  const long long rows = (long long)B * a.c.H * a.NC;
  DSRG_CHECK(rows < (1ll << 31), "dsrg_attention_paged: %lld query rows", rows);
  const dim3 grid(s.nsplit, a.c.H * cgs, B);
  const hipStream_t st = (hipStream_t)stream;
  const bool mix = causal && Nq > 1;
  // longest sequences first (in an instantiation of its own: it costs other calls 1 to 4 %): long sequences, several workgroups of four waves a CU.
  // One lane ranks a sequence, so 64 at most (of 1-2011 int8 tokens: 64 sequences in this order 24.2 us, 65 in theirs 29.1).
  const bool lf = s.nsplit == 1 && s.nw == 4 && B > 1 && B <= 64 && a.c.H * cgs * B > 256 && !a.window && (long long)width * a.c.S >= 1024;
  KV_SWITCH(cache->dtype, D_SWITCH(D_, {
    constexpr int MW = most_waves(KV, D, 1);
    const int lds = s.nw * std::min(16, a.NC) * (D + 6) * 4;
    auto four = [&](auto tiles, auto mixed, auto first) { launch_paged<KV, D, decltype(tiles)::value, 4, decltype(mixed)::value, decltype(first)::value>(a, grid, lds, st); };
    auto pick = [&](auto tiles) {
      if (lf) mix ? four(tiles, std::true_type(), std::true_type()) : four(tiles, std::false_type(), std::true_type());
      else mix ? four(tiles, std::true_type(), std::false_type()) : four(tiles, std::false_type(), std::false_type());
    };
    if (ct == 2) pick(std::integral_constant<int, 2>());
    else if (s.nw == 4) pick(std::integral_constant<int, 1>());
    else {
      if (mix) launch_paged<KV, D, 1, MW, true>(a, grid, lds, st);
      else launch_paged<KV, D, 1, MW, false>(a, grid, lds, st);
    }
  }))
  DSRG_LAUNCH_CHECK("dsrg_attention_paged");
  if (s.nsplit > 1) {
    const dim3 jgrid((unsigned)((rows + 3) / 4));
    D_SWITCH(D_, {
      if (dtype == DSRG_F32) hipLaunchKernelGGL((attention_paged_join_kernel<D, float>), jgrid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((attention_paged_join_kernel<D, bf16_t>), jgrid, dim3(256), 0, st, a);
    })
    DSRG_LAUNCH_CHECK("dsrg_attention_paged (join)");
  }
  return DSRG_OK;
}
