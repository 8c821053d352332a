// Draw of one entry per row of logits with temperature, top-k, top-p and min-p, from given random numbers (gfx950).
//
// The entries of a row in falling order (equal ones: the lowest index first) are cut three times, and each cut leaves a prefix of
// that order: after the k-th entry; after the first whose running weight reaches p of what the first cut left; where the weight
// falls under m times the largest.  So nothing is sorted: a cut is a threshold on the 64-bit number (value's order-preserving
// bits, ~index), found from a histogram (count or weight per bin of max - x) and the exact ranks inside the one bin that the cut
// falls into.  The draw is the inverse distribution function over what is left, in index order.
// Weights exp((x - max) / T) are fixed-point numbers with 44 bits behind the point, good to 1e-10 of themselves and cut off at 2^-44 of the
// largest (lighter entries weigh nothing): integer sums do not depend on the order of the atomics, and 2^-44 an entry is at most 2^-25 of
// the largest weight a row, half a step of a 24-bit random number.
// One workgroup a row.  Measured (fp32): 256 rows of 30522, k = 60, p = 0.92, m = 0.02: 14.1 us, of which the 31 MB take 5.3 (5.9 TB/s) and the
// rest is one workgroup's chain of barriers; 64 rows of 100 with top-p: 5.5 us, the launch and the same chain; 64 rows of 30522 with
// top-p alone (0.9) 33 us and unfiltered 16.5 us, bound by the weights' instructions (one or two weights an entry, 29 instructions each) on 64
// CUs; rows of 131072, read again by every pass: 55 us unfiltered and 124 us with top-p for one row, 58 and 129 for 64.
#include "common.h"
#include <math.h>

typedef unsigned long long u64;

namespace {

constexpr int WBITS = 44;

struct SampleArgs {
  const void* logits;
  long long ld;
  const float* u;
  const float* temp; const int32_t* topk; const float* topp; const float* minp;      // NULL: the number beside it
  float temp0; int topk0; float topp0, minp0;
  int64_t* token; float* logp;
  int V;
};

__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ u64 comp_of(float x, int j) { return ((u64)key_of(x) << 32) | (unsigned)~j; }

__constant__ const double EXP2_A[32] = {       // 2^(k / 32)
    1, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
    1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832, 1.4142135623730951, 1.4451808069770467,
    1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543,
    1.6457554781539649, 1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424,
    1.8741676341103, 1.9152065613971474, 1.9571441241754002};
__constant__ const double EXP2_B[32] = {       // 2^(k / 1024)
    1, 1.0006771306930664, 1.0013547198921082, 1.002032767907594, 1.0027112750502025, 1.0033902416308227,
    1.0040696679605541, 1.0047495543507072, 1.0054299011128027, 1.006110708558573, 1.0067919769999607, 1.0074737067491204,
    1.0081558981184175, 1.0088385514204294, 1.0095216669679448, 1.0102052450739643, 1.0108892860517005,
    1.0115737902145781, 1.0122587578762337, 1.0129441893505169, 1.0136300849514894, 1.0143164449934257,
    1.0150032697908125, 1.0156905596583505, 1.0163783149109531, 1.0170665358637463, 1.0177552228320703,
    1.0184443761314785, 1.0191339960777379, 1.0198240829868295, 1.0205146371749483, 1.0212056589585028};
// 2^(k / 1024) as a fixed-point number with 62 bits behind the point
__device__ __forceinline__ u64 exp2_table(int k) {
  const u64 bits = (u64)__double_as_longlong(EXP2_A[k >> 5] * EXP2_B[k & 31]);
  return ((bits & 0xfffffffffffffull) | 0x10000000000000ull) << 10;
}

// 2^(t / 1024) in WBITS-bit fixed point for t <= 0.  With k the whole number next to t, 2^(k / 1024) comes from the table and a shift, and
// e^y, |y| <= ln2 / 2048, is 1 + (y + y^2 / 2): the first term left out is y^3 / 6 < 7e-12, and the bracket, 2^-11 of the result at most, is
// fine in fp32 (2^-35 of it).  Adding 1.5 * 2^52 leaves k in the low word.
__device__ __forceinline__ u64 fixed_exp2(double t, const u64* tab) {
  constexpr double MAGIC = 0x1.8p52;
  t = fmax(t, -65536.0);
  const double kk = t + MAGIC;
  const int k = (int)(unsigned)(u64)__double_as_longlong(kk);
  const float y = (float)(t - (kk - MAGIC)) * (float)(0.69314718055994530942 / 1024);
  const u64 T = tab[k & 1023];
  const float more = fmaf(y * 0.5f, y, y) * ((float)(unsigned)(T >> 32) * 256.f);        // in units of 2^24
  return (u64)((long long)T + ((long long)(int)more << 24)) >> min(62 - WBITS - (k >> 10), 63);
}

template <int CTRL> __device__ __forceinline__ u64 dpp_u64(u64 v) {
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, 0xF, 0xF, true);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, 0xF, 0xF, true);
  return (u64)hi << 32 | lo;
}
// sum over the 16 lanes of a DPP row, in all of them
__device__ __forceinline__ u64 row_sum_u64(u64 v) {
  v += dpp_u64<0xB1>(v);
  v += dpp_u64<0x4E>(v);
  v += dpp_u64<0x141>(v);
  return v + dpp_u64<0x140>(v);
}
__device__ __forceinline__ u64 lane_u64(u64 v, int l) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), l) << 32 | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, l);
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
  v = row_sum_u64(v);
  return (lane_u64(v, 0) + lane_u64(v, 16)) + (lane_u64(v, 32) + lane_u64(v, 48));
}
// inclusive running sum over the wave
__device__ __forceinline__ unsigned wave_scan_u32(unsigned v) {
#define DSRG_STEP(ctrl, rows) v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xF, true)
  DSRG_STEP(0x111, 0xF);      // row_shr 1, 2, 4, 8: inside the rows of 16
  DSRG_STEP(0x112, 0xF);
  DSRG_STEP(0x114, 0xF);
  DSRG_STEP(0x118, 0xF);
  DSRG_STEP(0x142, 0xA);      // row_bcast 15: rows 1 and 3 get what rows 0 and 2 end with
  DSRG_STEP(0x143, 0xC);      // row_bcast 31: rows 2 and 3 get what row 1 ends with
#undef DSRG_STEP
  return v;
}

__device__ __forceinline__ u64 wave_scan_u64(u64 v) {
#define DSRG_STEP(ctrl, rows)                                                                                  \
  v += (u64)(unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), ctrl, rows, 0xF, true) << 32 |  \
       (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, ctrl, rows, 0xF, true)
  DSRG_STEP(0x111, 0xF);
  DSRG_STEP(0x112, 0xF);
  DSRG_STEP(0x114, 0xF);
  DSRG_STEP(0x118, 0xF);
  DSRG_STEP(0x142, 0xA);
  DSRG_STEP(0x143, 0xC);
#undef DSRG_STEP
  return v;
}

// -0 + 0 = +0: the two zeros are one value; NaN is no candidate
__device__ __forceinline__ float candidate(float x) { return fmaxf(x + 0.0f, -INFINITY); }
template <typename T> __device__ __forceinline__ float load_logit(const T* row, int j) { return candidate(Elem<T>::ld(row + j)); }
// A row through a buffer descriptor: what lies past the row is not read (it is 0) without a comparison a load.  The whole position goes into the
// lane's offset, which is what the hardware compares with the row's size: a scalar offset is no certain part of that, and could pass the
// size by itself.  One addition a load at most, neighbouring loads share theirs (constants fold into the instruction).
template <typename T> struct RowBuffer {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ RowBuffer(const T* row, int V) : r(__builtin_amdgcn_make_buffer_rsrc((void*)row, 0, V * (int)sizeof(T), 0x00027000)) {}
  __device__ __forceinline__ T raw(int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, j * 4, 0, 0));
    else return __builtin_amdgcn_raw_buffer_load_b16(r, j * 2, 0, 0);
  }
};

// Where the row is: VPT > 0: a thread holds VPT values of it in registers (64 rows of 30522: unfiltered 18.3 -> 17.2 us, top-p 37.7 ->
// 35.9 against reading them again); longer rows, and the passes that only crowded bins need, read the row from the cache, eight independent loads
// at a time.
template <typename T, int NT, int NB, int VPT>
__global__ __launch_bounds__(NT) void sample_rows_kernel(const SampleArgs a) {
  constexpr int NW = NT / 64, BPT = NB / NT;            // bins per thread
  __shared__ u64 mass[NB];
  __shared__ unsigned cnt[NB];
  // Ranks cost n^2 / NT: entries of a cut's bin that are ranked directly (more: by the bits of their values), candidates of the short way, the
  // k that goes there, and what a long way's end ranks.
  constexpr int LIST = NT == 1024 ? 512 : 256, FEW = 3 * NT / 8, SHORT = NT / 4;
  __shared__ ulonglong2 list[LIST];                     // (comp, weight)
  u64* const l_ahead = mass;                            // (the short way has no use for the bins' weights)
  unsigned* const l_rank = cnt;
  static_assert(NB >= LIST, "one word an entry");
  __shared__ u64 tab[1024];
  __shared__ u64 red_a[NW], red_b[NW];
  __shared__ float s_max[NW];
  __shared__ double s_c2, s_tlogm;
  __shared__ u64 s_thr, s_base, s_bin_v;
  __shared__ unsigned s_bin, s_n;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), b = blockIdx.x, V = a.V;
  const T* row = (const T*)a.logits + (long long)b * a.ld;
  const float Tm = a.temp ? a.temp[b] : a.temp0, P = a.topp ? a.topp[b] : a.topp0, M = a.minp ? a.minp[b] : a.minp0;
  const int Kk = a.topk ? a.topk[b] : a.topk0;
  const float u_raw = a.u[b], uu = u_raw >= 0.f ? fminf(u_raw, 0.99999994f) : 0.f;
  // wave w's part of the row: index order is (wave, step, lane)
  const int seg = (V + NW * 64 - 1) / (NW * 64) * 64, j0 = min(V, w * seg), j1 = min(V, j0 + seg);

  // f(value, index) for this thread's share of the row; -inf stands for what is no candidate
  const RowBuffer<T> buf(row, V);
  auto again = [&](auto&& f) {
    for (int jb = j0; jb < j1; jb += 512) {
      T x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = buf.raw(jb + lane + i * 64);
#pragma unroll
      for (int i = 0; i < 8; ++i) f(jb + i * 64 + lane < j1 ? candidate(Elem<T>::ld(&x[i])) : -INFINITY, jb + i * 64 + lane);
    }
  };
  auto constants = [&] {                                // (while the row is on its way)
    for (int k = tid; k < 1024; k += NT) tab[k] = exp2_table(k);
    if (tid == NT - 1) {
      s_c2 = 1024 * 1.44269504088896340736 / (double)Tm;
      s_tlogm = M > 0.f && Tm < INFINITY ? (double)Tm * log((double)M) : -INFINITY;      // (T infinite: all weigh 1)
    }
  };
  float xs[VPT ? VPT : 1];
  if constexpr (VPT > 0) {
    T x[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) x[i] = buf.raw(j0 + lane + i * 64);
    constants();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      xs[i] = candidate(Elem<T>::ld(&x[i]));
      if (j0 + i * 64 + 64 > j1) xs[i] = j0 + i * 64 + lane < j1 ? xs[i] : -INFINITY;
    }
  } else constants();
  auto each = [&](auto&& f) {
    if constexpr (VPT > 0) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) f(xs[i], j0 + i * 64 + lane);
    } else again(f);
  };

  // largest value
  float tmax = -INFINITY;
  each([&](float x, int) { tmax = fmaxf(tmax, x); });
  const float wmax = wave_max(tmax);
  if (lane == 0) s_max[w] = wmax;
  __syncthreads();
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < NW; ++i) mx = fmaxf(mx, s_max[i]);
  if (mx == -INFINITY) {                                // nothing to draw from
    if (tid == 0) { a.token[b] = -1; a.logp[b] = -INFINITY; }
    return;
  }
  if (!(Tm > 0.f)) {                                    // greedy: the lowest index of the largest value
    if (tid == 0) s_n = 0x7fffffff;
    __syncthreads();
    each([&](float x, int j) { if (x == mx) atomicMin(&s_n, (unsigned)j); });
    __syncthreads();
    if (tid == 0) { a.token[b] = (int)s_n; a.logp[b] = 0.f; }
    return;
  }
  const double c2 = s_c2, floor_ = (double)mx + s_tlogm;          // w >= m  <=>  x >= max + T ln m
  auto weight = [&](float x) -> u64 { return x == mx ? (u64)1 << WBITS : fixed_exp2(((double)x - (double)mx) * c2, tab); };
  auto logp_of = [&](float x, u64 total) -> float {
    return (float)((x == mx ? 0.0 : ((double)x - (double)mx) / (double)Tm) - log(ldexp((double)total, -WBITS)));
  };
  // bins of max - x: its float bits from 2^-8 to 2^8, NB / 16 an octave (monotone in x, whatever the logits' spread)
  constexpr int SH = 23 - (NB == 4096 ? 8 : 6);
  static_assert(NB == 4096 || NB == 1024, "NB / 16 bins an octave");
  auto bin_of = [&](float x) -> unsigned {
    const unsigned d = x == mx ? 0u : __float_as_uint(mx - x) >> SH;
    const unsigned lo = 0x3b800000u >> SH;              // 2^-8
    return d < lo ? 0u : min(d - lo, (unsigned)NB - 1);
  };

  // For every entry of the list: what the entries weigh for which `ahead(other, me)` holds, and how many they are.  The 16 lanes of a DPP row
  // walk the list together for an entry (or two).
  auto ranked = [&](int n, auto&& ahead, auto&& f) {
    constexpr int EB = NT == 1024 ? 1 : 2;
    const int sub = tid & 15;
    for (int i0 = 0; i0 < n; i0 += NT / 16 * EB) {
      const int i1 = i0 + (tid >> 4) * EB;
      if (__builtin_amdgcn_readfirstlane(i1) >= n) break;                // (the wave's lowest entry)
      ulonglong2 me[EB];
      unsigned c[EB];
      u64 m[EB];
#pragma unroll
      for (int e = 0; e < EB; ++e) { me[e] = list[min(i1 + e, n - 1)]; c[e] = 0; m[e] = 0; }
#pragma unroll 2
      for (int k = sub; k < n; k += 16) {
        const ulonglong2 o = list[k];
#pragma unroll
        for (int e = 0; e < EB; ++e) {
          const bool up = ahead(o, me[e]);
          c[e] += up;
          m[e] += up ? o.y : 0;
        }
      }
#pragma unroll
      for (int e = 0; e < EB; ++e) {
        const unsigned cs = (unsigned)row_sum_u64(c[e]);
        const u64 ms = row_sum_u64(m[e]);
        if (sub == e && i1 + e < n) f(i1 + e, me[e], cs, ms);
      }
    }
  };
  auto larger = [](const ulonglong2& o, const ulonglong2& me) { return o.x > me.x; };
  auto clear = [&](bool by_mass) {
    for (int i = tid; i < NB; i += NT)
      if (by_mass) mass[i] = 0; else cnt[i] = 0;
  };
  auto put = [&](bool by_mass, unsigned bin, float x) {
    if (by_mass) atomicAdd(&mass[bin], weight(x)); else atomicAdd(&cnt[bin], 1u);
  };
  // Running sum over the bins (of counts or of weights), behind what lies before them; the first bin at which it reaches the goal goes to
  // s_bin, with what lies before it.  *goal < 0: it is frac of the whole.  By weight the first entry is inside whatever the goal (it weighs
  // most; nothing weighs anything before it), and a bin whose weights all rounded to 0 never reaches one.
  auto locate = [&](bool by_mass, u64 want, double frac, u64 before, double* goal) {
    u64 t = 0;
#pragma unroll
    for (int i = 0; i < BPT; ++i) t += by_mass ? mass[tid * BPT + i] : cnt[tid * BPT + i];
    u64 inc = by_mass ? wave_scan_u64(t) : wave_scan_u32((unsigned)t);
    if (lane == 63) red_a[w] = inc;
    __syncthreads();
    u64 total = 0;
    inc += before;
#pragma unroll
    for (int i = 0; i < NW; ++i) { inc += i < w ? red_a[i] : 0; total += red_a[i]; }
    u64 ex = inc - t;
    if (*goal < 0) *goal = fmax(frac, 0.0) * (double)total;
    auto reached = [&](u64 v) { return by_mass ? (double)v >= *goal && v : v >= want; };
    if (t && !reached(ex) && reached(inc)) {
      bool done = false;
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        const u64 v = by_mass ? mass[tid * BPT + i] : cnt[tid * BPT + i];
        if (!done && reached(ex + v)) { done = true; s_bin = tid * BPT + i; s_base = ex; s_bin_v = v; }
        ex += v;
      }
    }
    __syncthreads();
  };
  u64 thr = 0;                                          // entries with comp >= thr are kept (comp of a valid entry is never 0)
  // One cut: by_mass false: after `want` entries; true: after the first whose running weight reaches frac of the whole.
  auto cut = [&](bool by_mass, u64 want, double frac) {
    double goal = -1.0;
    clear(by_mass);
    if (tid == 0) { s_thr = ~0ull; s_n = 0; }
    __syncthreads();
    each([&](float x, int j) {
      if (x > -INFINITY && comp_of(x, j) >= thr) put(by_mass, bin_of(x), x);
    });
    __syncthreads();
    locate(by_mass, want, frac, 0, &goal);
    const unsigned bin = s_bin;
    u64 base = s_base;
    // the bin's entries: values between its edges, widened a little for the rounding of max - x, then looked at exactly
    constexpr unsigned BLO = 0x3b800000u >> SH;
    const double e0 = bin ? (double)__uint_as_float((bin + BLO) << SH) : 0.0, e1 = bin < NB - 1 ? (double)__uint_as_float((bin + BLO + 1) << SH) : INFINITY;
    const double slack = fabs((double)mx) * 0x1p-22, top = (double)mx - e0 * (1.0 - 0x1p-22) + slack, bottom = (double)mx - e1 * (1.0 + 0x1p-22) - slack;
    const float vtop = top < 3.4e38 ? (float)top : INFINITY, vbottom = bottom > -3.4e38 ? (float)bottom : -3.4028235e38f;
    const bool exact_only = !(fabs((double)mx) < 3e38);
    // its parts: NB of equal width (the last bin, from 256 on: by the first bits of max - x)
    const unsigned part_lo = (bin + BLO) << SH, part_sh = bin < NB - 1 ? SH - (NB == 4096 ? 12 : 10) : NB == 4096 ? 18 : 20;
    auto part_of = [&](float x) -> unsigned {
      const float d = x == mx ? 0.f : mx - x;
      return bin ? (__float_as_uint(d) - part_lo) >> part_sh : (unsigned)(d * (NB * (NB == 4096 ? 255.f : 252.f)));      // (bin 0 ends at 2^-8 times 1 + 16 / NB)
    };
    int part = -1;                                        // (all of them)
    auto gather = [&] {
      each([&](float x, int j) {
        if ((exact_only ? x > -INFINITY : x >= vbottom && x <= vtop) && bin_of(x) == bin && (part < 0 || part_of(x) == (unsigned)part) && comp_of(x, j) >= thr) {
          const unsigned at = atomicAdd(&s_n, 1u);
          if (at < LIST) list[at].x = comp_of(x, j);
        }
      });
      __syncthreads();
      return (int)s_n;
    };
    int n = gather();
    const u64 bin_base = base;
    if (n > LIST) {
      // more than are ranked: the same once more over the bin's parts (64 rows of 30522 entries of which the cut falls among 30 thousand within 0.01:
      // 119 us without, 74 with; where they are all equal the way below is taken all the same: 147 and 184)
      __syncthreads();
      clear(by_mass);
      if (tid == 0) s_n = 0;
      __syncthreads();
      again([&](float x, int j) {
        if (x > -INFINITY && bin_of(x) == bin && comp_of(x, j) >= thr) put(by_mass, part_of(x), x);
      });
      __syncthreads();
      locate(by_mass, want, frac, base, &goal);
      part = (int)s_bin;
      base = s_base;
      n = gather();
    }
    if (n <= LIST) {
      for (int i = tid; i < n; i += NT) list[i].y = by_mass ? weight(of_key((unsigned)(list[i].x >> 32))) : 1;
      __syncthreads();
      ranked(n, larger, [&](int, const ulonglong2& me, unsigned, u64 m) {
        const u64 ahead = base + m;
        if (by_mass ? (double)ahead < goal || ahead == 0 : ahead < want) atomicMin(&s_thr, me.x);
      });
      __syncthreads();
      thr = s_thr;
    } else {
      // still many (equal values): by the value's 32 bits, LB of them a pass
      base = bin_base;
      __syncthreads();
      constexpr int LB = NB == 4096 ? 12 : 10;
      unsigned prefix = 0, pmask = 0;
      for (int sh = 32; sh > 0;) {
        const int nb = min(LB, sh);
        sh -= nb;
        clear(by_mass);
        __syncthreads();
        again([&](float x, int j) {
          const unsigned k = key_of(x);
          if (x > -INFINITY && comp_of(x, j) >= thr && bin_of(x) == bin && (k & pmask) == prefix) put(by_mass, ~(k >> sh) & ((1u << nb) - 1), x);       // falling values
        });
        __syncthreads();
        locate(by_mass, want, frac, base, &goal);
        base = s_base;
        prefix |= (~s_bin & ((1u << nb) - 1)) << sh;
        pmask |= ((1u << nb) - 1) << sh;
        __syncthreads();
      }
      // what is left are equal values: as many of them as the goal asks, the lowest indices first
      const u64 one = by_mass ? weight(of_key(prefix)) : 1, ties = s_bin_v / one;
      u64 r;
      if (by_mass) {
        const double left = goal - (double)base;
        r = left > 0 ? (u64)ceil(left / (double)one) : 1;
        while (r > 1 && (double)(base + (r - 1) * one) >= goal) --r;
        while ((double)(base + r * one) < goal && r < ties) ++r;
      } else r = want - base;
      r = r < 1 ? 1 : r > ties ? ties : r;
      unsigned mine = 0;
      for (int j = j0 + lane; j - lane < j1; j += 64) mine += __popcll(__ballot(j < j1 && key_of(load_logit(row, j < V ? j : V - 1)) == prefix));
      if (lane == 0) red_a[w] = mine;
      __syncthreads();
      u64 before = 0;
      for (int i = 0; i < w; ++i) before += red_a[i];
      if (before < r && before + mine >= r) {           // this wave holds the r-th of them
        u64 left = r - before;
        for (int j = j0 + lane; j - lane < j1; j += 64) {
          const u64 hit = __ballot(j < j1 && key_of(load_logit(row, j < V ? j : V - 1)) == prefix);
          const u64 n = __popcll(hit);
          if (left <= n) {
            if ((hit >> lane & 1) && __popcll(hit & (((u64)1 << lane) - 1)) == left - 1) s_thr = ((u64)prefix << 32) | (unsigned)~j;
            break;
          }
          left -= n;
        }
      }
      __syncthreads();
      thr = s_thr;
    }
    __syncthreads();
  };

  // The rest, once the list holds everything that can still be drawn (s_n entries, weights not yet filled in): the first `want`, of them
  // what top-p keeps (p >= 1: all), of them what min-p keeps, and the draw.
  auto draw_from_list = [&](unsigned want, float p) {
    const int n = (int)s_n;
    auto value = [&](u64 comp) { return of_key((unsigned)(comp >> 32)); };
    for (int i = tid; i < n; i += NT) list[i].y = weight(value(list[i].x));
    __syncthreads();
    // rank and the weight ahead of every entry; what the first `want` weigh (only top-p asks for it)
    u64 sum = 0;
    const bool cuts = want < (unsigned)n || p < 1.f;
    double goal = 0.0;
    if (cuts) {
      ranked(n, larger, [&](int i, const ulonglong2& me, unsigned c, u64 m) {
        l_rank[i] = c;
        l_ahead[i] = m;
        if (c < want) sum += me.y;
      });
      sum = wave_sum_u64(sum);
      if (lane == 0) red_a[w] = sum;
      __syncthreads();
      u64 all = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) all += red_a[i];
      goal = fmax((double)p, 0.0) * (double)all;
      sum = 0;
    }
    for (int i = tid; i < n; i += NT) {                 // what is not kept loses its weight: it is not drawn then
      const ulonglong2 me = list[i];
      const float x = value(me.x);
      // (without cuts all entries are among the first `want`, and the largest stays by min-p)
      const unsigned rank = cuts ? l_rank[i] : 0u;
      const bool first = cuts && rank == 0, in = rank < want && (!(p < 1.f) || (double)l_ahead[i] < goal);
      const bool keep = first || (in && (x == mx || (double)x >= floor_));
      if (keep) sum += me.y; else list[i].y = 0;
    }
    sum = wave_sum_u64(sum);
    if (lane == 0) red_b[w] = sum;
    __syncthreads();
    u64 total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) total += red_b[i];
    const double draw = (double)uu * (double)total;
    if constexpr (VPT == 1) {                           // the list is in index order, an entry a thread
      const u64 own = tid < n ? list[tid].y : 0;
      u64 c = wave_scan_u64(own);
      if (lane == 63) red_a[w] = c;
      __syncthreads();
      c -= own;
#pragma unroll
      for (int i = 0; i < NW; ++i) c += i < w ? red_a[i] : 0;
      if (own && (double)c <= draw && (double)(c + own) > draw) { a.token[b] = (int)~(unsigned)list[tid].x; a.logp[b] = logp_of(value(list[tid].x), total); }
    } else {
      // (the low word is ~index: the entries before have a larger one)
      ranked(n, [](const ulonglong2& o, const ulonglong2& me) { return (unsigned)o.x > (unsigned)me.x; }, [&](int, const ulonglong2& me, unsigned, u64 m) {
        if (me.y && (double)m <= draw && (double)(m + me.y) > draw) { a.token[b] = (int)~(unsigned)me.x; a.logp[b] = logp_of(value(me.x), total); }
      });
    }
  };

  // The short way: everything that can be drawn fits a list.  Short rows: all of them (measured, 64 rows with top-p: V = 100 6.9 us against 8.8
  // the long way, 170 the same, 256 12.1 against 9.3).  Top-k with a small k: the k-th largest of the threads' largest entries is no larger
  // than the k-th largest of all, so the entries of its bin and above hold the k wanted ones, and few others (256 rows of 30522: k = 60 11.7 us
  // against 28.5, k = 256 25.5 against 34.8, k = 400 50.9 against 38.5).  One bin a thread here (NT / 16 an octave): coarser ones cost a few
  // entries more, a longer scan more time.
  const bool small = VPT == 1, few = Kk > 0 && Kk <= SHORT;
  if (small || few) {
    float lim = -3.4028235e38f;                         // entries from here on (every candidate: -inf and NaN are none)
    if (tid == 0) s_n = 0;
    if (!small) {
      constexpr int SN = 23 - (NT == 1024 ? 6 : 4);
      static_assert(NT == 1024 || NT == 256, "NT / 16 bins an octave");
      constexpr unsigned lo = 0x3b800000u >> SN;
      cnt[tid] = 0;
      if (tid == 0) s_bin = NT;                         // (fewer than k threads have an entry at all: everything)
      __syncthreads();
      if (tmax > -INFINITY) {
        const unsigned d = __float_as_uint(mx == tmax ? 0.f : mx - tmax) >> SN;
        atomicAdd(&cnt[d < lo ? 0u : min(d - lo, (unsigned)NT - 1)], 1u);
      }
      __syncthreads();
      const unsigned tc = cnt[tid];
      unsigned ic = wave_scan_u32(tc);
      if (lane == 63) red_b[w] = ic;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NW; ++i) ic += i < w ? (unsigned)red_b[i] : 0u;
      if (ic >= (unsigned)Kk && ic - tc < (unsigned)Kk) s_bin = tid;
      __syncthreads();
      const unsigned last = s_bin;
      // fl(max - x) < edge means max - x < edge (1 + 2^-24): all of those are above this, rounded down by 2^-22 of edge and of the result
      if (last < NT - 1) {
        const double edge = __uint_as_float((last + lo + 1) << SN), at = (double)mx - edge * (1.0 + 0x1p-22);
        lim = fmaxf((float)(at - fabs(at) * 0x1p-22), lim);
      }
    }
    if constexpr (VPT == 1) {                           // packed in index order
      const bool in = xs[0] > -INFINITY;
      const u64 hit = __ballot(in);
      if (lane == 0) red_a[w] = __popcll(hit);
      __syncthreads();
      unsigned at = __popcll(hit & (((u64)1 << lane) - 1)), all = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) { at += i < w ? (unsigned)red_a[i] : 0u; all += (unsigned)red_a[i]; }
      if (in) list[at].x = comp_of(xs[0], j0 + lane);
      if (tid == 0) s_n = all;
    } else {
      if constexpr (VPT >= 8) {                         // counted first: one atomic a wave
        unsigned mine = 0;
        each([&](float x, int) { mine += x >= lim; });
        const unsigned upto = wave_scan_u32(mine), total = (unsigned)__builtin_amdgcn_readlane((int)upto, 63);
        if (total) {
          unsigned at = 0;
          if (lane == 0) at = atomicAdd(&s_n, total);
          at = (unsigned)__builtin_amdgcn_readfirstlane((int)at) + upto - mine;
#pragma unroll
          for (int i = 0; i < VPT; i += 8) {            // (one test for eight: few of a wave's 512 are taken)
            float m = xs[i];
#pragma unroll
            for (int t = 1; t < 8; ++t) m = fmaxf(m, xs[i + t]);
            if (__any(m >= lim))
#pragma unroll
              for (int t = 0; t < 8; ++t)
                if (xs[i + t] >= lim) {
                  if (at < LIST) list[at].x = comp_of(xs[i + t], j0 + (i + t) * 64 + lane);
                  ++at;
                }
          }
        }
      } else {
        each([&](float x, int j) {
          if (x >= lim) {
            const unsigned at = atomicAdd(&s_n, 1u);
            if (at < LIST) list[at].x = comp_of(x, j);
          }
        });
      }
    }
    __syncthreads();
    if (VPT == 1 || s_n <= FEW) {
      draw_from_list(Kk > 0 ? (unsigned)Kk : ~0u, P);
      return;
    }
    __syncthreads();
  }
  // sum over the workgroup (of whole numbers below 2^24: exact)
  auto count = [&](float v) {
    __syncthreads();
    v = wave_sum(v);
    if (lane == 0) s_max[w] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += s_max[i];
    return v;
  };
  if (Kk > 0) {
    float n = 0.f;
    each([&](float x, int) { n += x > -INFINITY ? 1.f : 0.f; });
    if ((float)Kk < count(n)) cut(false, (u64)Kk, 0.0);
  }
  if (P < 1.f) cut(true, 0, (double)P);
  auto kept = [&](float x, int j) { return x > -INFINITY && comp_of(x, j) >= thr && (x == mx || (double)x >= floor_); };
  __syncthreads();

  // what is left, in index order: each wave's part is summed; little of it in all is drawn from a list
  if (thr || M > 0.f) {
    if (tid == 0) s_n = 0;
    __syncthreads();
    // (a float below which nothing is kept: the smallest value the threshold lets through, or min-p's; the largest entry always is)
    const float least = fminf(mx, fmaxf(thr ? of_key((unsigned)(thr >> 32)) : -3.4028235e38f, (float)(floor_ - fabs(floor_) * 0x1p-22)));
    float over = 0.f;
    each([&](float x, int) { over += x >= least ? 1.f : 0.f; });
    over = count(over);
    if (over <= SHORT) {
      each([&](float x, int j) {
        if (x >= least && kept(x, j)) list[atomicAdd(&s_n, 1u)].x = comp_of(x, j);
      });
      __syncthreads();
      draw_from_list(~0u, 1.f);
      return;
    }
  }
  u64 sum = 0;
  each([&](float x, int j) {
    if (kept(x, j)) sum += weight(x);
  });
  sum = wave_sum_u64(sum);
  if (lane == 0) red_a[w] = sum;
  __syncthreads();
  u64 total = 0, before = 0;
  for (int i = 0; i < NW; ++i) { if (i < w) before += red_a[i]; total += red_a[i]; }
  const double goal = (double)uu * (double)total;
  if (lane == 0 && sum && (double)before <= goal && (double)(before + sum) > goal) { s_bin = w; s_base = before; }       // one wave: the running sums rise
  __syncthreads();
  // its part again, by all threads: a run of neighbouring entries each
  const int p0 = min(V, (int)s_bin * seg), p1 = min(V, p0 + seg), run = (p1 - p0 + NT - 1) / NT, r0 = min(p1, p0 + tid * run), r1 = min(p1, r0 + run);
  u64 own = 0, first[4] = {0, 0, 0, 0};                  // (the weights of the run's first four, for the walk below)
  for (int j = r0; j < r1; j += 4) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = load_logit(row, min(j + i, V - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u64 v = j + i < r1 && kept(x[i], j + i) ? weight(x[i]) : 0;
      if (j == r0) first[i] = v;
      own += v;
    }
  }
  u64 c = wave_scan_u64(own);
  if (lane == 63) red_b[w] = c;
  __syncthreads();
  c += s_base - own;
#pragma unroll
  for (int i = 0; i < NW; ++i) c += i < w ? red_b[i] : 0;
  if (own && (double)c <= goal && (double)(c + own) > goal)
    for (int j = r0; j < r1; ++j) {
      const int i = j - r0;
      u64 v = i == 0 ? first[0] : i == 1 ? first[1] : i == 2 ? first[2] : first[3];
      if (i > 3) { const float x = load_logit(row, j); v = kept(x, j) ? weight(x) : 0; }
      c += v;
      if ((double)c > goal) { a.token[b] = j; a.logp[b] = logp_of(load_logit(row, j), total); break; }
    }
}

template <typename T> void launch(const SampleArgs& a, int B, hipStream_t st) {
  if (a.V <= 160) hipLaunchKernelGGL((sample_rows_kernel<T, 256, 1024, 1>), dim3(B), dim3(256), 0, st, a);
  else if (a.V <= 4096) hipLaunchKernelGGL((sample_rows_kernel<T, 256, 1024, 16>), dim3(B), dim3(256), 0, st, a);
  else if (a.V <= 8192) hipLaunchKernelGGL((sample_rows_kernel<T, 1024, 4096, 8>), dim3(B), dim3(1024), 0, st, a);
  else if (a.V <= 32768) hipLaunchKernelGGL((sample_rows_kernel<T, 1024, 4096, 32>), dim3(B), dim3(1024), 0, st, a);
  else hipLaunchKernelGGL((sample_rows_kernel<T, 1024, 4096, 0>), dim3(B), dim3(1024), 0, st, a);
}

}  // namespace

extern "C" int dsrg_sample_rows(const void* logits, int64_t ld, int dtype, const float* u, const float* temperature, float temperature0,
                                const int32_t* top_k, int top_k0, const float* top_p, float top_p0, const float* min_p, float min_p0,
                                int64_t* token, float* logp, int B, int V, void* stream) {
  DSRG_CHECK(dtype == DSRG_F32 || dtype == DSRG_BF16, "dsrg_sample_rows: unsupported dtype %d", dtype);
  DSRG_CHECK(B >= 0 && V >= 1 && V <= (1 << 19), "dsrg_sample_rows: %d x %d logits (1 to 524288 a row)", B, V);
  if (B == 0) return DSRG_OK;
  DSRG_CHECK(logits && u && token && logp && (ld >= V || B == 1), "dsrg_sample_rows: bad arguments");
  DSRG_CHECK(temperature || (temperature0 >= 0.f && temperature0 < INFINITY), "dsrg_sample_rows: temperature %g", (double)temperature0);
  DSRG_CHECK(top_k || top_k0 >= 0, "dsrg_sample_rows: top_k %d", top_k0);
  DSRG_CHECK(top_p || top_p0 >= 0.f, "dsrg_sample_rows: top_p %g", (double)top_p0);
  DSRG_CHECK(min_p || (min_p0 >= 0.f && min_p0 <= 1.f), "dsrg_sample_rows: min_p %g", (double)min_p0);
  const SampleArgs a{logits, ld, u, temperature, top_k, top_p, min_p, temperature0, top_k0, top_p0, min_p0, token, logp, V};
  if (dtype == DSRG_F32) launch<float>(a, B, (hipStream_t)stream);
  else launch<bf16_t>(a, B, (hipStream_t)stream);
  DSRG_LAUNCH_CHECK("dsrg_sample_rows");
  return DSRG_OK;
}
