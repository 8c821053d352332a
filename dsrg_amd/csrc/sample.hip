// Draw of one entry per row of logits with temperature, top-k, top-p and min-p, from given random numbers (gfx950).
//
// The entries of a row in falling order (equal ones: the lowest index first) are cut three times, and each cut leaves a prefix of
// that order: after the k-th entry; after the first whose running weight reaches p of what the first cut left; where the weight
// falls under m times the largest.  So nothing is sorted: a cut is a threshold on the 64-bit number (value's order-preserving
// bits, ~index), found from a histogram (count or weight per bin of max - x) and the exact ranks inside the one bin that the cut
// falls into.  The draw is the inverse distribution function over what is left, in index order.
// Weights exp((x - max) / T) are fixed-point numbers of 44 bits behind the point, from a double exponential: integer sums do not
// depend on the order of the atomics, and 2^-45 an entry is far below what a 24-bit random number resolves.
#include "common.h"
#include <math.h>

typedef unsigned long long u64;

namespace {

constexpr int LIST = 1024;           // entries of the cut's bin that are ranked directly
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

__constant__ const double EXP2_32[32] = {      // 2^(k / 32)
    1, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
    1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832, 1.4142135623730951, 1.4451808069770467,
    1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543,
    1.6457554781539649, 1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424,
    1.8741676341103, 1.9152065613971474, 1.9571441241754002};

// 2^(t32 / 32) in WBITS-bit fixed point for t32 <= 0: 2^(n/32) from a table, the rest as e^y, |y| <= ln2 / 64, by its series (the
// first term left out is y^5 / 120 < 1.3e-12 of the weight).  Adding 2^(52 - WBITS) leaves the rounded fixed-point number in the mantissa.
__device__ __forceinline__ u64 fixed_exp2(double t32, const double* tab) {
  if (!(t32 > -46.0 * 32)) return 0;
  const double s = rint(t32), y = (t32 - s) * (0.69314718055994530942 / 32);
  const int n = (int)s;
  double e = fma(y, 1.0 / 24.0, 1.0 / 6.0);
  e = fma(y, e, 0.5);
  e = fma(y, e, 1.0);
  e = fma(y, e, 1.0);
  constexpr double MAGIC = (double)(1ull << (52 - WBITS));
  return (u64)__double_as_longlong(ldexp(e * tab[n & 31], n >> 5) + MAGIC) - (u64)__builtin_bit_cast(long long, MAGIC);
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

template <typename T> __device__ __forceinline__ float load_logit(const T* row, int j) {
  const float x = Elem<T>::ld(row + j) + 0.0f;          // (-0 + 0 = +0: the two zeros are one value)
  return x != x ? -INFINITY : x;
}

// Where the row is: VPT > 0: a thread holds VPT values of it in registers for the passes of the short way (top-k with a small k, short
// rows); the long way, taken by the others, reads the row again from the cache, eight independent loads at a time.
template <typename T, int NT, int NB, int VPT>
__global__ __launch_bounds__(NT) void sample_rows_kernel(const SampleArgs a) {
  constexpr int NW = NT / 64, BPT = NB / NT;            // bins per thread
  __shared__ u64 mass[NB];
  __shared__ unsigned cnt[NB];
  __shared__ ulonglong2 list[LIST];                     // (comp, weight)
  u64* const l_ahead = mass;                            // (the short way has no use for the bins' weights)
  unsigned* const l_rank = cnt;
  static_assert(NB >= LIST, "one word an entry");
  __shared__ double tab[32];
  __shared__ u64 red_a[NW], red_b[NW];
  __shared__ float s_max[NW], s_valid[NW];
  __shared__ double s_c2, s_tlogm;
  __shared__ u64 s_thr, s_base_m, s_base_c, s_bin_m;
  __shared__ unsigned s_bin, s_n, s_bin_n;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, b = blockIdx.x, V = a.V;
  const T* row = (const T*)a.logits + (long long)b * a.ld;
  const float Tm = a.temp ? a.temp[b] : a.temp0, P = a.topp ? a.topp[b] : a.topp0, M = a.minp ? a.minp[b] : a.minp0;
  const int Kk = a.topk ? a.topk[b] : a.topk0;
  const float u_raw = a.u[b], uu = u_raw >= 0.f ? fminf(u_raw, 0.99999994f) : 0.f;
  // wave w's part of the row: index order is (wave, step, lane)
  const int seg = (V + NW * 64 - 1) / (NW * 64) * 64, j0 = min(V, w * seg), j1 = min(V, j0 + seg);

  // f(value, index) for this thread's share of the row; -inf stands for what is no candidate
  auto again = [&](auto&& f) {
    for (int jb = j0 + lane; jb - lane < j1; jb += 512) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = load_logit(row, min(jb + i * 64, V - 1));
#pragma unroll
      for (int i = 0; i < 8; ++i) f(jb + i * 64 < j1 ? x[i] : -INFINITY, jb + i * 64);
    }
  };
  float xs[VPT ? VPT : 1];
  if constexpr (VPT > 0) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) xs[i] = load_logit(row, min(j0 + i * 64 + lane, V - 1));
#pragma unroll
    for (int i = 0; i < VPT; ++i) xs[i] = j0 + i * 64 + lane < j1 ? xs[i] : -INFINITY;
  }
  // (while the row is on its way)
  if (tid < 32) tab[tid] = EXP2_32[tid];
  if (tid == NT - 1) {
    s_c2 = 32 * 1.44269504088896340736 / (double)Tm;
    s_tlogm = M > 0.f ? (double)Tm * log((double)M) : -INFINITY;
  }
  auto each = [&](auto&& f) {
    if constexpr (VPT > 0) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) f(xs[i], j0 + i * 64 + lane);
    } else again(f);
  };

  // largest value, and how many entries can be drawn at all
  float tmax = -INFINITY;
  unsigned valid = 0;
  each([&](float x, int) {
    valid += x > -INFINITY;
    tmax = fmaxf(tmax, x);
  });
  const float wmax = wave_max(tmax), wvalid = wave_sum((float)valid);
  if (lane == 0) { s_max[w] = wmax; s_valid[w] = wvalid; }
  __syncthreads();
  float mx = -INFINITY, fvalid = 0.f;                   // (counts up to 2^19: exact)
#pragma unroll
  for (int i = 0; i < NW; ++i) { mx = fmaxf(mx, s_max[i]); fvalid += s_valid[i]; }
  const int nvalid = (int)fvalid;
  if (nvalid == 0) {                                    // nothing to draw from
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

  // For every entry of the list, by the 16 lanes of a DPP row together: how many entries `ahead(other, me)` holds for and what they weigh.
  auto ranked = [&](int n, auto&& ahead, auto&& f) {
    const int sub = tid & 15;
    for (int i0 = 0; i0 < n; i0 += NT / 16) {
      const int i = i0 + (tid >> 4);
      const ulonglong2 me = list[min(i, n - 1)];
      unsigned c = 0;
      u64 m = 0;
#pragma unroll 4
      for (int k = sub; k < n; k += 16) {
        const ulonglong2 o = list[k];
        const bool up = ahead(o, me);
        c += up;
        m += up ? o.y : 0;
      }
      const u64 cs = row_sum_u64(c);
      m = row_sum_u64(m);
      if (sub == 0 && i < n) f(i, me, (unsigned)cs, m);
    }
  };
  auto larger = [](const ulonglong2& o, const ulonglong2& me) { return o.x > me.x; };
  // Running count and weight over the bins, behind (c0, m0); the first bin that reaches the goal goes to s_bin, with what lies
  // before it and what it holds.  *goal < 0: it is frac of what all bins weigh.  (Entries so far down that their weight rounds to
  // 0 never reach a goal: the last bin that weighs anything does.)
  auto locate = [&](bool by_mass, u64 want, double frac, u64 c0, u64 m0, double* goal) {
    u64 tc = 0, tm = 0;
#pragma unroll
    for (int i = 0; i < BPT; ++i) { tc += cnt[tid * BPT + i]; tm += mass[tid * BPT + i]; }
    u64 ic = wave_scan_u32((unsigned)tc), im = by_mass ? wave_scan_u64(tm) : 0;
    if (lane == 63) { red_a[w] = ic; red_b[w] = im; }
    __syncthreads();
    u64 bc = c0, bm = m0, total = 0;
    for (int i = 0; i < NW; ++i) { if (i < w) { bc += red_a[i]; bm += red_b[i]; } total += red_b[i]; }
    ic += bc; im += bm;
    u64 ec = ic - tc, em = im - tm;
    if (*goal < 0) *goal = fmax(frac, 0.0) * (double)total;
    if (tc && (by_mass ? ((double)em < *goal || ec == 0) && (double)im >= *goal : ec < want && ic >= want)) {
      bool done = false;
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        const u64 nc = cnt[tid * BPT + i], nm = mass[tid * BPT + i];
        if (!done && nc && (by_mass ? (double)(em + nm) >= *goal : ec + nc >= want)) {
          done = true;
          s_bin = tid * BPT + i; s_base_c = ec; s_base_m = em; s_bin_n = (unsigned)nc; s_bin_m = nm;
        }
        ec += nc; em += nm;
      }
    }
    __syncthreads();
  };
  u64 thr = 0;                                          // entries with comp >= thr are kept (comp of a valid entry is never 0)
  // One cut: by_mass false: after `want` entries; true: after the first whose running weight reaches frac of the whole.
  auto cut = [&](bool by_mass, u64 want, double frac) {
    double goal = -1.0;
    for (int i = tid; i < NB; i += NT) { cnt[i] = 0; mass[i] = 0; }
    if (tid == 0) { s_thr = ~0ull; s_n = 0; }
    __syncthreads();
    again([&](float x, int j) {
      if (x > -INFINITY && comp_of(x, j) >= thr) {
        const unsigned bin = bin_of(x);
        atomicAdd(&cnt[bin], 1u);
        if (by_mass) atomicAdd(&mass[bin], weight(x));
      }
    });
    __syncthreads();
    locate(by_mass, want, frac, 0, 0, &goal);
    const unsigned bin = s_bin;
    u64 base_c = s_base_c, base_m = s_base_m;
    if (s_bin_n <= LIST) {
      again([&](float x, int j) {
        if (x > -INFINITY && comp_of(x, j) >= thr && bin_of(x) == bin) {
          const unsigned at = atomicAdd(&s_n, 1u);
          list[at] = make_ulonglong2(comp_of(x, j), by_mass ? weight(x) : 0);
        }
      });
      __syncthreads();
      const int n = (int)s_n;
      ranked(n, larger, [&](int, const ulonglong2& me, unsigned c, u64 m) {
        if (by_mass ? (double)(base_m + m) < goal || base_c + c == 0 : base_c + c < want) atomicMin(&s_thr, me.x);
      });
      __syncthreads();
      thr = s_thr;
    } else {
      // many entries in one bin (a flat row, or equal values): by the value's 32 bits, LB of them a pass
      constexpr int LB = NB == 4096 ? 12 : 10;
      unsigned prefix = 0, pmask = 0;
      for (int sh = 32; sh > 0;) {
        const int nb = min(LB, sh);
        sh -= nb;
        for (int i = tid; i < NB; i += NT) { cnt[i] = 0; mass[i] = 0; }
        __syncthreads();
        again([&](float x, int j) {
          const unsigned k = key_of(x);
          if (x > -INFINITY && comp_of(x, j) >= thr && bin_of(x) == bin && (k & pmask) == prefix) {
            const unsigned dig = ~(k >> sh) & ((1u << nb) - 1);            // falling values
            atomicAdd(&cnt[dig], 1u);
            if (by_mass) atomicAdd(&mass[dig], weight(x));
          }
        });
        __syncthreads();
        locate(by_mass, want, frac, base_c, base_m, &goal);
        base_c = s_base_c; base_m = s_base_m;
        prefix |= (~s_bin & ((1u << nb) - 1)) << sh;
        pmask |= ((1u << nb) - 1) << sh;
        __syncthreads();
      }
      // s_bin_n equal values of weight s_bin_m / s_bin_n: as many of them as the goal asks, the lowest indices first
      u64 r;
      const u64 each = s_bin_m / s_bin_n;
      if (by_mass) {
        const double left = goal - (double)base_m;
        r = each && left > 0 ? (u64)ceil(left / (double)each) : 1;
        while (r > 1 && (double)(base_m + (r - 1) * each) >= goal) --r;
        while ((double)(base_m + r * each) < goal && r < s_bin_n) ++r;
      } else r = want - base_c;
      if (r < 1) r = 1;
      if (r > s_bin_n) r = s_bin_n;
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
    const double goal = fmax((double)p, 0.0) * (double)all;
    sum = 0;
    for (int i = tid; i < n; i += NT) {                 // what is not kept loses its weight: it is not drawn then
      const ulonglong2 me = list[i];
      const float x = value(me.x);
      const unsigned rank = l_rank[i];
      const bool keep = rank == 0 || (rank < want && (!(p < 1.f) || (double)l_ahead[i] < goal) && (x == mx || (double)x >= floor_));
      if (keep) sum += me.y; else list[i].y = 0;
    }
    sum = wave_sum_u64(sum);
    if (lane == 0) red_b[w] = sum;
    __syncthreads();
    u64 total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) total += red_b[i];
    const double draw = (double)uu * (double)total;
    // (the low word is ~index: the entries before have a larger one)
    ranked(n, [](const ulonglong2& o, const ulonglong2& me) { return (unsigned)o.x > (unsigned)me.x; }, [&](int, const ulonglong2& me, unsigned, u64 m) {
      if (me.y && (double)m <= draw && (double)(m + me.y) > draw) { a.token[b] = (int)~(unsigned)me.x; a.logp[b] = logp_of(value(me.x), total); }
    });
  };

  // The short way: everything that can be drawn fits a list.  Rows of up to 256 entries: all of them.  Top-k with a small k: the k-th
  // largest of the threads' largest entries is no larger than the k-th largest of all, so the entries of its bin and above hold the k
  // wanted ones, and few others.  One bin a thread here (NT / 16 an octave): a bin costs a few more entries, a scan more costs time.
  const bool small = VPT == 1, few = Kk > 0 && Kk <= 256 && Kk < nvalid;
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
    } else __syncthreads();
    auto take = [&](float x, int j) {
      if (x >= lim) {
        const unsigned at = atomicAdd(&s_n, 1u);
        if (at < LIST) list[at].x = comp_of(x, j);
      }
    };
    if constexpr (VPT >= 8) {
#pragma unroll
      for (int i = 0; i < VPT; i += 8) {                // (one test for eight: few of a wave's 512 are taken)
        float m = xs[i];
#pragma unroll
        for (int t = 1; t < 8; ++t) m = fmaxf(m, xs[i + t]);
        if (__any(m >= lim))
#pragma unroll
          for (int t = 0; t < 8; ++t) take(xs[i + t], j0 + (i + t) * 64 + lane);
      }
    } else each(take);
    __syncthreads();
    if (s_n <= LIST) {
      draw_from_list(Kk > 0 ? (unsigned)Kk : ~0u, P);
      return;
    }
    __syncthreads();
  }
  u64 certain = 0;                                      // entries that are left at least
  if (Kk > 0 && Kk < nvalid) { cut(false, (u64)Kk, 0.0); certain = Kk; }
  if (P < 1.f) { cut(true, 0, (double)P); certain = s_base_c; }
  auto kept = [&](float x, int j) { return x > -INFINITY && comp_of(x, j) >= thr && (x == mx || (double)x >= floor_); };
  __syncthreads();

  // what is left, where that is little
  constexpr int SHORT = NT / 4;                         // (ranks cost n^2 / NT, another pass of weights V / NT)
  if ((thr || M > 0.f) && certain <= SHORT) {
    if (tid == 0) s_n = 0;
    __syncthreads();
    again([&](float x, int j) {
      if (kept(x, j)) {
        const unsigned at = atomicAdd(&s_n, 1u);
        if (at < LIST) list[at].x = comp_of(x, j);
      }
    });
    __syncthreads();
    if (s_n <= SHORT) {
      draw_from_list(~0u, 1.f);
      return;
    }
  }

  // what is left, in index order
  u64 sum = 0;
  again([&](float x, int j) {
    if (kept(x, j)) sum += weight(x);
  });
  sum = wave_sum_u64(sum);
  if (lane == 0) red_a[w] = sum;
  __syncthreads();
  u64 total = 0, before = 0;
  for (int i = 0; i < NW; ++i) { if (i < w) before += red_a[i]; total += red_a[i]; }
  const double goal = (double)uu * (double)total;
  if (sum && (double)before <= goal && (double)(before + sum) > goal) {       // one wave: the running sums rise
    u64 base = before;
    for (int s0 = j0; s0 < j1; s0 += 64) {
      const int j = s0 + lane;
      const float x = j < j1 ? load_logit(row, j) : -INFINITY;
      const bool in = j < j1 && kept(x, j);
      if (!__ballot(in)) continue;
      u64 c = in ? weight(x) : 0;
      const u64 own = c;
      c = wave_scan_u64(c);
      const u64 hit = __ballot(own && (double)(base + c) > goal);
      if (hit) {
        if (lane == __builtin_ctzll(hit)) {
          a.token[b] = j;
          a.logp[b] = logp_of(x, total);
        }
        break;
      }
      base += lane_u64(c, 63);
    }
  }
}

template <typename T> void launch(const SampleArgs& a, int B, hipStream_t st) {
  if (a.V <= 256) hipLaunchKernelGGL((sample_rows_kernel<T, 256, 1024, 1>), dim3(B), dim3(256), 0, st, a);
  else if (a.V <= 4096) hipLaunchKernelGGL((sample_rows_kernel<T, 256, 1024, 16>), dim3(B), dim3(256), 0, st, a);
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
