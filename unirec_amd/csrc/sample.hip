// Sampling from scores with temperature, top-k, top-p and min-p, the random numbers given by the caller (beside eval.hip's top-k: an answer
// drawn from the distribution instead of its head).  Per row of N scores x:
//   z_n = (x_n - max x) / T, weight w_n = exp(z_n); NaN and -inf carry none; a row with +inf: those entries 1, the others 0
//   top-k: the first k in the order (score descending, index ascending); top-p: of those, in that order, every entry before which less
//   than p of their weight lies; min-p: w >= min_p.  The answer to u: the first index n, in INDEX order, with sum_{j <= n} kept w_j > u W.
// No sort: the order only decides a threshold (a key and how many of its ties stay), found by radix selection over 11, 11 and 10 bits.
//
// Arithmetic.  Which entry a sum's border falls on is a whole number, so sums are exact: a weight is exp in double (2 10^-16), rounded down
// once to a multiple of 2^-62 and added as integers, in two 32-bit limbs summed in 64 bits each (the top-p selection sums multiples of
// 2^-(62 - log2 N) in one).  No result depends on an order of additions or on how a row was cut into pieces.
//
// Two forms.  A row that fits into LDS (32 768 entries; 65 536 of 16 bits): one workgroup, one read of the row, every pass from LDS.
// Longer rows: workgroups of 16 384 entries, a pass over memory each for the maximum, every round of a selection and the kept sums, the
// decisions between the passes taken by the workgroup that arrives last.
#include <math.h>

#include <algorithm>

#include "common.h"

namespace ur {

typedef unsigned long long u64;
typedef unsigned __int128 u128;

struct SampleArgs {
  const void* scores; int type; long long N, ld; int B, S;
  const float* rand;                    // [B, S]
  double T, top_p, min_p; int top_k;    // for every row, unless the row has its own:
  const float *T_rows, *p_rows, *minp_rows; const int* k_rows;
  const long long* ids; long long ld_ids;
  long long* out_id; float* out_logp;   // [B, S]
};

// ascending unsigned order == ascending float order; -0 counts as 0 (equal scores tie), NaN as -inf
__device__ __forceinline__ unsigned sample_key(float x) {
  if (!(x > -INFINITY)) return 0u;
  const unsigned u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sample_value(unsigned key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key); }
__device__ __forceinline__ float sample_load(const void* p, int type, long long i) {
  if (type == UR_F16) return (float)((const _Float16*)p)[i];
  if (type == UR_BF16) return __uint_as_float((unsigned)((const unsigned short*)p)[i] << 16);
  return ((const float*)p)[i];
}
// exp(z) 2^62, rounded down, z <= 0.  r = z - n ln 2 in two pieces, |r| <= ln 2 / 2, the Taylor polynomial of degree 12 (remainder 2 10^-16)
__device__ __forceinline__ u64 exp_fixed(double z) {
  if (!(z > -43.0)) return 0;                                    // below 2^-62
  const double n = rint(z * 1.4426950408889634);
  constexpr double LN2_HI = 2977044471.0 / 4294967296.0;         // the first 32 bits of ln 2 (n LN2_HI is exact), and the rest
  const double r = fma(n, -1.9082149292705877e-10, fma(n, -LN2_HI, z));
  double p = 1.0 / 479001600.0;
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const double v = ldexp(p, (int)n + 30);                        // <= 2^30 (z <= 0: p 2^n <= 1 up to its rounding)
  const unsigned hi = (unsigned)v;
  return ((u64)hi << 32) + (unsigned)((v - (double)hi) * 4294967296.0);
}
// a row's parameters
struct SampleRow {
  double inv_T, p, min_z; long long k; bool greedy, flat;
  float m;
  __device__ __forceinline__ void load(const SampleArgs& a, int b) {
    const double T = a.T_rows ? (double)a.T_rows[b] : a.T;
    double min_p = a.minp_rows ? (double)a.minp_rows[b] : a.min_p;
    p = a.p_rows ? (double)a.p_rows[b] : a.top_p;
    k = a.k_rows ? a.k_rows[b] : a.top_k;
    if (k <= 0) k = a.N;
    greedy = !(T > 1e-300);              // (1 / T stays finite)
    inv_T = greedy ? 1.0 : 1.0 / T;
    if (!(min_p < 1.0)) min_p = 1.0;     // (the largest stays)
    min_z = min_p > 0.0 ? log(min_p) : -INFINITY;
  }
  __device__ __forceinline__ void set_max(unsigned key) { m = sample_value(key); flat = greedy || m == INFINITY; }
  __device__ __forceinline__ double z(unsigned key) const {
    const float x = sample_value(key);
    if (flat) return x == m ? 0.0 : -INFINITY;
    return ((double)x - (double)m) * inv_T;
  }
  __device__ __forceinline__ u64 weight(unsigned key) const { return exp_fixed(z(key)); }
  // of an entry that the selections leave: 0 if min-p takes it
  __device__ __forceinline__ u64 kept(unsigned key) const {
    const double v = z(key);
    return v >= min_z ? exp_fixed(v) : 0;
  }
};
// entries above `cut` stay, and of those equal to it the first `ties` in index order
struct SampleCut { unsigned cut; unsigned ties; };
constexpr unsigned ALL_TIES = 0xFFFFFFFFu;

struct WSum {   // a sum of weights
  u64 hi, lo;
  __device__ __forceinline__ void add(u64 w) { hi += w >> 32; lo += w & 0xFFFFFFFFull; }
  __device__ __forceinline__ void add(const WSum& o) { hi += o.hi; lo += o.lo; }
  __device__ __forceinline__ u128 all() const { return ((u128)hi << 32) + lo; }
};
__device__ __forceinline__ u64 shfl_xor64(u64 v, int o) {
  return ((u64)(unsigned)__shfl_xor((int)(v >> 32), o, 64) << 32) | (unsigned)__shfl_xor((int)(unsigned)v, o, 64);
}
__device__ __forceinline__ u64 shfl_up64(u64 v, int o) {
  return ((u64)(unsigned)__shfl_up((int)(v >> 32), o, 64) << 32) | (unsigned)__shfl_up((int)(unsigned)v, o, 64);
}
__device__ __forceinline__ WSum wave_total(WSum v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    v.hi += shfl_xor64(v.hi, o);
    v.lo += shfl_xor64(v.lo, o);
  }
  return v;
}
__device__ __forceinline__ WSum wave_upto(WSum v) {   // inclusive, lane order
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 h = shfl_up64(v.hi, o), l = shfl_up64(v.lo, o);
    if (lane >= o) { v.hi += h; v.lo += l; }
  }
  return v;
}
__device__ __forceinline__ double wide_to_double(u128 v) { return (double)(u64)(v >> 64) * 18446744073709551616.0 + (double)(u64)v; }
__device__ __forceinline__ u128 double_to_wide(double v) {   // v >= 0
  const u64 hi = (u64)(v * 5.42101086242752217e-20);          // 2^-64
  const double rest = v - (double)hi * 18446744073709551616.0;
  return ((u128)hi << 64) + (rest > 0.0 ? (u64)rest : 0);
}
__device__ __forceinline__ u128 sample_goal(float u, u128 W) {
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;                   // [0, 1): what lies outside is moved to the nearest end, NaN to 0
  return double_to_wide((double)u * wide_to_double(W));
}
// entries j = 0, 1, .. of one tied weight w stay while above + j w < limit (the first always)
__device__ __forceinline__ unsigned ties_within(u64 above, u64 w, double limit, unsigned most) {
  if (w == 0) return most;
  unsigned lo = 1, hi = most;           // the first j in [1, most] that does not stay
  while (lo < hi) {
    const unsigned mid = lo + (hi - lo) / 2;
    if ((double)(above + w * mid) < limit) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// ---- one round of a selection: 2 048 bins over the keys of one prefix
constexpr int SB = 2048, ROUNDS = 3;
__device__ __forceinline__ int round_shift(int round) { return round == 0 ? 21 : round == 1 ? 10 : 0; }
__device__ __forceinline__ unsigned round_bin(unsigned key, int round) { return (key >> round_shift(round)) & (round == 2 ? 1023u : 2047u); }
__device__ __forceinline__ bool round_in(unsigned key, int round, unsigned prefix) {
  return round == 0 || (round == 1 ? key >> 21 : key >> 10) == prefix;
}
struct Select {   // state of a selection (one per row)
  unsigned prefix; unsigned need;       // top-k: how many of the prefix's entries stay
  u64 above; double limit;              // top-p: the weight in front of the prefix, p times all of it
  unsigned done;
};
template <int NT>
__device__ __forceinline__ unsigned block_before(unsigned v, unsigned* tmp) {   // exclusive sum over the threads; tmp[NT / 64]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned t = __shfl_up((int)s, o, 64);
    if (lane >= o) s += t;
  }
  if (lane == 63) tmp[wave] = s;
  __syncthreads();
  unsigned base = 0;
  for (int w = 0; w < wave; ++w) base += tmp[w];
  __syncthreads();
  return base + s - v;
}
template <int NT>
__device__ __forceinline__ u64 block_before(u64 v, u64* tmp, u64* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 t = shfl_up64(s, o);
    if (lane >= o) s += t;
  }
  if (lane == 63) tmp[wave] = s;
  __syncthreads();
  u64 base = 0, all = 0;
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) base += tmp[w];
    all += tmp[w];
  }
  __syncthreads();
  *total = all;
  return base + s - v;
}
// the bin that the border falls into, found by the whole workgroup (bins from the highest key down); updates st, sets cut when it is final.
// cnt / wgt: the round's histogram (any address space), read through `count` and `weight`
template <int NT, typename C>
__device__ __forceinline__ void pick_k(int round, C count, Select* st, SampleCut* cut, unsigned* tmp) {
  constexpr int PB = SB / NT;
  const unsigned need = st->need, prefix = st->prefix;
  unsigned mine[PB], sum = 0;
#pragma unroll
  for (int j = 0; j < PB; ++j) { mine[j] = count(SB - 1 - ((int)threadIdx.x * PB + j)); sum += mine[j]; }
  unsigned before = block_before<NT>(sum, tmp);
  if (before < need && need <= before + sum) {
#pragma unroll
    for (int j = 0; j < PB; ++j) {
      if (before < need && need <= before + mine[j]) {
        const unsigned d = SB - 1 - (threadIdx.x * PB + j), p = round == 0 ? d : (prefix << (round == 1 ? 11 : 10)) | d, rest = need - before;
        st->prefix = p;
        st->need = rest;
        if (rest == mine[j]) { cut->cut = (p << round_shift(round)) - 1u; cut->ties = 0u; st->done = 1u; }   // all of the bin
        else if (round == ROUNDS - 1) { cut->cut = p; cut->ties = rest; st->done = 1u; }
      }
      before += mine[j];
    }
  } else if (threadIdx.x == NT - 1 && before + sum < need) {
    st->done = 1u;                      // fewer entries than k: nothing is cut
  }
  __syncthreads();
}
template <int NT, typename C, typename W>
__device__ __forceinline__ void pick_p(int round, C count, W weight, double p, Select* st, SampleCut* cut, u64* tmp) {
  constexpr int PB = SB / NT;
  const unsigned prefix = st->prefix;
  u64 mine[PB], sum = 0, total;
#pragma unroll
  for (int j = 0; j < PB; ++j) { mine[j] = weight(SB - 1 - ((int)threadIdx.x * PB + j)); sum += mine[j]; }
  u64 before = block_before<NT>(sum, tmp, &total) + st->above;
  const double limit = round == 0 ? p * (double)total : st->limit;
  __syncthreads();
  // the first entry of exactly one bin is the last whose forerunners weigh less than the limit (p <= 0: the first bin)
  const bool here = limit > 0.0 ? (double)before < limit && !((double)(before + sum) < limit) : false;
  if (here) {
#pragma unroll
    for (int j = 0; j < PB; ++j) {
      if ((double)before < limit && !((double)(before + mine[j]) < limit)) {
        const unsigned d = SB - 1 - (threadIdx.x * PB + j), q = round == 0 ? d : (prefix << (round == 1 ? 11 : 10)) | d, n = count(d);
        st->prefix = q;
        st->above = before;
        st->limit = limit;
        st->need = n;
        if (n == 1) { cut->cut = (q << round_shift(round)) - 1u; cut->ties = 0u; st->done = 1u; }
        else if (round == ROUNDS - 1) { cut->cut = q; cut->ties = ties_within(before, mine[j] / n, limit, n); st->done = 1u; }
      }
      before += mine[j];
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------------------------- rows that fit into LDS
constexpr int SBLK = 512;               // entries of a block of the kept sums
template <int NT, bool RAW>
__global__ __launch_bounds__(NT) void sample_row_kernel(SampleArgs a, int coarse) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int NWV = NT / 64;
  const int nblk = (int)((a.N + SBLK - 1) / SBLK), N = (int)a.N;
  u64* hw = (u64*)smem;                                          // [SB]
  u64* bs = hw + SB;                                             // [2 nblk] block sums, then what lies in front of a block
  unsigned* hc = (unsigned*)(bs + 2 * nblk);                     // [SB]
  unsigned* tb = hc + SB;                                        // [nblk] ties in front of a block
  unsigned* keys = tb + ((nblk + 3) & ~3);                       // [N], or 16-bit scores as they are
  unsigned short* raw = (unsigned short*)keys;
  __shared__ u64 tmp64[NWV];
  __shared__ unsigned tmp32[NWV], s_max[NWV];
  __shared__ Select st;
  __shared__ SampleCut cut_s;
  __shared__ WSum s_total;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long base = (long long)b * a.ld;
  SampleRow r;
  r.load(a, b);
  auto key_at = [&](int i) -> unsigned {
    if constexpr (RAW) return sample_key(a.type == UR_F16 ? (float)__builtin_bit_cast(_Float16, raw[i]) : __uint_as_float((unsigned)raw[i] << 16));
    else return keys[i];
  };
  unsigned mk = 0u;
  for (int i = tid; i < N; i += NT) {
    const unsigned k = sample_key(sample_load(a.scores, a.type, base + i));
    if constexpr (RAW) raw[i] = ((const unsigned short*)a.scores)[base + i];
    else keys[i] = k;
    mk = max(mk, k);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) mk = max(mk, (unsigned)__shfl_xor((int)mk, o, 64));
  if (lane == 0) s_max[wave] = mk;
  __syncthreads();
  mk = 0u;
  for (int w = 0; w < NWV; ++w) mk = max(mk, s_max[w]);
  if (mk == 0u) {                       // nothing to choose from
    for (int s = tid; s < a.S; s += NT) {
      a.out_id[(long long)b * a.S + s] = -1;
      a.out_logp[(long long)b * a.S + s] = -INFINITY;
    }
    return;
  }
  r.set_max(mk);
  SampleCut c{0u, ALL_TIES};            // (key 0: no entry)
  if (r.greedy) {
    c.cut = mk;
    c.ties = 1u;
  } else {
    if (r.k < N) {
      if (tid == 0) { st = Select{0u, (unsigned)r.k, 0, 0.0, 0u}; cut_s = c; }
      for (int round = 0; round < ROUNDS; ++round) {
        for (int i = tid; i < SB; i += NT) hc[i] = 0u;
        __syncthreads();
        const unsigned prefix = st.prefix;
        for (int i = tid; i < N; i += NT) {
          const unsigned k = key_at(i);
          if (k != 0u && round_in(k, round, prefix)) atomicAdd(&hc[round_bin(k, round)], 1u);
        }
        __syncthreads();
        pick_k<NT>(round, [&](int d) { return hc[d]; }, &st, &cut_s, tmp32);
        if (st.done) break;
      }
      c = cut_s;
      __syncthreads();
    }
    if (r.p < 1.0) {
      if (tid == 0) { st = Select{0u, 0u, 0, 0.0, 0u}; cut_s = SampleCut{mk, 1u}; }   // (p <= 0: the largest alone)
      for (int round = 0; round < ROUNDS && r.p > 0.0; ++round) {
        for (int i = tid; i < SB; i += NT) { hc[i] = 0u; hw[i] = 0; }
        __syncthreads();
        const unsigned prefix = st.prefix;
        for (int i = tid; i < N; i += NT) {
          const unsigned k = key_at(i);
          if (k <= c.cut || !round_in(k, round, prefix)) continue;
          const u64 w = r.weight(k) >> coarse;
          const unsigned d = round_bin(k, round);
          atomicAdd(&hc[d], 1u);
          atomicAdd(&hw[d], w);
        }
        if (tid == 0 && c.cut != 0u && c.ties != 0u && round_in(c.cut, round, prefix)) {   // the ties that top-k left
          atomicAdd(&hc[round_bin(c.cut, round)], c.ties);
          atomicAdd(&hw[round_bin(c.cut, round)], (r.weight(c.cut) >> coarse) * c.ties);
        }
        __syncthreads();
        pick_p<NT>(round, [&](int d) { return hc[d]; }, [&](int d) { return hw[d]; }, r.p, &st, &cut_s, tmp64);
        if (st.done) break;
      }
      __syncthreads();
      c = cut_s;
    }
  }
  // ---- ties in front of every block (where some of them go)
  const bool ranked = c.ties != 0u && c.ties != ALL_TIES;
  if (ranked) {
    for (int q = wave; q < nblk; q += NWV) {
      int n = 0;
      for (int i = q * SBLK + lane; i < min(N, (q + 1) * SBLK); i += 64) n += key_at(i) == c.cut;
      for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o, 64);
      if (lane == 0) tb[q] = (unsigned)n;
    }
    __syncthreads();
    const unsigned v = tid < nblk ? tb[tid] : 0u;               // (nblk <= 128 < NT)
    const unsigned before = block_before<NT>(v, tmp32);
    if (tid < nblk) tb[tid] = before;
    __syncthreads();
  }
  // whether this lane's entry (one of 64 consecutive ones) stays; `ties` = ties in front of the 64
  auto stays = [&](unsigned k, unsigned& ties) -> bool {
    if (!ranked) return k > c.cut || (k == c.cut && k != 0u && c.ties != 0u);
    const u64 eq = __ballot(k == c.cut);
    const unsigned rank = ties + __popcll(eq & ((1ull << lane) - 1ull));
    ties += __popcll(eq);
    return k > c.cut || (k == c.cut && rank < c.ties);
  };
  // ---- the kept weight of every block
  for (int q = wave; q < nblk; q += NWV) {
    WSum v{0, 0};
    unsigned ties = ranked ? tb[q] : 0u;
#pragma unroll 2
    for (int j = 0; j < SBLK / 64; ++j) {
      const int i = q * SBLK + 64 * j + lane;
      const unsigned k = i < N ? key_at(i) : 0u;
      if (stays(k, ties)) v.add(r.kept(k));
    }
    v = wave_total(v);
    if (lane == 0) { bs[2 * q] = v.hi; bs[2 * q + 1] = v.lo; }
  }
  __syncthreads();
  if (wave == 0) {                      // prefix over the blocks, 64 at a time
    WSum run{0, 0};
    for (int q0 = 0; q0 < nblk; q0 += 64) {
      const int q = q0 + lane;
      const WSum v = q < nblk ? WSum{bs[2 * q], bs[2 * q + 1]} : WSum{0, 0};
      const WSum up = wave_upto(v);
      if (q < nblk) { bs[2 * q] = run.hi + up.hi - v.hi; bs[2 * q + 1] = run.lo + up.lo - v.lo; }
      run.hi += ((u64)(unsigned)__shfl((int)(up.hi >> 32), 63, 64) << 32) | (unsigned)__shfl((int)(unsigned)up.hi, 63, 64);
      run.lo += ((u64)(unsigned)__shfl((int)(up.lo >> 32), 63, 64) << 32) | (unsigned)__shfl((int)(unsigned)up.lo, 63, 64);
    }
    if (lane == 0) s_total = run;
  }
  __syncthreads();
  const u128 W = s_total.all();
  const double log_W = log(wide_to_double(W) * 2.168404344971009e-19);   // 2^-62
  // ---- a wave a draw: the last block that does not begin behind the goal, its first entry behind it
  for (int s = wave; s < a.S; s += NWV) {
    const u128 goal = sample_goal(a.rand[(long long)b * a.S + s], W);
    int q = 0;
    for (int q0 = 0; q0 < nblk; q0 += 64) {
      const int t = q0 + lane;
      const bool before = t < nblk && WSum{bs[2 * t], bs[2 * t + 1]}.all() <= goal;
      q += __popcll(__ballot(before));
    }
    q -= 1;
    u128 run = WSum{bs[2 * q], bs[2 * q + 1]}.all();
    unsigned ties = ranked ? tb[q] : 0u;
    for (int j = 0; j < SBLK / 64; ++j) {
      const int i = q * SBLK + 64 * j + lane;
      const unsigned k = i < N ? key_at(i) : 0u;
      WSum v{0, 0};
      if (stays(k, ties)) v.add(r.kept(k));
      const WSum up = wave_upto(v);
      const u64 over = __ballot(run + up.all() > goal);
      if (over) {
        if (lane == __ffsll(over) - 1) {
          a.out_id[(long long)b * a.S + s] = a.ids ? a.ids[(long long)b * a.ld_ids + i] : i;
          a.out_logp[(long long)b * a.S + s] = r.greedy ? 0.f : (float)(r.z(k) - log_W);
        }
        break;
      }
      const u64 th = ((u64)(unsigned)__shfl((int)(up.hi >> 32), 63, 64) << 32) | (unsigned)__shfl((int)(unsigned)up.hi, 63, 64);
      const u64 tl = ((u64)(unsigned)__shfl((int)(up.lo >> 32), 63, 64) << 32) | (unsigned)__shfl((int)(unsigned)up.lo, 63, 64);
      run += WSum{th, tl}.all();
    }
  }
}

// ---------------------------------------------------------------------------------------------- longer rows
constexpr int LCH = 16384, LBLK = 2048;   // entries of a workgroup; of a block of the kept sums
struct SampleState {                      // per row, in the workspace
  Select st;
  SampleCut cut;                          // of the selections so far
  SampleCut kcut;                         // of top-k (the top-p rounds need it)
  unsigned maxkey, arrived;
};
struct SampleLong {
  SampleState* state; unsigned* hc; u64* hw;   // [B], [B][SB], [B][SB]
  unsigned* tb; u64* bs;                       // [B][nblk] ties of a block, [B][2 nblk] kept weight of a block
  int nblk, nchunk, coarse;
  int uses_k, uses_p;
};

__global__ __launch_bounds__(256) void sample_init_kernel(SampleArgs a, SampleLong g) {
  const int b = blockIdx.x;
  for (int i = threadIdx.x; i < SB; i += 256) { g.hc[(long long)b * SB + i] = 0u; g.hw[(long long)b * SB + i] = 0; }
  if (threadIdx.x == 0) {
    SampleState s{};
    s.cut = s.kcut = SampleCut{0u, ALL_TIES};
    g.state[b] = s;
  }
}
__device__ __forceinline__ unsigned agent_load(const unsigned* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ u64 agent_load(const u64* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// four consecutive entries a thread and step (one wide load where the row's address allows it); entries behind the end are key 0.
// f(key)
template <typename F>
__device__ __forceinline__ void sample_walk(const SampleArgs& a, long long base, long long i0, long long i1, F f) {
  const bool half = a.type != UR_F32;
  const bool wide = (((unsigned long long)a.scores + (unsigned long long)(base + i0) * (half ? 2 : 4)) & (half ? 7 : 15)) == 0;
#pragma unroll 2
  for (long long i = i0 + 4 * threadIdx.x; i < i1; i += 1024) {
    float x[4];
    if (wide && i + 4 <= i1) {
      if (half) {
        const ushort4 v = *(const ushort4*)((const unsigned short*)a.scores + base + i);
        const unsigned short u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = a.type == UR_F16 ? (float)__builtin_bit_cast(_Float16, u[j]) : __uint_as_float((unsigned)u[j] << 16);
      } else {
        const float4 v = *(const float4*)((const float*)a.scores + base + i);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = i + j < i1 ? sample_load(a.scores, a.type, base + i + j) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) f(sample_key(x[j]));
  }
}
__global__ __launch_bounds__(256) void sample_max_kernel(SampleArgs a, SampleLong g) {
  const int b = blockIdx.y;
  const long long i0 = (long long)blockIdx.x * LCH, i1 = min(a.N, i0 + LCH);
  unsigned mk = 0u;
  sample_walk(a, (long long)b * a.ld, i0, i1, [&](unsigned k) { mk = max(mk, k); });
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) mk = max(mk, (unsigned)__shfl_xor((int)mk, o, 64));
  if ((threadIdx.x & 63) == 0 && mk) atomicMax(&g.state[b].maxkey, mk);
}
// a round of the top-k (PHASE 0) or top-p (PHASE 1) selection: counts (and weights) of the prefix's entries by bin; the workgroup that
// arrives last takes the decision and clears the bins for the next round
template <int PHASE>
__global__ __launch_bounds__(256) void sample_round_kernel(SampleArgs a, SampleLong g, int round, int mode) {
  __shared__ unsigned hc[SB];
  __shared__ u64 hw[PHASE == 1 ? SB : 1];
  __shared__ unsigned tmp32[4], last;
  __shared__ u64 tmp64[4];
  __shared__ Select st;
  __shared__ SampleCut cut;
  const int b = blockIdx.y, tid = threadIdx.x;
  SampleState* S = g.state + b;
  SampleRow r;
  r.load(a, b);
  const unsigned mk = S->maxkey;
  const bool active = mk != 0u && !r.greedy && (PHASE == 0 ? r.k < a.N : r.p < 1.0 && r.p > 0.0) && !(round > 0 && S->st.done);
  if (!active) {
    // a row whose p is not positive keeps its largest entry alone
    if (PHASE == 1 && round == 0 && blockIdx.x == 0 && tid == 0 && mk != 0u && !r.greedy && r.p <= 0.0) S->cut = SampleCut{mk, 1u};
    return;
  }
  r.set_max(mk);
  unsigned* ghc = g.hc + (long long)b * SB;
  u64* ghw = g.hw + (long long)b * SB;
  const unsigned prefix = round ? S->st.prefix : 0u;
  const SampleCut kc = S->kcut;
  for (int i = tid; i < SB; i += 256) {
    hc[i] = 0u;
    if (PHASE == 1) hw[i] = 0;
  }
  __syncthreads();
  const long long i0 = (long long)blockIdx.x * LCH, i1 = min(a.N, i0 + LCH);
  sample_walk(a, (long long)b * a.ld, i0, i1, [&](unsigned k) {
    if (PHASE == 0 ? k == 0u : k <= kc.cut) return;
    if (!round_in(k, round, prefix)) return;
    const unsigned d = round_bin(k, round);
    atomicAdd(&hc[d], 1u);
    if constexpr (PHASE == 1) atomicAdd(&hw[d], r.weight(k) >> g.coarse);
  });
  if (PHASE == 1 && blockIdx.x == 0 && tid == 0 && kc.cut != 0u && kc.ties != 0u && round_in(kc.cut, round, prefix)) {
    atomicAdd(&hc[round_bin(kc.cut, round)], kc.ties);
    atomicAdd(&hw[PHASE == 1 ? round_bin(kc.cut, round) : 0], (r.weight(kc.cut) >> g.coarse) * kc.ties);
  }
  __syncthreads();
  for (int i = tid; i < SB; i += 256)
    if (hc[i]) {
      atomicAdd(&ghc[i], hc[i]);
      if constexpr (PHASE == 1) atomicAdd(&ghw[i], hw[i]);
    }
  __syncthreads();
  if (tid == 0) last = ur_arrive(&S->arrived, mode) == (unsigned)g.nchunk - 1u;
  __syncthreads();
  if (!last) return;
  if (tid == 0) {
    st = round ? S->st : Select{0u, (unsigned)min((long long)0x7FFFFFFF, r.k), 0, 0.0, 0u};
    cut = S->cut;
  }
  for (int i = tid; i < SB; i += 256) {
    hc[i] = agent_load(ghc + i);
    if constexpr (PHASE == 1) hw[i] = agent_load(ghw + i);
    ghc[i] = 0u;
    if (PHASE == 1) ghw[i] = 0;
  }
  __syncthreads();
  if constexpr (PHASE == 0) pick_k<256>(round, [&](int d) { return hc[d]; }, &st, &cut, tmp32);
  else pick_p<256>(round, [&](int d) { return hc[d]; }, [&](int d) { return hw[d]; }, r.p, &st, &cut, tmp64);
  if (tid == 0) {
    S->st = st;
    S->cut = cut;
    if (PHASE == 0) S->kcut = cut;
    S->arrived = 0u;
  }
}
__device__ __forceinline__ SampleCut final_cut(const SampleState* S, const SampleRow& r) {
  return r.greedy ? SampleCut{S->maxkey, 1u} : S->cut;
}
// ties of every block (rows where some of them go)
__global__ __launch_bounds__(256) void sample_ties_kernel(SampleArgs a, SampleLong g) {
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  SampleRow r;
  r.load(a, b);
  const SampleCut c = final_cut(g.state + b, r);
  if (c.ties == 0u || c.ties == ALL_TIES) return;
  for (int q = blockIdx.x * (LCH / LBLK) + wave; q < min(g.nblk, (int)(blockIdx.x + 1) * (LCH / LBLK)); q += 4) {
    int n = 0;
    for (long long i = (long long)q * LBLK + lane; i < min(a.N, (long long)(q + 1) * LBLK); i += 64)
      n += sample_key(sample_load(a.scores, a.type, (long long)b * a.ld + i)) == c.cut;
    for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o, 64);
    if (lane == 0) g.tb[(long long)b * g.nblk + q] = (unsigned)n;
  }
}
struct TieRank {   // whether this lane's entry (one of 64 consecutive ones) stays
  SampleCut c; bool ranked; unsigned ties;
  __device__ __forceinline__ bool stays(unsigned k) {
    if (!ranked) return k > c.cut || (k == c.cut && k != 0u && c.ties != 0u);
    const u64 eq = __ballot(k == c.cut);
    const unsigned rank = ties + __popcll(eq & ((1ull << (threadIdx.x & 63)) - 1ull));
    ties += __popcll(eq);
    return k > c.cut || (k == c.cut && rank < c.ties);
  }
};
__device__ __forceinline__ unsigned ties_before(const unsigned* tb, int q) {   // a wave sums what lies in front of block q
  unsigned n = 0;
  for (int t = threadIdx.x & 63; t < q; t += 64) n += tb[t];
  for (int o = 1; o < 64; o <<= 1) n += (unsigned)__shfl_xor((int)n, o, 64);
  return n;
}
__global__ __launch_bounds__(256) void sample_sums_kernel(SampleArgs a, SampleLong g) {
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  SampleRow r;
  r.load(a, b);
  const SampleState* S = g.state + b;
  if (S->maxkey == 0u) return;
  r.set_max(S->maxkey);
  TieRank t{final_cut(S, r), false, 0u};
  t.ranked = t.c.ties != 0u && t.c.ties != ALL_TIES;
  for (int q = blockIdx.x * (LCH / LBLK) + wave; q < min(g.nblk, (int)(blockIdx.x + 1) * (LCH / LBLK)); q += 4) {
    if (t.ranked) t.ties = ties_before(g.tb + (long long)b * g.nblk, q);
    WSum v{0, 0};
#pragma unroll 4
    for (int j = 0; j < LBLK / 64; ++j) {
      const long long i = (long long)q * LBLK + 64 * j + lane;
      const unsigned k = i < a.N ? sample_key(sample_load(a.scores, a.type, (long long)b * a.ld + i)) : 0u;
      if (t.stays(k)) v.add(r.kept(k));
    }
    v = wave_total(v);
    if (lane == 0) {
      u64* o = g.bs + ((long long)b * g.nblk + q) * 2;
      o[0] = v.hi;
      o[1] = v.lo;
    }
  }
}
// a workgroup of one wave a draw
__global__ __launch_bounds__(64) void sample_draw_kernel(SampleArgs a, SampleLong g) {
  const int s = blockIdx.x, b = blockIdx.y, lane = threadIdx.x;
  const long long at = (long long)b * a.S + s;
  SampleRow r;
  r.load(a, b);
  const SampleState* S = g.state + b;
  if (S->maxkey == 0u) {
    if (lane == 0) { a.out_id[at] = -1; a.out_logp[at] = -INFINITY; }
    return;
  }
  r.set_max(S->maxkey);
  TieRank t{final_cut(S, r), false, 0u};
  t.ranked = t.c.ties != 0u && t.c.ties != ALL_TIES;
  const u64* bs = g.bs + (long long)b * g.nblk * 2;
  WSum sum{0, 0};
  for (int q = lane; q < g.nblk; q += 64) sum.add(WSum{bs[2 * q], bs[2 * q + 1]});
  const u128 W = wave_total(sum).all();
  const double log_W = log(wide_to_double(W) * 2.168404344971009e-19);   // 2^-62
  const u128 goal = sample_goal(a.rand[at], W);
  WSum run{0, 0};                       // in front of the 64 blocks, then of the block, then of the 64 entries
  int q = 0;
  for (;; q += 64) {
    const WSum v = q + lane < g.nblk ? WSum{bs[2 * (q + lane)], bs[2 * (q + lane) + 1]} : WSum{0, 0};
    const WSum up = wave_upto(v);
    WSum end = run;
    end.add(up);
    const u64 over = __ballot(end.all() > goal);
    const int from = over ? __ffsll(over) - 1 : 63;
    const WSum at_end{((u64)(unsigned)__shfl((int)(up.hi >> 32), from, 64) << 32) | (unsigned)__shfl((int)(unsigned)up.hi, from, 64),
                      ((u64)(unsigned)__shfl((int)(up.lo >> 32), from, 64) << 32) | (unsigned)__shfl((int)(unsigned)up.lo, from, 64)};
    const WSum last{((u64)(unsigned)__shfl((int)(v.hi >> 32), from, 64) << 32) | (unsigned)__shfl((int)(unsigned)v.hi, from, 64),
                    ((u64)(unsigned)__shfl((int)(v.lo >> 32), from, 64) << 32) | (unsigned)__shfl((int)(unsigned)v.lo, from, 64)};
    if (over || q + 64 >= g.nblk) {     // (goal < W: some block passes it)
      run.hi += at_end.hi - last.hi;
      run.lo += at_end.lo - last.lo;
      q = min(q + from, g.nblk - 1);
      break;
    }
    run.add(at_end);
  }
  if (t.ranked) t.ties = ties_before(g.tb + (long long)b * g.nblk, q);
  for (int j = 0; j < LBLK / 64; ++j) {
    const long long i = (long long)q * LBLK + 64 * j + lane;
    const unsigned k = i < a.N ? sample_key(sample_load(a.scores, a.type, (long long)b * a.ld + i)) : 0u;
    WSum v{0, 0};
    if (t.stays(k)) v.add(r.kept(k));
    const WSum up = wave_upto(v);
    WSum end = run;
    end.add(up);
    const u64 over = __ballot(end.all() > goal);
    if (over) {
      if (lane == __ffsll(over) - 1) {
        a.out_id[at] = a.ids ? a.ids[(long long)b * a.ld_ids + i] : i;
        a.out_logp[at] = r.greedy ? 0.f : (float)(r.z(k) - log_W);
      }
      return;
    }
    run.hi += ((u64)(unsigned)__shfl((int)(up.hi >> 32), 63, 64) << 32) | (unsigned)__shfl((int)(unsigned)up.hi, 63, 64);
    run.lo += ((u64)(unsigned)__shfl((int)(up.lo >> 32), 63, 64) << 32) | (unsigned)__shfl((int)(unsigned)up.lo, 63, 64);
  }
}

// ---- host
static inline int log2_up(long long n) {
  int k = 0;
  while ((1LL << k) < n) ++k;
  return k;
}
static inline bool sample_in_lds(long long N, int type) { return N <= (type == UR_F32 ? 32768 : 65536); }
static size_t sample_long_bytes(long long N, int B, char* base, SampleLong* g) {
  size_t o = 0;
  auto take = [&](size_t n) {
    char* p = base ? base + o : nullptr;
    o += (n + 255) & ~(size_t)255;
    return p;
  };
  SampleLong w{};
  w.nchunk = cdiv(N, LCH); w.nblk = cdiv(N, LBLK); w.coarse = log2_up(N);
  w.state = (SampleState*)take(sizeof(SampleState) * B);
  w.hc = (unsigned*)take((size_t)B * SB * 4); w.hw = (u64*)take((size_t)B * SB * 8);
  w.tb = (unsigned*)take((size_t)B * w.nblk * 4); w.bs = (u64*)take((size_t)B * w.nblk * 16);
  if (g) *g = w;
  return o;
}
template <int NT, bool RAW>
static int launch_sample_row(const SampleArgs& a, hipStream_t st) {
  const int nblk = cdiv(a.N, SBLK);
  const size_t lds = (size_t)SB * 12 + nblk * 16 + ((nblk + 3) & ~3) * 4 + (size_t)a.N * (RAW ? 2 : 4) + 16;
  static const hipError_t attr = hipFuncSetAttribute((const void*)sample_row_kernel<NT, RAW>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024 - 512);
  (void)attr;
  hipLaunchKernelGGL((sample_row_kernel<NT, RAW>), dim3(a.B), dim3(NT), lds, st, a, log2_up(a.N));
  UR_LAUNCH_CHECK();
  return UR_OK;
}

}  // namespace ur

using namespace ur;

extern "C" int64_t ur_sample_scores_workspace_bytes(int32_t score_type, int64_t n, int32_t B) {
  if (B <= 0 || n <= 0 || n >= (1LL << 31) || (score_type != UR_F32 && score_type != UR_F16 && score_type != UR_BF16)) return UR_ERR_ARG;
  return sample_in_lds(n, score_type) ? 0 : (int64_t)sample_long_bytes(n, B, nullptr, nullptr);
}

extern "C" int ur_sample_scores(const void* scores, int32_t score_type, int64_t n, int64_t ld, int32_t B, const float* rand, int32_t S,
                                double temperature, int32_t top_k, double top_p, double min_p, const float* temperature_rows,
                                const int32_t* top_k_rows, const float* top_p_rows, const float* min_p_rows, const int64_t* ids, int64_t ld_ids,
                                int64_t* out_id, float* out_logp, void* ws, void* stream) {
  UR_TRACE_SCOPE();
  UR_REQUIRE(scores && rand && out_id && out_logp, UR_ERR_ARG, "ur_sample_scores: null pointer");
  UR_REQUIRE(score_type == UR_F32 || score_type == UR_F16 || score_type == UR_BF16, UR_ERR_ARG, "ur_sample_scores: score_type=%d", score_type);
  UR_REQUIRE(B > 0 && S > 0 && n > 0 && n < (1LL << 31) && ld >= n && (!ids || ld_ids >= n), UR_ERR_ARG, "ur_sample_scores: shape");
  UR_REQUIRE(temperature >= 0.0 && temperature < INFINITY, UR_ERR_ARG, "ur_sample_scores: temperature=%g", temperature);
  UR_REQUIRE(top_k >= 0 && top_p > 0.0 && min_p >= 0.0 && min_p <= 1.0, UR_ERR_ARG, "ur_sample_scores: top_k=%d top_p=%g min_p=%g", top_k, top_p, min_p);
  const bool lds = sample_in_lds(n, score_type);
  UR_REQUIRE(lds || ws, UR_ERR_ARG, "ur_sample_scores: rows of %lld entries need a workspace", (long long)n);
  UR_REQUIRE(lds || B <= 65535, UR_ERR_UNSUPPORTED, "ur_sample_scores: B=%d rows of %lld entries (at most 65535 that long)", B, (long long)n);
  hipStream_t st = as_stream(stream);
  ProfScope ps(PC_MISC, st, (double)B * n * (score_type == UR_F32 ? 4 : 2));
  SampleArgs a{};
  a.scores = scores; a.type = score_type; a.N = n; a.ld = ld; a.B = B; a.S = S; a.rand = rand;
  a.T = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
  a.T_rows = temperature_rows; a.k_rows = top_k_rows; a.p_rows = top_p_rows; a.minp_rows = min_p_rows;
  a.ids = (const long long*)ids; a.ld_ids = ld_ids; a.out_id = (long long*)out_id; a.out_logp = out_logp;
  if (lds) {
    // (threads: about 8 entries each for short rows, whose passes are latency; 1 024 where the row is most of a CU's LDS anyway)
    if (n > 32768) return launch_sample_row<1024, true>(a, st);
    return n <= 2048 ? launch_sample_row<256, false>(a, st) : n <= 8192 ? launch_sample_row<512, false>(a, st) : launch_sample_row<1024, false>(a, st);
  }
  SampleLong g;
  sample_long_bytes(n, B, (char*)ws, &g);
  g.uses_k = top_k_rows || (top_k > 0 && top_k < n);
  g.uses_p = top_p_rows || top_p < 1.0;
  const dim3 grid(g.nchunk, B);
  const int mode = ur_arrive_mode();
  hipLaunchKernelGGL(sample_init_kernel, dim3(B), dim3(256), 0, st, a, g);
  UR_LAUNCH_CHECK();
  hipLaunchKernelGGL(sample_max_kernel, grid, dim3(256), 0, st, a, g);
  UR_LAUNCH_CHECK();
  for (int round = 0; round < ROUNDS && g.uses_k; ++round) {
    hipLaunchKernelGGL((sample_round_kernel<0>), grid, dim3(256), 0, st, a, g, round, mode);
    UR_LAUNCH_CHECK();
  }
  for (int round = 0; round < ROUNDS && g.uses_p; ++round) {
    hipLaunchKernelGGL((sample_round_kernel<1>), grid, dim3(256), 0, st, a, g, round, mode);
    UR_LAUNCH_CHECK();
  }
  if (g.uses_k || g.uses_p || temperature_rows || temperature == 0.0) {
    hipLaunchKernelGGL(sample_ties_kernel, grid, dim3(256), 0, st, a, g);
    UR_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(sample_sums_kernel, grid, dim3(256), 0, st, a, g);
  UR_LAUNCH_CHECK();
  hipLaunchKernelGGL(sample_draw_kernel, dim3(S, B), dim3(64), 0, st, a, g);
  UR_LAUNCH_CHECK();
  return UR_OK;
}
