// Sampling from scores with temperature, top-k, top-p and min-p, the random numbers given by the caller (beside eval.hip's top-k: an answer
// drawn from the distribution instead of its head).  Per row of N scores x:
//   z_n = (x_n - max x) / T, weight w_n = exp(z_n); NaN and -inf carry none; a row with +inf: those entries 1, the others 0
//   top-k: the first k in the order (score descending, index ascending); top-p: of those, in that order, every entry before which less
//   than p of their weight lies; min-p: w >= min_p.  The answer to u: the first index n, in INDEX order, with sum_{j <= n} kept w_j > u W.
// No sort: the order only decides a threshold (a key and how many of its ties stay).  It is found by a histogram over 2 048 equal steps of
// the score (steps of the key's upper bits put most scores into a few dozen bins, whose LDS atomics then queue: with those the whole call
// took 756 us for 64 rows of a million with top-p, 587 us with these and the comparison), and inside the step that the border falls into by
// comparing up to 128 keys directly, or by radix selection over 11, 11 and 10 bits of the key.
//
// Arithmetic.  Which entry a sum's border falls on is a whole number, so sums are exact: a weight is exp in double, rounded down
// once to a multiple of 2^-57 (2^-53 is a double's own step) and added as integers: 64 of them in 64 bits, more in two limbs.  (With top-p's sums
// in 64 bits, log2 N - 6 bits of every weight dropped, the border came out up to 900 entries off among a million equal ones 22 T below one.)  No
// result depends on an order of additions or on how a row was cut into pieces.
//
// Two forms.  A row that fits into LDS (32 768 entries; 65 536 of 16 bits): one workgroup, one read of the row, every pass from LDS.
// Longer rows: many workgroups a row, a pass over memory each for the maximum, for a selection's histogram and its border's step, and for the
// kept sums.  Bound: short rows by the latency of the passes (1 x 1 000: 16 us, 512 x 1 000: 17 us), long rows with top-p by vector
// instructions, 48 an entry for a weight and its sum: 0.76 of the cycles of the kept sums, 0.66 of the steps', whose weights also go through 64-bit
// LDS atomics (64 x 1 M fp32: 371 - 376 us, without selections 168 us); 256 x 60 K bf16 with all three filters: 65 us, a workgroup a row and its passes
// over LDS, one key a read (vector instructions in 0.50 of the cycles, the waves wait 0.59 of theirs).
#include <math.h>

#include <algorithm>
#include <type_traits>

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

// ascending unsigned order == ascending float order; -0 counts as 0 (equal scores tie), NaN and -inf are 0: no entry.
// Scores of 16 bits keep their own 16-bit image, in the upper half (the last 10-bit round of a selection falls away).
__device__ __forceinline__ unsigned key_f32(float x) {
  if (!(x > -INFINITY)) return 0u;
  const unsigned u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned key_16(unsigned u, int type) {
  const unsigned mag = u & 0x7FFFu, top = type == UR_F16 ? 0x7C00u : 0x7F80u;   // infinity
  if (mag > top || u == (0x8000u | top)) return 0u;
  if (mag == 0u) u = 0u;
  return ((u & 0x8000u) ? (~u & 0xFFFFu) : (u | 0x8000u)) << 16;
}
__device__ __forceinline__ float key_value(unsigned key, int type) {
  if (type == UR_F32) return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
  const unsigned k = key >> 16, u = (k & 0x8000u) ? (k & 0x7FFFu) : (~k & 0xFFFFu);
  return type == UR_F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)u) : __uint_as_float(u << 16);
}
// a score x (a number) lies above it where x's key lies above `key`; NaN or -inf: every number does.  The place of -0, which no entry
// has, is read as the number below it: 0 > -0 is false
__device__ __forceinline__ float cut_value(unsigned key, int type) {
  const unsigned low = type == UR_F32 ? 0x7FFFFFFFu : 0x7FFF0000u, mask = type == UR_F32 ? 0xFFFFFFFFu : 0xFFFF0000u;
  const float v = key_value((key & mask) == low ? (type == UR_F32 ? low - 1u : low - 0x10000u) : key, type);
  return v == v ? v : -INFINITY;
}
__device__ __forceinline__ unsigned sample_key(const void* p, int type, long long i) {
  return type == UR_F32 ? key_f32(((const float*)p)[i]) : key_16(((const unsigned short*)p)[i], type);
}

// 2^(z + 57), rounded down, z <= 0.  r = z - n in [-1/2, 1/2] (exact; n by adding 1.5 2^52), the Taylor polynomial of 2^r of degree 11
// (remainder 6 10^-15 of it, of the order of the rounding of z itself), 2^n and the fixed point by shifting the result's mantissa
constexpr int WBITS = 57;
__device__ __forceinline__ u64 exp2_fixed(double z) {
  constexpr double L = 0.69314718055994530942, MAGIC = 6755399441055744.0;
  constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6, c7 = c6 * L / 7, c8 = c7 * L / 8,
                   c9 = c8 * L / 9, c10 = c9 * L / 10, c11 = c10 * L / 11;
  z = fmax(z, -100.0);
  const double t = z + MAGIC;
  const int n = (int)(unsigned)__double_as_longlong(t);
  const double r = z - (t - MAGIC);
  double p = fma(c11, r, c10);
  p = fma(p, r, c9);
  p = fma(p, r, c8);
  p = fma(p, r, c7);
  p = fma(p, r, c6);
  p = fma(p, r, c5);
  p = fma(p, r, c4);
  p = fma(p, r, c3);
  p = fma(p, r, c2);
  p = fma(p, r, L);
  p = fma(p, r, 1.0);
  const unsigned hi = (unsigned)((u64)__double_as_longlong(p) >> 32), lo = (unsigned)__double_as_longlong(p);   // p in [0.7, 1.5)
  const unsigned down = min(1023u - (hi >> 20) - (unsigned)n, 63u);                                             // 0 for z = 0; 63: nothing is left
  const u64 mant = ((u64)((hi & 0xFFFFFu) | 0x100000u) << 32) | lo;
  return (mant << (WBITS - 52)) >> down;
}
// a row's parameters
struct SampleRow {
  double scale, inv_T, p, min_z; long long k; int type; bool greedy, tiny, flat;   // scale: log2(e) / T
  float m;
  __device__ __forceinline__ void load(const SampleArgs& a, int b) {
    const double T = a.T_rows ? (double)a.T_rows[b] : a.T;
    double min_p = a.minp_rows ? (double)a.minp_rows[b] : a.min_p;
    p = a.p_rows ? (double)a.p_rows[b] : a.top_p;
    k = a.k_rows ? a.k_rows[b] : a.top_k;
    type = a.type;
    if (k <= 0) k = a.N;
    greedy = !(T > 0.0);                 // the first of the largest
    tiny = !(T > 1e-300);                // (1 / T stays finite) nothing but the largest has weight: two floats differ by 1e-45 at least
    inv_T = tiny ? 1.0 : 1.0 / T;
    scale = tiny ? 1.0 : 1.4426950408889634 / T;
    if (!(min_p < 1.0)) min_p = 1.0;     // (the largest stays)
    min_z = min_p > 0.0 ? log2(min_p) : -INFINITY;
  }
  __device__ __forceinline__ void set_max(unsigned key) { m = key_value(key, type); flat = tiny || m == INFINITY; }
  __device__ __forceinline__ double z(unsigned key) const {
    const float x = key_value(key, type);
    if (flat) return x == m ? 0.0 : -INFINITY;
    return ((double)x - (double)m) * inv_T;
  }
  __device__ __forceinline__ double z2(unsigned key) const {     // log2 of the weight
    const float x = key_value(key, type);
    if (flat) return x == m ? 0.0 : -INFINITY;
    return ((double)x - (double)m) * scale;
  }
  __device__ __forceinline__ u64 weight(unsigned key) const { return exp2_fixed(z2(key)); }
  // the smallest key that min-p leaves, searched by a wave, 64 keys at a time
  __device__ __forceinline__ unsigned min_key(unsigned mk) const {
    if (!(min_z > -INFINITY)) return 1u;
    const unsigned lane = threadIdx.x & 63;
    unsigned lo = 1u, hi = mk;
    while (lo < hi) {
      const unsigned probe = lo + (unsigned)(((u64)(hi - lo) * lane) >> 6);
      const u64 in = __ballot(z2(probe) >= min_z);
      if (in == 0ull) {
        lo = (unsigned)__builtin_amdgcn_readlane((int)probe, 63) + 1u;
      } else {
        const int f = __builtin_amdgcn_readfirstlane(__ffsll(in) - 1);
        hi = (unsigned)__builtin_amdgcn_readlane((int)probe, f);
        if (f > 0) lo = (unsigned)__builtin_amdgcn_readlane((int)probe, f - 1) + 1u;
      }
    }
    return hi;
  }
};
// entries above `cut` stay, and of those equal to it the first `ties` in index order
struct SampleCut { unsigned cut; unsigned ties; };
constexpr unsigned ALL_TIES = 0xFFFFFFFFu;
__device__ __forceinline__ SampleCut inside(SampleCut c, SampleCut outer) {   // a cut made among what `outer` left never lets more in: ties that all
  return c.cut < outer.cut ? outer : c;                                        // stay are those that `outer` left of them, not all of the row's
}
__device__ __forceinline__ SampleCut above_min_p(SampleCut c, unsigned min_key) {   // and what min-p leaves of them
  return min_key > 1u && min_key > c.cut ? SampleCut{min_key - 1u, 0u} : c;
}

struct WSum {   // a sum of weights
  u64 hi, lo;
  __device__ __forceinline__ void add(u64 w) { hi += w >> 32; lo += w & 0xFFFFFFFFull; }
  __device__ __forceinline__ void add(const WSum& o) { hi += o.hi; lo += o.lo; }
  __device__ __forceinline__ u128 all() const { return ((u128)hi << 32) + lo; }
};
// inclusive sums over the lanes of a wave, in lane order: DPP moves (row_shr 1, 2, 4, 8, then lane 15 / 31 of the rows before), VALU rate
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned dpp_from(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_from(u64 v) { return ((u64)dpp_from<CTRL, ROWS>((unsigned)(v >> 32)) << 32) | dpp_from<CTRL, ROWS>((unsigned)v); }
template <typename T>
__device__ __forceinline__ T wave_upto(T v) {
  v += dpp_from<0x111, 0xF>(v);
  v += dpp_from<0x112, 0xF>(v);
  v += dpp_from<0x114, 0xF>(v);
  v += dpp_from<0x118, 0xF>(v);
  v += dpp_from<0x142, 0xA>(v);
  v += dpp_from<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ u64 at_lane(u64 v, int lane) {
  return ((u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, lane);
}
__device__ __forceinline__ unsigned last_lane(unsigned v) { return (unsigned)__builtin_amdgcn_readlane((int)v, 63); }
__device__ __forceinline__ u64 last_lane(u64 v) { return ((u64)last_lane((unsigned)(v >> 32)) << 32) | last_lane((unsigned)v); }
template <typename T>
__device__ __forceinline__ T wave_total(T v) { return last_lane(wave_upto(v)); }
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
  return v;
}
// over the workgroup, in thread order: the sum in front of a thread, and the sum of all.  tmp[NT / 64]
template <int NT, typename T>
__device__ __forceinline__ T block_before(T v, T* tmp, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T s = wave_upto(v);
  __syncthreads();
  if (lane == 63) tmp[wave] = s;
  __syncthreads();
  T base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    const T t = tmp[w];
    if (w < wave) base += t;
    all += t;
  }
  *total = all;
  return base + s - v;
}
template <int NT>
__device__ __forceinline__ WSum block_before(const WSum& v, u64* tmp, WSum* total) {   // tmp[2 NT / 64]: both limbs between the same two barriers
  constexpr int NW = NT / 64;
  const int lane = threadIdx.x & 63, wave = NW <= 4 ? (int)(threadIdx.x >> 6) : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const WSum s{wave_upto(v.hi), wave_upto(v.lo)};
  __syncthreads();
  if (lane == 63) { tmp[wave] = s.hi; tmp[NW + wave] = s.lo; }
  __syncthreads();
  WSum r{s.hi - v.hi, s.lo - v.lo};
  if constexpr (NW <= 4) {
    *total = WSum{0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const WSum t{tmp[w], tmp[NW + w]};
      r.add(WSum{w < wave ? t.hi : 0, w < wave ? t.lo : 0});
      total->add(t);
    }
  } else {
    const WSum t{wave_upto(lane < NW ? tmp[lane] : 0ull), wave_upto(lane < NW ? tmp[NW + lane] : 0ull)};   // the waves' sums, a lane each
    *total = WSum{at_lane(t.hi, NW - 1), at_lane(t.lo, NW - 1)};
    if (wave > 0) r.add(WSum{at_lane(t.hi, wave - 1), at_lane(t.lo, wave - 1)});
  }
  return r;
}
__device__ __forceinline__ double wide_to_double(u128 v) {     // v < 2^88 (2^31 weights)
  return fma((double)(unsigned)(v >> 64), 18446744073709551616.0, (double)(u64)v);
}
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
__device__ __forceinline__ unsigned ties_within(u128 above, u64 w, double limit, unsigned most) {
  if (w == 0) return most;
  unsigned lo = 1, hi = most;           // the first j in [1, most] that does not stay
  while (lo < hi) {
    const unsigned mid = lo + (hi - lo) / 2;
    if (wide_to_double(above + (u128)w * mid) < limit) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// ---- a selection: a histogram over equal steps of the score (round -1), then rounds over the bits of the keys of one step
constexpr int SB = 2048, SBP = SB + 8;   // bins; their room in LDS
struct Steps {   // step of a score: (max / 2 - x / 2) c, never larger for a larger score (fp32 rounding keeps an order); halves: no difference overflows
  float half_m, c; float m; int type; bool flat;
  __device__ __forceinline__ void set(const SampleRow& r, unsigned minkey, bool weights) {
    m = r.m; type = r.type; flat = r.flat;
    half_m = 0.5f * m;
    double range = 0.5 * ((double)r.m - (double)key_value(minkey, r.type));
    if (weights) range = fmin(range, 21.5 / r.inv_T);            // (steps behind 43 T weigh nothing: one bin)
    c = range > 0.0 ? (float)fmin((double)SB / range, 1e38) : 0.f;
  }
  __device__ __forceinline__ int of(unsigned key) const { return of_value(key_value(key, type)); }
  __device__ __forceinline__ int of_value(float x) const {
    if (flat) return x == m ? 0 : SB - 1;
    const float t = fmaf(x, -0.5f, half_m) * c;
    return t < (float)(SB - 1) ? (int)t : SB - 1;                // (a pattern that is no number: the last)
  }
};
// the smallest key whose step is at most s, searched by a wave, 64 keys at a time (mk's step is 0)
__device__ __forceinline__ unsigned first_key(const Steps& steps, int s, unsigned mk) {
  const unsigned lane = threadIdx.x & 63;
  unsigned lo = 1u, hi = mk;
  while (lo < hi) {
    const unsigned probe = lo + (unsigned)(((u64)(hi - lo) * lane) >> 6);
    const u64 in = __ballot(steps.of(probe) <= s);
    if (in == 0ull) {
      lo = (unsigned)__builtin_amdgcn_readlane((int)probe, 63) + 1u;
    } else {
      const int f = __builtin_amdgcn_readfirstlane(__ffsll(in) - 1);
      hi = (unsigned)__builtin_amdgcn_readlane((int)probe, f);
      if (f > 0) lo = (unsigned)__builtin_amdgcn_readlane((int)probe, f - 1) + 1u;
    }
  }
  return hi;
}
__device__ __forceinline__ int round_shift(int round) { return round == 0 ? 21 : round == 1 ? 10 : 0; }
__device__ __forceinline__ int round_place(unsigned key, int round) {   // from the highest key down
  return SB - 1 - (int)((key >> round_shift(round)) & (round == 2 ? 1023u : 2047u));
}
__device__ __forceinline__ unsigned round_prefix(unsigned prefix, int round, int place) {
  const unsigned d = (unsigned)(SB - 1 - place);
  return round == 0 ? d : (prefix << (round == 1 ? 11 : 10)) | d;
}
__device__ __forceinline__ bool round_in(unsigned key, int round, unsigned prefix) {
  return round == 0 || (round == 1 ? key >> 21 : key >> 10) == prefix;
}
struct Select {   // state of a selection (one per row)
  int step; unsigned lo, hi;            // the border's step, its keys [lo, hi]
  unsigned prefix, count;               // the key's bits so far, and the entries that share them
  unsigned need;                        // top-k: how many of those stay
  u128 above; double limit;             // top-p: the weight in front of them, p times all of it
  unsigned done;
};
// bins lie in the order of the threads that sum them: thread t of NT takes places t SB / NT .. , place j of them at j (NT + 1) + t (a bank apart:
// scores next to each other fall into places next to each other)
template <int NT>
__device__ __forceinline__ int bin_at(int place) {
  constexpr int PB = SB / NT;
  return (place % PB) * (NT + 1) + place / PB;
}
// a bin of weights: 64 bits and, in units of 2^HI, 32 more.  Up to 65 536 entries go in without a carry (HI 42: a weight below 2^64 / entries into the
// lower part, of a larger one its last 42 bits); any number of them with one (HI 64)
constexpr int BIN_HI = 42;
__device__ __forceinline__ unsigned large_from(unsigned entries) { return entries > 128u ? 1u << __clz(entries - 1u) : 1u << 25; }   // 2^(64 - log2), upper word
__device__ __forceinline__ void add_weight(u64* lo, unsigned* hi, u64 w, unsigned times, unsigned large) {
  if ((unsigned)(w >> 32) >= large) {
    atomicAdd(hi, (unsigned)(w >> BIN_HI) * times);
    w &= (1ull << BIN_HI) - 1ull;
  }
  atomicAdd(lo, w * times);
}
__device__ __forceinline__ void add_wide(u64* lo, unsigned* hi, u128 v) {
  const u64 w = (u64)v, old = atomicAdd(lo, w);
  const unsigned up = (unsigned)(v >> 64) + (old + w < old);
  if (up) atomicAdd(hi, up);
}
// the place that the border falls into, found by the whole workgroup; updates st, sets cut when it is final.
// `last`: no key of this type has bits below this round's
template <int NT>
__device__ __forceinline__ void pick_k(int round, bool last, const unsigned* hc, Select* st, SampleCut* cut, unsigned* tmp) {
  constexpr int PB = SB / NT;
  const unsigned need = st->need, prefix = st->prefix;
  unsigned mine[PB], sum = 0, total;
#pragma unroll
  for (int j = 0; j < PB; ++j) { mine[j] = hc[j * (NT + 1) + threadIdx.x]; sum += mine[j]; }
  unsigned before = block_before<NT>(sum, tmp, &total);
  if (before < need && need <= before + sum) {
#pragma unroll
    for (int j = 0; j < PB; ++j) {
      if (before < need && need <= before + mine[j]) {
        const int place = (int)threadIdx.x * PB + j;
        const unsigned rest = need - before;
        st->need = rest;
        st->count = mine[j];
        if (round < 0) st->step = place;
        else {
          const unsigned q = round_prefix(prefix, round, place);
          st->prefix = q;
          if (last) {                   // one key: all of its entries, or the first of them
            const unsigned key = q << round_shift(round);
            cut->cut = rest == mine[j] ? key - 1u : key;
            cut->ties = rest == mine[j] ? 0u : rest;
            st->done = 1u;
          }
        }
      }
      before += mine[j];
    }
  } else if (threadIdx.x == 0 && total < need) {
    st->done = 1u;                      // fewer entries than k: nothing is cut
  }
  __syncthreads();
}
// the bins' weights in hw and hc (see add_weight)
template <int NT, int HI>
__device__ __forceinline__ void pick_p(int round, const unsigned* hc, const u64* hw, double p, Select* st, u64* tmp) {
  constexpr int PB = SB / NT;
  const unsigned prefix = st->prefix;
  const u128 above = st->above;
  const double given = st->limit;
  auto in_bin = [&](int j) { return ((u128)hc[j * (NT + 1) + threadIdx.x] << HI) + hw[j * (NT + 1) + threadIdx.x]; };
  u128 here = 0;
  WSum total;
#pragma unroll
  for (int j = 0; j < PB; ++j) here += in_bin(j);
  u128 before = block_before<NT>(WSum{(u64)(here >> 32), (u64)here & 0xFFFFFFFFull}, tmp, &total).all() + above;
  const double limit = round < 0 ? p * wide_to_double(total.all()) : given;
  // the first entry of exactly one bin is the last whose forerunners weigh less than the limit
  if (wide_to_double(before) < limit && !(wide_to_double(before + here) < limit)) {
    u128 mine[PB];                      // (read again: not worth registers across the sums)
#pragma unroll
    for (int j = 0; j < PB; ++j) mine[j] = in_bin(j);
    int found = 0;
    u128 upto = before;
#pragma unroll
    for (int j = 0; j < PB - 1; ++j) {
      upto += mine[j];
      if (wide_to_double(upto) < limit) { before = upto; ++found; }
    }
    const int place = (int)threadIdx.x * PB + found;
    st->above = before;
    st->limit = limit;
    if (round < 0) st->step = place;
    else st->prefix = round_prefix(prefix, round, place);
  }
  __syncthreads();
}
// the last round: hc are the entries of one key a bin, weight(key) each
template <int NT, typename W>
__device__ __forceinline__ void pick_p_key(int round, const unsigned* hc, const W& weight, Select* st, SampleCut* cut, u64* tmp) {
  constexpr int PB = SB / NT;
  const unsigned prefix = st->prefix;
  const u128 above = st->above;
  const double limit = st->limit;
  auto key_of = [&](int j) { return round_prefix(prefix, round, (int)threadIdx.x * PB + j) << round_shift(round); };
  auto in_bin = [&](int j) -> u128 {
    const unsigned c = hc[j * (NT + 1) + threadIdx.x];
    return c ? (u128)weight(key_of(j)) * c : 0;
  };
  u128 here = 0;
#pragma unroll 1
  for (int j = 0; j < PB; ++j) here += in_bin(j);
  WSum total;
  u128 before = block_before<NT>(WSum{(u64)(here >> 32), (u64)here & 0xFFFFFFFFull}, tmp, &total).all() + above;
  if (wide_to_double(before) < limit && !(wide_to_double(before + here) < limit)) {
#pragma unroll 1
    for (int j = 0; j < PB; ++j) {
      const u128 mine = in_bin(j);
      if (!(wide_to_double(before + mine) < limit)) {
        const unsigned n = hc[j * (NT + 1) + threadIdx.x], key = key_of(j), t = ties_within(before, weight(key), limit, n);
        cut->cut = t == n ? key - 1u : key;
        cut->ties = t == n ? 0u : t;
        st->done = 1u;
        break;
      }
      before += mine;
    }
  }
  __syncthreads();
}
// the keys of the step that the border fell into (two waves, a barrier)
__device__ __forceinline__ void step_keys(const Steps& steps, unsigned mk, Select* st) {
  const int wave = threadIdx.x >> 6, at = st->step;
  if (wave == 0) {
    const unsigned lo = first_key(steps, at, mk);
    if (threadIdx.x == 0) st->lo = lo;
  } else if (wave == 1) {
    const unsigned above = at > 0 ? first_key(steps, at - 1, mk) : 0u;
    if (threadIdx.x == 64) st->hi = at > 0 ? above - 1u : mk;
  }
  __syncthreads();
}
// the border among `n` <= DIRECT keys of one step, compared with each other (lists padded with key 0 to a multiple of 8)
constexpr int DIRECT = 128;
__device__ __forceinline__ void direct_k(const unsigned* keys, int n, const Select* st, SampleCut* cut) {
  if ((int)threadIdx.x < n) {
    const unsigned mine = keys[threadIdx.x], need = st->need;
    unsigned above = 0, equal = 0;
    for (int j = 0; j < n; j += 8) {
      const uint4 u = *(const uint4*)(keys + j), v = *(const uint4*)(keys + j + 4);
      const unsigned k[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int q = 0; q < 8; ++q) { above += k[q] > mine; equal += k[q] == mine; }
    }
    if (above < need && need <= above + equal) {                 // (threads of equal keys write the same)
      const bool all = need == above + equal;
      cut->cut = all ? mine - 1u : mine;
      cut->ties = all ? 0u : need - above;
    }
  }
  __syncthreads();
}
__device__ __forceinline__ void direct_p(const unsigned* keys, const u64* wgt, int n, const Select* st, SampleCut* cut) {
  if ((int)threadIdx.x < n) {
    const unsigned mine = keys[threadIdx.x];
    const u64 w = wgt[threadIdx.x];
    u64 larger = 0;                     // (of at most 127 others, 2^57 each)
    unsigned equal = 0;
    for (int j = 0; j < n; j += 8) {
      const uint4 u = *(const uint4*)(keys + j), v = *(const uint4*)(keys + j + 4);
      const unsigned k[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
      u64 x[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = wgt[j + q];
#pragma unroll
      for (int q = 0; q < 8; ++q) { larger += k[q] > mine ? x[q] : 0; equal += k[q] == mine; }
    }
    const double limit = st->limit;
    const u128 front = st->above + larger;
    if (wide_to_double(front) < limit && !(wide_to_double(front + (u128)w * equal) < limit)) {
      const unsigned t = ties_within(front, w, limit, equal);
      cut->cut = t == equal ? mine - 1u : mine;
      cut->ties = t == equal ? 0u : t;
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------------------------- rows that fit into LDS
constexpr int SLIST = 2048;
// Thread t owns the entries [t C, (t + 1) C): sums in index order are one scan over the threads.  When top-k leaves few entries they are
// copied out, in order, and everything behind it works on the copy.  A draw falls to one thread's entries; a wave looks at them together.
template <int NT, bool RAW>
__global__ __launch_bounds__(NT, 4) void sample_row_kernel(SampleArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int NWV = NT / 64, LAST = RAW ? 1 : 2;
  u64* hw = (u64*)smem;                                          // [SBP]; the copied entries on their way
  unsigned* hc = (unsigned*)(hw + SBP);                          // [SBP]
  unsigned* keys = hc + SBP;                                     // [N] (RAW: 16 bits each); then the copied entries, keys and indices
  unsigned short* keys16 = (unsigned short*)keys;
  __shared__ u64 tmp64[2 * NWV];
  __shared__ unsigned tmp32[NWV], s_min[NWV], s_n;
  __shared__ Select st;
  __shared__ SampleCut cut_s;
  __shared__ __attribute__((aligned(16))) unsigned near_k[DIRECT];
  __shared__ u64 near_w[DIRECT];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, N = (int)a.N;
  const long long base = (long long)b * a.ld;
  constexpr int DRAWS = 4;              // draws that a wave takes at a time
  const float u_first = lane < DRAWS && wave * DRAWS + lane < a.S ? a.rand[(long long)b * a.S + wave * DRAWS + lane] : 0.f;   // asked for early
  SampleRow r;
  r.load(a, b);
  int n = N;                            // entries in hand
  bool copied = false;
  auto key_at = [&](int i) -> unsigned {
    if constexpr (RAW) {
      if (!copied) return (unsigned)keys16[i] << 16;
    }
    return keys[i];
  };
  unsigned mk = 0u, least = 0xFFFFFFFFu;
  auto seen = [&](unsigned k) {
    mk = max(mk, k);
    if (k != 0u) least = min(least, k);
  };
  if constexpr (RAW) {
    const unsigned short* x = (const unsigned short*)a.scores + base;
    const int head = (int)min((long long)N, (long long)((8 - (((unsigned long long)x >> 1) & 7)) & 7));   // entries in front of a 16-byte boundary
    auto put = [&](int i, unsigned u) {
      const unsigned k = key_16(u, a.type);
      keys16[i] = (unsigned short)(k >> 16);
      seen(k);
    };
    if (tid < head) put(tid, x[tid]);
    const int wide = (N - head) / 8;
#pragma unroll 4
    for (int i = tid; i < wide; i += NT) {
      const uint4 v = *(const uint4*)(x + head + 8 * i);
      const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) { put(head + 8 * i + 2 * j, u[j] & 0xFFFFu); put(head + 8 * i + 2 * j + 1, u[j] >> 16); }
    }
    if (tid < N - head - 8 * wide) put(head + 8 * wide + tid, x[head + 8 * wide + tid]);
  } else {
    const float* x = (const float*)a.scores + base;
#pragma unroll 8
    for (int i = tid; i < N; i += NT) {
      const unsigned k = key_f32(x[i]);
      keys[i] = k;
      seen(k);
    }
  }
  mk = wave_max(mk);
  least = ~wave_max(~least);
  if (lane == 0) { tmp32[wave] = mk; s_min[wave] = least; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NWV; ++w) { mk = max(mk, tmp32[w]); least = min(least, s_min[w]); }
  if (mk == 0u) {                       // nothing to choose from
    for (int s = tid; s < a.S; s += NT) {
      a.out_id[(long long)b * a.S + s] = -1;
      a.out_logp[(long long)b * a.S + s] = -INFINITY;
    }
    return;
  }
  r.set_max(mk);
  SampleCut c{0u, ALL_TIES};            // (key 0: no entry)
  auto ranked = [&]() { return c.ties != 0u && c.ties != ALL_TIES; };
  auto span = [&]() { return ((n + NT - 1) / NT) | 1; };         // (odd: 64 threads a span apart are in 64 banks)
  auto in_front = [&](int i0, int i1) -> unsigned {              // ties in front of this thread's entries
    unsigned eq = 0, total;
    for (int i = i0; i < i1; ++i) eq += key_at(i) == c.cut;
    return block_before<NT>(eq, tmp32, &total);
  };
  auto stays = [&](unsigned k, unsigned& rank) -> bool {         // entries in order; rank = ties so far
    if (k > c.cut) return true;
    return k == c.cut && k != 0u && rank++ < c.ties;
  };
  Steps steps;
  if (r.greedy) {
    c.cut = mk;
    c.ties = 1u;
  } else {
    if (r.k < N) {
      steps.set(r, least, false);
      if (tid == 0) { st = Select{0, 0u, 0u, 0u, 0u, (unsigned)r.k, 0, 0.0, 0u}; cut_s = c; s_n = 0u; }
      if (tid < DIRECT) near_k[tid] = 0u;
      for (int round = -1; round <= LAST; ++round) {
        for (int i = tid; i < SBP; i += NT) hc[i] = 0u;
        __syncthreads();
        const unsigned prefix = st.prefix, lo = st.lo, hi = st.hi;
        if (round < 0) {
#pragma unroll 4
          for (int i = tid; i < N; i += NT) {
            const unsigned k = key_at(i);
            if (k != 0u) atomicAdd(&hc[bin_at<NT>(steps.of(k))], 1u);
          }
        } else {
#pragma unroll 4
          for (int i = tid; i < N; i += NT) {
            const unsigned k = key_at(i);
            if (k >= lo && k <= hi && round_in(k, round, prefix)) atomicAdd(&hc[bin_at<NT>(round_place(k, round))], 1u);
          }
        }
        __syncthreads();
        pick_k<NT>(round, round == LAST, hc, &st, &cut_s, tmp32);
        if (st.done) break;
        if (round < 0) step_keys(steps, mk, &st);
        if (round < 0 && st.count <= DIRECT) {
          const unsigned lo = st.lo, hi = st.hi;
#pragma unroll 4
          for (int i = tid; i < N; i += NT) {
            const unsigned k = key_at(i);
            if (k >= lo && k <= hi) near_k[atomicAdd(&s_n, 1u)] = k;
          }
          __syncthreads();
          direct_k(near_k, (int)st.count, &st, &cut_s);
          break;
        }
      }
      c = cut_s;
      __syncthreads();
      if (r.k <= SLIST && 4 * r.k <= N && c.cut != 0u) {         // exactly k entries are left: copy them out (through hw: they may overlap the row)
        const int C = span(), i0 = min(N, tid * C), i1 = min(N, i0 + C);
        unsigned rank = ranked() ? in_front(i0, i1) : 0u, count = 0, total;
        const unsigned rank0 = rank;
        for (int i = i0; i < i1; ++i) count += stays(key_at(i), rank);
        unsigned at = block_before<NT>(count, tmp32, &total);
        unsigned* list = (unsigned*)hw;                          // [2 SLIST]: key, index
        rank = rank0;
        if (count)
          for (int i = i0; i < i1; ++i) {
            const unsigned k = key_at(i);
            if (stays(k, rank)) { list[2 * at] = k; list[2 * at + 1] = (unsigned)i; ++at; }
          }
        __syncthreads();
        n = (int)total;
        for (int i = tid; i < n; i += NT) { keys[i] = list[2 * i]; keys[n + i] = list[2 * i + 1]; }
        copied = true;
        c = SampleCut{0u, ALL_TIES};
        __syncthreads();
      }
    }
    if (r.p < 1.0) {
      steps.set(r, least, true);
      if (tid == 0) { st = Select{0, 1u, mk, 0u, 0u, 0u, 0, 0.0, 0u}; cut_s = SampleCut{mk, 1u}; s_n = 0u; }   // (p <= 0: the largest alone)
      if (tid < DIRECT) { near_k[tid] = 0u; near_w[tid] = 0; }
      const unsigned large = large_from((unsigned)n);
      const bool few = n <= DIRECT && copied;                    // no histogram: all of them are compared
      auto gather = [&]() {                                      // the keys of the border's step (few: all), as many as can be compared
        const unsigned lo = st.lo, hi = st.hi;
        auto add = [&](unsigned k) {
          const unsigned q = atomicAdd(&s_n, 1u);
          if (q < DIRECT) { near_k[q] = k; near_w[q] = r.weight(k); }
        };
        for (int i = tid; i < n; i += NT) {
          const unsigned k = key_at(i);
          if (k > c.cut && k >= lo && k <= hi) add(k);
        }
        if (tid == 0 && c.cut != 0u && c.ties != 0u && c.cut >= lo && c.cut <= hi)
          for (unsigned t = 0; t < min(c.ties, (unsigned)DIRECT + 1u); ++t) add(c.cut);
        __syncthreads();
      };
      if (few) __syncthreads();                                  // (st)
      for (int round = few ? LAST + 1 : -1; round <= LAST && r.p > 0.0; ++round) {
        for (int i = tid; i < SBP; i += NT) { hc[i] = 0u; hw[i] = 0; }
        __syncthreads();
        const unsigned prefix = st.prefix, lo = st.lo, hi = st.hi;
        auto count = [&](unsigned k, unsigned times) {
          if (round >= 0 && !(k >= lo && k <= hi && round_in(k, round, prefix))) return;
          const int d = bin_at<NT>(round < 0 ? steps.of(k) : round_place(k, round));
          if (round == LAST) atomicAdd(&hc[d], times);
          else add_weight(hw + d, hc + d, r.weight(k), times, large);
        };
        for (int i = tid; i < n; i += NT) {
          const unsigned k = key_at(i);
          if (k > c.cut) count(k, 1u);
        }
        if (tid == 0 && c.cut != 0u && c.ties != 0u) count(c.cut, c.ties);   // the ties that top-k left
        __syncthreads();
        if (round == LAST) pick_p_key<NT>(round, hc, [&](unsigned k) { return r.weight(k); }, &st, &cut_s, tmp64);
        else pick_p<NT, BIN_HI>(round, hc, hw, r.p, &st, tmp64);
        if (round < 0) {
          step_keys(steps, mk, &st);
          gather();
          if (s_n <= DIRECT) break;
        }
        if (st.done) break;
      }
      if (few) gather();
      __syncthreads();
      if (r.p > 0.0 && !st.done) {
        if (few) {                                               // the limit: p times all of it
          WSum one{0, 0}, total;
          if (tid < DIRECT) one.add(near_w[tid]);
          block_before<NT>(one, tmp64, &total);
          if (tid == 0) st.limit = r.p * wide_to_double(total.all());
          __syncthreads();
        }
        direct_p(near_k, near_w, (int)s_n, &st, &cut_s);
      }
      c = inside(cut_s, c);
      __syncthreads();
    }
  }
  c = above_min_p(c, r.min_key(mk));
  // ---- the kept weight in front of every thread's entries
  const int C = span(), i0 = min(n, tid * C), i1 = min(n, i0 + C);
  const unsigned rank0 = ranked() ? in_front(i0, i1) : 0u;
  unsigned rank = rank0;
  WSum mine{0, 0}, all;
  {
    u64 sum = 0;                        // (at most 65 entries of at most 2^57)
    for (int i = i0; i < i1; ++i) {
      const unsigned k = key_at(i);
      if (stays(k, rank)) sum += r.weight(k);
    }
    mine.add(sum);
  }
  const WSum front = block_before<NT>(mine, tmp64, &all);
  const u128 W = all.all();
  const double log_W = log(wide_to_double(W) * 6.938893903907228e-18);   // 2^-57
  u64* from_hi = hw;                                             // [NT] (the histograms are done with): what lies in front of a thread's entries
  u64* from_lo = hw + NT;                                        // [NT]
  unsigned* ranks = hc;                                          // [NT]
  from_hi[tid] = front.hi;
  from_lo[tid] = front.lo;
  ranks[tid] = rank0;
  __syncthreads();
  // a wave takes a few draws, a lane of it finds the thread that a goal falls to (the last that does not begin behind it); then the wave looks
  // at 64 of that thread's entries at a time, draw after draw
  for (int s0 = wave * DRAWS; s0 < a.S; s0 += NWV * DRAWS) {
    const int ns = min(DRAWS, a.S - s0);
    u128 my_goal = 0;
    int owner = 0;
    if (lane < ns) {
      my_goal = sample_goal(s0 == wave * DRAWS ? u_first : a.rand[(long long)b * a.S + s0 + lane], W);
#pragma unroll
      for (int o = NT / 2; o > 0; o >>= 1)
        if (WSum{from_hi[owner + o], from_lo[owner + o]}.all() <= my_goal) owner += o;
    }
    for (int s = 0; s < ns; ++s) {
      const int t = __builtin_amdgcn_readlane(owner, s);
      const u128 goal = ((u128)(((u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(my_goal >> 96), s) << 32) |
                                (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(my_goal >> 64), s)) << 64) |
                        (((u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(my_goal >> 32), s) << 32) |
                         (unsigned)__builtin_amdgcn_readlane((int)(unsigned)my_goal, s));
      u128 run = WSum{from_hi[t], from_lo[t]}.all();
      const int j0 = min(n, t * C), j1 = min(n, j0 + C);
      unsigned ties = ranks[t];
      for (int j = j0; j < j1; j += 64) {
        const int i = j + lane;
        const unsigned k = i < j1 ? key_at(i) : 0u;
        const u64 eq = __ballot(k == c.cut && k != 0u);
        unsigned my_rank = ties + (unsigned)__popcll(eq & ((1ull << lane) - 1ull));
        ties += (unsigned)__popcll(eq);
        WSum v{0, 0};
        if (stays(k, my_rank)) v.add(r.weight(k));
        const WSum up{wave_upto(v.hi), wave_upto(v.lo)};
        const u64 over = __ballot(run + up.all() > goal);
        if (over) {
          if (lane == __ffsll(over) - 1) {
            const long long at = copied ? (long long)keys[n + i] : i, o = (long long)b * a.S + s0 + s;
            a.out_id[o] = a.ids ? a.ids[(long long)b * a.ld_ids + at] : at;
            a.out_logp[o] = r.greedy ? 0.f : (float)(r.z(k) - log_W);
          }
          break;
        }
        run += WSum{last_lane(up.hi), last_lane(up.lo)}.all();
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- longer rows
constexpr int LBLK = 2048;                // entries of a block of the kept sums
struct SampleState {                      // per row, in the workspace
  Select st;
  SampleCut cut;                          // of the selections so far
  SampleCut kcut;                         // of top-k (the top-p rounds need it)
  unsigned maxkey, minkey, arrived, listed;   // listed: entries of the border's step in the list
};
constexpr int LLIST = 8192;                   // a row's list
struct SampleLong {
  SampleState* state; unsigned* hc; u64* hw;   // [B], [B][SBP], [B][SBP]
  unsigned* tb; u64* bs;                       // [B][nblk] ties of a block, [B][2 nblk] kept weight of a block
  unsigned* list;                              // [B][LLIST] keys of the border's step
  int nblk, nchunk;
  int chunk;                                   // entries of a workgroup, a multiple of 4 096
  int uses_k, uses_p;
};

__global__ __launch_bounds__(256) void sample_init_kernel(SampleArgs a, SampleLong g) {
  const int b = blockIdx.x;
  for (int i = threadIdx.x; i < SBP; i += 256) { g.hc[(long long)b * SBP + i] = 0u; g.hw[(long long)b * SBP + i] = 0; }
  if (threadIdx.x == 0) {
    SampleState s{};
    s.cut = s.kcut = SampleCut{0u, ALL_TIES};
    s.minkey = 0xFFFFFFFFu;
    g.state[b] = s;
  }
}
__device__ __forceinline__ unsigned agent_load(const unsigned* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ u64 agent_load(const u64* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// four consecutive entries (one wide load where `wide`: the address allows it); entries behind the end are key 0
struct Four { unsigned k[4]; };
__device__ __forceinline__ bool sample_wide(const SampleArgs& a, long long first) {
  return (((unsigned long long)a.scores + (unsigned long long)first * (a.type == UR_F32 ? 4 : 2)) & (a.type == UR_F32 ? 15 : 7)) == 0;
}
__device__ __forceinline__ Four sample_four(const SampleArgs& a, long long base, long long i, long long end, bool wide) {
  Four r;
  if (wide && i + 4 <= end) {
    if (a.type == UR_F32) {
      const float4 v = *(const float4*)((const float*)a.scores + base + i);
      r.k[0] = key_f32(v.x); r.k[1] = key_f32(v.y); r.k[2] = key_f32(v.z); r.k[3] = key_f32(v.w);
    } else {
      const ushort4 v = *(const ushort4*)((const unsigned short*)a.scores + base + i);
      r.k[0] = key_16(v.x, a.type); r.k[1] = key_16(v.y, a.type); r.k[2] = key_16(v.z, a.type); r.k[3] = key_16(v.w, a.type);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.k[j] = i + j < end ? sample_key(a.scores, a.type, base + i + j) : 0u;
  }
  return r;
}
// a workgroup's entries, f(key): four wide loads of a thread under way while the four before them are looked at
template <typename F>
__device__ __forceinline__ void sample_walk(const SampleArgs& a, long long base, long long i0, long long i1, F f) {
  const bool wide = sample_wide(a, base + i0);
  Four v[4];
  long long i = i0 + 4 * threadIdx.x;
#pragma unroll
  for (int u = 0; u < 4; ++u) v[u] = sample_four(a, base, i + 1024 * u, i1, wide);
  for (; i < i1; i += 4096) {
    Four w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] = sample_four(a, base, i + 4096 + 1024 * u, i1, wide);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) f(v[u].k[j]);
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = w[u];
  }
}
__global__ __launch_bounds__(256) void sample_max_kernel(SampleArgs a, SampleLong g) {
  const int b = blockIdx.y;
  const long long i0 = (long long)blockIdx.x * g.chunk, i1 = min(a.N, i0 + g.chunk);
  unsigned mk = 0u, least = 0xFFFFFFFFu;
  sample_walk(a, (long long)b * a.ld, i0, i1, [&](unsigned k) {
    mk = max(mk, k);
    if (k != 0u) least = min(least, k);
  });
  mk = wave_max(mk);
  least = ~wave_max(~least);
  if ((threadIdx.x & 63) == 0 && mk) {
    atomicMax(&g.state[b].maxkey, mk);
    atomicMin(&g.state[b].minkey, least);
  }
}
template <int PHASE>
__device__ __forceinline__ bool sample_active(const SampleArgs& a, const SampleRow& r, unsigned mk) {
  return mk != 0u && !r.greedy && (PHASE == 0 ? r.k < a.N : r.p < 1.0 && r.p > 0.0);
}
// four consecutive scores as floats; behind the end: -inf
struct FourX { float x[4]; };
template <int TYPE>
__device__ __forceinline__ FourX four_scores(const SampleArgs& a, long long base, long long i, long long end, bool wide) {
  FourX r;
  auto narrow = [](unsigned u) { return TYPE == UR_F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)u) : __uint_as_float(u << 16); };
  if (wide && i + 4 <= end) {
    if constexpr (TYPE == UR_F32) {
      const float4 v = *(const float4*)((const float*)a.scores + base + i);
      r.x[0] = v.x; r.x[1] = v.y; r.x[2] = v.z; r.x[3] = v.w;
    } else {
      const ushort4 v = *(const ushort4*)((const unsigned short*)a.scores + base + i);
      r.x[0] = narrow(v.x); r.x[1] = narrow(v.y); r.x[2] = narrow(v.z); r.x[3] = narrow(v.w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.x[j] = -INFINITY;
      if (i + j < end) r.x[j] = TYPE == UR_F32 ? ((const float*)a.scores)[base + i + j] : narrow(((const unsigned short*)a.scores)[base + i + j]);
    }
  }
  return r;
}
// a workgroup's bins added to the row's, up to nine adds of a thread under way.  Every thread waits for its adds' old values: an add without one
// may still be on its way when the barrier in front of the arrival is passed (that barrier waits for LDS, the arrival for its own wave only), and the
// workgroup that arrives last would read, and clear, bins that lack it
template <int FIRST = 0, typename T>
__device__ __forceinline__ void add_bins(const T* mine, T* row) {
  const int i = (int)threadIdx.x + FIRST;
  const T v = i < SBP ? mine[i] : (T)0;
  T old = 0;
  if (v) old = __hip_atomic_fetch_add(row + i, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if constexpr (FIRST + 256 < SBP) add_bins<FIRST + 256>(mine, row);
  asm volatile("" ::"v"(old));
}
// the same of bins of weights (HI 42), into the row's (HI 64)
template <int FIRST = 0>
__device__ __forceinline__ void add_bins(const u64* lo, const unsigned* hi, u64* row_lo, unsigned* row_hi) {
  const int i = (int)threadIdx.x + FIRST;
  const u128 v = i < SBP ? ((u128)hi[i] << BIN_HI) + lo[i] : 0;
  const u64 w = (u64)v;
  u64 old = 0;
  unsigned up = (unsigned)(v >> 64), old_up = 0;
  if (w) old = __hip_atomic_fetch_add(row_lo + i, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if constexpr (FIRST + 256 < SBP) add_bins<FIRST + 256>(lo, hi, row_lo, row_hi);
  up += old + w < old;
  if (up) old_up = __hip_atomic_fetch_add(row_hi + i, up, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("" ::"v"(old), "v"(old_up));
}
// the top-k (PHASE 0) or top-p (PHASE 1) selection: counts (and weights) of the steps; the workgroup that arrives last finds the border's step
// and clears the bins
template <int PHASE, int TYPE>
__global__ __launch_bounds__(256) void sample_steps_kernel(SampleArgs a, SampleLong g, int mode) {
  __shared__ unsigned hc[SBP];
  __shared__ u64 hw[PHASE == 1 ? SBP : 1];
  __shared__ unsigned tmp32[4], last;
  __shared__ u64 tmp64[8];
  __shared__ Select st;
  __shared__ SampleCut cut;
  const int b = blockIdx.y, tid = threadIdx.x;
  SampleState* S = g.state + b;
  SampleRow r;
  r.load(a, b);
  const unsigned mk = S->maxkey;
  if (!sample_active<PHASE>(a, r, mk)) {
    // a row whose p is not positive keeps its largest entry alone
    if (PHASE == 1 && blockIdx.x == 0 && tid == 0 && mk != 0u && !r.greedy && r.p <= 0.0) S->cut = SampleCut{mk, 1u};
    return;
  }
  r.set_max(mk);
  Steps steps;
  steps.set(r, S->minkey, PHASE == 1);
  unsigned* ghc = g.hc + (long long)b * SBP;
  u64* ghw = g.hw + (long long)b * SBP;
  const SampleCut kc = S->kcut;
  for (int i = tid; i < SBP; i += 256) {
    hc[i] = 0u;
    if constexpr (PHASE == 1) hw[i] = 0;
  }
  __syncthreads();
  const long long i0 = (long long)blockIdx.x * g.chunk, i1 = min(a.N, i0 + g.chunk);
  const float above = PHASE == 1 ? cut_value(kc.cut, TYPE) : -INFINITY;
  const double m = (double)r.m, scale = r.scale;
  const unsigned large = large_from((unsigned)g.chunk);
  auto weight = [&](float x) { return exp2_fixed(r.flat ? (x == r.m ? 0.0 : -100.0) : ((double)x - m) * scale); };
  auto count = [&](float x) {
    const int d = bin_at<256>(steps.of_value(x));
    if constexpr (PHASE == 0) atomicAdd(&hc[d], 1u);
    else add_weight(hw + d, hc + d, weight(x), 1u, large);       // (a chunk is 65 536 entries at most)
  };
  {
    const long long base = (long long)b * a.ld;
    const bool wide = sample_wide(a, base + i0);
    FourX v[4];
    long long i = i0 + 4 * tid;
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = four_scores<TYPE>(a, base, i + 1024 * u, i1, wide);
    for (; i < i1; i += 4096) {
      FourX w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = four_scores<TYPE>(a, base, i + 4096 + 1024 * u, i1, wide);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (v[u].x[j] > above) count(v[u].x[j]);
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = w[u];
    }
  }
  __syncthreads();
  if constexpr (PHASE == 0) add_bins(hc, ghc);
  else add_bins(hw, hc, ghw, ghc);
  __syncthreads();
  if (tid == 0) last = ur_arrive(&S->arrived, mode) == (unsigned)g.nchunk - 1u;
  __syncthreads();
  if (!last) return;
  if (tid == 0) {
    st = Select{0, 1u, mk, 0u, 0u, (unsigned)min((long long)0x7FFFFFFF, r.k), 0, 0.0, 0u};
    cut = S->cut;
  }
  constexpr int PER = (SBP + 255) / 256;                         // all of a thread's bins under way at once
  unsigned c[PER];
  u64 w[PHASE == 1 ? PER : 1];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = min(tid + 256 * j, SBP - 1);
    c[j] = agent_load(ghc + i);
    if constexpr (PHASE == 1) w[j] = agent_load(ghw + i);
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = tid + 256 * j;
    if (i >= SBP) break;
    hc[i] = c[j];
    if constexpr (PHASE == 1) hw[i] = w[j];
  }
  __syncthreads();
  for (int i = tid; i < SBP; i += 256) {
    ghc[i] = 0u;
    if constexpr (PHASE == 1) ghw[i] = 0;
  }
  __syncthreads();
  if constexpr (PHASE == 0) pick_k<256>(-1, false, hc, &st, &cut, tmp32);
  else {
    if (tid == 0 && kc.cut != 0u && kc.ties != 0u) {             // the ties that top-k left
      const int d = bin_at<256>(steps.of_value(above));
      add_wide(hw + d, hc + d, (u128)weight(above) * kc.ties);
    }
    __syncthreads();
    pick_p<256, 64>(-1, hc, hw, r.p, &st, tmp64);
  }
  step_keys(steps, mk, &st);
  if (tid == 0) {
    S->st = st;
    S->arrived = 0u;
    S->listed = 0u;
  }
}
// the keys of the border's step, put together (a list that holds them all)
template <int PHASE>
__global__ __launch_bounds__(256) void sample_near_kernel(SampleArgs a, SampleLong g) {
  __shared__ unsigned lk[LLIST], n_s, at_s;
  const int b = blockIdx.y, tid = threadIdx.x;
  SampleState* S = g.state + b;
  SampleRow r;
  r.load(a, b);
  if (!sample_active<PHASE>(a, r, S->maxkey) || S->st.done) return;
  const unsigned lo = PHASE == 0 ? S->st.lo : max(S->st.lo, S->kcut.cut + 1u), hi = S->st.hi;
  if (tid == 0) n_s = 0u;
  __syncthreads();
  const long long i0 = (long long)blockIdx.x * g.chunk, i1 = min(a.N, i0 + g.chunk);
  sample_walk(a, (long long)b * a.ld, i0, i1, [&](unsigned k) {
    if (k >= lo && k <= hi) {
      const unsigned q = atomicAdd(&n_s, 1u);
      if (q < LLIST) lk[q] = k;
    }
  });
  __syncthreads();
  const unsigned n = n_s;
  if (n == 0u) return;
  if (tid == 0) at_s = atomicAdd(&S->listed, n);
  __syncthreads();
  unsigned* list = g.list + (long long)b * LLIST;
  for (unsigned i = tid; at_s + i < LLIST && i < n; i += 256) list[at_s + i] = lk[i];   // (more than the list holds: counted only)
}
// the border among them: compared directly, or radix rounds over the list (over the row where the list could not hold them)
template <int PHASE>
__global__ __launch_bounds__(1024) void sample_border_kernel(SampleArgs a, SampleLong g) {
  constexpr int NT = 1024;
  __shared__ unsigned hc[SBP];
  __shared__ u64 hw[PHASE == 1 ? SBP : 1];
  __shared__ __attribute__((aligned(16))) unsigned near_k[DIRECT];
  __shared__ u64 near_w[PHASE == 1 ? DIRECT : 1];
  __shared__ unsigned tmp32[NT / 64];
  __shared__ u64 tmp64[2 * NT / 64];
  __shared__ Select st;
  __shared__ SampleCut cut;
  const int b = blockIdx.x, tid = threadIdx.x;
  SampleState* S = g.state + b;
  SampleRow r;
  r.load(a, b);
  const unsigned mk = S->maxkey;
  if (!sample_active<PHASE>(a, r, mk) || S->st.done) return;
  r.set_max(mk);
  const SampleCut kc = S->kcut;
  const unsigned n = S->listed;
  const bool listed = n <= LLIST;
  const unsigned* list = g.list + (long long)b * LLIST;
  if (tid == 0) { st = S->st; cut = S->cut; }
  __syncthreads();
  const unsigned lo = st.lo, hi = st.hi;
  const bool tied = PHASE == 1 && kc.cut != 0u && kc.ties != 0u && kc.cut >= lo && kc.cut <= hi;   // ties that top-k left are among them
  if (listed && n <= DIRECT && !tied) {
    if (tid < DIRECT) {
      const unsigned k = tid < (int)n ? list[tid] : 0u;
      near_k[tid] = k;
      if constexpr (PHASE == 1) near_w[tid] = k ? r.weight(k) : 0;
    }
    __syncthreads();
    if constexpr (PHASE == 0) direct_k(near_k, (int)n, &st, &cut);
    else direct_p(near_k, near_w, (int)n, &st, &cut);
    if (tid == 0) st.done = 1u;
    __syncthreads();
  }
  const int rounds = a.type == UR_F32 ? 3 : 2;
  for (int round = 0; round < rounds && !st.done; ++round) {
    for (int i = tid; i < SBP; i += NT) {
      hc[i] = 0u;
      if (PHASE == 1) hw[i] = 0;
    }
    __syncthreads();
    const unsigned prefix = st.prefix;
    auto count = [&](unsigned k, unsigned times) {
      if (!round_in(k, round, prefix)) return;
      const int d = bin_at<NT>(round_place(k, round));
      if (PHASE == 0 || round == rounds - 1) atomicAdd(&hc[d], times);
      else add_wide(hw + d, hc + d, (u128)r.weight(k) * times);
    };
    if (listed) {
      for (unsigned i = tid; i < n; i += NT) count(list[i], 1u);
    } else {
      const long long base = (long long)b * a.ld;
      const unsigned from = PHASE == 0 ? lo : max(lo, kc.cut + 1u);
      const bool wide = sample_wide(a, base);
      for (long long i = 4 * tid; i < a.N; i += 4 * NT) {
        const Four v = sample_four(a, base, i, a.N, wide);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (v.k[j] >= from && v.k[j] <= hi) count(v.k[j], 1u);
      }
    }
    if (tied && tid == 0) count(kc.cut, kc.ties);
    __syncthreads();
    if constexpr (PHASE == 0) pick_k<NT>(round, round == rounds - 1, hc, &st, &cut, tmp32);
    else if (round == rounds - 1) pick_p_key<NT>(round, hc, [&](unsigned k) { return r.weight(k); }, &st, &cut, tmp64);
    else pick_p<NT, 64>(round, hc, hw, r.p, &st, tmp64);
  }
  if (tid == 0) {
    S->cut = inside(cut, kc);
    if (PHASE == 0) S->kcut = cut;
  }
}
__device__ __forceinline__ SampleCut final_cut(const SampleState* S, const SampleRow& r) {   // (set_max has been called)
  return r.greedy ? SampleCut{S->maxkey, 1u} : above_min_p(S->cut, r.min_key(S->maxkey));
}
__device__ __forceinline__ bool some_ties(const SampleCut& c) { return c.ties != 0u && c.ties != ALL_TIES; }
// ties of every block (rows where some of them go)
__global__ __launch_bounds__(256) void sample_ties_kernel(SampleArgs a, SampleLong g) {
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  SampleRow r;
  r.load(a, b);
  const SampleState* S = g.state + b;
  if (S->maxkey == 0u || (!r.greedy && !some_ties(S->cut))) return;
  r.set_max(S->maxkey);
  const SampleCut c = final_cut(S, r);
  if (!some_ties(c)) return;
  const long long base = (long long)b * a.ld;
  for (int q = blockIdx.x * (g.chunk / LBLK) + wave; q < min(g.nblk, (int)(blockIdx.x + 1) * (g.chunk / LBLK)); q += 4) {
    const long long i0 = (long long)q * LBLK, i1 = min(a.N, i0 + LBLK);
    const bool wide = sample_wide(a, base + i0);
    unsigned n = 0;
#pragma unroll 4
    for (int j = 0; j < LBLK / 256; ++j) {
      const Four v = sample_four(a, base, i0 + 256 * j + 4 * lane, i1, wide);
#pragma unroll
      for (int u = 0; u < 4; ++u) n += v.k[u] == c.cut;
    }
    n = wave_total(n);
    if (lane == 0) g.tb[(long long)b * g.nblk + q] = n;
  }
}
__device__ __forceinline__ unsigned ties_before(const unsigned* tb, int q) {   // a wave sums what lies in front of block q
  unsigned n = 0;
  for (int t = threadIdx.x & 63; t < q; t += 64) n += tb[t];
  return wave_total(n);
}
// the kept weight of every block: a wave a block of 2 048, four consecutive entries a lane.  Scores are compared as floats (a key's order is
// theirs, the keys in front of the first number are -inf)
template <int TYPE>
__global__ __launch_bounds__(256) void sample_sums_kernel(SampleArgs a, SampleLong g) {
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  SampleRow r;
  r.load(a, b);
  const SampleState* S = g.state + b;
  if (S->maxkey == 0u) return;
  r.set_max(S->maxkey);
  const SampleCut c = final_cut(S, r);
  const bool ranked = some_ties(c);
  const float above = cut_value(c.cut, TYPE);
  const double m = (double)r.m, scale = r.scale;
  const long long base = (long long)b * a.ld;
  for (int q = blockIdx.x * (g.chunk / LBLK) + wave; q < min(g.nblk, (int)(blockIdx.x + 1) * (g.chunk / LBLK)); q += 4) {
    const long long i0 = (long long)q * LBLK, i1 = min(a.N, i0 + LBLK);
    const bool wide = sample_wide(a, base + i0);
    unsigned ties = ranked ? ties_before(g.tb + (long long)b * g.nblk, q) : 0u;
    u64 sum = 0;                        // (32 entries of at most 2^57)
    FourX next[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) next[u] = four_scores<TYPE>(a, base, i0 + 256 * u + 4 * lane, i1, wide);
#pragma unroll
    for (int j = 0; j < LBLK / 256; ++j) {
      const FourX f = next[j & 3];
      if (j + 4 < LBLK / 256) next[j & 3] = four_scores<TYPE>(a, base, i0 + 256 * (j + 4) + 4 * lane, i1, wide);
      unsigned rank = 0;
      if (ranked) {
        unsigned eq = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) eq += f.x[u] == above;
        const unsigned upto = wave_upto(eq);
        rank = ties + upto - eq;
        ties += last_lane(upto);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float x = f.x[u];
        bool stays = x > above;
        if (ranked) stays |= x == above && rank++ < c.ties;
        const double z = r.flat ? (x == r.m ? 0.0 : -100.0) : ((double)x - m) * scale;
        sum += stays ? exp2_fixed(z) : 0;
      }
    }
    WSum v{0, 0};
    v.add(sum);
    v.hi = wave_total(v.hi);
    v.lo = wave_total(v.lo);
    if (lane == 0) {
      u64* o = g.bs + ((long long)b * g.nblk + q) * 2;
      o[0] = v.hi;
      o[1] = v.lo;
    }
  }
}
// a workgroup a draw: the block that the goal falls into (a thread takes a run of blocks), then its entry (a thread takes eight)
__global__ __launch_bounds__(256) void sample_draw_kernel(SampleArgs a, SampleLong g) {
  __shared__ u64 tmp64[8];
  __shared__ unsigned tmp32[4];
  __shared__ int q_s;
  __shared__ WSum run_s;
  const int s = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const long long at = (long long)b * a.S + s, base = (long long)b * a.ld;
  SampleRow r;
  r.load(a, b);
  const SampleState* S = g.state + b;
  if (S->maxkey == 0u) {
    if (tid == 0) { a.out_id[at] = -1; a.out_logp[at] = -INFINITY; }
    return;
  }
  r.set_max(S->maxkey);
  if (tid == 0) { q_s = 0; run_s = WSum{0, 0}; }
  const SampleCut c = final_cut(S, r);
  const u64* bs = g.bs + (long long)b * g.nblk * 2;
  const int per = (g.nblk + 255) / 256, q0 = min(g.nblk, tid * per), q1 = min(g.nblk, q0 + per);
  WSum mine{0, 0}, all;
  for (int q = q0; q < q1; ++q) mine.add(WSum{bs[2 * q], bs[2 * q + 1]});
  WSum run = block_before<256>(mine, tmp64, &all);
  const u128 W = all.all(), goal = sample_goal(a.rand[at], W);
  WSum end = run;
  end.add(mine);
  if (run.all() <= goal && goal < end.all()) {   // one thread (goal < W)
    for (int q = q0; q < q1; ++q) {
      end = run;
      end.add(WSum{bs[2 * q], bs[2 * q + 1]});
      if (goal < end.all()) { q_s = q; run_s = run; break; }
      run = end;
    }
  }
  __syncthreads();
  const int q = q_s;
  run = run_s;
  const long long i0 = (long long)q * LBLK + 8 * tid, i1 = min(a.N, (long long)(q + 1) * LBLK);
  unsigned k[8];
  {
    const bool wide = sample_wide(a, base + i0);
    const Four f = sample_four(a, base, i0, i1, wide), h = sample_four(a, base, i0 + 4, i1, wide);
#pragma unroll
    for (int u = 0; u < 4; ++u) { k[u] = f.k[u]; k[4 + u] = h.k[u]; }
  }
  unsigned rank = 0;
  if (some_ties(c)) {
    unsigned eq = 0, total;
#pragma unroll
    for (int u = 0; u < 8; ++u) eq += k[u] == c.cut;
    rank = block_before<256>(eq, tmp32, &total) + ties_before(g.tb + (long long)b * g.nblk, q);
  }
  u64 w[8];
  mine = WSum{0, 0};
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const bool stays = k[u] > c.cut || (k[u] == c.cut && k[u] != 0u && rank++ < c.ties);
    w[u] = stays ? r.weight(k[u]) : 0;
    mine.add(w[u]);
  }
  run.add(block_before<256>(mine, tmp64, &all));
  u128 sum = run.all();
  if (sum <= goal && goal < sum + mine.all()) {
    const double log_W = log(wide_to_double(W) * 6.938893903907228e-18);   // 2^-57
    bool found = false;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      sum += w[u];
      if (!found && sum > goal) {
        found = true;
        a.out_id[at] = a.ids ? a.ids[(long long)b * a.ld_ids + i0 + u] : i0 + u;
        a.out_logp[at] = r.greedy ? 0.f : (float)(r.z(k[u]) - log_W);
      }
    }
  }
}

// ---- host
// what fits into a workgroup's LDS beside the histograms.  Rows in LDS or over many workgroups, k 50 and p 0.9: 256 x 20 000 28 / 135 us, 4 x 30 000
// 34 / 51
static inline bool sample_in_lds(long long N, int type) { return N <= (type == UR_F32 ? 32768 : 65536); }
static size_t sample_long_bytes(long long N, int B, char* base, SampleLong* g) {
  size_t o = 0;
  auto take = [&](size_t n) {
    char* p = base ? base + o : nullptr;
    o += (n + 255) & ~(size_t)255;
    return p;
  };
  SampleLong w{};
  // about 2 048 workgroups where there is work for them, of 4 096 to 65 536 entries
  const long long want = (N * (long long)B + 2047) / 2048;
  w.chunk = (int)std::min<long long>(65536, std::max<long long>(4096, (want + 4095) / 4096 * 4096));
  w.nchunk = cdiv(N, w.chunk); w.nblk = cdiv(N, LBLK);
  w.state = (SampleState*)take(sizeof(SampleState) * B);
  w.hc = (unsigned*)take((size_t)B * SBP * 4); w.hw = (u64*)take((size_t)B * SBP * 8);
  w.tb = (unsigned*)take((size_t)B * w.nblk * 4); w.bs = (u64*)take((size_t)B * w.nblk * 16);
  w.list = (unsigned*)take((size_t)B * LLIST * 4);
  if (g) *g = w;
  return o;
}
template <int NT, bool RAW>
static int launch_sample_row(const SampleArgs& a, hipStream_t st) {
  const size_t lds = (size_t)SBP * 12 + (size_t)a.N * (RAW ? 2 : 4) + 16;
  static const hipError_t attr = hipFuncSetAttribute((const void*)sample_row_kernel<NT, RAW>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024 - 6144);
  (void)attr;
  hipLaunchKernelGGL((sample_row_kernel<NT, RAW>), dim3(a.B), dim3(NT), lds, st, a);
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
    // threads for a row, 256 / 512 / 1 024, p 0.9: fp32 512 x 1 000 17.3 / 17.5 / 25.7 us, 256 x 6 000 31.0 / 23.5 / 22.3, 256 x 20 000 73 / 49 / 40;
    // bf16 20.0 / 19.9 / 28.5, 39.0 / 28.0 / 25.8, 99 / 62 / 48 (one rule for both)
    if (score_type == UR_F32)
      return n <= 2048 ? launch_sample_row<256, false>(a, st) : n <= 8192 ? launch_sample_row<512, false>(a, st) : launch_sample_row<1024, false>(a, st);
    return n <= 2048 ? launch_sample_row<256, true>(a, st) : n <= 8192 ? launch_sample_row<512, true>(a, st) : launch_sample_row<1024, true>(a, st);
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
  auto select = [&](auto phase) -> int {
    constexpr int PHASE = decltype(phase)::value;
    if (score_type == UR_F32) hipLaunchKernelGGL((sample_steps_kernel<PHASE, UR_F32>), grid, dim3(256), 0, st, a, g, mode);
    else if (score_type == UR_F16) hipLaunchKernelGGL((sample_steps_kernel<PHASE, UR_F16>), grid, dim3(256), 0, st, a, g, mode);
    else hipLaunchKernelGGL((sample_steps_kernel<PHASE, UR_BF16>), grid, dim3(256), 0, st, a, g, mode);
    UR_LAUNCH_CHECK();
    hipLaunchKernelGGL((sample_near_kernel<PHASE>), grid, dim3(256), 0, st, a, g);
    UR_LAUNCH_CHECK();
    hipLaunchKernelGGL((sample_border_kernel<PHASE>), dim3(B), dim3(1024), 0, st, a, g);
    UR_LAUNCH_CHECK();
    return UR_OK;
  };
  int rc = g.uses_k ? select(std::integral_constant<int, 0>()) : UR_OK;
  if (rc) return rc;
  if (g.uses_p && (rc = select(std::integral_constant<int, 1>()))) return rc;
  if (g.uses_k || g.uses_p || temperature_rows || temperature == 0.0) {
    hipLaunchKernelGGL(sample_ties_kernel, grid, dim3(256), 0, st, a, g);
    UR_LAUNCH_CHECK();
  }
  if (score_type == UR_F32) hipLaunchKernelGGL((sample_sums_kernel<UR_F32>), grid, dim3(256), 0, st, a, g);
  else if (score_type == UR_F16) hipLaunchKernelGGL((sample_sums_kernel<UR_F16>), grid, dim3(256), 0, st, a, g);
  else hipLaunchKernelGGL((sample_sums_kernel<UR_BF16>), grid, dim3(256), 0, st, a, g);
  UR_LAUNCH_CHECK();
  hipLaunchKernelGGL(sample_draw_kernel, dim3(S, B), dim3(256), 0, st, a, g);
  UR_LAUNCH_CHECK();
  return UR_OK;
}
