// Sampling from scores with temperature, top-k, top-p and min-p, the random numbers given by the caller (beside eval.hip's top-k: an answer
// drawn from the distribution instead of its head).  Per row of N scores x:
//   z_n = (x_n - max x) / T, weight w_n = exp(z_n); NaN and -inf carry none; a row with +inf: those entries 1, the others 0
//   top-k: the first k in the order (score descending, index ascending); top-p: of those, in that order, every entry before which less
//   than p of their weight lies; min-p: w >= min_p.  The answer to u: the first index n, in INDEX order, with sum_{j <= n} kept w_j > u W.
// No sort: the order only decides a threshold (a key and how many of its ties stay), found by radix selection.
//
// Arithmetic.  Which entry a sum's border falls on is a whole number, so every sum is exact: weights are exp in double, rounded once to
// multiples of 2^-62 and added as integers (two 64-bit limbs).  Sums do not depend on an order, partial sums of any cut agree.
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
// a row's parameters; the weight of a key as a multiple of 2^-62
struct SampleRow {
  double inv_T, p, min_p; long long k; bool greedy;
  float m;
  __device__ __forceinline__ void load(const SampleArgs& a, int b) {
    const double T = a.T_rows ? (double)a.T_rows[b] : a.T;
    p = a.p_rows ? (double)a.p_rows[b] : a.top_p;
    min_p = a.minp_rows ? (double)a.minp_rows[b] : a.min_p;
    k = a.k_rows ? a.k_rows[b] : a.top_k;
    if (k <= 0) k = a.N;
    greedy = !(T > 1e-300);              // (1 / T stays finite)
    inv_T = greedy ? 1.0 : 1.0 / T;
    if (!(min_p < 1.0)) min_p = 1.0;    // (the largest stays)
  }
  __device__ __forceinline__ double z(unsigned key) const {
    const float x = sample_value(key);
    if (m == INFINITY) return x == INFINITY ? 0.0 : -INFINITY;
    return ((double)x - (double)m) * inv_T;
  }
  __device__ __forceinline__ u64 weight(unsigned key) const { return (u64)(exp(z(key)) * 4611686018427387904.0 + 0.5); }
  __device__ __forceinline__ bool min_ok(unsigned key) const { return !(min_p > 0.0) || exp(z(key)) >= min_p; }
};
struct WSum {   // a sum of weights: limbs of 32 bits, each summed in 64
  u64 hi, lo;
  __device__ __forceinline__ void add(u64 w) { hi += w >> 32; lo += w & 0xFFFFFFFFull; }
  __device__ __forceinline__ u128 all() const { return ((u128)hi << 32) + lo; }
};
__device__ __forceinline__ double wide_to_double(u128 v) { return (double)(u64)(v >> 64) * 18446744073709551616.0 + (double)(u64)v; }
__device__ __forceinline__ u128 double_to_wide(double v) {   // v >= 0
  const u64 hi = (u64)(v * 5.42101086242752217e-20);          // 2^-64
  const double rest = v - (double)hi * 18446744073709551616.0;
  return ((u128)hi << 64) + (rest > 0.0 ? (u64)rest : 0);
}
// entries j = 0, 1, .. of one tied weight w stay while above + j w < limit
__device__ __forceinline__ long long ties_within(u128 above, u64 w, double limit, long long most) {
  if (w == 0) return most;
  long long lo = 0, hi = most;          // the first j in [0, most] that does not stay
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if (wide_to_double(above + (u128)w * (u64)mid) < limit) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// Simple form: one workgroup a row, every pass over the row in memory.
__global__ __launch_bounds__(1024) void sample_row_kernel(SampleArgs a) {
  constexpr int NT = 1024;
  __shared__ unsigned hist[256];
  __shared__ u64 whi[256], wlo[256];
  __shared__ u64 s_hi[NT], s_lo[NT];
  __shared__ int s_cnt[NT];
  __shared__ unsigned s_max, s_prefix, s_mask;
  __shared__ long long s_need;
  __shared__ u64 s_above[2], s_tot[2];
  const int b = blockIdx.x, tid = threadIdx.x;
  const long long base = (long long)b * a.ld;
  auto key_at = [&](long long i) { return sample_key(sample_load(a.scores, a.type, base + i)); };
  SampleRow r;
  r.load(a, b);
  if (tid == 0) s_max = 0u;
  __syncthreads();
  unsigned mk = 0u;
  for (long long i = tid; i < a.N; i += NT) mk = max(mk, key_at(i));
  atomicMax(&s_max, mk);
  __syncthreads();
  mk = s_max;
  if (mk == 0u) {   // nothing to choose from
    for (int s = tid; s < a.S; s += NT) {
      a.out_id[(long long)b * a.S + s] = -1;
      a.out_logp[(long long)b * a.S + s] = -INFINITY;
    }
    return;
  }
  r.m = sample_value(mk);
  unsigned cut = 1u;                    // entries above this key stay, `ties` of those equal to it (in index order)
  long long ties = a.N;
  if (r.greedy) { cut = mk; ties = 1; }
  else {
    if (r.k < a.N) {                    // ---- top-k: the k-th largest key
      if (tid == 0) { s_prefix = 0u; s_mask = 0u; s_need = r.k; }
      __syncthreads();
      for (int pass = 0; pass < 4; ++pass) {
        const int sh = 24 - 8 * pass;
        for (int i = tid; i < 256; i += NT) hist[i] = 0u;
        __syncthreads();
        const unsigned prefix = s_prefix, mask = s_mask;
        for (long long i = tid; i < a.N; i += NT) {
          const unsigned k = key_at(i);
          if (k != 0u && (k & mask) == prefix) atomicAdd(&hist[(k >> sh) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
          long long need = s_need;
          int d = 255;
          for (; d > 0; --d) {
            if ((long long)hist[d] >= need) break;
            need -= hist[d];
          }
          s_need = need;
          s_prefix = prefix | ((unsigned)d << sh);
          s_mask = mask | (255u << sh);
        }
        __syncthreads();
      }
      cut = max(s_prefix, 1u);          // (fewer than k entries: the walk ends at key 0, nothing is cut)
      ties = s_prefix ? s_need : a.N;
      __syncthreads();
    }
    if (r.p < 1.0) {                    // ---- top-p over what is left
      if (tid == 0) { s_prefix = 0u; s_mask = 0u; s_above[0] = s_above[1] = 0; s_tot[0] = s_tot[1] = 0; }
      __syncthreads();
      for (int pass = 0; pass < 4; ++pass) {
        const int sh = 24 - 8 * pass;
        for (int i = tid; i < 256; i += NT) { hist[i] = 0u; whi[i] = 0; wlo[i] = 0; }
        if (tid == 0) s_cnt[0] = 0;
        __syncthreads();
        const unsigned prefix = s_prefix, mask = s_mask;
        for (long long i = tid; i < a.N; i += NT) {
          const unsigned k = key_at(i);
          if (k < cut || (k & mask) != prefix) continue;
          if (k == cut && ties < a.N && atomicAdd((unsigned*)&s_cnt[0], 1u) >= (unsigned)ties) continue;   // any `ties` of the equal ones: equal weights
          const u64 w = r.weight(k);
          const int d = (k >> sh) & 255;
          atomicAdd(&hist[d], 1u);
          atomicAdd(&whi[d], w >> 32);
          atomicAdd(&wlo[d], w & 0xFFFFFFFFull);
        }
        __syncthreads();
        if (tid == 0) {
          if (pass == 0)
            for (int d = 0; d < 256; ++d) { s_tot[0] += whi[d]; s_tot[1] += wlo[d]; }
          const WSum tot{s_tot[0], s_tot[1]};
          const double limit = r.p * wide_to_double(tot.all());
          WSum above{s_above[0], s_above[1]}, at = above;
          int best = -1;
          for (int d = 255; d >= 0; --d) {
            if (!hist[d]) continue;
            if (best >= 0 && !(wide_to_double(above.all()) < limit)) break;
            best = d;                   // its first entry stays
            at = above;
            above.hi += whi[d];
            above.lo += wlo[d];
          }
          s_above[0] = at.hi; s_above[1] = at.lo;
          s_prefix = prefix | ((unsigned)best << sh);
          s_mask = mask | (255u << sh);
          s_need = hist[best];
        }
        __syncthreads();
      }
      const WSum above{s_above[0], s_above[1]}, tot{s_tot[0], s_tot[1]};
      const unsigned kp = s_prefix;
      const long long t = max(1LL, ties_within(above.all(), r.weight(kp), r.p * wide_to_double(tot.all()), s_need));
      cut = kp;
      ties = t;
      __syncthreads();
    }
  }
  // ---- the kept weights in index order: thread t owns entries [t c, (t + 1) c)
  const long long c = (a.N + NT - 1) / NT, i0 = min(a.N, tid * c), i1 = min(a.N, i0 + c);
  int eq = 0;
  for (long long i = i0; i < i1; ++i) eq += key_at(i) == cut;
  s_cnt[tid] = eq;
  __syncthreads();
  if (tid == 0) {
    int run = 0;
    for (int t = 0; t < NT; ++t) { const int v = s_cnt[t]; s_cnt[t] = run; run += v; }
  }
  __syncthreads();
  long long rank = s_cnt[tid];
  WSum mine{0, 0};
  for (long long i = i0; i < i1; ++i) {
    const unsigned k = key_at(i);
    const bool stays = (k > cut || (k == cut && rank < ties)) && r.min_ok(k);
    rank += k == cut;
    if (stays) mine.add(r.greedy ? 1ull << 62 : r.weight(k));
  }
  s_hi[tid] = mine.hi; s_lo[tid] = mine.lo;
  __syncthreads();
  if (tid == 0) {
    WSum run{0, 0};
    for (int t = 0; t < NT; ++t) {
      const WSum v{s_hi[t], s_lo[t]};
      s_hi[t] = run.hi; s_lo[t] = run.lo;
      run.hi += v.hi; run.lo += v.lo;
    }
    s_tot[0] = run.hi; s_tot[1] = run.lo;
  }
  __syncthreads();
  const WSum tot{s_tot[0], s_tot[1]}, start{s_hi[tid], s_lo[tid]};
  const double W = wide_to_double(tot.all()), log_W = log(W * 2.168404344971009e-19);   // 2^-62
  const u128 from = start.all(), to = from + mine.all();
  for (int s = 0; s < a.S; ++s) {
    float u = a.rand[(long long)b * a.S + s];
    u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
    const u128 goal = double_to_wide((double)u * W);
    if (!(from <= goal && goal < to)) continue;
    u128 run = from;
    rank = s_cnt[tid];
    for (long long i = i0; i < i1; ++i) {
      const unsigned k = key_at(i);
      const bool stays = (k > cut || (k == cut && rank < ties)) && r.min_ok(k);
      rank += k == cut;
      if (!stays) continue;
      run += r.greedy ? 1ull << 62 : r.weight(k);
      if (run > goal) {
        a.out_id[(long long)b * a.S + s] = a.ids ? a.ids[(long long)b * a.ld_ids + i] : i;
        a.out_logp[(long long)b * a.S + s] = r.greedy ? 0.f : (float)(r.z(k) - log_W);
        break;
      }
    }
  }
}

}  // namespace ur

using namespace ur;

extern "C" int ur_sample_scores(const void* scores, int32_t score_type, int64_t n, int64_t ld, int32_t B, const float* rand, int32_t S,
                                double temperature, int32_t top_k, double top_p, double min_p, const float* temperature_rows,
                                const int32_t* top_k_rows, const float* top_p_rows, const float* min_p_rows, const int64_t* ids, int64_t ld_ids,
                                int64_t* out_id, float* out_logp, void* stream) {
  UR_TRACE_SCOPE();
  UR_REQUIRE(scores && rand && out_id && out_logp, UR_ERR_ARG, "ur_sample_scores: null pointer");
  UR_REQUIRE(score_type == UR_F32 || score_type == UR_F16 || score_type == UR_BF16, UR_ERR_ARG, "ur_sample_scores: score_type=%d", score_type);
  UR_REQUIRE(B > 0 && S > 0 && n > 0 && n < (1LL << 31) && ld >= n && (!ids || ld_ids >= n), UR_ERR_ARG, "ur_sample_scores: shape");
  UR_REQUIRE(temperature >= 0.0 && temperature < INFINITY, UR_ERR_ARG, "ur_sample_scores: temperature=%g", temperature);
  UR_REQUIRE(top_k >= 0 && top_p > 0.0 && min_p >= 0.0 && min_p <= 1.0, UR_ERR_ARG, "ur_sample_scores: top_k=%d top_p=%g min_p=%g", top_k, top_p, min_p);
  hipStream_t st = as_stream(stream);
  ProfScope ps(PC_MISC, st, (double)B * n * (score_type == UR_F32 ? 4 : 2));
  SampleArgs a{};
  a.scores = scores; a.type = score_type; a.N = n; a.ld = ld; a.B = B; a.S = S; a.rand = rand;
  a.T = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
  a.T_rows = temperature_rows; a.k_rows = top_k_rows; a.p_rows = top_p_rows; a.minp_rows = min_p_rows;
  a.ids = (const long long*)ids; a.ld_ids = ld_ids; a.out_id = (long long*)out_id; a.out_logp = out_logp;
  hipLaunchKernelGGL(sample_row_kernel, dim3(B), dim3(1024), 0, st, a);
  UR_LAUNCH_CHECK();
  return UR_OK;
}
