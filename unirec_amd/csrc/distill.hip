// Distillation from a teacher's top logits over the whole catalogue, forward and backward (beside fullsoftmax.hip: every item is a
// candidate, no [B, N] score matrix ever exists).
//   s(b,n) = clip((u_b . E_n + item_bias[n]) / tau),  q_b = softmax_n(s(b,:) / T),  p_b = softmax of the teacher's present entries / T
//   loss   = T^2 / C * sum_b sum_k p_bk (log p_bk - s(b, y_bk) / T + lse_b),        C = rows with an entry
//   d loss / d (u_b . E_n) = g (q_bn - sum_{k: y_bk = n} p_bk),  g = d_loss T / (C tau), 0 where the score was clipped
// The dense halves  O_b = sum_n q_bn E_n  (the expected embedding: d u_b = g (O_b - sum_k p_bk E_{y_bk})) and  dE_n = g sum_b q_bn u_b
// are the SAME computation with the two operands swapped: an OWNER row x (a user in the forward, an item in the backward) against a
// STREAM of rows y, weights exp2(z - M), a sum l of the weights and a weighted sum of the stream's rows, one pass, nothing of size
// B x N written.  The forward finds its maximum M on the way (online softmax); the backward knows q's denominator from the forward
// pass (it rides in the stream rows' bias as -log2 of it), its M is a per-item reference that keeps q in fp16's range.
// The teacher's K entries a row are sparse: gathered once in the forward, added to the table gradient through a row plan (rows.hip).
#include <math.h>

#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace ur {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr float DS_LOG2E = 1.44269504088896340736f, DS_LN2 = 0.69314718055994530942f;
constexpr int DS_MAX_D = 256;

// ---- fp32 products on the fp16 matrix pipes.  x 2^k = hi + lo with hi = fp16(x 2^k), lo = fp16(x 2^k - hi): 22 bits of every value that
// is within 2^-17 of its group's largest (k puts that at 2^13), an absolute floor of 2^-38 of the largest below.  x y is accumulated in
// fp32 from hi hi, hi lo and lo hi; the dropped lo lo is below 2^-22 |x y|, of the order of one fp32 rounding.  Three products where the
// bf16 split of gemm.hip needs six: fp16's short exponent is what the group exponents k pay for.
__device__ __forceinline__ int group_exponent(float largest) {   // k: largest 2^k in [2^13, 2^14); limited so that every 2^k stays normal
  const int e = (int)((__float_as_uint(largest) >> 23) & 0xFF) - 127;
  return min(30, max(-60, 13 - e));
}
__device__ __forceinline__ float pow2i(int k) { return __uint_as_float((unsigned)(k + 127) << 23); }
__device__ __forceinline__ float finite_abs(float x) {   // |x|, 0 for infinities and NaN: those do not set a group's exponent
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
// two values at a time: v_cvt_pk_f16_f32 and v_fma_mix_f32 (the residual in one instruction), 3 VALU slots a value, 2 without the scale
__device__ __forceinline__ void split_pair(float x, float y, float up, half2_t& hi, half2_t& lo) {
  hi = __builtin_convertvector((float2_t){x * up, y * up}, half2_t);
  lo = __builtin_convertvector((float2_t){fmaf(x, up, -(float)hi[0]), fmaf(y, up, -(float)hi[1])}, half2_t);
}

struct DistillStream {
  const float* X; long long nx;        // owner rows [nx, d]
  const float* Y; long long ny;        // stream rows [ny, d]
  int d;
  const float* y_bias;                 // added to the log2 score of a stream row (forward: item bias * cz; nullable)
  const float* row_stat; int B;        // backward: the forward's per-user statistics, row_stat[2 B + b] = log2 sum_n 2^s2 (+inf: no teacher)
  const float* x_bias;                 // backward: item bias of an owner row (* cz; nullable)
  float cz;                            // log2(e) / (tau T): dot + bias -> log2 units
  float clip2;                         // score_clip / T in log2 units
  int owner_blocks, splits; long long tiles_per_split;
  float *part_m, *part_l, *part_o;     // forward: [splits][nx], [splits][nx], [splits][nx][d]
  const float* loss_out; const float* d_loss; float g_num;   // backward: g = g_num * d_loss / max(1, loss_out[1]),  g_num = T / tau
  float *dX, *d_bias;                  // backward: [nx, d] (row 0 = 0), [nx] (nullable)
};

__device__ __forceinline__ float distill_scale(const float* loss_out, const float* d_loss, float g_num) {
  return g_num * (d_loss ? d_loss[0] : 1.f) / fmaxf(loss_out[1], 1.f);
}

// One wave owns 32 rows of X (lane & 31 = its row, for good: as the B operand of both products and the column of both results), held as
// split fragments in registers; the workgroup streams tiles of 32 rows of Y (64 with eight waves: a wave stages 8 rows) through LDS.
//   product 1: S^T [32 stream, 32 owner] = Y X^T     -> a lane has 16 stream rows of ONE owner: maximum and sum are lane-local
//   product 2: O^T [d, 32 owner] += Y^T W            -> W is the B operand as it stands in the registers (the order of the stream rows
//              inside a K step is free: Y^T is fetched in the same order, transposed on the way out of LDS by ds_read_b64_tr_b16)
// so the running maximum, the rescale and the final scale are per-lane scalars.  Two LDS stages, one barrier a tile: the next tile's rows
// are requested before the products of this one and split into the other stage behind them.
constexpr int ds_rows(int nw) { return nw == 8 ? 64 : 32; }

template <int D, int NW, bool FWD, bool GRAD, bool CLIP>
__global__ __launch_bounds__(NW * 64, D <= 128 && NW >= 4 ? 2 : 1) void distill_stream_kernel(DistillStream a) {
  constexpr int KS = D / 16, DB = D / 32, LS = D + 8;            // LS: row stride in halves, 16 bytes of padding (b128 reads conflict-free)
  constexpr int F4 = D / 4, PER = 2 * D / 64;                    // float4 of a row; float4 a lane stages of 8 rows
  constexpr int TR = ds_rows(NW), GW = TR / 8 / NW;              // stream rows of a stage; groups of 8 rows a wave stages
  __shared__ __attribute__((aligned(16))) _Float16 Ys[2][2][TR * LS];
  __shared__ __attribute__((aligned(16))) float rb_s[2][TR];
  __shared__ int ky_s[2][TR / 8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
  // all owner blocks of one split sit on one XCD at neighbouring ids: the stream rows they share come from HBM into one L2 once
  int ob = blockIdx.x;
  long long t0 = 0, t1 = (a.ny + TR - 1) / TR;
  int split = 0;
  if constexpr (FWD) {
    const int xcd = blockIdx.x & 7, q = blockIdx.x >> 3;
    ob = q % a.owner_blocks;
    split = (q / a.owner_blocks) * 8 + xcd;
    t0 = split * a.tiles_per_split;
    t1 = min(t1, t0 + a.tiles_per_split);
  }
  const long long own = ((long long)ob * NW + wave) * 32 + col;
  const bool live = own < a.nx;

  // ---- staging: lane = (row sr of the group, columns sc .. sc + 3), rows sr + p * 64 / F4
  const int sr = lane / F4, sc = (lane % F4) * 4;
  const bool son = sc < a.d;
  float4 v[GW][PER];
  auto request = [&](long long tile) {
#pragma unroll
    for (int g = 0; g < GW; ++g)
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const long long y = min(tile * TR + (g * NW + wave) * 8 + sr + p * (64 / F4), a.ny - 1);   // (behind the end: the last row again, its bias is -inf)
        v[g][p] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (son) v[g][p] = *(const float4*)(a.Y + y * a.d + sc);
      }
  };
  auto stage = [&](long long tile, int buf) {
#pragma unroll
    for (int g = 0; g < GW; ++g) {
      const int grp = g * NW + wave;
      float mx = 0.f;
#pragma unroll
      for (int p = 0; p < PER; ++p) mx = fmaxf(fmaxf(fmaxf(mx, fabsf(v[g][p].x)), fmaxf(fabsf(v[g][p].y), fabsf(v[g][p].z))), fabsf(v[g][p].w));
      const int ky = group_exponent(group_max<64>(mx));
      const float up = pow2i(ky);
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const int at = (grp * 8 + sr + p * (64 / F4)) * LS + sc;
        half2_t h0, h1, l0, l1;
        split_pair(v[g][p].x, v[g][p].y, up, h0, l0);
        split_pair(v[g][p].z, v[g][p].w, up, h1, l1);
        *(half4*)(&Ys[buf][0][at]) = (half4){h0[0], h0[1], h1[0], h1[1]};
        *(half4*)(&Ys[buf][1][at]) = (half4){l0[0], l0[1], l1[0], l1[1]};
      }
      if (lane == 0) ky_s[buf][grp] = ky;
      if (lane < 8) {
        const long long y = tile * TR + grp * 8 + lane;
        float rb = -INFINITY;                                    // rows behind the end carry no weight
        if (y < a.ny) {
          if constexpr (FWD) rb = a.y_bias ? a.y_bias[y] * a.cz : 0.f;
          else rb = -a.row_stat[2 * (long long)a.B + y];
        }
        rb_s[buf][grp * 8 + lane] = rb;
      }
    }
  };
  if (t0 < t1) request(t0);

  // ---- owner fragments: lane (col, h) holds x[16 t + 8 h .. + 8] of its row for every K step t
  half8 xh[KS], xl[KS];
  float fl;
  {
    float mx = 0.f;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const int c = 16 * t + 8 * h;
      float4 u = make_float4(0.f, 0.f, 0.f, 0.f), w = u;
      if (live && c < a.d) u = *(const float4*)(a.X + own * a.d + c);
      if (live && c + 4 < a.d) w = *(const float4*)(a.X + own * a.d + c + 4);
      mx = fmaxf(mx, fmaxf(fmaxf(finite_abs(u.x), finite_abs(u.y)), fmaxf(finite_abs(u.z), finite_abs(u.w))));
      mx = fmaxf(mx, fmaxf(fmaxf(finite_abs(w.x), finite_abs(w.y)), fmaxf(finite_abs(w.z), finite_abs(w.w))));
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const int kx = group_exponent(mx);
    const float up = pow2i(kx);
    fl = a.cz * pow2i(-kx);
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const int c = 16 * t + 8 * h;
      float4 u = make_float4(0.f, 0.f, 0.f, 0.f), w = u;
      if (live && c < a.d) u = *(const float4*)(a.X + own * a.d + c);
      if (live && c + 4 < a.d) w = *(const float4*)(a.X + own * a.d + c + 4);
      const float x[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        half2_t hi, lo;
        split_pair(x[j], x[j + 1], up, hi, lo);
        xh[t][j] = hi[0]; xh[t][j + 1] = hi[1];
        xl[t][j] = lo[0]; xl[t][j + 1] = lo[1];
      }
    }
  }
  float xb = 0.f;
  if constexpr (!FWD) xb = (live && a.x_bias) ? a.x_bias[own] * a.cz : 0.f;

  float M = -1e30f, l = 0.f;
  int kappa = 36;                                                // O is held in units of 2^-kappa: min over the groups seen of k, + 6
  floatx16 O[GRAD ? DB : 1];
  if constexpr (GRAD) {
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) O[b][r] = 0.f;
  }

  auto compute = [&](long long tile, int buf, int sub) {
    const long long y0 = tile * TR + sub * 32;
    const _Float16 *Yh = &Ys[buf][0][sub * 32 * LS], *Yl = &Ys[buf][1][sub * 32 * LS];
    // ---- product 1
    floatx16 S;
#pragma unroll
    for (int r = 0; r < 16; ++r) S[r] = 0.f;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const half8 yh = *(const half8*)(Yh + col * LS + 16 * t + 8 * h), yl = *(const half8*)(Yl + col * LS + 16 * t + 8 * h);
      S = __builtin_amdgcn_mfma_f32_32x32x16_f16(yl, xh[t], S, 0, 0, 0);
      S = __builtin_amdgcn_mfma_f32_32x32x16_f16(yh, xl[t], S, 0, 0, 0);
      S = __builtin_amdgcn_mfma_f32_32x32x16_f16(yh, xh[t], S, 0, 0, 0);
    }
    // ---- log2 scores: register r is stream row 8 (r >> 2) + 4 h + (r & 3)
    float z[16];
    bool in[16];
    int ky[4];
    float tmax = -INFINITY;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      ky[q] = __builtin_amdgcn_readfirstlane(ky_s[buf][sub * 4 + q]);
      const float fq = fl * pow2i(-ky[q]);
      const float4 rb = *(const float4*)(&rb_s[buf][sub * 32 + 8 * q + 4 * h]);
      const float rbv[4] = {rb.x, rb.y, rb.z, rb.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * q + i;
        if constexpr (!CLIP) {
          z[r] = fmaf(S[r], fq, rbv[i]);
        } else {
          const float s = fmaf(S[r], fq, FWD ? rbv[i] : xb);
          const float c = s > a.clip2 ? a.clip2 : (s < -a.clip2 ? -a.clip2 : s);   // (a NaN stays one)
          in[r] = !(s > a.clip2) && !(s < -a.clip2);
          if constexpr (FWD) z[r] = y0 + 8 * q + 4 * h + i < a.ny ? c : -INFINITY;
          else z[r] = c + rbv[i];
        }
      }
      tmax = fmaxf(fmaxf(tmax, fmaxf(z[4 * q], z[4 * q + 1])), fmaxf(z[4 * q + 2], z[4 * q + 3]));
    }
    const int kmin = min(min(ky[0], ky[1]), min(ky[2], ky[3])) + 6;
    // ---- a new reference only when a weight would pass 2^8 (or a larger group arrives): weights reach 2^(8 + 6) = fp16's range
    if (kmin < kappa || __any(tmax > M + 8.f)) {
      const float m2 = fmaxf(tmax, __shfl_xor(tmax, 32, 64)), Mn = m2 > M + 8.f ? m2 : M;
      const int kn = min(kmin, kappa);
      const float f = __builtin_amdgcn_exp2f(M - Mn), fo = f * exp2f((float)(kn - kappa));
      l *= f;
      if constexpr (GRAD) {
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) O[b][r] *= fo;
      }
      M = Mn;
      kappa = kn;
    }
    half8 wh[2], wl[2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float mk = M - (float)(kappa - ky[q]);
      float w[4], lq = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * q + i;
        w[i] = __builtin_amdgcn_exp2f(z[r] - mk);
        if constexpr (CLIP && !FWD) w[i] = in[r] ? w[i] : 0.f;
        lq += w[i];
        if constexpr (CLIP && FWD) w[i] = in[r] ? w[i] : 0.f;
      }
      l = fmaf(lq, pow2i(ky[q] - kappa), l);
      if constexpr (GRAD) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          half2_t hi, lo;
          split_pair(w[i], w[i + 1], 1.f, hi, lo);
          wh[q >> 1][4 * (q & 1) + i] = hi[0]; wh[q >> 1][4 * (q & 1) + i + 1] = hi[1];
          wl[q >> 1][4 * (q & 1) + i] = lo[0]; wl[q >> 1][4 * (q & 1) + i + 1] = lo[1];
        }
      }
    }
    // ---- product 2
    if constexpr (GRAD) {
      const int i16 = lane & 15, cg = (lane >> 4) & 1;
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          half8 yh, yl;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int off = (16 * t + 8 * q + 4 * h + (i16 >> 2)) * LS + 32 * b + 16 * cg + 4 * (i16 & 3);
            const half4 th = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(Yh + off)));
            const half4 tl = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(Yl + off)));
#pragma unroll
            for (int j = 0; j < 4; ++j) { yh[4 * q + j] = th[j]; yl[4 * q + j] = tl[j]; }
          }
          O[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(yl, wh[t], O[b], 0, 0, 0);
          O[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(yh, wl[t], O[b], 0, 0, 0);
          O[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(yh, wh[t], O[b], 0, 0, 0);
        }
    }
  };
  if (t0 < t1) stage(t0, 0);
  __syncthreads();
  int buf = 0;
  for (long long tile = t0; tile < t1; ++tile, buf ^= 1) {
    if (tile + 1 < t1) request(tile + 1);
#pragma unroll
    for (int sub = 0; sub < TR / 32; ++sub) compute(tile, buf, sub);
    if (tile + 1 < t1) stage(tile + 1, buf ^ 1);                 // (its last readers passed the barrier of the tile before)
    __syncthreads();
  }
  // ---- out
  l += __shfl_xor(l, 32, 64);
  if (!live) return;
  if constexpr (FWD) {
    const long long at = (long long)split * a.nx + own;
    if (h == 0) {
      a.part_m[at] = M;
      a.part_l[at] = l;
    }
    if constexpr (GRAD) {
      const float down = exp2f((float)-kappa);
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 32 * b + 8 * q + 4 * h;
          if (c < a.d)
            *(float4*)(a.part_o + at * a.d + c) = make_float4(O[b][4 * q] * down, O[b][4 * q + 1] * down, O[b][4 * q + 2] * down, O[b][4 * q + 3] * down);
        }
    }
  } else {
    const float g = distill_scale(a.loss_out, a.d_loss, a.g_num), e = CLIP ? 0.f : xb;
    if (h == 0 && a.d_bias) a.d_bias[own] = l * exp2f(M + e) * g;
    const float down = own == 0 ? 0.f : exp2f(M + e - (float)kappa) * g;   // padding row: no gradient
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = 32 * b + 8 * q + 4 * h;
        if (c < a.d)
          *(float4*)(a.dX + own * a.d + c) = own == 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
              : make_float4(O[b][4 * q] * down, O[b][4 * q + 1] * down, O[b][4 * q + 2] * down, O[b][4 * q + 3] * down);
      }
  }
}

// ---- teacher scores in the type they were stored in
__device__ __forceinline__ float teacher_at(const void* p, int type, long long i) {
  if (type == UR_F16) return (float)((const _Float16*)p)[i];
  if (type == UR_BF16) return __uint_as_float((unsigned)((const unsigned short*)p)[i] << 16);
  return ((const float*)p)[i];
}

struct DistillRow {
  const float* U; const float* E; long long N; int B, d, K, splits;
  const float *part_m, *part_l, *part_o;
  const long long* id; const void* score; int score_type;
  const float* item_bias;
  float inv_tau, inv_T, clip;
  float* lse;
  float* stat;                         // [0, B) loss of the row, [B, 2B) 1 = has a teacher, [2B, 3B) log2 of the softmax sum (+inf without a teacher)
  float* coef; long long* tid;         // [B, K]: p (0 where the gradient is cut), item (0 = absent)
  float* d_unit;                       // [B, d]: O_b - sum_k p E
  IdGuard guard;
};

__device__ __forceinline__ float ds_block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}
__device__ __forceinline__ float ds_block_max(float v, float* red) {
  v = group_max<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// One workgroup per user: the splits' partials folded in order, the teacher's softmax, its K rows gathered once (dot for the loss and
// weighted sum for the gradient).  TPR lanes hold a row as float4.
template <int TPR, bool GRAD>
__global__ __launch_bounds__(256) void distill_row_kernel(DistillRow a) {
  constexpr int G = 256 / TPR;
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) float4 acc_s[256];
  const int b = blockIdx.x, tid = threadIdx.x, g = tid / TPR, t = tid % TPR, d4 = a.d / 4;
  const bool on = t < d4;
  float m = -INFINITY;
  for (int s = tid; s < a.splits; s += 256) m = fmaxf(m, a.part_m[(long long)s * a.B + b]);
  m = ds_block_max(m, red);
  float l = 0.f;
  for (int s = tid; s < a.splits; s += 256) l += a.part_l[(long long)s * a.B + b] * exp2f(a.part_m[(long long)s * a.B + b] - m);
  l = ds_block_sum(l, red);
  const float lse2 = m + log2f(l), lse = lse2 * DS_LN2;
  // ---- the teacher's softmax
  float tm = -INFINITY, ts = 0.f;
  for (int k = tid; k < a.K; k += 256) {
    const long long i = (long long)b * a.K + k;
    long long id = a.id[i];
    if (id < -1 || id >= a.N) id = ur_guard_id(id, a.N, a.guard);   // not an item at all: the guard goes up, the entry is absent
    const float v = teacher_at(a.score, a.score_type, i) * a.inv_T;
    if (id >= 1 && v > -INFINITY) tm = fmaxf(tm, v);
  }
  tm = ds_block_max(tm, red);
  const bool some = tm > -INFINITY;
  for (int k = tid; k < a.K; k += 256) {
    const long long i = (long long)b * a.K + k, id = a.id[i];
    const float v = teacher_at(a.score, a.score_type, i) * a.inv_T;
    if (id >= 1 && id < a.N && v > -INFINITY) ts += expf(v - tm);
  }
  ts = ds_block_sum(ts, red);
  const float log_ts = logf(ts);
  // ---- its rows
  float4 u = make_float4(0.f, 0.f, 0.f, 0.f), acc = u;
  if (on) u = ((const float4*)a.U)[(long long)b * d4 + t];
  float loss = 0.f;
  for (int k = g; k < a.K; k += G) {
    const long long i = (long long)b * a.K + k, id = a.id[i];
    const float v = teacher_at(a.score, a.score_type, i) * a.inv_T;
    const bool there = some && id >= 1 && id < a.N && v > -INFINITY;
    float p = 0.f;
    if (there) {
      float4 e = make_float4(0.f, 0.f, 0.f, 0.f);
      if (on) e = ((const float4*)a.E)[id * d4 + t];
      const float dot = group_sum<TPR>((u.x * e.x + u.y * e.y) + (u.z * e.z + u.w * e.w));
      float s = (dot + (a.item_bias ? a.item_bias[id] : 0.f)) * a.inv_tau;
      const bool cut = a.clip > 0.f && (s > a.clip || s < -a.clip);
      if (cut) s = s > 0.f ? a.clip : -a.clip;
      const float logp = v - tm - log_ts;
      p = expf(logp);
      if (t == 0) loss += p * (logp - s * a.inv_T + lse);
      if (cut) p = 0.f;
      acc.x -= p * e.x; acc.y -= p * e.y; acc.z -= p * e.z; acc.w -= p * e.w;
    }
    if (GRAD && t == 0) {
      a.coef[i] = p;
      a.tid[i] = there ? id : 0;
    }
  }
  loss = ds_block_sum(loss, red);
  if (tid == 0) {
    a.lse[b] = lse;
    a.stat[b] = loss;
    a.stat[a.B + b] = some ? 1.f : 0.f;
    a.stat[2 * (long long)a.B + b] = some ? lse2 : INFINITY;
  }
  if constexpr (GRAD) {
    for (int s = g; s < a.splits; s += G) {
      const long long at = (long long)s * a.B + b;
      const float f = exp2f(a.part_m[at] - lse2);
      if (on) {
        const float4 o = ((const float4*)a.part_o)[at * d4 + t];
        acc.x += f * o.x; acc.y += f * o.y; acc.z += f * o.z; acc.w += f * o.w;
      }
    }
    acc_s[tid] = acc;
    __syncthreads();
    if (tid < d4) {
      float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = 0; q < G; ++q) {
        const float4 v = acc_s[q * TPR + tid];
        r.x += v.x; r.y += v.y; r.z += v.z; r.w += v.w;
      }
      if (!some) r = make_float4(0.f, 0.f, 0.f, 0.f);
      ((float4*)a.d_unit)[(long long)b * d4 + tid] = r;
    }
  }
}

// loss_out = [T^2 / C sum of the rows' losses, C, update guard, -] (single block, fixed order)
__global__ __launch_bounds__(256) void distill_loss_kernel(const float* __restrict__ stat, int B, float T2, float* __restrict__ loss_out) {
  __shared__ float red[4];
  float s = 0.f, c = 0.f;
  for (int b = threadIdx.x; b < B; b += 256) {
    s += stat[b];
    c += stat[B + b];
  }
  s = ds_block_sum(s, red);
  c = ds_block_sum(c, red);
  if (threadIdx.x == 0) {
    loss_out[0] = T2 * s / fmaxf(c, 1.f);
    loss_out[1] = c;
    loss_out[2] = s != s ? -1.f : 1.f;   // update guard (see ur_gather_dot_loss_fwd)
    loss_out[3] = 0.f;
  }
}

struct DistillApply {
  const int *uniq, *seg, *pos, *n_uniq;
  const float *coef, *U, *d_unit;
  int B, d, K;
  const float* loss_out; const float* d_loss; float g_num;
  float *d_user, *d_table, *d_bias;
  int user_blocks;
};
// the first user_blocks workgroups: d_user = g d_unit; the others: a group of TPR lanes per distinct teacher item,
// dE[item] -= g sum p u (the plan's order: bit-reproducible), d_bias[item] -= g sum p
template <int TPR>
__global__ __launch_bounds__(256) void distill_apply_kernel(DistillApply a) {
  constexpr int G = 256 / TPR;
  const float g = distill_scale(a.loss_out, a.d_loss, a.g_num);
  const int d4 = a.d / 4;
  if ((int)blockIdx.x < a.user_blocks) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < (long long)a.B * d4) {
      const float4 v = ((const float4*)a.d_unit)[i];
      ((float4*)a.d_user)[i] = make_float4(g * v.x, g * v.y, g * v.z, g * v.w);
    }
    return;
  }
  const int n = *a.n_uniq, t = threadIdx.x % TPR;
  for (long long q = (long long)(blockIdx.x - a.user_blocks) * G + threadIdx.x / TPR; q < n; q += (long long)(gridDim.x - a.user_blocks) * G) {
    const int item = a.uniq[q];
    if (item == 0) continue;                                    // absent entries
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float pb = 0.f;
    for (int s = a.seg[q]; s < a.seg[q + 1]; ++s) {
      const int at = a.pos[s];
      const float p = a.coef[at];
      pb += p;
      if (t < d4) {
        const float4 u = ((const float4*)a.U)[(long long)(at / a.K) * d4 + t];
        acc.x += p * u.x; acc.y += p * u.y; acc.z += p * u.z; acc.w += p * u.w;
      }
    }
    if (t < d4) {
      float4* o = (float4*)a.d_table + (long long)item * d4 + t;
      const float4 v = *o;
      *o = make_float4(v.x - g * acc.x, v.y - g * acc.y, v.z - g * acc.z, v.w - g * acc.w);
    }
    if (t == 0 && a.d_bias) a.d_bias[item] -= g * pb;
  }
}

static inline int ds_tpr(int d) { return d <= 64 ? 16 : d <= 128 ? 32 : 64; }
static inline int ds_nw(int B, int d) { return B <= 32 ? 1 : B <= 64 ? 2 : B <= 128 || d > 128 ? 4 : 8; }

// the catalogue is cut into splits (a multiple of the 8 XCDs) so that about two workgroups per CU are in flight
static void ds_splits(int B, int d, long long N, int* owner_blocks, int* splits, long long* per) {
  const int nw = ds_nw(B, d);
  *owner_blocks = cdiv(B, 32 * nw);
  const long long tiles = (N + ds_rows(nw) - 1) / ds_rows(nw);
  const long long want = std::max<long long>(1, 2048 / nw / *owner_blocks);
  long long s = std::min(want, (tiles + 1) / 2);
  s = std::max<long long>(8, (s + 7) / 8 * 8);
  *per = (tiles + s - 1) / s;
  *splits = (int)s;
}

struct DistillWs {
  float *part_m, *part_l, *part_o;                                   // forward
  int *uniq, *seg, *pos, *n_uniq; char* plan;                       // backward
  int64_t bytes;
};
static DistillWs ds_carve(int B, int d, long long N, int K, int grad, char* base) {
  DistillWs w{};
  int64_t o = 0;
  auto take = [&](int64_t n) {
    char* p = base ? base + o : nullptr;
    o += (n + 255) & ~(int64_t)255;
    return p;
  };
  int ob, splits;
  long long per;
  ds_splits(B, d, N, &ob, &splits, &per);
  w.part_m = (float*)take((int64_t)splits * B * 4);
  w.part_l = (float*)take((int64_t)splits * B * 4);
  if (grad) {
    w.part_o = (float*)take((int64_t)splits * B * d * 4);
    const int64_t n = (int64_t)B * K, fwd = o;
    o = 0;                                                          // the backward reuses the forward's partials
    w.uniq = (int*)take(n * 4); w.seg = (int*)take((n + 1) * 4); w.pos = (int*)take(n * 4); w.n_uniq = (int*)take(4);
    w.plan = take(ur_rows_plan_workspace_bytes(n));
    o = std::max(o, fwd);
  }
  w.bytes = o;
  return w;
}

template <int D, int NW, bool FWD, bool GRAD>
static int ds_launch_stream(const DistillStream& a, bool clip, int grid, hipStream_t st) {
  if (clip) hipLaunchKernelGGL((distill_stream_kernel<D, NW, FWD, GRAD, true>), dim3(grid), dim3(NW * 64), 0, st, a);
  else hipLaunchKernelGGL((distill_stream_kernel<D, NW, FWD, GRAD, false>), dim3(grid), dim3(NW * 64), 0, st, a);
  UR_LAUNCH_CHECK();
  return UR_OK;
}
template <int D>
static int ds_launch_fwd(const DistillStream& a, bool grad, bool clip, int nw, int grid, hipStream_t st) {
#define GO(W) (grad ? ds_launch_stream<D, W, true, true>(a, clip, grid, st) : ds_launch_stream<D, W, true, false>(a, clip, grid, st))
  if constexpr (D <= 128) {
    if (nw == 8) return GO(8);
  }
  return nw == 1 ? GO(1) : nw == 2 ? GO(2) : GO(4);
#undef GO
}

static int ds_check(const float* user_emb, const float* table, int64_t N, int B, int d, int K, float tau, float T, const char* who) {
  UR_REQUIRE(user_emb && table, UR_ERR_ARG, "%s: null pointer", who);
  UR_REQUIRE(B > 0 && d > 0 && d % 4 == 0 && N > 1 && N < (1LL << 31) && K > 0, UR_ERR_ARG, "%s: shape", who);
  UR_REQUIRE(d <= DS_MAX_D, UR_ERR_UNSUPPORTED, "%s: d=%d (at most %d)", who, d, DS_MAX_D);
  UR_REQUIRE((int64_t)B * K < (1LL << 31), UR_ERR_ARG, "%s: B * K = %lld", who, (long long)B * K);
  UR_REQUIRE(tau > 0.f && T > 0.f && tau < INFINITY && T < INFINITY, UR_ERR_ARG, "%s: tau=%g and temperature=%g must be positive", who, tau, T);
  return UR_OK;
}

}  // namespace ur

using namespace ur;

extern "C" int64_t ur_full_distill_workspace_bytes(int32_t B, int32_t d, int64_t n_items, int32_t K, int32_t need_grad) {
  if (B <= 0 || d <= 0 || n_items <= 1 || K <= 0 || (int64_t)B * K >= (1LL << 31)) return UR_ERR_ARG;
  return ds_carve(B, d, n_items, K, need_grad, nullptr).bytes;
}

extern "C" int ur_full_distill_fwd(const float* user_emb, const float* item_table, int64_t n_items, int32_t B, int32_t d,
                                   const int64_t* teacher_id, const void* teacher_score, int32_t score_type, int32_t K, const float* item_bias,
                                   float tau, float score_clip, float temperature, float* lse, float* loss_out, float* row_stat, float* coef,
                                   int64_t* entry_id, float* d_unit, void* ws, void* stream) {
  UR_TRACE_SCOPE();
  int rc = ds_check(user_emb, item_table, n_items, B, d, K, tau, temperature, "ur_full_distill_fwd");
  if (rc) return rc;
  UR_REQUIRE(teacher_id && teacher_score && lse && loss_out && row_stat && ws, UR_ERR_ARG, "ur_full_distill_fwd: null pointer");
  UR_REQUIRE(score_type == UR_F32 || score_type == UR_F16 || score_type == UR_BF16, UR_ERR_ARG, "ur_full_distill_fwd: score_type=%d", score_type);
  const bool grad = d_unit != nullptr;
  UR_REQUIRE(grad == (coef != nullptr) && grad == (entry_id != nullptr), UR_ERR_ARG,
             "ur_full_distill_fwd: coef, entry_id and d_unit go together (all of them for a backward pass, none without)");
  hipStream_t st = as_stream(stream);
  ProfScope ps(PC_LOSS, st, (grad ? 4.0 : 2.0) * B * (double)n_items * d);
  const DistillWs w = ds_carve(B, d, n_items, K, grad, (char*)ws);
  DistillStream a{};
  a.X = user_emb; a.nx = B; a.Y = item_table; a.ny = n_items; a.d = d; a.y_bias = item_bias; a.B = B;
  a.cz = DS_LOG2E / (tau * temperature); a.clip2 = score_clip > 0.f ? score_clip / temperature * DS_LOG2E : 0.f;
  ds_splits(B, d, n_items, &a.owner_blocks, &a.splits, &a.tiles_per_split);
  a.part_m = w.part_m; a.part_l = w.part_l; a.part_o = w.part_o;
  const int nw = ds_nw(B, d), grid = a.owner_blocks * a.splits;
  const bool clip = score_clip > 0.f;
  rc = d <= 32 ? ds_launch_fwd<32>(a, grad, clip, nw, grid, st) : d <= 64 ? ds_launch_fwd<64>(a, grad, clip, nw, grid, st)
     : d <= 128 ? ds_launch_fwd<128>(a, grad, clip, nw, grid, st) : ds_launch_fwd<256>(a, grad, clip, nw, grid, st);
  if (rc) return rc;
  DistillRow r{};
  r.U = user_emb; r.E = item_table; r.N = n_items; r.B = B; r.d = d; r.K = K; r.splits = a.splits;
  r.part_m = w.part_m; r.part_l = w.part_l; r.part_o = w.part_o;
  r.id = (const long long*)teacher_id; r.score = teacher_score; r.score_type = score_type; r.item_bias = item_bias;
  r.inv_tau = 1.f / tau; r.inv_T = 1.f / temperature; r.clip = score_clip;
  r.lse = lse; r.stat = row_stat; r.coef = coef; r.tid = (long long*)entry_id; r.d_unit = d_unit; r.guard = id_guard();
#define GO(T) do { if (grad) hipLaunchKernelGGL((distill_row_kernel<T, true>), dim3(B), dim3(256), 0, st, r); \
                   else hipLaunchKernelGGL((distill_row_kernel<T, false>), dim3(B), dim3(256), 0, st, r); } while (0)
  switch (ds_tpr(d)) {
    case 16: GO(16); break;
    case 32: GO(32); break;
    default: GO(64); break;
  }
#undef GO
  UR_LAUNCH_CHECK();
  hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(256), 0, st, row_stat, B, temperature * temperature, loss_out);
  UR_LAUNCH_CHECK();
  return UR_OK;
}

extern "C" int ur_full_distill_bwd(const float* user_emb, const float* item_table, int64_t n_items, int32_t B, int32_t d, int32_t K,
                                   const float* item_bias, float tau, float score_clip, float temperature, const float* loss_out,
                                   const float* row_stat, const float* coef, const int64_t* entry_id, const float* d_unit, const float* d_loss,
                                   float* d_user_emb, float* d_item_table, float* d_item_bias, void* ws, void* stream) {
  UR_TRACE_SCOPE();
  int rc = ds_check(user_emb, item_table, n_items, B, d, K, tau, temperature, "ur_full_distill_bwd");
  if (rc) return rc;
  UR_REQUIRE(loss_out && row_stat && coef && entry_id && d_unit && d_user_emb && d_item_table && ws, UR_ERR_ARG, "ur_full_distill_bwd: null pointer");
  UR_REQUIRE(!item_bias || d_item_bias, UR_ERR_ARG, "ur_full_distill_bwd: d_item_bias is required when item_bias is given");
  hipStream_t st = as_stream(stream);
  const DistillWs w = ds_carve(B, d, n_items, K, 1, (char*)ws);
  rc = ur_rows_plan(nullptr, 0, entry_id, (int64_t)B * K, n_items, w.uniq, w.seg, w.pos, w.n_uniq, w.plan, stream);
  if (rc) return rc;
  ProfScope ps(PC_LOSS, st, 4.0 * B * (double)n_items * d);
  DistillStream a{};
  a.X = item_table; a.nx = n_items; a.Y = user_emb; a.ny = B; a.d = d; a.row_stat = row_stat; a.B = B; a.x_bias = item_bias;
  a.cz = DS_LOG2E / (tau * temperature); a.clip2 = score_clip > 0.f ? score_clip / temperature * DS_LOG2E : 0.f;
  a.loss_out = loss_out; a.d_loss = d_loss; a.g_num = temperature / tau; a.dX = d_item_table; a.d_bias = d_item_bias;
  const bool clip = score_clip > 0.f;
  const int grid = cdiv(n_items, 128);
  rc = d <= 32 ? ds_launch_stream<32, 4, false, true>(a, clip, grid, st) : d <= 64 ? ds_launch_stream<64, 4, false, true>(a, clip, grid, st)
     : d <= 128 ? ds_launch_stream<128, 4, false, true>(a, clip, grid, st) : ds_launch_stream<256, 4, false, true>(a, clip, grid, st);
  if (rc) return rc;
  DistillApply p{};
  p.uniq = w.uniq; p.seg = w.seg; p.pos = w.pos; p.n_uniq = w.n_uniq; p.coef = coef; p.U = user_emb; p.d_unit = d_unit;
  p.B = B; p.d = d; p.K = K; p.loss_out = loss_out; p.d_loss = d_loss; p.g_num = temperature / tau;
  p.d_user = d_user_emb; p.d_table = d_item_table; p.d_bias = d_item_bias; p.user_blocks = cdiv((long long)B * (d / 4), 256);
  const int tpr = ds_tpr(d), item_blocks = (int)std::min<int64_t>(cdiv((int64_t)B * K, 256 / tpr), 4096);
#define GO(T) hipLaunchKernelGGL((distill_apply_kernel<T>), dim3(p.user_blocks + item_blocks), dim3(256), 0, st, p)
  switch (tpr) {
    case 16: GO(16); break;
    case 32: GO(32); break;
    default: GO(64); break;
  }
#undef GO
  UR_LAUNCH_CHECK();
  return UR_OK;
}
