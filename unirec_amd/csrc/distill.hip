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
// The teacher's K entries a row are sparse: gathered once in the forward, which leaves them as short lists by (tile of 32 users, bucket of
// items); a workgroup per bucket adds them to the table gradient, in the order of the users.  Nothing is sorted over the whole batch (that
// took 6 launches and 32 of 115 us at 60 K items, 512 users x 50 entries); taking the lists inside the stream kernel cost more than it saved
// (35 -> 47 - 55 us there, its one barrier a tile waits for the wave that has entries, and D = 128 has no register left for it).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace ur {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr float DS_LOG2E = 1.44269504088896340736f, DS_LN2 = 0.69314718055994530942f;
constexpr int DS_MAX_D = 256;
constexpr int DS_MAX_K = 65536;   // an item listed twice is found by comparing a list's entries with each other: 2.3 ms for 4 096 of them, 34 for 16 384, 135 for 32 768

// ---- fp32 products on the fp16 matrix pipes.  x 2^k = hi + lo with hi = fp16(x 2^k), lo = fp16(x 2^k - hi): 22 bits of every value that
// is within 2^-17 of its group's largest (k puts that at 2^13), an absolute floor of 2^-38 of the largest below.  x y is accumulated in
// fp32 from hi hi, hi lo and lo hi; the dropped lo lo is below 2^-22 |x y|, of the order of one fp32 rounding.  Three products where the
// bf16 split of gemm.hip needs six: fp16's short exponent is what the group exponents k pay for.
// The softmax' weights have no exponent of their own: the largest of a row stands at 2^6 to 2^14, so one that is 2^-31 of it or less is 0 or 2^-30 of
// it to product 2 (l has it in fp32).  The sum it goes into is fp32 and takes 32 weights at a time, of which it loses what is below 2^-25 of it: 2^-30 a
// weight.  (Carrying what a weight loses on to the next one changed d_user's error by 3 in 100 in rows of a peak and a flat tail 16 to 22 below.)
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

// ---- a tile of 32 stream rows, split: [hi | lo][32][D] halves.  Rows are not padded; the 16-byte units of row r are permuted by XOR with
// ds_swizzle(r), which keeps both readers free of bank conflicts: the 8 consecutive rows of a b128 read and the 4 rows x 32 bytes of a
// transposing read land in 8 different 16-byte bank groups.
constexpr int DS_TILE = 32;
template <int D>
__device__ __forceinline__ int ds_swizzle(int r) {
  return D >= 64 ? ((r & 3) << 1) | ((r >> 2) & 1) : (((r >> 1) & 1) << 1) | ((r >> 2) & 1);
}
template <int D>
__device__ __forceinline__ int ds_at(int r, int c) { return r * D + (((c >> 3) ^ ds_swizzle<D>(r)) << 3) + (c & 7); }

struct DistillStream {
  const float* X; long long nx;        // owner rows [nx, d]
  const float* Y; long long ny;        // stream rows [ny, d] (forward; the backward's come from the image)
  int d;
  const float* y_bias;                 // forward: added to the log2 score of a stream row (item bias * cz; nullable)
  const _Float16* img; const float* rb_img; const int* ky_img;   // backward: the users' rows split tile by tile, their bias, a tile's exponent
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

// One wave owns 32 rows of X as two column blocks of 16 (lane & 15 = the row of a block, for good: the B operand of both products and the
// column of both results), held as split fragments in registers; the workgroup streams tiles of 32 rows of Y through LDS.
//   product 1: S^T [32 stream, 32 owner] = Y X^T     -> a lane has 8 stream rows (16 rb + 4 (lane >> 4) + r) of each of TWO owners
//   product 2: O^T [d, 32 owner] += Y^T W            -> W is the B operand as it stands in the registers (the order of the stream rows
//              inside a K step is free: Y^T is fetched in the same order, transposed on the way out of LDS by ds_read_b64_tr_b16)
// so the running maximum, the rescale and the final scale are per-lane.  v_mfma_f32_16x16x32_f16 rather than 32x32x16: the same flops
// ran at 2 050 - 2 160 TFLOP/s against 1 720 - 1 820 in a loop of nothing else (the part is power-limited there).
// Three LDS stages, one barrier a tile: while the weights of tile t are made (VALU), product 1 of tile t + 1 runs on the matrix pipe, and
// tile t + 2 or t + 3 arrives (forward: fp32 rows through registers, split here with one exponent a tile, which the waves agree on a
// barrier ahead; backward: the image's bytes straight into LDS).
typedef __attribute__((address_space(1))) const void* ds_gptr;
typedef __attribute__((address_space(3))) void* ds_lptr;

template <int D, int NW, bool FWD, bool GRAD, bool CLIP>
__global__ __launch_bounds__(NW * 64, D <= 128 && NW >= 4 ? 2 : 1) void distill_stream_kernel(DistillStream a) {
  constexpr int KS = D / 32, DB = D / 16;                        // K steps of product 1; 16-column blocks of product 2
  constexpr int N1 = 2 * KS, N1a = N1 > 4 ? 2 : 1;               // steps of product 1 (K step, row block); those in front of the maximum
  constexpr int F4 = D / 4, PER = DS_TILE * F4 / (64 * NW);      // float4 of a row; float4 a thread stages of a tile
  constexpr int HALF = DS_TILE * D;                              // lo plane, in halves behind the hi plane
  __shared__ __attribute__((aligned(1024))) _Float16 Ys[3][2 * HALF];
  __shared__ __attribute__((aligned(16))) float rb_s[3][DS_TILE];
  __shared__ int kw_s[2][NW];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  // all owner blocks of one split sit on one XCD at neighbouring ids: the stream rows they share come from HBM into one L2 once
  int ob = blockIdx.x;
  long long t0 = 0, t1 = (a.ny + DS_TILE - 1) / DS_TILE;
  int split = 0;
  if constexpr (FWD) {
    const int xcd = blockIdx.x & 7, q = blockIdx.x >> 3;
    ob = q % a.owner_blocks;
    split = (q / a.owner_blocks) * 8 + xcd;
    t0 = split * a.tiles_per_split;
    t1 = min(t1, t0 + a.tiles_per_split);
  }
  const long long own0 = ((long long)ob * NW + wave) * 32 + col;   // and own0 + 16

  // ---- staging, forward: thread = (row sr + p * 64 NW / F4, columns sc .. sc + 3)
  const int sr = threadIdx.x / F4, sc = (threadIdx.x % F4) * 4;
  const bool son = sc < a.d;
  float4 v[FWD ? PER : 1];
  float rb_next = 0.f;
  auto request = [&](long long tile, int buf) {
    if constexpr (FWD) {
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const long long y = min(tile * DS_TILE + sr + p * (64 * NW / F4), a.ny - 1);   // (behind the end: the last row again, its bias is -inf)
        v[p] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (son) v[p] = *(const float4*)(a.Y + y * a.d + sc);
      }
      if (threadIdx.x < DS_TILE) {
        const long long y = tile * DS_TILE + threadIdx.x;
        rb_next = y < a.ny ? (a.y_bias ? a.y_bias[y] * a.cz : 0.f) : -INFINITY;        // rows behind the end carry no weight
      }
    } else {
      const char* src = (const char*)(a.img + tile * (2 * HALF)) + lane * 16;
      char* dst = (char*)&Ys[buf][0];
#pragma unroll
      for (int i = 0; i < 4 * HALF / 1024 / NW; ++i) {
        const int piece = (i * NW + wave) * 1024;
        __builtin_amdgcn_global_load_lds((ds_gptr)(src + piece), (ds_lptr)(dst + piece), 16, 0, 0);
      }
      if (threadIdx.x < DS_TILE) rb_next = a.rb_img[tile * DS_TILE + threadIdx.x];
    }
  };
  auto publish = [&](int par) {   // this wave's exponent for the rows it holds
    float mx = 0.f;
#pragma unroll
    for (int p = 0; p < PER; ++p) mx = fmaxf(fmaxf(fmaxf(mx, fabsf(v[p].x)), fmaxf(fabsf(v[p].y), fabsf(v[p].z))), fabsf(v[p].w));
    mx = group_max<64>(mx);
    if (lane == 0) kw_s[par][wave] = group_exponent(mx);
  };
  auto agreed = [&](int par) {
    int k = kw_s[par][0];
#pragma unroll
    for (int w = 1; w < NW; ++w) k = min(k, kw_s[par][w]);
    return __builtin_amdgcn_readfirstlane(k);
  };
  auto convert = [&](int buf, int ky) {
    const float up = pow2i(ky);
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = ds_at<D>(sr + p * (64 * NW / F4), sc);
      half2_t h0, h1, l0, l1;
      split_pair(v[p].x, v[p].y, up, h0, l0);
      split_pair(v[p].z, v[p].w, up, h1, l1);
      *(half4*)(&Ys[buf][at]) = (half4){h0[0], h0[1], h1[0], h1[1]};
      *(half4*)(&Ys[buf][HALF + at]) = (half4){l0[0], l0[1], l1[0], l1[1]};
    }
  };
  auto put_bias = [&](int buf) {
    if (threadIdx.x < DS_TILE) rb_s[buf][threadIdx.x] = rb_next;
  };
  auto arrive = [&]() {   // backward: this wave's bytes are in LDS (the barrier speaks for every wave's)
    if constexpr (!FWD) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  if (t0 < t1) request(t0, 0);

  // ---- owner fragments: lane (col, g) holds x[32 t + 8 g .. + 8] of its two rows for every K step t
  half8 xh[2][KS], xl[2][KS];
  float fl[2], xb[2] = {0.f, 0.f};
#pragma unroll
  for (int cb = 0; cb < 2; ++cb) {
    const long long own = own0 + 16 * cb;
    const bool live = own < a.nx;
    float4 u[KS], w[KS];
    float mx = 0.f;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const int c = 32 * t + 8 * g;
      u[t] = w[t] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (live && c < a.d) u[t] = *(const float4*)(a.X + own * a.d + c);
      if (live && c + 4 < a.d) w[t] = *(const float4*)(a.X + own * a.d + c + 4);
      mx = fmaxf(mx, fmaxf(fmaxf(finite_abs(u[t].x), finite_abs(u[t].y)), fmaxf(finite_abs(u[t].z), finite_abs(u[t].w))));
      mx = fmaxf(mx, fmaxf(fmaxf(finite_abs(w[t].x), finite_abs(w[t].y)), fmaxf(finite_abs(w[t].z), finite_abs(w[t].w))));
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const int kx = group_exponent(mx);
    const float up = pow2i(kx);
    fl[cb] = a.cz * pow2i(-kx);
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const float x[8] = {u[t].x, u[t].y, u[t].z, u[t].w, w[t].x, w[t].y, w[t].z, w[t].w};
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        half2_t hi, lo;
        split_pair(x[j], x[j + 1], up, hi, lo);
        xh[cb][t][j] = hi[0]; xh[cb][t][j + 1] = hi[1];
        xl[cb][t][j] = lo[0]; xl[cb][t][j + 1] = lo[1];
      }
    }
    if constexpr (!FWD) xb[cb] = (live && a.x_bias) ? a.x_bias[own] * a.cz : 0.f;
  }

  float M[2] = {-1e30f, -1e30f}, l[2] = {0.f, 0.f};
  int kappa = 36;                                                // O is held in units of 2^-kappa: min over the tiles seen of k, + 6
  floatx4 O[GRAD ? DB : 1][2];
  if constexpr (GRAD) {
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) O[b][cb] = (floatx4){0.f, 0.f, 0.f, 0.f};
  }
  // byte offsets of this lane's fragments inside a tile (K step t: ^ 64 t; row block: + 16 rows; column block b: ^ 32 b)
  const int frag = 2 * ds_at<D>(col, 8 * g), frag_t = 2 * ds_at<D>(4 * g + (col >> 2), 4 * (col & 3));

  // a fragment pair (hi, lo): step i of product 1 is (K step i >> 1, row block i & 1), step b of product 2 a block of 16 columns
  auto read1 = [&](int buf, int i, half8& yh, half8& yl) {
    const char* at = (const char*)&Ys[buf][0] + (frag ^ (64 * (i >> 1))) + (i & 1) * 32 * D;
    yh = *(const half8*)at;
    yl = *(const half8*)(at + 2 * HALF);
  };
  auto read2 = [&](int buf, int b, half8& yh, half8& yl) {
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const char* at = (const char*)&Ys[buf][0] + (frag_t ^ (32 * b)) + rb * 32 * D;
      const half4 th = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)at));
      const half4 tl = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(at + 2 * HALF)));
#pragma unroll
      for (int j = 0; j < 4; ++j) { yh[4 * rb + j] = th[j]; yl[4 * rb + j] = tl[j]; }
    }
  };
  auto mac = [](floatx4& P0, floatx4& P1, const half8& yh, const half8& yl, const half8& h0, const half8& l0, const half8& h1, const half8& l1) {
    P0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(yl, h0, P0, 0, 0, 0);
    P1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(yl, h1, P1, 0, 0, 0);
    P0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(yh, l0, P0, 0, 0, 0);
    P1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(yh, l1, P1, 0, 0, 0);
    P0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(yh, h0, P0, 0, 0, 0);
    P1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(yh, h1, P1, 0, 0, 0);
  };
  struct Scores { floatx4 at[2][2]; };                           // [row block][owner block]
  auto clear = [](Scores& P) {
#pragma unroll
    for (int i = 0; i < 4; ++i) P.at[i >> 1][i & 1] = (floatx4){0.f, 0.f, 0.f, 0.f};
  };
  auto product1 = [&](Scores& P, int i, const half8& yh, const half8& yl) {
    mac(P.at[i & 1][0], P.at[i & 1][1], yh, yl, xh[0][i >> 1], xl[0][i >> 1], xh[1][i >> 1], xl[1][i >> 1]);
  };
  // one tile: weights of `tile` (exponent ky) from S (stage buf), product 1 of the next one (stage nb, into Sn) beside them, product 2.
  // Fragments are read one step (six matrix instructions) ahead of their use.
  auto step = [&](long long tile, int buf, int nb, int ky, Scores& S, Scores& Sn, auto has_next) {
    constexpr bool NEXT = decltype(has_next)::value;
    float z[2][8];                                               // [owner block][4 rb + r]: stream row 16 rb + 4 g + r
    bool in[2][8];
    float tmax[2] = {-INFINITY, -INFINITY};
    half8 fh[2], fo[2];                                          // the fragment pair in use and the one on its way
    if constexpr (NEXT) {
      read1(nb, 0, fh[0], fo[0]);
      clear(Sn);
    }
    const float down = pow2i(-ky), fq[2] = {fl[0] * down, fl[1] * down};
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const float4 rb4 = *(const float4*)(&rb_s[buf][16 * rb + 4 * g]);
      const float rbv[4] = {rb4.x, rb4.y, rb4.z, rb4.w};
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (!CLIP) {
            z[cb][4 * rb + r] = fmaf(S.at[rb][cb][r], fq[cb], rbv[r]);
          } else {
            const float s = fmaf(S.at[rb][cb][r], fq[cb], FWD ? rbv[r] : xb[cb]);
            const float c = s > a.clip2 ? a.clip2 : (s < -a.clip2 ? -a.clip2 : s);   // (a NaN stays one)
            in[cb][4 * rb + r] = !(s > a.clip2) && !(s < -a.clip2);
            if constexpr (FWD) z[cb][4 * rb + r] = tile * DS_TILE + 16 * rb + 4 * g + r < a.ny ? c : -INFINITY;
            else z[cb][4 * rb + r] = c + rbv[r];
          }
        }
        tmax[cb] = fmaxf(fmaxf(tmax[cb], fmaxf(z[cb][4 * rb], z[cb][4 * rb + 1])), fmaxf(z[cb][4 * rb + 2], z[cb][4 * rb + 3]));
      }
    }
    if constexpr (NEXT) {
#pragma unroll
      for (int i = 0; i < N1a; ++i) {
        read1(nb, i + 1, fh[(i + 1) & 1], fo[(i + 1) & 1]);
        product1(Sn, i, fh[i & 1], fo[i & 1]);
      }
    }
    // ---- a new reference only when a weight would pass 2^8 (or a larger tile arrives): weights reach 2^(8 + 6) = fp16's range
    if (ky + 6 < kappa || __any(fmaxf(tmax[0] - M[0], tmax[1] - M[1]) > 8.f)) {
      const int kn = min(ky + 6, kappa);
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) {
        float m2 = fmaxf(tmax[cb], __shfl_xor(tmax[cb], 16, 64));
        m2 = fmaxf(m2, __shfl_xor(m2, 32, 64));
        // (a whole number, so that what is added to M or taken off it is hardly rounded: that would be in all the weights of a row alike.  Not floorf or
        // rintf: with those D = 128 spills four registers more, 377 -> 382 us at 512 x 200 K)
        const float Mn = m2 > M[cb] + 8.f ? m2 - __builtin_amdgcn_fractf(m2) : M[cb];
        const float f = __builtin_amdgcn_exp2f(M[cb] - Mn), fk = f * exp2f((float)(kn - kappa));
        l[cb] *= f;
        if constexpr (GRAD) {
#pragma unroll
          for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) O[b][cb][r] *= fk;
        }
        M[cb] = Mn;
      }
      kappa = kn;
    }
    if constexpr (NEXT) {
#pragma unroll
      for (int i = N1a; i < N1; ++i) {
        if (i + 1 < N1) read1(nb, i + 1, fh[(i + 1) & 1], fo[(i + 1) & 1]);
        product1(Sn, i, fh[i & 1], fo[i & 1]);
      }
    }
    half8 wh[2], wl[2];
    const float unit = pow2i(ky - kappa);
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
      const float mk = M[cb] - (float)(kappa - ky);
      float w[8], sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = __builtin_amdgcn_exp2f(z[cb][j] - mk);
        if constexpr (CLIP && !FWD) w[j] = in[cb][j] ? w[j] : 0.f;
        sum += w[j];
        if constexpr (CLIP && FWD) w[j] = in[cb][j] ? w[j] : 0.f;
      }
      l[cb] = fmaf(sum, unit, l[cb]);
      if constexpr (GRAD) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          half2_t hi, lo;
          split_pair(w[j], w[j + 1], 1.f, hi, lo);
          wh[cb][j] = hi[0]; wh[cb][j + 1] = hi[1];
          wl[cb][j] = lo[0]; wl[cb][j + 1] = lo[1];
        }
      }
    }
    // ---- product 2
    if constexpr (GRAD) {
      half8 gh[2], gl[2];
      read2(buf, 0, gh[0], gl[0]);
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        if (b + 1 < DB) read2(buf, b + 1, gh[(b + 1) & 1], gl[(b + 1) & 1]);
        mac(O[b][0], O[b][1], gh[b & 1], gl[b & 1], wh[0], wl[0], wh[1], wl[1]);
      }
    }
    // the order the scheduler is asked for, from the branch on: a step's reads, then its six matrix instructions with the weights' VALU
    // work between them (0x100 LDS reads, 0x8 matrix, 0x2 VALU)
    if constexpr (NEXT) {
#pragma unroll
      for (int i = N1a; i + 1 < N1; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
        for (int j = 0; j < 6; ++j) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x2, 3, 0);
        }
      }
      if constexpr (GRAD) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int j = 0; j < 6; ++j) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 3, 0);
      }
    }
    if constexpr (GRAD) {
#pragma unroll
      for (int b = 0; b + 1 < DB; ++b) {
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, 6, 0);
      }
    }
  };
  if (t0 < t1) {
    Scores Sa, Sb;
    int k0 = 0, k1 = 0, k2 = 0, par = 0;                         // exponents of the tile in hand and of the two behind it
    auto exponent = [&](long long tile) { return FWD ? agreed(par) : a.ky_img[min(tile, t1 - 1)]; };
    if constexpr (FWD) {
      publish(0);
      __syncthreads();
      k0 = agreed(0);
      convert(0, k0);
      put_bias(0);
      request(t0 + 1, 0);                                        // (behind the last tile: its last row again, never used)
      publish(1);
      __syncthreads();
      k1 = agreed(1);
      convert(1, k1);
      put_bias(1);
      request(t0 + 2, 0);
      publish(0);
    } else {
      put_bias(0);
      k0 = exponent(t0);
      if (t0 + 1 < t1) {
        request(t0 + 1, 1);
        put_bias(1);
      }
      k1 = exponent(t0 + 1);
    }
    arrive();
    clear(Sa);
#pragma unroll
    for (int i = 0; i < N1; ++i) {
      half8 yh, yl;
      read1(0, i, yh, yl);
      product1(Sa, i, yh, yl);
    }
    int b0 = 0, b1 = 1, b2 = 2;
    auto advance = [&](long long tile, Scores& S, Scores& Sn) {
      // (stage b2's last readers passed the barrier of the tile before)
      if constexpr (FWD) {
        k2 = agreed(par);
        par ^= 1;
        convert(b2, k2);
        put_bias(b2);
        request(tile + 3, 0);
      } else {
        k2 = exponent(tile + 2);
        if (tile + 2 < t1) request(tile + 2, b2);
      }
      step(tile, b0, b1, k0, S, Sn, std::true_type());
      if constexpr (FWD) publish(par);
      else put_bias(b2);
      arrive();
      const int b = b0;
      b0 = b1; b1 = b2; b2 = b;
      k0 = k1; k1 = k2;
    };
    long long tile = t0;
    for (; tile + 2 < t1; tile += 2) {
      advance(tile, Sa, Sb);
      advance(tile + 1, Sb, Sa);
    }
    if (tile + 1 < t1) {
      advance(tile, Sa, Sb);
      step(tile + 1, b0, b1, k0, Sb, Sa, std::false_type());
    } else {
      step(tile, b0, b1, k0, Sa, Sb, std::false_type());
    }
  }
  // ---- out
#pragma unroll
  for (int cb = 0; cb < 2; ++cb) {
    const long long own = own0 + 16 * cb;
    float lt = l[cb] + __shfl_xor(l[cb], 16, 64);
    lt += __shfl_xor(lt, 32, 64);
    if (own >= a.nx) continue;
    float down;
    float* out;
    if constexpr (FWD) {
      const long long at = (long long)split * a.nx + own;
      if (g == 0) {
        a.part_m[at] = M[cb];
        a.part_l[at] = lt;
      }
      down = exp2f((float)-kappa);
      out = a.part_o + at * a.d;
    } else {
      const float gs = distill_scale(a.loss_out, a.d_loss, a.g_num), e = CLIP ? 0.f : xb[cb];
      // 2^(M + e), M + e in two pieces: its rounding would be in every term of the item's sums
      const float at = M[cb] + e, back = at - M[cb], rest = at > -1e30f ? (M[cb] - (at - back)) + (e - back) : 0.f;
      const float scale = exp2f(at) * fmaf(rest, DS_LN2, 1.f);
      if (g == 0 && a.d_bias) a.d_bias[own] = lt * scale * gs;
      down = ldexpf(scale, -kappa) * gs;
      out = a.dX + own * a.d;
    }
    if constexpr (GRAD) {
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        const int c = 16 * b + 4 * g;
        if (c < a.d)
          *(float4*)(out + c) = !FWD && own == 0 ? make_float4(0.f, 0.f, 0.f, 0.f)   // padding row: no gradient
                                                 : make_float4(O[b][cb][0] * down, O[b][cb][1] * down, O[b][cb][2] * down, O[b][cb][3] * down);
      }
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
  float inv_tau, inv_T, T, clip;
  float* lse;
  float* stat;                         // [0, B) loss of the row, [B, 2B) 1 = has a teacher, [2B, 3B) log2 of the softmax sum (+inf without a teacher)
  float* coef; int* tid;               // [B, K]: p (0 where the gradient is cut), item (0: absent; negative: a second time)
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
  __shared__ __attribute__((aligned(16))) int items_s[GRAD ? 1024 : 4];
  const int b = blockIdx.x, tid = threadIdx.x, g = tid / TPR, t = tid % TPR, d4 = a.d / 4;
  const bool on = t < d4;
  float m = -INFINITY;
  for (int s = tid; s < a.splits; s += 256) m = fmaxf(m, a.part_m[(long long)s * a.B + b]);
  m = ds_block_max(m, red);
  float l = 0.f;
  for (int s = tid; s < a.splits; s += 256) l += a.part_l[(long long)s * a.B + b] * exp2f(a.part_m[(long long)s * a.B + b] - m);
  l = ds_block_sum(l, red);
  // (log2f is 0.46 of a step low on average, and every q of the row would be as much too large: one step of Newton's, in the residual)
  const float lg = log2f(l), lse2 = m + fmaf(fmaf(l, exp2f(-lg), -1.f), DS_LOG2E, lg), lse = lse2 * DS_LN2;
  // ---- the teacher's softmax
  float tm = -INFINITY, ts = 0.f;
  for (int k = tid; k < a.K; k += 256) {
    const long long i = (long long)b * a.K + k;
    long long id = a.id[i];
    if (id < -1 || id >= a.N) id = ur_guard_id(id, a.N, a.guard);   // not an item at all: the guard goes up, the entry is absent
    const float v = teacher_at(a.score, a.score_type, i) / a.T;
    if (id >= 1 && v > -INFINITY) tm = fmaxf(tm, v);
  }
  tm = ds_block_max(tm, red);
  const bool some = tm > -INFINITY;
  for (int k = tid; k < a.K; k += 256) {
    const long long i = (long long)b * a.K + k, id = a.id[i];
    const float v = teacher_at(a.score, a.score_type, i) / a.T;
    if (id >= 1 && id < a.N && v > -INFINITY) ts += expf(v - tm);
  }
  ts = ds_block_sum(ts, red);
  const float log_ts = logf(ts), inv_ts = 1.f / ts;
  // ---- its rows
  float4 u = make_float4(0.f, 0.f, 0.f, 0.f), acc = u;
  if (on) u = ((const float4*)a.U)[(long long)b * d4 + t];
  float loss = 0.f;
  constexpr int AHEAD = 4;                                       // rows of a group under way at once
  for (int k0 = g; k0 < a.K; k0 += AHEAD * G) {
    long long id[AHEAD];
    float v[AHEAD], bias[AHEAD];
    bool there[AHEAD];
    float4 e[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int k = k0 + j * G;
      const long long i = (long long)b * a.K + min(k, a.K - 1);
      id[j] = a.id[i];
      v[j] = teacher_at(a.score, a.score_type, i) / a.T;
      there[j] = k < a.K && some && id[j] >= 1 && id[j] < a.N && v[j] > -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      e[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      bias[j] = 0.f;
      if (there[j] && on) e[j] = ((const float4*)a.E)[id[j] * d4 + t];
      if (there[j] && a.item_bias) bias[j] = a.item_bias[id[j]];
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int k = k0 + j * G;
      float p = 0.f;
      if (there[j]) {
        const float dot = group_sum<TPR>((u.x * e[j].x + u.y * e[j].y) + (u.z * e[j].z + u.w * e[j].w));
        float s = (dot + bias[j]) * a.inv_tau;
        const bool cut = a.clip > 0.f && (s > a.clip || s < -a.clip);
        if (cut) s = s > 0.f ? a.clip : -a.clip;
        const float logp = v[j] - tm - log_ts;
        p = expf(v[j] - tm) * inv_ts;                            // (not exp(logp): log_ts is rounded, once for all of the row)
        if (t == 0) loss += p * (logp - s * a.inv_T + lse);
        if (cut) p = 0.f;
        acc.x -= p * e[j].x; acc.y -= p * e[j].y; acc.z -= p * e[j].z; acc.w -= p * e[j].w;
      }
      if (GRAD && t == 0 && k < a.K) {
        a.coef[(long long)b * a.K + k] = p;
        a.tid[(long long)b * a.K + k] = there[j] ? (int)id[j] : 0;
      }
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
    // ---- an item listed again: the first of its entries takes their mass (in order)
    float* coef = a.coef + (long long)b * a.K;
    int* items = a.tid + (long long)b * a.K;
    for (int k0 = 0; k0 < a.K; k0 += 256) {
      const int k = k0 + tid, mine = k < a.K ? abs(items[k]) : 0;
      bool before = false, after = false;
      for (int c0 = 0; c0 < a.K; c0 += 1024) {
        const int n = min(1024, a.K - c0);
        __syncthreads();
        for (int i = tid; i < 1024; i += 256) items_s[i] = i < n ? abs(items[c0 + i]) : -1;
        __syncthreads();
        if (mine)
          for (int j = 0; j < n; j += 4) {
            const int4 v = *(const int4*)(items_s + j);
            const int q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              before |= q[e] == mine && c0 + j + e < k;
              after |= q[e] == mine && c0 + j + e > k;
            }
          }
      }
      if (before) items[k] = -mine;
      else if (after) {
        float p = coef[k];
        for (int j = k + 1; j < a.K; ++j)
          if (abs(items[j]) == mine) p += coef[j];
        coef[k] = p;
      }
    }
#pragma unroll 8
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

struct DistillLoss {
  const float* stat; int B, d, K; float T2; float* loss_out;
  const float* U; _Float16* img; float* rb_img; int* ky_img;
  const float* coef; const int* tid; int buckets, log2b; int* offs; uint2* list;
};
// Workgroup 0: loss_out = [T^2 / C sum of the rows' losses, C, update guard, -] (fixed order).  The others (a forward pass that will be
// followed by a backward), two for a tile of 32 users, leave what the backward needs of it.  One the image that every workgroup streams: one
// exponent, [hi | lo][32][D] halves in the swizzled order, the row biases -log2(softmax sum) (-inf without a teacher and behind the last user).
// The other its teacher's entries (item / buckets, user; p) by bucket item % buckets, a counting sort in LDS: the order inside a bucket is free.
template <int D>
__global__ __launch_bounds__(256) void distill_loss_kernel(DistillLoss a) {
  __shared__ float red[4];
  __shared__ unsigned wave_s[4];
  extern __shared__ unsigned count_s[];                          // [buckets]
  const float* stat = a.stat;
  const int B = a.B, d = a.d, tid = threadIdx.x;
  if (blockIdx.x == 0) {
    float s = 0.f, c = 0.f;
    for (int b = tid; b < B; b += 256) {
      s += stat[b];
      c += stat[B + b];
    }
    s = ds_block_sum(s, red);
    c = ds_block_sum(c, red);
    if (tid == 0) {
      a.loss_out[0] = a.T2 * s / fmaxf(c, 1.f);
      a.loss_out[1] = c;
      a.loss_out[2] = s != s ? -1.f : 1.f;   // update guard (see ur_gather_dot_loss_fwd)
      a.loss_out[3] = 0.f;
    }
    return;
  }
  const int tile = (blockIdx.x - 1) >> 1;
  if (blockIdx.x & 1) {
    constexpr int F4 = D / 4, PER = DS_TILE * F4 / 256;
    float4 v[PER];
    float mx = 0.f;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int i = threadIdx.x + 256 * p, b = tile * DS_TILE + i / F4, c = (i % F4) * 4;
      v[p] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (b < B && c < d) v[p] = *(const float4*)(a.U + (long long)b * d + c);
      mx = fmaxf(mx, fmaxf(fmaxf(finite_abs(v[p].x), finite_abs(v[p].y)), fmaxf(finite_abs(v[p].z), finite_abs(v[p].w))));
    }
    const int ky = group_exponent(ds_block_max(mx, red));
    const float up = pow2i(ky);
    _Float16* out = a.img + (long long)tile * 2 * DS_TILE * D;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int i = threadIdx.x + 256 * p, at = ds_at<D>(i / F4, (i % F4) * 4);
      half2_t h0, h1, l0, l1;
      split_pair(v[p].x, v[p].y, up, h0, l0);
      split_pair(v[p].z, v[p].w, up, h1, l1);
      *(half4*)(out + at) = (half4){h0[0], h0[1], h1[0], h1[1]};
      *(half4*)(out + DS_TILE * D + at) = (half4){l0[0], l0[1], l1[0], l1[1]};
    }
    if (tid == 0) a.ky_img[tile] = ky;
    if (tid < DS_TILE) {
      const int b = tile * DS_TILE + tid;
      a.rb_img[b] = b < B ? -stat[2 * (long long)B + b] : -INFINITY;
    }
    return;
  }
  // ---- the lists
  const int rows = min(DS_TILE, B - tile * DS_TILE);
  const unsigned n = (unsigned)rows * (unsigned)a.K;
  const long long e0 = (long long)tile * DS_TILE * a.K;
  const int* items = a.tid + e0;
  const float* coef = a.coef + e0;
  for (int i = tid; i < a.buckets; i += 256) count_s[i] = 0u;
  __syncthreads();
  constexpr int AHEAD = 8;                                       // entries of a thread under way at once
  int item[AHEAD];
  float p[AHEAD];
  auto fetch = [&](unsigned i0) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const unsigned i = i0 + tid + 256u * j;
      item[j] = i < n ? items[i] : 0;
      p[j] = i < n ? coef[i] : 0.f;
    }
  };
  const unsigned batch = 256u * AHEAD;
  for (unsigned i0 = 0; i0 < n; i0 += batch) {
    fetch(i0);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (item[j] > 0 && p[j] != 0.f) atomicAdd(&count_s[item[j] & (a.buckets - 1)], 1u);
  }
  __syncthreads();
  const int per = (a.buckets + 255) / 256, i0 = min(a.buckets, tid * per), i1 = min(a.buckets, i0 + per);
  unsigned mine = 0u;
  for (int i = i0; i < i1; ++i) mine += count_s[i];
  unsigned upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned v = (unsigned)__shfl_up((int)upto, o, 64);
    if ((tid & 63) >= o) upto += v;
  }
  if ((tid & 63) == 63) wave_s[tid >> 6] = upto;
  __syncthreads();
  unsigned at = upto - mine;
#pragma unroll
  for (int w = 0; w < 3; ++w)
    if (w < (tid >> 6)) at += wave_s[w];
  int* offs = a.offs + (long long)tile * (a.buckets + 1);
  for (int i = i0; i < i1; ++i) {
    const unsigned c = count_s[i];
    count_s[i] = at;
    offs[i] = (int)at;
    at += c;
  }
  if (tid == 255) offs[a.buckets] = (int)at;
  __syncthreads();
  uint2* list = a.list + e0;
  for (unsigned i0 = 0; i0 < n; i0 += batch) {
    if (n > batch) fetch(i0);                                    // (else they are still at hand)
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (item[j] > 0 && p[j] != 0.f)
        list[atomicAdd(&count_s[item[j] & (a.buckets - 1)], 1u)] =
            make_uint2(((unsigned)item[j] >> a.log2b) << 5 | (i0 + tid + 256u * j) / (unsigned)a.K, __float_as_uint(p[j]));
  }
}

struct DistillApply {
  const int* offs; const uint2* list; int buckets, log2b; unsigned items;   // items: of a bucket, at most
  const float *U, *d_unit;
  int B, d, K;
  const float* loss_out; const float* d_loss; float g_num;
  float *d_user, *d_table, *d_bias;
};
// A workgroup per bucket: dE[item] -= g sum p u, d_bias[item] -= g sum p over its lists of up to 16 tiles of users (512 users) at a time, put
// in the order of (item, user) by a bitonic sort in LDS.  Lists longer than the room there: one tile at a time, as many items at a time as have
// their entries in the room, 32 (32 x 32 entries at the most) at least.  TPR lanes hold a row; a group of them takes an item, all groups one that many list (a popular item).  The
// workgroups behind: d_user = g d_unit.  Latency bound: a chain of range, entries, rows, gradient.
template <int TPR>
__global__ __launch_bounds__(128) void distill_apply_kernel(DistillApply a) {
  constexpr int NT = 128, G = NT / TPR, ROOM = 1024, LONG = 32, AHEAD = 8;
  typedef unsigned long long u64;
  __shared__ u64 entry_s[ROOM];                                  // item of the bucket << 41 | user of the 512 << 32 | p
  __shared__ unsigned short run_s[ROOM + 1], long_s[ROOM];       // where an item's entries begin
  __shared__ int first_s[16], count_s[16], reach_s[32], n_s, runs_s, nlong_s;
  __shared__ __attribute__((aligned(16))) float4 acc_s[NT];
  __shared__ float accp_s[G];
  const float gs = distill_scale(a.loss_out, a.d_loss, a.g_num);
  const int d4 = a.d / 4, tid = threadIdx.x, grp = tid / TPR, t = tid % TPR;
  if ((int)blockIdx.x >= a.buckets) {
    const long long i = (long long)(blockIdx.x - a.buckets) * NT + tid;
    if (i < (long long)a.B * d4) {
      const float4 v = ((const float4*)a.d_unit)[i];
      ((float4*)a.d_user)[i] = make_float4(gs * v.x, gs * v.y, gs * v.z, gs * v.w);
    }
    return;
  }
  const int bucket = blockIdx.x, tiles = (a.B + DS_TILE - 1) / DS_TILE;
  for (int t0 = 0, m = 0; t0 < tiles; t0 += m) {
    const int some = min(16, tiles - t0);
    __syncthreads();
    if (tid < 16) {
      int f = 0, e = 0;
      if (tid < some) {
        const int* o = a.offs + (long long)(t0 + tid) * (a.buckets + 1) + bucket;
        f = o[0];
        e = o[1];
      }
      first_s[tid] = f;
      count_s[tid] = e - f;
    }
    __syncthreads();
    int total = 0;
    m = 0;
    while (m < some && (m == 0 || total + count_s[m] <= ROOM)) total += count_s[m++];   // as many tiles as fit
    if (total == 0) continue;
    const int lanes = m > 8 ? 8 : m > 4 ? 16 : m > 2 ? 32 : m > 1 ? 64 : 128, tile = tid / lanes;   // threads of a tile
    const int n_tile = tile < m ? count_s[tile] : 0;
    const uint2* list = a.list + ((long long)(t0 + tile) * DS_TILE * a.K + (tile < m ? first_s[tile] : 0));
    const bool fits = total <= ROOM;
    const unsigned items = a.items;
    auto each = [&](auto f) {                                    // of the entries, AHEAD of a thread on their way at once
      for (int i0 = tid % lanes; i0 < n_tile; i0 += AHEAD * lanes) {
        uint2 v[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) v[j] = list[min(i0 + j * lanes, n_tile - 1)];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
          if (i0 + j * lanes < n_tile) f(v[j]);
      }
    };
    for (unsigned w0 = 0, w1 = items; w0 < items; w0 = w1, w1 = items) {
      if (tid == 0) n_s = nlong_s = 0;
      if (!fits) {                                               // entries by the bits of their distance from w0: the widest 2^bits that fits
        if (tid < 32) reach_s[tid] = 0;
        __syncthreads();
        each([&](const uint2& v) {
          const unsigned o = v.x >> 5;
          if (o >= w0) atomicAdd(&reach_s[o == w0 ? 0 : 32 - __clz(o - w0)], 1);
        });
        __syncthreads();
        int bits = 0, sum = reach_s[0];
        while ((1u << bits) < items && (bits < 5 || sum + reach_s[bits + 1] <= ROOM)) sum += reach_s[++bits];
        w1 = min(items, w0 + (1u << bits));
        if (sum == 0) { __syncthreads(); continue; }
      }
      __syncthreads();
      each([&](const uint2& v) {
        const unsigned o = v.x >> 5;
        if (o >= w0 && o < w1) entry_s[atomicAdd(&n_s, 1)] = ((u64)o << 41) | ((u64)(unsigned)(tile * DS_TILE + (v.x & 31u)) << 32) | v.y;
      });
      __syncthreads();
      const int n = n_s;
      if (n == 0) { __syncthreads(); continue; }
      int size = 2;
      while (size < n) size *= 2;
      for (int i = n + tid; i < size; i += NT) entry_s[i] = ~0ull;
      __syncthreads();
      for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
          for (int i = tid; i < size / 2; i += NT) {
            const int x = ((i & ~(j - 1)) << 1) | (i & (j - 1)), y = x | j;
            const u64 vx = entry_s[x], vy = entry_s[y];
            if ((vx > vy) == ((x & k) == 0)) { entry_s[x] = vy; entry_s[y] = vx; }
          }
          __syncthreads();
        }
      if (tid < 64) {
        int runs = 0;
        for (int i0 = 0; i0 < n; i0 += 64) {
          const int i = i0 + tid;
          const bool head = i < n && (i == 0 || (entry_s[i] >> 41) != (entry_s[i - 1] >> 41));
          const u64 heads = __ballot(head);
          if (head) run_s[runs + __popcll(heads & ((1ull << tid) - 1ull))] = (unsigned short)i;
          runs += __popcll(heads);
        }
        if (tid == 0) { run_s[runs] = (unsigned short)n; runs_s = runs; }
      }
      __syncthreads();
      const int runs = runs_s;
      const float4* U = (const float4*)a.U + (long long)t0 * DS_TILE * d4 + t;
      const bool on = t < d4;
      auto sum = [&](int from, int to, int step, float4& acc, float& pb) {
#pragma unroll 4
        for (int e = from; e < to; e += step) {
          const u64 v = entry_s[e];
          const float p = __uint_as_float((unsigned)v);
          pb += p;
          if (on) {
            const float4 u = U[(long long)((unsigned)(v >> 32) & 511u) * d4];
            acc.x += p * u.x; acc.y += p * u.y; acc.z += p * u.z; acc.w += p * u.w;
          }
        }
      };
      auto put = [&](int from, const float4& acc, float pb) {
        const long long item = (long long)(entry_s[from] >> 41) << a.log2b | bucket;
        if (on) {
          float4* e = (float4*)a.d_table + item * d4 + t;
          const float4 v = *e;
          *e = make_float4(v.x - gs * acc.x, v.y - gs * acc.y, v.z - gs * acc.z, v.w - gs * acc.w);
        }
        if (t == 0 && a.d_bias) a.d_bias[item] -= gs * pb;
      };
      for (int r = grp; r < runs; r += G) {
        const int from = run_s[r], to = run_s[r + 1];
        if (to - from > LONG) {
          if (t == 0) long_s[atomicAdd(&nlong_s, 1)] = (unsigned short)r;   // (their order is free: an item is its own sum)
          continue;
        }
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float pb = 0.f;
        sum(from, to, 1, acc, pb);
        put(from, acc, pb);
      }
      __syncthreads();
      const int nl = nlong_s;
      for (int q = 0; q < nl; ++q) {
        const int from = run_s[long_s[q]], to = run_s[long_s[q] + 1];
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float pb = 0.f;
        sum(from + grp, to, G, acc, pb);
        acc_s[tid] = acc;
        if (t == 0) accp_s[grp] = pb;
        __syncthreads();
        if (grp == 0) {
          for (int w = 1; w < G; ++w) {
            const float4 v = acc_s[w * TPR + t];
            acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
            pb += accp_s[w];
          }
          put(from, acc, pb);
        }
        __syncthreads();
      }
      __syncthreads();
    }
  }
}

static inline int ds_tpr(int d) { return d <= 64 ? 16 : d <= 128 ? 32 : 64; }
// waves of a workgroup of the forward, 32 users each, the stream's tiles staged once for all of them.  Eight where they have users (512 x 60 K,
// d 64: 49.8 us with eight, 50.7 with four) and registers; else four, also where some have none: 16 x 500 K, d 128: 147 us with four, 218 with
// one, 182 with eight; 64 x 500 K: 151, 163 with two, 180 with eight; 128 x 500 K: 157 and 182; above, eight also where many have none: 130 x 500 K 189 and
// 234 with four, 260 x 500 K 340 and 492, 400 x 500 K 356 and 434 (d 64: 145 and 150, 224 and 267, 223 and 242)
static inline int ds_nw(int B, int d) { return B <= 128 || d <= 32 || d > 128 ? 4 : 8; }
static inline int ds_width(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// tiles of a split at most (8 192 items): its sums stand in fp32, where a tile that weighs less than 2^-25 of what is there already is lost.  (4 000
// users x 1 M items in 8 splits, scores 21.5 below the 20 best for all but those: d_user off by 5e-6, by 6e-7 in these 128)
constexpr int DS_RUN = 256;
static void ds_splits(int B, int d, long long N, int* owner_blocks, int* splits, long long* per) {
  const int nw = ds_nw(B, d);
  *owner_blocks = cdiv(B, 32 * nw);
  const long long tiles = (N + DS_TILE - 1) / DS_TILE;
  const long long want = std::max<long long>(1, 2048 / nw / *owner_blocks);
  long long s = std::min(want, (tiles + 1) / 2);
  s = std::max<long long>(8, (std::max(s, (tiles + DS_RUN - 1) / DS_RUN) + 7) / 8 * 8);
  *per = (tiles + s - 1) / s;
  *splits = (int)s;
}

// buckets of the lists, a power of two: some 4 to 16 entries a bucket (32 to 64: 512 x 60 K 103 us, 8 to 16 100), and no more buckets than a tile of
// users can count in LDS.  (512 users x 100, 1 M items: buckets of 128 items left 7 a workgroup, 86 us of workgroups waiting for memory; 400 x 20,
// 1 682 items: 14 workgroups of 610, 21 us.)  An item's bucket is its id modulo their number: ids next to each other, which are often alike popular, fall
// into different ones.  (With ranges of ids, 512 users x 100 entries on 200 neighbours of 1 M items, d 64, had one workgroup do it all: the
// backward 4 375 us, 508 with lists all over the catalogue; as it is 529 and 523; 120 items with one remainder, which still share a list, 3 617)
static inline int ds_log2_buckets(long long N, long long entries) {
  int s = 0, k = 0;
  while (s < 22 && ((entries << s) < 8 * N || ((N - 1) >> s) >= 8192)) ++s;
  while ((1LL << k) < ((N - 1) >> s) + 1) ++k;
  return k;
}
struct DistillWs {
  float *part_m, *part_l, *part_o, *stat, *coef; int* tid;          // the forward's own
  _Float16* img; float* rb_img; int* ky_img; int* offs; uint2* list; float* d_unit;   // from the forward to the backward
  int buckets, log2b;
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
  w.log2b = ds_log2_buckets(N, (long long)B * K);
  w.buckets = 1 << w.log2b;
  if (grad) {
    const int64_t ut = cdiv(B, DS_TILE);
    w.img = (_Float16*)take(ut * 4 * DS_TILE * ds_width(d)); w.rb_img = (float*)take(ut * DS_TILE * 4); w.ky_img = (int*)take(ut * 4);
    w.offs = (int*)take(ut * (w.buckets + 1) * 4); w.list = (uint2*)take((int64_t)B * K * 8);
    w.d_unit = (float*)take((int64_t)B * d * 4);
  }
  w.part_m = (float*)take((int64_t)splits * B * 4); w.part_l = (float*)take((int64_t)splits * B * 4);
  w.stat = (float*)take((int64_t)B * 12);
  if (grad) {
    w.part_o = (float*)take((int64_t)splits * B * d * 4);
    w.coef = (float*)take((int64_t)B * K * 4); w.tid = (int*)take((int64_t)B * K * 4);
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
  if constexpr (D == 64 || D == 128) {
    if (nw == 8) return GO(8);
  }
  return GO(4);
#undef GO
}

// waves of a workgroup of the backward, 32 items each: one where four would leave most compute units without a workgroup (1 682 items, 400
// users: step of 55.3 us with one, 57.6 with four; 20 011 items, 333 users: 65.4 and 65.9, and two waves 70.7, so no size takes two)
static inline int ds_nw_bwd(long long N) { return N <= 256 * 32 ? 1 : 4; }
template <int D>
static int ds_launch_bwd(const DistillStream& a, bool clip, hipStream_t st) {
  const int nw = ds_nw_bwd(a.nx), grid = cdiv(a.nx, 32 * nw);
  return nw == 1 ? ds_launch_stream<D, 1, false, true>(a, clip, grid, st) : ds_launch_stream<D, 4, false, true>(a, clip, grid, st);
}

// (rounded once: a scale that is off is off for every score of the batch, and what is off the same way everywhere stays in sums over the users)
static inline void ds_scales(DistillStream& a, float tau, float score_clip, float temperature) {
  constexpr double log2e = 1.4426950408889634074;
  a.cz = (float)(log2e / ((double)tau * (double)temperature));
  a.clip2 = score_clip > 0.f ? (float)((double)score_clip / (double)temperature * log2e) : 0.f;
}

static int ds_check(const float* table, int64_t N, int B, int d, int K, float tau, float T, const char* who) {
  UR_REQUIRE(table, UR_ERR_ARG, "%s: null pointer", who);
  UR_REQUIRE(B > 0 && d > 0 && d % 4 == 0 && N > 1 && N < (1LL << 31) && K > 0, UR_ERR_ARG, "%s: shape", who);
  UR_REQUIRE(d <= DS_MAX_D, UR_ERR_UNSUPPORTED, "%s: d=%d (at most %d)", who, d, DS_MAX_D);
  UR_REQUIRE((int64_t)B * K < (1LL << 31), UR_ERR_ARG, "%s: B * K = %lld", who, (long long)B * K);
  UR_REQUIRE(K <= DS_MAX_K, UR_ERR_UNSUPPORTED, "%s: K=%d entries a list (at most %d)", who, K, DS_MAX_K);
  UR_REQUIRE(tau > 0.f && T > 0.f && tau < INFINITY && T < INFINITY, UR_ERR_ARG, "%s: tau=%g and temperature=%g must be positive", who, tau, T);
  return UR_OK;
}

}  // namespace ur

using namespace ur;

extern "C" int64_t ur_full_distill_workspace_bytes(int32_t B, int32_t d, int64_t n_items, int32_t K, int32_t need_grad) {
  if (B <= 0 || d <= 0 || n_items <= 1 || K <= 0 || K > DS_MAX_K || (int64_t)B * K >= (1LL << 31)) return UR_ERR_ARG;
  return ds_carve(B, d, n_items, K, need_grad, nullptr).bytes;
}

extern "C" int ur_full_distill_fwd(const float* user_emb, const float* item_table, int64_t n_items, int32_t B, int32_t d,
                                   const int64_t* teacher_id, const void* teacher_score, int32_t score_type, int32_t K, const float* item_bias,
                                   float tau, float score_clip, float temperature, float* lse, float* loss_out, int32_t need_grad, void* ws,
                                   void* stream) {
  UR_TRACE_SCOPE();
  int rc = ds_check(item_table, n_items, B, d, K, tau, temperature, "ur_full_distill_fwd");
  if (rc) return rc;
  UR_REQUIRE(user_emb && teacher_id && teacher_score && lse && loss_out && ws, UR_ERR_ARG, "ur_full_distill_fwd: null pointer");
  UR_REQUIRE(score_type == UR_F32 || score_type == UR_F16 || score_type == UR_BF16, UR_ERR_ARG, "ur_full_distill_fwd: score_type=%d", score_type);
  const bool grad = need_grad != 0;
  hipStream_t st = as_stream(stream);
  ProfScope ps(PC_LOSS, st, (grad ? 4.0 : 2.0) * B * (double)n_items * d);
  const DistillWs w = ds_carve(B, d, n_items, K, grad, (char*)ws);
  DistillStream a{};
  a.X = user_emb; a.nx = B; a.Y = item_table; a.ny = n_items; a.d = d; a.y_bias = item_bias;
  ds_scales(a, tau, score_clip, temperature);
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
  r.inv_tau = 1.f / tau; r.inv_T = 1.f / temperature; r.T = temperature; r.clip = score_clip;
  r.lse = lse; r.stat = w.stat; r.coef = w.coef; r.tid = w.tid; r.d_unit = w.d_unit; r.guard = id_guard();
#define GO(T) do { if (grad) hipLaunchKernelGGL((distill_row_kernel<T, true>), dim3(B), dim3(256), 0, st, r); \
                   else hipLaunchKernelGGL((distill_row_kernel<T, false>), dim3(B), dim3(256), 0, st, r); } while (0)
  switch (ds_tpr(d)) {
    case 16: GO(16); break;
    case 32: GO(32); break;
    default: GO(64); break;
  }
#undef GO
  UR_LAUNCH_CHECK();
  DistillLoss l{};
  l.stat = w.stat; l.B = B; l.d = d; l.K = K; l.T2 = temperature * temperature; l.loss_out = loss_out; l.U = user_emb;
  l.img = w.img; l.rb_img = w.rb_img; l.ky_img = w.ky_img; l.coef = w.coef; l.tid = w.tid;
  l.buckets = w.buckets; l.log2b = w.log2b; l.offs = w.offs; l.list = w.list;
  const int tiles = grad ? cdiv(B, DS_TILE) : 0;
  const size_t lds = grad ? (size_t)w.buckets * 4 : 0;
#define GO(W) hipLaunchKernelGGL((distill_loss_kernel<W>), dim3(1 + 2 * tiles), dim3(256), lds, st, l)
  switch (ds_width(d)) {
    case 32: GO(32); break;
    case 64: GO(64); break;
    case 128: GO(128); break;
    default: GO(256); break;
  }
#undef GO
  UR_LAUNCH_CHECK();
  return UR_OK;
}

extern "C" int ur_full_distill_bwd(const float* user_emb, const float* item_table, int64_t n_items, int32_t B, int32_t d, int32_t K, const float* item_bias, float tau,
                                   float score_clip, float temperature, const float* loss_out, const float* d_loss, float* d_user_emb,
                                   float* d_item_table, float* d_item_bias, const void* ws, void* stream) {
  UR_TRACE_SCOPE();
  int rc = ds_check(item_table, n_items, B, d, K, tau, temperature, "ur_full_distill_bwd");
  if (rc) return rc;
  UR_REQUIRE(user_emb && loss_out && d_user_emb && d_item_table && ws, UR_ERR_ARG, "ur_full_distill_bwd: null pointer");
  UR_REQUIRE(!item_bias || d_item_bias, UR_ERR_ARG, "ur_full_distill_bwd: d_item_bias is required when item_bias is given");
  hipStream_t st = as_stream(stream);
  const DistillWs w = ds_carve(B, d, n_items, K, 1, (char*)ws);
  ProfScope ps(PC_LOSS, st, 4.0 * B * (double)n_items * d);
  DistillStream a{};
  a.X = item_table; a.nx = n_items; a.ny = B; a.d = d; a.img = w.img; a.rb_img = w.rb_img; a.ky_img = w.ky_img; a.x_bias = item_bias;
  ds_scales(a, tau, score_clip, temperature);
  a.loss_out = loss_out; a.d_loss = d_loss; a.g_num = temperature / tau; a.dX = d_item_table; a.d_bias = d_item_bias;
  const bool clip = score_clip > 0.f;
  rc = d <= 32 ? ds_launch_bwd<32>(a, clip, st) : d <= 64 ? ds_launch_bwd<64>(a, clip, st)
     : d <= 128 ? ds_launch_bwd<128>(a, clip, st) : ds_launch_bwd<256>(a, clip, st);
  if (rc) return rc;
  DistillApply p{};
  p.offs = w.offs; p.list = w.list; p.buckets = w.buckets; p.log2b = w.log2b; p.items = (unsigned)((n_items - 1) >> w.log2b) + 1u; p.U = user_emb; p.d_unit = w.d_unit;
  p.B = B; p.d = d; p.K = K; p.loss_out = loss_out; p.d_loss = d_loss; p.g_num = temperature / tau;
  p.d_user = d_user_emb; p.d_table = d_item_table; p.d_bias = d_item_bias;
  const int blocks = w.buckets + cdiv((long long)B * (d / 4), 128);
  switch (ds_tpr(d)) {
    case 16: hipLaunchKernelGGL((distill_apply_kernel<16>), dim3(blocks), dim3(128), 0, st, p); break;
    case 32: hipLaunchKernelGGL((distill_apply_kernel<32>), dim3(blocks), dim3(128), 0, st, p); break;
    default: hipLaunchKernelGGL((distill_apply_kernel<64>), dim3(blocks), dim3(128), 0, st, p); break;
  }
  UR_LAUNCH_CHECK();
  return UR_OK;
}
