// Attention over the rows of scenes, backward.  Two kernels and no atomics: one owns queries (dQ, the rows' sum(dO O), the slopes'
// gradient), one owns keys (dK, dV, summed over the heads that share them); both form the scores again from the operands and the kept
// softmax statistics.  With P and D = sum(dO O):
//   dV = P^T dO      dL = P (dO V^T - D)      dslope = -sum dL |xy - kv_xy|      dS = dL (1 - tanh^2)      dQ = scale dS K      dK = scale dS^T Q
// P and dS are rounded to the operands' type where they enter a product, as every operand is (Coef in blk_attn.h); what is summed without a
// product -- sum(dO O), the slopes' gradient -- takes them in f32.
#include <limits.h>
#include "blk_attn.h"
#include "../../include/mggan_hip.h"

int blk_attn_check(const BlkAttnArgs* a, const char* name);

namespace {

// Tiles of 32 rows: the scores' gradients need registers next to the scores.  (bf16 of width 32 and 96: 64, whole passes of 256 copies.)
template <class T, int DP>
using BwdGeo = Geo<T, DP, sizeof(T) == 2 && DP % 64 ? 64 : 32>;

// dQ of 64 QF rows of one head (this wave's start at w0), and the sum that the rows' slopes' gradient is.  Three products a tile: keys are read
// twice (rows, then transposed), values once.  Bound by the waves' instructions around the products (width 128 with a distance: vector instructions
// 62 % of the time, matrix cores 36 %; width 64 with a cap: 82 and 17 %): 16,384 causal rows of 8 heads at width 128, 1.14 ms; packed 8,192 rows of
// 16 heads at width 64, 107 us.
template <class T, int DP, int QF, int X, bool SAFE>
__device__ __forceinline__ float attn_dq_rows(const BlkAttnArgs& p, int np, float* delta, int h, int glo, int ghi, int w0, u32x4* lk, u32x4* lv,
                                              float* lx, int* odd) {
  using G = BwdGeo<T, DP>;
  using W = Soft<T, X>;
  constexpr int AXES = W::AXES;
  const int lane = mg_lane(), wave = mg_wave(), i16 = lane & 15, g = lane >> 4, hk = h / (p.H / p.Hkv), nd = p.D / G::CH;
  int lo[QF], hi[QF], wlo = INT_MAX, whi = 0, flo = 0, fhi = INT_MAX;
  float qx[QF], qy[QF], top[QF], inv[QF], dsum[QF];
  u32x4 q[QF][G::SK], dO[QF][G::SK];
#pragma unroll
  for (int j = 0; j < QF; ++j) {
    const int r = w0 + 16 * j + i16, rc = min(r, p.N - 1);
    lo[j] = p.spans[r];
    hi[j] = p.spans[np + r];
    if (hi[j] > lo[j]) wlo = min(wlo, lo[j]), whi = max(whi, hi[j]);
    flo = max(flo, hi[j] > lo[j] ? lo[j] : INT_MAX);
    fhi = min(fhi, hi[j]);
    const T* row = (const T*)p.q + rc * p.q_row + h * p.q_head;
    const long at = ((long)rc * p.H + h) * p.D;
    float d = 0.f;
#pragma unroll
    for (int s = 0; s < G::SK; ++s) {
      q[j][s] = owner_chunk(row, 4 * s + g, nd);
      dO[j][s] = owner_chunk((const T*)p.dout + at, 4 * s + g, nd);
      const float* o = p.out32 + at + (4 * s + g) * G::CH;
      if (4 * s + g < nd) {
#pragma unroll
        for (int e = 0; e < G::CH; ++e) {
          if constexpr (sizeof(T) == 2)
            d = fmaf(o[e], (float)__builtin_bit_cast(bf16x8, dO[j][s])[e], d);
          else
            d = fmaf(o[e], __builtin_bit_cast(f32x4, dO[j][s])[e], d);
        }
      }
    }
    dsum[j] = quarters_sum(d);
    top[j] = p.lse[((W::NATURAL ? 0 : 2L * p.H) + h) * p.N + rc];
    inv[j] = W::NATURAL ? p.lse[(long)(p.H + h) * p.N + rc] : 1.f;
    if (r < p.N && g == 0) delta[(long)h * p.N + r] = dsum[j];
    qx[j] = AXES ? p.xy[(long)rc * AXES] : 0.f;
    qy[j] = AXES > 1 ? p.xy[(long)rc * AXES + 1] : 0.f;
  }
  wave_span(wlo, whi, flo, fhi);

  const T* kb = (const T*)p.k + hk * p.k_head;
  const T* vb = (const T*)p.v + hk * p.v_head;
  auto fetch = [&](int k0, int buf) {
    copy_tile<G>(kb, p.k_row, k0, glo, ghi, nd, lk + buf * G::TILE);
    copy_tile<G>(vb, p.v_row, k0, glo, ghi, nd, lv + buf * G::TILE);
    if (wave < AXES) copy_meta(p.kv_xy, AXES, wave, k0, p.M, lx + (2 * buf + wave) * 64);
  };

  f32x4 acc[QF][G::DF];
#pragma unroll
  for (int j = 0; j < QF; ++j)
#pragma unroll
    for (int d = 0; d < G::DF; ++d) acc[j][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  // the slopes' gradient is f32 and a sum over all pairs, so it takes the rows' sum(P dO V^T) from the same P: -sum (P dP dist) + sum(P dP)
  // sum(P dist) row by row, with nothing in it that was rounded to the operands' type
  float sa[QF] = {}, sb[QF] = {}, sc[QF] = {};
  const W soft(p, AXES ? p.slopes[h] : 0.f);
  Lane<G> at;
  at.init(lane);

  if (glo < ghi) fetch(glo, 0);
  int buf = 0;
  for (int k0 = glo; k0 < ghi; k0 += G::BK, buf ^= 1) {
    copies_done();
    if (k0 + G::BK < ghi) fetch(k0 + G::BK, buf ^ 1);
    if (k0 >= whi || k0 + G::BK <= wlo) continue;
    const u32x4 *tk = lk + buf * G::TILE, *tv = lv + buf * G::TILE;
    const bool part = k0 < flo || k0 + G::BK > fhi;
    if (!SAFE && part && tile_not_finite<G>(tk, lane)) *odd = 1;
    float ta[QF] = {}, tb[QF] = {}, tc[QF] = {};
    f32x4 s[QF][G::F], dp[QF][G::F];
    Coef<T> ds[QF][G::F];
    scores<G, QF>(tk, q, s, at);
    scores<G, QF>(tv, dO, dp, at);
#pragma unroll
    for (int f = 0; f < G::F; ++f) {
      const int kr = G::row4(f, g);
      f32x4 bx = {}, by = {};
      if (AXES) bx = *(const f32x4*)(lx + 2 * buf * 64 + kr);
      if (AXES > 1) by = *(const f32x4*)(lx + (2 * buf + 1) * 64 + kr);
#pragma unroll
      for (int j = 0; j < QF; ++j) {
        f32x4 dl;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = s[j][f][r], fac = 1.f, dist = 0.f;
          if (!W::RAW) x = soft.score(x, qx[j], qy[j], bx[r], by[r], fac, dist);
          float w = soft.weight(x, top[j]);
          if (W::NATURAL) w *= inv[j];
          float wd = w * dp[j][f][r];
          dl[r] = fmaf(-w, dsum[j], wd);
          if (W::CAP) dl[r] *= fac;
          if (part) {
            const int key = k0 + kr + r;
            const bool seen = key >= lo[j] && key < hi[j];
            dl[r] = seen ? dl[r] : 0.f;
            if (AXES) {
              w = seen ? w : 0.f;
              wd = seen ? wd : 0.f;
              dist = seen ? dist : 0.f;
            }
          }
          if (AXES) {
            ta[j] = fmaf(wd, dist, ta[j]);
            tb[j] = fmaf(w, dist, tb[j]);
            tc[j] += wd;
          }
        }
        ds[j][f].set(dl);
      }
    }
    if (AXES) {
#pragma unroll
      for (int j = 0; j < QF; ++j) sa[j] += ta[j], sb[j] += tb[j], sc[j] += tc[j];
    }
    if (SAFE && part && tile_not_finite<G>(tk, lane))
      accumulate_seen<G, QF>(tk, ds, acc, at, lane, [&](int j, int row) { return k0 + row >= lo[j] && k0 + row < hi[j]; });
    else
      accumulate<G, QF>(tk, ds, acc, at);
  }
  if (!SAFE) {
    __syncthreads();
    if (*odd) return 0.f;
  }

#pragma unroll
  for (int j = 0; j < QF; ++j) {
    const int r = w0 + 16 * j + i16;
    if (r >= p.N) continue;
    T* out = (T*)p.dq + ((long)r * p.H + h) * p.D;
#pragma unroll
    for (int d = 0; d < G::DF; ++d)
      if (16 * d + 4 * g < p.D) store4<T>(out + 16 * d + 4 * g, acc[j][d], p.scale);
  }
  float slope_sum = 0.f;
#pragma unroll
  for (int j = 0; j < QF; ++j) {
    const float a = quarters_sum(sa[j]), b = quarters_sum(sb[j]), c = quarters_sum(sc[j]);
    if (g == 0 && w0 + 16 * j + i16 < p.N) slope_sum += fmaf(-c, b, a);
  }
  return slope_sum;
}

template <class T, int DP, int QF, int X>
__global__ __launch_bounds__(256, QF == 1 && DP <= 64 ? 3 : 2) void blk_attn_dq_kernel(BlkAttnArgs p, int np, float* delta, float* slope_part, int2* ranges) {
  using G = BwdGeo<T, DP>;
  __shared__ struct {
    u32x4 k[2 * G::TILE], v[2 * G::TILE];
    float x[2 * 2 * 64];
    int odd, order[RANK_MAX + 1], range[2];
  } lds;
  // for the keys' side: the rows that see any of 64 keys lie between the first and the last 32 that do
  for (int kt = blockIdx.x; kt < (p.M + 63) / 64; kt += gridDim.x) {
    if (threadIdx.x == 0) lds.range[0] = INT_MAX, lds.range[1] = -1;
    __syncthreads();
    for (int u = threadIdx.x; u < np / 32; u += 256) {
      const int4 s = *(const int4*)(p.spans + 2 * np + 4 * u);
      if (s.x < kt * 64 + 64 && s.y > kt * 64) {
        atomicMin(&lds.range[0], u);
        atomicMax(&lds.range[1], u);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) ranges[kt] = make_int2(lds.range[0], lds.range[1]);
  }
  const int wave = mg_wave(), h = blockIdx.x % p.H, nqt = gridDim.x / p.H;
  const int qt = by_work(blockIdx.x / p.H, nqt, [&](int i) {
    const int2 k = group_span<2 * QF>(p, np, i * 64 * QF);
    return k.y - k.x;
  }, lds.order);
  const int r0 = qt * 64 * QF, w0 = r0 + wave * 16 * QF;
  if (threadIdx.x == 0) lds.odd = 0;
  __syncthreads();
  const int2 keys = group_span<2 * QF>(p, np, r0);
  float sum = attn_dq_rows<T, DP, QF, X, false>(p, np, delta, h, keys.x, keys.y, w0, lds.k, lds.v, lds.x, &lds.odd);
  if (lds.odd) {
    sum = 0.f;
    for (int j = 0; j < QF; ++j) {
      __syncthreads();
      sum += attn_dq_rows<T, DP, 1, X, true>(p, np, delta, h, keys.x, keys.y, afresh(w0 + 16 * j), lds.k, lds.v, lds.x, &lds.odd);
    }
  }
  if (Soft<T, X>::AXES && p.dslopes) {
    __syncthreads();
    sum = wave_sum(sum);
    if (mg_lane() == 0) lds.x[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) slope_part[(long)h * nqt + qt] = (lds.x[0] + lds.x[1]) + (lds.x[2] + lds.x[3]);
  }
}

// dK and dV of 64 keys of one key head (this wave's 16 start at w0) from the queries [qa, qb) of `heads` heads from h0 on, in tiles of BK
// rows; `part`: of some of the key head's heads, left in f32 for blk_attn_sum_kernel as the slot-th of `slots` such results.  Four products a tile, both streamed operands read twice.  Bound by LDS at width 128:
// 16 keys a wave take a kilobyte of reads for every multiplication, and LDS is busy 75 % of the time, 45 % of that with bank conflicts (1.58 ms at 16,384
// causal rows).  At width 64 with a cap vector instructions fill 57 % and LDS 38 % (packed 8,192 rows: 170 us).  32 keys a wave would halve the reads, but two results, keys and values of 32 rows leave too few registers (1.8 to 9
// ms, spilled or with two waves a SIMD).
template <class T, int DP, int X, bool SAFE>
__device__ __forceinline__ void attn_dkv_rows(const BlkAttnArgs& p, int np, const float* delta, float* part, int slot, int slots, int h0, int heads, int qa, int qb, int w0,
                                              u32x4* lq, u32x4* lo_, float* lm, int* odd) {
  using G = BwdGeo<T, DP>;
  using W = Soft<T, X>;
  constexpr int AXES = W::AXES;
  constexpr bool ONE = sizeof(T) == 2;  // one statistic a row
  const int lane = mg_lane(), wave = mg_wave(), i16 = lane & 15, g = lane >> 4, hk = h0 / (p.H / p.Hkv), nd = p.D / G::CH;
  u32x4 k[G::SK], v[G::SK];
  f32x4 dk[1][G::DF], dv[1][G::DF];
  const int rc = min(w0 + i16, p.M - 1);
  const T* kr = (const T*)p.k + rc * p.k_row + hk * p.k_head;
  const T* vr = (const T*)p.v + rc * p.v_row + hk * p.v_head;
#pragma unroll
  for (int s = 0; s < G::SK; ++s) {
    k[s] = owner_chunk(kr, 4 * s + g, nd);
    v[s] = owner_chunk(vr, 4 * s + g, nd);
  }
  const float kx = AXES ? p.kv_xy[(long)rc * AXES] : 0.f, ky = AXES > 1 ? p.kv_xy[(long)rc * AXES + 1] : 0.f;
#pragma unroll
  for (int d = 0; d < G::DF; ++d) dk[0][d] = dv[0][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  Lane<G> at;
  at.init(lane);

  auto meta = [&](int buf, int i) { return lm + (8 * buf + i) * 64; };
  // (head, tile) pairs in one sequence, so that the copies of the next head's first tile are under way too
  const int nt = qb > qa ? (qb - qa + G::BK - 1) / G::BK : 0, total = nt * heads;
  auto fetch = [&](int t, int buf) {
    const int h = h0 + t / nt, q0 = qa + t % nt * G::BK;
    copy_tile<G>((const T*)p.q + h * p.q_head, p.q_row, q0, 0, p.N, nd, lq + buf * G::TILE);
    copy_tile<G>((const T*)p.dout + (long)h * p.D, (long)p.H * p.D, q0, 0, p.N, nd, lo_ + buf * G::TILE);
    if (wave == 0) copy_meta(p.lse + ((ONE ? 2L * p.H : 0) + h) * p.N, 1, 0, q0, p.N, meta(buf, 0));
    if (wave == 3 && !ONE) copy_meta(p.lse + (long)(p.H + h) * p.N, 1, 0, q0, p.N, meta(buf, 6));
    if (wave == 1) copy_meta(delta + (long)h * p.N, 1, 0, q0, p.N, meta(buf, 1));
    if (wave == 2) copy_meta(p.spans, 1, 0, q0, np, meta(buf, 2));
    if (wave == 3) copy_meta(p.spans + np, 1, 0, q0, np, meta(buf, 3));
    if (wave == 2) copy_meta(p.spans + 2 * np, 1, 0, q0 >> 3, np >> 3, meta(buf, 7));
    if (wave < AXES) copy_meta(p.xy, AXES, wave, q0, p.N, meta(buf, 4 + wave));
  };
  if (total > 0) fetch(0, 0);
  float slope = 0.f;
  for (int t = 0; t < total; ++t) {
    const int buf = t & 1, q0 = qa + t % nt * G::BK, h = h0 + t / nt;
    copies_done();
    if (AXES && t % nt == 0) slope = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(p.slopes[h])));
    if (t + 1 < total) fetch(t + 1, buf ^ 1);
    int slo = INT_MAX, shi = 0, flo = 0, fhi = INT_MAX;
#pragma unroll
    for (int i = 0; i < G::BK / 32; ++i) {
      const int4 u = *(const int4*)(meta(buf, 7) + 4 * i);  // (a load from memory would be waited for behind the copies)
      slo = min(slo, u.x), shi = max(shi, u.y), flo = max(flo, u.z), fhi = min(fhi, u.w);
    }
    slo = __builtin_amdgcn_readfirstlane(slo), shi = __builtin_amdgcn_readfirstlane(shi);
    if (slo >= w0 + 16 || shi <= w0) continue;
    const bool cut = __builtin_amdgcn_readfirstlane(w0 < flo || w0 + 16 > fhi);
    const W soft(p, slope);
    const u32x4 *tq = lq + buf * G::TILE, *to = lo_ + buf * G::TILE;
    const int key = w0 + i16;
    Coef<T> w[1][G::F], ds[1][G::F];
#pragma unroll
    for (int f = 0; f < G::F; ++f) {
      f32x4 x, dp;
      scores2<G>(tq, to, k, v, f, x, dp, at);
      const int qr = G::row4(f, g);
      const f32x4 top = *(const f32x4*)(meta(buf, 0) + qr), dsum = *(const f32x4*)(meta(buf, 1) + qr);
      f32x4 inv = {}, ax = {}, ay = {};
      if (!ONE) inv = *(const f32x4*)(meta(buf, 6) + qr);
      if (AXES) ax = *(const f32x4*)(meta(buf, 4) + qr);
      if (AXES > 1) ay = *(const f32x4*)(meta(buf, 5) + qr);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float z = x[r], fac = 1.f, dist;
        if (!W::RAW) z = soft.score(z, ax[r], ay[r], kx, ky, fac, dist);
        float p_ = soft.weight(z, top[r]);
        if (!ONE) p_ *= inv[r];
        float dl = p_ * (dp[r] - dsum[r]);
        if (W::CAP) dl *= fac;
        x[r] = p_;
        dp[r] = dl;
      }
      if (cut) {
        const f32x4 from = *(const f32x4*)(meta(buf, 2) + qr), to_ = *(const f32x4*)(meta(buf, 3) + qr);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool seen = key >= __float_as_int(from[r]) && key < __float_as_int(to_[r]);
          x[r] = seen ? x[r] : 0.f;
          dp[r] = seen ? dp[r] : 0.f;
        }
      }
      w[0][f].set(x);
      ds[0][f].set(dp);
      __builtin_amdgcn_sched_barrier(0);
    }
    auto sees = [&](int, int row) { return key >= __float_as_int(meta(buf, 2)[row]) && key < __float_as_int(meta(buf, 3)[row]); };
    const bool bad = cut && (tile_not_finite<G>(to, lane) || tile_not_finite<G>(tq, lane));
    if (!SAFE && bad) *odd = 1;
    if (SAFE && bad) {
      accumulate_seen<G, 1>(to, w, dv, at, lane, sees);
      accumulate_seen<G, 1>(tq, ds, dk, at, lane, sees);
    } else {
      accumulate<G, 1>(to, w, dv, at);
      accumulate<G, 1>(tq, ds, dk, at);
    }
  }
  if (!SAFE) {
    __syncthreads();
    if (*odd) return;
  }
  const int r = w0 + i16;
  if (r >= p.M) return;
  const long o = ((long)r * p.Hkv + hk) * p.D, po = ((long)slot * p.M + r) * p.D;
#pragma unroll
  for (int d = 0; d < G::DF; ++d)
    if (16 * d + 4 * g < p.D) {
      if (part) {
        store4<float>(part + po + 16 * d + 4 * g, dk[0][d], p.scale);
        store4<float>(part + (long)slots * p.M * p.D + po + 16 * d + 4 * g, dv[0][d], 1.f);
      } else {
        store4<T>((T*)p.dk + o + 16 * d + 4 * g, dk[0][d], p.scale);
        store4<T>((T*)p.dv + o + 16 * d + 4 * g, dv[0][d], 1.f);
      }
    }
}

template <class T, int DP, int X>
__global__ __launch_bounds__(256, DP <= 64 || (sizeof(T) == 2 && DP == 128) ? 3 : 2) void blk_attn_dkv_kernel(BlkAttnArgs p, int np, const float* delta,
                                                                                                                         float* part, int parts, int per, const float* slope_part,
                                                                                                                         int nqt, const int2* ranges) {
  using G = BwdGeo<T, DP>;
  __shared__ struct {
    u32x4 q[2 * G::TILE], o[2 * G::TILE];
    float m[2 * 8 * 64];  // of each streamed row: top, sum(dO O), lo, hi, x, y, 1 / sum; then what 32 rows see
    int odd, order[RANK_MAX + 1];
  } lds;
  const int group = p.H / p.Hkv, nh = p.Hkv * parts, slot = blockIdx.x % nh, sub = slot % parts;
  const int h0 = slot / parts * group + sub * per, heads = min(per, group - sub * per);
  const int kt = by_work(blockIdx.x / nh, gridDim.x / nh, [&](int i) { return ranges[i].y - ranges[i].x; }, lds.order);
  const int w0 = kt * 64 + mg_wave() * 16;

  // the slopes' gradient: a head's partial sums of the dQ kernel, in a fixed order, by the first wave of each of the first workgroups
  if (Soft<T, X>::AXES && p.dslopes && threadIdx.x < 64) {
    for (int h = blockIdx.x; h < p.H; h += gridDim.x) {
      double s = 0.;
      for (int i = threadIdx.x; i < nqt; i += 64) s += (double)slope_part[(long)h * nqt + i];
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
      if (threadIdx.x == 0) p.dslopes[h] = (float)-s;
    }
  }
  if (threadIdx.x == 0) lds.odd = 0;
  __syncthreads();
  const int first = ranges[kt].x, last = ranges[kt].y, qa = last < 0 ? 0 : first * 32 / G::BK * G::BK, qb = (last + 1) * 32;
  attn_dkv_rows<T, DP, X, false>(p, np, delta, part, slot, nh, h0, heads, qa, qb, w0, lds.q, lds.o, lds.m, &lds.odd);
  if (!lds.odd) return;
  __syncthreads();
  attn_dkv_rows<T, DP, X, true>(p, np, delta, part, slot, nh, h0, heads, qa, qb, afresh(w0), lds.q, lds.o, lds.m, &lds.odd);
}

// dK and dV (blockIdx.y) of a key head: the sum of its `parts` partial results, in their order; four columns a thread.  Bound by bytes (12 us for the
// packed 8,192 rows at width 64).
template <class T>
__global__ __launch_bounds__(256) void blk_attn_sum_kernel(BlkAttnArgs p, const float* part, int parts) {
  const long per = (long)p.M * p.D, id = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (id >= per * p.Hkv) return;
  const long hk = id / per, at = id - hk * per, r = at / p.D, d = at - r * p.D;
  const float* in = part + (blockIdx.y * (long)p.Hkv + hk) * parts * per + at;
  f32x4 s = {};
  for (int g = 0; g < parts; ++g) s += *(const f32x4*)(in + g * per);
  store4<T>((T*)(blockIdx.y ? p.dv : p.dk) + (r * p.Hkv + hk) * p.D + d, s, 1.f);
}

// The workspace: sum(dO O), the slopes' partial sums, the rows that see each 64 keys, and -- where the heads of a key head are taken apart -- dK and dV
// of each `per` of them, `parts` a key head.
// They are where a key head's keys alone are too few workgroups: the first keys behind a causal mask are seen by all rows of all those
// heads, and one workgroup's walk over them would be the whole time (backward pass, together / apart, causal: 256 workgroups 1.16 / 0.51 ms,
// 1,024: 5.21 / 4.34; 2,048: 5.76 / 5.73, not worth the memory).  One head each while their f32 results stay within PART_BYTES, else as many
// together as it takes: below 2,048 workgroups a key head's dK and dV are 134 MB at most, so eight parts always fit, and the memory does not grow
// with the heads.
constexpr size_t PART_BYTES = (size_t)1 << 30;
struct Parts {
  size_t slopes, ranges, heads, bytes;
  int parts, per;
};
Parts parts_of(int N, int M, int H, int Hkv, int D) {
  Parts w;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  w.slopes = up((size_t)H * N * 4);
  w.ranges = w.slopes + up((size_t)H * cdiv(N, 64) * 4);
  w.heads = w.ranges + up((size_t)cdiv(M, 64) * 8);
  const int group = H / Hkv;
  const size_t one = (size_t)2 * Hkv * M * D * 4;  // dK and dV of one part of each key head
  w.per = group;
  if (group > 1 && (long)cdiv(M, 64) * Hkv < 2048) w.per = cdiv(group, (long)(PART_BYTES / one));
  w.parts = cdiv(group, w.per);
  w.bytes = w.heads + (w.parts > 1 ? w.parts * one : 0);
  return w;
}

template <class T, int DP, int QF, int X>
void launch_bwd_tile(const BlkAttnArgs& p, hipStream_t st) {
  const int np = cdiv(p.N, 128) * 128, nqt = cdiv(p.N, 64 * QF);
  const Parts w = parts_of(p.N, p.M, p.H, p.Hkv, p.D);
  float* delta = (float*)p.ws;
  float* slopes = (float*)((char*)p.ws + w.slopes);
  int2* ranges = (int2*)((char*)p.ws + w.ranges);
  float* heads = w.bytes > w.heads ? (float*)((char*)p.ws + w.heads) : nullptr;
  MG_LAUNCH((blk_attn_dq_kernel<T, DP, QF, X>), dim3(nqt * p.H), dim3(256), 0, st, p, np, delta, slopes, ranges);
  MG_LAUNCH((blk_attn_dkv_kernel<T, DP, X>), dim3(cdiv(p.M, 64) * p.Hkv * w.parts), dim3(256), 0, st, p, np, (const float*)delta, heads, w.parts, w.per,
            (const float*)slopes, nqt, (const int2*)ranges);
  if (heads) MG_LAUNCH((blk_attn_sum_kernel<T>), dim3(cdiv((long)p.M * p.Hkv * p.D, 1024), 2), dim3(256), 0, st, p, (const float*)heads, w.parts);
}
template <class T, int DP, int X>
void launch_bwd_x(const BlkAttnArgs& p, hipStream_t st) {
  // rows a workgroup: as in the forward pass (width 128, 16,384 rows: dQ 1.08 against 1.23 ms; width 64: 142 against 125 us).  On the keys'
  // side, with two results, 16 keys a wave and three waves a SIMD are better at every width (width 128: 1.71 ms against 1.91 with two).
  constexpr int QF = sizeof(T) == 2 && DP > 64 ? 2 : 1;
  if (QF > 1 && (long)cdiv(p.N, 128) * p.H >= 256)
    launch_bwd_tile<T, DP, QF, X>(p, st);
  else
    launch_bwd_tile<T, DP, 1, X>(p, st);
}
template <class T, int DP>
void launch_bwd(const BlkAttnArgs& p, hipStream_t st) {
  const int x = blk_attn_x<T>(p);
  if constexpr (sizeof(T) == 2) {
    switch (x) {
      case 9: return launch_bwd_x<T, DP, 9>(p, st);
      case 11: return launch_bwd_x<T, DP, 11>(p, st);
      case 13: return launch_bwd_x<T, DP, 13>(p, st);
    }
  }
  switch (x) {
    case 0: return launch_bwd_x<T, DP, 0>(p, st);
    case 1: return launch_bwd_x<T, DP, 1>(p, st);
    case 2: return launch_bwd_x<T, DP, 2>(p, st);
    case 3: return launch_bwd_x<T, DP, 3>(p, st);
    case 4: return launch_bwd_x<T, DP, 4>(p, st);
    default: return launch_bwd_x<T, DP, 5>(p, st);
  }
}
template <class T>
void launch_bwd_width(const BlkAttnArgs& p, hipStream_t st) {
  if (p.D <= 32)
    launch_bwd<T, 32>(p, st);
  else if (p.D <= 64)
    launch_bwd<T, 64>(p, st);
  else if (p.D <= 96)
    launch_bwd<T, 96>(p, st);
  else
    launch_bwd<T, 128>(p, st);
}

}  // namespace

extern "C" {

size_t mggan_block_attention_bwd_workspace(int rows, int keys, int heads, int kv_heads, int width) {
  return rows > 0 && keys > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && width > 0 && width <= 128 ? parts_of(rows, keys, heads, kv_heads, width).bytes : 0;
}

int mggan_block_attention_bwd(const void* args, hipStream_t stream) {
  const BlkAttnArgs* a = (const BlkAttnArgs*)args;
  const int rc = blk_attn_check(a, "block_attention_bwd");
  if (rc != MGGAN_OK) return rc;
  MG_CHECK_ARG(a->out32 && a->lse && a->dout && a->dq && a->dk && a->dv, "block_attention_bwd: null operand");
  MG_CHECK_ARG((long)cdiv(a->M, 64) * a->H <= 1 << 23, "block_attention_bwd: %d keys of %d heads are too many workgroups", a->M, a->H);
  MG_CHECK_ARG(((size_t)a->out32 | (size_t)a->dout | (size_t)a->dq | (size_t)a->dk | (size_t)a->dv | (size_t)a->spans) % 16 == 0,
               "block_attention_bwd: operands have to be 16-byte aligned");
  const size_t need = parts_of(a->N, a->M, a->H, a->Hkv, a->D).bytes;
  MG_CHECK_ARG(a->ws && (size_t)a->ws_bytes >= need && (size_t)a->ws % 256 == 0, "block_attention_bwd: workspace of %zu bytes, 256-byte aligned (got %ld)", need,
               a->ws_bytes);
  if (a->dtype == BLK_BF16)
    launch_bwd_width<bf16>(*a, stream);
  else
    launch_bwd_width<float>(*a, stream);
  MG_LAUNCH_CHECK("block_attention_bwd");
  return MGGAN_OK;
}
}
