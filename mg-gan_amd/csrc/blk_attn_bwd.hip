// Attention over the rows of scenes, backward.  Two kernels and no atomics: one owns queries (dQ, the rows' sum(dO O), the slopes'
// gradient), one owns keys (dK, dV, summed over the heads that share them); both form the scores again from the operands and the kept
// softmax statistics.  With P and D = sum(dO O):
//   dV = P^T dO      dL = P (dO V^T - D)      dslope = -sum dL |xy - kv_xy|      dS = dL (1 - tanh^2)      dQ = scale dS K      dK = scale dS^T Q
// P and dS are rounded to the operands' type where they enter a product, as every operand is.
#include <limits.h>
#include "blk_attn.h"
#include "../../include/mggan_hip.h"

int blk_attn_check(const BlkAttnArgs* a, const char* name);

namespace {

template <class T, int DP, int QF, int X>
__global__ __launch_bounds__(256, 2) void blk_attn_dq_kernel(BlkAttnArgs p, int np, float* delta, float* slope_part) {
  using G = Geo<T, DP>;
  using W = Soft<T, X>;
  constexpr int AXES = W::AXES;
  __shared__ u32x4 lk[2][G::TILE], lv[2][G::TILE];
  __shared__ __attribute__((aligned(16))) float lx[2][2][64];
  const int lane = mg_lane(), wave = mg_wave(), i16 = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % p.H, hk = h / (p.H / p.Hkv);
  const int nqt = gridDim.x / p.H, qt = nqt - 1 - (int)(blockIdx.x / p.H);
  const int r0 = qt * 64 * QF, w0 = r0 + wave * 16 * QF;
  const int nd = p.D / G::CH;

  int glo = INT_MAX, ghi = 0;
#pragma unroll
  for (int i = 0; i < 2 * QF; ++i) {
    const int4 s = *(const int4*)(p.spans + 2 * np + 4 * ((r0 >> 5) + i));
    glo = min(glo, s.x);
    ghi = max(ghi, s.y);
  }
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
    top[j] = p.lse[(long)h * p.N + rc];
    inv[j] = p.lse[(long)(p.H + h) * p.N + rc];
    if (r < p.N && g == 0) delta[(long)h * p.N + r] = dsum[j];
    qx[j] = AXES ? p.xy[(long)rc * AXES] : 0.f;
    qy[j] = AXES > 1 ? p.xy[(long)rc * AXES + 1] : 0.f;
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    wlo = min(wlo, __shfl_xor(wlo, o, 64));
    whi = max(whi, __shfl_xor(whi, o, 64));
    flo = max(flo, __shfl_xor(flo, o, 64));
    fhi = min(fhi, __shfl_xor(fhi, o, 64));
  }
  wlo = __builtin_amdgcn_readfirstlane(wlo), whi = __builtin_amdgcn_readfirstlane(whi);
  flo = __builtin_amdgcn_readfirstlane(flo), fhi = __builtin_amdgcn_readfirstlane(fhi);

  const T* kb = (const T*)p.k + hk * p.k_head;
  const T* vb = (const T*)p.v + hk * p.v_head;
  auto fetch = [&](int k0, int buf) {
    copy_tile<G>(kb, p.k_row, k0, glo, ghi, nd, lk[buf]);
    copy_tile<G>(vb, p.v_row, k0, glo, ghi, nd, lv[buf]);
    if (wave < AXES) copy_meta(p.kv_xy, AXES, wave, k0, p.M, lx[buf][wave]);
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
    __syncthreads();
    if (k0 + G::BK < ghi) fetch(k0 + G::BK, buf ^ 1);
    if (k0 >= whi || k0 + G::BK <= wlo) continue;
    f32x4 s[QF][G::F], dp[QF][G::F];
    scores<G, QF>(lk[buf], q, s, at);
    scores<G, QF>(lv[buf], dO, dp, at);
    const bool part = k0 < flo || k0 + G::BK > fhi;
    float ta[QF] = {}, tb[QF] = {}, tc[QF] = {};
#pragma unroll
    for (int f = 0; f < G::F; ++f) {
      const int kr = G::row4(f, g);
      f32x4 bx = {}, by = {};
      if (AXES) bx = *(const f32x4*)&lx[buf][0][kr];
      if (AXES > 1) by = *(const f32x4*)&lx[buf][1][kr];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < QF; ++j) {
          float x = s[j][f][r], fac = 1.f, dist = 0.f;
          if (!W::RAW) x = soft.score(x, qx[j], qy[j], bx[r], by[r], fac, dist);
          float w = soft.weight(x, top[j]) * inv[j], dl = w * (dp[j][f][r] - dsum[j]);
          if (W::CAP) dl *= fac;
          float wd = w * dp[j][f][r];
          if (part) {
            const int key = k0 + kr + r;
            const bool seen = key >= lo[j] && key < hi[j];
            dl = seen ? dl : 0.f;
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
          s[j][f][r] = dl;
        }
    }
    if (AXES) {
#pragma unroll
      for (int j = 0; j < QF; ++j) sa[j] += ta[j], sb[j] += tb[j], sc[j] += tc[j];
    }
    if (part && tile_not_finite<G>(lk[buf], lane))
      accumulate_seen<G, QF>(lk[buf], s, acc, lane, [&](int j, int row) { return k0 + row >= lo[j] && k0 + row < hi[j]; });
    else
      accumulate<G, QF>(lk[buf], s, acc, at);
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
  if (AXES && p.dslopes) {
    float slope_sum = 0.f;
#pragma unroll
    for (int j = 0; j < QF; ++j) {
      const float a = quarters_sum(sa[j]), b = quarters_sum(sb[j]), c = quarters_sum(sc[j]);
      if (g == 0 && w0 + 16 * j + i16 < p.N) slope_sum += fmaf(-c, b, a);
    }
    __syncthreads();
    const float w = wave_sum(slope_sum);
    if (lane == 0) lx[0][0][wave] = w;
    __syncthreads();
    if (threadIdx.x == 0) slope_part[(long)h * nqt + qt] = (lx[0][0][0] + lx[0][0][1]) + (lx[0][0][2] + lx[0][0][3]);
  }
}

// The slopes' gradient: a head's partial sums in their order.
__global__ __launch_bounds__(64) void blk_slopes_kernel(const float* part, int n, float* out) {
  const int lane = threadIdx.x;
  double s = 0.;
  for (int i = lane; i < n; i += 64) s += (double)part[(long)blockIdx.x * n + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) out[blockIdx.x] = (float)-s;
}

// A workgroup: 64 QF keys of one key head; the queries of every head that shares it, in tiles of BK rows.
template <class T, int DP, int QF, int X>
__global__ __launch_bounds__(256, 2) void blk_attn_dkv_kernel(BlkAttnArgs p, int np, const float* delta) {
  using G = Geo<T, DP>;
  using W = Soft<T, X>;
  constexpr int AXES = W::AXES;
  __shared__ u32x4 lq[2][G::TILE], lo_[2][G::TILE];
  __shared__ __attribute__((aligned(16))) float lm[2][7][64];  // of each streamed row: largest score, sum(dO O), lo, hi, x, y, 1 / sum
  __shared__ int range[2];
  const int lane = mg_lane(), wave = mg_wave(), i16 = lane & 15, g = lane >> 4;
  const int hk = blockIdx.x % p.Hkv, kt = blockIdx.x / p.Hkv, group = p.H / p.Hkv;
  const int b0 = kt * 64 * QF, w0 = b0 + wave * 16 * QF;
  const int nd = p.D / G::CH;

  // the rows that see any of the workgroup's keys lie between the first and the last 32 that do
  if (threadIdx.x == 0) range[0] = INT_MAX, range[1] = -1;
  __syncthreads();
  for (int u = threadIdx.x; u < np / 32; u += 256) {
    const int4 s = *(const int4*)(p.spans + 2 * np + 4 * u);
    if (s.x < b0 + 64 * QF && s.y > b0) {
      atomicMin(&range[0], u);
      atomicMax(&range[1], u);
    }
  }
  __syncthreads();
  const int first = range[0], last = range[1];
  const int qa = last < 0 ? 0 : first * 32 / G::BK * G::BK, qb = (last + 1) * 32;

  float kx[QF], ky[QF];
  u32x4 k[QF][G::SK], v[QF][G::SK];
#pragma unroll
  for (int j = 0; j < QF; ++j) {
    const int rc = min(w0 + 16 * j + i16, p.M - 1);
    const T* kr = (const T*)p.k + rc * p.k_row + hk * p.k_head;
    const T* vr = (const T*)p.v + rc * p.v_row + hk * p.v_head;
#pragma unroll
    for (int s = 0; s < G::SK; ++s) {
      k[j][s] = owner_chunk(kr, 4 * s + g, nd);
      v[j][s] = owner_chunk(vr, 4 * s + g, nd);
    }
    kx[j] = AXES ? p.kv_xy[(long)rc * AXES] : 0.f;
    ky[j] = AXES > 1 ? p.kv_xy[(long)rc * AXES + 1] : 0.f;
  }
  f32x4 dk[QF][G::DF], dv[QF][G::DF];
#pragma unroll
  for (int j = 0; j < QF; ++j)
#pragma unroll
    for (int d = 0; d < G::DF; ++d) dk[j][d] = dv[j][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  Lane<G> at;
  at.init(lane);

  // (head, tile) pairs in one sequence, so that the copies of the next head's first tile are under way too
  const int nt = qb > qa ? (qb - qa + G::BK - 1) / G::BK : 0, total = nt * group;
  auto fetch = [&](int t, int buf) {
    const int h = hk * group + t / nt, q0 = qa + t % nt * G::BK;
    copy_tile<G>((const T*)p.q + h * p.q_head, p.q_row, q0, 0, p.N, nd, lq[buf]);
    copy_tile<G>((const T*)p.dout + (long)h * p.D, (long)p.H * p.D, q0, 0, p.N, nd, lo_[buf]);
    if (wave == 0) copy_meta(p.lse + (long)h * p.N, 1, 0, q0, p.N, lm[buf][0]);
    if (wave == 3) copy_meta(p.lse + (long)(p.H + h) * p.N, 1, 0, q0, p.N, lm[buf][6]);
    if (wave == 1) copy_meta(delta + (long)h * p.N, 1, 0, q0, p.N, lm[buf][1]);
    if (wave == 2) copy_meta(p.spans, 1, 0, q0, np, lm[buf][2]);
    if (wave == 3) copy_meta(p.spans + np, 1, 0, q0, np, lm[buf][3]);
    if (wave < AXES) copy_meta(p.xy, AXES, wave, q0, p.N, lm[buf][4 + wave]);
  };
  if (total > 0) fetch(0, 0);
  for (int t = 0; t < total; ++t) {
    const int buf = t & 1, q0 = qa + t % nt * G::BK, h = hk * group + t / nt;
    __syncthreads();
    if (t + 1 < total) fetch(t + 1, buf ^ 1);
    int slo = INT_MAX, shi = 0, flo = 0, fhi = INT_MAX;
#pragma unroll
    for (int i = 0; i < G::BK / 32; ++i) {
      const int4 u = *(const int4*)(p.spans + 2 * np + 4 * ((q0 >> 5) + i));
      slo = min(slo, u.x), shi = max(shi, u.y), flo = max(flo, u.z), fhi = min(fhi, u.w);
    }
    if (slo >= w0 + 16 * QF || shi <= w0) continue;
    const bool part = w0 < flo || w0 + 16 * QF > fhi;
    const W soft(p, AXES ? p.slopes[h] : 0.f);
    f32x4 s[QF][G::F], dp[QF][G::F];
    scores<G, QF>(lq[buf], k, s, at);
    scores<G, QF>(lo_[buf], v, dp, at);
#pragma unroll
    for (int f = 0; f < G::F; ++f) {
      const int qr = G::row4(f, g);
      const f32x4 top = *(const f32x4*)&lm[buf][0][qr], dsum = *(const f32x4*)&lm[buf][1][qr], inv = *(const f32x4*)&lm[buf][6][qr];
      f32x4 ax = {}, ay = {};
      if (AXES) ax = *(const f32x4*)&lm[buf][4][qr];
      if (AXES > 1) ay = *(const f32x4*)&lm[buf][5][qr];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < QF; ++j) {
          float x = s[j][f][r], fac = 1.f, dist;
          if (!W::RAW) x = soft.score(x, ax[r], ay[r], kx[j], ky[j], fac, dist);
          float w = soft.weight(x, top[r]) * inv[r], dl = w * (dp[j][f][r] - dsum[r]);
          if (W::CAP) dl *= fac;
          s[j][f][r] = w;
          dp[j][f][r] = dl;
        }
      if (part) {
        const f32x4 from = *(const f32x4*)&lm[buf][2][qr], to = *(const f32x4*)&lm[buf][3][qr];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < QF; ++j) {
            const int key = w0 + 16 * j + i16;
            const bool seen = key >= __float_as_int(from[r]) && key < __float_as_int(to[r]);
            s[j][f][r] = seen ? s[j][f][r] : 0.f;
            dp[j][f][r] = seen ? dp[j][f][r] : 0.f;
          }
      }
    }
    auto sees = [&](int j, int row) {
      const int key = w0 + 16 * j + i16;
      return key >= __float_as_int(lm[buf][2][row]) && key < __float_as_int(lm[buf][3][row]);
    };
    if (part && (tile_not_finite<G>(lo_[buf], lane) || tile_not_finite<G>(lq[buf], lane))) {
      accumulate_seen<G, QF>(lo_[buf], s, dv, lane, sees);
      accumulate_seen<G, QF>(lq[buf], dp, dk, lane, sees);
    } else {
      accumulate<G, QF>(lo_[buf], s, dv, at);
      accumulate<G, QF>(lq[buf], dp, dk, at);
    }
  }
#pragma unroll
  for (int j = 0; j < QF; ++j) {
    const int r = w0 + 16 * j + i16;
    if (r >= p.M) continue;
    const long o = ((long)r * p.Hkv + hk) * p.D;
#pragma unroll
    for (int d = 0; d < G::DF; ++d)
      if (16 * d + 4 * g < p.D) {
        store4<T>((T*)p.dk + o + 16 * d + 4 * g, dk[j][d], p.scale);
        store4<T>((T*)p.dv + o + 16 * d + 4 * g, dv[j][d], 1.f);
      }
  }
}

template <class T, int DP, int X>
void launch_bwd_x(const BlkAttnArgs& p, hipStream_t st) {
  constexpr int QF = 1;
  const int np = cdiv(p.N, 128) * 128, nqt = cdiv(p.N, 64 * QF);
  float* delta = (float*)p.ws;
  float* part = delta + (size_t)p.H * p.N;
  MG_LAUNCH((blk_attn_dq_kernel<T, DP, QF, X>), dim3(nqt * p.H), dim3(256), 0, st, p, np, delta, part);
  if (X > 1 && p.dslopes) MG_LAUNCH(blk_slopes_kernel, dim3(p.H), dim3(64), 0, st, (const float*)part, nqt, p.dslopes);
  MG_LAUNCH((blk_attn_dkv_kernel<T, DP, QF, X>), dim3(cdiv(p.M, 64 * QF) * p.Hkv), dim3(256), 0, st, p, np, (const float*)delta);
}
template <class T, int DP>
void launch_bwd(const BlkAttnArgs& p, hipStream_t st) {
  switch ((p.cap > 0.f ? 1 : 0) + 2 * p.axes) {
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

size_t mggan_block_attention_bwd_workspace(int rows, int heads) {
  return rows > 0 && heads > 0 ? ((size_t)heads * rows + (size_t)heads * cdiv(rows, 64)) * 4 : 0;
}

int mggan_block_attention_bwd(const void* args, hipStream_t stream) {
  const BlkAttnArgs* a = (const BlkAttnArgs*)args;
  const int rc = blk_attn_check(a, "block_attention_bwd");
  if (rc != MGGAN_OK) return rc;
  MG_CHECK_ARG(a->out32 && a->lse && a->dout && a->dq && a->dk && a->dv, "block_attention_bwd: null operand");
  MG_CHECK_ARG(((size_t)a->out32 | (size_t)a->dout | (size_t)a->dq | (size_t)a->dk | (size_t)a->dv | (size_t)a->spans) % 16 == 0,
               "block_attention_bwd: operands have to be 16-byte aligned");
  const size_t need = mggan_block_attention_bwd_workspace(a->N, a->H);
  MG_CHECK_ARG(a->ws && (size_t)a->ws_bytes >= need, "block_attention_bwd: workspace of %zu bytes (got %ld)", need, a->ws_bytes);
  if (a->dtype == BLK_BF16)
    launch_bwd_width<bf16>(*a, stream);
  else
    launch_bwd_width<float>(*a, stream);
  MG_LAUNCH_CHECK("block_attention_bwd");
  return MGGAN_OK;
}
}
