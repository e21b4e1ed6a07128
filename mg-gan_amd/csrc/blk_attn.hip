// Attention over the rows of scenes, forward: intervals of visible keys, one pass over the keys with running maximum and sum.
#include <limits.h>
#include "blk_attn.h"
#include "../../include/mggan_hip.h"

namespace {

// The interval of keys that row r of scene s sees (s < 0: of none).  What the tables say is clamped to the operands' rows.
__device__ __forceinline__ int2 blk_span(const BlkAttnArgs& p, int s, int r) {
  if (s < 0) return make_int2(0, 0);
  const int q0 = max(p.scenes[2 * s], 0), q1 = min(p.scenes[2 * s + 1], p.N);
  const int k0 = min(max(p.kv_scenes[2 * s], 0), p.M), k1 = min(max(p.kv_scenes[2 * s + 1], k0), p.M);
  int n = k1 - k0;
  if (p.causal) {
    const int pre = p.prefix ? p.prefix[s] : 0;
    n = max(0, min(n, max(pre, r - q0 + 1 + n - (q1 - q0))));
  }
  return n > 0 ? make_int2(k0, k0 + n) : make_int2(0, 0);
}

// The interval of keys that each of 64 rows sees, and what every 32 rows have in common.  All scenes are looked through (in any
// order; the last one that names a row counts), so that nothing is asked of a list in device memory.
__global__ __launch_bounds__(256) void blk_spans_kernel(BlkAttnArgs p, int np) {
  __shared__ int scene[64];
  const int r0 = blockIdx.x * 64, tid = threadIdx.x;
  if (tid < 64) scene[tid] = -1;
  __syncthreads();
  for (int s = tid; s < p.S; s += 256) {
    const int a = max(p.scenes[2 * s], r0), b = min(p.scenes[2 * s + 1], min(r0 + 64, p.N));
    for (int r = a; r < b; ++r) atomicMax(&scene[r - r0], s);
  }
  __syncthreads();
  if (tid >= 64) return;
  const int s = scene[tid];
  const int2 span = blk_span(p, s, r0 + tid);
  const int lo = span.x, hi = span.y;
  p.spans[r0 + tid] = lo;
  p.spans[np + r0 + tid] = hi;
  const bool some = hi > lo;
  int v[4] = {some ? lo : INT_MAX, some ? hi : 0, some ? lo : INT_MAX, some ? hi : 0};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    v[0] = min(v[0], __shfl_xor(v[0], o, 64));
    v[1] = max(v[1], __shfl_xor(v[1], o, 64));
    v[2] = max(v[2], __shfl_xor(v[2], o, 64));
    v[3] = min(v[3], __shfl_xor(v[3], o, 64));
  }
  if ((tid & 31) == 0) *(int4*)(p.spans + 2 * np + 4 * ((r0 + tid) >> 5)) = make_int4(v[0], v[1], v[2], v[3]);
}

// 64 QF query rows of one head: four waves of 16 QF rows each (this one's start at w0); keys and values in tiles of BK rows, two buffers.
//   m' = max(m, max_j s_j)    l' = l 2^(m-m') + sum_j 2^(s_j-m')    acc' = acc 2^(m-m') + sum_j 2^(s_j-m') v_j    out = acc / l
// Bound by the vector instructions around the softmax: they fill 71 % of the time (an exp2 or rcp counts as two), both at width 64 with a cap, where
// the matrix cores are busy 12 %, and at width 128 with a distance, 35 %.  16,384 causal rows of 8 heads at width 128 take 0.85 ms, packed 8,192
// rows of 16 heads at width 64 with a cap 95 us.
template <class T, int DP, int QF, int X, bool SAFE>
__device__ __forceinline__ void attn_fwd_rows(const BlkAttnArgs& p, int np, int h, int glo, int ghi, int w0, u32x4* lk, u32x4* lv, float* lx, int* odd) {
  using G = Geo<T, DP>;
  using W = Soft<T, X>;
  constexpr int AXES = W::AXES;
  const int lane = mg_lane(), wave = mg_wave(), i16 = lane & 15, g = lane >> 4, hk = h / (p.H / p.Hkv), nd = p.D / G::CH;
  int lo[QF], hi[QF], wlo = INT_MAX, whi = 0, flo = 0, fhi = INT_MAX;
  float qx[QF], qy[QF];
  u32x4 q[QF][G::SK];
#pragma unroll
  for (int j = 0; j < QF; ++j) {
    const int r = w0 + 16 * j + i16, rc = min(r, p.N - 1);
    lo[j] = p.spans[r];
    hi[j] = p.spans[np + r];
    if (hi[j] > lo[j]) wlo = min(wlo, lo[j]), whi = max(whi, hi[j]);
    flo = max(flo, hi[j] > lo[j] ? lo[j] : INT_MAX);
    fhi = min(fhi, hi[j]);
    const T* row = (const T*)p.q + rc * p.q_row + h * p.q_head;
#pragma unroll
    for (int s = 0; s < G::SK; ++s) q[j][s] = owner_chunk(row, 4 * s + g, nd);
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
  float m[QF], l[QF];
#pragma unroll
  for (int j = 0; j < QF; ++j) {
    m[j] = -INFINITY;
    l[j] = 0.f;
#pragma unroll
    for (int d = 0; d < G::DF; ++d) acc[j][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const W soft(p, AXES ? p.slopes[h] : 0.f);
  Lane<G> at;
  at.init(lane);

  if (glo < ghi) fetch(glo, 0);
  int buf = 0;
  for (int k0 = glo; k0 < ghi; k0 += G::BK, buf ^= 1) {
    copies_done();
    if (k0 + G::BK < ghi) fetch(k0 + G::BK, buf ^ 1);
    if (k0 >= whi || k0 + G::BK <= wlo) continue;  // (the wave's: nothing of this tile is seen)
    const u32x4* tv = lv + buf * G::TILE;
    f32x4 s[QF][G::F];
    scores<G, QF>(lk + buf * G::TILE, q, s, at);
    const bool part = k0 < flo || k0 + G::BK > fhi;
    if (!W::RAW) {
#pragma unroll
      for (int f = 0; f < G::F; ++f) {
        const int kr = G::row4(f, g);
        f32x4 bx = {}, by = {};
        if (AXES) bx = *(const f32x4*)(lx + 2 * buf * 64 + kr);
        if (AXES > 1) by = *(const f32x4*)(lx + (2 * buf + 1) * 64 + kr);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < QF; ++j) {
            float fac, dist;
            s[j][f][r] = soft.score(s[j][f][r], qx[j], qy[j], bx[r], by[r], fac, dist);
          }
      }
    }
    if (part) {
      if (!SAFE && tile_not_finite<G>(tv, lane)) *odd = 1;
#pragma unroll
      for (int f = 0; f < G::F; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = k0 + G::row4(f, g) + r;
#pragma unroll
          for (int j = 0; j < QF; ++j) s[j][f][r] = key >= lo[j] && key < hi[j] ? s[j][f][r] : -INFINITY;
        }
    }
    Coef<T> w[QF][G::F];
#pragma unroll
    for (int j = 0; j < QF; ++j) {
      float t = -INFINITY;
#pragma unroll
      for (int f = 0; f < G::F; ++f) t = fmaxf(t, fmaxf(fmaxf(s[j][f][0], s[j][f][1]), fmaxf(s[j][f][2], s[j][f][3])));
      t = quarters_max(t) * soft.E;
      if (__ballot(t > m[j] + 8.f)) {  // (weights up to 2^8 are as good: most tiles leave the sums as they are)
        const float mn = fmaxf(m[j], t), al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[j] - mn);
        m[j] = mn;
        l[j] *= al;
#pragma unroll
        for (int d = 0; d < G::DF; ++d) acc[j][d] *= al;
      }
      const float mm = m[j] == -INFINITY ? 0.f : m[j];
      float sum = 0.f;
#pragma unroll
      for (int f = 0; f < G::F; ++f) {
        f32x4 e;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          e[r] = soft.weight(s[j][f][r], mm);
          sum += e[r];
        }
        w[j][f].set(e);
      }
      l[j] += sum;
    }
    if (SAFE && part && tile_not_finite<G>(tv, lane))
      accumulate_seen<G, QF>(tv, w, acc, at, lane, [&](int j, int row) { return k0 + row >= lo[j] && k0 + row < hi[j]; });
    else
      accumulate<G, QF>(tv, w, acc, at);
  }
  if (!SAFE) {
    __syncthreads();
    if (*odd) return;
  }

#pragma unroll
  for (int j = 0; j < QF; ++j) {
    const int r = w0 + 16 * j + i16;
    const float sum = quarters_sum(l[j]), inv = hi[j] > lo[j] ? 1.f / sum : 0.f;
    if (r >= p.N) continue;
    if (g == 0 && p.lse) {
      p.lse[(long)h * p.N + r] = m[j];
      p.lse[(long)(p.H + h) * p.N + r] = inv;
      p.lse[(long)(2 * p.H + h) * p.N + r] = m[j] + __log2f(sum);
    }
    const long o = ((long)r * p.H + h) * p.D;
#pragma unroll
    for (int d = 0; d < G::DF; ++d)
      if (16 * d + 4 * g < p.D) {
        store4<T>((T*)p.out + o + 16 * d + 4 * g, acc[j][d], inv);
        if (sizeof(T) == 2 && p.out32) store4<float>(p.out32 + o + 16 * d + 4 * g, acc[j][d], inv);
      }
  }
}

template <class T, int DP, int QF, int X>
__global__ __launch_bounds__(256, QF == 1 && DP <= 64 ? 3 : 2) void blk_attn_fwd_kernel(BlkAttnArgs p, int np) {
  using G = Geo<T, DP>;
  __shared__ struct {
    u32x4 k[2 * G::TILE], v[2 * G::TILE];
    float x[2 * 2 * 64];
    int odd, order[RANK_MAX + 1];
  } lds;
  const int h = blockIdx.x % p.H;
  const int qt = by_work(blockIdx.x / p.H, gridDim.x / p.H, [&](int i) {
    const int2 k = group_span<2 * QF>(p, np, i * 64 * QF);
    return k.y - k.x;
  }, lds.order);
  const int r0 = qt * 64 * QF, w0 = r0 + mg_wave() * 16 * QF;
  if (threadIdx.x == 0) lds.odd = 0;
  __syncthreads();
  const int2 keys = group_span<2 * QF>(p, np, r0);  // (what the workgroup's rows see)
  attn_fwd_rows<T, DP, QF, X, false>(p, np, h, keys.x, keys.y, w0, lds.k, lds.v, lds.x, &lds.odd);
  if (!lds.odd) return;
  for (int j = 0; j < QF; ++j) {
    __syncthreads();
    attn_fwd_rows<T, DP, 1, X, true>(p, np, h, keys.x, keys.y, afresh(w0 + 16 * j), lds.k, lds.v, lds.x, &lds.odd);
  }
}

// Few rows over long caches.  A workgroup takes one row, the heads of one key head (up to 16: the columns of the matrix
// instruction) and one of `splits` shares of the row's keys; its four waves take the share's tiles in turn, each with LDS of its own and
// no barrier between them: what counts is bytes in flight (two tiles of keys and values a wave, 64 KB a CU at width 128).  Bound by the cache's
// bytes: 32 rows over 16,384 keys each, width 128, 1.62 GB in 287 us, 5.6 TB/s.  Shares leave
// maximum, sum and unnormalised output, which blk_attn_join_kernel puts together in their order.
template <class T, int DP, int X>
__global__ __launch_bounds__(256) void blk_attn_row_kernel(BlkAttnArgs p, int splits, int hgroups, float* part) {
  using G = Geo<T, DP, 64 / (int)sizeof(T)>;
  using W = Soft<T, X>;
  constexpr int AXES = W::AXES;
  constexpr int LOADS = 2 * G::TILE / 64;  // copies of a tile of keys and one of values
  __shared__ struct {
    u32x4 tiles[4][2][2][G::TILE];
    int scene;
  } lds;
  auto& tiles = lds.tiles;
  const int lane = mg_lane(), wave = mg_wave(), i16 = lane & 15, g = lane >> 4, nd = p.D / G::CH;
  int id = blockIdx.x;
  const int sp = id % splits;
  id /= splits;
  const int hg = id % hgroups;
  id /= hgroups;
  const int hk = id % p.Hkv, r = id / p.Hkv, group = p.H / p.Hkv;
  const int head = hk * group + hg * 16 + i16;
  const bool mine = hg * 16 + i16 < group;

  if (threadIdx.x == 0) lds.scene = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < p.S; s += 256)
    if (p.scenes[2 * s] <= r && r < p.scenes[2 * s + 1]) atomicMax(&lds.scene, s);
  __syncthreads();
  const int2 span = blk_span(p, lds.scene, r);
  const int n = span.y - span.x, per = ((n + splits - 1) / splits + G::BK - 1) / G::BK * G::BK;
  const int lo = min(span.x + sp * per, span.y), hi = min(lo + per, span.y);

  u32x4 q[1][G::SK];
#pragma unroll
  for (int s = 0; s < G::SK; ++s)
    q[0][s] = mine ? owner_chunk((const T*)p.q + r * p.q_row + head * p.q_head, 4 * s + g, nd) : u32x4{0, 0, 0, 0};
  const float qx = AXES ? p.xy[(long)r * AXES] : 0.f, qy = AXES > 1 ? p.xy[(long)r * AXES + 1] : 0.f;
  const W soft(p, AXES && mine ? p.slopes[head] : 0.f);
  Lane<G> at;
  at.init(lane);
  f32x4 acc[1][G::DF];
#pragma unroll
  for (int d = 0; d < G::DF; ++d) acc[0][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  auto fetch = [&](int k0, int buf) {
    copy_tile<G, 64>((const T*)p.k + hk * p.k_head, p.k_row, k0, lo, hi, nd, tiles[wave][buf][0]);
    copy_tile<G, 64>((const T*)p.v + hk * p.v_head, p.v_row, k0, lo, hi, nd, tiles[wave][buf][1]);
  };
  int buf = 0;
  const int first = lo + wave * G::BK;
  if (first < hi) fetch(first, 0);
  for (int k0 = first; k0 < hi; k0 += 4 * G::BK, buf ^= 1) {
    if (k0 + 4 * G::BK < hi) {
      fetch(k0 + 4 * G::BK, buf ^ 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");  // (copies end in their order: this tile's have)
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    f32x4 s[1][G::F];
    scores<G, 1>(tiles[wave][buf][0], q, s, at);
    float t = -INFINITY;
#pragma unroll
    for (int f = 0; f < G::F; ++f)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = k0 + G::row4(f, g) + e;
        float x = s[0][f][e];
        if (!W::RAW) {
          const long k = (long)min(key, p.M - 1) * AXES;
          float fac, dist;
          x = soft.score(x, qx, qy, AXES ? p.kv_xy[k] : 0.f, AXES > 1 ? p.kv_xy[k + 1] : 0.f, fac, dist);
        }
        x = key < hi ? x : -INFINITY;
        s[0][f][e] = x;
        t = fmaxf(t, x);
      }
    t = quarters_max(t) * soft.E;
    if (__ballot(t > m + 8.f)) {
      const float mn = fmaxf(m, t), al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int d = 0; d < G::DF; ++d) acc[0][d] *= al;
    }
    const float mm = m == -INFINITY ? 0.f : m;
    Coef<T> w[1][G::F];
#pragma unroll
    for (int f = 0; f < G::F; ++f) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = soft.weight(s[0][f][e], mm);
        l += x[e];
      }
      w[0][f].set(x);
    }
    accumulate<G, 1>(tiles[wave][buf][1], w, acc, at);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (this tile is read before the next copy goes into it)
  }
  l = quarters_sum(l);

  // the four waves' results, joined by wave 0 .. 3 in turn order
  __syncthreads();
  float* sm = (float*)&tiles[0][0][0][0];  // [wave][16 heads][m, l], then [wave][DP][16 heads]
  if (g == 0) sm[wave * 32 + i16] = m, sm[wave * 32 + 16 + i16] = l;
  float* so = sm + 128 + wave * DP * 16;
#pragma unroll
  for (int d = 0; d < G::DF; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) so[(16 * d + 4 * g + e) * 16 + i16] = acc[0][d][e];
  __syncthreads();
  const int heads = min(16, group - hg * 16);
  for (int i = threadIdx.x; i < heads * p.D; i += 256) {
    const int d = i % p.D, hh = i / p.D;
    float mt = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, sm[w * 32 + hh]);
    float lt = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = mt == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sm[w * 32 + hh] - mt);
      lt = fmaf(f, sm[w * 32 + 16 + hh], lt);
      o = fmaf(f, sm[128 + (w * DP + d) * 16 + hh], o);
    }
    const int h = hk * group + hg * 16 + hh;
    if (splits > 1) {
      float* out = part + (((long)r * p.H + h) * splits + sp) * (p.D + 4);
      out[d] = o;
      if (d == 0) out[p.D] = mt, out[p.D + 1] = lt, out[p.D + 2] = n > 0 ? 1.f : 0.f;
    } else {
      const float inv = n > 0 ? 1.f / lt : 0.f;
      ((T*)p.out)[((long)r * p.H + h) * p.D + d] = (T)(o * inv);
    }
  }
}

template <class T>
__global__ __launch_bounds__(128) void blk_attn_join_kernel(BlkAttnArgs p, int splits, const float* part) {
  const int d = threadIdx.x;
  const float* in = part + (long)blockIdx.x * splits * (p.D + 4);
  float mt = -INFINITY;
  for (int s = 0; s < splits; ++s) mt = fmaxf(mt, in[(long)s * (p.D + 4) + p.D]);
  float lt = 0.f, o = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float* x = in + (long)s * (p.D + 4);
    const float f = mt == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(x[p.D] - mt);
    lt = fmaf(f, x[p.D + 1], lt);
    if (d < p.D) o = fmaf(f, x[d], o);
  }
  const float inv = in[p.D + 2] != 0.f ? 1.f / lt : 0.f;
  if (d < p.D) ((T*)p.out)[(long)blockIdx.x * p.D + d] = (T)(o * inv);
}

// Few rows a scene over long caches (no gradient kept): how many shares of the keys; 0 where the tile kernel runs instead.
// A row's keys are read for it alone here; the tile kernel reads them once for 64 rows, but by few workgroups where rows are few, and through
// the keys of every scene that its 64 rows span.  So this one is taken while its workgroups are at most 400 for each round of the tile kernel's
// (512 of them run at once) and each scene spanned.  Measured, this kernel / the tiles, us: one row over 1,000 keys 9.4 / 35; 32 x 1 over 16,384,
// 223 / 23,580; 16 x 16 over 1,000 (102) 13 / 55; 64 x 16 over 500 (410) 29 / 36; 64 rows of one scene over 4,000, 8 key heads (512) 89 / 80; 64 x 32
// over 200 (5,461) 119 / 19.  Below 64 keys a scene both are
// launches (4.6 / 8.0).
int row_splits(const BlkAttnArgs& p) {
  if (p.lse || p.S == 0 || p.N > 64L * p.S || p.M / p.S < 64) return 0;
  const long blocks = (long)p.N * p.Hkv * cdiv(p.H / p.Hkv, 16), rounds = cdiv((long)cdiv(p.N, 64) * p.H, 512);
  const long spanned = 64L * p.S / p.N + 1;
  if (blocks > 400 * rounds * (spanned < p.S ? spanned : p.S)) return 0;
  if ((long)p.N * p.H > 1 << 22) return 0;  // (more workgroups than a launch takes)
  long n = cdiv(1024, blocks);
  if (n > p.M / p.S / 512) n = p.M / p.S / 512;  // (a share of fewer keys is not worth the launch that joins: 1,000 keys 20 -> 17 us)
  return n < 1 ? 1 : n > 64 ? 64 : (int)n;
}

template <class T, int DP, int X>
void launch_fwd_x(const BlkAttnArgs& p, hipStream_t st) {
  const int splits = row_splits(p);
  if (splits) {
    const int hgroups = cdiv(p.H / p.Hkv, 16);
    const dim3 grid((unsigned)((long)p.N * p.Hkv * hgroups * splits));
    MG_LAUNCH((blk_attn_row_kernel<T, DP, X>), grid, dim3(256), 0, st, p, splits, hgroups, (float*)p.ws);
    if (splits > 1)
      MG_LAUNCH((blk_attn_join_kernel<T>), dim3(p.N * p.H), dim3(128), 0, st, p, splits, (const float*)p.ws);
    return;
  }
  const int np = cdiv(p.N, 128) * 128;
  MG_LAUNCH(blk_spans_kernel, dim3(np / 64), dim3(256), 0, st, p, np);
  // 128 rows a workgroup read every key once for 32 rows of a wave instead of 16, which pays where LDS is what they wait for (width 128,
  // 16,384 rows: 0.80 against 1.10 ms); below that three smaller waves a SIMD are better (width 64: 127 against 101 us)
  constexpr int QF = DP > 64 ? 2 : 1;
  if (QF > 1 && (long)cdiv(p.N, 128) * p.H >= 256)
    MG_LAUNCH((blk_attn_fwd_kernel<T, DP, QF, X>), dim3(cdiv(p.N, 64 * QF) * p.H), dim3(256), 0, st, p, np);
  else
    MG_LAUNCH((blk_attn_fwd_kernel<T, DP, 1, X>), dim3(cdiv(p.N, 64) * p.H), dim3(256), 0, st, p, np);
}
template <class T, int DP>
void launch_fwd(const BlkAttnArgs& p, hipStream_t st) {
  const int x = blk_attn_x<T>(p);
  if constexpr (sizeof(T) == 2) {
    switch (x) {
      case 9: return launch_fwd_x<T, DP, 9>(p, st);
      case 11: return launch_fwd_x<T, DP, 11>(p, st);
      case 13: return launch_fwd_x<T, DP, 13>(p, st);
    }
  }
  switch (x) {
    case 0: return launch_fwd_x<T, DP, 0>(p, st);
    case 1: return launch_fwd_x<T, DP, 1>(p, st);
    case 2: return launch_fwd_x<T, DP, 2>(p, st);
    case 3: return launch_fwd_x<T, DP, 3>(p, st);
    case 4: return launch_fwd_x<T, DP, 4>(p, st);
    default: return launch_fwd_x<T, DP, 5>(p, st);
  }
}
template <class T>
void launch_fwd_width(const BlkAttnArgs& p, hipStream_t st) {
  if (p.D <= 32)
    launch_fwd<T, 32>(p, st);
  else if (p.D <= 64)
    launch_fwd<T, 64>(p, st);
  else if (p.D <= 96)
    launch_fwd<T, 96>(p, st);
  else
    launch_fwd<T, 128>(p, st);
}

size_t fwd_workspace(const BlkAttnArgs& p) {
  const int splits = row_splits(p);
  return splits > 1 ? (size_t)p.N * p.H * splits * (p.D + 4) * 4 : 0;
}

}  // namespace

int blk_attn_check(const BlkAttnArgs* a, const char* name) {
  MG_CHECK_ARG(a, "%s: no arguments", name);
  const BlkAttnArgs& p = *a;
  MG_CHECK_ARG(p.dtype == BLK_F32 || p.dtype == BLK_BF16, "%s: dtype %d (0 = f32, 1 = bf16)", name, p.dtype);
  MG_CHECK_ARG(p.N > 0 && p.M > 0 && p.N <= (1 << 24) && p.M <= (1 << 30), "%s: %d rows, %d keys", name, p.N, p.M);
  MG_CHECK_ARG(p.H > 0 && p.Hkv > 0 && p.H % p.Hkv == 0 && p.H <= 1024, "%s: %d heads over %d key heads", name, p.H, p.Hkv);
  MG_CHECK_ARG((long)cdiv(p.N, 64) * p.H <= 1 << 23, "%s: %d rows of %d heads are too many workgroups", name, p.N, p.H);
  MG_CHECK_ARG(p.D > 0 && p.D <= 128 && p.D % 8 == 0, "%s: width %d (a multiple of 8 up to 128)", name, p.D);
  auto in_range = [](float x) { return x >= 0x1p-60f && x <= 0x1p60f; };  // (quotient and products stay normal numbers)
  MG_CHECK_ARG(p.S >= 0 && p.axes >= 0 && p.axes <= 2 && in_range(p.scale) && (p.cap == 0.f || in_range(p.cap)),
               "%s: %d scenes, %d axes, scale %g, cap %g", name, p.S, p.axes, p.scale, p.cap);
  MG_CHECK_ARG(p.q && p.k && p.v && p.spans && (p.S == 0 || (p.scenes && p.kv_scenes)), "%s: null operand", name);
  MG_CHECK_ARG(!p.axes || (p.xy && p.kv_xy && p.slopes), "%s: positions without coordinates or slopes", name);
  const long ch = p.dtype == BLK_BF16 ? 8 : 4;
  MG_CHECK_ARG(((size_t)p.q | (size_t)p.k | (size_t)p.v) % 16 == 0 && (p.q_row | p.q_head | p.k_row | p.k_head | p.v_row | p.v_head) % ch == 0,
               "%s: operands and their strides have to be multiples of 16 bytes", name);
  return MGGAN_OK;
}

extern "C" {

size_t mggan_block_attention_span_ints(int rows) {
  const size_t np = (size_t)cdiv(rows, 128) * 128;
  return 2 * np + np / 8;
}

size_t mggan_block_attention_fwd_workspace(int rows, int keys, int heads, int kv_heads, int width, int scenes) {
  BlkAttnArgs p = {};
  p.N = rows, p.M = keys, p.H = heads, p.Hkv = kv_heads, p.D = width, p.S = scenes;
  return rows > 0 && keys > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && width > 0 && scenes > 0 ? fwd_workspace(p) : 0;
}

int mggan_block_attention_fwd(const void* args, hipStream_t stream) {
  const BlkAttnArgs* a = (const BlkAttnArgs*)args;
  const int rc = blk_attn_check(a, "block_attention_fwd");
  if (rc != MGGAN_OK) return rc;
  MG_CHECK_ARG(a->out && ((size_t)a->out | (size_t)a->out32 | (size_t)a->spans) % 16 == 0, "block_attention_fwd: output or spans null or unaligned");
  const size_t need = fwd_workspace(*a);
  MG_CHECK_ARG(!need || (a->ws && (size_t)a->ws_bytes >= need), "block_attention_fwd: workspace of %zu bytes (got %ld)", need, a->ws_bytes);
  if (a->dtype == BLK_BF16)
    launch_fwd_width<bf16>(*a, stream);
  else
    launch_fwd_width<float>(*a, stream);
  MG_LAUNCH_CHECK("block_attention_fwd");
  return MGGAN_OK;
}
}
