// Attention over the rows of scenes, forward: intervals of visible keys, one pass over the keys with running maximum and sum.
#include <limits.h>
#include "blk_attn.h"
#include "../../include/mggan_hip.h"

namespace {

// The interval of keys that each of 64 rows sees, and what every 32 rows have in common.  All scenes are looked through (in any
// order; the last one that names a row counts), so that nothing is asked of a list in device memory; what it says is clamped to the
// operands' rows.
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
  int lo = 0, hi = 0;
  if (s >= 0) {
    const int q0 = max(p.scenes[2 * s], 0), q1 = min(p.scenes[2 * s + 1], p.N);
    const int k0 = min(max(p.kv_scenes[2 * s], 0), p.M), k1 = min(max(p.kv_scenes[2 * s + 1], k0), p.M);
    int n = k1 - k0;
    if (p.causal) {
      const int pre = p.prefix ? p.prefix[s] : 0;
      n = max(0, min(n, max(pre, r0 + tid - q0 + 1 + n - (q1 - q0))));
    }
    if (n > 0) lo = k0, hi = k0 + n;
  }
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

// A workgroup: 64 QF query rows of one head, four waves of 16 QF rows each; keys and values in tiles of BK rows, two buffers.
template <class T, int DP, int QF, bool EXTRA>
__global__ __launch_bounds__(256) void blk_attn_fwd_kernel(BlkAttnArgs p, int np) {
  using G = Geo<T, DP>;
  __shared__ u32x4 lk[2][G::TILE], lv[2][G::TILE];
  __shared__ float lx[2][2][64];
  const int lane = mg_lane(), wave = mg_wave(), i16 = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % p.H, hk = h / (p.H / p.Hkv);
  const int qt = gridDim.x / p.H - 1 - (int)(blockIdx.x / p.H);  // the rows at the end first: behind a causal mask they see the most
  const int r0 = qt * 64 * QF, w0 = r0 + wave * 16 * QF;
  const int nd = p.D / G::CH;

  // what the workgroup's rows and this wave's rows see
  int glo = INT_MAX, ghi = 0;
#pragma unroll
  for (int i = 0; i < 2 * QF; ++i) {
    const int4 s = *(const int4*)(p.spans + 2 * np + 4 * ((r0 >> 5) + i));
    glo = min(glo, s.x);
    ghi = max(ghi, s.y);
  }
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
    if (EXTRA && p.axes) {
      qx[j] = p.xy[(long)rc * p.axes];
      qy[j] = p.axes > 1 ? p.xy[(long)rc * p.axes + 1] : 0.f;
    }
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
    copy_tile<T, DP>(kb, p.k_row, k0, glo, ghi, nd, lk[buf]);
    copy_tile<T, DP>(vb, p.v_row, k0, glo, ghi, nd, lv[buf]);
    if (EXTRA && wave < p.axes) copy_meta(p.kv_xy, p.axes, wave, k0, p.M, lx[buf][wave]);
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
  const float c2 = p.scale * LOG2E, slope2 = EXTRA && p.axes ? p.slopes[h] * LOG2E : 0.f, icap = EXTRA && p.cap > 0.f ? p.scale / p.cap : 0.f;

  if (glo < ghi) fetch(glo, 0);
  int buf = 0;
  for (int k0 = glo; k0 < ghi; k0 += G::BK, buf ^= 1) {
    __syncthreads();
    if (k0 + G::BK < ghi) fetch(k0 + G::BK, buf ^ 1);
    if (k0 >= whi || k0 + G::BK <= wlo) continue;  // (the wave's: nothing of this tile is seen)
    f32x4 s[QF][G::F];
    scores<T, DP, QF>(lk[buf], q, s, lane);
    const bool part = k0 < flo || k0 + G::BK > fhi;
    if (EXTRA) {
#pragma unroll
      for (int f = 0; f < G::F; ++f) {
        const int kr = G::row4(f, g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float bx = p.axes ? lx[buf][0][kr + r] : 0.f, by = p.axes > 1 ? lx[buf][1][kr + r] : 0.f;
#pragma unroll
          for (int j = 0; j < QF; ++j) {
            float x = s[j][f][r];
            x = p.cap > 0.f ? p.cap * LOG2E * blk_tanh<T>(x * icap) : x * c2;
            if (p.axes) x = fmaf(-slope2, blk_dist(p.axes, qx[j], qy[j], bx, by), x);
            s[j][f][r] = x;
          }
        }
      }
    }
    const float cs = EXTRA ? 1.f : c2;
    if (part) {
#pragma unroll
      for (int f = 0; f < G::F; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = k0 + G::row4(f, g) + r;
#pragma unroll
          for (int j = 0; j < QF; ++j) s[j][f][r] = key >= lo[j] && key < hi[j] ? s[j][f][r] : -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < QF; ++j) {
      float t = -INFINITY;
#pragma unroll
      for (int f = 0; f < G::F; ++f) t = fmaxf(t, fmaxf(fmaxf(s[j][f][0], s[j][f][1]), fmaxf(s[j][f][2], s[j][f][3])));
      t = quarters_max(t) * cs;
      if (__ballot(t > m[j])) {
        const float mn = fmaxf(m[j], t), al = __builtin_amdgcn_exp2f(mn == -INFINITY ? 0.f : m[j] - mn);
        m[j] = mn;
        l[j] *= al;
#pragma unroll
        for (int d = 0; d < G::DF; ++d) acc[j][d] *= al;
      }
      const float mm = m[j] == -INFINITY ? 0.f : m[j];
      float sum = 0.f;
#pragma unroll
      for (int f = 0; f < G::F; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[j][f][r], cs, -mm));
          s[j][f][r] = e;
          sum += e;
        }
      l[j] += sum;
    }
    if (part && tile_not_finite<T, DP>(lv[buf], lane))
      accumulate_seen<T, DP, QF>(lv[buf], s, acc, lane, [&](int j, int row) { return k0 + row >= lo[j] && k0 + row < hi[j]; });
    else
      accumulate<T, DP, QF>(lv[buf], s, acc, lane);
  }

#pragma unroll
  for (int j = 0; j < QF; ++j) {
    const int r = w0 + 16 * j + i16;
    const float sum = quarters_sum(l[j]), inv = hi[j] > lo[j] ? 1.f / sum : 0.f;
    if (r >= p.N) continue;
    if (g == 0 && p.lse) p.lse[(long)h * p.N + r] = m[j] + __log2f(sum);
    T* out = (T*)p.out + ((long)r * p.H + h) * p.D;
#pragma unroll
    for (int d = 0; d < G::DF; d += 2)
      if (16 * d + 8 * g < p.D) store_pair<T>(out + 16 * d + 8 * g, acc[j][d], acc[j][d + 1], inv);
  }
}

template <class T, int DP>
void launch_fwd(const BlkAttnArgs& p, hipStream_t st) {
  const int np = cdiv(p.N, 128) * 128;
  const bool extra = p.cap > 0.f || p.axes > 0;
  const bool wide = (long)cdiv(p.N, 128) * p.H >= 256;  // enough workgroups of 128 rows to fill the chip
  const dim3 grid(cdiv(p.N, wide ? 128 : 64) * p.H);
  if (wide) {
    if (extra)
      MG_LAUNCH((blk_attn_fwd_kernel<T, DP, 2, true>), grid, dim3(256), 0, st, p, np);
    else
      MG_LAUNCH((blk_attn_fwd_kernel<T, DP, 2, false>), grid, dim3(256), 0, st, p, np);
  } else {
    if (extra)
      MG_LAUNCH((blk_attn_fwd_kernel<T, DP, 1, true>), grid, dim3(256), 0, st, p, np);
    else
      MG_LAUNCH((blk_attn_fwd_kernel<T, DP, 1, false>), grid, dim3(256), 0, st, p, np);
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

}  // namespace

int blk_attn_check(const BlkAttnArgs* a, const char* name) {
  MG_CHECK_ARG(a, "%s: no arguments", name);
  const BlkAttnArgs& p = *a;
  MG_CHECK_ARG(p.dtype == BLK_F32 || p.dtype == BLK_BF16, "%s: dtype %d (0 = f32, 1 = bf16)", name, p.dtype);
  MG_CHECK_ARG(p.N > 0 && p.M > 0 && p.N <= (1 << 24) && p.M <= (1 << 30), "%s: %d rows, %d keys", name, p.N, p.M);
  MG_CHECK_ARG(p.H > 0 && p.Hkv > 0 && p.H % p.Hkv == 0 && p.H <= 1024, "%s: %d heads over %d key heads", name, p.H, p.Hkv);
  MG_CHECK_ARG(p.D > 0 && p.D <= 128 && p.D % 8 == 0, "%s: width %d (a multiple of 8 up to 128)", name, p.D);
  MG_CHECK_ARG(p.S >= 0 && p.axes >= 0 && p.axes <= 2 && p.scale > 0.f && p.cap >= 0.f, "%s: %d scenes, %d axes, scale %g, cap %g", name, p.S,
               p.axes, p.scale, p.cap);
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

int mggan_block_attention_fwd(const void* args, hipStream_t stream) {
  const BlkAttnArgs* a = (const BlkAttnArgs*)args;
  const int rc = blk_attn_check(a, "block_attention_fwd");
  if (rc != MGGAN_OK) return rc;
  MG_CHECK_ARG(a->out && (size_t)a->out % 16 == 0 && (size_t)a->spans % 16 == 0, "block_attention_fwd: output or spans null or unaligned");
  const int np = cdiv(a->N, 128) * 128;
  MG_LAUNCH(blk_spans_kernel, dim3(np / 64), dim3(256), 0, stream, *a, np);
  if (a->dtype == BLK_BF16)
    launch_fwd_width<bf16>(*a, stream);
  else
    launch_fwd_width<float>(*a, stream);
  MG_LAUNCH_CHECK("block_attention_fwd");
  return MGGAN_OK;
}
}
