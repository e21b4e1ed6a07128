// Shared pieces of the attention kernels (blk_attn.hip: forward, blk_attn_bwd.hip: backward).
//
//   out_i = sum_j P_ij v_j,   P_i = softmax over the keys j that row i sees of   cap tanh(scale q_i.k_j / cap) - slope_h |xy_i - kv_xy_j|
//
// Which keys a row sees is one interval [lo_i, hi_i): those of its scene, cut off behind the row's own place (causal) or behind the
// prefix.  blk_spans_kernel writes the intervals, every kernel compares indices with them: documents, prefixes and padding are one test.
//
// All products run transposed on the matrix cores.  The side that owns the result (queries, or keys in the dK / dV kernel) lies in
// registers as the second operand, one row per lane; the other side streams through LDS in tiles of BK rows.  S^T = K Q^T leaves
// lane 16 g + i with row i's scores of keys 32 p + 8 g + {0..7} (the rows of K are read in that order: a product may number its
// result rows as it likes) -- which is how the next product wants its second operand: P never leaves the registers.
#pragma once
#include "blk.h"

struct BlkAttnArgs {  // mirrored by mggan/hip/blocks.py
  const void *q, *k, *v, *dout;
  void *out, *dq, *dk, *dv;
  float* dslopes;
  const int *scenes, *kv_scenes, *prefix;
  const float *xy, *kv_xy, *slopes;
  float* lse;    // (2, H, N): the row's largest score (as the exponent takes it) and one over its sum of exp(score - largest)
  float* out32;  // the output before it is rounded (f32: the output): what sum(dO O) is formed of -- from the rounded one every row's
                 // gradient would carry a common error, which the sums over rows (the slopes' gradient) do not average away
  int* spans;   // mggan_block_attention_span_ints(N): lo, hi, and {min lo, max hi, max lo, min hi} of every 32 rows
  void* ws;
  long ws_bytes;
  long q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  int N, M, H, Hkv, D, S, causal, axes, dtype;
  float scale, cap;
};

namespace {

__device__ __attribute__((aligned(16))) const unsigned blk_attn_zeros[4] = {0, 0, 0, 0};

constexpr float LOG2E = 1.44269504f;

// tanh.  f32 operands: near zero by its series (to x^11: 2^-26 of the value at 0.35), so that a score keeps its relative precision
// through the cap; bf16 operands carry 2^-9 themselves, there the quotient does everywhere.
template <class T>
__device__ __forceinline__ float blk_tanh(float x) {
  const float big = fmaf(-2.0f, mg_rcp(__builtin_amdgcn_exp2f(x * (2.f * LOG2E)) + 1.0f), 1.0f);
  if constexpr (sizeof(T) == 2) return big;
  const float y = x * x;
  const float s = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -0.0088632355f, 0.0218694885f), -0.0539682540f), 0.1333333333f), -0.3333333333f), 1.f) * x;
  return fabsf(x) < 0.35f ? s : big;
}

// What is done to a score q.k, by the kernels' template argument X: bit 0 a cap, bits 1-2 the axes of the distance.
// Scores are exponentiated as exp2((s - max) log2e) where their last bits matter (f32; scores with a distance, whose slopes' gradient is
// f32): log2e rounded into the scores first would stretch all of them by a common 2^-25, which shows in the slopes' gradient.  The others
// (bf16, gradients rounded at 2^-9) are kept times log2e and take exp2(s - max), an operation less.
template <class T, int X>
struct Soft {
  static constexpr bool CAP = X & 1, NATURAL = (X >> 1) || sizeof(T) == 4;
  static constexpr int AXES = X >> 1;
  float c, k, cap, slope;  // c: a plain score's factor
  __device__ __forceinline__ Soft(const BlkAttnArgs& p, float slope_) {
    c = p.scale * (NATURAL ? 1.f : LOG2E);
    cap = p.cap * (NATURAL ? 1.f : LOG2E);
    k = CAP ? p.scale / p.cap : 0.f;
    slope = slope_;
  }
  // the score as it is exponentiated; fac = d(capped)/d(score), dist: what the slope multiplies
  __device__ __forceinline__ float score(float x, float ax, float ay, float bx, float by, float& fac, float& dist) const {
    fac = 1.f, dist = 0.f;
    if constexpr (CAP) {
      const float t = blk_tanh<T>(x * k);
      fac = fmaf(-t, t, 1.f);
      x = cap * t;
    } else {
      x *= c;
    }
    if constexpr (AXES == 1) dist = fabsf(ax - bx);
    if constexpr (AXES == 2) {
      const float dx = ax - bx, dy = ay - by;
      dist = __builtin_amdgcn_sqrtf(fmaf(dx, dx, dy * dy));
    }
    if constexpr (AXES) x = fmaf(-slope, dist, x);
    return x;
  }
  // whether scores are left as the product gives them and weight() multiplies (one operation for both)
  static constexpr bool RAW = X == 0 && !NATURAL;
  __device__ __forceinline__ float weight(float s, float top) const {
    if (RAW) return __builtin_amdgcn_exp2f(fmaf(s, c, -top));
    return __builtin_amdgcn_exp2f(NATURAL ? (s - top) * LOG2E : s - top);
  }
  // exp(a - b) of two maxima
  static __device__ __forceinline__ float ratio(float a, float b) { return __builtin_amdgcn_exp2f(NATURAL ? (a - b) * LOG2E : a - b); }
};

template <class T_, int DP_, int BK_ = 128 / (int)sizeof(T_)>
struct Geo {
  using T = T_;
  static constexpr int DP = DP_, CH = Mf<T>::CH;
  static constexpr int NCH = DP / CH;          // 16-byte chunks of a row
  static constexpr int SK = NCH / 4;           // steps of a product over the width
  static constexpr int BK = BK_;               // streamed rows of a tile: 64 bf16, 32 f32
  static constexpr int F = BK / 16;            // their 16-row fragments
  static constexpr int DF = DP / 16;           // 16-column fragments of the width
  static constexpr int TILE = BK * NCH;        // chunks of a tile
  // the streamed row that fragment f's row i is, and the row of a lane's r-th value (r, g -> i = 4 g + r)
  static __device__ __forceinline__ int row_of(int f, int i) {
    return sizeof(T) == 2 ? 32 * (f >> 1) + 8 * (i >> 2) + 4 * (f & 1) + (i & 3) : 16 * f + i;
  }
  static __device__ __forceinline__ int row4(int f, int g) { return sizeof(T) == 2 ? 32 * (f >> 1) + 8 * g + 4 * (f & 1) : 16 * f + 4 * g; }
  // Place of a chunk in its row.  Row reads take one chunk of 16 rows ({0-3, 8-11, ..} (+4) with bf16, 0-15 with f32): any eight lanes meet
  // eight bank groups.  The transposing reads of bf16 take two chunks of rows 8 g + {0..3}: eight bank groups again.  Neither depends on which
  // fragment it is, so a lane's addresses are a few bases plus constants (Lane).
  static __device__ __forceinline__ int swz(int r) {
    if (sizeof(T) == 4) return (r & 7) ^ ((r >> 1) & 4);
    return NCH % 8 == 0 ? (r & 3) << 1 | ((r >> 3) & 1) : (r & 2) | ((r >> 3) & 1);
  }
};

// Byte offsets of a lane's reads in a tile.
template <class G>
struct Lane {
  static constexpr int ROW = G::NCH * 16;
  static constexpr bool WIDE = G::NCH % 8 == 0;
  int row[2];  // of a row's chunk 4 s + g, by s & 1
  int col[8];  // of the transposed reads: bf16 by column fragment, f32 by r + 4 (column fragment & 1)
  __device__ __forceinline__ void init(int lane) {
    const int i16 = lane & 15, g = lane >> 4, r = G::row_of(0, i16);
#pragma unroll
    for (int k = 0; k < 2; ++k) row[k] = r * ROW + (WIDE ? ((4 * k + g) ^ G::swz(r)) & 7 : g ^ G::swz(r)) * 16;
    if (sizeof(typename G::T) == 2) {
      const int k = 8 * g + (i16 >> 2);
#pragma unroll
      for (int f = 0; f < 4; ++f)
        col[f] = k * ROW + 8 * (i16 & 1) + (WIDE ? ((2 * f + ((i16 & 3) >> 1)) ^ G::swz(k)) & 7 : ((2 * (f & 1) + ((i16 & 3) >> 1)) ^ G::swz(k)) & 3) * 16;
    } else {
#pragma unroll
      for (int f = 0; f < 8; ++f) {
        const int k = 4 * g + (f & 3);
        col[f] = k * ROW + 4 * (i16 & 3) + (((4 * (f >> 2) + (i16 >> 2)) ^ G::swz(k)) & 7) * 16;
      }
    }
  }
  // fragment f's rows, chunk 4 s + g: first operand of a product over the width
  __device__ __forceinline__ u32x4 rows(const char* tile, int f, int s) const {
    const int at = sizeof(typename G::T) == 2 ? (32 * (f >> 1) + 4 * (f & 1)) * ROW : 16 * f * ROW;
    return *(const u32x4*)(tile + row[WIDE ? s & 1 : 0] + at + (WIDE ? (s >> 1) * 128 : s * 64));
  }
  // bf16: columns 16 fd + i of rows 32 p + 8 g + {0..7}, transposed: first operand of a product over the tile's rows
  __device__ __forceinline__ bf16x8 cols(const char* tile, int p, int fd) const {
    const char* a = tile + col[WIDE ? fd & 3 : fd & 1] + 32 * p * ROW + (WIDE ? (fd >> 2) * 128 : (fd >> 1) * 64);
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MG_LDS s16x4*)a);
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MG_LDS s16x4*)(a + 4 * ROW));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // f32: column 16 fd + i of row 16 f + 4 g + r
  __device__ __forceinline__ float col1(const char* tile, int f, int r, int fd) const {
    return *(const float*)(tile + col[r + 4 * (fd & 1)] + 16 * f * ROW + (fd >> 1) * 128);
  }
};

// Rows [first, first + BK) of a (rows, heads, D) operand into LDS; rows outside [lo, hi) and columns from D on as zeros.
// The workgroup's (threads = 256) or one wave's (64) work.
template <class G, int threads = 256>
__device__ __forceinline__ void copy_tile(const typename G::T* base, long row_stride, int first, int lo, int hi, int nd, u32x4* lds) {
  const int wave = threads == 64 ? 0 : mg_wave();
#pragma unroll
  for (int i = 0; i < G::TILE / threads; ++i) {
    const int slot = i * threads + (threads == 64 ? mg_lane() : (int)threadIdx.x), row = slot / G::NCH, c = (slot % G::NCH) ^ G::swz(row), at = first + row;
    const bool in = at >= lo && at < hi && c < nd;
    const char* src = (const char*)(base + (long)at * row_stride) + c * 16;
    lds_copy16(in ? src : (const char*)blk_attn_zeros, lds + i * threads + wave * 64);
  }
}
// 4 bytes of each of 64 rows: element `at` of row `first + lane` of rows of `stride` (rows clamped to [0, n)).
__device__ __forceinline__ void copy_meta(const void* base, long stride, long at, int first, int n, void* lds) {
  const int r = first + mg_lane(), row = r < 0 ? 0 : r < n ? r : n - 1;
  __builtin_amdgcn_global_load_lds((MG_GLB const void*)((const char*)base + 4 * (row * stride + at)), (MG_LDS void*)lds, 4, 0, 0);
}

// The chunk of an owner row that a lane holds as second operand; zeros outside.
template <class T>
__device__ __forceinline__ u32x4 owner_chunk(const T* row, int c, int nd) {
  if (c < nd) return *(const u32x4*)((const char*)row + c * 16);
  return u32x4{0, 0, 0, 0};
}

// D fragments of scores: sum over the width of streamed rows x owner rows.
template <class G, int QF>
__device__ __forceinline__ void scores(const void* tile, const u32x4 (&own)[QF][G::SK], f32x4 (&out)[QF][G::F], const Lane<G>& at) {
#pragma unroll
  for (int f = 0; f < G::F; ++f) {
#pragma unroll
    for (int j = 0; j < QF; ++j) out[j][f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < G::SK; ++s) {
      const u32x4 a = at.rows((const char*)tile, f, s);
#pragma unroll
      for (int j = 0; j < QF; ++j) out[j][f] = Mf<typename G::T>::step(a, own[j][s], out[j][f]);
    }
  }
}

// acc[d][owner row] += sum over streamed rows of tile[row][d] * coef[row][owner row], the tile read transposed.  Column fragment fd's row
// i is column 16 fd + i: a lane ends up with columns 16 fd + 4 g + {0..3} of its owner row.
template <class G, int QF>
__device__ __forceinline__ void accumulate(const void* tile, const f32x4 (&coef)[QF][G::F], f32x4 (&acc)[QF][G::DF], const Lane<G>& at) {
  if constexpr (sizeof(typename G::T) == 2) {
#pragma unroll
    for (int p = 0; p < G::F / 2; ++p) {
      bf16x8 b[QF];
#pragma unroll
      for (int j = 0; j < QF; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) b[j][r] = (bf16)coef[j][2 * p][r], b[j][4 + r] = (bf16)coef[j][2 * p + 1][r];
#pragma unroll
      for (int fd = 0; fd < G::DF; ++fd) {
        const bf16x8 a = at.cols((const char*)tile, p, fd);
#pragma unroll
        for (int j = 0; j < QF; ++j) acc[j][fd] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[j], acc[j][fd], 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int f = 0; f < G::F; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int fd = 0; fd < G::DF; ++fd) {
          const float a = at.col1((const char*)tile, f, r, fd);
#pragma unroll
          for (int j = 0; j < QF; ++j) acc[j][fd] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, coef[j][f][r], acc[j][fd], 0, 0, 0);
        }
  }
}

// Whether any value of the tile is infinite or not a number (a masked place's zero coefficient would turn it into one).
template <class G>
__device__ __forceinline__ bool tile_not_finite(const u32x4* tile, int lane) {
  bool bad = false;
  for (int i = lane; i < G::TILE; i += 64) {
    const u32x4 v = tile[i];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (sizeof(typename G::T) == 2)
        bad |= (v[w] & 0x7f80u) == 0x7f80u || (v[w] & 0x7f800000u) == 0x7f800000u;
      else
        bad |= (v[w] & 0x7f800000u) == 0x7f800000u;
    }
  }
  return __ballot(bad) != 0;
}
// accumulate() row by row over the places that `sees` only: the way of tiles that are partly masked AND hold such a value.
template <class G, int QF, class See>
__device__ __forceinline__ void accumulate_seen(const u32x4* tile, const f32x4 (&coef)[QF][G::F], f32x4 (&acc)[QF][G::DF], int lane, See sees) {
  using T = typename G::T;
  const int i16 = lane & 15, g = lane >> 4;
  for (int row = 0; row < G::BK; ++row) {
    int f, gg, r = row & 3;
    if (sizeof(T) == 2)
      f = 2 * (row >> 5) + ((row >> 2) & 1), gg = (row >> 3) & 3;
    else
      f = row >> 4, gg = (row >> 2) & 3;
    const T* t = (const T*)(tile + row * G::NCH);
    const int sw = G::swz(row);
#pragma unroll
    for (int j = 0; j < QF; ++j) {
      float c = 0.f;
#pragma unroll
      for (int a = 0; a < G::F; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) c = a == f && b == r ? coef[j][a][b] : c;
      c = __shfl(c, i16 + 16 * gg, 64);
      if (!sees(j, row)) continue;
#pragma unroll
      for (int fd = 0; fd < G::DF; ++fd)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = 16 * fd + 4 * g + e;
          acc[j][fd][e] = fmaf(c, (float)t[((d / G::CH) ^ sw) * G::CH + d % G::CH], acc[j][fd][e]);
        }
    }
  }
}

// Four neighbouring columns of an owner row, scaled.
template <class T>
__device__ __forceinline__ void store4(T* p, const f32x4& a, float scale) {
  if constexpr (sizeof(T) == 2) {
    bf16x4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = (bf16)(a[r] * scale);
    *(bf16x4*)p = x;
  } else {
    *(f32x4*)p = a * scale;
  }
}

}  // namespace
