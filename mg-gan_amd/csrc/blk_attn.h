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
  float* lse;    // (3, H, N): what the exponents of a row's weights were taken less (about the largest), one over the weights' sum, and both in
                 // one (the exponent less this is the log2 of the softmax: exact to 2^-21 or so, which is enough where bf16 follows)
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

// tanh(x) from z = 2 log2e x.  The quotient is off by up to 12 steps of 2^-24 however small x is, and the cap multiplies that.  SERIES: near
// zero by the series instead (to x^11: 2^-26 of the value at 0.35), so that a score keeps its relative precision through any cap.
template <bool SERIES>
__device__ __forceinline__ float blk_tanh(float z) {
  const float big = fmaf(-2.0f, mg_rcp(__builtin_amdgcn_exp2f(z) + 1.0f), 1.0f);
  if constexpr (!SERIES) return big;
  const float x = z * (0.5f / LOG2E), y = x * x;
  const float s = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -0.0088632355f, 0.0218694885f), -0.0539682540f), 0.1333333333f), -0.3333333333f), 1.f) * x;
  return fabsf(x) < 0.35f ? s : big;
}

// What is done to a score q.k, by the kernels' template argument X: bit 0 a cap, bits 1-2 the axes of the distance, bit 3 (bf16 with a cap
// above SERIES_FROM; f32 does so always) the cap's tanh by its series near zero.  bf16 up to there takes the quotient alone: 64 times its 12 F
// are 2^-14.4 of a weight, which is rounded to 2^-8 of itself anyway, and the series would be seven instructions more a score.
// Weights are exp2(s E - top), one fused operation, with top = max s E.  E = log2e over scores in their own units where the last bits
// matter (f32; scores with a distance, whose slopes' gradient is f32): scale log2e and slope log2e rounded into one factor first would
// stretch all scores by a common 2^-25, which shows in the slopes' gradient (log2e itself is 2^-26 off, top's rounding divides out).
// bf16, with gradients rounded at 2^-9: plain scores are left as the product gives them and E = scale log2e, capped ones as their tanh and
// E = cap log2e.
template <class T, int X>
struct Soft {
  static constexpr int AXES = (X >> 1) & 3;
  static constexpr bool CAP = X & 1, SERIES = (X & 8) || sizeof(T) == 4, NATURAL = AXES || sizeof(T) == 4;
  static constexpr bool RAW = X == 0 && !NATURAL;  // score() is not called
  float scale, k, cap, slope, E;
  __device__ __forceinline__ Soft(const BlkAttnArgs& p, float slope_) {
    scale = p.scale;
    cap = p.cap;
    k = CAP ? p.scale / p.cap * (2.f * LOG2E) : 0.f;
    slope = slope_;
    E = LOG2E * (NATURAL ? 1.f : CAP ? p.cap : p.scale);
  }
  // the score as weight() takes it; fac = d(capped)/d(score), dist: what the slope multiplies
  __device__ __forceinline__ float score(float x, float ax, float ay, float bx, float by, float& fac, float& dist) const {
    fac = 1.f, dist = 0.f;
    if constexpr (CAP) {
      x = blk_tanh<SERIES>(x * k);
      fac = fmaf(-x, x, 1.f);
      if (NATURAL) x *= cap;
    } else {
      x *= scale;
    }
    if constexpr (AXES == 1) dist = fabsf(ax - bx);
    if constexpr (AXES == 2) {
      const float dx = ax - bx, dy = ay - by;
      dist = __builtin_amdgcn_sqrtf(fmaf(dx, dx, dy * dy));
    }
    if constexpr (AXES) x = fmaf(-slope, dist, x);
    return x;
  }
  __device__ __forceinline__ float weight(float s, float top) const { return __builtin_amdgcn_exp2f(fmaf(s, E, -top)); }
};

constexpr float SERIES_FROM = 64.f;
template <class T>
int blk_attn_x(const BlkAttnArgs& p) {
  return (p.cap > 0.f ? 1 : 0) + 2 * p.axes + (sizeof(T) == 2 && p.cap > SERIES_FROM ? 8 : 0);
}

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
  // eight groups of four banks.  The transposing reads of bf16 take two chunks of rows 8 g + {0..3}: eight groups again.  Neither depends on which
  // fragment it is, so a lane's addresses are a few bases plus constants (Lane).  Eight groups are 128 of the 256 bytes that LDS serves in a
  // cycle, so the reads are not free of conflicts: 1.9 to 2.5 cycles of them an LDS instruction (counters, widths 64 and 128).
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
    const s16x4 x = lds_transposed(a);
    const s16x4 y = lds_transposed(a + 4 * ROW);
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
  static_assert(G::TILE % threads == 0, "a tile is copied in whole passes");
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

// D fragments of scores: sum over the width of streamed rows x owner rows.  The reads of a fragment's rows are issued before the
// multiplications of the one before (and no earlier: left to itself the compiler reads everything ahead and runs out of registers).
template <class G, int QF>
__device__ __forceinline__ void scores(const void* tile, const u32x4 (&own)[QF][G::SK], f32x4 (&out)[QF][G::F], const Lane<G>& at) {
  u32x4 a[2][G::SK];
#pragma unroll
  for (int s = 0; s < G::SK; ++s) a[0][s] = at.rows((const char*)tile, 0, s);
#pragma unroll
  for (int f = 0; f < G::F; ++f) {
    if (f + 1 < G::F) {
#pragma unroll
      for (int s = 0; s < G::SK; ++s) a[(f + 1) & 1][s] = at.rows((const char*)tile, f + 1, s);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < QF; ++j) out[j][f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < G::SK; ++s)
#pragma unroll
      for (int j = 0; j < QF; ++j) out[j][f] = Mf<typename G::T>::step(a[f & 1][s], own[j][s], out[j][f]);
  }
}

// Both score-like products of a fragment's streamed rows (Q K and dO V) for one group of 16 owner rows.
template <class G>
__device__ __forceinline__ void scores2(const void* ta, const void* tb, const u32x4 (&a)[G::SK], const u32x4 (&b)[G::SK], int f, f32x4& x, f32x4& y,
                                        const Lane<G>& at) {
  x = y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < G::SK; ++s) {
    const u32x4 ra = at.rows((const char*)ta, f, s), rb = at.rows((const char*)tb, f, s);
    x = Mf<typename G::T>::step(ra, a[s], x);
    y = Mf<typename G::T>::step(rb, b[s], y);
  }
}

// Four weights or score gradients of a lane as the next product takes them.  bf16 operands: rounded to bf16 here, once -- the matrix
// instructions take both operands in one type, so P V, P^T dO, dS K and dS^T Q carry half a step of P or dS (2^-8) beside that of their other operand.
// Against 64 bits that makes 0.0023 to 0.0024 of outputs and gradients that are 0.0017 off with P and dS in f32 (the final rounding alone); P as the
// sum of two bf16 numbers would take each of these products twice.
template <class T>
struct Coef {
  f32x4 v;
  __device__ __forceinline__ void set(const f32x4& x) { v = x; }
};
template <>
struct Coef<bf16> {
  bf16x4 v;
  __device__ __forceinline__ void set(const f32x4& x) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (bf16)x[r];
  }
};

// acc[d][owner row] += sum over streamed rows of tile[row][d] * coef[row][owner row], the tile read transposed.  Column fragment fd's row
// i is column 16 fd + i: a lane ends up with columns 16 fd + 4 g + {0..3} of its owner row.
template <class G, int QF>
__device__ __forceinline__ void accumulate(const void* tile, const Coef<typename G::T> (&coef)[QF][G::F], f32x4 (&acc)[QF][G::DF], const Lane<G>& at) {
  if constexpr (sizeof(typename G::T) == 2) {
    constexpr int C = 2;  // column fragments read together
#pragma unroll
    for (int p = 0; p < G::F / 2; ++p) {
      bf16x8 a[2][C], b[QF];
#pragma unroll
      for (int c = 0; c < C; ++c) a[0][c] = at.cols((const char*)tile, p, c);
#pragma unroll
      for (int j = 0; j < QF; ++j) b[j] = __builtin_shufflevector(coef[j][2 * p].v, coef[j][2 * p + 1].v, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int k = 0; k < G::DF / C; ++k) {
        if (k + 1 < G::DF / C) {
#pragma unroll
          for (int c = 0; c < C; ++c) a[(k + 1) & 1][c] = at.cols((const char*)tile, p, (k + 1) * C + c);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < QF; ++j)
            acc[j][k * C + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[k & 1][c], b[j], acc[j][k * C + c], 0, 0, 0);
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
          for (int j = 0; j < QF; ++j) acc[j][fd] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, coef[j][f].v[r], acc[j][fd], 0, 0, 0);
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
// accumulate() for a tile that is partly masked AND holds such values: they are taken as zeros, and where a row sees some the sum becomes the
// infinity or the NaN that it would have been, by two more products: of ones where they are with ones where the row sees (how many terms are not
// finite) and of their signs with the coefficients' signs (how many are +inf less how many -inf; a NaN and a coefficient of zero count nothing, so
// a term that is a NaN, as zero times infinity is, leaves the two apart; an infinite coefficient that meets one gives a NaN).  It is in a second copy of the kernels' loops (SAFE) that a workgroup
// runs, from the start, only if its first run came upon such a tile: beside the plain way in one loop it would cost every run 40 to 100 registers.
// (One product after the other: their operands together would cost the plain run's waves theirs, width 64 with a cap 342 -> 350 us.)
__device__ __forceinline__ float sign_of(float x) { return x > 0.f ? 1.f : x < 0.f ? -1.f : 0.f; }
template <class G, int QF, class See>
__device__ __forceinline__ void accumulate_seen(const void* tile, const Coef<typename G::T> (&coef)[QF][G::F], f32x4 (&acc)[QF][G::DF], const Lane<G>& at, int lane,
                                                See sees) {
  constexpr bool HALF = sizeof(typename G::T) == 2;
  const int g = lane >> 4;
#pragma unroll
  for (int fd = 0; fd < G::DF; ++fd) {
    f32x4 many[QF] = {}, sign[QF] = {};
#pragma unroll
    for (int p = 0; p < (HALF ? G::F / 2 : G::F * 4); ++p) {
      if constexpr (HALF) {
        const bf16x8 a = at.cols((const char*)tile, p, fd);
        auto product = [&](f32x4(&to)[QF], auto left, auto right) {
          bf16x8 x, y;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = (bf16)left((float)a[e], !(fabsf((float)a[e]) < INFINITY));
#pragma unroll
          for (int j = 0; j < QF; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = (bf16)right(j, (float)coef[j][2 * p + (e >> 2)].v[e & 3], 32 * p + 8 * g + e);
            to[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, to[j], 0, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        };
        f32x4 t[QF];
#pragma unroll
        for (int j = 0; j < QF; ++j) t[j] = acc[j][fd];
        product(t, [](float x, bool odd) { return odd ? 0.f : x; }, [](int, float c, int) { return c; });
#pragma unroll
        for (int j = 0; j < QF; ++j) acc[j][fd] = t[j];
        product(many, [](float, bool odd) { return odd ? 1.f : 0.f; }, [&](int j, float, int row) { return sees(j, row) ? 1.f : 0.f; });
        product(sign, [](float x, bool odd) { return odd ? sign_of(x) : 0.f; }, [&](int j, float c, int row) { return sees(j, row) ? sign_of(c) : 0.f; });
      } else {
        const float x = at.col1((const char*)tile, p >> 2, p & 3, fd);
        const bool odd = !(fabsf(x) < INFINITY);
#pragma unroll
        for (int j = 0; j < QF; ++j) {
          const float c = coef[j][p >> 2].v[p & 3];
          const bool seen = sees(j, 16 * (p >> 2) + 4 * g + (p & 3));
          acc[j][fd] = __builtin_amdgcn_mfma_f32_16x16x4f32(odd ? 0.f : x, c, acc[j][fd], 0, 0, 0);
          many[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(odd ? 1.f : 0.f, seen ? 1.f : 0.f, many[j], 0, 0, 0);
          sign[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(odd ? sign_of(x) : 0.f, seen ? sign_of(c) : 0.f, sign[j], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < QF; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (many[j][e] > 0.f) acc[j][fd][e] += many[j][e] == sign[j][e] ? INFINITY : many[j][e] == -sign[j][e] ? -INFINITY : NAN;
    __builtin_amdgcn_sched_barrier(0);
  }
}

// What 32 n rows from row r0 on see between them: the first and the end of it.
template <int n>
__device__ __forceinline__ int2 group_span(const BlkAttnArgs& p, int np, int r0) {
  int lo = 0x7fffffff, hi = 0;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const int4 s = *(const int4*)(p.spans + 2 * np + 4 * ((r0 >> 5) + i));
    lo = min(lo, s.x);
    hi = max(hi, s.y);
  }
  return make_int2(lo, hi);
}
// From the 16 lanes' own: the first and the end of what any row of the wave sees, and of what all do.
__device__ __forceinline__ void wave_span(int& wlo, int& whi, int& flo, int& fhi) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    wlo = min(wlo, __shfl_xor(wlo, o, 64));
    whi = max(whi, __shfl_xor(whi, o, 64));
    flo = max(flo, __shfl_xor(flo, o, 64));
    fhi = min(fhi, __shfl_xor(fhi, o, 64));
  }
  wlo = __builtin_amdgcn_readfirstlane(wlo), whi = __builtin_amdgcn_readfirstlane(whi);
  flo = __builtin_amdgcn_readfirstlane(flo), fhi = __builtin_amdgcn_readfirstlane(fhi);
}

// The tile that comes `rank`-th when n of them are taken by falling work (ties by index): workgroups start in the order of their numbers, and
// a long one that starts last is waited for by the whole chip (packed sequences, dK / dV: 203 -> 165 us).  Every workgroup finds its own,
// so at most RANK_MAX are ranked; beyond that the last ones come first (behind a causal mask they see the most).
constexpr int RANK_MAX = 512;
template <class Work>
__device__ __forceinline__ int by_work(int rank, int n, Work work, int* lds) {
  if (n > RANK_MAX) return n - 1 - rank;
  for (int i = threadIdx.x; i < n; i += 256) lds[i] = work(i);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 256) {
    const int mine = lds[i];
    int before = 0;
    for (int k = 0; k < n; ++k) before += lds[k] > mine || (lds[k] == mine && k < i);
    if (before == rank) lds[RANK_MAX] = i;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(lds[RANK_MAX]);
}

// A value that the compiler knows nothing of: what is computed from it is not kept from an earlier computation.
__device__ __forceinline__ int afresh(int x) {
  asm volatile("" : "+v"(x));
  return __builtin_amdgcn_readfirstlane(x);
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
