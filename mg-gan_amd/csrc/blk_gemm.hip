// The layers of a transformer block that are matrix products: linear with bias, activation and residual, and the gated layer
// act(x Wg^T + bg) * (x Wu^T + bu); forward and backward, f32 and bf16.
//
// One kernel does all products, C[m][n] = sum_k A(m, k) B(n, k); an operand lies in memory with k contiguous ("rows": x, W in the
// forward pass, dZ in dX = dZ W) or with k as the row index ("columns": W in dX, both operands of dW = dZ^T x) and goes through LDS as it
// lies; columns are read out transposed.  So nothing is transposed in memory.  The gated layer takes its B rows from two weights, so that
// one wave holds the gate and the up value of the same outputs and multiplies them in registers.
#include "blk.h"
#include "../../include/mggan_hip.h"

struct BlkLayerArgs {  // mirrored by mggan/hip/blocks.py
  const void *x, *w, *w2, *b, *b2, *res, *dy;  // w2: the up weight of a gated layer, NULL for a linear one
  float *z, *z2;
  void *y, *dx, *dw, *db, *ws;
  long ws_bytes, ldx;
  int M, K, N, act, dtype;
  float slope;
};

namespace {

__device__ __attribute__((aligned(16))) const unsigned blk_zeros[4] = {0, 0, 0, 0};

struct GemmP {
  const void* A;
  const void* B;
  const void* B2;  // gated: the up weight
  long lda, ldb;   // elements; rows are 16-byte aligned
  int ca, cb;      // columns that may be read of an operand that lies in columns (a multiple of the chunk)
  int kb, seg;     // B in columns: its k; seg > 0: after so many steps B2's follow
  int M, N, K;     // an operand in rows: K a multiple of the chunk (8 bf16 / 4 f32)
  int tiles_m, tiles_n, kt_split;
  void* C;
  long ldc;
  float* Z;  // inputs of the activation, kept for the backward pass (or null) in f32: rounded to bf16 they would put a second
  float* Z2; // half step next to dZ's own into every gradient
  const void* bias;
  const void* bias2;
  const void* res;  // (M, N) contiguous
  int act;
  float slope;
  float* part;  // split reduction: (splits, M, N or 2 N)
};


enum { EPI_LINEAR = 0, EPI_GATED = 1 };

template <class T, int W>
__device__ __forceinline__ void load_n(const T* p, bool vec, int left, float (&v)[W]) {
  if (vec && left >= W) {
    if constexpr (sizeof(T) == 2) {
      typedef bf16 V __attribute__((ext_vector_type(W)));
      const V x = *(const V*)p;
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = (float)x[i];
    } else {
#pragma unroll
      for (int j = 0; j < W; j += 4) {
        const f32x4 x = *(const f32x4*)(p + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j + i] = x[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = i < left ? (float)p[i] : 0.f;
  }
}
template <class T, int W>
__device__ __forceinline__ void store_n(T* p, bool vec, int left, const float (&v)[W]) {
  if (vec && left >= W) {
    if constexpr (sizeof(T) == 2) {
      typedef bf16 V __attribute__((ext_vector_type(W)));
      V x;
#pragma unroll
      for (int i = 0; i < W; ++i) x[i] = (bf16)v[i];
      *(V*)p = x;
    } else {
#pragma unroll
      for (int j = 0; j < W; j += 4) *(f32x4*)(p + j) = f32x4{v[j], v[j + 1], v[j + 2], v[j + 3]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < left) p[i] = (T)v[i];
  }
}

// The epilogue of W neighbouring outputs of row m from column n on.
template <class T, int EPI, int W>
__device__ __forceinline__ void epilogue(const GemmP& p, int m, int n, float (&v)[W], float (&u)[W], bool vec) {
  const int left = p.N - n;
  if (left <= 0) return;
  float t[W];
  const long at = (long)m * p.N + n;
  if (p.bias) {
    load_n<T, W>((const T*)p.bias + n, vec, left, t);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] += t[i];
  }
  if (EPI == EPI_GATED && p.bias2) {
    load_n<T, W>((const T*)p.bias2 + n, vec, left, t);
#pragma unroll
    for (int i = 0; i < W; ++i) u[i] += t[i];
  }
  if (p.Z) store_n<float, W>(p.Z + at, vec, left, v);
  if (EPI == EPI_GATED && p.Z2) store_n<float, W>(p.Z2 + at, vec, left, u);
  if (p.act != ACT_NONE) {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = blk_act(v[i], p.act, p.slope);
  }
  if (EPI == EPI_GATED) {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] *= u[i];
  }
  if (p.res) {
    load_n<T, W>((const T*)p.res + at, vec, left, t);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] += t[i];
  }
  store_n<T, W>((T*)p.C + (long)m * p.ldc + n, vec, left, v);
}

// One operand of a tile in LDS: R outputs by 64 bytes of k, filled by NT threads.  The copies land lane by lane, so the swizzle that
// keeps a wave's reads off each other's banks is in which chunk a lane fetches.
//   rows:    [R][4 chunks], chunk c of row r at c ^ s(r): a wave reads one chunk of 16 rows, rows 0-15 or {0-3, 8-11, 16-19, 24-27} (+4);
//            any eight lanes of either set fall on eight bank groups.
//   columns: [64 / sizeof(T) values of k][R / CH chunks]: bf16 is read by the transposing LDS read (16 lanes take 4 k x 16 columns: four
//            rows of two chunks each, on eight bank groups), f32 element by element (4 k x 16 columns: two passes, the least for 256 bytes).
// Eight groups of four banks are half of what LDS serves in a cycle, so conflicts remain: 2.7 cycles beside the 4 of a 16-byte read, 2.0 beside
// the 2 of a transposing one (counters).
template <class T, int R, int NT, bool COLS>
struct Side {
  static constexpr int CH = Mf<T>::CH, KS = 4 * CH, L = R * 4 / NT, NC = COLS ? R / CH : 4, SIZE = R * 4;
  const char* src[L];
  int c;         // the chunk this lane copies
  long step;     // bytes from one k step to the next
  int k_row;     // columns: the k of this lane's first copy

  static __device__ __forceinline__ int swz(int r) {
    if (!COLS) return ((r >> 1) & 3) ^ ((r >> 2) & 2);
    return sizeof(T) == 2 ? (r & 3) << 1 : r & 4;
  }
  // base(row) -> first byte of an operand row; o0: the tile's first output, cols: columns that may be read, k0: first k
  template <class Base>
  __device__ __forceinline__ void init(Base base, long ld, int o0, int cols, long k0) {
    const int tid = threadIdx.x;
    if constexpr (!COLS) {
      c = (tid & 3) ^ swz(tid >> 2);  // (a lane's rows differ by multiples of 16)
      step = 64;
#pragma unroll
      for (int i = 0; i < L; ++i) src[i] = base((i * NT + tid) >> 2, true) + k0 * sizeof(T) + c * 16;
    } else {
      k_row = tid / NC;  // (a lane's k differ by NT / NC: multiples of 8)
      c = min((tid % NC) ^ swz(k_row), (cols - o0) / CH - 1);  // (outputs past the end are not stored: any column will do for them)
      step = ld * KS * sizeof(T);
#pragma unroll
      for (int i = 0; i < L; ++i) src[i] = base(0, false) + ((k0 + k_row + i * (NT / NC)) * ld + o0) * sizeof(T) + c * 16;
    }
  }
  // the copies of one k step into d; WHOLE: it lies inside k, else `left` values of k do and zeros stand for the rest
  template <bool WHOLE>
  __device__ __forceinline__ void fetch(u32x4* d, int left, const char* zeros) {
    d += mg_wave() * 64;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const bool ok = WHOLE || (COLS ? k_row + i * (NT / NC) < left : c * CH < left);
      lds_copy16(ok ? src[i] : zeros, d + i * NT);
      src[i] += step;
    }
  }
  // fragment of 16 outputs: rows given by `row` (this lane's), columns by their first
  static __device__ __forceinline__ u32x4 frag(const u32x4* t, int row, int first, int lane) {
    const int i16 = lane & 15, g = lane >> 4;
    if constexpr (!COLS) {
      return t[row * 4 + (g ^ swz(row))];
    } else if constexpr (sizeof(T) == 2) {
      const int k = 8 * g + (i16 >> 2), sw = swz(k), ch = (first >> 3) + ((i16 & 3) >> 1);
      const char* a = (const char*)(t + k * NC + (ch ^ sw)) + 8 * (i16 & 1);
      const s16x4 x = lds_transposed(a);
      const s16x4 y = lds_transposed(a + 4 * NC * 16);  // (k + 4: the same swizzle)
      return __builtin_bit_cast(u32x4, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      u32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 4 * g + e, col = first + i16;
        v[e] = ((const unsigned*)(t + k * NC + ((col >> 2) ^ swz(k))))[col & 3];
      }
      return v;
    }
  }
};

// Waits until at most n of this wave's copies are under way (they end in their order) and its LDS reads are done (the next copies go into
// what they read), then for the other waves.
template <int n>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(n) : "memory");
}

// A tile of BM x BN outputs, WM x WN waves; k in steps of 64 bytes through a ring of four LDS buffers.  In step t the copies of step
// t+3 start, the fragments of step t+1 are read into registers and those of step t are multiplied: the matrix cores wait neither for
// memory (two steps of slack) nor for LDS (one step).
// Bound by the matrix cores from about 256 tiles on.  A tile of 256 x 256 takes 32 KB of copies for 4.2 MFLOP, so that its bytes come out of the
// L2; its eight waves of 128 x 64 read 12 fragments for 32 multiplications (four waves of 128 x 128 would read less, but 256 accumulators
// leave no room for a second set of fragments: 634 TFLOP/s).  8,192 x 4,096 x 4,096 bf16: 204 us, 1.35 PFLOP/s (the library: 1.24-1.6), the
// gated training pass' products of four times that work 1.05 (forward), 1.15 (dX) and 1.24 (dW); f32, 4,096 each way: 145 TFLOP/s (136).  Its matrix
// cores are busy 65, 70 and 76 % of the time in these; copies of two steps behind one barrier made it 964 instead of 1,150 TFLOP/s.
template <class T, int BM, int BN, int WM, int WN, int EPI, bool SPLIT, bool CA, bool CB>
__global__ __launch_bounds__(WM* WN * 64) void blk_gemm_kernel(GemmP p) {
  constexpr int NT = WM * WN * 64, CH = Mf<T>::CH, KS = 4 * CH;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int NB = EPI == EPI_GATED ? BN / 2 : BN;  // output columns of the tile
  using SA = Side<T, BM, NT, CA>;
  using SB = Side<T, BN, NT, CB>;
  constexpr int BUF = SA::SIZE + SB::SIZE, LOADS = SA::L + SB::L;
  __shared__ u32x4 lds[4 * BUF];

  int t = blockIdx.x;
  {  // neighbouring tiles to the same XCD (blocks are dealt round the eight of them), in columns of four row tiles
    const int nb = p.tiles_m * p.tiles_n, n8 = nb >> 3;
    if (t < n8 * 8) t = (t & 7) * n8 + (t >> 3);
  }
  const int per = 4 * p.tiles_n, grp = t / per, gm = min(4, p.tiles_m - 4 * grp), rem = t - grp * per;
  const int m0 = (4 * grp + rem % gm) * BM, n0 = (rem / gm) * NB;
  const int lane = mg_lane(), wave = mg_wave(), i16 = lane & 15, g = lane >> 4;
  const int steps = (p.K + KS - 1) / KS;
  const int kt0 = SPLIT ? blockIdx.y * p.kt_split : 0, n = (SPLIT ? min(kt0 + p.kt_split, steps) : steps) - kt0;

  SA sa;
  SB sb;
  sa.init([&](int row, bool rows) { return (const char*)p.A + (rows ? (long)min(m0 + row, p.M - 1) * p.lda * sizeof(T) : 0); }, p.lda, m0,
          p.ca, (long)kt0 * KS);
  auto base_b = [&](bool second) {
    return [&, second](int row, bool rows) {
      const bool up = EPI == EPI_GATED && row >= NB;
      return (const char*)(up || second ? p.B2 : p.B) + (rows ? (long)min(n0 + (up ? row - NB : row), p.N - 1) * p.ldb * sizeof(T) : 0);
    };
  };
  const bool second = CB && p.seg && kt0 >= p.seg;
  sb.init(base_b(second), p.ldb, n0, p.cb, (long)(second ? kt0 - p.seg : kt0) * KS);
  auto fetch = [&](int t) {
    const int kt = kt0 + t;
    int kb = kt;
    if (CB && p.seg && kt >= p.seg) {
      kb -= p.seg;
      if (kb == 0 && t) sb.init(base_b(true), p.ldb, n0, p.cb, 0);
    }
    u32x4* d = lds + (t & 3) * BUF;
    const int la = p.K - kt * KS, lb = (CB ? p.kb : p.K) - kb * KS;
    if (la >= KS)
      sa.template fetch<true>(d, la, (const char*)blk_zeros);
    else
      sa.template fetch<false>(d, la, (const char*)blk_zeros);
    if (lb >= KS)
      sb.template fetch<true>(d + SA::SIZE, lb, (const char*)blk_zeros);
    else
      sb.template fetch<false>(d + SA::SIZE, lb, (const char*)blk_zeros);
  };

  f32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // B's fragments of rows are numbered so that a lane's results of a pair of fragments are eight neighbouring outputs; those of columns
  // have to keep their order (four neighbouring outputs).
  const int wm = wave % WM, wn = wave / WM;
  int rb[FN];
#pragma unroll
  for (int f = 0; f < FN; ++f) {
    const int q = EPI == EPI_GATED ? f % (FN / 2) : f;
    rb[f] = (EPI == EPI_GATED ? (f / (FN / 2)) * NB + wn * (TN / 2) : wn * TN);
    rb[f] += CB ? 16 * q : 32 * (q >> 1) + 8 * (i16 >> 2) + 4 * (q & 1) + (i16 & 3);
  }
  struct Frags {
    u32x4 a[FM], b[FN];
  };
  auto read = [&](int t, Frags& f) {
    const u32x4* la = lds + (t & 3) * BUF;
    const u32x4* lb = la + SA::SIZE;
#pragma unroll
    for (int i = 0; i < FN; ++i) f.b[i] = SB::frag(lb, rb[i], rb[i], lane);
#pragma unroll
    for (int j = 0; j < FM; ++j) f.a[j] = SA::frag(la, wm * TM + 16 * j + i16, wm * TM + 16 * j, lane);
  };
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] = Mf<T>::step(f.b[i], f.a[j], acc[i][j]);
  };
  // a step whose copies and multiplications are all there: straight code, in which the reads of the next fragments and the copies are
  // dealt out among the multiplications
  auto steady = [&](int t, const Frags& now, Frags& next) {
    wait_copies<LOADS>();
    read(t + 1, next);
    u32x4* d = lds + ((t + 3) & 3) * BUF;
    sa.template fetch<true>(d, 0, nullptr);
    sb.template fetch<true>(d + SA::SIZE, 0, nullptr);
    multiply(now);
    constexpr int READS = (CA ? (sizeof(T) == 2 ? 2 : 4) : 1) * FM + (CB ? (sizeof(T) == 2 ? 2 : 4) : 1) * FN;
    constexpr int MM = FM * FN * (sizeof(T) == 2 ? 1 : 4), EACH = MM / (READS + LOADS) > 0 ? MM / (READS + LOADS) : 1;
#pragma unroll
    for (int i = 0; i < READS / 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);  // multiplications
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);     // an LDS read
      __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);  // multiplications
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // a copy
      __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
    }
  };
  auto any = [&](int t, const Frags& now, Frags& next) {
    if (t + 2 < n)
      wait_copies<LOADS>();
    else
      wait_copies<0>();
    if (t + 3 < n) fetch(t + 3);
    read(t + 1 < n ? t + 1 : t, next);  // (after the last step: read again, not used)
    multiply(now);
  };

  if (n > 0) {
    Frags f0, f1;
    fetch(0);
    if (n > 1) fetch(1);
    if (n > 2) fetch(2);
    if (n > 2)
      wait_copies<2 * LOADS>();
    else
      wait_copies<0>();
    read(0, f0);
    int t = 0;
    const int kw = (CB ? min(p.K, p.kb) : p.K) / KS;  // steps that lie inside k (with two segments: inside either)
    auto walk = [&](int end) {
      for (; t + 4 < end; t += 2) {
        steady(t, f0, f1);
        steady(t + 1, f1, f0);
      }
    };
    int whole = min(kw - kt0, n);
    if (CB && p.seg) {
      const int s = p.seg - kt0;  // the second segment's first step
      if (s > 0 && s < n) {
        walk(min(kw - kt0, s));
        for (; t < n && t + 3 <= s; t += 2) {
          any(t, f0, f1);
          if (t + 1 < n) any(t + 1, f1, f0);
        }
      }
      whole = min(n, s < n ? s + kw : kw - kt0);
    }
    walk(whole);
    for (; t < n; t += 2) {
      any(t, f0, f1);
      if (t + 1 < n) any(t + 1, f1, f0);
    }
  }

  constexpr int FO = EPI == EPI_GATED ? FN / 2 : FN, W = CB ? 4 : 8, P = W / 4;
  const bool vec = p.N % (SPLIT && EPI != EPI_GATED ? 4 : CH) == 0;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int m = m0 + wm * TM + 16 * j + i16;
    if (m >= p.M) continue;
#pragma unroll
    for (int f = 0; f < FO; f += P) {
      const int n = n0 + wn * (FO * 16) + 16 * f + W * g;  // (the lane's first output)
      float v[W], u[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        v[e] = acc[f + e / 4][j][e % 4];
        u[e] = EPI == EPI_GATED ? acc[FO % FN + f + e / 4][j][e % 4] : 0.f;
      }
      if (SPLIT) {
        if (n >= p.N) continue;
        const long cols = EPI == EPI_GATED ? 2L * p.N : p.N;
        float* out = p.part + ((long)blockIdx.y * p.M + m) * cols + n;
        store_n<float, W>(out, vec, p.N - n, v);
        if (EPI == EPI_GATED) store_n<float, W>(out + p.N, vec, p.N - n, u);
      } else {
        epilogue<T, EPI, W>(p, m, n, v, u, vec);
      }
    }
  }
}

// The partial sums of a split reduction, then the epilogue: four outputs a thread, whose partial sums four threads add up (each every
// fourth, in their order, so that the result does not depend on which workgroup ends first).  Bound by the partial sums' bytes and, where
// they are few, by the launch (4 to 6 us beside products of 30).
template <class T, int EPI>
__global__ __launch_bounds__(256) void blk_join_kernel(GemmP p, int splits) {
  __shared__ f32x4 part[EPI == EPI_GATED ? 2 : 1][4][64];
  const int per = (p.N + 3) >> 2, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const long id = (long)blockIdx.x * 64 + x;
  const int m = (int)(id / per), n = (int)(id % per) * 4;
  const bool mine = id < (long)per * p.M, vec = p.N % 4 == 0;
  const long cols = EPI == EPI_GATED ? 2L * p.N : p.N;
  float v[4] = {}, u[4] = {}, t[4];
  if (mine) {
#pragma unroll 4
    for (int s = y; s < splits; s += 4) {
      const float* in = p.part + ((long)s * p.M + m) * cols + n;
      load_n<float, 4>(in, vec, p.N - n, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += t[i];
      if (EPI == EPI_GATED) {
        load_n<float, 4>(in + p.N, vec, p.N - n, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] += t[i];
      }
    }
  }
  part[0][y][x] = f32x4{v[0], v[1], v[2], v[3]};
  if (EPI == EPI_GATED) part[EPI == EPI_GATED][y][x] = f32x4{u[0], u[1], u[2], u[3]};
  __syncthreads();
  if (y || !mine) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = (part[0][0][x][i] + part[0][1][x][i]) + (part[0][2][x][i] + part[0][3][x][i]);
    if constexpr (EPI == EPI_GATED) u[i] = (part[1][0][x][i] + part[1][1][x][i]) + (part[1][2][x][i] + part[1][3][x][i]);
  }
  epilogue<T, EPI, 4>(p, m, n, v, u, p.N % Mf<T>::CH == 0);
}

// 16 bytes of a row from element k on, rows of any alignment; what lies past the row's end is zero.
template <class T>
__device__ __forceinline__ u32x4 row_chunk(const T* row, int k, int K) {
  u32x4 v = {0, 0, 0, 0};
  if (k + Mf<T>::CH <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
    T t[Mf<T>::CH];
#pragma unroll
    for (int i = 0; i < Mf<T>::CH; ++i) t[i] = k + i < K ? row[k + i] : (T)0.f;
    __builtin_memcpy(&v, t, 16);
  }
  return v;
}

// The forward product of up to 16 rows of x: weights stream from memory straight into matrix-instruction operands, once, with nothing
// between.  A workgroup takes 16 outputs (of both weights where gated), its waves a share of k each; x comes out of the caches.
// Bound by the weights' bytes, so what counts is how many loads are under way (8 of 16 bytes a lane and operand).  8 rows of 4,096, a weight of
// 16,384 x 4,096 (134 MB): 26.5 us, 5.1 TB/s; a small one by the launch (16 rows of 512, 512 outputs, f32: 4 us).
template <class T, int EPI, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void blk_few_rows_kernel(GemmP p) {
  constexpr int CH = Mf<T>::CH, U = 8, two = EPI == EPI_GATED ? 2 : 1;
  __shared__ f32x4 part[WAVES][two][64];
  const int lane = mg_lane(), wave = mg_wave(), i16 = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;
  const T* w = (const T*)p.B + (long)min(n0 + i16, p.N - 1) * p.ldb;
  const T* w2 = (const T*)p.B2 + (long)min(n0 + i16, p.N - 1) * p.ldb;
  const T* x = (const T*)p.A + (long)min(i16, p.M - 1) * p.lda;  // (rows past the last give outputs that are not stored)
  const int steps = (p.K + 4 * CH - 1) / (4 * CH), share = (steps + WAVES - 1) / WAVES;
  const int s0 = wave * share, s1 = min(s0 + share, steps), whole = min(s1, p.K / (4 * CH));
  f32x4 acc[two] = {};
  int s = s0;
  for (; s + U <= whole; s += U) {
    u32x4 a[U], b[U], c[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = (4 * (s + i) + g) * CH;
      __builtin_memcpy(&a[i], w + k, 16);
      if (two == 2) __builtin_memcpy(&b[i], w2 + k, 16);
      __builtin_memcpy(&c[i], x + k, 16);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      acc[0] = Mf<T>::step(a[i], c[i], acc[0]);
      if (two == 2) acc[two - 1] = Mf<T>::step(b[i], c[i], acc[two - 1]);
    }
  }
  for (; s < s1; ++s) {
    const int k = (4 * s + g) * CH;
    const u32x4 c = row_chunk(x, k, p.K);
    acc[0] = Mf<T>::step(row_chunk(w, k, p.K), c, acc[0]);
    if (two == 2) acc[two - 1] = Mf<T>::step(row_chunk(w2, k, p.K), c, acc[two - 1]);
  }
#pragma unroll
  for (int i = 0; i < two; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave || i16 >= p.M) return;
  float v[4], u[4] = {};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = part[0][0][lane][e];
    if (two == 2) u[e] = part[0][two - 1][lane][e];
    for (int k = 1; k < WAVES; ++k) {
      v[e] += part[k][0][lane][e];
      if (two == 2) u[e] += part[k][two - 1][lane][e];
    }
  }
  epilogue<T, EPI, 4>(p, i16, n0 + 4 * g, v, u, p.N % CH == 0);
}

// Rows of `cols` elements into rows of `ldo` (>= cols), the rest zeros.
template <class T>
__global__ __launch_bounds__(256) void blk_pad_kernel(const T* in, long ldi, T* out, long ldo, int rows, int cols) {
  for (long id = (long)blockIdx.x * 256 + threadIdx.x; id < (long)rows * ldo; id += (long)gridDim.x * 256) {
    const long r = id / ldo, cc = id - r * ldo;
    out[id] = cc < cols ? in[r * ldi + cc] : (T)0.f;
  }
}

// dY -> dZ = dY act'(z) (linear) or dG = dY u act'(g), dU = dY act(g) (gated), as rows of ld ldz (dU `off` behind dG, zeros up to the
// end of each), and the columns' sums of DZ_ROWS rows in f32 for the bias gradients.  dZ is rounded to the operands' type once: it is an
// operand of both products, and half a step is what every operand has (bf16 gradients 0.0023 to 0.0024 off against 64 bits, 0.0017 with dZ in f32).  A thread takes eight columns of every eighth row.
// Bound by bytes (gated bf16: 10 read and 4 written an output): 8,192 x 8,192 gated 200 us, 4.7 TB/s.
constexpr int DZ_ROWS = 64;
struct DzP {
  const void* dY;
  const float* Z;
  const float* Z2;
  void* dZ;
  float* sums;  // (ceil(M / DZ_ROWS), N or 2 N)
  int M, N, act;
  float slope;
  long ldz, off;
};
template <class T, bool GATED>
__global__ __launch_bounds__(256) void blk_dz_kernel(DzP p) {
  constexpr int two = GATED ? 2 : 1;
  __shared__ float part[two][8][256];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, n = blockIdx.x * 256 + 8 * x, r0 = blockIdx.y * DZ_ROWS;
  const int left = p.N - n;
  const bool vec = p.N % 8 == 0;
  float s[two][8] = {};
  if (n < p.off) {
#pragma unroll 2
    for (int i = y; i < DZ_ROWS; i += 8) {
      const int m = r0 + i;
      if (m >= p.M) break;
      const long at = (long)m * p.N + n;
      float dy[8], z[8], a[8], b[8];
      load_n<T, 8>((const T*)p.dY + at, vec, left, dy);
      if (GATED || p.Z) load_n<float, 8>(p.Z + at, vec, left, z);
      if constexpr (GATED) {
        float u[8];
        load_n<float, 8>(p.Z2 + at, vec, left, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          b[e] = dy[e] * blk_act(z[e], p.act, p.slope);
          a[e] = dy[e] * u[e] * blk_act_grad(z[e], p.act, p.slope);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = p.Z ? dy[e] * blk_act_grad(z[e], p.act, p.slope) : dy[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[0][e] += a[e];
        if (GATED) s[GATED][e] += b[e];
      }
      if (p.dZ) {  // (columns from N to `off` are loaded as zeros)
        const bool v16 = p.off % 8 == 0;
        store_n<T, 8>((T*)p.dZ + m * p.ldz + n, v16, (int)p.off - n, a);
        if (GATED) store_n<T, 8>((T*)p.dZ + m * p.ldz + p.off + n, v16, (int)p.off - n, b);
      }
    }
  }
  if (!p.sums) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    part[0][y][8 * x + e] = s[0][e];
    if (GATED) part[GATED][y][8 * x + e] = s[GATED][e];
  }
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.N) return;
#pragma unroll
  for (int k = 0; k < two; ++k) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += part[k][i][threadIdx.x];
    p.sums[(long)blockIdx.y * two * p.N + (long)k * p.N + c] = t;
  }
}

// Column sums of (rows, cols) partials in a fixed order, rounded to the bias' type.  A launch's worth of work (4 to 6 us).
template <class T>
__global__ __launch_bounds__(1024) void blk_colsum_kernel(const float* in, int rows, int cols, T* out) {
  __shared__ float part[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int r = y; r < rows; r += 32) s += in[(long)r * cols + c];
  }
  part[y][x] = s;
  __syncthreads();
  if (y != 0 || c >= cols) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += part[i][x];
  out[c] = (T)s;
}

// ---- host side -------------------------------------------------------------------------------------------------------------

inline long up(long a, long b) { return (a + b - 1) / b * b; }

// Tile and split of one product, by an estimate of its time: rounds of workgroups over the 256 CUs, each round its multiplications (at the
// rate the tile reaches) and what a workgroup costs before and after them; a split adds the partial sums' way through memory and a launch.
// Measured, all tiles and splits of ten products forced (rows x k x outputs, us, tile/splits): f32 256 x 512 x 512: 64/1 13.4, 64/4 9.5 (chosen),
// 128/4 16.6; f32 4,096 x 512 x 512: 64/1 23.4 (chosen), 128/2 36.4; bf16 2,048 each way: 128/1 26.9 (chosen), 256/1 42.2, 64/1 47.5; bf16 8,192 x
// 4,096 x 4,096: 256/1 204 (chosen), 128/1 323, 64/1 540.  The choice is the best or within 7 % of it but for two: 1,024 x 4,096 x 1,024, 28.7 against
// 24.4 with 128/4, and 100 x 4,096 x 4,096, 19.2 against 17.4 with 128/8.
struct Plan {
  int tile, splits, kt_split;
  size_t bytes;
};
Plan plan_of(int M, int N, long K, int ch, bool gated) {
  const int half = gated ? 2 : 1;
  const long steps = (K + 4 * ch - 1) / (4 * ch);
  Plan best = {};
  double least = 1e30;
  const int tiles[3] = {256, 128, 64};
  for (int i = 0; i < 3; ++i) {
    const int b = tiles[i];
    const long nt = (long)cdiv(M, b) * cdiv(N, b / half);
    // cycles of one step of one tile on a CU, per workgroup with the CU to itself; a CU holds `res` of them
    const double flops = 2. * b * b * 4 * ch, rate = ch == 4 ? (b == 256 ? 230. : b == 128 ? 220. : 200.) : (b == 256 ? 2600. : b == 128 ? 1900. : 1000.);
    const int res = b == 256 ? 1 : b == 128 ? 2 : 4;
    for (int splits = 1; splits <= 64 && splits <= steps; splits *= 2) {
      if (splits > 1 && nt * splits > 2048) break;
      const long per = (steps + splits - 1) / splits, blocks = nt * ((steps + per - 1) / per);
      const double busy = (double)((blocks + 255) / 256);  // workgroups of the fullest CU
      const double work = busy * per * flops / rate;       // (they share its matrix cores)
      const double fixed = 2000. + 1200. * ((busy + res - 1) / res);
      const double join = splits > 1 ? 8000. + 8. * splits * (double)M * N * half / 1500. : 0.;
      const double t = work + fixed + join;
      if (t < least) {
        least = t;
        best.tile = b;
        best.kt_split = (int)per;
        best.splits = (int)((steps + per - 1) / per);
        best.bytes = best.splits > 1 ? (size_t)best.splits * M * N * half * 4 : 0;
      }
    }
  }
  return best;
}

template <class T, int B, int WM, int WN, int EPI, bool CA, bool CB>
int gemm_tile(GemmP& p, const Plan& q, hipStream_t st) {
  p.tiles_m = cdiv(p.M, B);
  p.tiles_n = cdiv(p.N, EPI == EPI_GATED ? B / 2 : B);
  p.kt_split = q.kt_split;
  if (q.splits > 1) {
    MG_LAUNCH((blk_gemm_kernel<T, B, B, WM, WN, EPI, true, CA, CB>), dim3(p.tiles_m * p.tiles_n, q.splits), dim3(WM * WN * 64), 0, st, p);
    MG_LAUNCH((blk_join_kernel<T, EPI>), dim3(cdiv((long)cdiv(p.N, 4) * p.M, 64)), dim3(256), 0, st, p, q.splits);
  } else {
    MG_LAUNCH((blk_gemm_kernel<T, B, B, WM, WN, EPI, false, CA, CB>), dim3(p.tiles_m * p.tiles_n), dim3(WM * WN * 64), 0, st, p);
  }
  MG_LAUNCH_CHECK("block gemm");
  return MGGAN_OK;
}
template <class T, int EPI, bool CA, bool CB>
int gemm(GemmP p, void* ws, hipStream_t st) {
  const Plan q = plan_of(p.M, p.N, p.K, Mf<T>::CH, EPI == EPI_GATED);
  p.part = (float*)ws;
  switch (q.tile) {
    case 256: return gemm_tile<T, 256, 2, 4, EPI, CA, CB>(p, q, st);
    case 128: return gemm_tile<T, 128, 2, 2, EPI, CA, CB>(p, q, st);
    default: return gemm_tile<T, 64, 4, 1, EPI, CA, CB>(p, q, st);
  }
}

struct Arena {  // 256-byte aligned pieces of the caller's workspace; without a base it only counts
  char* base;
  size_t at;
  void* take(size_t bytes) {
    void* p = base ? base + at : nullptr;
    at += up((long)bytes, 256);
    return p;
  }
};

template <class T>
void pad(const void* in, long ldi, void* out, long ldo, int rows, int cols, hipStream_t st) {
  const long n = (long)rows * ldo;
  MG_LAUNCH((blk_pad_kernel<T>), dim3((unsigned)(n / 256 + 1 < 4096 ? n / 256 + 1 : 4096)), dim3(256), 0, st, (const T*)in, ldi, (T*)out, ldo,
            rows, cols);
}

// x and the weights with rows of whole chunks: as they are, or copied with zeros behind where K is odd.
template <class T, bool GATED>
struct Padded {
  int Kp;
  const void *x, *w, *w2;
  long ldx;
  Padded(const BlkLayerArgs& l, Arena& ws, bool run, bool want_x, bool want_w, hipStream_t st) {
    Kp = (int)up(l.K, Mf<T>::CH);
    x = l.x, w = l.w, w2 = l.w2, ldx = l.ldx;
    if (Kp == l.K) return;
    void* xp = ws.take((size_t)l.M * Kp * sizeof(T));
    void* wp = ws.take((size_t)l.N * Kp * sizeof(T));
    void* wp2 = GATED ? ws.take((size_t)l.N * Kp * sizeof(T)) : nullptr;
    if (!run) return;
    if (want_x) pad<T>(l.x, l.ldx, xp, Kp, l.M, l.K, st), x = xp, ldx = Kp;
    if (want_w) pad<T>(l.w, l.K, wp, Kp, l.N, l.K, st), w = wp;
    if (want_w && GATED) pad<T>(l.w2, l.K, wp2, Kp, l.N, l.K, st), w2 = wp2;
  }
};

template <class T, bool GATED>
int layer_fwd(const BlkLayerArgs& l, Arena ws, size_t* need, hipStream_t st) {
  constexpr int EPI = GATED ? EPI_GATED : EPI_LINEAR;
  GemmP p = {};
  p.M = l.M, p.N = l.N;
  p.C = l.y, p.ldc = l.N, p.Z = l.z, p.Z2 = l.z2, p.bias = l.b, p.bias2 = l.b2, p.res = l.res, p.act = l.act, p.slope = l.slope;
  // one matrix instruction's worth of rows: bound by the weights' bytes (us against the tile kernel's: 16 rows of 512, 512 outputs, f32 4.0 / 6.8;
  // 16 rows of 4,096, gated 8,192, bf16 27.7 / 31.1; 24 rows, which take two such instructions, are left to the tiles: 31.7)
  if (l.M <= 16) {
    p.A = l.x, p.lda = l.ldx, p.B = l.w, p.B2 = l.w2, p.ldb = l.K, p.K = l.K;
    if (need) {
      *need = 0;
      return MGGAN_OK;
    }
    const unsigned blocks = cdiv(l.N, 16);
    // few workgroups: eight waves in each, for bytes in flight; else four, with fewer sums to join (8 rows of 4,096, four waves / eight, us:
    // linear 4,096 outputs 9.8 / 8.7, 8,192: 16.9 / 15.1, 16,384: 26.5 / 26.4; gated 8,192: 26.0 / 27.6)
    if (blocks * (GATED ? 2 : 1) < 1024)
      MG_LAUNCH((blk_few_rows_kernel<T, EPI, 8>), dim3(blocks), dim3(512), 0, st, p);
    else
      MG_LAUNCH((blk_few_rows_kernel<T, EPI, 4>), dim3(blocks), dim3(256), 0, st, p);
    MG_LAUNCH_CHECK("block layer forward");
    return MGGAN_OK;
  }
  const Padded<T, GATED> o(l, ws, !need, true, true, st);
  void* part = ws.take(plan_of(l.M, l.N, o.Kp, Mf<T>::CH, GATED).bytes);
  if (need) {
    *need = ws.at;
    return MGGAN_OK;
  }
  p.A = o.x, p.lda = o.ldx, p.B = o.w, p.B2 = o.w2, p.ldb = o.Kp, p.K = o.Kp;
  return gemm<T, EPI, false, false>(p, part, st);
}

template <class T, bool GATED>
int layer_bwd(const BlkLayerArgs& l, Arena ws, size_t* need, hipStream_t st) {
  constexpr int CH = Mf<T>::CH, two = GATED ? 2 : 1;
  const long tiles = cdiv(l.M, DZ_ROWS);
  const long off = up(l.N, GATED ? 4 * CH : CH), ldz = two * off;  // (gated: dU starts with a step of dX's product)
  const bool plain = !GATED && l.act == ACT_NONE && off == l.N;    // dZ is dY
  const Padded<T, GATED> o(l, ws, !need, l.dw != nullptr, l.dx != nullptr, st);
  void* dz = plain ? nullptr : ws.take((size_t)l.M * ldz * sizeof(T));
  float* sums = (float*)ws.take((size_t)tiles * two * l.N * 4);
  const int mw = GATED ? (int)off + l.N : l.N;  // rows of dw
  const size_t px = plan_of(l.M, l.K, ldz, CH, false).bytes, pw = plan_of(mw, l.K, l.M, CH, false).bytes;
  void* part = ws.take(px > pw ? px : pw);
  if (need) {
    *need = ws.at;
    return MGGAN_OK;
  }
  if (!plain || l.db) {
    DzP d = {};
    d.dY = l.dy, d.Z = l.z, d.Z2 = l.z2, d.dZ = dz, d.sums = l.db ? sums : nullptr;
    d.M = l.M, d.N = l.N, d.act = l.act, d.slope = l.slope, d.ldz = ldz, d.off = off;
    MG_LAUNCH((blk_dz_kernel<T, GATED>), dim3(cdiv(off, 256), (unsigned)tiles), dim3(256), 0, st, d);
    if (l.db)
      MG_LAUNCH((blk_colsum_kernel<T>), dim3(cdiv((long)two * l.N, 32)), dim3(1024), 0, st, (const float*)sums, (int)tiles, two * l.N, (T*)l.db);
  }
  GemmP p = {};
  p.act = ACT_NONE;
  p.A = plain ? l.dy : dz, p.lda = ldz, p.ldc = l.K, p.N = l.K;
  if (l.dx) {
    p.B = o.w, p.B2 = o.w2, p.ldb = o.Kp, p.cb = o.Kp, p.kb = l.N, p.seg = GATED ? (int)(off / (4 * CH)) : 0;
    p.M = l.M, p.K = (int)ldz, p.C = l.dx;
    const int rc = gemm<T, EPI_LINEAR, false, true>(p, part, st);
    if (rc != MGGAN_OK) return rc;
  }
  if (l.dw) {
    p.ca = (int)ldz, p.B = o.x, p.ldb = o.ldx, p.cb = o.Kp, p.kb = l.M, p.seg = 0;
    p.M = mw, p.K = l.M, p.C = l.dw;
    const int rc = gemm<T, EPI_LINEAR, true, true>(p, part, st);
    if (rc != MGGAN_OK) return rc;
  }
  MG_LAUNCH_CHECK("block layer backward");
  return MGGAN_OK;
}

int layer(const BlkLayerArgs& l, bool gated, bool bwd, void* ws, size_t* need, hipStream_t st) {
  const Arena a = {(char*)ws, 0};
  if (l.dtype == BLK_BF16) {
    if (bwd) return gated ? layer_bwd<bf16, true>(l, a, need, st) : layer_bwd<bf16, false>(l, a, need, st);
    return gated ? layer_fwd<bf16, true>(l, a, need, st) : layer_fwd<bf16, false>(l, a, need, st);
  }
  if (bwd) return gated ? layer_bwd<float, true>(l, a, need, st) : layer_bwd<float, false>(l, a, need, st);
  return gated ? layer_fwd<float, true>(l, a, need, st) : layer_fwd<float, false>(l, a, need, st);
}

bool sizes_fit(int M, int K, int N) { return M > 0 && K > 0 && N > 0 && M <= (1 << 21) && K <= (1 << 20) && N <= (1 << 20); }

int check(const char* name, const BlkLayerArgs* a, bool bwd) {
  MG_CHECK_ARG(a, "%s: no arguments", name);
  const BlkLayerArgs& l = *a;
  const bool gated = l.w2 != nullptr;
  MG_CHECK_ARG(l.dtype == BLK_F32 || l.dtype == BLK_BF16, "%s: dtype %d (0 = f32, 1 = bf16)", name, l.dtype);
  MG_CHECK_ARG(sizes_fit(l.M, l.K, l.N), "%s: sizes %d x %d x %d (limits 2^21 x 2^20 x 2^20)", name, l.M, l.K, l.N);
  MG_CHECK_ARG(l.x && l.w, "%s: null operand", name);
  MG_CHECK_ARG((l.act >= ACT_NONE && l.act <= ACT_SIGMOID) || l.act == ACT_SILU || l.act == ACT_GELU, "%s: activation %d", name, l.act);
  const int ch = l.dtype == BLK_BF16 ? 8 : 4;
  MG_CHECK_ARG(l.ldx >= l.K && (l.K % ch || (l.ldx % ch == 0 && ((size_t)l.x | (size_t)l.w | (size_t)l.w2) % 16 == 0)),
               "%s: row stride %ld of %d columns, or an operand that is not 16-byte aligned", name, l.ldx, l.K);
  MG_CHECK_ARG(((size_t)l.b | (size_t)l.b2 | (size_t)l.res | (size_t)l.y | (size_t)l.z | (size_t)l.z2 | (size_t)l.dy | (size_t)l.dx | (size_t)l.dw) % 16 == 0,
               "%s: an operand or output is not 16-byte aligned", name);
  size_t need = 0;
  layer(l, gated, bwd, nullptr, &need, nullptr);
  MG_CHECK_ARG(!need || (l.ws && (size_t)l.ws_bytes >= need && (size_t)l.ws % 256 == 0), "%s: workspace of %zu bytes, 256-byte aligned (got %ld)",
               name, need, l.ws_bytes);
  return MGGAN_OK;
}

}  // namespace

extern "C" {

size_t mggan_block_layer_workspace(int rows, int K, int N, int gated, int backward, int act, int dtype) {
  if (!sizes_fit(rows, K, N)) return 0;
  BlkLayerArgs l = {};
  l.M = rows, l.K = K, l.N = N, l.ldx = K, l.act = act, l.dtype = dtype;
  size_t need = 0;
  layer(l, gated != 0, backward != 0, nullptr, &need, nullptr);
  return need;
}

int mggan_block_layer_fwd(const void* args, hipStream_t stream) {
  const BlkLayerArgs* l = (const BlkLayerArgs*)args;
  const int rc = check("block_layer_fwd", l, false);
  if (rc != MGGAN_OK) return rc;
  MG_CHECK_ARG(l->y && (!l->w2 || ((!l->z) == (!l->z2) && !l->res)), "block_layer_fwd: null output, one kept input of two, or a gated residual");
  return layer(*l, l->w2 != nullptr, false, l->ws, nullptr, stream);
}

int mggan_block_layer_bwd(const void* args, hipStream_t stream) {
  const BlkLayerArgs* l = (const BlkLayerArgs*)args;
  const int rc = check("block_layer_bwd", l, true);
  if (rc != MGGAN_OK) return rc;
  MG_CHECK_ARG(l->dy && (l->z || (l->act == ACT_NONE && !l->w2)) && (!l->w2 || l->z2), "block_layer_bwd: null gradient or activation input");
  return layer(*l, l->w2 != nullptr, true, l->ws, nullptr, stream);
}
}
