// The layers of a transformer block that are matrix products: linear with bias, activation and residual, and the gated layer
// act(x Wg^T + bg) * (x Wu^T + bu); forward and backward, f32 and bf16.
//
// One product does all of it: C[m][n] = sum_k A[m][k] B[n][k], both operands with k contiguous.  Forward: A = x, B = W.
// Backward: dX = dZ (W^T)^T and dW = dZ^T (x^T)^T; the pass that turns dY into dZ writes dZ^T beside it, W and x are transposed
// by a copy.  The gated layer takes its B rows from two weights, so that one wave holds the gate and the up value of the same
// outputs and multiplies them in registers.
#include "blk.h"
#include "../../include/mggan_hip.h"

namespace {

__device__ __attribute__((aligned(16))) const unsigned blk_zeros[4] = {0, 0, 0, 0};

struct GemmP {
  const void* A;
  const void* B;
  const void* B2;  // gated: the up weight
  long lda, ldb;   // elements; rows are 16-byte aligned
  int M, N, K;     // K: a multiple of the chunk (8 bf16 / 4 f32)
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

template <class T>
__device__ __forceinline__ void load8(const T* p, bool vec, int left, float (&v)[8]) {
  if (vec && left >= 8) {
    if constexpr (sizeof(T) == 2) {
      const bf16x8 x = *(const bf16x8*)p;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
    } else {
      const f32x4 x = *(const f32x4*)p, y = *(const f32x4*)(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = x[i], v[4 + i] = y[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? (float)p[i] : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, bool vec, int left, const float (&v)[8]) {
  if (vec && left >= 8) {
    if constexpr (sizeof(T) == 2) {
      bf16x8 x;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (bf16)v[i];
      *(bf16x8*)p = x;
    } else {
      f32x4 x, y;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = v[i], y[i] = v[4 + i];
      *(f32x4*)p = x;
      *(f32x4*)(p + 4) = y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (T)v[i];
  }
}

// The epilogue of eight neighbouring outputs of row m from column n on.
template <class T, int EPI>
__device__ __forceinline__ void epilogue8(const GemmP& p, int m, int n, float (&v)[8], float (&u)[8], bool vec) {
  const int left = p.N - n;
  if (left <= 0) return;
  float t[8];
  const long at = (long)m * p.N + n;
  if (p.bias) {
    load8<T>((const T*)p.bias + n, vec, left, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += t[i];
  }
  if (EPI == EPI_GATED && p.bias2) {
    load8<T>((const T*)p.bias2 + n, vec, left, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] += t[i];
  }
  if (p.Z) store8<float>(p.Z + at, vec, left, v);
  if (EPI == EPI_GATED && p.Z2) store8<float>(p.Z2 + at, vec, left, u);
  if (p.act != ACT_NONE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = blk_act(v[i], p.act, p.slope);
  }
  if (EPI == EPI_GATED) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= u[i];
  }
  if (p.res) {
    load8<T>((const T*)p.res + at, vec, left, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += t[i];
  }
  store8<T>((T*)p.C + (long)m * p.ldc + n, vec, left, v);
}

// Position of 16-byte chunk c of LDS row r: a wave reads 16 rows' chunks at once, either rows 0-15 or {0-3, 8-11, 16-19, 24-27}
// (+4); any eight lanes of either set fall on eight different positions, so the reads meet no bank twice.
__device__ __forceinline__ int swz(int r) { return (r & 7) ^ ((r >> 1) & 4); }

// A tile of BM x BN outputs, WM x WN waves; k in steps of 128 bytes a row, two LDS buffers: the copies of step t+1 are under way
// while step t is multiplied.
template <class T, int BM, int BN, int WM, int WN, int EPI, bool SPLIT>
__global__ __launch_bounds__(WM* WN * 64) void blk_gemm_kernel(GemmP p) {
  constexpr int NT = WM * WN * 64, CH = Mf<T>::CH;
  constexpr int LA = BM * 8 / NT, LB = BN * 8 / NT;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int NB = EPI == EPI_GATED ? BN / 2 : BN;  // output columns of the tile
  __shared__ u32x4 lds[2][(BM + BN) * 8];

  int t = blockIdx.x;
  {  // neighbouring tiles to the same XCD (blocks are dealt round the eight of them), in columns of eight row tiles
    const int nb = p.tiles_m * p.tiles_n, n8 = nb >> 3;
    if (t < n8 * 8) t = (t & 7) * n8 + (t >> 3);
  }
  const int per = 8 * p.tiles_n, grp = t / per, gm = min(8, p.tiles_m - 8 * grp), rem = t - grp * per;
  const int m0 = (8 * grp + rem % gm) * BM, n0 = (rem / gm) * NB;

  const int tid = threadIdx.x, lane = tid & 63, wave = mg_wave();
  const int c = (tid & 7) ^ swz(tid >> 3);  // this lane's chunk of every row it copies (rows differ by multiples of 16)
  const int nch = p.K / CH;
  const int kt0 = SPLIT ? blockIdx.y * p.kt_split : 0;
  const int kt1 = SPLIT ? min(kt0 + p.kt_split, (nch + 7) >> 3) : (nch + 7) >> 3;

  const char *sa[LA], *sb[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int row = (i * NT + tid) >> 3;
    sa[i] = (const char*)p.A + ((long)min(m0 + row, p.M - 1) * p.lda + (long)kt0 * 8 * CH) * sizeof(T) + c * 16;
  }
#pragma unroll
  for (int i = 0; i < LB; ++i) {
    const int row = (i * NT + tid) >> 3;
    const char* base = (const char*)(EPI == EPI_GATED && row >= NB ? p.B2 : p.B);
    const int r = EPI == EPI_GATED && row >= NB ? row - NB : row;
    sb[i] = base + ((long)min(n0 + r, p.N - 1) * p.ldb + (long)kt0 * 8 * CH) * sizeof(T) + c * 16;
  }
  auto fetch = [&](int kt, int buf) {
    u32x4* d = &lds[buf][wave * 64];
    if (kt * 8 + 8 <= nch) {
#pragma unroll
      for (int i = 0; i < LA; ++i) lds_copy16(sa[i], d + i * NT);
#pragma unroll
      for (int i = 0; i < LB; ++i) lds_copy16(sb[i], d + BM * 8 + i * NT);
    } else {  // the last step of a reduction that is no multiple of 128 bytes: chunks past its end come from a page of zeros
      const bool in = kt * 8 + c < nch;
#pragma unroll
      for (int i = 0; i < LA; ++i) lds_copy16(in ? sa[i] : (const char*)blk_zeros, d + i * NT);
#pragma unroll
      for (int i = 0; i < LB; ++i) lds_copy16(in ? sb[i] : (const char*)blk_zeros, d + BM * 8 + i * NT);
    }
#pragma unroll
    for (int i = 0; i < LA; ++i) sa[i] += 128;
#pragma unroll
    for (int i = 0; i < LB; ++i) sb[i] += 128;
  };

  f32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int wm = wave % WM, wn = wave / WM, i16 = lane & 15, g = lane >> 4;
  const int ra = wm * TM + i16, ha = swz(i16);
  int rb[FN];
#pragma unroll
  for (int f = 0; f < FN; ++f) {
    const int q = EPI == EPI_GATED ? f % (FN / 2) : f;
    rb[f] = (EPI == EPI_GATED ? (f / (FN / 2)) * NB + wn * (TN / 2) : wn * TN) + 32 * (q >> 1) + 8 * (i16 >> 2) + 4 * (q & 1) + (i16 & 3);
  }

  if (kt0 < kt1) fetch(kt0, 0);
  for (int kt = kt0; kt < kt1; ++kt) {
    const int buf = (kt - kt0) & 1;
    __syncthreads();  // (waits for this step's copies; everyone is done reading the other buffer)
    if (kt + 1 < kt1) fetch(kt + 1, buf ^ 1);
    const u32x4* la = &lds[buf][0];
    const u32x4* lb = &lds[buf][BM * 8];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 fa[FM], fb[FN];
#pragma unroll
      for (int j = 0; j < FM; ++j) fa[j] = la[(ra + 16 * j) * 8 + ((4 * s + g) ^ ha)];
#pragma unroll
      for (int i = 0; i < FN; ++i) fb[i] = lb[rb[i] * 8 + ((4 * s + g) ^ swz(rb[i]))];
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = Mf<T>::step(fb[i], fa[j], acc[i][j]);
    }
  }

  constexpr int FO = EPI == EPI_GATED ? FN / 2 : FN;
  const bool vec = p.N % (EPI == EPI_GATED || !SPLIT ? CH : 4) == 0;
  float u[8];
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int m = m0 + wm * TM + 16 * j + i16;
    if (m >= p.M) continue;
#pragma unroll
    for (int f = 0; f < FO; f += 2) {
      const int n = n0 + wn * (FO * 16) + 16 * f + 8 * g;
      float v[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = acc[f][j][r], v[4 + r] = acc[f + 1][j][r];
      if (EPI == EPI_GATED) {
#pragma unroll
        for (int r = 0; r < 4; ++r) u[r] = acc[FO + f][j][r], u[4 + r] = acc[FO + f + 1][j][r];
      }
      if (SPLIT) {
        const long cols = EPI == EPI_GATED ? 2L * p.N : p.N;
        float* out = p.part + ((long)blockIdx.y * p.M + m) * cols + n;
        store8<float>(out, vec, p.N - n, v);
        if (EPI == EPI_GATED) store8<float>(out + p.N, vec, p.N - n, u);
      } else {
        epilogue8<T, EPI>(p, m, n, v, u, vec);
      }
    }
  }
}

// The partial sums of a split reduction joined in their order, then the epilogue; eight outputs a thread.
template <class T, int EPI>
__global__ __launch_bounds__(256) void blk_join_kernel(GemmP p, int splits) {
  const int per = (p.N + 7) >> 3;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long)per * p.M) return;
  const int m = (int)(id / per), n = (int)(id % per) * 8;
  const long cols = EPI == EPI_GATED ? 2L * p.N : p.N;
  const bool vec4 = p.N % 4 == 0;
  float v[8] = {}, u[8] = {}, t[8];
  for (int s = 0; s < splits; ++s) {
    const float* in = p.part + ((long)s * p.M + m) * cols + n;
    load8<float>(in, vec4, p.N - n, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += t[i];
    if (EPI == EPI_GATED) {
      load8<float>(in + p.N, vec4, p.N - n, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] += t[i];
    }
  }
  epilogue8<T, EPI>(p, m, n, v, u, p.N % Mf<T>::CH == 0);
}

// Rows of `cols` elements into rows of `ldo` (>= cols), the rest zeros.
template <class T>
__global__ __launch_bounds__(256) void blk_pad_kernel(const T* in, long ldi, T* out, long ldo, int rows, int cols) {
  for (long id = (long)blockIdx.x * 256 + threadIdx.x; id < (long)rows * ldo; id += (long)gridDim.x * 256) {
    const long r = id / ldo, cc = id - r * ldo;
    out[id] = cc < cols ? in[r * ldi + cc] : (T)0.f;
  }
}

// out[c][r] = in[r][c] in tiles of 64 x 64 through LDS; zeros for r in [rows, rpad).
template <class T>
__global__ __launch_bounds__(256) void blk_transpose_kernel(const T* in, long ldi, T* out, long ldo, int rows, int cols, int rpad) {
  __shared__ T tile[64][65];
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
#pragma unroll 4
  for (int i = y; i < 64; i += 4) tile[i][x] = r0 + i < rows && c0 + x < cols ? in[(long)(r0 + i) * ldi + c0 + x] : (T)0.f;
  __syncthreads();
#pragma unroll 4
  for (int i = y; i < 64; i += 4)
    if (c0 + i < cols && r0 + x < rpad) out[(long)(c0 + i) * ldo + r0 + x] = tile[x][i];
}

// dY -> dZ = dY act'(z) (linear) or dG = dY u act'(g), dU = dY act(g) (gated), as rows (ld ldz, dU `off` behind dG, zeros up to
// there) and transposed (ld ldt), and each tile's column sums in f32 for the bias gradients.  dZ is rounded to the operands'
// type once: it is an operand of both products, and half a step is what every operand has.
struct DzP {
  const void* dY;
  const float* Z;
  const float* Z2;
  void* dZ;
  void* dZt;
  float* sums;  // (tiles of rows, N or 2 N)
  int M, N, act;
  float slope;
  long ldz, off, ldt;
};
template <class T, bool GATED>
__global__ __launch_bounds__(256) void blk_dz_kernel(DzP p) {
  __shared__ T tile[GATED ? 2 : 1][64][65];
  __shared__ float part[4][GATED ? 2 : 1][64];
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const int n = c0 + x;
  float s0 = 0.f, s1 = 0.f;
#pragma unroll 4
  for (int i = y; i < 64; i += 4) {
    const int m = r0 + i;
    float a = 0.f, b = 0.f;
    if (m < p.M && n < p.N) {
      const long at = (long)m * p.N + n;
      const float dy = (float)((const T*)p.dY)[at];
      if (GATED) {
        const float z = p.Z[at], u = p.Z2[at];
        a = dy * u * blk_act_grad(z, p.act, p.slope);
        b = dy * blk_act(z, p.act, p.slope);
      } else {
        a = p.Z ? dy * blk_act_grad(p.Z[at], p.act, p.slope) : dy;
      }
    }
    s0 += a;
    s1 += b;
    tile[0][i][x] = (T)a;
    if (GATED) tile[GATED][i][x] = (T)b;
    if (m < p.M && n < (GATED ? p.off : p.ldz)) {
      if (p.dZ) {
        ((T*)p.dZ)[m * p.ldz + n] = (T)a;
        if (GATED) ((T*)p.dZ)[m * p.ldz + p.off + n] = (T)b;
      }
    }
  }
  part[y][0][x] = s0;
  if (GATED) part[y][GATED][x] = s1;
  __syncthreads();
  if (p.dZt) {
#pragma unroll 4
    for (int i = y; i < 64; i += 4)
      if (c0 + i < p.N && r0 + x < p.ldt) {
        ((T*)p.dZt)[(long)(c0 + i) * p.ldt + r0 + x] = tile[0][x][i];
        if (GATED) ((T*)p.dZt)[(long)(p.N + c0 + i) * p.ldt + r0 + x] = tile[GATED][x][i];
      }
  }
  if (p.sums && y < (GATED ? 2 : 1) && n < p.N) {
    const long cols = GATED ? 2L * p.N : p.N;
    p.sums[blockIdx.y * cols + (long)y * p.N + n] = (part[0][y][x] + part[1][y][x]) + (part[2][y][x] + part[3][y][x]);
  }
}

// Column sums of (rows, cols) partials in a fixed order, rounded to the bias' type.
template <class T>
__global__ __launch_bounds__(256) void blk_colsum_kernel(const float* in, int rows, int cols, T* out) {
  __shared__ float part[4][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), y = threadIdx.x >> 6;
  float s = 0.f;
  if (c < cols)
    for (int r = y; r < rows; r += 4) s += in[(long)r * cols + c];
  part[y][threadIdx.x & 63] = s;
  __syncthreads();
  if (y == 0 && c < cols) out[c] = (T)((part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]));
}

// ---- host side -------------------------------------------------------------------------------------------------------------

inline long up(long a, long b) { return (a + b - 1) / b * b; }

// Tile and split of one product; workspace for the partial sums.
struct Plan {
  int bm, bn, splits, kt_split;
  size_t bytes;
};
Plan plan_of(int M, int N, long K, int ch, bool gated) {
  Plan q;
  auto tiles = [&](int b, int n) { return (long)cdiv(M, b) * cdiv(N, n); };
  const int half = gated ? 2 : 1;
  q.bm = tiles(256, 256 / half) >= 192 ? 256 : tiles(128, 128 / half) >= 192 ? 128 : 64;
  q.bn = q.bm;
  const long nt = tiles(q.bm, q.bn / half), kts = (K / ch + 7) / 8;
  q.splits = 1;
  if (nt < 192) {
    const long want = cdiv(256, nt), most = kts / 4;
    q.splits = (int)(want < most ? want : most);
    if (q.splits > 32) q.splits = 32;
    if (q.splits < 1) q.splits = 1;
  }
  q.kt_split = (int)((kts + q.splits - 1) / q.splits);
  q.splits = (int)((kts + q.kt_split - 1) / q.kt_split);
  q.bytes = q.splits > 1 ? (size_t)q.splits * M * N * half * 4 : 0;
  return q;
}

template <class T, int B, int WM, int WN, int EPI>
int gemm_tile(GemmP& p, const Plan& q, hipStream_t st) {
  p.tiles_m = cdiv(p.M, B);
  p.tiles_n = cdiv(p.N, EPI == EPI_GATED ? B / 2 : B);
  p.kt_split = q.kt_split;
  if (q.splits > 1) {
    MG_LAUNCH((blk_gemm_kernel<T, B, B, WM, WN, EPI, true>), dim3(p.tiles_m * p.tiles_n, q.splits), dim3(WM * WN * 64), 0, st, p);
    MG_LAUNCH((blk_join_kernel<T, EPI>), dim3(cdiv((long)cdiv(p.N, 8) * p.M, 256)), dim3(256), 0, st, p, q.splits);
  } else {
    MG_LAUNCH((blk_gemm_kernel<T, B, B, WM, WN, EPI, false>), dim3(p.tiles_m * p.tiles_n), dim3(WM * WN * 64), 0, st, p);
  }
  MG_LAUNCH_CHECK("block gemm");
  return MGGAN_OK;
}
template <class T, int EPI>
int gemm(GemmP p, void* ws, hipStream_t st) {
  const Plan q = plan_of(p.M, p.N, p.K, Mf<T>::CH, EPI == EPI_GATED);
  p.part = (float*)ws;
  switch (q.bm) {
    case 256: return gemm_tile<T, 256, 2, 4, EPI>(p, q, st);
    case 128: return gemm_tile<T, 128, 2, 2, EPI>(p, q, st);
    default: return gemm_tile<T, 64, 4, 1, EPI>(p, q, st);
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
template <class T>
void transpose(const void* in, long ldi, void* out, long ldo, int rows, int cols, int rpad, hipStream_t st) {
  MG_LAUNCH((blk_transpose_kernel<T>), dim3(cdiv(cols, 64), cdiv(rpad, 64)), dim3(256), 0, st, (const T*)in, ldi, (T*)out, ldo, rows, cols, rpad);
}

struct LayerP {
  const void *x, *w, *w2, *b, *b2, *res, *dy;
  long ldx;
  float *z, *z2;
  void *y, *dx, *dw, *db;
  int M, K, N, act;
  float slope;
};

template <class T, int EPI>
int layer_fwd(const LayerP& l, Arena ws, size_t* need, hipStream_t st) {
  constexpr int CH = Mf<T>::CH;
  const int Kp = (int)up(l.K, CH);
  const bool odd = Kp != l.K;
  const bool px = odd || l.ldx % CH || (size_t)l.x % 16, pw = odd || (size_t)l.w % 16 || (EPI == EPI_GATED && (size_t)l.w2 % 16);
  // (what the size asks for does not depend on the pointers: the workspace holds the padded operands in every case)
  void* xp = ws.take((size_t)l.M * Kp * sizeof(T));
  void* wp = ws.take((size_t)l.N * Kp * sizeof(T));
  void* wp2 = EPI == EPI_GATED ? ws.take((size_t)l.N * Kp * sizeof(T)) : nullptr;
  void* part = ws.take(plan_of(l.M, l.N, Kp, CH, EPI == EPI_GATED).bytes);
  if (need) {
    *need = ws.at;
    return MGGAN_OK;
  }
  if (px) pad<T>(l.x, l.ldx, xp, Kp, l.M, l.K, st);
  if (pw) {
    pad<T>(l.w, l.K, wp, Kp, l.N, l.K, st);
    if (EPI == EPI_GATED) pad<T>(l.w2, l.K, wp2, Kp, l.N, l.K, st);
  }
  GemmP p = {};
  p.A = px ? xp : l.x, p.lda = px ? Kp : l.ldx;
  p.B = pw ? wp : l.w, p.B2 = pw ? wp2 : l.w2, p.ldb = Kp;
  p.M = l.M, p.N = l.N, p.K = Kp;
  p.C = l.y, p.ldc = l.N, p.Z = l.z, p.Z2 = l.z2, p.bias = l.b, p.bias2 = l.b2, p.res = l.res, p.act = l.act, p.slope = l.slope;
  return gemm<T, EPI>(p, part, st);
}

template <class T, bool GATED>
int layer_bwd(const LayerP& l, Arena ws, size_t* need, hipStream_t st) {
  constexpr int CH = Mf<T>::CH, two = GATED ? 2 : 1;
  const long Np = up(l.N, CH), Mp = up(l.M, CH), tiles = cdiv(l.M, 64);
  void* dz = ws.take((size_t)l.M * two * Np * sizeof(T));
  void* dzt = ws.take((size_t)two * l.N * Mp * sizeof(T));
  void* wt = ws.take((size_t)l.K * two * Np * sizeof(T));
  void* xt = ws.take((size_t)l.K * Mp * sizeof(T));
  float* sums = (float*)ws.take((size_t)tiles * two * l.N * 4);
  const size_t p1 = plan_of(l.M, l.K, two * Np, CH, false).bytes, p2 = plan_of(two * l.N, l.K, Mp, CH, false).bytes;
  void* part = ws.take(p1 > p2 ? p1 : p2);
  if (need) {
    *need = ws.at;
    return MGGAN_OK;
  }
  DzP d = {};
  d.dY = l.dy, d.Z = l.z, d.Z2 = l.z2, d.dZ = l.dx ? dz : nullptr, d.dZt = l.dw ? dzt : nullptr, d.sums = l.db ? sums : nullptr;
  d.M = l.M, d.N = l.N, d.act = l.act, d.slope = l.slope, d.ldz = two * Np, d.off = Np, d.ldt = Mp;
  MG_LAUNCH((blk_dz_kernel<T, GATED>), dim3(cdiv(Np, 64), cdiv(Mp, 64)), dim3(256), 0, st, d);
  if (l.db) MG_LAUNCH((blk_colsum_kernel<T>), dim3(cdiv((long)two * l.N, 64)), dim3(256), 0, st, (const float*)sums, (int)tiles, two * l.N, (T*)l.db);
  GemmP p = {};
  p.act = ACT_NONE;
  if (l.dx) {
    transpose<T>(l.w, l.K, wt, two * Np, l.N, l.K, (int)Np, st);
    if (GATED) transpose<T>(l.w2, l.K, (T*)wt + Np, two * Np, l.N, l.K, (int)Np, st);
    p.A = dz, p.lda = two * Np, p.B = wt, p.ldb = two * Np, p.M = l.M, p.N = l.K, p.K = (int)(two * Np), p.C = l.dx, p.ldc = l.K;
    const int rc = gemm<T, EPI_LINEAR>(p, part, st);
    if (rc != MGGAN_OK) return rc;
  }
  if (l.dw) {
    transpose<T>(l.x, l.ldx, xt, Mp, l.M, l.K, (int)Mp, st);
    p.A = dzt, p.lda = Mp, p.B = xt, p.ldb = Mp, p.M = two * l.N, p.N = l.K, p.K = (int)Mp, p.C = l.dw, p.ldc = l.K;
    const int rc = gemm<T, EPI_LINEAR>(p, part, st);
    if (rc != MGGAN_OK) return rc;
  }
  MG_LAUNCH_CHECK("block layer backward");
  return MGGAN_OK;
}

int layer(const LayerP& l, bool gated, bool bwd, int dtype, void* ws, size_t* need, hipStream_t st) {
  const Arena a = {(char*)ws, 0};
  if (dtype == BLK_BF16) {
    if (bwd) return gated ? layer_bwd<bf16, true>(l, a, need, st) : layer_bwd<bf16, false>(l, a, need, st);
    return gated ? layer_fwd<bf16, EPI_GATED>(l, a, need, st) : layer_fwd<bf16, EPI_LINEAR>(l, a, need, st);
  }
  if (bwd) return gated ? layer_bwd<float, true>(l, a, need, st) : layer_bwd<float, false>(l, a, need, st);
  return gated ? layer_fwd<float, EPI_GATED>(l, a, need, st) : layer_fwd<float, EPI_LINEAR>(l, a, need, st);
}

int check(const char* name, const LayerP& l, int dtype, const void* ws, size_t ws_bytes, bool gated, bool bwd) {
  MG_CHECK_ARG(dtype == BLK_F32 || dtype == BLK_BF16, "%s: dtype %d (0 = f32, 1 = bf16)", name, dtype);
  MG_CHECK_ARG(l.M > 0 && l.K > 0 && l.N > 0, "%s: sizes %d x %d x %d", name, l.M, l.K, l.N);
  MG_CHECK_ARG(l.M <= (1 << 21) && l.K <= (1 << 20) && l.N <= (1 << 20), "%s: sizes %d x %d x %d over the limits 2^21 x 2^20 x 2^20", name,
               l.M, l.K, l.N);
  MG_CHECK_ARG(l.ldx >= l.K, "%s: row stride %ld below %d", name, l.ldx, l.K);
  MG_CHECK_ARG(l.x && l.w && (!gated || l.w2), "%s: null operand", name);
  MG_CHECK_ARG((l.act >= ACT_NONE && l.act <= ACT_SIGMOID) || l.act == ACT_SILU || l.act == ACT_GELU, "%s: activation %d", name, l.act);
  MG_CHECK_ARG(((size_t)l.b | (size_t)l.b2 | (size_t)l.res | (size_t)l.y | (size_t)l.z | (size_t)l.z2 | (size_t)l.dx | (size_t)l.dw) % 16 == 0,
               "%s: bias, residual, outputs and kept inputs have to be 16-byte aligned", name);
  size_t need = 0;
  layer(l, gated, bwd, dtype, nullptr, &need, nullptr);
  MG_CHECK_ARG(ws && ws_bytes >= need && (size_t)ws % 256 == 0, "%s: workspace of %zu bytes, 256-byte aligned (got %zu)", name, need, ws_bytes);
  return MGGAN_OK;
}

}  // namespace

extern "C" {

size_t mggan_block_layer_workspace(int rows, int K, int N, int gated, int backward, int dtype) {
  if (rows <= 0 || K <= 0 || N <= 0) return 0;
  LayerP l = {};
  l.M = rows, l.K = K, l.N = N, l.ldx = K;
  size_t need = 0;
  layer(l, gated != 0, backward != 0, dtype, nullptr, &need, nullptr);
  return need;
}

int mggan_block_linear_fwd(const void* x, long ldx, const void* w, const void* bias, const void* residual, void* y, float* z, int rows, int K,
                           int N, int act, float slope, int dtype, void* ws, size_t ws_bytes, hipStream_t stream) {
  LayerP l = {};
  l.x = x, l.ldx = ldx, l.w = w, l.b = bias, l.res = residual, l.y = y, l.z = z, l.M = rows, l.K = K, l.N = N, l.act = act, l.slope = slope;
  const int rc = check("block_linear_fwd", l, dtype, ws, ws_bytes, false, false);
  if (rc != MGGAN_OK) return rc;
  MG_CHECK_ARG(y, "block_linear_fwd: null output");
  return layer(l, false, false, dtype, ws, nullptr, stream);
}

int mggan_block_linear_bwd(const void* dy, const float* z, const void* x, long ldx, const void* w, void* dx, void* dw, void* db, int rows, int K,
                           int N, int act, float slope, int dtype, void* ws, size_t ws_bytes, hipStream_t stream) {
  LayerP l = {};
  l.dy = dy, l.z = (float*)z, l.x = x, l.ldx = ldx, l.w = w, l.dx = dx, l.dw = dw, l.db = db, l.M = rows, l.K = K, l.N = N, l.act = act,
  l.slope = slope;
  const int rc = check("block_linear_bwd", l, dtype, ws, ws_bytes, false, true);
  if (rc != MGGAN_OK) return rc;
  MG_CHECK_ARG(dy && (z || act == ACT_NONE), "block_linear_bwd: null gradient or activation input");
  return layer(l, false, true, dtype, ws, nullptr, stream);
}

int mggan_block_gated_fwd(const void* x, long ldx, const void* w_gate, const void* w_up, const void* b_gate, const void* b_up, void* y, float* z_gate,
                          float* z_up, int rows, int K, int N, int act, float slope, int dtype, void* ws, size_t ws_bytes, hipStream_t stream) {
  LayerP l = {};
  l.x = x, l.ldx = ldx, l.w = w_gate, l.w2 = w_up, l.b = b_gate, l.b2 = b_up, l.y = y, l.z = z_gate, l.z2 = z_up, l.M = rows, l.K = K, l.N = N;
  l.act = act, l.slope = slope;
  const int rc = check("block_gated_fwd", l, dtype, ws, ws_bytes, true, false);
  if (rc != MGGAN_OK) return rc;
  MG_CHECK_ARG(y && (!z_gate) == (!z_up), "block_gated_fwd: null output, or one of the two kept inputs only");
  return layer(l, true, false, dtype, ws, nullptr, stream);
}

int mggan_block_gated_bwd(const void* dy, const float* z_gate, const float* z_up, const void* x, long ldx, const void* w_gate, const void* w_up,
                          void* dx, void* dw, void* db, int rows, int K, int N, int act, float slope, int dtype, void* ws, size_t ws_bytes,
                          hipStream_t stream) {
  LayerP l = {};
  l.dy = dy, l.z = (float*)z_gate, l.z2 = (float*)z_up, l.x = x, l.ldx = ldx, l.w = w_gate, l.w2 = w_up, l.dx = dx, l.dw = dw, l.db = db;
  l.M = rows, l.K = K, l.N = N, l.act = act, l.slope = slope;
  const int rc = check("block_gated_bwd", l, dtype, ws, ws_bytes, true, true);
  if (rc != MGGAN_OK) return rc;
  MG_CHECK_ARG(dy && z_gate && z_up, "block_gated_bwd: null gradient or activation input");
  return layer(l, true, true, dtype, ws, nullptr, stream);
}
}
