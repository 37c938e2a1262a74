// The linear layer y = act(x W^T + b) + r (models.py's fc1..fc4 at any size and
// type), its gradients and its form for a few rows.
//
//   z = x W^T + b,  y = act(z) + r             act: none, relu, gelu (erf), silu
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// One tile kernel serves the three products: each operand is either "kc" (the
// reduction index runs along memory: x and W of the forward pass, dz of dx) or
// "ks" (it runs down the rows: W of dx, both of dW); the ks operands of 16-bit
// types are transposed on their way out of LDS (ds_read_tr16_b64), so no
// transposed copy is ever written.  Sums are fp32 in the matrix cores'
// accumulators from the first product to the epilogue; the one rounding to the
// element type is the store.
#include "cit_ops.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 fp16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((__vector_size__(8)));

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

// Phi(z) = erfc(-z / sqrt(2)) / 2 and exp(-z^2 / 2).  fp32 takes the library's erfc
// (no cancellation at z < 0).  For 16-bit results it is Abramowitz and
// Stegun's 7.1.26, off by at most 0.75e-7 absolute, whose exponential gelu's
// derivative needs anyhow: a fifth of the instructions.
template <typename T>
__device__ __forceinline__ void normal_cdf(float z, float& cdf, float& e) {
  if (sizeof(T) == 4) {
    e = expf(-0.5f * z * z);
    cdf = 0.5f * erfcf(-z * 0.70710678118654752f);
    return;
  }
  e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(fmaf(x, 0.3275911f, 1.0f));
  float p = fmaf(t, 1.061405429f, -1.453152027f);
  p = fmaf(t, p, 1.421413741f);
  p = fmaf(t, p, -0.284496736f);
  p = fmaf(t, p, 0.254829592f);
  const float tail = 0.5f * p * t * e;
  cdf = z < 0.0f ? tail : 1.0f - tail;
}
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  if (sizeof(T) == 4) return 1.0f / (1.0f + expf(-z));
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}

template <typename T>
__device__ __forceinline__ float act_fwd(int act, float z) {
  if (act == ACT_RELU) return z < 0.0f ? 0.0f : z;                  // NaN stays
  if (act == ACT_GELU) {
    float cdf, e;
    normal_cdf<T>(z, cdf, e);
    return z * cdf;
  }
  if (act == ACT_SILU) return z * sigmoid<T>(z);
  return z;
}
template <typename T>
__device__ __forceinline__ float act_grad(int act, float z) {
  if (act == ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (act == ACT_GELU) {
    float cdf, e;
    normal_cdf<T>(z, cdf, e);
    return fmaf(z * 0.39894228040143268f, e, cdf);
  }
  if (act == ACT_SILU) {
    const float s = sigmoid<T>(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  return 1.0f;
}

// z kept for the backward pass in the element type.  The rounding is to
// nearest, except that a finite z stays finite and a nonzero one nonzero: relu
// asks for its sign (fp16 underflows below 2^-25), and gelu's z * exp(-z^2 / 2)
// is inf * 0 at an infinity that only the rounding made.
template <typename T> __device__ __forceinline__ T keep_z(float z) { return from_f<T>(z); }
template <> __device__ __forceinline__ fp16_t keep_z<fp16_t>(float z) {
  const float a = fabsf(z);
  if (a > 65504.0f && a <= 3.4028234663852886e38f) return (fp16_t)copysignf(65504.0f, z);
  if (a < 5.9604644775390625e-08f && a > 0.0f) return (fp16_t)copysignf(5.9604644775390625e-08f, z);
  return (fp16_t)z;
}
template <> __device__ __forceinline__ bf16_t keep_z<bf16_t>(float z) {
  if (fabsf(z) > 3.3895313892515355e38f && fabsf(z) <= 3.4028234663852886e38f)
    return (bf16_t)copysignf(3.3895313892515355e38f, z);
  return (bf16_t)z;
}

struct Epilogue {               // what follows a product's sum at row m, column n
  const void* bias;             // [N] or null
  const void* res;              // [M][ldr] or null
  void* out;                    // [M][ldo]
  void* z;                      // [M][N] pre-activation for the backward pass, or null
  float* part;                  // split sums: [split][M][N] fp32 instead of out
  int64_t ldr, ldo;
  int act;
};

template <typename T>
__device__ __forceinline__ void finish(const Epilogue& e, int64_t m, int n, int N, float v) {
  if (e.bias) v += to_f(static_cast<const T*>(e.bias)[n]);
  if (e.z) static_cast<T*>(e.z)[m * N + n] = keep_z<T>(v);
  v = act_fwd<T>(e.act, v);
  if (e.res) v += to_f(static_cast<const T*>(e.res)[m * e.ldr + n]);
  static_cast<T*>(e.out)[m * e.ldo + n] = from_f<T>(v);
}

// Eight neighbouring columns of one row, from n on (those inside N).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  Pack16<T> u[sizeof(T) / 2];
#pragma unroll
  for (int h = 0; h < (int)sizeof(T) / 2; h++) u[h].raw = load16(p + h * Pack16<T>::N);
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = to_f(u[i / Pack16<T>::N].e[i % Pack16<T>::N]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const T (&v)[8]) {
  Pack16<T> u[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < 8; i++) u[i / Pack16<T>::N].e[i % Pack16<T>::N] = v[i];
#pragma unroll
  for (int h = 0; h < (int)sizeof(T) / 2; h++) store16(p + h * Pack16<T>::N, u[h].raw);
}

template <typename T>
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t m, int n, int N, float (&v)[8], int split,
                                        int64_t M) {
  if (e.part) {
    float* p = e.part + ((int64_t)split * M + m) * N + n;
    if (n + 8 <= N) {
      store8<float>(p, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (n + i < N) p[i] = v[i];
    }
    return;
  }
  if (n + 8 > N) {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (n + i < N) finish<T>(e, m, n + i, N, v[i]);
    return;
  }
  float t[8];
  T o[8];
  if (e.bias) {
    load8<T>(static_cast<const T*>(e.bias) + n, t);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += t[i];
  }
  if (e.z) {
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = keep_z<T>(v[i]);
    store8<T>(static_cast<T*>(e.z) + m * N + n, o);
  }
  if (e.act != ACT_NONE) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = act_fwd<T>(e.act, v[i]);
  }
  if (e.res) {
    load8<T>(static_cast<const T*>(e.res) + m * e.ldr + n, t);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += t[i];
  }
#pragma unroll
  for (int i = 0; i < 8; i++) o[i] = from_f<T>(v[i]);
  store8<T>(static_cast<T*>(e.out) + m * e.ldo + n, o);
}

// A wave's sums, TM x TN blocks of 16 x 16 from (m0, n0) on, through its own
// `bytes` of LDS so that rows leave in whole lines: a lane holds 4 columns of
// one row (a 16-byte chunk; chunks permuted by the row against bank conflicts) and
// writes out 8.  B went into the products as the instruction's rows, hence the
// neighbouring columns.
template <typename T, int TM, int TN, int BYTES>
__device__ __forceinline__ void write_out(const Epilogue& e, const f32x4 (&acc)[TM][TN], char* lds, int m0, int n0,
                                          int M, int N, int split) {
  constexpr int ROW = TN * 64, CHUNKS = TN * 4;                        // bytes and chunks of a row
  constexpr int FIT = BYTES / (16 * ROW), PER = FIT < TM ? FIT : TM;   // row blocks of a pass
  static_assert(PER >= 1, "a row block fits");
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int i0 = 0; i0 < TM; i0 += PER) {
#pragma unroll
    for (int i = i0; i < i0 + PER && i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) {
        const int r = (i - i0) * 16 + (l & 15), c = j * 4 + (l >> 4);
        *reinterpret_cast<f32x4*>(lds + r * ROW + ((c ^ (r & (CHUNKS - 1))) << 4)) = acc[i][j];
      }
    const int rows = (TM - i0 < PER ? TM - i0 : PER) * 16;
    for (int k = l; k < rows * (CHUNKS / 2); k += 64) {
      const int r = k / (CHUNKS / 2), c = k % (CHUNKS / 2) * 2, x = r & (CHUNKS - 1);
      const int m = m0 + i0 * 16 + r, n = n0 + c * 4;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(lds + r * ROW + ((c ^ x) << 4));
      const f32x4 hi = *reinterpret_cast<const f32x4*>(lds + r * ROW + (((c + 1) ^ x) << 4));
      if (m < M && n < N) {
        float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        finish8<T>(e, m, n, N, v, split, M);
      }
    }
  }
}

// ---- operand tiles ------------------------------------------------------------
//
// A tile holds R rows (of the output's m or n) by 128 bytes of the reduction:
// BK = 64 16-bit or 32 32-bit elements.  kc tiles lie as [R][128 B], ks tiles as
// [BK][R elements]; both are R * 128 bytes in chunks of 16, and a row's chunks
// are permuted (xor) so that the lanes of one LDS read, which walk down rows
// or along k, meet different banks.

template <typename T> constexpr int BK = 128 / (int)sizeof(T);

template <typename T, bool KS, int R>
struct Tile {
  static constexpr int E = 16 / sizeof(T);            // elements of a chunk
  static constexpr int CPR = KS ? R / E : 8;          // chunks of a tile row
  static constexpr int CHUNKS = R * 8;

  __device__ static __forceinline__ int swz(int row) {
    if (!KS) return row & 7;
    return sizeof(T) == 2 ? (row & 3) << 1 : ((row >> 2) & 3) << 2;
  }
  // Byte offset of the 16-byte chunk c of tile row `row`.
  __device__ static __forceinline__ int at(int row, int c) { return (row * CPR + (c ^ swz(row))) << 4; }

  // Global chunk behind LDS chunk `id`: (tile row, chunk of the row).
  __device__ static __forceinline__ void from(int id, int& row, int& c) {
    row = id / CPR;
    c = (id % CPR) ^ swz(row);
  }
};

// A matrix of `rows` x `cols` elements, ld elements apart.
struct Mat {
  const void* p;
  int64_t ld;
  int rows, cols;
};

// 16 bytes of row r from column c on, zero outside the matrix: any alignment.
template <typename T>
__device__ __forceinline__ u32x4 fetch(const Mat& a, int r, int c) {
  constexpr int E = 16 / sizeof(T);
  Pack16<T> v;
  v.raw = u32x4{0, 0, 0, 0};
  if (r < a.rows && c < a.cols) {
    const T* p = static_cast<const T*>(a.p) + (int64_t)r * a.ld + c;
    if (c + E <= a.cols) {
      v.raw = load16(p);
    } else {
#pragma unroll
      for (int i = 0; i < E; i++)
        if (c + i < a.cols) v.e[i] = p[i];
    }
  }
  return v.raw;
}

// Loads of one thread for one tile, through registers (THREADS threads).
template <typename T, bool KS, int R, int THREADS>
struct Stage {
  typedef Tile<T, KS, R> L;
  static constexpr int PER = L::CHUNKS / THREADS;
  u32x4 v[PER];
  __device__ __forceinline__ void load(const Mat& a, int r0, int k0) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      int row, c;
      L::from(i * THREADS + (int)threadIdx.x, row, c);
      v[i] = KS ? fetch<T>(a, k0 + row, r0 + c * L::E) : fetch<T>(a, r0 + row, k0 + c * L::E);
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < PER; i++)
      *reinterpret_cast<u32x4*>(lds + ((i * THREADS + (int)threadIdx.x) << 4)) = v[i];
  }
};

// ---- matrix instructions --------------------------------------------------------

__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, fp16_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fp16x8, a), __builtin_bit_cast(fp16x8, b), c, 0, 0,
                                                0);
}
// Four k of each lane: the k a lane group holds differ from the instruction's
// own order, but A and B hold the same ones, and a sum has no order.
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, float) {
  const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
  return c;
}

typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// The 16 rows from `r0` on of a tile, k step s (32 16-bit or 16 32-bit
// elements): lane l holds row r0 + l % 16 and its quarter l / 16 of the k.
template <typename T, bool KS, int R>
__device__ __forceinline__ u32x4 frag(const char* lds, int r0, int s) {
  typedef Tile<T, KS, R> L;
  const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
  if (!KS) return *reinterpret_cast<const u32x4*>(lds + L::at(r0 + i, s * 4 + g));
  if (sizeof(T) == 2) {
    // Two transposing reads of 4 k x 16 rows: lane i of a group reads 4 elements
    // of k row i / 4 and receives the 4 k of row i.
    union { u32x4 raw; s16x4 h[2]; } v;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int k = s * 32 + g * 8 + h * 4 + (i >> 2);
      const int off = L::at(k, (r0 >> 3) + ((i & 3) >> 1)) + ((i & 1) << 3);
      v.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(lds + off));
    }
    return v.raw;
  }
  union { u32x4 raw; float f[4]; } v;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int k = s * 16 + g * 4 + j, c = r0 + i;
    v.f[j] = *reinterpret_cast<const float*>(lds + L::at(k, c >> 2) + ((c & 3) << 2));
  }
  return v.raw;
}

// ---- the tile kernel ------------------------------------------------------------
//
// Workgroup (tile, split): BM x BN outputs by WM x WN waves, over the split's
// share of the reduction.  Two LDS buffers: while the matrix cores work on one
// tile, the next one's loads are in flight.

template <typename T, bool AKS, bool BKS, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64) void k_gemm(Mat A, Mat B, Epilogue e, int M, int N, int K, int tiles_n,
                                                      int k_per_split) {
  constexpr int THREADS = WM * WN * 64;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int STEPS = 2;                              // k steps of a tile: 64 bytes of each row
  __shared__ __attribute__((aligned(16))) char lds[2][(BM + BN) * 128];

  const int tile = blockIdx.x, split = blockIdx.y;
  const int m0 = (tile / tiles_n) * BM, n0 = (tile % tiles_n) * BN;
  const int kb = split * k_per_split, ke = min(K, kb + k_per_split);
  Mat a = A, b = B;                                     // the split's share of the reduction
  if (AKS) a.rows = ke; else a.cols = ke;
  if (BKS) b.rows = ke; else b.cols = ke;

  const int w = threadIdx.x >> 6;
  const int wm = (w / WN) * (BM / WM), wn = (w % WN) * (BN / WN);
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0, 0, 0, 0};

  Stage<T, AKS, BM, THREADS> sa;
  Stage<T, BKS, BN, THREADS> sb;
  sa.load(a, m0, kb);
  sb.load(b, n0, kb);
  sa.store(lds[0]);
  sb.store(lds[0] + BM * 128);
  __syncthreads();
  int cur = 0;
  for (int k = kb; k < ke; k += BK<T>) {
    const bool more = k + BK<T> < ke;
    if (more) {
      sa.load(a, m0, k + BK<T>);
      sb.load(b, n0, k + BK<T>);
    }
    const char* la = lds[cur];
    const char* lb = lds[cur] + BM * 128;
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      u32x4 fa[TM], fb[TN];
#pragma unroll
      for (int i = 0; i < TM; i++) fa[i] = frag<T, AKS, BM>(la, wm + i * 16, s);
#pragma unroll
      for (int j = 0; j < TN; j++) fb[j] = frag<T, BKS, BN>(lb, wn + j * 16, s);
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = mma(fb[j], fa[i], acc[i][j], T{});
    }
    if (more) {
      sa.store(lds[cur ^ 1]);
      sb.store(lds[cur ^ 1] + BM * 128);
    }
    __syncthreads();
    cur ^= 1;
  }

  constexpr int SHARE = (BM + BN) * 256 / (WM * WN);
  write_out<T, TM, TN, SHARE>(e, acc, &lds[0][0] + w * SHARE, m0 + wm, n0 + wn, M, N, split);
}

// ---- the tile kernel with direct loads --------------------------------------------
//
// The same product for matrices whose rows start on 16 bytes (and, ks, whose
// columns are whole chunks): global memory goes straight to LDS
// (global_load_lds_dwordx4), so a tile costs no registers and no LDS write
// instructions.  The chunk permutation of Tile is applied to the address each
// lane reads, since a wave's 64 chunks land side by side.
//
// Two tiles of LDS, two k steps a tile, and two sets of fragments, so that the
// matrix cores never wait for a load that was asked for in the same step:
//
//   read step 1 of tile t      multiply step 0 of tile t
//   --- tile t + 1 has arrived, every wave has read tile t ---
//   ask for tile t + 2 in tile t's place
//   read step 0 of tile t + 1  multiply step 1 of tile t

typedef const __attribute__((address_space(1))) void* global_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

// One thread's share of a tile, asked for but not waited for.  Rows (ks:
// chunks) past the edge repeat the last one; nothing of them is stored.
template <typename T, bool KS, int R, int THREADS>
struct Direct {
  typedef Tile<T, KS, R> L;
  static constexpr int PER = L::CHUNKS / THREADS;
  const char* base;              // the next tile's first row, the same for all lanes
  uint32_t off[PER];             // this thread's chunks behind it
  int64_t step;                  // bytes to the tile after it

  __device__ __forceinline__ void start(const Mat& a, int r0, int k0) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      int row, c;
      L::from(i * THREADS + (int)threadIdx.x, row, c);
      int64_t at;
      if (KS) {
        int col = r0 + c * L::E;
        if (col + L::E > a.cols) col = a.cols - L::E;
        at = row * a.ld + (col - r0);
      } else {
        int r = row;
        if (r0 + r >= a.rows) r = a.rows - 1 - r0;
        at = r * a.ld + c * L::E;
      }
      off[i] = (uint32_t)(at * (int64_t)sizeof(T));
    }
    base = static_cast<const char*>(a.p) + (KS ? k0 * a.ld + r0 : r0 * a.ld + k0) * (int64_t)sizeof(T);
    step = KS ? a.ld * BK<T> * (int64_t)sizeof(T) : 128;
  }
  __device__ __forceinline__ void next(char* lds) {
    char* to = lds + (__builtin_amdgcn_readfirstlane((int)threadIdx.x & ~63) << 4);   // the wave's place; lane i lands 16 i behind it
#pragma unroll
    for (int i = 0; i < PER; i++)
      __builtin_amdgcn_global_load_lds((global_ptr)(base + off[i]), (lds_ptr)(to + i * THREADS * 16), 16, 0, 0);
    base += step;
  }
};

// Workgroup `b` of `n` runs on XCD b % 8: each XCD takes a run of neighbouring
// tiles, in columns of 4 tile rows, so that what its L2 holds of A and B is
// shared by its 32 compute units.
__device__ __forceinline__ void place(int b, int n, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int per = n / 8, rest = n % 8, x = b & 7;
  const int t = x * per + (x < rest ? x : rest) + (b >> 3);
  constexpr int GROUP = 4;
  const int wide = GROUP * tiles_n, g = t / wide, first = g * GROUP;
  const int rows = tiles_m - first < GROUP ? tiles_m - first : GROUP;
  tm = first + (t - g * wide) % rows;
  tn = (t - g * wide) / rows;
}

template <typename T, bool AKS, bool BKS, int BM, int BN, int WM, int WN, bool AHEAD>
__global__ __launch_bounds__(WM* WN * 64) void k_gemm_direct(Mat A, Mat B, Epilogue e, int M, int N, int K, int tiles_m,
                                                             int tiles_n, int k_per_split) {
  constexpr int THREADS = WM * WN * 64;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int STEPS = 2;
  // four arrays, not one: the compiler then sees that a load under way into one does not concern reads of another
  __shared__ __attribute__((aligned(16))) char a0[BM * 128], b0[BN * 128], a1[BM * 128], b1[BN * 128];

  int tm, tn;
  place(blockIdx.x, gridDim.x, tiles_m, tiles_n, tm, tn);
  const int split = blockIdx.y, m0 = tm * BM, n0 = tn * BN;
  const int kb = split * k_per_split, ke = min(K, kb + k_per_split);
  const int whole = (ke - kb) / BK<T>;
  const int w = threadIdx.x >> 6;
  const int wm = (w / WN) * (BM / WM), wn = (w % WN) * (BN / WN);
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0, 0, 0, 0};

  Direct<T, AKS, BM, THREADS> da;
  Direct<T, BKS, BN, THREADS> db;
  da.start(A, m0, kb);
  db.start(B, n0, kb);
  auto ask = [&](int t, char* la, char* lb) {
    if (t < whole) {
      da.next(la);
      db.next(lb);
    }
  };
  u32x4 fa[AHEAD ? 2 : 1][TM], fb[AHEAD ? 2 : 1][TN];
  auto read = [&](int s, const char* la, const char* lb) {
#pragma unroll
    for (int i = 0; i < TM; i++) fa[AHEAD ? s : 0][i] = frag<T, AKS, BM>(la, wm + i * 16, s);
#pragma unroll
    for (int j = 0; j < TN; j++) fb[AHEAD ? s : 0][j] = frag<T, BKS, BN>(lb, wn + j * 16, s);
  };
  auto multiply = [&](int s) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) acc[i][j] = mma(fb[AHEAD ? s : 0][j], fa[AHEAD ? s : 0][i], acc[i][j], T{});
  };
  auto tile = [&](int t, char* la, char* lb, char* na, char* nb) {
    if (AHEAD) {
      read(1, la, lb);
      multiply(0);
      __syncthreads();
      ask(t + 2, la, lb);
      if (t + 1 < whole) read(0, na, nb);
      multiply(1);
    } else {
      ask(t + 1, na, nb);
      read(0, la, lb);
      multiply(0);
      read(1, la, lb);
      multiply(1);
      __syncthreads();
    }
  };
  ask(0, a0, b0);
  __syncthreads();
  if (AHEAD) {
    ask(1, a1, b1);
    if (whole) read(0, a0, b0);
  }
  for (int t = 0; t < whole; t += 2) {
    tile(t, a0, b0, a1, b1);
    if (t + 1 < whole) tile(t + 1, a1, b1, a0, b0);
  }
  if (kb + whole * BK<T> < ke) {
    // the reduction ends inside a tile: that one through registers, zeros behind the end
    Mat a = A, b = B;
    if (AKS) a.rows = ke; else a.cols = ke;
    if (BKS) b.rows = ke; else b.cols = ke;
    __syncthreads();
    {
      Stage<T, AKS, BM, THREADS> sa;
      sa.load(a, m0, kb + whole * BK<T>);
      sa.store(a0);
    }
    {
      Stage<T, BKS, BN, THREADS> sb;
      sb.load(b, n0, kb + whole * BK<T>);
      sb.store(b0);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      read(s, a0, b0);
      multiply(s);
    }
  }

  __syncthreads();
  static_assert(BM == BN && WM * WN % 4 == 0, "the waves share the four arrays evenly");
  constexpr int EACH = WM * WN / 4, SHARE = BM * 128 / EACH;
  char* mine = w / EACH == 0 ? a0 : w / EACH == 1 ? b0 : w / EACH == 2 ? a1 : b1;
  write_out<T, TM, TN, SHARE>(e, acc, mine + (w % EACH) * SHARE, m0 + wm, n0 + wn, M, N, split);
}

// The splits' sums in their order, then the epilogue.
template <typename T>
__global__ __launch_bounds__(256) void k_join(Epilogue e, int64_t M, int N, int splits) {
  const int64_t count = M * N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    float v = 0.0f;
    for (int s = 0; s < splits; s++) v += e.part[s * count + i];
    const int64_t m = i / N;
    finish<T>(e, m, (int)(i - m * N), N, v);
  }
}

// ---- dz and db --------------------------------------------------------------------
//
// Workgroup (column block, row share): 16 lanes across 8 columns each, 16 rows
// down, over the share's rows.  dz = dy act'(z) rounded once to the element
// type (the matrix cores' input), its column sums taken before that rounding.
// Bound by memory: dy and z read, dz written.

#define DZ_COLUMNS 128

template <typename T>
__global__ __launch_bounds__(256) void k_dz(const T* dy, int64_t ldy, const T* z, T* dz, T* db, float* part, int M,
                                            int N, int act, int rows_per) {
  __shared__ float sums[16][DZ_COLUMNS + 4];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
  const int n = blockIdx.x * DZ_COLUMNS + x * 8;
  const int mb = blockIdx.y * rows_per, me = min(M, mb + rows_per);
  float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (n + 8 <= N) {
#pragma unroll 2
    for (int m = mb + y; m < me; m += 16) {
      float v[8], u[8];
      load8<T>(dy + m * ldy + n, v);
      if (act != ACT_NONE) {
        load8<T>(z + (int64_t)m * N + n, u);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= act_grad<T>(act, u[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; i++) s[i] += v[i];
      if (dz) {
        T o[8];
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = from_f<T>(v[i]);
        store8<T>(dz + (int64_t)m * N + n, o);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (n + i < N)
        for (int m = mb + y; m < me; m += 16) {
          float v = to_f(dy[m * ldy + n + i]);
          if (act != ACT_NONE) v *= act_grad<T>(act, to_f(z[(int64_t)m * N + n + i]));
          s[i] += v;
          if (dz) dz[(int64_t)m * N + n + i] = from_f<T>(v);
        }
  }
  if (!db && !part) return;
#pragma unroll
  for (int i = 0; i < 8; i++) sums[y][x * 8 + i] = s[i];
  __syncthreads();
  const int c = blockIdx.x * DZ_COLUMNS + threadIdx.x;
  if (threadIdx.x >= DZ_COLUMNS || c >= N) return;
  float t = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; i++) t += sums[i][threadIdx.x];
  if (part) part[(int64_t)blockIdx.y * N + c] = t;
  else db[c] = from_f<T>(t);
}

// The shares' column sums: 4 waves over the shares, in a fixed order.
template <typename T>
__global__ __launch_bounds__(256) void k_db(const float* part, T* db, int N, int shares) {
  __shared__ float sums[4][64];
  const int x = threadIdx.x & 63, w = threadIdx.x >> 6, n = blockIdx.x * 64 + x;
  float s = 0.0f;
  if (n < N)
    for (int i = w; i < shares; i += 4) s += part[(int64_t)i * N + n];
  sums[w][x] = s;
  __syncthreads();
  if (w == 0 && n < N) db[n] = from_f<T>((sums[0][x] + sums[1][x]) + (sums[2][x] + sums[3][x]));
}

// ---- host side ---------------------------------------------------------------------

int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

struct Plan {
  int tiles_m, tiles_n, splits, k_per;
};

Plan plan_tiles(int M, int N, int K, int bm, int bn, int bk) {
  Plan p;
  p.tiles_m = cdiv(M, bm);
  p.tiles_n = cdiv(N, bn);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  // fewer tiles than half the compute units: the reduction is shared out too, in shares of at least 4 k tiles
  int want = tiles < 128 ? (int)(256 / tiles) : 1;
  const int kt = cdiv(K, bk);
  want = want < kt / 4 ? want : kt / 4;
  if (want < 1) want = 1;
  p.k_per = cdiv(kt, want) * bk;
  p.splits = K > 0 ? cdiv(K, p.k_per) : 1;
  return p;
}

int elt(int dtype) { return dtype == CIT_FP32 ? 4 : 2; }

enum { TILE_64, TILE_128, TILE_256 };

// The tile of a product of aligned operands.
int tile_of(int M, int N, int es) {
  if (es == 2 && (int64_t)cdiv(M, 256) * cdiv(N, 256) >= 128) return TILE_256;
  if ((int64_t)cdiv(M, 128) * cdiv(N, 128) >= 128) return TILE_128;
  return TILE_64;
}
Plan plan_of(int tile, int M, int N, int K, int bk) {
  const int t = tile == TILE_256 ? 256 : tile == TILE_128 ? 128 : 64;
  return plan_tiles(M, N, K, t, t, bk);
}

// Room for split sums, whatever the operands' alignment makes of the tile.
int64_t product_work(int M, int N, int K, int dtype) {
  if (M <= 0 || N <= 0) return 0;
  int64_t most = 0;
  for (int tile : {(int)TILE_64, tile_of(M, N, elt(dtype))}) {
    const Plan p = plan_of(tile, M, N, K, 128 / elt(dtype));
    if (p.splits > 1 && p.splits > most) most = p.splits;
  }
  return align256(most * M * N * 4);
}

template <typename T>
bool direct(const Mat& a, bool ks) {
  if (((uintptr_t)a.p & 15) || (a.ld * (int64_t)sizeof(T)) % 16) return false;
  if (a.ld * (int64_t)sizeof(T) >= 1 << 23) return false;             // a tile's rows within 31 bits of its first
  return !ks || a.cols % (16 / (int)sizeof(T)) == 0;
}

template <typename T, bool AKS, bool BKS, int TILE, int WM, int WN, bool AHEAD>
void launch_direct(const Mat& A, const Mat& B, const Epilogue& e, int M, int N, int K, const Plan& p,
                   hipStream_t stream) {
  hipLaunchKernelGGL((k_gemm_direct<T, AKS, BKS, TILE, TILE, WM, WN, AHEAD>), dim3(p.tiles_m * p.tiles_n, p.splits),
                     dim3(WM * WN * 64), 0, stream, A, B, e, M, N, K, p.tiles_m, p.tiles_n, p.k_per);
}

template <typename T, bool AKS, bool BKS>
int product(Mat A, Mat B, Epilogue e, int M, int N, int K, void* work, hipStream_t stream) {
  const bool d = K > 0 && direct<T>(A, AKS) && direct<T>(B, BKS);
  const int tile = d ? tile_of(M, N, sizeof(T)) : TILE_64;
  const Plan p = plan_of(tile, M, N, K, BK<T>);
  if (p.splits > 1) e.part = static_cast<float*>(work);
  if (!d)
    hipLaunchKernelGGL((k_gemm<T, AKS, BKS, 64, 64, 2, 2>), dim3(p.tiles_m * p.tiles_n, p.splits), dim3(256), 0, stream,
                       A, B, e, M, N, K, p.tiles_n, p.k_per);
  else if (tile == TILE_64) launch_direct<T, AKS, BKS, 64, 2, 2, true>(A, B, e, M, N, K, p, stream);
  else if (tile == TILE_128) launch_direct<T, AKS, BKS, 128, 2, 2, true>(A, B, e, M, N, K, p, stream);
  else if constexpr (sizeof(T) == 2) launch_direct<T, AKS, BKS, 256, 2, 4, false>(A, B, e, M, N, K, p, stream);
  if (p.splits > 1) {
    const int64_t blocks = ((int64_t)M * N + 255) / 256;
    hipLaunchKernelGGL((k_join<T>), dim3(blocks < 4096 ? (unsigned)blocks : 4096), dim3(256), 0, stream, e, (int64_t)M,
                       N, p.splits);
  }
  return launch_status();
}

// Rows of a share: about 4 workgroups for each compute unit, at least 64 rows each.
int dz_rows(int M, int N) {
  int shares = cdiv(1024, cdiv(N, DZ_COLUMNS));
  const int most = cdiv(M, 64);
  if (shares > most) shares = most;
  if (shares < 1) shares = 1;
  return cdiv(cdiv(M, shares), 16) * 16;
}

template <typename T>
int forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const Epilogue& e, int M, int N, int K, void* work,
            hipStream_t stream) {
  return product<T, false, false>(Mat{x, ldx, M, K}, Mat{w, ldw, N, K}, e, M, N, K, work, stream);
}

template <typename T>
int backward(const void* dy, int64_t ldy, const void* z, const void* x, int64_t ldx, const void* w, int64_t ldw,
             void* dx, void* dw, void* db, int M, int N, int K, int act, char* work, hipStream_t stream) {
  const T* d = static_cast<const T*>(dy);
  int64_t ldd = ldy;
  const int rows = dz_rows(M, N), shares = cdiv(M, rows);
  T* dz = nullptr;
  float* sums = nullptr;
  if (act != ACT_NONE && (dx || dw)) {
    dz = reinterpret_cast<T*>(work);
    work += align256((int64_t)M * N * sizeof(T));
  }
  if (db && shares > 1) {
    sums = reinterpret_cast<float*>(work);
    work += align256((int64_t)shares * N * 4);
  }
  if (dz || db) {
    hipLaunchKernelGGL((k_dz<T>), dim3(cdiv(N, DZ_COLUMNS), shares), dim3(256), 0, stream, d, ldy,
                       static_cast<const T*>(z), dz, static_cast<T*>(db), sums, M, N, act, rows);
    if (sums)
      hipLaunchKernelGGL((k_db<T>), dim3(cdiv(N, 64)), dim3(256), 0, stream, sums, static_cast<T*>(db), N, shares);
  }
  if (dz) d = dz, ldd = N;
  int rc = 0;
  if (dx && K > 0) {
    Epilogue e = {};
    e.out = dx;
    e.ldo = K;
    rc = product<T, false, true>(Mat{d, ldd, M, N}, Mat{w, ldw, N, K}, e, M, K, N, work, stream);
  }
  if (!rc && dw && K > 0) {
    Epilogue e = {};
    e.out = dw;
    e.ldo = K;
    rc = product<T, true, true>(Mat{d, ldd, M, N}, Mat{x, ldx, M, K}, e, N, K, M, work, stream);
  }
  return rc ? rc : launch_status();
}

bool bad_types(int dtype, int act) { return dtype < CIT_FP32 || dtype > CIT_FP16 || act < ACT_NONE || act > ACT_SILU; }

}  // namespace

extern "C" {

size_t cit_linear_forward_work_bytes(int M, int N, int K, int dtype) {
  return bad_types(dtype, 0) ? 0 : (size_t)product_work(M, N, K, dtype);
}

size_t cit_linear_backward_work_bytes(int M, int N, int K, int dtype, int act) {
  if (bad_types(dtype, act) || M <= 0 || N <= 0 || K < 0) return 0;
  const int64_t a = product_work(M, K, N, dtype), b = product_work(N, K, M, dtype);
  const int64_t dz = act != ACT_NONE ? align256((int64_t)M * N * elt(dtype)) : 0;
  return (size_t)(dz + align256((int64_t)cdiv(M, dz_rows(M, N)) * N * 4) + (a > b ? a : b));
}

int cit_linear_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual,
                       int64_t ldr, void* y, void* z, int M, int N, int K, int dtype, int act, void* work,
                       size_t work_bytes, hipStream_t stream) {
  if (M < 0 || N < 0 || K < 0 || bad_types(dtype, act)) return -1;
  if (!M || !N) return 0;
  if (!y || (K && (!x || !w || ldx < K || ldw < K)) || (residual && ldr < N)) return -1;
  const size_t need = cit_linear_forward_work_bytes(M, N, K, dtype);
  if (need && (!work || work_bytes < need)) return -1;
  Epilogue e = {};
  e.bias = bias, e.res = residual, e.out = y, e.z = z, e.ldr = ldr, e.ldo = N, e.act = act;
  if (dtype == CIT_FP32) return forward<float>(x, ldx, w, ldw, e, M, N, K, work, stream);
  if (dtype == CIT_BF16) return forward<bf16_t>(x, ldx, w, ldw, e, M, N, K, work, stream);
  return forward<fp16_t>(x, ldx, w, ldw, e, M, N, K, work, stream);
}

int cit_linear_backward(const void* dy, int64_t ldy, const void* z, const void* x, int64_t ldx, const void* w,
                        int64_t ldw, void* dx, void* dw, void* db, int M, int N, int K, int dtype, int act, void* work,
                        size_t work_bytes, hipStream_t stream) {
  if (M <= 0 || N <= 0 || K < 0 || bad_types(dtype, act)) return -1;
  if (!dy || ldy < N || (act != ACT_NONE && !z) || (dx && (!w || ldw < K)) || (dw && (!x || ldx < K))) return -1;
  const size_t need = cit_linear_backward_work_bytes(M, N, K, dtype, act);
  if (need && (!work || work_bytes < need)) return -1;
  char* p = static_cast<char*>(work);
  if (dtype == CIT_FP32) return backward<float>(dy, ldy, z, x, ldx, w, ldw, dx, dw, db, M, N, K, act, p, stream);
  if (dtype == CIT_BF16) return backward<bf16_t>(dy, ldy, z, x, ldx, w, ldw, dx, dw, db, M, N, K, act, p, stream);
  return backward<fp16_t>(dy, ldy, z, x, ldx, w, ldw, dx, dw, db, M, N, K, act, p, stream);
}

}  // extern "C"
