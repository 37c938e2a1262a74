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
#include <type_traits>

#include "cit_ops.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 fp16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((__vector_size__(8)));

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

// Phi(z) = erfc(-z / sqrt(2)) / 2 and exp(-z^2 / 2).  fp32 takes the library's erfc
// (no cancellation at z < 0).  For 16-bit results it is Abramowitz and
// Stegun's 7.1.26, off by at most 0.75e-7 absolute, whose exponential gelu's
// derivative needs anyhow: a fifth of the instructions.  Of Phi itself that is
// 6e-8 at z = -1, 5e-4 at -4 and 1e-2 at -8: past half a step of bf16 below
// z = -5, where gelu is under 1.5e-6 (fp16's steps are absolute there, 6e-8).
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
  if (act == ACT_RELU) return z <= 0.0f ? 0.0f : 1.0f;              // NaN lets dy through: no 0 hides it
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

// z kept for the backward pass in the element type: half the bytes of a 32-bit
// z, whose writing and reading are a part of what the passes around the products
// cost; act' is then that of a z off by half a step, as it is where a layer's pre-activation is a
// tensor of its own.  The rounding is to
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

// Until this wave's LDS writes are there for its other lanes, and its reads done before they are written over.  (A wave's
// LDS accesses run in their order; this keeps the compiler from moving one past another, whatever it knows of their
// addresses.)
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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
    wave_fence();
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
    wave_fence();
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
    return (sizeof(T) == 2 ? (row & 3) << 1 : ((row >> 2) & 3) << 2) & (CPR - 1);
  }
  // Byte offset of the 16-byte chunk c of tile row `row`.
  __device__ static __forceinline__ int at(int row, int c) { return (row * CPR + (c ^ swz(row))) << 4; }

  // Global chunk behind LDS chunk `id`: (tile row, chunk of the row).
  __device__ static __forceinline__ void from(int id, int& row, int& c) {
    row = id / CPR;
    c = (id % CPR) ^ swz(row);
  }
};

// A matrix of `rows` x `cols` elements, ld elements apart; of each row `edge`
// elements may be read (more than cols in a padded copy).
struct Mat {
  const void* p;
  int64_t ld;
  int rows, cols, edge;
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

// Loads of thread `me` of THREADS for one tile, through registers.  DZ: the
// operand is dy act'(z), made on the way (rounded to the type, as k_dz does).
template <typename T, bool KS, int R, int THREADS, bool DZ = false>
struct Stage {
  typedef Tile<T, KS, R> L;
  static constexpr int PER = L::CHUNKS / THREADS;
  u32x4 v[PER], u[DZ ? PER : 1];
  __device__ __forceinline__ void load(const Mat& a, int r0, int k0, int me, const Mat* z = nullptr) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      int row, c;
      L::from(i * THREADS + me, row, c);
      const int y = KS ? k0 + row : r0 + row, x = KS ? r0 + c * L::E : k0 + c * L::E;
      v[i] = fetch<T>(a, y, x);
      if (DZ) u[i] = fetch<T>(*z, y, x);
    }
  }
  __device__ __forceinline__ void store(char* lds, int me, int act = ACT_NONE) const {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      Pack16<T> p;
      p.raw = v[i];
      if (DZ) {
        Pack16<T> q;
        q.raw = u[i];
#pragma unroll
        for (int k = 0; k < L::E; k++) p.e[k] = from_f<T>(to_f(p.e[k]) * act_grad<T>(act, to_f(q.e[k])));
      }
      *reinterpret_cast<u32x4*>(lds + ((i * THREADS + me) << 4)) = p.raw;
    }
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
// tile, the next one's loads are in flight.  Any alignment; bound by those
// loads' latency: a second tile ahead in registers gained nothing, but HALVES of a
// workgroup that take the reduction's tiles in turn did where all workgroups
// are on the chip at once, two a compute unit (fp16 1023 x 1537 x 2051, 400 tiles, 33
// -> 29 us; 1100 x 1100 x 3001 43 -> 35; but 3000 x 1001 x 999, 752 tiles, 25 -> 30).
// fp32 comes here only with rows 8 MB apart.

template <typename T, bool AKS, bool BKS, int BM, int BN, int WM, int WN, int HALVES>
__global__ __launch_bounds__(WM* WN * 64 * HALVES) void k_gemm(Mat A, Mat B, Epilogue e, int M, int N, int K, int tiles_n,
                                                               int k_per_split) {
  constexpr int THREADS = WM * WN * 64;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int STEPS = 2;                              // k steps of a tile: 64 bytes of each row
  __shared__ __attribute__((aligned(16))) char lds[HALVES][2][(BM + BN) * 128];

  const int64_t tile = (int64_t)blockIdx.z * gridDim.x + blockIdx.x;
  if (tile >= (int64_t)((M + BM - 1) / BM) * tiles_n) return;
  const int split = blockIdx.y, m0 = (int)(tile / tiles_n) * BM, n0 = (int)(tile % tiles_n) * BN;
  const int kb = split * k_per_split, ke = min(K, kb + k_per_split);
  Mat a = A, b = B;                                     // the split's share of the reduction
  if (AKS) a.rows = ke; else a.cols = ke;
  if (BKS) b.rows = ke; else b.cols = ke;

  const int half = HALVES > 1 ? threadIdx.x / THREADS : 0, me = threadIdx.x % THREADS;
  const int w = me >> 6;
  const int wm = (w / WN) * (BM / WM), wn = (w % WN) * (BN / WN);
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0, 0, 0, 0};

  Stage<T, AKS, BM, THREADS> sa;
  Stage<T, BKS, BN, THREADS> sb;
  constexpr int STEP = HALVES * BK<T>;                  // (a half's tile past the end is zeros)
  const int mine = half * BK<T>;
  sa.load(a, m0, kb + mine, me);
  sb.load(b, n0, kb + mine, me);
  sa.store(lds[half][0], me);
  sb.store(lds[half][0] + BM * 128, me);
  __syncthreads();
  int cur = 0;
  for (int k = kb; k < ke; k += STEP) {
    const bool more = k + STEP < ke;
    if (more) {
      sa.load(a, m0, k + STEP + mine, me);
      sb.load(b, n0, k + STEP + mine, me);
    }
    const char* la = lds[half][cur];
    const char* lb = lds[half][cur] + BM * 128;
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
      sa.store(lds[half][cur ^ 1], me);
      sb.store(lds[half][cur ^ 1] + BM * 128, me);
    }
    __syncthreads();
    cur ^= 1;
  }

  if (HALVES > 1) {                                     // the halves' sums meet in the second one's place
    f32x4* other = reinterpret_cast<f32x4*>(&lds[HALVES - 1][0][0]) + me;
    static_assert(TM * TN * 16 * THREADS <= (BM + BN) * 256, "the sums fit");
    if (half)
#pragma unroll
      for (int i = 0; i < TM * TN; i++) other[i * THREADS] = acc[i / TN][i % TN];
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int i = 0; i < TM * TN; i++) acc[i / TN][i % TN] += other[i * THREADS];
  }
  constexpr int SHARE = (BM + BN) * 256 / (WM * WN);
  write_out<T, TM, TN, SHARE>(e, acc, &lds[0][0][0] + w * SHARE, m0 + wm, n0 + wn, M, N, split);
}

// ---- the tile kernel with direct loads --------------------------------------------
//
// The same product for matrices whose rows start on 16 bytes (and, ks, whose
// columns are whole chunks), and for fp32 ones of any width in single words:
// global memory goes straight to LDS (global_load_lds_dwordx4, _dword), so a
// tile costs no registers and no LDS write instructions.  The chunk permutation of Tile is applied to the address each
// lane reads, since a wave's 64 chunks land side by side.
//
// STAGES tiles of LDS, all but one of them under way while the last is worked
// on, two k steps a tile, and (AHEAD) two sets of fragments, so that the matrix
// cores never wait for a load that was asked for in the same step:
//
//   read step 1 of tile t      multiply step 0 of tile t
//   --- tile t + 1 has arrived, every wave has read tile t ---
//   ask for tile t + STAGES in tile t's place
//   read step 0 of tile t + 1  multiply step 1 of tile t
//
// A tile takes about 0.9 us to arrive and a 64 x 64 one 0.1 us to multiply:
// where there are not enough workgroups to hide that, four stages do.
//
// Bound by the matrix cores (fp32) and by the L2s' 10 TB/s and the LDS reads
// (16-bit types).  8192 x 4096 x 4096: bf16 forward 217 us, dx 217, dw 202, 1,270
// to 1,360 TFLOP/s (a library's 8192^3 reaches 1,390 here, its products of this
// size 970 to 1,220); fp32 1,986 us, 138 TFLOP/s (library 136 to 150).  fp32 in words,
// 4096 x 512 x 418: 25 us (through registers 27), the matrix cores at work for 12.

typedef const __attribute__((address_space(1))) void* global_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

// One thread's share of a tile, asked for but not waited for, in pieces of W
// bytes: 16, or 4 for fp32 matrices whose rows are off 16 bytes.  Rows (ks:
// pieces) past the edge repeat the last one; nothing of them is stored.
template <typename T, bool KS, int R, int THREADS, int W>
struct Direct {
  typedef Tile<T, KS, R> L;
  static constexpr int PER = L::CHUNKS * (16 / W) / THREADS, E = W / (int)sizeof(T);
  const char* base;              // the next tile's first row, the same for all lanes
  uint32_t off[PER];             // this thread's chunks behind it
  int64_t step;                  // bytes to the tile after it

  __device__ __forceinline__ void start(const Mat& a, int r0, int k0) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int id = i * THREADS + (int)threadIdx.x;
      int row, c;
      L::from(id / (16 / W), row, c);
      const int in = id % (16 / W) * E;                // the piece within its chunk
      int64_t at;
      if (KS) {
        int col = r0 + c * L::E + in;
        if (col + E > a.edge) col = a.edge - E;
        at = row * a.ld + (col - r0);
      } else {
        int r = row;
        if (r0 + r >= a.rows) r = a.rows - 1 - r0;
        at = r * a.ld + c * L::E + in;
      }
      off[i] = (uint32_t)(at * (int64_t)sizeof(T));
    }
    base = static_cast<const char*>(a.p) + (KS ? k0 * a.ld + r0 : r0 * a.ld + k0) * (int64_t)sizeof(T);
    step = KS ? a.ld * BK<T> * (int64_t)sizeof(T) : 128;
  }
  __device__ __forceinline__ void next(char* lds) {
    char* to = lds + __builtin_amdgcn_readfirstlane((int)threadIdx.x & ~63) * W;   // the wave's place; lane i lands W i behind it
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const global_ptr from = (global_ptr)(base + off[i]);
      const lds_ptr at = (lds_ptr)(to + i * THREADS * W);
      if constexpr (W == 16) __builtin_amdgcn_global_load_lds(from, at, 16, 0, 0);
      else __builtin_amdgcn_global_load_lds(from, at, 4, 0, 0);
    }
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

// Until all but N of this wave's loads to LDS have landed and its reads of LDS
// are done, then until every wave is here.  (A plain barrier would wait for all
// loads, the ones for later tiles too.)
template <int N>
__device__ __forceinline__ void arrive() {
  static_assert(N < 64, "the counter's field");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);      // lgkmcnt 0; the builtin, since the compiler counts along
  asm volatile("s_barrier" ::: "memory");
}

// The same for all of its loads, stated rather than left to what a fence at a barrier happens to wait for.
__device__ __forceinline__ void arrive_all() {
  __builtin_amdgcn_s_waitcnt(15 << 8 | 7 << 4);                        // vmcnt 0
  __syncthreads();
}

template <typename T, bool AKS, bool BKS, int BM, int BN, int WM, int WN, int STAGES, bool AHEAD, int W>
__global__ __launch_bounds__(WM* WN * 64) void k_gemm_direct(Mat A, Mat B, Epilogue e, int M, int N, int K, int tiles_m,
                                                             int tiles_n, int k_per_split) {
  constexpr int THREADS = WM * WN * 64;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int STEPS = 2, BYTES = (BM + BN) * 128;
  // an array a stage, not one: the compiler then sees that loads under way into one do not concern reads of another
  __shared__ __attribute__((aligned(16))) char s0[BYTES], s1[BYTES], s2[STAGES > 2 ? BYTES : 16],
      s3[STAGES > 3 ? BYTES : 16];

  const int block = (int)(blockIdx.z * gridDim.x + blockIdx.x), tiles = tiles_m * tiles_n;
  if (block >= tiles) return;
  int tm, tn;
  place(block, tiles, tiles_m, tiles_n, tm, tn);
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

  Direct<T, AKS, BM, THREADS, W> da;
  Direct<T, BKS, BN, THREADS, W> db;
  constexpr int LOADS = decltype(da)::PER + decltype(db)::PER;         // a tile's, for each wave
  da.start(A, m0, kb);
  db.start(B, n0, kb);
  auto ask = [&](int t, char* to) __attribute__((always_inline)) {
    if (t < whole) {
      da.next(to);
      db.next(to + BM * 128);
    }
  };
  u32x4 fa[AHEAD ? 2 : 1][TM], fb[AHEAD ? 2 : 1][TN];
  auto read = [&](int s, const char* from) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; i++) fa[AHEAD ? s : 0][i] = frag<T, AKS, BM>(from, wm + i * 16, s);
#pragma unroll
    for (int j = 0; j < TN; j++) fb[AHEAD ? s : 0][j] = frag<T, BKS, BN>(from + BM * 128, wn + j * 16, s);
  };
  auto multiply = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++)
        acc[i][j] = mma(fb[AHEAD ? s : 0][j], fa[AHEAD ? s : 0][i], acc[i][j], T{});
  };
  // tile t in `here`, the one after it in `next`; `steady`: there is a tile t + STAGES
  auto tile = [&](auto steady, int t, char* here, char* next) __attribute__((always_inline)) {
    if (AHEAD) {
      read(1, here);
      multiply(0);
      // tiles t + 1 .. t + STAGES - 1 are under way, near the end fewer
      if (STAGES == 2) arrive_all();
      else if (steady.value || t + STAGES <= whole) arrive<(STAGES - 2) * LOADS>();
      else arrive<0>();
      if (steady.value || t + STAGES < whole) {
        da.next(here);
        db.next(here + BM * 128);
      }
      if (steady.value || t + 1 < whole) read(0, next);
      multiply(1);
    } else {
      static_assert(AHEAD || STAGES == 2, "one tile ahead");
      ask(t + 1, next);
      read(0, here);
      multiply(0);
      read(1, here);
      multiply(1);
      arrive_all();
    }
  };
  auto round = [&](auto steady, int t) __attribute__((always_inline)) {
    tile(steady, t, s0, s1);
    if (steady.value || t + 1 < whole) tile(steady, t + 1, s1, STAGES == 2 ? s0 : s2);
    if (STAGES > 2 && (steady.value || t + 2 < whole)) tile(steady, t + 2, s2, STAGES == 3 ? s0 : s3);
    if (STAGES > 3 && (steady.value || t + 3 < whole)) tile(steady, t + 3, s3, s0);
  };
  ask(0, s0);
  if (AHEAD) {
    ask(1, s1);
    if (STAGES > 2) ask(2, s2);
    if (STAGES > 3) ask(3, s3);
    if (whole >= STAGES) arrive<(STAGES - 1) * LOADS>();
    else arrive<0>();
    if (whole) read(0, s0);
  } else {
    arrive_all();
  }
  int t = 0;
  for (; STAGES > 2 && t + 2 * STAGES <= whole; t += STAGES) round(std::true_type{}, t);    // without a branch
  for (; t < whole; t += STAGES) round(std::false_type{}, t);
  if (kb + whole * BK<T> < ke) {
    // the reduction ends inside a tile: that one through registers, zeros behind the end
    Mat a = A, b = B;
    if (AKS) a.rows = ke; else a.cols = ke;
    if (BKS) b.rows = ke; else b.cols = ke;
    __syncthreads();
    {
      Stage<T, AKS, BM, THREADS> sa;
      sa.load(a, m0, kb + whole * BK<T>, threadIdx.x);
      sa.store(s0, threadIdx.x);
    }
    {
      Stage<T, BKS, BN, THREADS> sb;
      sb.load(b, n0, kb + whole * BK<T>, threadIdx.x);
      sb.store(s0 + BM * 128, threadIdx.x);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      read(s, s0);
      multiply(s);
    }
  }

  __syncthreads();
  static_assert(WM * WN % 2 == 0, "the waves share two stages evenly");
  constexpr int EACH = WM * WN / 2, SHARE = BYTES / EACH;
  char* mine = w < EACH ? s0 : s1;
  write_out<T, TM, TN, SHARE>(e, acc, mine + (w % EACH) * SHARE, m0 + wm, n0 + wn, M, N, split);
}

// ---- few outputs --------------------------------------------------------------------
//
// 32 x 32 outputs by 8 waves that share out the reduction, k tile by k tile:
// each wave stages its own tiles in its own 8 KB of LDS (no barrier until the
// end), and the 8 partial sums meet in LDS in the waves' order.  For layers too
// small to fill the chip with larger tiles, and for some rows against a wide
// weight, whose bytes are then what there is to do: bf16 8 x 16,384 x 4096 35 us,
// 3.9 TB/s, as fast as a sum over a large tensor reads.

#define SMALL_WAVES 8
#define SMALL_LDS (SMALL_WAVES * 64 * 128)

template <typename T, bool AKS, bool BKS, bool DZ>
__device__ __forceinline__ void small_tile(const Mat& A, const Mat* Z, const Mat& B, const Epilogue& e, int act, int M,
                                           int N, int K, int m0, int n0, int split, int k_per_split, char* lds) {
  const int kb = split * k_per_split, ke = min(K, kb + k_per_split);
  Mat a = A, b = B;
  if (AKS) a.rows = ke; else a.cols = ke;
  if (BKS) b.rows = ke; else b.cols = ke;
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  char* la = lds + w * (64 * 128);
  char* lb = la + 32 * 128;
  f32x4 acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; i++) acc[i >> 1][i & 1] = f32x4{0, 0, 0, 0};
  // the next tile's loads are under way while this one is at work; two tiles ahead spilled registers and gained nothing
  Stage<T, AKS, 32, 64, DZ> sa;
  Stage<T, BKS, 32, 64> sb;
  constexpr int STEP = SMALL_WAVES * BK<T>;
  int k = kb + w * BK<T>;
  if (k < ke) {
    sa.load(a, m0, k, l, Z);
    sb.load(b, n0, k, l);
  }
  for (; k < ke; k += STEP) {
    sa.store(la, l, act);
    sb.store(lb, l);
    if (k + STEP < ke) {
      sa.load(a, m0, k + STEP, l, Z);
      sb.load(b, n0, k + STEP, l);
    }
    wave_fence();
#pragma unroll
    for (int s = 0; s < 2; s++) {
      u32x4 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        fa[i] = frag<T, AKS, 32>(la, i * 16, s);
        fb[i] = frag<T, BKS, 32>(lb, i * 16, s);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) acc[i >> 1][i & 1] = mma(fb[i & 1], fa[i >> 1], acc[i >> 1][i & 1], T{});
    }
    wave_fence();
  }
  // [wave][row][chunk of 4 columns, permuted by the row]
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int r = i * 16 + (l & 15), c = j * 4 + (l >> 4);
      *reinterpret_cast<f32x4*>(la + r * 128 + ((c ^ (r & 7)) << 4)) = acc[i][j];
    }
  __syncthreads();
  if (threadIdx.x >= 128) return;
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 2, m = m0 + r, n = n0 + c * 4;
  if (m >= M || n >= N) return;
  f32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < SMALL_WAVES; i++) {
    const char* p = lds + i * (64 * 128) + r * 128;
    lo += *reinterpret_cast<const f32x4*>(p + ((c ^ (r & 7)) << 4));
    hi += *reinterpret_cast<const f32x4*>(p + (((c + 1) ^ (r & 7)) << 4));
  }
  float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  finish8<T>(e, m, n, N, v, split, M);
}

template <typename T, bool AKS, bool BKS>
__global__ __launch_bounds__(SMALL_WAVES * 64, 4) void k_gemm_small(Mat A, Mat B, Epilogue e, int M, int N, int K,
                                                                 int tiles_n, int k_per_split) {
  __shared__ __attribute__((aligned(16))) char lds[SMALL_LDS];
  const int64_t tile = (int64_t)blockIdx.z * gridDim.x + blockIdx.x;
  if (tile >= (int64_t)((M + 31) / 32) * tiles_n) return;
  small_tile<T, AKS, BKS, false>(A, nullptr, B, e, ACT_NONE, M, N, K, (int)(tile / tiles_n) * 32,
                                 (int)(tile % tiles_n) * 32, blockIdx.y, k_per_split, lds);
}

// A small layer's whole backward pass in one launch: workgroups for 4 columns
// each of db, then the tiles of dw (the long ones first), then those of dx; dz
// is made from dy and z wherever it is read.  fp32 64 x 418 x 512 9 us, mostly
// latency; 2048 x 512 x 256 27 us.
template <typename T>
__global__ __launch_bounds__(SMALL_WAVES * 64, 4) void k_backward_small(Mat dy, Mat z, Mat x, Mat w, T* dx, T* dw, T* db,
                                                                     int act, int M, int N, int K, int sums,
                                                                     int dw_tiles) {
  __shared__ __attribute__((aligned(16))) char lds[SMALL_LDS];
  const int tiles_k = (K + 31) / 32;
  int b = blockIdx.x;
  if (b >= sums) {
    b -= sums;
    Epilogue e = {};
    e.ldo = K;
    if (b < dw_tiles) {
      e.out = dw;
      const int m0 = b / tiles_k * 32, n0 = b % tiles_k * 32;
      if (act == ACT_NONE) small_tile<T, true, true, false>(dy, &z, x, e, act, N, K, M, m0, n0, 0, M, lds);
      else small_tile<T, true, true, true>(dy, &z, x, e, act, N, K, M, m0, n0, 0, M, lds);
      return;
    }
    b -= dw_tiles;
    e.out = dx;
    const int m0 = b / tiles_k * 32, n0 = b % tiles_k * 32;
    if (act == ACT_NONE) small_tile<T, false, true, false>(dy, &z, w, e, act, M, K, N, m0, n0, 0, N, lds);
    else small_tile<T, false, true, true>(dy, &z, w, e, act, M, K, N, m0, n0, 0, N, lds);
    return;
  }
  // 128 rows of 4 columns at a time, then the 16 rows of a wave, then the waves
  const int c = threadIdx.x & 3, n = b * 4 + c;
  float s = 0.0f;
  if (n < N)
#pragma unroll 4
    for (int m = threadIdx.x >> 2; m < M; m += SMALL_WAVES * 16) {
      float v = to_f(static_cast<const T*>(dy.p)[m * dy.ld + n]);
      if (act != ACT_NONE) v *= act_grad<T>(act, to_f(static_cast<const T*>(z.p)[m * z.ld + n]));
      s += v;
    }
#pragma unroll
  for (int d = 4; d < 64; d <<= 1) s += __shfl_xor(s, d, 64);
  float* part = reinterpret_cast<float*>(lds);
  if ((threadIdx.x & 63) < 4) part[(threadIdx.x >> 6) * 4 + c] = s;
  __syncthreads();
  if (threadIdx.x >= 4 || n >= N) return;
  float t = 0.0f;
#pragma unroll
  for (int i = 0; i < SMALL_WAVES; i++) t += part[i * 4 + c];
  db[n] = from_f<T>(t);
}

// The splits' sums in their order, then the epilogue.
template <typename T>
__global__ __launch_bounds__(256) void k_join(Epilogue e, int64_t M, int N, int splits) {
  const int64_t count = M * N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    float v = 0.0f;
#pragma unroll 8
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
// Bound by memory: dy and z read, dz written; 8192 x 4096 bf16 gelu 42 us, 4.8 TB/s.

#define DZ_COLUMNS 128

template <typename T>
__global__ __launch_bounds__(256) void k_dz(const T* dy, int64_t ldy, const T* z, T* dz, int64_t ldd, T* db, float* part,
                                            int M, int N, int act, int rows_per) {
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
        store8<T>(dz + m * ldd + n, o);
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
          if (dz) dz[m * ldd + n + i] = from_f<T>(v);
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

// ---- padded copies -----------------------------------------------------------------
//
// Rows that do not start on 16 bytes cost the tile kernel guarded loads through
// registers.  The backward products, which read them down the rows, are
// faster over copies with padded rows (bf16 3000 x 1001 x 999: dw 95 -> 42 us);
// the forward product and fp32 only where they are large.

struct Copies {
  Mat from[2];
  void* to[2];
  int64_t ld[2];                 // of the copies, a whole number of chunks
};

// A wave a row.
template <typename T>
__global__ __launch_bounds__(256) void k_pack(Copies c) {
  constexpr int E = 16 / sizeof(T);
  const int64_t all = (int64_t)c.from[0].rows + c.from[1].rows;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < all; r += (int64_t)gridDim.x * 4) {
    const int w = r >= c.from[0].rows;
    const int row = (int)(w ? r - c.from[0].rows : r);
    T* to = static_cast<T*>(c.to[w]) + row * c.ld[w];
#pragma unroll 2
    for (int at = (threadIdx.x & 63) * E; at < c.ld[w]; at += 64 * E)
      *reinterpret_cast<u32x4*>(to + at) = fetch<T>(c.from[w], row, at);
  }
}

// ---- a few rows ----------------------------------------------------------------------
//
// y for up to ROWS rows of x: a wave reads OUT rows of the weight at a time, 1 KB of
// each with one load a lane, and multiplies in fp32; `share` waves of a workgroup
// share the rows of a long reduction.  The weight's bytes are what there is to do:
// 1 x 4096 x 16,384 bf16 23 us, 5.9 TB/s (the tiles of k_gemm_small: 34 us), fp32 50
// us, 5.4 TB/s (69).

#define FEW_WAVES 8

template <typename T, int ROWS, int OUT>
__global__ __launch_bounds__(FEW_WAVES * 64) void k_few(Mat x, Mat w, Epilogue e, int M, int N, int K, int share) {
  constexpr int E = 16 / sizeof(T), SUMS = ROWS * OUT;
  __shared__ float sums[FEW_WAVES][SUMS];
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, groups = FEW_WAVES / share;
  const int64_t first = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * groups * OUT;
  const int64_t n0 = first + wave / share * OUT;
  float acc[ROWS][OUT];
#pragma unroll
  for (int m = 0; m < ROWS; m++)
#pragma unroll
    for (int o = 0; o < OUT; o++) acc[m][o] = 0.0f;
  if (n0 < N) {
    const T *px[ROWS], *pw[OUT];                     // rows past the last one repeat it
#pragma unroll
    for (int m = 0; m < ROWS; m++) px[m] = static_cast<const T*>(x.p) + (m < M ? m : M - 1) * x.ld;
#pragma unroll
    for (int o = 0; o < OUT; o++) pw[o] = static_cast<const T*>(w.p) + (n0 + o < N ? n0 + o : N - 1) * w.ld;
    const int step = share * 64 * E;
    int64_t k = (int64_t)(wave % share * 64 + l) * E;
#pragma unroll 2
    for (; k + E <= K; k += step) {
      Pack16<T> u[ROWS], v[OUT];
#pragma unroll
      for (int o = 0; o < OUT; o++) v[o].raw = load16(pw[o] + k);
#pragma unroll
      for (int m = 0; m < ROWS; m++) u[m].raw = load16(px[m] + k);
#pragma unroll
      for (int i = 0; i < E; i++)
#pragma unroll
        for (int m = 0; m < ROWS; m++)
#pragma unroll
          for (int o = 0; o < OUT; o++) acc[m][o] = fmaf(to_f(u[m].e[i]), to_f(v[o].e[i]), acc[m][o]);
    }
    for (; k < K; k++)                               // the lane in whose chunk the rows end; others are past it
#pragma unroll
      for (int m = 0; m < ROWS; m++)
#pragma unroll
        for (int o = 0; o < OUT; o++) acc[m][o] = fmaf(to_f(px[m][k]), to_f(pw[o][k]), acc[m][o]);
  }
#pragma unroll
  for (int m = 0; m < ROWS; m++)
#pragma unroll
    for (int o = 0; o < OUT; o++) {
      const float t = wave_sum(acc[m][o]);
      if (l == 0) sums[wave][m * OUT + o] = t;
    }
  __syncthreads();
  if ((int)threadIdx.x >= groups * SUMS) return;
  const int g = threadIdx.x / SUMS, j = threadIdx.x % SUMS, m = j / OUT;
  const int64_t n = first + g * OUT + j % OUT;
  if (m >= M || n >= N) return;
  float t = 0.0f;
  for (int i = 0; i < share; i++) t += sums[g * share + i][j];
  finish<T>(e, m, (int)n, N, t);
}

// ---- host side ---------------------------------------------------------------------

int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

struct Plan {
  int tile, tiles_m, tiles_n, splits, k_per;
  bool deep;                     // four stages instead of two
};

int elt(int dtype) { return dtype == CIT_FP32 ? 4 : 2; }

enum { TILE_32, TILE_64, TILE_128, TILE_256 };

// Outputs for 32 x 32 tiles: a few rows or columns, or less than a 64 x 64 tile for each compute unit.  Measured,
// forward, 32 against 64: bf16 1 x 4096 x 16384 34 / 46 us, 512 x 1024 x 1024 6.7 / 7.8, 2048 x 512 x 512 8.4 / 5.6
// (that one has 256 tiles); fp32 1 x 4096 x 16384 68 / 262 us, 512 x 1024 x 1024 17 / 21, 2048 x 512 x 512 19 / 14.
bool small(int M, int N) { return M <= 32 || N <= 32 || (int64_t)cdiv(M, 64) * cdiv(N, 64) < 256; }

// The tile of a product whose operands take direct loads.  Larger tiles load less (what the L2s deliver, about
// 10 TB/s, bounds 64 x 64 ones of 16-bit types) but fill the last round of the 256 compute units less.  Measured,
// us at K = 1024, by tiles of 128 in steps s of 256, r = steps of 256 tiles of 256:
//   bf16   s   1   2   3   4   5   6   7   8   9  10  12      128: 19 ceil(s / 2), 4 less where s is odd
//         128 13  21  34  40  53  59  71  77  88  96 114
//         256 30  30  31  34  58  60  61  67  93  94  98      r = 1, 1, 1, 1, 2, 2, 2, 2, 3, 3, 3: 30.5 r + 1
//          64 14  28  38  53  66  78  90 105 117 128 152
//   fp32  the matrix cores: 64 x 64 tiles 18.3 a round of 256, 128 x 128 ones 65: by the rounds alone
// Under K = 512 what a tile starts and ends with counts more: 64 longer (bf16 K = 256, s = 2: 10.5 / 11.0 / 15.0).
int direct_tile(int M, int N, int K, int es) {
  const auto steps = [&](int t) { return ((int64_t)cdiv(M, t) * cdiv(N, t) + 255) / 256; };
  const int64_t s = steps(128);
  if (es == 4) return K >= 512 && 36 * s < 10 * steps(64) ? TILE_128 : TILE_64;
  if (K < 512 && s <= 3) return TILE_64;
  if (61 * steps(256) + 2 < 38 * ((s + 1) / 2) - (s & 1 ? 8 : 0)) return TILE_256;
  return s > 1 || (int64_t)cdiv(M, 128) * cdiv(N, 128) >= 208 ? TILE_128 : TILE_64;
}

// Splits of a long reduction for few outputs, and the tile they take; 1: not of that kind.  For operands that take
// direct loads (ks: one is read down its rows).  Split so / as before, us: bf16 dw of 65,536 rows x 256 x 512 51 / 111,
// 32,768 x 768 x 768 72 / 261, 9000 x 1024 x 512 29 / 58, 4096 x 512 x 416 15 / 18, forward 256 x 4096 x 16,384 51 / 109,
// 256 x 4096 x 4096 25 / 33 (but 512 x 1024 x 4096 19 / 16, dw 4096 x 256 x 128 11 / 9); fp32 dw 32,768 x 768 x 768
// 314 / 557, forward 256 x 4096 x 16,384 281 / 445 (but dw 65,536 x 128 x 128 52 / 41).
int long_splits(int M, int N, int K, int es, bool ks, int& tile) {
  const int64_t c64 = (int64_t)cdiv(M, 64) * cdiv(N, 64), c128 = (int64_t)cdiv(M, 128) * cdiv(N, 128);
  const int from = c128 > 64 || (es == 2 && !ks && c64 <= 128) ? 8192 : 4096;
  if (K < from || M < 64 || N < 64 || c128 > 128 || c64 < (K < 32768 ? 16 : 8)) return 1;
  tile = c64 > 96 ? TILE_128 : TILE_64;
  // a workgroup a compute unit of large tiles, two of small ones; each split long enough to pay for its sums
  int64_t want = tile == TILE_128 ? 256 / c128 : 512 / c64;
  const int most = K / (es == 2 ? 1024 : 512);
  if (want > most) want = most;
  return (int)(want > 32 ? 32 : want);
}

Plan plan(int M, int N, int K, int es, bool aligned, bool ks) {
  Plan p;
  p.tile = small(M, N) ? TILE_32 : aligned ? direct_tile(M, N, K, es) : TILE_64;
  int split = 1;
  if (aligned) split = long_splits(M, N, K, es, ks, p.tile);
  const int t = 32 << p.tile, bk = 128 / es, kt = cdiv(K, bk);
  p.tiles_m = cdiv(M, t);
  p.tiles_n = cdiv(N, t);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  p.deep = p.tile == TILE_128 && tiles * split <= 256;   // one workgroup on a compute unit: 2048^3 bf16 31 -> 25 us
  int want = split;
  // A few small tiles: the launch shares the reduction out too, at least 4 k tiles for each wave (fp32 dw of 4096 rows x
  // 512 x 418: 39 -> 34 us).
  if (p.tile == TILE_32 && tiles < 256) {
    want = (int)(512 / tiles);
    if (want > kt / (SMALL_WAVES * 4)) want = kt / (SMALL_WAVES * 4);
  }
  if (want < 1) want = 1;
  p.k_per = cdiv(kt, want) * bk;
  p.splits = K > 0 ? cdiv(K, p.k_per) : 1;
  return p;
}
// Of either kind of operands: what the matrices' addresses allow is not known here.
int64_t split_bytes(int M, int N, int K, int es, bool ks) {
  const int a = plan(M, N, K, es, false, ks).splits, b = plan(M, N, K, es, true, ks).splits;
  return a > 1 || b > 1 ? align256((int64_t)(a > b ? a : b) * M * N * 4) : 0;
}

bool aligned(const void* p, int64_t ld, int es) {
  // 31 bits reach a tile's rows from its first
  return !((uintptr_t)p & 15) && (ld * es) % 16 == 0 && ld * es < 1 << 23;
}
bool direct(const Mat& a, bool ks, int es) { return aligned(a.p, a.ld, es) && (!ks || a.edge % (16 / es) == 0); }

// fp32 matrices of any width take direct loads too, 4 bytes a lane.
bool by_words(const Mat& a) { return !((uintptr_t)a.p & 3) && a.ld * 4 < 1 << 23; }

int64_t padded(int cols, int es) { return ((int64_t)cols * es + 15) / 16 * 16 / es; }

// Whether the backward pass copies unaligned operands of an M x N x K product first.  16-bit types: of many outputs, or
// of few over a reduction long enough to be split (bf16 dw of 65,536 rows x 512 x 418, us with / without: 100 / 413, of
// 8192 rows 35 / 35).  fp32, which has loads of 4 bytes: of much work (with / without: dx 30,000 x 301 over 1000 183 / 210,
// dw of 4096 rows x 1100 x 2051 220 / 248; dw of 3000 rows x 1001 x 999 85 / 70, of 65,536 rows x 512 x 418 311 / 284).
bool worth_copies(int M, int N, int K, int es) {
  int tile;
  if (es == 4) return !small(M, N) && (double)M * N * K >= 8e9;
  return !small(M, N) ? K >= 256 : K >= 16384 && long_splits(M, N, K, es, true, tile) > 1;
}

// Whether a forward product whose rows cannot start on 16 bytes copies its operands first: of enough work, and of
// enough work for each copied element.  With copies / without, us: fp16 4001 x 4003 x 2001 84 / 205, 65,536 x 200 x
// 418 47 / 59, 3000 x 1001 x 999 27 / 24, 4096 x 512 x 418 13 / 10; fp32 4001 x 4003 x 2001 535 / 562, 65,536 x 200 x
// 418 171 / 148, 3000 x 1001 x 999 67 / 68.
bool forward_copies(int M, int N, int K, int es) {
  return padded(K, es) != K && !small(M, N) && (double)M * N * K >= 4e9 &&
         (int64_t)M * N / ((int64_t)M + N) >= (es == 4 ? 512 : 192);
}

template <typename T, bool AKS, bool BKS, int TILE, int WM, int WN, int STAGES, bool AHEAD, int W = 16>
void launch_direct(const Mat& A, const Mat& B, const Epilogue& e, int M, int N, int K, const Plan& p,
                   hipStream_t stream) {
  const dim3 tiles = wide_grid((int64_t)p.tiles_m * p.tiles_n);
  hipLaunchKernelGGL((k_gemm_direct<T, AKS, BKS, TILE, TILE, WM, WN, STAGES, AHEAD, W>), dim3(tiles.x, p.splits, tiles.y),
                     dim3(WM * WN * 64), 0, stream, A, B, e, M, N, K, p.tiles_m, p.tiles_n, p.k_per);
}

template <typename T, bool AKS, bool BKS>
int product(Mat A, Mat B, Epilogue e, int M, int N, int K, void* work, hipStream_t stream) {
  const bool d = K > 0 && direct(A, AKS, sizeof(T)) && direct(B, BKS, sizeof(T));
  const bool words = !d && K > 0 && sizeof(T) == 4 && by_words(A) && by_words(B);
  const Plan p = plan(M, N, K, sizeof(T), d || words, AKS || BKS);
  const dim3 tiles = wide_grid((int64_t)p.tiles_m * p.tiles_n), grid(tiles.x, p.splits, tiles.y);
  if (p.splits > 1) e.part = static_cast<float*>(work);
  if (p.tile == TILE_32)
    hipLaunchKernelGGL((k_gemm_small<T, AKS, BKS>), grid, dim3(SMALL_WAVES * 64), 0, stream, A, B, e, M, N, K,
                       p.tiles_n, p.k_per);
  else if (words) {
    if constexpr (sizeof(T) == 4) {
      if (p.tile == TILE_64) launch_direct<T, AKS, BKS, 64, 2, 2, 2, true, 4>(A, B, e, M, N, K, p, stream);
      else launch_direct<T, AKS, BKS, 128, 2, 2, 2, true, 4>(A, B, e, M, N, K, p, stream);
    }
  } else if (!d && sizeof(T) == 2 && (int64_t)p.tiles_m * p.tiles_n <= 512) {
    if constexpr (sizeof(T) == 2)
      hipLaunchKernelGGL((k_gemm<T, AKS, BKS, 64, 64, 2, 2, 2>), grid, dim3(512), 0, stream, A, B, e, M, N, K, p.tiles_n,
                         p.k_per);
  } else if (!d)
    hipLaunchKernelGGL((k_gemm<T, AKS, BKS, 64, 64, 2, 2, 1>), grid, dim3(256), 0, stream, A, B, e, M, N, K, p.tiles_n,
                       p.k_per);
  else if (p.tile == TILE_64) launch_direct<T, AKS, BKS, 64, 2, 2, 2, true>(A, B, e, M, N, K, p, stream);
  else if (p.tile == TILE_128 && p.deep) launch_direct<T, AKS, BKS, 128, 2, 2, 4, true>(A, B, e, M, N, K, p, stream);
  else if (p.tile == TILE_128) launch_direct<T, AKS, BKS, 128, 2, 2, 2, true>(A, B, e, M, N, K, p, stream);
  else if constexpr (sizeof(T) == 2) launch_direct<T, AKS, BKS, 256, 2, 4, 2, false>(A, B, e, M, N, K, p, stream);
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

// Whether the backward pass goes in one launch, where act' is worked out again by every 32 columns of K: cells of
// that work, and rows for the column sums to walk.  One launch against five, us: fp32 relu 64 x 418 x 512 8.5 / 15,
// 2048 x 512 x 256 25 / 32, 512 x 1024 x 1024 (34e6 cells) 42 / 41; fp32 gelu (erfc) 512 x 418 x 512 (7e6) 23 / 25,
// 1024 x 418 x 512 (14e6) 40 / 36; bf16 gelu 2048 x 418 x 512 (27e6) 30 / 35, 512 x 1024 x 1024 33 / 22.
bool one_launch(int M, int N, int K, int es, int act) {
  if (K <= 0 || M > 2048 || N > 4096) return false;
  const int64_t k = cdiv(K, 32), cells = (int64_t)M * N * k;
  return cdiv(M, 32) * k <= 1024 && cdiv(N, 32) * k <= 1024 && cells <= (es == 4 && act > ACT_RELU ? 7 << 20 : 30 << 20);
}

// The pieces of a workspace, in their order; bytes 0: not needed.
struct Layout {
  int64_t copy[2], dz, sums, split;
  int64_t bytes() const { return copy[0] + copy[1] + dz + sums + split; }
};

Layout backward_layout(const void* x, int64_t ldx, const void* w, int64_t ldw, bool dx, bool dw, bool db, int M, int N,
                       int K, int es, int act) {
  Layout l = {};
  if (M <= 0 || N <= 0 || one_launch(M, N, K, es, act)) return l;
  if (K <= 0) dx = dw = false;
  // dz in rows of its own; where there is no activation dy stands for it, unless its rows are off 16 bytes, which
  // the size alone decides here
  const bool big_x = dx && worth_copies(M, K, N, es), big_w = dw && worth_copies(N, K, M, es);
  const bool odd = padded(N, es) != N;
  if ((dx || dw) && (act != ACT_NONE || (odd && (big_x || big_w)))) l.dz = align256(M * padded(N, es) * es);
  // the products' other operands are read down their rows: their width has to be whole chunks too
  const bool odd_k = padded(K, es) != K;
  if (big_w && (!aligned(x, ldx, es) || odd_k)) l.copy[0] = align256(M * padded(K, es) * es);
  if (big_x && (!aligned(w, ldw, es) || odd_k)) l.copy[1] = align256(N * padded(K, es) * es);
  if (db && cdiv(M, dz_rows(M, N)) > 1) l.sums = align256((int64_t)cdiv(M, dz_rows(M, N)) * N * 4);
  const int64_t a = dx ? split_bytes(M, K, N, es, true) : 0, b = dw ? split_bytes(N, K, M, es, true) : 0;
  l.split = a > b ? a : b;
  return l;
}

// The copies a layout asks for, at `work`; x and w become them.
template <typename T>
void make_copies(const Layout& l, Mat& x, Mat& w, char* work, hipStream_t stream) {
  if (!l.copy[0] && !l.copy[1]) return;
  Copies c = {};
  for (int i = 0; i < 2; i++) {
    Mat& m = i ? w : x;
    if (!l.copy[i]) continue;
    c.from[i] = m;
    c.to[i] = work + (i ? l.copy[0] : 0);
    c.ld[i] = padded(m.cols, sizeof(T));
    m = Mat{c.to[i], c.ld[i], m.rows, m.cols, (int)c.ld[i]};
  }
  const int64_t blocks = ((int64_t)c.from[0].rows + c.from[1].rows + 3) / 4;
  hipLaunchKernelGGL((k_pack<T>), dim3(blocks < 4096 ? (unsigned)blocks : 4096), dim3(256), 0, stream, c);
}

template <typename T>
int backward(Mat dy, const void* z, Mat x, Mat w, void* dx, void* dw, void* db, int M, int N, int K, int act,
             char* work, hipStream_t stream) {
  if (one_launch(M, N, K, sizeof(T), act)) {
    const int dx_tiles = dx ? cdiv(M, 32) * cdiv(K, 32) : 0, dw_tiles = dw ? cdiv(N, 32) * cdiv(K, 32) : 0;
    const int sums = db ? cdiv(N, 4) : 0;
    if (dx_tiles + dw_tiles + sums)
      hipLaunchKernelGGL((k_backward_small<T>), dim3(dx_tiles + dw_tiles + sums), dim3(SMALL_WAVES * 64), 0, stream, dy,
                         Mat{z, N, M, N, N}, x, w, static_cast<T*>(dx), static_cast<T*>(dw), static_cast<T*>(db), act,
                         M, N, K, sums, dw_tiles);
    return launch_status();
  }
  const Layout l =
      backward_layout(x.p, x.ld, w.p, w.ld, dx != nullptr, dw != nullptr, db != nullptr, M, N, K, sizeof(T), act);
  make_copies<T>(l, x, w, work, stream);
  work += l.copy[0] + l.copy[1];
  T* dz = l.dz ? reinterpret_cast<T*>(work) : nullptr;
  float* sums = l.sums ? reinterpret_cast<float*>(work + l.dz) : nullptr;
  const int64_t ldd = padded(N, sizeof(T));
  const int rows = dz_rows(M, N);
  if (dz || db) {
    hipLaunchKernelGGL((k_dz<T>), dim3(cdiv(N, DZ_COLUMNS), cdiv(M, rows)), dim3(256), 0, stream,
                       static_cast<const T*>(dy.p), dy.ld, static_cast<const T*>(z), dz, ldd, static_cast<T*>(db), sums,
                       M, N, act, rows);
    if (sums)
      hipLaunchKernelGGL((k_db<T>), dim3(cdiv(N, 64)), dim3(256), 0, stream, sums, static_cast<T*>(db), N,
                         cdiv(M, rows));
  }
  if (dz) dy = Mat{dz, ldd, M, N, (int)ldd};
  work += l.dz + l.sums;
  int rc = 0;
  Epilogue e = {};
  e.ldo = K;
  if (dx && K > 0) {
    e.out = dx;
    rc = product<T, false, true>(dy, w, e, M, K, N, work, stream);
  }
  if (!rc && dw && K > 0) {
    e.out = dw;
    rc = product<T, true, true>(dy, x, e, N, K, M, work, stream);
  }
  return rc ? rc : launch_status();
}

// Rows that k_few takes.  Against k_gemm_small, us at 4096 -> 4096 / 50,000 x 1001 / 65,536 x 512: bf16 1 row 6.0 / 18 /
// 12 against 9.3 / 29 / 17, 2 rows 7.1 / 22 / 18 against 9.4 / 29 / 17, 4 rows 10 / 36 / 30 against 9.4 / 29 / 17; fp32
// 4 rows 15 / 41 / 36 against 21 / 52 / 35, 8 rows 19 / 64 / 60 against 21 / 52 / 35.
bool few(int M, int K, int es) { return M <= (es == 4 ? 4 : 2) && (int64_t)K * es >= 1024; }

// Copies of both operands of a forward product, where their rows cannot start on 16 bytes, and the splits' sums.
Layout forward_layout(int M, int N, int K, int es) {
  Layout l = {};
  if (few(M, K, es)) return l;
  if (forward_copies(M, N, K, es)) {
    l.copy[0] = align256((int64_t)M * padded(K, es) * es);
    l.copy[1] = align256((int64_t)N * padded(K, es) * es);
  }
  l.split = split_bytes(M, N, K, es, false);
  return l;
}

template <typename T, int ROWS, int OUT>
void launch_few(const Mat& x, const Mat& w, const Epilogue& e, int M, int N, int K, hipStream_t stream) {
  // waves that have 2 KB of each row: as many as 4,096, of a large weight and 1 or 2 rows 8,192 (1 x 4096 x 16,384 bf16:
  // 34 and 23 us; 1 x 4096 x 4096 5.9 and 6.3; 3 x 4096 x 4096 fp32 15 and 20)
  const int64_t waves = ROWS > 2 || (int64_t)N * K * sizeof(T) < 48 << 20 ? 4096 : 8192;
  int share = 1;
  while (share < FEW_WAVES && (int64_t)cdiv(N, OUT) * share < waves && K >= share * 256 * (16 / (int)sizeof(T))) share *= 2;
  hipLaunchKernelGGL((k_few<T, ROWS, OUT>), wide_grid(cdiv(N, FEW_WAVES / share * OUT)), dim3(FEW_WAVES * 64), 0, stream,
                     x, w, e, M, N, K, share);
}

template <typename T>
int forward(Mat x, Mat w, const Epilogue& e, int M, int N, int K, char* work, hipStream_t stream) {
  if (few(M, K, sizeof(T))) {
    if (M == 1) launch_few<T, 1, 4>(x, w, e, M, N, K, stream);
    else if (M == 2) launch_few<T, 2, 4>(x, w, e, M, N, K, stream);
    else if constexpr (sizeof(T) == 4) launch_few<T, 4, 4>(x, w, e, M, N, K, stream);
    return launch_status();
  }
  Layout l = forward_layout(M, N, K, sizeof(T));
  char* sums = work + l.copy[0] + l.copy[1];
  if (aligned(x.p, x.ld, sizeof(T))) l.copy[0] = 0;
  if (aligned(w.p, w.ld, sizeof(T))) l.copy[1] = 0;
  make_copies<T>(l, x, w, work, stream);
  return product<T, false, false>(x, w, e, M, N, K, sums, stream);
}

// Sides whose 32-bit indexes have room for a tile past the end.
bool bad_sides(int M, int N, int K) {
  constexpr int MOST = INT32_MAX - 1023;
  return M < 0 || N < 0 || K < 0 || M > MOST || N > MOST || K > MOST;
}
bool bad_types(int dtype, int act) { return dtype < CIT_FP32 || dtype > CIT_FP16 || act < ACT_NONE || act > ACT_SILU; }

}  // namespace

extern "C" {

size_t cit_linear_forward_work_bytes(int M, int N, int K, int dtype) {
  return bad_types(dtype, 0) || bad_sides(M, N, K) || !M || !N || !K ? 0 : (size_t)forward_layout(M, N, K, elt(dtype)).bytes();
}

size_t cit_linear_backward_work_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* dx,
                                      const void* dw, const void* db, int M, int N, int K, int dtype, int act) {
  return bad_types(dtype, act) || bad_sides(M, N, K) ? 0
                               : (size_t)backward_layout(x, ldx, w, ldw, dx != nullptr, dw != nullptr, db != nullptr, M,
                                                         N, K, elt(dtype), act)
                                     .bytes();
}

int cit_linear_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual,
                       int64_t ldr, void* y, void* z, int M, int N, int K, int dtype, int act, void* work,
                       size_t work_bytes, hipStream_t stream) {
  if (bad_sides(M, N, K) || bad_types(dtype, act)) return -1;
  if (!M || !N) return 0;
  if (!y || (K && (!x || !w || ldx < K || ldw < K)) || (residual && ldr < N)) return -1;
  const size_t need = cit_linear_forward_work_bytes(M, N, K, dtype);
  if (need && (!work || work_bytes < need || ((uintptr_t)work & 15))) return -1;
  Epilogue e = {};
  e.bias = bias, e.res = residual, e.out = y, e.z = z, e.ldr = ldr, e.ldo = N, e.act = act;
  const Mat a = {x, ldx, M, K, K}, b = {w, ldw, N, K, K};
  char* p = static_cast<char*>(work);
  if (dtype == CIT_FP32) return forward<float>(a, b, e, M, N, K, p, stream);
  if (dtype == CIT_BF16) return forward<bf16_t>(a, b, e, M, N, K, p, stream);
  return forward<fp16_t>(a, b, e, M, N, K, p, stream);
}

int cit_linear_backward(const void* dy, int64_t ldy, const void* z, const void* x, int64_t ldx, const void* w,
                        int64_t ldw, void* dx, void* dw, void* db, int M, int N, int K, int dtype, int act, void* work,
                        size_t work_bytes, hipStream_t stream) {
  if (bad_sides(M, N, K) || !M || !N || bad_types(dtype, act)) return -1;
  if (!dy || ldy < N || (act != ACT_NONE && !z) || (dx && K && (!w || ldw < K)) || (dw && K && (!x || ldx < K)))
    return -1;
  const size_t need = cit_linear_backward_work_bytes(x, ldx, w, ldw, dx, dw, db, M, N, K, dtype, act);
  if (need && (!work || work_bytes < need || ((uintptr_t)work & 15))) return -1;
  const Mat a = {dy, ldy, M, N, N}, b = {x, ldx, M, K, K}, c = {w, ldw, N, K, K};
  char* p = static_cast<char*>(work);
  if (dtype == CIT_FP32) return backward<float>(a, z, b, c, dx, dw, db, M, N, K, act, p, stream);
  if (dtype == CIT_BF16) return backward<bf16_t>(a, z, b, c, dx, dw, db, M, N, K, act, p, stream);
  return backward<fp16_t>(a, z, b, c, dx, dw, db, M, N, K, act, p, stream);
}

}  // extern "C"
