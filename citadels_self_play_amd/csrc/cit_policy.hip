// The clipped policy loss with a KL term, and its gradient.  Row i of N holds
// the logits of one position's options: a row of [N][width], or entries
// offsets[i] .. offsets[i + 1] of one list (the ragged option rows of
// cit_cfr_targets); a mask leaves illegal entries out.  Over a row's legal
// entries
//
//   lp = l - logsumexp(l),  p = exp(lp),  rho = exp(lp_a - old),  d = lp - lq
//   L  = -min(rho A, clip(rho, 1 - low, 1 + high) A) + beta KL,  KL = sum p d
//   loss = sum_i w_i L_i
//   dloss/dl_j = w (g (1[j = a] - p_j) + beta p_j (d_j - KL))
//   g  = -rho A where the unclipped side is the minimum, else 0
//
// lq is the reference's log softmax.  KL is summed as p (d + exp(-d) - 1), which
// adds sum q - sum p = 0: every term is >= 0, so policies close together
// keep their digits (sum p d cancels to nothing there); where the reference is
// much the flatter one, whose sum then outweighs KL, as p d.  A row of weight 0 is
// not read; a row that leaves no entry counts nothing, and the gradients of
// both are 0.  An action outside its row makes the row NaN.  Where beta is 0 KL is
// told and no part of the loss, also where it is infinite.
#include <type_traits>

#include "cit_ops.h"

#define LONGEST (1 << 30)          // entries of a row: 32-bit indexes, with room for a step past the end

namespace {

struct Policy {
  const void *logits, *ref;      // ref: null without a KL term
  const uint8_t* mask;           // null: every entry is legal
  const int64_t* offsets;        // null: dense rows
  const int64_t* actions;
  const float *old, *adv, *weights;
  int64_t ld, ld_ref, ld_mask;   // dense: elements between rows
  int64_t rows, total;           // total: entries of the ragged list
  int32_t width;
  float low, high, beta, uniform;
  float *logp, *kl;
  double* part;                  // one sum of w L per workgroup
  void* grad;                    // null: no gradient
  const float* upstream;         // backward pass: the loss's gradient; null in the forward pass
  int32_t skip_one;              // backward pass: grad holds upstream = 1 already
  // a few long rows in parts, a workgroup each: first their sums, then (join) the row's, then the gradient
  int32_t parts, part_len, mode; // parts 1: whole rows, mode 0; else mode 1 sums, 2 gradient
  float* part_sums;              // [rows][parts] PartSums
  float* row_state;              // [rows] RowState
};

struct PartSums {                // maxima and sums of k_policy's pass 2 over one part
  float m, mr, s, sr, f, d;
};
struct RowState {                // what the gradient needs of a row
  float top, top_q, inv_s, L, dlogp, kl, live;
};

struct Row {
  int64_t at, at_ref, at_mask, at_grad;
  int len;
  bool bad;
};

__device__ __forceinline__ Row row_of(const Policy& a, int64_t i) {
  Row r;
  r.bad = false;
  if (a.offsets) {
    const int64_t s = a.offsets[i], e = a.offsets[i + 1];
    r.bad = s < 0 || e < s || e > a.total || e - s > LONGEST;
    r.at = r.at_ref = r.at_mask = r.at_grad = r.bad ? 0 : s;
    r.len = r.bad ? 0 : (int)(e - s);
  } else {
    r.at = i * a.ld, r.at_ref = i * a.ld_ref, r.at_mask = i * a.ld_mask, r.at_grad = i * a.width;
    r.len = a.width;
  }
  return r;
}

// e (x + exp(-x) - 1) from e, w = e x and er = e exp(-x); where the three would cancel, x w times
// the Chebyshev interpolation of (x + exp(-x) - 1) / x^2 on |x| <= 1/2 (off by 2^-24).
__device__ __forceinline__ float kl_term(float e, float er, float x, float w) {
  float s = -0.00019944873929489404f;
  s = fmaf(s, x, 0.0013982185628265142f);
  s = fmaf(s, x, -0.0083332359790802f);
  s = fmaf(s, x, 0.04166579246520996f);
  s = fmaf(s, x, -0.1666666716337204f);
  s = fmaf(s, x, 0.5f);
  // both sides worked out: as a branch a lane takes, either costs both and the exec mask's bookkeeping
  const float near = x * s * w, far = (w - e) + er;
  return fabsf(x) < 0.5f ? near : far;
}

// Sums and maxima over the G lanes that share a row: shuffles, and LDS between the waves of a wide row.
template <int G>
struct Lanes {
  static constexpr int WAVES = G > 64 ? G / 64 : 1;
  float (*lds)[4];               // [WAVES][4], wide rows only

  template <int N, bool MAX>
  __device__ __forceinline__ void all(float (&v)[N]) const {
#pragma unroll
    for (int d = (G > 64 ? 64 : G) / 2; d; d >>= 1)
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float o = __shfl_xor(v[i], d, 64);
        v[i] = MAX ? fmaxf(v[i], o) : v[i] + o;
      }
    if (G <= 64) return;
    const int w = threadIdx.x >> 6;
    __syncthreads();                                 // the last round's readers are done
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; i++) lds[w][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = lds[0][i];
    for (int k = 1; k < WAVES; k++)
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = MAX ? fmaxf(v[i], lds[k][i]) : v[i] + lds[k][i];
  }
};

// What a row's statistics say about the loss: from the action's shifted logit
// l = l_a - m, the sum s of exp(l_j - m), and kl.  The rows' values have either
// sign and a batch's sum is smaller than they are, so they are worked out and
// summed in 64 bits.  DOUBLE: the logarithm and exponential too, about 2,400
// cycles of a wave, where a wave has several rows or a row several waves; a row
// to a wave takes the 32-bit functions (65,536 x 1,000 bf16: 125 us, 145 with the
// others).
struct RowLoss {
  float logp, kl, dlogp;
  double loss;
};

template <bool DOUBLE>
__device__ __forceinline__ RowLoss row_loss(const Policy& a, int64_t i, double l, double s, float kl) {
  RowLoss v;
  const double logp = l - (DOUBLE ? log(s) : (double)logf((float)s));
  const double adv = a.adv[i], past = logp - (double)a.old[i];
  const double ratio = DOUBLE ? exp(past) : (double)expf((float)past);
  const double low = 1.0 - (double)a.low, high = 1.0 + (double)a.high;
  const double free = ratio * adv, held = (ratio < low ? low : ratio > high ? high : ratio) * adv;
  v.logp = (float)logp, v.kl = kl;
  v.dlogp = (float)(free <= held ? -free : held < free ? 0.0 : (double)NAN);
  v.loss = (free <= held || free != free ? -free : -held) + (a.ref && a.beta != 0.0f ? (double)a.beta * (double)kl : 0.0);
  return v;
}

__device__ __forceinline__ float weight_of(const Policy& a, int64_t i) { return a.weights ? a.weights[i] : a.uniform; }

// The logit of the row's action; NaN outside the row, -inf where it is illegal.
template <typename T>
__device__ __forceinline__ float action_logit(const Policy& a, const Row& r, int64_t i) {
  const int64_t k = a.actions[i];
  if (k < 0 || k >= r.len) return NAN;
  if (a.mask && !a.mask[r.at_mask + k]) return -INFINITY;
  return to_f(static_cast<const T*>(a.logits)[r.at + k]);
}

// E neighbouring entries of a row, in the words they were loaded as.
template <typename T, int E>
struct Pack {
  static constexpr int W = E * (int)sizeof(T) > 4 ? E * (int)sizeof(T) / 4 : 1;
  uint32_t w[W];

  __device__ __forceinline__ float get(int k) const {
    if (sizeof(T) == 4) return __builtin_bit_cast(float, w[k]);
    const uint16_t h = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
    return to_f(__builtin_bit_cast(T, (typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type)h));
  }
  __device__ __forceinline__ void set(int k, float f) {
    const T v = from_f<T>(f);
    if (sizeof(T) == 4) {
      w[k] = __builtin_bit_cast(uint32_t, f);
      return;
    }
    uint16_t h;
    __builtin_memcpy(&h, &v, 2);
    w[k >> 1] = k & 1 ? (w[k >> 1] & 0xffffu) | ((uint32_t)h << 16) : (w[k >> 1] & 0xffff0000u) | h;
  }
  // All of them at once: two 16-bit conversions are one instruction.
  __device__ __forceinline__ void set_all(const float (&f)[E]) {
    if (sizeof(T) == 4 || E == 1) {
#pragma unroll
      for (int k = 0; k < E; k++) set(k, f[k]);
      return;
    }
    typedef T Two __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int k = 0; k + 1 < E; k += 2) {
      const Two t = {from_f<T>(f[k]), from_f<T>(f[k + 1])};
      __builtin_memcpy(&w[k >> 1], &t, 4);
    }
  }
  // Not to be unpacked once for all passes: that doubles the registers a row takes.
  __device__ __forceinline__ void keep_packed() {
#pragma unroll
    for (int i = 0; i < W; i++) asm volatile("" : "+v"(w[i]));
  }
};
template <typename T, int E>
__device__ __forceinline__ Pack<T, E> load_pack(const T* row, const uint8_t* ok, int j, int len) {
  Pack<T, E> v;
  if (E > 1 && j + E <= len) {
    const u32x4 u = load16(row + j);
#pragma unroll
    for (int i = 0; i < Pack<T, E>::W; i++) v.w[i] = u[i & 3];
  } else {
#pragma unroll
    for (int i = 0; i < Pack<T, E>::W; i++) v.w[i] = 0;
#pragma unroll
    for (int i = 0; i < E; i++) v.set(i, j + i < len ? to_f(row[j + i]) : -INFINITY);
  }
  if (ok) {                      // illegal entries are -inf from here on
    if (E > 1 && j + E <= len) {
      struct __attribute__((packed, aligned(1))) Bytes { uint8_t b[E]; };
      const Bytes m = *reinterpret_cast<const Bytes*>(ok + j);
#pragma unroll
      for (int i = 0; i < E; i++)
        if (!m.b[i]) v.set(i, -INFINITY);
    } else {
#pragma unroll
      for (int i = 0; i < E; i++)
        if (j + i < len && !ok[j + i]) v.set(i, -INFINITY);
    }
  }
  return v;
}
template <typename T, int E>
__device__ __forceinline__ void store_pack(T* row, int j, int len, const Pack<T, E>& v) {
  if (E > 1 && j + E <= len) {
    u32x4 u;
#pragma unroll
    for (int i = 0; i < Pack<T, E>::W; i++) u[i & 3] = v.w[i];
    store16(row + j, u);
  } else {
#pragma unroll
    for (int i = 0; i < E; i++)
      if (j + i < len) row[j + i] = from_f<T>(v.get(i));
  }
}

// Entries of the list in front of the first row and behind the last: no gradient.
template <typename T>
__device__ void clear_ends(const Policy& a, int block, int blocks) {
  T* grad = static_cast<T*>(a.grad);
  const int64_t n = a.total;
  int64_t first = a.offsets[0], last = a.offsets[a.rows];
  first = first < 0 ? 0 : first > n ? n : first;
  last = last < first ? first : last > n ? n : last;
  const int64_t at = (int64_t)block * blockDim.x + threadIdx.x, step = (int64_t)blocks * blockDim.x;
  for (int64_t j = at; j < first; j += step) grad[j] = from_f<T>(0.0f);
  for (int64_t j = last + at; j < n; j += step) grad[j] = from_f<T>(0.0f);
}

#define LOG2E 1.44269504088896341f

// exp(x).  FINE: to the last place, for short rows; over long ones what the product x log2(e) is off by, |x| last
// places, averages out, and the instruction alone does (fp32 2,048 x 16,384: 93 us, 108).
template <bool FINE>
__device__ __forceinline__ float exp_of(float x) {
  return FINE ? expf(x) : __builtin_amdgcn_exp2f(x * LOG2E);
}

// A row by G lanes, each with up to NV packs of E entries in registers, so that
// the logits come from memory once; a longer row is read again in each pass.
//
//   pass 1  the maxima m of l and mr of the reference r
//   pass 2  e = exp(l - m), er = exp(r - mr) (a difference first, so
//           that no error is shared by all entries and a type's lowest value is
//           a number like others), x = (l - m) - (r - mr), hence er = e exp(-x).
//           s = sum e, sr = sum er, F = sum e (x + exp(-x) - 1): with
//           eta = 1 - sr / s,  d = x - L, L = -log1p(-eta), and
//           KL = F / s + eta - L.  One pass gives KL without its cancellation.
//           Where sr > 2 s that would take sr away from F: D = sum e x, and
//           KL = D / s - L.
//   pass 3  the gradient: exp(l - m) once more, 1 / s in what it is multiplied
//           with: rounded by half a step, where a log s in the exponent would put its
//           own rounding, up to ten steps, on all of a row alike
//
// bf16 with a reference is bound by the vector units (52 instructions an entry,
// three of them exponentials at a quarter of the rate), the others by memory.
// 4096 x 32,768 bf16, gradient included: 236 us, 3.4 TB/s, the vector units at
// work for 190 of them; without a reference 120 us, 4.5 TB/s; 509 x 50,001 masked,
// evaluated only, 23 us, 3.3 TB/s.
template <typename T, int G, int NV, int E, bool REF, bool PARTED>
__global__ __launch_bounds__(G > 256 ? G : 256, G == 1024 && !REF ? 8 : G > 256 ? 4 : E > 1 && REF && !PARTED ? 5 : 2) void k_policy(Policy a, int64_t row_blocks, int tail) {
  constexpr int THREADS = G > 256 ? G : 256, GROUPS = THREADS / G;
  constexpr bool FINE = E == 1;
  __shared__ double sums[GROUPS];
  __shared__ float between[G > 64 ? G / 64 : 1][4];
  __shared__ RowLoss said;
  const float up = a.upstream ? *a.upstream : 1.0f;
  if (a.upstream && a.skip_one && up == 1.0f) return;
  const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (b >= row_blocks) {
    if (b < row_blocks + tail) clear_ends<T>(a, (int)(b - row_blocks), tail);
    return;
  }
  const int lane = threadIdx.x % G;
  int64_t i = b * GROUPS + threadIdx.x / G;
  int part = 0;
  if (PARTED) {
    part = (int)(i % a.parts);
    i /= a.parts;
  }
  const Lanes<G> lanes{between};
  double counted = 0.0;
  if (i < a.rows) {              // the same for all lanes of a row: barriers inside are met by all of a wide row
    Row r = row_of(a, i);
    if (PARTED) {
      const int skip = part * a.part_len;
      r.at += skip, r.at_ref += skip, r.at_mask += skip, r.at_grad += skip;
      r.len = r.len - skip < a.part_len ? r.len - skip : a.part_len;
    }
    const float w = weight_of(a, i);
    const T* lrow = static_cast<const T*>(a.logits) + r.at;
    const T* qrow = REF ? static_cast<const T*>(a.ref) + r.at_ref : nullptr;
    const uint8_t* ok = a.mask ? a.mask + r.at_mask : nullptr;
    T* grow = a.grad ? static_cast<T*>(a.grad) + r.at_grad : nullptr;
    RowLoss v = {0.0f, 0.0f, 0.0f, 0.0};
    bool live = w != 0.0f && !r.bad;
    const float of_action = !PARTED && live ? action_logit<T>(a, r, i) : 0.0f;
    float top = 0.0f, top_q = 0.0f, inv_s = 0.0f, L = 0.0f;
    const bool held = r.len <= G * NV * E;
    Pack<T, E> l[NV], q[NV];
    // f(j, l, q) for every pack of the row this lane has
    auto visit = [&](auto&& f) {
      if (held) {
#pragma unroll
        for (int n = 0; n < NV; n++)
          if ((n * G + lane) * E < r.len) {
            l[n].keep_packed();
            if (REF) q[n].keep_packed();
            f((n * G + lane) * E, l[n], q[n]);
          }
      } else {
        for (int j = lane * E; j < r.len; j += G * E) {
          const Pack<T, E> x = load_pack<T, E>(lrow, ok, j, r.len);
          f(j, x, REF ? load_pack<T, E>(qrow, ok, j, r.len) : x);
        }
      }
    };
    if (live) {
      if (held) {
#pragma unroll
        for (int n = 0; n < NV; n++) {
          const int j = (n * G + lane) * E;
          if (j < r.len) {
            l[n] = load_pack<T, E>(lrow, ok, j, r.len);
            if (REF) q[n] = load_pack<T, E>(qrow, ok, j, r.len);
          }
        }
      }
    }
    if (PARTED && a.mode == 2) {
      const RowState* state = reinterpret_cast<const RowState*>(a.row_state) + i;
      live = state->live != 0.0f;
      top = state->top, top_q = state->top_q, inv_s = state->inv_s, L = state->L;
      v.dlogp = state->dlogp, v.kl = state->kl;
    } else if (live) {
      float m[REF ? 2 : 1];
      for (float& k : m) k = -INFINITY;
      visit([&](int, const Pack<T, E>& x, const Pack<T, E>& y) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < E; k++) {
          m[0] = fmaxf(m[0], x.get(k));
          if (REF) m[REF ? 1 : 0] = fmaxf(m[REF ? 1 : 0], y.get(k));
        }
      });
      lanes.template all<REF ? 2 : 1, true>(m);
      top = m[0] == -INFINITY ? 0.0f : m[0];
      if (REF) top_q = m[REF ? 1 : 0] == -INFINITY ? 0.0f : m[REF ? 1 : 0];
      constexpr int SUMS = REF ? 4 : 1;
      float t[SUMS] = {};
      visit([&](int, const Pack<T, E>& x, const Pack<T, E>& y) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < E; k++) {
          const float dl = x.get(k) - top;
          const float e = exp_of<FINE>(dl);
          t[0] += e;
          if (REF) {
            const float dr = y.get(k) - top_q;
            const float er = exp_of<FINE>(dr);
            t[REF ? 1 : 0] += er;
            // An entry of no probability (l = -inf, and r perhaps too) is finite here: it counts er.  r = -inf
            // counts nothing where p is 0 to its last bit.
            const float d = fmaxf(dl - dr, -200.0f), w = e == 0.0f ? 0.0f : e * d;
            t[REF ? 2 : 0] += kl_term(e, er, d, w);
            t[SUMS - 1] += w;
          }
        }
      });
      lanes.template all<SUMS, false>(t);
      if (PARTED && a.mode == 1) {
        if (lane == 0)
          reinterpret_cast<PartSums*>(a.part_sums)[i * a.parts + part] =
              PartSums{m[0], m[REF ? 1 : 0], t[0], REF ? t[REF ? 1 : 0] : 0.0f, REF ? t[REF ? 2 : 0] : 0.0f,
                       REF ? t[SUMS - 1] : 0.0f};
        return;
      }
      live = !(t[0] == 0.0f);
      if (live) {
        inv_s = 1.0f / t[0];
        float kl = 0.0f;
        if (REF) {
          const float eta = (t[0] - t[REF ? 1 : 0]) / t[0];
          // where the reference's sum is much the smaller, 1 - eta has lost what it is (fp32, an even row of 4,000
          // against a reference that is sure of one entry: KL 9.70138 for 9.70151)
          L = eta > 0.5f ? logf(t[0] / t[REF ? 1 : 0]) : -log1pf(-eta);
          kl = eta < -1.0f ? t[SUMS - 1] / t[0] - L
                           : t[REF ? 2 : 0] / t[0] + (fabsf(eta) < 0.01f ? -eta * eta * fmaf(eta, fmaf(eta, 0.25f, 1.0f / 3.0f), 0.5f) : eta - L);
          kl = kl < 0.0f ? 0.0f : kl;
        }
        const double l_a = (double)of_action - top;
        if (G > 64) {            // the first wave for all
          if (threadIdx.x < 64) {
            v = row_loss<true>(a, i, l_a, t[0], kl);
            if (threadIdx.x == 0) said = v;
          }
          __syncthreads();
          v = said;
        } else {
          v = row_loss<G != 64>(a, i, l_a, t[0], kl);
        }
      }
    }
    if (PARTED && a.mode == 1) return;
    if (r.bad && w != 0.0f) v = {NAN, NAN, NAN, (double)NAN};
    if (!a.upstream && !PARTED && lane == 0) {
      a.logp[i] = v.logp, a.kl[i] = v.kl;
      counted = w != 0.0f ? (double)w * v.loss : 0.0;
    }
    if (grow) {
      const int64_t action = PARTED ? a.actions[i] - (int64_t)part * a.part_len : a.actions[i];
      const float uw = up * w;
      if (live) {
        const float bw = REF ? uw * a.beta : 0.0f;
        // exp(l - m) (by_x x + flat), 1 / s in both
        const float flat = (-uw * v.dlogp - (bw != 0.0f ? bw * (L + v.kl) : 0.0f)) * inv_s, by_x = bw * inv_s;
        auto prob = [&](float lx) __attribute__((always_inline)) { return exp_of<FINE>(lx - top); };
        // x within what times 0 is 0: an entry of no probability has no gradient
        auto slope = [&](float lx, float qx) __attribute__((always_inline)) {
          return REF ? fmaf(by_x, fminf(fmaxf((lx - top) - (qx - top_q), -1e30f), 1e30f), flat) : flat;
        };
        visit([&](int j, const Pack<T, E>& x, const Pack<T, E>& y) __attribute__((always_inline)) {
          Pack<T, E> g = {};
          float o[E];
#pragma unroll
          for (int k = 0; k < E; k++) {
            const float lx = x.get(k);
            o[k] = prob(lx) * slope(lx, REF ? y.get(k) : 0.0f);
          }
          g.set_all(o);
          store_pack<T, E>(grow, j, r.len, g);
          if (action >= j && action < j + E && action < r.len) {
            // the chosen entry has uw dlogp besides; its lane has just stored the pack
            const int k = (int)(action - j);
            float lx = -INFINITY, qx = -INFINITY;
#pragma unroll
            for (int c = 0; c < E; c++)
              if (c == k) {
                lx = x.get(c);
                if (REF) qx = y.get(c);
              }
            if (!(ok && !ok[action])) grow[action] = from_f<T>(fmaf(prob(lx), slope(lx, qx), uw * v.dlogp));
          }
        });
      } else {
        Pack<T, E> zero = {};
        for (int j = lane * E; j < r.len; j += G * E) store_pack<T, E>(grow, j, r.len, zero);
      }
    }
  }
  if (a.upstream || PARTED) return;
  if (lane == 0) sums[threadIdx.x / G] = counted;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int k = 0; k < GROUPS; k++) s += sums[k];
    a.part[b] = s;
  }
}

// The parts of a row together, a wave a row.  With a = exp(m_part - m) and the
// shift of x, delta = (m_part - m) - (mr_part - mr):
//   sum e x = a (D_part + delta s_part)
//   sum e (x + exp(-x) - 1) = a (F_part + delta (s_part - sr_part) + (delta + exp(-delta) - 1) sr_part)
// where a exp(-delta) = exp(mr_part - mr) stands for the product once delta is
// not small: either factor may be 0 or infinite alone.
template <typename T>
__global__ __launch_bounds__(64) void k_policy_join(Policy a) {
  const float up = a.upstream ? *a.upstream : 1.0f;
  if (a.upstream && a.skip_one && up == 1.0f) return;
  const int64_t i = blockIdx.x;
  const int lane = threadIdx.x;
  const float w = weight_of(a, i);
  const Row r = row_of(a, i);
  const bool ref = a.ref != nullptr;
  PartSums p = {-INFINITY, -INFINITY, 0.0f, 0.0f, 0.0f, 0.0f};
  if (w != 0.0f && lane < a.parts) p = reinterpret_cast<const PartSums*>(a.part_sums)[i * a.parts + lane];
  const float m = wave_max(p.m), mr = wave_max(p.mr);
  const float top = m == -INFINITY ? 0.0f : m, top_q = !ref || mr == -INFINITY ? 0.0f : mr;
  double s = 0.0, sr = 0.0, f = 0.0, d = 0.0;
  if (ref && p.sr != 0.0f) f = sr = exp((double)p.mr - top_q) * p.sr;  // f: of a part that has no weight in the row
  if (p.s != 0.0f) {                                 // NaN too
    const double x = (double)p.m - top, y = exp(x);
    s = y * p.s;
    if (ref && y != 0.0) {
      const double delta = x - ((double)p.mr - top_q);
      d = y * (p.d + delta * p.s);
      f = fabs(delta) < 1.0 ? y * (p.f + delta * ((double)p.s - p.sr) + (delta + expm1(-delta)) * p.sr)
                            : y * (p.f + delta * p.s - p.sr) + sr;
    }
  }
  s = wave_sum(s), sr = wave_sum(sr), f = wave_sum(f), d = wave_sum(d);
  if (lane) return;
  RowLoss v = {0.0f, 0.0f, 0.0f, 0.0};
  RowState state = {top, top_q, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (w != 0.0f && !(s == 0.0)) {
    float kl = 0.0f;
    if (ref) {
      const double eta = (s - sr) / s, L = -log1p(-eta);
      state.L = (float)L;
      kl = (float)(eta < -1.0 ? d / s - L : f / s + (fabs(eta) < 1e-4 ? -eta * eta * (0.5 + eta / 3.0) : eta - L));
      kl = kl < 0.0f ? 0.0f : kl;
    }
    state.inv_s = (float)(1.0 / s);
    v = row_loss<true>(a, i, (double)action_logit<T>(a, r, i) - top, s, kl);
    state.dlogp = v.dlogp, state.kl = v.kl, state.live = 1.0f;
  }
  reinterpret_cast<RowState*>(a.row_state)[i] = state;
  if (a.upstream) return;
  a.logp[i] = v.logp, a.kl[i] = v.kl;
  a.part[i] = w != 0.0f ? (double)w * v.loss : 0.0;
}

#define SUM_BLOCKS 256

// Sums in a fixed order: each workgroup its share to part2, or one workgroup the whole to loss.
__global__ __launch_bounds__(1024) void k_policy_sum(const double* part, int64_t count, double* part2, float* loss) {
  __shared__ double sums[16];
  const int64_t share = (count + gridDim.x - 1) / gridDim.x;
  const int64_t first = share * blockIdx.x, last = first + share < count ? first + share : count;
  double s = 0.0;
  for (int64_t i = first + threadIdx.x; i < last; i += 1024) s += part[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = 0.0;
  for (int i = 0; i < 16; i++) s += sums[i];
  if (part2) part2[blockIdx.x] = s;
  else *loss = (float)s;
}

// Lanes of a row and entries they hold: `width` is a dense row's, or twice a
// ragged batch's mean (its rows' lengths stay on the device).
struct Shape {
  int lanes, packs;              // lanes of a row; packs of 16 bytes (packs = 0: single entries, 4 a lane)
};
Shape shape_of(int64_t width, int dtype) {
  const int64_t e = dtype == CIT_FP32 ? 4 : 8;
  if (width <= 64) return {16, 0};
  if (width <= 256) return {64, 0};
  if (width <= 64 * 4 * e) return {64, 4};
  if (width <= 256 * 4 * e) return {256, 4};
  if (width <= 512 * 8 * e) return {512, 8};
  return {1024, 8};
}
int64_t width_of(int64_t rows, int64_t total, int width, bool ragged) {
  return ragged ? (rows > 0 ? 2 * (total / rows) : 0) : width;
}
int64_t row_blocks(int64_t rows, const Shape& s) {
  const int groups = s.lanes > 256 ? 1 : 256 / s.lanes;
  return (rows + groups - 1) / groups;
}

// Workgroups for each of a few long dense rows, 1 where the rows fill the chip or are short; parts of whole packs.
// 8 rows of 131,072 bf16 entries, gradient included: 46 us whole, 25 in parts.
int parts_of(int64_t rows, int width, bool ragged) {
  if (ragged || rows > 128 || width < 16384) return 1;
  int64_t parts = 512 / rows;
  if (parts > 64) parts = 64;
  const int most = (int)(((int64_t)width + 4095) / 4096);              // 4,096 entries are held by 256 lanes in any type
  return parts < most ? (int)parts : most;
}
int part_len(int width, int parts) { return ((width - 1) / parts + 1 + 7) / 8 * 8; }

template <typename T, int G, int NV, int E, bool PARTED = false>
void launch_shape(const Policy& a, int64_t blocks, hipStream_t stream) {
  const int tail = a.grad && a.offsets ? 64 : 0;
  const dim3 grid = wide_grid(blocks + tail), block(G > 256 ? G : 256);
  if (a.ref) hipLaunchKernelGGL((k_policy<T, G, NV, E, true, PARTED>), grid, block, 0, stream, a, blocks, tail);
  else hipLaunchKernelGGL((k_policy<T, G, NV, E, false, PARTED>), grid, block, 0, stream, a, blocks, tail);
}

template <typename T>
int launch(Policy a, const Shape& s, hipStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  if (a.parts > 1) {
    a.mode = 1;
    launch_shape<T, 256, 4, E, true>(a, a.rows * a.parts, stream);
    hipLaunchKernelGGL((k_policy_join<T>), dim3((unsigned)a.rows), dim3(64), 0, stream, a);
    a.mode = 2;
    if (a.grad) launch_shape<T, 256, 4, E, true>(a, a.rows * a.parts, stream);
    return launch_status();
  }
  const int64_t blocks = row_blocks(a.rows, s);
  if (s.lanes == 16) launch_shape<T, 16, 4, 1>(a, blocks, stream);
  else if (s.lanes == 64 && !s.packs) launch_shape<T, 64, 4, 1>(a, blocks, stream);
  else if (s.lanes == 64) launch_shape<T, 64, 4, E>(a, blocks, stream);
  else if (s.lanes == 256) launch_shape<T, 256, 4, E>(a, blocks, stream);
  else if (s.lanes == 512) launch_shape<T, 512, 8, E>(a, blocks, stream);
  else launch_shape<T, 1024, 8, E>(a, blocks, stream);
  return launch_status();
}

// Sums and row states of rows in parts, at `work`.
size_t part_bytes(int64_t rows, int parts) {
  return parts > 1 ? (size_t)rows * (parts * sizeof(PartSums) + sizeof(RowState)) : 0;
}
void set_parts(Policy& a, void* work) {
  a.parts = parts_of(a.rows, a.width, a.offsets != nullptr);
  a.part_len = a.parts > 1 ? part_len(a.width, a.parts) : 0;
  a.mode = 0;
  a.part_sums = static_cast<float*>(work);
  a.row_state = a.part_sums + (a.parts > 1 ? a.rows * a.parts * (int64_t)(sizeof(PartSums) / 4) : 0);
}

int run(const Policy& a, int dtype, hipStream_t stream) {
  const Shape s = shape_of(width_of(a.rows, a.total, a.width, a.offsets != nullptr), dtype);
  if (dtype == CIT_FP32) return launch<float>(a, s, stream);
  if (dtype == CIT_BF16) return launch<bf16_t>(a, s, stream);
  return launch<fp16_t>(a, s, stream);
}

bool bad(const Policy& a, int dtype) {
  if (dtype < CIT_FP32 || dtype > CIT_FP16 || a.rows < 0 || a.rows > INT32_MAX / 2) return true;
  if (!(a.low >= 0.0f) || !(a.high >= 0.0f) || !(a.beta >= 0.0f)) return true;
  if (!a.rows) return false;
  if (!a.actions || !a.old || !a.adv) return true;
  if (a.offsets) return a.total < 0 || (a.total && !a.logits);
  if (a.width < 0 || a.width > LONGEST || (a.width && !a.logits)) return true;
  return a.ld < a.width || (a.ref && a.ld_ref < a.width) || (a.mask && a.ld_mask < a.width);
}

}  // namespace

extern "C" {

size_t cit_policy_loss_work_bytes(int64_t rows, int width, int ragged) {
  if (rows <= 0 || (!ragged && width < 0)) return 0;
  return ((size_t)rows + SUM_BLOCKS) * sizeof(double) + part_bytes(rows, parts_of(rows, width, ragged != 0));
}

int cit_policy_loss(const void* logits, int64_t ld, const void* ref, int64_t ld_ref, const uint8_t* mask,
                    int64_t ld_mask, const int64_t* offsets, int64_t total, int64_t rows, int width,
                    const int64_t* actions, const float* old_logp, const float* advantages, const float* weights,
                    float low, float high, float kl_coef, int dtype, float* loss, float* logp, float* kl, void* grad,
                    void* work, size_t work_bytes, hipStream_t stream) {
  Policy a = {logits, ref, mask, offsets, actions, old_logp, advantages, weights, ld, ld_ref, ld_mask, rows, total,
              width, low, high, kl_coef, rows > 0 ? (float)(1.0 / (double)rows) : 0.0f, logp, kl,
              static_cast<double*>(work), grad, nullptr, 0};
  if (bad(a, dtype) || !loss || (rows && (!logp || !kl))) return -1;
  const size_t need = cit_policy_loss_work_bytes(rows, width, offsets != nullptr);
  if (need && (!work || work_bytes < need || ((uintptr_t)work & 15))) return -1;
  set_parts(a, a.part + rows + SUM_BLOCKS);
  if (rows) {
    const int rc = run(a, dtype, stream);
    if (rc) return rc;
  }
  const int64_t parts =
      !rows ? 0
            : a.parts > 1 ? rows : row_blocks(rows, shape_of(width_of(rows, total, width, offsets != nullptr), dtype));
  if (parts > 64 * SUM_BLOCKS) {                     // one workgroup would be at it for longer than two launches take
    double* part = a.part + rows;
    hipLaunchKernelGGL(k_policy_sum, dim3(SUM_BLOCKS), dim3(1024), 0, stream, a.part, parts, part, nullptr);
    hipLaunchKernelGGL(k_policy_sum, dim3(1), dim3(1024), 0, stream, part, (int64_t)SUM_BLOCKS, nullptr, loss);
  } else {
    hipLaunchKernelGGL(k_policy_sum, dim3(1), dim3(1024), 0, stream, a.part, parts, nullptr, loss);
  }
  return launch_status();
}

int cit_policy_loss_backward(const void* logits, int64_t ld, const void* ref, int64_t ld_ref, const uint8_t* mask,
                             int64_t ld_mask, const int64_t* offsets, int64_t total, int64_t rows, int width,
                             const int64_t* actions, const float* old_logp, const float* advantages,
                             const float* weights, float low, float high, float kl_coef, int dtype,
                             const float* upstream, int skip_one, void* grad, void* work, size_t work_bytes,
                             hipStream_t stream) {
  Policy a = {logits, ref, mask, offsets, actions, old_logp, advantages, weights, ld, ld_ref, ld_mask, rows, total,
              width, low, high, kl_coef, rows > 0 ? (float)(1.0 / (double)rows) : 0.0f, nullptr, nullptr, nullptr,
              grad, upstream, skip_one};
  if (bad(a, dtype) || !upstream || (rows && !grad)) return -1;
  const size_t need = part_bytes(rows, parts_of(rows, width, offsets != nullptr));
  if (need && (!work || work_bytes < need || ((uintptr_t)work & 15))) return -1;
  set_parts(a, work);
  return rows ? run(a, dtype, stream) : 0;
}

}  // extern "C"
