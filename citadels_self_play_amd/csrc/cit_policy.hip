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
// keep their digits (sum p d cancels to nothing there).  A row of weight 0 is
// not read; a row that leaves no entry counts nothing, and the gradients of
// both are 0.  An action outside its row makes the row NaN.
#include "cit_ops.h"

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
    r.bad = s < 0 || e < s || e > a.total || e - s > INT32_MAX;
    r.at = r.at_ref = r.at_mask = r.at_grad = r.bad ? 0 : s;
    r.len = r.bad ? 0 : (int)(e - s);
  } else {
    r.at = i * a.ld, r.at_ref = i * a.ld_ref, r.at_mask = i * a.ld_mask, r.at_grad = i * a.width;
    r.len = a.width;
  }
  return r;
}

// p (d + exp(-d) - 1) for p > 0: the series where the three cancel.
__device__ __forceinline__ float kl_term(float p, float q, float d) {
  if (!(p > 0.0f)) return q;
  float s = 1.0f / 40320.0f;
  s = fmaf(s, -d, 1.0f / 5040.0f);
  s = fmaf(s, -d, 1.0f / 720.0f);
  s = fmaf(s, -d, 1.0f / 120.0f);
  s = fmaf(s, -d, 1.0f / 24.0f);
  s = fmaf(s, -d, 1.0f / 6.0f);
  s = fmaf(s, -d, 0.5f);
  return fabsf(d) < 0.5f ? p * (d * d * s) : fmaf(p, d, q - p);
}

struct Lse {                     // running maximum and sum of exp(x - maximum)
  float m = -INFINITY, s = 0.0f;
  __device__ __forceinline__ void add(float x) {
    if (x == -INFINITY) return;                      // nothing, also before the first entry
    if (x > m) {
      s = fmaf(s, expf(m - x), 1.0f);
      m = x;
    } else {
      s += m == INFINITY ? NAN : expf(x - m);        // a NaN comes through here too
    }
  }
  __device__ __forceinline__ void join(float m2, float s2) {
    const float t = fmaxf(m, m2);
    const float a = m == t ? 1.0f : expf(m - t), b = m2 == t ? 1.0f : expf(m2 - t);
    s = t == -INFINITY ? s + s2 : fmaf(s, a, s2 * b);
    m = t;
  }
};

template <int G>
__device__ __forceinline__ void join_lanes(Lse& v) {
#pragma unroll
  for (int d = G / 2; d; d >>= 1) {
    const float m = __shfl_xor(v.m, d, 64), s = __shfl_xor(v.s, d, 64);
    v.join(m, s);
  }
}
template <int G>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int d = G / 2; d; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

// What a row's statistics say about the loss: from lse, the action's logit and kl.
struct Verdict {
  float logp, kl, dlogp, loss;
};

__device__ __forceinline__ Verdict judge(const Policy& a, int64_t i, float logp, float kl) {
  Verdict v;
  v.logp = logp, v.kl = kl;
  const float adv = a.adv[i], ratio = expf(logp - a.old[i]);
  const float free = ratio * adv;
  const float clipped = ratio < 1.0f - a.low ? 1.0f - a.low : ratio > 1.0f + a.high ? 1.0f + a.high : ratio;
  const float held = clipped * adv;
  v.dlogp = free <= held ? -free : held < free ? 0.0f : NAN;
  v.loss = (free <= held || free != free ? -free : -held) + (a.ref ? a.beta * kl : 0.0f);
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

__device__ __forceinline__ float grad_of(const Policy& a, float p, float d, const Verdict& v, bool chosen, float w) {
  float t = a.ref && a.beta != 0.0f ? a.beta * (d - v.kl) - v.dlogp : -v.dlogp;
  t = p > 0.0f ? p * t : p * 0.0f;                   // an entry of no probability has no gradient of its own
  return w * (chosen ? t + v.dlogp : t);
}

// A row by G lanes, entry by entry (short rows).
template <typename T, int G>
__global__ __launch_bounds__(256) void k_policy_rows(Policy a, int row_blocks) {
  __shared__ double sums[256 / G];
  const float up = a.upstream ? *a.upstream : 1.0f;
  if (a.upstream && a.skip_one && up == 1.0f) return;
  T* grad = static_cast<T*>(a.grad);
  if ((int)blockIdx.x >= row_blocks) {               // entries in front of the first row and behind the last: no gradient
    const int64_t n = a.total;
    int64_t first = a.offsets[0], last = a.offsets[a.rows];
    first = first < 0 ? 0 : first > n ? n : first;
    last = last < first ? first : last > n ? n : last;
    const int64_t at = (int64_t)((int)blockIdx.x - row_blocks) * 256 + threadIdx.x;
    const int64_t step = (int64_t)((int)gridDim.x - row_blocks) * 256;
    for (int64_t j = at; j < first; j += step) grad[j] = from_f<T>(0.0f);
    for (int64_t j = last + at; j < n; j += step) grad[j] = from_f<T>(0.0f);
    return;
  }
  const int lane = threadIdx.x % G;
  const int64_t i = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  double counted = 0.0;
  if (i < a.rows) {
    const Row r = row_of(a, i);
    const float w = weight_of(a, i);
    const T* l = static_cast<const T*>(a.logits) + r.at;
    const T* q = a.ref ? static_cast<const T*>(a.ref) + r.at_ref : nullptr;
    const uint8_t* ok = a.mask ? a.mask + r.at_mask : nullptr;
    Verdict v = {0.0f, 0.0f, 0.0f, 0.0f};
    float lse = 0.0f, lse_q = 0.0f;
    bool live = w != 0.0f && !r.bad;
    if (live) {
      Lse x, y;
      for (int j = lane; j < r.len; j += G) {
        if (ok && !ok[j]) continue;
        x.add(to_f(l[j]));
        if (q) y.add(to_f(q[j]));
      }
      join_lanes<G>(x);
      join_lanes<G>(y);
      live = !(x.s == 0.0f);
      if (live) {
        lse = x.m + logf(x.s), lse_q = y.m + logf(y.s);
        float kl = 0.0f;
        if (q) {
          for (int j = lane; j < r.len; j += G) {
            if (ok && !ok[j]) continue;
            const float lp = to_f(l[j]) - lse, lq = to_f(q[j]) - lse_q;
            kl += kl_term(expf(lp), expf(lq), lp - lq);
          }
          kl = sum_lanes<G>(kl);
        }
        v = judge(a, i, action_logit<T>(a, r, i) - lse, kl);
      }
    }
    if (r.bad && w != 0.0f) v = {NAN, NAN, NAN, NAN};
    if (!a.upstream && lane == 0) {
      a.logp[i] = v.logp, a.kl[i] = v.kl;
      counted = w != 0.0f ? (double)w * (double)v.loss : 0.0;
    }
    if (grad) {
      const int64_t act = a.actions[i];
      T* g = grad + r.at_grad;
      for (int j = lane; j < r.len; j += G) {
        float t = 0.0f;
        if (live && !(ok && !ok[j])) {
          const float lp = to_f(l[j]) - lse;
          t = grad_of(a, expf(lp), q ? lp - (to_f(q[j]) - lse_q) : 0.0f, v, j == act, up * w);
        }
        g[j] = from_f<T>(t);
      }
    }
  }
  if (a.upstream) return;
  if (lane == 0) sums[threadIdx.x / G] = counted;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int k = 0; k < 256 / G; k++) s += sums[k];
    a.part[blockIdx.x] = s;
  }
}

__global__ __launch_bounds__(1024) void k_policy_sum(const double* part, int64_t count, float* loss) {
  __shared__ double sums[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += 1024) s += part[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = 0.0;
  for (int i = 0; i < 16; i++) s += sums[i];
  *loss = (float)s;
}

int64_t row_blocks(int64_t rows) { return (rows + 3) / 4; }            // 64 lanes a row, 4 rows a workgroup

template <typename T>
int launch(const Policy& a, hipStream_t stream) {
  const int64_t blocks = row_blocks(a.rows);
  const int tail = a.grad && a.offsets ? 64 : 0;
  hipLaunchKernelGGL((k_policy_rows<T, 64>), dim3((unsigned)(blocks + tail)), dim3(256), 0, stream, a, (int)blocks);
  return launch_status();
}

int run(const Policy& a, int dtype, hipStream_t stream) {
  if (dtype == CIT_FP32) return launch<float>(a, stream);
  if (dtype == CIT_BF16) return launch<bf16_t>(a, stream);
  return launch<fp16_t>(a, stream);
}

bool bad(const Policy& a, int dtype) {
  if (dtype < CIT_FP32 || dtype > CIT_FP16 || a.rows < 0 || row_blocks(a.rows) > INT32_MAX / 2) return true;
  if (!(a.low >= 0.0f) || !(a.high >= 0.0f) || !(a.beta >= 0.0f)) return true;
  if (!a.rows) return false;
  if (!a.actions || !a.old || !a.adv) return true;
  if (a.offsets) return a.total < 0 || (a.total && !a.logits);
  if (a.width < 0 || (a.width && !a.logits)) return true;
  return a.ld < a.width || (a.ref && a.ld_ref < a.width) || (a.mask && a.ld_mask < a.width);
}

}  // namespace

extern "C" {

size_t cit_policy_loss_work_bytes(int64_t rows) { return rows > 0 ? (size_t)row_blocks(rows) * sizeof(double) : 0; }

int cit_policy_loss(const void* logits, int64_t ld, const void* ref, int64_t ld_ref, const uint8_t* mask,
                    int64_t ld_mask, const int64_t* offsets, int64_t total, int64_t rows, int width,
                    const int64_t* actions, const float* old_logp, const float* advantages, const float* weights,
                    float low, float high, float kl_coef, int dtype, float* loss, float* logp, float* kl, void* grad,
                    void* work, size_t work_bytes, hipStream_t stream) {
  Policy a = {logits, ref, mask, offsets, actions, old_logp, advantages, weights, ld, ld_ref, ld_mask, rows, total,
              width, low, high, kl_coef, rows > 0 ? (float)(1.0 / (double)rows) : 0.0f, logp, kl,
              static_cast<double*>(work), grad, nullptr, 0};
  if (bad(a, dtype) || !loss || (rows && (!logp || !kl))) return -1;
  const size_t need = cit_policy_loss_work_bytes(rows);
  if (need && (!work || work_bytes < need)) return -1;
  if (rows) {
    const int rc = run(a, dtype, stream);
    if (rc) return rc;
  }
  hipLaunchKernelGGL(k_policy_sum, dim3(1), dim3(1024), 0, stream, a.part, rows ? row_blocks(rows) : 0, loss);
  return launch_status();
}

int cit_policy_loss_backward(const void* logits, int64_t ld, const void* ref, int64_t ld_ref, const uint8_t* mask,
                             int64_t ld_mask, const int64_t* offsets, int64_t total, int64_t rows, int width,
                             const int64_t* actions, const float* old_logp, const float* advantages,
                             const float* weights, float low, float high, float kl_coef, int dtype,
                             const float* upstream, int skip_one, void* grad, hipStream_t stream) {
  Policy a = {logits, ref, mask, offsets, actions, old_logp, advantages, weights, ld, ld_ref, ld_mask, rows, total,
              width, low, high, kl_coef, rows > 0 ? (float)(1.0 / (double)rows) : 0.0f, nullptr, nullptr, nullptr,
              grad, upstream, skip_one};
  if (bad(a, dtype) || !upstream || (rows && !grad)) return -1;
  return rows ? run(a, dtype, stream) : 0;
}

}  // extern "C"
