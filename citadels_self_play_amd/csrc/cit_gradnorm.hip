// The global norm of many gradients and their clipping:
//
//   n = sqrt(sum_t sum_i g_ti^2),  c = min(1, max_norm / (n + 1e-6)),  out_ti = c g_ti
//
// Bound by memory: the norm has to be whole before the first scaled value is
// written, so the gradients are read twice and written once.  Squares are
// summed in fp64 (they neither overflow nor vanish for any value of the element
// types, and 4e8 of them lose nothing); every sum has a fixed order, so the
// norm is the same from run to run.
#include "cit_ops.h"

namespace {

#define GN_LIST 96               // tensors of one launch: their list travels in the kernel's arguments (2.9 KB)
#define GN_BLOCKS 2048           // most workgroups (and partial sums) of one launch

struct GradList {
  const void* in[GN_LIST];
  void* out[GN_LIST];
  int64_t n[GN_LIST];
  int32_t first[GN_LIST + 1];    // chunks before tensor t
  uint8_t type[GN_LIST];         // element type | out type << 4
  int32_t count, chunk;          // tensors, elements of a chunk
};

__device__ __forceinline__ int tensor_of(const GradList& g, int c) {
  int lo = 0, hi = g.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (g.first[mid] <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Four loads of 16 bytes at a time: 4e8 bf16 elements in 4 launches of 45 us each, 4.4 TB/s (one load at a time: 2.8).
template <typename T>
__device__ __forceinline__ double sum_squares(const T* p, int64_t n) {
  constexpr int E = 16 / sizeof(T), U = 4;
  double s[U] = {0.0, 0.0, 0.0, 0.0};
  const int64_t whole = n / E;
  int64_t i = threadIdx.x;
  for (; i + (U - 1) * 256 < whole; i += U * 256) {
    Pack16<T> v[U];
#pragma unroll
    for (int u = 0; u < U; u++) v[u].raw = load16(p + (i + u * 256) * E);
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < E; j++) {
        const double d = (double)to_f(v[u].e[j]);
        s[u] = fma(d, d, s[u]);
      }
  }
  for (; i < whole; i += 256) {
    Pack16<T> v;
    v.raw = load16(p + i * E);
#pragma unroll
    for (int j = 0; j < E; j++) {
      const double d = (double)to_f(v.e[j]);
      s[0] = fma(d, d, s[0]);
    }
  }
  for (i = whole * E + threadIdx.x; i < n; i += 256) {
    const double d = (double)to_f(p[i]);
    s[1] = fma(d, d, s[1]);
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ __launch_bounds__(256) void k_sum_squares(GradList g, double* part) {
  __shared__ double sums[4];
  double s = 0.0;
  const int chunks = g.first[g.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(g, c);
    const int64_t at = (int64_t)(c - g.first[t]) * g.chunk;
    const int64_t n = g.n[t] - at < g.chunk ? g.n[t] - at : g.chunk;
    const int type = g.type[t] & 15;
    if (type == CIT_FP32) s += sum_squares(static_cast<const float*>(g.in[t]) + at, n);
    else if (type == CIT_BF16) s += sum_squares(static_cast<const bf16_t*>(g.in[t]) + at, n);
    else s += sum_squares(static_cast<const fp16_t*>(g.in[t]) + at, n);
  }
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// The norm and the factor from the partial sums, the same in every workgroup that asks (THREADS threads, all of them).
template <int THREADS>
__device__ __forceinline__ double norm_of(const double* part, int count, double (&sums)[THREADS / 64]) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += THREADS) s += part[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0.0;
  for (int i = 0; i < THREADS / 64; i++) s += sums[i];
  return sqrt(s);
}
__device__ __forceinline__ float factor_of(double n, double max_norm) {
  const double c = max_norm / (n + 1e-6);
  return c >= 1.0 ? 1.0f : (float)c;                                   // a NaN norm makes NaN gradients, inf / inf too
}

// work: [0] the factor (fp32), [2] on the partial sums.
__global__ __launch_bounds__(1024) void k_norm(const double* part, int count, double max_norm, float* norm,
                                               float* factor) {
  __shared__ double sums[16];
  const double n = norm_of<1024>(part, count, sums);
  if (threadIdx.x) return;
  *norm = (float)n;
  *factor = factor_of(n, max_norm);
}

// A lane writes 16 neighbouring bytes and reads what they are made of, four times over: 4e8 bf16 elements to fp32 in
// 4 launches of 121 us each, 5.0 TB/s, what a copy reaches (16 bytes read and 32 written a lane: 3.4).  Scaling the
// last tensors first, for what the cache before memory still holds of them, changed nothing.
template <typename T, typename O>
__device__ __forceinline__ void scale(const T* p, O* o, int64_t n, float c) {
  constexpr int W = 16 / sizeof(O), U = 4;
  struct __attribute__((packed, aligned(2))) In { T e[W]; };
  const int64_t whole = n / W;
  auto write = [&](int64_t i, const In& v) {
    Pack16<O> r;
#pragma unroll
    for (int j = 0; j < W; j++) r.e[j] = from_f<O>(to_f((T)v.e[j]) * c);
    store16(o + i * W, r.raw);
  };
  int64_t i = threadIdx.x;
  for (; i + (U - 1) * 256 < whole; i += U * 256) {
    In v[U];
#pragma unroll
    for (int u = 0; u < U; u++) v[u] = *reinterpret_cast<const In*>(p + (i + u * 256) * W);
#pragma unroll
    for (int u = 0; u < U; u++) write(i + u * 256, v[u]);
  }
  for (; i < whole; i += 256) write(i, *reinterpret_cast<const In*>(p + i * W));
  for (i = whole * W + threadIdx.x; i < n; i += 256) o[i] = from_f<O>(to_f(p[i]) * c);
}

// `parts` > 0: every workgroup works the norm out of that many partial sums itself, which saves a launch.
__global__ __launch_bounds__(256) void k_scale(GradList g, const float* factor, const double* part, int parts,
                                               double max_norm, float* norm) {
  __shared__ double sums[4];
  float f;
  if (parts) {
    const double n = norm_of<256>(part, parts, sums);
    f = factor_of(n, max_norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  } else {
    f = *factor;
  }
  const int chunks = g.first[g.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(g, c);
    if (g.in[t] == g.out[t] && f == 1.0f) continue;                    // in place, not clipped: as they are
    const int64_t at = (int64_t)(c - g.first[t]) * g.chunk;
    const int64_t n = g.n[t] - at < g.chunk ? g.n[t] - at : g.chunk;
    const int in = g.type[t] & 15, out = g.type[t] >> 4;
    const void* p = g.in[t];
    void* o = g.out[t];
    if (in == CIT_FP32) scale((const float*)p + at, (float*)o + at, n, f);
    else if (in == CIT_BF16 && out == CIT_BF16) scale((const bf16_t*)p + at, (bf16_t*)o + at, n, f);
    else if (in == CIT_BF16) scale((const bf16_t*)p + at, (float*)o + at, n, f);
    else if (out == CIT_FP16) scale((const fp16_t*)p + at, (fp16_t*)o + at, n, f);
    else scale((const fp16_t*)p + at, (float*)o + at, n, f);
  }
}

}  // namespace

extern "C" {

size_t cit_clip_grad_norm_work_bytes(int tensors) {
  return tensors < 0 ? 0 : ((size_t)(tensors + GN_LIST - 1) / GN_LIST * GN_BLOCKS + 2) * sizeof(double);
}

int cit_clip_grad_norm(const void* const* grads, void* const* out, const int64_t* sizes, const int32_t* types,
                       const int32_t* out_types, int tensors, double max_norm, float* norm, void* work,
                       size_t work_bytes, hipStream_t stream) {
  if (tensors < 0 || !norm || !work || work_bytes < cit_clip_grad_norm_work_bytes(tensors)) return -1;
  if ((uintptr_t)work & 15) return -1;
  if (tensors && (!grads || !sizes || !types || (out && !out_types))) return -1;
  if (out && !(max_norm >= 0.0)) return -1;
  int64_t total = 0;
  int count = 0;
  for (int t = 0; t < tensors; t++) {
    if (sizes[t] < 0 || sizes[t] > (int64_t)1 << 48 || (sizes[t] && !grads[t])) return -1;
    if (types[t] < CIT_FP32 || types[t] > CIT_FP16) return -1;
    if (out && ((sizes[t] && !out[t]) || (out_types[t] != types[t] && out_types[t] != CIT_FP32))) return -1;
    total += sizes[t];
    count += sizes[t] > 0;
  }
  // lists of equal length: none left with a few; of at least one, also where no tensor holds anything
  const int lists_needed = (count + GN_LIST - 1) / GN_LIST;
  const int each = count ? (count + lists_needed - 1) / lists_needed : 1;
  // about 8 GN_BLOCKS chunks in all, so that each launch of a long list has enough workgroups
  int64_t chunk = (total / (8 * GN_BLOCKS) + 2047) / 2048 * 2048;
  if (chunk < 2048) chunk = 2048;
  if (chunk > (int64_t)1 << 30) chunk = (int64_t)1 << 30;
  float* factor = static_cast<float*>(work);
  double* part = static_cast<double*>(work) + 2;
  int parts = 0, lists = 0;
  bool own_norm = false;                             // the scaling workgroups take the norm from the partial sums
  for (int pass = 0; pass < (out ? 2 : 1); pass++) {
    for (int t = 0; t < tensors;) {
      GradList g;
      g.count = 0, g.chunk = (int32_t)chunk;
      int64_t chunks = 0;
      for (; t < tensors && g.count < each; t++) {
        if (!sizes[t]) continue;
        const int64_t more = (sizes[t] + chunk - 1) / chunk;
        if (chunks + more > INT32_MAX / 2) return -1;
        const int i = g.count++;
        g.in[i] = grads[t], g.out[i] = out ? out[t] : nullptr, g.n[i] = sizes[t];
        g.first[i] = (int32_t)chunks;
        g.type[i] = (uint8_t)(types[t] | (out ? out_types[t] << 4 : 0));
        chunks += more;
      }
      if (!g.count) continue;
      g.first[g.count] = (int32_t)chunks;
      const int blocks = chunks < GN_BLOCKS ? (int)chunks : GN_BLOCKS;
      if (pass == 0) {
        hipLaunchKernelGGL(k_sum_squares, dim3(blocks), dim3(256), 0, stream, g, part + parts);
        parts += blocks;
        lists++;
      } else {
        hipLaunchKernelGGL(k_scale, dim3(blocks), dim3(256), 0, stream, g, factor, part, own_norm ? parts : 0, max_norm,
                           norm);
      }
    }
    if (pass == 0) {
      own_norm = out && lists == 1 && parts <= 1024;
      if (!own_norm)
        hipLaunchKernelGGL(k_norm, dim3(1), dim3(1024), 0, stream, part, parts, out ? max_norm : INFINITY, norm,
                           factor);
    }
  }
  return launch_status();
}

}  // extern "C"
