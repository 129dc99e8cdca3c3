// Rows of class scores: log probability of given labels, entropy, best alternatives (vitta_label_logprobs_*) and distillation from a
// teacher's top list (vitta_top_distill_*), forward and gradient.
//
// With x the scores of a row, T the temperature, c = log2(e) / T, m = max x, a_j = (x_j - m) c, e_j = 2^a_j, s = sum e, t = sum e a:
//   log p_j = ln2 (a_j - log2 s)        entropy = ln2 (log2 s - t / s)        lse = m / T + ln2 log2 s
// The difference x - m is taken first, so the best score's term is exactly 1 and a row of the type's lowest value stays finite.
// m starts at the lowest finite float: a row of minus infinities keeps s = 0 and is answered as a row without a distribution.
// Sums, maxima and statistics are 32 bits wide; a gradient is rounded once, to the scores' type.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.h"

namespace {

using namespace vitta;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLowest = -3.402823466e+38f;
constexpr int kThreads = 256;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __hip_bfloat16 from_float<__hip_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ _Float16 from_float<_Float16>(float v) { return (_Float16)v; }

__device__ __forceinline__ float exp2_fast(float a) { return __builtin_amdgcn_exp2f(a); }
__device__ __forceinline__ float log2_fast(float a) { return __builtin_amdgcn_logf(a); }
__device__ __forceinline__ float nan_f() { return __builtin_nanf(""); }

// (x - m) / T; halved first, for two finite scores may lie further apart than a float reaches while this does not
__device__ __forceinline__ float below(float x, float m, float inv_t) { return (0.5f * x - 0.5f * m) * (2.f * inv_t); }

// (max, sum of 2^a, sum of a 2^a); a is clamped where its power is 0 anyway, so that 0 * -inf never forms
struct Sum {
  float m, s, t;
};
__device__ __forceinline__ float clamped(float a) { return a < -200.f ? -200.f : a; }  // (NaN stays)
__device__ __forceinline__ Sum merge(Sum a, Sum b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float da = clamped((a.m - m) * c), db = clamped((b.m - m) * c);
  const float ea = exp2_fast(da), eb = exp2_fast(db);
  return Sum{m, a.s * ea + b.s * eb, ea * (a.t + a.s * da) + eb * (b.t + b.s * db)};
}
__device__ __forceinline__ Sum wave_merge(Sum v, float c) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = merge(v, Sum{__shfl_xor(v.m, d), __shfl_xor(v.s, d), __shfl_xor(v.t, d)}, c);
  return v;
}

// orders scores by value, then by lowest class; 0 is below every finite score
__device__ __forceinline__ uint64_t key_of(float x, uint32_t j) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 becomes +0)
  return ((uint64_t)(b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u)) << 32) | (uint32_t)~j;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}

struct FwdArgs {
  const void* x;
  int64_t rows, stride;
  int32_t classes;
  float c, inv_t;
  float* stats;
  // readout
  const int64_t* labels;
  int64_t ignore;
  int32_t top;
  float *logprob, *entropy, *lse, *top_logprob;
  int64_t* top_index;
  // distillation
  const int64_t* index;
  const void* value;
  int32_t value_type, list, tail;
  float *loss, *q;
};

template <typename T>
__device__ Sum row_sum(const T* x, int n, float c, Sum* red) {
  Sum v{kLowest, 0.f, 0.f};
  for (int j = threadIdx.x; j < n; j += kThreads) {
    const float f = to_float(x[j]);
    if (f > v.m) {
      const float d = clamped((v.m - f) * c), r = exp2_fast(d);
      v = Sum{f, v.s * r, r * (v.t + v.s * d)};
    }
    const float a = clamped((f - v.m) * c), e = exp2_fast(a);
    v.s += e;
    v.t += e * a;
  }
  v = wave_merge(v, c);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < kThreads / 64; ++w) v = merge(v, red[w], c);
  return v;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void readout_kernel(FwdArgs A) {
  __shared__ Sum red[kThreads / 64];
  __shared__ uint64_t best[kThreads / 64];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(A.x) + row * A.stride;
  const int n = A.classes, tid = threadIdx.x;
  const Sum v = row_sum(x, n, A.c, red);
  const float l2 = log2_fast(v.s);
  if (tid == 0) {
    if (A.stats) reinterpret_cast<float4*>(A.stats)[row] = make_float4(v.m, v.s, v.t, 0.f);
    if (A.lse) A.lse[row] = v.s == 0.f ? -INFINITY : v.m * A.inv_t + kLn2 * l2;
    if (A.entropy) A.entropy[row] = v.s == 0.f ? 0.f : kLn2 * (l2 - v.t / v.s);
    if (A.logprob) {
      const int64_t y = A.labels[row];
      float lp = nan_f();
      if (y == A.ignore) lp = 0.f;
      else if (y >= 0 && y < n) lp = v.s == 0.f ? -INFINITY : below(to_float(x[y]), v.m, A.inv_t) - kLn2 * l2;
      A.logprob[row] = lp;
    }
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < A.top; ++k) {
    uint64_t mine = 0;
    for (int j = tid; j < n; j += kThreads) {
      const float f = to_float(x[j]);
      if (f >= kLowest) {
        const uint64_t key = key_of(f, j);
        if (key < last && key > mine) mine = key;
      }
    }
    for (int d = 32; d >= 1; d >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)mine, d);
      mine = o > mine ? o : mine;
    }
    __syncthreads();
    if ((tid & 63) == 0) best[tid >> 6] = mine;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) mine = best[w] > mine ? best[w] : mine;
    last = mine;
    if (tid == 0) {
      const bool some = mine != 0 && v.s == v.s;
      A.top_index[row * A.top + k] = some ? (int64_t)(uint32_t)~(uint32_t)mine : -1;
      A.top_logprob[row * A.top + k] = v.s != v.s ? nan_f() : mine == 0 ? -INFINITY : below(value_of(mine), v.m, A.inv_t) - kLn2 * l2;
    }
  }
}

__device__ __forceinline__ float load_value(const FwdArgs& A, int64_t i) {
  if (A.value_type == VITTA_SCORES_F32) return static_cast<const float*>(A.value)[i];
  if (A.value_type == VITTA_SCORES_BF16) return to_float(static_cast<const __hip_bfloat16*>(A.value)[i]);
  return to_float(static_cast<const _Float16*>(A.value)[i]);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_kernel(FwdArgs A) {
  __shared__ Sum red[kThreads / 64];
  __shared__ int64_t idx[VITTA_SCORES_MAX_LIST];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(A.x) + row * A.stride;
  const int n = A.classes, tid = threadIdx.x, K = A.list;
  for (int k = tid; k < K; k += kThreads) {
    const int64_t i = A.index[row * K + k];
    idx[k] = i >= 0 && i < n ? i : -1;
  }
  __syncthreads();
  Sum v = row_sum(x, n, A.c, red);
  // what the classes outside the list hold: summed apart, for 1 minus the listed mass cancels
  float rest = 0.f;
  if (A.tail) {
    for (int j = tid; j < n; j += kThreads) {
      bool in = false;
      for (int k = 0; k < K; ++k) in |= idx[k] == j;
      if (!in) rest += exp2_fast((to_float(x[j]) - v.m) * A.c);
    }
    rest = wave_sum(rest);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6].s = rest;
    __syncthreads();
    rest = 0.f;
    for (int w = 0; w < kThreads / 64; ++w) rest += red[w].s;
  }
  if (tid != 0) return;
  // the teacher's list and the loss, one thread
  const float l2 = log2_fast(v.s);
  bool some = false;
  float vm = kLowest, qs = 0.f;
  for (int k = 0; k < K; ++k)
    if (idx[k] >= 0) some = true, vm = fmaxf(vm, load_value(A, row * K + k));
  const float cv = A.tail ? kLog2e : A.c;
  const float ref = A.tail ? 0.f : vm;
  for (int k = 0; k < K; ++k)
    if (idx[k] >= 0) qs += exp2_fast((load_value(A, row * K + k) - ref) * cv);
  const float ql2 = A.tail ? 0.f : log2_fast(qs), qinv = A.tail ? 1.f : 1.f / qs;
  float loss = 0.f, sum = 0.f;
  for (int k = 0; k < K; ++k) {
    float q = 0.f;
    if (idx[k] >= 0) {
      const float b = (load_value(A, row * K + k) - ref) * cv;
      q = exp2_fast(b) * qinv;
      if (q != 0.f) {
        const float log_q = A.tail ? load_value(A, row * K + k) : below(load_value(A, row * K + k), ref, A.inv_t) - kLn2 * ql2;
        loss += q * (log_q - (v.s == 0.f ? -INFINITY : below(to_float(x[idx[k]]), v.m, A.inv_t) - kLn2 * l2));
      }
    }
    sum += q;
    A.q[row * K + k] = q;
  }
  float inside = some ? sum : 0.f, outside = inside;
  if (A.tail && some) {
    const float q_rest = fmaxf(1.f - sum, 0.f);
    if (q_rest > 0.f && rest > 0.f) {
      loss += q_rest * kLn2 * (log2_fast(q_rest) - log2_fast(rest / v.s));
      inside = sum + q_rest;
      outside = inside - q_rest * v.s / rest;
    }
  }
  A.loss[row] = some ? loss : 0.f;
  reinterpret_cast<float4*>(A.stats)[row] = make_float4(v.m, v.s, inside, outside);
}

struct BwdArgs {
  const void* x;
  void* dx;
  int64_t rows, stride;
  int32_t classes;
  float c, inv_t;
  const float* stats;
  const int64_t* labels;
  int64_t ignore;
  int32_t top;
  const int64_t* top_index;
  const float *g_logprob, *g_entropy, *g_lse, *g_top;
  int64_t s_logprob, s_entropy, s_lse;
  const int64_t* index;
  int32_t list;
  const float *q, *g;
  int64_t s_g;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void readout_grad_kernel(BwdArgs A) {
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(A.x) + row * A.stride;
  T* dx = static_cast<T*>(A.dx) + row * (int64_t)A.classes;
  const float4 st = reinterpret_cast<const float4*>(A.stats)[row];
  const float m = st.x, is = st.y == 0.f ? 0.f : 1.f / st.y;
  const int64_t y = A.g_logprob ? A.labels[row] : -1;
  const bool given = A.g_logprob && y != A.ignore;
  float gl = given ? A.g_logprob[row * A.s_logprob] : 0.f;
  if (given && (y < 0 || y >= A.classes)) gl = nan_f();
  const float gh = A.g_entropy ? A.g_entropy[row * A.s_entropy] : 0.f;
  float all = -gl + (A.g_lse ? A.g_lse[row * A.s_lse] : 0.f);
  if (A.g_top)
    for (int k = 0; k < A.top; ++k)
      if (A.top_index[row * A.top + k] >= 0) all -= A.g_top[row * A.top + k];
  // dx_j = (e_j / s) / T (all - g_H ln2 (a_j - t / s)) + what the label and the alternatives add
  for (int j = threadIdx.x; j < A.classes; j += kThreads) {
    const float a = clamped((to_float(x[j]) - m) * A.c);
    float g = 0.f;
    if (all != 0.f || gh != 0.f) g = exp2_fast(a) * is * (all - gh * kLn2 * (a - st.z * is));
    if (given && j == y && st.y != 0.f) g += gl;
    if (A.g_top)
      for (int k = 0; k < A.top; ++k)
        if (A.top_index[row * A.top + k] == j) g += A.g_top[row * A.top + k];
    dx[j] = from_float<T>(g * A.inv_t);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_grad_kernel(BwdArgs A) {
  __shared__ int64_t idx[VITTA_SCORES_MAX_LIST];
  __shared__ float q[VITTA_SCORES_MAX_LIST];
  const int64_t row = blockIdx.x;
  const int K = A.list;
  for (int k = threadIdx.x; k < K; k += kThreads) {
    idx[k] = A.index[row * K + k];
    q[k] = A.q[row * K + k];
  }
  __syncthreads();
  const T* x = static_cast<const T*>(A.x) + row * A.stride;
  T* dx = static_cast<T*>(A.dx) + row * (int64_t)A.classes;
  const float4 st = reinterpret_cast<const float4*>(A.stats)[row];
  const float is = st.y == 0.f ? 0.f : 1.f / st.y, g = A.g[row * A.s_g] * A.inv_t;
  for (int j = threadIdx.x; j < A.classes; j += kThreads) {
    float pull = 0.f;
    bool in = false;
    for (int k = 0; k < K; ++k)
      if (idx[k] == j) pull += q[k], in = true;
    const float f = in ? st.z : st.w;
    const float p = f == 0.f ? 0.f : exp2_fast((to_float(x[j]) - st.x) * A.c) * is * f;
    dx[j] = from_float<T>(g * (p - pull));
  }
}

bool bad_stats(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15u); }
bool bad_out(const void* p, int32_t type) { return !p || reinterpret_cast<uintptr_t>(p) % (type == VITTA_SCORES_F32 ? 4 : 2); }

bool bad_scores(const void* x, int32_t type, int64_t rows, int32_t classes, int64_t stride, float temperature) {
  if (!x || type < VITTA_SCORES_F32 || type > VITTA_SCORES_F16 || rows <= 0 || classes <= 0 || stride < 0) return true;
  if (!(temperature > 0.f) || !(1.f / temperature > 0.f) || temperature > 3e38f) return true;
  return reinterpret_cast<uintptr_t>(x) % (type == VITTA_SCORES_F32 ? 4 : 2) != 0;
}

#define SCORES_LAUNCH(kernel, type, args)                                                                                    \
  do {                                                                                                                       \
    const dim3 grid((unsigned)(args).rows);                                                                                  \
    if ((type) == VITTA_SCORES_F32) VITTA_LAUNCH(kernel<float>, grid, dim3(kThreads), 0, st, args);                          \
    else if ((type) == VITTA_SCORES_BF16) VITTA_LAUNCH(kernel<__hip_bfloat16>, grid, dim3(kThreads), 0, st, args);           \
    else VITTA_LAUNCH(kernel<_Float16>, grid, dim3(kThreads), 0, st, args);                                                  \
  } while (0)

}  // namespace

extern "C" {

size_t vitta_scores_workspace_bytes(int64_t, int32_t, int32_t, int32_t) { return 0; }

int vitta_label_logprobs_fwd(const void* d_x, int32_t dtype, int64_t rows, int32_t classes, int64_t row_stride, float temperature,
                             const int64_t* d_labels, int64_t ignore_index, int32_t top, float* d_logprob, float* d_entropy,
                             float* d_lse, float* d_top_logprob, int64_t* d_top_index, float* d_stats, void* d_workspace,
                             size_t workspace_bytes, void* stream) {
  if (bad_scores(d_x, dtype, rows, classes, row_stride, temperature)) return VITTA_ERR_INVALID_ARG;
  if (top < 0 || top > VITTA_SCORES_MAX_TOP || top > classes || (top > 0 && (!d_top_logprob || !d_top_index))) return VITTA_ERR_INVALID_ARG;
  if (!d_labels != !d_logprob || (!d_logprob && !d_entropy && !d_lse && top == 0)) return VITTA_ERR_INVALID_ARG;
  if (d_stats && bad_stats(d_stats)) return VITTA_ERR_INVALID_ARG;
  if (rows > 0x7fffffff) return VITTA_ERR_UNSUPPORTED;
  if (workspace_bytes < vitta_scores_workspace_bytes(rows, classes, dtype, top)) return VITTA_ERR_WORKSPACE;
  (void)d_workspace;
  FwdArgs a{};
  a.x = d_x, a.rows = rows, a.stride = row_stride, a.classes = classes, a.c = kLog2e / temperature, a.inv_t = 1.f / temperature;
  a.stats = d_stats, a.labels = d_labels, a.ignore = ignore_index, a.top = top, a.logprob = d_logprob, a.entropy = d_entropy, a.lse = d_lse;
  a.top_logprob = d_top_logprob, a.top_index = d_top_index;
  hipStream_t st = static_cast<hipStream_t>(stream);
  SCORES_LAUNCH(readout_kernel, dtype, a);
  return VITTA_OK;
}

int vitta_label_logprobs_bwd(const void* d_x, int32_t dtype, int64_t rows, int32_t classes, int64_t row_stride, float temperature,
                             const int64_t* d_labels, int64_t ignore_index, int32_t top, const int64_t* d_top_index,
                             const float* d_stats, const float* d_glogprob, int64_t glogprob_stride, const float* d_gentropy,
                             int64_t gentropy_stride, const float* d_glse, int64_t glse_stride, const float* d_gtop, void* d_dx,
                             void* stream) {
  if (bad_scores(d_x, dtype, rows, classes, row_stride, temperature) || bad_stats(d_stats) || bad_out(d_dx, dtype)) return VITTA_ERR_INVALID_ARG;
  if ((d_glogprob && !d_labels) || (d_gtop && (!d_top_index || top <= 0 || top > VITTA_SCORES_MAX_TOP))) return VITTA_ERR_INVALID_ARG;
  if (rows > 0x7fffffff) return VITTA_ERR_UNSUPPORTED;
  BwdArgs a{};
  a.x = d_x, a.dx = d_dx, a.rows = rows, a.stride = row_stride, a.classes = classes, a.c = kLog2e / temperature, a.inv_t = 1.f / temperature;
  a.stats = d_stats, a.labels = d_labels, a.ignore = ignore_index, a.top = top, a.top_index = d_top_index;
  a.g_logprob = d_glogprob, a.g_entropy = d_gentropy, a.g_lse = d_glse, a.g_top = d_gtop;
  a.s_logprob = glogprob_stride, a.s_entropy = gentropy_stride, a.s_lse = glse_stride;
  hipStream_t st = static_cast<hipStream_t>(stream);
  SCORES_LAUNCH(readout_grad_kernel, dtype, a);
  return VITTA_OK;
}

int vitta_top_distill_fwd(const void* d_x, int32_t dtype, int64_t rows, int32_t classes, int64_t row_stride, float temperature,
                          const int64_t* d_index, const void* d_value, int32_t value_dtype, int32_t list, int32_t tail, float* d_loss,
                          float* d_stats, float* d_q, void* d_workspace, size_t workspace_bytes, void* stream) {
  if (bad_scores(d_x, dtype, rows, classes, row_stride, temperature)) return VITTA_ERR_INVALID_ARG;
  if (!d_index || !d_value || !d_loss || bad_stats(d_stats) || !d_q || list <= 0 || list > VITTA_SCORES_MAX_LIST) return VITTA_ERR_INVALID_ARG;
  if (value_dtype < VITTA_SCORES_F32 || value_dtype > VITTA_SCORES_F16) return VITTA_ERR_INVALID_ARG;
  if (rows > 0x7fffffff) return VITTA_ERR_UNSUPPORTED;
  if (workspace_bytes < vitta_scores_workspace_bytes(rows, classes, dtype, 0)) return VITTA_ERR_WORKSPACE;
  (void)d_workspace;
  FwdArgs a{};
  a.x = d_x, a.rows = rows, a.stride = row_stride, a.classes = classes, a.c = kLog2e / temperature, a.inv_t = 1.f / temperature;
  a.stats = d_stats, a.index = d_index, a.value = d_value, a.value_type = value_dtype, a.list = list, a.tail = tail != 0;
  a.loss = d_loss, a.q = d_q;
  hipStream_t st = static_cast<hipStream_t>(stream);
  SCORES_LAUNCH(distill_kernel, dtype, a);
  return VITTA_OK;
}

int vitta_top_distill_bwd(const void* d_x, int32_t dtype, int64_t rows, int32_t classes, int64_t row_stride, float temperature,
                          const int64_t* d_index, int32_t list, const float* d_stats, const float* d_q, const float* d_g,
                          int64_t g_stride, void* d_dx, void* stream) {
  if (bad_scores(d_x, dtype, rows, classes, row_stride, temperature)) return VITTA_ERR_INVALID_ARG;
  if (!d_index || bad_stats(d_stats) || !d_q || !d_g || bad_out(d_dx, dtype) || list <= 0 || list > VITTA_SCORES_MAX_LIST) return VITTA_ERR_INVALID_ARG;
  if (rows > 0x7fffffff) return VITTA_ERR_UNSUPPORTED;
  BwdArgs a{};
  a.x = d_x, a.dx = d_dx, a.rows = rows, a.stride = row_stride, a.classes = classes, a.c = kLog2e / temperature, a.inv_t = 1.f / temperature;
  a.stats = d_stats, a.index = d_index, a.list = list, a.q = d_q, a.g = d_g, a.s_g = g_stride;
  hipStream_t st = static_cast<hipStream_t>(stream);
  SCORES_LAUNCH(distill_grad_kernel, dtype, a);
  return VITTA_OK;
}

}  // extern "C"
