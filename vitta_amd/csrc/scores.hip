// Rows of class scores: log probability of given labels, entropy, best alternatives (vitta_label_logprobs_*) and distillation from a
// teacher's top list (vitta_top_distill_*), forward and gradient.
//
// With x the scores of a row, T the temperature, c = log2(e) / T, m = max x, a_j = (x_j - m) c, e_j = 2^a_j, s = sum e, t = sum e a:
//   log p_j = (x_j - m) / T - ln2 log2 s        entropy = ln2 (log2 s - t / s)        lse = m / T + ln2 log2 s
// The difference x - m is taken first, so the best score's term is exactly 1 and a row of the type's lowest value stays finite.
// m starts at the lowest finite float: a row of minus infinities keeps s = 0 and is answered as a row without a distribution.
// Sums, maxima and statistics are 32 bits wide, what a teacher's list leaves of 1 is summed in 64; a gradient is rounded once, to the scores' type.
//
// Forward: one pass, bound by memory (4096 x 131072 bfloat16: 170 us = 6.3 TB/s with label and entropy, 200 us with 64 alternatives, where the
// candidates' instructions add up; 2048 x 32003 float16 with 5: 36 us).  A lane holds four 16-byte loads while the next four are on
// their way, takes their maximum, moves its running sums to it and adds; the lanes' (m, s, t) are joined at the end.  A short row belongs to
// one wave, a longer one to a workgroup (wave_rows), and few long rows are cut into segments (fwd_cut) that the last one of a row joins.
// Best alternatives in the same pass: a lower bound of the k-th best (from the lanes' maxima of the first loads, raised later) lets all but a
// few scores pass by; these few wait with their classes in LDS, and at the end 64 at a time are sorted across the lanes of a wave and merged
// into its list of 64.  Equal scores order by class, so the answer does not depend on which wave saw what.  (Sorting as they come,
// or keeping only their classes and reading the scores again, took 330 and 297 us of the first case.)
// Gradient: elementwise from the row statistics, e_j (A + B a_j), bound by memory (4096 x 131072 bfloat16: 356 us = 6.0 TB/s); the few classes
// that a label or a list adds to are written again at the end by the workgroup that wrote them.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.h"

namespace {

using namespace vitta;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLowest = -3.402823466e+38f;
constexpr int kU = 4;              // 16-byte loads of a lane that are consumed together
// Waves of a workgroup that share a long row: eight, four where it collects alternatives (2048 x 32003 float16: 27.0 us with eight and 29.5 with four
// without alternatives, 40.3 and 36.5 with five of them; 4096 x 131072 bfloat16 with 64 of them 223 and 203).
constexpr int waves_of(bool top) { return top ? 4 : 8; }
constexpr int kWaveRow = 4096;     // classes up to which a row may belong to one wave, in the forward
constexpr int kWaveGrad = 2048;    // and does, in the gradient
constexpr int kWorkgroups = 512;   // workgroups that few long rows are cut into (1024: 400 x 131072 27 -> 25 us, 64 x 131072 with alternatives 15 -> 17)
constexpr int kKeys = 256;         // candidates that a wave keeps: 2 KiB of LDS
constexpr int kMaxSegments = 64;
constexpr int kTailSegment = 1 << 18;  // classes whose membership bits fit 32 KiB

// ---- element types -------------------------------------------------------------------------------------------------------------
template <typename T> struct Pack;
template <> struct Pack<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint4 empty() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static __device__ __forceinline__ void open(const uint4& w, float* f) {
    f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 close(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <> struct Pack<__hip_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint4 empty() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  static __device__ __forceinline__ void open(const uint4& w, float* f) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(u[i] << 16), f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, bf2));
  }
  static __device__ __forceinline__ uint4 close(const float* f) { return make_uint4(two(f[0], f[1]), two(f[2], f[3]), two(f[4], f[5]), two(f[6], f[7])); }
};
template <> struct Pack<_Float16> {
  static constexpr int N = 8;
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ uint4 empty() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  static __device__ __forceinline__ void open(const uint4& w, float* f) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const h2 h = __builtin_bit_cast(h2, u[i]);
      f[2 * i] = (float)h[0], f[2 * i + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ uint32_t two(float a, float b) { return __builtin_bit_cast(uint32_t, (h2){(_Float16)a, (_Float16)b}); }
  static __device__ __forceinline__ uint4 close(const float* f) { return make_uint4(two(f[0], f[1]), two(f[2], f[3]), two(f[4], f[5]), two(f[6], f[7])); }
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __hip_bfloat16 from_float<__hip_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ _Float16 from_float<_Float16>(float v) { return (_Float16)v; }

// Streamed loads: a score is used once.  Reading 1 GiB of scores 5.7 -> 6.2 TB/s, and a gradient that reads them again loses nothing (1024 x 50021
// floats forward and backward 127 -> 118 us).
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const u4 v = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ void store_once(uint4* p, uint4 w) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store((u4){w.x, w.y, w.z, w.w}, reinterpret_cast<u4*>(p));
}

__device__ __forceinline__ float exp2_fast(float a) { return __builtin_amdgcn_exp2f(a); }
__device__ __forceinline__ float log2_fast(float a) { return __builtin_amdgcn_logf(a); }
__device__ __forceinline__ float nan_f() { return __builtin_nanf(""); }
// (x - m) / T; halved first, for two finite scores may lie further apart than a float reaches while this does not
__device__ __forceinline__ float below(float x, float m, float inv_t) { return (0.5f * x - 0.5f * m) * (2.f * inv_t); }

// ---- lanes ------------------------------------------------------------------------------------------------------------------------------
// the value of lane ^ D: within a row of 16 by DPP, across rows by the swaps (a shuffle through LDS costs several times as much)
template <int CTRL, int BANKS> __device__ __forceinline__ int dpp(int old, int v) { return __builtin_amdgcn_update_dpp(old, v, CTRL, 0xf, BANKS, false); }
template <int D> __device__ __forceinline__ uint32_t lane_xor(uint32_t x, int lane) {
  const int v = (int)x;
  if (D == 1) return dpp<0xb1, 0xf>(v, v);                     // quad_perm 1 0 3 2
  if (D == 2) return dpp<0x4e, 0xf>(v, v);                     // quad_perm 2 3 0 1
  if (D == 4) return dpp<0x114, 0xa>(dpp<0x104, 0x5>(v, v), v);  // row_shl:4 into the even quads, row_shr:4 into the odd ones
  if (D == 8) return dpp<0x128, 0xf>(v, v);                    // row_ror:8
  if (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (lane & 16) ? r[0] : r[1];
  }
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return (lane & 32) ? r[0] : r[1];
}
template <int D> __device__ __forceinline__ uint64_t lane_xor(uint64_t v, int lane) {
  return ((uint64_t)lane_xor<D>((uint32_t)(v >> 32), lane) << 32) | lane_xor<D>((uint32_t)v, lane);
}

template <class Op> __device__ __forceinline__ float wave_all(float v, int lane, Op op) {
  v = op(v, __uint_as_float(lane_xor<1>(__float_as_uint(v), lane)));
  v = op(v, __uint_as_float(lane_xor<2>(__float_as_uint(v), lane)));
  v = op(v, __uint_as_float(lane_xor<4>(__float_as_uint(v), lane)));
  v = op(v, __uint_as_float(lane_xor<8>(__float_as_uint(v), lane)));
  v = op(v, __uint_as_float(lane_xor<16>(__float_as_uint(v), lane)));
  return op(v, __uint_as_float(lane_xor<32>(__float_as_uint(v), lane)));
}
__device__ __forceinline__ float all_max(float v, int lane) { return wave_all(v, lane, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float all_sum(float v, int lane) { return wave_all(v, lane, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ double all_sum(double v, int lane) {
  v += __longlong_as_double((long long)lane_xor<1>((uint64_t)__double_as_longlong(v), lane));
  v += __longlong_as_double((long long)lane_xor<2>((uint64_t)__double_as_longlong(v), lane));
  v += __longlong_as_double((long long)lane_xor<4>((uint64_t)__double_as_longlong(v), lane));
  v += __longlong_as_double((long long)lane_xor<8>((uint64_t)__double_as_longlong(v), lane));
  v += __longlong_as_double((long long)lane_xor<16>((uint64_t)__double_as_longlong(v), lane));
  return v + __longlong_as_double((long long)lane_xor<32>((uint64_t)__double_as_longlong(v), lane));
}

// ---- running sums ----------------------------------------------------------------------------------------------------------------
// (max, sum of 2^a, sum of a 2^a); a is clamped where its power is 0 anyway, so that 0 * -inf never forms (a NaN reaches s unclamped)
struct Sum {
  float m, s, t;
};
__device__ __forceinline__ float clamped(float a) { return fmaxf(a, -200.f); }
__device__ __forceinline__ Sum moved(Sum v, float m, float c) {
  const float d = clamped((v.m - m) * c), r = exp2_fast(d);
  return Sum{m, v.s * r, r * (v.t + v.s * d)};
}
__device__ __forceinline__ Sum wave_merge(Sum v, float c, int lane) {
  v = moved(v, all_max(v.m, lane), c);
  return Sum{v.m, all_sum(v.s, lane), all_sum(v.t, lane)};
}

// ---- best alternatives -------------------------------------------------------------------------------------------------------------
// orders scores by value, then by lowest class; 0 is below every finite score
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t key_of(float x, uint32_t j) { return ((uint64_t)ordered(x + 0.f) << 32) | (uint32_t)~j; }  // (-0 becomes +0)
__device__ __forceinline__ float value_of(uint64_t key) { return unordered((uint32_t)(key >> 32)); }

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
  __builtin_amdgcn_wave_barrier();
}

// a lower bound, good to 16 bits, of the r-th largest of the lanes' M values: bit by bit, by counting
template <int M> __device__ __forceinline__ float rth_largest(const float* v, int r) {
  uint32_t o[M], t = 0;
#pragma unroll
  for (int i = 0; i < M; ++i) o[i] = ordered(v[i]);
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const uint32_t u = t | (1u << b);
    int n = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) n += __popcll(__ballot(o[i] >= u));
    if (n >= r) t = u;
  }
  return t <= ordered(kLowest) ? kLowest : unordered(t);
}

// one exchange of a bitonic network: the lane keeps the larger key where its bit D equals its bit K (K = 64: none has it), or the smaller
template <int D, int K, bool RISING> __device__ __forceinline__ uint64_t exchange(uint64_t v, int lane) {
  const uint64_t o = lane_xor<D>(v, lane);
  const bool larger = (((lane & D) == 0) == ((lane & K) == 0)) != RISING;
  return (o > v) == larger ? o : v;
}
template <int K, bool RISING> __device__ __forceinline__ uint64_t exchanges(uint64_t v, int lane) {
  if (K >= 64) v = exchange<32, K, RISING>(v, lane);
  if (K >= 32) v = exchange<16, K, RISING>(v, lane);
  if (K >= 16) v = exchange<8, K, RISING>(v, lane);
  if (K >= 8) v = exchange<4, K, RISING>(v, lane);
  if (K >= 4) v = exchange<2, K, RISING>(v, lane);
  return exchange<1, K, RISING>(v, lane);
}
// n <= 64 keys in the first lanes (0 behind them), sorted; falling with n <= 32 leaves out the stages that only move zeros
template <bool RISING> __device__ __forceinline__ uint64_t sort64(uint64_t v, int n, int lane) {
  v = exchanges<2, RISING>(v, lane);
  v = exchanges<4, RISING>(v, lane);
  v = exchanges<8, RISING>(v, lane);
  v = exchanges<16, RISING>(v, lane);
  if (RISING || n > 16) v = exchanges<32, RISING>(v, lane);
  if (RISING || n > 32) v = exchanges<64, RISING>(v, lane);
  return v;
}
// the 64 best of a falling and a rising list, falling
__device__ __forceinline__ uint64_t merge64(uint64_t falling, uint64_t rising, int lane) {
  return exchanges<64, false>(falling > rising ? falling : rising, lane);
}

// a wave's list: lane i holds the i-th best key seen (0: none)
struct Best {
  uint64_t mine;
  bool some;

  __device__ __forceinline__ void take(uint64_t key, int n, int lane) {  // n <= 64 keys in the first lanes, 0 behind them
    mine = some ? merge64(mine, sort64<true>(key, n, lane), lane) : sort64<false>(key, n, lane);
    some = true;
  }

  // every score of a row that the wave's lanes have, for rows of which the bound lets too many pass (scores that rise along the row, many
  // equal ones, or a row too short to give each of its four waves a bound: 512 x 1200 bfloat16 with 5 alternatives 8.8 us, 512 x 1024 4.4,
  // 512 x 2048 5.2): those from the list's k-th on wait in `buf` and are taken by 64.  all(e, &f): the lane's e-th class, and its score
  template <class All> __device__ void take_all(int n, int k, uint64_t* buf, All all, int lane) {
    int waiting = 0;
    float bound = kLowest;
    for (int e = 0; e <= n; ++e) {
      if (e < n) {
        float f;
        const uint32_t j = all(e, f);
        const bool in = f >= bound;  // (false for NaN and -inf: the bound is finite)
        const uint64_t who = __ballot(in);
        if (who == 0) continue;
        if (in) buf[waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = key_of(f, j);
        waiting += __popcll(who);
        wave_fence();
      }
      while (waiting >= 64 || (e == n && waiting > 0)) {
        const int m = min(waiting, 64);
        waiting -= m;
        take(lane < m ? buf[waiting + lane] : 0, m, lane);
        const uint32_t o = __builtin_amdgcn_readlane((uint32_t)(mine >> 32), k - 1);
        if (o) bound = fmaxf(bound, unordered(o));
        wave_fence();
      }
    }
  }
};

// ---- arguments ---------------------------------------------------------------------------------------------------------------------
struct FwdArgs {
  const void* x;
  int64_t rows, stride, outer, row0;  // row0: the launch's first row
  uint32_t inner;                     // rows at `stride` from one another, groups of them at `outer`
  int32_t classes, segments, per_segment;
  float c, inv_t;
  float* stats;
  float4* part;       // [rows][segments] (m, s, t) of a segment
  uint64_t* keys;     // [rows][segments][top]
  uint32_t* tickets;  // [rows] segments that are done, 0 at rest; NULL: a launch of its own joins them
  // readout
  const int64_t* labels;
  int64_t ignore;
  int32_t top;
  float *logprob, *entropy, *lse, *top_logprob;
  int64_t* top_index;
  // distillation
  const int64_t* index;
  const void* value;
  int32_t value_type, list;
  float *loss, *q;
};

template <typename T, class Args> __device__ __forceinline__ const T* row_of(const Args& A, int64_t row) {
  const int64_t group = A.inner < A.rows ? (uint32_t)row / A.inner : 0;  // (rows < 2^31)
  return static_cast<const T*>(A.x) + group * A.outer + (row - group * A.inner) * A.stride;
}

enum Mode { kReadout, kDistill, kDistillTail };

__device__ __forceinline__ float load_value(const FwdArgs& A, int64_t i) {
  if (A.value_type == VITTA_SCORES_F32) return static_cast<const float*>(A.value)[i];
  if (A.value_type == VITTA_SCORES_BF16) return to_float(static_cast<const __hip_bfloat16*>(A.value)[i]);
  return to_float(static_cast<const _Float16*>(A.value)[i]);
}

// ---- a row's answer, by one wave -----------------------------------------------------------------------------------------------------
template <typename T>
__device__ void finish_readout(const FwdArgs& A, int64_t row, const T* x, Sum v, uint64_t mine, int lane) {
  const float l2 = log2_fast(v.s);
  if (lane == 0) {
    if (A.stats) reinterpret_cast<float4*>(A.stats)[row] = make_float4(v.m, v.s, v.t, 0.f);
    if (A.lse) A.lse[row] = v.s == 0.f ? -INFINITY : v.m * A.inv_t + kLn2 * l2;
    if (A.entropy) A.entropy[row] = v.s == 0.f ? 0.f : kLn2 * (l2 - v.t / v.s);
    if (A.logprob) {
      const int64_t y = A.labels[row];
      float lp = nan_f();
      if (y == A.ignore) lp = 0.f;
      else if (y >= 0 && y < A.classes) lp = v.s == 0.f ? -INFINITY : below(to_float(x[y]), v.m, A.inv_t) - kLn2 * l2;
      A.logprob[row] = lp;
    }
  }
  if (lane < A.top) {
    const bool whole = v.s == v.s;
    A.top_index[row * A.top + lane] = mine != 0 && whole ? (int64_t)(uint32_t)~(uint32_t)mine : -1;
    A.top_logprob[row * A.top + lane] = !whole ? nan_f() : mine == 0 ? -INFINITY : below(value_of(mine), v.m, A.inv_t) - kLn2 * l2;
  }
}

// Bit i: entry i * 64 + lane of a list names a class that stands earlier in it already (-1: no class).  Entries meet in kSlots words of LDS by a
// multiplicative hash (Knuth, The Art of Computer Programming 3, 6.4); of a slot the lowest (class, entry) stays, its class is done, and the
// others meet again: one to four rounds for random classes.  (2048 x 32003 bfloat16 with lists of 32: 25.7 us forward, 24.9 without looking for repeats, 30 by every
// entry against every other.)
constexpr int kList = VITTA_SCORES_MAX_LIST / 64;
constexpr int kSlots = 1024;
static_assert(VITTA_SCORES_MAX_LIST <= 256 && kMaxSegments * kTailSegment <= 1 << 24, "a class and an entry share a word");
__device__ __forceinline__ uint32_t repeats_of(const int32_t (&at)[kList], uint32_t* slots, int lane) {
  uint32_t open = 0, again = 0;
#pragma unroll
  for (int i = 0; i < kList; ++i) open |= at[i] >= 0 ? 1u << i : 0u;
  auto slot = [&](int i) { return slots + ((uint32_t)at[i] * 2654435769u >> 22); };
  auto key = [&](int i) { return (uint32_t)at[i] << 8 | (uint32_t)(i * 64 + lane); };
  while (__ballot(open != 0) != 0) {
#pragma unroll
    for (int i = 0; i < kList; ++i)
      if (open >> i & 1) *slot(i) = ~0u;
    wave_fence();
#pragma unroll
    for (int i = 0; i < kList; ++i)
      if (open >> i & 1) atomicMin(slot(i), key(i));
    wave_fence();
#pragma unroll
    for (int i = 0; i < kList; ++i)
      if (open >> i & 1) {
        const uint32_t least = *slot(i);
        if (least >> 8 == (uint32_t)at[i]) open &= ~(1u << i), again |= least != key(i) ? 1u << i : 0u;
      }
    wave_fence();
  }
  return again;
}

// v: the row's sums, without the listed classes where these are one side of a tail
template <typename T, bool TAIL>
__device__ void finish_distill(const FwdArgs& A, int64_t row, const T* x, Sum v, uint32_t* slots, int lane) {
  constexpr int R = kList;
  const int K = A.list;
  int32_t at[R];
  float val[R], z[R];
  bool some = false;
  float vm = kLowest;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int k = i * 64 + lane;
    at[i] = -1;
    if (k < K) {
      const int64_t j = A.index[row * K + k];
      if (j >= 0 && j < A.classes) at[i] = (int32_t)j;
    }
    val[i] = at[i] >= 0 ? load_value(A, row * K + k) : -INFINITY;
    z[i] = at[i] >= 0 ? to_float(x[at[i]]) : -INFINITY;
    some |= at[i] >= 0;
    vm = fmaxf(vm, val[i]);
  }
  some = __ballot(some) != 0;
  const uint32_t again = repeats_of(at, slots, lane);
  float m = v.m, s = v.s, rest = 0.f;
  if (TAIL) {  // the listed classes' own sum, each once
#pragma unroll
    for (int i = 0; i < R; ++i) m = fmaxf(m, z[i]);
    m = all_max(m, lane);
    float in = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (at[i] >= 0 && !(again >> i & 1)) in += exp2_fast((z[i] - m) * A.c);
    rest = v.s * exp2_fast((v.m - m) * A.c);
    s = rest + all_sum(in, lane);
  }
  const float l2 = log2_fast(s);
  const float ref = TAIL ? 0.f : all_max(vm, lane);
  float q[R], sum = 0.f, q_rest = 0.f;
  if (TAIL) {  // in 64 bits, once a row: 32 bits of 1 - sum are all lost where a confident teacher leaves 1e-7
    double in = 0.;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      q[i] = 0.f;
      if (i * 64 >= K) continue;
      const double each = at[i] >= 0 ? exp((double)val[i]) : 0.;
      q[i] = (float)each;
      in += each;
    }
    in = all_sum(in, lane);
    sum = (float)in;
    q_rest = (float)fmax(1. - in, 0.);
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      q[i] = at[i] >= 0 ? exp2_fast((val[i] - ref) * A.c) : 0.f;
      sum += q[i];
    }
    sum = all_sum(sum, lane);
  }
  const float inv = TAIL ? 1.f : 1.f / sum, ql = TAIL ? 0.f : kLn2 * log2_fast(sum);
  float log_q[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    q[i] *= at[i] >= 0 ? inv : 0.f;
    log_q[i] = TAIL ? val[i] : below(val[i], ref, A.inv_t) - ql;
  }
  bool repeats = false;
#pragma unroll
  for (int i = 0; i < R; ++i) repeats |= at[i] >= 0 && (again >> i & 1);
  if (__ballot(repeats) != 0) {  // a class listed more than once is one class with the sum of its probabilities
    float all[R] = {};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int n = min(64, K - i * 64);
      for (int l = 0; l < n; ++l) {
        const int32_t j = __builtin_amdgcn_readlane(at[i], l);
        const float more = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(q[i]), l));
#pragma unroll
        for (int o = 0; o < R; ++o) all[o] += at[o] == j ? more : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool low = all[i] < 1e-30f;  // (the logarithm takes a subnormal number for 0)
      if (all[i] != q[i]) log_q[i] = kLn2 * (log2_fast(low ? all[i] * 0x1p64f : all[i]) - (low ? 64.f : 0.f));
    }
  }
  float loss = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int k = i * 64 + lane;
    if (at[i] >= 0 && q[i] != 0.f) loss += q[i] * (log_q[i] - (s == 0.f ? -INFINITY : below(z[i], m, A.inv_t) - kLn2 * l2));
    if (k < K) A.q[row * K + k] = q[i];
  }
  loss = all_sum(loss, lane);
  if (lane != 0) return;
  // The gradient is e_j a - q_j: (m, a) of the listed classes, and of the others, whose e_j is taken against their own maximum: their share of
  // the rest, q_rest e_j / sum e, then holds however little the student gives them.
  const bool lost = s != s || (TAIL ? sum != sum : !(sum > 0.f));  // no distribution on one of the sides: NaN throughout
  const float share = s == 0.f ? 0.f : (TAIL ? sum : 1.f) / s;
  float4 st = make_float4(m, share, m, share);
  if (TAIL) {
    const bool both = q_rest > 0.f && v.s > 0.f;  // (of a NaN neither is true)
    if (both) loss += q_rest * (kLn2 * (log2_fast(q_rest) + l2 - log2_fast(v.s)) - below(v.m, m, A.inv_t));
    const float all = both ? 1.f : sum;
    st.y = s == 0.f ? 0.f : all / s;
    st.z = v.m;
    st.w = v.s == 0.f ? 0.f : all * (rest / s) / v.s - (both ? q_rest / v.s : 0.f);
  }
  if (lost) loss = st.y = st.w = nan_f();
  A.loss[row] = some ? loss : 0.f;
  reinterpret_cast<float4*>(A.stats)[row] = some ? st : make_float4(m, 0.f, m, 0.f);
}

// ---- the segments of a row ----------------------------------------------------------------------------------------------------------------
// Their sums and lists pass through memory past the XCDs' caches: stored and loaded at device scope.
template <typename V> __device__ __forceinline__ void put(V* p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename V> __device__ __forceinline__ V get(const V* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// NW waves merge the lists (64 keys at a time, four loads ahead), the first one the sums
template <typename T, int MODE, bool TOP, int NW>
__device__ void join_segments(const FwdArgs& A, int64_t row, uint64_t* lists, uint32_t* slots, int lane, int wave) {
  const T* x = row_of<T>(A, row);
  Best best{0, false};
  if (TOP) {
    const int all = A.segments * A.top;
    const uint64_t* keys = A.keys + row * all;
    for (int at = wave * 64; at < all; at += 4 * NW * 64) {
      uint64_t key[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) key[i] = at + i * NW * 64 + lane < all ? get(keys + at + i * NW * 64 + lane) : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + i * NW * 64 < all) best.take(key[i], min(all - at - i * NW * 64, 64), lane);
    }
    lists[wave * 64 + lane] = best.mine;
    __syncthreads();
  }
  if (wave != 0) return;
  if (TOP)
    for (int w = 1; w < NW && w * 64 < A.segments * A.top; ++w) best.mine = merge64(best.mine, lists[w * 64 + 63 - lane], lane);
  Sum v{kLowest, 0.f, 0.f};
  if (lane < A.segments) {
    const float* p = reinterpret_cast<const float*>(A.part + row * A.segments + lane);
    v = Sum{get(p), get(p + 1), get(p + 2)};
  }
  v = wave_merge(v, A.c, lane);
  if (MODE == kReadout) finish_readout<T>(A, row, x, v, best.mine, lane);
  else finish_distill<T, MODE == kDistillTail>(A, row, x, v, slots, lane);
}

// ---- forward ---------------------------------------------------------------------------------------------------------------------------
// NW waves share a (segment of a) row; with NW == 1 the four waves of a workgroup take four rows.
template <typename T, int NW, int MODE, bool ENT, bool TOP>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64, 4) void scores_kernel(FwdArgs A) {
  constexpr int N = Pack<T>::N, NT = NW * 64, G = NW == 1 ? 4 : 1;  // G groups in a workgroup
  extern __shared__ __attribute__((aligned(16))) uint32_t bits_all[];  // kDistillTail: one bit per class of the group's segment
  __shared__ uint64_t keys_all[TOP ? (NW == 1 ? G : NW) * kKeys : 1];  // the waves' candidates, later their lists
  __shared__ uint32_t slots_all[MODE == kReadout ? 1 : G * kSlots];
  __shared__ int counts[NW], last_all;
  __shared__ Sum red[NW];
  __shared__ float bounds[NW];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = NW == 1 ? lane : threadIdx.x;
  int64_t row;
  int seg = 0;
  if (NW == 1) {
    row = A.row0 + (int64_t)blockIdx.x * G + wave;
    if (row >= A.rows) return;  // (no workgroup barrier in this form)
  } else if (A.segments == 1) {
    row = A.row0 + blockIdx.x;
  } else {
    const uint32_t at = blockIdx.x / (uint32_t)A.segments;
    row = A.row0 + at;
    seg = (int)(blockIdx.x - at * (uint32_t)A.segments);
  }
  const T* whole = row_of<T>(A, row);
  const int j0 = seg * A.per_segment, n = min(A.per_segment, A.classes - j0);
  const T* x = whole + j0;
  const int head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
  const int nv = (n - head) / N, body = head + nv * N;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);

  // the vectors at + u * NT of this lane (those from nv on are empty)
  auto load = [&](uint4* w, int at) {
#pragma unroll
    for (int u = 0; u < kU; ++u) w[u] = at + u * NT < nv ? load_once(xv + at + u * NT) : Pack<T>::empty();
  };
  uint4 now[kU], next[kU];
  load(now, tid);

  uint32_t* bits = bits_all;
  if (MODE == kDistillTail) {  // class j0 + i at bit i - head + 16: a vector's bits never straddle a byte
    const int words = (A.per_segment + 16 + 31) / 32 + 1;
    bits += (NW == 1 ? wave : 0) * words;
    for (int i = tid; i < words; i += NT) bits[i] = 0;
    if (NW > 1) __syncthreads(); else wave_fence();
    for (int k = tid; k < A.list; k += NT) {
      const int64_t j = A.index[row * A.list + k];
      if (j < j0 || j >= j0 + (int64_t)n) continue;
      const uint32_t bit = (uint32_t)(j - j0) - head + 16;
      atomicOr(&bits[bit >> 5], 1u << (bit & 31));
    }
    if (NW > 1) __syncthreads(); else wave_fence();
  }

  Sum v{kLowest, 0.f, 0.f};
  const float c = A.c;
  float bound = kLowest;  // a lower bound of the row's top-th score
  uint64_t* keys = keys_all + (TOP ? wave * kKeys : 0);
  int waiting = 0;        // candidates found; beyond kKeys: not all of them are kept
  auto offer = [&](float f, int j) {
    const bool in = f >= bound;  // (never for NaN and -inf: the bound is finite)
    const uint64_t who = __ballot(in);
    if (who == 0) return;
    const int many = __popcll(who);
    if (in && waiting + many <= kKeys)
      keys[waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = key_of(f, (uint32_t)(j0 + j));
    waiting += many;
  };

  const int steps = max(1, (nv + kU * NT - 1) / (kU * NT));
  auto consume = [&](const uint4* w, int base, int step) {
    float f[kU][N], cu[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      cu[u] = -INFINITY;
      if (base + u * NT >= nv) continue;  // (the same for the whole group)
      Pack<T>::open(w[u], f[u]);
      if (MODE == kDistillTail) {
        const int at = base + u * NT + tid;
        uint32_t in = 0;
        if (at < nv) in = reinterpret_cast<const uint8_t*>(bits)[2 + (N == 8 ? at : at >> 1)];
        if (N == 4) in = (at & 1) ? in >> 4 : in & 15;
        if (in) {
#pragma unroll
          for (int i = 0; i < N; ++i) f[u][i] = in >> i & 1 ? -INFINITY : f[u][i];
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) cu[u] = fmaxf(cu[u], f[u][i]);
    }
    float cm = cu[0];
#pragma unroll
    for (int u = 1; u < kU; ++u) cm = fmaxf(cm, cu[u]);
    const float m = fmaxf(v.m, cm);
    if (ENT) {
      v = moved(v, m, c);
    } else {
      v.s *= exp2_fast((v.m - m) * c);
      v.m = m;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (base + u * NT >= nv) continue;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float a = (f[u][i] - m) * c, e = exp2_fast(a);
        v.s += e;
        if (ENT) v.t = fmaf(e, clamped(a), v.t);
      }
    }
    if (TOP) {
      // Each of the waves has r of its lanes' maxima at or above what it gives into `bounds`, so NW r >= top scores of the row lie at or
      // above the least of these.  After the first step all wait for it; later, on steps 1, 2, 4, ..., the waves take what stands there.
      const int r = (A.top + NW - 1) / NW;
      if (step == 0) {
        bound = r <= 32 ? rth_largest<1>(&cm, r) : rth_largest<kU>(cu, r);
        if (NW > 1) {
          if (lane == 0) bounds[wave] = bound;
          __syncthreads();
        }
      }
      if (NW > 1) {
        float least = __hip_atomic_load(&bounds[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
#pragma unroll
        for (int o = 1; o < NW; ++o) least = fminf(least, __hip_atomic_load(&bounds[o], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
        bound = least;
      }
      // Where most lanes pass (masked classes came first, or scores rise along the row) the wave's own top-th maximum of this step is a bound too.
      if (step > 0 && __popcll(__ballot(cm >= bound)) > 48) bound = fmaxf(bound, rth_largest<kU>(cu, A.top));
      if (__ballot(cm >= bound) != 0) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          if (base + u * NT >= nv || __ballot(cu[u] >= bound) == 0) continue;
#pragma unroll
          for (int i = 0; i < N; ++i) offer(f[u][i], head + (base + u * NT + tid) * N + i);
        }
      }
      if (NW > 1 && step > 0 && (step & (step - 1)) == 0 && step + 1 < steps) {
        const float mine = rth_largest<1>(&v.m, r);
        if (lane == 0) __hip_atomic_store(&bounds[wave], mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
    }
  };

  for (int step = 0; step < steps; ++step) {
    const int base = step * kU * NT;
    if (step + 1 < steps) load(next, base + kU * NT + tid);
    consume(now, base, step);
#pragma unroll
    for (int u = 0; u < kU; ++u) now[u] = next[u];
  }
  // what lies before the first and behind the last whole vector: at most 2 (N - 1) <= 14 elements, one a lane
  if (NW == 1 || wave == 0) {
    const int rest = n - nv * N, i = lane < head ? lane : body + lane - head;
    if (rest > 0) {
      float f = lane < rest ? to_float(x[i]) : -INFINITY;
      if (TOP) offer(f, i);
      if (MODE == kDistillTail && lane < rest && (bits[(i - head + 16) >> 5] >> ((i - head + 16) & 31) & 1)) f = -INFINITY;
      v = moved(v, fmaxf(v.m, f), c);
      const float a = (f - v.m) * c, e = exp2_fast(a);
      v.s += e;
      v.t = fmaf(e, clamped(a), v.t);
    }
  }
  v = wave_merge(v, c, lane);
  Best best{0, false};
  if (NW > 1) {
    if (lane == 0) red[wave] = v, counts[wave] = waiting;
    __syncthreads();
  } else {
    wave_fence();
  }
  if (TOP) {
    int most = waiting, before = 0, all = waiting;
    if (NW > 1) {
      all = most = 0;
#pragma unroll
      for (int o = 0; o < NW; ++o) most = max(most, counts[o]), all += counts[o];
    }
    if (most > kKeys) {
      best.take_all((n + NT - 1) / NT, A.top, keys, [&](int e, float& f) {
        const int j = e * NT + tid;
        f = j < n ? to_float(x[j]) : -INFINITY;
        return (uint32_t)(j0 + j);
      }, lane);
    } else if (NW > 1 && all <= 64) {  // one sort for all of them
      uint64_t key = 0;
#pragma unroll
      for (int o = 0; o < NW; ++o) {
        if (lane >= before && lane < before + counts[o]) key = keys_all[o * kKeys + lane - before];
        before += counts[o];
      }
      if (wave == 0) best.take(key, all, lane);
    } else {
      for (int at = 0; at < waiting; at += 64) best.take(at + lane < waiting ? keys[at + lane] : 0, min(waiting - at, 64), lane);
    }
    if (NW > 1 && (all > 64 || most > kKeys)) {  // the waves' lists, pair by pair
      keys[lane] = best.mine;
      __syncthreads();
#pragma unroll
      for (int d = 1; d < NW; d <<= 1) {
        if ((wave & (2 * d - 1)) == 0) {
          best.mine = merge64(best.mine, keys[d * kKeys + 63 - lane], lane);
          keys[lane] = best.mine;
        }
        __syncthreads();
      }
    }
  }
  if (NW > 1) {
    if (wave != 0 && !(TOP && A.segments > 1)) return;
    if (wave == 0) {
      v = lane < NW ? red[lane] : Sum{kLowest, 0.f, 0.f};
      v = wave_merge(v, c, lane);
    }
    if (A.segments > 1) {
      int last = 0;
      if (wave == 0) {
        const int64_t at = row * A.segments + seg;
        float* p = reinterpret_cast<float*>(A.part + at);
        if (lane == 0) put(p, v.m), put(p + 1, v.s), put(p + 2, v.t);
        if (TOP && lane < A.top) put(A.keys + at * A.top + lane, best.mine);
        if (A.tickets) {  // who comes last joins the row: what it reads was in memory before the others took their tickets
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          if (lane == 0) {
            last = __hip_atomic_fetch_add(A.tickets + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)A.segments - 1;
            if (last) put(A.tickets + row, 0u);
          }
          last = __builtin_amdgcn_readfirstlane(last);
          asm volatile("" ::: "memory");
        }
        if (TOP && lane == 0) last_all = last;
      }
      if (TOP) {
        __syncthreads();
        last = last_all;
      }
      if (last) join_segments<T, MODE, TOP, TOP ? NW : 1>(A, row, keys_all, slots_all, lane, wave);
      return;
    }
  }
  if (MODE == kReadout) finish_readout<T>(A, row, whole, v, best.mine, lane);
  else finish_distill<T, MODE == kDistillTail>(A, row, whole, v, slots_all + (NW == 1 && MODE != kReadout ? wave * kSlots : 0), lane);
}

// a launch of its own for the joins
template <typename T, int MODE, bool TOP>
__global__ __launch_bounds__(256) void scores_join_kernel(FwdArgs A) {
  __shared__ uint64_t lists[TOP ? 4 * 64 : 1];
  __shared__ uint32_t slots[MODE == kReadout ? 1 : kSlots];
  join_segments<T, MODE, TOP, 4>(A, A.row0 + blockIdx.x, lists, slots, threadIdx.x & 63, threadIdx.x >> 6);
}

// ---- gradient --------------------------------------------------------------------------------------------------------------------------
struct BwdArgs {
  const void* x;
  void* dx;
  int64_t rows, stride, outer, row0;
  uint32_t inner;
  int32_t classes, segments, per_segment;
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
  int32_t stream_out;
};

// dx_j = e_j (a0 + a1 a_j), with a0 = at0 for the classes of the group's list, to which it adds `add`.
// A workgroup takes what its threads hold in kU loads each (32 KiB with what it writes), a wave a row of up to kWaveGrad classes.
template <typename T, int NT, bool DISTILL, bool ENT>
__global__ __launch_bounds__(256) void scores_grad_kernel(BwdArgs A) {
  constexpr int N = Pack<T>::N, G = 256 / NT, L = DISTILL ? VITTA_SCORES_MAX_LIST : VITTA_SCORES_MAX_TOP + 1;
  __shared__ int32_t at_all[G * L];
  __shared__ float add_all[G * L];
  __shared__ int many_all[G];
  const int group = threadIdx.x / NT, tid = threadIdx.x - group * NT, lane = threadIdx.x & 63;
  int32_t* at = at_all + group * L;
  float* add = add_all + group * L;
  const uint32_t unit = G > 1 ? blockIdx.x * G + group : blockIdx.x / (uint32_t)A.segments;  // (a row by a wave has one segment)
  const int64_t row = A.row0 + unit;
  if (row >= A.rows) return;  // (G > 1 only: a wave for itself)
  const int seg = G > 1 ? 0 : (int)(blockIdx.x - unit * (uint32_t)A.segments);
  const int j0 = seg * A.per_segment, n = min(A.per_segment, A.classes - j0);
  const T* x = row_of<T>(A, row) + j0;
  T* dx = static_cast<T*>(A.dx) + row * (int64_t)A.classes + j0;
  const int head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
  const int nv = (n - head) / N, body = head + nv * N;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);

  uint4 w[kU];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < kU; ++u) w[u] = i + u * NT < nv ? load_once(xv + i + u * NT) : Pack<T>::empty();
  };
  load(tid);

  const float4 st = reinterpret_cast<const float4*>(A.stats)[row];
  const float m = DISTILL ? st.z : st.x, is = st.y == 0.f ? 0.f : 1.f / st.y, c = A.c;  // (distillation: see finish_distill)
  float a0, a1 = 0.f, at0;
  int many = 0;  // the listed classes that lie here, in the list's order: the group's first wave collects them
  auto collect = [&](int64_t j, float value, bool valid) {
    const bool in = valid && j >= j0 && j < j0 + (int64_t)n;
    const uint64_t who = __ballot(in);
    if (in) {
      const int i = many + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
      at[i] = (int32_t)(j - j0);
      add[i] = value;
    }
    many += __popcll(who);
  };
  if (DISTILL) {
    const float g = A.g[row * A.s_g] * A.inv_t;
    if (tid < 64) {
      for (int k = lane; k - lane < A.list; k += 64) {
        const bool valid = k < A.list;
        collect(valid ? A.index[row * A.list + k] : 0, valid && g != 0.f ? -g * A.q[row * A.list + k] : 0.f, valid);
      }
    }
    at0 = g == 0.f ? 0.f : g * st.y;
    a0 = g == 0.f ? 0.f : g * st.w;
  } else {
    const int64_t y = A.g_logprob ? A.labels[row] : A.ignore;
    float gl = y != A.ignore ? A.g_logprob[row * A.s_logprob] : 0.f;
    if (y != A.ignore && (y < 0 || y >= A.classes) && gl != 0.f) gl = nan_f();
    const float gh = ENT ? A.g_entropy[row * A.s_entropy] : 0.f, gs = A.g_lse ? A.g_lse[row * A.s_lse] : 0.f;
    float all = gs - gl;
    bool used = gl != 0.f || gs != 0.f || gh != 0.f;
    if (tid < 64) collect(y, st.y == 0.f ? 0.f : gl * A.inv_t, y != A.ignore && lane == 0);
    if (A.g_top) {  // (every wave the whole list, of at most 64: all of them need its sum)
      const bool valid = lane < A.top;
      const int64_t j = valid ? A.top_index[row * A.top + lane] : -1;
      const float g = valid ? A.g_top[row * A.top + lane] : 0.f;
      if (tid < 64) collect(j, g * A.inv_t, j >= 0);
      all -= all_sum(j >= 0 ? g : 0.f, lane);
      used |= __ballot(g != 0.f) != 0;
    }
    a0 = is * A.inv_t * (all + (ENT ? gh * kLn2 * st.z * is : 0.f));
    a1 = ENT ? -is * A.inv_t * gh * kLn2 : 0.f;
    if (!used) a0 = a1 = 0.f;  // (zeros whatever the row holds; a row of NaN that is used gets NaN, also where the gradients cancel)
    at0 = a0;
  }
  if (tid == 0) many_all[group] = many;
  const bool dead = a0 == 0.f && a1 == 0.f;  // zeros whatever the row holds
  auto grad = [&](float f, float m, float b) {
    const float a = (f - m) * c, e = exp2_fast(a);
    return e * (ENT ? fmaf(a1, clamped(a), b) : b);
  };

  const bool straight = (reinterpret_cast<uintptr_t>(dx + head) & 15) == 0;
  for (int i0 = tid;;) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = i0 + u * NT;
      if (i < nv) {
        float f[N];
        Pack<T>::open(w[u], f);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = dead ? 0.f : grad(f[e], m, a0);
        const uint4 o = Pack<T>::close(f);
        if (straight && A.stream_out) store_once(reinterpret_cast<uint4*>(dx + head) + i, o);
        else if (straight) reinterpret_cast<uint4*>(dx + head)[i] = o;
        else __builtin_memcpy(__builtin_assume_aligned(dx + head + (int64_t)i * N, sizeof(T)), &o, 16);
      }
    }
    i0 += kU * NT;
    if (i0 - tid >= nv) break;
    load(i0);
  }
  if (tid < n - nv * N) {
    const int i = tid < head ? tid : body + tid - head;
    dx[i] = from_float<T>(dead ? 0.f : grad(to_float(x[i]), m, a0));
  }
  // the listed classes again, each with all that is added to it
  if (NT > 64) __syncthreads(); else wave_fence();
  many = many_all[group];
  for (int k = tid; k < many; k += NT) {
    const int j = at[k];
    float sum = 0.f;
    for (int o = 0; o < many; ++o) sum += at[o] == j ? add[o] : 0.f;
    dx[j] = from_float<T>((at0 == 0.f && a1 == 0.f ? 0.f : grad(to_float(x[j]), st.x, at0)) + sum);
  }
}

// ---- launches ----------------------------------------------------------------------------------------------------------------------------
bool bad_stats(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15u); }
bool bad_out(const void* p, int32_t type) { return !p || reinterpret_cast<uintptr_t>(p) % (type == VITTA_SCORES_F32 ? 4 : 2); }

bool bad_scores(const void* x, int32_t type, int64_t rows, int32_t classes, int64_t stride, int64_t inner, int64_t outer, float temperature) {
  if (!x || type < VITTA_SCORES_F32 || type > VITTA_SCORES_F16 || rows <= 0 || classes <= 0 || stride < 0 || inner <= 0 || outer < 0) return true;
  // 1 / T and c stay finite, and where a difference of finite scores overflows its term is 0 beyond doubt
  if (!(temperature >= 1e-30f && temperature <= 1e30f)) return true;
  return reinterpret_cast<uintptr_t>(x) % (type == VITTA_SCORES_F32 ? 4 : 2) != 0;
}

struct Cut {
  int32_t segments, per_segment;
};
Cut cut_into(int32_t classes, int64_t segments) {
  int64_t per = (classes + segments - 1) / segments;
  per = (per + 511) / 512 * 512;  // (whole 16-byte vectors: a segment starts as the row is aligned)
  return Cut{(int32_t)((classes + per - 1) / per), (int32_t)per};
}
// Whether a row of the forward belongs to one wave.  Up to 1024 classes it always does, up to kWaveRow where there are rows for every wave or no
// alternatives to sort, which four waves do in a quarter of the time (512 x 4000 bfloat16 with 20 alternatives: 10.6 us by waves, 6.7 by
// workgroups; 8192 x 4000: 27.0 and 30.1; without alternatives 512 x 4000: 4.9 and 4.7, 8192 x 4000: 16.7 and 24.3).
bool wave_rows(int64_t rows, int32_t classes, bool top) { return classes <= 1024 || (classes <= kWaveRow && (!top || rows >= 2048)); }
// Segments of a row in the forward: enough workgroups for the chip, none with less than one step of its threads.
Cut fwd_cut(int64_t rows, int32_t classes, int32_t type, bool top) {
  if (wave_rows(rows, classes, top)) return Cut{1, classes};
  int64_t s = (kWorkgroups + rows - 1) / rows;
  const int32_t floor = top || type == VITTA_SCORES_F32 ? 8192 : 16384;
  s = s < classes / floor ? s : classes / floor;
  s = s > kMaxSegments ? kMaxSegments : s;
  const int64_t least = ((int64_t)classes + kTailSegment - 1) / kTailSegment;  // (membership bits)
  s = s < least ? least : s;
  return s <= 1 ? Cut{1, classes} : cut_into(classes, s);
}
// A row of the gradient of up to 2048 classes belongs to one wave (512 x 4000 bfloat16: 6.0 us by waves, 4.6 by workgroups; 512 x 2000: 4.9 and
// 4.8), a workgroup takes one load of its 256 threads, 16 KiB of a row (2 x 32 KiB: 4096 x 131072 bfloat16 360 -> 381 us).
Cut bwd_cut(int32_t classes, int32_t type) {
  const int32_t per = 256 * kU * (type == VITTA_SCORES_F32 ? 4 : 8);
  return classes <= kWaveGrad || classes <= per ? Cut{1, classes} : Cut{(int32_t)(((int64_t)classes + per - 1) / per), per};
}
// Rows of one launch: its threads stay below 2^31 (a grid of 2^32 and more is refused); a multiple of 4, the rows of a workgroup by waves.
int64_t launch_rows(int32_t segments, int threads) {
  const int64_t n = (int64_t)0x7fffffff / ((int64_t)segments * threads) & ~(int64_t)3;
  return n < 4 ? 4 : n;
}

// rows that no 64 segments of kTailSegment classes hold
bool too_large(int64_t rows, int32_t classes) { return classes > kMaxSegments * kTailSegment || rows > 0x7fffffff; }

template <typename T, int MODE, bool ENT, bool TOP>
int launch_fwd(FwdArgs a, void* ws, uint32_t* tickets, hipStream_t st) {
  const Cut cut = fwd_cut(a.rows, a.classes, Pack<T>::N == 4 ? VITTA_SCORES_F32 : VITTA_SCORES_BF16, TOP);
  a.segments = cut.segments, a.per_segment = cut.per_segment;
  const size_t bits = MODE == kDistillTail ? ((size_t)(cut.per_segment + 16 + 31) / 32 + 1) * 4 : 0;
  constexpr int NW = waves_of(TOP);
  const bool waves = wave_rows(a.rows, a.classes, TOP);
  if (cut.segments > 1) {
    a.part = static_cast<float4*>(ws);
    a.keys = reinterpret_cast<uint64_t*>(a.part + a.rows * cut.segments);
    a.tickets = tickets;
  }
  const int64_t most = launch_rows(cut.segments, waves ? 64 : NW * 64);
  for (a.row0 = 0; a.row0 < a.rows; a.row0 += most) {
    const int64_t rows = a.rows - a.row0 < most ? a.rows - a.row0 : most;
    if (waves) {
      VITTA_LAUNCH((scores_kernel<T, 1, MODE, ENT, TOP>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 4 * bits, st, a);
      continue;
    }
    VITTA_LAUNCH((scores_kernel<T, NW, MODE, ENT, TOP>), dim3((unsigned)(rows * cut.segments)), dim3(NW * 64), bits, st, a);
    if (cut.segments > 1 && !tickets) VITTA_LAUNCH((scores_join_kernel<T, MODE, TOP>), dim3((unsigned)rows), dim3(256), 0, st, a);
  }
  return VITTA_OK;
}

template <int MODE, bool ENT, bool TOP>
int launch_fwd(int32_t type, const FwdArgs& a, void* ws, uint32_t* tickets, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (type == VITTA_SCORES_F32) return launch_fwd<float, MODE, ENT, TOP>(a, ws, tickets, st);
  if (type == VITTA_SCORES_BF16) return launch_fwd<__hip_bfloat16, MODE, ENT, TOP>(a, ws, tickets, st);
  return launch_fwd<_Float16, MODE, ENT, TOP>(a, ws, tickets, st);
}

template <typename T, bool DISTILL, bool ENT>
int launch_bwd(BwdArgs a, hipStream_t st) {
  const Cut cut = bwd_cut(a.classes, Pack<T>::N == 4 ? VITTA_SCORES_F32 : VITTA_SCORES_BF16);
  a.segments = cut.segments, a.per_segment = cut.per_segment;
  // A gradient of 512 MiB and more is streamed past the 256 MiB cache (2048 x 131072 bfloat16 188 -> 180 us); a smaller one stays in it, for the
  // store itself and for who reads it next (1024 x 131072 87 -> 91 us, 1024 x 50021 floats 58 -> 75 if it were streamed).
  a.stream_out = a.rows * a.classes * (int64_t)sizeof(T) >= (512ll << 20);
  const bool waves = a.classes <= kWaveGrad;
  const int64_t most = launch_rows(cut.segments, waves ? 64 : 256);
  for (a.row0 = 0; a.row0 < a.rows; a.row0 += most) {
    const int64_t rows = a.rows - a.row0 < most ? a.rows - a.row0 : most;
    if (waves) VITTA_LAUNCH((scores_grad_kernel<T, 64, DISTILL, ENT>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
    else VITTA_LAUNCH((scores_grad_kernel<T, 256, DISTILL, ENT>), dim3((unsigned)(rows * cut.segments)), dim3(256), 0, st, a);
  }
  return VITTA_OK;
}

template <bool DISTILL, bool ENT>
int launch_bwd(int32_t type, const BwdArgs& a, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (type == VITTA_SCORES_F32) return launch_bwd<float, DISTILL, ENT>(a, st);
  if (type == VITTA_SCORES_BF16) return launch_bwd<__hip_bfloat16, DISTILL, ENT>(a, st);
  return launch_bwd<_Float16, DISTILL, ENT>(a, st);
}

}  // namespace

extern "C" {

size_t vitta_scores_workspace_bytes(int64_t rows, int32_t classes, int32_t dtype, int32_t top) {
  if (rows <= 0 || classes <= 0 || top < 0 || top > VITTA_SCORES_MAX_TOP || too_large(rows, classes)) return 0;
  const int64_t s = fwd_cut(rows, classes, dtype, top > 0).segments;
  return s == 1 ? 0 : (size_t)rows * s * (16 + 8 * (size_t)top);
}

int vitta_label_logprobs_fwd(const void* d_x, int32_t dtype, int64_t rows, int32_t classes, int64_t row_stride, int64_t inner_rows,
                             int64_t outer_stride, float temperature,
                             const int64_t* d_labels, int64_t ignore_index, int32_t top, float* d_logprob, float* d_entropy,
                             float* d_lse, float* d_top_logprob, int64_t* d_top_index, float* d_stats, void* d_workspace,
                             size_t workspace_bytes, uint32_t* d_tickets, void* stream) {
  if (bad_scores(d_x, dtype, rows, classes, row_stride, inner_rows, outer_stride, temperature)) return VITTA_ERR_INVALID_ARG;
  if (top < 0 || top > VITTA_SCORES_MAX_TOP || top > classes || (top > 0 && (!d_top_logprob || !d_top_index))) return VITTA_ERR_INVALID_ARG;
  if (!d_labels != !d_logprob || (!d_logprob && !d_entropy && !d_lse && top == 0)) return VITTA_ERR_INVALID_ARG;
  if (d_stats && bad_stats(d_stats)) return VITTA_ERR_INVALID_ARG;
  if (too_large(rows, classes)) return VITTA_ERR_UNSUPPORTED;
  const size_t need = vitta_scores_workspace_bytes(rows, classes, dtype, top);
  if (workspace_bytes < need || (need && bad_stats(d_workspace))) return VITTA_ERR_WORKSPACE;
  FwdArgs a{};
  a.x = d_x, a.rows = rows, a.stride = row_stride, a.outer = outer_stride, a.classes = classes, a.c = kLog2e / temperature, a.inv_t = 1.f / temperature;
  a.inner = (uint32_t)(inner_rows < rows ? inner_rows : rows);
  a.stats = d_stats, a.labels = d_labels, a.ignore = ignore_index, a.top = top, a.logprob = d_logprob, a.entropy = d_entropy, a.lse = d_lse;
  a.top_logprob = d_top_logprob, a.top_index = d_top_index;
  if (d_entropy) return top ? launch_fwd<kReadout, true, true>(dtype, a, d_workspace, d_tickets, stream) : launch_fwd<kReadout, true, false>(dtype, a, d_workspace, d_tickets, stream);
  return top ? launch_fwd<kReadout, false, true>(dtype, a, d_workspace, d_tickets, stream) : launch_fwd<kReadout, false, false>(dtype, a, d_workspace, d_tickets, stream);
}

int vitta_label_logprobs_bwd(const void* d_x, int32_t dtype, int64_t rows, int32_t classes, int64_t row_stride, int64_t inner_rows,
                             int64_t outer_stride, float temperature,
                             const int64_t* d_labels, int64_t ignore_index, int32_t top, const int64_t* d_top_index,
                             const float* d_stats, const float* d_glogprob, int64_t glogprob_stride, const float* d_gentropy,
                             int64_t gentropy_stride, const float* d_glse, int64_t glse_stride, const float* d_gtop, void* d_dx,
                             void* stream) {
  if (bad_scores(d_x, dtype, rows, classes, row_stride, inner_rows, outer_stride, temperature) || bad_stats(d_stats) || bad_out(d_dx, dtype)) return VITTA_ERR_INVALID_ARG;
  if ((d_glogprob && !d_labels) || (d_gtop && (!d_top_index || top <= 0 || top > VITTA_SCORES_MAX_TOP))) return VITTA_ERR_INVALID_ARG;
  if (too_large(rows, classes)) return VITTA_ERR_UNSUPPORTED;
  BwdArgs a{};
  a.x = d_x, a.dx = d_dx, a.rows = rows, a.stride = row_stride, a.outer = outer_stride, a.classes = classes, a.c = kLog2e / temperature, a.inv_t = 1.f / temperature;
  a.inner = (uint32_t)(inner_rows < rows ? inner_rows : rows);
  a.stats = d_stats, a.labels = d_labels, a.ignore = ignore_index, a.top = top, a.top_index = d_top_index;
  a.g_logprob = d_glogprob, a.g_entropy = d_gentropy, a.g_lse = d_glse, a.g_top = d_gtop;
  a.s_logprob = glogprob_stride, a.s_entropy = gentropy_stride, a.s_lse = glse_stride;
  return d_gentropy ? launch_bwd<false, true>(dtype, a, stream) : launch_bwd<false, false>(dtype, a, stream);
}

int vitta_top_distill_fwd(const void* d_x, int32_t dtype, int64_t rows, int32_t classes, int64_t row_stride, int64_t inner_rows,
                             int64_t outer_stride, float temperature,
                          const int64_t* d_index, const void* d_value, int32_t value_dtype, int32_t list, int32_t tail, float* d_loss,
                          float* d_stats, float* d_q, void* d_workspace, size_t workspace_bytes, uint32_t* d_tickets, void* stream) {
  if (bad_scores(d_x, dtype, rows, classes, row_stride, inner_rows, outer_stride, temperature)) return VITTA_ERR_INVALID_ARG;
  if (!d_index || !d_value || !d_loss || bad_stats(d_stats) || !d_q || list <= 0 || list > VITTA_SCORES_MAX_LIST) return VITTA_ERR_INVALID_ARG;
  if (value_dtype < VITTA_SCORES_F32 || value_dtype > VITTA_SCORES_F16) return VITTA_ERR_INVALID_ARG;
  if (too_large(rows, classes)) return VITTA_ERR_UNSUPPORTED;
  const size_t need = vitta_scores_workspace_bytes(rows, classes, dtype, 0);
  if (workspace_bytes < need || (need && bad_stats(d_workspace))) return VITTA_ERR_WORKSPACE;
  FwdArgs a{};
  a.x = d_x, a.rows = rows, a.stride = row_stride, a.outer = outer_stride, a.classes = classes, a.c = kLog2e / temperature, a.inv_t = 1.f / temperature;
  a.inner = (uint32_t)(inner_rows < rows ? inner_rows : rows);
  a.stats = d_stats, a.index = d_index, a.value = d_value, a.value_type = value_dtype, a.list = list;
  a.loss = d_loss, a.q = d_q;
  return tail ? launch_fwd<kDistillTail, false, false>(dtype, a, d_workspace, d_tickets, stream) : launch_fwd<kDistill, false, false>(dtype, a, d_workspace, d_tickets, stream);
}

int vitta_top_distill_bwd(const void* d_x, int32_t dtype, int64_t rows, int32_t classes, int64_t row_stride, int64_t inner_rows,
                             int64_t outer_stride, float temperature,
                          const int64_t* d_index, int32_t list, const float* d_stats, const float* d_q, const float* d_g,
                          int64_t g_stride, void* d_dx, void* stream) {
  if (bad_scores(d_x, dtype, rows, classes, row_stride, inner_rows, outer_stride, temperature)) return VITTA_ERR_INVALID_ARG;
  if (!d_index || bad_stats(d_stats) || !d_q || !d_g || bad_out(d_dx, dtype) || list <= 0 || list > VITTA_SCORES_MAX_LIST) return VITTA_ERR_INVALID_ARG;
  if (too_large(rows, classes)) return VITTA_ERR_UNSUPPORTED;
  BwdArgs a{};
  a.x = d_x, a.dx = d_dx, a.rows = rows, a.stride = row_stride, a.outer = outer_stride, a.classes = classes, a.c = kLog2e / temperature, a.inv_t = 1.f / temperature;
  a.inner = (uint32_t)(inner_rows < rows ? inner_rows : rows);
  a.stats = d_stats, a.index = d_index, a.list = list, a.q = d_q, a.g = d_g, a.s_g = g_stride;
  return launch_bwd<true, false>(dtype, a, stream);
}

}  // extern "C"
