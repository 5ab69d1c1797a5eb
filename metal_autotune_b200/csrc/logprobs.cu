// Log-probabilities of given tokens with entropy, logsumexp and the top
// alternatives of each row of logits, in one pass over the logits.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "paged_common.cuh"

namespace cg = cooperative_groups;

namespace mt {
namespace {

// 5 CTAs of 256 threads per SM, 64 bytes in flight a thread: 2048 x 151936 bf16 with 20 alternatives 126 us when it was
// chosen (120 now); 4 CTAs 133, 6 (40 registers, spilled) 165, 3 vectors in flight 133, 3 CTAs of 512 threads 142.
constexpr int kThreads = 256;
constexpr int kCtasPerSm = 5;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;    // one key per lane
constexpr int kMaxSplit = 8;   // CTAs to a row
static_assert(kMaxSplit <= kWarps, "the first CTA joins a list per warp");
// 16-byte loads a thread has in flight (a batch). Rows that several CTAs share leave a thread few vectors (151936 values
// over 8 CTAs 9 or 10), so twice as many at once, at 4 CTAs per SM, whose registers that takes: one row 8.4 -> 8.1 us,
// 256 rows 28.0 -> 25.2. (12 at 3 CTAs: 8.4 and 29.1.)
constexpr int kUnrollMany = 4, kUnrollFew = 8, kCtasPerSmFew = 4;
constexpr int kGroups = 64;    // groups of threads whose maxima bound the k-th largest value
constexpr int kEntries = 32;   // maxima of its batches that a thread keeps
constexpr int kCap = 2048;     // candidates kept before the exact form takes over
constexpr int kNothingSeen = 2;  // Smem::exact: sums of 0, no NaN: every value is -inf or far below kFloor
constexpr float kLog2e = 1.4426950408889634f;
// what a unit of the sums' exponents is worth: by the constant that they were scaled with, not by ln 2, or the largest
// logit would come back 1.3e-8 of itself off (2.7e-4 at 20000)
constexpr double kUnit = 1.0 / static_cast<double>(kLog2e);

// Larger keys first: the value's order, then the lower index. NaN sorts above
// every number, -0 equals +0. No element's key is 0.
__device__ __forceinline__ uint64_t top_key(float v, uint32_t i) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t u = isnan(v) ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return static_cast<uint64_t>(u) << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ int key_index(uint64_t key) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
}

// A 16-byte vector of logits: its maxima (NaN skipped where there is another
// value), its values as they are, and its values with -inf raised to a finite
// bound far below kFloor, NaN kept: 0 * -inf never arises in the sums. The
// maxima of 16-bit values stay two to a register until a batch's are joined
// (32 rows 11.8 -> 11.6 us, 256 25.2 -> 24.6, 2048 121.2 -> 120.3).
template <typename T2> struct Vec16 {
  static constexpr int E = 8;
  using Max = T2;
  static __device__ __forceinline__ Max maxima(const uint4& u) {
    const T2* h = reinterpret_cast<const T2*>(&u);
    return __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return __hmax2(a, b); }
  static __device__ __forceinline__ Max across(Max a) { return __hmax2(a, __lowhigh2highlow(a)); }  // in both halves
  static __device__ __forceinline__ bool holds(Max a, Max whole) { return __heq2_mask(a, whole) != 0; }
  static __device__ __forceinline__ float value(Max whole) { return __low2float(whole); }
};
template <int DT> struct Vec;
template <> struct Vec<MT_BF16> : Vec16<__nv_bfloat162> {
  static __device__ __forceinline__ __nv_bfloat16 round_up(Max whole) { return __low2bfloat16(whole); }
  static __device__ __forceinline__ float raw(const uint4& u, int e) {
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(&u)[e]);
  }
  static __device__ __forceinline__ float2 pair(const uint4& u, int p) {
    const __nv_bfloat162 low = __float2bfloat162_rn(-1e30f);
    return __bfloat1622float2(__hmax2_nan(reinterpret_cast<const __nv_bfloat162*>(&u)[p], low));
  }
};
template <> struct Vec<MT_F16> : Vec16<__half2> {
  static __device__ __forceinline__ __nv_bfloat16 round_up(Max whole) { return __float2bfloat16_ru(value(whole)); }
  static __device__ __forceinline__ float raw(const uint4& u, int e) {
    return __half2float(reinterpret_cast<const __half*>(&u)[e]);
  }
  static __device__ __forceinline__ float2 pair(const uint4& u, int p) {
    const __half2 low = __float2half2_rn(-65504.f);
    return __half22float2(__hmax2_nan(reinterpret_cast<const __half2*>(&u)[p], low));
  }
};
template <> struct Vec<MT_F32> {
  static constexpr int E = 4;
  using Max = float;
  static __device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
  }
  static __device__ __forceinline__ Max maxima(const uint4& u) {
    return fmaxf(fmaxf(raw(u, 0), raw(u, 1)), fmaxf(raw(u, 2), raw(u, 3)));
  }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return fmaxf(a, b); }
  static __device__ __forceinline__ Max across(Max a) { return a; }
  static __device__ __forceinline__ bool holds(Max a, Max whole) { return a == whole; }
  static __device__ __forceinline__ float value(Max whole) { return whole; }
  static __device__ __forceinline__ __nv_bfloat16 round_up(Max whole) { return __float2bfloat16_ru(whole); }
  static __device__ __forceinline__ float raw(const uint4& u, int e) {
    return reinterpret_cast<const float*>(&u)[e];
  }
  static __device__ __forceinline__ float2 pair(const uint4& u, int p) {
    return make_float2(max_nan(raw(u, 2 * p), -1e30f), max_nan(raw(u, 2 * p + 1), -1e30f));
  }
};
constexpr float kFloor = -3e4f;  // rows whose maximum lies below it take the exact form

// The running sums of a thread: s = sum 2^z, t = sum 2^z z, z = x log2(e) - M,
// in two halves for the packed instructions. M is a whole number at most 1/2
// off the largest x log2(e) seen, so z is rounded once, z of the largest value
// is near 0, and neither sum cancels or overflows.
struct Sums {
  float2 s, t;
  float M, ref;  // ref: the value M belongs to
  __device__ __forceinline__ void raise(float v) {
    const float m = rintf(v * kLog2e), d = M - m, f = exp2_approx(d);
    t.x = f * fmaf(d, s.x, t.x);
    t.y = f * fmaf(d, s.y, t.y);
    s.x *= f;
    s.y *= f;
    M = m;
    ref = v;
  }
  __device__ __forceinline__ void add(float2 x) {
    const float2 z = fma2(x, make_float2(kLog2e, kLog2e), make_float2(-M, -M));
    const float2 p = make_float2(exp2_approx(z.x), exp2_approx(z.y));
    s = add2(s, p);
    t = fma2(p, z, t);
  }
};

// ------------------------------------------------ a warp's sorted top 32 keys
__device__ __forceinline__ uint64_t pick(uint64_t a, int o, bool larger) {
  const uint64_t b = __shfl_xor_sync(0xffffffffu, a, o);
  return (b > a) == larger ? b : a;
}
// bitonic sequence -> falling
__device__ __forceinline__ uint64_t merge_down(uint64_t a, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = pick(a, o, (lane & o) == 0);
  return a;
}
// any order -> rising
__device__ __forceinline__ uint64_t sort_up(uint64_t a, int lane) {
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int o = n >> 1; o > 0; o >>= 1) a = pick(a, o, ((lane & o) == 0) == ((lane & n) != 0 && n < 32));
  return a;
}
// any order -> falling
__device__ __forceinline__ uint64_t sort_down(uint64_t a, int lane) {
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int o = n >> 1; o > 0; o >>= 1) a = pick(a, o, ((lane & o) == 0) == ((lane & n) == 0 || n == 32));
  return a;
}
// falling list + rising batch -> falling list of the 32 largest
__device__ __forceinline__ uint64_t take(uint64_t list, uint64_t rising, int lane) {
  return merge_down(list > rising ? list : rising, lane);
}

struct Slice {  // what a CTA found in its part of a row
  double m;    // a whole number of units, or the largest logit itself: neither is rounded to fp32
  float s, t;  // sum e^(x-m), sum e^(x-m) (x-m); s = 0 where every logit is -inf
  uint64_t list[kMaxTop];
};

struct Smem {
  uint64_t buf[kCap];
  uint64_t lists[kWarps][32];
  uint64_t group[kGroups];
  uint64_t thr_key;
  __nv_bfloat16 batch_max[kEntries][kThreads];
  float red[3][kWarps];
  double red_d[2][kWarps];
  int count, hits, exact;  // exact: the sums of one pass will not do
  Slice out;
};

// The top 32 keys of the first `live` warps' falling lists, in warp 0, joined
// in pairs. All threads take part.
__device__ __forceinline__ uint64_t join_lists(Smem& sm, uint64_t list, int live) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  while (live > 1) {
    const int half = (live + 1) >> 1;
    if (warp >= half && warp < live) sm.lists[warp][lane] = list;
    __syncthreads();
    if (warp + half < live) list = take(list, sm.lists[warp + half][31 - lane], lane);
    live = half;  // the lists written next belong to warps that read here, none is read twice
  }
  return list;
}

struct LogprobArgs {
  const void* logits;
  int64_t stride, V;
  const int32_t* tokens;
  int top_k, split_bits;  // 2^split_bits CTAs to a row
  float *logprob, *entropy, *lse;
  int32_t* top_ids;
  float* top_lp;
};

// The part of a row that one CTA reads: vectors [v0, v1) of the aligned body,
// and, for the first part, the unaligned values before and after the body.
template <int DT>
struct Part {
  const typename Elem<DT>::T* x;
  int head, tail;       // values before / after the body that belong to this part
  int64_t body, tail0;  // index of the body's first value, of the first value after it
  int64_t v0, v1;
  __device__ __forceinline__ const uint4* vec() const { return reinterpret_cast<const uint4*>(x + body); }
};

// A part of one value throughout, as a mask (-inf, or the type's lowest value)
// that allows one range of ids leaves beside it: the sums are known, and its
// first values are the candidates. True if it is one. (By the exact form below,
// with a barrier for each 256 values, such a part held up its row: a hundredth of
// 151936 ids in one range took 79 us for one row and 305 for 256, where as many
// anywhere in the row take 9 and 25.)
template <int DT>
__device__ __forceinline__ bool constant_slice(Smem& sm, const Part<DT>& p) {
  using V = Vec<DT>;
  const int tid = threadIdx.x;
  const int64_t a0 = p.body + p.v0 * V::E, n_body = (p.v1 - p.v0) * V::E;
  const int64_t n = n_body + p.head + p.tail;
  if (n == 0) return false;
  const float c = Elem<DT>::to_f(p.x[n_body > 0 ? a0 : p.head > 0 ? 0 : p.tail0]);
  bool other = false;
#pragma unroll 4
  for (int64_t j = p.v0 + tid; j < p.v1; j += kThreads) {
    const uint4 w = p.vec()[j];
#pragma unroll
    for (int e = 0; e < V::E; ++e) other |= V::raw(w, e) != c;
  }
  if (tid < p.head) other |= Elem<DT>::to_f(p.x[tid]) != c;
  if (tid < p.tail) other |= Elem<DT>::to_f(p.x[p.tail0 + tid]) != c;
  if (__syncthreads_or(other)) return false;
  if (tid < 32) {
    const int64_t b = tid - p.head, t = b - n_body;
    const int64_t i = b < 0 ? tid : t < 0 ? a0 + b : t < p.tail ? p.tail0 + t : -1;
    sm.out.list[tid] = i >= 0 ? top_key(c, static_cast<uint32_t>(i)) : 0;
  }
  if (tid == 0) {
    sm.out.m = c;
    sm.out.s = c == -INFINITY ? 0.f : static_cast<float>(n);
    sm.out.t = 0.f;
  }
  return true;
}

// Any input, several passes: every logit tiny, NaN, +inf, or more candidates
// than the buffer holds (values that keep rising along the row).
template <int DT>
__device__ __noinline__ void exact_slice(Smem& sm, const Part<DT>& p, int top_k) {
  if (sm.exact == kNothingSeen && constant_slice<DT>(sm, p)) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int E = Vec<DT>::E;
  const int64_t a0 = p.body + p.v0 * E, n_body = (p.v1 - p.v0) * E;
  const int64_t n = n_body + p.head + p.tail;
  auto index = [&](int64_t j) {
    return j < n_body ? a0 + j : j < n_body + p.head ? j - n_body : p.tail0 + (j - n_body - p.head);
  };
  float m = -INFINITY;
  for (int64_t j = tid; j < n; j += kThreads) m = fmaxf(m, Elem<DT>::to_f(p.x[index(j)]));
  m = warp_max(m);
  if (lane == 0) sm.red[0][warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sm.red[0][w]);
  double s = 0, t = 0;
  for (int64_t j = tid; j < n; j += kThreads) {
    const float x = Elem<DT>::to_f(p.x[index(j)]);
    if (x == -INFINITY) continue;
    const float z = x - m, e = expf(z);
    s += e;
    if (e != 0.f) t += static_cast<double>(e) * z;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  if (lane == 0) {
    sm.red_d[0][warp] = s;
    sm.red_d[1][warp] = t;
  }
  if (tid == 0) sm.count = 0;
  if (tid < 32) sm.lists[0][tid] = 0;
  __syncthreads();
  if (tid == 0) {
    s = t = 0;
    for (int w = 0; w < kWarps; ++w) {
      s += sm.red_d[0][w];
      t += sm.red_d[1][w];
    }
    sm.out.m = m;
    sm.out.s = static_cast<float>(s);
    sm.out.t = static_cast<float>(t);
  }
  if (top_k == 0) return;
  for (int64_t j0 = 0; j0 < n; j0 += kThreads) {
    const uint64_t least = sm.lists[0][top_k - 1];
    if (j0 + tid < n) {
      const int64_t i = index(j0 + tid);
      const uint64_t key = top_key(Elem<DT>::to_f(p.x[i]), static_cast<uint32_t>(i));
      if (key > least) sm.buf[atomicAdd(&sm.count, 1)] = key;
    }
    __syncthreads();
    const int c = sm.count;  // at most kThreads
    if (c > 0) {
      if (warp == 0) {
        uint64_t list = sm.lists[0][lane];
        for (int b = 0; b < c; b += 32) list = take(list, sort_up(b + lane < c ? sm.buf[b + lane] : 0, lane), lane);
        sm.lists[0][lane] = list;
      }
      __syncthreads();
      if (tid == 0) sm.count = 0;
    }
    __syncthreads();
  }
  if (tid < 32) sm.out.list[tid] = sm.lists[0][tid];
}

// One pass over the logits for the sums, with a note of where large values are:
// each thread keeps the maximum of every batch of 4 vectors that it read (in
// bf16, rounded up) and its largest value. Of the maxima of 64 groups of
// threads, the k-th largest bounds the k-th largest logit from below, at about
// 1.2 k values above it for logits in no particular order; only batches that
// reach the bound are read a second time, and their values that do are sorted.
// An equal value counts up to the bound's own place in the row (ties go to the
// lower index), so constant or masked stretches stay within the buffer too.
// Which thread stores a candidate where does not matter: keys are unique and
// the sort is by key.
//
// Many rows: 2048 x 151936 bf16 with 20 alternatives in 120 us = 5.2 TB/s, 79%
// of the copy rate (223 us when the bound came from the row's beginning and
// candidates left the loop one by one). Instructions and the ends of rows bound
// it, not memory: issue slots are 67% busy, DRAM 61%. What follows the loop, 20%
// of a CTA's time, is covered by the SM's other CTAs only in part: without
// alternatives 107 us, 89%. A quarter of the powers as polynomials of degree 5,
// off the special-function units, took 132 us; and call after call under the
// power limit, at a lower clock, the 120 become 127 to 135.
template <int DT, int kUnroll>
__device__ __forceinline__ bool one_pass(Smem& sm, const Part<DT>& p, int top_k) {
  using V = Vec<DT>;
  constexpr int E = V::E, kBatch = kThreads * kUnroll;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = static_cast<int>(p.v1 - p.v0);                   // an index is below 2^31
  const uint32_t i0 = static_cast<uint32_t>(p.body + p.v0 * E);  // index of the slice's first value
  const uint4* v = p.vec() + p.v0;
  const int batches = (n + kBatch - 1) / kBatch;
  const int per = (batches + kEntries - 1) / kEntries;  // batches to an entry
  uint4 none;                                           // -inf throughout
  none.x = none.y = none.z = none.w = DT == MT_BF16 ? 0xff80ff80u : DT == MT_F16 ? 0xfc00fc00u : 0xff800000u;

  Sums a;
  a.s = a.t = make_float2(0.f, 0.f);
  a.ref = kFloor;
  a.M = rintf(kFloor * kLog2e);
  // a value before or after the aligned body; it stays out of the bound (one after the body ranks behind its equals)
  float extra = 0.f;
  int extra_i = -1;
  if (tid < p.head) extra_i = tid;
  else if (tid >= 32 && tid < 32 + p.tail) extra_i = static_cast<int>(p.tail0) + (tid - 32);
  if (extra_i >= 0) {
    extra = Elem<DT>::to_f(p.x[extra_i]);
    if (extra > a.ref) a.raise(extra);
    a.add(make_float2(extra == -INFINITY ? -1e30f : extra, -1e30f));
    a.s.y = a.t.y = 0.f;
  }
  float top = 0.f;  // the thread's largest value, in vector `at` (the first that holds it)
  int at = -1, entry = 0, in_entry = 0;
  auto take_batch = [&](const uint4 (&r)[kUnroll], int j0, int left) {  // left: vectors from the warp's first on
    typename V::Max m[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) m[u] = V::maxima(r[u]);
    typename V::Max whole = m[0];
#pragma unroll
    for (int u = 1; u < kUnroll; ++u) whole = V::larger(whole, m[u]);
    whole = V::across(whole);
    const float mb = V::value(whole);
    if (top_k > 0) {
      if (at < 0 || mb > top) {
        top = mb;
        int first = kUnroll - 1;
#pragma unroll
        for (int u = kUnroll - 2; u >= 0; --u) first = V::holds(m[u], whole) ? u : first;
        at = j0 + first * kThreads;
      }
      __nv_bfloat16 up = V::round_up(whole);
      if (in_entry > 0) up = __hmax(up, sm.batch_max[entry][tid]);
      sm.batch_max[entry][tid] = up;
      if (++in_entry == per) {
        in_entry = 0;
        ++entry;
      }
    }
    if (mb > a.ref + 1.0f) a.raise(mb);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (u * kThreads < left) {
#pragma unroll
        for (int q = 0; q < E / 2; ++q) a.add(V::pair(r[u], q));
      }
  };
  int j0 = 0;
  for (; j0 + kBatch <= n; j0 += kBatch) {
    uint4 r[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) r[u] = __ldcs(v + j0 + u * kThreads + tid);
    take_batch(r, j0, kBatch);
  }
  if (j0 < n) {
    uint4 r[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int j = j0 + u * kThreads + tid;
      r[u] = j < n ? __ldcs(v + j) : none;
    }
    take_batch(r, j0, n - j0 - warp * 32);
  }

  // the bound: the k-th largest of the groups' maxima
  uint64_t mine = 0;
  if (tid < n && top_k > 0) mine = top_key(top, i0 + static_cast<uint32_t>(at + tid) * E + E - 1);
#pragma unroll
  for (int o = 1; o < kThreads / kGroups; o <<= 1) {
    const uint64_t k = __shfl_xor_sync(0xffffffffu, mine, o);
    mine = k > mine ? k : mine;
  }
  constexpr int kPer = kThreads / kGroups;  // threads to a group; together they compare its key with all groups'
  const int group = tid / kPer;
  if (tid % kPer == 0) sm.group[group] = mine;
  if (tid == 0) {
    sm.count = sm.hits = 0;
    sm.thr_key = 0;
  }

  // the block's sums, relative to the largest M
  const float mw = warp_max(a.M);
  float d = a.M - mw, f = exp2_approx(d);
  float s = a.s.x + a.s.y, t = a.t.x + a.t.y;
  t = warp_sum(f * fmaf(d, s, t));
  s = warp_sum(f * s);
  if (lane == 0) {
    sm.red[0][warp] = mw;
    sm.red[1][warp] = s;
    sm.red[2][warp] = t;
  }
  __syncthreads();
  {
    int rank = 0;  // groups ahead of this one; empty ones (key 0) by their number
#pragma unroll
    for (int i = 0; i < kGroups / kPer; ++i) {
      const int g = i * kPer + tid % kPer;
      const uint64_t k = sm.group[g];
      rank += k > mine || (k == mine && g < group);
    }
#pragma unroll
    for (int o = 1; o < kPer; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (tid % kPer == 0 && rank == top_k - 1) sm.thr_key = mine;
  }
  auto join_sums = [&]() {  // a warp
    const float mr = lane < kWarps ? sm.red[0][lane] : -INFINITY;
    const float mb = warp_max(mr);
    d = lane < kWarps ? mr - mb : 0.f;
    f = lane < kWarps ? exp2_approx(d) : 0.f;
    s = lane < kWarps ? sm.red[1][lane] : 0.f;
    t = lane < kWarps ? sm.red[2][lane] : 0.f;
    t = warp_sum(f * fmaf(d, s, t));
    s = warp_sum(f * s);
    if (lane == 0) {
      sm.out.m = static_cast<double>(mb) * kUnit;
      sm.out.s = s;
      sm.out.t = t * static_cast<float>(kUnit);
      // the largest value alone adds over 1/2, unless it lies below kFloor or the row holds NaN or +inf
      sm.exact = s >= 0.25f && s < INFINITY && t == t ? 0 : s == 0.f && t == 0.f ? kNothingSeen : 1;
    }
  };
  if (top_k == 0) {
    if (warp == 0) join_sums();
    __syncthreads();
    return !sm.exact;
  }
  __syncthreads();
  const uint64_t thr_key = sm.thr_key;
  const float thr = key_value(thr_key);  // NaN where fewer than k groups hold anything: all count
  auto push = [&](uint64_t key) {
    if (key < thr_key) return;
    const int c = atomicAdd(&sm.count, 1);
    if (c < kCap) sm.buf[c] = key;
  };
  auto look = [&](int j) {
    const uint4 w = v[j];
    if (V::value(V::across(V::maxima(w))) < thr) return;
#pragma unroll
    for (int i = 0; i < E; ++i) push(top_key(V::raw(w, i), i0 + static_cast<uint32_t>(j) * E + i));
  };
  // the batches that reach the bound, as their first vectors; read again by all threads at once
  int* hits = reinterpret_cast<int*>(sm.lists);
  constexpr int kHits = sizeof(sm.lists) / sizeof(int);
  const int span = per * kBatch;
  if (warp == kWarps - 1) join_sums();
  for (int e = 0; e * span < n; ++e)
    if (!(__bfloat162float(sm.batch_max[e][tid]) < thr)) {
      const int h = atomicAdd(&sm.hits, 1);
      if (h < kHits) hits[h] = e * span + tid;
    }
  __syncthreads();
  if (sm.exact) return false;
  if (sm.hits <= kHits) {
    for (int i = tid; i < sm.hits * per * kUnroll; i += kThreads) {
      const int h = i / (per * kUnroll), j = hits[h] + (i - h * per * kUnroll) * kThreads;
      if (j < n) look(j);
    }
  } else {  // long stretches of equal values
    for (int e = 0; e * span < n; ++e)
      if (!(__bfloat162float(sm.batch_max[e][tid]) < thr))
        for (int j = e * span + tid; j < min(n, (e + 1) * span); j += kThreads) look(j);
  }
  if (extra_i >= 0) push(top_key(extra, static_cast<uint32_t>(extra_i)));
  __syncthreads();
  if (sm.count > kCap) return false;
  // top 32 of the candidates: batches of 32 sorted by the warps, their lists joined in pairs
  const int c = sm.count;
  uint64_t list = 0;
  if (warp * 32 < c) list = sort_down(warp * 32 + lane < c ? sm.buf[warp * 32 + lane] : 0, lane);
  for (int b = warp * 32 + kThreads; b < c; b += kThreads)
    list = take(list, sort_up(b + lane < c ? sm.buf[b + lane] : 0, lane), lane);
  list = join_lists(sm, list, min(kWarps, (c + 31) >> 5));
  if (warp == 0) sm.out.list[lane] = list;
  return true;
}

// A row per CTA, or `split` CTAs of a cluster per row where there are few rows;
// the first joins the others' sums and lists through distributed shared memory.
template <int DT, int kUnroll, int kPerSm>
__global__ void __launch_bounds__(kThreads, kPerSm) logprobs_kernel(const LogprobArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int E = Vec<DT>::E;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x, lane = tid & 31;
  const int split = 1 << a.split_bits;
  const int64_t row = blockIdx.x >> a.split_bits;
  const int rank = blockIdx.x & (split - 1);
  Part<DT> p;
  p.x = static_cast<const T*>(a.logits) + row * a.stride;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(p.x) & 15) / sizeof(T));
  p.body = min(static_cast<int64_t>((E - off) % E), a.V);
  const int64_t nvec = (a.V - p.body) / E;
  p.tail0 = p.body + nvec * E;
  p.v0 = nvec * rank >> a.split_bits;
  p.v1 = nvec * (rank + 1) >> a.split_bits;
  p.head = rank == 0 ? static_cast<int>(p.body) : 0;
  p.tail = rank == 0 ? static_cast<int>(a.V - p.tail0) : 0;
  if (!one_pass<DT, kUnroll>(sm, p, a.top_k)) exact_slice<DT>(sm, p, a.top_k);
  __syncthreads();
  double m = sm.out.m;
  float s = sm.out.s, t = sm.out.t;
  uint64_t list = tid < 32 ? sm.out.list[lane] : 0;
  if (split > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (rank == 0) {
      const int warp = tid >> 5;
      if (a.top_k > 0) {  // a list per warp
        if (warp < split) list = cluster.map_shared_rank(&sm.out, warp)->list[lane];
        list = join_lists(sm, list, split);
      }
      if (warp == 0) {  // sums, a slice per lane of each eight
        const int c = lane & (kMaxSplit - 1);
        const Slice* o = cluster.map_shared_rank(&sm.out, c < split ? c : 0);
        const double om = o->m;
        const float os = c < split ? o->s : 0.f, ot = o->t;
        m = os == 0.f ? -INFINITY : om;  // a slice of -inf alone, or a lane without one
#pragma unroll
        for (int q = kMaxSplit / 2; q > 0; q >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, q));
        const float d = static_cast<float>(om - m), f = exp2_approx(d * kLog2e);
        s = os == 0.f ? 0.f : f * os;
        t = f == 0.f || os == 0.f ? 0.f : f * fmaf(d, os, ot);  // (d may be past the range of floats)
#pragma unroll
        for (int q = kMaxSplit / 2; q > 0; q >>= 1) {
          s += __shfl_xor_sync(0xffffffffu, s, q);
          t += __shfl_xor_sync(0xffffffffu, t, q);
        }
      }
    }
    cluster.sync();  // the other CTAs' shared memory stays alive until it has been read
    if (rank != 0) return;
  }
  if (tid >= 32) return;
  const float ls = s > 0.f ? logf(s) : NAN;  // no distribution: NaN throughout
  const double lse = m + ls;
  // of a token that carries the row, rounding (the powers': 2^-22) can put the logarithm, and the entropy, past 0
  auto log_prob = [&](float x) {
    const float lp = static_cast<float>(x - lse);
    return lp > 0.f ? 0.f : lp;
  };
  if (lane == 0) {
    if (a.lse) a.lse[row] = static_cast<float>(lse);
    const float entropy = ls - t / s;
    if (a.entropy) a.entropy[row] = entropy < 0.f ? 0.f : entropy;
    if (a.tokens) {
      const int tok = a.tokens[row];
      if (tok >= a.V) report_status(0x801);
      a.logprob[row] = tok >= 0 && tok < a.V ? log_prob(Elem<DT>::to_f(p.x[tok])) : 0.f;
    }
  }
  if (lane < a.top_k) {
    a.top_ids[row * a.top_k + lane] = key_index(list);
    a.top_lp[row * a.top_k + lane] = log_prob(key_value(list));
  }
}

}  // namespace
}  // namespace mt

using namespace mt;

extern "C" int mt_token_logprobs(const void* logits, int64_t row_stride, const int32_t* tokens, int64_t R, int64_t V,
                                 int top_k, float* logprob, float* entropy, float* lse, int32_t* top_ids,
                                 float* top_logprobs, int dtype, mt_stream_t stream) {
  clear_error();
  MT_CHECK_ARG(R >= 0 && R < (1ll << 24) && V > 0 && V < (1ll << 31) - 1 && row_stride >= V,
               "mt_token_logprobs: R=%lld V=%lld row_stride=%lld", (long long)R, (long long)V, (long long)row_stride);
  MT_CHECK_ARG(top_k >= 0 && top_k <= kMaxTop && top_k <= V, "mt_token_logprobs: top_k=%d outside 0..min(%d, V)",
               top_k, kMaxTop);
  if (dtype != MT_BF16 && dtype != MT_F16 && dtype != MT_F32) {
    set_error("mt_token_logprobs: unsupported dtype %d", dtype);
    return MT_ERR_UNSUPPORTED;
  }
  if (R == 0) return MT_OK;
  MT_CHECK_ARG(logits && (!tokens || logprob) && (top_k == 0 || (top_ids && top_logprobs)),
               "mt_token_logprobs: null pointer");
  MT_CHECK_ARG(aligned(logits, dtype == MT_F32 ? 4 : 2), "mt_token_logprobs: logits not aligned to their type");
  int sms = 148;
  if (int rc = device_sm_count(&sms)) return rc;
  int bits = 0;
  while ((2 << bits) <= kMaxSplit && (R << (bits + 1)) <= kCtasPerSmFew * sms && (V >> (bits + 1)) >= 4096) ++bits;
  const LogprobArgs a = {logits, row_stride, V, tokens, top_k, bits, logprob, entropy, lse, top_ids, top_logprobs};
  // where there are fewer CTAs than fit, as much shared memory as leaves every SM its share of them: clusters are else
  // packed onto some of the SMs
  // (and a little more room for clusters of 8, which do not come out even over the SMs)
  const int64_t ctas = R << bits, share = ((bits == 3 ? ctas + ctas / 4 : ctas) + sms - 1) / sms;
  size_t smem = sizeof(Smem);
  if (share < (bits > 0 ? kCtasPerSmFew : kCtasPerSm)) smem = std::max(smem, static_cast<size_t>(228 * 1024 / share - 1024) / 1024 * 1024);
  auto run = [&](auto kern) -> int {
    if (int e = ensure_smem(kern, 227 * 1024)) return e;
    return launch_cluster(kern, dim3((unsigned)(R << bits)), dim3(kThreads), smem, 1 << bits, (cudaStream_t)stream, a);
  };
  auto pick_unroll = [&](auto type) -> int {
    constexpr int DT = decltype(type)::value;
    return bits > 0 ? run(logprobs_kernel<DT, kUnrollFew, kCtasPerSmFew>) : run(logprobs_kernel<DT, kUnrollMany, kCtasPerSm>);
  };
  return dtype == MT_BF16  ? pick_unroll(std::integral_constant<int, MT_BF16>())
         : dtype == MT_F16 ? pick_unroll(std::integral_constant<int, MT_F16>())
                           : pick_unroll(std::integral_constant<int, MT_F32>());
}
