// Paged serving, per step and per layer: the step's plan (block tables, slots
// and positions from request lengths) and the q/k prologue that rotates each
// row at its own position and writes k and v to their slots of the cache.
#include "mt_common.cuh"

namespace mt {
namespace {

// ------------------------------------------------------------------ step plan
// Two prefix sums over the requests decide everything: new tokens (where each
// request's rows start) and new pages (which free pages it gets). Both are
// sums of non-negative numbers that saturate at INT32_MAX, so adding in any
// grouping gives the same result and nothing overflows, whatever the lengths.
constexpr int kPlanThreads = 512;
constexpr int kPlanItems = 8;
constexpr int kPlanChunk = kPlanThreads * kPlanItems;  // requests scanned at a time
constexpr int kPlanMax = 0x7fffffff;

__device__ __forceinline__ int sat_add(int a, int b) {
  const uint32_t s = static_cast<uint32_t>(a) + static_cast<uint32_t>(b);
  return s > static_cast<uint32_t>(kPlanMax) ? kPlanMax : static_cast<int>(s);
}

struct PlanScan {
  int warp_sum[kPlanThreads / 32];
};

// Inclusive saturating scan of `own` over the block, plus `carry`; returns the
// exclusive prefix of this thread and the block's total through `total`.
__device__ __forceinline__ int plan_scan(int own, int carry, PlanScan& sm, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc = sat_add(inc, u);
  }
  int before = __shfl_up_sync(0xffffffffu, inc, 1);
  if (lane == 0) before = 0;
  if (lane == 31) sm.warp_sum[warp] = inc;
  __syncthreads();
  int w = lane < kPlanThreads / 32 ? sm.warp_sum[lane] : 0;
#pragma unroll
  for (int o = 1; o < kPlanThreads / 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w = sat_add(w, u);
  }
  const int prev = warp > 0 ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
  total = sat_add(carry, __shfl_sync(0xffffffffu, w, kPlanThreads / 32 - 1));
  __syncthreads();  // sm.warp_sum is written again by the next scan
  return sat_add(carry, sat_add(prev, before));
}

struct PlanArgs {
  const int32_t *ctx, *fresh;
  int64_t B;
  int32_t* table;
  int64_t table_stride, max_pages;
  const int32_t *free_pages, *free_head;
  int64_t n_free;
  int page_size;
  int64_t cap;
  int32_t *seq_lens, *query_start, *positions, *token_seq;
  int64_t* slots;
  int32_t* counts;
};

// Every CTA scans the lengths for itself (a few microseconds of latency would
// go into any exchange between CTAs, and 4096 lengths are 32 KB out of L2) and
// keeps the chunk's prefixes in shared memory; tokens, new pages and request
// outputs are then shared out over the grid, each found by a binary search. A
// token on a new page takes the page from the free list directly, so no CTA
// reads a table entry that another one writes.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a) {
  extern __shared__ int plan_smem[];
  int* tok_end = plan_smem;                  // inclusive sums of new tokens
  int* page_end = tok_end + kPlanChunk;      // inclusive sums of new pages
  int* ctx_of = page_end + kPlanChunk;       // cached tokens; ~cached where the request is refused
  __shared__ PlanScan scan;
  __shared__ int red[3];
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ps = a.page_size;
  const int n_free = static_cast<int>(a.n_free);
  int head = a.free_head ? *a.free_head : 0;
  head = head < 0 ? 0 : head > n_free ? n_free : head;
  const int avail = n_free - head;
  const int64_t room = a.max_pages * ps < kPlanMax ? a.max_pages * ps : kPlanMax;
  if (tid < 3) red[tid] = 0;
  int tok_base = 0, page_base = 0, refused = 0, taken = 0;
  for (int64_t r0 = 0; r0 < a.B; r0 += kPlanChunk) {
    const int n = static_cast<int>(a.B - r0 < kPlanChunk ? a.B - r0 : kPlanChunk);
    int ctx[kPlanItems], fresh[kPlanItems], need[kPlanItems];
    int own = 0;
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
      const int r = tid * kPlanItems + i;
      ctx[i] = r < n ? max(a.ctx[r0 + r], 0) : 0;
      fresh[i] = r < n ? max(a.fresh[r0 + r], 0) : 0;
      own = sat_add(own, fresh[i]);
    }
    int tok_total, page_total;
    int t = plan_scan(own, tok_base, scan, tok_total);
    own = 0;
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
      t = sat_add(t, fresh[i]);
      const int64_t total = static_cast<int64_t>(ctx[i]) + fresh[i];
      const bool fits = t <= a.cap && total <= room;
      need[i] = fits ? static_cast<int>((total + ps - 1) / ps) - static_cast<int>((static_cast<int64_t>(ctx[i]) + ps - 1) / ps) : -1;
      own = sat_add(own, max(need[i], 0));
      if (tid * kPlanItems + i < n) tok_end[tid * kPlanItems + i] = t;
    }
    int p = plan_scan(own, page_base, scan, page_total);
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
      const int r = tid * kPlanItems + i;
      p = sat_add(p, max(need[i], 0));
      const bool ok = need[i] == 0 || (need[i] > 0 && p <= avail);
      if (r < n) {
        page_end[r] = p;
        ctx_of[r] = ok ? ctx[i] : ~ctx[i];
        refused += !ok;
        if (ok && need[i] > 0) taken = p;
        if (warp % gridDim.x == blockIdx.x) {
          a.seq_lens[r0 + r] = ok ? ctx[i] + fresh[i] : ctx[i];
          a.query_start[r0 + r + 1] = tok_end[r];
        }
      }
    }
    __syncthreads();
    // new pages of this chunk's admitted requests
    const int page_last = min(page_total, avail);
    for (int64_t e = page_base + static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid; e < page_last;
         e += static_cast<int64_t>(gridDim.x) * kPlanThreads) {
      int lo = 0, hi = n - 1;  // first request with page_end > e
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (page_end[mid] > e) hi = mid; else lo = mid + 1;
      }
      const int c = ctx_of[lo];
      if (c < 0) continue;
      const int first = lo > 0 ? page_end[lo - 1] : page_base;
      const int had = static_cast<int>((static_cast<int64_t>(c) + ps - 1) / ps);
      a.table[(r0 + lo) * a.table_stride + had + (e - first)] = a.free_pages[head + e];
    }
    // tokens of this chunk
    const int64_t tok_last = tok_total < a.cap ? tok_total : a.cap;
    for (int64_t k = tok_base + static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid; k < tok_last;
         k += static_cast<int64_t>(gridDim.x) * kPlanThreads) {
      int lo = 0, hi = n - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (tok_end[mid] > k) hi = mid; else lo = mid + 1;
      }
      const int c0 = ctx_of[lo];
      const int c = c0 < 0 ? ~c0 : c0;
      const int start = lo > 0 ? tok_end[lo - 1] : tok_base;
      const int64_t pos = static_cast<int64_t>(c) + (k - start);
      int64_t slot = -1;
      if (c0 >= 0) {
        const int block = static_cast<int>(pos / ps);
        const int had = static_cast<int>((static_cast<int64_t>(c) + ps - 1) / ps);
        const int first = lo > 0 ? page_end[lo - 1] : page_base;
        const int page = block < had ? a.table[(r0 + lo) * a.table_stride + block]
                                     : a.free_pages[head + first + (block - had)];
        if (page >= 0) slot = static_cast<int64_t>(page) * ps + static_cast<int>(pos - static_cast<int64_t>(block) * ps);
      }
      a.positions[k] = static_cast<int>(pos < kPlanMax ? pos : kPlanMax);
      a.token_seq[k] = static_cast<int>(r0 + lo);
      a.slots[k] = slot;
    }
    tok_base = tok_total;
    page_base = page_total;
    __syncthreads();  // the prefixes are overwritten by the next chunk
  }
  for (int64_t k = tok_base + static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid; k < a.cap;
       k += static_cast<int64_t>(gridDim.x) * kPlanThreads) {
    a.positions[k] = 0;
    a.token_seq[k] = -1;
    a.slots[k] = -1;
  }
  if (blockIdx.x != 0) return;
  refused = __reduce_add_sync(0xffffffffu, refused);
  taken = __reduce_max_sync(0xffffffffu, taken);
  if (lane == 0) {
    atomicAdd(&red[0], refused);
    atomicMax(&red[1], taken);
  }
  __syncthreads();
  if (tid == 0) {
    a.query_start[0] = 0;
    a.counts[0] = tok_base;
    a.counts[1] = page_base;
    a.counts[2] = red[1];
    a.counts[3] = red[0];
    a.counts[4] = head + red[1];
  }
}

// ---------------------------------------------------- rotary + paged append
struct AppendArgs {
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  const void *q_w, *k_w;
  float eps, mscale;
  const int32_t* positions;
  const int64_t* slots;
  const float* inv_freq;
  int dims;
  void* q_out;
  int64_t qo_st, qo_sh;
  void* k_out;
  void *k_cache, *v_cache;
  int64_t num_pages, page_stride, head_stride, slot_stride;
  int page_size;
  int Hq, Hkv, D;
  int splits;  // CTAs per token
};

// 8 consecutive elements of a row as fp32
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* p, float (&x)[8]) {
  if constexpr (DT == MT_F32) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const typename Elem<DT>::T2* e = reinterpret_cast<const typename Elem<DT>::T2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<DT>::unpack2(e[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::T* p, const float (&x)[8]) {
  if constexpr (DT == MT_F32) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint4 u;
    typename Elem<DT>::T2* e = reinterpret_cast<typename Elem<DT>::T2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = Elem<DT>::pack2(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

constexpr int kAppendThreads = 256;

// cos and sin (times mscale) of the token's angles, each once, in shared
// memory. The angle is reduced to a fraction of a turn in double, so a position
// of 2^30 rotates as exactly as position 1.
__device__ __forceinline__ void angles(const AppendArgs& a, int64_t t, float2* turn) {
  for (int j = threadIdx.x; j < a.dims >> 1; j += kAppendThreads) {
    const double turns = static_cast<double>(a.positions[t]) * static_cast<double>(a.inv_freq[j]) * 0.15915494309189533577;
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    turn[j] = make_float2(c * a.mscale, s * a.mscale);
  }
}

// offset of the token's cache row (without the head), -1 where it has none
__device__ __forceinline__ int64_t slot_offset(const AppendArgs& a, int64_t t) {
  const int64_t slot = a.slots[t];
  if (slot < 0) return -1;
  const int64_t page = slot < (1ll << 31) ? static_cast<int64_t>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.page_size))
                                           : slot / a.page_size;
  if (page < a.num_pages) return page * a.page_stride + (slot - page * a.page_size) * a.slot_stride;
  report_status(0x701);
  return -1;
}

// 4 consecutive elements as they are in memory
template <int DT> struct Quad;
template <> struct Quad<MT_BF16> { using U = uint2; };
template <> struct Quad<MT_F16> { using U = uint2; };
template <> struct Quad<MT_F32> { using U = float4; };
template <int DT>
__device__ __forceinline__ void unpack4(const typename Quad<DT>::U& u, float* x) {
  if constexpr (DT == MT_F32) {
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
  } else {
    const typename Elem<DT>::T2* e = reinterpret_cast<const typename Elem<DT>::T2*>(&u);
    const float2 a = Elem<DT>::unpack2(e[0]), b = Elem<DT>::unpack2(e[1]);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
  }
}
template <int DT>
__device__ __forceinline__ typename Quad<DT>::U pack4(const float* x) {
  if constexpr (DT == MT_F32) {
    return make_float4(x[0], x[1], x[2], x[3]);
  } else {
    typename Quad<DT>::U u;
    typename Elem<DT>::T2* e = reinterpret_cast<typename Elem<DT>::T2*>(&u);
    e[0] = Elem<DT>::pack2(x[0], x[1]);
    e[1] = Elem<DT>::pack2(x[2], x[3]);
    return u;
  }
}

// One token (or one of `splits` parts of its rows) per CTA, LPR lanes to a row
// (8, 16 or 32 for heads of up to 64, 128, 256), for `dims` in whole eights. A
// lane holds two pieces of four values that rotate with each other: (j, j +
// dims/2), or eight adjacent ones; past `dims`, eight that are copied. So its
// four angles and its norm weights stay in registers for all rows, no value
// crosses lanes but the norm's sum, and the rows' loads are under way before
// the position is known. Norm and rotation in fp32, rounded once.
#ifndef AP_ROWS
#define AP_ROWS 3
#define AP_MIN 3
#endif
template <int DT, int LPR, bool TRAD, bool NORM, int ROWS>
__global__ void __launch_bounds__(kAppendThreads, ROWS > 1 ? AP_MIN : 2) append_kernel(const AppendArgs a) {
  using T = typename Elem<DT>::T;
  using Q = typename Quad<DT>::U;
  constexpr int kRows = kAppendThreads / LPR;
  __shared__ __align__(16) float2 turn[128];
  __shared__ int64_t dst;
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x;
  const int64_t t = blockIdx.x / a.splits;
  const int part = blockIdx.x - static_cast<int>(t) * a.splits;
  const int half = a.dims >> 1, sub = tid % LPR;
  const bool in = sub * 8 < a.D, turned = sub * 8 < a.dims;
  // the lane's two pieces of a row
  const int pa = !in ? 0 : TRAD || !turned ? sub * 8 : sub * 4;
  const int pb = !in ? 0 : TRAD || !turned ? sub * 8 + 4 : half + sub * 4;
  const int H = a.Hq + 2 * a.Hkv;
  const T* q = static_cast<const T*>(a.q) + t * a.q_st;
  const T* k = static_cast<const T*>(a.k) + t * a.k_st;
  const T* v = static_cast<const T*>(a.v) + t * a.v_st;
  Q ra[ROWS], rb[ROWS];
  int row = part * kRows + tid / LPR;
  auto load = [&]() {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = row + i * a.splits * kRows;
      if (r < H && in) {
        const T* src = r < a.Hq ? q + r * a.q_sh : r < a.Hq + a.Hkv ? k + (r - a.Hq) * a.k_sh : v + (r - a.Hq - a.Hkv) * a.v_sh;
        ra[i] = *reinterpret_cast<const Q*>(src + pa);
        rb[i] = *reinterpret_cast<const Q*>(src + pb);
      }
    }
  };
  load();
  Q wq[2], wk[2];
  if constexpr (NORM) {
    if (a.q_w) {
      wq[0] = *reinterpret_cast<const Q*>(static_cast<const T*>(a.q_w) + pa);
      wq[1] = *reinterpret_cast<const Q*>(static_cast<const T*>(a.q_w) + pb);
    }
    if (a.k_w) {
      wk[0] = *reinterpret_cast<const Q*>(static_cast<const T*>(a.k_w) + pa);
      wk[1] = *reinterpret_cast<const Q*>(static_cast<const T*>(a.k_w) + pb);
    }
  }
  angles(a, t, turn);
  if (tid == kAppendThreads - 1) dst = slot_offset(a, t);
  __syncthreads();
  const int64_t off = dst;
  float2 cs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) cs[i] = in && turned ? turn[sub * 4 + i] : make_float2(1.f, 0.f);
  while (true) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = row + i * a.splits * kRows;
      const bool live = r < H && in;
      const bool is_q = r < a.Hq, is_v = r >= a.Hq + a.Hkv;
      const int h = is_q ? r : is_v ? r - a.Hq - a.Hkv : r - a.Hq;
      Q oa = ra[i], ob = rb[i];
      float x[8];
      if (live) {
        unpack4<DT>(ra[i], x);
        unpack4<DT>(rb[i], x + 4);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
      }
      if constexpr (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (!is_v && (is_q ? a.q_w : a.k_w)) {
          const float g = 1.0f / sqrtf(ss / static_cast<float>(a.D) + a.eps);
          float w[8];
          unpack4<DT>(is_q ? wq[0] : wk[0], w);
          unpack4<DT>(is_q ? wq[1] : wk[1], w + 4);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= g * w[e];
        }
      }
      if (!live) continue;
      if (!is_v) {
        float y[8];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int i0 = TRAD ? 2 * p : p, i1 = TRAD ? 2 * p + 1 : p + 4;
          y[i0] = x[i0] * cs[p].x - x[i1] * cs[p].y;
          y[i1] = x[i1] * cs[p].x + x[i0] * cs[p].y;
        }
        if (!turned) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = x[e];
        }
        oa = pack4<DT>(y);
        ob = pack4<DT>(y + 4);
      }
      T* to = nullptr;
      if (is_q) {
        to = static_cast<T*>(a.q_out) + t * a.qo_st + h * a.qo_sh;
      } else {
        if (!is_v && a.k_out) {
          T* ko = static_cast<T*>(a.k_out) + (t * a.Hkv + h) * a.D;
          *reinterpret_cast<Q*>(ko + pa) = oa;
          *reinterpret_cast<Q*>(ko + pb) = ob;
        }
        if (off >= 0) to = static_cast<T*>(is_v ? a.v_cache : a.k_cache) + off + h * a.head_stride;
      }
      if (to) {
        *reinterpret_cast<Q*>(to + pa) = oa;
        *reinterpret_cast<Q*>(to + pb) = ob;
      }
    }
    row += ROWS * a.splits * kRows;
    if (__all_sync(0xffffffffu, row >= H)) break;
    load();
  }
}

// `dims` not a multiple of 8: a lane's values rotate with others anywhere in
// the row, fetched one by one. Such heads are rare and small.
template <int DT, int LPR, bool TRAD>
__global__ void __launch_bounds__(kAppendThreads) append_any_kernel(const AppendArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int kRows = kAppendThreads / LPR;
  __shared__ float2 turn[128];
  __shared__ int64_t dst;
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x;
  const int64_t t = blockIdx.x / a.splits;
  const int part = blockIdx.x % a.splits;
  const int half = a.dims >> 1;
  angles(a, t, turn);
  if (tid == kAppendThreads - 1) dst = slot_offset(a, t);
  __syncthreads();
  const int64_t off = dst;
  const int sub = tid % LPR, e0 = sub * 8;
  const bool in = e0 < a.D;
  const int H = a.Hq + 2 * a.Hkv;
  for (int row = part * kRows + tid / LPR; ; row += a.splits * kRows) {
    // a warp's rows run out together or not at all as far as the shuffles are concerned
    const bool live = row < H;
    if (!__any_sync(0xffffffffu, live)) break;
    const bool is_q = row < a.Hq, is_v = row >= a.Hq + a.Hkv;
    const int h = is_q ? row : is_v ? row - a.Hq - a.Hkv : row - a.Hq;
    const T* src = is_q ? static_cast<const T*>(a.q) + t * a.q_st + h * a.q_sh
                 : is_v ? static_cast<const T*>(a.v) + t * a.v_st + h * a.v_sh
                        : static_cast<const T*>(a.k) + t * a.k_st + h * a.k_sh;
    float x[8], y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
    if (live && in) load8<DT>(src + e0, x);
    // the other value of each rotated pair: inside the lane for adjacent pairs, half a rotation away otherwise
    if constexpr (!TRAD) {
      if (live && !is_v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = e0 + i;
          if (e < a.dims) y[i] = Elem<DT>::to_f(src[e < half ? e + half : e - half]);
        }
      }
    }
    const T* w = static_cast<const T*>(is_q ? a.q_w : a.k_w);
    if (a.q_w != nullptr || a.k_w != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (live && in && !is_v && w != nullptr) {
        const float r = 1.0f / sqrtf(ss / static_cast<float>(a.D) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = e0 + i;
          x[i] *= r * Elem<DT>::to_f(w[e]);
          if (!TRAD && e < a.dims) y[i] *= r * Elem<DT>::to_f(w[e < half ? e + half : e - half]);
        }
      }
    }
    __syncwarp();  // every lane's loads of the row come before any store to it (q_out may be q)
    if (!live || !in) continue;
    if (!is_v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (TRAD) {
          if ((i & 1) == 0 && e0 + i < a.dims) {
            const float2 cs = turn[(e0 + i) >> 1];
            const float u = x[i], v = x[i + 1];
            x[i] = u * cs.x - v * cs.y;
            x[i + 1] = v * cs.x + u * cs.y;
          }
        } else {
          const int e = e0 + i;
          if (e < half) {
            const float2 cs = turn[e];
            x[i] = x[i] * cs.x - y[i] * cs.y;
          } else if (e < a.dims) {
            const float2 cs = turn[e - half];
            x[i] = x[i] * cs.x + y[i] * cs.y;
          }
        }
      }
    }
    if (is_q) {
      store8<DT>(static_cast<T*>(a.q_out) + t * a.qo_st + h * a.qo_sh + e0, x);
    } else {
      if (!is_v && a.k_out) store8<DT>(static_cast<T*>(a.k_out) + (t * a.Hkv + h) * a.D + e0, x);
      if (off >= 0) store8<DT>(static_cast<T*>(is_v ? a.v_cache : a.k_cache) + off + h * a.head_stride + e0, x);
    }
  }
}

}  // namespace
}  // namespace mt

using namespace mt;

extern "C" {

int mt_paged_plan(const int32_t* ctx_lens, const int32_t* new_lens, int64_t B, int32_t* block_table,
                  int64_t table_stride, int64_t max_pages, const int32_t* free_pages, int64_t n_free,
                  const int32_t* free_head, int64_t page_size, int64_t token_cap, int32_t* seq_lens,
                  int32_t* query_start, int32_t* positions, int32_t* token_seq, int64_t* slots, int32_t* counts,
                  mt_stream_t stream) {
  clear_error();
  MT_CHECK_ARG(B >= 0 && B < (1ll << 30) && token_cap >= 0 && token_cap < (1ll << 31) - 1,
               "mt_paged_plan: B=%lld token_cap=%lld", (long long)B, (long long)token_cap);
  MT_CHECK_ARG(page_size > 0 && page_size <= (1 << 20), "mt_paged_plan: page_size %lld outside 1..2^20",
               (long long)page_size);
  MT_CHECK_ARG(max_pages >= 0 && max_pages < (1ll << 31) && table_stride >= max_pages,
               "mt_paged_plan: max_pages=%lld does not fit the table's row stride %lld", (long long)max_pages,
               (long long)table_stride);
  MT_CHECK_ARG(n_free >= 0 && n_free < (1ll << 31) - 1, "mt_paged_plan: n_free=%lld", (long long)n_free);
  MT_CHECK_ARG(query_start && counts && (B == 0 || (ctx_lens && new_lens && seq_lens)) &&
                   (B == 0 || max_pages == 0 || block_table) && (n_free == 0 || free_pages) &&
                   (token_cap == 0 || (positions && token_seq && slots)),
               "mt_paged_plan: null pointer");
  int sms = 148;
  if (int rc = device_sm_count(&sms)) return rc;
  const PlanArgs a = {ctx_lens, new_lens, B, block_table, table_stride, max_pages, free_pages, free_head, n_free,
                      (int)page_size, token_cap, seq_lens, query_start, positions, token_seq, slots, counts};
  const size_t smem = 3 * sizeof(int) * kPlanChunk;
  if (int rc = ensure_smem(plan_kernel, smem)) return rc;
  const int64_t want = (token_cap + kPlanThreads - 1) / kPlanThreads;
  const int64_t grid = want < 1 ? 1 : want < sms ? want : sms;
  return launch(plan_kernel, dim3((unsigned)grid), dim3(kPlanThreads), smem, (cudaStream_t)stream, a);
}

int mt_rope_paged_append(const void* q, const void* k, const void* v, int64_t q_st, int64_t q_sh, int64_t k_st,
                         int64_t k_sh, int64_t v_st, int64_t v_sh, const void* q_norm_w, const void* k_norm_w,
                         float eps, const int32_t* positions, const int64_t* slots, const float* inv_freq, int dims,
                         int traditional, float mscale, void* q_out, int64_t qo_st, int64_t qo_sh, void* k_out,
                         void* k_cache, void* v_cache, int64_t num_pages, int64_t page_size, int64_t page_stride,
                         int64_t head_stride, int64_t slot_stride, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                         int dtype, mt_stream_t stream) {
  clear_error();
  MT_CHECK_ARG(T >= 0 && T < (1ll << 24) && Hq >= 0 && Hkv > 0 && Hq < 4096 && Hkv < 4096,
               "mt_rope_paged_append: T=%lld Hq=%lld Hkv=%lld", (long long)T, (long long)Hq, (long long)Hkv);
  MT_CHECK_ARG(D > 0 && D <= 256 && D % 8 == 0, "mt_rope_paged_append: head_dim %lld must be a multiple of 8 up to 256",
               (long long)D);
  MT_CHECK_ARG(dims >= 0 && dims <= D && dims % 2 == 0, "mt_rope_paged_append: dims=%d must be even, within 0..%lld",
               dims, (long long)D);
  MT_CHECK_ARG(num_pages >= 0 && page_size > 0 && page_size <= (1 << 20),
               "mt_rope_paged_append: num_pages=%lld page_size=%lld", (long long)num_pages, (long long)page_size);
  if (dtype != MT_BF16 && dtype != MT_F16 && dtype != MT_F32) {
    set_error("mt_rope_paged_append: unsupported dtype %d", dtype);
    return MT_ERR_UNSUPPORTED;
  }
  if (T == 0) return MT_OK;
  MT_CHECK_ARG((Hq == 0 || (q && q_out)) && k && v && positions && slots && (dims == 0 || inv_freq) &&
                   (num_pages == 0 || (k_cache && v_cache)),
               "mt_rope_paged_append: null pointer");
  MT_CHECK_ARG(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_out, 16) && aligned(k_out, 16) &&
                   aligned(k_cache, 16) && aligned(v_cache, 16) &&
                   (q_st | q_sh | k_st | k_sh | v_st | v_sh | qo_st | qo_sh | page_stride | head_stride | slot_stride) % 8 == 0,
               "mt_rope_paged_append: rows must be 16-byte aligned, strides multiples of 8 elements");
  AppendArgs a = {q, k, v, q_st, q_sh, k_st, k_sh, v_st, v_sh, q_norm_w, k_norm_w, eps, mscale, positions, slots,
                  inv_freq, dims, q_out, qo_st, qo_sh, k_out, k_cache, v_cache, num_pages, page_stride, head_stride,
                  slot_stride, (int)page_size, (int)Hq, (int)Hkv, (int)D, 1};
  const int lpr = D <= 64 ? 8 : D <= 128 ? 16 : 32;
  int sms = 148;
  if (int rc = device_sm_count(&sms)) return rc;
  const int64_t parts = (Hq + 2 * Hkv + kAppendThreads / lpr - 1) / (kAppendThreads / lpr);
  if (T < sms * 4) a.splits = (int)parts;
  const dim3 grid(static_cast<unsigned>(T * a.splits));
  auto run = [&](auto kern) { return launch(kern, grid, dim3(kAppendThreads), 0, (cudaStream_t)stream, a); };
  const bool norm = q_norm_w != nullptr || k_norm_w != nullptr;
// one row per lane group where the rows are spread over CTAs, else three under way at once
#define MT_APPEND_K(DT, L, TR, N) (a.splits > 1 ? run(append_kernel<DT, L, TR, N, 1>) : run(append_kernel<DT, L, TR, N, AP_ROWS>))
#define MT_APPEND_L(DT, L)                                                                                      \
  (dims % 8 != 0 ? (traditional ? run(append_any_kernel<DT, L, true>) : run(append_any_kernel<DT, L, false>))   \
   : traditional ? (norm ? MT_APPEND_K(DT, L, true, true) : MT_APPEND_K(DT, L, true, false))                    \
                 : (norm ? MT_APPEND_K(DT, L, false, true) : MT_APPEND_K(DT, L, false, false)))
#define MT_APPEND(DT) (lpr == 8 ? MT_APPEND_L(DT, 8) : lpr == 16 ? MT_APPEND_L(DT, 16) : MT_APPEND_L(DT, 32))
  return dtype == MT_BF16 ? MT_APPEND(MT_BF16) : dtype == MT_F16 ? MT_APPEND(MT_F16) : MT_APPEND(MT_F32);
#undef MT_APPEND_K
#undef MT_APPEND_L
#undef MT_APPEND
}

}  // extern "C"
