// Paged serving, per step and per layer: the step's plan (block tables, slots
// and positions from request lengths) and the q/k prologue that rotates each
// row at its own position and writes k and v to their slots of the cache.
#include "paged_common.cuh"

namespace mt {
namespace {

// ------------------------------------------------------------------ step plan
// Two prefix sums over the requests decide everything: new tokens (where each
// request's rows start) and new pages (which free pages it gets). Both are
// sums of non-negative numbers that saturate at INT32_MAX, so adding in any
// grouping gives the same result and nothing overflows, whatever the lengths.
constexpr int kPlanMax = 0x7fffffff;

__device__ __forceinline__ int sat_add(int a, int b) {
  const uint32_t s = static_cast<uint32_t>(a) + static_cast<uint32_t>(b);
  return s > static_cast<uint32_t>(kPlanMax) ? kPlanMax : static_cast<int>(s);
}

struct PlanScan {
  int warp_sum[32];
};

// Inclusive saturating scan of `own` over the block, plus `carry`; returns the
// exclusive prefix of this thread and the block's total through `total`.
template <int kThreads>
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
  int w = lane < kThreads / 32 ? sm.warp_sum[lane] : 0;
#pragma unroll
  for (int o = 1; o < kThreads / 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w = sat_add(w, u);
  }
  const int prev = warp > 0 ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
  total = sat_add(carry, __shfl_sync(0xffffffffu, w, kThreads / 32 - 1));
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
  FastDiv page;
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
// reads a table entry that another one writes. Latency bounds it: lengths,
// scans, then a table or free-list entry for each token. 8 requests 3.6 us
// (6.8 with 64-bit divisions), 4096 requests with 131072 token places 9.0 us
// (9.2 with 512 threads of eight requests, 9.8 while those met in shared-memory
// banks), where the 2.2 MB it moves would take 0.3.
template <int kThreads, int kItems>
__global__ void __launch_bounds__(kThreads) plan_kernel(const PlanArgs a) {
  constexpr int kPlanChunk = kThreads * kItems;
  // a place in kItems is left out, so that threads with so many requests each do not meet in a bank
  auto pad = [](int r) { return kItems == 1 ? r : r + r / kItems; };
  extern __shared__ int plan_smem[];
  int* tok_end = plan_smem;                  // inclusive sums of new tokens
  int* page_end = tok_end + pad(kPlanChunk);  // inclusive sums of new pages
  int* ctx_of = page_end + pad(kPlanChunk);       // cached tokens; ~cached where the request is refused
  __shared__ PlanScan scan;
  __shared__ int red[3];
  griddep_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ps = a.page.d;
  const int n_free = static_cast<int>(a.n_free);
  int head = a.free_head ? *a.free_head : 0;
  head = head < 0 ? 0 : head > n_free ? n_free : head;
  const int avail = n_free - head;
  const int64_t room = a.max_pages * ps < kPlanMax ? a.max_pages * ps : kPlanMax;
  if (tid < 3) red[tid] = 0;
  if (a.B == 0) __syncthreads();  // no scan below whose barriers would order it before the sums
  const bool vec = ((reinterpret_cast<uintptr_t>(a.ctx) | reinterpret_cast<uintptr_t>(a.fresh)) & 15) == 0;
  auto pages_of = [&](int len) { return len > 0 ? a.page.div(len - 1) + 1 : 0; };
  int tok_base = 0, page_base = 0, refused = 0, taken = 0;
  for (int64_t r0 = 0; r0 < a.B; r0 += kPlanChunk) {
    const int n = static_cast<int>(a.B - r0 < kPlanChunk ? a.B - r0 : kPlanChunk);
    const int top_bit = 1 << (31 - __clz(n));
    alignas(16) int ctx[kItems], fresh[kItems];
    int need[kItems];
    int own = 0;
    if (kItems % 4 == 0 && vec && tid * kItems + kItems <= n) {
#pragma unroll
      for (int i = 0; i + 3 < kItems; i += 4) {
        *reinterpret_cast<int4*>(ctx + i) = *reinterpret_cast<const int4*>(a.ctx + r0 + tid * kItems + i);
        *reinterpret_cast<int4*>(fresh + i) = *reinterpret_cast<const int4*>(a.fresh + r0 + tid * kItems + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int r = tid * kItems + i;
        ctx[i] = r < n ? a.ctx[r0 + r] : 0;
        fresh[i] = r < n ? a.fresh[r0 + r] : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      ctx[i] = max(ctx[i], 0);
      fresh[i] = max(fresh[i], 0);
      own = sat_add(own, fresh[i]);
    }
    int tok_total, page_total;
    int t = plan_scan<kThreads>(own, tok_base, scan, tok_total);
    own = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int r = tid * kItems + i;
      need[i] = -1;
      if (r >= n) continue;
      t = sat_add(t, fresh[i]);
      const int64_t total = static_cast<int64_t>(ctx[i]) + fresh[i];
      if (t <= a.cap && total <= room) need[i] = pages_of(static_cast<int>(total)) - pages_of(ctx[i]);
      own = sat_add(own, max(need[i], 0));
      tok_end[pad(r)] = t;
    }
    int p = plan_scan<kThreads>(own, page_base, scan, page_total);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int r = tid * kItems + i;
      p = sat_add(p, max(need[i], 0));
      const bool ok = need[i] == 0 || (need[i] > 0 && p <= avail);
      if (r < n) {
        page_end[pad(r)] = p;
        ctx_of[pad(r)] = ok ? ctx[i] : ~ctx[i];
        refused += !ok;
        if (ok && need[i] > 0) taken = p;
        if (warp % gridDim.x == blockIdx.x) {
          a.seq_lens[r0 + r] = ok ? ctx[i] + fresh[i] : ctx[i];
          a.query_start[r0 + r + 1] = tok_end[pad(r)];
        }
      }
    }
    __syncthreads();
    // new pages of this chunk's admitted requests
    const int page_last = min(page_total, avail);
    for (int64_t e = page_base + static_cast<int64_t>(blockIdx.x) * kThreads + tid; e < page_last;
         e += static_cast<int64_t>(gridDim.x) * kThreads) {
      int lo = 0, hi = n - 1;  // first request with page_end > e
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (page_end[pad(mid)] > e) hi = mid; else lo = mid + 1;
      }
      const int c = ctx_of[pad(lo)];
      if (c < 0) continue;
      const int first = lo > 0 ? page_end[pad(lo - 1)] : page_base;
      const int had = pages_of(c);
      a.table[(r0 + lo) * a.table_stride + had + (e - first)] = a.free_pages[head + e];
    }
    // tokens of this chunk, two of a thread's at a time so that their searches and loads overlap
    const int64_t tok_last = tok_total < a.cap ? tok_total : a.cap;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t k0 = tok_base + static_cast<int64_t>(blockIdx.x) * kThreads + tid; k0 < tok_last; k0 += 2 * stride) {
      int at[2] = {0, 0}, block[2], page[2];
      int64_t pos[2];
#pragma unroll 1
      for (int w = top_bit; w > 0; w >>= 1)  // requests that end at the token or before it
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (at[i] + w <= n && tok_end[pad(at[i] + w - 1)] <= k0 + i * stride) at[i] += w;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t k = k0 + i * stride;
        page[i] = -1;
        if (k >= tok_last) continue;
        const int lo = at[i], c0 = ctx_of[pad(lo)], c = c0 < 0 ? ~c0 : c0;
        pos[i] = static_cast<int64_t>(c) + (k - (lo > 0 ? tok_end[pad(lo - 1)] : tok_base));
        if (c0 >= 0) {
          block[i] = a.page.div(static_cast<int>(pos[i]));  // an admitted request ends below 2^31
          const int had = pages_of(c), first = lo > 0 ? page_end[pad(lo - 1)] : page_base;
          page[i] = block[i] < had ? a.table[(r0 + lo) * a.table_stride + block[i]]
                                   : a.free_pages[head + first + (block[i] - had)];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t k = k0 + i * stride;
        if (k >= tok_last) continue;
        a.positions[k] = static_cast<int>(pos[i] < kPlanMax ? pos[i] : kPlanMax);
        a.token_seq[k] = static_cast<int>(r0 + at[i]);
        a.slots[k] = page[i] >= 0 ? static_cast<int64_t>(page[i]) * ps + (static_cast<int>(pos[i]) - block[i] * ps) : -1;
      }
    }
    tok_base = tok_total;
    page_base = page_total;
    __syncthreads();  // the prefixes are overwritten by the next chunk
  }
  griddep_launch();  // not at the top: the next kernel's CTAs beside these cost 1.7 us of 11.6 in a stream
  for (int64_t k = tok_base + static_cast<int64_t>(blockIdx.x) * kThreads + tid; k < a.cap;
       k += static_cast<int64_t>(gridDim.x) * kThreads) {
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
  int splits;  // items per token
  int64_t T;
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

// Three rows to a group of lanes, two stages, 5 CTAs of 128 threads per SM (91 registers, 24 KB of ring each): 8192
// tokens of 32/8 heads of 128 with norms in 36.7 us = 5.5 TB/s, 84% of the copy rate, in replays of a graph (38.4 to 40.1
// call after call). 6 CTAs, or a third stage, 38.6 to 38.9; 4 with three stages 38.3.
constexpr int kAppendRows = 3;
constexpr int kAppendStages = 2;
constexpr int kAppendCtas = 5;
constexpr int kAppendThreads = 128;

// cos and sin (times mscale) of one angle. The angle is reduced to a fraction
// of a turn in double, so a position of 2^30 rotates as exactly as position 1.
__device__ __forceinline__ float2 cos_sin(int pos, float inv_freq, float mscale) {
  const double turns = static_cast<double>(pos) * static_cast<double>(inv_freq) * 0.15915494309189533577;
  float s, c;
  sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
  return make_float2(c * mscale, s * mscale);
}

// offset of the token's cache row (without the head), -1 where it has none
__device__ __forceinline__ int64_t slot_offset(const AppendArgs& a, int64_t slot) {
  if (slot < 0) return -1;
  const int64_t page = slot < (1ll << 31) ? static_cast<int64_t>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.page_size))
                                           : slot / a.page_size;
  if (page < a.num_pages) return page * a.page_stride + (slot - page * a.page_size) * a.slot_stride;
  report_status(0x701);
  return -1;
}

// the 16 bytes of a piece of a row as pairs of fp32, and back with one rounding
template <int DT>
__device__ __forceinline__ void unpack(const uint4& u, float2* x) {
  if constexpr (DT == MT_F32) {
    x[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    x[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  } else {
    const typename Elem<DT>::T2* e = reinterpret_cast<const typename Elem<DT>::T2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = Elem<DT>::unpack2(e[i]);
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack(const float2* x) {
  uint4 u;
  if constexpr (DT == MT_F32) {
    u = make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x), __float_as_uint(x[1].y));
  } else {
    typename Elem<DT>::T2* e = reinterpret_cast<typename Elem<DT>::T2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = Elem<DT>::pack2(x[i].x, x[i].y);
  }
  return u;
}

// An item is a token's rows, or as many of them as a CTA takes at a time: ROWS
// to each group of LPR lanes. A lane holds two 16-byte pieces of a row whose
// values rotate with each other: (j, j + dims/2), or adjacent ones; past
// `dims`, two that are copied. No value crosses lanes but the norm's sum, and a
// thread reads back only what it copied to shared memory itself: the rows of
// the next STAGES - 1 items are always under way and need no barrier. The
// angles of the next item are worked out, one by a thread, while this one's
// rows arrive; one barrier per item hands them over. What limited it was
// instructions (0.48 a cycle, 724 for a warp's three rows: 72 us for the prompt
// above) and then shared memory (75% busy with the angles read for each row,
// 39.6 us): so two fp32 values to an instruction, a row's addresses and the
// weights out of shared memory, the angles in registers for all rows. Norm and
// rotation in fp32, rounded once.
template <int DT, int LPR, bool TRAD, int ROWS, int STAGES>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) append_kernel(const AppendArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int P = 16 / sizeof(T);  // values to a piece
  constexpr int kRows = kAppendThreads / LPR, kGroup = ROWS * kRows;
  struct Row {
    const T* src;  // token 0's row, and the way from token to token
    int64_t st;
    T* to;     // where it goes, but for the token's offset in q_out or its slot's in the cache
    int kind;  // 0 q, 1 k, 2 v, -1 no row
    int head;
  };
  extern __shared__ __align__(16) uint8_t append_smem[];
  uint4(*ring)[ROWS][2][kAppendThreads] = reinterpret_cast<uint4(*)[ROWS][2][kAppendThreads]>(append_smem);
  __shared__ __align__(16) float cos_of[2][128], sin_of[2][128];
  __shared__ __align__(16) T weight[2][256];
  __shared__ __align__(16) Row rows[kGroup];
  __shared__ int64_t dst[2];
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x;
  const int half = a.dims >> 1, sub = tid % LPR;
  const bool in = sub * 2 * P < a.D, turned = sub * 2 * P < a.dims;
  // the lane's two pieces of a row
  const int pa = !in ? 0 : TRAD || !turned ? sub * 2 * P : sub * P;
  const int pb = !in ? 0 : TRAD || !turned ? sub * 2 * P + P : half + sub * P;
  // the grid is a multiple of `splits`: this CTA's part of the rows, its first token and the way to the next
  const int part = blockIdx.x % a.splits;
  const int64_t step = gridDim.x / a.splits;
  int64_t t = blockIdx.x / a.splits;
  // position and slot of the next token, for the threads that use them
  const bool has_angle = tid < half, has_slot = tid == kAppendThreads - 1;
  const float inv = has_angle ? a.inv_freq[tid] : 0.f;
  int pos = has_angle ? a.positions[t] : 0;
  int64_t slot = has_slot ? a.slots[t] : -1;
  const bool norm_q = a.q_w != nullptr, norm_k = a.k_w != nullptr;
  for (int i = tid; i < kGroup; i += kAppendThreads) {
    const int r = part * kGroup + i;
    Row w = {nullptr, 0, nullptr, -1, 0};
    if (r < a.Hq)
      w = {static_cast<const T*>(a.q) + r * a.q_sh, a.q_st, static_cast<T*>(a.q_out) + r * a.qo_sh, 0, r};
    else if (r < a.Hq + a.Hkv)
      w = {static_cast<const T*>(a.k) + (r - a.Hq) * a.k_sh, a.k_st,
           static_cast<T*>(a.k_cache) + (r - a.Hq) * a.head_stride, 1, r - a.Hq};
    else if (r < a.Hq + 2 * a.Hkv)
      w = {static_cast<const T*>(a.v) + (r - a.Hq - a.Hkv) * a.v_sh, a.v_st,
           static_cast<T*>(a.v_cache) + (r - a.Hq - a.Hkv) * a.head_stride, 2, r - a.Hq - a.Hkv};
    rows[i] = w;
  }
  for (int i = tid; i < a.D; i += kAppendThreads) {
    if (norm_q) weight[0][i] = static_cast<const T*>(a.q_w)[i];
    if (norm_k) weight[1][i] = static_cast<const T*>(a.k_w)[i];
  }
  __syncthreads();
  int64_t ahead = t;  // the token whose rows are fetched next
  auto issue = [&](int stage) {
    if (ahead < a.T && in) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const Row& w = rows[i * kRows + tid / LPR];
        if (w.src) {
          const T* src = w.src + ahead * w.st;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(&ring[stage][i][0][tid])), "l"(src + pa) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(&ring[stage][i][1][tid])), "l"(src + pb) : "memory");
        }
      }
    }
    ahead += step;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(s);
  const float inv_d = 1.0f / static_cast<float>(a.D);
  auto hand_over = [&](int buf, int64_t next) {  // the angles of the token that pos and slot are of; then the next one's
    if (has_angle) {
      const float2 cs = cos_sin(pos, inv, a.mscale);
      cos_of[buf][tid] = cs.x;
      sin_of[buf][tid] = cs.y;
    }
    if (has_slot) dst[buf] = slot_offset(a, slot);
    if (next < a.T) {
      if (has_angle) pos = a.positions[next];
      if (has_slot) slot = a.slots[next];
    }
  };
  hand_over(0, t + step);
  __syncthreads();
  int buf = 0, get = 0, put = STAGES - 1;
  for (; t < a.T; t += step) {
    issue(put);
    put = put + 1 == STAGES ? 0 : put + 1;
    if (t + step < a.T) hand_over(buf ^ 1, t + 2 * step);
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    const int64_t off = dst[buf], q_off = t * a.qo_st;
    float2 c[P / 2], s[P / 2], ns[P / 2];
    if (turned) {
#pragma unroll
      for (int e = 0; e < P / 2; ++e) {
        c[e] = reinterpret_cast<const float2*>(&cos_of[buf][sub * P])[e];
        s[e] = reinterpret_cast<const float2*>(&sin_of[buf][sub * P])[e];
        ns[e] = make_float2(-s[e].x, -s[e].y);
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const Row& w = rows[i * kRows + tid / LPR];
      const int kind = w.kind;
      uint4 oa = ring[get][i][0][tid], ob = ring[get][i][1][tid];  // (where there is no row, whatever is there)
      if (__any_sync(0xffffffffu, kind == 0 || kind == 1)) {
        float2 x[P / 2], y[P / 2];
        unpack<DT>(oa, x);
        unpack<DT>(ob, y);
        if (norm_q || norm_k) {
          float2 ss = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < P / 2; ++e) ss = fma2(y[e], y[e], fma2(x[e], x[e], ss));
          float sum = in ? ss.x + ss.y : 0.f;
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          if (kind == 1 ? norm_k : norm_q) {
            const float g = rsqrtf(fmaf(sum, inv_d, a.eps));
            const float2 gg = make_float2(g, g);
            const T* ws = weight[kind == 1];
            float2 wf[P / 2];
            unpack<DT>(*reinterpret_cast<const uint4*>(ws + pa), wf);
#pragma unroll
            for (int e = 0; e < P / 2; ++e) x[e] = mul2(x[e], mul2(wf[e], gg));
            unpack<DT>(*reinterpret_cast<const uint4*>(ws + pb), wf);
#pragma unroll
            for (int e = 0; e < P / 2; ++e) y[e] = mul2(y[e], mul2(wf[e], gg));
          }
        }
        if (turned) {
          if constexpr (TRAD) {  // pairs within a piece: angles 0.. of the lane in x, then in y
#pragma unroll
            for (int e = 0; e < P / 2; ++e) {
              const float2 c0 = c[e / 2], s0 = s[e / 2], c1 = c[(P / 2 + e) / 2], s1 = s[(P / 2 + e) / 2];
              const float cx = (e & 1) ? c0.y : c0.x, sx = (e & 1) ? s0.y : s0.x;
              const float cy = (e & 1) ? c1.y : c1.x, sy = (e & 1) ? s1.y : s1.x;
              x[e] = make_float2(x[e].x * cx - x[e].y * sx, x[e].y * cx + x[e].x * sx);
              y[e] = make_float2(y[e].x * cy - y[e].y * sy, y[e].y * cy + y[e].x * sy);
            }
          } else {
#pragma unroll
            for (int e = 0; e < P / 2; ++e) {
              const float2 u = x[e], v = y[e];
              x[e] = fma2(u, c[e], mul2(v, ns[e]));
              y[e] = fma2(v, c[e], mul2(u, s[e]));
            }
          }
        }
        if (kind < 2) {
          oa = pack<DT>(x);
          ob = pack<DT>(y);
        }
      }
      if (!in || kind < 0) continue;
      if (kind == 1 && a.k_out) {
        T* ko = static_cast<T*>(a.k_out) + (t * a.Hkv + w.head) * a.D;
        *reinterpret_cast<uint4*>(ko + pa) = oa;
        *reinterpret_cast<uint4*>(ko + pb) = ob;
      }
      if (kind == 0 || off >= 0) {
        T* d = w.to + (kind == 0 ? q_off : off);
        *reinterpret_cast<uint4*>(d + pa) = oa;
        *reinterpret_cast<uint4*>(d + pb) = ob;
      }
    }
    get = get + 1 == STAGES ? 0 : get + 1;
    buf ^= 1;
    __syncthreads();
  }
}

// `dims` or the head not in whole pieces: a lane's values rotate with others anywhere in
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
  if (tid < half) turn[tid] = cos_sin(a.positions[t], a.inv_freq[tid], a.mscale);
  if (tid == kAppendThreads - 1) dst = slot_offset(a, a.slots[t]);
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

// ------------------------------------------------------- arguments in memory
struct Span {
  const char* name;
  const void* p;
  int64_t bytes;
  bool meets(const Span& o) const {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(o.p);
    return bytes > 0 && o.bytes > 0 && a < b + o.bytes && b < a + bytes;
  }
};
struct TableSpan {  // rows with room between them, which is not theirs
  const void* p;
  int64_t rows, stride, bytes;
  bool meets(const Span& o) const {
    if (rows == 0 || bytes == 0 || o.bytes == 0) return false;
    const int64_t at = static_cast<int64_t>(reinterpret_cast<uintptr_t>(o.p) - reinterpret_cast<uintptr_t>(p));
    const int64_t end = at + o.bytes;
    if (at < 0) return end > 0;
    const int64_t row = at / stride;
    return row < rows && (at - row * stride < bytes || (row + 1 < rows && end > (row + 1) * stride));
  }
};

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
  // CTAs read the inputs while others write: no output may lie over an input, the table or another output
  {
    const Span in[] = {{"ctx_lens", ctx_lens, 4 * B}, {"new_lens", new_lens, 4 * B}, {"free_pages", free_pages, 4 * n_free},
                       {"free_head", free_head, free_head ? 4 : 0}};
    const Span out[] = {{"seq_lens", seq_lens, 4 * B},          {"query_start", query_start, 4 * (B + 1)},
                        {"positions", positions, 4 * token_cap}, {"token_seq", token_seq, 4 * token_cap},
                        {"slots", slots, 8 * token_cap},         {"counts", counts, 20}};
    const TableSpan table = {block_table, B, 4 * table_stride, 4 * max_pages};
    const char *one = nullptr, *other = nullptr;
    for (const Span& i : in)
      if (table.meets(i)) one = "block_table", other = i.name;
    for (int k = 0; k < 6; ++k) {
      if (table.meets(out[k])) one = out[k].name, other = "block_table";
      for (const Span& i : in)
        if (out[k].meets(i)) one = out[k].name, other = i.name;
      for (int l = 0; l < k; ++l)
        if (out[k].meets(out[l])) one = out[k].name, other = out[l].name;
    }
    MT_CHECK_ARG(one == nullptr, "mt_paged_plan: %s overlaps %s in memory (a step's outputs are the next one's inputs by a copy or a second set of buffers)",
                 one, other);
  }
  int sms = 148;
  if (int rc = device_sm_count(&sms)) return rc;
  const PlanArgs a = {ctx_lens, new_lens, B, block_table, table_stride, max_pages, free_pages, free_head, n_free,
                      FastDiv::of((int)page_size), token_cap, seq_lens, query_start, positions, token_seq, slots, counts};
  auto run = [&](auto kern, int threads, int items) -> int {
    const int64_t want = (token_cap + threads - 1) / threads;
    const int64_t grid = want < 1 ? 1 : want < sms ? want : sms;
    const size_t smem = 3 * sizeof(int) * (threads * items + threads);
    if (int rc = ensure_smem(kern, smem)) return rc;
    return launch(kern, dim3((unsigned)grid), dim3(threads), smem, (cudaStream_t)stream, a);
  };
  // one request to a thread where there are few, else four to each of 1024, 4096 scanned at a time
  return B <= 512 ? run(plan_kernel<512, 1>, 512, 1) : run(plan_kernel<1024, 4>, 1024, 4);
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
                  slot_stride, (int)page_size, (int)Hq, (int)Hkv, (int)D, 1, T};
  int sms = 148;
  if (int rc = device_sm_count(&sms)) return rc;
  const int64_t rows = Hq + 2 * Hkv;
  const int piece = dtype == MT_F32 ? 4 : 8;
  const bool pieces = dims % (2 * piece) == 0 && D % (2 * piece) == 0;
  int lpr = pieces && piece == 8 ? 4 : 8;  // lanes to a row: whole pairs of pieces, or eights
  while (lpr * (pieces ? 2 * piece : 8) < D) lpr *= 2;
  const int per_pass = kAppendThreads / lpr;
  // few tokens: one row to a group of lanes, spread over as many CTAs; else three to a group
  const bool few = T * ((rows + per_pass - 1) / per_pass) <= sms * kAppendCtas;
  const int per_cta = pieces ? per_pass * (few ? 1 : kAppendRows) : few ? per_pass : 1 << 20;
  a.splits = (int)((rows + per_cta - 1) / per_cta);
  int64_t grid = T * a.splits;
  auto run = [&](auto kern, size_t smem) -> int {
    if (int e = ensure_smem(kern, smem)) return e;
    return launch(kern, dim3((unsigned)grid), dim3(kAppendThreads), smem, (cudaStream_t)stream, a);
  };
  if (pieces && grid > sms * kAppendCtas) grid = sms * kAppendCtas < a.splits ? a.splits : sms * kAppendCtas / a.splits * a.splits;
#define MT_APPEND_K(DT, L, TR)                                                              \
  (few ? run(append_kernel<DT, L, TR, 1, 2>, sizeof(uint4) * 2 * kAppendThreads * 2)        \
       : run(append_kernel<DT, L, TR, kAppendRows, kAppendStages>, sizeof(uint4) * 2 * kAppendThreads * kAppendRows * kAppendStages))
#define MT_APPEND_L(DT, L) (traditional ? MT_APPEND_K(DT, L, true) : MT_APPEND_K(DT, L, false))
#define MT_APPEND_ANY(DT, L) (traditional ? run(append_any_kernel<DT, L, true>, 0) : run(append_any_kernel<DT, L, false>, 0))
#define MT_APPEND_16(DT)                                                                     \
  (!pieces ? (lpr == 8 ? MT_APPEND_ANY(DT, 8) : lpr == 16 ? MT_APPEND_ANY(DT, 16) : MT_APPEND_ANY(DT, 32)) \
           : lpr == 4 ? MT_APPEND_L(DT, 4) : lpr == 8 ? MT_APPEND_L(DT, 8) : MT_APPEND_L(DT, 16))
#define MT_APPEND_32(DT)                                                                     \
  (!pieces ? (lpr == 8 ? MT_APPEND_ANY(DT, 8) : lpr == 16 ? MT_APPEND_ANY(DT, 16) : MT_APPEND_ANY(DT, 32)) \
           : lpr <= 8 ? MT_APPEND_L(DT, 8) : lpr == 16 ? MT_APPEND_L(DT, 16) : MT_APPEND_L(DT, 32))
  return dtype == MT_BF16 ? MT_APPEND_16(MT_BF16) : dtype == MT_F16 ? MT_APPEND_16(MT_F16) : MT_APPEND_32(MT_F32);
#undef MT_APPEND_32
#undef MT_APPEND_16
#undef MT_APPEND_ANY
#undef MT_APPEND_L
#undef MT_APPEND_K
}

}  // extern "C"
