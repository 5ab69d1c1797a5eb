// Attention of one new token per request over a paged key-value cache.
#include <type_traits>

#include "mma_sync.cuh"
#include "mt_tma.h"
#include "paged_common.cuh"

namespace mt {
namespace {

template <int N> using Int = std::integral_constant<int, N>;

struct PagedParams {
  const void* q;
  int64_t q_sb, q_sh;
  const void *kc, *vc;
  int64_t num_pages, page_stride, head_stride, slot_stride;
  FastDiv page;
  const int32_t* table;
  int64_t table_stride;
  int max_len;  // rows a table row can address (and the largest length used)
  const int32_t* lens;
  void* o;
  int64_t o_sb, o_sh;
  int B, Hkv, G, RB;  // RB: blocks of R query rows per kv head
  int box_rows;       // rows of a box of the copy engine
  float scale_log2;
  float* part;
  uint32_t* counters;
};

constexpr int kWarps = 4;                   // that compute; as many fetch, one for each
constexpr int kThreads = kWarps * 32;       // that compute
constexpr int kCtaThreads = 2 * kThreads;
// What a unit's beginning and end count as, in steps, when the work is cut (32/8 heads of 128, bf16): 64 requests of
// 64..8192 keys 85.6 us without, 80.3 with 1, 78.4 with 2 or 3; 256 of 1..512 40.8, 29.9, 28.4, 27.7; 37 of 0..1500
// with 20 heads of 64 17.8 with 2, 15.1 with 3 (and the next rule).
constexpr int kUnitCost = 3;
// The least run of a CTA, in places, where requests are that long. One request of 32/8 heads of 128 at least runs of 1, 3,
// 6 and 12: 129 keys 7.3, 7.0, 5.7 and 5.8 us (from 6 on a CTA to a head, no parts to join), 512 keys 7.5, 8.4, 9.8, 7.7;
// 1024 7.8, 8.9, 11.4, 11.4; 4096 10.1, 10.5, 12.2, 17.4; 16384 17.7, 17.8, 17.8, 19.2; four of 4096 keys 16.7 up to 6,
// 18.5. So 6 serves requests of a step or two, decides those up to some 13000 keys, and costs single ones of 512 to 4096
// 2 to 3.5 us.
constexpr int kLeastRun = 6;
// Warps work by themselves where a request has fewer places than this on average (of 16 keys), and runs are at least so
// long: 256 requests of 1..512 keys 28.5 us, 34.2 by CTAs; 32 of 1024 33.6, 29.6 by CTAs.
constexpr int kSoloMean = 24, kSoloRun = 4;
// The largest probability as a power of 2 where they are rounded to f16, whose normal numbers end at 2^-14: with 1 as the
// largest, a key 10 nats below it lost bits and one 18 below vanished from the output but not from the sum. So they are
// whole down to 2^-29 of the largest (20 nats) and 2^-40 of it off at most. Sum, output and a request's parts are in
// these units, which cancel at the end. (bf16 has fp32's exponents.)
constexpr float kTopF16 = 15.f;
constexpr int kMaxCtas = 296;  // bounds the workspace; 2 CTAs on each of 148 SMs
// arrival counters, one per warp of the grid, in the workspace's control words (the quantised matmul's: both leave
// them zero, and the workspace is used by one kernel at a time)
constexpr size_t kWsPagedCtl = kWsQmmDone;
static_assert(kWsPagedCtl + 4 * kMaxCtas * kWarps <= kWsCtlBytes, "the counters are control words");

// Byte offset of a 16-byte chunk of a staged row: 64-element halves of the KEYS
// rows one after another, each as the copy engine's 128-byte swizzle lays it out.
template <int KEYS>
__device__ __forceinline__ uint32_t swz(int row, int chunk) {
  return static_cast<uint32_t>((chunk >> 3) * (KEYS * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// a / b for non-negative numbers, by 32-bit division where they fit
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// Where a worker's copies stand in the flattened steps of (request, kv head x
// row block): KEYS keys of a warp that works by itself, four times as many of a
// CTA whose warps take KEYS each. A unit of nt steps takes nt + kUnitCost places in the order:
// its beginning and end cost as much as that many steps.
//
// The table's entries come in by windows of 32, a lane each, the next window
// (of this request or the one after it) while this one is used; the next
// request's length likewise.
struct Loader {
  int b, h, t, nt, len, next_len;
  int64_t left;  // places of this worker from here on
  int hk, rb;    // h's kv head and row block
  int base, win, ahead;        // first entry of the window, the lane's entry in it and in the next one
  int ahead_b, ahead_base;     // what the next one is of

  __device__ __forceinline__ void enter(const PagedParams& p, int keys) {
    nt = (len + keys - 1) / keys;
    next_len = b + 1 < p.B ? p.lens[b + 1] : 0;
  }
  __device__ __forceinline__ int entry(const PagedParams& p, int b_, int base_, int len_, int lane) const {
    const int i = base_ + lane;
    return i < (len_ > 0 ? p.page.div(len_ - 1) + 1 : 0) ? p.table[b_ * p.table_stride + i] : -1;
  }
  // fetch the window that follows (b, base): the request's next entries, else its first ones for its next head, else
  // the next request's first ones
  __device__ __forceinline__ void look_ahead(const PagedParams& p, int heads, int lane) {
    ahead_b = b;
    ahead_base = base + 32;
    int len_ = len;
    if (ahead_base > p.page.div(len - 1)) {
      ahead_base = 0;
      if (h + 1 >= heads) {
        ahead_b = b + 1;
        len_ = min(max(next_len, 0), p.max_len);
      }
    }
    ahead = ahead_b == b && ahead_base == base ? win : entry(p, ahead_b, ahead_base, len_, lane);
  }
  // the page of this lane's key (lane modulo KEYS) of the step at key0
  template <int KEYS>
  __device__ __forceinline__ int page_of(const PagedParams& p, int key0, int heads, int lane) {
    const int i0 = p.page.div(min(key0, len - 1));
    if (ahead_b == b && ahead_base == (i0 & ~31) && base != ahead_base) {
      win = ahead;
      base = ahead_base;
      look_ahead(p, heads, lane);
    } else if (base != (i0 & ~31)) {  // further on than the next window (pages of a few rows), or a request skipped
      base = i0 & ~31;
      win = entry(p, b, base, len, lane);
      look_ahead(p, heads, lane);
    }
    const int key = key0 + (lane & (KEYS - 1));
    const int i = p.page.div(min(key, len - 1)) - base;
    int page = __shfl_sync(0xffffffffu, win, i & 31);
    if (__any_sync(0xffffffffu, i >= 32)) {  // (only then wait for the next window)
      const int next = __shfl_sync(0xffffffffu, ahead, i & 31);
      if (i >= 32) page = ahead_b == b && ahead_base == base + 32 ? next : p.table[b * p.table_stride + base + i];
    }
    return key < len ? page : -1;
  }
  // to the next step that there is; true if it is of another request
  __device__ __forceinline__ bool advance(const PagedParams& p, int heads, int keys) {
    --left;
    if (++t < nt) return false;
    left -= kUnitCost;
    t = 0;
    if (++rb == p.RB) {
      rb = 0;
      ++hk;
    }
    if (++h < heads) return false;
    h = hk = rb = 0;
    if (left <= 0) return false;
    do {
      ++b;
      len = min(max(next_len, 0), p.max_len);
      enter(p, keys);
    } while (nt == 0);
    return true;
  }
};

// Keys and values are read once in a step and again only in the next one, after
// all other layers': first to be evicted (32 requests of 1024 keys 29.8 -> 27.5
// us, 256 of 1..512 27.8 -> 26.6), unless other rows of the head read them too.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(smem_addr(dst)),
      "l"(map), "r"(smem_addr(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy)
      : "memory");
}
__device__ __forceinline__ uint64_t l2_evict_normal() {
  uint64_t pol;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(pol));
  return pol;
}

// The step's KEYS rows of K and V into stage memory, completing on `bar`. Rows
// without a key (past the length, or on a page id outside the cache) stay out
// of the mask. BOX: the copy engine fetches boxes of 8, 16 or 32 rows that lie
// in one page (the page size is a multiple of that), 128 bytes of each row.
// Otherwise 16-byte asynchronous copies, each row from where its page is.
template <int D, int KEYS, bool BOX>
__device__ __forceinline__ void load_step(const PagedParams& p, const CUtensorMap* kmap, const CUtensorMap* vmap,
                                          const Loader& c, int page, int key0, int lane, uint8_t* stage,
                                          uint32_t* mask, uint64_t* bar, uint64_t policy) {
  const int key = key0 + (lane & (KEYS - 1));
  const bool there = static_cast<uint32_t>(page) < static_cast<uint32_t>(p.num_pages);
  if (key < c.len && !there) report_status(0x702);
  const uint32_t m = __ballot_sync(0xffffffffu, key < c.len && there) & (KEYS == 32 ? ~0u : 0xffffu);
  if (lane == 0) *mask = m;
  if constexpr (BOX) {
    int pages[KEYS / 8];
    uint32_t boxes = 0;
#pragma unroll
    for (int g = 0; g < KEYS / 8; ++g) {
      pages[g] = __shfl_sync(0xffffffffu, page, 8 * g);
      boxes += (8 * g & (p.box_rows - 1)) == 0 && (m >> (8 * g)) & 1;
    }
    if (lane == 0) {
      mbar_arrive_expect_tx(bar, boxes * p.box_rows * D * 4);
#pragma unroll
      for (int g = 0; g < KEYS / 8; ++g) {
        if ((8 * g & (p.box_rows - 1)) != 0 || !((m >> (8 * g)) & 1)) continue;
        const int first = key0 + 8 * g, slot = first - p.page.div(first) * p.page.d;
#pragma unroll
        for (int half = 0; half < D / 64; ++half) {
          uint8_t* dst = stage + half * KEYS * 128 + g * 1024;
          tma_load_4d(dst, kmap, bar, half * 64, slot, c.hk, pages[g], policy);
          tma_load_4d(dst + KEYS * D * 2, vmap, bar, half * 64, slot, c.hk, pages[g], policy);
        }
      }
    }
  } else {
    constexpr int CPR = D / 8;     // 16-byte chunks per row
    constexpr int RPI = 32 / CPR;  // rows per instruction
    const int chunk = lane % CPR;
    int64_t off = 0;
    if ((m >> (lane & (KEYS - 1))) & 1)
      off = page * p.page_stride + (key - p.page.div(key) * p.page.d) * p.slot_stride + c.hk * p.head_stride;
#pragma unroll
    for (int i = 0; i < KEYS / RPI; ++i) {
      const int row = i * RPI + lane / CPR;
      const int64_t src = __shfl_sync(0xffffffffu, off, row) + chunk * 8;
      if ((m >> row) & 1) {
        const uint32_t at = swz<KEYS>(row, chunk);
        cp_async16(stage + at, static_cast<const uint16_t*>(p.kc) + src, true);
        cp_async16(stage + KEYS * D * 2 + at, static_cast<const uint16_t*>(p.vc) + src, true);
      }
    }
    // this lane's arrival when its copies have landed, and one that the mask's store comes before
    if (lane == 0) mbar_arrive(bar);
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
  }
}

// 8 x 8 matrix of 16-bit values transposed across the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

template <int D, int R, int KEYS, int kStages>
struct PagedSmem {
  static constexpr int kStageBytes = 2 * KEYS * D * 2;
  static constexpr int kOStride = D + 4;
  alignas(1024) uint8_t stage[kWarps][kStages][kStageBytes];
  uint64_t full[kWarps][kStages], empty[kWarps][kStages];
  float m[kWarps][R], l[kWarps][R];
  uint32_t mask[kWarps][kStages];
  int sum_solo[2 * kWarps], sum_group[2 * kWarps];
  int longest[2 * kWarps];
  int64_t at_step[kWarps];
  int at_b[kWarps];
  int flag, abort;
  // followed by the warps' accumulators while they are joined: [kWarps][rows][kOStride]
  static size_t bytes(int rows) { return 1024 + sizeof(PagedSmem) + sizeof(float) * kWarps * rows * kOStride; }
};

// Joins the parts c0..c1 of a unit (in key order: the result does not depend on
// who joins) and writes its output rows. `threads` threads, this one `id`, each
// with the loads of ROWS rows of BATCH parts under way at once.
template <int DT, int D, int R, int ROWS, int BATCH>
__device__ __forceinline__ void join_parts(const PagedParams& p, int64_t c0, int64_t c1, int rows, typename Elem<DT>::T* ob,
                                           int id, int threads) {
  constexpr int kPart = R * (D + 2);
  const int apart = threads / (D / 4);  // rows side by side
  const int d = (id % (D / 4)) * 4;
  for (int r0 = id / (D / 4); r0 < rows; r0 += apart * ROWS) {
    float M[ROWS], L[ROWS], x[ROWS][4];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      M[j] = -INFINITY;
      L[j] = x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
    }
    // the unit begins in c0's second slot and goes on in the first slots of those after it
    for (int64_t c = c0; c <= c1; c += BATCH) {
      float m[ROWS][BATCH], l[ROWS][BATCH];
      float4 v[ROWS][BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int64_t at = c + k;
        const float* q = p.part + (at * 2 + (at == c0)) * kPart;
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          const int r = min(r0 + j * apart, rows - 1);
          m[j][k] = -INFINITY;
          l[j][k] = 0.f;
          v[j][k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (at > c1) continue;
          m[j][k] = __ldcg(q + r);
          l[j][k] = __ldcg(q + R + r);
          v[j][k] = __ldcg(reinterpret_cast<const float4*>(q + 2 * R + r * D + d));
        }
      }
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        float nm = M[j];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) nm = fmaxf(nm, m[j][k]);
        // parts whose maximum is -inf count 0 times what they hold, not nothing: NaN scores leave no maximum but a NaN sum
        const float ref = nm == -INFINITY ? 0.f : nm, f0 = exp2_approx(M[j] - ref);
        L[j] *= f0;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] *= f0;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const float f = exp2_approx(m[j][k] - ref);
          L[j] = fmaf(f, l[j][k], L[j]);
          x[j][0] = fmaf(f, v[j][k].x, x[j][0]);
          x[j][1] = fmaf(f, v[j][k].y, x[j][1]);
          x[j][2] = fmaf(f, v[j][k].z, x[j][2]);
          x[j][3] = fmaf(f, v[j][k].w, x[j][3]);
        }
        M[j] = nm;
      }
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int r = r0 + j * apart;
      if (r >= rows) continue;
      const float inv = L[j] > 0.f ? 1.f / L[j] : L[j];  // a row that saw no key is zero; NaN stays NaN
      uint2 u;
      u.x = pack2<DT>(x[j][0] * inv, x[j][1] * inv);
      u.y = pack2<DT>(x[j][2] * inv, x[j][3] * inv);
      *reinterpret_cast<uint2*>(ob + r * p.o_sh + d) = u;
    }
  }
}

// The flattened steps of all requests and kv heads are cut into equal runs, one
// per worker, whatever the lengths are; a run starts and ends anywhere inside a
// request. A worker is a warp, where runs are long enough and no request spans
// many of them: then nothing in the loop or at a request's end waits for
// another warp. Else it is a CTA whose 4 warps take a quarter each of a step's
// keys and join through shared memory at the request's end. Where a request's keys span
// several workers, each leaves its part (maximum, sum, unnormalised output) in
// the workspace, and the one that arrives last joins them.
//
// A warp that computes is fed by one that fetches, through a ring of stages:
// finding the next keys' page and issuing their copies takes about as long as
// computing on them does (1050 and 720 cycles of a step of 16 keys when one
// warp did both). The tensor instructions take 16 keys as their rows and the
// query rows of a kv head as their 8 columns: S^T = K Q^T, then O^T += V^T P^T,
// so up to 8 query heads of a kv head fill them without padding, and an
// accumulator takes D/2 registers. The probabilities are rounded to 16 bits for
// the product with V, since a tensor instruction takes both operands in one
// type and V has 16 bits: an error of the size of the output's own rounding.
// Maximum, sum and output stay in fp32.
//
// Memory bounds it where contexts are long: 4 flops a byte at 4 query heads to
// a kv head. Heads of 128, 32/8, bf16, pages of 16: 64 requests of 64..8192
// keys 75 us = 6.0 TB/s, 92% of the copy rate (92.5 us with one warp doing
// both, by 16-byte copies); one of 131072 88 us, 93%. Few or short requests
// wait for a chain of loads (lengths, page, keys: 2.6 us before the first
// product) and the joins of split requests (1.5 us): one of 129 keys 5.8 us.
template <int DT, int D, int R, int KEYS, int kStages, bool BOX, int kPerSm>
__global__ void __launch_bounds__(kCtaThreads, kPerSm)
    paged_kernel(const PagedParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using T = typename Elem<DT>::T;
  constexpr int KS = D / 16;  // mma steps over the head
  constexpr int NB = R / 8;   // blocks of 8 query rows
  constexpr int NK = KEYS / 16;  // blocks of 16 keys
  constexpr int kGroup = kWarps * KEYS;
  constexpr uint32_t kAll = KEYS == 32 ? ~0u : 0xffffu;
  constexpr int kPart = R * (D + 2);
  extern __shared__ uint8_t smem_raw[];
  using Smem = PagedSmem<D, R, KEYS, kStages>;
  uint8_t* smem = smem_raw + (1024 - (smem_addr(smem_raw) & 1023)) % 1024;
  Smem& sm = *reinterpret_cast<Smem*>(smem);
  const int rmax = min(R, p.G);
  float* so = reinterpret_cast<float*>(smem + sizeof(Smem));
  const int tid = threadIdx.x, lane = tid & 31, cta_warp = tid >> 5;
  const int warp = cta_warp % kWarps;  // the warp that computes, or is fetched for
  const bool fetches = cta_warp >= kWarps;
  const int heads = p.Hkv * p.RB;
  if (tid == 0) {
    sm.abort = 0;
    for (int w = 0; w < kWarps; ++w)
      for (int s = 0; s < kStages; ++s) {
        mbar_init(&sm.full[w][s], BOX ? 1 : 33);
        mbar_init(&sm.empty[w][s], 1);
      }
    fence_barrier_init();
    if (BOX) {
      prefetch_tmap(&kmap);
      prefetch_tmap(&vmap);
    }
  }
  griddep_wait();
  griddep_launch();

  // all places, of a warp's steps and of a CTA's, and the longest request (the host bounds their sums below 2^31)
  auto len_of = [&](int b) { return min(max(p.lens[b], 0), p.max_len); };
  auto places = [](int len, int keys) { return len > 0 ? (len + keys - 1) / keys + kUnitCost : 0; };
  const int my_len = tid < p.B ? len_of(tid) : 0;
  bool empty = false;  // of the empty requests, those with b = CTA modulo the grid are this CTA's
  {
    empty = tid < p.B && my_len == 0 && tid % gridDim.x == blockIdx.x;
    int n_solo = places(my_len, KEYS), n_group = places(my_len, kGroup), longest = my_len;
    for (int b = tid + kCtaThreads; b < p.B; b += kCtaThreads) {
      const int len = len_of(b);
      empty = empty || (len == 0 && b % gridDim.x == blockIdx.x);
      n_solo += places(len, KEYS);
      n_group += places(len, kGroup);
      longest = max(longest, len);
    }
    n_solo = __reduce_add_sync(0xffffffffu, n_solo);
    n_group = __reduce_add_sync(0xffffffffu, n_group);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) {
      sm.sum_solo[cta_warp] = n_solo;
      sm.sum_group[cta_warp] = n_group;
      sm.longest[cta_warp] = longest;
    }
  }
  if (__syncthreads_or(empty))  // their rows are zeros
    for (int b = blockIdx.x; b < p.B; b += gridDim.x)
      if (len_of(b) == 0)
        for (int i = tid; i < p.Hkv * p.G * D; i += kCtaThreads)
          static_cast<T*>(p.o)[b * p.o_sb + (i / D) * p.o_sh + i % D] = Elem<DT>::from_f(0.f);
  int n_solo = 0, n_group = 0, longest = 0;
#pragma unroll
  for (int w = 0; w < 2 * kWarps; ++w) {
    n_solo += sm.sum_solo[w];
    n_group += sm.sum_group[w];
    longest = max(longest, sm.longest[w]);
  }
  // Which worker: a warp where requests are short (their ends then cost more than the splits) and no request spans
  // many of them.
  const int64_t solo_quota = quotient(static_cast<int64_t>(n_solo) * heads + gridDim.x * kWarps - 1, gridDim.x * kWarps);
  const bool solo = solo_quota >= kSoloRun && n_solo / (kSoloMean * 16 / KEYS) < p.B && longest / KEYS < 24 * solo_quota;
  const int keys = solo ? KEYS : kGroup, first = solo ? 0 : warp * KEYS;
  const int64_t total = static_cast<int64_t>(solo ? n_solo : n_group) * heads;
  // a CTA's run is no shorter than a short request, or a few steps of a long one: a split costs about four steps
  const int64_t quota =
      solo ? solo_quota
           : max(quotient(total + gridDim.x - 1, gridDim.x), static_cast<int64_t>(min(places(longest, kGroup), kLeastRun)));
  const int64_t worker = solo ? static_cast<int64_t>(blockIdx.x) * kWarps + warp : blockIdx.x;
  const int64_t lo = worker * quota, hi = min(lo + quota, total);
  if (blockIdx.x * quota * (solo ? kWarps : 1) >= total) return;
  // the request that each worker's run begins in
  {
    const int64_t w0 = solo ? static_cast<int64_t>(blockIdx.x) * kWarps : blockIdx.x;
    int base = 0;  // places of the requests before this chunk, for one head
    for (int b0 = 0; b0 < p.B; b0 += kCtaThreads) {
      const int own = places(b0 == 0 ? my_len : b0 + tid < p.B ? len_of(b0 + tid) : 0, keys);
      int inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      int* sums = solo ? sm.sum_solo : sm.sum_group;
      if (p.B > kCtaThreads) {  // (one chunk: its warps' sums are there already)
        __syncthreads();
        if (lane == 31) sums[cta_warp] = inc;
        __syncthreads();
      }
      int all = base;
#pragma unroll
      for (int w = 0; w < 2 * kWarps; ++w) {
        if (w < cta_warp) inc += sums[w];
        all += sums[w];
      }
      inc += base;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int64_t at = (w0 + w) * quota;
        if (at < static_cast<int64_t>(inc) * heads && at >= static_cast<int64_t>(inc - own) * heads) {
          sm.at_b[w] = b0 + tid;
          sm.at_step[w] = at - static_cast<int64_t>(inc - own) * heads;
        }
      }
      base = all;
      if ((w0 + (solo ? kWarps - 1 : 0)) * quota < static_cast<int64_t>(all) * heads) break;
    }
    __syncthreads();
  }
  if (lo >= hi) return;  // (a warp by itself and the one that fetches for it; nothing below waits for them)

  Loader ld;
  ld.b = sm.at_b[solo ? warp : 0];
  ld.len = len_of(ld.b);
  ld.enter(p, keys);
  ld.left = hi - lo;
  const int64_t at_step = sm.at_step[solo ? warp : 0];
  ld.h = static_cast<int>(quotient(at_step, ld.nt + kUnitCost));
  ld.t = static_cast<int>(at_step - static_cast<int64_t>(ld.h) * (ld.nt + kUnitCost));
  ld.hk = ld.h / p.RB;
  ld.rb = ld.h - ld.hk * p.RB;

  uint8_t* stages = sm.stage[warp][0];
  int at = 0, phase = 0;  // stage and the parity of its round
  if (fetches) {
    if (ld.t >= ld.nt) {  // the run begins past the unit's last step
      ld.left -= ld.nt + kUnitCost - ld.t;
      ld.t = ld.nt - 1;
      ld.left += kUnitCost + 1;
      ld.advance(p, heads, keys);
    }
    ld.base = -1;
    ld.ahead_b = -1;
    ld.ahead_base = -1;
    int64_t step = 0;
    const uint64_t policy = p.RB > 1 ? l2_evict_normal() : l2_evict_first();
    while (ld.left > 0) {
      const int key0 = ld.t * keys + first;
      const int page = ld.page_of<KEYS>(p, key0, heads, lane);
      if (step >= kStages && !mbar_wait_warp(&sm.empty[warp][at], phase ^ 1, &sm.abort, 0x704)) return;  // reported
      load_step<D, KEYS, BOX>(p, &kmap, &vmap, ld, page, key0, lane, stages + at * Smem::kStageBytes, &sm.mask[warp][at],
                              &sm.full[warp][at], policy);
      if (ld.advance(p, heads, keys)) {  // another request: its first window has come in, or has not
        const bool come = ld.ahead_b == ld.b && ld.ahead_base == 0;
        ld.win = ld.ahead;
        ld.base = come ? 0 : -1;
        if (come) ld.look_ahead(p, heads, lane);
      } else if (ld.t == 0 && ld.base == 0) {  // another head of a request within one window
        ld.look_ahead(p, heads, lane);
      }
      ++step;
      if (++at == kStages) {
        at = 0;
        phase ^= 1;
      }
    }
    return;
  }

  // the unit computed on: request, kv head and row block, its step, steps in all
  int b = ld.b, hk = ld.hk, rb = ld.rb, t0 = ld.t, nt = ld.nt, next_len = ld.next_len;
  int64_t done = lo;  // flattened index of step t0
  bool dead = false;
  // the query rows of a unit as mma fragments
  uint32_t qn[KS][2 * NB];
  auto load_q = [&](int b_, int hk_, int rb_) {
    const int row0 = rb_ * R, rows = min(R, p.G - row0);
    const T* qb = static_cast<const T*>(p.q) + b_ * p.q_sb + (static_cast<int64_t>(hk_) * p.G + row0) * p.q_sh;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int r = (lane >> 2) + j * 8;
      const T* row = qb + r * p.q_sh + (lane & 3) * 2;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          qn[k][i * NB + j] = r < rows ? *reinterpret_cast<const uint32_t*>(row + k * 16 + i * 8) : 0u;
    }
  };
  load_q(b, hk, rb);

  while (done < hi) {
    const int rows = min(R, p.G - rb * R);
    const int t_past = static_cast<int>(min(static_cast<int64_t>(nt + kUnitCost), t0 + (hi - done)));  // places
    const int t_end = min(nt, t_past);                                                                // steps
    uint32_t qf[KS][2 * NB];
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) qf[k][i] = qn[k][i];
    // the unit after this one, whose query rows come in meanwhile
    int b2 = b, hk2 = hk, rb2 = rb + 1, nt2 = nt, next2 = next_len;
    if (done + (t_past - t0) < hi) {
      if (rb2 == p.RB) {
        rb2 = 0;
        ++hk2;
      }
      if (hk2 == p.Hkv) {
        hk2 = 0;
        do {
          ++b2;
          nt2 = (min(max(next2, 0), p.max_len) + keys - 1) / keys;
          next2 = b2 + 1 < p.B ? p.lens[b2 + 1] : 0;
        } while (nt2 == 0);
      }
      load_q(b2, hk2, rb2);
    }
    float acc[KS][NB][4];  // d = 16 n + lane / 4 (+ 8 in 2, 3), row 8 j + 2 (lane % 4) (+ 1 in 1, 3)
#pragma unroll
    for (int n = 0; n < KS; ++n)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][j][i] = 0.f;
    float mx[NB][2], sum[NB][2];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[j][i] = -INFINITY;
        sum[j][i] = 0.f;
      }
    for (int t = t0; t < t_end; ++t) {
      if (!dead && !mbar_try_wait(&sm.full[warp][at], phase)) dead = !mbar_wait(&sm.full[warp][at], phase, &sm.abort, 0x703);
      dead = __any_sync(0xffffffffu, dead);  // reported; nothing more is computed
      const uint32_t mask = dead ? 0u : sm.mask[warp][at];
      uint8_t* stage = stages + at * Smem::kStageBytes;
      const uint32_t kaddr = smem_addr(stage), vaddr = kaddr + KEYS * D * 2;
      if (mask != 0) {
        constexpr int CH = NK == 1 ? 2 : 1;  // chains over the head for a block of keys, added at the end
        float s[NK][NB][CH][4];
#pragma unroll
        for (int kb = 0; kb < NK; ++kb)
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
              for (int i = 0; i < 4; ++i) s[kb][j][c][i] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int kb = 0; kb < NK; ++kb) {
            uint32_t a[4];
            ldsm_x4(kaddr + swz<KEYS>(kb * 16 + (lane & 15), 2 * k + (lane >> 4)), a[0], a[1], a[2], a[3]);
#pragma unroll
            for (int j = 0; j < NB; ++j) mma16816<DT>(s[kb][j][k % CH], a, qf[k][j], qf[k][NB + j]);
          }
        uint32_t pb[NK][NB][2];
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          // key 16 kb + lane / 4 (+ 8 in x[2], x[3]) and rows 2 (lane % 4), + 1
          float x[NK][4];
          float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
          for (int kb = 0; kb < NK; ++kb) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[kb][i] = (CH == 2 ? s[kb][j][0][i] + s[kb][j][CH - 1][i] : s[kb][j][0][i]) * p.scale_log2;
            if (mask != kAll) {
              if (!((mask >> (kb * 16 + (lane >> 2))) & 1)) x[kb][0] = x[kb][1] = -INFINITY;
              if (!((mask >> (kb * 16 + (lane >> 2) + 8)) & 1)) x[kb][2] = x[kb][3] = -INFINITY;
            }
            m0 = fmaxf(m0, fmaxf(x[kb][0], x[kb][2]));
            m1 = fmaxf(m1, fmaxf(x[kb][1], x[kb][3]));
          }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
            m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
          }
          if (__any_sync(0xffffffffu, m0 > mx[j][0] || m1 > mx[j][1])) {
            const float n0 = fmaxf(mx[j][0], m0), n1 = fmaxf(mx[j][1], m1);
            const float f0 = n0 == -INFINITY ? 1.f : exp2_approx(mx[j][0] - n0);
            const float f1 = n1 == -INFINITY ? 1.f : exp2_approx(mx[j][1] - n1);
            mx[j][0] = n0;
            mx[j][1] = n1;
            sum[j][0] *= f0;
            sum[j][1] *= f1;
#pragma unroll
            for (int n = 0; n < KS; ++n) {
              acc[n][j][0] *= f0;
              acc[n][j][1] *= f1;
              acc[n][j][2] *= f0;
              acc[n][j][3] *= f1;
            }
          }
          const float r0 = mx[j][0] == -INFINITY ? 0.f : mx[j][0], r1 = mx[j][1] == -INFINITY ? 0.f : mx[j][1];
          auto power = [](float z) { return exp2_approx(DT == MT_F16 ? z + kTopF16 : z); };
#pragma unroll
          for (int kb = 0; kb < NK; ++kb) {
            const float e0 = power(x[kb][0] - r0), e1 = power(x[kb][1] - r1);
            const float e2 = power(x[kb][2] - r0), e3 = power(x[kb][3] - r1);
            sum[j][0] += e0 + e2;
            sum[j][1] += e1 + e3;
            // the probabilities in 16 bits, as the product with V takes them
            pb[kb][j][0] = transpose8(pack2<DT>(e0, e1));
            pb[kb][j][1] = transpose8(pack2<DT>(e2, e3));
          }
        }
        // O^T += V^T P^T. Rows of V without a key count as zeros, whatever the page or the stage holds there (a probability
        // of 0 would not clear a NaN): their fragments are masked in registers; zeros written to the stage instead
        // made one request of 129 keys 6.3 us for 5.8, 2048 of one key 46.4 for 42.8. Whole steps have a loop of their own.
        auto product = [&](auto part) {
#pragma unroll
          for (int kb = 0; kb < NK; ++kb) {
            // this lane's keys: 16 kb + 2 (lane % 4) and the next, + 8 in `upper`
            const uint32_t bits = mask >> (kb * 16 + (lane & 3) * 2);
            const uint32_t lower = ((bits & 1) ? 0xffffu : 0u) | ((bits & 2) ? 0xffff0000u : 0u);
            const uint32_t upper = ((bits & 0x100) ? 0xffffu : 0u) | ((bits & 0x200) ? 0xffff0000u : 0u);
#pragma unroll
            for (int n = 0; n < KS; ++n) {
              uint32_t a[4];
              ldsm_x4_t(vaddr + swz<KEYS>(kb * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * n + ((lane >> 3) & 1)), a[0], a[1],
                        a[2], a[3]);
              if constexpr (decltype(part)::value) {
                a[0] &= lower;
                a[1] &= lower;
                a[2] &= upper;
                a[3] &= upper;
              }
#pragma unroll
              for (int j = 0; j < NB; ++j) mma16816<DT>(acc[n][j], a, pb[kb][j][0], pb[kb][j][1]);
            }
          }
        };
        if (mask == kAll) product(std::false_type());
        else product(std::true_type());
      }
      __syncwarp();
      if (dead) continue;  // the stage stays taken: the warp that fetches gives up too
      if (lane == 0) mbar_arrive(&sm.empty[warp][at]);
      if (++at == kStages) {
        at = 0;
        phase ^= 1;
      }
    }

    const bool whole = t0 == 0 && t_end == nt;
    int64_t c0 = 0, c1 = 0;  // the workers that share the unit
    if (!whole) {
      c0 = quotient(done - t0, quota);
      c1 = quotient(done - t0 + nt - 1, quota);
    }
    // part slots of a worker: 0 the unit its run begins inside, 1 the unit that goes on after it
    float* mine = p.part + (worker * 2 + (t0 == 0 ? 1 : 0)) * kPart;
    T* ob = static_cast<T*>(p.o) + b * p.o_sb + (static_cast<int64_t>(hk) * p.G + rb * R) * p.o_sh;
    if (t0 < nt) {  // (a run may begin past a unit's last step)
    // the warp's rows in shared memory
    float* own = so + warp * rmax * Smem::kOStride;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = j * 8 + (lane & 3) * 2 + i;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum[j][i] += __shfl_xor_sync(0xffffffffu, sum[j][i], o);
        if (r < rows) {
          if (lane < 4) {
            sm.m[warp][r] = mx[j][i];
            sm.l[warp][r] = sum[j][i];
          }
#pragma unroll
          for (int n = 0; n < KS; ++n) {
            own[r * Smem::kOStride + n * 16 + (lane >> 2)] = acc[n][j][i];
            own[r * Smem::kOStride + n * 16 + 8 + (lane >> 2)] = acc[n][j][2 + i];
          }
        }
      }
    // rows of the worker's warps joined: to the output, or to the worker's part
    auto write_row = [&](int r, int d, float M, float L, const float (&x)[4]) {
      if (whole) {
        const float inv = L > 0.f ? 1.f / L : L;  // a row that saw no key is zero; NaN stays NaN
        uint2 u;
        u.x = pack2<DT>(x[0] * inv, x[1] * inv);
        u.y = pack2<DT>(x[2] * inv, x[3] * inv);
        *reinterpret_cast<uint2*>(ob + r * p.o_sh + d) = u;
      } else {
        __stcg(reinterpret_cast<float4*>(mine + 2 * R + r * D + d), make_float4(x[0], x[1], x[2], x[3]));
        if (d == 0) {
          __stcg(mine + r, M);
          __stcg(mine + R + r, L);
        }
      }
    };
    if (solo) {
      __syncwarp();
      for (int i = lane; i < rows * (D / 4); i += 32) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4;
        const float4 v = *reinterpret_cast<const float4*>(own + r * Smem::kOStride + d);
        const float x[4] = {v.x, v.y, v.z, v.w};
        write_row(r, d, sm.m[warp][r], sm.l[warp][r], x);
      }
      if (!whole) {
        __syncwarp();
        int last = 0;
        if (lane == 0) {
          __threadfence();
          last = atomicAdd(&p.counters[c0], 1u) == static_cast<uint32_t>(c1 - c0);
          if (last) p.counters[c0] = 0u;
        }
        if (__shfl_sync(0xffffffffu, last, 0)) {
          __threadfence();
          join_parts<DT, D, R, 2, 4>(p, c0, c1, rows, ob, lane, 32);
        }
      }
      __syncwarp();
    } else {
      named_barrier(1, kThreads);
      for (int i = tid; i < rows * (D / 4); i += kThreads) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.m[w][r]);
        float L = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = sm.m[w][r] == -INFINITY ? 0.f : exp2_approx(sm.m[w][r] - M);
          L = fmaf(f, sm.l[w][r], L);
          const float4 v = *reinterpret_cast<const float4*>(so + (w * rmax + r) * Smem::kOStride + d);
          x[0] = fmaf(f, v.x, x[0]);
          x[1] = fmaf(f, v.y, x[1]);
          x[2] = fmaf(f, v.z, x[2]);
          x[3] = fmaf(f, v.w, x[3]);
        }
        write_row(r, d, M, L, x);
      }
      if (!whole) {
        named_barrier(1, kThreads);
        if (tid == 0) {
          __threadfence();
          sm.flag = atomicAdd(&p.counters[c0], 1u) == static_cast<uint32_t>(c1 - c0);
          if (sm.flag) p.counters[c0] = 0u;
        }
        named_barrier(1, kThreads);
        if (sm.flag) {
          __threadfence();
          join_parts<DT, D, R, 1, 8>(p, c0, c1, rows, ob, tid, kThreads);
        }
      }
      named_barrier(1, kThreads);  // the joined rows' memory and the flag are used again
    }
    }
    done += t_past - t0;
    b = b2;
    hk = hk2;
    rb = rb2;
    nt = nt2;
    next_len = next2;
    t0 = 0;
  }
  if (BOX && dead)  // copies still under way must not outlive the CTA
    for (int s = 0; s < kStages; ++s) mbar_wait_drain(&sm.full[warp][s], s < at ? phase ^ 1 : phase, 100000000ull);
}

}  // namespace
}  // namespace mt

using namespace mt;

extern "C" {

size_t mt_paged_sdpa_decode_workspace_bytes(int64_t D) {
  return kWsCtlBytes + static_cast<size_t>(kMaxCtas) * kWarps * 2 * 16 * (D + 2) * sizeof(float);
}

int mt_paged_sdpa_decode(const void* q, int64_t q_sb, int64_t q_sh, const void* k_cache, const void* v_cache,
                         int64_t num_pages, int64_t page_size, int64_t page_stride, int64_t head_stride,
                         int64_t slot_stride, const int32_t* block_table, int64_t table_stride, int64_t max_pages,
                         const int32_t* seq_lens, void* o, int64_t o_sb, int64_t o_sh, int64_t B, int64_t Hq,
                         int64_t Hkv, int64_t D, float scale, int dtype, void* workspace, size_t workspace_bytes,
                         mt_stream_t stream) {
  clear_error();
  MT_CHECK_ARG(D == 64 || D == 128, "mt_paged_sdpa_decode: head_dim %lld, only 64 and 128 are built", (long long)D);
  if (dtype != MT_BF16 && dtype != MT_F16) {
    set_error("mt_paged_sdpa_decode: dtype must be bf16 or f16");
    return MT_ERR_UNSUPPORTED;
  }
  MT_CHECK_ARG(B >= 0 && B < (1 << 24) && Hkv > 0 && Hq > 0 && Hq < 4096 && Hq % Hkv == 0,
               "mt_paged_sdpa_decode: B=%lld, Hq=%lld must be a multiple of Hkv=%lld", (long long)B, (long long)Hq,
               (long long)Hkv);
  MT_CHECK_ARG(num_pages >= 0 && num_pages < (1ll << 31) && page_size > 0 && page_size <= (1 << 20) && max_pages >= 0 && max_pages < (1ll << 31) &&
                   table_stride >= max_pages,
               "mt_paged_sdpa_decode: num_pages=%lld page_size=%lld max_pages=%lld table stride=%lld",
               (long long)num_pages, (long long)page_size, (long long)max_pages, (long long)table_stride);
  if (B == 0) return MT_OK;
  MT_CHECK_ARG(q && seq_lens && o && (num_pages == 0 || (k_cache && v_cache)) && (max_pages == 0 || block_table),
               "mt_paged_sdpa_decode: null pointer");
  MT_CHECK_ARG(aligned(q, 4) && (q_sb | q_sh) % 2 == 0 && aligned(o, 8) && (o_sb | o_sh) % 4 == 0 && aligned(k_cache, 16) && aligned(v_cache, 16) &&
                   (page_stride | head_stride | slot_stride) % 8 == 0,
               "mt_paged_sdpa_decode: cache rows must be 16-byte aligned, output rows 8, query rows 4");
  if (workspace == nullptr || workspace_bytes < mt_paged_sdpa_decode_workspace_bytes(D)) {
    set_error("mt_paged_sdpa_decode: needs a workspace of %zu bytes, got %zu", mt_paged_sdpa_decode_workspace_bytes(D),
              workspace ? workspace_bytes : (size_t)0);
    return MT_ERR_WORKSPACE;
  }
  MT_CHECK_ARG(aligned(workspace, 16), "mt_paged_sdpa_decode: workspace must be 16-byte aligned");
  if (B * (max_pages * page_size / 16 + 1 + kUnitCost) >= 1ll << 31) {
    set_error("mt_paged_sdpa_decode: %lld requests of %lld pages of %lld rows: 2^35 rows in all are the limit", (long long)B,
              (long long)max_pages, (long long)page_size);
    return MT_ERR_UNSUPPORTED;
  }
  int sms = 148;
  if (int rc = device_sm_count(&sms)) return rc;
  const int G = static_cast<int>(Hq / Hkv), R = G <= 8 ? 8 : 16, RB = (G + R - 1) / R;
  const int64_t room = max_pages * page_size < 0x7fffffff - 64 ? max_pages * page_size : 0x7fffffff - 64;
  PagedParams p = {q, q_sb, q_sh, k_cache, v_cache, num_pages, page_stride, head_stride, slot_stride, FastDiv::of((int)page_size),
                   block_table, table_stride, (int)room, seq_lens, o, o_sb, o_sh, (int)B, (int)Hkv, G, RB, 8,
                   scale * 1.4426950408889634f,
                   reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kWsCtlBytes),
                   reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + kWsPagedCtl)};
  const int64_t most = B * Hkv * RB * ((room + 63) / 64 + kUnitCost);  // steps if every request were as long as its table row
  // the copy engine where pages hold whole boxes and its strides can express the cache
  const int64_t bytes[3] = {slot_stride * 2, head_stride * 2, page_stride * 2};
  const int64_t extent[3] = {page_size, Hkv, num_pages};
  bool box = page_size % 8 == 0 && num_pages > 0;
  uint64_t dims[4] = {(uint64_t)D}, strides[3];
  for (int i = 0; i < 3; ++i) {
    dims[i + 1] = (uint64_t)extent[i];
    strides[i] = extent[i] > 1 ? (uint64_t)bytes[i] : 16;
    box = box && extent[i] < (1ll << 32) && (extent[i] == 1 || (bytes[i] > 0 && bytes[i] < (1ll << 40)));
  }
  // Steps of 32 keys for heads of 64, and for heads of 128 where there are few units: then one CTA to an SM, fewer parts
  // to join and more bytes to a copy of the copy engine. With 8 units to a request, 16 keys a step against 32: 64..8192
  // keys 16 requests 25.4 and 24.2 us, 64 77.3 and 74.5, 128 146 and 143; four of 4096 18.9 and 16.9, one of 131072 90.6
  // and 87.8, 96 of 4096 251 and 247. But 64..2048 keys 16 requests 13.9 and 14.9, 64 31.6 and 34.3, 256 101 and 107; 1..512
  // keys 64 13.6 and 13.1, 256 26.3 and 28.7; and by 16-byte copies 16 of 64..2048 15.4 and 16.6. It is the lengths and
  // their spread that decide, which the host does not know; many units stand for short ragged requests here, 3% to 8%
  // off where they are few and short or many and long.
  const bool wide = D == 64 || (R == 8 && box && B * Hkv * RB <= 512);
  p.box_rows = wide && page_size % 32 == 0 ? 32 : page_size % 16 == 0 ? 16 : 8;
  CUtensorMap kmap = {}, vmap = {};
  if (box) {
    const uint32_t shape[4] = {64, (uint32_t)p.box_rows, 1, 1};
    const CUtensorMapDataType type = dtype == MT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (int e = make_tmaps(&kmap, k_cache, &vmap, v_cache, type, 2, 4, dims, strides, shape, CU_TENSOR_MAP_SWIZZLE_128B))
      return e;
  }
  auto run = [&](auto kern, size_t smem, int per_sm) -> int {
    if (int e = ensure_smem(kern, smem)) return e;
    int64_t grid = static_cast<int64_t>(sms) * per_sm;
    if (grid > kMaxCtas) grid = kMaxCtas;
    if (grid > most) grid = most < 1 ? 1 : most;
    return launch(kern, dim3((unsigned)grid), dim3(kCtaThreads), smem, (cudaStream_t)stream, p, kmap, vmap);
  };
  const int rows = G < R ? G : R;
  // by head size and query rows: ring stages and CTAs to an SM that its shared memory holds beside the rows to join
  auto pick = [&](auto type, auto dim) -> int {
    constexpr int DT = decltype(type)::value, D_ = decltype(dim)::value;
    auto with = [&](auto r, auto keys, auto stages, auto per_sm) -> int {
      constexpr int R_ = decltype(r)::value, K_ = decltype(keys)::value, S_ = decltype(stages)::value,
                    N_ = decltype(per_sm)::value;
      const size_t smem = PagedSmem<D_, R_, K_, S_>::bytes(rows);
      return box ? run(paged_kernel<DT, D_, R_, K_, S_, true, N_>, smem, N_)
                 : run(paged_kernel<DT, D_, R_, K_, S_, false, N_>, smem, N_);
    };
    if constexpr (D_ == 64)
      return R == 16 ? with(Int<16>(), Int<32>(), Int<2>(), Int<2>()) : with(Int<8>(), Int<32>(), Int<3>(), Int<2>());
    else
      return R == 16  ? with(Int<16>(), Int<16>(), Int<4>(), Int<1>())
             : wide   ? with(Int<8>(), Int<32>(), Int<3>(), Int<1>())
             : G <= 4 ? with(Int<8>(), Int<16>(), Int<3>(), Int<2>())
                      : with(Int<8>(), Int<16>(), Int<2>(), Int<2>());
  };
  if (dtype == MT_BF16) return D == 128 ? pick(Int<MT_BF16>(), Int<128>()) : pick(Int<MT_BF16>(), Int<64>());
  return D == 128 ? pick(Int<MT_F16>(), Int<128>()) : pick(Int<MT_F16>(), Int<64>());
}

}  // extern "C"
