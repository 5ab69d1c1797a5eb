// Attention of one new token per request over a paged key-value cache.
#include "mma_sync.cuh"
#include "mt_common.cuh"

namespace mt {
namespace {

struct PagedParams {
  const void* q;
  int64_t q_sb, q_sh;
  const void *kc, *vc;
  int64_t num_pages, page_stride, head_stride, slot_stride;
  int page_size;
  const int32_t* table;
  int64_t table_stride;
  int max_len;  // rows a table row can address (and the largest length used)
  const int32_t* lens;
  void* o;
  int64_t o_sb, o_sh;
  int B, Hkv, G, RB;  // RB: blocks of R query rows per kv head
  float scale_log2;
  float* part;
  uint32_t* counters;
};

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 16;                // keys of one warp's step
constexpr int kTile = kWarps * kKeys;    // keys of one CTA's step
constexpr int kMaxCtas = 444;            // bounds the workspace; 3 CTAs on each of 148 SMs
constexpr size_t kWsPagedCtl = 2304;     // arrival counters, one per CTA, in the workspace's control words
static_assert(kWsPagedCtl + 4 * kMaxCtas <= kWsQmmDone, "the counters end before the next kernel's words");

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Position in the flattened work: tiles of (request, kv head x row block), the
// requests of length 0 left out.
struct Cursor {
  int b, h, t, nt, len;
  int64_t left;  // tiles of this CTA from here on
  __device__ __forceinline__ void enter(const PagedParams& p) {
    len = min(max(p.lens[b], 0), p.max_len);
    nt = (len + kTile - 1) / kTile;
  }
  __device__ __forceinline__ void advance(const PagedParams& p, int heads) {
    --left;
    if (++t < nt) return;
    t = 0;
    if (++h < heads) return;
    h = 0;
    if (left <= 0) return;
    do {
      ++b;
      enter(p);
    } while (nt == 0);
  }
};

template <int D>
__device__ __forceinline__ uint32_t swz(int row, int chunk) {  // byte offset of a 16-byte chunk of a row
  return static_cast<uint32_t>(row * (D * 2) + ((chunk ^ (row & 7)) << 4));
}

// Warp-private step loads: the 16 keys' rows of K and V into stage memory by
// 16-byte asynchronous copies; rows without a key (past the length, or on a
// page id outside the cache) are filled with zeros and left out of the mask.
template <int D>
__device__ __forceinline__ void load_step(const PagedParams& p, const Cursor& c, int warp, int lane, uint8_t* stage,
                                          uint32_t* mask) {
  constexpr int CPR = D / 8;  // 16-byte chunks per row
  const int key = c.t * kTile + warp * kKeys + (lane & 15);
  int64_t off = -1;
  if (key < c.len) {
    const int block = key / p.page_size;
    const int page = p.table[c.b * p.table_stride + block];
    if (page >= 0 && page < p.num_pages)
      off = page * p.page_stride + (key - block * p.page_size) * p.slot_stride + (c.h / p.RB) * p.head_stride;
    else if (lane < 16)
      report_status(0x702);
  }
  const uint32_t m = __ballot_sync(0xffffffffu, off >= 0) & 0xffffu;
  if (lane == 0) *mask = m;
  const int chunk = lane % CPR;
#pragma unroll
  for (int i = 0; i < 16 * CPR / 32; ++i) {
    const int row = i * (32 / CPR) + lane / CPR;
    const int64_t ro = __shfl_sync(0xffffffffu, off, row);
    const int64_t src = ro >= 0 ? ro + chunk * 8 : 0;
    const uint32_t at = swz<D>(row, chunk);
    cp_async16(stage + at, static_cast<const uint16_t*>(p.kc) + src, ro >= 0);
    cp_async16(stage + 16 * D * 2 + at, static_cast<const uint16_t*>(p.vc) + src, ro >= 0);
  }
}

template <int D, int R, int kStages>
struct PagedSmem {
  static constexpr int kStageBytes = 2 * kKeys * D * 2;
  static constexpr int kOStride = D + 8;
  alignas(128) uint8_t stage[kWarps][kStages][kStageBytes];
  float m[kWarps][R], l[kWarps][R];
  uint32_t mask[kWarps][kStages];
  int64_t red[kWarps];
  int64_t at_tile;
  int at_b, flag;
  // followed by the warps' accumulators while they are joined: [kWarps][rows][kOStride]
  static size_t bytes(int rows) { return sizeof(PagedSmem) + sizeof(float) * kWarps * rows * kOStride; }
};

// The flattened tiles of all requests and kv heads are cut into equal runs,
// one per CTA, whatever the lengths are; a run starts and ends anywhere inside
// a request. Each of the 4 warps walks its own 16 keys of every tile with a
// ring of asynchronous copies of its own, a running maximum and sum per query
// row and its own accumulators: no barrier until the request's (kv head's)
// keys end. Then the warps join through shared memory. Where a request's keys
// span several CTAs, each leaves its part (maximum, sum, unnormalised output)
// in the workspace, and the one that arrives last joins the parts in key
// order, so the result does not depend on who that is.
template <int DT, int D, int R, int kStages>
__global__ void __launch_bounds__(kThreads) paged_kernel(const PagedParams p) {
  using T = typename Elem<DT>::T;
  constexpr int KS = D / 16;  // mma steps over the head
  constexpr int HALVES = R / 8;
  extern __shared__ uint8_t smem_raw[];
  using Smem = PagedSmem<D, R, kStages>;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int rmax = min(R, p.G);
  float* so = reinterpret_cast<float*>(smem_raw + sizeof(Smem));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = p.Hkv * p.RB;
  griddep_wait();
  griddep_launch();

  // empty requests: zeros
  for (int b = blockIdx.x; b < p.B; b += gridDim.x)
    if (p.lens[b] <= 0 || p.max_len == 0)
      for (int i = tid; i < p.Hkv * p.G * D; i += kThreads)
        static_cast<T*>(p.o)[b * p.o_sb + (i / D) * p.o_sh + i % D] = Elem<DT>::from_f(0.f);

  // this CTA's run of tiles
  auto tiles_of = [&](int b) -> int64_t {
    const int len = min(max(p.lens[b], 0), p.max_len);
    return static_cast<int64_t>((len + kTile - 1) / kTile) * heads;
  };
  int64_t total = 0;
  for (int b = tid; b < p.B; b += kThreads) total += tiles_of(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) sm.red[warp] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += sm.red[w];
  const int64_t quota = (total + gridDim.x - 1) / gridDim.x;
  const int64_t lo = blockIdx.x * quota;
  const int64_t hi = min(lo + quota, total);
  if (lo >= hi) return;
  int64_t base = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int64_t own = b0 + tid < p.B ? tiles_of(b0 + tid) : 0;
    int64_t inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) sm.red[warp] = inc;
    __syncthreads();
    int64_t all = base;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) inc += sm.red[w];
      all += sm.red[w];
    }
    inc += base;
    if (lo < inc && lo >= inc - own) {
      sm.at_b = b0 + tid;
      sm.at_tile = lo - (inc - own);
    }
    if (lo < all) break;
    base = all;
  }
  __syncthreads();

  Cursor cur;
  cur.b = sm.at_b;
  cur.enter(p);
  cur.h = static_cast<int>(sm.at_tile / cur.nt);
  cur.t = static_cast<int>(sm.at_tile - static_cast<int64_t>(cur.h) * cur.nt);
  cur.left = hi - lo;
  Cursor ld = cur;
  int64_t done = lo;  // flattened index of cur

  uint8_t* stages = sm.stage[warp][0];
  int put = 0, get = 0;
  auto issue = [&]() {
    if (ld.left > 0) {
      load_step<D>(p, ld, warp, lane, stages + put * Smem::kStageBytes, &sm.mask[warp][put]);
      ld.advance(p, heads);
    }
    cp_async_commit();
    put = put + 1 == kStages ? 0 : put + 1;
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue();

  while (cur.left > 0) {
    const int b = cur.b, h = cur.h, t0 = cur.t, nt = cur.nt;
    const int hk = h / p.RB, row0 = (h - hk * p.RB) * R;
    const int rows = min(R, p.G - row0);
    const T* qb = static_cast<const T*>(p.q) + b * p.q_sb + (static_cast<int64_t>(hk) * p.G + row0) * p.q_sh;
    uint32_t qf[KS][4];
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (lane >> 2) + (i & 1) * 8, col = k * 16 + (i >> 1) * 8 + (lane & 3) * 2;
        qf[k][i] = r < rows ? *reinterpret_cast<const uint32_t*>(qb + r * p.q_sh + col) : 0u;
      }
    float acc[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
    float mx[HALVES], sum[HALVES];
#pragma unroll
    for (int i = 0; i < HALVES; ++i) {
      mx[i] = -INFINITY;
      sum[i] = 0.f;
    }
    int t = t0;
    do {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      issue();
      const uint32_t mask = sm.mask[warp][get];
      const uint32_t kb = smem_addr(stages + get * Smem::kStageBytes), vb = kb + 16 * D * 2;
      get = get + 1 == kStages ? 0 : get + 1;
      if (mask != 0) {
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t r0, r1, r2, r3;
          // keys 0-7 / 8-15 by d halves of this step
          const int row = (lane & 7) + ((lane >> 4) << 3), chunk = 2 * k + ((lane >> 3) & 1);
          ldsm_x4(kb + swz<D>(row, chunk), r0, r1, r2, r3);
          mma16816<DT>(s[0], qf[k], r0, r1);
          mma16816<DT>(s[1], qf[k], r2, r3);
        }
        uint32_t pf[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < HALVES; ++i) {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = (e >> 1) * 8 + (lane & 3) * 2 + (e & 1);
            x[e] = (mask >> key) & 1 ? s[e >> 1][2 * i + (e & 1)] * p.scale_log2 : -INFINITY;
          }
          float m = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          if (__any_sync(0xffffffffu, m > mx[i])) {
            const float nm = fmaxf(mx[i], m);
            const float f = nm == -INFINITY ? 1.f : exp2_approx(mx[i] - nm);
            mx[i] = nm;
            sum[i] *= f;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              acc[n][2 * i] *= f;
              acc[n][2 * i + 1] *= f;
            }
          }
          const float ref = mx[i] == -INFINITY ? 0.f : mx[i];
          float e0 = exp2_approx(x[0] - ref), e1 = exp2_approx(x[1] - ref);
          float e2 = exp2_approx(x[2] - ref), e3 = exp2_approx(x[3] - ref);
          sum[i] += (e0 + e1) + (e2 + e3);
          pf[i] = pack2<DT>(e0, e1);
          pf[2 + i] = pack2<DT>(e2, e3);
        }
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          uint32_t r0, r1, r2, r3;
          const int row = (lane & 7) + (((lane >> 3) & 1) << 3), chunk = 2 * n + (lane >> 4);
          ldsm_x4_t(vb + swz<D>(row, chunk), r0, r1, r2, r3);
          mma16816<DT>(acc[2 * n], pf, r0, r1);
          mma16816<DT>(acc[2 * n + 1], pf, r2, r3);
        }
      }
      cur.advance(p, heads);
      ++t;
    } while (t < nt && cur.left > 0);

    // join the warps
#pragma unroll
    for (int i = 0; i < HALVES; ++i) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
      const int r = (lane >> 2) + 8 * i;
      if (r < rows) {
        if ((lane & 3) == 0) {
          sm.m[warp][r] = mx[i];
          sm.l[warp][r] = sum[i];
        }
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(so + (warp * rmax + r) * Smem::kOStride + n * 8 + (lane & 3) * 2) = make_float2(acc[n][2 * i], acc[n][2 * i + 1]);
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t == nt;
    const int64_t first = done - t0, last = first + nt - 1;  // the unit's tiles
    const int c0 = static_cast<int>(first / quota), c1 = static_cast<int>(last / quota);
    // part slots of a CTA: 0 the unit its run begins inside, 1 the unit that goes on after it
    constexpr int kPart = R * (D + 2);
    float* mine = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + (t0 == 0 ? 1 : 0)) * kPart;
    T* ob = static_cast<T*>(p.o) + b * p.o_sb + (static_cast<int64_t>(hk) * p.G + row0) * p.o_sh;
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
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const uint32_t old = atomicAdd(&p.counters[c0], 1u);
        sm.flag = old == static_cast<uint32_t>(c1 - c0);
        if (sm.flag) p.counters[c0] = 0u;
      }
      __syncthreads();
      if (sm.flag) {
        __threadfence();
        for (int i = tid; i < rows * (D / 4); i += kThreads) {
          const int r = i / (D / 4), d = (i % (D / 4)) * 4;
          float M = -INFINITY;
          for (int c = c0; c <= c1; ++c)
            M = fmaxf(M, __ldcg(p.part + (static_cast<int64_t>(c) * 2 + (c == c0)) * kPart + r));
          float L = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
          for (int c = c0; c <= c1; ++c) {
            const float* q = p.part + (static_cast<int64_t>(c) * 2 + (c == c0)) * kPart;
            const float m = __ldcg(q + r);
            const float f = m == -INFINITY ? 0.f : exp2_approx(m - M);
            L = fmaf(f, __ldcg(q + R + r), L);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(q + 2 * R + r * D + d));
            x[0] = fmaf(f, v.x, x[0]);
            x[1] = fmaf(f, v.y, x[1]);
            x[2] = fmaf(f, v.z, x[2]);
            x[3] = fmaf(f, v.w, x[3]);
          }
          const float inv = L > 0.f ? 1.f / L : L;
          uint2 u;
          u.x = pack2<DT>(x[0] * inv, x[1] * inv);
          u.y = pack2<DT>(x[2] * inv, x[3] * inv);
          *reinterpret_cast<uint2*>(ob + r * p.o_sh + d) = u;
        }
      }
    }
    __syncthreads();  // the joined rows' memory and the flag are used again
    done += t - t0;
  }
}

}  // namespace
}  // namespace mt

using namespace mt;

extern "C" {

size_t mt_paged_sdpa_decode_workspace_bytes(int64_t D) {
  return kWsCtlBytes + static_cast<size_t>(kMaxCtas) * 2 * 16 * (D + 2) * sizeof(float);
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
  MT_CHECK_ARG(num_pages >= 0 && page_size > 0 && page_size <= (1 << 20) && max_pages >= 0 && max_pages < (1ll << 31) &&
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
  int sms = 148;
  if (int rc = device_sm_count(&sms)) return rc;
  const int G = static_cast<int>(Hq / Hkv), R = G <= 8 ? 8 : 16, RB = (G + R - 1) / R;
  const int64_t room = max_pages * page_size < 0x7fffffff - kTile ? max_pages * page_size : 0x7fffffff - kTile;
  PagedParams p = {q, q_sb, q_sh, k_cache, v_cache, num_pages, page_stride, head_stride, slot_stride, (int)page_size,
                   block_table, table_stride, (int)room, seq_lens, o, o_sb, o_sh, (int)B, (int)Hkv, G, RB,
                   scale * 1.4426950408889634f,
                   reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kWsCtlBytes),
                   reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + kWsPagedCtl)};
  const int64_t most = B * Hkv * RB * ((room + kTile - 1) / kTile);  // tiles if every request were as long as its table row
  auto run = [&](auto kern, size_t smem) -> int {
    if (int e = ensure_smem(kern, smem)) return e;
    const int per_sm = static_cast<int>((228 * 1024) / (smem + 1024));
    int64_t grid = static_cast<int64_t>(sms) * (per_sm < 1 ? 1 : per_sm);
    if (grid > kMaxCtas) grid = kMaxCtas;
    if (grid > most) grid = most < 1 ? 1 : most;
    return launch(kern, dim3((unsigned)grid), dim3(kThreads), smem, (cudaStream_t)stream, p);
  };
#define MT_PAGED(DT, D_, R_, S_) run(paged_kernel<DT, D_, R_, S_>, PagedSmem<D_, R_, S_>::bytes(G < R_ ? G : R_))
// three ring stages where two CTAs with them fit an SM
#define MT_PAGED_R(DT, D_) \
  (R == 16 ? MT_PAGED(DT, D_, 16, 2) : (D_ == 64 || G <= 4) ? MT_PAGED(DT, D_, 8, 3) : MT_PAGED(DT, D_, 8, 2))
  if (dtype == MT_BF16) return D == 128 ? MT_PAGED_R(MT_BF16, 128) : MT_PAGED_R(MT_BF16, 64);
  return D == 128 ? MT_PAGED_R(MT_F16, 128) : MT_PAGED_R(MT_F16, 64);
#undef MT_PAGED_R
#undef MT_PAGED
}

}  // extern "C"
