// Log-probabilities of given tokens with entropy, logsumexp and the top
// alternatives of each row of logits.
#include "mt_common.cuh"

namespace mt {
namespace {

constexpr int kLpThreads = 512;
constexpr int kLpMaxTop = 32;

// Larger keys first: the value's order, then the lower index. NaN sorts above
// every number, -0 equals +0.
__device__ __forceinline__ uint64_t top_key(float v, uint32_t i) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t u = isnan(v) ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return static_cast<uint64_t>(u) << 32 | (0xffffffffu - i);
}

struct LogprobArgs {
  const void* logits;
  int64_t stride, V;
  const int32_t* tokens;
  int top_k;
  float *logprob, *entropy, *lse;
  int32_t* top_ids;
  float* top_lp;
};

// One row per CTA, three passes: maximum, sums, then top_k rounds.
template <int DT>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(const LogprobArgs a) {
  using T = typename Elem<DT>::T;
  __shared__ float red_f[kLpThreads / 32];
  __shared__ double red_d[2][kLpThreads / 32];
  __shared__ uint64_t red_k[kLpThreads / 32];
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  float m = -INFINITY;
  for (int64_t i = tid; i < a.V; i += kLpThreads) m = fmaxf(m, Elem<DT>::to_f(x[i]));
  m = warp_max(m);
  if (lane == 0) red_f[warp] = m;
  __syncthreads();
  for (int w = 0; w < kLpThreads / 32; ++w) m = fmaxf(m, red_f[w]);
  double s = 0, t = 0;
  for (int64_t i = tid; i < a.V; i += kLpThreads) {
    const float z = Elem<DT>::to_f(x[i]) - m;
    const float e = expf(z);
    s += e;
    if (e > 0.f) t += static_cast<double>(e) * z;
  }
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  if (lane == 0) {
    red_d[0][warp] = s;
    red_d[1][warp] = t;
  }
  __syncthreads();
  s = t = 0;
  for (int w = 0; w < kLpThreads / 32; ++w) {
    s += red_d[0][w];
    t += red_d[1][w];
  }
  const double lse = m + log(s);
  if (tid == 0) {
    if (a.lse) a.lse[row] = static_cast<float>(lse);
    if (a.entropy) a.entropy[row] = static_cast<float>(log(s) - t / s);
    if (a.tokens) {
      const int tok = a.tokens[row];
      if (tok >= a.V) report_status(0x801);
      a.logprob[row] = tok >= 0 && tok < a.V ? static_cast<float>(Elem<DT>::to_f(x[tok]) - lse) : 0.f;
    }
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    uint64_t best = 0;
    for (int64_t i = tid; i < a.V; i += kLpThreads) {
      const uint64_t key = top_key(Elem<DT>::to_f(x[i]), static_cast<uint32_t>(i));
      if (key < last && key > best) best = key;
    }
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t u = __shfl_xor_sync(0xffffffffu, best, o);
      best = u > best ? u : best;
    }
    __syncthreads();
    if (lane == 0) red_k[warp] = best;
    __syncthreads();
    for (int w = 0; w < kLpThreads / 32; ++w) best = red_k[w] > best ? red_k[w] : best;
    last = best;
    if (tid == 0) {
      const uint32_t i = 0xffffffffu - static_cast<uint32_t>(best);
      a.top_ids[row * a.top_k + k] = static_cast<int32_t>(i);
      a.top_lp[row * a.top_k + k] = static_cast<float>(Elem<DT>::to_f(x[i]) - lse);
    }
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
  MT_CHECK_ARG(top_k >= 0 && top_k <= kLpMaxTop && top_k <= V, "mt_token_logprobs: top_k=%d outside 0..min(%d, V)",
               top_k, kLpMaxTop);
  if (dtype != MT_BF16 && dtype != MT_F16 && dtype != MT_F32) {
    set_error("mt_token_logprobs: unsupported dtype %d", dtype);
    return MT_ERR_UNSUPPORTED;
  }
  if (R == 0) return MT_OK;
  MT_CHECK_ARG(logits && (!tokens || logprob) && (top_k == 0 || (top_ids && top_logprobs)),
               "mt_token_logprobs: null pointer");
  MT_CHECK_ARG(aligned(logits, dtype == MT_F32 ? 4 : 2), "mt_token_logprobs: logits not aligned to their type");
  const LogprobArgs a = {logits, row_stride, V, tokens, top_k, logprob, entropy, lse, top_ids, top_logprobs};
  auto run = [&](auto kern) {
    return launch(kern, dim3((unsigned)R), dim3(kLpThreads), 0, (cudaStream_t)stream, a);
  };
  return dtype == MT_BF16  ? run(logprobs_kernel<MT_BF16>)
         : dtype == MT_F16 ? run(logprobs_kernel<MT_F16>)
                           : run(logprobs_kernel<MT_F32>);
}
