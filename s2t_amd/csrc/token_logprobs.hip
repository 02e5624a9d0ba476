// Scores of given tokens over a row of logits (log probability, entropy, best alternatives) and their gradient.
// Semantics: include/s2t_hip.h, s2t_token_logprobs_fwd / _bwd.
#include "common.h"

namespace {

constexpr int MAX_TOP = 64;

// Statistics of a set of z: maximum, s = sum exp(z - m), t = sum exp(z - m) (z - m).  lse = m + log s, entropy = log s - t / s.
struct Stats {
  float m, s, t;
};
__device__ __forceinline__ Stats merged(Stats a, Stats b) {
  const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
  const float da = a.m - ref, db = b.m - ref, fa = __expf(da), fb = __expf(db);
  // a side that fades out contributes no t either: its s * da may be infinite (maximum -inf, or the type's lowest value)
  const float ta = fa == 0.f ? 0.f : fa * (a.t + a.s * da), tb = fb == 0.f ? 0.f : fb * (b.t + b.s * db);
  return {m, a.s * fa + b.s * fb, ta + tb};
}
struct Best {
  float v;
  int i;
};
__device__ __forceinline__ bool before(Best a, Best b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }

template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_kernel(const T* __restrict__ logits, int64_t ld, int V, const int64_t* __restrict__ tokens,
                                                             int64_t ignore, float inv_temp, int top, float* __restrict__ logprob,
                                                             float* __restrict__ lse_out, float* __restrict__ entropy,
                                                             float* __restrict__ top_lp, int64_t* __restrict__ top_idx) {
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t y = tokens ? tokens[r] : 0;
  if (tokens && y == ignore) {
    if (tid == 0) {
      if (logprob) logprob[r] = 0.f;
      if (lse_out) lse_out[r] = 0.f;
      if (entropy) entropy[r] = 0.f;
    }
    for (int k = tid; k < top; k += 256) {
      top_lp[r * top + k] = 0.f;
      top_idx[r * top + k] = -1;
    }
    return;
  }
  const T* row = logits + r * ld;
  __shared__ Stats part[4];
  __shared__ Best best[4];
  Stats st{-INFINITY, 0.f, 0.f};
  for (int c = tid; c < V; c += 256) st = merged(st, Stats{ld_as_f32<T>(row + c) * inv_temp, 1.f, 0.f});
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) st = merged(st, Stats{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.t, o, 64)});
  if (lane == 0) part[w] = st;
  __syncthreads();
  st = merged(merged(part[0], part[1]), merged(part[2], part[3]));
  const float ls = __logf(st.s), lse = st.m + ls;
  if (tid == 0) {
    if (lse_out) lse_out[r] = lse;
    if (entropy) entropy[r] = ls - st.t / st.s;
    if (logprob && tokens) logprob[r] = (uint64_t)y < (uint64_t)V ? (ld_as_f32<T>(row + y) * inv_temp - st.m) - ls : __builtin_nanf("");
  }
  Best last{INFINITY, -1};
  for (int k = 0; k < top; ++k) {
    Best b{-INFINITY, 0x7fffffff};
    for (int c = tid; c < V; c += 256) {
      const Best x{ld_as_f32<T>(row + c), c};
      if (before(last, x) && before(x, b)) b = x;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const Best x{__shfl_xor(b.v, o, 64), __shfl_xor(b.i, o, 64)};
      if (before(x, b)) b = x;
    }
    __syncthreads();
    if (lane == 0) best[w] = b;
    __syncthreads();
    b = best[0];
    for (int q = 1; q < 4; ++q)
      if (before(best[q], b)) b = best[q];
    last = b;
    if (tid == 0) {
      top_lp[r * top + k] = (b.v * inv_temp - st.m) - ls;
      top_idx[r * top + k] = b.i == 0x7fffffff ? -1 : b.i;
    }
  }
}

// d logits of one row: -p (W + g_entropy (log p + H)) / T with W = g_logprob + sum g_top, and the columns of the token and of the
// alternatives written once more with their own gradient added before the rounding.
template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(const T* __restrict__ logits, int64_t ld, int V,
                                                                 const int64_t* __restrict__ tokens, int64_t ignore, float inv_temp, int top,
                                                                 const float* __restrict__ lse, const float* __restrict__ entropy,
                                                                 const float* __restrict__ g_lp, const float* __restrict__ g_ent,
                                                                 const float* __restrict__ g_top, const int64_t* __restrict__ top_idx,
                                                                 T* __restrict__ dlogits, int64_t ldd) {
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const T* row = logits + r * ld;
  T* out = dlogits + r * ldd;
  const int64_t y = tokens ? tokens[r] : -1;
  if (tokens && y == ignore) {
    for (int c = tid; c < V; c += 256) st_from_f32<T>(out + c, 0.f);
    return;
  }
  float gl = g_lp ? g_lp[r] : 0.f;
  const float ge = g_ent ? g_ent[r] : 0.f, L = lse[r], H = g_ent ? entropy[r] : 0.f;
  if (g_lp && (uint64_t)y >= (uint64_t)V) gl = __builtin_nanf("");  // as its score
  float W = gl;
  if (g_top)
    for (int k = 0; k < top; ++k) W += g_top[r * top + k];
  auto dense = [&](int c) {
    const float lp = ld_as_f32<T>(row + c) * inv_temp - L, p = __expf(lp);
    return p == 0.f && W == W ? 0.f : -p * (W + ge * (lp + H));
  };
  for (int c = tid; c < V; c += 256) st_from_f32<T>(out + c, inv_temp * dense(c));
  __syncthreads();
  for (int k = tid; k <= (g_top ? top : 0); k += 256) {
    const int64_t c = k == 0 ? y : top_idx[r * top + k - 1];
    if ((uint64_t)c >= (uint64_t)V || (k == 0 && !g_lp)) continue;
    float add = c == y ? gl : 0.f;
    if (g_top)
      for (int q = 0; q < top; ++q)
        if (top_idx[r * top + q] == c) add += g_top[r * top + q];
    st_from_f32<T>(out + c, inv_temp * (dense((int)c) + add));
  }
}

}  // namespace

extern "C" int s2t_token_logprobs_fwd(int dtype, const void* logits, int64_t ld, int64_t rows, int V, const int64_t* tokens,
                                      int64_t ignore_index, float inv_temp, int top, float* logprob, float* lse, float* entropy,
                                      float* top_logprob, int64_t* top_index, void* stream) {
  if (rows < 0 || rows > 0x7fffffff || V <= 0 || V > 0x7fffff00 || ld < V || top < 0 || top > V) return S2T_ERR_ARG;
  if (top > MAX_TOP) return S2T_ERR_UNSUPPORTED;
  if (dtype != S2T_F32 && dtype != S2T_BF16) return S2T_ERR_DTYPE;
  if (rows == 0) return S2T_OK;  // (an empty tensor has no address)
  if (!logits || (logprob && !tokens) || (top > 0 && (!top_logprob || !top_index))) return S2T_ERR_ARG;
  const dim3 grid((unsigned)rows);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == S2T_F32)
    hipLaunchKernelGGL(token_logprobs_kernel<float>, grid, dim3(256), 0, s, (const float*)logits, ld, V, tokens, ignore_index, inv_temp, top, logprob, lse, entropy, top_logprob, top_index);
  else
    hipLaunchKernelGGL(token_logprobs_kernel<bf16_t>, grid, dim3(256), 0, s, (const bf16_t*)logits, ld, V, tokens, ignore_index, inv_temp, top, logprob, lse, entropy, top_logprob, top_index);
  return S2T_LAUNCH_CHECK();
}

extern "C" int s2t_token_logprobs_bwd(int dtype, const void* logits, int64_t ld, int64_t rows, int V, const int64_t* tokens,
                                      int64_t ignore_index, float inv_temp, int top, const float* lse, const float* entropy,
                                      const float* g_logprob, const float* g_entropy, const float* g_top, const int64_t* top_index,
                                      void* dlogits, int64_t ldd, void* stream) {
  if (rows < 0 || rows > 0x7fffffff || V <= 0 || V > 0x7fffff00 || ld < V || ldd < V || top < 0 || top > V) return S2T_ERR_ARG;
  if (top > MAX_TOP) return S2T_ERR_UNSUPPORTED;
  if (dtype != S2T_F32 && dtype != S2T_BF16) return S2T_ERR_DTYPE;
  if (rows == 0) return S2T_OK;
  if (!logits || !dlogits || !lse || (g_logprob && !tokens) || (g_entropy && !entropy) || (g_top && (!top_index || top == 0))) return S2T_ERR_ARG;
  const dim3 grid((unsigned)rows);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == S2T_F32)
    hipLaunchKernelGGL(token_logprobs_bwd_kernel<float>, grid, dim3(256), 0, s, (const float*)logits, ld, V, tokens, ignore_index, inv_temp, top, lse, entropy, g_logprob, g_entropy, g_top, top_index, (float*)dlogits, ldd);
  else
    hipLaunchKernelGGL(token_logprobs_bwd_kernel<bf16_t>, grid, dim3(256), 0, s, (const bf16_t*)logits, ld, V, tokens, ignore_index, inv_temp, top, lse, entropy, g_logprob, g_entropy, g_top, top_index, (bf16_t*)dlogits, ldd);
  return S2T_LAUNCH_CHECK();
}
