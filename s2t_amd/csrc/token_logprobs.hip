// Scores of given tokens over a row of logits (log probability, entropy, best alternatives) and their gradient.
// Semantics: include/s2t_hip.h, s2t_token_logprobs_fwd / _bwd.
#include <type_traits>

#include "common.h"

namespace {

constexpr int MAX_TOP = 64;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// Statistics of a set of logits in powers of two, c2 = log2(e) / T: maximum m, s = sum 2^d, t = sum 2^d d with d = c2 (x - m).
// log p = (d - log2 s) ln 2, entropy = (log2 s - t / s) ln 2.  The difference is taken of the logits as they are: m is one of them, so that
// rows of numbers far from zero (all of the type's lowest value, or around 10^30) lose nothing; and the backward pass is handed m and log2 s,
// not their sum, which would hide log2 s behind a large m.
struct Stats {
  float m, s, t;
};
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ Stats merged(Stats a, Stats b, float c2) {
  const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
  const float da = (a.m - ref) * c2, db = (b.m - ref) * c2, fa = exp2_(da), fb = exp2_(db);
  // a side that fades out contributes no t either: its s * da may be infinite (maximum -inf, or the type's lowest value)
  const float ta = fa == 0.f ? 0.f : fa * (a.t + a.s * da), tb = fb == 0.f ? 0.f : fb * (b.t + b.s * db);
  return {m, a.s * fa + b.s * fb, ta + tb};
}

// 16 bytes of a row at any element's address (the hardware takes them there)
struct __attribute__((packed, aligned(2))) Vec {
  uint32_t w[4];
};
template <typename T>
constexpr int EPV = 16 / (int)sizeof(T);
template <typename T>
__device__ __forceinline__ void unpack(const Vec& v, float (&x)[EPV<T>]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (sizeof(T) == 2) {
      x[2 * q] = __uint_as_float(v.w[q] << 16);
      x[2 * q + 1] = __uint_as_float(v.w[q] & 0xffff0000u);
    } else x[q] = __uint_as_float(v.w[q]);
  }
}

struct Best {
  float v;
  int i;
};
__device__ __forceinline__ bool before(Best a, Best b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }

// log p_y = z_y - lse, H = -sum p log p and the best columns from one read of the row: bound by its bytes (8192 x 10000 bf16 with entropy:
// 143 MB of rows that are not ignored in 27 us, 5.3 TB/s; 35 behind a kernel that has written 164 MB, whose lines go out as these come in,
// 43 behind the backward pass; 2047 x 32001 fp32 with 8 alternatives: 230 MB in 48 us, 4.8 TB/s).
// One workgroup to a row, one pass: every thread keeps the statistics of its vectors (relative to its own running maximum, moved once
// for each NB vectors) and, for the alternatives, the maximum of its raw logits.  The top-th largest of the 64 maxima of every 64th thread
// each bounds the alternatives from below, since as many columns reach it; the columns of the threads that reach it are read once more
// (from the caches, dealt to all threads), those that reach it are collected and ranked by (logit, column).  Of independent logits 11 columns
// reach the bound of 10 alternatives, 45 that of 32 and 90 that of 48; at 64 it is the least of the maxima, which 300 reach.  Rows with more than
// CAND such columns (ties without end; 2 of 100 rows at 64) are ranked one column after the other instead (8192 x 10000 bf16 with 0, 10, 32,
// 48 and 64 alternatives: 31, 41, 48, 68 and 700 us).
constexpr int CAND = 512;
template <typename T, int THREADS, bool TOP, bool ENTROPY>
__global__ __launch_bounds__(THREADS) void token_logprobs_kernel(const T* __restrict__ logits, int64_t ld, int V, const int64_t* __restrict__ tokens,
                                                                 int64_t ignore, float inv_temp, int top, float* __restrict__ logprob,
                                                                 float2* __restrict__ stats, float* __restrict__ entropy,
                                                                 float* __restrict__ top_lp, int64_t* __restrict__ top_idx) {
  constexpr int E = EPV<T>, NB = 5, WAVES = THREADS / 64;  // (five vectors of 256 threads: a row of 10 000 bf16 logits in one go)
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t y = tokens ? tokens[r] : 0;
  if (tokens && y == ignore) {
    if (tid == 0) {
      if (logprob) logprob[r] = 0.f;
      if (stats) stats[r] = make_float2(0.f, 0.f);
      if (ENTROPY) entropy[r] = 0.f;
    }
    if (TOP)
      for (int k = tid; k < top; k += THREADS) {
        top_lp[r * top + k] = 0.f;
        top_idx[r * top + k] = -1;
      }
    return;
  }
  const T* row = logits + r * ld;
  const float c2 = inv_temp * LOG2E;
  const int nvec = V / E, tail = nvec * E + tid;  // thread `tid`: vectors tid, tid + THREADS .., and one of the V % E last columns
  Stats st{-INFINITY, 0.f, 0.f};
  float most = -INFINITY;
  // N columns: the maximum first, so that the sums are moved once for all of them
  auto take = [&](const auto& x) __attribute__((always_inline)) {
    constexpr int N = sizeof(x) / sizeof(float);
    float hi = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) hi = fmaxf(hi, x[e]);
    if (TOP) most = fmaxf(most, hi);
    if (hi > st.m) {
      const float d = (st.m - hi) * c2, f = exp2_(d);
      st.t = ENTROPY && f != 0.f ? f * (st.t + st.s * d) : 0.f;
      st.s *= f;
      st.m = hi;
    }
    const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = (x[e] - ref) * c2, p = exp2_(d);
      st.s += p;
      if (ENTROPY) st.t = fmaf(p, fmaxf(d, -1e3f), st.t);  // (a column of -inf: 0 * -1e3)
    }
  };
  for (int v0 = tid; v0 < nvec; v0 += THREADS * NB) {
    Vec buf[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u) buf[u] = *reinterpret_cast<const Vec*>(row + (int64_t)min(v0 + u * THREADS, nvec - 1) * E);
    float x[NB * E];
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      if (v0 + u * THREADS >= nvec)  // -inf: adds nothing
#pragma unroll
        for (int q = 0; q < 4; ++q) buf[u].w[q] = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
      float y8[E];
      unpack<T>(buf[u], y8);
#pragma unroll
      for (int e = 0; e < E; ++e) x[u * E + e] = y8[e];
    }
    take(x);
  }
  if (tail < V) {
    const float x[1] = {ld_as_f32<T>(row + tail)};
    take(x);
  }
  __shared__ Stats part[WAVES];
  __shared__ float maxima[TOP ? THREADS : 1];
  __shared__ Best cand[TOP ? CAND : 1];
  __shared__ int winner[TOP ? THREADS : 1];
  __shared__ int n_cand, n_win;
  {  // of a wave: the common maximum, then sums
    const float m = wave_max(st.m), ref = m == -INFINITY ? 0.f : m, d = (st.m - ref) * c2, f = exp2_(d);
    const float sum = wave_sum(st.s * f);
    st.t = ENTROPY ? wave_sum(f == 0.f ? 0.f : f * (st.t + st.s * d)) : 0.f;
    st.s = sum;
    st.m = m;
  }
  if (lane == 0) part[w] = st;
  if (TOP) maxima[tid] = most;
  if (tid == 0) n_cand = n_win = 0;
  __syncthreads();
  st = part[0];
#pragma unroll
  for (int q = 1; q < WAVES; ++q) st = merged(st, part[q], c2);
  const float l2 = log2f(st.s);
  auto score = [&](float x) { return fmaf(x - st.m, inv_temp, -l2 * LN2); };  // (in nats: c2 times a difference that fp32 just holds is infinite)
  if (tid == 0) {
    if (stats) stats[r] = make_float2(st.m, l2);
    if (ENTROPY) entropy[r] = (l2 - st.t / st.s) * LN2;
    if (logprob) logprob[r] = (uint64_t)y < (uint64_t)V ? score(ld_as_f32<T>(row + y)) : __builtin_nanf("");
  }
  if constexpr (TOP) {
    // the bound: the largest of the 64 that `top` of them reach; every wave finds it for itself
    float mine = maxima[lane];
#pragma unroll
    for (int q = 1; q < WAVES; ++q) mine = fmaxf(mine, maxima[q * 64 + lane]);
    int reach = 0;
#pragma unroll
    for (int q = 0; q < 64; ++q) reach += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine), q)) >= mine ? 1 : 0;
    const float bound = wave_max(reach >= top ? mine : -INFINITY);
    auto offer = [&](float v, int i) {
      if (v >= bound) {
        const int at = atomicAdd(&n_cand, 1);
        if (at < CAND) cand[at] = Best{v, i};
      }
    };
    if (most >= bound) winner[atomicAdd(&n_win, 1)] = tid;
    if (tail < V) offer(ld_as_f32<T>(row + tail), tail);
    __syncthreads();
    // the vectors of the threads that reach it, dealt to all threads: each of them one load
    const int of_one = (nvec + THREADS - 1) / THREADS, all = n_win * of_one;
    for (int q = tid; q < all; q += THREADS) {
      const int v = winner[q / of_one] + q % of_one * THREADS;
      if (v < nvec) {
        float x[E];
        unpack<T>(*reinterpret_cast<const Vec*>(row + (int64_t)v * E), x);
#pragma unroll
        for (int e = 0; e < E; ++e) offer(x[e], v * E + e);
      }
    }
    __syncthreads();
    const int n = n_cand;
    auto put = [&](int k, Best x) {
      top_lp[r * top + k] = score(x.v);
      top_idx[r * top + k] = x.i;
    };
    if (n <= CAND) {  // (the order in which they were collected does not matter: no two columns rank alike)
      for (int j = tid; j < n; j += THREADS) {
        const Best x = cand[j];
        int rank = 0;
        for (int q = 0; q < n; ++q) rank += before(cand[q], x) ? 1 : 0;
        if (rank < top) put(rank, x);
      }
      for (int k = n + tid; k < top; k += THREADS) put(k, Best{__builtin_nanf(""), -1});  // (only NaN left)
    } else {
      Best last{INFINITY, -1};
      for (int k = 0; k < top; ++k) {
        Best b{-INFINITY, 0x7fffffff};
        for (int c = tid; c < V; c += THREADS) {
          const Best x{ld_as_f32<T>(row + c), c};
          if (before(last, x) && before(x, b)) b = x;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
          const Best x{__shfl_xor(b.v, o, 64), __shfl_xor(b.i, o, 64)};
          if (before(x, b)) b = x;
        }
        __syncthreads();
        if (lane == 0) cand[w] = b;
        __syncthreads();
        b = cand[0];
        for (int q = 1; q < WAVES; ++q)
          if (before(cand[q], b)) b = cand[q];
        last = b;
        if (tid == 0) put(k, b);
      }
    }
  }
}

// Bound by its bytes: 8192 x 10000 bf16 read (143 MB) and written (164 MB) in 50 us.
// d logits of one row: -p (W + g_entropy (log p + H)) / T with W = g_logprob + sum g_top; the thread that stored the column of the token or of
// an alternative stores it once more with its own gradient added before the rounding.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void token_logprobs_bwd_kernel(const T* __restrict__ logits, int64_t ld, int V,
                                                                 const int64_t* __restrict__ tokens, int64_t ignore, float inv_temp, int top,
                                                                 const float2* __restrict__ stats, const float* __restrict__ entropy,
                                                                 const float* __restrict__ g_lp, const float* __restrict__ g_ent,
                                                                 const float* __restrict__ g_top, const int64_t* __restrict__ top_idx,
                                                                 T* __restrict__ dlogits, int64_t ldd) {
  constexpr int E = EPV<T>, NB = 5;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const T* row = logits + r * ld;
  T* out = dlogits + r * ldd;
  const int nvec = V / E, tail = nvec * E + tid;
  const int64_t y = tokens ? tokens[r] : -1;
  if (tokens && y == ignore) {
    for (int v = tid; v < nvec; v += THREADS) *reinterpret_cast<Vec*>(out + (int64_t)v * E) = Vec{{0, 0, 0, 0}};
    if (tail < V) st_from_f32<T>(out + tail, 0.f);
    return;
  }
  float gl = g_lp ? g_lp[r] : 0.f;
  const float ge = g_ent ? g_ent[r] : 0.f, H = g_ent ? entropy[r] : 0.f;
  if (g_lp && (uint64_t)y >= (uint64_t)V) gl = __builtin_nanf("");  // as its score
  float W = gl;
  if (g_top)
    for (int k = 0; k < top; ++k) W += g_top[r * top + k];
  const float c2 = inv_temp * LOG2E, gw = W + ge * H, gp = ge * LN2;
  const float2 st = stats[r];
  // (a column of -inf: p is 0, and so is its gradient)
  auto dense = [&](float x) {
    const float lp = fmaf(x - st.x, c2, -st.y);
    return -exp2_(lp) * fmaf(gp, fmaxf(lp, -1e3f), gw);
  };
  for (int v0 = tid; v0 < nvec; v0 += THREADS * NB) {
    Vec buf[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u) buf[u] = *reinterpret_cast<const Vec*>(row + (int64_t)min(v0 + u * THREADS, nvec - 1) * E);
#pragma unroll
    for (int u = 0; u < NB; ++u)
      if (v0 + u * THREADS < nvec) {
        float x[E];
        unpack<T>(buf[u], x);
        Vec o;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (sizeof(T) == 2) o.w[q] = bf16pack(inv_temp * dense(x[2 * q]), inv_temp * dense(x[2 * q + 1]));
          else o.w[q] = __float_as_uint(inv_temp * dense(x[q]));
        }
        *reinterpret_cast<Vec*>(out + (int64_t)(v0 + u * THREADS) * E) = o;
      }
  }
  if (tail < V) st_from_f32<T>(out + tail, inv_temp * dense(ld_as_f32<T>(row + tail)));
  for (int k = 0; k <= (g_top ? top : 0); ++k) {
    const int64_t c = k == 0 ? y : top_idx[r * top + k - 1];
    if ((uint64_t)c >= (uint64_t)V || (k == 0 && !g_lp)) continue;
    if (tid != (c < (int64_t)nvec * E ? (int)(c / E % THREADS) : (int)(c - (int64_t)nvec * E))) continue;
    float add = c == y ? gl : 0.f;
    if (g_top)
      for (int q = 0; q < top; ++q)
        if (top_idx[r * top + q] == c) add += g_top[r * top + q];
    st_from_f32<T>(out + c, inv_temp * (dense(ld_as_f32<T>(row + c)) + add));
  }
}

// Threads of a row: five vectors each take all of a row of up to 5, 10 and 20 KB at once, and short rows leave room for many workgroups on a
// compute unit (8000 x 2500 bf16 with 10 alternatives: 36 us with 256 threads, 18 with 64; 8000 x 5000: 36 and, with 128, 24; 2047 x 32001
// fp32: 53 with 256, 50 with 512; 8192 x 10000 bf16: 28 with 256, 46 with 512).
template <typename F>
void for_threads(int64_t row_bytes, F&& f) {
  if (row_bytes <= 5120) f(std::integral_constant<int, 64>{});
  else if (row_bytes <= 10240) f(std::integral_constant<int, 128>{});
  else if (row_bytes <= 65536) f(std::integral_constant<int, 256>{});
  else f(std::integral_constant<int, 512>{});
}

template <typename T>
void launch_fwd(const void* logits, int64_t ld, int64_t rows, int V, const int64_t* tokens, int64_t ignore, float inv_temp, int top, float* logprob,
                float2* stats, float* entropy, float* top_lp, int64_t* top_idx, hipStream_t s) {
  for_threads((int64_t)V * sizeof(T), [&](auto n) {
    constexpr int THREADS = decltype(n)::value;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(THREADS), 0, s, (const T*)logits, ld, V, tokens, ignore, inv_temp, top, logprob, stats, entropy, top_lp, top_idx);
    };
    if (top > 0) {
      if (entropy) go(token_logprobs_kernel<T, THREADS, true, true>);
      else go(token_logprobs_kernel<T, THREADS, true, false>);
    } else {
      if (entropy) go(token_logprobs_kernel<T, THREADS, false, true>);
      else go(token_logprobs_kernel<T, THREADS, false, false>);
    }
  });
}
template <typename T>
void launch_bwd(const void* logits, int64_t ld, int64_t rows, int V, const int64_t* tokens, int64_t ignore, float inv_temp, int top, const float2* stats,
                const float* entropy, const float* g_lp, const float* g_ent, const float* g_top, const int64_t* top_idx, void* dlogits, int64_t ldd, hipStream_t s) {
  for_threads((int64_t)V * sizeof(T), [&](auto n) {
    constexpr int THREADS = decltype(n)::value;
    hipLaunchKernelGGL((token_logprobs_bwd_kernel<T, THREADS>), dim3((unsigned)rows), dim3(THREADS), 0, s, (const T*)logits, ld, V, tokens, ignore, inv_temp, top, stats, entropy, g_lp, g_ent, g_top, top_idx, (T*)dlogits, ldd);
  });
}

}  // namespace

extern "C" int s2t_token_logprobs_fwd(int dtype, const void* logits, int64_t ld, int64_t rows, int V, const int64_t* tokens,
                                      int64_t ignore_index, float inv_temp, int top, float* logprob, float* stats, float* entropy,
                                      float* top_logprob, int64_t* top_index, void* stream) {
  if (rows < 0 || rows > 0x7fffffff || V <= 0 || V > 0x7fffff00 || ld < V || top < 0 || top > V) return S2T_ERR_ARG;
  if (top > MAX_TOP) return S2T_ERR_UNSUPPORTED;
  if (dtype != S2T_F32 && dtype != S2T_BF16) return S2T_ERR_DTYPE;
  if (rows == 0) return S2T_OK;  // (an empty tensor has no address)
  if (!logits || ((uintptr_t)stats & 7) || (logprob && !tokens) || (top > 0 && (!top_logprob || !top_index))) return S2T_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == S2T_F32) launch_fwd<float>(logits, ld, rows, V, tokens, ignore_index, inv_temp, top, logprob, (float2*)stats, entropy, top_logprob, top_index, s);
  else launch_fwd<bf16_t>(logits, ld, rows, V, tokens, ignore_index, inv_temp, top, logprob, (float2*)stats, entropy, top_logprob, top_index, s);
  return S2T_LAUNCH_CHECK();
}

extern "C" int s2t_token_logprobs_bwd(int dtype, const void* logits, int64_t ld, int64_t rows, int V, const int64_t* tokens,
                                      int64_t ignore_index, float inv_temp, int top, const float* stats, const float* entropy,
                                      const float* g_logprob, const float* g_entropy, const float* g_top, const int64_t* top_index,
                                      void* dlogits, int64_t ldd, void* stream) {
  if (rows < 0 || rows > 0x7fffffff || V <= 0 || V > 0x7fffff00 || ld < V || ldd < V || top < 0 || top > V) return S2T_ERR_ARG;
  if (top > MAX_TOP) return S2T_ERR_UNSUPPORTED;
  if (dtype != S2T_F32 && dtype != S2T_BF16) return S2T_ERR_DTYPE;
  if (rows == 0) return S2T_OK;
  if (!logits || !dlogits || !stats || ((uintptr_t)stats & 7) || (g_logprob && !tokens) || (g_entropy && !entropy) || (g_top && (!top_index || top == 0))) return S2T_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == S2T_F32) launch_bwd<float>(logits, ld, rows, V, tokens, ignore_index, inv_temp, top, (const float2*)stats, entropy, g_logprob, g_entropy, g_top, top_index, dlogits, ldd, s);
  else launch_bwd<bf16_t>(logits, ld, rows, V, tokens, ignore_index, inv_temp, top, (const float2*)stats, entropy, g_logprob, g_entropy, g_top, top_index, dlogits, ldd, s);
  return S2T_LAUNCH_CHECK();
}
