// Paged key/value cache of an incremental decoder: append (with rotary positions on the way) and attention of several new tokens of a
// sequence over it, chain or tree of drafts.  Layout, bounds and semantics: include/s2t_hip.h, s2t_paged_args.
#include "common.h"

namespace {

// place -> element offset of (page, place in page), or -1 where the table does not lead to a page
struct Pages {
  const int32_t* table;  // this sequence's row
  int shift, mask, n_table, num_pages;
  int64_t sp, sr;
  __device__ __forceinline__ int64_t at(int place) const {
    const int i = place >> shift;
    if (place < 0 || i >= n_table) return -1;
    const int p = table[i];
    return (uint32_t)p < (uint32_t)num_pages ? p * sp + (place & mask) * sr : -1;
  }
};
__device__ __forceinline__ Pages pages_of(const s2t_paged_args& a, int shift, int b) {
  return {a.page_table + b * a.table_stride, shift, a.page_size - 1, a.table_pages, a.num_pages, a.p_sp, a.p_sr};
}
// the rows of sequence b: first row, number of them (bounded by N), length of its cache (bounded by the table)
struct Span {
  int row0, n, len;
};
__device__ __forceinline__ Span span_of(const s2t_paged_args& a, int b) {
  const int r0 = min(max(a.cu[b], 0), a.N), r1 = min(max(a.cu[b + 1], 0), a.N);
  return {r0, max(r1 - r0, 0), a.lens[b]};
}

// ---- append -----------------------------------------------------------------------------------------------------------------
// One workgroup per new token; a thread moves 16 bytes (two times 16 where elements turn in pairs).
template <typename T>
__global__ __launch_bounds__(256) void paged_append_kernel(const s2t_paged_args a, int shift) {
  const int b = blockIdx.y, i = blockIdx.x;
  const Span s = span_of(a, b);
  if (i >= s.n) return;
  const int t = s.row0 + i, place = s.len - s.n + i;
  const int64_t to = pages_of(a, shift, b).at(place);
  constexpr int E = 16 / (int)sizeof(T);
  const int rot = a.rotary ? a.rot_dim : 0, half = rot / 2;
  const int pos = a.positions ? a.positions[t] : place;
  const bool known = (uint32_t)pos < (uint32_t)a.rotary_positions;
  const float* cs = a.rotary + (int64_t)(known ? pos : 0) * rot;
  const int row = a.rows ? a.rows[t] : t;
  const bool stored = to >= 0 && (!a.rows || (uint32_t)row < (uint32_t)a.src_rows);
  // units of a head: `half / E` pairs of vectors that turn together, then the vectors that pass
  const int pairs = half / E, units = pairs + (a.dk - rot) / E;
  auto turn = [&](const T* src, T* dst, int u) {
    if (u >= pairs) {
      const int c = rot + (u - pairs) * E;
      *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
      return;
    }
    float x[E], y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[e] = ld_as_f32<T>(src + u * E + e);
      y[e] = ld_as_f32<T>(src + half + u * E + e);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float c = known ? cs[u * E + e] : __builtin_nanf(""), sn = known ? cs[half + u * E + e] : __builtin_nanf("");
      st_from_f32<T>(dst + u * E + e, x[e] * c - y[e] * sn);
      st_from_f32<T>(dst + half + u * E + e, y[e] * c + x[e] * sn);
    }
  };
  if (stored) {
    for (int w = threadIdx.x; w < a.kv_heads * units; w += 256) {
      const int h = w / units, u = w % units;
      turn((const T*)a.k + row * a.k_st + h * a.k_sh, (T*)a.k_pages + to + h * a.p_sh, u);
    }
    const int vecs = a.dk / E;
    for (int w = threadIdx.x; w < a.kv_heads * vecs; w += 256) {
      const int h = w / vecs, c = (w % vecs) * E;
      *reinterpret_cast<uint4*>((T*)a.v_pages + to + h * a.p_sh + c) =
          *reinterpret_cast<const uint4*>((const T*)a.v + row * a.v_st + h * a.v_sh + c);
    }
  }
  if (a.q) {
    for (int w = threadIdx.x; w < a.q_heads * units; w += 256) {
      const int h = w / units, u = w % units;
      turn((const T*)a.q + t * a.q_st + h * a.q_sh, (T*)a.q_out + t * a.qo_st + h * a.qo_sh, u);
    }
  }
}

// ---- attention --------------------------------------------------------------------------------------------------------------
// One wave per (new token, query head): a lane scores one key of each 64, the running maximum and sum are the wave's, and every lane
// keeps dk / 64 columns of the output.
template <typename T>
__global__ __launch_bounds__(64) void paged_attention_kernel(const s2t_paged_args a, int shift) {
  const int b = blockIdx.z, h = blockIdx.y, i = blockIdx.x, lane = threadIdx.x;
  const Span s = span_of(a, b);
  if (i >= s.n) return;
  const int t = s.row0 + i, prefix = s.len - s.n;
  const int64_t kvh = (int64_t)(h / (a.q_heads / a.kv_heads)) * a.p_sh;
  const Pages pg = pages_of(a, shift, b);
  const int len = (int)min((int64_t)s.len, (int64_t)a.table_pages << shift);
  __shared__ float qs[256];
  for (int c = lane; c < a.dk; c += 64) qs[c] = ld_as_f32<T>((const T*)a.q + t * a.q_st + h * a.q_sh + c) * a.scale;
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < len; k0 += 64) {
    const int key = k0 + lane, j = key - prefix;
    bool sees = key < len;
    if (j >= 0) {
      if (a.tree) sees = sees && j < 64 * a.tree_words && ((a.tree[t * a.tree_stride + (j >> 6)] >> (j & 63)) & 1);
      else sees = sees && j <= i;
    }
    const int64_t at = sees ? pg.at(key) : -1;
    float sc = -INFINITY;
    if (at >= 0) {
      const T* kr = (const T*)a.k_pages + at + kvh;
      sc = 0.f;
      for (int c = 0; c < a.dk; ++c) sc += qs[c] * ld_as_f32<T>(kr + c);
    }
    const float mn = fmaxf(m, wave_max(sc)), ref = mn == -INFINITY ? 0.f : mn;
    const float p = at >= 0 ? __expf(sc - ref) : 0.f, fade = __expf(m - ref);
    m = mn;
    l = l * fade + wave_sum(p);
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] *= fade;
    for (int u = 0; u < 64; ++u) {
      const int64_t au = __shfl(at, u, 64);
      if (au < 0) continue;
      const float pu = __shfl(p, u, 64);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r * 64 + lane < a.dk) o[r] += pu * ld_as_f32<T>((const T*)a.v_pages + au + kvh + r * 64 + lane);
    }
  }
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (r * 64 + lane < a.dk) st_from_f32<T>((T*)a.out + t * a.o_st + h * a.o_sh + r * 64 + lane, m == -INFINITY ? 0.f : o[r] * inv);
  if (a.lse && lane == 0) a.lse[(int64_t)t * a.q_heads + h] = m == -INFINITY ? -INFINITY : m + __logf(l);
}

int paged_args_bad(const s2t_paged_args* a) {
  if (!a || !a->k_pages || !a->v_pages || !a->page_table || !a->lens || !a->cu) return S2T_ERR_ARG;
  if (a->dtype != S2T_F32 && a->dtype != S2T_BF16) return S2T_ERR_DTYPE;
  if (a->B <= 0 || a->B > 65535 || a->N < 0 || a->max_new < 0 || a->q_heads <= 0 || a->kv_heads <= 0 || a->q_heads % a->kv_heads) return S2T_ERR_ARG;
  if (a->num_pages <= 0 || a->table_pages <= 0 || a->page_size <= 0 || (a->page_size & (a->page_size - 1))) return S2T_ERR_ARG;
  if ((int64_t)a->table_pages * a->page_size > 0x7fffff00ll) return S2T_ERR_UNSUPPORTED;  // places are 32-bit numbers
  if (a->dk <= 0 || a->dk % 16 || a->dk > 256) return S2T_ERR_UNSUPPORTED;
  return S2T_OK;
}
bool misaligned(const s2t_paged_args* a, const void* p, int64_t st, int64_t sh) {
  const int e = a->dtype == S2T_F32 ? 4 : 8;  // elements of 16 bytes
  return ((uintptr_t)p & 15) || st % e || sh % e;
}
int shift_of(const s2t_paged_args* a) { return __builtin_ctz((unsigned)a->page_size); }

}  // namespace

extern "C" int s2t_paged_kv_append(const s2t_paged_args* a, void* stream) {
  if (int bad = paged_args_bad(a)) return bad;
  if ((a->q && a->rows) || (a->rows && a->src_rows < 0)) return S2T_ERR_ARG;
  if (a->rotary && (a->rot_dim <= 0 || a->rot_dim % 16 || a->rot_dim > a->dk || a->rotary_positions <= 0)) return S2T_ERR_ARG;
  if (misaligned(a, a->k_pages, a->p_sp, a->p_sh) || misaligned(a, a->v_pages, a->p_sr, 0) || misaligned(a, a->k, a->k_st, a->k_sh) ||
      misaligned(a, a->v, a->v_st, a->v_sh) || (a->q && (misaligned(a, a->q, a->q_st, a->q_sh) || misaligned(a, a->q_out, a->qo_st, a->qo_sh))) ||
      ((uintptr_t)a->rotary & 15))
    return S2T_ERR_ALIGN;
  if (a->N == 0 || a->max_new == 0 || (a->rows && a->src_rows == 0)) return S2T_OK;  // (an empty tensor has no address)
  if (!a->k || !a->v || (a->q && !a->q_out)) return S2T_ERR_ARG;
  const dim3 grid((unsigned)a->max_new, (unsigned)a->B);
  if (a->dtype == S2T_F32) hipLaunchKernelGGL(paged_append_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, *a, shift_of(a));
  else hipLaunchKernelGGL(paged_append_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, *a, shift_of(a));
  return S2T_LAUNCH_CHECK();
}

extern "C" int64_t s2t_paged_attention_ws_bytes(const s2t_paged_args* a) { return paged_args_bad(a) ? -1 : 0; }

extern "C" int s2t_paged_attention(const s2t_paged_args* a, void* stream) {
  if (int bad = paged_args_bad(a)) return bad;
  if ((a->tree && a->tree_words <= 0) || a->q_heads > 65535) return S2T_ERR_ARG;
  if (misaligned(a, a->k_pages, a->p_sp, a->p_sh) || misaligned(a, a->v_pages, a->p_sr, 0) || misaligned(a, a->q, a->q_st, a->q_sh) ||
      misaligned(a, a->out, a->o_st, a->o_sh) || ((uintptr_t)a->tree & 7))
    return S2T_ERR_ALIGN;
  if (a->N == 0 || a->max_new == 0) return S2T_OK;
  if (!a->q || !a->out) return S2T_ERR_ARG;
  const dim3 grid((unsigned)a->max_new, (unsigned)a->q_heads, (unsigned)a->B);
  if (a->dtype == S2T_F32) hipLaunchKernelGGL(paged_attention_kernel<float>, grid, dim3(64), 0, (hipStream_t)stream, *a, shift_of(a));
  else hipLaunchKernelGGL(paged_attention_kernel<bf16_t>, grid, dim3(64), 0, (hipStream_t)stream, *a, shift_of(a));
  return S2T_LAUNCH_CHECK();
}
