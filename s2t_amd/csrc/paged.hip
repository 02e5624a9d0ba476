// Paged key/value cache of an incremental decoder: append (with rotary positions on the way) and attention of several new tokens of a
// sequence over it, chain or tree of drafts.  Layout, bounds and semantics: include/s2t_hip.h, s2t_paged_args.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace {

// Table, lens, cu and the like are uniform over a wave and only read here: through the constant address space they come by scalar loads,
// which do not queue behind the vector loads of keys and values.
typedef const __attribute__((address_space(4))) int32_t* Entries;

// place -> element offset of (page, place in page), or -1 where the table does not lead to a page
struct Pages {
  const int32_t* table;  // this sequence's row
  int shift, mask, n_table, num_pages;
  int64_t sp, sr;
  __device__ __forceinline__ int64_t at(int place) const {
    const int i = place >> shift;
    if (place < 0 || i >= n_table) return -1;
    const int p = ((Entries)table)[i];
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
  const Entries cu = (Entries)a.cu;
  const int r0 = min(max(cu[b], 0), a.N), r1 = min(max(cu[b + 1], 0), a.N);
  return {r0, max(r1 - r0, 0), ((Entries)a.lens)[b]};
}

// ---- append -----------------------------------------------------------------------------------------------------------------
// A wave takes a new token; its lanes go over the token's units: 16 bytes that pass, or two times 16 that turn together, first all of k, then
// v, then q.  (Bound by memory, and kept busy by many small waves: two, four and eight tokens to a wave, with as many loads of each
// lane on their way, were slower, 48, 57 and 63 us against 42 for 17 000 tokens of 4 + 4 + 16 heads x 128 in bf16, 210 MB: 5.0 TB/s.)
template <typename T>
struct Turned {
  static constexpr int E = 16 / (int)sizeof(T);
  // (x, y) -> (x cos - y sin, y cos + x sin), cs: cosines of this unit, sines `half` floats behind; rounded once
  static __device__ __forceinline__ void turn(uint4& xv, uint4& yv, const float* cs, int half, bool known) {
    uint32_t* xw = reinterpret_cast<uint32_t*>(&xv);
    uint32_t* yw = reinterpret_cast<uint32_t*>(&yv);
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      float4 c = reinterpret_cast<const float4*>(cs)[q], s = reinterpret_cast<const float4*>(cs + half)[q];
      if (!known) c.x = c.y = c.z = c.w = __builtin_nanf("");  // NaN both ways: x nan - y s, y nan + x s
      if constexpr (sizeof(T) == 2) {
        const float x0 = __uint_as_float(xw[2 * q] << 16), x1 = __uint_as_float(xw[2 * q] & 0xffff0000u);
        const float x2 = __uint_as_float(xw[2 * q + 1] << 16), x3 = __uint_as_float(xw[2 * q + 1] & 0xffff0000u);
        const float y0 = __uint_as_float(yw[2 * q] << 16), y1 = __uint_as_float(yw[2 * q] & 0xffff0000u);
        const float y2 = __uint_as_float(yw[2 * q + 1] << 16), y3 = __uint_as_float(yw[2 * q + 1] & 0xffff0000u);
        xw[2 * q] = bf16pack(x0 * c.x - y0 * s.x, x1 * c.y - y1 * s.y);
        xw[2 * q + 1] = bf16pack(x2 * c.z - y2 * s.z, x3 * c.w - y3 * s.w);
        yw[2 * q] = bf16pack(y0 * c.x + x0 * s.x, y1 * c.y + x1 * s.y);
        yw[2 * q + 1] = bf16pack(y2 * c.z + x2 * s.z, y3 * c.w + x3 * s.w);
      } else {
        const float x0 = __uint_as_float(xw[0]), x1 = __uint_as_float(xw[1]), x2 = __uint_as_float(xw[2]), x3 = __uint_as_float(xw[3]);
        const float y0 = __uint_as_float(yw[0]), y1 = __uint_as_float(yw[1]), y2 = __uint_as_float(yw[2]), y3 = __uint_as_float(yw[3]);
        xw[0] = __float_as_uint(x0 * c.x - y0 * s.x);
        xw[1] = __float_as_uint(x1 * c.y - y1 * s.y);
        xw[2] = __float_as_uint(x2 * c.z - y2 * s.z);
        xw[3] = __float_as_uint(x3 * c.w - y3 * s.w);
        yw[0] = __float_as_uint(y0 * c.x + x0 * s.x);
        yw[1] = __float_as_uint(y1 * c.y + x1 * s.y);
        yw[2] = __float_as_uint(y2 * c.z + x2 * s.z);
        yw[3] = __float_as_uint(y3 * c.w + x3 * s.w);
      }
    }
  }
};

template <typename T>
__global__ __launch_bounds__(256) void paged_append_kernel(const s2t_paged_args a, const int shift, const uint32_t by_units, const uint32_t by_vecs) {
  constexpr int E = Turned<T>::E;
  const int b = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = blockIdx.x * 4 + wave;
  const Span s = span_of(a, b);
  if (i >= min(s.n, a.max_new)) return;
  const int rot = a.rotary ? a.rot_dim : 0, half = rot / 2;
  const int pairs = half / E, units = pairs + (a.dk - rot) / E, vecs = a.dk / E;
  const int nk = a.kv_heads * units, nv = a.kv_heads * vecs, nq = a.q ? a.q_heads * units : 0;
  const int t = s.row0 + i, place = s.len - s.n + i;
  const int64_t to = pages_of(a, shift, b).at(place);
  const int row = a.rows ? ((Entries)a.rows)[t] : t, pos = a.positions ? ((Entries)a.positions)[t] : place;
  const bool there = !a.rows || (uint32_t)row < (uint32_t)a.src_rows, stored = to >= 0 && there;
  const bool known = (uint32_t)pos < (uint32_t)a.rotary_positions;
  const float* cs = a.rotary + (int64_t)(known ? pos : 0) * rot;
  for (int u = threadIdx.x & 63; u < nk + nv + nq; u += 64) {
    // what this unit is
    const bool is_v = u >= nk && u < nk + nv, is_q = u >= nk + nv;
    const int w = is_q ? u - nk - nv : is_v ? u - nk : u, per = is_v ? vecs : units;
    const int h = per == 1 ? w : (int)__umulhi((uint32_t)w, is_v ? by_vecs : by_units), c = w - h * per;
    const bool pair = !is_v && c < pairs;
    const int col = is_v || pair ? c * E : rot + (c - pairs) * E;
    const T* src = (is_v ? (const T*)a.v + row * a.v_st + h * a.v_sh : is_q ? (const T*)a.q + t * a.q_st + h * a.q_sh : (const T*)a.k + row * a.k_st + h * a.k_sh) + col;
    T* dst = (is_v ? (T*)a.v_pages + to + h * a.p_sh : is_q ? (T*)a.q_out + t * a.qo_st + h * a.qo_sh : (T*)a.k_pages + to + h * a.p_sh) + col;
    if (!is_q && !there) continue;
    uint4 x = *reinterpret_cast<const uint4*>(src), y = x;
    if (pair) {
      y = *reinterpret_cast<const uint4*>(src + half);
      Turned<T>::turn(x, y, cs + c * E, half, known);
    }
    if (!is_q && !stored) continue;
    *reinterpret_cast<uint4*>(dst) = x;
    if (pair) *reinterpret_cast<uint4*>(dst + half) = y;
  }
}

// ---- attention --------------------------------------------------------------------------------------------------------------
// out = softmax(scale q k^T) v in one pass over the keys, the running maximum and sum of a row carried along.
// Single tokens are bound by the bytes of the cache (128 sequences x 8 heads of 64 over 2050 keys: 538 MB in 111 us, 4.8 TB/s; 5 tokens of
// 16 + 4 heads of 128 over 131 000 keys: 268 MB in 50 us and 5 for the ranges), prompts by vector instructions (8 heads of 64, 8100 tokens
// over up to 3000 keys: 58 us among other work and 66 back to back, 372 and 330 TFLOP/s of products; half of the vector work is exponentials
// and splitting p; in fp32 255 us, 85 TFLOP/s), a beam step by a chain of five memory latencies (5.6 us).  A memory of 16 sentences x 4 heads
// of 64 under 17 rows each: 5.5 us (250 frames) and 10.6 (1000), in fp32 8.2 and 16.4, whether its heads lie side by side or apart.
// A workgroup takes 16 * MT rows (new token x query head of one key/value head's group) and a range of keys, its four waves every
// fourth tile of 32 keys; their results meet in LDS, those of several ranges in paged_combine_kernel.  Nothing but that goes through LDS:
// the products are laid out so that what a matrix instruction returns is what the next one takes, and K and V go from the pages to
// its operands by plain 16-byte loads.
//   S^T = K Q^T      A: lane (c, g) holds key c of a half tile, 8 (fp32: 4) elements; it returns lane (c, g) query c, keys 4g .. 4g + 3
//   O^T += V^T P^T   B: lane (c, g) holds query c, its 8 keys 4g .. 4g + 3 of both halves: those; the keys of A in the same order.
//                    A: lane (c, g) loads columns c * NDT .. of its 8 keys, 16 lanes a whole row, and (bf16) pairs keys by v_perm.
// Scores, running reference and sums are fp32, in powers of two.  The reference of a row moves only when a score passes it by 2^8
// (a vote; no exchange between lanes otherwise), so p < 2^8.  bf16 P is held as two bf16 numbers (2^-16 of the value): one rounding to
// bf16 would add an error as large as the output's own (and save 6 of 58 us with prompts, nothing where bytes count).
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float LOWEST = -3.402823466e38f;  // the reference of a row that has seen nothing: every score passes it, and -inf less it is -inf

__device__ __forceinline__ bool finite_(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// keys of each of n_split ranges of a row tile that sees keys 0 .. kend - 1, at least `least` (a multiple of 128)
__device__ __forceinline__ int chunk_of(int kend, int n_split, int least) {
  return n_split == 1 ? max(least, kend) : max(least, ((kend + n_split - 1) / n_split + 127) & ~127);
}
__device__ __forceinline__ int ranges_of(int kend, int chunk) { return kend <= chunk ? 1 : (kend + chunk - 1) / chunk; }
__device__ __forceinline__ int over(int n, int group) { return group == 1 ? n : n / group; }  // (a division is some thirty instructions)

// what a row tile sees: rows of this launch, first key after the last that any of its rows may see
struct Reach {
  int rows, len, prefix, kend;
};
__device__ __forceinline__ Reach reach_of(const s2t_paged_args& a, const Span& s, int shift, int group, int row_base, int tile_rows) {
  Reach r;
  r.rows = min(s.n, a.max_new) * group;
  r.len = min(s.len, a.table_pages << shift);
  r.prefix = a.memory ? r.len : s.len - s.n;
  const int last = over(min(row_base + tile_rows, r.rows) - 1, group);
  r.kend = a.tree ? r.len : min(r.len, r.prefix + last + 1);
  return r;
}

// bits of new tokens j0 .. j0 + 31 (bits of tokens below 0 are clear)
__device__ __forceinline__ uint32_t tree_window(const int64_t* __restrict__ row, int words, int j0) {
  const int lo = j0 >> 6, sh = j0 & 63;
  const uint64_t x = (uint32_t)lo < (uint32_t)words ? (uint64_t)row[lo] : 0, y = (uint32_t)(lo + 1) < (uint32_t)words ? (uint64_t)row[lo + 1] : 0;
  return (uint32_t)((x >> sh) | (sh ? y << (64 - sh) : 0));
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// T: type of the cache; DK: head_dim rounded up to 32, 64, 128 or 256; BIG: a half tile of 16 keys lies in one page
// BYROWS: the four waves have 16 * MT rows each and go over all keys (n_split is 1)
// (64 rows of 64-wide bf16 heads: held to two waves of a SIMD at the price of a spill outside the loop, 69 us instead of 96 with prompts)
template <typename T, int DK, int MT, bool BIG, bool BYROWS>
__global__ __launch_bounds__(256, sizeof(T) == 2 && DK == 64 && MT == 4 ? 2 : 1) void paged_attention_kernel(
    const s2t_paged_args a, const int shift, const int group, const int spread, const int n_tiles, const int n_split, const int least, const float c2, const int flip,
    float* __restrict__ part) {
  constexpr bool BF = sizeof(T) == 2;
  constexpr int NDT = DK / 16;          // 16-column tiles of the output
  constexpr int KE = BF ? 8 : 4;        // elements of 16 bytes
  constexpr int NK = DK / (4 * KE);     // 16-byte loads of a key
  constexpr int VB = NDT * (int)sizeof(T);  // bytes that a lane loads of a value row
  constexpr int STEP = BYROWS ? 32 : 128;   // from a tile of a wave to its next
  __shared__ float obuf[4][MT][4][64][NDT];
  __shared__ float mlbuf[4][MT][16][2];

  // spread: grid (8 * units, pairs / 8): all row tiles and ranges of a (sequence, key/value head) on one XCD (workgroups go round the eight),
  // the longest tiles first; otherwise (pairs, units)
  const int pair = spread ? blockIdx.y * 8 + (blockIdx.x & 7) : blockIdx.x, unit = spread ? blockIdx.x >> 3 : blockIdx.y;
  if (pair >= a.B * a.kv_heads) return;
  const int b = a.kv_heads == 1 ? pair : pair / a.kv_heads, h = pair - b * a.kv_heads;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slow = BYROWS || n_split == 1 ? unit : unit / n_split;
  const int split = unit - slow * n_split, tile = n_tiles - 1 - slow;
  const int row_base = (BYROWS ? tile * 4 + wave : tile) * 16 * MT;
  const Span sp = span_of(a, b);
  const Reach rc = reach_of(a, sp, shift, group, row_base, 16 * MT);
  if (row_base >= rc.rows) return;
  const int chunk = BYROWS ? 0 : chunk_of(rc.kend, n_split, least), used = BYROWS ? 1 : ranges_of(rc.kend, chunk);
  if (split >= used) return;
  const int k_hi = BYROWS ? rc.kend : min(rc.kend, (split + 1) * chunk);
  const int all_see = rc.prefix + (a.tree ? 0 : over(row_base, group) + 1);  // every row of the tile sees the keys before this one

  const int c = lane & 15, g = lane >> 4;
  const int d = a.dk;
  const T* kpool = (const T*)a.k_pages + h * a.p_sh;
  const T* vpool = (const T*)a.v_pages + h * a.p_sh;
  const int32_t* table = a.page_table + b * a.table_stride;
  const int sr = (int)a.p_sr, mask = a.page_size - 1;

  // queries: operand B of S^T
  u32x4 qf[MT][NK];
  int tok[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row_base + mt * 16 + c;
    const bool live = row < rc.rows;
    tok[mt] = !live ? 0 : over(row, group);
    const T* q = (const T*)a.q + (int64_t)(sp.row0 + tok[mt]) * a.q_st + (int64_t)(h * group + (live ? row - tok[mt] * group : 0)) * a.q_sh;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      const int col = (ks * 4 + g) * KE;
      u32x4 v = {0, 0, 0, 0};
      if (live && col < d) v = *reinterpret_cast<const u32x4*>(q + col);
      if (flip) v ^= BF ? 0x80008000u : 0x80000000u;  // a negative scale
      qf[mt][ks] = v;
    }
  }

  f32x4 acc[MT][NDT];
  float m[MT], l[MT];
  const int vcol = min(c * NDT, d - NDT);  // padded columns repeat the last ones; they are not written

  // where 32 keys lie: the two half tiles' first keys (BIG), or this lane's key
  struct Where {
    int64_t half0, half1;  // BIG
    int64_t row;           // !BIG: offset of key key0 + (lane & 31)
    uint32_t exist;        // bit of each of the 32 keys: it lies on a page
  };
  // (the entries of the tile after the next are asked for a tile ahead; an index beyond the table is read at its end and then left out)
  struct Pair {
    int p0, p1;
  };
  auto entries = [&](int key0) {
    const Entries e = (Entries)table;
    const int last = a.table_pages - 1;
    if constexpr (BIG) return Pair{e[min(key0 >> shift, last)], e[min((key0 + 16) >> shift, last)]};
    else return Pair{table[min((key0 + (lane & 31)) >> shift, last)], 0};
  };
  auto find = [&](int key0, Pair e) {
    Where w;
    if constexpr (BIG) {
      const bool ok0 = (uint32_t)e.p0 < (uint32_t)a.num_pages && (key0 >> shift) < a.table_pages;
      const bool ok1 = (uint32_t)e.p1 < (uint32_t)a.num_pages && ((key0 + 16) >> shift) < a.table_pages;
      w.half0 = (ok0 ? e.p0 : 0) * a.p_sp + (int64_t)(key0 & mask) * sr;
      w.half1 = (ok1 ? e.p1 : 0) * a.p_sp + (int64_t)((key0 + 16) & mask) * sr;
      w.exist = (ok0 ? 0xffffu : 0u) | (ok1 ? 0xffff0000u : 0u);
    } else {
      const int key = key0 + (lane & 31);
      const bool ok = (uint32_t)e.p0 < (uint32_t)a.num_pages && (key >> shift) < a.table_pages;
      w.row = ok ? e.p0 * a.p_sp + (int64_t)(key & mask) * sr : 0;
      w.exist = (uint32_t)__ballot(ok);
    }
    return w;
  };
  // BIG: offsets of the lane from a tile's base that hold for every tile
  uint32_t koff[NK];
#pragma unroll
  for (int ks = 0; ks < NK; ++ks) koff[ks] = (uint32_t)((BIG ? c * sr : 0) + min((ks * 4 + g) * KE, d - KE)) * (uint32_t)sizeof(T);
  const uint32_t voff = (uint32_t)((BIG ? 4 * g * sr : 0) + vcol) * (uint32_t)sizeof(T);
  auto load_k = [&](const Where& w, u32x4 (&kf)[2][NK]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* p = (const char*)(kpool + (BIG ? (t ? w.half1 : w.half0) : (int64_t)__shfl(w.row, 16 * t + c, 64)));
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) kf[t][ks] = *reinterpret_cast<const u32x4*>(p + koff[ks]);
    }
    if (d != DK) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int ks = 0; ks < NK; ++ks)
          if ((ks * 4 + g) * KE >= d) kf[t][ks] = u32x4{0, 0, 0, 0};
    }
  };
  constexpr int VW = VB / 4;  // dwords of a lane's piece of a value row
  auto load_v = [&](const Where& w, uint32_t (&vr)[8][VW]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const char* p = (const char*)(vpool + (BIG ? (e >> 2 ? w.half1 : w.half0) + (e & 3) * sr : (int64_t)__shfl(w.row, 16 * (e >> 2) + 4 * g + (e & 3), 64)));
      if constexpr (VB == 4) vr[e][0] = *reinterpret_cast<const uint32_t*>(p + voff);
      else if constexpr (VB == 8) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p + voff);
        vr[e][0] = x.x;
        vr[e][1] = x.y;
      } else {
#pragma unroll
        for (int q = 0; q < VW / 4; ++q) {
          const u32x4 x = reinterpret_cast<const u32x4*>(p + voff)[q];
          vr[e][4 * q] = x.x;
          vr[e][4 * q + 1] = x.y;
          vr[e][4 * q + 2] = x.z;
          vr[e][4 * q + 3] = x.w;
        }
      }
    }
  };

  // The first time round trusts the values that are seen: a 0 times infinity or NaN (a value that some rows of the tile do not see, or a
  // low half of p) leaves a result that is not finite.  Then the wave goes over its keys once more, taking those values out of the
  // matrix product and adding them to the rows that see them.
  float* seen = &obuf[wave][0][0][0][0];  // that round's [row tile][key][query]: p, -1 where the row does not see the key (obuf is free until the end)
  auto go = [&](auto again) {
    constexpr bool careful = decltype(again)::value;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt] = LOWEST;
      l[mt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) acc[mt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool huge = false;
    u32x4 kf[2][NK];
    int key0 = BYROWS ? 0 : split * chunk + 32 * wave;
    Where w;
    uint32_t vr[8][VW];
    Pair e{0, 0};
    if (!careful && key0 < k_hi) {
      w = find(key0, entries(key0));
      load_k(w, kf);
      load_v(w, vr);
      e = entries(key0 + STEP);
    }
    // A tile's keys and values are both on their way while the tile before it is worked on.  (The last tile asks for itself once more
    // instead of for nothing: behind a branch the compiler would have every wait for keys wait for the values as well.)
    while (key0 < k_hi) {
      if constexpr (careful) {  // (with nothing on its way, and the corrections last: this round is not to need more registers)
        w = find(key0, entries(key0));
        load_k(w, kf);
      }
      // scores of all rows, then the next tile's keys can be fetched
      f32x4 s[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < NK; ++ks) {
            if constexpr (BF)
              x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf[t][ks]), __builtin_bit_cast(bf16x8, qf[mt][ks]), x, 0, 0, 0);
            else
#pragma unroll
              for (int e = 0; e < 4; ++e)
                x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[t][ks][e]), __uint_as_float(qf[mt][ks][e]), x, 0, 0, 0);
          }
          s[mt][t] = x;
        }
      const Where now = w;
      const int next = key0 + STEP;
      if constexpr (careful) load_v(now, vr);
      else {
        if (next < k_hi) w = find(next, e);
        load_k(w, kf);
        e = entries(next + STEP);
      }
      __builtin_amdgcn_sched_barrier(0);
      // keys of this tile that exist, and whether every row sees all of them
      const uint32_t exist = low_bits(rc.len - key0) & now.exist;
      const bool whole = exist == 0xffffffffu && key0 + 32 <= all_see;
      uint32_t vis[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) vis[mt] = 0xffffffffu;
      if (!whole) {
        const int j0 = key0 - rc.prefix;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t x;
          if (a.tree) x = tree_window(a.tree + (int64_t)(sp.row0 + tok[mt]) * a.tree_stride, a.tree_words, j0) | low_bits(-j0);
          else x = low_bits(tok[mt] - j0 + 1);
          vis[mt] = x & exist;
          const uint32_t mine = vis[mt] >> (4 * g);
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!((mine >> (16 * t + r)) & 1)) s[mt][t][r] = -INFINITY;
        }
      }
      // one vote for all row tiles whether a reference has to move, then the exponents.  Equal scores have equal exponents at a reference, a rounded
      // score * c2 itself, however large it is; but where half a step of it is no longer small, the exponent of the score that it came from is not
      // near 0 by a fused product and difference: from then on the product is rounded as the reference was.  (Exponents first, against a
      // reference that moves by their maximum: 55 instead of 58 us with prompts, but from 2^28 on a move is lost and 2^x infinite.)
      bool grow = false;
      float top[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        top[mt] = fmaxf(fmaxf(fmaxf(s[mt][0][0], s[mt][0][1]), fmaxf(s[mt][0][2], s[mt][0][3])),
                        fmaxf(fmaxf(s[mt][1][0], s[mt][1][1]), fmaxf(s[mt][1][2], s[mt][1][3])));
        grow = grow || fmaf(top[mt], c2, -m[mt]) > 8.f;
      }
      if (__any(grow)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float mn = fmaxf(m[mt], s2t_xmax<16>(s2t_xmax<32>(top[mt])) * c2), fade = exp2_(m[mt] - mn);
          m[mt] = mn;
          l[mt] *= fade;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) acc[mt][dt] *= fade;
          huge = huge || __any(fabsf(mn) > 0x1p20f && mn != LOWEST);
        }
      }
      if (huge) {
        asm volatile("");  // (a branch, not both and a choice)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[mt][t][r] *= c2;
      }
      const float left = huge ? 1.f : c2;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[mt][t][r] = fmaf(s[mt][t][r], left, -m[mt]);
      __builtin_amdgcn_s_setprio(1);  // (the wave that has its scores before the one that waits for keys: prompts 69.7 -> 66.7 us)
      // values: operand A of O^T
      if (exist != 0xffffffffu) {  // what lies behind the end is not to be multiplied with anything
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!((exist >> (16 * (e >> 2) + 4 * g + (e & 3))) & 1))
#pragma unroll
            for (int q = 0; q < VW; ++q) vr[e][q] = 0;
      }
      if constexpr (careful) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int q = 0; q < VW; ++q) {
            if constexpr (BF) {
              if ((vr[e][q] & 0x7f80u) == 0x7f80u) vr[e][q] &= 0xffff0000u;
              if ((vr[e][q] & 0x7f800000u) == 0x7f800000u) vr[e][q] &= 0xffffu;
            } else if (!finite_(__uint_as_float(vr[e][q]))) vr[e][q] = 0;
          }
      }
      u32x4 va[BF ? NDT : 1];
      if constexpr (BF) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            va[dt][q] = __builtin_amdgcn_perm(vr[2 * q + 1][dt >> 1], vr[2 * q][dt >> 1], dt & 1 ? 0x07060302u : 0x05040100u);
        if constexpr (!careful) load_v(w, vr);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float p[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) p[t][r] = exp2_(s[mt][t][r]);
        l[mt] += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
        if constexpr (BF) {
          u32x4 hi, lo;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float x = p[q >> 1][2 * (q & 1)], y = p[q >> 1][2 * (q & 1) + 1];
            hi[q] = bf16pack(x, y);
            lo[q] = bf16pack(x - __uint_as_float(hi[q] << 16), y - __uint_as_float(hi[q] & 0xffff0000u));
          }
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) {
            acc[mt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va[dt]), __builtin_bit_cast(bf16x8, hi), acc[mt][dt], 0, 0, 0);
            acc[mt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va[dt]), __builtin_bit_cast(bf16x8, lo), acc[mt][dt], 0, 0, 0);
          }
        } else {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int dt = 0; dt < NDT; ++dt)
                acc[mt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[4 * t + r][dt]), p[t][r], acc[mt][dt], 0, 0, 0);
        }
        if constexpr (careful) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) seen[(mt * 32 + 16 * t + 4 * g + r) * 16 + c] = (vis[mt] >> (16 * t + 4 * g + r)) & 1 ? p[t][r] : -1.f;
        }
      }
      if constexpr (careful) {
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
        for (int key = 0; key < 32; ++key) {
          int64_t at = 0;
          if constexpr (!BIG) at = (int64_t)__shfl(now.row, key, 64);
          if (!((exist >> key) & 1)) continue;
          if constexpr (BIG) at = (key >> 4 ? now.half1 : now.half0) + (key & 15) * sr;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
              const float v = ld_as_f32<T>(vpool + at + min((4 * g + r) * NDT + dt, d - 1));
              if (!finite_(v))
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  const float pk = seen[(mt * 32 + key) * 16 + c];
                  if (!(pk < 0.f)) acc[mt][dt][r] += pk * v;
                }
              __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_wave_barrier();
      }
      __builtin_amdgcn_s_setprio(0);
      if constexpr (!BF && !careful) load_v(w, vr);
      key0 = next;
    }
  };
  go(std::false_type{});
  float sick = 0.f;  // a sum of 0 * x: 0, or NaN if any x is not finite
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) sick = fmaf(acc[mt][dt][r], 0.f, sick);
  if (__any(sick != sick)) go(std::true_type{});

  // columns col .. of a row: o / total, or both for paged_combine_kernel
  auto finish = [&](int row, int col, const auto& o, float top, float total) {
    constexpr int NC = sizeof(o) / 4, CH = NC < KE ? NC : KE;  // CH columns are all there or none
    if (row >= rc.rows) return;
    const int i = over(row, group), t = sp.row0 + i, hq = h * group + row - i * group;
    if (used == 1) {
      const float inv = total == 0.f ? 0.f : 1.f / total;  // (nothing seen; a NaN score leaves a sum of NaN, and so does its row)
      T* out = (T*)a.out + (int64_t)t * a.o_st + (int64_t)hq * a.o_sh + col;
#pragma unroll
      for (int e = 0; e < NC; e += CH)
        if (col + e < d) {
          if constexpr (BF) {
            uint32_t y[CH / 2];
#pragma unroll
            for (int q = 0; q < CH / 2; ++q) y[q] = bf16pack(o[e + 2 * q] * inv, o[e + 2 * q + 1] * inv);
            if constexpr (CH == 8) *reinterpret_cast<u32x4*>(out + e) = u32x4{y[0], y[1], y[2], y[3]};
            else if constexpr (CH == 4) *reinterpret_cast<u32x2*>(out + e) = u32x2{y[0], y[1]};
            else *reinterpret_cast<uint32_t*>(out + e) = y[0];
          } else if constexpr (CH == 4) *reinterpret_cast<f32x4*>(out + e) = f32x4{o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv};
          else *reinterpret_cast<float2*>(out + e) = make_float2(o[e] * inv, o[e + 1] * inv);
        }
      if (a.lse && col == 0) a.lse[(int64_t)t * a.q_heads + hq] = total == 0.f ? -INFINITY : (top + log2f(total)) * LN2;
    } else {  // part: [split][token][query head][d], then their [2]: reference and sum
      const int64_t heads = (int64_t)a.N * a.q_heads, at = split * heads + (int64_t)t * a.q_heads + hq;
      float* to = part + at * d + col;
#pragma unroll
      for (int e = 0; e < NC; e += CH)
        if (col + e < d) {
#pragma unroll
          for (int q = 0; q < CH; q += 2) *reinterpret_cast<float2*>(to + e + q) = make_float2(o[e + q], o[e + q + 1]);
        }
      if (col == 0) reinterpret_cast<float2*>(part + n_split * heads * d)[at] = make_float2(top, total);
    }
  };
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) l[mt] = s2t_xadd<16>(s2t_xadd<32>(l[mt]));
  if constexpr (BYROWS) {  // the lane holds columns (4g + r) * NDT + dt of query c
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float o[4 * NDT];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[r * NDT + dt] = acc[mt][dt][r];
      finish(row_base + mt * 16 + c, 4 * g * NDT, o, m[mt], l[mt]);
    }
    return;
  }
  // The four waves' results meet; with 64 rows each wave then finishes a row tile (its lanes write 16 columns, four of them a row), with fewer
  // half a tile or a quarter.
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (g == 0) {
      mlbuf[wave][mt][c][0] = m[mt];
      mlbuf[wave][mt][c][1] = l[mt];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) obuf[wave][mt][r][lane][dt] = acc[mt][dt][r];
  }
  __syncthreads();
  const int mine = wave * MT >> 2, r0 = wave * MT & 3;
  float mw[4], top = LOWEST;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    mw[w] = mlbuf[w][mine][c][0];
    top = fmaxf(top, mw[w]);
  }
  float total = 0.f, o[MT * NDT];
#pragma unroll
  for (int e = 0; e < MT * NDT; ++e) o[e] = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {  // (a wave that saw nothing has sums of 0, or of NaN)
    const float f = exp2_(mw[w] - top);
    total += f * mlbuf[w][mine][c][1];
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[r * NDT + dt] += f * obuf[w][mine][r0 + r][lane][dt];
  }
  finish(row_base + mine * 16 + c, (4 * g + r0) * NDT, o, top, total);
}

// Joins the ranges of the (new token, query head) rows, weights 2^(m - max m): WAVES waves to a row, `lanes` (a power of two) of them to a
// range's columns, so that 64 * WAVES / lanes ranges are on their way at a time; the order of every sum is fixed.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void paged_combine_kernel(const s2t_paged_args a, const int shift, const int tile_rows, const int n_split,
                                                            const int least, const int lanes, const float* __restrict__ part) {
  __shared__ float sums[4][256];
  const int b = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6, sub = WAVES == 1 ? 0 : w;
  const int rowid = WAVES == 1 ? blockIdx.x * 4 + w : blockIdx.x;
  const int i = rowid / a.q_heads, hq = rowid % a.q_heads, group = a.q_heads / a.kv_heads, d = a.dk;
  const Span sp = span_of(a, b);
  const bool live = i < min(sp.n, a.max_new);
  const Reach rc = reach_of(a, sp, shift, group, (i * group + hq % group) / tile_rows * tile_rows, tile_rows);
  const int chunk = chunk_of(rc.kend, n_split, least), used = ranges_of(rc.kend, chunk);
  if (!live || used == 1) return;  // (WAVES == 4: the whole workgroup)
  const int64_t heads = (int64_t)a.N * a.q_heads, t = sp.row0 + i, at = t * a.q_heads + hq;
  const float2* ml = reinterpret_cast<const float2*>(part + n_split * heads * d) + at;
  float top = LOWEST;
  for (int s = lane; s < used; s += 64) top = fmaxf(top, ml[s * heads].x);
  top = wave_max(top);
  const int col = (lane & (lanes - 1)) * 4, first = sub * (64 / lanes) + lane / lanes, step = WAVES * (64 / lanes);
  float total = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = first; s < used; s += step) {
    const float2 x = ml[s * heads];
    const float f = exp2_(x.x - top);
    const f32x4 y = col < d ? *reinterpret_cast<const f32x4*>(part + (s * heads + at) * d + col) : f32x4{0.f, 0.f, 0.f, 0.f};
    total += f * x.y;
    o += f * y;
  }
  for (int x = lanes; x < 64; x *= 2) {
    total += __shfl_xor(total, x, 64);
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] += __shfl_xor(o[r], x, 64);
  }
  if constexpr (WAVES == 4) {
    if (lane < lanes) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < d) sums[w][col + r] = o[r];
    }
    __shared__ float totals[4];
    if (lane == 0) totals[w] = total;
    __syncthreads();
    if (w != 0) return;
    total = (totals[0] + totals[1]) + (totals[2] + totals[3]);
    if (col < d)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (sums[0][col + r] + sums[1][col + r]) + (sums[2][col + r] + sums[3][col + r]);
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (lane < lanes && col < d) {
    const float y[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    st4_from_f32<T>((T*)a.out + t * a.o_st + hq * a.o_sh + col, y);
  }
  if (a.lse && lane == 0) a.lse[at] = total == 0.f ? -INFINITY : (top + log2f(total)) * LN2;
}

// How a call is cut: row tiles of 16 rows to a wave, whether the waves of a workgroup have rows of their own, tiles of a sequence, ranges of
// the keys.
struct Cut {
  int mt, by_rows, tiles, splits, least;
};
Cut cut_of(const s2t_paged_args* a) {
  const int64_t rows = (int64_t)a->max_new * (a->q_heads / a->kv_heads), keys = (int64_t)a->table_pages * a->page_size;
  const int64_t pairs = (int64_t)a->kv_heads * a->B;
  Cut c;
  // Few keys and many rows: a wave's rows go over all keys, and nothing has to be put together (147 sequences x 8 heads x 160 rows over 76
  // keys, fp32 heads of 64: 137 us by keys, 55 by rows; 105 x 4 x 51 over 263, bf16 heads of 128: 31.6 and 19.0), where that gives every
  // compute unit a workgroup (2 x 8 x 164 over 288: 11.5 by keys, 15.2 by rows).
  c.by_rows = rows > 16 && keys <= 512 && (rows + 63) / 64 * pairs >= 256;
  if (c.by_rows) {
    c.mt = c.splits = 1;
    c.least = 128;
    c.tiles = (int)((rows + 63) / 64);
    return c;
  }
  // as many rows to a wave as registers allow, unless that leaves most of the chip without work also with the keys in ranges (568 rows of
  // one fp32 head of 128, four sequences: 19.1 us with 32 rows, 13.6 with 16; 1248 rows of 8 heads of 32 over 2600 keys: 26.3 with 64,
  // 22.6 with 32; but 20 rows of 4 heads of 128 over 131 000 keys: 56 with 32, 81 with 16, which reads the keys twice)
  const int most = a->dk <= 64 ? 4 : a->dk <= 128 ? 2 : 1;
  c.mt = rows <= 16 || most == 1 ? 1 : rows <= 32 || most == 2 ? 2 : 4;
  while (c.mt > 1 && (rows + 16 * c.mt - 1) / (16 * c.mt) * pairs * std::max<int64_t>(1, keys / 2048) < 256) c.mt /= 2;
  c.tiles = (int)((rows + 16 * c.mt - 1) / (16 * c.mt));
  // Ranges of the keys where there is less than a workgroup for every compute unit, as many as fill the chip and no more; each holds 128 KB
  // of keys and values at least, as the second launch that joins them costs some 2 us.  Sequences x heads, one row each unless said:
  //   workgroups, at most                          128     256     512   |   KB in a range       32      64     128     256    no cut
  //   bf16, 64 wide, 4 x 16 over 4000 keys        19.2    15.0    17.0   |                     14.9    15.0    15.0    15.9    26.0 us
  //   bf16, 64 wide, 24 x 8 over 1500             13.8    13.7    18.2   |                     13.8    13.8    13.7    13.7    13.6
  //   bf16, 64 wide, 16 x 4 over 500               6.3     6.3     6.3   |                      7.9     8.5     6.3     6.3     6.4
  //   bf16, 64 wide, 2 x 2 over 6000              10.3    10.4    10.4   |                      8.6     9.0    10.4    13.5    33.9
  //   fp32, 64 wide, trees of 13, 24 x 4 over 300  9.2     9.2     9.2   |                     11.8    11.7     9.2     9.2     9.3
  //   fp32, 128 wide, 16 x 4 over 1000            21.3    17.2    20.7   |                     17.2    17.3    17.2    19.2    26.7
  //   fp32, 128 wide, 4 rows of 8 x 8 over 3000   40.0    30.6    38.1   |                     30.7    30.7    30.6    30.7    63.2
  int64_t s = 256 / (c.tiles * pairs);
  c.least = std::max(128, 131072 / (2 * a->dk * (a->dtype == S2T_F32 ? 4 : 2)) & ~127);
  if (s > keys / c.least) s = keys / c.least;
  if (s > 256) s = 256;
  if (s < 1) s = 1;
  c.splits = (int)s;
  return c;
}

template <typename T, int DK, int MT, bool BYROWS = false>
void launch_attention(const s2t_paged_args* a, const Cut& c, hipStream_t st) {
  const int pairs = a->B * a->kv_heads, units = c.tiles * c.splits, spread = c.tiles > 1 && pairs >= 8;
  const dim3 grid = spread ? dim3(8u * units, (unsigned)((pairs + 7) / 8)) : dim3((unsigned)pairs, (unsigned)units);
  const int shift = __builtin_ctz((unsigned)a->page_size), flip = a->scale < 0.f, group = a->q_heads / a->kv_heads;
  const float c2 = fmaxf(fabsf(a->scale) * LOG2E, 1e-30f);  // never 0: 0 times the -inf of a hidden key is not 0
  if (a->page_size >= 16) hipLaunchKernelGGL((paged_attention_kernel<T, DK, MT, true, BYROWS>), grid, dim3(256), 0, st, *a, shift, group, spread, c.tiles, c.splits, c.least, c2, flip, (float*)a->ws);
  else hipLaunchKernelGGL((paged_attention_kernel<T, DK, MT, false, BYROWS>), grid, dim3(256), 0, st, *a, shift, group, spread, c.tiles, c.splits, c.least, c2, flip, (float*)a->ws);
}
template <typename T>
void launch_attention(const s2t_paged_args* a, const Cut& c, hipStream_t st) {
  if (c.by_rows) {
    if (a->dk <= 32) launch_attention<T, 32, 1, true>(a, c, st);
    else if (a->dk <= 64) launch_attention<T, 64, 1, true>(a, c, st);
    else if (a->dk <= 128) launch_attention<T, 128, 1, true>(a, c, st);
    else launch_attention<T, 256, 1, true>(a, c, st);
  } else if (a->dk <= 32) {
    if (c.mt == 1) launch_attention<T, 32, 1>(a, c, st);
    else if (c.mt == 2) launch_attention<T, 32, 2>(a, c, st);
    else launch_attention<T, 32, 4>(a, c, st);
  } else if (a->dk <= 64) {
    if (c.mt == 1) launch_attention<T, 64, 1>(a, c, st);
    else if (c.mt == 2) launch_attention<T, 64, 2>(a, c, st);
    else launch_attention<T, 64, 4>(a, c, st);
  } else if (a->dk <= 128) {
    if (c.mt == 1) launch_attention<T, 128, 1>(a, c, st);
    else launch_attention<T, 128, 2>(a, c, st);
  } else {
    launch_attention<T, 256, 1>(a, c, st);
  }
  if (c.splits > 1) {
    const int rows = a->max_new * a->q_heads, shift = __builtin_ctz((unsigned)a->page_size);
    const int lanes = a->dk <= 16 ? 4 : a->dk <= 32 ? 8 : a->dk <= 64 ? 16 : a->dk <= 128 ? 32 : 64;
    if (c.splits <= 8)
      hipLaunchKernelGGL((paged_combine_kernel<T, 1>), dim3((unsigned)((rows + 3) / 4), (unsigned)a->B), dim3(256), 0, st, *a, shift, 16 * c.mt, c.splits, c.least, lanes, (const float*)a->ws);
    else
      hipLaunchKernelGGL((paged_combine_kernel<T, 4>), dim3((unsigned)rows, (unsigned)a->B), dim3(256), 0, st, *a, shift, 16 * c.mt, c.splits, c.least, lanes, (const float*)a->ws);
  }
}

int paged_args_bad(const s2t_paged_args* a) {
  if (!a || !a->k_pages || !a->v_pages || !a->page_table || !a->lens || !a->cu) return S2T_ERR_ARG;
  if (a->dtype != S2T_F32 && a->dtype != S2T_BF16) return S2T_ERR_DTYPE;
  if (a->B <= 0 || a->B > 65535 || a->N < 0 || a->max_new < 0 || a->q_heads <= 0 || a->kv_heads <= 0 || a->q_heads % a->kv_heads) return S2T_ERR_ARG;
  if (a->num_pages <= 0 || a->table_pages <= 0 || a->page_size <= 0 || (a->page_size & (a->page_size - 1))) return S2T_ERR_ARG;
  if ((int64_t)a->table_pages * a->page_size > 0x7fff0000ll) return S2T_ERR_UNSUPPORTED;  // places are 32-bit numbers
  if (a->dk <= 0 || a->dk % 16 || a->dk > 256) return S2T_ERR_UNSUPPORTED;
  return S2T_OK;
}
// A sequence brings no more new tokens than there are rows: a loose bound neither sizes a launch nor chooses how the keys are cut.
s2t_paged_args bounded(const s2t_paged_args* a) {
  s2t_paged_args b = *a;
  b.max_new = std::min(b.max_new, b.N);
  return b;
}
bool misaligned(const s2t_paged_args* a, const void* p, int64_t st, int64_t sh) {
  const int e = a->dtype == S2T_F32 ? 4 : 8;  // elements of 16 bytes
  return ((uintptr_t)p & 15) || st % e || sh % e;
}
int shift_of(const s2t_paged_args* a) { return __builtin_ctz((unsigned)a->page_size); }

}  // namespace

extern "C" int s2t_paged_kv_append(const s2t_paged_args* args, void* stream) {
  if (int bad = paged_args_bad(args)) return bad;
  const s2t_paged_args bound = bounded(args), *a = &bound;
  if ((a->q && a->rows) || (a->rows && a->src_rows < 0)) return S2T_ERR_ARG;
  if (a->rotary && (a->rot_dim <= 0 || a->rot_dim % 16 || a->rot_dim > a->dk || a->rotary_positions <= 0)) return S2T_ERR_ARG;
  if (misaligned(a, a->k_pages, a->p_sp, a->p_sh) || misaligned(a, a->v_pages, a->p_sr, 0) || misaligned(a, a->k, a->k_st, a->k_sh) ||
      misaligned(a, a->v, a->v_st, a->v_sh) || (a->q && (misaligned(a, a->q, a->q_st, a->q_sh) || misaligned(a, a->q_out, a->qo_st, a->qo_sh))) ||
      ((uintptr_t)a->rotary & 15))
    return S2T_ERR_ALIGN;
  if (a->N == 0 || a->max_new == 0 || (a->rows && a->src_rows == 0)) return S2T_OK;  // (an empty tensor has no address)
  if (!a->k || !a->v || (a->q && !a->q_out)) return S2T_ERR_ARG;
  const int e = a->dtype == S2T_F32 ? 4 : 8, rot = a->rotary ? a->rot_dim : 0, units = rot / 2 / e + (a->dk - rot) / e, vecs = a->dk / e;
  if ((int64_t)std::max(a->q_heads, a->kv_heads) * vecs * vecs >= (1ll << 31)) return S2T_ERR_UNSUPPORTED;  // (divisions by reciprocals)
  const auto by = [](int n) { return n > 1 ? (uint32_t)((1ull << 32) / n + 1) : 0u; };
  if (a->max_new > (1 << 26) - 4) return S2T_ERR_UNSUPPORTED;  // (a launch's dimension is below 2^32 threads, 64 of them to a token)
  const dim3 grid((unsigned)((a->max_new + 3) / 4), (unsigned)a->B);
  if (a->dtype == S2T_F32) hipLaunchKernelGGL(paged_append_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, *a, shift_of(a), by(units), by(vecs));
  else hipLaunchKernelGGL(paged_append_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, *a, shift_of(a), by(units), by(vecs));
  return S2T_LAUNCH_CHECK();
}

extern "C" int64_t s2t_paged_attention_ws_bytes(const s2t_paged_args* args) {
  if (paged_args_bad(args)) return -1;
  const s2t_paged_args bound = bounded(args), *a = &bound;
  if (a->N == 0 || a->max_new == 0) return 0;
  const Cut c = cut_of(a);
  return c.splits > 1 ? (int64_t)c.splits * a->N * a->q_heads * (a->dk + 2) * 4 : 0;
}

extern "C" int s2t_paged_attention(const s2t_paged_args* args, void* stream) {
  if (int bad = paged_args_bad(args)) return bad;
  const s2t_paged_args bound = bounded(args), *a = &bound;
  if ((a->tree && (a->tree_words <= 0 || a->memory)) || !(a->scale == a->scale)) return S2T_ERR_ARG;
  if (misaligned(a, a->k_pages, a->p_sp, a->p_sh) || misaligned(a, a->v_pages, a->p_sr, 0) || misaligned(a, a->q, a->q_st, a->q_sh) ||
      misaligned(a, a->out, a->o_st, a->o_sh) || ((uintptr_t)a->tree & 7))
    return S2T_ERR_ALIGN;
  if (a->N == 0 || a->max_new == 0) return S2T_OK;
  if (!a->q || !a->out) return S2T_ERR_ARG;
  const Cut c = cut_of(a);
  // launch bounds (a grid's second dimension is 16 bits), and 32-bit offsets of the 16 rows of a half tile
  const int64_t pairs = (int64_t)a->B * a->kv_heads, units = (int64_t)c.tiles * c.splits;
  const bool spread = c.tiles > 1 && pairs >= 8;
  if ((spread ? (pairs + 7) / 8 : units) > 65535 || (spread ? 8 * units : pairs) > (1 << 23) || (int64_t)a->max_new * a->q_heads > (1 << 23) || a->p_sr < 0 || a->p_sr > (1 << 24))
    return S2T_ERR_UNSUPPORTED;
  if (c.splits > 1 && (!a->ws || ((uintptr_t)a->ws & 15) || a->ws_bytes < s2t_paged_attention_ws_bytes(a))) return S2T_ERR_ARG;
  if (a->dtype == S2T_F32) launch_attention<float>(a, c, (hipStream_t)stream);
  else launch_attention<bf16_t>(a, c, (hipStream_t)stream);
  return S2T_LAUNCH_CHECK();
}
