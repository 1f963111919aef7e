// The key/value cache in pages: kv_store_paged, attention_decode_paged, kv_evict_paged.
//
// Keys and values live in pages of page_size positions, (num_pages, kv_heads, page_size,
// head_size) each, so that one head's rows of a page are one run of consecutive bytes; a table
// lists every sequence's pages in order.  Arithmetic is fp32 throughout; only what is stored in
// a 16-bit cache is rounded, once, to nearest even.
#include <cmath>
#include <type_traits>

#include "common.hpp"

namespace g2 {

typedef _Float16 f16;
struct bf16 {
  unsigned short bits;
};

// ---- the three element types of a cache -----------------------------------------------------
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(f16 v) { return (float)v; }
__device__ __forceinline__ float widen(bf16 v) { return __builtin_bit_cast(float, (unsigned)v.bits << 16); }

template <class E>
__device__ __forceinline__ E narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ f16 narrow<f16>(float v) { return (f16)v; }
template <>
__device__ __forceinline__ bf16 narrow<bf16>(float v) {
  // to nearest even; a NaN keeps its sign and stays a NaN
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const unsigned r = (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
  return bf16{(unsigned short)(v != v ? ((u >> 16) | 0x40u) : r)};
}

// 16 bytes of a row as floats.
template <class E>
constexpr int kPer16 = 16 / (int)sizeof(E);
__device__ __forceinline__ void widen16(float (&to)[4], u32x4 raw, float) {
  const f32x4 f = __builtin_bit_cast(f32x4, raw);
#pragma unroll
  for (int j = 0; j < 4; j++) to[j] = f[j];
}
__device__ __forceinline__ void widen16(float (&to)[8], u32x4 raw, f16) {
  typedef f16 f16x8 __attribute__((ext_vector_type(8)));
  const f16x8 h = __builtin_bit_cast(f16x8, raw);
#pragma unroll
  for (int j = 0; j < 8; j++) to[j] = (float)h[j];
}
__device__ __forceinline__ void widen16(float (&to)[8], u32x4 raw, bf16) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const unsigned lo = raw[j] << 16, hi = raw[j] & 0xffff0000u;
    to[2 * j] = __builtin_bit_cast(float, lo);
    to[2 * j + 1] = __builtin_bit_cast(float, hi);
  }
}

// ---- position -> row of the pages -----------------------------------------------------------
// Division by the page size as one high product and a shift, exact for every 31-bit position:
// with shift = ceil(log2 d) and magic = ceil(2^(31 + shift) / d), magic fits 32 bits and
// floor(n * magic / 2^(31 + shift)) = floor(n / d) for n < 2^31, because magic * d exceeds
// 2^(31 + shift) by less than d <= 2^shift.
struct PageDivide {
  unsigned magic;
  int shift;  // after the high half of the 64-bit product: 31 + log - 32
  unsigned size;
  explicit PageDivide(int d = 1) : size((unsigned)d) {
    int log = 0;
    while ((1LL << log) < d) log++;
    magic = (unsigned)(((1ULL << (31 + log)) + d - 1) / d);
    shift = 31 + log;
  }
  __host__ __device__ __forceinline__ unsigned operator()(unsigned n) const {
    return (unsigned)(((unsigned long long)n * magic) >> shift);
  }
};

// What a kernel has to know of a cache.
struct Pages {
  void *keys, *values;
  const int* table;
  PageDivide divide;
  int num_pages, max_pages, kv_heads, head_size;
  int capacity;  // positions a table row can name
  // The row (of head_size elements) that holds a position of sequence b for one kv head; ok is
  // cleared where the table names a page that does not exist.  Rows are counted in 32 bits: the
  // launchers refuse larger pools.
  __host__ __device__ __forceinline__ unsigned row(int b, int head, int pos, bool& ok) const {
    const unsigned p = divide((unsigned)pos);
    const int page = table[(size_t)b * max_pages + p];
    const bool there = (unsigned)page < (unsigned)num_pages;
    ok &= there;
    return there ? ((unsigned)page * kv_heads + head) * divide.size + ((unsigned)pos - p * divide.size) : 0u;
  }
};

// ---- kv_store_paged -------------------------------------------------------------------------
// One wave per row of the prompts: it finds the row's sequence by counting the starts that are
// not behind it, 64 at a time, and moves the row's keys and values, VEC floats per lane and step.
template <class E, int VEC>
__global__ __launch_bounds__(256) void kv_store_paged_kernel(Pages pg, const float* __restrict__ inp, int stride,
                                                             const int* __restrict__ starts,
                                                             const int* __restrict__ lengths, int N, int B, int NH) {
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= N) return;
  int b = -1;
  for (int i = 0; i <= B; i += 64) {
    const bool begun = i + lane <= B && starts[i + lane] <= r;
    const unsigned long long m = __ballot(begun);
    b += __popcll(m);
    if (m != ~0ull) break;
  }
  if (b < 0 || b >= B || starts[b] > r || starts[b + 1] <= r) return;  // in front of the first row or behind the last
  const int n = lengths[b];
  const long long pos = (long long)n + (r - starts[b]);
  if (n < 0 || pos >= pg.capacity) return;
  const int HS = pg.head_size, half = pg.kv_heads * HS;
  bool ok = true;
  const unsigned row0 = pg.row(b, 0, (int)pos, ok);
  if (!ok) return;
  const float* src = inp + (size_t)r * stride + (size_t)NH * HS;
  for (int i = lane * VEC; i < 2 * half; i += 64 * VEC) {
    const bool value = i >= half;
    const int c = value ? i - half : i;
    const int head = c / HS, d = c - head * HS;
    E* to = (E*)(value ? pg.values : pg.keys) + ((size_t)row0 + (size_t)head * pg.divide.size) * HS + d;
    if constexpr (VEC == 4) {
      const f32x4 x = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(src + i));
      struct alignas(4 * sizeof(E)) Four {
        E e[4];
      };
      *reinterpret_cast<Four*>(to) = Four{{narrow<E>(x[0]), narrow<E>(x[1]), narrow<E>(x[2]), narrow<E>(x[3])}};
    } else {
      to[0] = narrow<E>(src[i]);
    }
  }
}

// ---- attention_decode_paged -----------------------------------------------------------------
struct AttendPaged {
  Pages pg;
  float* out;
  const float* inp;
  const int* lengths;
  const float* weights_in;
  float* weights_out;
  float *part_o, *part_ml;  // (B, NH, S, HS) and (B, NH, S, 2): unnormalised outputs, (maximum, sum) in the exponent's base-2 scale
  float* scores;            // (B, NH, capacity) base-2 scores, where weights are asked for
  int B, NH, G, chunks;     // G query heads per kv head, in `chunks` groups of GQ
  int stride, S, append;
  float scale_log2e;
};

// How the n positions held by a sequence are dealt to at most S workgroups.
constexpr int kMinRange = 128;
__device__ __forceinline__ int range_of(int n, int S) {
  const int each = (n + S - 1) / S;
  return each < kMinRange ? kMinRange : (each + 63) & ~63;
}
__device__ __forceinline__ int ranges_of(int n, int range) { return n <= range ? 1 : (n + range - 1) / range; }

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  if (LPR >= 16) v += dpp<0x140>(v);
  if (LPR >= 32) v += __shfl_xor(v, 16, 64);
  if (LPR >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// exp2(a - m) where m is the running maximum: a maximum of -inf (nothing seen, or only scores of
// -inf) counts as 0, so that such scores weigh 0 instead of NaN.
__device__ __forceinline__ float above(float m) { return m == -INFINITY ? 0.f : m; }

constexpr int kAttWaves = 4;

// A workgroup takes one range of positions of one (sequence, kv head) for GQ of the query heads
// that share it.  LPR lanes hold one row of keys or values, 16 bytes each, so that a wave's load
// covers 64 / LPR rows; every such group of lanes keeps a softmax (maximum, sum, output) of its
// own over the rows it has seen, and the groups, the waves and the ranges meet only at the end.
// SCALAR: rows of any size and alignment, a row per wave, one element per lane and load.
template <class E, int LPR, int GQ, int U, bool SCALAR>
__global__ __launch_bounds__(kAttWaves* kWave) void attention_paged_kernel(const AttendPaged a) {
  constexpr int VEC = SCALAR ? 4 : kPer16<E>;
  constexpr int RPW = 64 / LPR;
  constexpr int TILE = U * RPW;
  static_assert(TILE <= 64, "a tile's rows are looked up by one lane each");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sub = lane & (LPR - 1), rg = lane / LPR;
  const int HS = a.pg.head_size, KVH = a.pg.kv_heads;
  int id = blockIdx.x;
  const int s = id % a.S;
  id /= a.S;
  const int hc = id % a.chunks;
  id /= a.chunks;
  const int kvh = id % KVH, b = id / KVH;
  const int head0 = kvh * a.G + hc * GQ;
  const int heads = min(GQ, a.G - hc * GQ);

  const int n = a.lengths[b];
  if (n < 0) return;  // an unused place in the batch
  const bool too_long = n > a.pg.capacity - a.append;
  if (too_long || n + a.append == 0) {
    if (s == 0) {
      const float fill = too_long ? __builtin_nanf("") : 0.f;
      for (int i = tid; i < heads * HS; i += kAttWaves * kWave) a.out[((size_t)b * a.NH + head0) * HS + i] = fill;
    }
    return;
  }
  const int range = range_of(n, a.S), ranges = ranges_of(n, range);
  if (s >= ranges) return;

  // element j of this lane's part of a row
  auto at = [&](int j) { return SCALAR ? sub + 64 * j : sub * VEC + j; };
  float q[GQ][VEC], o[GQ][VEC], m[GQ], l[GQ];
#pragma unroll
  for (int g = 0; g < GQ; g++) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      o[g][j] = 0.f;
      q[g][j] = g < heads && at(j) < HS
                    ? a.inp[(size_t)b * a.stride + (size_t)(head0 + g) * HS + at(j)] * a.scale_log2e
                    : 0.f;
    }
  }

  auto load = [&](float (&to)[VEC], const void* base, unsigned row) {
    const E* p = (const E*)base + (size_t)row * HS;
    if constexpr (SCALAR) {
#pragma unroll
      for (int j = 0; j < VEC; j++) to[j] = at(j) < HS ? widen(p[at(j)]) : 0.f;
    } else {
      u32x4 raw = {0u, 0u, 0u, 0u};
      if (sub * VEC < HS) raw = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + sub * VEC));
      widen16(to, raw, E{});
    }
  };
  // The softmax of this lane's row group over U more rows: keys k, values v; sc[g][u] base-2 scores.
  float* const scores = a.scores ? a.scores + ((size_t)b * a.NH + head0) * a.pg.capacity : nullptr;

  const int p0 = s * range, p1 = min(n, p0 + range);
  bool ok = true;
  int t = p0 + wave * TILE;
  unsigned next = t < p1 ? a.pg.row(b, kvh, min(t + (lane & (TILE - 1)), p1 - 1), ok) : 0u;
  for (; t < p1; t += kAttWaves * TILE) {
    const unsigned rows = next;
    if (t + kAttWaves * TILE < p1)
      next = a.pg.row(b, kvh, min(t + kAttWaves * TILE + (lane & (TILE - 1)), p1 - 1), ok);
    float k[U][VEC], v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; u++) load(k[u], a.pg.keys, __shfl(rows, u * RPW + rg, 64));
#pragma unroll
    for (int u = 0; u < U; u++) load(v[u], a.pg.values, __shfl(rows, u * RPW + rg, 64));
    const bool full = t + TILE <= p1;
    if (!full) {
      // rows behind the range were read as copies of its last one: they weigh nothing, whatever they hold
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int j = 0; j < VEC; j++) v[u][j] = t + u * RPW + rg < p1 ? v[u][j] : 0.f;
    }
#pragma unroll
    for (int g = 0; g < GQ; g++) {
      float sc[U], top = m[g];
#pragma unroll
      for (int u = 0; u < U; u++) {
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; j++) d = fmaf(q[g][j], k[u][j], d);
        d = row_sum<LPR>(d);
        const bool in = t + u * RPW + rg < p1;
        if (scores && sub == 0 && in && g < heads) scores[(size_t)g * a.pg.capacity + t + u * RPW + rg] = d;
        sc[u] = in ? d : -INFINITY;
        top = fmaxf(top, sc[u]);
      }
      const float base = above(top);
      const float fade = __builtin_amdgcn_exp2f(m[g] - base);
      m[g] = top;
      l[g] *= fade;
#pragma unroll
      for (int j = 0; j < VEC; j++) o[g][j] *= fade;
#pragma unroll
      for (int u = 0; u < U; u++) {
        const float p = __builtin_amdgcn_exp2f(sc[u] - base);
        l[g] += p;
#pragma unroll
        for (int j = 0; j < VEC; j++) o[g][j] = fmaf(p, v[u][j], o[g][j]);
      }
    }
  }

  // The new row: stored where position n belongs, and attended to as it is stored.
  if (a.append && s == ranges - 1 && wave == 0) {
    const float* kn = a.inp + (size_t)b * a.stride + (size_t)a.NH * HS + (size_t)kvh * HS;
    const float* vn = kn + (size_t)KVH * HS;
    const unsigned row = a.pg.row(b, kvh, n, ok);
    float k[VEC], v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      k[j] = v[j] = 0.f;
      if (at(j) < HS) {
        const E ke = narrow<E>(kn[at(j)]), ve = narrow<E>(vn[at(j)]);
        if (ok && hc == 0 && rg == 0) {
          ((E*)a.pg.keys)[(size_t)row * HS + at(j)] = ke;
          ((E*)a.pg.values)[(size_t)row * HS + at(j)] = ve;
        }
        k[j] = widen(ke);
        v[j] = widen(ve);
      }
    }
#pragma unroll
    for (int g = 0; g < GQ; g++) {
      float d = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; j++) d = fmaf(q[g][j], k[j], d);
      d = row_sum<LPR>(d);
      if (scores && lane == 0 && g < heads) scores[(size_t)g * a.pg.capacity + n] = d;
      if (rg == 0) {
        const float top = fmaxf(m[g], d), base = above(top);
        const float fade = __builtin_amdgcn_exp2f(m[g] - base), p = __builtin_amdgcn_exp2f(d - base);
        m[g] = top;
        l[g] = l[g] * fade + p;
#pragma unroll
        for (int j = 0; j < VEC; j++) o[g][j] = fmaf(p, v[j], o[g][j] * fade);
      }
    }
  }

  // row groups of the wave
#pragma unroll
  for (int g = 0; g < GQ; g++)
#pragma unroll
    for (int off = LPR; off < 64; off *= 2) {
      const float mo = __shfl_xor(m[g], off, 64), lo = __shfl_xor(l[g], off, 64);
      const float top = fmaxf(m[g], mo), base = above(top);
      const float x = __builtin_amdgcn_exp2f(m[g] - base), y = __builtin_amdgcn_exp2f(mo - base);
      m[g] = top;
      l[g] = l[g] * x + lo * y;
#pragma unroll
      for (int j = 0; j < VEC; j++) o[g][j] = o[g][j] * x + __shfl_xor(o[g][j], off, 64) * y;
    }
  // waves of the workgroup
  __shared__ float lds_o[kAttWaves][GQ][LPR * VEC], lds_m[kAttWaves][GQ], lds_l[kAttWaves][GQ];
  const bool all_ok = __ballot(!ok) == 0;
  if (rg == 0) {
#pragma unroll
    for (int g = 0; g < GQ; g++) {
#pragma unroll
      for (int j = 0; j < VEC; j++) lds_o[wave][g][at(j)] = o[g][j];
      if (sub == 0) {
        lds_m[wave][g] = m[g];
        lds_l[wave][g] = all_ok ? l[g] : __builtin_nanf("");  // a page that does not exist: NaN, not a stray read
      }
    }
  }
  __syncthreads();
  const size_t bh0 = (size_t)b * a.NH + head0;
  for (int i = tid; i < heads * HS; i += kAttWaves * kWave) {
    const int g = i / HS, d = i - g * HS;
    float top = lds_m[0][g];
#pragma unroll
    for (int w = 1; w < kAttWaves; w++) top = fmaxf(top, lds_m[w][g]);
    const float base = above(top);
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kAttWaves; w++) {
      const float x = __builtin_amdgcn_exp2f(lds_m[w][g] - base);
      sum = fmaf(x, lds_l[w][g], sum);
      acc = fmaf(x, lds_o[w][g][d], acc);
    }
    const size_t bh = bh0 + g;
    if (ranges == 1)
      a.out[bh * HS + d] = acc / sum;
    else
      a.part_o[(bh * a.S + s) * HS + d] = acc;
    if (d == 0 && a.part_ml) {
      a.part_ml[(bh * a.S + s) * 2] = top;
      a.part_ml[(bh * a.S + s) * 2 + 1] = sum;
    }
  }
}

constexpr int kJoinPositions = 1024;  // positions per workgroup of the weights' part

// Joins the ranges: the first B * NH workgroups the outputs, the others the weights.
__global__ __launch_bounds__(256) void attention_paged_join_kernel(const AttendPaged a) {
  const int HS = a.pg.head_size, tid = threadIdx.x;
  __shared__ float wgt[256], red[256];
  const bool outputs = (int)blockIdx.x < a.B * a.NH;
  if (outputs) {
    const size_t bh = blockIdx.x;
    const int n = a.lengths[bh / a.NH];
    if (n < 0 || n > a.pg.capacity - a.append || n + a.append == 0) return;
    const int ranges = ranges_of(n, range_of(n, a.S));
    if (ranges == 1) return;  // written already
    const float* ml = a.part_ml + bh * a.S * 2;
    red[tid] = tid < ranges ? ml[2 * tid] : -INFINITY;
    __syncthreads();
    float top = -INFINITY;
    for (int s = 0; s < ranges; s++) top = fmaxf(top, red[s]);
    const float base = above(top);
    if (tid < ranges) wgt[tid] = __builtin_amdgcn_exp2f(red[tid] - base);
    __syncthreads();
    float sum = 0.f;
    for (int s = 0; s < ranges; s++) sum = fmaf(wgt[s], ml[2 * s + 1], sum);
    for (int d = tid; d < HS; d += 256) {
      float acc = 0.f;
      for (int s = 0; s < ranges; s++) acc = fmaf(wgt[s], a.part_o[(bh * a.S + s) * HS + d], acc);
      a.out[bh * HS + d] = acc / sum;
    }
    return;
  }
  int id = blockIdx.x - a.B * a.NH;
  const int per = (a.pg.capacity + kJoinPositions - 1) / kJoinPositions;
  const int c = id % per;
  id /= per;
  const int kvh = id % a.pg.kv_heads, b = id / a.pg.kv_heads;
  const int n = a.lengths[b];
  if (n < 0 || n > a.pg.capacity - a.append || n + a.append <= c * kJoinPositions) return;
  const int total = n + a.append, ranges = ranges_of(n, range_of(n, a.S));
  float w[kJoinPositions / 256] = {};
  for (int g = 0; g < a.G; g++) {
    const size_t bh = (size_t)b * a.NH + kvh * a.G + g;
    const float* ml = a.part_ml + bh * a.S * 2;
    float top = -INFINITY, sum = 0.f;
    for (int s = 0; s < ranges; s++) top = fmaxf(top, ml[2 * s]);
    const float base = above(top);
    for (int s = 0; s < ranges; s++) sum = fmaf(__builtin_amdgcn_exp2f(ml[2 * s] - base), ml[2 * s + 1], sum);
#pragma unroll
    for (int j = 0; j < kJoinPositions / 256; j++) {
      const int i = c * kJoinPositions + j * 256 + tid;
      if (i < total) w[j] += __builtin_amdgcn_exp2f(a.scores[bh * a.pg.capacity + i] - base) / sum;
    }
  }
  const size_t at = ((size_t)b * a.pg.kv_heads + kvh) * a.pg.capacity;
#pragma unroll
  for (int j = 0; j < kJoinPositions / 256; j++) {
    const int i = c * kJoinPositions + j * 256 + tid;
    if (i < total) a.weights_out[at + i] = i < n ? a.weights_in[at + i] + w[j] : w[j];
  }
}

// ---- kv_evict_paged -------------------------------------------------------------------------
// The order of weights as unsigned integers: -0 equals 0, and a NaN is the largest of all.
__device__ __forceinline__ unsigned rank_of(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.0f);
  return w != w ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kPickWaves = 16;

// One workgroup per (sequence, kv head) chooses the positions that stay: the `recent` last ones
// and, of the others, the budget - recent of largest weight.  The smallest rank that stays is
// found two bits at a time by counting how many ranks reach each of three candidates (ballots:
// no histogram, no atomics on data, the same result on every run); a wave owns consecutive
// positions, so that the places in the output follow from counts alone.  R ranks per thread are
// kept in registers; R = 0: any length, read again for every count.
template <int R>
__global__ __launch_bounds__(kPickWaves* kWave) void kv_evict_pick_kernel(
    int* __restrict__ kept, int* __restrict__ lengths_out, const float* __restrict__ weights,
    const int* __restrict__ lengths, int KVH, int capacity, int budget, int recent) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t bh = blockIdx.x;
  const int b = (int)(bh / KVH);
  const int n = lengths[b];
  if (n < 0) return;
  const bool too_long = n > capacity;
  const int stay = too_long ? 0 : min(n, budget);
  if (bh % KVH == 0 && tid == 0) lengths_out[b] = too_long ? -1 : stay;
  int* out = kept + bh * budget;
  for (int j = stay + tid; j < budget; j += kPickWaves * kWave) out[j] = -1;
  if (stay == n || too_long) {  // nothing has to go
    for (int j = tid; j < stay; j += kPickWaves * kWave) out[j] = j;
    return;
  }
  const int older = n - recent, want = budget - recent;  // want < older
  for (int j = tid; j < recent; j += kPickWaves * kWave) out[want + j] = older + j;
  if (want == 0) return;

  const float* w = weights + bh * capacity;
  const int span = R ? 64 * R : ((older + kPickWaves - 1) / kPickWaves + 63) & ~63;
  const int first = wave * span, groups = span / 64;
  unsigned rank[R ? R : 1];
  if constexpr (R > 0) {
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int i = first + r * 64 + lane;
      rank[r] = i < older ? rank_of(w[i]) : 0u;
    }
  }
  // group r of this wave's ranks; 0, which no weight has, behind the last position
  auto get = [&](int r) -> unsigned {
    const int i = first + r * 64 + lane;
    return i < older ? rank_of(w[i]) : 0u;
  };
  __shared__ int counts[16][3], waves[2][kPickWaves];
  if (tid < 48) (&counts[0][0])[tid] = 0;
  __syncthreads();
  unsigned low = 0u;
  for (int step = 0; step < 16; step++) {
    const int shift = 30 - 2 * step;
    int c1 = 0, c2 = 0, c3 = 0;
    const unsigned t1 = low | (1u << shift), t2 = low | (2u << shift), t3 = low | (3u << shift);
    if constexpr (R > 0) {
#pragma unroll
      for (int r = 0; r < R; r++) {
        c1 += __popcll(__ballot(rank[r] >= t1));
        c2 += __popcll(__ballot(rank[r] >= t2));
        c3 += __popcll(__ballot(rank[r] >= t3));
      }
    } else {
      for (int r = 0; r < groups; r++) {
        const unsigned x = get(r);
        c1 += __popcll(__ballot(x >= t1));
        c2 += __popcll(__ballot(x >= t2));
        c3 += __popcll(__ballot(x >= t3));
      }
    }
    if (lane == 0) {
      atomicAdd(&counts[step][0], c1);
      atomicAdd(&counts[step][1], c2);
      atomicAdd(&counts[step][2], c3);
    }
    __syncthreads();
    low = counts[step][2] >= want ? t3 : counts[step][1] >= want ? t2 : counts[step][0] >= want ? t1 : low;
  }
  // low is the smallest rank that stays: all above it, and of its equals as many as there is room for
  int gt = 0, eq = 0;
  if constexpr (R > 0) {
#pragma unroll
    for (int r = 0; r < R; r++) {
      gt += __popcll(__ballot(rank[r] > low));
      eq += __popcll(__ballot(rank[r] == low));
    }
  } else {
    for (int r = 0; r < groups; r++) {
      const unsigned x = get(r);
      gt += __popcll(__ballot(x > low));
      eq += __popcll(__ballot(x == low));
    }
  }
  if (lane == 0) {
    waves[0][wave] = gt;
    waves[1][wave] = eq;
  }
  __syncthreads();
  int above_all = 0, gt_before = 0, eq_before = 0;
  for (int i = 0; i < kPickWaves; i++) {
    above_all += waves[0][i];
    if (i < wave) {
      gt_before += waves[0][i];
      eq_before += waves[1][i];
    }
  }
  const int room = want - above_all;  // for ranks that equal low: the lowest positions have it
  const unsigned long long before = (1ull << lane) - 1ull;
  auto place = [&](int r, unsigned x) {
    const unsigned long long g = __ballot(x > low), e = __ballot(x == low);
    const int eq_at = eq_before + __popcll(e & before);
    const bool stays = x > low || (x == low && eq_at < room);
    if (stays) out[gt_before + __popcll(g & before) + min(eq_at, room)] = first + r * 64 + lane;
    gt_before += __popcll(g);
    eq_before += __popcll(e);
  };
  if constexpr (R > 0) {
#pragma unroll
    for (int r = 0; r < R; r++) place(r, rank[r]);
  } else {
    for (int r = 0; r < groups; r++) place(r, get(r));
  }
}

// Copies what stays into the pages of the other table: a wave moves the keys and values of ROWS
// rows of one (sequence, kv head), 16 bytes per lane, and their weights.
template <int UNIT>  // bytes per lane and load: 16, or the size of an element
__global__ __launch_bounds__(256) void kv_evict_copy_kernel(Pages dst, Pages src, const int* __restrict__ kept,
                                                            float* __restrict__ weights_out,
                                                            const float* __restrict__ weights_in,
                                                            const int* __restrict__ lengths, int B, int budget,
                                                            int row_bytes, int groups) {
  const int lane = threadIdx.x & 63;
  const size_t id = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int KVH = src.kv_heads;
  const size_t bh = id / groups;
  const int b = (int)(bh / KVH), h = (int)(bh % KVH);
  if (b >= B) return;
  const int n = lengths[b];
  if (n < 0 || n > src.capacity) return;
  const int j0 = (int)(id % groups) * 64, stay = min(n, budget);
  if (j0 >= stay) return;
  const int j = j0 + lane;
  unsigned from = 0, to = 0;
  bool ok = j < stay;
  if (ok) {
    const int i = kept[bh * budget + j];
    from = src.row(b, h, i, ok);
    to = dst.row(b, h, j, ok);
    weights_out[bh * dst.capacity + j] = ok ? weights_in[bh * src.capacity + i] : __builtin_nanf("");
  }
  const unsigned long long live = __ballot(ok);
  const int units = row_bytes / UNIT, per = 64 / units > 0 ? 64 / units : 1;  // rows per load
  for (int r = 0; r < 64; r += per) {
    const int mine = r + lane / units;
    const unsigned f = __shfl(from, mine & 63, 64), t = __shfl(to, mine & 63, 64);
    if (mine >= 64 || mine >= r + per || !((live >> (mine & 63)) & 1ull)) continue;
    for (int c = lane % units; c < units; c += 64) {
      const size_t x = (size_t)f * row_bytes + (size_t)c * UNIT, y = (size_t)t * row_bytes + (size_t)c * UNIT;
      if constexpr (UNIT == 16) {
        const u32x4 kk = *(const u32x4*)((const char*)src.keys + x), vv = *(const u32x4*)((const char*)src.values + x);
        *(u32x4*)((char*)dst.keys + y) = kk;
        *(u32x4*)((char*)dst.values + y) = vv;
      } else {
        typedef typename std::conditional<UNIT == 4, unsigned, unsigned short>::type W;
        const W kk = *(const W*)((const char*)src.keys + x), vv = *(const W*)((const char*)src.values + x);
        *(W*)((char*)dst.keys + y) = kk;
        *(W*)((char*)dst.values + y) = vv;
      }
    }
  }
}

// ---- launchers ------------------------------------------------------------------------------
static size_t type_bytes(int type) { return type == GPT2HIP_F32 ? 4 : 2; }

static int check_cache(const char* name, const GPT2PagedCache* c, Pages& pg) {
  if (!c) return fail(GPT2HIP_EINVAL, "%s: null cache", name);
  if (c->type != GPT2HIP_F32 && c->type != GPT2HIP_F16 && c->type != GPT2HIP_BF16)
    return fail(GPT2HIP_EINVAL, "%s: unknown cache type %d", name, c->type);
  if (c->num_pages < 1 || c->page_size < 1 || c->max_pages < 1 || c->kv_heads < 1 || c->head_size < 1)
    return fail(GPT2HIP_EINVAL, "%s: bad cache shape num_pages=%d page_size=%d max_pages=%d kv_heads=%d head_size=%d", name,
                c->num_pages, c->page_size, c->max_pages, c->kv_heads, c->head_size);
  if (c->head_size > 256) return fail(GPT2HIP_EINVAL, "%s: head size %d > 256", name, c->head_size);
  if ((long long)c->max_pages * c->page_size > 0x3fffffffLL)
    return fail(GPT2HIP_EINVAL, "%s: %d pages of %d positions: a sequence holds at most 2^30 - 1", name, c->max_pages, c->page_size);
  if ((double)c->num_pages * c->kv_heads * c->page_size > 4294967295.0)
    return fail(GPT2HIP_EINVAL, "%s: num_pages * kv_heads * page_size must be below 2^32", name);
  if (!c->keys || !c->values || !c->table) return fail(GPT2HIP_EINVAL, "%s: null pointer in the cache", name);
  const size_t size = type_bytes(c->type);
  if (((uintptr_t)c->keys | (uintptr_t)c->values) % size)
    return fail(GPT2HIP_EINVAL, "%s: keys and values must be aligned to their element", name);
  pg.keys = c->keys;
  pg.values = c->values;
  pg.table = c->table;
  pg.divide = PageDivide(c->page_size);
  pg.num_pages = c->num_pages;
  pg.max_pages = c->max_pages;
  pg.kv_heads = c->kv_heads;
  pg.head_size = c->head_size;
  pg.capacity = c->max_pages * c->page_size;
  return GPT2HIP_OK;
}

// Rows can be moved 16 bytes per lane.
static bool rows_by_16(const GPT2PagedCache* c) {
  return c->head_size * type_bytes(c->type) % 16 == 0 && aligned16(c->keys) && aligned16(c->values);
}

template <class E>
static void launch_store(const Pages& pg, const float* inp, int stride, const int* starts, const int* lengths, int N,
                         int B, int NH, bool vec) {
  const dim3 grid((unsigned)((N + 3) / 4)), block(256);
  if (vec)
    hipLaunchKernelGGL((kv_store_paged_kernel<E, 4>), grid, block, 0, stream(), pg, inp, stride, starts, lengths, N, B, NH);
  else
    hipLaunchKernelGGL((kv_store_paged_kernel<E, 1>), grid, block, 0, stream(), pg, inp, stride, starts, lengths, N, B, NH);
}

// Query heads that one workgroup takes at once.
static int heads_at_once(int G) { return G >= 5 ? 8 : G >= 3 ? 4 : G; }

// Ranges that a sequence's positions may be split into: enough workgroups to fill the chip.
constexpr int kMaxRanges = 256;
static int ranges_for(int B, int KVH, int G, int capacity) {
  const int gq = heads_at_once(G);
  const long long groups = (long long)B * KVH * ((G + gq - 1) / gq);
  const long long want = (2048 + groups - 1) / groups;
  const long long most = (capacity + kMinRange - 1) / kMinRange;
  const long long s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > kMaxRanges ? kMaxRanges : s);
}

static size_t part_bytes(int B, int NH, int HS, int S) { return (size_t)B * NH * S * (HS + 2) * sizeof(float); }
static size_t score_bytes(int B, int NH, int capacity) { return (size_t)B * NH * capacity * sizeof(float); }

template <class E, int LPR, bool SCALAR>
static void launch_attend(const AttendPaged& a, unsigned blocks) {
  const dim3 grid(blocks), block(kAttWaves * kWave);
  const int gq = heads_at_once(a.G);
  if (gq == 1)
    hipLaunchKernelGGL((attention_paged_kernel<E, LPR, 1, 8, SCALAR>), grid, block, 0, stream(), a);
  else if (gq == 2)
    hipLaunchKernelGGL((attention_paged_kernel<E, LPR, 2, 8, SCALAR>), grid, block, 0, stream(), a);
  else if (gq == 4)
    hipLaunchKernelGGL((attention_paged_kernel<E, LPR, 4, 4, SCALAR>), grid, block, 0, stream(), a);
  else
    hipLaunchKernelGGL((attention_paged_kernel<E, LPR, 8, 4, SCALAR>), grid, block, 0, stream(), a);
}

template <class E>
static void launch_attend(const AttendPaged& a, unsigned blocks, bool vec) {
  const int lanes = (a.pg.head_size + kPer16<E> - 1) / kPer16<E>;
  if (!vec)
    launch_attend<E, 64, true>(a, blocks);
  else if (lanes <= 8)
    launch_attend<E, 8, false>(a, blocks);
  else if (lanes <= 16)
    launch_attend<E, 16, false>(a, blocks);
  else if (lanes <= 32)
    launch_attend<E, 32, false>(a, blocks);
  else if constexpr (sizeof(E) == 4)
    launch_attend<E, 64, false>(a, blocks);
}

}  // namespace g2

extern "C" {

int kv_store_paged_status(const GPT2PagedCache* cache, const float* inp, int inp_stride, const int* starts,
                          const int* lengths, int N, int B, int NH) {
  using namespace g2;
  Pages pg;
  if (int rc = check_cache("kv_store_paged", cache, pg)) return rc;
  if (N < 0 || B < 0 || NH < 0) return fail(GPT2HIP_EINVAL, "kv_store_paged: bad shape N=%d B=%d NH=%d", N, B, NH);
  const long long need = ((long long)NH + 2LL * pg.kv_heads) * pg.head_size;
  if (inp_stride < need)
    return fail(GPT2HIP_EINVAL, "kv_store_paged: rows of %lld floats at a stride of %d", need, inp_stride);
  if (N == 0 || B == 0) return GPT2HIP_OK;
  if (!inp || !starts || !lengths) return fail(GPT2HIP_EINVAL, "kv_store_paged: null pointer");
  const bool vec = pg.head_size % 4 == 0 && inp_stride % 4 == 0 && aligned16(inp) && aligned16(pg.keys) && aligned16(pg.values);
  if (cache->type == GPT2HIP_F32)
    launch_store<float>(pg, inp, inp_stride, starts, lengths, N, B, NH, vec);
  else if (cache->type == GPT2HIP_F16)
    launch_store<f16>(pg, inp, inp_stride, starts, lengths, N, B, NH, vec);
  else
    launch_store<bf16>(pg, inp, inp_stride, starts, lengths, N, B, NH, vec);
  G2_LAUNCH_CHECK("kv_store_paged");
  return GPT2HIP_OK;
}

size_t attention_decode_paged_workspace(const GPT2PagedCache* cache, int B, int NH, int weights) {
  using namespace g2;
  Pages pg;
  if (check_cache("attention_decode_paged_workspace", cache, pg)) return 0;
  if (B < 1 || NH < 1 || NH % pg.kv_heads != 0) return 0;
  const int S = ranges_for(B, pg.kv_heads, NH / pg.kv_heads, pg.capacity);
  return part_bytes(B, NH, pg.head_size, S) + (weights ? score_bytes(B, NH, pg.capacity) : 0);
}

int attention_decode_paged_status(float* out, const GPT2PagedCache* cache, const float* inp, int inp_stride,
                                  const int* lengths, const float* weights_in, float* weights_out, int B, int NH,
                                  int append, void* workspace, size_t workspace_bytes) {
  using namespace g2;
  AttendPaged a;
  if (int rc = check_cache("attention_decode_paged", cache, a.pg)) return rc;
  const int KVH = a.pg.kv_heads, HS = a.pg.head_size;
  if (B < 0 || NH < 1 || NH % KVH != 0)
    return fail(GPT2HIP_EINVAL, "attention_decode_paged: bad shape B=%d NH=%d kv_heads=%d", B, NH, KVH);
  const long long need = ((long long)NH + (append ? 2LL * KVH : 0)) * HS;
  if (inp_stride < need)
    return fail(GPT2HIP_EINVAL, "attention_decode_paged: rows of %lld floats at a stride of %d", need, inp_stride);
  if (!weights_in != !weights_out)
    return fail(GPT2HIP_EINVAL, "attention_decode_paged: weights_in and weights_out go together");
  if (B == 0) return GPT2HIP_OK;
  if (!out || !inp || !lengths) return fail(GPT2HIP_EINVAL, "attention_decode_paged: null pointer");
  if ((uintptr_t)workspace % 256) return fail(GPT2HIP_EINVAL, "attention_decode_paged: workspace must be 256-byte aligned");
  const bool weights = weights_out != nullptr;
  a.out = out;
  a.inp = inp;
  a.lengths = lengths;
  a.weights_in = weights_in;
  a.weights_out = weights_out;
  a.B = B;
  a.NH = NH;
  a.G = NH / KVH;
  const int gq = heads_at_once(a.G);
  a.chunks = (a.G + gq - 1) / gq;
  a.stride = inp_stride;
  a.append = append ? 1 : 0;
  a.scale_log2e = (1.0f / sqrtf((float)HS)) * 1.4426950408889634f;
  // as many ranges as the workspace holds, behind the scores
  const size_t scores = weights ? score_bytes(B, NH, a.pg.capacity) : 0;
  if (!workspace) workspace_bytes = 0;
  a.S = ranges_for(B, KVH, a.G, a.pg.capacity);
  const size_t one = part_bytes(B, NH, HS, 1);
  const size_t room = workspace_bytes > scores ? (workspace_bytes - scores) / one : 0;
  if (weights && room < 1)
    return fail(GPT2HIP_EINVAL, "attention_decode_paged: weights need a workspace of at least %zu bytes, got %zu", scores + one,
                workspace_bytes);
  if (room < (size_t)a.S) a.S = room < 1 ? 1 : (int)room;
  const bool parts = a.S > 1 || weights;
  float* at = (float*)workspace;
  a.part_o = parts ? at : nullptr;
  a.part_ml = parts ? at + (size_t)B * NH * a.S * HS : nullptr;
  a.scores = weights ? a.part_ml + (size_t)B * NH * a.S * 2 : nullptr;
  const long long blocks = (long long)B * KVH * a.chunks * a.S;
  const long long joins = (long long)B * NH +
      (weights ? (long long)B * KVH * ((a.pg.capacity + kJoinPositions - 1) / kJoinPositions) : 0);
  if (blocks > 0x7fffffffLL || joins > 0x7fffffffLL) return fail(GPT2HIP_EINVAL, "attention_decode_paged: grid too large");
  const bool vec = rows_by_16(cache);
  if (cache->type == GPT2HIP_F32)
    launch_attend<float>(a, (unsigned)blocks, vec);
  else if (cache->type == GPT2HIP_F16)
    launch_attend<f16>(a, (unsigned)blocks, vec);
  else
    launch_attend<bf16>(a, (unsigned)blocks, vec);
  G2_LAUNCH_CHECK("attention_decode_paged");
  if (parts) {
    hipLaunchKernelGGL(attention_paged_join_kernel, dim3((unsigned)joins), dim3(256), 0, stream(), a);
    G2_LAUNCH_CHECK("attention_decode_paged (join)");
  }
  return GPT2HIP_OK;
}

int kv_evict_paged_status(const GPT2PagedCache* dst, const GPT2PagedCache* src, int* kept, float* weights_out,
                          int* lengths_out, const float* weights_in, const int* lengths, int B, int budget,
                          int recent) {
  using namespace g2;
  Pages to, from;
  if (int rc = check_cache("kv_evict_paged", dst, to)) return rc;
  if (int rc = check_cache("kv_evict_paged", src, from)) return rc;
  if (dst->type != src->type || to.kv_heads != from.kv_heads || to.head_size != from.head_size)
    return fail(GPT2HIP_EINVAL, "kv_evict_paged: the two caches differ in type, kv_heads or head_size");
  if (B < 0 || budget < 1 || recent < 0 || recent > budget)
    return fail(GPT2HIP_EINVAL, "kv_evict_paged: bad shape B=%d budget=%d recent=%d", B, budget, recent);
  if (budget > to.capacity)
    return fail(GPT2HIP_EINVAL, "kv_evict_paged: a budget of %d does not fit %d pages of %d", budget, dst->max_pages,
                dst->page_size);
  if (dst->keys == src->keys && dst->table == src->table)
    return fail(GPT2HIP_EINVAL, "kv_evict_paged: the rows that stay are copied: dst needs pages of its own");
  if (B == 0) return GPT2HIP_OK;
  if (!kept || !weights_out || !lengths_out || !weights_in || !lengths)
    return fail(GPT2HIP_EINVAL, "kv_evict_paged: null pointer");
  if (weights_out == weights_in || lengths_out == lengths)
    return fail(GPT2HIP_EINVAL, "kv_evict_paged: weights_out and lengths_out must not be the inputs");
  const int KVH = from.kv_heads;
  const int groups = (budget + 63) / 64;
  const long long pairs = (long long)B * KVH, blocks = (pairs * groups + 3) / 4;
  if (pairs > 0x7fffffffLL || blocks > 0x7fffffffLL) return fail(GPT2HIP_EINVAL, "kv_evict_paged: grid too large");
  const dim3 picks((unsigned)pairs), pick_block(kPickWaves * kWave);
  const int most = from.capacity - recent;  // weights that can take part
#define G2_PICK(R)                                                                                              \
  hipLaunchKernelGGL((kv_evict_pick_kernel<R>), picks, pick_block, 0, stream(), kept, lengths_out, weights_in,   \
                     lengths, KVH, from.capacity, budget, recent)
  if (most <= 1024)
    G2_PICK(1);
  else if (most <= 4 * 1024)
    G2_PICK(4);
  else if (most <= 16 * 1024)
    G2_PICK(16);
  else if (most <= 32 * 1024)
    G2_PICK(32);
  else
    G2_PICK(0);
#undef G2_PICK
  G2_LAUNCH_CHECK("kv_evict_paged (choice)");
  const int row_bytes = (int)(from.head_size * type_bytes(src->type));
  const dim3 grid((unsigned)blocks), block(256);
#define G2_COPY(UNIT)                                                                                             \
  hipLaunchKernelGGL((kv_evict_copy_kernel<UNIT>), grid, block, 0, stream(), to, from, kept, weights_out, weights_in, \
                     lengths, B, budget, row_bytes, groups)
  if (rows_by_16(src) && rows_by_16(dst))
    G2_COPY(16);
  else if (src->type == GPT2HIP_F32)
    G2_COPY(4);
  else
    G2_COPY(2);
#undef G2_COPY
  G2_LAUNCH_CHECK("kv_evict_paged (copy)");
  return GPT2HIP_OK;
}

}  // extern "C"
