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
// Division by the page size as one product and a shift, exact for every 31-bit position:
// with log = ceil(log2 d) and magic = ceil(2^(31 + log) / d), magic fits 32 bits and
// floor(n * magic / 2^(31 + log)) = floor(n / d) for n < 2^31, because magic * d exceeds
// 2^(31 + log) by less than d <= 2^log.
struct PageDivide {
  unsigned magic;
  int shift;  // 31 + log
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
// A copy, bound by memory: 8 prompts of 129-1023 rows, 12 heads, fp32: 13.5 us = 4.8 TB/s; 4 of
// 4001-8192 rows, 8 heads of 128, bf16: 57.5 us = 5.5 TB/s (a streaming copy of 192 MiB reaches 6.2,
// one that writes half of what it reads 6.3-6.5, torch's copy of 2 GiB 4.9).  16-bit rows are stored
// past the caches (12 x 5-496 rows, 20 heads, fp16: 13.8 -> 11.9 us; fp32 gains nothing).
// The first loads of the row are under way while its place is looked up.
template <class E, int VEC>
__global__ __launch_bounds__(256) void kv_store_paged_kernel(Pages pg, const float* __restrict__ inp, int stride,
                                                             const int* __restrict__ starts,
                                                             const int* __restrict__ lengths, int N, int B, int NH) {
  constexpr int U = 4, STEP = 64 * VEC;  // loads at a time, floats of one
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= N) return;
  const int HS = pg.head_size, half = pg.kv_heads * HS;
  const float* src = inp + (size_t)r * stride + (size_t)NH * HS;
  typedef float In __attribute__((ext_vector_type(VEC)));
  In x[U];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = min(i0 + u * STEP + lane * VEC, 2 * half - VEC);
      if constexpr (VEC == 4)
        x[u] = __builtin_nontemporal_load(reinterpret_cast<const In*>(src + i));
      else
        x[u][0] = src[i];
    }
  };
  load(0);
  int b = -1, begin = 0, n = 0;
  for (int i = 0; i <= B; i += 64) {
    const int mine = min(i + lane, B);
    const int start = starts[mine], held = lengths[min(mine, B - 1)];
    const unsigned long long m = __ballot(i + lane <= B && start <= r);
    const int before = __popcll(m);
    if (before > 0) {
      begin = __builtin_amdgcn_readlane(start, before - 1);
      n = __builtin_amdgcn_readlane(held, before - 1);
    }
    b += before;
    if (m != ~0ull) break;
  }
  // in front of the first row or behind the last; starts that do not ascend are nobody's either
  if (b < 0 || b >= B || begin > r || starts[b + 1] <= r) return;
  const long long pos = (long long)n + r - begin;  // begin may be below 0
  if (n < 0 || pos >= pg.capacity) return;
  bool ok = true;
  const unsigned row0 = pg.row(b, 0, (int)pos, ok);
  if (!ok) return;
  for (int i0 = 0; i0 < 2 * half; i0 += U * STEP) {
    if (i0 > 0) load(i0);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * STEP + lane * VEC;
      if (i >= 2 * half) break;
      const bool value = i >= half;
      const int c = value ? i - half : i;
      const int head = c / HS, d = c - head * HS;
      E* to = (E*)(value ? pg.values : pg.keys) + ((size_t)row0 + (size_t)head * pg.divide.size) * HS + d;
      if constexpr (VEC == 4) {
        typedef unsigned Words __attribute__((ext_vector_type(sizeof(E))));
        struct Four {
          E e[4];
        };
        const Four y{{narrow<E>(x[u][0]), narrow<E>(x[u][1]), narrow<E>(x[u][2]), narrow<E>(x[u][3])}};
        if constexpr (sizeof(E) == 2)
          __builtin_nontemporal_store(__builtin_bit_cast(Words, y), reinterpret_cast<Words*>(to));
        else
          *reinterpret_cast<Words*>(to) = __builtin_bit_cast(Words, y);
      } else {
        to[0] = narrow<E>(x[u][0]);
      }
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
  // workspace, where the work is split or weights are asked for
  unsigned* counters;  // (B, kv_heads, chunks) ranges that have arrived: zero between calls
  float* part_o;       // (kv_heads, chunks, slots, part_heads, part_stride) unnormalised outputs of the ranges
  float* part_ml;      // (kv_heads, chunks, slots, part_heads, 2) their maxima and sums, in the exponent's base-2 scale
  float* joined;       // (B, NH, 2) the whole row's
  float* scores;       // (B, NH, score_stride) base-2 scores
  int B, NH, G, chunks;  // G query heads per kv head, in `chunks` groups of at most GQ
  int stride, append;
  int slots, min_range;  // workgroups per kv head and chunk: B, or more, for ranges of at least min_range positions
  int weigh_here;        // weights by the same workgroup (no splitting, one chunk)
  int part_heads, part_stride, score_stride;
  float scale_log2e;
};

constexpr int kCounterStride = 32;  // a cache line each: counters that share one are counted one after the other
constexpr int kMostSplit = 256;     // sequences whose lengths a wave looks through, four per lane

// exp2(s - above(m)) where m is the running maximum: a maximum of -inf (nothing seen, or only
// scores of -inf) counts as 0, so that such scores weigh 0 instead of NaN.
__device__ __forceinline__ float above(float m) { return m == -INFINITY ? 0.f : m; }

// What one workgroup is to do.
struct Range {
  int b, kvh, hc;            // sequence, kv head, chunk of its query heads
  int head0, heads;          // the chunk's query heads
  int n, ranges, s, first;   // positions held, ranges they are dealt to, this one, the slot of the first
  int p0, p1;                // this range
  bool adds;                 // the new row belongs to it
};

__device__ __forceinline__ int across_rows(int v) {  // the sum over the lanes 16, 32 and 48 apart
  const auto h = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
  v = (int)(h[0] + h[1]);
  const auto r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
  return (int)(r[0] + r[1]);
}
__device__ __forceinline__ int wave_sum_int(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true);
  return across_rows(v);
}
// The sum of this lane's value and of those in front of it.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// Ranges of `size` positions that n positions make, at least one; 0 for an unused place (n < 0).
__device__ __forceinline__ int ranges_of(int n, int size, float inverse) {
  int q = (int)((float)n * inverse);  // off by one at most: sizes are an even share or more, so q <= slots
  int rest = n - q * size;
  if (rest < 0) {
    q--;
    rest += size;
  }
  q += rest > size ? 2 : rest > 0 ? 1 : 0;
  return n < 0 ? 0 : max(q, 1);
}

// Deals the positions of all sequences to a.slots workgroups in ranges of one size, so that a long
// sequence gets more of them: slot `slot`'s sequence and range.  The size is the smallest of 16
// between what an even share would be and what fits whatever the lengths (sum of n / size, and one
// more range per sequence); four lanes at a time count a size's ranges.  Every wave of every
// workgroup comes to the same result.  (4 sequences of 1-30000 positions, 4 of 32 heads of 128,
// bf16: 31.7 us, where every sequence is cut into as many ranges 40.6.)
__device__ __forceinline__ bool deal(const AttendPaged& a, int slot, int lane, Range& w, int& size) {
  const int most = a.pg.capacity - a.append;  // a sequence that does not fit is a range of nothing
  if (a.B == 1) {
    w.n = a.lengths[0];
    const int n = w.n > most ? 0 : max(w.n, 0);
    size = max(a.min_range, ((n + a.slots - 1) / a.slots + 63) & ~63);
    w.ranges = max((n + size - 1) / size, 1);
    w.b = w.first = 0;
    w.s = slot;
    return slot < w.ranges;
  }
  const int per = (a.B + 63) >> 6, lanes = (a.B + per - 1) / per;
  int held[4], n[4], places = 0;  // `per` sequences in this lane
#pragma unroll
  for (int k = 0; k < 4; k++) held[k] = k < per ? a.lengths[min(lane * per + k, a.B - 1)] : -1;
  float total = 0.f;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    if (k >= per || lane * per + k >= a.B) held[k] = -1;
    n[k] = held[k] > most ? 0 : held[k];
    places += __popcll(__ballot(n[k] >= 0));
    total += (float)max(n[k], 0);
  }
  total = wave_sum(total);
  if (places == 0) return false;
  const float even = total / (float)a.slots, safe = total / (float)(a.slots - places) * 1.0001f + 1.f;
  const float share = even + (safe - even) * (float)(lane & 15) * (1.f / 15.f);
  const int mine = max(a.min_range, ((int)fminf(share, 1073741824.f) + 64) & ~63);
  const float inverse = 1.f / (float)mine;
  int count = 0;
  for (int j = 0; j < lanes; j += 4)
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (k < per) count += ranges_of(__shfl(n[k], j + (lane >> 4), 64), mine, inverse);
  count = across_rows(count);
  const unsigned fits = (unsigned)__ballot(count <= a.slots) & 0xffffu;  // the last one always does
  size = __builtin_amdgcn_readlane(mine, fits ? __builtin_ctz(fits) : 15);
  const float by = 1.f / (float)size;
  int c[4], sum = 0;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    c[k] = ranges_of(n[k], size, by);
    sum += c[k];
  }
  const int upto = wave_scan(sum);
  const int who = __popcll(__ballot(upto <= slot));
  if (who == 64) return false;
  int left = slot - __builtin_amdgcn_readlane(upto - sum, who);
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int ck = __builtin_amdgcn_readlane(c[k], who);
    if (left >= 0 && left < ck) {
      w.b = who * per + k;
      w.n = __builtin_amdgcn_readlane(held[k], who);
      w.ranges = ck;
      w.s = left;
      w.first = slot - left;
      left = -1;
    } else if (left >= 0) {
      left -= ck;
    }
  }
  return true;
}

// False where there is nothing (left) to do: unused places, slots past the last range, sequences
// that do not fit (NaN) or hold nothing (zeros).
template <int W>
__device__ __forceinline__ bool take_range(const AttendPaged& a, int GQ, int tid, Range& w) {
  const int per = a.pg.kv_heads * a.chunks;
  const int slot = blockIdx.x / per, rest = blockIdx.x - slot * per;
  w.kvh = rest / a.chunks;
  w.hc = rest - w.kvh * a.chunks;
  w.head0 = w.kvh * a.G + w.hc * GQ;
  w.heads = min(GQ, a.G - w.hc * GQ);
  int size = 0x7fffffff;
  if (a.slots > a.B) {
    if (!deal(a, slot, tid & 63, w, size)) return false;
  } else {
    w.b = w.first = slot;
    w.ranges = 1;
    w.s = 0;
    w.n = a.lengths[slot];
  }
  if (w.n < 0) return false;
  const bool too_long = w.n > a.pg.capacity - a.append;
  if (too_long || w.n + a.append == 0) {
    const float fill = too_long ? __builtin_nanf("") : 0.f;
    for (int i = tid; i < w.heads * a.pg.head_size; i += W * kWave)
      a.out[((size_t)w.b * a.NH + w.head0) * a.pg.head_size + i] = fill;
    return false;
  }
  w.p0 = w.s == 0 ? 0 : w.s * size;
  w.p1 = w.s == w.ranges - 1 ? w.n : w.p0 + size;
  w.adds = a.append && w.s == w.ranges - 1;
  return true;
}

// What the waves of a workgroup hand each other: per wave and head the unnormalised output, the
// maximum and the sum, and as one more "wave" the new row (sum 1, output its value).  Later the
// same memory holds what joins the ranges.
template <int W, int GQ, int ROW>
struct Meeting {
  static_assert(ROW % 4 == 0, "rows are read four floats at a time");
  union {
    float o[W][GQ][ROW];
    struct {
      f32x4 sum[W * kWave];
      float m[W * kWave], l[W * kWave];
    } join;
  };
  float v[ROW];
  float m[W + 1][GQ], l[W][GQ];
  float base[GQ], sum[GQ];  // the whole row's, where one workgroup has it all
  int last;
};

// 16 bytes of floats at any address that floats may have.
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

// The new row: rounded as the cache holds it, stored (by the first wave, once per kv head), and
// scored against the chunk's queries, a head per wave at a time.
template <class E, int W, int GQ, int ROW>
__device__ __forceinline__ bool add_row(const AttendPaged& a, const Range& w, int lane, int wave,
                                        Meeting<W, GQ, ROW>& meet) {
  constexpr int N = (ROW + 63) / 64;
  if (wave > 0 && wave >= w.heads) return true;
  const int HS = a.pg.head_size;
  const float* row = a.inp + (size_t)w.b * a.stride;
  const float* kn = row + ((size_t)a.NH + w.kvh) * HS;
  const float* vn = kn + (size_t)a.pg.kv_heads * HS;
  bool ok = true;
  float k[N];
#pragma unroll
  for (int j = 0; j < N; j++) k[j] = lane + 64 * j < HS ? kn[lane + 64 * j] : 0.f;
  if (wave == 0) {
    const size_t to = (size_t)a.pg.row(w.b, w.kvh, w.n, ok) * HS;
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int d = lane + 64 * j;
      const E ve = narrow<E>(d < HS ? vn[d] : 0.f);
      if (d < HS && ok && w.hc == 0) {
        ((E*)a.pg.keys)[to + d] = narrow<E>(k[j]);
        ((E*)a.pg.values)[to + d] = ve;
      }
      if (d < ROW) meet.v[d] = widen(ve);
    }
  }
#pragma unroll
  for (int j = 0; j < N; j++) k[j] = widen(narrow<E>(k[j]));
  for (int g = wave; g < w.heads; g += W) {
    const float* q = row + (size_t)(w.head0 + g) * HS;
    float d = 0.f;
#pragma unroll
    for (int j = 0; j < N; j++)
      if (lane + 64 * j < HS) d = fmaf(q[lane + 64 * j] * a.scale_log2e, k[j], d);
    d = wave_sum(d);
    if (lane == 0) {
      meet.m[W][g] = d;
      if (a.scores) a.scores[((size_t)w.b * a.NH + w.head0 + g) * a.score_stride + w.n] = d;
    }
  }
  return ok;
}

// Joins the waves and, where the sequence was dealt to several workgroups, the ranges: each leaves
// its part in the workspace, and whichever of them arrives last (a counter tells it, nobody waits)
// joins all of them in order, so that the result does not depend on which one that was.  The
// parts cross XCDs: they are written and read with the cache-bypassing policy, and every wave
// waits for its stores before the workgroup counts itself in.
template <int W, int GQ, int ROW>
__device__ __forceinline__ void finish(const AttendPaged& a, const Range& w, int tid, Meeting<W, GQ, ROW>& meet) {
  constexpr int THREADS = W * kWave;
  const int HS = a.pg.head_size, HP4 = a.part_stride >> 2;
  const size_t bh0 = (size_t)w.b * a.NH + w.head0;
  const size_t part0 = w.ranges > 1 ? ((size_t)(w.kvh * a.chunks + w.hc) * a.slots + w.first) * a.part_heads : 0;
  const Bypass parts(a.part_o + part0 * a.part_stride, w.ranges > 1 ? (size_t)w.ranges * a.part_heads * a.part_stride : 0);
  unsigned long long* const part_ml = reinterpret_cast<unsigned long long*>(a.part_ml) + part0;
  __syncthreads();
  for (int i = tid; i < w.heads * HP4; i += THREADS) {
    const int g = i / HP4, d = (i - g * HP4) * 4;
    float top = meet.m[0][g];
#pragma unroll
    for (int k = 1; k < W; k++) top = fmaxf(top, meet.m[k][g]);
    if (w.adds) top = fmaxf(top, meet.m[W][g]);
    const float base = above(top);
    float sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < W; k++) {
      const float x = __builtin_amdgcn_exp2f(meet.m[k][g] - base);
      sum = fmaf(x, meet.l[k][g], sum);
      acc += x * *reinterpret_cast<const f32x4*>(&meet.o[k][g][d]);
    }
    if (w.adds) {
      const float x = __builtin_amdgcn_exp2f(meet.m[W][g] - base);
      sum += x;
      acc += x * *reinterpret_cast<const f32x4*>(&meet.v[d]);
    }
    if (w.ranges == 1) {
      float* out = a.out + (bh0 + g) * HS + d;
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (d + e < HS) out[e] = acc[e] / sum;
      if (d == 0 && a.joined) {
        a.joined[(bh0 + g) * 2] = base;
        a.joined[(bh0 + g) * 2 + 1] = sum;
      }
      if (d == 0) {
        meet.base[g] = base;
        meet.sum[g] = sum;
      }
    } else {
      const int at = w.s * a.part_heads + g;
      parts.store4(at * a.part_stride + d, acc);
      if (d == 0) {
        const unsigned long long both = (unsigned long long)__builtin_bit_cast(unsigned, sum) << 32 | __builtin_bit_cast(unsigned, top);
        __hip_atomic_store(part_ml + at, both, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if (w.ranges == 1) return;
  wait_vm();
  __syncthreads();
  if (tid == 0) {
    unsigned* counter = a.counters + kCounterStride * (((size_t)w.b * a.pg.kv_heads + w.kvh) * a.chunks + w.hc);
    const unsigned old = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool last = old + 1u == (unsigned)w.ranges;
    if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    meet.last = last;
  }
  __syncthreads();
  if (!meet.last) return;
  // As many threads per four channels as there are to spare, each with every so manieth range and
  // a softmax of its own over them; all loads of a thread are under way at once.
  constexpr int MOST = 8;
  int per = 1;
  while (per < w.heads * HP4 && per < THREADS) per *= 2;
  const int slices = THREADS / per, slice = tid / per;
  for (int i0 = 0; i0 < w.heads * HP4; i0 += per) {
    const int i = min(i0 + (tid & (per - 1)), w.heads * HP4 - 1);
    const int g = i / HP4, d = (i - g * HP4) * 4;
    float m = -INFINITY, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = slice; s0 < w.ranges; s0 += MOST * slices) {
      unsigned long long x[MOST];
      f32x4 p[MOST];
#pragma unroll
      for (int u = 0; u < MOST; u++) {
        const int s = s0 + u * slices;
        x[u] = 0;
        p[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (s < w.ranges) {
          const int at = s * a.part_heads + g;
          x[u] = __hip_atomic_load(part_ml + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          p[u] = parts.load4(at * a.part_stride + d);
        }
      }
      float mu[MOST], top = m;
#pragma unroll
      for (int u = 0; u < MOST; u++) {
        const unsigned bits = (unsigned)x[u];
        mu[u] = s0 + u * slices < w.ranges ? __builtin_bit_cast(float, bits) : -INFINITY;
        top = fmaxf(top, mu[u]);
      }
      const float base = above(top), fade = __builtin_amdgcn_exp2f(m - base);
      m = top;
      l *= fade;
      acc *= fade;
#pragma unroll
      for (int u = 0; u < MOST; u++)
        if (s0 + u * slices < w.ranges) {
          const unsigned bits = (unsigned)(x[u] >> 32);
          const float f = __builtin_amdgcn_exp2f(mu[u] - base);
          l = fmaf(f, __builtin_bit_cast(float, bits), l);
          acc += f * p[u];
        }
    }
    if (slices > 1) {
      meet.join.sum[tid] = acc;
      meet.join.m[tid] = m;
      meet.join.l[tid] = l;
      __syncthreads();
      if (slice == 0) {
        float top = m;
        for (int k = 1; k < slices; k++) top = fmaxf(top, meet.join.m[tid + k * per]);
        const float base = above(top), fade = __builtin_amdgcn_exp2f(m - base);
        m = top;
        l *= fade;
        acc *= fade;
        for (int k = 1; k < slices; k++) {
          const float f = __builtin_amdgcn_exp2f(meet.join.m[tid + k * per] - base);
          l = fmaf(f, meet.join.l[tid + k * per], l);
          acc += f * meet.join.sum[tid + k * per];
        }
      }
    }
    if (slice == 0 && i0 + (tid & (per - 1)) < w.heads * HP4) {
      float* out = a.out + (bh0 + g) * HS + d;
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (d + e < HS) out[e] = acc[e] / l;
      if (d == 0 && a.joined) {
        a.joined[(bh0 + g) * 2] = above(m);
        a.joined[(bh0 + g) * 2 + 1] = l;
      }
    }
  }
}

// weights_out = weights_in + sum over the group's heads of exp2(score - maximum) / sum, where this
// workgroup has all positions and heads of a kv head.
template <int W, int GQ, int ROW>
__device__ __forceinline__ void weigh(const AttendPaged& a, const Range& w, int tid, Meeting<W, GQ, ROW>& meet) {
  __syncthreads();  // the scores of all waves and meet.base, meet.sum
  const size_t at = ((size_t)w.b * a.pg.kv_heads + w.kvh) * a.pg.capacity;
  const float* scores = a.scores + ((size_t)w.b * a.NH + w.head0) * a.score_stride;
  for (int i = tid; i < w.n + a.append; i += W * kWave) {
    float x = i < w.n ? a.weights_in[at + i] : 0.f, p = 0.f;
#pragma unroll 4
    for (int g = 0; g < w.heads; g++)
      p += __builtin_amdgcn_exp2f(scores[(size_t)g * a.score_stride + i] - meet.base[g]) / meet.sum[g];
    a.weights_out[at + i] = x + p;
  }
}

// Sums across the four rows of 16 lanes, two values for the price of one: v_permlane32_swap puts
// x's halves side by side with y's, v_permlane16_swap rows with rows.
__device__ __forceinline__ float halves_sum(float x, float y) {  // lanes 0-31: x's, lanes 32-63: y's
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
  const unsigned lo = r[0], hi = r[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float rows_sum(float x, float y) {  // rows 0, 2: x's; rows 1, 3: y's
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
  const unsigned lo = r[0], hi = r[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}
// The maximum across the lanes that are LPR and more apart, for every lane.
template <int LPR>
__device__ __forceinline__ float rows_max(float v) {
  if constexpr (LPR <= 32) {
    const auto h = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned lo = h[0], hi = h[1];
    v = fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
  }
  if constexpr (LPR <= 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned lo = r[0], hi = r[1];
    v = fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
  }
  if constexpr (LPR <= 8) v = fmaxf(v, dpp<0x128>(v));  // row_ror:8
  return v;
}
// The sums of four values over the four rows: row i of 16 lanes receives that of value quad_value(i).
__device__ __forceinline__ float quads_sum(float x0, float x1, float x2, float x3) {
  return rows_sum(halves_sum(x0, x1), halves_sum(x2, x3));
}
__device__ __forceinline__ int quad_value(int quad) { return quad == 1 ? 2 : quad == 2 ? 1 : quad; }

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

// One or two query heads per kv head: LPR lanes hold one row of keys or values, 16 bytes each, so
// that a wave's load covers 64 / LPR rows; every such group of lanes keeps a softmax (maximum,
// sum, output) of its own over the rows it has seen, and the groups, the waves and the ranges meet
// only at the end.  Bound by reading the cache: 64 sequences of 200-1023 positions, 25 heads, bf16:
// 44 us = 5.7 TB/s; one of 65001, 20 heads, fp16: 56 us = 5.9 TB/s (a streaming read: 6.4-7.1).
// Eight rows per lane group and tile (U) at one workgroup per unit, four at two: see plan_attend.
// SCALAR: rows of any size and alignment and any number of heads, GQ at a time: a row per wave,
// one element per lane and load.
template <class E, int LPR, int GQ, int U, int W, bool SCALAR>
__global__ __launch_bounds__(W* kWave) void attention_paged_kernel(const AttendPaged a) {
  constexpr int VEC = SCALAR ? 4 : kPer16<E>;
  constexpr int RPW = 64 / LPR;
  constexpr int TILE = U * RPW;
  constexpr int ROW = LPR * VEC;
  static_assert(TILE <= 64, "a tile's rows are looked up by one lane each");
  __shared__ Meeting<W, GQ, ROW> meet;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sub = lane & (LPR - 1), rg = lane / LPR;
  const int HS = a.pg.head_size;
  Range w;
  if (!take_range<W>(a, GQ, tid, w)) return;
  // element j of this lane's part of a row
  auto at = [&](int j) { return SCALAR ? sub + 64 * j : sub * VEC + j; };
  const bool live = SCALAR || sub * VEC < HS;  // lanes behind the row's end read its last piece and count for nothing
  const int piece = SCALAR ? 0 : min(sub * VEC, HS - VEC);
  float q[GQ][VEC], o[GQ][VEC], m[GQ], l[GQ];
#pragma unroll
  for (int g = 0; g < GQ; g++) {
    const float* src = a.inp + (size_t)w.b * a.stride + (size_t)(w.head0 + (g < w.heads ? g : 0)) * HS;
    if constexpr (SCALAR) {
#pragma unroll
      for (int j = 0; j < VEC; j++) q[g][j] = src[min(at(j), HS - 1)];
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        const f32x4 f = *reinterpret_cast<const f32x4_any*>(src + piece + j);
#pragma unroll
        for (int e = 0; e < 4; e++) q[g][j + e] = f[e];
      }
    }
  }
  bool ok = true;
  const int p1 = w.p1;
  int t = w.p0 + wave * TILE;
  // the rows of the tile at `from`, one per lane (behind the range: of its last position)
  auto look_up = [&](int from) { return a.pg.row(w.b, w.kvh, min(from + (lane & (TILE - 1)), p1 - 1), ok); };
  unsigned rows = 0, rows_next = 0;
  if (t < p1) rows = look_up(t);
  if (t + W * TILE < p1) rows_next = look_up(t + W * TILE);

  // Rows are kept as they are loaded until they are used.  The keys' registers are free once the
  // scores are known and the values' once they are added up: the next tile's loads go there at
  // once, so that half of a tile is always under way.
  typedef typename std::conditional<SCALAR, E[VEC], u32x4>::type Raw;
  struct Piece {
    Raw x;
  };
  auto load = [&](const void* base, unsigned row) {
    const E* p = (const E*)base + (size_t)row * HS;
    Piece r;
    if constexpr (SCALAR) {
#pragma unroll
      for (int j = 0; j < VEC; j++) r.x[j] = p[min(at(j), HS - 1)];
    } else {
      r.x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + piece));
    }
    return r;
  };
  auto unpack = [&](float (&to)[VEC], const Piece& r) {
    if constexpr (SCALAR) {
#pragma unroll
      for (int j = 0; j < VEC; j++) to[j] = at(j) < HS ? widen(r.x[j]) : 0.f;
    } else {
      widen16(to, r.x, E{});
    }
  };
  float* const scores = a.scores ? a.scores + ((size_t)w.b * a.NH + w.head0) * a.score_stride : nullptr;

  Piece kr[U], vr[U];
  // one tile; MORE: another follows, so that this one is whole
  auto step = [&](auto more) {
    constexpr bool MORE = decltype(more)::value;
    unsigned rows_after = 0;
    if constexpr (MORE) {
      if (t + 2 * W * TILE < p1) rows_after = look_up(t + 2 * W * TILE);
    }
    float sc[GQ][U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      float k[VEC];
      unpack(k, kr[u]);
      const bool in = MORE || t + u * RPW + rg < p1;
#pragma unroll
      for (int g = 0; g < GQ; g++) {
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; j++) d = fmaf(q[g][j], k[j], d);
        d = row_sum<LPR>(live ? d : 0.f);
        if (scores && sub == 0 && in && g < w.heads) scores[(size_t)g * a.score_stride + t + u * RPW + rg] = d;
        sc[g][u] = in ? d : -INFINITY;
      }
    }
    if constexpr (MORE) {
#pragma unroll
      for (int u = 0; u < U; u++) kr[u] = load(a.pg.keys, __shfl(rows_next, u * RPW + rg, 64));
    }
#pragma unroll
    for (int g = 0; g < GQ; g++) {
      float top = m[g];
#pragma unroll
      for (int u = 0; u < U; u++) top = fmaxf(top, sc[g][u]);
      const float base = above(top);
      const float fade = __builtin_amdgcn_exp2f(m[g] - base);
      m[g] = top;
      l[g] *= fade;
#pragma unroll
      for (int j = 0; j < VEC; j++) o[g][j] *= fade;
#pragma unroll
      for (int u = 0; u < U; u++) {
        sc[g][u] = __builtin_amdgcn_exp2f(sc[g][u] - base);
        l[g] += sc[g][u];
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      float v[VEC];
      unpack(v, vr[u]);
      // rows behind the range were read as copies of its last one: they weigh nothing, whatever they hold
      if (!MORE && t + u * RPW + rg >= p1) {
#pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = 0.f;
      }
#pragma unroll
      for (int g = 0; g < GQ; g++)
#pragma unroll
        for (int j = 0; j < VEC; j++) o[g][j] = fmaf(sc[g][u], v[j], o[g][j]);
    }
    if constexpr (MORE) {
#pragma unroll
      for (int u = 0; u < U; u++) vr[u] = load(a.pg.values, __shfl(rows_next, u * RPW + rg, 64));
      rows_next = rows_after;
      t += W * TILE;
    }
  };
  if (t < p1) {
#pragma unroll
    for (int u = 0; u < U; u++) kr[u] = load(a.pg.keys, __shfl(rows, u * RPW + rg, 64));
#pragma unroll
    for (int u = 0; u < U; u++) vr[u] = load(a.pg.values, __shfl(rows, u * RPW + rg, 64));
  }
  if (w.adds) ok &= add_row<E>(a, w, lane, wave, meet);
#pragma unroll
  for (int g = 0; g < GQ; g++) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      o[g][j] = 0.f;
      q[g][j] *= a.scale_log2e;
    }
  }
  if (t < p1) {
    while (t + W * TILE < p1) step(std::true_type{});
    step(std::false_type{});
  }

  // row groups of the wave
  const bool all_ok = __ballot(!ok) == 0;
#pragma unroll
  for (int g = 0; g < GQ; g++) {
    const float top = rows_max<LPR>(m[g]);
    const float fade = __builtin_amdgcn_exp2f(m[g] - above(top));
    float sum = l[g] * fade;
#pragma unroll
    for (int j = 0; j < VEC; j++) o[g][j] *= fade;
    if constexpr (LPR <= 8) {  // row_ror:8: the two groups of a row of 16 lanes
      sum += dpp<0x128>(sum);
#pragma unroll
      for (int j = 0; j < VEC; j++) o[g][j] += dpp<0x128>(o[g][j]);
    }
    if constexpr (LPR <= 16) {
      sum = quads_sum(sum, sum, sum, sum);
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        const float x = quads_sum(o[g][j], o[g][j + 1], o[g][j + 2], o[g][j + 3]);
        if ((lane & 15) < LPR) meet.o[wave][g][sub * VEC + j + quad_value(lane >> 4)] = x;
      }
    } else if constexpr (LPR == 32) {
      sum = halves_sum(sum, sum);
#pragma unroll
      for (int j = 0; j < VEC; j += 2) meet.o[wave][g][sub * VEC + j + rg] = halves_sum(o[g][j], o[g][j + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j++) meet.o[wave][g][at(j)] = o[g][j];
    }
    if (lane == 0) {
      meet.m[wave][g] = top;
      meet.l[wave][g] = all_ok ? sum : __builtin_nanf("");  // a page that does not exist: NaN, not a stray read
    }
  }
  finish(a, w, tid, meet);
  if (a.weigh_here) weigh(a, w, tid, meet);
}

// ---- several query heads per kv head: matrix instructions -----------------------------------
// Scores and outputs of 16 positions by 16 heads are 16x16 tiles.  Transposed scores
// S^T = K Q^T: a lane loads 16 bytes of the key row of position (lane % 16), which is an operand
// as it comes from memory, and receives the scores of four positions 4 (lane / 16) + r for head
// (lane % 16).  That is at once how the other product wants its left operand: O = P V with V's
// rows loaded by the lanes of the same four positions.  Neither K, V nor P pass through LDS.
//
// The matrix instructions for a 16-bit cache would round the fp32 queries and weights.  So each is
// cut into as many pieces of 8 (bf16: 3) or 11 (fp16: 2) bits as make up its 24, and their
// products, exact in fp32, are added up.  Heads beyond the group's are computed on zeros: the
// kernel is bound by reading the cache (at 16 heads as at 3), not by these instructions: 8 sequences
// of 28000-32767 positions, 8 of 32 heads of 128 channels, bf16: 160 us = 6.3 TB/s.  One query head
// per kv head is faster without them (64 sequences of 25 heads, bf16: 54 against 44 us).
template <class E>
struct Mx;
template <>
struct Mx<float> {
  static constexpr int PIECES = 1;
};
template <>
struct Mx<f16> {
  static constexpr int PIECES = 2;
};
template <>
struct Mx<bf16> {
  static constexpr int PIECES = 3;
};
constexpr int kMatrixHeads = 16;
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ unsigned bits_of(float v) { return __builtin_bit_cast(unsigned, v); }
__device__ __forceinline__ float float_of(unsigned v) { return __builtin_bit_cast(float, v); }
// the upper, the lower halves of two words as one
__device__ __forceinline__ unsigned upper_halves(unsigned lo, unsigned hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}
__device__ __forceinline__ unsigned lower_halves(unsigned lo, unsigned hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
// The pieces of two floats, packed: bf16 by cutting off (8 + 8 + 8 bits are all of a float's 24),
// fp16 by rounding (11 + 11 bits and two signs leave half a step of fp32 at most).
__device__ __forceinline__ void cut(unsigned (&to)[3], float a, float b, bf16) {
  const float a1 = a - float_of(bits_of(a) & 0xffff0000u), b1 = b - float_of(bits_of(b) & 0xffff0000u);
  const float a2 = a1 - float_of(bits_of(a1) & 0xffff0000u), b2 = b1 - float_of(bits_of(b1) & 0xffff0000u);
  to[0] = upper_halves(bits_of(a), bits_of(b));
  to[1] = upper_halves(bits_of(a1), bits_of(b1));
  to[2] = upper_halves(bits_of(a2), bits_of(b2));
}
__device__ __forceinline__ void cut(unsigned (&to)[2], float a, float b, f16) {
  typedef f16 f16x2 __attribute__((ext_vector_type(2)));
  const f16x2 hi = {(f16)a, (f16)b};
  const f16x2 lo = {(f16)(a - (float)hi[0]), (f16)(b - (float)hi[1])};
  to[0] = __builtin_bit_cast(unsigned, hi);
  to[1] = __builtin_bit_cast(unsigned, lo);
}

__device__ __forceinline__ f32x4 mfma32(u32x4 x, u32x4 y, f32x4 c, f16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma32(u32x4 x, u32x4 y, f32x4 c, bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(u32x2 x, u32x2 y, f32x4 c, f16) {
  return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, x), __builtin_bit_cast(f16x4, y), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(u32x2 x, u32x2 y, f32x4 c, bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, x), __builtin_bit_cast(s16x4, y), c, 0, 0, 0);
}

// CPL: output channels per lane (16 CPL cover the head size); P16: 16-position blocks of a tile.
template <class E, int CPL, int P16, int W>
__global__ __launch_bounds__(W* kWave) void attention_paged_matrix_kernel(const AttendPaged a) {
  constexpr int GQ = kMatrixHeads, NP = Mx<E>::PIECES;
  constexpr int PER = kPer16<E>;             // elements per 16 bytes
  constexpr int ROW = 16 * CPL;              // channels, padded
  constexpr int KS = ROW / (4 * PER);        // 16-byte loads of a key row's lane
  constexpr int TILE = 16 * P16;
  constexpr bool HALF = sizeof(E) == 2;
  constexpr int VP = CPL < PER ? CPL : PER;  // channels per load of a value row
  constexpr int VS = CPL / VP;
  constexpr int VW = VP * (int)sizeof(E) / 4;
  // fp16 weights are scaled up so that the small ones keep all bits of both pieces
  constexpr float LIFT = std::is_same<E, f16>::value ? 14.f : 0.f;
  static_assert(TILE <= 64, "a tile's rows are looked up by one lane each");
  __shared__ Meeting<W, GQ, ROW> meet;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // what follows from it stays in scalar registers
  const int col = lane & 15, quad = lane >> 4;
  const int HS = a.pg.head_size;
  Range w;
  if (!take_range<W>(a, GQ, tid, w)) return;
  // queries of head col, channels 4 PER j + PER quad + e
  f32x4 raw[KS][PER / 4];
  {
    const float* src = a.inp + (size_t)w.b * a.stride + (size_t)(w.head0 + (col < w.heads ? col : 0)) * HS;
#pragma unroll
    for (int j = 0; j < KS; j++)
#pragma unroll
      for (int e = 0; e < PER; e += 4)
        raw[j][e / 4] = *reinterpret_cast<const f32x4_any*>(src + min(4 * PER * j + PER * quad + e, HS - 4));
  }
  bool ok = true;
  const int p1 = w.p1;
  int t = w.p0 + wave * TILE;
  // the rows of the tile at `from`, one per lane (behind the range: of its last position)
  auto look_up = [&](int from) { return a.pg.row(w.b, w.kvh, min(from + (lane & (TILE - 1)), p1 - 1), ok); };
  unsigned rows = 0, rows_next = 0;
  if (t < p1) rows = look_up(t);
  if (t + W * TILE < p1) rows_next = look_up(t + W * TILE);

  u32x4 q[NP][KS];
  float unscale = 1.f;
  auto cut_queries = [&] {
    float x[KS][PER], most = 0.f;
#pragma unroll
    for (int j = 0; j < KS; j++)
#pragma unroll
      for (int e = 0; e < PER; e++) {
        x[j][e] = col < w.heads && 4 * PER * j + PER * quad + e < HS ? raw[j][e / 4][e % 4] * a.scale_log2e : 0.f;
        most = fmaxf(most, fabsf(x[j][e]));
      }
    if constexpr (std::is_same<E, f16>::value) {
      // a power of two per head takes its largest entry to 2^13 .. 2^14
      most = rows_max<16>(most);
      const int up = 14 - max(-100, min(100, __builtin_amdgcn_frexp_expf(most)));
      unscale = __builtin_amdgcn_ldexpf(1.f, -up);
#pragma unroll
      for (int j = 0; j < KS; j++)
#pragma unroll
        for (int e = 0; e < PER; e++) x[j][e] = __builtin_amdgcn_ldexpf(x[j][e], up);
    }
#pragma unroll
    for (int j = 0; j < KS; j++) {
      if constexpr (HALF) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          unsigned c[NP];
          cut(c, x[j][2 * e], x[j][2 * e + 1], E{});
#pragma unroll
          for (int i = 0; i < NP; i++) q[i][j][e] = c[i];
        }
      } else {
        const f32x4 f = {x[j][0], x[j][1], x[j][2], x[j][3]};
        q[0][j] = __builtin_bit_cast(u32x4, f);
      }
    }
  };

  f32x4 o[CPL];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < CPL; c++) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  float* const scores = a.scores && col < w.heads
                            ? a.scores + ((size_t)w.b * a.NH + w.head0 + col) * a.score_stride : nullptr;

  u32x4 k[P16][KS];
  unsigned v[P16][4][VS][VW];  // [positions 4 quad + r][piece of the row]
  auto load_keys = [&](unsigned of) {
#pragma unroll
    for (int p = 0; p < P16; p++) {
      const E* src = (const E*)a.pg.keys + (size_t)__shfl(of, 16 * p + col, 64) * HS;
#pragma unroll
      for (int j = 0; j < KS; j++) {
        if (j > KS / 2 && 4 * PER * j >= HS) break;  // nothing but what is behind the row's end
        // behind the row's end: its last piece, against queries that are 0 there
        const int d = min(4 * PER * j + PER * quad, HS - PER);
        k[p][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + d));
      }
    }
  };
  auto load_values = [&](unsigned of) {
#pragma unroll
    for (int p = 0; p < P16; p++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const E* src = (const E*)a.pg.values + (size_t)__shfl(of, 16 * p + 4 * quad + r, 64) * HS;
#pragma unroll
        for (int j = 0; j < VS; j++) {
          // behind the row's end: its last piece, for outputs that nobody takes
          const int d = min(16 * VP * j + VP * col, HS - VP);
          if constexpr (VW == 4) {
            const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + d));
#pragma unroll
            for (int e = 0; e < 4; e++) v[p][r][j][e] = x[e];
          } else {
            const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(src + d));
            v[p][r][j][0] = x[0];
            v[p][r][j][1] = x[1];
          }
        }
      }
  };

  // One tile; MORE: another follows, so that this one is whole.  The keys' registers are free once
  // the scores are known and the values' once they are added up: the next tile's loads go there at
  // once, so that half of a tile is always under way.
  // SPECIAL: every position that weighs anything weighs the same, in one piece, see below.
  auto step = [&](auto more, auto special) {
    constexpr bool MORE = decltype(more)::value, SPECIAL = decltype(special)::value;
    unsigned rows_after = 0;
    if constexpr (MORE) {
      if (t + 2 * W * TILE < p1) rows_after = look_up(t + 2 * W * TILE);
    }
    const bool full = MORE || t + TILE <= p1;

    f32x4 sc[P16];
    if constexpr (HALF) {
#pragma unroll
      for (int p = 0; p < P16; p++) sc[p] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = NP - 1; i >= 0; i--)  // the smallest pieces first
#pragma unroll
        for (int j = 0; j < KS; j++) {
          if (j > KS / 2 && 4 * PER * j >= HS) break;
#pragma unroll
          for (int p = 0; p < P16; p++) sc[p] = mfma32(k[p][j], q[i][j], sc[p], E{});
        }
    } else {
#pragma unroll
      for (int p = 0; p < P16; p++) {
        f32x4 s4[4] = {};  // four chains: a quarter of the roundings in each
#pragma unroll
        for (int j = 0; j < KS; j++) {
          if (j > KS / 2 && 4 * PER * j >= HS) break;
          const f32x4 kf = __builtin_bit_cast(f32x4, k[p][j]), qf = __builtin_bit_cast(f32x4, q[0][j]);
#pragma unroll
          for (int e = 0; e < 4; e++) s4[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[e], s4[e], 0, 0, 0);
        }
        sc[p] = (s4[0] + s4[1]) + (s4[2] + s4[3]);
      }
    }
    bool odd = false;
#pragma unroll
    for (int p = 0; p < P16; p++) {
      if constexpr (LIFT != 0.f) sc[p] *= unscale;
      odd |= __builtin_isunordered(sc[p][0], sc[p][1]) || __builtin_isunordered(sc[p][2], sc[p][3]);
    }
    if (__ballot(odd)) {
      // an infinity in a key has met a 0 (a piece, or behind the row's end): in one piece it would
      // not have, unless the score is a NaN indeed
      const float* qs = a.inp + (size_t)w.b * a.stride + (size_t)(w.head0 + (col < w.heads ? col : 0)) * HS;
#pragma unroll
      for (int p = 0; p < P16; p++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const E* ks = (const E*)a.pg.keys + (size_t)__shfl(rows, 16 * p + 4 * quad + r, 64) * HS;
          float x = 0.f;
          for (int d = 0; d < HS; d++) x = fmaf(qs[d] * a.scale_log2e, widen(ks[d]), x);
          sc[p][r] = x;
        }
    }
    if constexpr (MORE) load_keys(rows_next);
    if constexpr (SPECIAL) load_values(rows);
    if (!SPECIAL && scores) {
#pragma unroll
      for (int p = 0; p < P16; p++) {
        float* to = scores + t + 16 * p + 4 * quad;
        if (full)
          *reinterpret_cast<f32x4*>(to) = sc[p];
        else
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (t + 16 * p + 4 * quad + r < p1) to[r] = sc[p][r];
      }
    }
    if (!full) {
      // rows behind the range are copies of its last one: they weigh nothing, whatever they hold
#pragma unroll
      for (int p = 0; p < P16; p++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (t + 16 * p + 4 * quad + r >= p1) {
            sc[p][r] = -INFINITY;
#pragma unroll
            for (int j = 0; j < VS; j++)
#pragma unroll
              for (int e = 0; e < VW; e++) v[p][r][j][e] = 0u;
          }
    }

    if constexpr (SPECIAL) {
      // a weight of 2^-31 keeps sums of bf16 values finite
      constexpr float ONE = std::is_same<E, f16>::value ? 1.f : 0x1p-31f;
#pragma unroll
      for (int p = 0; p < P16; p++)
#pragma unroll
        for (int r = 0; r < 4; r++) sc[p][r] = sc[p][r] > -INFINITY ? ONE : 0.f;
    } else {
      // the maximum over all positions of the tile: a head's outputs are added up over them
      float top = m;
#pragma unroll
      for (int p = 0; p < P16; p++) top = fmaxf(top, fmaxf(fmaxf(sc[p][0], sc[p][1]), fmaxf(sc[p][2], sc[p][3])));
      top = rows_max<16>(top);
      if (__ballot(top > m)) {
        const float fade = __builtin_amdgcn_exp2f(m - above(top));
        l *= fade;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float f = __shfl(fade, 4 * quad + r, 64);
#pragma unroll
          for (int c = 0; c < CPL; c++) o[c][r] *= f;
        }
        m = top;
      }
      const float base = above(m) - LIFT;
#pragma unroll
      for (int p = 0; p < P16; p++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          sc[p][r] = __builtin_amdgcn_exp2f(sc[p][r] - base);
          l += sc[p][r];
        }
    }

    if constexpr (!HALF) {
#pragma unroll
      for (int p = 0; p < P16; p++)
#pragma unroll
        for (int j = 0; j < VS; j++)
#pragma unroll
          for (int e = 0; e < VP; e++)
#pragma unroll
            for (int r = 0; r < 4; r++)
              o[j * VP + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(sc[p][r], float_of(v[p][r][j][e]), o[j * VP + e], 0, 0, 0);
    } else {
      // two blocks of positions make one product of 32, where there are two
      constexpr int PP = P16 % 2 == 0 ? 2 : 1;
#pragma unroll
      for (int p = 0; p < P16; p += PP) {
        unsigned wt[NP][2 * PP];
#pragma unroll
        for (int h = 0; h < PP; h++) {
          unsigned c01[NP], c23[NP];
          cut(c01, sc[p + h][0], sc[p + h][1], E{});
          cut(c23, sc[p + h][2], sc[p + h][3], E{});
#pragma unroll
          for (int i = 0; i < NP; i++) {
            wt[i][2 * h] = c01[i];
            wt[i][2 * h + 1] = c23[i];
          }
        }
#pragma unroll
        for (int j = 0; j < VS; j++)
#pragma unroll
          for (int e = 0; e < VW; e++) {
            unsigned even[2 * PP], odds[2 * PP];
#pragma unroll
            for (int h = 0; h < PP; h++) {
              const auto& x = v[p + h];
              even[2 * h] = lower_halves(x[0][j][e], x[1][j][e]);
              even[2 * h + 1] = lower_halves(x[2][j][e], x[3][j][e]);
              odds[2 * h] = upper_halves(x[0][j][e], x[1][j][e]);
              odds[2 * h + 1] = upper_halves(x[2][j][e], x[3][j][e]);
            }
            f32x4 &oe = o[j * VP + 2 * e], &oo = o[j * VP + 2 * e + 1];
#pragma unroll
            for (int i = SPECIAL ? 0 : NP - 1; i >= 0; i--) {
              if constexpr (PP == 2) {
                const u32x4 l4 = {wt[i][0], wt[i][1], wt[i][2], wt[i][3]};
                oe = mfma32(l4, u32x4{even[0], even[1], even[2], even[3]}, oe, E{});
                oo = mfma32(l4, u32x4{odds[0], odds[1], odds[2], odds[3]}, oo, E{});
              } else {
                const u32x2 l2 = {wt[i][0], wt[i][1]};
                oe = mfma16(l2, u32x2{even[0], even[1]}, oe, E{});
                oo = mfma16(l2, u32x2{odds[0], odds[1]}, oo, E{});
              }
            }
          }
      }
    }
    if constexpr (MORE) {
      load_values(rows_next);
      rows = rows_next;
      rows_next = rows_after;
      t += W * TILE;
    }
  };
  if (t < p1) {
    load_keys(rows);
    load_values(rows);
  }
  if (w.adds) ok &= add_row<E>(a, w, lane, wave, meet);
  cut_queries();
  if (t < p1) {
    while (t + W * TILE < p1) step(std::true_type{}, std::false_type{});
    step(std::false_type{}, std::false_type{});
  }

  const bool all_ok = __ballot(!ok) == 0;
  l = quads_sum(l, l, l, l);
  if (quad == 0) {
    meet.m[wave][col] = m == -INFINITY ? m : m - LIFT;
    meet.l[wave][col] = all_ok ? l : __builtin_nanf("");  // a page that does not exist: NaN, not a stray read
  }
  // row 4 quad + r of o is head 4 quad + r
  auto each_output = [&](auto f) {
#pragma unroll
    for (int r = 0; r < 4; r++)
      if (4 * quad + r < w.heads) {
#pragma unroll
        for (int j = 0; j < VS; j++)
#pragma unroll
          for (int e = 0; e < VP; e++) f(meet.o[wave][4 * quad + r][16 * VP * j + VP * col + e], o[j * VP + e][r]);
      }
  };
  each_output([](float& to, float x) { to = x; });
  if constexpr (HALF) {
    // A NaN can come from an infinite value that met a weight's lower pieces, which are 0 or
    // negative.  Which infinity belongs there, if not a NaN, does not depend on how large the
    // weights are, so that the range is gone through once more, from its end, with weights of one
    // piece, and outputs that are NaN take an infinity that comes of it.  (8 sequences of 4000
    // positions, 8 of 32 heads of 128, bf16, an infinity in each: 28.0 -> 32.8 us; without any 28.0
    // as before.)
    bool odd = false;
    each_output([&](float&, float x) { odd |= x != x; });
    if (__ballot(odd)) {
#pragma unroll
      for (int c = 0; c < CPL; c++) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (; t >= w.p0; t -= W * TILE) {
        rows = look_up(t);
        load_keys(rows);
        step(std::false_type{}, std::true_type{});
      }
      each_output([](float& to, float x) { to = to != to && fabsf(x) == INFINITY ? x : to; });
    }
  }
  finish(a, w, tid, meet);
  if (a.weigh_here) weigh(a, w, tid, meet);
}

constexpr int kWeighPositions = 256;  // positions per workgroup

// The same where the work is split: a thread per position.  TURNS: as many workgroups as a launch
// holds, which take the rest of the `blocks` in further turns (a loop that costs narrower tables
// 0.3 of 21.4 us: 4 sequences of 5000-9001 positions, 4 of 32 heads of 96, bf16).
template <bool TURNS>
__global__ __launch_bounds__(kWeighPositions) void attention_paged_weights_kernel(const AttendPaged a, unsigned blocks) {
  const unsigned per = (unsigned)(a.pg.capacity + kWeighPositions - 1) / kWeighPositions;
  unsigned turn = blockIdx.x;
  do {
    const unsigned pair = turn / per, kvh = pair % a.pg.kv_heads, b = pair / a.pg.kv_heads;
    const int i = (int)(turn - pair * per) * kWeighPositions + threadIdx.x;
    const int n = a.lengths[b];
    if (n >= 0 && n <= a.pg.capacity - a.append && i < n + a.append) {
      const size_t at = ((size_t)b * a.pg.kv_heads + kvh) * a.pg.capacity + i;
      const size_t bh = (size_t)b * a.NH + kvh * a.G;
      const float x = i < n ? a.weights_in[at] : 0.f;
      float p = 0.f;
#pragma unroll 8
      for (int g = 0; g < a.G; g++)
        p += __builtin_amdgcn_exp2f(a.scores[(bh + g) * a.score_stride + i] - a.joined[(bh + g) * 2]) / a.joined[(bh + g) * 2 + 1];
      a.weights_out[at] = x + p;
    }
    turn += gridDim.x;
  } while (TURNS && turn < blocks);
}

// ---- kv_evict_paged -------------------------------------------------------------------------
// The order of weights as unsigned integers: -0 equals 0, and a NaN is the largest of all.  No
// weight has rank 0.
__device__ __forceinline__ unsigned rank_of(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.0f);
  return w != w ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// base + the set bits of m in front of this lane's
__device__ __forceinline__ int lanes_before(unsigned long long m, int base) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, base));
}

// The sum over WAVES consecutive lanes of a row of 16, in each of them.
template <int WAVES>
__device__ __forceinline__ int waves_sum(int v) {
  static_assert(WAVES == 4 || WAVES == 16, "quads or rows");
  v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);
  if constexpr (WAVES == 16) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true);
  }
  return v;
}

constexpr int kFew = 4096;  // ranks that are worth a list of their own

struct Evict {
  Pages dst, src;
  int* kept;
  float* weights_out;
  int* lengths_out;
  const float* weights_in;
  const int* lengths;
  int B, budget, recent;
  int row_bytes, rows, groups;  // rows that a wave copies, waves (or, with the choice, workgroups) per (sequence, kv head)
};

// Which of the `older` first positions stay: the `want` (0 < want < older) of largest weight w,
// for each of which put(place, position) is called.  A workgroup of WAVES waves, all of it.
// The first 10 or 12 bits of the smallest rank that stays come from counts in LDS of how many
// ranks begin with each value (before, two bits at a time from the start: 4 x 32000 weights, 8
// heads, to 3200: 39.8 -> 33.2 us; 13 x 3-31, 12 heads: 8.9 -> 7.8), the others two at a time from
// how many ranks go each of the four ways: sums of integers, the same on every run.  Once few
// ranks are left that could be it, they are listed in LDS and the rest is not looked at again
// until the end; the search ends early where a candidate is reached by exactly as many ranks as
// are wanted.  A wave owns consecutive positions, so that the places in the output follow from
// counts alone.  R ranks per thread are kept in registers; R = 0: any length, read again for
// every count (200000 weights, 4 heads, to 20000: 147 us).
template <int WAVES, int R, class Put>
__device__ __forceinline__ void pick(const float* __restrict__ w, int older, int want, int tid, Put put) {
  constexpr int THREADS = WAVES * kWave;
  constexpr bool LISTS = R == 0 || R * THREADS > 2 * kFew;
  constexpr int FEW = LISTS ? kFew / THREADS : 1;
  constexpr int BITS = WAVES == 16 ? 12 : 10, BINS = 1 << BITS;
  static_assert(BINS == 4 * THREADS, "four bins per thread");
  __shared__ unsigned list[LISTS ? kFew : 1];
  constexpr int COPIES = 4;
  __shared__ __align__(16) int bins[COPIES * BINS];
  __shared__ int counts[2][WAVES][3], waves[2][WAVES], chosen[3], listed;
  const int lane = tid & 63, wave = tid >> 6;
  if (tid == 0) listed = 0;
#pragma unroll
  for (int k = 0; k < COPIES; k++) *reinterpret_cast<int4*>(bins + 4 * (tid + k * THREADS)) = make_int4(0, 0, 0, 0);
  constexpr int AHEAD = 8;  // loads under way, where nothing is kept
  const int span = R ? 64 * R : (older + WAVES * AHEAD * 64 - 1) / (WAVES * AHEAD * 64) * AHEAD * 64;
  const int first = wave * span;
  unsigned rank[R ? R : 1];
  if constexpr (R > 0) {
    float x[R];
#pragma unroll
    for (int r = 0; r < R; r++) x[r] = w[min(first + r * 64 + lane, older - 1)];
#pragma unroll
    for (int r = 0; r < R; r++) rank[r] = first + r * 64 + lane < older ? rank_of(x[r]) : 0u;
  }
  // calls f(group, its ranks): 0, which no weight has, behind the last position
  auto each = [&](auto f) {
    if constexpr (R > 0) {
#pragma unroll
      for (int r = 0; r < R; r++) f(r, rank[r]);
    } else {
      for (int r0 = 0; r0 < span / 64; r0 += AHEAD) {
        float x[AHEAD];
#pragma unroll
        for (int r = 0; r < AHEAD; r++) x[r] = w[min(first + (r0 + r) * 64 + lane, older - 1)];
#pragma unroll
        for (int r = 0; r < AHEAD; r++) f(r0 + r, first + (r0 + r) * 64 + lane < older ? rank_of(x[r]) : 0u);
      }
    }
  };
  unsigned few[FEW];
  bool from_list = false;
  __syncthreads();

  // How many ranks begin with each value of BITS bits, in COPIES counts, so that equal ones wait
  // less for each other (32000 equal weights: 68 us with one, 48 with four).  What is behind the
  // last position counts as 0, where no weight is.
  each([&](int, unsigned x) { atomicAdd(&bins[(x >> (32 - BITS)) * COPIES + (lane & (COPIES - 1))], 1); });
  __syncthreads();
  {
    int c[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      c[k] = 0;
#pragma unroll
      for (int i = 0; i < COPIES; i++) c[k] += bins[(4 * tid + k) * COPIES + i];
    }
    const int sum = c[0] + c[1] + c[2] + c[3], upto = wave_scan(sum);
    if (lane == 63) waves[0][wave] = upto;
    __syncthreads();
    int at_least = span * WAVES - (upto - sum);  // ranks from this thread's bins on
#pragma unroll
    for (int i = 0; i < WAVES; i++) at_least -= i < wave ? waves[0][i] : 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (at_least >= want && at_least - c[k] < want) {
        chosen[0] = 4 * tid + k;
        chosen[1] = at_least;
        chosen[2] = at_least - c[k];
      }
      at_least -= c[k];
    }
  }
  __syncthreads();
  unsigned low = (unsigned)chosen[0] << (32 - BITS);  // at least `want` ranks reach it ...
  int reach = chosen[1], over = chosen[2];  // ... this many; and this many are too large to be the one sought
  auto to_list = [&](int shift) {
    if constexpr (LISTS) {
      if (from_list || reach - over > kFew || reach == want) return;
      int mine = 0;  // low is above 0 by now, so that nothing behind the last position counts
      each([&](int, unsigned x) { mine += (x - low) >> shift == 0u; });
      const int upto = wave_scan(mine);
      int at = 0;
      if (lane == 63) at = atomicAdd(&listed, upto);
      at = __builtin_amdgcn_readlane(at, 63) + upto - mine;
      each([&](int, unsigned x) {
        if ((x - low) >> shift == 0u && at < kFew) list[at++] = x;
      });
      __syncthreads();
#pragma unroll
      for (int k = 0; k < FEW; k++) few[k] = k * THREADS + tid < min(listed, kFew) ? list[k * THREADS + tid] : 0u;
      from_list = true;
    }
  };
  to_list(32 - BITS);
  for (int step = BITS / 2; step < 16 && reach != want; step++) {
    // the four ways the next two bits can go, for ranks that agree with low in front of them
    const int shift = 30 - 2 * step;
    int n1, n2, n3;
    if (R > 0 || from_list) {
      // four counts of 7 bits, and what is elsewhere runs out at the top
      unsigned c = 0u;
      auto count = [&](unsigned x) { c += 1u << (7u * min((x - low) >> shift, 4u)); };
      if (LISTS && from_list) {
#pragma unroll
        for (int k = 0; k < FEW; k++) count(few[k]);
      } else {
        each([&](int, unsigned x) { count(x); });
      }
      n1 = wave_sum_int((c >> 7) & 127u);
      n2 = wave_sum_int(((c >> 14) & 127u) | ((c >> 21) & 127u) << 16);
      n3 = n2 >> 16;
      n2 &= 0xffff;
    } else {
      n1 = n2 = n3 = 0;
      each([&](int, unsigned x) {
        const unsigned d = (x - low) >> shift;
        n1 += d == 1u;
        n2 += d == 2u;
        n3 += d == 3u;
      });
      n1 = wave_sum_int(n1);
      n2 = wave_sum_int(n2);
      n3 = wave_sum_int(n3);
    }
    if (lane == 0) {
      counts[step & 1][wave][0] = n1;
      counts[step & 1][wave][1] = n2;
      counts[step & 1][wave][2] = n3;
    }
    __syncthreads();  // the counts of the step before last have been read by then
    n1 = waves_sum<WAVES>(counts[step & 1][lane & (WAVES - 1)][0]);
    n2 = waves_sum<WAVES>(counts[step & 1][lane & (WAVES - 1)][1]);
    n3 = waves_sum<WAVES>(counts[step & 1][lane & (WAVES - 1)][2]);
    const int c3 = over + n3, c2 = c3 + n2, c1 = c2 + n1;
    if (c3 >= want) {
      low |= 3u << shift;
      reach = c3;
    } else if (c2 >= want) {
      low |= 2u << shift;
      reach = c2;
      over = c3;
    } else if (c1 >= want) {
      low |= 1u << shift;
      reach = c1;
      over = c2;
    } else {
      over = c1;
    }
    to_list(shift);
  }

  // All ranks above low stay, and of its equals as many as there is room for: all of them, where
  // exactly as many as are wanted reach low.
  const bool exact = reach == want;
  int gt = 0, eq = 0;
  each([&](int, unsigned x) { gt += x >= low; });
  if (!exact) {
    each([&](int, unsigned x) { eq += x == low; });
    eq = wave_sum_int(eq);
  }
  gt = wave_sum_int(gt) - eq;
  if (lane == 0) {
    waves[0][wave] = gt;
    waves[1][wave] = eq;
  }
  __syncthreads();
  int above_all = 0, gt_before = 0, eq_before = 0;
#pragma unroll
  for (int i = 0; i < WAVES; i++) {
    above_all += waves[0][i];
    gt_before += i < wave ? waves[0][i] : 0;
    eq_before += i < wave ? waves[1][i] : 0;
  }
  if (exact) {
    each([&](int r, unsigned x) {
      const unsigned long long g = __ballot(x >= low);
      const int at = lanes_before(g, gt_before);
      if (x >= low && at < want) put(at, first + r * 64 + lane);
      gt_before += __popcll(g);
    });
    return;
  }
  const int room = want - above_all;  // the lowest positions have it
  each([&](int r, unsigned x) {
    const unsigned long long g = __ballot(x > low), e = __ballot(x == low);
    const int eq_at = lanes_before(e, eq_before), at = lanes_before(g, gt_before) + min(eq_at, room);
    if ((x > low || (x == low && eq_at < room)) && at < want) put(at, first + r * 64 + lane);
    gt_before += __popcll(g);
    eq_before += __popcll(e);
  });
}

// Copies the keys and values of `rows` rows of one (sequence, kv head), kCopyLoads times as many
// as one load of the wave holds, all loads ahead of the stores, and their weights.  Lane r < rows
// says that row j comes from position i.  UNIT: bytes per lane and load, 16 or the size of an
// element; STREAM: stores past the caches (rows of whole cache lines).
constexpr int kCopyLoads = 4;
static int copy_rows(int row_bytes, int unit) {  // rows per wave
  const int units = row_bytes / unit, per = units < 64 ? 64 / units : 1;
  return per * kCopyLoads < 64 ? per * kCopyLoads : 64;
}
template <int UNIT, bool STREAM>
__device__ __forceinline__ void copy_kept(const Evict& e, size_t bh, int b, int h, int lane, bool ok, int i, int j) {
  unsigned from = 0, to = 0;
  if (ok) {
    const float w = e.weights_in[bh * e.src.capacity + i];
    from = e.src.row(b, h, i, ok);
    to = e.dst.row(b, h, j, ok);
    e.weights_out[bh * e.dst.capacity + j] = ok ? w : __builtin_nanf("");
  }
  const unsigned long long live = __ballot(ok);
  const int units = e.row_bytes / UNIT, per = units < 64 ? 64 / units : 1;  // units per row, rows per load
  const int mine = lane / units;
  typedef typename std::conditional<UNIT == 16, u32x4, typename std::conditional<UNIT == 4, unsigned, unsigned short>::type>::type Word;
  const Word *ks = (const Word*)e.src.keys, *vs = (const Word*)e.src.values;
  Word *kd = (Word*)e.dst.keys, *vd = (Word*)e.dst.values;
  const int c0 = lane - mine * units;  // a row of more than 64 units takes more than one round, all lanes in each
  for (int round = 0; round < units; round += 64) {
    const int c = min(c0 + round, units - 1);
    Word k[kCopyLoads], v[kCopyLoads];
#pragma unroll
    for (int u = 0; u < kCopyLoads; u++) {
      const size_t x = (size_t)__shfl(from, (u * per + mine) & 63, 64) * units + c;  // row 0 where there is none
      k[u] = __builtin_nontemporal_load(ks + x);
      v[u] = __builtin_nontemporal_load(vs + x);
    }
#pragma unroll
    for (int u = 0; u < kCopyLoads; u++) {
      const int r = u * per + mine;
      const size_t x = (size_t)__shfl(to, r & 63, 64) * units + c;
      if (mine < per && r < e.rows && c0 + round < units && ((live >> (r & 63)) & 1ull)) {
        if constexpr (STREAM) {
          __builtin_nontemporal_store(k[u], kd + x);
          __builtin_nontemporal_store(v[u], vd + x);
        } else {
          kd[x] = k[u];
          vd[x] = v[u];
        }
      }
    }
  }
}

// One workgroup per (sequence, kv head) chooses the positions that stay: the `recent` last ones
// and, of the others, the budget - recent of largest weight.
// COPY (up to 4096 weights, where a second launch would cost as much as the choice): several
// workgroups per (sequence, kv head), each of which makes the whole choice and copies its share of
// the rows.  8 sequences of 900-1024 positions, 12 heads, fp32, to 512: 14.5 us (two launches: 17.9).
// Alone, 4 of 32768, 8 heads: 20 us on 32 compute units: loading 3.4, first counts 4.5, the list 3,
// the other bits 3, what stays 4 (the 100 MHz clock's stamps).
template <int WAVES, int R, bool COPY, int UNIT, bool STREAM>
__global__ __launch_bounds__(WAVES* kWave) void kv_evict_pick_kernel(const Evict e) {
  constexpr int THREADS = WAVES * kWave;
  __shared__ int here[COPY ? WAVES * 64 : 1];  // this workgroup's share of the positions
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int KVH = e.src.kv_heads;
  const size_t bh = COPY ? blockIdx.x / (unsigned)e.groups : blockIdx.x;
  const int b = (int)(bh / KVH), h = (int)(bh % KVH);
  const int share = COPY ? WAVES * e.rows : e.budget;
  const int j0 = COPY ? (int)(blockIdx.x % (unsigned)e.groups) * share : 0, j1 = min(j0 + share, e.budget);
  const int n = e.lengths[b];
  if (n < 0) return;
  const bool too_long = n > e.src.capacity;
  const int stay = too_long ? 0 : min(n, e.budget);
  if (h == 0 && j0 == 0 && tid == 0) e.lengths_out[b] = too_long ? -1 : stay;
  int* out = e.kept + bh * e.budget;
  for (int j = max(stay, j0) + tid; j < j1; j += THREADS) out[j] = -1;
  if (j0 >= stay) return;
  auto put = [&](int j, int i) {
    if constexpr (COPY) {
      if (j < j0 || j >= j1) return;
      here[j - j0] = i;
    }
    out[j] = i;
  };
  if (stay == n) {  // nothing has to go
    for (int j = j0 + tid; j < min(j1, stay); j += THREADS) put(j, j);
  } else {
    const int older = n - e.recent, want = e.budget - e.recent;  // want < older
    for (int j = max(want, j0) + tid; j < j1; j += THREADS) put(j, older + j - want);
    if (want > j0) pick<WAVES, R>(e.weights_in + bh * e.src.capacity, older, want, tid, put);
  }
  if constexpr (COPY) {
    __syncthreads();
    const int r = wave * e.rows + lane, j = j0 + r;
    const bool ok = lane < e.rows && j < min(j1, stay);
    copy_kept<UNIT, STREAM>(e, bh, b, h, lane, ok, ok ? min(max(here[r], 0), n - 1) : 0, j);
  }
}

// The copy alone: 4 of 32768 positions, 8 heads of 128, bf16, to 8192: 57 us = 4.7 TB/s.
template <int UNIT, bool STREAM>
__global__ __launch_bounds__(256) void kv_evict_copy_kernel(const Evict e) {
  const int lane = threadIdx.x & 63;
  const size_t id = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const size_t bh = id / e.groups;
  const int b = (int)(bh / e.src.kv_heads), h = (int)(bh % e.src.kv_heads);
  if (b >= e.B) return;
  const int j0 = (int)(id % e.groups) * e.rows, j = j0 + lane;
  const int n = e.lengths[b];
  if (n < 0 || n > e.src.capacity || j0 >= min(n, e.budget)) return;
  const bool ok = lane < e.rows && j < min(n, e.budget);
  copy_kept<UNIT, STREAM>(e, bh, b, h, lane, ok, ok ? min(max(e.kept[bh * e.budget + j], 0), n - 1) : 0, j);
}

// ---- launchers ------------------------------------------------------------------------------
// A launch holds fewer than 2^32 threads in all; what is beyond is left out without an error.
static bool too_many(long long blocks, int threads) { return blocks > 0xffffffffLL / threads; }

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
  const dim3 grid((unsigned)((N + 3LL) / 4)), block(256);
  if (vec)
    hipLaunchKernelGGL((kv_store_paged_kernel<E, 4>), grid, block, 0, stream(), pg, inp, stride, starts, lengths, N, B, NH);
  else
    hipLaunchKernelGGL((kv_store_paged_kernel<E, 1>), grid, block, 0, stream(), pg, inp, stride, starts, lengths, N, B, NH);
}

// Which kernel a problem takes, and how it is cut up.
struct AttendPlan {
  bool rows16, matrix, deep;
  int gq, chunks, slots, min_range, waves;
};

static AttendPlan plan_attend(const GPT2PagedCache* c, int B, int NH, bool weights) {
  AttendPlan p;
  const int G = NH / c->kv_heads;
  p.rows16 = rows_by_16(c);
  p.matrix = p.rows16 && G >= 3;
  p.gq = p.matrix ? kMatrixHeads : G >= 3 ? 4 : G;
  p.chunks = (G + p.gq - 1) / p.gq;
  const long long groups = (long long)B * c->kv_heads * p.chunks;
  const long long capacity = (long long)c->max_pages * c->page_size, row_bytes = 2LL * c->head_size * type_bytes(c->type);
  const long long each = capacity * row_bytes;  // of keys and values, per group
  // As many workgroups as compute units, or, where that is less than two per sequence, there is
  // much to do and whole sequences would not fill the units evenly, twice as many.  A range is
  // worth a workgroup from 64 KB on.  The capacity is all that is known of the lengths here: dealing
  // to twice as many gains where they are uneven (8 of 32 heads of 128, bf16, 24 sequences of
  // 100-6000: 94.7 -> 68.9 us) and costs where they are even (24 of 1535: 31.9 -> 44.6; 36 of 4071:
  // 138.0 -> 139.5); from 205 to 256 groups the loss is taken to matter more (28 of 1535: 33.5
  // whole, 45.6 dealt; but 28 of 1-8900: 141 whole, 106 dealt).
  p.min_range = (int)((65536 / row_bytes + 63) & ~63LL);
  if (p.min_range < 128) p.min_range = 128;
  const long long per = (long long)c->kv_heads * p.chunks, ranges = capacity / p.min_range;  // ranges of a sequence, at most
  long long slots = 256 / per;
  if (slots < 2LL * B) {
    slots = each >= 768 * 1024 && (groups < 205 || groups > 256) ? 512 / per : 0;
  } else {
    // Splitting costs 4 us (parts to memory, the counter, parts back) and, with weights, a second
    // launch.  A workgroup takes 18 ns for a KB of cache, 27 in the matrix kernel, and all of them
    // together at least 0.12 ns per KB.  (12 heads, fp32: whole or split, one sequence of 383
    // positions 6.4 or 8.0 us, of 895 10.9 or 8.5; 8 of 895 13.3 or 15.2, of 1791 23.2 or 20.5, with
    // weights 25.1 or 24.3.  4 sequences, 8 of 32 heads of 128, bf16: 383 10.1 or 11.1, with weights
    // 11.5 or 14.8; 639 14.5 or 11.7, with weights 15.8 or 15.2.)
    const double alone = p.matrix ? 27. : 18., parts = (double)(slots < B * ranges ? slots : B * ranges) / B;
    const double split = parts > 1. ? alone / parts : alone, together = 0.12 * (double)groups;
    if ((double)each / 1024. * (alone - (split > together ? split : together)) < (weights ? 5300. : 4000.)) slots = 0;
  }
  if (slots > B * ranges) slots = B * ranges;
  if (B > kMostSplit || groups * kCounterStride * 4 > GPT2HIP_PAGED_COUNTER_BYTES) slots = 0;
  p.slots = slots > B ? (int)slots : B;
  // Four waves instead of eight for many short caches (64 sequences of 12 heads, bf16, of 100
  // positions: 7.2 against 9.9 us; 64 of 16 heads of 128, of 2000, the other way: 164 against 161)
  // and where eight would take all of a unit's registers: the matrix kernel from 257 groups on
  // (8 of 32 heads, fp32, 55 sequences of 350: 18.0 against 22.9 us) and for head sizes above 128
  // -- or where four have one tile each and no more (30 sequences of 8 of 32 heads of 128, fp16, of
  // 60: 7.3 against 7.5 us).
  p.waves = 8;
  if (!p.rows16 || (groups > 512 && each < 768 * 1024)) p.waves = 4;
  if (p.matrix && (groups > 256 || (capacity <= 128 && type_bytes(c->type) == 2) || c->head_size > 128)) p.waves = 4;
  // one workgroup per compute unit with much to do: twice the loads under way (16 sequences of 12
  // heads, fp32, up to 1024 positions: 15.8 -> 15.0 us; short ranges would leave waves idle)
  p.deep = (long long)p.slots * c->kv_heads * p.chunks <= 256 && each * B / p.slots >= 256 * 1024;
  return p;
}

// What a call puts into the workspace behind the counters.
struct AttendSpace {
  size_t part, ml, joined, scores, total;  // offsets in floats
  AttendSpace(const AttendPlan& p, int B, int NH, int KVH, int part_stride, int score_stride, int slots, bool weights) {
    const size_t rows = (size_t)B * NH;
    const int G = NH / KVH;
    const size_t parts = slots > B ? (size_t)slots * KVH * p.chunks * (p.gq < G ? p.gq : G) : 0;
    part = 0;
    ml = part + parts * part_stride;
    joined = ml + parts * 2;
    scores = (joined + (weights ? rows * 2 : 0) + 3) & ~(size_t)3;
    total = scores + (weights ? rows * score_stride : 0);
  }
};

template <class E>
static void launch_attend(const AttendPaged& a, const AttendPlan& p, unsigned blocks) {
  const int HS = a.pg.head_size, lanes = (HS + kPer16<E> - 1) / kPer16<E>;
#define G2_KERNEL(W, ...) hipLaunchKernelGGL((__VA_ARGS__), dim3(blocks), dim3(W * kWave), 0, stream(), a)
#define G2_MATRIX(CPL, P16)                                            \
  if (p.waves == 8)                                                    \
    G2_KERNEL(8, attention_paged_matrix_kernel<E, CPL, P16, 8>);       \
  else                                                                 \
    G2_KERNEL(4, attention_paged_matrix_kernel<E, CPL, P16, 4>);
#define G2_ROWS(LPR)                                                   \
  if (p.waves == 8 && p.gq == 1 && p.deep)                             \
    G2_KERNEL(8, attention_paged_kernel<E, LPR, 1, 8, 8, false>);      \
  else if (p.waves == 8 && p.gq == 1)                                  \
    G2_KERNEL(8, attention_paged_kernel<E, LPR, 1, 4, 8, false>);      \
  else if (p.waves == 8)                                               \
    G2_KERNEL(8, attention_paged_kernel<E, LPR, 2, 4, 8, false>);      \
  else if (p.gq == 1)                                                  \
    G2_KERNEL(4, attention_paged_kernel<E, LPR, 1, 8, 4, false>);      \
  else                                                                 \
    G2_KERNEL(4, attention_paged_kernel<E, LPR, 2, 4, 4, false>);
  if (p.matrix && HS <= 64) {
    G2_MATRIX(4, (sizeof(E) == 4 ? 2 : 4))
  } else if (p.matrix && HS <= 128) {
    G2_MATRIX(8, (sizeof(E) == 4 ? 1 : 2))
  } else if (p.matrix) {
    G2_KERNEL(4, attention_paged_matrix_kernel<E, 16, 1, 4>);
  } else if (!p.rows16) {
    if (p.gq == 1)
      G2_KERNEL(4, attention_paged_kernel<E, 64, 1, 8, 4, true>);
    else if (p.gq == 2)
      G2_KERNEL(4, attention_paged_kernel<E, 64, 2, 8, 4, true>);
    else
      G2_KERNEL(4, attention_paged_kernel<E, 64, 4, 4, 4, true>);
  } else if (lanes <= 8) {
    G2_ROWS(8)
  } else if (lanes <= 16) {
    G2_ROWS(16)
  } else if (lanes <= 32) {
    G2_ROWS(32)
  } else if constexpr (sizeof(E) == 4) {
    G2_ROWS(64)
  }
#undef G2_ROWS
#undef G2_MATRIX
#undef G2_KERNEL
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
  if (too_many((N + 3LL) / 4, 256)) return fail(GPT2HIP_EINVAL, "kv_store_paged: grid too large (N=%d rows)", N);
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
  size_t most = 0;  // with weights, what a call without them needs too
  for (int w = 0; w <= (weights != 0); w++) {
    const AttendPlan plan = plan_attend(cache, B, NH, w);
    const AttendSpace space(plan, B, NH, pg.kv_heads, (pg.head_size + 3) & ~3, (pg.capacity + 63) & ~63, plan.slots, w);
    if (space.total > most) most = space.total;
  }
  return GPT2HIP_PAGED_COUNTER_BYTES + most * sizeof(float);
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
  AttendPlan plan = plan_attend(cache, B, NH, weights);
  a.out = out;
  a.inp = inp;
  a.lengths = lengths;
  a.weights_in = weights_in;
  a.weights_out = weights_out;
  a.B = B;
  a.NH = NH;
  a.G = NH / KVH;
  a.chunks = plan.chunks;
  a.stride = inp_stride;
  a.append = append ? 1 : 0;
  a.part_stride = (HS + 3) & ~3;
  a.score_stride = (a.pg.capacity + 63) & ~63;
  a.scale_log2e = (1.0f / sqrtf((float)HS)) * 1.4426950408889634f;
  a.part_heads = plan.gq < a.G ? plan.gq : a.G;
  // as many ranges as the workspace holds
  const size_t room = workspace && workspace_bytes > GPT2HIP_PAGED_COUNTER_BYTES
                          ? (workspace_bytes - GPT2HIP_PAGED_COUNTER_BYTES) / sizeof(float) : 0;
  auto space = [&](int slots) { return AttendSpace(plan, B, NH, KVH, a.part_stride, a.score_stride, slots, weights); };
  while (plan.slots > B && space(plan.slots).total > room) plan.slots--;
  const AttendSpace use = space(plan.slots);
  if (use.total > room)
    return fail(GPT2HIP_EINVAL, "attention_decode_paged: weights need a workspace of at least %zu bytes, got %zu",
                GPT2HIP_PAGED_COUNTER_BYTES + use.total * sizeof(float), workspace_bytes);
  a.slots = plan.slots;
  a.min_range = plan.min_range;
  a.counters = (unsigned*)workspace;
  float* at = workspace ? (float*)((char*)workspace + GPT2HIP_PAGED_COUNTER_BYTES) : nullptr;
  a.part_o = at;
  a.part_ml = at + use.ml;
  a.joined = weights ? at + use.joined : nullptr;
  a.scores = weights ? at + use.scores : nullptr;
  a.weigh_here = weights && a.slots == B && a.chunks == 1;
  const long long blocks = (long long)a.slots * KVH * a.chunks;
  const long long weighs = (long long)B * KVH * ((a.pg.capacity + kWeighPositions - 1) / kWeighPositions);
  if (too_many(blocks, plan.waves * kWave) || weighs > 0x7fffffffLL)
    return fail(GPT2HIP_EINVAL, "attention_decode_paged: grid too large (B=%d, NH=%d)", B, NH);
  if (cache->type == GPT2HIP_F32)
    launch_attend<float>(a, plan, (unsigned)blocks);
  else if (cache->type == GPT2HIP_F16)
    launch_attend<f16>(a, plan, (unsigned)blocks);
  else
    launch_attend<bf16>(a, plan, (unsigned)blocks);
  G2_LAUNCH_CHECK("attention_decode_paged");
  if (weights && !a.weigh_here) {
    if (too_many(weighs, kWeighPositions))
      hipLaunchKernelGGL(attention_paged_weights_kernel<true>, dim3(0xffffffffu / kWeighPositions), dim3(kWeighPositions), 0,
                         stream(), a, (unsigned)weighs);
    else
      hipLaunchKernelGGL(attention_paged_weights_kernel<false>, dim3((unsigned)weighs), dim3(kWeighPositions), 0, stream(), a,
                         (unsigned)weighs);
    G2_LAUNCH_CHECK("attention_decode_paged (weights)");
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
  Evict e{to, from, kept, weights_out, lengths_out, weights_in, lengths, B, budget, recent, 0, 0, 0};
  e.row_bytes = (int)(from.head_size * type_bytes(src->type));
  const int unit = rows_by_16(src) && rows_by_16(dst) ? 16 : (int)type_bytes(src->type);
  e.rows = copy_rows(e.row_bytes, unit);
  const int most = from.capacity - recent;  // weights that can take part
  // Choice and copy in one launch, the choice made again by every workgroup: up to 4096 weights
  // (48 pairs, bf16, 2000 -> 1000 positions: 15.4 -> 13.0 us; 768 pairs, 4000 -> 2000: 178 -> 168).
  // Where many workgroups would copy nearly everything it is two launches, a bound from before the
  // first bits were counted in LDS: now one launch is the faster there too (768 pairs, 4000 -> 3600:
  // 301 against 313 us; fp32, 250 -> 225: 43 against 68).
  const long long pairs = (long long)B * KVH, groups4 = (budget + 4 * e.rows - 1) / (4 * e.rows);
  const bool together = most <= 4096 && (4LL * budget <= 3LL * from.capacity || pairs * groups4 <= 1024);
  e.groups = together ? (int)groups4 : (budget + e.rows - 1) / e.rows;
  const long long copies = together ? pairs * e.groups : (pairs * e.groups + 3) / 4;
  if (too_many(copies, 256) || (!together && too_many(pairs, 16 * kWave)))
    return fail(GPT2HIP_EINVAL, "kv_evict_paged: grid too large (B=%d, budget=%d)", B, budget);
#define G2_UNITS(KERNEL)                                                                           \
  if (unit == 16 && e.row_bytes % 128 == 0) /* whole cache lines */                                \
    KERNEL(16, true);                                                                              \
  else if (unit == 16)                                                                             \
    KERNEL(16, false);                                                                             \
  else if (unit == 4)                                                                              \
    KERNEL(4, false);                                                                              \
  else                                                                                             \
    KERNEL(2, false);
#define G2_BOTH_1(UNIT, STREAM) \
  hipLaunchKernelGGL((kv_evict_pick_kernel<4, 1, true, UNIT, STREAM>), dim3((unsigned)copies), dim3(256), 0, stream(), e)
#define G2_BOTH_4(UNIT, STREAM) \
  hipLaunchKernelGGL((kv_evict_pick_kernel<4, 4, true, UNIT, STREAM>), dim3((unsigned)copies), dim3(256), 0, stream(), e)
#define G2_BOTH_16(UNIT, STREAM) \
  hipLaunchKernelGGL((kv_evict_pick_kernel<4, 16, true, UNIT, STREAM>), dim3((unsigned)copies), dim3(256), 0, stream(), e)
#define G2_PICK(WAVES, R)                                                                                               \
  hipLaunchKernelGGL((kv_evict_pick_kernel<WAVES, R, false, 16, false>), dim3((unsigned)pairs), dim3(WAVES * kWave), 0, \
                     stream(), e)
#define G2_COPY(UNIT, STREAM) \
  hipLaunchKernelGGL((kv_evict_copy_kernel<UNIT, STREAM>), dim3((unsigned)copies), dim3(256), 0, stream(), e)
  if (together) {
    if (most <= 256) {
      G2_UNITS(G2_BOTH_1)
    } else if (most <= 1024) {
      G2_UNITS(G2_BOTH_4)
    } else {
      G2_UNITS(G2_BOTH_16)
    }
    G2_LAUNCH_CHECK("kv_evict_paged");
    return GPT2HIP_OK;
  }
  if (most <= 4 * 1024)
    G2_PICK(16, 4);
  else if (most <= 16 * 1024)
    G2_PICK(16, 16);
  else if (most <= 32 * 1024)
    G2_PICK(16, 32);
  else
    G2_PICK(16, 0);
  G2_LAUNCH_CHECK("kv_evict_paged (choice)");
  G2_UNITS(G2_COPY)
#undef G2_COPY
#undef G2_PICK
#undef G2_BOTH_16
#undef G2_BOTH_4
#undef G2_BOTH_1
#undef G2_UNITS
  G2_LAUNCH_CHECK("kv_evict_paged (copy)");
  return GPT2HIP_OK;
}

}  // extern "C"
