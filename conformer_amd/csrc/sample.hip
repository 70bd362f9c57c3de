// Drawing a token per row of logits (gfx950).
//
// With x the logits of a row as fp32 and t its temperature:  w_i = exp((x_i - max x) / t).  The tokens are ordered by
// falling x, equal ones by rising index, and three filters keep a head of that order:
//   top-k : the first k;                                             (k <= 0: all)
//   top-p : token i while the mass of those before it is below p times the mass that top-k left;    (p >= 1: all)
//   min-p : tokens with w_i >= min_p                                 (w of the largest is 1)
// The first token is always kept.  Over the kept ones in index order, with C_i the running sum of w and C the whole sum,
// the token drawn for a given u in [0, 1) is the first with C_i > u C.  t <= 0 takes the first maximum.
//
// A token is a comparison of a sum with a border, so sums must not depend on the order of their terms: weights are
// formed in fp64 and rounded to integers in units of 2^-b, b = min(51, 63 - ceil(log2 vocab)), so that no sum passes
// 2^63, and integers add up exactly in any order, LDS atomics included.  A weight below half a unit (2^-52 of the largest one up to 4096
// logits, 2^-46 at the most there can be) counts as 0 and can be drawn only at u = 0, which takes the first kept token whose
// weight is a number at all (as a double: (max - x) / t < 745.13).  A filter that is NaN is off; a temperature that is takes the maximum.
//
// One workgroup per row; a wave takes a contiguous piece of it.  The head's last token is found by counting, not
// sorting: a histogram (counts or masses) over equal steps of (max - x) / t gives the step it lies in, histograms over
// the bit patterns inside that step give its value, and a count over equal values gives the token.  Elements that the
// first histogram leaves in question go to a list in LDS (in index order, a segment per wave): everything above the k-th when
// top-k is on, so that the rest of the work runs on the list, or the one step that top-p ends in.  A list that does not
// fit is not made, and the same code runs over the row again.
//
// A long row of bf16 logits has few different values (4736 per sign between 2^-30 and 2^7, and 0): there one pass over the
// row counts every value, the borders and the kept mass follow from the counts times the values' weights, and one more pass
// adds up the weights, read from a table, in index order.  A value outside that range, if it can matter, sends
// the row to the general form.
#include <float.h>
#include <math.h>

#include "common.h"
#include "kernels.h"

namespace fcenc {

namespace {

constexpr int MAX_WAVES = 16;
constexpr int BINS_PER_WAVE = 128;                // two bins per thread
constexpr int SEG = 512;                          // list entries per wave
constexpr float RANGE = 32.f;                     // the first histogram reaches down to exp(-32), about where weights end
constexpr int MAX_VOCAB = 1 << 18;
constexpr int TABLE = 256;
constexpr double MAGIC = 4503599627370496.0;      // 2^52: adding it leaves a rounded integer in the low 52 bits
using u64 = unsigned long long;

// 2^(j / 256)
struct ExpTable {
  double v[TABLE];
  constexpr ExpTable() : v() {
    for (int j = 0; j < TABLE; ++j) {
      const double x = j * (0.693147180559945309417 / TABLE);
      double term = 1.0, sum = 1.0;
      for (int i = 1; i < 24; ++i) {
        term *= x / i;
        sum += term;
      }
      v[j] = sum;
    }
  }
};
__device__ constexpr ExpTable exp_table{};

struct SampleLds {
  u64* mass;                 // [bins]
  unsigned* count;           // [bins], also read in fours: at a multiple of 16 bytes
  double* table;             // [TABLE]
  float* seg_x;              // [waves][SEG]
  int* seg_i;                // [waves][SEG]
  u64* part_m;               // [waves]
  u64* found_m;              // a border found in the bins: mass before it,
  unsigned* found;           //   bin, count before it; [2]: a token index
  unsigned* part_c;          // [waves]
  unsigned* seg_n;           // [waves] list entries
  unsigned* lo;              // range of keys: lo, hi
};
__host__ __device__ constexpr int lds_bytes(int waves) {
  return waves * BINS_PER_WAVE * 12 + waves * (8 + 4 + 4) + TABLE * 8 + waves * SEG * 8 + 8 + 8 + 16;
}
__host__ __device__ constexpr int count_at(int waves) { return waves * BINS_PER_WAVE * 8; }
static_assert(count_at(1) % 16 == 0 && count_at(2) % 16 == 0 && count_at(4) % 16 == 0 && count_at(8) % 16 == 0 && count_at(16) % 16 == 0,
              "by_few loads four counts at a time");

__device__ __forceinline__ SampleLds carve(char* p, int waves) {
  SampleLds l;
  char* at = p + count_at(waves);
  auto take = [&](int bytes) { char* q = at; at += bytes; return q; };
  l.mass = reinterpret_cast<u64*>(p);
  l.count = reinterpret_cast<unsigned*>(take(waves * BINS_PER_WAVE * 4));
  l.table = reinterpret_cast<double*>(take(TABLE * 8));
  l.seg_x = reinterpret_cast<float*>(take(waves * SEG * 4));
  l.seg_i = reinterpret_cast<int*>(take(waves * SEG * 4));
  l.part_m = reinterpret_cast<u64*>(take(waves * 8));
  l.found_m = reinterpret_cast<u64*>(take(8));
  l.found = reinterpret_cast<unsigned*>(take(16));
  l.part_c = reinterpret_cast<unsigned*>(take(waves * 4));
  l.seg_n = reinterpret_cast<unsigned*>(take(waves * 4));
  l.lo = reinterpret_cast<unsigned*>(take(8));
  return l;
}

// smaller values have larger keys; -0 counts as 0
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x == 0.f ? 0.f : x);
  return u & 0x80000000u ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key : ~key & 0x7fffffffu);
}
// NaN counts as -inf, +inf as the largest finite number
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }

struct Raw8F { f32x4 lo, hi; };
__device__ __forceinline__ float raw_at(const Raw8F& r, int i) { return i < 4 ? r.lo[i] : r.hi[i - 4]; }
__device__ __forceinline__ float raw_at(const u32x4& r, int i) {
  return __builtin_bit_cast(float, i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
}
// eight logits, at any alignment of the type
__device__ __forceinline__ Raw8F load_whole(const float* p) {
  struct __attribute__((packed, aligned(4))) V { f32x4 a, b; };
  const V v = *reinterpret_cast<const V*>(p);
  return Raw8F{v.a, v.b};
}
__device__ __forceinline__ u32x4 load_whole(const bf16* p) {
  struct __attribute__((packed, aligned(2))) V { u32x4 a; };
  return reinterpret_cast<const V*>(p)->a;
}
// the same from element e of the row on; -inf behind the row's end
__device__ __forceinline__ Raw8F load_raw(const float* row, int e, int n) {
  Raw8F r;
  if (e + 8 <= n) {
    r = load_whole(row + e);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = e + i < n ? row[e + i] : -INFINITY;
      if (i < 4) r.lo[i] = x; else r.hi[i - 4] = x;
    }
  }
  return r;
}
__device__ __forceinline__ u32x4 load_raw(const bf16* row, int e, int n) {
  if (e + 8 <= n) return load_whole(row + e);
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = e + 2 * i < n ? p[e + 2 * i] : 0xff80u, b = e + 2 * i + 1 < n ? p[e + 2 * i + 1] : 0xff80u;
    r[i] = a | (b << 16);
  }
  return r;
}

struct RowParams {
  float top;                 // the largest logit
  float bins;                // steps of the first histogram per unit of logit
  int nbins;
  double c;                  // 256 / (t ln 2)
};

// exp((x - top) / t) in weight units, not yet rounded: with s = 256 log2(...) = 256 n + j + f, |f| <= 1/2, it is 2^n table[j]
// exp(f ln 2 / 256); the Taylor sum to the third power leaves (0.00136)^4 / 24 = 1.4e-13.
__device__ __forceinline__ double weight(float x, const RowParams& p, const double* table) {
  constexpr double L = 0.693147180559945309417 / TABLE;
  const double s = fmax(((double)x - (double)p.top) * p.c, -40.0 / L);
  const double k = s + 1.5 * MAGIC;                    // an integer in the low word
  const int n = (int)(unsigned)__builtin_bit_cast(u64, k);
  const double f = s - (k - 1.5 * MAGIC);
  double q = fma(f, L * L * L / 6.0, L * L / 2.0);
  q = fma(f, q, L);
  q = fma(f, q, 1.0);
  return ldexp(q * table[n & (TABLE - 1)], n >> 8);
}
// the same without the table, for few values
__device__ __forceinline__ double weight_by(float x, const RowParams& p, double unit) {
  constexpr double L = 0.693147180559945309417 / TABLE;
  return exp2(fmax(((double)x - (double)p.top) * p.c, -40.0 / L) * (1.0 / TABLE)) * unit;
}
__device__ __forceinline__ u64 rounded(double w) { return __builtin_bit_cast(u64, w + MAGIC) & 0xfffffffffffffull; }
__device__ __forceinline__ u64 units(float x, const RowParams& p, const double* table) { return rounded(weight(x, p, table)); }
__device__ __forceinline__ int bin_of(float x, const RowParams& p) {
  const float d = (p.top - x) * p.bins;                // both steps round monotonically
  return d < (float)(p.nbins - 1) ? (int)d : p.nbins - 1;
}

template <typename V>
__device__ __forceinline__ V wave_total(V v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
template <typename V>
__device__ __forceinline__ V wave_running(V v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// ---- where the elements come from: the row in memory, or the list in LDS ----
template <typename T>
struct RowSource {
  static constexpr int AHEAD = 2;         // vectors in flight per lane
  const T* row;
  int n, wave, waves, lane;

  // f(index of the first, eight raw logits) for the vectors of [from, to) in this wave's piece of that range
  template <typename F>
  __device__ __forceinline__ void vectors(int from, int to, F f) const {
    const int per = piece(from, to) >> 3, vecs = (to - from + 7) >> 3;
    const int end = (wave + 1) * per < vecs ? (wave + 1) * per : vecs;
    int v0 = wave * per;
    for (; v0 + 64 * AHEAD <= end && from + 8 * (v0 + 64 * AHEAD) <= n; v0 += 64 * AHEAD) {
      decltype(load_raw(row, 0, 0)) raw[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) raw[a] = load_whole(row + from + 8 * (v0 + 64 * a + lane));
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) f(from + 8 * (v0 + 64 * a + lane), raw[a]);
    }
    for (; v0 < end; v0 += 64) {                       // every lane takes part; those past the piece see nothing but -inf
      const int e = v0 + lane < end ? from + 8 * (v0 + lane) : n;
      f(e, load_raw(row, e, n));
    }
  }
  // f(index, value) for the elements of that piece, and -inf at indices >= n that fill up the last wave instruction
  template <typename F>
  __device__ __forceinline__ void each(int from, int to, F f) const {
    vectors(from, to, [&](int e, const auto& raw) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f(e + i, clean(raw_at(raw, i)));
    });
  }
  template <typename F>
  __device__ __forceinline__ void all(F f) const { each(0, n, f); }
  // elements of a wave's piece: whole wave instructions
  __device__ __forceinline__ int piece(int from, int to) const {
    const int vecs = (to - from + 7) >> 3;
    return (((vecs + waves - 1) / waves + 63) & ~63) * 8;
  }
};

struct ListSource {
  const SampleLds& lds;
  int wave, waves, lane;
  template <typename F>
  __device__ __forceinline__ void all(F f) const {
    const int n = (int)lds.seg_n[wave];
    for (int i = lane; i < n; i += 64) f(lds.seg_i[wave * SEG + i], lds.seg_x[wave * SEG + i]);
  }
};

// `locate` finds the first element, in index order, at which the running sum of g(index, value) exceeds target_of(total),
// and gives its index to every thread.  The wave whose piece it lies in:
template <typename F>
__device__ __forceinline__ int pick_wave(const SampleLds& lds, u64 mine, int waves, int wave, int lane, u64& target, bool first,
                                         F target_of) {
  const u64 m = wave_total(mine);
  __syncthreads();
  if (lane == 0) lds.part_m[wave] = m;
  __syncthreads();
  if (first) {
    u64 total = 0;
    for (int w = 0; w < waves; ++w) total += lds.part_m[w];
    target = target_of(total);
  }
  int w = 0;
  u64 before = 0;
  while (w < waves - 1 && before + lds.part_m[w] <= target) before += lds.part_m[w++];
  target -= before;
  return w;
}
// eight values per lane, in order: the position (lane and element) at which the running sum exceeds `target`, -1 if none
__device__ __forceinline__ int pick_in_wave(const u64 (&v)[8], int lane, u64& target) {
  u64 sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += v[i];
  const u64 incl = wave_running(sum, lane);
  const u64 hit = __ballot(incl > target);
  if (!hit) {
    target -= __shfl(incl, 63);
    return -1;
  }
  const int l = __ffsll(hit) - 1;
  u64 run = incl - sum;
  int at = 7;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    u64 upto = run;
#pragma unroll
    for (int j = 0; j <= i; ++j) upto += v[j];
    if (upto > target) at = i;
  }
  return 8 * l + __shfl(at, l);
}

template <typename T, typename G, typename F>
__device__ __forceinline__ int locate(const SampleLds& lds, const RowSource<T>& s, G g, F target_of) {
  u64 target = 0;
  int from = 0, to = s.n;
  for (int level = 0; level < 2; ++level) {
    u64 m = 0;
    s.each(from, to, [&](int e, float x) { m += g(e, x); });
    const int w = pick_wave(lds, m, s.waves, s.wave, s.lane, target, level == 0, target_of);
    const int step = s.piece(from, to);
    from += w * step;
    to = from + step < to ? from + step : to;
    if (s.waves == 1) break;
  }
  __syncthreads();
  if (s.wave == 0) {                                           // 512 to 1024 elements
    int at = -1;
    for (int e0 = from; e0 < to && at < 0; e0 += 512) {
      const auto raw = load_raw(s.row, e0 + 8 * s.lane < to ? e0 + 8 * s.lane : s.n, s.n);
      u64 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + 8 * s.lane + i;
        v[i] = e < to ? g(e, clean(raw_at(raw, i))) : 0;
      }
      at = pick_in_wave(v, s.lane, target);
      if (at >= 0) at += e0;
    }
    if (s.lane == 0) lds.found[2] = (unsigned)at;
  }
  __syncthreads();
  return (int)lds.found[2];
}
template <typename G, typename F>
__device__ __forceinline__ int locate(const SampleLds& lds, const ListSource& s, G g, F target_of) {
  u64 target = 0, m = 0;
  s.all([&](int e, float x) { m += g(e, x); });
  const int w = pick_wave(lds, m, s.waves, s.wave, s.lane, target, true, target_of);
  __syncthreads();
  if (s.wave == 0) {
    static_assert(SEG == 512, "a segment is eight entries per lane");
    const int n = (int)lds.seg_n[w];
    u64 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = 8 * s.lane + i;
      v[i] = k < n ? g(lds.seg_i[w * SEG + k], lds.seg_x[w * SEG + k]) : 0;
    }
    const int at = pick_in_wave(v, s.lane, target);
    if (s.lane == 0) lds.found[2] = (unsigned)(at >= 0 && at < n ? lds.seg_i[w * SEG + at] : -1);
  }
  __syncthreads();
  return (int)lds.found[2];
}

// Puts the elements that `want` names into the list; false (for every thread) if a segment does not hold its wave's share.
template <typename T, typename W>
__device__ __forceinline__ bool make_list(const SampleLds& lds, const RowSource<T>& s, W want) {
  unsigned n = 0;
  s.vectors(0, s.n, [&](int e, const auto& raw) {
    unsigned mask = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (want(clean(raw_at(raw, i)))) mask |= 1u << i;
    const int left = s.n - e;                                  // no index behind the row's end
    if (left < 8) mask &= (1u << left) - 1;
    if (!__any(mask != 0)) return;
    const unsigned c = __popc(mask);
    const unsigned incl = wave_running(c, s.lane);
    unsigned at = n + incl - c;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (mask >> i & 1) {
        if (at < SEG) {
          lds.seg_x[s.wave * SEG + at] = clean(raw_at(raw, i));
          lds.seg_i[s.wave * SEG + at] = e + i;
        }
        ++at;
      }
    n = __builtin_amdgcn_readlane(n + incl, 63);
  });
  __syncthreads();
  if (s.lane == 0) lds.seg_n[s.wave] = n;
  __syncthreads();
  bool fits = true;
  for (int w = 0; w < s.waves; ++w) fits = fits && lds.seg_n[w] <= SEG;
  return fits;
}

__device__ __forceinline__ void clear_bins(const SampleLds& lds) {
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    lds.count[i * blockDim.x + threadIdx.x] = 0;
    lds.mass[i * blockDim.x + threadIdx.x] = 0;
  }
  __syncthreads();
}

struct Found {
  int bin;
  unsigned count;            // before the bin
  u64 mass;
};
// The bin in which the running count reaches `k` (k > 0) or else the running mass reaches `target`, counting from `count0` /
// `mass0` in front of bin 0.
__device__ __forceinline__ Found find_bin(const SampleLds& lds, unsigned k, double target, unsigned count0, u64 mass0, int waves) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __syncthreads();
  const unsigned c0 = lds.count[2 * tid], c1 = lds.count[2 * tid + 1];
  const u64 m0 = lds.mass[2 * tid], m1 = lds.mass[2 * tid + 1];
  const unsigned ci = wave_running(c0 + c1, lane);
  const u64 mi = wave_running(m0 + m1, lane);
  if (lane == 63) {
    lds.part_c[wave] = ci;
    lds.part_m[wave] = mi;
  }
  __syncthreads();
  unsigned cb = count0 + ci - (c0 + c1);
  u64 mb = mass0 + mi - (m0 + m1);
  for (int w = 0; w < wave; ++w) {
    cb += lds.part_c[w];
    mb += lds.part_m[w];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const unsigned cn = i ? c1 : c0;
    const u64 mn = i ? m1 : m0;
    const bool here = k > 0 ? cb < k && k <= cb + cn : (double)mb < target && (double)(mb + mn) >= target;
    if (here) {
      lds.found[0] = (unsigned)(2 * tid + i);
      lds.found[1] = cb;
      *lds.found_m = mb;
    }
    cb += cn;
    mb += mn;
  }
  __syncthreads();
  return Found{(int)lds.found[0], lds.found[1], *lds.found_m};
}

struct Border {              // the last kept token: its key, how many of the tokens with that key are kept, what lies before
  unsigned key, ties;
  u64 mass_before;
};
// Narrows step `at` of the first histogram down to one value; the source holds at least that step's elements.
template <typename S>
__device__ __forceinline__ Border refine(const SampleLds& lds, const S& s, const RowParams& p, unsigned k, double target, Found at) {
  const int bin0 = at.bin;
  __syncthreads();
  if (threadIdx.x == 0) {
    lds.lo[0] = 0xffffffffu;
    lds.lo[1] = 0;
  }
  __syncthreads();
  unsigned klo = 0xffffffffu, khi = 0;
  s.all([&](int e, float x) {
    if (bin_of(x, p) == bin0) {
      const unsigned key = key_of(x);
      klo = key < klo ? key : klo;
      khi = key > khi ? key : khi;
    }
  });
  if (klo <= khi) {
    atomicMin(&lds.lo[0], klo);
    atomicMax(&lds.lo[1], khi);
  }
  __syncthreads();
  unsigned base = lds.lo[0], top = lds.lo[1];
  const int log_bins = 31 - __clz(p.nbins);
  while (top > base) {                                   // every trip narrows the range to one bin of it
    const int bits = 32 - __clz((int)(top - base));
    const int shift = bits > log_bins ? bits - log_bins : 0;
    clear_bins(lds);
    s.all([&](int e, float x) {
      const unsigned key = key_of(x);
      if (key >= base && key <= top) {
        atomicAdd(&lds.count[(key - base) >> shift], 1u);
        atomicAdd(&lds.mass[(key - base) >> shift], units(x, p, lds.table));
      }
    });
    at = find_bin(lds, k, target, at.count, at.mass, s.waves);
    base += (unsigned)at.bin << shift;
    const unsigned span = (1u << shift) - 1;                 // base + span may lie behind the last key there is
    top = top > base && top - base > span ? base + span : top;
  }
  Border b;
  b.key = base;
  b.mass_before = at.mass;
  if (k > 0) {
    b.ties = k - at.count;
  } else {
    const double r = ceil((target - (double)at.mass) / (double)units(value_of(base), p, lds.table));   // kept while mass + i w < target
    b.ties = r < 1.0 ? 1u : (r > (double)MAX_VOCAB ? (unsigned)MAX_VOCAB : (unsigned)r);
  }
  return b;
}

struct Limit {               // the tokens that are kept: values above x, and those equal to it up to an index
  float x;
  int index;
};

template <typename S>
__device__ __forceinline__ int draw(const SampleLds& lds, const S& s, const RowParams& p, Limit lim, float min_p, float u) {
  if (min_p > 0.f) {                                           // w >= min_p in terms of x, rounded up to a float
    const double least = (double)p.top + log((double)fminf(min_p, 1.f)) * (TABLE / 0.693147180559945309417) / p.c;
    float x = (float)least;
    if ((double)x < least) x = nextafterf(x, INFINITY);
    x = fminf(x, p.top);
    if (x > lim.x) lim = Limit{x, 0x7fffffff};
  }
  if (!(u > 0.f))            // u = 0 (or NaN): the first kept token whose weight is a number at all, however small
    return locate(lds, s, [&](int e, float x) -> u64 {
      const bool kept = x > lim.x || (x == lim.x && e <= lim.index);
      return kept && ((double)x - (double)p.top) * p.c > -745.13 * (TABLE / 0.693147180559945309417);
    }, [](u64) -> u64 { return 0; });
  u = u < 1.f ? u : 0.99999994f;
  return locate(lds, s, [&](int e, float x) -> u64 {
    const u64 w = units(x, p, lds.table);
    return x > lim.x || (x == lim.x && e <= lim.index) ? w : 0;
  }, [&](u64 total) -> u64 {
    const u64 t = (u64)((double)u * (double)total);
    return t < total ? t : total - 1;
  });
}
template <typename S>
__device__ __forceinline__ int tie_index(const SampleLds& lds, const S& s, float value, unsigned ties) {
  return locate(lds, s, [&](int e, float x) -> u64 { return x == value; },
                [&](u64 total) -> u64 { return (ties < total ? ties : total) - 1; });
}

// the mass histogram of the elements above `floor`, and its total
template <typename S>
__device__ __forceinline__ u64 mass_bins(const SampleLds& lds, const S& s, const RowParams& p, float floor) {
  clear_bins(lds);
  u64 m = 0;
  s.all([&](int e, float x) {
    u64 w = units(x, p, lds.table);
    w = x > floor ? w : 0;
    m += w;
    atomicAdd(&lds.mass[w ? bin_of(x, p) : s.lane], w);        // no branch; nothing is added to some bin rather than to the last one
  });
  m = wave_total(m);
  if (s.lane == 0) lds.part_m[s.wave] = m;
  __syncthreads();
  u64 total = 0;
  for (int w = 0; w < s.waves; ++w) total += lds.part_m[w];
  __syncthreads();
  return total;
}

// inclusive prefix sum of one value per thread, and the sum of all
__device__ __forceinline__ u64 block_running(const SampleLds& lds, u64 v, int waves, u64& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 incl = wave_running(v, lane);
  __syncthreads();
  if (lane == 63) lds.part_m[wave] = incl;
  __syncthreads();
  u64 base = 0;
  total = 0;
  for (int w = 0; w < waves; ++w) {
    if (w < wave) base += lds.part_m[w];
    total += lds.part_m[w];
  }
  return base + incl;
}

// A list of few entries (one per thread at most): every entry finds its rank by comparing with all others, and the rest
// is two prefix sums, one by rank and one by index.  A dozen barriers where the histograms take fifty: 19 against 34 us for
// 32001 logits with top-k 40 and the other filters; the comparisons grow with the square (1000 entries: 128 against 27 us).
// The bins hold the entries in index order, then the weights by rank.
constexpr int FEW = 256;
__device__ __forceinline__ int by_few(const SampleLds& lds, const RowParams& p, int n, unsigned k, float top_p, float min_p, float u,
                                      int waves) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float* xs = reinterpret_cast<float*>(lds.count);           // [64 waves]
  int base = 0;
  for (int w = 0; w < wave; ++w) base += (int)lds.seg_n[w];
  int* is = reinterpret_cast<int*>(lds.count) + 64 * waves;
  for (int i = lane; i < (int)lds.seg_n[wave]; i += 64) {
    xs[base + i] = lds.seg_x[wave * SEG + i];
    is[base + i] = lds.seg_i[wave * SEG + i];
  }
  __syncthreads();
  const bool mine = tid < n;
  const float x = mine ? xs[tid] : -INFINITY;
  const u64 w = mine ? units(x, p, lds.table) : 0;
  int rank = 0;
  for (int j0 = 0; j0 < n && 64 * wave < n; j0 += 4) {       // 128 bins a wave: xs is readable up to 64 waves + 3
    const f32x4 o = *reinterpret_cast<const f32x4*>(xs + j0);
#pragma unroll
    for (int j = 0; j < 4; ++j) rank += (j0 + j < n) & ((o[j] > x) | ((o[j] == x) & (j0 + j < tid)));
  }
  if (mine) lds.mass[rank] = w;
  __syncthreads();
  u64 total;
  const u64 wr = mine && tid < (int)k ? lds.mass[tid] : 0;   // of rank tid
  const u64 before = block_running(lds, wr, waves, total) - wr;
  const double target = (double)top_p * (double)total;
  const bool in = mine && tid < (int)k && (!(top_p < 1.f) || (double)before < target || tid == 0);
  // what top-k and top-p keep is a head of the ranks
  const u64 head = __ballot(in);
  __syncthreads();
  if (lane == 0) lds.part_c[wave] = (unsigned)__popcll(head);
  __syncthreads();
  int keep = 0;
  for (int v = 0; v < waves; ++v) keep += (int)lds.part_c[v];
  const bool first = !(u > 0.f);
  bool kept = mine && rank < keep;
  if (min_p > 0.f) kept = kept && ((double)x >= (double)p.top + log((double)fminf(min_p, 1.f)) * (TABLE / 0.693147180559945309417) / p.c || x == p.top);
  u64 v = kept ? w : 0;
  if (first) v = kept && ((double)x - (double)p.top) * p.c > -745.13 * (TABLE / 0.693147180559945309417);
  const u64 run = block_running(lds, v, waves, total);
  u64 t = 0;
  if (!first) {
    t = (u64)((double)(u < 1.f ? u : 0.99999994f) * (double)total);
    t = t < total ? t : total - 1;
  }
  if (run > t && run - v <= t) lds.found[2] = (unsigned)is[tid];
  __syncthreads();
  return (int)lds.found[2];
}

// top-k on, its step of the first histogram known: the rest of the row's work
template <typename S>
__device__ __forceinline__ int by_rank(const SampleLds& lds, const S& s, const RowParams& p, unsigned k, float top_p, float min_p,
                                       float u, Found at) {
  const Border b = refine(lds, s, p, k, 0.0, at);
  float value = value_of(b.key);
  unsigned ties = b.ties;
  if (top_p < 1.f) {
    // masses before the border's own value, then `ties` times that value's
    const u64 before = mass_bins(lds, s, p, value);
    const u64 w = units(value, p, lds.table);
    const double target = (double)top_p * (double)(before + ties * w);
    if ((double)before >= target) {
      const Found f = find_bin(lds, 0, target, 0, 0, s.waves);
      const Border c = refine(lds, s, p, 0, target, f);
      value = value_of(c.key);
      ties = c.ties;
    } else {
      const double r = ceil((target - (double)before) / (double)w);
      ties = r < (double)ties ? (r < 1.0 ? 1u : (unsigned)r) : ties;
    }
  }
  return draw(lds, s, p, Limit{value, tie_index(lds, s, value, ties)}, min_p, u);
}

// ---- rows of bf16 by value ----
constexpr int BV_LO = (127 - 30) << 7, BV_HI = (127 + 7) << 7;            // bits of 2^-30 and 2^7
constexpr int BV_SIDE = BV_HI - BV_LO;                                    // values of one sign
constexpr int BV_ZERO = BV_SIDE, BV_LOW = 2 * BV_SIDE + 1;                // index of 0; of everything at or below -2^7
constexpr int BV_BINS = BV_LOW + 1;                                       // indices rise with falling value
constexpr int BV_PER = (BV_BINS + 64 * MAX_WAVES - 1) / (64 * MAX_WAVES);
constexpr int BV_MIN_VOCAB = 64 * 8 * MAX_WAVES + 1;   // a workgroup of 16 waves; shorter rows would spend their time on the bins
constexpr int BV_BYTES = BV_PER * 64 * MAX_WAVES * 12 + MAX_WAVES * 12 + 64;

struct ByValueLds {
  u64* weight;               // [bins], then of the kept values only
  unsigned* count;           // [bins]
  u64* part_m;               // [waves]
  unsigned* part_c;          // [waves]
  u64* mass;                 // 0: total of the last scan, 1: mass before the border found
  unsigned* word;            // 0: first bin in use, 1: a row that does not fit, 2: border, 3: count before it, 4: token
};
__device__ __forceinline__ ByValueLds carve_by_value(char* p) {
  ByValueLds l;
  l.weight = reinterpret_cast<u64*>(p);
  l.part_m = l.weight + BV_PER * 64 * MAX_WAVES;
  l.mass = l.part_m + MAX_WAVES;
  l.count = reinterpret_cast<unsigned*>(l.mass + 2);
  l.part_c = l.count + BV_PER * 64 * MAX_WAVES;
  l.word = l.part_c + MAX_WAVES;
  return l;
}

__device__ __forceinline__ unsigned bits16(const u32x4& r, int i) { return i & 1 ? r[i >> 1] >> 16 : r[i >> 1] & 0xffffu; }
// index of a value, not yet kept within the bins: negative for values of 2^7 and more, > BV_LOW for those below -2^7; values
// between 0 and 2^-30 share the index of 0
__device__ __forceinline__ int index_of(unsigned u) {
  const int d = max((int)(u & 0x7fffu) - (BV_LO - 1), 0);
  return u & 0x8000u ? BV_ZERO + d : BV_ZERO - d;
}
__device__ __forceinline__ float value_at(int i) {
  const int d = i < BV_ZERO ? BV_ZERO - i : i - BV_ZERO;
  const unsigned u = d == 0 ? 0u : (unsigned)(d + BV_LO - 1) | (i > BV_ZERO ? 0x8000u : 0u);
  return __builtin_bit_cast(float, u << 16);
}

// Two values at once, in packed 16-bit integers: the vector unit is busy for 37 % of the cycles, waits fill the rest (with the
// weights found by neighbouring lanes, 50 -> 46 us for 256 rows of 131072).
using u16x2 = __attribute__((ext_vector_type(2))) unsigned short;
using i16x2 = __attribute__((ext_vector_type(2))) short;
__device__ __forceinline__ i16x2 both(int x) { return i16x2{(short)x, (short)x}; }
__device__ __forceinline__ u16x2 magnitudes(unsigned u) { return __builtin_bit_cast(u16x2, u & 0x7fff7fffu); }
// index_of of both
__device__ __forceinline__ i16x2 indices_of(unsigned u) {
  const u16x2 d = __builtin_elementwise_sub_sat(magnitudes(u), __builtin_bit_cast(u16x2, both(BV_LO - 1)));
  unsigned negative = __builtin_bit_cast(unsigned, __builtin_bit_cast(i16x2, u) >> 15);    // all ones or none
  asm("" : "+v"(negative));                                  // or it becomes two selects
  // BV_ZERO + d or BV_ZERO - d = BV_ZERO + ~d + 1
  return __builtin_bit_cast(i16x2, ~(__builtin_bit_cast(unsigned, d) ^ negative)) + __builtin_bit_cast(i16x2, negative) + both(BV_ZERO + 1);
}

// prefix sums over the bins of this thread's first one; lds.mass[0] becomes the whole mass
__device__ __forceinline__ void before_mine(const ByValueLds& lds, unsigned c, u64 m, int wave, int lane, unsigned& cb, u64& mb) {
  const unsigned ci = wave_running(c, lane);
  const u64 mi = wave_running(m, lane);
  __syncthreads();
  if (lane == 63) {
    lds.part_c[wave] = ci;
    lds.part_m[wave] = mi;
  }
  __syncthreads();
  cb = ci - c;
  mb = mi - m;
  u64 total = 0;
#pragma unroll 4
  for (int w = 0; w < MAX_WAVES; ++w) {
    if (w < wave) {
      cb += lds.part_c[w];
      mb += lds.part_m[w];
    }
    total += lds.part_m[w];
  }
  if (wave == 0 && lane == 0) lds.mass[0] = total;
  __syncthreads();
}

// false: the row does not fit (for every thread)
__device__ __forceinline__ bool sample_by_value(char* smem, const RowSource<bf16>& s, float t, int top_k, float top_p, float min_p,
                                                float u, double unit, int& token) {
  const ByValueLds lds = carve_by_value(smem);
  const int tid = threadIdx.x, lane = s.lane, wave = s.wave, n = s.n;
#pragma unroll
  for (int j = 0; j < BV_PER; ++j) lds.count[j * 64 * MAX_WAVES + tid] = 0;
  if (tid == 0) {
    lds.word[0] = BV_BINS;
    lds.word[1] = 0;
    lds.word[2] = BV_LOW;
  }
  __syncthreads();
  // ---- one pass: count every value ----
  {
    i16x2 least = both(0);
    u16x2 tiny = {0xffff, 0xffff};
    s.vectors(0, n, [&](int e, const u32x4& raw) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const i16x2 i = indices_of(raw[k]), c = __builtin_elementwise_min(__builtin_elementwise_max(i, both(0)), both(BV_LOW));
        least = __builtin_elementwise_min(least, i);
        tiny = __builtin_elementwise_min(tiny, magnitudes(raw[k]) - u16x2{1, 1});       // of 0: 0xffff
        atomicAdd(&lds.count[c.x], 1u);                      // -inf and NaN among the low ones, and what fills up the row
        atomicAdd(&lds.count[c.y], 1u);
      }
    });
    if (least.x < 0 || least.y < 0 || tiny.x < BV_LO - 1 || tiny.y < BV_LO - 1) lds.word[1] = 1;      // 2^7 and more; between 0 and 2^-30
  }
  __syncthreads();
  unsigned cnt[BV_PER];
  int first = BV_BINS;
#pragma unroll
  for (int j = BV_PER - 1; j >= 0; --j) {
    const int i = tid * BV_PER + j;
    cnt[j] = i < BV_LOW ? lds.count[i] : 0;
    first = cnt[j] ? i : first;
  }
  if (first < BV_BINS) atomicMin(&lds.word[0], (unsigned)first);
  __syncthreads();
  const int top_i = (int)lds.word[0];
  if (lds.word[1] || top_i >= BV_LOW) return false;
  const float top = value_at(top_i);
  // low values that may matter: those of half a unit and more, and at u = 0 (or NaN) every weight that is a number at all
  if ((double)top + 128.0 < (u > 0.f ? 40.0 : 745.14) * (double)t && lds.count[BV_LOW] > 0) return false;
  RowParams p;
  p.top = top;
  p.bins = 0.f;
  p.nbins = 0;
  p.c = TABLE / 0.693147180559945309417 / (double)t;

  // ---- weights, and the borders ----
  unsigned c = 0;
  // (values that occur lie close together: neighbours go to neighbouring lanes here)
  for (int i = tid; i < BV_LOW; i += 64 * MAX_WAVES) lds.weight[i] = lds.count[i] ? rounded(weight_by(value_at(i), p, unit)) : 0;
  __syncthreads();
  u64 m = 0, w[BV_PER];
#pragma unroll
  for (int j = 0; j < BV_PER; ++j) {
    w[j] = cnt[j] ? lds.weight[tid * BV_PER + j] : 0;
    c += cnt[j];
    m += cnt[j] * w[j];
  }
  unsigned cb;
  u64 mb;
  before_mine(lds, c, m, wave, lane, cb, mb);
  int border = BV_LOW;                                       // the last value kept, how many of it, and the mass before it
  unsigned ties = 0;
  u64 before = lds.mass[0], total = before;
  auto publish = [&](int j, unsigned count_before, u64 mass_before) {
    lds.word[2] = (unsigned)(tid * BV_PER + j);
    lds.word[3] = count_before;
    lds.mass[1] = mass_before;
    lds.part_m[0] = w[j];
  };
  if (top_k > 0 && top_k < n) {
    unsigned cc = cb;
    u64 mm = mb;
#pragma unroll
    for (int j = 0; j < BV_PER; ++j) {
      if (cc < (unsigned)top_k && (unsigned)top_k <= cc + cnt[j]) publish(j, cc, mm);
      cc += cnt[j];
      mm += cnt[j] * w[j];
    }
    __syncthreads();
    if (lds.word[2] != BV_LOW) {                             // else k reaches the low values: all others are kept
      border = (int)lds.word[2];
      ties = (unsigned)top_k - lds.word[3];
      before = lds.mass[1];
      total = before + ties * lds.part_m[0];
    }
    __syncthreads();
  }
  if (top_p < 1.f) {
    const double target = (double)top_p * (double)total;
    u64 mm = mb;
#pragma unroll
    for (int j = 0; j < BV_PER; ++j) {
      if ((double)mm < target && target <= (double)(mm + cnt[j] * w[j])) publish(j, cnt[j], mm);
      mm += cnt[j] * w[j];
    }
    __syncthreads();
    const double r = ceil((target - (double)lds.mass[1]) / (double)lds.part_m[0]);      // kept while mass + i w < target
    // (sums are rounded to doubles here: r may come out above the number there is)
    const unsigned rr = r < 1.0 ? 1u : (r > (double)lds.word[3] ? lds.word[3] : (unsigned)r);
    const int at = (int)lds.word[2];
    ties = at == border && rr > ties ? ties : rr;
    border = at;
    before = lds.mass[1];
    total = before + ties * lds.part_m[0];
    __syncthreads();
  }
  if (min_p > 0.f) {                                         // values whose weight is below min_p fall away whole
    const double least = (double)top + log((double)fminf(min_p, 1.f)) * (double)t;
    u64 cut = 0;
    int last = -1;
#pragma unroll
    for (int j = 0; j < BV_PER; ++j) {
      const int i = tid * BV_PER + j;
      if (i < border && cnt[j] && ((double)value_at(i) >= least || i == top_i)) {
        cut += cnt[j] * w[j];
        last = i;
      }
    }
    const bool whole = border < BV_LOW && ((double)value_at(border) >= least || border == top_i);
    cut = wave_total(cut);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o));
    if (lane == 0) {
      lds.part_m[wave] = cut;
      lds.part_c[wave] = (unsigned)(last + 1);
    }
    __syncthreads();
    if (!whole) {                                            // every kept value lies before the border, with all its tokens
      before = 0;
      int end = 0;
      for (int k = 0; k < MAX_WAVES; ++k) {
        before += lds.part_m[k];
        end = max(end, (int)lds.part_c[k]);
      }
      border = end;
      ties = 0;
      total = before;
    }
    __syncthreads();
  }

  // ---- the draw: weights of the kept values by index, the border's apart ----
  const bool zero = !(u > 0.f);                              // u = 0 (or NaN): the first kept token whose weight is a number at all
#pragma unroll
  for (int j = 0; j < BV_PER; ++j) {
    const int i = tid * BV_PER + j;
    if (zero && cnt[j]) w[j] = ((double)value_at(i) - (double)top) * p.c > -745.13 * (TABLE / 0.693147180559945309417);
    lds.weight[i] = i < border ? w[j] : 0;
    if (i == border) lds.mass[1] = w[j];
  }
  __syncthreads();
  const u64 w_border = ties > 0 ? lds.mass[1] : 0;
  u64 target = 0;
  if (!zero) {
    target = (u64)((double)(u < 1.f ? u : 0.99999994f) * (double)total);
    target = target < total ? target : total - 1;
  }
  int from = 0, to = n;
  const i16x2 last_kept = both(border);
  for (int level = 0; level < 2; ++level) {
    u64 sum = 0;
    unsigned seen = 0;
    u16x2 others = {0, 0};
    s.vectors(from, to, [&](int e, const u32x4& raw) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const i16x2 i = indices_of(raw[k]);
        const u16x2 c = __builtin_bit_cast(u16x2, __builtin_elementwise_min(i, last_kept));
        unsigned apart = __builtin_bit_cast(unsigned, i ^ last_kept);
        asm("" : "+v"(apart));                               // or the line after the next becomes comparisons
        sum += lds.weight[c.x] + lds.weight[c.y];            // 0 from the border on; one address, so those lanes do not collide
        others += __builtin_elementwise_min(__builtin_bit_cast(u16x2, apart), u16x2{1, 1});
      }
      seen += 8;
    });
    unsigned eq = seen - others.x - others.y;                // of the border's value
    sum = wave_total(sum);
    eq = wave_total(eq);
    __syncthreads();
    if (lane == 0) {
      lds.part_m[wave] = sum;
      lds.part_c[wave] = eq;
    }
    __syncthreads();
    int k = 0;
    for (; k < MAX_WAVES; ++k) {                             // the wave's piece in which the running sum passes the target
      const unsigned e = min(lds.part_c[k], ties);
      const u64 piece_sum = lds.part_m[k] + e * w_border;
      if (piece_sum > target || k == MAX_WAVES - 1) break;
      target -= piece_sum;
      ties -= e;
    }
    const int step = s.piece(from, to);
    from += k * step;
    to = from + step < to ? from + step : to;
  }
  if (wave == 0) {
    int at = -1;
    for (int e0 = from; e0 < to && at < 0; e0 += 512) {
      const int e = e0 + 8 * lane;
      const u32x4 raw = load_raw(s.row, e < to ? e : n, n);
      u64 v[8];
      unsigned eq = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) eq += min(index_of(bits16(raw, k)), BV_LOW) == border;
      unsigned rank = wave_running(eq, lane) - eq;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = min(index_of(bits16(raw, k)), BV_LOW);
        v[k] = i == border ? (rank++ < ties ? w_border : 0) : lds.weight[i];
      }
      const unsigned here = wave_total(eq);
      at = pick_in_wave(v, lane, target);
      if (at >= 0) at += e0;
      ties -= min(here, ties);
    }
    if (lane == 0) lds.word[4] = (unsigned)at;
  }
  __syncthreads();
  token = (int)lds.word[4];
  return true;
}

template <typename T>
__global__ __launch_bounds__(64 * MAX_WAVES) void sample_kernel(const SampleArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  const SampleLds lds = carve(smem, waves);
  const int r = blockIdx.x, n = a.vocab;
  const RowSource<T> s{reinterpret_cast<const T*>(a.logits) + (long long)r * a.row_stride, n, wave, waves, lane};
  const int log_n = n > 1 ? 32 - __clz(n - 1) : 0;
  const double unit = ldexp(1.0, log_n > 12 ? 63 - log_n : 51);
  const float t = a.temperature ? a.temperature[r] : 1.f;
  const int top_k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.f;
  const float min_p = a.min_p ? a.min_p[r] : 0.f;
  const bool greedy = !(t > 0.f) || top_k == 1 || top_p <= 0.f;
  int token;
  if constexpr (sizeof(T) == 2) {
    if (n >= BV_MIN_VOCAB && !greedy) {
      if (sample_by_value(smem, s, t, top_k, top_p, min_p, a.u[r], unit, token)) {
        if (tid == 0) a.tokens[r] = token;
        return;
      }
      __syncthreads();
    }
  }
  for (int i = tid; i < TABLE; i += blockDim.x) lds.table[i] = exp_table.v[i] * unit;

  // the largest logit, and the lane's first vector that holds its own largest
  float top = -INFINITY;
  int top_at = 0;
  s.vectors(0, n, [&](int e, const auto& raw) {
    float m = clean(raw_at(raw, 0));
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, clean(raw_at(raw, i)));
    top_at = m > top ? e : top_at;
    top = fmaxf(top, m);
  });
  const float lane_top = top;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (lane == 0) lds.part_c[wave] = __builtin_bit_cast(unsigned, top);
  __syncthreads();
  for (int w = 0; w < waves; ++w) top = fmaxf(top, __builtin_bit_cast(float, lds.part_c[w]));
  __syncthreads();

  if (top == -INFINITY) {
    token = -1;
  } else if (greedy) {
    if (tid == 0) lds.lo[0] = 0xffffffffu;
    __syncthreads();
    if (lane_top == top) atomicMin(&lds.lo[0], (unsigned)top_at);
    __syncthreads();
    const int e = (int)lds.lo[0];
    const auto raw = load_raw(s.row, e, n);
    token = e;
#pragma unroll
    for (int i = 7; i >= 0; --i) token = clean(raw_at(raw, i)) == top ? e + i : token;
  } else {
    RowParams p;
    p.top = top;
    p.nbins = waves * BINS_PER_WAVE;
    p.bins = fminf((float)p.nbins / RANGE / t, 1e30f);         // finite, so that the largest logit lies in bin 0
    p.c = TABLE / 0.693147180559945309417 / (double)t;
    const float u = a.u[r];
    if (top_k > 0 && top_k < n) {
      clear_bins(lds);
      s.all([&](int e, float x) { atomicAdd(&lds.count[bin_of(x, p)], 1u); });
      const Found at = find_bin(lds, (unsigned)top_k, 0.0, 0, 0, waves);
      if (make_list(lds, s, [&](float x) { return bin_of(x, p) <= at.bin; })) {
        int entries = 0;
        for (int w = 0; w < waves; ++w) entries += (int)lds.seg_n[w];
        if (entries <= (64 * waves < FEW ? 64 * waves : FEW)) token = by_few(lds, p, entries, (unsigned)top_k, top_p, min_p, u, waves);
        else token = by_rank(lds, ListSource{lds, wave, waves, lane}, p, (unsigned)top_k, top_p, min_p, u, at);
      } else {
        token = by_rank(lds, s, p, (unsigned)top_k, top_p, min_p, u, at);
      }
    } else {
      Limit lim{-INFINITY, n};
      if (top_p < 1.f) {
        const double target = (double)top_p * (double)mass_bins(lds, s, p, -INFINITY);
        const Found at = find_bin(lds, 0, target, 0, 0, waves);
        if (make_list(lds, s, [&](float x) { return bin_of(x, p) == at.bin; })) {
          const ListSource l{lds, wave, waves, lane};
          const Border b = refine(lds, l, p, 0, target, at);
          lim.x = value_of(b.key);
          lim.index = tie_index(lds, l, lim.x, b.ties);
        } else {
          const Border b = refine(lds, s, p, 0, target, at);
          lim.x = value_of(b.key);
          lim.index = tie_index(lds, s, lim.x, b.ties);
        }
      }
      token = draw(lds, s, p, lim, min_p, u);
    }
  }
  if (tid == 0) a.tokens[r] = token;
}

}  // namespace

int launch_sample_tokens(int dtype, const SampleArgs& a, hipStream_t stream) {
  if (dtype != DT_BF16 && dtype != DT_F32) return fail("sample_tokens: dtype %d", dtype);
  if (a.rows < 0 || a.vocab < 1 || a.vocab > MAX_VOCAB) return fail("sample_tokens: %d rows, vocabulary %d out of range (1..%d)", a.rows, a.vocab, MAX_VOCAB);
  if (a.rows == 0) return 0;
  if (a.rows > 1 && a.row_stride < a.vocab) return fail("sample_tokens: rows of %d logits overlap (stride %lld)", a.vocab, a.row_stride);
  if (!a.logits || !a.u || !a.tokens) return fail("sample_tokens: null operand");
  if ((uintptr_t)a.logits % (dtype == DT_BF16 ? 2 : 4)) return fail("sample_tokens: logits are not aligned to their type");
  // a wave takes 512 logits at a time: as many waves as have some, in powers of two (the histogram has 128 bins per wave)
  int waves = 1;
  while (waves < MAX_WAVES && waves * 512 < a.vocab) waves *= 2;
  auto k = dtype == DT_BF16 ? sample_kernel<bf16> : sample_kernel<float>;
  const int bytes = dtype == DT_BF16 && a.vocab >= BV_MIN_VOCAB && BV_BYTES > lds_bytes(waves) ? BV_BYTES : lds_bytes(waves);
  if (reserve_lds(reinterpret_cast<const void*>(k), bytes) != hipSuccess) return fail("sample_tokens: cannot reserve %d bytes of LDS", bytes);
  k<<<a.rows, 64 * waves, bytes, stream>>>(a);
  return check_launch("sample_tokens");
}

}  // namespace fcenc
