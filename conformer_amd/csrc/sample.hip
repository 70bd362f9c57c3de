// Drawing a token per row of logits (gfx950).
//
// With x the logits of a row as fp32 and t its temperature:  w_i = exp((x_i - max x) / t).  The tokens are ordered by
// falling x, equal ones by rising index, and three filters keep a head of that order:
//   top-k : the first k;                                             (k <= 0: all)
//   top-p : token i while the mass of those before it is below p times the mass that top-k left;    (p >= 1: all)
//   min-p : tokens with w_i >= min_p                                 (w of the largest is 1)
// The first token is always kept.  Over the kept ones in index order, with C_i the running sum of w and C the whole sum,
// the token drawn for a given u in [0, 1) is the first with C_i > u C.  t <= 0 takes the largest logit.
//
// A token is a comparison of a sum with a border, so sums must not depend on the order of their terms: weights are
// formed in fp64 and rounded to integers in units of 2^-45 (the largest is 2^45; up to 2^18 of them stay below 2^63),
// and integers add up exactly in any order, LDS atomics included.  A weight below 2^-46 of the largest counts as 0.
//
// One workgroup per row.  The head's last token is found by counting, not sorting: a histogram (counts and masses) over
// 2048 equal steps of (max - x) / t gives the step it lies in, finer histograms over the values' bit patterns inside
// that step give its value, and among equal values an index count gives the token.
#include <math.h>

#include "common.h"
#include "kernels.h"

namespace fcenc {

namespace {

constexpr int NBINS = 2048;
constexpr float BINS_PER_UNIT = 64.f;             // 2048 steps reach down to exp(-32), below a weight's last bit
constexpr int MAX_VOCAB = 1 << 18;
constexpr int MAX_WAVES = 16;
constexpr double UNIT = 35184372088832.0;         // 2^45
using u64 = unsigned long long;

struct SampleLds {
  u64 mass[NBINS];
  u64 part_m[MAX_WAVES];
  double table[32];                               // 2^(j / 32)
  unsigned count[NBINS];
  unsigned part_c[MAX_WAVES];
  unsigned lo, hi;                                // range of keys
  // a border found in the bins
  u64 mass_before;
  unsigned count_before;
  int bin;
  int token;
};

// larger values have larger keys; -0 counts as 0, NaN as -inf
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ float clean(float x) { return x == x ? (x == 0.f ? 0.f : x) : -INFINITY; }

// eight logits from element e of the row on; elements behind the row are -inf
__device__ __forceinline__ void load_logits(const float* row, int e, int n, float (&x)[8]) {
  struct __attribute__((packed, aligned(4))) V { float v[8]; };
  if (e + 8 <= n) {
    const V v = *reinterpret_cast<const V*>(row + e);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = clean(v.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = e + i < n ? clean(row[e + i]) : -INFINITY;
  }
}
__device__ __forceinline__ void load_logits(const bf16* row, int e, int n, float (&x)[8]) {
  struct __attribute__((packed, aligned(2))) V { bf16 v[8]; };
  if (e + 8 <= n) {
    const V v = *reinterpret_cast<const V*>(row + e);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = clean((float)v.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = e + i < n ? clean((float)row[e + i]) : -INFINITY;
  }
}

// exp of z <= 0 with z > -40, relative error below 1e-14: z = (32 n + j + f) ln 2 / 32, |f| <= 1/2, and the Taylor sum of
// exp(f ln 2 / 32) to the fifth power leaves (0.0109)^6 / 720 = 2e-15
__device__ __forceinline__ double exp_neg(double z, const double* table) {
  const double s = z * (32.0 / M_LN2);
  const double k = rint(s);
  const double f = (s - k) * (M_LN2 / 32.0);
  const int n = (int)k;
  double p = fma(f, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(f, p, 1.0 / 6.0);
  p = fma(f, p, 0.5);
  p = fma(f, p, 1.0);
  p = fma(f, p, 1.0);
  return ldexp(p * table[n & 31], n >> 5);
}

struct RowParams {
  float top;                 // the largest logit
  float bins;                // steps per unit of logit
  double inv_t;
};

__device__ __forceinline__ double weight(float x, const RowParams& p, const double* table) {
  if (x == p.top) return 1.0;
  const double z = ((double)x - (double)p.top) * p.inv_t;
  return z > -33.0 ? exp_neg(z, table) : 0.0;
}
__device__ __forceinline__ u64 units(double w) { return (u64)(w * UNIT + 0.5); }
__device__ __forceinline__ int bin_of(float x, const RowParams& p) {
  if (x == p.top) return 0;
  const float d = (p.top - x) * p.bins;              // both steps round monotonically
  return d < (float)(NBINS - 1) ? (int)d : NBINS - 1;
}

__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// calls f(index, eight logits) for the vectors of [from, to) that belong to this wave: a contiguous piece per wave
template <typename T, typename F>
__device__ __forceinline__ void for_row(const T* row, int from, int to, int n, int wave, int waves, int lane, F f) {
  const int vecs = (to - from + 7) >> 3;
  const int per = ((vecs + waves - 1) / waves + 63) & ~63;      // whole wave instructions
  const int end = (wave + 1) * per < vecs ? (wave + 1) * per : vecs;
  for (int v = wave * per + lane; v < end; v += 64) {
    float x[8];
    load_logits(row, from + 8 * v, n, x);
    f(from + 8 * v, x);
  }
}
__device__ __forceinline__ int piece(int from, int to, int waves) {           // elements of a wave's piece
  const int vecs = (to - from + 7) >> 3;
  return (((vecs + waves - 1) / waves + 63) & ~63) * 8;
}

// The bin in which the running count reaches `k` (k > 0) or else the running mass reaches `target`, starting from
// count0 / mass0 in front of bin 0: into lds.bin, .count_before, .mass_before.
__device__ __forceinline__ void find_bin(SampleLds& lds, unsigned k, double target, unsigned count0, u64 mass0, int waves) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = NBINS / (64 * waves);
  __syncthreads();
  unsigned c = 0;
  u64 m = 0;
  for (int i = 0; i < per; ++i) {
    c += lds.count[tid * per + i];
    m += lds.mass[tid * per + i];
  }
  unsigned ci = c;
  u64 mi = m;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned cu = __shfl_up(ci, o);
    const u64 mu = __shfl_up(mi, o);
    if (lane >= o) {
      ci += cu;
      mi += mu;
    }
  }
  if (lane == 63) {
    lds.part_c[wave] = ci;
    lds.part_m[wave] = mi;
  }
  __syncthreads();
  unsigned cb = count0 + ci - c;
  u64 mb = mass0 + mi - m;
  for (int w = 0; w < wave; ++w) {
    cb += lds.part_c[w];
    mb += lds.part_m[w];
  }
  for (int i = 0; i < per; ++i) {
    const unsigned cn = lds.count[tid * per + i];
    const u64 mn = lds.mass[tid * per + i];
    const bool here = k > 0 ? cb < k && k <= cb + cn : (double)mb < target && (double)(mb + mn) >= target;
    if (here) {
      lds.bin = tid * per + i;
      lds.count_before = cb;
      lds.mass_before = mb;
    }
    cb += cn;
    mb += mn;
  }
  __syncthreads();
}

__device__ __forceinline__ void clear_bins(SampleLds& lds, int threads) {
  __syncthreads();
  for (int i = threadIdx.x; i < NBINS; i += threads) {
    lds.count[i] = 0;
    lds.mass[i] = 0;
  }
  __syncthreads();
}

struct Border {              // the last kept token: its key, how many of the tokens with that key are kept, what lies before
  unsigned key, ties;
  u64 mass_before;
};

// Narrows the step `bin0` of the first histogram down to one value.
template <typename T>
__device__ __forceinline__ Border refine(SampleLds& lds, const T* row, int n, const RowParams& p, unsigned k, double target,
                                         int waves) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int bin0 = lds.bin;
  unsigned count0 = lds.count_before;
  u64 mass0 = lds.mass_before;
  __syncthreads();
  if (tid == 0) {
    lds.lo = 0xffffffffu;
    lds.hi = 0;
  }
  __syncthreads();
  unsigned klo = 0xffffffffu, khi = 0;                   // inverted keys: rising with falling value
  for_row(row, 0, n, n, wave, waves, lane, [&](int e, const float(&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i < n && bin_of(x[i], p) == bin0) {
        const unsigned key = ~key_of(x[i]);
        klo = key < klo ? key : klo;
        khi = key > khi ? key : khi;
      }
  });
  if (klo <= khi) {
    atomicMin(&lds.lo, klo);
    atomicMax(&lds.hi, khi);
  }
  __syncthreads();
  unsigned base = lds.lo, top = lds.hi;
  while (top != base) {
    const int bits = 32 - __clz((int)(top - base));
    const int shift = bits > 11 ? bits - 11 : 0;
    clear_bins(lds, 64 * waves);
    for_row(row, 0, n, n, wave, waves, lane, [&](int e, const float(&x)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned key = ~key_of(x[i]);
        if (e + i < n && key >= base && key <= top) {
          atomicAdd(&lds.count[(key - base) >> shift], 1u);
          atomicAdd(&lds.mass[(key - base) >> shift], units(weight(x[i], p, lds.table)));
        }
      }
    });
    find_bin(lds, k, target, count0, mass0, waves);
    count0 = lds.count_before;
    mass0 = lds.mass_before;
    base += (unsigned)lds.bin << shift;
    const unsigned end = base + ((1u << shift) - 1);
    top = end < top ? end : top;
  }
  Border b;
  b.key = base;
  b.mass_before = mass0;
  if (k > 0) {
    b.ties = k - count0;
  } else {
    const double w = (double)units(weight(value_of(~base), p, lds.table));
    const double r = ceil((target - (double)mass0) / w);       // kept while mass0 + i w < target
    b.ties = r < 1.0 ? 1u : (r > (double)MAX_VOCAB ? (unsigned)MAX_VOCAB : (unsigned)r);
  }
  return b;
}

template <typename T>
__global__ __launch_bounds__(64 * MAX_WAVES) void sample_kernel(const SampleArgs a) {
  __shared__ SampleLds lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, threads = blockDim.x, waves = threads >> 6;
  const int r = blockIdx.x, n = a.vocab;
  const T* row = reinterpret_cast<const T*>(a.logits) + (long long)r * a.row_stride;
  if (tid < 32) lds.table[tid] = exp2(tid / 32.0);

  // ---- the first of the largest ----
  u64 best = 0;                                            // key, then the smaller index
  for_row(row, 0, n, n, wave, waves, lane, [&](int e, const float(&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const u64 c = ((u64)key_of(x[i]) << 32) | (unsigned)~(e + i);
      best = e + i < n && c > best ? c : best;
    }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 c = __shfl_xor(best, o);
    best = c > best ? c : best;
  }
  if (lane == 0) lds.part_m[wave] = best;
  __syncthreads();
  for (int w = 0; w < waves; ++w) best = lds.part_m[w] > best ? lds.part_m[w] : best;
  RowParams p;
  p.top = value_of((unsigned)(best >> 32));
  const float t = a.temperature ? a.temperature[r] : 1.f;
  const int top_k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.f;
  const float min_p = a.min_p ? a.min_p[r] : 0.f;
  if (p.top == -INFINITY || !(t > 0.f) || top_k == 1 || top_p <= 0.f) {
    if (tid == 0) a.tokens[r] = p.top == -INFINITY ? -1 : (int)~(unsigned)best;
    return;
  }
  p.bins = BINS_PER_UNIT / t;
  p.inv_t = 1.0 / (double)t;

  // ---- the last token that top-k and top-p keep ----
  const bool by_k = top_k > 0 && top_k < n, by_p = top_p < 1.f;
  unsigned last_key = 0xffffffffu, last_ties = 0xffffffffu;      // everything
  if (by_k || by_p) {
    clear_bins(lds, threads);
    for_row(row, 0, n, n, wave, waves, lane, [&](int e, const float(&x)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e + i < n) {
          const int bin = bin_of(x[i], p);
          if (by_k) atomicAdd(&lds.count[bin], 1u);
          if (by_p) atomicAdd(&lds.mass[bin], units(weight(x[i], p, lds.table)));
        }
    });
    __syncthreads();
    u64 total = 0;
    if (by_p) {
      u64 m = 0;
      for (int i = tid; i < NBINS; i += threads) m += lds.mass[i];
      m = wave_sum(m);
      if (lane == 0) lds.part_m[wave] = m;
      __syncthreads();
      for (int w = 0; w < waves; ++w) total += lds.part_m[w];
      __syncthreads();
    }
    if (by_k) {
      find_bin(lds, (unsigned)top_k, 0.0, 0, 0, waves);
      const Border b = refine(lds, row, n, p, (unsigned)top_k, 0.0, waves);
      last_key = b.key;
      last_ties = b.ties;
      if (by_p) {
        total = b.mass_before + b.ties * units(weight(value_of(~b.key), p, lds.table));
        clear_bins(lds, threads);
        for_row(row, 0, n, n, wave, waves, lane, [&](int e, const float(&x)[8]) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (e + i < n && ~key_of(x[i]) <= last_key) atomicAdd(&lds.mass[bin_of(x[i], p)], units(weight(x[i], p, lds.table)));
        });
        __syncthreads();
      }
    }
    if (by_p) {
      const double target = (double)top_p * (double)total;
      find_bin(lds, 0, target, 0, 0, waves);
      const Border b = refine(lds, row, n, p, 0, target, waves);
      if (b.key < last_key) {
        last_key = b.key;
        last_ties = b.ties;
      } else if (b.ties < last_ties) {
        last_ties = b.ties;
      }
    }
  }

  // ---- among equal values the smaller indices: the last index kept ----
  int last_index = n;
  if (last_ties != 0xffffffffu) {
    int from = 0, to = n;
    unsigned want = last_ties;
    for (int level = 0; level < 3 && to - from > 0; ++level) {    // 1/waves of the range per level, then one wave alone
      unsigned c = 0;
      for_row(row, from, to, n, wave, waves, lane, [&](int e, const float(&x)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c += e + i < to && ~key_of(x[i]) == last_key;
      });
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
      __syncthreads();
      if (lane == 0) lds.part_c[wave] = c;
      __syncthreads();
      const int step = piece(from, to, waves);
      int w = 0;
      unsigned before = 0;
      while (w < waves && before + lds.part_c[w] < want) before += lds.part_c[w++];
      if (w == waves) {                                            // fewer than asked for: all of them are kept
        from = to;
        break;
      }
      want -= before;
      const int f = from + w * step;
      to = f + step < to ? f + step : to;
      from = f;
      __syncthreads();
    }
    if (from < to) {
      if (wave == 0) {
        int found = n;
        for (int e0 = from; e0 < to; e0 += 64) {                   // 512 to 1024 elements at most
          const int e = e0 + lane;
          float x = -INFINITY;
          if (e < to) x = clean((float)row[e]);
          const u64 hit = __ballot(e < to && ~key_of(x) == last_key);
          const unsigned c = (unsigned)__popcll(hit);
          if (c >= want) {
            u64 h = hit;
            for (unsigned i = 1; i < want; ++i) h &= h - 1;
            found = e0 + __ffsll(h) - 1;
            break;
          }
          want -= c;
        }
        if (lane == 0) lds.token = found;
      }
      __syncthreads();
      last_index = lds.token;
      __syncthreads();
    }
  }

  // ---- the draw ----
  auto kept = [&](int e, float x, u64& m) {
    const unsigned key = ~key_of(x);
    m = 0;
    if (key < last_key || (key == last_key && e <= last_index)) {
      const double w = weight(x, p, lds.table);
      if (w >= (double)min_p || x == p.top) m = units(w);
    }
  };
  float u = a.u[r];
  u = u > 0.f ? (u < 1.f ? u : 0.99999994f) : 0.f;                 // NaN draws as 0
  int from = 0, to = n;
  u64 target = 0;
  for (int level = 0; level < 2; ++level) {
    u64 m = 0;
    for_row(row, from, to, n, wave, waves, lane, [&](int e, const float(&x)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        u64 v;
        kept(e + i, x[i], v);
        m += e + i < to ? v : 0;
      }
    });
    m = wave_sum(m);
    __syncthreads();
    if (lane == 0) lds.part_m[wave] = m;
    __syncthreads();
    if (level == 0) {
      u64 c = 0;
      for (int w = 0; w < waves; ++w) c += lds.part_m[w];
      target = (u64)((double)u * (double)c);
      target = target < c ? target : c - 1;
    }
    const int step = piece(from, to, waves);
    int w = 0;
    u64 before = 0;
    while (w < waves - 1 && before + lds.part_m[w] <= target) before += lds.part_m[w++];
    target -= before;
    const int f = from + w * step;
    to = f + step < to ? f + step : to;
    from = f;
  }
  if (wave == 0) {
    int token = -1;
    for (int e0 = from; e0 < to; e0 += 64) {
      const int e = e0 + lane;
      u64 v = 0;
      if (e < to) kept(e, clean((float)row[e]), v);
      u64 incl = v;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const u64 up = __shfl_up(incl, o);
        if (lane >= o) incl += up;
      }
      const u64 hit = __ballot(incl > target);
      if (hit) {
        token = e0 + __ffsll(hit) - 1;
        break;
      }
      target -= __shfl(incl, 63);
    }
    if (lane == 0) a.tokens[r] = token;
  }
}

}  // namespace

int launch_sample_tokens(int dtype, const SampleArgs& a, hipStream_t stream) {
  if (dtype != DT_BF16 && dtype != DT_F32) return fail("sample_tokens: dtype %d", dtype);
  if (a.rows < 0 || a.vocab < 1 || a.vocab > MAX_VOCAB) return fail("sample_tokens: %d rows, vocabulary %d out of range (1..%d)", a.rows, a.vocab, MAX_VOCAB);
  if (a.rows == 0) return 0;
  if (a.rows > 1 && a.row_stride < a.vocab) return fail("sample_tokens: rows of %d logits overlap (stride %lld)", a.vocab, a.row_stride);
  if (!a.logits || !a.u || !a.tokens) return fail("sample_tokens: null operand");
  if ((uintptr_t)a.logits % (dtype == DT_BF16 ? 2 : 4)) return fail("sample_tokens: logits are not aligned to their type");
  // a wave takes 512 logits at a time: as many waves as have some, in powers of two (the bins divide among them)
  int waves = 1;
  while (waves < MAX_WAVES && waves * 512 < a.vocab) waves *= 2;
  if (dtype == DT_BF16) sample_kernel<bf16><<<a.rows, 64 * waves, 0, stream>>>(a);
  else sample_kernel<float><<<a.rows, 64 * waves, 0, stream>>>(a);
  return check_launch("sample_tokens");
}

}  // namespace fcenc
