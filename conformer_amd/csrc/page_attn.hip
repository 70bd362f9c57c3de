// Attention of a chunk of new rows over a paged key/value cache (gfx950).
//
// Request b brings rows cu_rows[b] .. cu_rows[b + 1] - 1 (n of them) and holds kv = kv_lens[b] tokens, the chunk's own
// among them: its row i sits at position p = kv - n + i and sees the tokens j with
//     j < kv,   causal: j <= p,   window w > 0: j > p - w or j < sinks.
//   out = softmax_j(scale * q . k_j) . v_j;   a row that sees nothing gives zeros.
// Query head h reads kv head h / (heads / kv_heads).  Token j is slot j mod page_size of page table[b][j / page_size]; the
// tokens of a page whose id is outside the pool are seen by nobody.
//
// One pass over the keys with a running maximum m and sum l per row (fp32, base-2 exponents):
//     m' = max(m, max_j s_j),  l' = l 2^(m - m') + sum_j 2^(s_j - m'),  O' = O 2^(m - m') + sum_j 2^(s_j - m') v_j.
// In bf16 p_j = 2^(s_j - m') has to be given to the product with v in bf16.  The kernel of short requests, bound by the bytes of K
// and V, takes it as a sum of two bf16 numbers (good to 2^-15; 64 requests of up to 8192 tokens 257.1 us, 257.4 rounded
// once).  The kernel of chunks and prompts, where a second product for every one of v would be half as much matrix work again,
// rounds it once, and l adds up the rounded ones: what is rounded off in the numerator is then missing in the
// denominator too, and a row that one key dominates loses nothing.
//
// A tile is a set of rows of one (request, kv head): `tt` neighbouring rows of the chunk times the gc query heads that
// share the kv head, so that a key read once serves all of them.  Workgroup t finds its request without any table:
// start(b) = cu_rows[b] / tt + min(b, cu_rows[b]) grows by at least ceil(n / tt) over a request of n rows (n > 0: the second
// term grows by one or more, the first by n / tt rounded down) and never falls, so the request of t is the last one
// with start(b) <= t, and rows / tt + min(B, rows) + 1 workgroups cover every batch, however many requests bring nothing
// (a table of 16384 requests of which 25 bring 64 rows, 32 heads of 128 over 8: 24 ms with B in place of min(B, rows)).
//
// Everything is computed transposed: S^T = K Q^T has the query row on the lane's column and tokens on the accumulator
// rows, and those rows are, as they are, the k elements of the B operand of O^T = V^T P^T once the V fragment is read
// in the same token order.  P never leaves the registers; V^T fragments come out of LDS with transposing reads.
//
// K and V are looked up by 16 tokens (a page holds at least as many).  Of those, what no row of the tile sees (stale slots,
// tokens in front of the window, bad pages, head dims up to the padded width) arrives as zero, so garbage there can reach
// neither the scores nor, as 0 * NaN, the sums: in the step kernel by buffer descriptors that end behind the last token seen,
// in the chunk kernel, which loads straight into LDS, by lanes that read a row of zeros instead.
#include <math.h>

#include "common.h"
#include "kernels.h"

namespace fcenc {

namespace {

constexpr uint32_t OOB = 0xE0000000u;       // an offset outside every descriptor, 16 slots of 2^24 bytes further on as well
constexpr int MAX_SPLITS = 256;
constexpr int STEP_WAVES = 4;
constexpr int STEP_ROWS = 16;
constexpr int CHUNK_ROWS = 128;             // rows of a tile of the chunk kernel
constexpr int CHUNK_MIN = 32;               // requests with more rows (times heads per kv head) than this are its share

// How a launch divides the work.  `share` 0: every request; 1: those of up to CHUNK_MIN rows, `per_request` > 0 rows of
// the chunk at most; 2: the longer ones and the rows behind the last request.
struct Split {
  int gc = 1, hchunks = 1, tt = 1, share = 0, per_request = 0;
  int pieces = 1;                            // of the key axis, at most; the results of more than one go to the workspace from float `ws` on
  int piece = 1 << 30;                       // longest piece, in the kernel's blocks of tokens
  long long ws = 0;
  long long ws_rows = 0;                     // (row, head) pairs there: of every row, or
  bool by_request = false;                   // of per_request rows of every request (share 1, where that is less), which is then also how tiles go
};

// Partial results of a split key axis: (m, l) of every (row, head, piece), then the unnormalised sums.
__device__ __host__ __forceinline__ long long ws_sums(long long rows, int pieces) { return (2 * rows * pieces + 3) & ~3ll; }

// first tile of request b, whose rows begin at c0
__device__ __forceinline__ int first_tile(int b, int c0, int tt) { return c0 / tt + (b < c0 ? b : c0); }

struct TileInfo {
  int b, t0, n, c0, kv;                      // request (B: rows behind the last one), first row, rows, offset, tokens
};

constexpr int STEP_BLOCK = 5, CHUNK_BLOCK = 6;               // log2 of the tokens that the kernels take at a time

// The tokens that some row of a tile sees, [0, sinks) and [lo, hi), as `count` blocks: the first `sb`, then those from `lob` on.
struct Span {
  int first, last, lo, hi, sinks, sb, lob, count;
};
__device__ __forceinline__ Span span_of(const PageAttnArgs& a, const TileInfo& ti, int tt, int log) {
  Span s;
  s.first = ti.kv - ti.n + ti.t0;                            // position of the tile's first row
  s.last = s.first + (ti.n - ti.t0 < tt ? ti.n - ti.t0 : tt) - 1;
  s.hi = a.causal ? s.last + 1 : ti.kv;
  if (ti.b == a.B || s.hi < 0) s.hi = 0;
  s.lo = a.window > 0 && s.first > 0 ? s.first - a.window + 1 : 0;
  s.lo = s.lo < 0 ? 0 : (s.lo > s.hi ? s.hi : s.lo);
  s.sinks = a.window > 0 ? a.sinks : 0;
  const int up = (1 << log) - 1;
  s.lob = s.lo >> log;
  s.sb = ((s.sinks < s.hi ? s.sinks : s.hi) + up) >> log;
  s.sb = s.sb < s.lob ? s.sb : s.lob;
  s.count = s.hi > 0 ? s.sb + ((s.hi + up) >> log) - s.lob : 0;
  return s;
}
// Pieces of a tile's key axis: equal ones, none longer than sp.piece as far as sp.pieces are enough (so a long request does not hold up
// the launch, and a short one needs no join).
__device__ __forceinline__ int pieces_of(const Split& sp, int count) {
  if (sp.pieces == 1) return 1;
  const int n = (count + sp.piece - 1) / sp.piece;
  return n < 1 ? 1 : (n > sp.pieces ? sp.pieces : n);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int clamp_rows(int v, int rows) { return v < 0 ? 0 : (v > rows ? rows : v); }

// false: no such tile, or not of this launch's share
__device__ __forceinline__ bool find_tile(const PageAttnArgs& a, int tile, const Split& sp, TileInfo& ti) {
  const int tt = sp.tt;
  int lo = 0, c0, c1, kv;
  if (sp.by_request) {                         // as many tiles for every request
    const int each = (sp.per_request + tt - 1) / tt;
    lo = tile / each;
    c0 = clamp_rows(uniform(a.cu_rows[lo]), a.rows);
    c1 = clamp_rows(uniform(a.cu_rows[lo + 1]), a.rows);
    kv = uniform(a.kv_lens[lo]);
    tile = tile - lo * each + first_tile(lo, c0, tt);
  } else {
    // 64 candidates at a time, their lengths along with the last ones: one memory latency for up to 63 requests, two for up to
    // 4095
    const int lane = threadIdx.x & 63;
    int hi = a.B + 1, k = 0, start = 0, length = 0, step;
    do {                                       // the last trip looks at neighbours, also where one candidate was left
      step = (hi - lo + 63) >> 6;
      const int b = lo + lane * step;
      if (b <= a.B) start = clamp_rows(a.cu_rows[b], a.rows);
      if (step == 1 && b < a.B) length = a.kv_lens[b];
      k = __popcll(__ballot(b < hi && first_tile(b, start, tt) <= tile)) - 1;     // starts rise with b
      k = k > 0 ? k : 0;
      lo = lo + k * step;
      hi = hi < lo + step ? hi : lo + step;
    } while (step > 1);
    k = uniform(k);
    lo = uniform(lo);
    c0 = __builtin_amdgcn_readlane(start, k);
    kv = __builtin_amdgcn_readlane(length, k);
    c1 = lo == a.B ? a.rows : k < 63 ? __builtin_amdgcn_readlane(start, k + 1) : clamp_rows(uniform(a.cu_rows[lo + 1]), a.rows);
  }
  ti.b = lo;
  ti.c0 = c0;
  ti.n = c1 - c0;
  ti.t0 = (tile - first_tile(lo, c0, tt)) * tt;
  ti.kv = 0;
  if (ti.t0 < 0 || ti.t0 >= ti.n) return false;
  if (sp.share == 1 && ti.n > sp.per_request) return false;
  if (sp.share == 2 && lo < a.B && ti.n <= sp.per_request) return false;
  if (lo < a.B) {
    const int cap = a.width << a.shift;
    ti.kv = kv < 0 ? 0 : (kv > cap ? cap : kv);
  }
  return true;
}

// where the partial results of a (row of request b, head) lie
__device__ __forceinline__ long long ws_row(const PageAttnArgs& a, const Split& sp, const TileInfo& ti, int row, int head) {
  return (sp.by_request ? (long long)ti.b * sp.per_request + row : (long long)ti.c0 + row) * a.heads + head;
}

// V^T fragment of a [32 tokens][DP] tile in LDS: element j of lane (g, r) is V[token 16 (j >> 2) + 4 g + (j & 3)][dim 16 db + r]
template <int ROWB>
__device__ __forceinline__ bf16x8 v_frag(const char* vt, int db, int g, int r, bf16) {
  using lds_bf16x4 = __attribute__((address_space(3))) bf16x4;
  bf16x8 f;
#pragma unroll
  for (int hi = 0; hi < 2; ++hi) {
    const int key = 16 * hi + 4 * g + (r >> 2);
    const char* p = vt + tile_off<ROWB>(key, 2 * db + ((r & 3) >> 1)) + 8 * (r & 1);
    const bf16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(p));
#pragma unroll
    for (int q = 0; q < 4; ++q) f[4 * hi + q] = v[q];
  }
  return f;
}
template <int ROWB>
__device__ __forceinline__ f32x8 v_frag(const char* vt, int db, int g, int r, float) {
  f32x8 f;
  const int dv = 16 * db + r;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int key = 16 * (j >> 2) + 4 * g + (j & 3);
    const float v = *reinterpret_cast<const float*>(vt + tile_off<ROWB>(key, dv >> 2) + 4 * (dv & 3));
    if (j < 4) f.lo[j] = v; else f.hi[j - 4] = v;
  }
  return f;
}
__device__ __forceinline__ bf16x8 p_frag(const float (&x)[8], bf16) {
  bf16x8 f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (bf16)x[i];
  return f;
}
__device__ __forceinline__ f32x8 p_frag(const float (&x)[8], float) {
  f32x8 f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f.lo[i] = x[i];
    f.hi[i] = x[4 + i];
  }
  return f;
}

// sum of a fragment's eight elements on top of l
__device__ __forceinline__ float add_frag(float l, const f32x8& f) {
  return l + (((f.lo[0] + f.lo[1]) + (f.lo[2] + f.lo[3])) + ((f.hi[0] + f.hi[1]) + (f.hi[2] + f.hi[3])));
}

// eight elements of a row through a descriptor
__device__ __forceinline__ bf16x8 load_frag(__amdgpu_buffer_rsrc_t r, uint32_t off, bf16) {
  return __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}
__device__ __forceinline__ f32x8 load_frag(__amdgpu_buffer_rsrc_t r, uint32_t off, float) {
  f32x8 f;
  f.lo = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
  f.hi = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 16, 0));
  return f;
}

__device__ __forceinline__ void store_row(bf16* p, float v) { *p = (bf16)v; }
__device__ __forceinline__ void store_row(float* p, float v) { *p = v; }

// ---------------------------------------------------------------------------------------------------------------
// Tiles of up to 16 rows: single tokens and short chunks.  Bound by the bytes of K and V.  The four waves of a workgroup
// take every fourth block of 32 tokens, on their own (K straight into MFMA fragments, V through a wave-private LDS
// tile), with the next block's loads in flight; their partial results meet in LDS.  With few tiles the key axis is
// also cut into `splits` pieces, whose results a second launch joins.  64 requests of up to 8192 tokens, 8 kv heads of 128 in
// bf16 under 32 heads: 257 us, 5.4 TB/s of K and V (a large copy reaches 5.2); 2 of up to 131072 over 4 kv heads: 75 us.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int DP>
struct StepTile {
  static constexpr int ROWB = DP * (int)sizeof(T);
  static constexpr int CPR = ROWB / 16;                     // 16-byte pieces of a row
  static constexpr int OROW = DP + 4;                       // floats per row of the merge buffer
  static constexpr int WAVE_BYTES = 32 * ROWB > STEP_ROWS * OROW * 4 ? 32 * ROWB : STEP_ROWS * OROW * 4;
  static constexpr int BYTES = STEP_WAVES * WAVE_BYTES + STEP_WAVES * STEP_ROWS * 8;
};

template <typename T, int DP>
__device__ __forceinline__ void step_tile(const PageAttnArgs& a, const Split& sp, unsigned block, char* smem) {
  using TL = StepTile<T, DP>;
  using Frag = typename Traits<T>::Frag;
  constexpr int ROWB = TL::ROWB, CPR = TL::CPR, ES = (int)sizeof(T);
  constexpr int KS = DP / 32, NDB = DP / 16, NV = CPR / 4;   // k32 steps, 16-dim blocks, V loads per 16 tokens
  constexpr int RPI = 64 / CPR;                              // V rows per load instruction
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int gc = sp.gc, tt = sp.tt;
  // pieces fastest, tiles slowest: workgroups go round the 8 XCDs by their number, and with the tile (of which some are
  // empty) in front, a batch of two requests left half of the XCDs without work (146 against 77 us at 2 x 131072 tokens)
  const unsigned per_tile = a.kv_heads * sp.hchunks * sp.pieces;
  const int tile = (int)(block / per_tile);
  const int rest = (int)(block - tile * per_tile), column = rest / sp.pieces, split = rest - column * sp.pieces;
  const int kvh = column / sp.hchunks, hc = column - kvh * sp.hchunks;
  const int group = a.heads / a.kv_heads;

  TileInfo ti;
  if (!find_tile(a, tile, sp, ti)) return;
  const Span at_tile = span_of(a, ti, tt, STEP_BLOCK);
  const int first = at_tile.first, last = at_tile.last, lo = at_tile.lo, hi = at_tile.hi, sinks = at_tile.sinks;
  const int sb = at_tile.sb, lob = at_tile.lob, count = at_tile.count, pieces = pieces_of(sp, count);
  if (split >= pieces) return;
  const int i0 = (int)((long long)count * split / pieces), i1 = (int)((long long)count * (split + 1) / pieces);

  // this lane's row of the tile
  const int rt = r / gc, rh = hc * gc + r - rt * gc;
  const bool live = rt < tt && ti.t0 + rt < ti.n && rh < group;
  const int pos = first + rt;
  const int see_hi = a.causal ? pos : ti.kv - 1;             // last token it sees
  const int see_lo = a.window > 0 && pos > 0 ? pos - a.window + 1 : 0;  // first one, next to the sinks
  Frag q[KS];
  {
    const char* qrow = a.q + (long long)(ti.c0 + ti.t0 + (live ? rt : 0)) * a.q_row + (long long)(kvh * group + (live ? rh : 0)) * a.q_head;
    const __amdgpu_buffer_rsrc_t none = buffer_of(nullptr, 0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      q[ks] = load_frag(none, OOB, T{});
      if (live && 32 * ks + 8 * g < a.dim) q[ks] = *reinterpret_cast<const Frag*>(qrow + (32 * ks + 8 * g) * ES);
    }
  }

  f32x4 ot[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i) ot[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;
  const float c = a.scale * kLog2e;
  char* vt = smem + wave * TL::WAVE_BYTES;
  const int32_t* trow = a.table + (long long)(ti.b < a.B ? ti.b : 0) * a.table_row;
  const char* kbase = a.k + kvh * a.k_head;
  const char* vbase = a.v + kvh * a.v_head;

  Frag kf[2][KS];
  u32x4 vr[2][NV];
  bool page_ok[2];
  auto block_of = [&](int i) { return i < sb ? i : lob + i - sb; };
  // of the block to fetch next, so that its loads need not wait for the table; left in vector registers until then (made
  // uniform here, the wait for them would also wait for the K and V loads in front of them)
  int pages[2];
  auto find_pages = [&](int i) {
    const int j0 = block_of(i) * 32;
#pragma unroll
    for (int t = 0; t < 2; ++t) pages[t] = i < i1 && j0 + 16 * t < hi ? trow[(j0 + 16 * t) >> a.shift] : -1;
  };
  // descriptors of the 16 tokens from tok0 on: bytes up to the last one that the tile sees
  auto fetch = [&](int i) {
    const int j0 = block_of(i) * 32;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int tok0 = j0 + 16 * t;
      int left = hi - tok0;
      left = left > 16 ? 16 : left;
      const int page = uniform(pages[t]);
      const bool ok = (page >= 0) & (page < a.n_pages) & (left > 0);
      page_ok[t] = ok | (left <= 0);
      const int slot0 = tok0 & ((1 << a.shift) - 1);
      const char* kp = kbase + (long long)(ok ? page : 0) * a.k_page + (long long)slot0 * a.k_slot;
      const char* vp = vbase + (long long)(ok ? page : 0) * a.v_page + (long long)slot0 * a.v_slot;
      const __amdgpu_buffer_rsrc_t kd = buffer_of(kp, ok ? (left - 1) * a.k_slot + a.dim * ES : 0);
      const __amdgpu_buffer_rsrc_t vd = buffer_of(vp, ok ? (left - 1) * a.v_slot + a.dim * ES : 0);
      // tokens in front of the window and behind the sinks are seen by no row of the tile
      const bool dead_k = (tok0 + r < lo) & (tok0 + r >= sinks);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d0 = 32 * ks + 8 * g;
        kf[t][ks] = load_frag(kd, (dead_k | (d0 >= a.dim)) ? OOB : (uint32_t)(r * a.k_slot + d0 * ES), T{});
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int row = lane / CPR + v * RPI, ch = lane % CPR;
        const bool dead_v = (tok0 + row < lo) & (tok0 + row >= sinks);
        vr[t][v] = __builtin_amdgcn_raw_buffer_load_b128(vd, (int)((dead_v | (ch * 16 >= a.dim * ES)) ? OOB : (uint32_t)(row * a.v_slot + ch * 16)), 0, 0);
      }
    }
  };

  int i = i0 + wave;
  find_pages(i);
  if (i < i1) fetch(i);
  find_pages(i + STEP_WAVES);
  for (; i < i1; i += STEP_WAVES) {
    const int j0 = block_of(i) * 32;
    const bool ok0 = page_ok[0], ok1 = page_ok[1];
    // ---- S^T = K Q^T: lane (g, r), register e of tile t: token j0 + 16 t + 4 g + e, row r ----
    f32x4 st[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) mma(st[t], kf[t][ks], q[ks]);
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");         // the tile of the block before has been read
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int v = 0; v < NV; ++v)
        *reinterpret_cast<u32x4*>(vt + tile_off<ROWB>(16 * t + lane / CPR + v * RPI, lane % CPR)) = vr[t][v];
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    if (i + STEP_WAVES < i1) {
      fetch(i + STEP_WAVES);
      find_pages(i + 2 * STEP_WAVES);
    }

    bool inside = ok0 && ok1 && j0 + 31 <= (a.causal ? first : ti.kv - 1);
    if (a.window > 0) inside = inside && (j0 >= last - a.window + 1 || j0 + 31 < sinks);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float s = st[t][e] * c;
        if (!inside) {
          const int j = j0 + 16 * t + 4 * g + e;
          const bool see = (t ? ok1 : ok0) && j <= see_hi && (j >= see_lo || j < sinks);
          s = see ? s : -INFINITY;
        }
        st[t][e] = s;
      }
    float tmax = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) tmax = fmaxf(tmax, st[t][e]);
    const float m_new = fmaxf(m_run, rows4_max(tmax));
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
    m_run = m_new;
    float pk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) pk[e] = __builtin_amdgcn_exp2f(st[e >> 2][e & 3] - m_use);
    l_run = l_run * alpha + (((pk[0] + pk[1]) + (pk[2] + pk[3])) + ((pk[4] + pk[5]) + (pk[6] + pk[7])));
    // bf16: p as the sum of two bf16 numbers.  The first is the largest one below p, so that the second is above 0 as well, and
    // an infinite v gives infinity as it does with p itself; 0 stays 0.
    float ph[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ph[e] = pk[e];
      if constexpr (sizeof(T) == 2) {
        const int below = __builtin_bit_cast(int, pk[e]) - 1;
        ph[e] = __builtin_bit_cast(float, (below > 0 ? below : 0) & 0xffff0000);
        pk[e] -= ph[e];
      }
    }
    const Frag pf = p_frag(ph, T{}), pr = p_frag(pk, T{});
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      ot[db] *= alpha;
      const Frag vf = v_frag<ROWB>(vt, db, g, r, T{});
      mma(ot[db], vf, pf);
      if constexpr (sizeof(T) == 2) mma(ot[db], vf, pr);
    }
  }

  // ---- the four waves' results ----
  l_run = rows4_sum(l_run);
  float* ob = reinterpret_cast<float*>(vt);
  float2* ml = reinterpret_cast<float2*>(smem + STEP_WAVES * TL::WAVE_BYTES);
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int db = 0; db < NDB; ++db) *reinterpret_cast<f32x4*>(ob + r * TL::OROW + 16 * db + 4 * g) = ot[db];
  if (g == 0) ml[wave * STEP_ROWS + r] = float2{m_run, l_run};
  __syncthreads();
  constexpr int DPT = DP / 16;                              // dims per thread: 16 threads a row
  const int row = tid >> 4, d0 = (tid & 15) * DPT;
  const int ort = row / gc, orh = hc * gc + row - ort * gc;
  if (!(ort < tt && ti.t0 + ort < ti.n && orh < group)) return;
  float m = -INFINITY, l = 0.f, acc[DPT];
#pragma unroll
  for (int w = 0; w < STEP_WAVES; ++w) m = fmaxf(m, ml[w * STEP_ROWS + row].x);
#pragma unroll
  for (int d = 0; d < DPT; ++d) acc[d] = 0.f;
#pragma unroll
  for (int w = 0; w < STEP_WAVES; ++w) {
    const float2 p = ml[w * STEP_ROWS + row];
    if (p.y == 0.f) continue;                                // nothing seen by that wave
    const float f = __builtin_amdgcn_exp2f(p.x - m);
    l += p.y * f;
    const float* src = reinterpret_cast<const float*>(smem + w * TL::WAVE_BYTES) + row * TL::OROW + d0;
#pragma unroll
    for (int d = 0; d < DPT; ++d) acc[d] += src[d] * f;
  }
  const long long orow = (long long)(ti.c0 + ti.t0 + ort) * a.heads + kvh * group + orh;
  if (pieces == 1) {
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);       // NaN stays NaN
    T* o = reinterpret_cast<T*>(a.out) + orow * a.dim;
#pragma unroll
    for (int d = 0; d < DPT; ++d)
      if (d0 + d < a.dim) store_row(o + d0 + d, acc[d] * inv);
  } else {
    const long long at = ws_row(a, sp, ti, ti.t0 + ort, kvh * group + orh) * sp.pieces + split;
    float* o = a.ws + sp.ws + ws_sums(sp.ws_rows, sp.pieces) + at * a.dim;
#pragma unroll
    for (int d = 0; d < DPT; ++d)
      if (d0 + d < a.dim) o[d0 + d] = acc[d];
    if ((tid & 15) == 0) reinterpret_cast<float2*>(a.ws + sp.ws)[at] = float2{m, l};
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(64 * STEP_WAVES, (StepTile<T, DP>::ROWB > 256 ? 1 : 2))
    page_attn_step_kernel(const PageAttnArgs a, const Split sp) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  step_tile<T, DP>(a, sp, blockIdx.x, lds);
}

// ---------------------------------------------------------------------------------------------------------------
// Tiles of up to 128 rows: chunks and prompts.  Four waves of 32 rows share each K / V tile of 64 tokens through LDS;
// 32x32 MFMAs, so a wave reads a fragment once for 32 rows and a row's statistics need one exchange between the two
// halves of the wave.  Tiles go from memory straight into LDS (wave w: tokens 16 w .. 16 w + 15, one page lookup), two of each
// in flight or in use, K a tile ahead of V: the products for tile i + 1's scores stand beside tile i's exponentials.
// Bound by the matrix and vector units together: at 128 head dims they are busy 57 and 49 % of the cycles, and what one wave
// needs of one the other wave of the SIMD must leave.  3 prompts of up to 8192 rows, 32 heads of 128 over 8, window 4096:
// 0.87 ms, 1016 TFLOP/s in bf16, where a large matrix product reaches 1320; 2 of up to 2048 rows, 16 heads, in fp32 77 (143).
//
// C layout of a 32x32 product: lane (h = lane / 32, c = lane % 32), register i: row 8 (i / 4) + 4 h + i % 4, column c.  With
// rows = tokens, registers 8 s .. 8 s + 7 are the eight tokens {4 h + 0..3, 8 + 4 h + 0..3} of 16-token step s: the k
// elements of lane half h of the next product, whose V^T fragment is read in that order.
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma32(f32x16& acc, const bf16x8& a, const bf16x8& b) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma32(f32x16& acc, const f32x8& a, const f32x8& b) {
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.lo[j], b.lo[j], acc, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.hi[j], b.hi[j], acc, 0, 0, 0);
}

template <typename T, int DP>
struct ChunkTile {
  static constexpr int ROWB = DP * (int)sizeof(T);
  static constexpr int CPR = ROWB / 16;
  static constexpr int KT = 64;                                  // tokens of a tile
  static constexpr int TILE = KT * ROWB;
  static constexpr int V_OFF = 2 * TILE;                         // two K tiles, two V tiles; all at multiples of 256: see lds_at
  static constexpr int BYTES = 4 * TILE;
};

// Where 16-byte piece `ch` of row `row` lies, so that reads spread over the 256 bytes of the 64 LDS banks.  K: 16 rows that are
// read at one piece hit 16 different ones.  V: a transposing read takes 4 rows x 32 bytes per 16 lanes, 64 bytes per 32
// lanes, rows 4 apart in the wave's other half.
template <int ROWB>
__device__ __forceinline__ uint32_t k_off(int row, int ch) {
  return (uint32_t)(row * ROWB + ((ch ^ (ROWB >= 256 ? row & 15 : (row >> 1) & 7)) << 4));
}
template <int ROWB>
__device__ __forceinline__ uint32_t v_off(int row, int ch, bf16) {
  const int x = ROWB >= 256 ? (row & 3) << 2 : (row & 2) << 1;
  return (uint32_t)(row * ROWB + ((ch ^ (x | (row >> 1 & 2))) << 4));
}
template <int ROWB>
__device__ __forceinline__ uint32_t v_off(int row, int ch, float) { return k_off<ROWB>(row, ch); }

// Tile addresses are formed as (what belongs to the lane) xor (a constant per fragment): rows are 128, 256 or 512 bytes, chunk
// bits lie below them, and a tile starts at a multiple of 256.  One register per tile instead of one per fragment.
template <typename V>
__device__ __forceinline__ V lds_at(uint32_t addr) {
  using LV = const __attribute__((address_space(3))) V;
  return *(LV*)(uintptr_t)addr;
}
// k_lane: address of chunk h (bf16) or 2 h (fp32) of token c; the fragment of step ks of token 32 t + c
template <int ROWB>
__device__ __forceinline__ bf16x8 k_frag32(uint32_t k_lane, int t, int ks, bf16) {
  return lds_at<bf16x8>((k_lane ^ (uint32_t)(ks << 5)) + t * 32 * ROWB);
}
template <int ROWB>
__device__ __forceinline__ f32x8 k_frag32(uint32_t k_lane, int t, int ks, float) {
  f32x8 f;
  f.lo = lds_at<f32x4>((k_lane ^ (uint32_t)(ks << 6)) + t * 32 * ROWB);
  f.hi = lds_at<f32x4>((k_lane ^ (uint32_t)(ks << 6) ^ 16u) + t * 32 * ROWB);
  return f;
}
// V^T of dims 32 dt .. + 31, 16-token step s: element j of lane (h, c) is V[16 s + 8 (j >> 2) + 4 h + (j & 3)][32 dt + c].
// v_lane (bf16): address of this lane's 8 bytes of step 0, dims 0 .. 31.
template <int ROWB>
__device__ __forceinline__ bf16x8 v_frag32(uint32_t v_lane, int dt, int s, int lane, bf16) {
  using lds_bf16x4 = __attribute__((address_space(3))) bf16x4;
  bf16x8 f;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const bf16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(uintptr_t)((v_lane ^ (uint32_t)(dt << 6)) + (16 * s + 8 * u) * ROWB));
#pragma unroll
    for (int q = 0; q < 4; ++q) f[4 * u + q] = v[q];
  }
  return f;
}
template <int ROWB>
__device__ __forceinline__ f32x8 v_frag32(uint32_t v_tile, int dt, int s, int lane, float) {
  const int h = lane >> 5, d = 32 * dt + (lane & 31);
  f32x8 f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int key = 16 * s + 8 * (j >> 2) + 4 * h + (j & 3);
    const float v = lds_at<float>(v_tile + v_off<ROWB>(key, d >> 2, float{}) + 4 * (d & 3));
    if (j < 4) f.lo[j] = v; else f.hi[j - 4] = v;
  }
  return f;
}

// 16 bytes per lane from memory to 1 KiB of LDS at `dst`, lane after lane, without a register on the way.  Written as
// assembly because the compiler, which cannot tell the LDS tiles apart, would wait for such a load before every LDS
// read; nothing but lds_loads_done and the barrier behind it says that the data is there.  There is no result register that
// could be written late; the s_nop is the wait state between a write of m0 and its use here.
__device__ __forceinline__ void lds_load16(uint32_t dst, const char* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void lds_load16(uint32_t dst, const char* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory");
}
// N of them, to `dst` + 1024 v.  The offset in the instruction counts for both addresses (and reaches 4095), so load v's
// `off` is what its 16 bytes are away from base + 1024 (v % 4).
template <int N>
__device__ __forceinline__ void lds_loads(uint32_t dst, const char* base, const uint32_t (&off)[N]) {
  static_assert(N == 2 || N % 4 == 0, "pairs or fours");
  if constexpr (N == 2) {
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 1\n\t"
        "global_load_lds_dwordx4 %1, %3\n\t"
        "global_load_lds_dwordx4 %2, %3 offset:0x400" ::"s"(dst), "v"(off[0]), "v"(off[1]), "s"(base) : "memory");
  } else {
#pragma unroll
    for (int v = 0; v < N; v += 4)
      asm volatile(
          "s_mov_b32 m0, %0\n\ts_nop 1\n\t"
          "global_load_lds_dwordx4 %1, %5\n\t"
          "global_load_lds_dwordx4 %2, %5 offset:0x400\n\t"
          "global_load_lds_dwordx4 %3, %5 offset:0x800\n\t"
          "global_load_lds_dwordx4 %4, %5 offset:0xc00"
          ::"s"(dst + v * 1024), "v"(off[v]), "v"(off[v + 1]), "v"(off[v + 2]), "v"(off[v + 3]), "s"(base) : "memory");
  }
}
__device__ __forceinline__ void lds_loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ const u32x4 zero16 = {0, 0, 0, 0};

// Sum of a lane's p.  bf16: as products of 4x4x4 blocks with ones, in which a lane's four elements meet no other lane's: 16
// cycles of the matrix unit for eight tokens instead of 64 of the vector unit (64 head dims 883 -> 834 us, 128: 1106 -> 1099, over
// prompts of 8192 tokens).
template <typename T>
struct RowSum {
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(const bf16x8& p) {
    using i16x4 = __attribute__((ext_vector_type(4))) short;
    using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
    const i16x4 ones = {0x3f80, 0x3f80, 0x3f80, 0x3f80};
    const u32x4 x = __builtin_bit_cast(u32x4, p);
    acc = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(ones, __builtin_bit_cast(i16x4, u32x2{x[0], x[1]}), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(ones, __builtin_bit_cast(i16x4, u32x2{x[2], x[3]}), acc, 0, 0, 0);
  }
  __device__ __forceinline__ void scale(float f) { acc *= f; }
  __device__ __forceinline__ float of_lane() const { return acc[0]; }
};
template <>
struct RowSum<float> {
  float acc = 0.f;
  __device__ __forceinline__ void add(const f32x8& p) { acc = add_frag(acc, p); }
  __device__ __forceinline__ void scale(float f) { acc *= f; }
  __device__ __forceinline__ float of_lane() const { return acc; }
};

// DP: head dims of a row in LDS (64 or 128), DC <= DP: those that are multiplied
template <typename T, int DP, int DC>
__device__ __forceinline__ void chunk_tile(const PageAttnArgs& a, const Split& sp, unsigned block, unsigned blocks, char* tiles) {
  using TL = ChunkTile<T, DP>;
  using Frag = typename Traits<T>::Frag;
  constexpr int ROWB = TL::ROWB, CPR = TL::CPR, ES = (int)sizeof(T);
  constexpr int KS = DC / 16, NDT = DC / 32, NL = CPR / 4, RPI = 64 / CPR;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int h = lane >> 5, c = lane & 31;
  // workgroups of one kv head are dispatched to one XCD where the number of kv heads allows it (their tiles read the same
  // keys), long tiles (the late rows of a causal chunk) first
  const int columns = a.kv_heads * sp.hchunks;
  const int split = (int)(block / blocks);
  block -= split * blocks;
  const int tile = (int)((blocks - 1 - block) / columns), column = (int)(block % columns);
  const int kvh = column / sp.hchunks, hc = column - kvh * sp.hchunks;
  const int gc = sp.gc, tt = sp.tt;
  const int group = a.heads / a.kv_heads;

  TileInfo ti;
  if (!find_tile(a, tile, sp, ti)) return;
  const Span at_tile = span_of(a, ti, tt, CHUNK_BLOCK);
  const int first = at_tile.first, lo = at_tile.lo, hi = at_tile.hi, sinks = at_tile.sinks;
  const int sb = at_tile.sb, lot = at_tile.lob, count = at_tile.count, pieces = pieces_of(sp, count);
  if (split >= pieces) return;
  const int live_tt = at_tile.last - first + 1;
  const int i0 = (int)((long long)count * split / pieces), i1 = (int)((long long)count * (split + 1) / pieces);

  // this lane's row and this wave's rows
  const int R = 32 * wave + c;
  const int rt = R / gc, rh = hc * gc + R - rt * gc;
  const bool live = rt < live_tt && rh < group;
  const int pos = first + rt;
  const int see_hi = a.causal ? pos : ti.kv - 1;
  const int see_lo = a.window > 0 && pos > 0 ? pos - a.window + 1 : 0;
  const int wt0 = (32 * wave) / gc;
  int wt1 = (32 * wave + 31) / gc;
  wt1 = wt1 < live_tt - 1 ? wt1 : live_tt - 1;
  const bool busy = wt0 <= wt1;
  const int wfirst = first + wt0, wlast = first + wt1;       // positions of the wave's first and last row

  Frag q[KS];
  {
    const char* qrow = a.q + (long long)(ti.c0 + ti.t0 + (live ? rt : 0)) * a.q_row + (long long)(kvh * group + (live ? rh : 0)) * a.q_head;
    const __amdgpu_buffer_rsrc_t none = buffer_of(nullptr, 0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      q[ks] = load_frag(none, OOB, T{});
      if (live && 16 * ks + 8 * h < a.dim) q[ks] = *reinterpret_cast<const Frag*>(qrow + (16 * ks + 8 * h) * ES);
    }
  }

  f32x16 ot[NDT];
#pragma unroll
  for (int i = 0; i < NDT; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) ot[i][e] = 0.f;
  float m_run = -INFINITY;                                   // m in units of the raw scores
  RowSum<T> l_run;
  const float cs = a.scale * kLog2e;
  const int32_t* trow = a.table + (long long)(ti.b < a.B ? ti.b : 0) * a.table_row;
  const char* kbase = a.k + kvh * a.k_head;
  const char* vbase = a.v + kvh * a.v_head;

  const uint32_t lds0 = (uint32_t)(uintptr_t)tiles;
  auto start_of = [&](int i) { return (i < sb ? i : lot + i - sb) * 64; };   // first token of tile i
  // Lane l: the page of tokens 16 (l % 4) .. + 15 of a tile (behind hi: that of the last token; nobody looks at it).  Left in a
  // vector register until it is needed: made uniform at once, the wait for it would also wait for the loads in front of it.
  auto pages_of = [&](int start) {
    const int tok = start + 16 * (lane & 3);
    return *reinterpret_cast<const int32_t*>(reinterpret_cast<const char*>(trow) + (uint32_t)((tok < hi ? tok : hi - 1) >> a.shift) * 4u);
  };
  // Where lane l's 16 bytes of load v come from: LDS position l % CPR of row v RPI + l / CPR holds another piece of that row.
  // Less 1024 (v % 4): see lds_loads.  (A slot is at least as long as an LDS row when the loads below use that, so this is
  // not negative.)
  uint32_t koff[NL], voff[NL];
  uint32_t alive = 0;                                        // bit v: load v of K holds head dims; bit 8 + v: of V
#pragma unroll
  for (int v = 0; v < NL; ++v) {
    const int row = v * RPI + lane / CPR;
    const uint32_t kp = k_off<ROWB>(row, lane % CPR) - row * ROWB, vp = v_off<ROWB>(row, lane % CPR, T{}) - row * ROWB;
    koff[v] = (uint32_t)(row * a.k_slot) + kp;
    voff[v] = (uint32_t)(row * a.v_slot) + vp;
    if (a.dim == DP) {
      koff[v] -= 1024 * (v % 4);
      voff[v] -= 1024 * (v % 4);
    }
    alive |= (uint32_t)((int)kp < a.dim * ES) << v | (uint32_t)((int)vp < a.dim * ES) << (8 + v);
  }
  // this wave's 16 tokens of a tile whose tokens all are within [lo, hi): tok0 - lo < whole
  const uint32_t whole = hi - 15 > lo ? hi - 15 - lo : 0;
  // K or V of this wave's 16 tokens from tok0 on into LDS
  auto fetch = [&](uint32_t lds_tile, int tok0, bool good, const char* src, const uint32_t (&off)[NL], uint32_t live) {
    const uint32_t dst = lds_tile + 16 * wave * ROWB;
    if (good & ((uint32_t)(tok0 - lo) < whole)) {
      if (a.dim == DP) {
        lds_loads(dst, src, off);
      } else {                                               // the other lanes' bytes are zero from the start
#pragma unroll
        for (int v = 0; v < NL; ++v)
          if (live >> v & 1) lds_load16(dst + v * 1024, src, off[v]);
      }
    } else {                                                 // what nobody sees comes from a row of zeros
#pragma unroll
      for (int v = 0; v < NL; ++v) {
        const int row = v * RPI + lane / CPR, j = tok0 + row;
        const bool dead = !good | (j >= hi) | ((j < lo) & (j >= sinks)) | !(live >> v & 1);
        lds_load16(dst + v * 1024, dead ? reinterpret_cast<const char*>(&zero16) : src + off[v] + (a.dim == DP ? 1024 * (v % 4) : 0));
      }
    }
  };
  // What is known of a tile on its way: its first token, which of its four pages exist, and where this wave's part of V is
  struct Coming { int start; uint32_t ok; const char* v; };
  auto fetch_v = [&](int buf, const Coming& t) {
    fetch(lds0 + TL::V_OFF + buf * TL::TILE, t.start + 16 * wave, t.ok >> wave & 1, t.v, voff, alive >> 8);
  };
  auto fetch_k = [&](int buf, int start, int pages) {
    Coming t;
    t.start = start;
    t.ok = (uint32_t)__ballot((unsigned)pages < (unsigned)a.n_pages) & 15u;
    const bool good = t.ok >> wave & 1;
    const uint32_t page = good ? __builtin_amdgcn_readlane(pages, wave) : 0, slot0 = (start + 16 * wave) & ((1 << a.shift) - 1);
    t.v = vbase + page * (unsigned long long)(uint32_t)a.v_page + slot0 * (uint32_t)a.v_slot;
    fetch(lds0 + buf * TL::TILE, start + 16 * wave, good, kbase + page * (unsigned long long)(uint32_t)a.k_page + slot0 * (uint32_t)a.k_slot, koff, alive);
    return t;
  };
  const uint32_t k_lane = lds0 + k_off<ROWB>(c, sizeof(T) == 2 ? h : 2 * h);
  uint32_t v_lane = lds0 + TL::V_OFF;
  if constexpr (sizeof(T) == 2) {
    const int r = lane & 15;
    v_lane += v_off<ROWB>(4 * h + (r >> 2), 2 * ((lane >> 4) & 1) + ((r & 3) >> 1), T{}) + 8 * (r & 1);
  }
  if (a.dim != DP) {                                         // head dims up to the padded width stay zero
    for (int o = tid * 16; o < TL::BYTES; o += 256 * 16) *reinterpret_cast<u32x4*>(tiles + o) = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  // tiles of this wave that need no mask: all pages exist, last token <= in_hi, first one >= in_lo or last one < sinks
  const int in_hi = a.causal ? wfirst : ti.kv - 1, in_lo = a.window > 0 ? wlast - a.window + 1 : 0;

  // Tile i + 1's scores are formed beside tile i's softmax: the products of one fill the time that the exponentials of the
  // other take.  K therefore runs a tile ahead of V.
  f32x16 s[2];
  Coming t0{0, 0, vbase}, t1{0, 0, vbase};                   // tile i and tile i + 1
  int pages = 0;                                             // of tile i + 2
  if (i0 < i1) {
    const int first_pages = pages_of(start_of(i0)), second_pages = pages_of(start_of(i0 + 1));
    t0 = fetch_k(0, start_of(i0), first_pages);
    fetch_v(0, t0);
    if (i0 + 1 < i1) t1 = fetch_k(1, start_of(i0 + 1), second_pages);
    pages = pages_of(start_of(i0 + 2));
    lds_loads_done();
    __syncthreads();
    if (busy) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[t][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) mma32(s[t], k_frag32<ROWB>(k_lane, t, ks, T{}), q[ks]);
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);    // vmcnt(0): q has arrived, said once, or every first product in the loop would wait for the tiles on their way
  for (int i = i0; i < i1; ++i) {
    const int cur = (i - i0) & 1;
    lds_loads_done();
    __syncthreads();                                         // K of tile i + 1 and V of tile i are in place
    Coming t2 = t1;
    if (i + 2 < i1) t2 = fetch_k(cur, start_of(i + 2), pages);
    if (i + 1 < i1) fetch_v(cur ^ 1, t1);
    pages = pages_of(start_of(i + 3));
    if (busy) {
      const int j0 = t0.start;
      const uint32_t kl = k_lane + (cur ^ 1) * TL::TILE, vl = v_lane + cur * TL::TILE;
      constexpr int RING = sizeof(T) == 2 ? 4 : 1, NX = 4 * NDT;                  // fragments on their way: RING products ahead
      Frag kf[RING], vf[RING];
#pragma unroll
      for (int x = 0; x < RING; ++x) {
        kf[x] = k_frag32<ROWB>(kl, x / KS, x % KS, T{});
        vf[x] = v_frag32<ROWB>(vl, x % NDT, x / NDT, lane, T{});
      }
      const bool inside = (t0.ok == 15) & (j0 + 63 <= in_hi) & ((j0 >= in_lo) | (j0 + 63 < sinks));
      if (!inside) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int j = j0 + 32 * t + 8 * (e >> 2) + 4 * h + (e & 3);
            const bool see = (t0.ok >> (2 * t + (e >> 3)) & 1) & (j <= see_hi) & ((j >= see_lo) | (j < sinks));
            s[t][e] = see ? s[t][e] : -INFINITY;
          }
      }
      float tmax = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) tmax = fmaxf(tmax, s[t][e]);
      {
        float x, y;
        swap_halves32(tmax, x, y);
        tmax = fmaxf(x, y);
      }
      // The reference point of the exponents follows the maximum only when it lags by more than 2^8: with 32 rows a wave the
      // maximum of some row moves in most tiles, and every move costs a multiplication per accumulator (a third of
      // the vector work).  Sums of terms up to 2^8 are as good in fp32, and the rounding of p is relative.
      if (__any((tmax - m_run) * cs > 8.f)) {
        const float m_new = fmaxf(m_run, tmax);
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run - m_new) * cs);
        l_run.scale(alpha);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) ot[dt] *= alpha;
        m_run = m_new;
      }
      const float m_use = m_run == -INFINITY ? 0.f : m_run * cs;
      auto step_p = [&](int u) {
        float pk[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) pk[e] = __builtin_amdgcn_exp2f(fmaf(s[u >> 1][8 * (u & 1) + e], cs, -m_use));
        Frag f = p_frag(pk, T{});
        if constexpr (sizeof(T) == 2) asm("" : "+v"(f));         // or its halves are converted once more for the row sums
        return f;
      };
      f32x16 sn[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) sn[t][e] = 0.f;
      Frag pf = step_p(0);
      // Where two waves share a vector unit (128 head dims), the one in its products goes first: it keeps the matrix unit fed and
      // its exponentials fall into the other's loads and maximum (1168 -> 1123 us).  With 64 head dims there are three and
      // less to multiply: 834 us so, 874 with the priority.
      if constexpr (DC > 64) __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        Frag pn = pf;
        if (u < 3) pn = step_p(u + 1);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const int x = u * NDT + dt;                        // product of the next tile's scores: tokens 32 (x / KS), k step x % KS
          const int y = x + RING;
          mma32(sn[x / KS], kf[x % RING], q[x % KS]);
          if (y < NX) kf[x % RING] = k_frag32<ROWB>(kl, y / KS, y % KS, T{});
          mma32(ot[dt], vf[x % RING], pf);
          if (y < NX) vf[x % RING] = v_frag32<ROWB>(vl, y % NDT, y / NDT, lane, T{});
        }
        l_run.add(pf);
        if constexpr (sizeof(T) == 2) {
          if (u < 3) {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x002, 16 / NDT, 0);
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
              __builtin_amdgcn_sched_group_barrier(0x002, 16 / NDT, 0);
            }
          }
        } else {
          __builtin_amdgcn_sched_barrier(0);                 // or the fragments of all steps are read at once, and spilled
        }
        pf = pn;
      }
      if constexpr (DC > 64) __builtin_amdgcn_s_setprio(0);
      s[0] = sn[0];
      s[1] = sn[1];
    }
    t0 = t1;
    t1 = t2;
  }

  float l;
  {
    float x, y;
    swap_halves32(l_run.of_lane(), x, y);
    l = x + y;
  }
  if (!live) return;
  const long long orow = (long long)(ti.c0 + ti.t0 + rt) * a.heads + kvh * group + rh;
  if (pieces == 1) {
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);       // NaN stays NaN
    T* o = reinterpret_cast<T*>(a.out) + orow * a.dim;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 32 * dt + 8 * e + 4 * h;
        if (d < a.dim) store4(o + d, f32x4{ot[dt][4 * e], ot[dt][4 * e + 1], ot[dt][4 * e + 2], ot[dt][4 * e + 3]} * inv);
      }
  } else {
    const long long at = ws_row(a, sp, ti, ti.t0 + rt, kvh * group + rh) * sp.pieces + split;
    float* o = a.ws + sp.ws + ws_sums(sp.ws_rows, sp.pieces) + at * a.dim;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 32 * dt + 8 * e + 4 * h;
        if (d < a.dim) store4(o + d, f32x4{ot[dt][4 * e], ot[dt][4 * e + 1], ot[dt][4 * e + 2], ot[dt][4 * e + 3]});
      }
    if (h == 0) reinterpret_cast<float2*>(a.ws + sp.ws)[at] = float2{m_run * cs, l};    // the join works in base-2 exponents
  }
}

// Workgroups of the short requests behind those of the long ones: they are bound by memory and fill what the last chunks
// leave idle (12 requests, a third of them single tokens, up to 512 rows and 16384 tokens: 558 us in two launches and 510 in one as this
// was built, 473 now).
template <typename T, int DP, int DC>
__global__ void __launch_bounds__(256, (ChunkTile<T, DP>::ROWB > 256 ? 1 : ChunkTile<T, DP>::ROWB > 128 ? 2 : 3))
    page_attn_chunk_kernel(const PageAttnArgs a, const Split sp, const Split step, const unsigned blocks) {
  static_assert(ChunkTile<T, DP>::BYTES >= StepTile<T, DP>::BYTES, "one size of LDS for both");
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const unsigned chunks = blocks * sp.pieces;
  if (__builtin_expect(blockIdx.x >= chunks, 0)) {
    step_tile<T, DP>(a, step, blockIdx.x - chunks, lds);
    return;
  }
  chunk_tile<T, DP, DC>(a, sp, blockIdx.x, blocks, lds);
}

// The output row of row `wrow` of a launch's workspace and how many pieces its results are in; 0: it is written already.
__device__ __forceinline__ int joined_pieces(const PageAttnArgs& a, const Split& sp, int wrow, int log, int& row) {
  TileInfo ti;
  if (sp.by_request) {
    ti.b = wrow / sp.per_request;
    row = wrow - ti.b * sp.per_request;
    ti.c0 = clamp_rows(a.cu_rows[ti.b], a.rows);
    ti.n = clamp_rows(a.cu_rows[ti.b + 1], a.rows) - ti.c0;
    if (row >= ti.n || ti.n > sp.per_request) return 0;
    row += ti.c0;
  } else {
    // the last request that starts at or before this row (B: behind all of them), 32 candidates at a time
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = a.B + 1;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) >> 5, b = lo + lane * step;
      const unsigned long long starts = __ballot(b < hi && a.cu_rows[b] <= wrow);
      const int k = __popc((unsigned)(starts >> (threadIdx.x & 32))) - 1;
      lo += (k > 0 ? k : 0) * step;
      hi = hi < lo + step ? hi : lo + step;
    }
    row = wrow;
    if (lo == a.B) return 0;
    ti.b = lo;
    ti.c0 = clamp_rows(a.cu_rows[lo], a.rows);
    ti.n = clamp_rows(a.cu_rows[lo + 1], a.rows) - ti.c0;
    if (row - ti.c0 >= ti.n || (sp.share != 0 && (ti.n <= sp.per_request) == (sp.share == 2))) return 0;
  }
  ti.t0 = (row - ti.c0) / sp.tt * sp.tt;
  const int cap = a.width << a.shift, kv = a.kv_lens[ti.b];
  ti.kv = kv < 0 ? 0 : (kv > cap ? cap : kv);
  const int n = pieces_of(sp, span_of(a, ti, sp.tt, log).count);
  return n > 1 ? n : 0;
}

// Joins few pieces: 32 threads per (row, head), four dims each.  (A workgroup per pair, as below, moved 1 TB/s of the
// partial results of 80 000 pairs x 3 pieces.)
constexpr int JOIN_FEW = 32;
template <typename T>
__global__ __launch_bounds__(256) void page_attn_join_few_kernel(const PageAttnArgs a, const Split chunk, const Split step, const unsigned chunks) {
  const bool of_chunk = blockIdx.x < chunks;
  const Split& sp = of_chunk ? chunk : step;
  const int log = of_chunk ? CHUNK_BLOCK : STEP_BLOCK;
  const long long slot = (long long)(of_chunk ? blockIdx.x : blockIdx.x - chunks) * 8 + (threadIdx.x >> 5);
  const bool there = slot < sp.ws_rows;
  const long long at = there ? slot : 0;                     // (all lanes of a wave take part in the search for the request)
  const int lane = threadIdx.x & 31, d = lane * 4;
  const int wrow = (int)(at / a.heads), head = (int)(at - (long long)wrow * a.heads);
  int row;
  const int pieces = joined_pieces(a, sp, wrow, log, row);
  if (!there || pieces == 0) return;
  float2 p{-INFINITY, 0.f};
  if (lane < pieces) p = reinterpret_cast<const float2*>(a.ws + sp.ws)[at * sp.pieces + lane];
  float m = p.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 32));
  const float f = p.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(p.x - m);     // a piece that saw nothing has no part
  float l = p.y * f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor(l, o, 32);
  const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
  const float* src = a.ws + sp.ws + ws_sums(sp.ws_rows, sp.pieces) + at * sp.pieces * a.dim + d;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < pieces; k0 += 4) {
    f32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (k0 + k < pieces && d < a.dim) v[k] = *reinterpret_cast<const f32x4*>(src + (long long)(k0 + k) * a.dim);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float w = __shfl(f, (k0 + k) & 31, 32);
      if (k0 + k < pieces) acc += v[k] * w;
    }
  }
  if (d < a.dim) store4(reinterpret_cast<T*>(a.out) + ((long long)row * a.heads + head) * a.dim + d, acc * inv);
}

// Joins many pieces: a workgroup per (row, head).  32 threads hold the dims, four each; the eight groups of 32 take every
// eighth piece, four loads in flight, and meet in LDS.
template <typename T>
__global__ __launch_bounds__(256) void page_attn_join_kernel(const PageAttnArgs a, const Split sp, const int log) {
  __shared__ float s_m[4], s_l[4];
  __shared__ float s_w[MAX_SPLITS];
  __shared__ f32x4 s_acc[8][32];
  const int at = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wrow = at / a.heads, head = at - wrow * a.heads;
  int row;
  const int pieces = joined_pieces(a, sp, wrow, log, row);
  if (pieces == 0) return;
  float2 p{-INFINITY, 0.f};                                  // MAX_SPLITS pieces: one per thread
  if (tid < pieces) p = reinterpret_cast<const float2*>(a.ws + sp.ws)[(long long)at * sp.pieces + tid];
  float m = p.x;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (lane == 0) s_m[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const float f = p.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(p.x - m);     // a piece that saw nothing has no part
  float l = p.y * f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  if (lane == 0) s_l[wave] = l;
  s_w[tid] = f;
  __syncthreads();
  l = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
  const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
  const int g = tid >> 5, d = (tid & 31) * 4;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (d < a.dim) {
    const float* src = a.ws + sp.ws + ws_sums(sp.ws_rows, sp.pieces) + (long long)at * sp.pieces * a.dim + d;
    for (int k0 = g; k0 < pieces; k0 += 32) {
      f32x4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (k0 + 8 * k < pieces) v[k] = *reinterpret_cast<const f32x4*>(src + (long long)(k0 + 8 * k) * a.dim);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k0 + 8 * k < pieces) acc += v[k] * s_w[k0 + 8 * k];
    }
  }
  s_acc[g][tid & 31] = acc;
  __syncthreads();
  if (g != 0 || d >= a.dim) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) acc += s_acc[k][tid & 31];
  store4(reinterpret_cast<T*>(a.out) + ((long long)row * a.heads + head) * a.dim + d, acc * inv);
}

// ---------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------
struct Plan {
  Split step, chunk;
  long long step_tiles = 0, chunk_tiles = 0;                 // 0: not launched
  long long ws = 0;                                          // floats
};

// Pieces of the key axis for a launch with `busy` workgroups per piece, by the longest request that the table can
// describe: enough to fill the chip with 512 workgroups (two per CU) as long as a piece has 256 tokens, and up to `most`, which
// the dispatcher can balance, as long as it has 2048.  Single tokens: 2 requests of up to 131072 tokens x 4 kv heads 76 us with
// 64 pieces, 87 with 256; 64 x 8192 x 8 258 us with 4, 265 with 2.  Chunks, in the example above: 473 us with 2560, 483 with 2048,
// 530 with 1280, 504 with 4096, 517 with 6144 (64 head dims: 269, 270, 319, 271, 276; in fp32, with 8 heads, with 24 requests or
// under a window all alike).  Below 768 tokens the join costs more than it saves (one token, 32 heads of 64 over 8 kv
// heads: 512 tokens 9.6 us cut, 7.8 whole; 1024 tokens 9.7 and 11.3).  Shorter requests have fewer pieces: chunks as many as
// keep each within the longest's, so that no workgroup ends much later than the others; single tokens, which wait for memory
// only, down to 512 tokens each (64 requests of 1 to 8192 tokens 238 us, 268 with the longest's, both with caches cold).
void divide(const PageAttnArgs& a, Split& s, long long busy, int most, int log) {
  long long longest = (long long)a.width << a.shift;
  const long long seen = (long long)a.window + a.sinks + CHUNK_ROWS;
  if (a.window > 0 && seen < longest) longest = seen;
  if (busy < 1) busy = 1;
  long long n = 512 / busy, m = most / busy;
  if (n > longest / 256) n = longest / 256;
  if (m > longest / 2048) m = longest / 2048;
  if (m > n) n = m;
  if (n > MAX_SPLITS) n = MAX_SPLITS;
  if (longest < 768) n = 1;
  s.pieces = n < 1 ? 1 : (int)n;
  s.piece = (int)((((longest + (1 << log) - 1) >> log) + s.pieces - 1) / s.pieces);
}

long long ws_floats(const PageAttnArgs& a, const Split& s) {
  return s.pieces > 1 ? ws_sums(s.ws_rows, s.pieces) + s.ws_rows * s.pieces * a.dim : 0;
}

Plan make_plan(const PageAttnArgs& a) {
  Plan p;
  const int group = a.heads / a.kv_heads;
  const int few = CHUNK_MIN / group;                                                          // rows of a short request
  const long long longest = a.max_rows > 0 && a.max_rows < a.rows ? a.max_rows : a.rows;      // rows of one request
  // without a hint a batch of as many rows as requests is taken for single tokens
  const bool chunks = longest > few && (a.max_rows > 0 || a.rows > a.B || few == 0);
  const long long some = a.rows < a.B ? a.rows : a.B;                                         // requests with rows, at most
  if (few > 0 || !chunks) {
    Split& s = p.step;
    s.gc = group < STEP_ROWS ? group : STEP_ROWS;
    s.hchunks = (group + s.gc - 1) / s.gc;
    s.tt = STEP_ROWS / s.gc;
    s.share = chunks ? 1 : 0;
    s.per_request = chunks ? few : 0;
    const long long full = chunks ? 0 : (a.rows + s.tt - 1) / s.tt;
    divide(a, s, (full > some ? full : some) * a.kv_heads * s.hchunks, 2048, STEP_BLOCK);
    s.piece = s.piece < 16 ? s.piece : 16;
    // a large table with a small step must not pay for the rows that its requests do not bring
    s.by_request = chunks && (long long)a.B * few < a.rows;
    p.step_tiles = s.by_request ? (long long)a.B * ((few + s.tt - 1) / s.tt) : (long long)a.rows / s.tt + some + 1;
    s.ws_rows = (s.by_request ? (long long)a.B * few : (long long)a.rows) * a.heads;
  }
  if (chunks) {
    Split& s = p.chunk;
    s.gc = group < CHUNK_ROWS ? group : CHUNK_ROWS;
    s.hchunks = (group + s.gc - 1) / s.gc;
    s.tt = CHUNK_ROWS / s.gc;
    s.share = 2;
    s.per_request = few;
    p.chunk_tiles = (long long)a.rows / s.tt + some + 1;
    divide(a, s, (long long)(a.rows + s.tt - 1) / s.tt * a.kv_heads * s.hchunks, 2560, CHUNK_BLOCK);
    s.ws_rows = (long long)a.rows * a.heads;
    s.ws = (ws_floats(a, p.step) + 3) & ~3ll;
  }
  p.ws = p.chunk.ws + ws_floats(a, p.chunk);
  if (p.chunk_tiles == 0) p.ws = ws_floats(a, p.step);
  return p;
}

int check_args(int dtype, const PageAttnArgs& a) {
  const int es = dtype == DT_BF16 ? 2 : 4;
  if (dtype != DT_BF16 && dtype != DT_F32) return fail("page_attention: dtype %d", dtype);
  if (a.B <= 0 || a.rows < 0 || a.kv_heads <= 0 || a.heads <= 0 || a.heads % a.kv_heads) return fail("page_attention: B=%d rows=%d, %d heads over %d kv heads", a.B, a.rows, a.heads, a.kv_heads);
  if (a.dim <= 0 || a.dim > 128 || a.dim % 8) return fail("page_attention: head dim %d unsupported (<= 128, multiple of 8)", a.dim);
  if (a.shift < 0) return fail("page_attention: the page size must be a power of two, 16 to 1024");
  if (a.n_pages <= 0 || a.width <= 0 || a.table_row < a.width) return fail("page_attention: %d pages, table of %d columns in rows of %lld", a.n_pages, a.width, a.table_row);
  if (((long long)a.width << a.shift) > 0x7fffffffll - 1024)       // positions a few tiles further on stay within 32 bits
     return fail("page_attention: a table of %d pages describes too many tokens", a.width);
  if (a.window < 0 || a.sinks < 0 || a.max_rows < 0) return fail("page_attention: window, sinks and max_rows must not be negative");
  if (!(a.scale > 0.f) || !isfinite(a.scale)) return fail("page_attention: the scale must be positive and finite");
  const long long strides[] = {a.q_row, a.q_head, a.k_page, a.k_head, a.k_slot, a.v_page, a.v_head, a.v_slot};
  for (long long s : strides)
    if (s % 16) return fail("page_attention: strides must be multiples of 16 bytes");
  if (a.k_slot < a.dim * es || a.v_slot < a.dim * es || a.k_slot > (1 << 24) || a.v_slot > (1 << 24)) return fail("page_attention: slots of %d / %d bytes for %d dims", a.k_slot, a.v_slot, a.dim);
  // page and slot offsets are formed in 32 bits, addresses in 64
  if (a.k_page < 0 || a.v_page < 0 || a.k_page > 0xffffffffll || a.v_page > 0xffffffffll) return fail("page_attention: page strides of %lld / %lld bytes (at most 2^32 - 1)", a.k_page, a.v_page);
  if (((long long)a.k_slot << a.shift) > 0x7fffffffll || ((long long)a.v_slot << a.shift) > 0x7fffffffll) return fail("page_attention: pages of more than 2 GiB");
  if ((long long)a.rows * a.heads > 0x7fffffffll || a.kv_heads > 65535) return fail("page_attention: too many rows or heads");
  return 0;
}

// few pieces of both launches' shares in one, many of either in one each
template <typename T>
void join(const PageAttnArgs& a, const Plan& p, hipStream_t stream) {
  const bool chunk = p.chunk_tiles > 0 && p.chunk.pieces > 1, step = p.step_tiles > 0 && p.step.pieces > 1;
  if (chunk && p.chunk.pieces > JOIN_FEW) page_attn_join_kernel<T><<<(unsigned)p.chunk.ws_rows, 256, 0, stream>>>(a, p.chunk, CHUNK_BLOCK);
  if (step && p.step.pieces > JOIN_FEW) page_attn_join_kernel<T><<<(unsigned)p.step.ws_rows, 256, 0, stream>>>(a, p.step, STEP_BLOCK);
  const unsigned chunks = chunk && p.chunk.pieces <= JOIN_FEW ? (unsigned)((p.chunk.ws_rows + 7) / 8) : 0;
  const unsigned steps = step && p.step.pieces <= JOIN_FEW ? (unsigned)((p.step.ws_rows + 7) / 8) : 0;
  if (chunks + steps > 0) page_attn_join_few_kernel<T><<<chunks + steps, 256, 0, stream>>>(a, p.chunk, p.step, chunks);
}

template <typename T, int DP, int DC>
int run(const PageAttnArgs& a, const Plan& p, hipStream_t stream) {
  using ST = StepTile<T, DP>;
  using CT = ChunkTile<T, DP>;
  auto sk = page_attn_step_kernel<T, DP>;
  auto ck = page_attn_chunk_kernel<T, DP, DC>;
  const long long chunk_blocks = p.chunk_tiles * a.kv_heads * p.chunk.hchunks;
  const long long step_grid = p.step_tiles * a.kv_heads * p.step.hchunks * p.step.pieces;
  if (chunk_blocks * p.chunk.pieces + step_grid > 0x7fffffffll) return fail("page_attention: too many rows or heads");
  if (p.chunk_tiles > 0) {
    if (reserve_lds(reinterpret_cast<const void*>(ck), CT::BYTES) != hipSuccess) return fail("page_attention: cannot reserve %d bytes of LDS", CT::BYTES);
    ck<<<(unsigned)(chunk_blocks * p.chunk.pieces + step_grid), 256, CT::BYTES, stream>>>(a, p.chunk, p.step, (unsigned)chunk_blocks);
  } else {
    if (reserve_lds(reinterpret_cast<const void*>(sk), ST::BYTES) != hipSuccess) return fail("page_attention: cannot reserve %d bytes of LDS", ST::BYTES);
    sk<<<(unsigned)step_grid, 64 * STEP_WAVES, ST::BYTES, stream>>>(a, p.step);
  }
  join<T>(a, p, stream);
  return check_launch("page_attention");
}

template <typename T>
int run(const PageAttnArgs& a, const Plan& p, hipStream_t stream) {
  return a.dim <= 64 ? run<T, 64, 64>(a, p, stream) : a.dim <= 96 ? run<T, 128, 96>(a, p, stream) : run<T, 128, 128>(a, p, stream);
}

}  // namespace

size_t page_attention_workspace_bytes(int dtype, const PageAttnArgs& a) {
  if (check_args(dtype, a) != 0) return 0;
  return (size_t)make_plan(a).ws * sizeof(float);
}

int launch_page_attention(int dtype, const PageAttnArgs& a, size_t ws_bytes, hipStream_t stream) {
  if (check_args(dtype, a) != 0) return -1;
  if (a.rows == 0) return 0;
  if (!a.q || !a.k || !a.v || !a.table || !a.kv_lens || !a.cu_rows || !a.out) return fail("page_attention: null operand");
  if ((uintptr_t)a.q % 16 || (uintptr_t)a.k % 16 || (uintptr_t)a.v % 16 || (uintptr_t)a.out % 16) return fail("page_attention: operands must be 16-byte aligned");
  const Plan p = make_plan(a);
  const size_t need = (size_t)p.ws * sizeof(float);
  if (need > 0 && (!a.ws || ws_bytes < need || (uintptr_t)a.ws % 16)) return fail("page_attention: workspace of %zu bytes, %zu needed", ws_bytes, need);
  return dtype == DT_BF16 ? run<bf16>(a, p, stream) : run<float>(a, p, stream);
}

}  // namespace fcenc
