// Pages of a key/value cache: the plan of a step (page table, slots, lengths, free list) and the write of its rows.
//
// The cache is a pool of pages of `page_size` slots (a power of two).  A request of length n holds ceil(n / page_size)
// pages, listed in order in its row of the block table; pages that nobody holds lie on a stack (`free_pages`, height
// `free_count`).  One step of a batch:
//
//   1. rows that finished push their pages in row order and become empty;
//   2. row b wants need_b = ceil((kv_b + new_b) / page_size) - ceil(kv_b / page_size) pages.  It is granted if its
//      tokens fit the table's width and the rows of the step, and need_b = 0 or sum_{j <= b} need_j <= height (the sum
//      runs over every row that fits, so that a row is never overtaken by a later one);
//   3. the i-th page handed out, in row order, is free_pages[height - 1 - i];
//   4. slot of row cu_rows[b] + i = table[b][(kv_b + i) / page_size] * page_size + (kv_b + i) % page_size, -1 if refused.
//
// All of it is integer arithmetic on prefix sums, so results do not depend on the order of execution.
#include "common.h"
#include "kernels.h"

namespace fcenc {

namespace {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_WAVES = PLAN_THREADS / 64;
// Steps with up to this many rows (and PLAN_THREADS requests) find their slots in the planning workgroup itself, out of
// LDS; longer ones leave them to a second launch over all CUs.
constexpr int PLAN_INLINE_ROWS = 4 * PLAN_THREADS;

__device__ __forceinline__ long long wave_scan(long long v, int lane) {      // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// inclusive prefix sum of one value per thread; `total` receives the sum.  `part` holds a value per wave.
__device__ __forceinline__ long long block_scan(long long v, long long* part, int waves, long long& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long incl = wave_scan(v, lane);
  if (waves == 1) {
    total = __shfl(incl, 63);
    return incl;
  }
  __syncthreads();                       // the last use of `part` is over
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  long long base = 0;
  total = 0;
  for (int w = 0; w < waves; ++w) {
    if (w < wave) base += part[w];
    total += part[w];
  }
  return base + incl;
}

__device__ __forceinline__ int pages_of(int tokens, int shift) { return (int)(((long long)tokens + (1 << shift) - 1) >> shift); }

__device__ __forceinline__ long long slot_of(const int32_t* row, int pos, int shift) {
  return ((long long)row[pos >> shift] << shift) + (pos & ((1 << shift) - 1));
}

constexpr int OWN_PAGES = 2;

// n ids from `src` (going up or, with STEP -1, down) to `dst`, by one wave
template <int STEP>
__device__ __forceinline__ void move_pages(const int32_t* src, int32_t* dst, int n, int lane) {
  for (int c0 = lane; c0 < n; c0 += 256) {
    int32_t v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = c0 + 64 * k < n ? src[STEP * (c0 + 64 * k)] : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c0 + 64 * k < n) dst[c0 + 64 * k] = v[k];
  }
}

// the last of `n` rising starts that is at or before i (starts[0] = 0); its row is not empty if i lies before the end
__device__ __forceinline__ int last_at(const int* starts, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

// One workgroup: a plan is a chain of prefix sums over a few hundred requests, bound by latency, and one workgroup
// needs no hand-over between CUs.  With one wave no scan waits at a barrier.  A thread moves up to OWN_PAGES pages of its
// request by itself; longer ones are listed and taken by a wave each, four pages a lane in flight.  (One page per thread,
// its request found by bisection of the prefix sums, took 18 us for 256 requests with 13 000 pages to move, this 12.)
__global__ __launch_bounds__(PLAN_THREADS) void page_plan_kernel(const PagePlanArgs a, int inline_slots) {
  __shared__ long long part[PLAN_WAVES];
  __shared__ int s_kv[PLAN_THREADS];                 // length before the step (0 for rows that finished), -1 if refused
  __shared__ int s_cu[PLAN_THREADS + 1];
  __shared__ int s_take[PLAN_THREADS];               // where a listed row's pages begin: in the stack,
  __shared__ int s_held[PLAN_THREADS];               // in its table row,
  __shared__ int s_move[PLAN_THREADS];               // and how many there are
  __shared__ int s_list[PLAN_THREADS];
  __shared__ int s_listed;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, threads = blockDim.x, waves = threads >> 6;
  const int cap = a.width << a.shift;                // the longest request the table can describe
  int top = *a.free_count;
  top = top < 0 ? 0 : (top > a.pool ? a.pool : top);

  // ---- 1. rows that finished ----
  if (a.finished) {
    for (int b0 = 0; b0 < a.B; b0 += threads) {
      const int b = b0 + tid;
      int count = 0;
      if (b < a.B && a.finished[b]) {
        int kv = a.kv_lens[b];
        kv = kv < 0 ? 0 : (kv > cap ? cap : kv);
        count = pages_of(kv, a.shift);
      }
      long long total;
      const long long before = block_scan(count, part, waves, total) - count;
      const int room = a.pool - top;
      const int pushed = total < room ? (int)total : room;      // a pool never gets back more pages than it has
      if (tid == 0) s_listed = 0;
      __syncthreads();
      if (count > 0 && before < pushed) {
        s_take[tid] = top + (int)before;
        s_move[tid] = count < pushed - (int)before ? count : pushed - (int)before;
        s_list[atomicAdd(&s_listed, 1)] = tid;
      }
      __syncthreads();
      for (int q = wave; q < s_listed; q += waves) {
        const int k = s_list[q];
        move_pages<1>(a.table + (size_t)(b0 + k) * a.table_row, a.free_pages + s_take[k], s_move[k], lane);
      }
      top += pushed;
      __syncthreads();
    }
    __threadfence_block();
    __syncthreads();                                 // pages pushed are visible to the pops below
  }

  // ---- 2. - 3. lengths, grants, pages ----
  long long rows_before = 0, asked_before = 0, taken_before = 0;
  for (int b0 = 0; b0 < a.B; b0 += threads) {
    const int b = b0 + tid;
    int kv = 0, n = 0;
    if (b < a.B) {
      kv = a.kv_lens[b];
      kv = kv < 0 || (a.finished && a.finished[b]) ? 0 : kv;
      n = a.new_lens[b];
      n = n < 0 ? 0 : n;
    }
    long long total;
    const long long rows_end = rows_before + block_scan(n, part, waves, total);
    rows_before += total;
    const bool fits = b < a.B && (long long)kv + n <= cap && rows_end <= a.rows;
    const int held = pages_of(kv, a.shift);
    int need = fits ? pages_of(kv + n, a.shift) - held : 0;
    const long long asked = asked_before + block_scan(need, part, waves, total);
    asked_before += total;
    const bool granted = fits && (need == 0 || asked <= top);
    need = granted ? need : 0;
    const long long taken = taken_before + block_scan(need, part, waves, total);
    taken_before += total;
    const long long cu = rows_end - n;
    s_kv[tid] = granted ? kv : -1;
    s_cu[tid] = cu > 0x7fffffff ? 0x7fffffff : (int)cu;
    if (b < a.B) {
      a.cu_rows[b] = s_cu[tid];
      a.granted[b] = granted;
      a.kv_lens[b] = granted ? kv + n : kv;
    }
    if (b == a.B - 1) {
      const int end = rows_end > 0x7fffffff ? 0x7fffffff : (int)rows_end;
      s_cu[tid + 1] = end;
      a.cu_rows[a.B] = end;
    }
    const int from = top - 1 - (int)(taken - need);  // of the stack, downwards
    if (tid == 0) s_listed = 0;
    __syncthreads();
    if (need > OWN_PAGES) {
      s_take[tid] = from;
      s_held[tid] = held;
      s_move[tid] = need;
      s_list[atomicAdd(&s_listed, 1)] = tid;
    } else if (need > 0) {
      int32_t* row = a.table + (size_t)b * a.table_row + held;
#pragma unroll
      for (int c = 0; c < OWN_PAGES; ++c)
        if (c < need) row[c] = a.free_pages[from - c];
    }
    __syncthreads();
    for (int q = wave; q < s_listed; q += waves) {
      const int k = s_list[q];
      move_pages<-1>(a.free_pages + s_take[k], a.table + (size_t)(b0 + k) * a.table_row + s_held[k], s_move[k], lane);
    }
    if (b0 + threads < a.B) __syncthreads();
  }
  if (tid == 0) *a.free_count = top - (int)taken_before;

  // ---- 4. slots of a short step (one trip of the loop above: the LDS arrays describe every request) ----
  if (!inline_slots) return;
  __threadfence_block();
  __syncthreads();
  for (int i = tid; i < a.rows; i += threads) {
    long long slot = -1;
    if (i < s_cu[a.B]) {
      const int lo = last_at(s_cu, a.B, i);
      if (s_kv[lo] >= 0) slot = slot_of(a.table + (size_t)lo * a.table_row, s_kv[lo] + i - s_cu[lo], a.shift);
    }
    a.slots[i] = slot;
  }
}

// slots of a long step: one row per thread, its request by bisection of cu_rows
__global__ __launch_bounds__(256) void page_slots_kernel(const PagePlanArgs a) {
  const unsigned at = blockIdx.x * 256u + threadIdx.x;
  if (at >= (unsigned)a.rows) return;
  const int i = (int)at;
  long long slot = -1;
  if (i < a.cu_rows[a.B]) {
    const int lo = last_at(a.cu_rows, a.B, i);
    if (a.granted[lo]) {
      const int pos = a.kv_lens[lo] - (a.cu_rows[lo + 1] - i);        // kv_lens already counts the step's rows
      slot = slot_of(a.table + (size_t)lo * a.table_row, pos, a.shift);
    }
  }
  a.slots[i] = slot;
}

// New K and V rows to their slots, 16 bytes per thread and tensor.  Bound by memory: every byte is read and written
// once, and a head's row of a page is contiguous.  16411 rows of 8 heads of 128 bf16 values: 21 us, 6.3 TB/s.
__global__ __launch_bounds__(256) void page_write_kernel(const PageWriteArgs a, uint32_t chunks_per_row, uint32_t chunks_per_head) {
  const size_t step = (size_t)gridDim.x * 256;
  const size_t count = (size_t)a.rows * chunks_per_row;
  for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < count; e += step) {
    const uint32_t row = (uint32_t)(e / chunks_per_row), c = (uint32_t)(e - (size_t)row * chunks_per_row);
    const long long slot = a.slots[row];
    if (slot < 0 || (slot >> a.shift) >= a.n_pages) continue;
    const uint32_t h = c / chunks_per_head, o = (c - h * chunks_per_head) * 16;
    const long long page = slot >> a.shift, off = slot & ((1 << a.shift) - 1);
    *reinterpret_cast<u32x4*>(a.k_pages + page * a.k_page + h * a.k_phead + off * a.k_slot + o) =
        *reinterpret_cast<const u32x4*>(a.k + row * a.k_row + h * a.k_head + o);
    *reinterpret_cast<u32x4*>(a.v_pages + page * a.v_page + h * a.v_phead + off * a.v_slot + o) =
        *reinterpret_cast<const u32x4*>(a.v + row * a.v_row + h * a.v_head + o);
  }
}

}  // namespace

int page_shift(int page_size) {
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return -1;
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

int launch_page_plan(const PagePlanArgs& a, hipStream_t stream) {
  if (a.B <= 0 || a.width <= 0 || a.pool <= 0 || a.rows < 0) return fail("page_plan: empty batch, table or pool (B=%d width=%d pool=%d rows=%d)", a.B, a.width, a.pool, a.rows);
  if (a.shift < 0) return fail("page_plan: the page size must be a power of two, 16 to 1024");
  if (a.table_row < a.width) return fail("page_plan: table rows overlap (%lld < %d)", a.table_row, a.width);
  if (((long long)a.width << a.shift) > 0x7fffffffll) return fail("page_plan: a table of %d pages describes more than 2^31 - 1 tokens", a.width);
  if (!a.kv_lens || !a.new_lens || !a.table || !a.free_pages || !a.free_count || !a.cu_rows || !a.granted || (a.rows > 0 && !a.slots)) return fail("page_plan: null operand");
  const bool inl = a.B <= PLAN_THREADS && a.rows <= PLAN_INLINE_ROWS;
  // a thread per request, or per row of a short step; all of them where whole prompts or whole requests' pages may move
  int threads = a.B > a.rows ? a.B : a.rows;
  threads = !inl || a.finished || threads > PLAN_THREADS ? PLAN_THREADS : (threads + 63) / 64 * 64;
  page_plan_kernel<<<1, threads, 0, stream>>>(a, inl ? 1 : 0);
  if (!inl && a.rows > 0) page_slots_kernel<<<(a.rows - 1) / 256 + 1, 256, 0, stream>>>(a);
  return check_launch("page_plan");
}

int launch_page_write(const PageWriteArgs& a, hipStream_t stream) {
  if (a.rows < 0 || a.heads <= 0 || a.head_bytes <= 0 || a.head_bytes % 16) return fail("page_write: rows %d, heads %d, %d bytes a head (a multiple of 16)", a.rows, a.heads, a.head_bytes);
  if (a.shift < 0) return fail("page_write: the page size must be a power of two, 16 to 1024");
  if (a.n_pages <= 0) return fail("page_write: no pages");
  if (a.rows == 0) return 0;
  if (!a.k || !a.v || !a.k_pages || !a.v_pages || !a.slots) return fail("page_write: null operand");
  const long long strides[] = {a.k_row, a.k_head, a.v_row, a.v_head, a.k_page, a.k_phead, a.k_slot, a.v_page, a.v_phead, a.v_slot};
  for (long long s : strides)
    if (s % 16) return fail("page_write: strides must be multiples of 16 bytes");
  if ((uintptr_t)a.k % 16 || (uintptr_t)a.v % 16 || (uintptr_t)a.k_pages % 16 || (uintptr_t)a.v_pages % 16) return fail("page_write: operands must be 16-byte aligned");
  const uint32_t cph = (uint32_t)a.head_bytes / 16, cpr = cph * (uint32_t)a.heads;
  const size_t blocks = ((size_t)a.rows * cpr + 255) / 256;
  page_write_kernel<<<(unsigned)(blocks < 16384 ? blocks : 16384), 256, 0, stream>>>(a, cpr, cph);
  return check_launch("page_write");
}

}  // namespace fcenc
